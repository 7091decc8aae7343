"""A decoder layer's attention over the paged 4-bit KV cache: prompts in, then tokens one at a time.

int8 q/k/v and output linears (``qrow``), one plan a step (``paging``), rotary positions and the
4-bit cache (``rotary``, ``kv4``).  Run from the repository's root on an MI355X:

    python3 examples/attention_step.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import __graft_entry__  # noqa: E402

__graft_entry__.load_package()

from mrun_pub_amd import codecs, kv4, paging, qrow, rotary  # noqa: E402

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, PAGE = 1536, 12, 2, 128, 16


class AttentionLayer:
    """Fused q/k/v linear, attention over the cache's layer ``index``, output linear."""

    def __init__(self, index: int, device, seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed + index)
        rows = (HEADS + 2 * KV_HEADS) * HEAD_DIM
        self.index = index
        self.qkv = codecs.quant_row_int8(torch.randn(rows, HIDDEN, device=device, generator=g) / HIDDEN**0.5)
        self.out = codecs.quant_row_int8(torch.randn(HIDDEN, HEADS * HEAD_DIM, device=device, generator=g) / HIDDEN**0.5)

    def __call__(self, x, cache, tables, plan, spec, max_query, max_context):
        qkv = qrow.qrow_matmul(*self.qkv, x).view(-1, HEADS + 2 * KV_HEADS, HEAD_DIM)
        q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
        q = kv4.append(cache, self.index, k, v, plan.slots, q=q, positions=plan.positions, rotary=spec)
        o = kv4.attend(q, cache, self.index, tables, plan.query_starts, plan.context_lens, max_query=max_query,
                       max_context=max_context)
        return qrow.qrow_matmul(*self.out, o.view(-1, HEADS * HEAD_DIM))


class Requests:
    """Block tables, lengths and the page pool of a batch."""

    def __init__(self, prompts: list[int], most: int, device):
        self.device, self.lens = device, torch.zeros(len(prompts), dtype=torch.int32, device=device)
        columns = -(-most // PAGE)
        self.tables = torch.full((len(prompts), columns), -1, dtype=torch.int32, device=device)
        self.pages = len(prompts) * columns
        self.ring, self.pool = paging.free_pages(self.pages, device)

    def plan(self, new: torch.Tensor, tokens: int) -> paging.StepPlan:
        plan = paging.plan_step(self.ring, self.pool, self.tables, self.lens, new, page_size=PAGE, tokens=tokens)
        self.pool, self.lens = plan.free_state, plan.context_lens
        return plan

    def finish(self) -> None:
        done = torch.ones(self.lens.numel(), dtype=torch.bool, device=self.device)
        self.pool = paging.release_pages(self.ring, self.pool, self.tables, self.lens, done, page_size=PAGE)


def run(prompts: list[int], steps: int, layers: int = 2, device="cuda:0"):
    """Outputs of the prompts' step and of every decode step, and the requests afterwards."""
    device = torch.device(device)
    g = torch.Generator(device=device).manual_seed(1)
    most = max(prompts) + steps
    batch = Requests(prompts, most, device)
    cache = kv4.KV4Cache(layers=layers, kv_heads=KV_HEADS, head_dim=HEAD_DIM, pages=batch.pages, page_size=PAGE, device=device)
    spec = rotary.RotarySpec(HEAD_DIM, base=1e6)
    stack = [AttentionLayer(i, device) for i in range(layers)]
    outputs = []
    for step in range(steps + 1):
        lens = prompts if step == 0 else [1] * len(prompts)
        x = torch.randn(sum(lens), HIDDEN, device=device, generator=g).to(torch.bfloat16)
        plan = batch.plan(torch.tensor(lens, dtype=torch.int32, device=device), sum(lens))
        for layer in stack:
            x = x + layer(x, cache, batch.tables, plan, spec, max(lens), max(prompts) + step)
        outputs.append(x)
    return outputs, batch, cache


def main() -> None:
    outputs, batch, cache = run([513, 40, 7], steps=8)
    print(f"prompts: {list(outputs[0].shape)}, then {len(outputs) - 1} steps of {list(outputs[1].shape)}")
    print(f"lengths {batch.lens.tolist()}, {cache.nbytes >> 10} KiB of cache, pool {batch.pool.tolist()}")
    batch.finish()
    print(f"pages back: pool {batch.pool.tolist()}")


if __name__ == "__main__":
    main()
