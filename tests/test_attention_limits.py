"""Limits of the operators around the 4-bit KV cache that the host refuses before any launch."""

from __future__ import annotations

import pytest
import torch

from mrun_pub_amd import rotary

FAKE = 1 << 20  # an aligned pointer that is never read: the checks come first


def _lib():
    import mrun_pub_amd._native as nat

    if not nat.LIB_PATH.exists():
        pytest.skip("library not built")
    return nat, nat.load()


@pytest.mark.parametrize("tokens,heads,kv_heads,dtype", [(1 << 26, 12, 2, 1), (1 << 25, 32, 8, 0), (1 << 30, 1, 1, 2)])
def test_attention_of_more_threads_than_a_grid_has(tokens, heads, kv_heads, dtype):
    nat, lib = _lib()
    a = [FAKE, dtype, heads * 128, 128, FAKE, 9, 16, kv_heads, heads, 128, FAKE, 4, 4, FAKE, FAKE, 2, tokens, 1, 60, 0.1, 0, FAKE,
         None, 0, None]
    assert lib.qs_kv4_attend(*a) == nat.QS_ERR_LIMIT
    assert b"threads" in lib.qs_last_error()


def test_rotary_frequencies_are_not_laid_out_in_a_capture(monkeypatch):
    """The copy and the wait of the first use would end a graph's capture with an error of their own."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        rotary.RotarySpec(64).on(torch.device("cuda:0"))


@pytest.mark.parametrize("tokens,requests,kv_heads,heads,d,new,context", [
    (4095, 1, 8, 32, 128, 4095, 4095), (8000, 1, 8, 32, 128, 8000, 8000), (2048, 4, 8, 32, 128, 512, 30000),
    (4095, 1, 8, 32, 256, 4095, 4095), (64, 64, 8, 32, 128, 1, 131072), (320, 64, 8, 32, 256, 5, 131072), (1, 1, 2, 12, 128, 1, 131072),
])
def test_attention_workspace_holds_cut_tiles_alone(tokens, requests, kv_heads, heads, d, new, context):
    """A place a block that runs at once, 512 of 128 rows or 1024 of 16, each its rows' sums, maxima and
    totals in fp32: whatever the number of tiles.  (Two tiles of 16 rows a block: half as many run.)"""
    _nat, lib = _lib()
    size = lib.qs_kv4_attend_workspace_bytes(tokens, requests, kv_heads, heads, d, 64, new, context, 0)
    rows = 512 * 128 if new * heads // kv_heads > 32 else 1024 * 16
    assert 0 < size <= 4 * (8192 + rows * (d + 2))
