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
