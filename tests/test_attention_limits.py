"""Calls past what one launch takes (2^32 threads) are refused before it."""

from __future__ import annotations

import pytest

from flatrun_amd import _lib, device
from test_attention import decode, prefill


class Cache:
    """A large cache's shape without its memory."""
    page_tokens, head_dim = 32, 64

    def __init__(self, pages, kv_heads):
        self.pages, self.kv_heads = pages, kv_heads
        self.nbytes = pages * kv_heads * 32 * 2 * 64 * 9 // 16      # no call while tests are collected: torch loads first

    def data_ptr(self):
        return 0x10000


@pytest.mark.parametrize("call,kw", [
    (prefill, dict(seqs=1 << 16, tokens_q=1 << 20, tokens_k=1 << 20, max_q=1 << 14, max_k=1 << 14, q_heads=32, kv_heads=8)),
    (prefill, dict(seqs=1 << 20, tokens_q=1 << 21, tokens_k=1 << 21, max_q=1, max_k=1, q_heads=64, kv_heads=64)),
    (prefill, dict(seqs=1, tokens_q=(1 << 31) - 257, max_q=(1 << 31) - 257, max_k=1, tokens_k=8, q_heads=64, kv_heads=1)),
    (decode, dict(cache=Cache(1 << 20, 16), batch=1 << 20, q_heads=16, max_len=30)),
    (decode, dict(cache=Cache(1 << 20, 1), batch=1 << 18, q_heads=64, max_len=4000, ld_table=200)),
])
def test_more_than_a_launch(call, kw):
    with pytest.raises(_lib.FrqError) as ei:
        call(**kw)
    assert ei.value.code == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("move", [device.kv4_write, device.kv4_read])
@pytest.mark.parametrize("tokens,kv_heads", [(1 << 29, 1), (1 << 25, 16), (1 << 24, 32)])
def test_more_heads_than_a_launch(move, tokens, kv_heads):
    with pytest.raises(_lib.FrqError) as ei:
        move(Cache(1 << 20, kv_heads), 0x10000, 0x20000, 0x30000, tokens)
    assert ei.value.code == _lib.ERR_UNSUPPORTED
