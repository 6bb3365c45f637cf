"""add_rms_norm, attn_chunk and sample without a GPU: refusals, and calls with
nothing to do."""

from __future__ import annotations

import pytest
import torch

from flatrun_amd import _lib, device
from test_attention import FakeCache


def norm(**kw):
    a = dict(x=0x10000, out=0x20000, rows=3, hidden=256, weight=0x30000, residual=0x40000, sum_out=0x50000)
    a.update(kw)
    device.add_rms_norm(**a)


def chunk(cache=None, **kw):
    a = dict(q=0x10000, cache=cache or FakeCache(), table=0x20000, lens=0x30000, cu_q=0x40000, out=0x50000, seqs=2,
             tokens_q=9, q_heads=4, max_q=8, max_len=100)
    a.update(kw)
    device.attn_chunk(**a)


def sample(**kw):
    a = dict(logits=0x10000, u=0x20000, tokens=0x30000, rows=3, vocab=1000, probs=0x40000)
    a.update(kw)
    device.sample(**a)


REFUSED = [
    (norm, dict(x_dtype=8), _lib.ERR_INVALID),
    (norm, dict(res_dtype=2), _lib.ERR_INVALID),
    (norm, dict(out_dtype=2), _lib.ERR_INVALID),
    (norm, dict(x=0), _lib.ERR_INVALID),
    (norm, dict(out=0), _lib.ERR_INVALID),
    (norm, dict(eps=-1e-6), _lib.ERR_INVALID),
    (norm, dict(eps=float("nan")), _lib.ERR_INVALID),
    (norm, dict(eps=float("inf")), _lib.ERR_INVALID),
    (norm, dict(residual=None), _lib.ERR_INVALID),
    (norm, dict(sum_out=0x20000), _lib.ERR_INVALID),
    (norm, dict(rows=-1), _lib.ERR_SHAPE),
    (norm, dict(hidden=0), _lib.ERR_SHAPE),
    (norm, dict(hidden=(1 << 24) + 8), _lib.ERR_SHAPE),
    (norm, dict(ld_x=255), _lib.ERR_SHAPE),
    (norm, dict(ld_res=255), _lib.ERR_SHAPE),
    (norm, dict(ld_sum=255), _lib.ERR_SHAPE),
    (norm, dict(ld_out=255), _lib.ERR_SHAPE),
    (norm, dict(hidden=250, out_dtype="q8_0"), _lib.ERR_SHAPE),
    (norm, dict(ld_out=260, out_dtype="q8_0"), _lib.ERR_SHAPE),
    (norm, dict(x=0x10002), _lib.ERR_ALIGN),
    (norm, dict(x=0x10001, x_dtype="bf16"), _lib.ERR_ALIGN),
    (norm, dict(residual=0x40002), _lib.ERR_ALIGN),
    (norm, dict(sum_out=0x50001, res_dtype="f16"), _lib.ERR_ALIGN),
    (norm, dict(weight=0x30002), _lib.ERR_ALIGN),
    (norm, dict(out=0x20001, out_dtype="q8_0"), _lib.ERR_ALIGN),
    (chunk, dict(dtype="f32"), _lib.ERR_INVALID),
    (chunk, dict(out_dtype="f16"), _lib.ERR_INVALID),
    (chunk, dict(scale=0.0), _lib.ERR_INVALID),
    (chunk, dict(q=0), _lib.ERR_INVALID),
    (chunk, dict(table=0), _lib.ERR_INVALID),
    (chunk, dict(lens=0), _lib.ERR_INVALID),
    (chunk, dict(cu_q=0), _lib.ERR_INVALID),
    (chunk, dict(q_heads=5), _lib.ERR_SHAPE),
    (chunk, dict(max_q=10), _lib.ERR_SHAPE),
    (chunk, dict(seqs=-1), _lib.ERR_SHAPE),
    (chunk, dict(ld_table=1), _lib.ERR_SHAPE),
    (chunk, dict(ld_q=500), _lib.ERR_SHAPE),
    (chunk, dict(ld_out=511), _lib.ERR_SHAPE),
    (chunk, dict(max_len=-1), _lib.ERR_UNSUPPORTED),
    (chunk, dict(max_len=(1 << 29) + 1, ld_table=1 << 24), _lib.ERR_UNSUPPORTED),
    (chunk, dict(seqs=1 << 20, tokens_q=1 << 20, max_q=256), _lib.ERR_UNSUPPORTED),
    (chunk, dict(out=0x50008), _lib.ERR_ALIGN),
    (chunk, dict(ld_q=516), _lib.ERR_ALIGN),
    (chunk, dict(cu_q=0x40002), _lib.ERR_ALIGN),
    (sample, dict(dtype=2), _lib.ERR_INVALID),
    (sample, dict(temperature=-0.5), _lib.ERR_INVALID),
    (sample, dict(temperature=float("inf")), _lib.ERR_INVALID),
    (sample, dict(top_k=-1), _lib.ERR_INVALID),
    (sample, dict(top_p=1.5), _lib.ERR_INVALID),
    (sample, dict(min_p=float("nan")), _lib.ERR_INVALID),
    (sample, dict(u=0), _lib.ERR_INVALID),
    (sample, dict(tokens=0), _lib.ERR_INVALID),
    (sample, dict(rows=-1), _lib.ERR_SHAPE),
    (sample, dict(ld=999), _lib.ERR_SHAPE),
    (sample, dict(vocab=0), _lib.ERR_UNSUPPORTED),
    (sample, dict(vocab=(1 << 20) + 1), _lib.ERR_UNSUPPORTED),
    (sample, dict(logits=0x10002), _lib.ERR_ALIGN),
]


@pytest.mark.parametrize("call,kw,code", REFUSED, ids=[f"{c[0].__name__}-{i}" for i, c in enumerate(REFUSED)])
def test_refusals(call, kw, code):
    with pytest.raises(_lib.FrqError) as ei:
        call(**kw)
    assert ei.value.code == code


def test_a_cache_that_is_too_small():
    bad = FakeCache()
    bad.nbytes -= 1
    with pytest.raises(_lib.FrqError) as ei:
        chunk(bad)
    assert ei.value.code == _lib.ERR_SIZE


def test_nothing_to_do_needs_no_buffers():
    norm(rows=0, x=0, out=0, weight=None, residual=None, sum_out=None)
    chunk(seqs=0, q=0, out=0, lens=0, cu_q=0, table=0)
    chunk(tokens_q=0, max_q=0, q=0, out=0)
    sample(rows=0, logits=0, u=0, tokens=0, probs=None)


@pytest.mark.parametrize("call,kw,error", [
    (norm, dict(x=torch.zeros(3 * 256).half()), TypeError),
    (norm, dict(x=torch.zeros(3 * 256 - 1)), ValueError),
    (norm, dict(weight=torch.zeros(255)), ValueError),
    (norm, dict(out=torch.zeros((3, 8, 34), dtype=torch.uint8)), TypeError),
    (norm, dict(out=torch.zeros((3, 8, 33), dtype=torch.uint8), out_dtype="q8_0"), ValueError),
    (norm, dict(out=torch.zeros((3, 256)), out_dtype="q8_0"), TypeError),
    (norm, dict(out_dtype="q4_0"), ValueError),
    (norm, dict(x=torch.zeros((3, 256))), ValueError),                                # host memory
    (norm, dict(residual=torch.zeros((3, 512))[:, :256]), ValueError),                # strides
    (chunk, dict(q=torch.zeros((9, 4, 128))), TypeError),
    (chunk, dict(lens=torch.zeros(2, dtype=torch.int64)), TypeError),
    (chunk, dict(cu_q=torch.zeros(2, dtype=torch.int32)), ValueError),
    (chunk, dict(q=torch.zeros((9, 8, 128), dtype=torch.bfloat16)[:, ::2]), ValueError),
    (sample, dict(logits=torch.zeros((3, 1000)).half()), TypeError),
    (sample, dict(logits=torch.zeros((3, 1024))[:, :1000]), ValueError),
    (sample, dict(tokens=torch.zeros(3, dtype=torch.int64)), TypeError),
    (sample, dict(top_k=torch.zeros(3)), TypeError),
    (sample, dict(min_p=torch.zeros(2)), ValueError),
    (sample, dict(u=torch.zeros(3)), ValueError),                                     # host memory
    (sample, dict(dtype="q8"), ValueError),
])
def test_wrong_tensors_are_refused(call, kw, error):
    with pytest.raises(error):
        call(**kw)
