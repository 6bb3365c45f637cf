"""qk_norm_rope against the 64-bit form.

fp32 bound: the norm's factor carries at most 12 roundings (a sum of d squares
in 8 steps a lane and a tree, the mean, root, reciprocal), each product and
the pair's two products and sum one each: 20 * 2^-24 of |a| + |b| after the
norm. A 16-bit output adds half its last place (fp16: 2^-25 below its normal
range)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import HALF_ULP, TORCH, dev, f64, rope
from flatrun_amd import device
from flatrun_amd.attention import rope_table

pytestmark = pytest.mark.gpu


def make(tokens, heads, d, src, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, heads, d), generator=g) * torch.exp(torch.randn((heads, d), generator=g))
    return x.to(TORCH[src])


def check(got, want, size, out):
    for a, w, m in zip(got, want, size):
        tol = 20 * 2.0 ** -24 * m + (0 if out == "f32" else HALF_ULP[out] * np.abs(w) * 1.001)
        assert np.all(np.abs(f64(a) - w) <= tol + 2.0 ** -25)


CASES = [
    # tokens, hq, hkv, d, rot, interleaved, norm, src, out
    (1, 14, 2, 64, 64, False, False, "f32", "f32"),
    (1, 1, 1, 8, 8, True, True, "f32", "f32"),
    (7, 32, 8, 128, 128, False, True, "f32", "bf16"),
    (33, 4, 4, 256, 64, True, False, "bf16", "bf16"),
    (130, 8, 4, 256, 256, False, True, "bf16", "f32"),
    (5, 3, 1, 80, 20, False, True, "f32", "f16"),        # a part whose halves fall inside a lane's eight
    (5, 3, 3, 96, 96, True, True, "f16", "f16"),
    (9, 2, 1, 128, 2, False, False, "f32", "f32"),
    (9, 2, 1, 128, 0, False, True, "f32", "f32"),        # no position at all: the norm alone
    (1001, 16, 8, 128, 64, False, True, "f32", "bf16"),
]


@pytest.mark.parametrize("tokens,hq,hkv,d,rot,inter,norm,src,out", CASES)
def test_values(frq, tokens, hq, hkv, d, rot, inter, norm, src, out):
    x = make(tokens, hq + 2 * hkv, d, src, seed=tokens + d)
    table = rope_table(max(rot, 2), 4096)
    rng = np.random.default_rng(tokens)
    pos = rng.integers(0, 4096, tokens).astype(np.int32)
    wq, wk = ((1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if norm else None for _ in range(2))
    got = [torch.full((tokens, h, d), 7.0, dtype=TORCH[out], device="cuda") for h in (hq, hkv, hkv)]
    device.qk_norm_rope(x.cuda(), *got, tokens, hq, hkv, d, dev(table), dev(pos), rot=rot, interleaved=inter,
                        q_norm=None if wq is None else dev(wq), k_norm=None if wk is None else dev(wk), eps=1e-5,
                        x_dtype=src, out_dtype=out)
    torch.cuda.synchronize()
    cs = table[pos][:, :rot // 2]
    want, size = rope(f64(x), hq, hkv, d, rot, inter, cs, wq, wk, 1e-5)
    check(got, want, size, out)
    if src == out or out == "f32":
        assert np.array_equal(f64(got[2]), f64(x[:, hq + hkv:]))


def test_in_place_and_strided_rows_on_a_stream(frq):
    """The heads of a wider row, rewritten where they are; v untouched."""
    tokens, hq, hkv, d, ld = 50, 4, 2, 64, 640
    x = make(tokens, ld // d, d, "f32").view(tokens, ld)
    cu = x.cuda()
    table, pos = rope_table(d, 64), np.arange(tokens, dtype=np.int32)
    tc, pc = dev(table), dev(pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    device.qk_norm_rope(cu, cu.data_ptr(), cu.data_ptr() + 4 * hq * d, None, tokens, hq, hkv, d, tc, pc,
                        ld_x=ld, ld_q=ld, ld_k=ld, stream=s)
    s.synchronize()
    want, size = rope(f64(x).reshape(tokens, -1, d)[:, :hq + 2 * hkv], hq, hkv, d, d, False, table[pos])
    got = f64(cu).reshape(tokens, -1, d)
    check([torch.as_tensor(got[:, :hq]), torch.as_tensor(got[:, hq:hq + hkv])], want[:2], size[:2], "f32")
    assert np.array_equal(got[:, hq + hkv:], f64(x).reshape(tokens, -1, d)[:, hq + hkv:])


def test_unknown_positions_give_nan_and_nothing_else(frq):
    x = make(4, 3, 64, "f32")
    out = [torch.zeros((4, 1, 64), device="cuda") for _ in range(3)]
    pos = np.array([3, -1, 8, 7], np.int32)
    device.qk_norm_rope(x.cuda(), *out, 4, 1, 1, 64, dev(rope_table(64, 8)), dev(pos))
    torch.cuda.synchronize()
    for o in out[:2]:
        assert torch.isnan(o).all(-1).flatten().tolist() == [False, True, True, False]
        assert not torch.isnan(o[[0, 3]]).any()
    assert np.array_equal(f64(out[2]), f64(x[:, 2:]))


def test_zero_heads_and_special_values_stay_in_their_head(frq):
    x = make(2, 4, 64, "f32")
    x[0, 0] = 0
    x[1, 1, 5] = float("inf")
    w = torch.ones(64)
    out = [torch.zeros((2, h, 64), device="cuda") for h in (2, 1, 1)]
    device.qk_norm_rope(x.cuda(), *out, 2, 2, 1, 64, dev(rope_table(64, 4)), dev(np.zeros(2, np.int32)),
                        q_norm=w.cuda(), k_norm=w.cuda())
    torch.cuda.synchronize()
    assert torch.all(out[0][0, 0] == 0)
    assert torch.isnan(out[0][1, 1]).any()
    assert torch.isfinite(out[0][1, 0]).all() and torch.isfinite(out[1]).all()
