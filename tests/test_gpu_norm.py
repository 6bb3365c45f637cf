"""add_rms_norm against the 64-bit form.

The kernel computes in 64 bits and rounds to fp32 once: half a last place, and
2^-30 for where its 64-bit value and the oracle's, some 2^-50 apart, round
differently. A 16-bit output rounds the fp32 value again: half of its last
place and 2^-24 (fp16: 2^-25 below its normal range). The sum is an fp32
addition and one rounding: the same bits. So are Q8_0 blocks of equal fp32
values: quotients are correctly rounded."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import HALF_ULP, TORCH, dev, f64
from flatrun_amd import device

pytestmark = pytest.mark.gpu


def make(rows, hidden, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    ch = torch.exp(0.5 * torch.randn(hidden, generator=g))
    ch[::97] *= 30
    return (size * torch.randn((rows, hidden), generator=g) * ch).to(TORCH[dtype])


def oracle(h, w, eps):
    h = f64(h)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return y if w is None else y * w.astype(np.float64)


def blocks(y):
    """Q8_0 bytes of fp32 values."""
    b = y.astype(np.float32).reshape(-1, 32)
    d = np.minimum(np.abs(b).max(1) / np.float32(127), np.float32(65504)).astype(np.float16)
    f = d.astype(np.float32)[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(f == 0, 0, np.clip(np.rint(b / f), -127, 127)).astype(np.int8)
    return np.concatenate([d[:, None].view(np.uint8).reshape(-1, 2), q.view(np.uint8)], axis=1)


def check(got, want, out):
    tol = (2.0 ** -24 + 2.0 ** -30 + (0 if out == "f32" else HALF_ULP[out])) * np.abs(want) + (2.0 ** -25 if out == "f16" else 1e-44)
    assert np.all(np.abs(f64(got) - want) <= tol)


def empty(rows, hidden, out):
    if out == "q8_0":
        return torch.full((rows, hidden // 32, 34), 7, dtype=torch.uint8, device="cuda")
    return torch.full((rows, hidden), 7.0, dtype=TORCH[out], device="cuda")


CASES = [
    # rows, hidden, x, residual (None: the norm alone), out, weight
    (1, 896, "f32", "f32", "f32", True),
    (1, 1, "f32", "f32", "f32", True),
    (3, 7, "bf16", "f32", "f16", True),
    (2, 32, "f16", "f16", "q8_0", True),
    (5, 64, "f32", None, "bf16", False),
    (33, 512, "bf16", "bf16", "bf16", True),
    (33, 520, "f16", "f32", "f16", True),
    (4, 4096, "f32", "f32", "bf16", True),
    (4, 3584, "bf16", "bf16", "q8_0", True),
    (3, 5000, "f32", "bf16", "f32", True),              # more than eight elements a thread, an uneven end
    (2, 8192, "bf16", "f16", "f32", True),
    (2, 16384, "f32", "f32", "q8_0", False),
    (2, 16392, "bf16", "bf16", "f32", True),            # too long for a workgroup's registers
    (2, 20032, "f16", "f32", "q8_0", True),
    (300, 1001, "f32", "f32", "f32", True),             # odd rows: not aligned
    (3000, 96, "bf16", None, "q8_0", True),
]


@pytest.mark.parametrize("rows,hidden,src,res,out,weight", CASES)
def test_values(frq, rows, hidden, src, res, out, weight):
    x = make(rows, hidden, src, seed=hidden)
    r = None if res is None else make(rows, hidden, res, seed=hidden + 1, size=3.0)
    w = (1 + 0.3 * np.random.default_rng(hidden).standard_normal(hidden)).astype(np.float32) if weight else None
    h = x if r is None else (x.float() + r.float()).to(r.dtype)
    got, total = empty(rows, hidden, out), None if r is None else torch.full_like(r, 7.0).cuda()
    device.add_rms_norm(x.cuda(), got, rows, hidden, weight=None if w is None else dev(w), residual=None if r is None else r.cuda(),
                        sum_out=total, eps=1e-5, x_dtype=src, res_dtype=res or "f32", out_dtype=out)
    torch.cuda.synchronize()
    if r is not None:
        assert torch.equal(total.cpu(), h)
    want = oracle(h, w, 1e-5)
    if out == "q8_0":
        assert np.array_equal(got.cpu().numpy().reshape(-1, 34), blocks(want))
    else:
        check(got, want, out)


@pytest.mark.parametrize("hidden,ld", [(512, 640), (512, 513), (96, 100)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_in_place_on_strided_rows(frq, hidden, ld, out):
    """The residual is updated where it is; what lies between rows stays."""
    rows = 9
    x, r = make(rows, ld, "f32", 1), make(rows, ld, "f32", 2)
    xc, rc = x.cuda(), r.cuda()
    o = torch.full((rows, ld), 7.0, dtype=TORCH[out], device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    device.add_rms_norm(xc, o, rows, hidden, residual=rc, sum_out=rc, out_dtype=out, ld_x=ld, ld_res=ld, ld_sum=ld, ld_out=ld,
                        stream=s)
    s.synchronize()
    assert torch.equal(rc.cpu()[:, :hidden], (x + r)[:, :hidden]) and torch.equal(rc.cpu()[:, hidden:], r[:, hidden:])
    check(o[:, :hidden], oracle((x + r)[:, :hidden], None, 1e-6), out)
    assert torch.all(o[:, hidden:] == 7) and torch.equal(xc.cpu(), x)


@pytest.mark.parametrize("hidden", [256, 250])
@pytest.mark.parametrize("where", ["x", "residual"])
def test_outputs_in_the_place_of_inputs(frq, hidden, where):
    x, r = make(5, hidden, "f32", 3), make(5, hidden, "f32", 4)
    xc, rc = x.cuda(), r.cuda()
    other = torch.empty_like(xc)
    device.add_rms_norm(xc, xc if where == "x" else rc, 5, hidden, residual=rc, sum_out=other if where == "x" else xc)
    torch.cuda.synchronize()
    assert torch.equal((other if where == "x" else xc).cpu(), x + r)
    check(xc if where == "x" else rc, oracle(x + r, None, 1e-6), "f32")


@pytest.mark.parametrize("hidden", [64, 100])
def test_special_rows(frq, hidden):
    """Zeros, values whose squares pass fp32 either way, an inf, a NaN: each in its own row."""
    x = torch.ones((6, hidden))
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, 5] = float("inf")
    x[4, 7] = float("nan")
    for eps in (0.0, 1e-6):
        o = torch.full((6, hidden), 7.0, device="cuda")
        device.add_rms_norm(x.cuda(), o, 6, hidden, eps=eps)
        torch.cuda.synchronize()
        o = o.cpu()
        assert torch.isnan(o[0]).all() if eps == 0 else torch.all(o[0] == 0)
        check(o[[1, 2, 5]], oracle(x[[1, 2, 5]], None, eps), "f32")
        assert torch.isnan(o[3, 5]) and torch.all(o[3, :5] == 0) and torch.isnan(o[4]).all()


def test_q8_blocks_with_specials_and_large_values(frq):
    """A block with an inf or a NaN reads back as NaN, its neighbours as they are; scales are held to 65504."""
    x, w = torch.ones((1, 128)), torch.ones(128)
    w[3], w[40], w[64:96] = float("inf"), float("nan"), 3e7
    out, val = empty(1, 128, "q8_0"), torch.zeros(128, device="cuda")
    device.add_rms_norm(x.cuda(), out, 1, 128, weight=w.cuda(), eps=0.0, out_dtype="q8_0")
    device.dequant("Q8_0", out, val, 128)
    torch.cuda.synchronize()
    v = val.cpu()
    assert torch.isnan(v[:64]).all() and torch.all(v[64:96] == 127 * 65504)
    assert torch.equal(v[96:], torch.full((32,), float(np.float16(1 / 127)) * 127))


def test_q8_rows_are_a_matrix_for_gemv(frq):
    """Normed rows kept in 8 bits and searched by a vector."""
    rows, hidden = 37, 896
    x, q = make(rows, hidden, "f32", 5), make(1, hidden, "f32", 6)[0]
    out, y = empty(rows, hidden, "q8_0"), torch.empty(rows, device="cuda")
    device.add_rms_norm(x.cuda(), out, rows, hidden, out_dtype="q8_0")
    device.gemv("Q8_0", out, q.cuda(), y, rows, hidden)
    torch.cuda.synchronize()
    b = blocks(oracle(x, None, 1e-6)).reshape(rows, -1, 34)
    m = (b[..., 2:].view(np.int8) * b[..., :2].copy().view(np.float16).astype(np.float64)).reshape(rows, hidden)
    assert np.all(np.abs(f64(y) - m @ f64(q)) <= 1e-5 * (np.abs(m) @ np.abs(f64(q))))


def test_graph_replay(frq):
    """One step captured: the residual grows by x at each replay."""
    rows, hidden = 3, 896
    x, r = make(rows, hidden, "f32", 7).cuda(), make(rows, hidden, "f32", 8).cuda()
    o, total = torch.empty_like(x), r.clone()
    torch.cuda.synchronize()
    s = device.Stream()
    with device.Graph.capture(s) as g:
        device.add_rms_norm(x, o, rows, hidden, residual=total, sum_out=total, stream=s)
    want = r.clone()
    for _ in range(3):
        g.launch(s)
        s.synchronize()
        want += x
        assert torch.equal(total, want)
        check(o, oracle(want, None, 1e-6), "f32")
    g.destroy()
    s.destroy()


@pytest.mark.parametrize("hidden", [4096, 20032])
def test_codes_next_to_a_half(frq, hidden):
    """y one last place beside d (k + 1/2): the quotient rounded to fp32 may be the half itself, the code is the
    exact quotient's. A row of ones under weights w has y = w / sqrt(1 + eps), here w itself (eps 0)."""
    rng = np.random.default_rng(hidden)
    w = np.zeros((hidden // 32, 32), np.float32)
    d = np.exp2(rng.uniform(-14, 3, hidden // 32)).astype(np.float16).astype(np.float32)
    half = rng.integers(0, 126, w.shape) + 0.5
    step = rng.choice([-1, 0, 1], w.shape)
    w[:] = (half * d[:, None]).astype(np.float32)
    w = np.where(step < 0, np.nextafter(w, np.float32(-1)), np.where(step > 0, np.nextafter(w, np.float32(1e9)), w)).astype(np.float32)
    w[:, 7] = 127 * d                                    # the largest: the scale is d again
    w *= rng.choice(np.array([-1, 1], np.float32), w.shape)
    out = empty(1, hidden, "q8_0")
    device.add_rms_norm(torch.ones((1, hidden), device="cuda"), out, 1, hidden, weight=torch.as_tensor(w.reshape(-1)).cuda(), eps=0.0,
                        out_dtype="q8_0")
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(-1, 34)
    assert np.array_equal(got[:, :2].copy().view(np.float16)[:, 0].astype(np.float32), d)
    assert np.array_equal(got[:, 2:].view(np.int8), np.rint(w.astype(np.float64) / d.astype(np.float64)[:, None]))


@pytest.mark.parametrize("hidden", [8, 32, 64, 72, 128, 192, 256, 264, 97, 511, 8191, 8193, 16383])
@pytest.mark.parametrize("rows", [1, 31, 33, 259])
def test_rows_that_share_a_workgroup_or_hold_one_element_a_lane(frq, hidden, rows):
    for src, res, out in (("f32", "f32", "f32"), ("bf16", "f32", "bf16"), ("f16", "f16", "f16")) + (
            (("bf16", "bf16", "q8_0"),) if hidden % 32 == 0 else ()):
        x, r = make(rows, hidden, src, seed=hidden), make(rows, hidden, res, seed=rows)
        w = np.random.default_rng(hidden).standard_normal(hidden).astype(np.float32)
        h = (x.float() + r.float()).to(TORCH[res])
        total, o = torch.full_like(h, 9).cuda(), empty(rows + 1, hidden, out)
        device.add_rms_norm(x.cuda(), o, rows, hidden, weight=dev(w), residual=r.cuda(), sum_out=total, x_dtype=src, res_dtype=res,
                            out_dtype=out)
        torch.cuda.synchronize()
        assert torch.equal(total.cpu(), h) and torch.all(o[rows] == 7)
        want = oracle(h, w, 1e-6)
        if out == "q8_0":
            assert np.array_equal(o[:rows].cpu().numpy().reshape(-1, 34), blocks(want))
        else:
            check(o[:rows], want, out)


@pytest.mark.parametrize("hidden", [8, 7])
def test_more_rows_than_a_launch_takes(frq, hidden):
    rows = (1 << 21) + 5
    x = torch.arange(rows, device="cuda", dtype=torch.float32)[:, None] % 1000 + torch.arange(1, hidden + 1, device="cuda")
    out = torch.full((rows + 1, hidden), 7.0, device="cuda")
    torch.cuda.synchronize()
    device.add_rms_norm(x, out, rows, hidden)
    torch.cuda.synchronize()
    y = x.double()
    want = y / torch.sqrt((y * y).mean(-1, keepdim=True) + float(np.float32(1e-6)))
    assert torch.all((out[:rows].double() - want).abs() <= (2.0 ** -24 + 2.0 ** -30) * want.abs()) and torch.all(out[rows] == 7)


@pytest.mark.parametrize("hidden", [64, 67])
def test_rows_past_32_bits(frq, hidden):
    ld = (1 << 30) + 8
    x = torch.zeros((3, ld), dtype=torch.bfloat16, device="cuda")
    x[:, :hidden] = make(3, hidden, "bf16", seed=1).cuda()
    out = torch.empty((3, hidden), device="cuda")
    torch.cuda.synchronize()
    device.add_rms_norm(x, out, 3, hidden, x_dtype="bf16", ld_x=ld, residual=x, sum_out=x, res_dtype="bf16", ld_res=ld, ld_sum=ld)
    torch.cuda.synchronize()
    h = 2 * make(3, hidden, "bf16", seed=1).float()
    assert torch.equal(x[:, :hidden].float().cpu(), h) and torch.all(x[:, hidden:hidden + 64] == 0)
    check(out, oracle(h, None, float(np.float32(1e-6))), "f32")
