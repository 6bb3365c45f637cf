"""attn_prefill against 64-bit attention.

Bound: scores as in attn_ref.fp32_bound (without q's split), each weight
rounded to the inputs' type for its product (half its last place, and below
fp16's normal range 2^-25 of the largest), the result rounded once."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import HALF_ULP, TORCH, attend, dev, f64, fp32_bound
from flatrun_amd import device

pytestmark = pytest.mark.gpu


class Setup:
    def __init__(self, nq, nk, hq, hkv, d, dtype="bf16", seed=0, qmul=1.5):
        g = torch.Generator().manual_seed(seed)
        self.nq, self.nk, self.hq, self.hkv, self.d, self.dtype = nq, nk, hq, hkv, d, dtype
        t = TORCH[dtype]
        self.q = (qmul * torch.randn((sum(nq), hq, d), generator=g)).to(t)
        self.k = torch.randn((sum(nk), hkv, d), generator=g).to(t)
        self.v = torch.randn((sum(nk), hkv, d), generator=g).to(t)
        self.cu = [dev(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)) for n in (nq, nk)]

    def run(self, causal=True, out_dtype=None, scale=None):
        out = torch.full(self.q.shape, 5.0, dtype=TORCH[out_dtype or self.dtype], device="cuda")
        device.attn_prefill(self.q.cuda(), self.k.cuda(), self.v.cuda(), out, *self.cu, len(self.nq), sum(self.nq),
                            sum(self.nk), self.hq, self.hkv, self.d, max(self.nq), max(self.nk), causal=causal,
                            dtype=self.dtype, out_dtype=out_dtype, scale=scale)
        torch.cuda.synchronize()
        return f64(out)

    def check(self, got, causal=True, out_dtype=None, scale=None, heads=None):
        scale = self.d ** -0.5 if scale is None else scale
        aq = ak = 0
        q, k, v = f64(self.q), f64(self.k), f64(self.v)
        for nq, nk in zip(self.nq, self.nk):
            last = np.arange(nq) + nk - nq if causal else np.full(nq, nk - 1)
            for h in heads or range(self.hq):
                kv = h // (self.hq // self.hkv)
                vv = v[ak:ak + nk, kv]
                want, mag, size = attend(q[aq:aq + nq, h], k[ak:ak + nk, kv], vv, scale, last)
                tol = fp32_bound(mag, size, nk, self.d) + HALF_ULP[self.dtype] * mag
                if self.dtype == "f16" and nk:
                    tol = tol + 2.0 ** -25 * nk * np.abs(vv).max(initial=0)
                if (out_dtype or self.dtype) != "f32":
                    tol = tol + HALF_ULP[self.dtype] * np.abs(want) * 1.001
                err = np.abs(got[aq:aq + nq, h] - want)
                assert np.all(err <= tol + 1e-30), (nq, nk, h, float((err / np.maximum(tol, 1e-30)).max()))
            aq, ak = aq + nq, ak + nk


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257])
def test_lengths(frq, n):
    s = Setup([n], [n], 2, 1, 64, seed=n)
    s.check(s.run())


@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 64), (14, 2, 64), (4, 4, 128), (8, 2, 128), (7, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
def test_heads_and_types(frq, hq, hkv, d, dtype, causal):
    s = Setup([75, 140], [75, 140], hq, hkv, d, dtype=dtype, seed=hq + d)
    s.check(s.run(causal), causal)
    s.check(s.run(causal, out_dtype="f32"), causal, out_dtype="f32")


@pytest.mark.parametrize("nq,nk", [([1, 5, 130, 64], [300, 5, 200, 65]), ([3, 1, 1], [0, 1, 0]), ([5, 200], [3, 70]),
                                   ([100, 0, 7], [100, 50, 7]), ([1] * 9, list(range(60, 69)))])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_and_chunks(frq, nq, nk, causal):
    """Chunks of longer prompts, sequences without queries or keys, and fewer
    keys than queries: rows that see no key are zeros."""
    s = Setup(nq, nk, 4, 2, 64, seed=sum(nk))
    got = s.run(causal)
    s.check(got, causal)
    aq = 0
    for a, b in zip(nq, nk):
        empty = a if b == 0 else max(0, a - b) if causal else 0
        assert np.all(got[aq:aq + empty] == 0)
        aq += a


def test_long(frq):
    s = Setup([1500], [2100], 4, 1, 128, seed=1)
    s.check(s.run(), heads=[0, 3])


def test_peaked_rising_and_flat_scores(frq):
    s = Setup([190], [190], 2, 1, 64, seed=2, qmul=40.0)
    s.check(s.run())
    s = Setup([400], [400], 2, 1, 64, seed=3)
    s.k = (s.k.float() * torch.linspace(0.01, 8, 400)[:, None, None]).to(s.k.dtype)
    s.check(s.run())
    s.q[:] = 0
    s.check(s.run())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_special_values_in_masked_places(frq, dtype, bad):
    """Keys and values that a query does not see never reach it."""
    n, at = 150, 70
    s = Setup([n, 40], [n, 40], 2, 1, 64, dtype=dtype, seed=4)
    clean = s.run()
    s.k[at, 0, 5] = bad
    s.v[at, 0, 9] = bad
    got = s.run()
    s2 = Setup([n, 40], [n, 40], 2, 1, 64, dtype=dtype, seed=4)
    s2.check(np.concatenate([got[:at], clean[at:]]))
    assert np.isfinite(got[:at]).all() and np.array_equal(got[n:], clean[n:])
    assert not np.isfinite(got[at:n]).all()
    s2.v[at, 0, 9] = bad                                     # the value alone: its column only, for those who see it
    got = s2.run()
    assert np.isfinite(np.delete(got, 9, axis=2)).all()
    assert np.isfinite(got[:at]).all() and not np.isfinite(got[at:n, :, 9]).any()


def test_a_special_query_stays_in_its_row(frq):
    s = Setup([100], [100], 2, 1, 64, seed=5)
    clean = s.run()
    s.q[40, 1, 3] = float("nan")
    got = s.run()
    assert np.isnan(got[40, 1]).all()
    got[40, 1] = clean[40, 1]
    assert np.array_equal(got, clean)


def test_rows_of_a_wider_buffer_and_heads_first(frq):
    """q|k|v rows as a projection writes them, and head-major tensors."""
    n, hq, hkv, d = 90, 4, 2, 64
    s = Setup([n], [n], hq, hkv, d, seed=6)
    rows = torch.cat([s.q.view(n, -1), s.k.view(n, -1), s.v.view(n, -1)], dim=1).cuda()
    ld, out = rows.shape[1], torch.zeros((hq, n, d), dtype=torch.bfloat16, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    base = rows.data_ptr()
    device.attn_prefill(base, base + 2 * hq * d, base + 2 * (hq + hkv) * d, out, *s.cu, 1, n, n, hq, hkv, d, n, n,
                        ld_q=ld, ld_k=ld, ld_v=ld, ld_out=d, hs_out=n * d, stream=st)
    st.synchronize()
    s.check(f64(out.transpose(0, 1)))
    qh, kh, vh = (x.transpose(0, 1).contiguous().cuda() for x in (s.q, s.k, s.v))
    out2 = torch.zeros((n, hq, d), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    device.attn_prefill(qh, kh, vh, out2, *s.cu, 1, n, n, hq, hkv, d, n, n, ld_q=d, ld_k=d, ld_v=d, hs_q=n * d,
                        hs_k=n * d, hs_v=n * d)
    torch.cuda.synchronize()
    assert torch.equal(out2, out.transpose(0, 1))


def test_same_bits_every_time_and_other_scale(frq):
    s = Setup([300, 40], [340, 40], 4, 2, 128, seed=7)
    assert np.array_equal(s.run(), s.run())
    s.check(s.run(scale=0.2), scale=0.2)


def test_offsets_that_leave_the_buffers_are_not_computed(frq):
    s = Setup([20, 20, 20], [20, 20, 20], 2, 1, 64, seed=8)
    clean = s.run()
    s.cu[1] = dev(np.array([0, 20, 40, 61], np.int32))
    got = s.run()
    assert np.array_equal(got[:40], clean[:40]) and np.all(got[40:] == 5.0)


def test_offsets_past_32_bits(frq):
    """Keys and values 2 MiB apart: 2100 of them span more than 2^32 bytes, and
    a tile of 64 more than 2^26."""
    s = Setup([70], [2100], 2, 1, 64, seed=9)
    clean = s.run()
    ld = 1 << 20
    wide = torch.empty(2099 * ld + 128, dtype=torch.bfloat16, device="cuda")
    rows = torch.as_strided(wide, (2100, 128), (ld, 1))
    rows[:, :64] = s.k[:, 0].cuda()
    rows[:, 64:] = s.v[:, 0].cuda()
    out = torch.zeros((70, 2, 64), dtype=torch.bfloat16, device="cuda")
    device.attn_prefill(s.q.cuda(), wide.data_ptr(), wide.data_ptr() + 128, out, *s.cu, 1, 70, 2100, 2, 1, 64, 70, 2100,
                        ld_k=ld, ld_v=ld)
    torch.cuda.synchronize()
    assert np.array_equal(f64(out), clean)


@pytest.mark.parametrize("nq,nk,hq,hkv", [([1100, 40, 0, 513], [1100, 700, 9, 600], 4, 2), ([1030], [1090], 12, 4),
                                          ([1025, 1], [1025, 1], 5, 1)])
def test_long_packed_heads_of_128(frq, nq, nk, hq, hkv):
    """More than 1024 queries: eight waves to a key tile."""
    s = Setup(nq, nk, hq, hkv, 128, seed=sum(nq))
    s.check(s.run(), heads=range(0, hq, 3))


def test_special_values_in_masked_places_of_long_prompts(frq):
    s = Setup([1100], [1100], 4, 1, 128, seed=10)
    clean = s.run()
    s.v[1040, 0, 5], s.v[1041, 0, 6] = float("inf"), float("nan")
    got = s.run()
    assert np.array_equal(got[:1040], clean[:1040])
    assert np.all(got[1040:, :, 5] == np.inf) and np.isnan(got[1041:, :, 6]).all()
    got[1040:, :, 5:7] = clean[1040:, :, 5:7]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("nq,nk,hq,hkv,d,causal", [
    ([384], [384], 2, 1, 64, True), ([33, 1, 0, 200], [640, 385, 3, 200], 4, 2, 128, True),
    ([40, 450], [449, 300], 2, 2, 64, False), ([300, 20], [400, 0], 6, 2, 128, False),
    ([700], [700], 28, 4, 128, True), ([900, 31], [1000, 64], 14, 2, 64, True),
    ([200] * 7, [390] * 7, 32, 8, 128, True), ([1100], [1100], 32, 8, 128, True),
    ([1030, 40, 700, 5], [1030, 90, 700, 5], 32, 8, 128, True),
])
def test_few_queries_and_many(frq, nq, nk, hq, hkv, d, causal):
    """Tiles of a unit shared by two waves, in workgroups of four and of eight,
    and enough units that none are."""
    s = Setup(nq, nk, hq, hkv, d, seed=sum(nk) + d)
    got = s.run(causal=causal)
    s.check(got, causal=causal, heads=range(0, hq, max(1, hq // 4)))
    assert np.array_equal(got, s.run(causal=causal))


def test_peaked_rows_whose_tiles_two_waves_share(frq):
    """The reference rises from tile to tile, or is far apart in the two halves."""
    s = Setup([100], [900], 4, 2, 64, seed=11, qmul=6.0)
    s.k *= torch.linspace(0.1, 6, 900)[:, None, None].to(s.k.dtype)
    s.check(s.run())
    s = Setup([100], [900], 4, 2, 128, seed=12, qmul=6.0)
    s.k[64:128] *= 8                                         # one tile of the second half outweighs the rest
    s.check(s.run())
    s.k[:64] *= 30
    s.check(s.run())


@pytest.mark.parametrize("nq,nk,at,d", [([100], [100], 0, 64), ([100], [100], 40, 128), ([70, 20], [500, 20], 69, 64),
                                        ([40], [30], 10, 256)])
def test_queries_whose_keys_all_score_minus_infinity(frq, nq, nk, at, d):
    """A softmax of nothing but -inf is 0 / 0; zeros are for queries that see no key."""
    s = Setup(nq, nk, 2, 1, d, seed=14)
    clean = s.run(out_dtype="f32")
    s.q[at, 1, 7] = float("inf")
    s.k[:, 0, 7] = -s.k[:, 0, 7].abs() - 0.125
    want = s.run(out_dtype="f32")                            # of the other queries, with these keys
    assert np.isnan(want[at, 1]).all()
    s.q[at, 1, 7] = 1.0
    other = s.run(out_dtype="f32")
    other[at, 1], want[at, 1] = 0, 0
    assert np.array_equal(other, want) and np.isfinite(clean).all()
    if nk[0] < nq[0]:                                        # no key at all: zeros, also for a query with an inf
        s.q[3, 1, 7] = float("inf")
        assert np.all(s.run()[:nq[0] - nk[0]] == 0)


@pytest.mark.parametrize("most", [20, 64, 129])
@pytest.mark.parametrize("d,hq,hkv", [(64, 6, 2), (128, 4, 4)])
def test_sequences_longer_than_max_q_are_nan(frq, most, d, hq, hkv):
    """All their rows, and only theirs."""
    s = Setup([130, 20, 700, 0, 300], [130, 20, 700, 5, 500], hq, hkv, d, seed=15)
    clean = s.run()
    out = torch.full((1170, hq, d), 5.0, dtype=torch.bfloat16, device="cuda")
    device.attn_prefill(s.q.cuda(), s.k.cuda(), s.v.cuda(), out[:1150], *s.cu, 5, 1150, 1355, hq, hkv, d, most, 700)
    torch.cuda.synchronize()
    got = f64(out)
    assert np.isnan(got[:130]).all() and np.isnan(got[150:1150]).all() and np.all(got[1150:] == 5)
    s.check(np.concatenate([clean[:130], got[130:150], clean[150:]]))
