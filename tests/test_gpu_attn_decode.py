"""attn_decode against 64-bit attention over the values the cache holds
(bounds: attn_ref.fp32_bound; a 16-bit output adds half its last place)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import HALF_ULP, TORCH, attend, block4, dev, f64, fp32_bound
from flatrun_amd import device
from flatrun_amd.attention import KVCache4

pytestmark = pytest.mark.gpu


class Setup:
    def __init__(self, lens, hq, hkv, d, page, dtype="f32", seed=0, kmul=1.0, vmul=1.0, qmul=2.0, spare=1):
        g = torch.Generator().manual_seed(seed)
        per = [-(-n // page) for n in lens]
        self.lens, self.hq, self.hkv, self.d, self.dtype = lens, hq, hkv, d, dtype
        self.cache = KVCache4(sum(per) + spare, page, hkv, d)
        perm = torch.randperm(sum(per) + spare, generator=g).numpy()
        self.table = np.full((len(lens), max(per + [1])), -7, np.int32)
        slots, at = [], 0
        for i, (n, p) in enumerate(zip(lens, per)):
            self.table[i, :p] = perm[at:at + p]
            t = np.arange(n)
            slots.append(self.table[i, t // page].astype(np.int64) * page + t % page)
            at += p
        self.slots = np.concatenate(slots) if lens else np.zeros(0, np.int64)
        total = sum(lens)
        self.k = (kmul * torch.randn((total, hkv, d), generator=g)).numpy()
        self.v = (vmul * torch.randn((total, hkv, d), generator=g)).numpy()
        self.q = (qmul * torch.randn((len(lens), hq, d), generator=g)).to(TORCH[dtype])
        # what no token owns is poison: masked places that must not matter
        every = np.arange(self.cache.pages * page)
        nan = torch.full((len(every), hkv, d), float("nan"), device="cuda")
        self.cache.write(nan, nan, dev(every), len(every))
        if total:
            self.cache.write(dev(self.k), dev(self.v), dev(self.slots), total)

    def run(self, max_len=None, scale=None, stream=None):
        out = torch.full(self.q.shape, 5.0, dtype=TORCH[self.dtype], device="cuda")
        table = dev(self.table)
        device.attn_decode(self.q.cuda(), self.cache, table, dev(np.array(self.lens, np.int32)), out, len(self.lens),
                           self.hq, max(self.lens) if max_len is None else max_len, dtype=self.dtype, scale=scale,
                           stream=stream)
        torch.cuda.synchronize()
        return f64(out)

    def check(self, got, scale=None):
        scale = self.d ** -0.5 if scale is None else scale
        at, g = 0, self.hq // self.hkv
        for b, n in enumerate(self.lens):
            kk, vv = block4(self.k[at:at + n]), block4(self.v[at:at + n])
            at += n
            for h in range(self.hkv):
                q = f64(self.q)[b, h * g:(h + 1) * g]
                want, mag, size = attend(q, kk[:, h], vv[:, h], scale, np.full(g, n - 1))
                tol = fp32_bound(mag, size, n, self.d)
                if self.dtype != "f32":
                    tol = tol + HALF_ULP[self.dtype] * 1.001 * np.abs(want) + 2.0 ** -25
                err = np.abs(got[b, h * g:(h + 1) * g] - want)
                assert np.all(err <= tol), (b, h, n, float((err / np.maximum(tol, 1e-300)).max()))


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_lengths(frq, n):
    s = Setup([n, 5], 4, 2, 128, 32, seed=n)
    got = s.run()
    if n == 0:
        assert np.all(got[0] == 0)
    s.check(got)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (1, 1, 64), (8, 8, 128), (32, 8, 128), (28, 4, 128), (8, 4, 256),
                                      (16, 2, 64), (18, 2, 128), (24, 1, 128)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_heads_and_types(frq, hq, hkv, d, dtype):
    s = Setup([77, 0, 200, 1], hq, hkv, d, 64, dtype=dtype, seed=hq + d)
    s.check(s.run())


@pytest.mark.parametrize("batch,hi,page", [(1, 5000, 32), (3, 3000, 256), (40, 400, 96), (1, 40, 4096)])
def test_splits(frq, batch, hi, page):
    """Long and ragged: the splits of a sequence and their joining."""
    rng = np.random.default_rng(hi)
    s = Setup([int(x) for x in rng.integers(0, hi + 1, batch - 1)] + [hi], 4, 2, 64, page, seed=hi)
    got = s.run()
    s.check(got)
    assert np.array_equal(got, s.run())                    # the same bits every time
    s.check(s.run(max_len=3 * hi if s.table.shape[1] * page >= 3 * hi else s.table.shape[1] * page))


@pytest.mark.parametrize("kmul,vmul,qmul", [(1.0, 1e-6, 2.0), (1.0, 3e4, 2.0), (1e-4, 1.0, 3e4), (3e3, 1.0, 1e-4),
                                            (1.0, 1.0, 1e-30), (1e-3, 1.0, 1e3)])
def test_magnitudes(frq, kmul, vmul, qmul):
    s = Setup([150, 33], 8, 2, 64, 32, seed=3, kmul=kmul, vmul=vmul, qmul=qmul)
    s.check(s.run())


def test_scales_of_v_that_grow_and_shrink_along_the_sequence(frq):
    s = Setup([700], 8, 2, 64, 32, seed=4)
    s.v *= np.exp(np.linspace(-9, 9, 700))[:, None, None].astype(np.float32)
    s.v[300:420] = 0
    s.cache.write(dev(s.k), dev(s.v), dev(s.slots), 700)
    s.check(s.run())


def test_a_peaked_and_a_flat_softmax(frq):
    s = Setup([600], 8, 2, 128, 64, seed=5, qmul=40.0)
    s.check(s.run())
    s.q[:] = 0
    s.check(s.run())
    s = Setup([600], 8, 2, 128, 64, seed=6)
    s.k *= np.linspace(0.01, 6, 600)[:, None, None].astype(np.float32)     # maxima that keep rising
    s.cache.write(dev(s.k), dev(s.v), dev(s.slots), 600)
    s.check(s.run())


def test_special_values_reach_their_rows_only(frq):
    s = Setup([40, 40, 40], 4, 2, 64, 32, seed=6)
    clean = s.run()
    s.q[1, 2, 3] = float("nan")
    got = s.run()
    assert np.isnan(got[1, 2]).all()
    got[1, 2] = clean[1, 2]
    assert np.array_equal(got, clean)
    s.q[1, 2, 3] = float("inf")
    assert np.isnan(s.run()[1, 2]).all()
    s = Setup([40, 40, 40], 4, 2, 64, 32, seed=6)
    s.v[45, 1, 7] = float("inf")                             # a block of sequence 1's values
    s.cache.write(dev(s.k), dev(s.v), dev(s.slots), 120)
    got = s.run()
    assert np.isnan(got[1, 2:, :32]).all()
    got[1, 2:, :32] = clean[1, 2:, :32]
    assert np.array_equal(got, clean)
    s.k[85, 0, 0] = float("nan")
    s.cache.write(dev(s.k), dev(s.v), dev(s.slots), 120)
    assert np.isnan(s.run()[2, :2]).all() and np.isfinite(s.run()[2, 2:]).all()


def test_lengths_and_pages_that_do_not_fit_are_nan(frq):
    s = Setup([40, 40, 40], 4, 2, 64, 32, seed=7)
    clean = s.run()
    s.table[0, 1], s.table[2, 0] = s.cache.pages, -1
    got = s.run()
    assert np.isnan(got[0]).all() and np.isnan(got[2]).all() and np.array_equal(got[1], clean[1])
    s = Setup([40, 64, 40], 4, 2, 64, 32, seed=7)
    got = s.run(max_len=63)
    assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()
    s.lens[0] = -3
    assert np.all(s.run(max_len=64)[0] == 0)


def test_scale_strides_and_stream(frq):
    s = Setup([90, 20], 4, 2, 64, 32, seed=8)
    s.check(s.run(scale=0.31), scale=0.31)
    st = torch.cuda.Stream()
    wide = torch.zeros((2, 1024))
    wide[:, 256:512] = s.q.view(2, 256)
    cu, out = wide.cuda(), torch.full((2, 640), 4.0, device="cuda")
    table, lens = dev(s.table), dev(np.array(s.lens, np.int32))
    st.wait_stream(torch.cuda.current_stream())
    device.attn_decode(cu.data_ptr() + 4 * 256, s.cache, table, lens, out, 2, 4, 90, ld_q=1024, ld_out=640, stream=st)
    st.synchronize()
    s.check(f64(out)[:, :256].reshape(2, 4, 64))
    assert (out[:, 256:] == 4).all()


def test_graph_replays(frq):
    """Captured on a stream that has run the shape once; replayed with other
    lengths and eager work between."""
    s = Setup([2500, 900], 4, 2, 128, 64, seed=9)
    st = device.Stream()
    q, out = s.q.cuda(), torch.zeros(s.q.shape, device="cuda")
    table, lens = dev(s.table), dev(np.array(s.lens, np.int32))
    torch.cuda.synchronize()

    def call():
        device.attn_decode(q, s.cache, table, lens, out, 2, 4, 2560, stream=st)

    call()
    st.synchronize()
    with device.Graph.capture(st) as g:
        call()
    for a, b in ((2500, 900), (33, 0), (1, 900), (2500, 900)):
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.launch(st)
        st.synchronize()
        replay = out.clone()
        call()
        st.synchronize()
        assert torch.equal(replay, out)
    s.check(f64(out))
    g.destroy()


@pytest.mark.parametrize("lens,hq,hkv,d", [
    ([0] * 70 + [1400, 0, 1, 33] + [0] * 64 + [1000], 4, 2, 64),     # empty stretches longer than a wave's lanes
    ([1500, 7, 0, 901], 24, 1, 128),                                 # three chunks of query heads to a key head
    ([1000, 1, 1203], 8, 4, 256),
    ([3] * 30 + [2200] + [40] * 33, 8, 8, 64),                       # a pair at least for every workgroup
    ([0, 0, 950], 14, 2, 128),
])
def test_sequences_that_share_the_workgroups(frq, lens, hq, hkv, d):
    s = Setup(lens, hq, hkv, d, 32, seed=len(lens) + d)
    got = s.run()
    assert np.all(got[np.array(lens) == 0] == 0)
    s.check(got)
    assert np.array_equal(got, s.run())


def test_growth_and_special_values_in_shared_sequences(frq):
    """References that are outgrown, bad lengths, pages and values where rows
    are joined from several workgroups."""
    s = Setup([2000, 1200, 0, 1300], 8, 2, 64, 32, seed=11)
    s.v[:2000] *= np.exp(np.linspace(-9, 9, 2000))[:, None, None].astype(np.float32)
    s.k[2000:3200] *= np.linspace(0.01, 6, 1200)[:, None, None].astype(np.float32)
    s.cache.write(dev(s.k), dev(s.v), dev(s.slots), 4500)
    clean = s.run()
    s.check(clean)
    s.q[0, 5, 3] = float("nan")
    got = s.run()
    assert np.isnan(got[0, 5]).all()
    got[0, 5] = clean[0, 5]
    assert np.array_equal(got, clean)
    s = Setup([2000, 1200, 0, 1300], 8, 2, 64, 32, seed=12)
    clean = s.run()
    s.table[0, 60] = s.cache.pages                           # of its last tiles
    got = s.run()
    assert np.isnan(got[0]).all() and np.array_equal(got[1:], clean[1:])
    got = s.run(max_len=1999)
    assert np.isnan(got[0]).all() and np.all(got[2] == 0) and np.isfinite(got[1:]).all()


def test_offsets_past_32_bits(frq):
    """A cache of 5 GiB, the sequence's pages at its end."""
    c = KVCache4(1200, 4096, 8, 128)
    g = torch.Generator().manual_seed(13)
    k, v, q = (torch.randn((n, h, 128), generator=g) for n, h in ((300, 8), (300, 8), (1, 16)))
    t = np.arange(300)
    page = np.where(t < 100, 1199, 1100)                     # places 3996 .. 4095 of one page, then of another
    place = np.where(t < 100, 3996 + t, t - 100)
    pad = np.arange(3996)
    c.write(dev(np.zeros((3996, 8, 128), np.float32)), dev(np.zeros((3996, 8, 128), np.float32)), dev(1199 * 4096 + pad), 3996)
    c.write(k.cuda(), v.cuda(), dev((page * 4096 + place).astype(np.int64)), 300)
    out = torch.zeros((1, 16, 128), device="cuda")
    device.attn_decode(q.cuda(), c, dev(np.array([[1199, 1100]], np.int32)), dev(np.array([4296], np.int32)), out, 1, 16,
                       4296)
    torch.cuda.synchronize()
    kk, vv = (np.concatenate([np.zeros((3996, 8, 128)), block4(f64(x))]) for x in (k, v))
    got = f64(out)
    for h in range(16):
        want, mag, size = attend(f64(q)[:, h], kk[:, h // 2], vv[:, h // 2], 128 ** -0.5, np.array([4295]))
        assert np.all(np.abs(got[:, h] - want) <= fp32_bound(mag, size, 4296, 128)), h
    c.close()
