"""attn_chunk against 64-bit attention over the values that the cache holds.

Bound: k as a product's operand is off by half a last place of fp16 (2^-11 of
itself as HALF_ULP counts it), so a score by that of scale sum |q k|, besides
the fp32 sums of attn_ref.fp32_bound; a weight and v by as much of themselves,
the weights' sum too; a weight by 2^-30 of the largest at least; the result is
rounded once."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import HALF_ULP, TORCH, attend, block4, dev, f64, fp32_bound
from flatrun_amd import device
from flatrun_amd.attention import KVCache4

pytestmark = pytest.mark.gpu
NAN = float("nan")


class Setup:
    def __init__(self, new, lens, hq, hkv, d, page=64, dtype="bf16", seed=0, qmul=1.5, stale=False, k=None, v=None, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens, self.hq, self.hkv, self.d, self.dtype = list(new), list(lens), hq, hkv, d, dtype
        n = sum(self.lens)
        self.q = (qmul * torch.randn((sum(self.new), hq, d), generator=g)).to(TORCH[dtype])
        own = [torch.randn((n, hkv, d), generator=g) for _ in range(2)]
        self.k, self.v = own[0] if k is None else k, own[1] if v is None else v
        per = [max(1, -(-m // page)) for m in self.lens]
        self.pages = sum(per) + spare
        perm = np.random.default_rng(seed).permutation(self.pages).astype(np.int32)
        self.table = np.zeros((max(1, len(per)), max(per, default=1)), np.int32)
        slots, at = [], 0
        for i, (m, p) in enumerate(zip(self.lens, per)):
            self.table[i, :p] = perm[at:at + p]
            t = np.arange(m)
            slots.append(self.table[i, t // page].astype(np.int64) * page + t % page)
            at += p
        self.cache = KVCache4(self.pages, page, hkv, d)
        if stale:                                # what earlier sequences left behind the ends
            junk = torch.full((self.pages * page, hkv, d), NAN, device="cuda")
            self.cache.write(junk, junk, dev(np.arange(self.pages * page)), self.pages * page)
        if n:
            self.cache.write(self.k.cuda(), self.v.cuda(), dev(np.concatenate(slots)), n)
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        torch.cuda.synchronize()

    def run(self, out_dtype=None, scale=None, stream=None, tail=0, **kw):
        t = sum(self.new)
        out = torch.full((t + tail, self.hq, self.d), 5.0, dtype=TORCH[out_dtype or self.dtype], device="cuda")
        a = dict(max_q=max(self.new, default=0), max_len=max(self.lens, default=0))
        a.update(kw)
        table, lens, cu = a.pop("table", self.table), a.pop("lens", self.lens), a.pop("cu", self.cu)
        ops = dev(table), dev(np.array(lens, np.int32)), dev(np.array(cu, np.int32)), self.q.cuda()
        torch.cuda.synchronize()
        device.attn_chunk(ops[3], self.cache, ops[0], ops[1], ops[2], out, len(self.new), t, self.hq, a["max_q"], a["max_len"],
                          dtype=self.dtype, out_dtype=out_dtype, scale=scale, stream=stream)
        torch.cuda.synchronize()
        assert torch.all(out[t:] == 5.0)
        return f64(out[:t])

    def check(self, got, out_dtype=None, scale=None, heads=None, rows=None):
        scale = self.d ** -0.5 if scale is None else scale
        q, k, v = f64(self.q), block4(f64(self.k)), block4(f64(self.v))
        aq = ak = 0
        for n, m in zip(self.new, self.lens):
            pick = np.arange(n) if rows is None else np.array([r % n for r in rows if n] or [], int)
            for h in heads or range(self.hq):
                g = h // (self.hq // self.hkv)
                vv = v[ak:ak + m, g]
                want, mag, size = attend(q[aq:aq + n, h][pick], k[ak:ak + m, g], vv, scale, (np.arange(n) + m - n)[pick])
                tol = fp32_bound(mag, size, m, self.d) + (2 * 2.0 ** -11 * size[:, None] + 3 * 2.0 ** -11) * mag
                tol = tol + 2.0 ** -29 * m * np.abs(vv).max(initial=0)
                if (out_dtype or self.dtype) != "f32":
                    tol = tol + HALF_ULP[self.dtype] * np.abs(want) * 1.001 + 2.0 ** -25
                err = np.abs(got[aq:aq + n, h][pick] - want)
                assert np.all(err <= tol + 1e-30), (n, m, h, float((err / np.maximum(tol, 1e-30)).max()))
            aq, ak = aq + n, ak + m


@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64, 65, 130])
def test_chunk_lengths(frq, new):
    s = Setup([new], [new + 77], 4, 2, 64, seed=new)
    s.check(s.run())


@pytest.mark.parametrize("m", [5, 31, 32, 33, 63, 64, 65, 96, 127, 129, 160, 1000, 2049])
def test_context_lengths(frq, m):
    s = Setup([5], [m], 4, 1, 64, page=32, seed=m, stale=True)
    s.check(s.run(out_dtype="f32"), out_dtype="f32")


@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 64), (14, 2, 64), (4, 4, 128), (8, 2, 128), (7, 1, 128), (28, 4, 128), (4, 2, 256),
                                      (8, 1, 256), (64, 1, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("new", [[3, 20], [75, 140]])
def test_heads_and_types(frq, hq, hkv, d, dtype, new):
    s = Setup(new, [new[0] + 200, new[1]], hq, hkv, d, page=96, dtype=dtype, seed=hq + d + new[0], stale=True)
    s.check(s.run())
    s.check(s.run(out_dtype="f32"), out_dtype="f32")


@pytest.mark.parametrize("new,lens", [([1, 5, 130, 64], [300, 5, 200, 65]), ([3, 1, 1], [0, 1, 0]), ([5, 200], [3, 70]),
                                      ([100, 0, 7], [100, 50, 7]), ([1] * 9, list(range(60, 69))), ([0, 0], [10, 0]),
                                      ([33] * 40, [40 * i + 33 for i in range(40)])])
def test_packed_sequences(frq, new, lens):
    """Sequences without queries or tokens, and fewer tokens than queries: rows that see none are zeros."""
    s = Setup(new, lens, 4, 2, 64, page=32, seed=sum(lens), stale=True)
    got = s.run(tail=2)
    s.check(got)
    at = 0
    for n, m in zip(new, lens):
        assert np.all(got[at:at + max(0, n - m)] == 0)
        at += n


@pytest.mark.parametrize("new,lens,hq,hkv,d", [([7], [20000], 8, 2, 128), ([3, 17], [9000, 30], 28, 4, 128), ([16], [5000], 2, 1, 256),
                                               ([40], [12345], 14, 2, 64), ([2] * 5, [3000, 1, 40, 7000, 2], 16, 8, 128)])
def test_keys_split_over_workgroups(frq, new, lens, hq, hkv, d):
    s = Setup(new, lens, hq, hkv, d, page=128, seed=sum(lens), stale=True)
    s.check(s.run(out_dtype="f32"), out_dtype="f32", heads=[0, hq - 1])
    s.check(s.run(), heads=[0, hq - 1])


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 8, 2), (256, 2, 1)])
def test_long_chunks(frq, d, hq, hkv):
    s = Setup([700, 1], [1500, 900], hq, hkv, d, seed=d, stale=True)
    s.check(s.run(), heads=[hq - 1], rows=[0, 1, 15, 16, 31, 32, 255, 256, 511, 698, 699])


def test_a_dominant_token_among_many_small_ones(frq):
    """Weights of 2^-22 of one token's each, half as much together: kept, not rounded away."""
    m, d = 1 << 21, 64
    k, v = torch.zeros((m, 1, d)), torch.ones((m, 1, d))
    k[5, 0, 0] = 8.0
    v[5] = -1.0
    s = Setup([2], [m], 1, 1, d, page=4096, k=k, v=v, seed=1)
    s.q[:] = 0
    s.q[:, 0, 0] = 1.0
    scale = 22 * np.log(2) / 8
    got = s.run(out_dtype="f32", scale=float(scale))
    rest = (m - 1 - np.array([1, 0])) * 2.0 ** -22
    assert np.allclose(got[:, 0], ((rest - 1) / (rest + 1))[:, None], rtol=0, atol=2e-3)


def test_scores_that_grow_along_the_keys(frq):
    """The reference moves in every tile, by little and by much."""
    for step, new in ((0.5, 6), (30.0, 6), (0.5, 200), (30.0, 200)):
        m = 700
        k = torch.zeros((m, 1, 64))
        k[:, 0, 0] = torch.arange(m) // 32 * step
        s = Setup([new], [m], 2, 1, 64, k=k, seed=3)
        s.q[:] = 0
        s.q[:, 0, 0], s.q[:, 1, 0] = 8.0, -8.0
        s.check(s.run(out_dtype="f32"), out_dtype="f32")


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 3e4, 3e5])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("new,d", [(9, 64), (90, 64), (90, 128), (20, 256)])
def test_small_and_large_values(frq, what, size, new, d):
    g = torch.Generator().manual_seed(5)
    x = size * torch.randn((400, 2, d), generator=g).clamp(-1.7, 1.7)
    s = Setup([new], [400], 4, 2, d, seed=4, stale=True, **{what: x})
    if what == "k":
        s.q = (s.q.float() / max(size, 1e-3)).to(torch.bfloat16)
    s.check(s.run(out_dtype="f32"), out_dtype="f32")


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e4, 1e30])
def test_small_and_large_queries(frq, size):
    s = Setup([9], [200], 4, 2, 64, seed=6)
    s.q = (s.q.float() * size).to(torch.bfloat16)
    s.check(s.run(out_dtype="f32", scale=0.125 / size), out_dtype="f32", scale=0.125 / size)


@pytest.mark.parametrize("new", [20, 150])
@pytest.mark.parametrize("at", [40, 120, 299])
def test_large_values_beside_ordinary_ones(frq, new, at):
    """A tile with values past fp16: the channels of the others to 2^-21 beside."""
    v = Setup([new], [300], 2, 1, 128, seed=8).v
    v[at, 0, :32] = 4e5
    s = Setup([new], [300], 2, 1, 128, seed=8, v=v, stale=True)
    s.check(s.run(out_dtype="f32"), out_dtype="f32")


@pytest.mark.parametrize("d,hq", [(64, 2), (128, 4), (256, 2)])
@pytest.mark.parametrize("new,m,at", [(20, 100, 90), (20, 100, 3), (5, 600, 599), (40, 64, 63), (100, 300, 210)])
def test_no_number_reaches_a_query_that_does_not_see_it(frq, d, hq, new, m, at):
    """A NaN in one block of k or v at one token: every row that sees the token, and in v only the block's channels."""
    base = Setup([new], [m], hq, 1, d, seed=at, stale=True)
    clean = base.run(out_dtype="f32")
    sees = np.arange(new) + m - new >= at
    for what in "kv":
        x = getattr(base, what).clone()
        x[at, 0, 37] = NAN if at % 2 else float("inf")
        got = Setup([new], [m], hq, 1, d, seed=at, stale=True, **{what: x}).run(out_dtype="f32")
        hit = np.zeros((new, hq, d), bool)
        hit[sees] = True
        if what == "v":
            hit[..., :32] = hit[..., 64:] = False
        assert np.array_equal(np.isnan(got), hit), (what, np.argwhere(np.isnan(got) != hit)[:5])
        if what == "v":
            assert np.array_equal(got[~hit], clean[~hit])
        else:
            assert np.array_equal(got[~sees], clean[~sees])


@pytest.mark.parametrize("new", [9, 99])
def test_no_number_in_a_query_stays_in_its_row(frq, new):
    s = Setup([new], [150], 4, 2, 64, seed=2)
    want = s.run(out_dtype="f32")
    s.q[3, 1, 5], s.q[7, 2, 0] = NAN, float("inf")
    got = s.run(out_dtype="f32")
    hit = np.zeros((new, 4), bool)
    hit[3, 1] = hit[7, 2] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], want[~hit])


@pytest.mark.parametrize("more", [0, 200])
def test_what_the_device_arrays_must_not_say(frq, more):
    """Lengths and pages that are not the call's give NaN, offsets outside nothing; the others stay right."""
    n = [4, 6 + more, 5]
    s = Setup(n, [40, 300, 64], 4, 2, 64, seed=11)
    want = s.run(out_dtype="f32")
    a, b, c = slice(0, 4), slice(4, 10 + more), slice(10 + more, 15 + more)
    for kw, hit in ((dict(lens=[40, 301, 64]), b), (dict(max_q=5 + more), b), (dict(lens=[40, 1 << 30, 64]), b),
                    (dict(table=np.where(np.arange(3)[:, None] == 2, s.pages, s.table)), c),
                    (dict(table=np.where(np.arange(3)[:, None] == 0, -1, s.table)), a)):
        got = s.run(out_dtype="f32", **kw)
        miss = np.ones(15 + more, bool)
        miss[hit] = False
        assert np.isnan(got[hit]).all() and np.array_equal(got[miss], want[miss]), kw
    assert np.all(s.run(out_dtype="f32", lens=[-5, 300, 64])[a] == 0)
    got = s.run(out_dtype="f32", cu=[0, 4, 10 + more, 999])
    assert np.all(got[c] == 5) and np.array_equal(got[:10 + more], want[:10 + more])
    got = s.run(out_dtype="f32", cu=[-3, 4, 10 + more, 15 + more])
    assert np.all(got[a] == 5) and np.array_equal(got[4:], want[4:])


def test_strided_queries_and_outputs(frq):
    s = Setup([5, 12], [100, 12], 4, 2, 64, seed=12)
    want, t = s.run(), 17
    wide, out = torch.full((t, 6, 64), NAN, dtype=torch.bfloat16), torch.full((t, 5, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    wide[:, :4] = s.q
    device.attn_chunk(wide.cuda(), s.cache, dev(s.table), dev(np.array(s.lens, np.int32)), dev(s.cu), out, 2, t, 4, 12, 100,
                      ld_q=6 * 64, ld_out=5 * 64)
    torch.cuda.synchronize()
    assert np.array_equal(f64(out[:, :4]), want) and torch.all(out[:, 4:] == 5)


def test_pages_past_32_bits(frq):
    """Bytes 2^32 and on of a cache."""
    page, d = 4096, 256
    pages = (1 << 32) // (page // 32 * 8 * 1152) + 3
    s = Setup([3], [5000], 2, 1, d, page=page, seed=13, spare=pages)
    s.table = s.table.copy()
    big = np.array([[pages + 1, pages]], np.int32)
    t = np.arange(5000)
    s.cache.write(s.k.cuda(), s.v.cuda(), dev(big[0, t // page].astype(np.int64) * page + t % page), 5000)
    s.check(s.run(table=big), heads=[1])


def test_same_bits_on_another_stream_and_in_replays(frq):
    """Split keys: joined in a fixed order. The scratch is the stream's."""
    s, r = Setup([7], [6000], 8, 2, 128, seed=14), Setup([5], [9000], 8, 2, 128, seed=15)
    want, other = s.run(), r.run()
    assert np.array_equal(s.run(stream=torch.cuda.Stream()), want)
    st = device.Stream()
    ops = [(x.q.cuda(), dev(x.table), dev(np.array(x.lens, np.int32)), dev(x.cu), torch.zeros((x.new[0], 8, 128), dtype=torch.bfloat16, device="cuda"))
           for x in (s, r)]
    torch.cuda.synchronize()

    def call(x, o):
        device.attn_chunk(o[0], x.cache, o[1], o[2], o[3], o[4], 1, x.new[0], 8, x.new[0], x.lens[0], stream=st)

    for x, o in zip((s, r), ops):
        call(x, o)
    st.synchronize()
    graphs = []
    for x, o in zip((s, r), ops):
        with device.Graph.capture(st) as g:
            call(x, o)
        graphs.append(g)
    for _ in range(3):
        for o in ops:
            o[4].zero_()
        torch.cuda.synchronize()
        for g in graphs:
            g.launch(st)
        st.synchronize()
        assert np.array_equal(f64(ops[0][4]), want) and np.array_equal(f64(ops[1][4]), other)
    for g in graphs:
        g.destroy()
    st.destroy()


def test_one_token_agrees_with_decode(frq):
    s = Setup([1] * 6, [1, 50, 700, 32, 64, 9], 8, 2, 128, seed=16)
    got, out = s.run(out_dtype="f32"), torch.empty((6, 8, 128), device="cuda")
    device.attn_decode(s.q.float().cuda(), s.cache, dev(s.table), dev(np.array(s.lens, np.int32)), out, 6, 8, 700)
    torch.cuda.synchronize()
    assert np.abs(got - f64(out)).max() <= 4e-3


@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("new", [[2, 5, 8, 10, 13, 16, 0, 1], [1, 4, 12, 7], [30, 1, 17, 31, 9], [3, 8]])
def test_sequences_that_differ_in_rows(frq, hq, hkv, d, new):
    """Column tiles without rows are left out, a sequence at a time: each as it is alone."""
    lens = [n + 150 * i for i, n in enumerate(new)]
    s = Setup(new, lens, hq, hkv, d, page=32, seed=len(new), stale=True)
    s.check(s.run(out_dtype="f32"), out_dtype="f32")


@pytest.mark.parametrize("new,hq", [(3, 4), (37, 8)])
def test_more_sequences_than_lanes(frq, new, hq):
    """Past 64 the blocks go by number, not by length."""
    n = [new - i % 3 for i in range(70)]
    lens = [0 if i == 5 else m + (i * 37) % 211 for i, m in enumerate(n)]
    s = Setup(n, lens, hq, 1, 64, page=32, seed=new, stale=True)
    got = s.run(tail=1)
    s.check(got)
    at = sum(n[:5])
    assert np.all(got[at:at + n[5]] == 0)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 3e4, 3e5])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_and_large_values_of_many_rows(frq, what, size, d):
    x = size * torch.randn((300, 1, d), generator=torch.Generator().manual_seed(6)).clamp(-1.7, 1.7)
    s = Setup([150], [300], 2, 1, d, seed=5, stale=True, **{what: x})
    if what == "k":
        s.q = (s.q.float() / max(size, 1e-3)).to(torch.bfloat16)
    s.check(s.run(out_dtype="f32"), out_dtype="f32")


@pytest.mark.parametrize("size", [1e-30, 1e4, 1e30])
def test_small_and_large_queries_of_many_rows(frq, size):
    s = Setup([140], [200], 4, 2, 64, seed=6)
    s.q = (s.q.float() * size).to(torch.bfloat16)
    s.check(s.run(out_dtype="f32", scale=0.125 / size), out_dtype="f32", scale=0.125 / size)


def test_many_rows_in_replays(frq):
    """Two captured calls share the stream's scratch, the unpacked keys among it: the eager bits every time."""
    st = device.Stream()
    two = [Setup([90, 40], [900, 2000], 8, 2, 128, seed=17), Setup([70], [1500], 8, 2, 64, seed=18)]
    want = [s.run() for s in two]
    held, graphs = [], []

    def call(s, o):
        device.attn_chunk(o[0], s.cache, o[1], o[2], o[3], o[4], len(s.new), sum(s.new), 8, max(s.new), max(s.lens), stream=st)

    for s in two:
        held.append((s.q.cuda(), dev(s.table), dev(np.array(s.lens, np.int32)), dev(s.cu),
                     torch.zeros((sum(s.new), 8, s.d), dtype=torch.bfloat16, device="cuda")))
    torch.cuda.synchronize()
    for s, o in zip(two, held):
        call(s, o)
    st.synchronize()
    for s, o in zip(two, held):
        with device.Graph.capture(st) as g:
            call(s, o)
        graphs.append(g)
    for _ in range(3):
        for o in held:
            o[4].zero_()
        torch.cuda.synchronize()
        for g in graphs:
            g.launch(st)
        st.synchronize()
        assert all(np.array_equal(f64(o[4]), w) for o, w in zip(held, want))
        call(two[0], held[0])
        st.synchronize()
        assert np.array_equal(f64(held[0][4]), want[0])
    for g in graphs:
        g.destroy()
    st.destroy()
