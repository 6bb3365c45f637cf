"""The 4-bit cache: what is read back equals the block's definition, bit for
bit, at every place of a page, and nothing else in the cache changes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import TORCH, block4, dev, f64
from flatrun_amd.attention import KVCache4

pytestmark = pytest.mark.gpu


def heads(tokens, h, d, src, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((tokens, h, d), generator=g) * torch.exp(2 * torch.randn((1, h, d), generator=g))).to(TORCH[src])


def read(c, slots, out="f32"):
    n = len(slots)
    k, v = (torch.full((n, c.kv_heads, c.head_dim), 9.0, dtype=TORCH[out], device="cuda") for _ in range(2))
    c.read(k, v, dev(np.asarray(slots, np.int64)), n, dtype=out)
    torch.cuda.synchronize()
    return k, v


@pytest.mark.parametrize("tokens,h,d,page,src", [(1, 1, 64, 32, "f32"), (45, 2, 64, 32, "bf16"), (130, 8, 128, 64, "f32"),
                                                 (96, 3, 256, 96, "f16"), (1027, 4, 128, 256, "bf16")])
def test_round_trip(frq, tokens, h, d, page, src):
    pages = 2 * -(-tokens // page) + 1
    c = KVCache4(pages, page, h, d)
    rng = np.random.default_rng(tokens)
    slots = rng.permutation(pages * page)
    c.write(*(x.cuda() for x in (heads(len(slots), h, d, "f32", 5), heads(len(slots), h, d, "f32", 6))),
            dev(slots.astype(np.int64)), len(slots))
    before = read(c, np.arange(pages * page))
    some = slots[:tokens]
    k, v = heads(tokens, h, d, src, 7), heads(tokens, h, d, src, 8)
    c.write(k.cuda(), v.cuda(), dev(some.astype(np.int64)), tokens, dtype=src)
    for got, x in zip(read(c, some), (k, v)):
        assert np.array_equal(f64(got), block4(f64(x)))
    after = read(c, np.arange(pages * page))
    rest = np.setdiff1d(np.arange(pages * page), some)
    for a, b in zip(after, before):
        assert torch.equal(a[rest], b[rest])
    for out in ("f16", "bf16"):
        for got, full in zip(read(c, some, out), read(c, some)):
            assert torch.equal(got, full.to(TORCH[out]))


def test_appending_a_token_at_a_time_equals_writing_at_once(frq):
    n, h, d, page = 70, 2, 128, 64
    k, v = heads(n, h, d, "f32", 1), heads(n, h, d, "f32", 2)
    slots = np.concatenate([np.arange(64, 128), np.arange(6)])       # page 1, then page 0
    one, all_ = KVCache4(2, page, h, d), KVCache4(2, page, h, d)
    all_.write(k.cuda(), v.cuda(), dev(slots), n)
    for i in range(n):
        one.write(k[i:i + 1].cuda(), v[i:i + 1].cuda(), dev(slots[i:i + 1]), 1)
    for a, b in zip(read(one, slots), read(all_, slots)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("start,n,page", [(0, 320, 32), (64, 300, 64), (13, 299, 96), (32, 257, 256)])
@pytest.mark.parametrize("d,src", [(64, "f32"), (128, "bf16"), (256, "f16")])
def test_runs_of_slots(frq, start, n, page, d, src):
    """Prompts: slots one after another, from a tile's start and from within."""
    h, pages = 2, -(-(start + n) // page) + 1
    c = KVCache4(pages, page, h, d)
    fill = heads(pages * page, h, d, "f32", 3)
    c.write(fill.cuda(), fill.cuda(), dev(np.arange(pages * page)), pages * page)
    k, v = heads(n, h, d, src, 4), heads(n, h, d, src, 5)
    slots = np.arange(start, start + n)
    c.write(k.cuda(), v.cuda(), dev(slots), n, dtype=src)
    one = [np.concatenate([f64(x) for x in part]) for part in zip(*(read(c, [i]) for i in range(pages * page)))]
    want = [block4(f64(fill)) for _ in range(2)]
    for w, x in zip(want, (k, v)):
        w[start:start + n] = block4(f64(x))
    for a, b, w in zip(one, read(c, np.arange(pages * page)), want):
        assert np.array_equal(a, w) and np.array_equal(f64(b), w)
    for a, w in zip(read(c, slots), want):
        assert np.array_equal(f64(a), w[start:start + n])


def test_edges(frq):
    x = torch.zeros((12, 1, 64))
    x[0, 0, 3], x[0, 0, 9] = 5.0, -5.0             # the first of equals gives the sign
    x[1, 0, 3], x[1, 0, 9] = -5.0, 5.0
    x[2, 0, :32] = 1e-30                           # the scale underflows: zeros
    x[3, 0, 0] = 3e38                              # the scale is held at 65504
    x[4, 0, 0] = float("nan")
    x[5, 0, 40] = float("-inf")
    x[6] = -0.0
    x[7, 0, :32] = torch.linspace(-8, 8, 32)       # codes on their ties
    x[8, 0, :32] = torch.arange(32) * 0.25 - 4
    x[9, 0, 31] = 2.0 ** -22                       # a subnormal scale
    x[10, 0, 0], x[10, 0, 31] = 1.0, -1.0          # equals in different lanes
    x[11, 0, 7], x[11, 0, 8] = -1.0, 1.0
    c = KVCache4(1, 32, 1, 64)
    slots = np.arange(12)
    c.write(x.cuda(), (-x).cuda(), dev(slots), 12)
    k, v = read(c, slots)
    fine = [i for i in range(12) if i not in (4, 5)]
    assert np.array_equal(f64(k)[fine], block4(f64(x))[fine])
    assert np.array_equal(f64(v)[fine], block4(-f64(x))[fine])
    for t in (k, v):
        assert torch.isnan(t[4, 0, :32]).all() and (t[4, 0, 32:] == 0).all()
        assert torch.isnan(t[5, 0, 32:]).all() and (t[5, 0, :32] == 0).all()


def test_slots_outside_the_cache(frq):
    c = KVCache4(2, 32, 1, 64)
    k = heads(64, 1, 64, "f32", 3)
    c.write(k.cuda(), k.cuda(), dev(np.arange(64)), 64)
    before = read(c, np.arange(64))
    c.write(k[:3].cuda(), k[:3].cuda(), dev(np.array([-1, 64, 1 << 40])), 3)
    for a, b in zip(read(c, np.arange(64)), before):
        assert torch.equal(a, b)
    for t in read(c, np.array([-1, 64, 5, -(1 << 40)])):
        assert (t[0] == 0).all() and torch.isnan(t[1]).all() and torch.equal(t[2], before[0][5]) and (t[3] == 0).all()


def test_strided_rows_on_a_stream(frq):
    n, h, d, ld = 40, 2, 64, 512
    rows = torch.randn((n, ld))
    cu = rows.cuda()
    c = KVCache4(2, 32, h, d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    slots = dev(np.arange(n))
    s.wait_stream(torch.cuda.current_stream())
    c.write(cu, cu.data_ptr() + 4 * 256, slots, n, ld_k=ld, ld_v=ld, stream=s)
    back = torch.full((n, ld), 3.0, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    c.read(back, back.data_ptr() + 4 * 256, slots, n, ld_k=ld, ld_v=ld, stream=s)
    s.synchronize()
    assert np.array_equal(f64(back)[:, :128], block4(f64(rows)[:, :128]))
    assert np.array_equal(f64(back)[:, 256:384], block4(f64(rows)[:, 256:384]))
    assert (back[:, 128:256] == 3).all() and (back[:, 384:] == 3).all()


def test_offsets_past_32_bits(frq):
    """A cache of 5 GiB: slots at its end lie past 2^32 bytes."""
    c = KVCache4(1200, 4096, 8, 128)
    assert c.nbytes > 5 << 30
    slots = np.array([0, 1200 * 4096 - 1, 1100 * 4096 + 33, 7], np.int64)
    k, v = heads(4, 8, 128, "f32", 1), heads(4, 8, 128, "f32", 2)
    c.write(k.cuda(), v.cuda(), dev(slots), 4)
    for got, x in zip(read(c, slots), (k, v)):
        assert np.array_equal(f64(got), block4(f64(x)))
    c.close()
