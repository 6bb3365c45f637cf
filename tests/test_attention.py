"""The attention step without a GPU: refusals, the rotary table, pages."""

from __future__ import annotations

import math

import numpy as np
import pytest

from flatrun_amd import _lib, device
from flatrun_amd.attention import KVCache4, Sequence, rope_frequencies, rope_table


class FakeCache:
    """A cache's shape without its memory: for calls that are refused."""
    pages, page_tokens, kv_heads, head_dim, nbytes = 4, 64, 2, 128, 4 * 2 * 2 * 4608

    def data_ptr(self):
        return 0x10000


def rope(**kw):
    a = dict(x=0x10000, q=0x20000, k=0x30000, v=0x40000, tokens=3, q_heads=4, kv_heads=2, head_dim=128, table=0x50000,
             positions=0x60000, n_pos=16)
    a.update(kw)
    device.qk_norm_rope(**a)


def decode(cache=None, **kw):
    a = dict(q=0x10000, cache=cache or FakeCache(), table=0x20000, lens=0x30000, out=0x40000, batch=2, q_heads=4,
             max_len=100)
    a.update(kw)
    device.attn_decode(**a)


def prefill(**kw):
    a = dict(q=0x10000, k=0x20000, v=0x30000, out=0x40000, cu_q=0x50000, cu_k=0x60000, seqs=1, tokens_q=8, tokens_k=8,
             q_heads=4, kv_heads=2, head_dim=128, max_q=8, max_k=8)
    a.update(kw)
    device.attn_prefill(**a)


REFUSED = [
    (rope, dict(x_dtype=7), _lib.ERR_INVALID),
    (rope, dict(q=0), _lib.ERR_INVALID),
    (rope, dict(positions=0), _lib.ERR_INVALID),
    (rope, dict(table=0), _lib.ERR_INVALID),
    (rope, dict(n_pos=0), _lib.ERR_INVALID),
    (rope, dict(eps=-1.0), _lib.ERR_INVALID),
    (rope, dict(eps=float("nan")), _lib.ERR_INVALID),
    (rope, dict(tokens=-1), _lib.ERR_SHAPE),
    (rope, dict(q_heads=0), _lib.ERR_SHAPE),
    (rope, dict(rot=7), _lib.ERR_SHAPE),
    (rope, dict(rot=130), _lib.ERR_SHAPE),
    (rope, dict(ld_x=1000), _lib.ERR_SHAPE),
    (rope, dict(ld_q=508), _lib.ERR_SHAPE),
    (rope, dict(head_dim=100), _lib.ERR_UNSUPPORTED),
    (rope, dict(head_dim=264), _lib.ERR_UNSUPPORTED),
    (rope, dict(x=0x10004), _lib.ERR_ALIGN),
    (rope, dict(ld_x=1025), _lib.ERR_ALIGN),
    (rope, dict(out_dtype="bf16", ld_k=260), _lib.ERR_ALIGN),
    (rope, dict(q_norm=0x10008), _lib.ERR_ALIGN),
    (decode, dict(dtype=2), _lib.ERR_INVALID),
    (decode, dict(scale=0.0), _lib.ERR_INVALID),
    (decode, dict(scale=float("inf")), _lib.ERR_INVALID),
    (decode, dict(q=0), _lib.ERR_INVALID),
    (decode, dict(table=0), _lib.ERR_INVALID),
    (decode, dict(q_heads=5), _lib.ERR_SHAPE),
    (decode, dict(max_len=-1), _lib.ERR_UNSUPPORTED),
    (decode, dict(ld_table=1), _lib.ERR_SHAPE),
    (decode, dict(ld_q=500), _lib.ERR_SHAPE),
    (decode, dict(batch=-1), _lib.ERR_SHAPE),
    (decode, dict(out=0x40008), _lib.ERR_ALIGN),
    (decode, dict(lens=0x30002), _lib.ERR_ALIGN),
    (prefill, dict(dtype="f32"), _lib.ERR_INVALID),
    (prefill, dict(out_dtype="f16"), _lib.ERR_INVALID),
    (prefill, dict(scale=-1.0), _lib.ERR_INVALID),
    (prefill, dict(k=0), _lib.ERR_INVALID),
    (prefill, dict(q_heads=3), _lib.ERR_SHAPE),
    (prefill, dict(max_q=9), _lib.ERR_SHAPE),
    (prefill, dict(max_k=9), _lib.ERR_SHAPE),
    (prefill, dict(hs_k=64), _lib.ERR_SHAPE),
    (prefill, dict(head_dim=96), _lib.ERR_UNSUPPORTED),
    (prefill, dict(ld_v=257), _lib.ERR_ALIGN),
    (prefill, dict(ld_k=1 << 24), _lib.ERR_UNSUPPORTED),
    (prefill, dict(ld_v=1 << 24), _lib.ERR_UNSUPPORTED),
    (prefill, dict(hs_q=132), _lib.ERR_ALIGN),
    (prefill, dict(q=0x10002), _lib.ERR_ALIGN),
]


@pytest.mark.parametrize("call,kw,code", REFUSED, ids=[f"{c[0].__name__}-{i}" for i, c in enumerate(REFUSED)])
def test_refusals(call, kw, code):
    with pytest.raises(_lib.FrqError) as ei:
        call(**kw)
    assert ei.value.code == code


@pytest.mark.parametrize("move", [device.kv4_write, device.kv4_read])
def test_cache_refusals(move):
    c = FakeCache()
    bad = FakeCache()
    bad.nbytes -= 1
    for cache, kw, code in ((bad, {}, _lib.ERR_SIZE), (c, dict(tokens=-1), _lib.ERR_SHAPE), (c, dict(ld_k=200), _lib.ERR_SHAPE),
                            (c, dict(k=0), _lib.ERR_INVALID), (c, dict(slots=0), _lib.ERR_INVALID),
                            (c, dict(v=0x20001), _lib.ERR_ALIGN), (c, dict(slots=0x30004), _lib.ERR_ALIGN)):
        a = dict(k=0x10000, v=0x20000, slots=0x30000, tokens=5)
        a.update(kw)
        with pytest.raises(_lib.FrqError) as ei:
            move(cache, a.pop("k"), a.pop("v"), a.pop("slots"), a.pop("tokens"), **a)
        assert ei.value.code == code


def test_nothing_to_do_needs_no_buffers():
    rope(tokens=0, x=0, q=0, k=0, v=0, positions=0, table=0)
    decode(batch=0, q=0, out=0, lens=0, table=0)
    prefill(seqs=0, q=0, k=0, v=0, out=0, cu_q=0, cu_k=0)
    device.kv4_write(FakeCache(), 0, 0, 0, 0)


def test_wrong_tensors_are_refused_by_type_and_size():
    import torch

    f = torch.zeros(3 * 8 * 128)
    with pytest.raises(TypeError):
        rope(x=f.half())
    with pytest.raises(ValueError):
        rope(x=torch.zeros(3 * 8 * 128 - 1))
    with pytest.raises(ValueError):
        rope(x_dtype="q8")
    with pytest.raises(TypeError):
        rope(positions=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        decode(lens=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        prefill(out=torch.zeros((8, 4, 127), dtype=torch.bfloat16))


@pytest.mark.parametrize("pages,page,heads,d", [(0, 64, 2, 128), (3, 32, 1, 64), (5, 256, 8, 256)])
def test_cache_bytes(pages, page, heads, d):
    assert device.kv4_bytes(pages, page, heads, d) == pages * page * heads * 2 * (d // 2 + d // 32 * 2)


@pytest.mark.parametrize("args", [(-1, 64, 2, 128), (1, 48, 2, 128), (1, 0, 2, 128), (1, 64, 0, 128), (1, 64, 2, 96)])
def test_cache_shapes_refused(args):
    with pytest.raises(_lib.FrqError):
        device.kv4_bytes(*args)


def test_large_cache_needs_64_bits():
    assert device.kv4_bytes(1 << 16, 256, 8, 128) == (1 << 16) * 256 * 8 * 144


def test_rope_table():
    t = rope_table(64, 131072, base=500000.0)
    assert t.shape == (131072, 32, 2) and t.dtype == np.float32
    for p, i in ((0, 0), (1, 0), (131071, 0), (131071, 31), (77777, 13)):
        a = p * 500000.0 ** (-2 * i / 64)
        assert abs(t[p, i, 0] - math.cos(a)) <= 2 ** -24 and abs(t[p, i, 1] - math.sin(a)) <= 2 ** -24


def test_rope_scaling():
    plain, one = rope_frequencies(128, 500000.0)
    assert one == 1.0 and plain[0] == 1.0
    lin, one = rope_frequencies(128, 500000.0, {"kind": "linear", "factor": 4})
    assert one == 1.0 and np.array_equal(lin, plain / 4)
    sc = {"kind": "bands", "factor": 8, "low": 1, "high": 4, "trained": 8192}
    bands, one = rope_frequencies(128, 500000.0, sc)
    turns = 8192 * plain / (2 * math.pi)
    assert one == 1.0
    assert np.array_equal(bands[turns >= 4], plain[turns >= 4])
    assert np.allclose(bands[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and np.all(bands[mid] < plain[mid]) and np.all(bands[mid] > plain[mid] / 8)
    ramp, f = rope_frequencies(128, 10000.0, {"kind": "ramp", "factor": 4, "fast": 32, "slow": 1, "trained": 4096})
    base, _ = rope_frequencies(128, 10000.0)
    assert f == 0.1 * math.log(4) + 1.0
    assert np.array_equal(ramp[:16], base[:16]) and np.allclose(ramp[-8:], base[-8:] / 4, rtol=1e-15)
    assert np.all(np.diff(ramp) < 0)
    for bad in ({"kind": "other", "factor": 2}, {"kind": "linear", "factor": 0.5},
                {"kind": "bands", "factor": 2, "low": 4, "high": 1, "trained": 10}):
        with pytest.raises(ValueError):
            rope_frequencies(64, 1e4, bad)
    with pytest.raises(ValueError):
        rope_frequencies(63)


def test_pages(monkeypatch):
    class NoMemory:
        def __init__(self, nbytes):
            self.nbytes, self.ptr = nbytes, 0

        def free(self):
            pass

    monkeypatch.setattr(device, "DeviceBuffer", NoMemory)
    c = KVCache4(3, 32, 1, 64)
    a = c.take(2)
    assert sorted(a + c.take()) == [0, 1, 2]
    with pytest.raises(_lib.FrqError):
        c.take()
    c.give(a)
    with pytest.raises(ValueError):
        c.give(a[:1])
    with pytest.raises(ValueError):
        c.give([7])
    assert sorted(c.take(2)) == sorted(a)
    s = Sequence()
    assert s.pages == [] and s.length == 0
