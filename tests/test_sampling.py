"""Sampler, Residual and BlockAttention(direct=True) without a GPU: what they
refuse, and the order and arguments of their calls."""

from __future__ import annotations

import numpy as np
import pytest

from attn_host import Buffer, Lib, Stream, host, view    # noqa: F401  (host: fixture)
from flatrun_amd import _lib, device
from flatrun_amd.attention import BlockAttention, KVCache4, Sequence, rope_table
from flatrun_amd.layer import Residual
from flatrun_amd.sampling import Sampler


@pytest.fixture
def calls(monkeypatch):
    made, lib = [], Lib(_lib.lib())
    monkeypatch.setattr(device, "DeviceBuffer", Buffer)
    monkeypatch.setattr(device, "synchronize", lambda: made.append("wait"))
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(device, "add_rms_norm", lambda *a, **kw: made.append((a, kw)))
    monkeypatch.setattr(device, "sample", lambda *a, **kw: made.append((a, kw)))
    return made


def test_sampler_parameters(calls):
    s = Sampler(1000, max_rows=3)
    s.plan([dict(temperature=0.5, top_k=7), dict()])
    tokens = s("logits", "u", 2, ld=1024)
    assert calls[0] == "wait" and tokens is s.tokens
    a, kw = calls[1]
    assert a == ("logits", "u", s.tokens, 2, 1000) and kw["ld"] == 1024 and kw["probs"] is s.probs
    for name, dtype, want in (("temperature", np.float32, [0.5, 1]), ("top_k", np.int32, [7, 0]), ("top_p", np.float32, [1, 1]),
                              ("min_p", np.float32, [0, 0])):
        assert view(kw[name].data_ptr(), 2, dtype).tolist() == want
    with pytest.raises(ValueError):
        s("logits", "u", 3)
    for bad in ([], [{}] * 4, [dict(topk=3)], [dict(temperature=-1)], [dict(temperature=float("nan"))], [dict(top_k=-1)],
                [dict(top_p=1.5)], [dict(min_p=-0.1)]):
        with pytest.raises(ValueError):
            s.plan(bad)
    assert s.rows == 2
    for kw in (dict(vocab=0), dict(vocab=5, max_rows=0)):
        with pytest.raises(ValueError):
            Sampler(**kw)


def test_sampler_waits_for_its_stream(calls):
    s = Sampler(10, stream=7)
    s.plan([{}])
    assert _lib.lib().waits == [7]
    one = Stream()
    Sampler(10, stream=one).plan([{}])
    assert one.waits == 1


def test_residual(calls):
    r = Residual(64, max_rows=5, eps=1e-5)
    with pytest.raises(ValueError):
        r.add("d", "w", 2)
    assert r.start("x", "w0", 5) is r.xn and r.add("d", "w1", 5) is r.xn
    assert calls[0] == (("x", r.xn, 5, 64), dict(weight="w0", eps=1e-5, stream=None))
    assert calls[1] == (("d", r.xn, 5, 64), dict(weight="w1", eps=1e-5, stream=None, residual="x", sum_out="x"))
    for rows in (0, 6):
        with pytest.raises(ValueError):
            r.add("d", "w", rows)
    with pytest.raises(ValueError):
        Residual(0)


HQ, HKV, D = 4, 2, 64


def test_chunks_straight_from_the_cache(host, monkeypatch):
    """One launch for the chunks of a step; single tokens beside them have no tokens there."""
    made = []

    def chunk(q, cache, table, lens, cu_q, out, seqs, tokens_q, q_heads, max_q, max_len, dtype="bf16", out_dtype=None, ld_table=0,
              stream=None):
        made.append((seqs, tokens_q, q_heads, max_q, max_len, dtype, out_dtype, ld_table, view(lens, seqs, np.int32).tolist(),
                     view(cu_q, seqs + 1, np.int32).tolist(), np.lib.stride_tricks.as_strided(
                         view(table, seqs * ld_table, np.int32), (seqs, ld_table), (4 * ld_table, 4))[:, :4].tolist()))

    monkeypatch.setattr(device, "attn_chunk", chunk)
    table = device.DeviceBuffer.from_host(rope_table(D, 256))
    new = lambda **kw: BlockAttention(KVCache4(12, 32, HKV, D), HQ, table, 256, **kw)    # noqa: E731
    first = new(max_rows=100, max_seqs=3, max_context=200, stream=Stream(), direct=True)
    more = new(first=first)
    a, b, c = Sequence(), Sequence(), Sequence()

    def step(plan):
        first.plan(plan)
        host.calls.clear()
        made.clear()
        n = sum(plan.values())
        for one in (first, more):
            one(device.DeviceBuffer.from_host(np.zeros((n, (HQ + 2 * HKV) * D), np.float32)), n)
        return [x[0] for x in host.calls]

    assert step({a: 45, b: 7}) == ["rope", "write", "prefill"] * 2 and not made
    assert step({a: 40, b: 1, c: 3}) == ["rope", "write", "rope", "write", "decode"] * 2
    want = (3, 44, HQ, 40, 85, "bf16", "f32", 7, [85, 0, 3], [0, 40, 41, 44],
            [(a.pages + [0] * 4)[:4], (b.pages + [0] * 4)[:4], (c.pages + [0] * 4)[:4]])
    assert made == [want, want]
    assert step({a: 1, b: 1}) == ["rope", "write", "decode"] * 2 and not made
    with pytest.raises(ValueError):
        new(first=first, direct=True)
