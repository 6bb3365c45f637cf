"""BlockAttention on host memory: plans, pages, buffers and the order of its
calls, every row of every step against 64-bit attention over all that its
sequence has seen. What the cache rounds (4 bits, a prompt's heads to bf16
before) is rounded in the reference too; the heads that a prompt attends with
are given their rounding."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_host import Buffer, Stream, host, view    # noqa: F401  (host: fixture)
from attn_ref import attend, block4, rope
from flatrun_amd import _lib, device
from flatrun_amd.attention import BlockAttention, KVCache4, Sequence, rope_table

HQ, HKV, D = 4, 2, 64
WIDTH = (HQ + 2 * HKV) * D


class Model:
    """Layers of random q|k|v rows and what each has to answer."""

    def __init__(self, layers=1, pages=12, page=32, max_rows=160, max_seqs=4, max_context=200, n_pos=256):
        rng = np.random.default_rng(layers)
        self.table = rope_table(D, n_pos)
        self.norms = [[(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)] for _ in range(layers)]
        self.rng, self.seen = rng, [{} for _ in range(layers)]
        self.stream, self.steps, self.caches = Stream(), [], []
        kw = dict(max_rows=max_rows, max_seqs=max_seqs, max_context=max_context, stream=self.stream)
        up = device.DeviceBuffer.from_host
        for wq, wk in self.norms:
            self.caches.append(KVCache4(pages, page, HKV, D))
            more = {"first": self.steps[0]} if self.steps else kw
            self.steps.append(BlockAttention(self.caches[-1], HQ, up(self.table), n_pos, q_norm=up(wq), k_norm=up(wk), **more))

    def step(self, new, **kw):
        start = {s: s.length for s in new}
        self.steps[0].plan(new, **kw)
        n = sum(new.values())
        for i, one in enumerate(self.steps):
            qkv = self.rng.standard_normal((n, WIDTH)).astype(np.float32)
            got = one(device.DeviceBuffer.from_host(qkv), n).to_host(np.float32)[:n * HQ * D].reshape(n, HQ, D)
            self.check(i, new, start, qkv.reshape(n, -1, D), got)

    def check(self, layer, new, start, x, got):
        at, context = 0, any(start[s] and n > 1 for s, n in new.items())
        for s, n in new.items():
            pos = np.arange(start[s], start[s] + n)
            (q, k, v), _ = rope(x[at:at + n], HQ, HKV, D, D, False, self.table[pos], *self.norms[layer])
            one = n == 1
            if not one:                         # a prompt's heads are bf16, in the cache too
                k, v = (torch.as_tensor(np.float32(a)).bfloat16().double().numpy() for a in (k, v))
            kv = self.seen[layer].setdefault(s, [np.zeros((0, HKV, D))] * 2)
            kv[:] = [np.concatenate([a, b]) for a, b in zip(kv, (k, v))]
            for h in range(HQ):
                g = h // (HQ // HKV)
                kk, vv = ([block4(np.float32(a)) for a in kv] if one or context else kv)
                want, mag, _ = attend(q[:, h], kk[:, g], vv[:, g], D ** -0.5, pos)
                # one token: fp32 heads against the cache's own values. A prompt: q and what the cache reads back
                # rounded to bf16, some 2^-9.5 in the mean of scores of some units and of the values
                err = np.linalg.norm(got[at:at + n, h] - want) / np.linalg.norm(mag)
                assert err <= (2.0 ** -18 if one else 1.2e-2), (layer, n, start[s], h, err)
            at += n


@pytest.mark.parametrize("chunks", [(45, 40), (2, 3), (33, 64, 4), (31, 7)])
def test_chunks_of_any_total(host, chunks):
    """A chunk's context and new keys together may be an odd number."""
    m, s = Model(), Sequence()
    for n in chunks:
        m.step({s: n})
    assert s.length == sum(chunks) and len(s.pages) == -(-s.length // 32)


def test_a_context_buffer_that_grows(host):
    m = Model()
    a, b = Sequence(), Sequence()
    m.step({a: 3, b: 6})
    m.step({a: 4, b: 2})
    m.step({b: 97, a: 12, Sequence(): 21})     # one that the cache held nothing of reads it back too


def test_layers_share_a_plan(host):
    """A prompt, a chunk and single tokens through three layers, each with its own cache; one plan a step."""
    m = Model(layers=3)
    a, b = Sequence(), Sequence()
    for i, new in enumerate(({a: 45, b: 7}, {a: 40}, {a: 1, b: 1}, {b: 30, a: 2}, {a: 1, b: 1})):
        m.step(new)
        assert m.stream.waits == i + 1
    assert (a.length, b.length) == (89, 39) and (len(a.pages), len(b.pages)) == (3, 2)
    assert len(set(a.pages + b.pages)) == 5 and len(m.caches[0]._free) == 12 - 5


def test_a_sequence_has_one_planner(host):
    """Layers that each plan a sequence would advance it twice: refused, nothing changed."""
    m, s = Model(), Sequence()
    table = device.DeviceBuffer.from_host(m.table)
    other = BlockAttention(KVCache4(12, 32, HKV, D), HQ, table, 256, max_rows=160, max_seqs=4, max_context=200,
                           stream=m.stream)
    m.step({s: 40})
    pages = list(s.pages)
    with pytest.raises(ValueError):
        other.plan({Sequence(): 2, s: 1})
    assert s.length == 40 and s.pages == pages and len(other.cache._free) == 12
    more = BlockAttention(KVCache4(12, 32, HKV, D), HQ, table, 256, first=m.steps[0])
    with pytest.raises(ValueError):
        more.plan({s: 1})
    m.step({s: 1})
    for cache, kw in ((KVCache4(11, 32, HKV, D), {}), (KVCache4(12, 64, HKV, D), {}), (KVCache4(12, 32, 1, D), {}),
                      (m.caches[0], {}), (KVCache4(12, 32, HKV, D), dict(stream=7)),
                      (KVCache4(12, 32, HKV, D), dict(max_rows=10)), (KVCache4(12, 32, HKV, D), dict(first=more))):
        with pytest.raises(ValueError):
            BlockAttention(cache, HQ, table, 256, **{"first": m.steps[0], **kw})
    with pytest.raises(ValueError):
        BlockAttention(KVCache4(12, 32, HKV, D), HQ, table, 256)


MIXED = [(0, 1, 30, 1), (1, 30, 1, 1), (30, 1, 1, 12), (1, 1, 1, 9)]


@pytest.mark.parametrize("past", [(40, 33, 0, 5), (0, 40, 31, 0), (2, 2, 2, 2)])
@pytest.mark.parametrize("new", MIXED)
def test_single_tokens_beside_prompts(host, past, new):
    """fp32 and the cache for single tokens, bf16 for prompts, whatever stands beside them and in which order."""
    m, seqs = Model(layers=2, max_rows=200), [Sequence() for _ in past]
    for s, n in zip(seqs, past):
        if n:
            m.step({s: n})
    m.step({s: n for s, n in zip(seqs, new) if n})
    m.step({s: 1 for s in seqs})


def test_a_tokens_result_does_not_depend_on_its_neighbours(host):
    rng = np.random.default_rng(5)
    x = [rng.standard_normal((n, WIDTH)).astype(np.float32) for n in (45, 1, 1, 30)]
    got = []
    for beside in (False, True):
        m, a, b = Model(), Sequence(), Sequence()
        outs = []
        for i in range(3):
            new, at, qkv = {a: len(x[i])}, 0, x[i]
            if beside and i:
                new, qkv, at = ({b: 30, a: 1}, np.concatenate([x[3], x[i]]), 30)
            m.steps[0].plan(new)
            out = m.steps[0](device.DeviceBuffer.from_host(qkv), len(qkv)).to_host(np.float32)
            outs.append(out[at * HQ * D:len(qkv) * HQ * D])
        store = host.held[m.caches[0]]
        got.append(outs + [np.stack(store[a.pages[t // 32] * 32 + t % 32]) for t in range(47)])
    assert all(np.array_equal(p, q) for p, q in zip(*got))


def test_launches_of_a_step(host):
    """Single tokens side by side go together; a step of one kind has no launch of the other."""
    m, seqs = Model(), [Sequence() for _ in range(4)]
    m.step({seqs[0]: 3, seqs[1]: 5})
    assert [c[0] for c in host.calls] == ["rope", "write", "prefill"]
    host.calls.clear()
    m.step({s: 1 for s in seqs})
    assert [c[0] for c in host.calls] == ["rope", "write", "decode"] and host.calls[-1][1] == 4
    host.calls.clear()
    m.step({seqs[0]: 1, seqs[1]: 1, seqs[2]: 4, seqs[3]: 1})
    assert [c[0] for c in host.calls] == ["rope", "write", "read", "prefill"] + ["rope", "write", "decode"] * 2
    assert [c[1] for c in host.calls if c[0] == "decode"] == [2, 1] and host.calls[3][3] == 5    # keys: the prompt's only


def test_the_length_that_a_captured_step_is_made_for(host):
    m, s = Model(), Sequence()
    m.step({s: 40})
    m.step({s: 1})
    assert host.calls[-1][:3] == ("decode", 1, 41)
    m.step({s: 1}, max_len=200)
    assert host.calls[-1][:3] == ("decode", 1, 200)
    for bad in (42, 201, 0, -1):
        with pytest.raises(ValueError):
            m.steps[0].plan({s: 1}, max_len=bad)
    assert s.length == 42


def test_a_stream_given_by_its_handle(host):
    table = device.DeviceBuffer.from_host(rope_table(D, 64))
    step = BlockAttention(KVCache4(2, 32, HKV, D), HQ, table, 64, max_rows=8, max_seqs=2, max_context=64, stream=7)
    more = BlockAttention(KVCache4(2, 32, HKV, D), HQ, table, 64, first=step)
    step.plan({Sequence(): 3})
    assert more.stream == 7 and _lib.lib().waits == [7]
