"""BlockAttention over layers, chunks and mixed steps, on the values that each
layer's cache reads back.

Bounds. Single tokens, fp32: attn_ref.fp32_bound, and q's own error of 20 *
2^-24 of its pair (test_gpu_rope) in every score, on both sides of the
division. Prompts: q, keys, values and weights rounded to bf16, at most 2^-8 and
some 2^-9.5 in the mean each: 1.2e-2 normwise. A value of the cache is within its
block's scale (largest / 8) of the head, where the scale is off by the largest's
rounding to bf16 (2^-8) and its own to fp16 (2^-11), both up to 8 times."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from attn_ref import attend, dev, f64, fp32_bound, rope
from flatrun_amd import _lib, device
from flatrun_amd.attention import BlockAttention, KVCache4, Sequence, rope_table

pytestmark = pytest.mark.gpu

HQ, HKV, D = 8, 2, 64
WIDTH = (HQ + 2 * HKV) * D


def upload(buf, host):
    _lib.check(_lib.lib().frq_memcpy_h2d(buf.ptr, host.ctypes.data, host.nbytes))


def cached(cache, seq):
    t = np.arange(seq.length)
    slots = np.array(seq.pages)[t // cache.page_tokens] * cache.page_tokens + t % cache.page_tokens
    k, v = (torch.zeros((len(t), HKV, D), device="cuda") for _ in range(2))
    cache.read(k, v, dev(slots.astype(np.int64)), len(t))
    torch.cuda.synchronize()
    return f64(k), f64(v)


def bf16(a):
    return torch.as_tensor(np.asarray(a, np.float32)).bfloat16().double().numpy()


@pytest.mark.parametrize("page", [32, 96])
def test_layers_chunks_and_mixed_steps(frq, page):
    rng = np.random.default_rng(page)
    stream, table = device.Stream(), rope_table(D, 512)
    up = device.DeviceBuffer.from_host
    caches = [KVCache4(24, page, HKV, D) for _ in range(2)]
    norms = [[(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)] for _ in caches]
    first = dict(max_rows=128, max_seqs=3, max_context=300, stream=stream)
    steps = []
    for c, (wq, wk) in zip(caches, norms):
        steps.append(BlockAttention(c, HQ, up(table), 512, q_norm=up(wq), k_norm=up(wk),
                                    **({"first": steps[0]} if steps else first)))
    a, b, c = (Sequence() for _ in range(3))
    qkv = device.DeviceBuffer(4 * 128 * WIDTH)
    for new in ({a: 45, b: 7}, {a: 40, c: 33}, {b: 1, a: 1, c: 1}, {c: 1, a: 60, b: 1}, {b: 90, c: 1}, {a: 1, b: 1},
                {a: 128}, {a: 1, c: 2}, {c: 1, b: 1}):
        rows, start = sum(new.values()), {s: s.length for s in new}
        context = any(start[s] and n > 1 for s, n in new.items())      # a chunk: the step's prompts read the cache
        steps[0].plan(new)
        for step, cache, (wq, wk) in zip(steps, caches, norms):
            x = rng.standard_normal((rows, WIDTH)).astype(np.float32)
            upload(qkv, x)
            got = step(qkv, rows)
            stream.synchronize()
            got, x = got.to_host(np.float32)[:rows * HQ * D].reshape(rows, HQ, D), x.reshape(rows, -1, D)
            at = 0
            for s, n in new.items():
                pos = np.arange(start[s], s.length)
                (q, k, v), (size_q, _, _) = rope(x[at:at + n], HQ, HKV, D, D, False, table[pos], wq, wk)
                ck, cv = cached(cache, s)
                for held, fresh in ((ck[start[s]:], k), (cv[start[s]:], v)):
                    top = np.abs(fresh.reshape(n, HKV, -1, 32)).max(-1, keepdims=True)
                    err = np.abs(held - fresh).reshape(n, HKV, -1, 32)
                    assert np.all(err <= top / 8 * (1 + 8 * (2.0 ** -8 + 2.0 ** -11) * (1 + 2.0 ** -7))), (new, n)
                kk, vv = (ck, cv) if n == 1 or context else (bf16(k), bf16(v))
                for h in range(HQ):
                    g = h // (HQ // HKV)
                    want, mag, size = attend(q[:, h], kk[:, g], vv[:, g], D ** -0.5, pos)
                    err = np.abs(got[at:at + n, h] - want)
                    if n == 1:
                        pair = (np.abs(kk[:, g]) * size_q[0, h]).sum(-1).max() * D ** -0.5
                        tol = fp32_bound(mag, size, len(kk), D) + 2 * 20 * 2.0 ** -24 * pair * mag
                        assert np.all(err <= tol), (n, start[s], h, float((err / tol).max()))
                    else:
                        assert np.linalg.norm(err) <= 1.2e-2 * np.linalg.norm(mag), (n, start[s], h)
                at += n
    steps[0].close()
    for cache in caches:
        cache.close()


def test_a_captured_step_of_single_tokens(frq):
    """Captured once, replayed after later plans while the sequences grow: the eager step's bits every time."""
    cache, stream = KVCache4(60, 32, HKV, D), device.Stream()
    table = device.DeviceBuffer.from_host(rope_table(D, 2048))
    step = BlockAttention(cache, HQ, table, 2048, max_rows=96, max_seqs=2, max_context=1600, stream=stream)
    seqs = [Sequence(), Sequence()]
    qkv = device.DeviceBuffer(4 * 96 * WIDTH)
    rng = np.random.default_rng(1)
    upload(qkv, rng.standard_normal(67 * WIDTH).astype(np.float32))
    step.plan({seqs[0]: 60, seqs[1]: 7})
    step(qkv, 67)
    stream.synchronize()
    graph = None
    for i in range(70):                                      # over two page ends, the longest from 61 to 130
        upload(qkv, rng.standard_normal(2 * WIDTH).astype(np.float32))
        step.plan({s: 1 for s in seqs}, max_len=1600)
        if graph is None:
            step(qkv, 2)                                     # the scratch of this shape is there
            stream.synchronize()
            with device.Graph.capture(stream) as graph:
                step(qkv, 2)
        graph.launch(stream)
        stream.synchronize()
        got = step.out.to_host(np.float32)[:2 * HQ * D]
        step(qkv, 2)
        stream.synchronize()
        assert np.isfinite(got).all() and np.array_equal(got, step.out.to_host(np.float32)[:2 * HQ * D]), i
    assert seqs[0].length == 130
    graph.destroy()
    step.close()
    cache.close()
