"""The attention step's operators on host memory, so that what BlockAttention
does around its kernels runs without a GPU: buffers are host arrays, a call
checks what its entry point checks of addresses and computes the 64-bit form."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from attn_ref import TORCH, attend, block4, rope
from flatrun_amd import _lib, device

SIZE = {"f32": 4, "f16": 2, "bf16": 2}


class Buffer:
    """device.DeviceBuffer in host memory, filled with what nobody wrote."""

    def __init__(self, nbytes):
        self.nbytes = int(nbytes)
        self._raw = np.full(self.nbytes + 256, 0xFF, np.uint8)          # NaN in every type
        self.ptr = -(-self._raw.ctypes.data // 256) * 256

    @classmethod
    def from_host(cls, arr, stream=None):
        a = np.ascontiguousarray(arr)
        b = cls(a.nbytes)
        ctypes.memmove(b.ptr, a.ctypes.data, a.nbytes)
        return b

    def to_host(self, dtype=np.uint8, count=None):
        n = self.nbytes // np.dtype(dtype).itemsize if count is None else count
        return view(self.ptr, n, dtype).copy()

    def free(self):
        pass

    def data_ptr(self):
        return self.ptr


def view(ptr, count, dtype=np.float32):
    n = int(count) * np.dtype(dtype).itemsize
    return np.frombuffer((ctypes.c_uint8 * max(n, 1)).from_address(ptr), np.uint8, n).view(dtype)


def rows(obj, count, ld, width, dtype):
    """The rows of an operand as a tensor that shares its memory (16-byte aligned, as the entry points demand)."""
    p = device._addr(obj)
    assert p % 16 == 0 and ld * SIZE[dtype] % 16 == 0, (hex(p), ld)
    raw = torch.from_numpy(view(p, (count - 1) * ld + width, np.float32 if dtype == "f32" else np.int16))
    return torch.as_strided(raw if dtype == "f32" else raw.view(TORCH[dtype]), (count, width), (ld, 1))


class Lib:
    """The library with the calls that need a GPU replaced."""

    def __init__(self, real):
        self._real, self.waits = real, []

    def __getattr__(self, name):
        return getattr(self._real, name)

    def frq_memcpy_h2d(self, dst, src, n):
        ctypes.memmove(dst, src, n)
        return 0

    def frq_stream_synchronize(self, handle):
        self.waits.append(handle)
        return 0


class Stream:
    waits, cuda_stream = 0, 5

    def synchronize(self):
        self.waits += 1


class Host:
    """Calls in the order in which they were made: (name, arguments that matter)."""

    def __init__(self):
        self.calls = []
        self.held = {}                          # cache -> {slot: (k, v)}

    def rope(self, x, q, k, v, tokens, q_heads, kv_heads, head_dim, table, positions, rot=None, interleaved=False,
             q_norm=None, k_norm=None, eps=1e-6, x_dtype="f32", out_dtype="f32", ld_x=0, ld_q=0, ld_k=0, ld_v=0,
             n_pos=None, stream=None):
        d, nq, nk = head_dim, q_heads * head_dim, kv_heads * head_dim
        heads = q_heads + (1 if v is None else 2) * kv_heads
        rot = d if rot is None else rot
        xs = rows(x, tokens, ld_x or heads * d, heads * d, x_dtype).double().numpy().reshape(tokens, heads, d)
        at = view(device._addr(positions), tokens, np.int32)
        assert at.min() >= 0 and at.max() < n_pos
        cs = view(device._addr(table), n_pos * rot).reshape(n_pos, rot // 2, 2)[at]
        w = [None if a is None else view(device._addr(a), d) for a in (q_norm, k_norm)]
        out, _ = rope(xs, q_heads, kv_heads, d, rot, interleaved, cs, *w, eps)
        for dst, ld, width, y in ((q, ld_q, nq, out[0]), (k, ld_k, nk, out[1]), (v, ld_v, nk, out[2])):
            if dst is not None:
                rows(dst, tokens, ld or width, width, out_dtype).copy_(torch.from_numpy(y.reshape(tokens, width)))
        self.calls.append(("rope", tokens, q_heads, kv_heads, out_dtype))

    def write(self, cache, k, v, slots, tokens, dtype="f32", ld_k=0, ld_v=0, stream=None):
        w = cache.kv_heads * cache.head_dim
        at = view(device._addr(slots), tokens, np.int64)
        assert len(set(at)) == tokens
        kk, vv = (rows(a, tokens, ld or w, w, dtype).float().numpy().reshape(tokens, cache.kv_heads, -1)
                  for a, ld in ((k, ld_k), (v, ld_v)))
        store = self.held.setdefault(cache, {})
        for i, s in enumerate(at):
            assert 0 <= s < cache.pages * cache.page_tokens
            store[int(s)] = (block4(kk[i]), block4(vv[i]))
        self.calls.append(("write", tokens, dtype))

    def read(self, cache, k, v, slots, tokens, dtype="f32", ld_k=0, ld_v=0, stream=None):
        w = cache.kv_heads * cache.head_dim
        at = view(device._addr(slots), tokens, np.int64)
        for dst, ld, i in ((k, ld_k, 0), (v, ld_v, 1)):
            y = np.stack([self.held[cache][int(s)][i] for s in at]).reshape(tokens, w)    # KeyError: nobody wrote it
            rows(dst, tokens, ld or w, w, dtype).copy_(torch.from_numpy(y))
        self.calls.append(("read", tokens, dtype))

    def decode(self, q, cache, table, lens, out, batch, q_heads, max_len, dtype="f32", scale=None, ld_q=0, ld_out=0,
               ld_table=0, stream=None):
        d, w, p = cache.head_dim, q_heads * cache.head_dim, cache.page_tokens
        n = view(device._addr(lens), batch, np.int32)
        per = -(-max_len // p)
        pages = np.lib.stride_tricks.as_strided(view(device._addr(table), (batch - 1) * ld_table + per, np.int32), (batch, per),
                                                (4 * ld_table, 4))
        qs = rows(q, batch, ld_q or w, w, dtype).double().numpy().reshape(batch, q_heads, d)
        dst = rows(out, batch, ld_out or w, w, dtype)
        for b in range(batch):
            if n[b] > max_len:
                dst[b] = float("nan")
                continue
            kv = [self.held[cache][int(pages[b, t // p]) * p + t % p] for t in range(n[b])]
            for h in range(q_heads):
                g = h // (q_heads // cache.kv_heads)
                y, _, _ = attend(qs[b, h:h + 1], [a[0][g] for a in kv], np.stack([a[1][g] for a in kv]), d ** -0.5, [n[b] - 1])
                dst[b, h * d:(h + 1) * d] = torch.from_numpy(y[0])
        self.calls.append(("decode", batch, max_len, dtype))

    def prefill(self, q, k, v, out, cu_q, cu_k, seqs, tokens_q, tokens_k, q_heads, kv_heads, head_dim, max_q, max_k,
                causal=True, dtype="bf16", out_dtype=None, scale=None, ld_q=0, ld_k=0, ld_v=0, ld_out=0, hs_q=0, hs_k=0,
                hs_v=0, hs_out=0, stream=None):
        d, nq, nk = head_dim, q_heads * head_dim, kv_heads * head_dim
        cq, ck = (view(device._addr(a), seqs + 1, np.int32) for a in (cu_q, cu_k))
        assert cq[0] >= 0 and ck[0] >= 0 and cq[-1] <= tokens_q and ck[-1] <= tokens_k
        qs = rows(q, tokens_q, ld_q or nq, nq, dtype).double().numpy().reshape(tokens_q, q_heads, d)
        ks, vs = (rows(a, tokens_k, ld or nk, nk, dtype).double().numpy().reshape(tokens_k, kv_heads, d)
                  for a, ld in ((k, ld_k), (v, ld_v)))
        dst = rows(out, tokens_q, ld_out or nq, nq, out_dtype or dtype)
        for s in range(seqs):
            n, m = cq[s + 1] - cq[s], ck[s + 1] - ck[s]
            assert 0 <= n <= max_q and 0 <= m <= max_k
            for h in range(q_heads if n else 0):
                g = h // (q_heads // kv_heads)
                y, _, _ = attend(qs[cq[s]:cq[s + 1], h], ks[ck[s]:ck[s + 1], g], vs[ck[s]:ck[s + 1], g], d ** -0.5,
                                 np.arange(n) + m - n if causal else np.full(n, m - 1))
                dst[cq[s]:cq[s + 1], h * d:(h + 1) * d] = torch.from_numpy(y)
        self.calls.append(("prefill", seqs, tokens_q, tokens_k))


@pytest.fixture
def host(monkeypatch):
    h, lib = Host(), Lib(_lib.lib())
    monkeypatch.setattr(device, "DeviceBuffer", Buffer)
    monkeypatch.setattr(device, "synchronize", lambda: None)
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    for name, f in (("qk_norm_rope", h.rope), ("kv4_write", h.write), ("kv4_read", h.read), ("attn_decode", h.decode),
                    ("attn_prefill", h.prefill)):
        monkeypatch.setattr(device, name, f)
    return h
