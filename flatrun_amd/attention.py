"""The attention step of a decoder block on the device: what
:meth:`flatrun_amd.layer.DecoderProjections.forward` asks its caller for.

The reference runs it in NumPy on the host, K and V kept as growing fp32
buffers (model/qwen2.py:1520-1624, runtime/kv_cache.py:35-113). Here:

    qkv ─▶ qk_norm_rope ─▶ q, k, v ─▶ KVCache4.write ─▶ attn_decode   (one token a sequence)
                                └──────────────────────▶ attn_prefill (prompts)

:class:`KVCache4` holds K and V in 4 bits in pages, :func:`rope_table` makes
the rotary table (64-bit, once per model), :class:`BlockAttention` is the
step with its buffers. The kernels are ``device.qk_norm_rope``,
``device.kv4_write`` / ``kv4_read``, ``device.attn_decode`` and
``device.attn_prefill``.
"""

from __future__ import annotations

import math

import numpy as np

from . import _lib, device


def rope_frequencies(rot: int, base: float = 10000.0, scaling: dict | None = None) -> tuple[np.ndarray, float]:
    """(frequencies fp64 [rot/2], factor of cos and sin) of rotary positions.

    ``scaling`` stretches a model to contexts longer than it was trained on:
      {"kind": "linear", "factor": f}       every frequency / f
      {"kind": "bands", "factor": f, "low": a, "high": b, "trained": n}
          frequencies that turn more than b times in n positions stay, fewer
          than a times are divided by f, those between blend linearly in their
          number of turns
      {"kind": "ramp", "factor": f, "fast": a, "slow": b, "trained": n}
          the same idea over the dimension's index, between the indices whose
          frequencies turn a (fast) and b (slow) times in n positions; cos and
          sin are multiplied by 0.1 ln(f) + 1
    """
    if rot < 0 or rot % 2:
        raise ValueError(f"the rotated part must be even, got {rot}")
    inv = float(base) ** (-np.arange(0, rot, 2, dtype=np.float64) / max(rot, 1))
    if scaling is None:
        return inv, 1.0
    kind, f = scaling.get("kind"), float(scaling["factor"])
    if not f >= 1.0:
        raise ValueError(f"a scaling factor is at least 1, got {f}")
    if kind == "linear":
        return inv / f, 1.0
    turns = float(scaling["trained"]) * inv / (2 * math.pi) if kind in ("bands", "ramp") else None
    if kind == "bands":
        lo, hi = float(scaling["low"]), float(scaling["high"])
        if not hi > lo:
            raise ValueError("bands: high must exceed low")
        keep = np.clip((turns - lo) / (hi - lo), 0.0, 1.0)
        return inv * (keep + (1 - keep) / f), 1.0
    if kind == "ramp":
        n = float(scaling["trained"])

        def index(count: float) -> float:
            return rot * math.log(n / (2 * math.pi * count)) / (2 * math.log(base))

        first = max(0, math.floor(index(float(scaling["fast"]))))
        last = min(rot - 1, math.ceil(index(float(scaling["slow"]))))
        part = np.clip((np.arange(rot // 2) - first) / max(last - first, 1e-3), 0.0, 1.0)
        return inv * ((1 - part) + part / f), 0.1 * math.log(f) + 1.0
    raise ValueError(f"unknown rotary scaling {kind!r}")


def rope_table(rot: int, positions: int, base: float = 10000.0, scaling: dict | None = None) -> np.ndarray:
    """(positions, rot/2, 2) fp32: cos and sin of position * frequency, made in
    64 bits and rounded once (at position 131071 an angle made in fp32 is off
    by 0.004). Upload it once: ``DeviceBuffer.from_host(rope_table(...))``."""
    inv, factor = rope_frequencies(rot, base, scaling)
    out = np.empty((positions, rot // 2, 2), np.float32)
    for at in range(0, positions, 8192):
        angle = np.arange(at, min(positions, at + 8192), dtype=np.float64)[:, None] * inv
        out[at:at + 8192, :, 0] = factor * np.cos(angle)
        out[at:at + 8192, :, 1] = factor * np.sin(angle)
    return out


class KVCache4:
    """Keys and values of one layer in 4 bits, in pages of ``page_tokens``
    tokens (a multiple of 32) in one device allocation: 4.5 bits an element.

    A slot is ``page * page_tokens + place``. :meth:`take` and :meth:`give`
    hand out page ids; a caller with its own page allocator (one for all
    layers) need not use them."""

    def __init__(self, pages: int, page_tokens: int, kv_heads: int, head_dim: int):
        self.pages, self.page_tokens = int(pages), int(page_tokens)
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.nbytes = device.kv4_bytes(pages, page_tokens, kv_heads, head_dim)
        self._buf = device.DeviceBuffer(max(self.nbytes, 16))
        self._free = list(range(self.pages - 1, -1, -1))

    def data_ptr(self) -> int:
        return self._buf.ptr

    def write(self, k, v, slots, tokens: int, dtype="f32", ld_k: int = 0, ld_v: int = 0, stream=None) -> None:
        """Quantise tokens' heads into their slots (:func:`device.kv4_write`)."""
        device.kv4_write(self, k, v, slots, tokens, dtype=dtype, ld_k=ld_k, ld_v=ld_v, stream=stream)

    def read(self, k, v, slots, tokens: int, dtype="f32", ld_k: int = 0, ld_v: int = 0, stream=None) -> None:
        """The values at the slots (:func:`device.kv4_read`)."""
        device.kv4_read(self, k, v, slots, tokens, dtype=dtype, ld_k=ld_k, ld_v=ld_v, stream=stream)

    def take(self, count: int = 1) -> list[int]:
        """Ids of ``count`` free pages."""
        if count > len(self._free):
            raise _lib.FrqError(_lib.ERR_UNSUPPORTED, f"cache full: {count} pages asked, {len(self._free)} free")
        return [self._free.pop() for _ in range(count)]

    def give(self, ids) -> None:
        """Pages back; the caller's work on them must have been enqueued."""
        for i in ids:
            if not 0 <= int(i) < self.pages or int(i) in self._free:
                raise ValueError(f"page {i} is not a page in use")
            self._free.append(int(i))

    def close(self) -> None:
        self._buf.free()


class Sequence:
    """A sequence's place in a model's caches: its length and its pages, which
    have the same ids in every layer's cache. ``cache`` is the one that handed
    them out, the first layer's."""

    def __init__(self):
        self.pages: list[int] = []
        self.length = 0
        self.cache: KVCache4 | None = None


class BlockAttention:
    """The attention step of one decoder block over its :class:`KVCache4`.

    The blocks of a model share one plan: the first layer's has buffers and
    hands out pages, the others are made with ``first=`` that one, on the same
    stream and with caches of their own of the same shape. They use its
    buffers, so a layer's output is read before the next layer is enqueued, as
    ``DecoderProjections.forward`` on one stream does.

    ``plan(new)``, on the first layer and once per step, fixes the step for all:
    ``new`` maps each sequence of the batch, in the order of the rows of qkv, to
    its number of new tokens; it takes pages for them and uploads positions,
    slots, lengths and the page table. Then, layer by layer,
    ``attention(qkv, rows)`` -- what ``DecoderProjections.forward`` calls --
    enqueues the step on the stream and returns fp32 rows for the o
    projection:

    * one new token of a sequence: norms and rotary positions in fp32, the
      token into the cache, attn_decode against it;
    * prompts: the heads as bf16, into the cache, and attn_prefill on them;
      where a prompt of the step has tokens in the cache already (it comes in
      chunks), all keys of the step's prompts, new ones too, are what the cache
      reads back.

    A step may hold both; what a single token gets does not depend on its
    neighbours (but for the last bits of sums). Single tokens that stand side
    by side in ``new`` share their launches.

    ``plan`` waits for the stream's earlier steps before it reuses its
    buffers.

    A step of single tokens can be captured in a graph and replayed after later
    plans of as many sequences. Its launches keep the longest length that they
    were made for: give ``plan`` a ``max_len`` that the replays will not pass
    (default: the longest sequence of this step, past which a replay gives NaN)."""

    def __init__(self, cache: KVCache4, q_heads: int, table, n_pos: int, max_rows: int = 0, max_seqs: int = 0,
                 max_context: int = 0, rot: int | None = None, interleaved: bool = False, q_norm=None, k_norm=None,
                 eps: float = 1e-6, stream=None, first: BlockAttention | None = None):
        if q_heads % cache.kv_heads:
            raise ValueError("q_heads must be a multiple of the cache's kv_heads")
        self.cache, self.q_heads, self.table, self.n_pos = cache, int(q_heads), table, int(n_pos)
        self.rot, self.interleaved, self.eps = rot, interleaved, eps
        self.q_norm, self.k_norm, self.stream = q_norm, k_norm, stream
        self._first = first
        if first is not None:
            self._share(first, max_rows, max_seqs, max_context)
            return
        if min(int(max_rows), int(max_seqs), int(max_context)) < 1:
            raise ValueError("max_rows, max_seqs and max_context must be at least 1")
        self.max_rows, self.max_seqs, self.max_context = int(max_rows), int(max_seqs), int(max_context)
        self.max_pages = -(-self.max_context // cache.page_tokens)
        d, hkv, r = cache.head_dim, cache.kv_heads, self.max_rows
        new = device.DeviceBuffer
        self.q, self.k, self.v = new(4 * r * q_heads * d), new(4 * r * hkv * d), new(4 * r * hkv * d)
        self.out = new(4 * r * q_heads * d)
        self._ints = new(4 * (r + 3 * (self.max_seqs + 1) + self.max_seqs * self.max_pages) + 64)
        self._slots = new(8 * r)
        self._ctx = None                     # K and V of a chunk's context, made when a prompt first needs it
        self._plan = None

    def _share(self, first: BlockAttention, *sizes) -> None:
        c, f = self.cache, first.cache
        if first._first is not None:
            raise ValueError("first must be the layer that plans")
        if (c.pages, c.page_tokens, c.kv_heads, c.head_dim) != (f.pages, f.page_tokens, f.kv_heads, f.head_dim) or c is f:
            raise ValueError("the layers' caches must have the same shape, and be one per layer")
        if self.q_heads != first.q_heads or self.n_pos < first.n_pos:
            raise ValueError("the layers must have the same heads and tables of as many positions")
        if device._stream(self.stream or first.stream) != device._stream(first.stream) or any(sizes):
            raise ValueError("the stream, max_rows, max_seqs and max_context are those of the first layer")
        self.stream = first.stream
        self.q, self.k, self.v, self.out, self._slots = first.q, first.k, first.v, first.out, first._slots
        self.max_rows, self.max_seqs, self.max_context = first.max_rows, first.max_seqs, first.max_context
        self.max_pages = first.max_pages

    def plan(self, new: dict, max_len: int | None = None) -> None:
        if self._first is not None:
            raise ValueError("the first layer plans the step for all of them")
        seqs, counts = list(new), [int(n) for n in new.values()]
        rows, c = sum(counts), self.cache
        if any(s.cache not in (None, c) for s in seqs):
            raise ValueError("a sequence is planned by the first layer of its model only (BlockAttention's first=)")
        if not seqs or len(seqs) > self.max_seqs or rows > self.max_rows or min(counts) < 1:
            raise ValueError(f"a step takes 1..{self.max_seqs} sequences and {self.max_rows} rows, a token at least each")
        if max(s.length + n for s, n in zip(seqs, counts)) > min(self.max_context, self.n_pos):
            raise ValueError("a sequence would pass max_context or the rotary table")
        if max_len is not None and not max(s.length + n for s, n in zip(seqs, counts)) <= max_len <= self.max_context:
            raise ValueError("max_len is from the step's longest sequence to max_context")
        need = [-(-(s.length + n) // c.page_tokens) - len(s.pages) for s, n in zip(seqs, counts)]
        ids = c.take(sum(max(0, n) for n in need))
        table = np.zeros((len(seqs), self.max_pages), np.int32)
        slots, positions = [], []
        for i, (s, n) in enumerate(zip(seqs, counts)):
            s.cache = c
            for _ in range(max(0, need[i])):
                s.pages.append(ids.pop())
            table[i, :len(s.pages)] = s.pages
            t = np.arange(s.length, s.length + n)
            positions.append(t)
            slots.append(table[i, t // c.page_tokens].astype(np.int64) * c.page_tokens + t % c.page_tokens)
        past = [s.length for s in seqs]
        lens = np.array([p + n for p, n in zip(past, counts)], np.int32)
        single = [n == 1 for n in counts]
        context = any(p and not one for p, one in zip(past, single))
        # keys of the prompts' attention; a single token beside them has none, or, where the rows themselves are the
        # keys, its own: attn_decode overwrites what comes of it
        keys = np.where(single, 0, lens) if context else np.array(counts)
        cu_q = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        cu_k = np.concatenate([[0], np.cumsum(keys)]).astype(np.int32)
        ints = np.concatenate([np.concatenate(positions).astype(np.int32), lens, cu_q, cu_k, table.reshape(-1)])
        lib, check = _lib.lib(), _lib.check
        if self.stream is None:              # earlier steps still read these buffers
            device.synchronize()
        elif hasattr(self.stream, "synchronize"):
            self.stream.synchronize()
        else:                                # a stream's handle
            check(lib.frq_stream_synchronize(device._stream(self.stream)))
        check(lib.frq_memcpy_h2d(self._ints.ptr, ints.ctypes.data, ints.nbytes))
        sl = np.concatenate(slots)
        check(lib.frq_memcpy_h2d(self._slots.ptr, sl.ctypes.data, sl.nbytes))
        b, at = len(seqs), self._ints.ptr
        p = {"rows": rows, "batch": b, "positions": at, "lens": at + 4 * rows, "cu_q": at + 4 * (rows + b),
             "cu_k": at + 4 * (rows + 2 * b + 1), "table": at + 4 * (rows + 3 * b + 2), "max_q": max(counts),
             "max_k": int(keys.max()), "tokens_k": int(keys.sum()), "prompts": not all(single), "context": context,
             "max_len": max_len or max([int(n) for n, one in zip(lens, single) if one], default=0), "tokens": []}
        for i in range(b):                   # runs of single tokens: (sequence, row, count)
            if single[i] and i and single[i - 1]:
                p["tokens"][-1][2] += 1
            elif single[i]:
                p["tokens"].append([i, int(cu_q[i]), 1])
        if context:
            self._plan_context(p, table, keys)
        for s, n in zip(seqs, counts):
            s.length += n
        self._plan = p

    def _plan_context(self, p: dict, table, keys) -> None:
        """Slots of every key of the prompts, context and new, in packed order."""
        c = self.cache
        slots = np.concatenate([table[i, np.arange(n) // c.page_tokens].astype(np.int64) * c.page_tokens
                                + np.arange(n) % c.page_tokens for i, n in enumerate(keys)])
        size = 2 * p["tokens_k"] * c.kv_heads * c.head_dim   # whole rows of 64 elements and more: K and V stay aligned
        want = 2 * size + slots.nbytes
        if self._ctx is None or self._ctx.nbytes < want:
            self._ctx = device.DeviceBuffer(want)
        p["ctx_k"], p["ctx_v"], p["ctx_slots"] = (self._ctx.ptr + i * size for i in range(3))
        _lib.check(_lib.lib().frq_memcpy_h2d(p["ctx_slots"], slots.ctypes.data, slots.nbytes))

    def __call__(self, qkv, rows: int):
        p, c = (self._first or self)._plan, self.cache
        if p is None or rows != p["rows"]:
            raise ValueError("plan() this step's rows first")
        if p["prompts"]:
            self._prompts(p, qkv)
        for seq, row, count in p["tokens"]:
            self._tokens(p, qkv, seq, row, count)
        return self.out

    def _heads(self, p: dict, qkv, row: int, count: int, dtype: str) -> None:
        """q, k and v of `count` rows from `row` on, the new tokens into the cache."""
        c, slots = self.cache, (self._first or self)._slots
        width = (self.q_heads + 2 * c.kv_heads) * c.head_dim
        device.qk_norm_rope(qkv if row == 0 else device._addr(qkv) + 4 * row * width, self.q, self.k, self.v, count,
                            self.q_heads, c.kv_heads, c.head_dim, self.table, p["positions"] + 4 * row, rot=self.rot,
                            interleaved=self.interleaved, q_norm=self.q_norm, k_norm=self.k_norm, eps=self.eps,
                            out_dtype=dtype, n_pos=self.n_pos, stream=self.stream)
        c.write(self.k, self.v, slots.ptr + 8 * row, count, dtype=dtype, stream=self.stream)

    def _prompts(self, p: dict, qkv) -> None:
        c, rows, s = self.cache, p["rows"], self.stream
        self._heads(p, qkv, 0, rows, "bf16")
        k, v, cu_k = self.k, self.v, p["cu_q"]
        if p["context"]:
            k, v, cu_k = p["ctx_k"], p["ctx_v"], p["cu_k"]
            c.read(k, v, p["ctx_slots"], p["tokens_k"], dtype="bf16", stream=s)
        device.attn_prefill(self.q, k, v, self.out, p["cu_q"], cu_k, p["batch"], rows, p["tokens_k"], self.q_heads,
                            c.kv_heads, c.head_dim, max_q=p["max_q"], max_k=p["max_k"], out_dtype="f32", stream=s)

    def _tokens(self, p: dict, qkv, seq: int, row: int, count: int) -> None:
        c, s = self.cache, self.stream
        self._heads(p, qkv, row, count, "f32")
        device.attn_decode(self.q, c, p["table"] + 4 * seq * self.max_pages, p["lens"] + 4 * seq,
                           self.out.ptr + 4 * row * self.q_heads * c.head_dim, count, self.q_heads, p["max_len"],
                           ld_table=self.max_pages, stream=s)

    def close(self) -> None:
        """Frees the buffers, once for all layers: on the first."""
        if self._first is not None:
            return
        for b in (self.q, self.k, self.v, self.out, self._ints, self._slots, self._ctx):
            if b is not None:
                b.free()
