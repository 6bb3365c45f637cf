"""Device-resident buffers, streams and the device-pointer entry points.

This is the decode-time path: raw GGUF blocks are uploaded once
(:meth:`DeviceBuffer.from_host`) and every matvec reads them straight from
HBM through ``frq_dev_gemv``. Any object exposing ``data_ptr()`` (a torch
CUDA tensor) can be passed where a device buffer is expected, so callers that
keep activations in torch tensors need no copies.
"""

from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from ._lib import check, lib


def _addr(obj) -> int:
    if obj is None:
        return 0
    if isinstance(obj, DeviceBuffer):
        return obj.ptr
    if hasattr(obj, "data_ptr"):
        return int(obj.data_ptr())
    if isinstance(obj, int):
        return obj
    raise TypeError(f"expected a device buffer, got {type(obj).__name__}")


def _nbytes(obj) -> int:
    if isinstance(obj, DeviceBuffer):
        return obj.nbytes
    if hasattr(obj, "data_ptr") and isinstance(getattr(obj, "nbytes", None), int):   # DeviceWeight
        return obj.nbytes
    if hasattr(obj, "untyped_storage"):
        return int(obj.numel() * obj.element_size())
    raise TypeError(f"cannot size {type(obj).__name__}")


def _stream(s) -> int:
    if s is None:
        return 0
    if isinstance(s, Stream):
        return s.handle
    try:
        return s.cuda_stream             # torch's
    except AttributeError:
        return int(s)


class DeviceBuffer:
    """An allocation in device memory (hipMalloc), freed with the object."""

    def __init__(self, nbytes: int):
        self.nbytes = int(nbytes)
        p = ctypes.c_void_p()
        check(lib().frq_malloc(ctypes.byref(p), self.nbytes))
        self.ptr = int(p.value or 0)

    @classmethod
    def from_host(cls, arr: np.ndarray, stream=None) -> "DeviceBuffer":
        a = np.ascontiguousarray(arr)
        buf = cls(a.nbytes)
        if a.nbytes:
            if stream is None:
                check(lib().frq_memcpy_h2d(buf.ptr, a.ctypes.data, a.nbytes))
            else:
                check(lib().frq_memcpy_h2d_async(buf.ptr, a.ctypes.data, a.nbytes, _stream(stream)))
        return buf

    def to_host(self, dtype=np.uint8, count: int | None = None) -> np.ndarray:
        dt = np.dtype(dtype)
        n = self.nbytes // dt.itemsize if count is None else int(count)
        out = np.empty(n, dtype=dt)
        if out.nbytes:
            check(lib().frq_memcpy_d2h(out.ctypes.data, self.ptr, out.nbytes))
        return out

    def free(self) -> None:
        if getattr(self, "ptr", 0):
            try:
                lib().frq_free(self.ptr)
            finally:
                self.ptr = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def data_ptr(self) -> int:
        return self.ptr


class PinnedBuffer:
    """Page-locked host memory (hipHostMalloc) viewed as a numpy array."""

    def __init__(self, nbytes: int):
        self.nbytes = int(nbytes)
        p = ctypes.c_void_p()
        check(lib().frq_host_alloc(ctypes.byref(p), self.nbytes))
        self.ptr = int(p.value or 0)
        self.array = np.ctypeslib.as_array((ctypes.c_uint8 * max(self.nbytes, 1)).from_address(self.ptr))[: self.nbytes]

    def free(self) -> None:
        if getattr(self, "ptr", 0):
            self.array = None
            try:
                lib().frq_host_free(self.ptr)
            finally:
                self.ptr = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Stream:
    """A HIP stream at the default priority (non-blocking w.r.t. the null stream)."""

    def __init__(self):
        p = ctypes.c_void_p()
        check(lib().frq_stream_create(ctypes.byref(p)))
        self.handle = int(p.value or 0)

    def synchronize(self) -> None:
        check(lib().frq_stream_synchronize(self.handle))

    def wait(self, event: "Event") -> None:
        check(lib().frq_stream_wait_event(self.handle, event.handle))

    def destroy(self) -> None:
        if getattr(self, "handle", 0):
            try:
                lib().frq_stream_destroy(self.handle)
            finally:
                self.handle = 0

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class Event:
    def __init__(self):
        p = ctypes.c_void_p()
        check(lib().frq_event_create(ctypes.byref(p)))
        self.handle = int(p.value or 0)

    def record(self, stream=None) -> None:
        check(lib().frq_event_record(self.handle, _stream(stream)))

    def synchronize(self) -> None:
        check(lib().frq_event_synchronize(self.handle))

    def elapsed_ms(self, end: "Event") -> float:
        ms = ctypes.c_float()
        check(lib().frq_event_elapsed_ms(ctypes.byref(ms), self.handle, end.handle))
        return float(ms.value)

    def destroy(self) -> None:
        if getattr(self, "handle", 0):
            try:
                lib().frq_event_destroy(self.handle)
            finally:
                self.handle = 0

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class Graph:
    """A recorded launch sequence, replayed with one call.

    ``with Graph.capture(stream) as g: ...`` records every launch issued on
    ``stream`` inside the block (nothing runs then); ``g.launch(stream)``
    replays it. The stream must be a :class:`Stream`, not the null stream.
    """

    def __init__(self, handle: int):
        self.handle = handle

    @classmethod
    def capture(cls, stream: "Stream"):
        return _Capture(stream)

    def launch(self, stream=None) -> None:
        check(lib().frq_graph_launch(self.handle, _stream(stream)))

    def destroy(self) -> None:
        if getattr(self, "handle", 0):
            try:
                lib().frq_graph_destroy(self.handle)
            finally:
                self.handle = 0

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class _Capture:
    def __init__(self, stream: "Stream"):
        if not isinstance(stream, Stream):
            raise TypeError("graph capture needs a device.Stream")
        self.stream = stream
        self.graph: Graph | None = None

    def __enter__(self) -> "_Capture":
        check(lib().frq_stream_begin_capture(self.stream.handle))
        return self

    def __exit__(self, et, ev, tb) -> None:
        h = ctypes.c_void_p()
        rc = lib().frq_stream_end_capture(self.stream.handle, ctypes.byref(h))
        if et is None:
            check(rc)
            self.graph = Graph(int(h.value or 0))
        elif rc == 0 and h.value:
            lib().frq_graph_destroy(h.value)

    def launch(self, stream=None) -> None:
        self.graph.launch(stream)

    def destroy(self) -> None:
        if self.graph is not None:
            self.graph.destroy()


def synchronize() -> None:
    check(lib().frq_device_synchronize())


def qtype_id(q) -> int:
    if isinstance(q, str):
        return _lib.QTYPES[q.upper()]
    return int(q)


def gemv(qtype, w, x, y, n: int, k: int, batch: int = 1, stream=None, w_bytes: int | None = None) -> None:
    """y[b, :n] = W[n, k] . x[b, :k] on device buffers (enqueued, not synchronised)."""
    q = qtype_id(qtype)
    wb = _nbytes(w) if w_bytes is None else int(w_bytes)
    check(lib().frq_dev_gemv(q, _addr(w), wb, _addr(x), _addr(y), int(n), int(k), int(batch), _stream(stream)))


BATCH_ROUTES = ("rows", "small", "pair", "few", "gemm")


def batch_plan(qtype, n: int, k: int, batch: int) -> tuple[str, int, int, int]:
    """(route, rows per tile, splits of k, scratch bytes) of a batched gemv
    (frq_gemv_batch_plan); needs no GPU."""
    plan = (ctypes.c_int64 * 4)()
    check(lib().frq_gemv_batch_plan(qtype_id(qtype), int(n), int(k), int(batch), plan))
    return BATCH_ROUTES[plan[0]], plan[1], plan[2], plan[3]


def gemv_host(qtype, w, x: np.ndarray, y: np.ndarray, n: int, k: int, batch: int, scratch: DeviceBuffer,
              pinned: PinnedBuffer | None = None, w_bytes: int | None = None) -> None:
    """gemv with x and y in host memory (contiguous float32, (batch, k) and
    (batch, n)), synchronous, on the null stream (frq_dev_gemv_host)."""
    q = qtype_id(qtype)
    wb = _nbytes(w) if w_bytes is None else int(w_bytes)
    if x.dtype != np.float32 or y.dtype != np.float32 or not (x.flags.c_contiguous and y.flags.c_contiguous):
        raise ValueError("gemv_host: x and y must be contiguous float32")
    if x.size < batch * k or y.size < batch * n:
        raise ValueError(f"gemv_host: x or y holds fewer than {batch} rows")
    check(lib().frq_dev_gemv_host(q, _addr(w), wb, x.ctypes.data, y.ctypes.data, int(n), int(k), int(batch),
                                  scratch.ptr, scratch.nbytes, pinned.ptr if pinned else 0,
                                  pinned.nbytes if pinned else 0))


GROUP_MAX = 4


def _group_arrays(parts):
    if not 1 <= len(parts) <= GROUP_MAX:
        raise ValueError(f"a group holds 1..{GROUP_MAX} matrices, got {len(parts)}")
    qt = (ctypes.c_int * len(parts))(*[qtype_id(p[0]) for p in parts])
    wp = (ctypes.c_void_p * len(parts))(*[_addr(p[1]) for p in parts])
    return qt, wp


def gemv_group(parts, x, k: int, batch: int = 1, y_stride: int = 0, stream=None) -> None:
    """Matrices sharing x in one launch where possible (frq_dev_gemv_group;
    a single matrix runs frq_dev_gemv's kernel).

    ``parts``: up to 4 tuples ``(qtype, w, n, y[, w_bytes])``; ``y`` is the
    device output of batch row 0 (an int address is accepted, e.g. an offset
    into one concatenated buffer); row b of matrix i goes to
    ``y_i + b * (y_stride or n_i)`` floats."""
    qt, wp = _group_arrays(parts)
    c = len(parts)
    wb = (ctypes.c_size_t * c)(*[int(p[4]) if len(p) > 4 else _nbytes(p[1]) for p in parts])
    nn = (ctypes.c_int64 * c)(*[int(p[2]) for p in parts])
    yy = (ctypes.c_void_p * c)(*[_addr(p[3]) for p in parts])
    check(lib().frq_dev_gemv_group(c, qt, wp, wb, nn, _addr(x), int(k), yy, int(batch), int(y_stride),
                                   _stream(stream)))


def gemv_group_fusable(parts, k: int) -> bool:
    """True if ``parts`` ((qtype, w, ...) tuples) run as one launch."""
    qt, wp = _group_arrays(parts)
    return bool(lib().frq_gemv_group_fusable(len(parts), qt, wp, int(k)))


def gemv_tuned(qtype, w, x, y, n: int, k: int, kernel: int = 0, cpl: int = 0, rows: int = 0, unroll: int = 0,
               stream=None, w_bytes: int | None = None, slices: int = 0) -> dict:
    """One GEMV with an explicit launch geometry; returns the geometry used
    (fields of frq_gemv_config)."""
    q = qtype_id(qtype)
    wb = _nbytes(w) if w_bytes is None else int(w_bytes)
    cfg = _lib.GemvConfig(kernel=kernel, cpl=cpl, rows=rows, unroll=unroll, slices=slices)
    check(lib().frq_dev_gemv_tuned(q, _addr(w), wb, _addr(x), _addr(y), int(n), int(k), ctypes.addressof(cfg),
                                   _stream(stream)))
    return cfg.as_dict()


def gemm_bf16(qtype, w, x_bf16, y, m: int, n: int, k: int, stream=None, w_bytes: int | None = None) -> None:
    """y[m, n] = x[m, k] . W[n, k]^T on the matrix cores (W: Q4_K, Q6_K or Q8_0
    blocks; x: bf16 bits, row-major; y: fp32). Enqueued, not synchronised."""
    wb = _nbytes(w) if w_bytes is None else int(w_bytes)
    check(lib().frq_dev_gemm_bf16(qtype_id(qtype), _addr(w), wb, _addr(x_bf16), _addr(y), int(m), int(n), int(k),
                                  _stream(stream)))


def gemm_bf16_group(parts, x_bf16, m: int, k: int, y_stride: int = 0, stream=None) -> None:
    """Matrices sharing x in one GEMM launch (frq_dev_gemm_bf16_group).
    ``parts``: up to 4 tuples ``(qtype, w, n, y[, w_bytes])``; ``y`` is the
    device output (an int address is accepted, e.g. an offset into one
    concatenated buffer); row r of matrix i goes to ``y_i + r * (y_stride or n_i)``
    floats."""
    qt, wp = _group_arrays(parts)
    c = len(parts)
    wb = (ctypes.c_size_t * c)(*[int(p[4]) if len(p) > 4 else _nbytes(p[1]) for p in parts])
    nn = (ctypes.c_int64 * c)(*[int(p[2]) for p in parts])
    yy = (ctypes.c_void_p * c)(*[_addr(p[3]) for p in parts])
    check(lib().frq_dev_gemm_bf16_group(c, qt, wp, wb, nn, _addr(x_bf16), int(m), int(k), yy, int(y_stride),
                                        _stream(stream)))


def gemm_q4k_bf16(w, x_bf16, y, m: int, n: int, k: int, stream=None, w_bytes: int | None = None) -> None:
    gemm_bf16("Q4_K", w, x_bf16, y, m, n, k, stream=stream, w_bytes=w_bytes)


def memcpy_h2d_async(dst, src_host_ptr: int, nbytes: int, stream=None) -> None:
    """Enqueues a host -> device copy (the host memory should be pinned for it
    to run asynchronously)."""
    check(lib().frq_memcpy_h2d_async(_addr(dst), int(src_host_ptr), int(nbytes), _stream(stream)))


def copy(dst, src, nbytes: int, stream=None) -> None:
    """dst[:nbytes] = src[:nbytes] with the library's streaming copy kernel (enqueued)."""
    check(lib().frq_dev_copy(_addr(dst), _addr(src), int(nbytes), _stream(stream)))


READ_XOR_WORDS = 2048


def read_xor(src, nbytes: int, out, stream=None) -> None:
    """Read src[:nbytes] with the library's streaming read kernel (enqueued):
    out (READ_XOR_WORDS device words) receives per-workgroup XORs of its
    32-bit words, zeros past the grid; the XOR of all of out is that of src."""
    check(lib().frq_dev_read_xor(_addr(src), int(nbytes), _addr(out), _stream(stream)))


def dequant(qtype, w, y, n_elems: int, stream=None, w_bytes: int | None = None) -> None:
    """y[:n_elems] = dequant(w) on device buffers (enqueued)."""
    q = qtype_id(qtype)
    wb = _nbytes(w) if w_bytes is None else int(w_bytes)
    check(lib().frq_dev_dequant(q, _addr(w), wb, int(n_elems), _addr(y), _stream(stream)))


def dequant_f16(qtype, w, y, n_elems: int, stream=None, w_bytes: int | None = None) -> None:
    """y[:n_elems] = fp16 bit patterns of dequant(w), rounded to nearest even
    (enqueued)."""
    q = qtype_id(qtype)
    wb = _nbytes(w) if w_bytes is None else int(w_bytes)
    check(lib().frq_dev_dequant_f16(q, _addr(w), wb, int(n_elems), _addr(y), _stream(stream)))


def gemv_swiglu(gate, up, x, k: int, gateup, act, batch: int = 1, stream=None) -> None:
    """gateup[r] = [W_gate x_r | W_up x_r] and act[r] = silu(gate) * up for
    `batch` rows of x, enqueued (frq_dev_gemv_swiglu: one launch for a Q4_K
    pair at batch 1, else the grouped launch and frq_dev_silu_mul, same
    bits). ``gate`` / ``up``: ``(qtype, w, inter[, w_bytes])``."""
    qg, wg, inter = gate[0], gate[1], int(gate[2])
    qu, wu = up[0], up[1]
    gb = int(gate[3]) if len(gate) > 3 else _nbytes(wg)
    ub = int(up[3]) if len(up) > 3 else _nbytes(wu)
    if int(up[2]) != inter:
        raise ValueError(f"gate and up need the same output size, got {inter} and {up[2]}")
    check(lib().frq_dev_gemv_swiglu(qtype_id(qg), _addr(wg), gb, qtype_id(qu), _addr(wu), ub, inter, _addr(x),
                                    int(k), _addr(gateup), _addr(act), int(batch), _stream(stream)))


def gemv_swiglu_fusable(gate, up, k: int) -> bool:
    """True if gemv_swiglu runs ``gate`` and ``up`` ((qtype, w, ...)) and the
    activation as one launch at batch 1."""
    return bool(lib().frq_gemv_swiglu_fusable(qtype_id(gate[0]), _addr(gate[1]), qtype_id(up[0]), _addr(up[1]),
                                              int(k)))


def silu_mul(gateup, out, rows: int, inter: int, ld_in: int = 0, ld_out: int = 0, stream=None) -> None:
    """out[r, :inter] = silu(gate) * up for the grouped gate|up rows of
    gateup (gate first; rows ld_in floats apart, default 2 inter; out rows
    ld_out apart, default inter), enqueued (frq_dev_silu_mul)."""
    li = int(ld_in) or 2 * int(inter)
    lo = int(ld_out) or int(inter)
    check(lib().frq_dev_silu_mul(_addr(gateup), li, _addr(out), lo, int(rows), int(inter), _stream(stream)))


# ------------------------------------------------- a block's attention step

_VTYPE_OF = {**{n: i for n, i in _lib.VTYPES.items()}, **{i: i for i in _lib.VTYPES.values()}}


def vtype_id(t) -> int:
    """Type id of activations: "f32", "f16" or "bf16" (or the id itself)."""
    i = _VTYPE_OF.get(t)
    if i is None:
        if isinstance(t, str):
            i = _VTYPE_OF.get(t.lower())
            if i is None:
                raise ValueError(f"activations are f32, f16 or bf16, not {t!r}")
            return i
        return int(t)
    return i


_I32, _I64, _U8 = "int32", "int64", "torch.uint8"
_Q8 = _lib.QTYPES["Q8_0"]
_KINDS: dict = {}              # dtype object -> type id or integer kind (filled as dtypes are met)


def _kind_of(dtype):
    kind = {"torch.float32": _lib.F32, "torch.float16": _lib.F16, "torch.bfloat16": _lib.BF16, "torch.int32": _I32,
            "torch.int64": _I64}.get(str(dtype), str(dtype))
    _KINDS[dtype] = kind
    return kind


def _rows_of(obj, ld: int, hs: int) -> bool:
    """Whether a strided tensor lies as the call describes it: elements side by
    side, in rows ld or heads hs apart."""
    dims: list = []
    for n, step in zip(reversed(obj.shape), reversed(obj.stride())):
        if n == 1:
            continue
        if dims and step == dims[-1][0] * dims[-1][1]:
            dims[-1] = (n * dims[-1][0], dims[-1][1])       # one run with the dimension inside it
        else:
            dims.append((n, step))
    return not dims or (dims[0][1] == 1 and all(step > 0 and step in (ld, hs) for _, step in dims[1:]))


def _operand(name: str, obj, need: int, kind, ld: int = 0, hs: int = 0) -> int:
    """Address of a device operand that holds `need` bytes of `kind`. Refuses a
    buffer whose size is known and too small, and a tensor of another type, in
    host memory, or of strides other than the call's (an address says nothing of
    either)."""
    if obj is None:
        return 0
    t = type(obj)
    if t is int:
        return obj
    if t is DeviceBuffer:
        if obj.nbytes < need:
            raise ValueError(f"{name} holds {obj.nbytes} bytes, the call needs {need}")
        return obj.ptr
    try:
        if _KINDS[obj.dtype] == kind and obj.nbytes >= need and obj.is_cuda and obj.is_contiguous():
            return obj.data_ptr()
    except (AttributeError, KeyError):
        pass
    if hasattr(obj, "dtype") and hasattr(obj, "untyped_storage"):
        if _kind_of(obj.dtype) != kind:
            raise TypeError(f"{name} is {obj.dtype}, the call says otherwise")
        # a strided view reaches further than its own elements
        size = int(obj.untyped_storage().nbytes() - obj.storage_offset() * obj.element_size())
        if size < need:
            raise ValueError(f"{name} holds {size} bytes, the call needs {need}")
        if not obj.is_contiguous() and not _rows_of(obj, ld, hs):
            raise ValueError(f"{name} has strides {tuple(obj.stride())}, the call takes its rows {ld or 1} elements apart")
        if not obj.is_cuda and not obj.is_pinned():
            raise ValueError(f"{name} is in host memory")
        return obj.data_ptr()
    return _addr(obj)


def qk_norm_rope(x, q, k, v, tokens: int, q_heads: int, kv_heads: int, head_dim: int, table, positions,
                 rot: int | None = None, interleaved: bool = False, q_norm=None, k_norm=None, eps: float = 1e-6,
                 x_dtype="f32", out_dtype="f32", ld_x: int = 0, ld_q: int = 0, ld_k: int = 0, ld_v: int = 0,
                 n_pos: int | None = None, stream=None) -> None:
    """Norms of the query and key heads and rotary positions of the q|k|v rows
    of ``x`` in one pass (frq_dev_qk_norm_rope), enqueued.

    Row t of ``x`` (``ld_x`` elements apart, default the heads' width) goes to
    ``q[t]``, ``k[t]`` and ``v[t]`` (``v`` None: x has, or keeps, its v); ``rot``
    elements of each head turn (default all) by ``table[positions[t]]``
    (:func:`flatrun_amd.attention.rope_table`; ``n_pos`` rows, taken from its
    size where that is known); ``q_norm`` / ``k_norm``: fp32 weights or None."""
    hd, t = int(head_dim), int(tokens)
    rot = hd if rot is None else int(rot)
    nq, nk = q_heads * hd, kv_heads * hd
    lq, lk, lv = ld_q or nq, ld_k or nk, ld_v or nk
    width = nq + (nk if v is None else 2 * nk)
    lx = ld_x or width
    xi, oi = vtype_id(x_dtype), vtype_id(out_dtype)
    xs, os_ = (4 if xi == 0 else 2), (4 if oi == 0 else 2)
    if n_pos is None:
        n_pos = _nbytes(table) // (4 * rot) if rot and table is not None else 0
    check(lib().frq_dev_qk_norm_rope(
        xi, _operand("x", x, xs * ((t - 1) * lx + width), xi, lx), lx, oi, _operand("q", q, os_ * ((t - 1) * lq + nq), oi, lq), lq,
        _operand("k", k, os_ * ((t - 1) * lk + nk), oi, lk), lk, _operand("v", v, os_ * ((t - 1) * lv + nk), oi, lv), lv, t, q_heads,
        kv_heads, hd, rot, 1 if interleaved else 0, _operand("table", table, 4 * n_pos * rot, _lib.F32), n_pos,
        _operand("positions", positions, 4 * t, _I32), _operand("q_norm", q_norm, 4 * hd, _lib.F32),
        _operand("k_norm", k_norm, 4 * hd, _lib.F32), eps, _stream(stream)))


def kv4_bytes(pages: int, page_tokens: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of a 4-bit paged cache (frq_kv4_bytes); needs no GPU."""
    n = ctypes.c_size_t()
    check(lib().frq_kv4_bytes(int(pages), int(page_tokens), int(kv_heads), int(head_dim), ctypes.byref(n)))
    return int(n.value)


def _kv4_args(cache, k, v, slots, tokens, dtype, ld_k, ld_v):
    width, t = cache.kv_heads * cache.head_dim, int(tokens)
    lk, lv = ld_k or width, ld_v or width
    ti = vtype_id(dtype)
    size = 4 if ti == 0 else 2
    return (cache.data_ptr(), cache.nbytes, cache.pages, cache.page_tokens, cache.kv_heads, cache.head_dim, ti,
            _operand("k", k, size * ((t - 1) * lk + width), ti, lk), lk, _operand("v", v, size * ((t - 1) * lv + width), ti, lv), lv,
            _operand("slots", slots, 8 * t, _I64), t)


def kv4_write(cache, k, v, slots, tokens: int, dtype="f32", ld_k: int = 0, ld_v: int = 0, stream=None) -> None:
    """Quantise ``tokens`` tokens' heads into the slots (int64, on the device)
    of a :class:`flatrun_amd.attention.KVCache4`, enqueued (frq_dev_kv4_write)."""
    check(lib().frq_dev_kv4_write(*_kv4_args(cache, k, v, slots, tokens, dtype, ld_k, ld_v), _stream(stream)))


def kv4_read(cache, k, v, slots, tokens: int, dtype="f32", ld_k: int = 0, ld_v: int = 0, stream=None) -> None:
    """The values at the slots of a :class:`flatrun_amd.attention.KVCache4`
    into k and v, enqueued (frq_dev_kv4_read)."""
    check(lib().frq_dev_kv4_read(*_kv4_args(cache, k, v, slots, tokens, dtype, ld_k, ld_v), _stream(stream)))


def attn_decode(q, cache, table, lens, out, batch: int, q_heads: int, max_len: int, dtype="f32",
                scale: float | None = None, ld_q: int = 0, ld_out: int = 0, ld_table: int = 0, stream=None) -> None:
    """out[b] = attention of query token q[b] over the first lens[b] tokens of
    its sequence in a :class:`flatrun_amd.attention.KVCache4`, enqueued
    (frq_dev_attn_decode).

    ``table``: int32 page ids, one row per sequence (``ld_table`` apart,
    default what ``max_len`` tokens need, or a 2-d tensor's own row stride);
    ``lens``: int32; no length exceeds ``max_len``. ``scale`` defaults to
    1 / sqrt(head_dim)."""
    hd, b, n = cache.head_dim, int(batch), int(max_len)
    nq = q_heads * hd
    lq, lo = ld_q or nq, ld_out or nq
    per = (n + cache.page_tokens - 1) // cache.page_tokens
    lt = ld_table or (table.stride(0) if getattr(table, "ndim", 0) == 2 and hasattr(table, "stride") else per)
    ti = vtype_id(dtype)
    size = 4 if ti == 0 else 2
    check(lib().frq_dev_attn_decode(
        ti, _operand("q", q, size * ((b - 1) * lq + nq), ti, lq), lq, cache.data_ptr(), cache.nbytes, cache.pages,
        cache.page_tokens, cache.kv_heads, hd, _operand("table", table, 4 * ((b - 1) * lt + per), _I32, lt), lt,
        _operand("lens", lens, 4 * b, _I32), n, _operand("out", out, size * ((b - 1) * lo + nq), ti, lo), lo, b, q_heads,
        hd ** -0.5 if scale is None else scale, _stream(stream)))


def attn_prefill(q, k, v, out, cu_q, cu_k, seqs: int, tokens_q: int, tokens_k: int, q_heads: int, kv_heads: int,
                 head_dim: int, max_q: int, max_k: int, causal: bool = True, dtype="bf16", out_dtype=None,
                 scale: float | None = None, ld_q: int = 0, ld_k: int = 0, ld_v: int = 0, ld_out: int = 0, hs_q: int = 0,
                 hs_k: int = 0, hs_v: int = 0, hs_out: int = 0, stream=None) -> None:
    """Attention over ``seqs`` packed sequences (frq_dev_attn_prefill),
    enqueued: the queries [cu_q[s], cu_q[s + 1]) over the keys [cu_k[s],
    cu_k[s + 1]) (int32 on the device, seqs + 1 of each), causal from the last
    key back. Tokens are ``ld_*`` elements apart (default all heads side by
    side) and heads ``hs_*`` (default head_dim). ``dtype`` "bf16" or "f16";
    ``out_dtype`` the same (default) or "f32"."""
    hd, tq, tk, n = int(head_dim), int(tokens_q), int(tokens_k), int(seqs)
    ti = vtype_id(dtype)
    oi = ti if out_dtype is None else vtype_id(out_dtype)
    hq, hk, hv, ho = hs_q or hd, hs_k or hd, hs_v or hd, hs_out or hd
    nq, nk = q_heads * hd, kv_heads * hd
    lq, lk, lv, lo = ld_q or nq, ld_k or nk, ld_v or nk, ld_out or nq
    check(lib().frq_dev_attn_prefill(
        ti, _operand("q", q, 2 * ((tq - 1) * lq + (q_heads - 1) * hq + hd) if tq else 0, ti, lq, hq), lq, hq,
        _operand("k", k, 2 * ((tk - 1) * lk + (kv_heads - 1) * hk + hd) if tk else 0, ti, lk, hk), lk, hk,
        _operand("v", v, 2 * ((tk - 1) * lv + (kv_heads - 1) * hv + hd) if tk else 0, ti, lv, hv), lv, hv, oi,
        _operand("out", out, (4 if oi == 0 else 2) * ((tq - 1) * lo + (q_heads - 1) * ho + hd) if tq else 0, oi, lo, ho), lo, ho,
        _operand("cu_q", cu_q, 4 * (n + 1), _I32), _operand("cu_k", cu_k, 4 * (n + 1), _I32), n, tq, tk, int(max_q),
        int(max_k), q_heads, kv_heads, hd, 1 if causal else 0, hd ** -0.5 if scale is None else scale, _stream(stream)))


def attn_chunk(q, cache, table, lens, cu_q, out, seqs: int, tokens_q: int, q_heads: int, max_q: int, max_len: int,
               dtype="bf16", out_dtype=None, scale: float | None = None, ld_q: int = 0, ld_out: int = 0, ld_table: int = 0,
               stream=None) -> None:
    """Attention of each sequence's new tokens, the queries [cu_q[s], cu_q[s + 1])
    (int32 on the device, seqs + 1), over the lens[s] tokens that a
    :class:`flatrun_amd.attention.KVCache4` holds of it, the new ones among them,
    causal from the last token back; enqueued (frq_dev_attn_chunk).

    ``table``, ``lens`` and ``ld_table`` as for :func:`attn_decode`; no sequence
    has more than ``max_q`` queries or ``max_len`` tokens. ``dtype`` "bf16" or
    "f16"; ``out_dtype`` the same (default) or "f32"."""
    hd, n, tq, most = cache.head_dim, int(seqs), int(tokens_q), int(max_len)
    nq = q_heads * hd
    lq, lo = ld_q or nq, ld_out or nq
    per = (most + cache.page_tokens - 1) // cache.page_tokens
    lt = ld_table or (table.stride(0) if getattr(table, "ndim", 0) == 2 and hasattr(table, "stride") else per)
    ti = vtype_id(dtype)
    oi = ti if out_dtype is None else vtype_id(out_dtype)
    check(lib().frq_dev_attn_chunk(
        ti, _operand("q", q, 2 * ((tq - 1) * lq + nq) if tq else 0, ti, lq), lq, cache.data_ptr(), cache.nbytes, cache.pages,
        cache.page_tokens, cache.kv_heads, hd, _operand("table", table, 4 * ((n - 1) * lt + per), _I32, lt), lt,
        _operand("lens", lens, 4 * n, _I32), _operand("cu_q", cu_q, 4 * (n + 1), _I32), n, tq, int(max_q), most, oi,
        _operand("out", out, (4 if oi == 0 else 2) * ((tq - 1) * lo + nq) if tq else 0, oi, lo), lo, q_heads,
        hd ** -0.5 if scale is None else scale, _stream(stream)))


# ------------------------------ between blocks, and from logits to a token

def add_rms_norm(x, out, rows: int, hidden: int, weight=None, residual=None, sum_out=None, eps: float = 1e-6, x_dtype="f32",
                 res_dtype="f32", out_dtype="f32", ld_x: int = 0, ld_res: int = 0, ld_sum: int = 0, ld_out: int = 0,
                 stream=None) -> None:
    """sum_out = x + residual and out = its root-mean-square norm times
    ``weight`` (fp32, None for ones), row by row, enqueued (frq_dev_add_rms_norm).

    ``residual`` None: the norm of x alone. ``sum_out`` (of ``res_dtype``, None:
    not kept) may be the residual itself. ``out_dtype`` "f32", "f16", "bf16" or
    "q8_0": rows of hidden / 32 blocks of 34 bytes, as :func:`dequant` and
    :func:`gemv` read them (a uint8 tensor or a buffer). ``ld_*``: elements from a
    row to the next, default ``hidden``."""
    n, h = int(rows), int(hidden)
    lx, lr, ls, lo = ld_x or h, ld_res or h, ld_sum or h, ld_out or h
    xi, ri = vtype_id(x_dtype), vtype_id(res_dtype)
    q8 = out_dtype == _Q8 or (isinstance(out_dtype, str) and out_dtype.lower() == "q8_0")
    oi = _Q8 if q8 else vtype_id(out_dtype)
    xs, rs = (4 if xi == 0 else 2), (4 if ri == 0 else 2)
    last = (n - 1) * lo + h
    to = (_operand("out", out, last // 32 * 34, _U8, lo // 32 * 34) if q8
          else _operand("out", out, (4 if oi == 0 else 2) * last, oi, lo))
    check(lib().frq_dev_add_rms_norm(
        xi, _operand("x", x, xs * ((n - 1) * lx + h), xi, lx), lx, ri,
        _operand("residual", residual, rs * ((n - 1) * lr + h), ri, lr), lr,
        _operand("sum_out", sum_out, rs * ((n - 1) * ls + h), ri, ls), ls, _operand("weight", weight, 4 * h, _lib.F32), eps, oi,
        to, lo, n, h, _stream(stream)))


def sample(logits, u, tokens, rows: int, vocab: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, probs=None,
           dtype="f32", ld: int = 0, stream=None) -> None:
    """One token (int32) per row of ``logits``, rows ``ld`` elements apart
    (default ``vocab``), drawn with the random numbers ``u`` (fp32 in [0, 1), one a
    row); enqueued (frq_dev_sample).

    The ``top_k`` largest logits stay (0: all), of these the fewest whose
    probabilities at ``temperature`` sum to ``top_p`` of theirs, of these the ones
    at least ``min_p`` times as probable as the largest; temperature 0 takes the
    largest. Each parameter is a number for all rows or a device array of one a row
    (fp32, ``top_k`` int32). ``probs`` (fp32, None: not wanted): the tokens'
    probabilities among those that stayed."""
    n, v = int(rows), int(vocab)
    lx, ti = ld or v, vtype_id(dtype)
    one, many = [], []
    for name, p, kind, rest in (("temperature", temperature, _lib.F32, 1.0), ("top_k", top_k, _I32, 0),
                                ("top_p", top_p, _lib.F32, 1.0), ("min_p", min_p, _lib.F32, 0.0)):
        number = isinstance(p, (int, float, np.integer, np.floating))
        one.append(p if number else rest)
        many.append(0 if number else _operand(name, p, 4 * n, kind))
    check(lib().frq_dev_sample(
        ti, _operand("logits", logits, (4 if ti == 0 else 2) * ((n - 1) * lx + v), ti, lx), lx, n, v,
        _operand("u", u, 4 * n, _lib.F32), float(one[0]), many[0], int(one[1]), many[1], float(one[2]), many[2], float(one[3]), many[3],
        _operand("tokens", tokens, 4 * n, _I32), _operand("probs", probs, 4 * n, _lib.F32), _stream(stream)))
