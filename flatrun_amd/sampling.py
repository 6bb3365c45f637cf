"""From logits to tokens on the device: what the reference's sampler
(model/sampling.py) does in NumPy on the host for one sequence, for a batch whose
requests have parameters of their own.

    sampler = Sampler(vocab, max_rows=64, stream=stream)
    sampler.plan([dict(temperature=0.7, top_k=50, top_p=0.95), dict(temperature=0.0), ...])
    tokens = sampler(logits, u, rows)          # int32 on the device; u: fp32 in [0, 1), one a row

The kernels are ``device.sample``; the random numbers are the caller's, so that a
run can be repeated."""

from __future__ import annotations

import numpy as np

from . import _lib, device

_FIELDS = {"temperature": (np.float32, 1.0), "top_k": (np.int32, 0), "top_p": (np.float32, 1.0), "min_p": (np.float32, 0.0)}


class Sampler:
    """Parameters and outputs of up to ``max_rows`` rows of logits of ``vocab``.

    ``plan`` fixes the parameters of the rows until the next ``plan``; it waits
    for the stream's earlier draws before it overwrites them. A call can be
    captured in a graph and replayed after later plans of as many rows."""

    def __init__(self, vocab: int, max_rows: int = 1, stream=None):
        if int(vocab) < 1 or int(max_rows) < 1:
            raise ValueError("vocab and max_rows must be at least 1")
        self.vocab, self.max_rows, self.stream = int(vocab), int(max_rows), stream
        self._params = device.DeviceBuffer(4 * len(_FIELDS) * self.max_rows)
        self.tokens, self.probs = device.DeviceBuffer(4 * self.max_rows), device.DeviceBuffer(4 * self.max_rows)
        self.rows = 0

    def plan(self, params) -> None:
        """One dict a row: any of temperature, top_k, top_p and min_p."""
        params = list(params)
        if not 1 <= len(params) <= self.max_rows:
            raise ValueError(f"1..{self.max_rows} rows, got {len(params)}")
        cols = []
        for name, (dtype, default) in _FIELDS.items():
            cols.append(np.full(self.max_rows, default, dtype))
            cols[-1][:len(params)] = [p.get(name, default) for p in params]
        if any(set(p) - set(_FIELDS) for p in params):
            raise ValueError(f"a row's parameters are {', '.join(_FIELDS)}")
        t, k, p, m = (c[:len(params)] for c in cols)
        if not (np.all((t >= 0) & np.isfinite(t)) and np.all(k >= 0) and np.all((p >= 0) & (p <= 1)) and np.all((m >= 0) & (m <= 1))):
            raise ValueError("temperature and top_k must not be negative, top_p and min_p lie in [0, 1]")
        if self.stream is None:                  # earlier draws still read the parameters
            device.synchronize()
        elif hasattr(self.stream, "synchronize"):
            self.stream.synchronize()
        else:
            _lib.check(_lib.lib().frq_stream_synchronize(device._stream(self.stream)))
        host = np.concatenate([c.view(np.uint32) for c in cols])
        _lib.check(_lib.lib().frq_memcpy_h2d(self._params.ptr, host.ctypes.data, host.nbytes))
        self.rows = len(params)

    def __call__(self, logits, u, rows: int, dtype="f32", ld: int = 0):
        """Enqueues the draws of the planned rows; returns the tokens' buffer
        (``probs`` has their probabilities)."""
        if rows != self.rows:
            raise ValueError("plan() these rows first")
        t, k, p, m = (self._params.ptr + 4 * i * self.max_rows for i in range(4))
        device.sample(logits, u, self.tokens, rows, self.vocab, temperature=_At(t), top_k=_At(k), top_p=_At(p), min_p=_At(m),
                      probs=self.probs, dtype=dtype, ld=ld, stream=self.stream)
        return self.tokens

    def close(self) -> None:
        for b in (self._params, self.tokens, self.probs):
            b.free()


class _At:
    """A place on the device (a number would be a parameter's value)."""

    def __init__(self, ptr: int):
        self.ptr = ptr

    def data_ptr(self) -> int:
        return self.ptr
