"""Plain 64-bit forms of the attention step's operators, in NumPy, and the
bounds that the kernels' arithmetic gives."""

from __future__ import annotations

import numpy as np
import torch

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}    # rounding, relative to the value (2^-p)


def dev(a, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(TORCH[dtype])).cuda()


def f64(t) -> np.ndarray:
    return t.double().cpu().numpy()


def rope(x, hq, hkv, d, rot, interleaved, cs, wq=None, wk=None, eps=1e-6):
    """x (tokens, heads, d) -> q, k, v and the size that errors scale with."""
    x = x.astype(np.float64)
    out, size = [], []
    for lo, hi, w in ((0, hq, wq), (hq, hq + hkv, wk)):
        y = x[:, lo:hi].copy()
        if w is not None:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        r = y.copy()
        mag = np.abs(y)
        if interleaved:
            ia, ib = np.arange(0, rot, 2), np.arange(1, rot, 2)
        else:
            ia, ib = np.arange(rot // 2), np.arange(rot // 2) + rot // 2
        c, s = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
        r[..., ia] = y[..., ia] * c - y[..., ib] * s
        r[..., ib] = y[..., ib] * c + y[..., ia] * s
        both = np.abs(y[..., ia]) + np.abs(y[..., ib])
        mag[..., ia], mag[..., ib] = both, both
        out.append(r)
        size.append(mag)
    v = x[:, hq + hkv:]
    return out + [v], size + [np.abs(v)]


def block4(x) -> np.ndarray:
    """The values that 4-bit blocks of 32 keep of x (finite)."""
    b = np.asarray(x, np.float64).reshape(-1, 32)
    e = b[np.arange(len(b)), np.abs(b).argmax(1)]
    d = np.clip(-e / 8, -65504, 65504).astype(np.float16).astype(np.float64)[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(d == 0, 8, np.clip(np.rint(b / d) + 8, 0, 15))
    return ((code - 8) * d).reshape(np.shape(x))


def attend(q, k, v, scale, last):
    """One head: q (m, d), k and v (n, d), query i sees keys j <= last[i].
    Returns out, sum of p |v| and the largest scale sum |q k| of a row."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    out, mag = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    size = np.zeros(len(q))
    for i in range(len(q)):
        n = min(len(k), int(last[i]) + 1)
        if n <= 0:
            continue
        s = (k[:n] * q[i]).sum(-1) * scale
        size[i] = (np.abs(k[:n]) * np.abs(q[i])).sum(-1).max() * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i] = (p[:, None] * v[:n]).sum(0)
        mag[i] = (p[:, None] * np.abs(v[:n])).sum(0)
    return out, mag, size


def fp32_bound(mag, size, n, d):
    """Scores: products and sums in fp32 (d + 8 roundings of at most 2^-23 of
    scale sum |q k|, q itself kept to 2^-22), so every weight is off by that
    much on both sides of the division; the n weights are rounded (2^-22) and
    summed in fp32, 8 sqrt(n) roundings' worth."""
    score = (d + 8) * 2.0 ** -23 * size + 2.0 ** -22 * size
    return (2 * score[..., None] + 2.0 ** -20 + 8 * np.sqrt(max(n, 1)) * 2.0 ** -24) * mag
