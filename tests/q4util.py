"""The 4-bit storage mode in plain numpy, and the bounds that results are held to."""
from __future__ import annotations

import numpy as np

from oracle import oracle as O

DT = {"bf16": O.DT_BF16, "f16": O.DT_F16}
EPS = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}  # spacing relative to the value


def quantize(bits: np.ndarray, dt: str):
    """Codes u8 [..., D], scales and biases f16 [..., D/64] of rows of `dt` bits [..., D], from the
    definition, every step rounded as it says."""
    with np.errstate(all="ignore"):
        w = O.bits_to_f32(bits, DT[dt])
        w = w.reshape(*w.shape[:-1], w.shape[-1] // 64, 64)
        nan = np.isnan(w).any(-1, keepdims=True)
        w = np.clip(np.where(np.isnan(w), 0, w), np.float32(-65504), np.float32(65504))
        lo, hi = w.min(-1, keepdims=True) + np.float32(0), w.max(-1, keepdims=True)
        b = lo.astype(np.float16)
        s = (np.maximum(hi - b.astype(np.float32), np.float32(0)) / np.float32(15)).astype(np.float16)
        # (in 64 bits the quotient keeps the side of a tie it lies on)
        c = np.rint((w.astype(np.float64) - b.astype(np.float64)) / np.where(s > 0, s.astype(np.float64), 1.0))
        c = np.where(s > 0, np.clip(c, 0, 15), 0)
    s, b = np.where(nan, np.float16(np.nan), s), np.where(nan, np.float16(np.nan), b)
    return c.astype(np.uint8).reshape(bits.shape), s[..., 0], b[..., 0]


def values(c, s, b):
    """float64 values the codes stand for."""
    g = c.reshape(*c.shape[:-1], c.shape[-1] // 64, 64).astype(np.float64)
    return (g * s.astype(np.float64)[..., None] + b.astype(np.float64)[..., None]).reshape(c.shape)


def stored(bits, dt):
    return values(*quantize(bits, dt))


def read_back(x):
    """float64 values as the cache gives them out: fp16, within its range."""
    with np.errstate(over="ignore"):
        return np.clip(x.astype(np.float32), np.float32(-65504), np.float32(65504)).astype(np.float16)


def attention(q, k, v, lo, hi, scale):
    """float64 [n, D]: row i of q over keys [lo[i], hi[i]) of k, v [T, D]; no key: zeros."""
    out = np.zeros_like(q, dtype=np.float64)
    for i in range(q.shape[0]):
        if hi[i] <= lo[i]:
            continue
        x = k[lo[i]:hi[i]] @ q[i] * scale
        p = np.exp(x - x.max())
        out[i] = p @ v[lo[i]:hi[i]] / p.sum()
    return out


def weight_error(G):
    """What a weight errs by relative, scores' terms up to 8 in log2 units: the roundings of `bound`, half
    as large on average."""
    return (6 * G + 4) * 2.0 ** -24 * 8 + 2.0 ** -19


def bound(q, k, v, scale, want, out, sk=0.0, sv=0.0, long=False):
    """Largest error a row of the kernels' output may show, given float64 q [n, D], k, v [T, D].

    Queries and codes enter the products exactly, so a score errs by the roundings of its sums: per
    group of 64 dims two matrix steps, the scale's and the bias's multiply-add, and two at the end,
    each at most 2^-23 of the sum of the terms' sizes; a weight 2^x errs by as much relative (times
    ln 2) and by 2^-22 in the exponential, its split and the sums; the output by half a step.

    bf16 outputs: weights are rounded to fp16 (2^-11) and weigh |c - 8| s <= 8 sv, sv the largest
    scale of V; codes of K enter as 1024 + c or 1024 + 16 c (over 16 queries), so a group's three
    sums of products, from the offset's start to two matrix steps, are at most 2^-23 of 1040 times
    the group's |q| off, in units of the scale, sk the largest.  Long windows hold k and v as fp16
    numbers s (c - 8) + z, z = b + 8 s rounded too: 2^-11 of |k| and of |z| <= |k| + 8 sk, and
    weights of 2^-11."""
    G = k.shape[-1] // 64
    terms = np.abs(q) @ np.abs(k).max(0) * 2.0  # |s c| and |b| are each at most twice the value's range
    dx = (6 * G + 4) * 2.0 ** -23 * terms * abs(scale) * np.log2(np.e)
    low = 0.0
    if out == "bf16":
        dx = dx + 3 * 2.0 ** -23 * 1040 * np.abs(q).sum(-1) * sk * abs(scale) * np.log2(np.e)
        low = 2.0 ** -11 * 8 * sv
        if long:
            kmax, vmax = np.abs(k).max(), np.abs(v).max()
            dx = dx + 2.0 ** -11 * np.abs(q).sum(-1) * (2 * kmax + 8 * sk) * abs(scale) * np.log2(np.e)
            low = 2.0 ** -11 * (3 * vmax + 8 * sv)
    vmax = 2.0 * np.abs(v).max()
    rel = 2 * np.log(2.0) * dx + 2.0 ** -19
    return (rel * vmax)[:, None] + low + 0.5 * EPS[out] * np.abs(want) + 2.0 ** -25
