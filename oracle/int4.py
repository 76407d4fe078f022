"""Numpy restatement of the 4-bit K/V format and of attention over it (test oracle).

TEST INFRASTRUCTURE ONLY.  The integer output of the quantiser is defined by
fp32 arithmetic (differences and quotients rounded to fp32) and is reproduced
so, bit for bit; values and attention are float64.
"""

from __future__ import annotations

import numpy as np


def word_place(p: int, D: int) -> int:
    """Place of 32-bit word ``p`` (elements 8p .. 8p + 7) in a row of ``D`` codes."""
    if D == 16:
        return p
    block = min(D, 128)
    n = block // 8
    return (p // n) * n + (p % n % 4) * (block // 32) + p % n // 4


def pack(codes) -> np.ndarray:
    """Codes ``(..., D)`` -> bytes ``(..., D/2)``."""
    c = np.asarray(codes, np.uint8)
    D = c.shape[-1]
    words = np.zeros(c.shape[:-1] + (D // 8, 4), np.uint8)
    for p in range(D // 8):
        e = c[..., 8 * p:8 * p + 8]
        words[..., word_place(p, D), :] = e[..., 0::2] | (e[..., 1::2] << 4)
    return words.reshape(c.shape[:-1] + (D // 2,))


def unpack(packed) -> np.ndarray:
    """Bytes ``(..., D/2)`` -> codes ``(..., D)``."""
    b = np.asarray(packed, np.uint8)
    D = 2 * b.shape[-1]
    words = b.reshape(b.shape[:-1] + (D // 8, 4))
    out = np.zeros(b.shape[:-1] + (D,), np.uint8)
    for p in range(D // 8):
        w = words[..., word_place(p, D), :]
        out[..., 8 * p:8 * p + 8:2] = w & 15
        out[..., 8 * p + 1:8 * p + 8:2] = w >> 4
    return out


def _toward_zero_f16(x32) -> np.ndarray:
    h = x32.astype(np.float16)
    over = h.astype(np.float32) > x32
    return np.where(over, (h.view(np.uint16) - over).astype(np.uint16).view(np.float16), h)


def quantize(x, group: int):
    """fp32 rows ``(..., D)`` -> (codes ``(..., D)`` uint8, parameters ``(..., 2D/group)`` fp16)."""
    f = np.float32
    x = np.asarray(x, f)
    shape = x.shape
    x = x.reshape(-1, shape[-1] // group, group)
    bad = ~np.isfinite(x).all(-1)
    xc = np.clip(np.where(np.isnan(x), f(0), x), f(-65504), f(65504))
    lo, hi = xc.min(-1), xc.max(-1)
    m = lo.astype(np.float16)
    step = np.maximum((hi - m.astype(f)) / f(15), f(0))
    s = _toward_zero_f16(step)
    sf = s.astype(f)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.rint((xc - m.astype(f)[..., None]) / sf)
    n = np.where(sf > 0, np.clip(n, 0, 15), 0)
    n = np.where(bad[..., None], 0, n).astype(np.uint8)
    nan = np.float16(np.nan)
    params = np.stack([np.where(bad, nan, s), np.where(bad, nan, m)], -1)
    return n.reshape(shape), params.reshape(shape[:-1] + (2 * (shape[-1] // group),))


def values(codes, params) -> np.ndarray:
    """What codes ``(..., D)`` and parameters stand for, ``m + n s`` in float64."""
    D = codes.shape[-1]
    p = np.asarray(params, np.float64)
    g = 2 * D // p.shape[-1]
    s, m = np.repeat(p[..., 0::2], g, -1), np.repeat(p[..., 1::2], g, -1)
    return m + codes.astype(np.float64) * s


def decode(q, k, v, n: int, scale: float):
    """Attention of ``q (Hq, D)`` over the first ``n`` of ``k, v (Hkv, S, D)`` in float64.

    Returns the output, ``sum_t w_t |v_t|`` (what a relative error of the weights or values scales with) and the
    largest ``scale sum_i |q_i k_i|`` of each head (what a rounding of the scores scales with).
    """
    Hq, D = q.shape
    G = Hq // k.shape[0]
    out, wabs, sabs = np.zeros((Hq, D)), np.zeros((Hq, D)), np.zeros((Hq, 1))
    if n == 0:
        return out, wabs, sabs
    for h in range(Hq):
        kk, vv = k[h // G, :n], v[h // G, :n]
        s = kk @ q[h] * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h], wabs[h] = w @ vv, w @ np.abs(vv)
        sabs[h] = (np.abs(kk) @ np.abs(q[h])).max() * scale
    return out, wabs, sabs
