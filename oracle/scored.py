"""Float64 restatement of scored attention and of rotary positions from frequencies, on the CPU.

``scored_attention`` takes ``q (B, Hq, Tq, D)`` and ``k, v (B, Hkv, Tk, D)`` as
float64 and walks the definition: scores of all pairs, a truth value per pair
for each mask, a softmax of what is left, zeros where nothing is.
"""

from __future__ import annotations

import torch


def _each(x, B):
    return [None] * B if x is None else [int(x[b if len(x) > 1 else 0]) for b in range(B)]


def visible(Tq, Tk, causal, window=None, cuts=None, prefix=None, start=None, length=None):
    """Truth values (Tq, Tk) of one sequence."""
    p = torch.arange(Tk - Tq, Tk)[:, None]
    j = torch.arange(Tk)[None, :]
    see = torch.ones(Tq, Tk, dtype=torch.bool)
    if causal:
        see &= (j <= p) | (j < (0 if prefix is None else prefix))
    if window is not None:
        see &= (p - j).abs() < window
    for c in cuts or []:
        see &= (p >= c) == (j >= c)
    if start is not None:
        see &= j >= start
    if length is not None:
        see &= j < length
    return see


def scored_attention(q, k, v, causal=True, sm_scale=None, softcap=None, slopes=None, window=None, cuts=None, prefix=None,
                     start=None, length=None):
    """-> (B, Hq, Tq, D) float64; ``cuts`` a list of positions or one list per sequence."""
    B, Hq, Tq, D = q.shape
    H, Tk = k.shape[1], k.shape[2]
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    prefix, start, length = _each(prefix, B), _each(start, B), _each(length, B)
    out = torch.zeros(B, Hq, Tq, D, dtype=torch.float64)
    dist = (torch.arange(Tk - Tq, Tk)[:, None] - torch.arange(Tk)[None, :]).abs().double()
    for b in range(B):
        cb = cuts[b] if cuts and isinstance(cuts[0], (list, tuple)) else cuts
        see = visible(Tq, Tk, causal, window, cb, prefix[b], start[b], length[b])
        some = see.any(dim=1)
        for h in range(Hq):
            x = (q[b, h] @ k[b, h // (Hq // H)].T) * sm_scale
            if softcap is not None:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * dist
            w = torch.softmax(x[some].masked_fill(~see[some], float("-inf")), dim=1)
            # (a hidden key's value is no part of the sum: a NaN there stays out)
            vv = v[b, h // (Hq // H)]
            hidden = ~see[some].any(dim=0)
            out[b, h, some] = w @ vv.masked_fill(hidden[:, None], 0.0)
    return out


def rope(x, positions, freq, rotary_dim, interleaved=False, scale=1.0):
    """x (B, T, H, D) float64 with the pairs of its first rotary_dim elements turned by positions (B, T) x freq."""
    R = rotary_dim
    angle = positions.double()[:, :, None, None] * freq.double()
    c, s = scale * angle.cos(), scale * angle.sin()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    y = x.clone()
    if interleaved:
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :R // 2], y[..., R // 2:R] = a * c - b * s, b * c + a * s
    return y
