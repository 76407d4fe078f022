"""Writes through K and V tensors whose strides differ in dims of size 1 only, which have no stride to compare."""

from __future__ import annotations

import pytest
import torch

from helpers import announce
from test_int4_gpu import BF16, DEV, FP16, FP32, gen, randn

pytestmark = pytest.mark.gpu
D, GROUP, S = 128, 64, 40


def other_strides(t):
    """The same elements, the strides of dims of size 1 changed (to ones that keep rows aligned); None for None."""
    if t is None:
        return None
    return t.as_strided(t.shape, [s if n > 1 else 16 * 7 for n, s in zip(t.shape, t.stride())], t.storage_offset())


def cache(kind, B, H):
    """k, v and their scales or parameters, zeroed."""
    if kind == "int4":
        mk, par = (lambda: torch.zeros(B, H, S, D // 2, dtype=torch.uint8, device=DEV)), (B, H, S, 2 * D // GROUP)
    else:
        mk, par = (lambda: torch.zeros(B, H, S, D, dtype=kind, device=DEV)), (B, H, S)
    sc = [torch.zeros(par, dtype=FP16, device=DEV) for _ in range(2)] if kind in ("int4", torch.int8) else [None, None]
    return [mk(), mk(), *sc]


@pytest.mark.parametrize("kind", ["int4", torch.int8, BF16])
@pytest.mark.parametrize("B,H,T", [(1, 1, 1), (1, 2, 3), (2, 1, 1), (3, 2, 1)])
def test_write(gpu_pkg, kind, B, H, T):
    announce(f"kv_write dims of one {kind} {B} {H} {T}")
    g = gen(B + H + T)
    k, v = randn(g, B, H, T, D), randn(g, B, H, T, D)
    a, b = cache(kind, B, H), cache(kind, B, H)
    gpu_pkg.kv_write(k, v, *a, start_offset=5)
    kd, vd, ks, vs = b
    gpu_pkg.kv_write(k, other_strides(v), kd, other_strides(vd), ks, other_strides(vs), start_offset=5)
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        assert x is None or torch.equal(x, y)
    assert a[0].any()
    if kind == "int4":                                               # what was written reads back and decodes
        rk, rv = gpu_pkg.kv_read(kd, other_strides(vd), T, ks, other_strides(vs), start_offset=5)
        want = gpu_pkg.kv_read(a[0], a[1], T, a[2], a[3], start_offset=5)
        assert torch.equal(rk, want[0]) and torch.equal(rv, want[1])


@pytest.mark.parametrize("kind", ["int4", torch.int8])
@pytest.mark.parametrize("page", [0, 16])
def test_rope_write(gpu_pkg, kind, page):
    """One sequence, one token, one KV head: every dim but head_dim is of size 1."""
    announce(f"rope_kv_write dims of one {kind} page {page}")
    g = gen(page)
    q, k, v = randn(g, 1, 1, 2, D), randn(g, 1, 1, 1, D), randn(g, 1, 1, 1, D)
    cos, sin = gpu_pkg.RopeFrequencies(D, S, device=torch.device(DEV)).get(S, dtype=FP32)
    a, b = cache(kind, 1, 1), cache(kind, 1, 1)
    kw = dict(start_offset=3)
    if page:                                                         # the cache as a pool of one page
        a, b = ([t if t is None else t[:, :, :page] for t in c] for c in (a, b))
        kw.update(block_table=torch.zeros(1, 1, dtype=torch.int32, device=DEV), page_size=page)
    q1 = gpu_pkg.rope_kv_write(q, k, v, cos, sin, *a, **kw)
    kd, vd, ks, vs = b
    q2 = gpu_pkg.rope_kv_write(q, k, other_strides(v), cos, sin, kd, other_strides(vd), ks, other_strides(vs), **kw)
    torch.cuda.synchronize()
    assert torch.equal(q1, q2) and all(torch.equal(x, y) for x, y in zip(a, b)) and a[0].any()


def test_differing_strides_stay_refused(gpu_pkg):
    announce("kv_write differing strides")
    g = gen(1)
    k, v = randn(g, 2, 2, 3, D), randn(g, 2, 3, 2, D).transpose(1, 2)
    kd, vd, ks, vs = cache("int4", 2, 2)
    with pytest.raises(ValueError):
        gpu_pkg.kv_write(k, v, kd, vd, ks, vs)
    with pytest.raises(ValueError):
        gpu_pkg.kv_write(k, k, kd, vd.transpose(1, 2).contiguous().transpose(1, 2), ks, vs)
