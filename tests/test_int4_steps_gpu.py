"""Whole decode steps over 4-bit caches, and large batches of every short length.  Tolerances as in test_int4_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import announce
from oracle import int4 as I4
from test_int4_gpu import BF16, DEV, FP16, FP32, cache_case, check_decode, gen, randn

pytestmark = pytest.mark.gpu
POOLS = ("k_cache", "v_cache", "k_scale", "v_scale")


def caches(gpu_pkg, n, layers, batch, S, H, D, group, seed):
    """n equal 4-bit caches whose every layer holds S tokens."""
    out = [gpu_pkg.KVCache(layers, batch, S, H, D, device=DEV, kv_dtype="int4", group_size=group) for _ in range(n)]
    g = gen(seed)
    for layer in range(layers):
        k, v = randn(g, batch, H, S, D), randn(g, batch, H, S, D)
        for c in out:
            c.update(layer, 0, k, v)
    return out


def unfused(gpu_pkg, q, k, v, cos, sin, at, cache, layer, ctx):
    """RoPE of every sequence by its own table row, then the step on rotated q and k."""
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    for b, p in enumerate(at):
        qr[b:b + 1], kr[b:b + 1] = gpu_pkg.rope_triton(q[b:b + 1], k[b:b + 1], cos[p:p + 1], sin[p:p + 1])
    return gpu_pkg.decode_step_attention(qr.transpose(1, 2), kr.transpose(1, 2), v.contiguous().transpose(1, 2), cache,
                                         layer, ctx)


@pytest.mark.parametrize("D,group,heads,dtype", [(128, 64, (32, 8), BF16), (64, 32, (8, 8), FP16), (256, 128, (4, 2), BF16),
                                                 (32, 32, (8, 2), BF16), (128, 32, (8, 1), FP32)])
@pytest.mark.parametrize("layer,B", [(0, 4), (1, 3), (-1, 1)])
def test_rope_step(gpu_pkg, D, group, heads, dtype, layer, B):
    """rope_decode_step_attention over KVCache(kv_dtype="int4"): RoPE, write and attention of one layer, its first B
    sequences at their own positions; the other layers and sequences as they were."""
    announce(f"rope step int4 D {D} heads {heads} {dtype} layer {layer} B {B}")
    S, (Hq, H) = 300, heads
    a, b = caches(gpu_pkg, 2, 2, 4, S, H, D, group, D)
    cos, sin = gpu_pkg.RopeFrequencies(D, S, device=torch.device(DEV)).get(S, dtype=FP32 if dtype == FP32 else dtype)
    at = [100, S - 1, 0, 7][:B]
    ctx = gpu_pkg.DecodeCtx(D, DEV, batch=B, per_sequence=True)
    ctx.set_position(torch.tensor(at, dtype=torch.int32, device=DEV))
    g = gen(B)
    q, k, v = (randn(g, B, 1, n, D, dtype=dtype) for n in (Hq, H, H))
    out = gpu_pkg.rope_decode_step_attention(q, k, v, cos, sin, a, layer, ctx)
    want = unfused(gpu_pkg, q, k, v, cos, sin, at, b, layer, ctx)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and out.shape == (B, 1, Hq, D) and torch.isfinite(out).all()
    for name in POOLS:
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    q2 = a.write_decode_rope(layer, ctx.pos_index, q, k, v, cos, sin)         # the same token again: nothing changes
    torch.cuda.synchronize()
    assert q2.shape == q.shape and all(torch.equal(getattr(a, name), getattr(b, name)) for name in POOLS)
    kx, vx = ([I4.values(I4.unpack(getattr(a, c)[layer, i].cpu().numpy()), getattr(a, p)[layer, i].cpu().numpy())
               for i in range(B)] for c, p in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
    check_decode(out, q2.transpose(1, 2), kx, vx, [p + 1 for p in at], "step", dtype != FP32 and D >= 64)


def test_rope_step_in_a_graph(gpu_pkg):
    """One captured step, replayed at new positions: every replay equals the eager unfused step, output and cache."""
    announce("rope step int4 in a HIP graph")
    B, Hq, H, D, S = 3, 32, 8, 128, 600
    a, b = caches(gpu_pkg, 2, 1, B, S, H, D, 64, 1)
    cos, sin = gpu_pkg.RopeFrequencies(D, S, device=torch.device(DEV)).get(S, dtype=BF16)
    ctx = gpu_pkg.DecodeCtx(D, DEV, batch=B, per_sequence=True)
    q, k, v = (torch.zeros(B, 1, n, D, dtype=BF16, device=DEV) for n in (Hq, H, H))
    saved = [getattr(a, name).clone() for name in POOLS]
    ctx.set_position(torch.tensor([10, 20, 30], dtype=torch.int32, device=DEV))
    gpu_pkg.rope_decode_step_attention(q, k, v, cos, sin, a, 0, ctx)          # warm-up outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu_pkg.rope_decode_step_attention(q, k, v, cos, sin, a, 0, ctx)
    for name, t in zip(POOLS, saved):
        getattr(a, name).copy_(t)
    g = gen(5)
    for i, at in enumerate(([10, 20, 30], [11, 200, 31], [12, 201, S - 1], [400, 7, 0])):
        ctx.set_position(torch.tensor(at, dtype=torch.int32, device=DEV))
        for t in (q, k, v):
            t.copy_(randn(g, *t.shape))
        graph.replay()
        want = unfused(gpu_pkg, q, k, v, cos, sin, at, b, 0, ctx)
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {i}"
        for name in POOLS:
            assert torch.equal(getattr(a, name), getattr(b, name)), f"replay {i}: {name}"


@pytest.mark.parametrize("B", [4200, 8192, 8193])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 24), (256, 0)])
def test_large_batches_of_every_length(gpu_pkg, B, D, page):
    """Thousands of sequences of 0 to 40 tokens: none, one, two and three tiles, tile and page boundaries, in plans whose
    lengths, and then whose prefix, do not fit into LDS."""
    announce(f"int4 decode batch {B} of every length D {D} page {page}")
    S = 40
    c = cache_case(gpu_pkg, D, B, 1, D, 32, S, page)
    lens = [(17 * b) % (S + 1) for b in range(B)]                              # (17 and 41 have no common factor)
    gpu_pkg.kv_write(c.k, c.v, c.kc, c.vc, c.ks, c.vs, block_table=c.bt, page_size=page)
    q = randn(gen(4), B, 2, 1, D)
    out = c.run(gpu_pkg, q, torch.tensor(lens, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    some = list(range(0, B, 97)) + [B - 1]
    assert {lens[b] for b in some} == set(range(S + 1))
    k, v = (I4.values(*I4.quantize(t[some].float().cpu().numpy(), 32)) for t in (c.k, c.v))
    check_decode(out[some], q[some], k, v, [lens[b] for b in some], "every length", B <= 8192)
    empty = np.flatnonzero(np.array(lens) == 0)
    assert len(empty) > 100 and (out[empty] == 0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("D,page,qdt", [(128, 16, BF16), (64, 0, FP16), (256, 16, BF16), (128, 24, BF16), (128, 16, FP32),
                                        (32, 0, BF16)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_nothing_but_nan(gpu_pkg, D, page, qdt, what):
    """A sequence whose every key (or value) is NaN gives NaN, whoever merges its pieces; its neighbour is as without."""
    announce(f"int4 decode all NaN in {what} D {D} page {page} {qdt}")
    lens, H = [3000, 3000, 1], 2
    c = cache_case(gpu_pkg, D, 3, H, D, 32, 3000, page)
    c.fill(gpu_pkg, lens)
    q = randn(gen(2), 3, 8, 1, D, dtype=qdt)
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for tiles in (0, 3, 100000):
        with gpu_pkg.decode_options(tiles_per_split=tiles):
            clean = c.run(gpu_pkg, q, kl)
            t = getattr(c, what)
            saved = t.clone()
            t[[0, 2]] = float("nan")
            c.fill(gpu_pkg, lens)
            out = c.run(gpu_pkg, q, kl)
            t.copy_(saved)
            c.fill(gpu_pkg, lens)
        torch.cuda.synchronize()
        assert torch.isnan(out[[0, 2]]).all(), tiles
        assert torch.equal(out[1], clean[1]) and torch.isfinite(clean).all(), tiles
