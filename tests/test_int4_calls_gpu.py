"""The 4-bit cache's calls at the edges of what they take: long shares, extreme queries, dead rows beside NaN, offsets
past 32 bits, shared pages, strides, graphs.  Tolerances as in test_int4_gpu.py unless said otherwise."""

from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from helpers import announce, f64
from oracle import int4 as I4
from test_int4_gpu import BF16, DEV, FP16, FP32, cache_case, check_decode, gen, pools, quant, randn, rounded, same

pytestmark = pytest.mark.gpu
PKG = "simple-inference-autoresearch_amd"


def lens_tensor(lens):
    return torch.tensor(lens, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("D,group,page", [(64, 32, 16), (128, 64, 0), (128, 128, 64), (256, 64, 16)])
def test_one_wave_walks_hundreds_of_tiles(gpu_pkg, D, group, page):
    """The whole batch in one share: every wave takes all tiles of a head, far more than the 64 page ids it holds."""
    announce(f"int4 decode long shares D {D} page {page}")
    lens, H = [4113, 1, 0, 2048, 1039], 8
    c = cache_case(gpu_pkg, D, len(lens), H, D, group, max(lens), page)
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(4), len(lens), 2 * H, 1, D)
    with gpu_pkg.decode_options(tiles_per_split=100000):
        out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    check_decode(out, q, k, v, lens, "one share", True)


@pytest.mark.parametrize("D,group", [(64, 32), (128, 32), (128, 64), (128, 128), (256, 32), (256, 128)])
@pytest.mark.parametrize("heads", [(8, 8), (24, 2)])
def test_dead_rows_beside_nan(gpu_pkg, D, group, heads):
    """Sequences that end inside a tile, walked by the waves that read another sequence's NaN just before."""
    announce(f"int4 decode NaN neighbours D {D} group {group} heads {heads}")
    lens = [97, 17, 96, 1, 97, 15, 33]
    c = cache_case(gpu_pkg, D + 1, len(lens), heads[1], D, group, 97, 16)
    for b in (0, 2, 4):
        c.k[b, :, ::3, 5] = float("nan")
        c.v[b, :, 1::3, D - 1] = float("inf")
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(4), len(lens), heads[0], 1, D)
    with gpu_pkg.decode_options(tiles_per_split=100000):
        out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    live = [1, 3, 5, 6]
    check_decode(out[live], q[live], [k[b] for b in live], [v[b] for b in live], [lens[b] for b in live], "clean", True)
    assert torch.isnan(out[[0, 2, 4]]).any(-1).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [4, 12])
def test_minimum_and_query_sum_keep_their_bits(gpu_pkg, D, G):
    """A score that is left over when the parts of it, 2^14 times as large, cancel.

    Keys and queries are small integers and halves, so every score is exact in fp32.  Token 0 is -60 everywhere but at
    element 0 (0 there: step 4, code 15); token 1 is 0.  The query is 8192 at element 0 and 0.25 at element 1: scores
    -15 and 0.  Values 1 and 0: the output is token 0's weight, with one rounding of it (2^-11), and one of the result.
    """
    announce(f"int4 cancelling scores D {D} G {G}")
    k, v = torch.zeros(1, 1, 2, D, dtype=BF16, device=DEV), torch.zeros(1, 1, 2, D, dtype=BF16, device=DEV)
    k[0, 0, 0, :32] = -60
    k[0, 0, 0, 0] = 0
    v[0, 0, 0] = 1
    (kc, ks), (vc, vs) = (gpu_pkg.quantize_kv_int4(t, 32) for t in (k, v))
    assert torch.equal(gpu_pkg.dequantize_kv_int4(kc, ks), k)
    q = torch.zeros(1, G, 1, D, dtype=BF16, device=DEV)
    q[..., 0], q[..., 1] = 8192, 0.25
    out = gpu_pkg.attention_flash_decode_int4(q, kc, vc, ks, vs, 2, 0.125)
    want = 1 / (1 + np.exp(15 * 0.125))
    # (fp16 weight 2^-11, bf16 result 2^-8 + 2^-24's)
    assert (np.abs(f64(out) - want) <= want * (2.0 ** -8 + 2.0 ** -10)).all()


@pytest.mark.parametrize("D,page", [(64, 0), (128, 16), (256, 16), (128, 24)])
@pytest.mark.parametrize("scale", [2.0 ** 120, 2.0 ** 60, 2.0 ** -120])
def test_queries_of_extreme_size(gpu_pkg, D, page, scale):
    """Huge queries pick one token, tiny ones weigh all tokens alike."""
    announce(f"int4 decode queries x {scale} D {D} page {page}")
    lens = [130, 50]
    c = cache_case(gpu_pkg, D + 3, 2, 2, D, 32, 130, page)
    k, v = c.fill(gpu_pkg, lens)
    # (|q k| stays below fp32's largest number: 2^120 x 5 x 256 x ... would not)
    q = (torch.randn(2, 8, 1, D, generator=gen(2), device=DEV) * 2.0 ** -6).to(BF16) * scale
    out = f64(c.run(gpu_pkg, q.to(BF16), lens_tensor(lens)))
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        for h in range(8):
            s = f64(q)[b, h, 0] @ k[b][h // 4][:n].T * D ** -0.5
            w = np.exp(s - s.max())
            w /= w.sum()
            assert scale < 1 or np.sort(w)[-2] < 1e-30        # one token stands alone
            ref, wabs = w @ v[b][h // 4][:n], w @ np.abs(v[b][h // 4][:n])
            # weights and values rounded to fp16, fp32 sums of up to 130 weights, the result to bf16
            assert (np.abs(out[b, 0, h] - ref) <= (2.0 ** -10 + 130 * 2.0 ** -23) * wabs + 2.0 ** -8 * (np.abs(ref) + wabs * 2.0 ** -9)).all()


@pytest.mark.parametrize("T", [1, 15, 16, 17, 33])
@pytest.mark.parametrize("D,group", [(16, 16), (32, 32), (64, 32), (64, 64), (128, 128), (256, 32)])
def test_write_lengths(gpu_pkg, D, group, T):
    """Row orders of short and long writes, with sequences that begin before the cache and end behind it."""
    announce(f"kv_write int4 D {D} group {group} T {T}")
    B, H, S = 4, 3, 40
    g = gen(D + T)
    k, v = randn(g, B, H, T, D), randn(g, B, H, T, D)
    (kc, ks), (vc, vs) = pools(B, H, S, D, group), pools(B, H, S, D, group)
    want = [t.cpu().numpy().copy() for t in (kc, ks, vc, vs)]
    src = [*quant(k, group), *quant(v, group)]
    first = [0, -4, S - 3, 1 << 30]
    for b, at in enumerate(first):
        for t in range(T):
            if 0 <= at + t < S:
                for w, s in zip(want, src):
                    w[b, :, at + t] = s[b, :, t]
    gpu_pkg.kv_write(k, v, kc, vc, ks, vs, start_pos=lens_tensor(first))
    torch.cuda.synchronize()
    for got, ref in zip((kc, ks, vc, vs), want):
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
    rk, rv = gpu_pkg.kv_read(kc, vc, T, ks, vs, start_pos=lens_tensor(first), dtype=FP32)
    for b, at in enumerate(first):
        for t in range(T):
            for r, (codes, par) in ((rk, src[:2]), (rv, src[2:])):
                ref = I4.values(I4.unpack(codes[b, :, t]), par[b, :, t]) if 0 <= at + t < S else np.zeros((H, D))
                np.testing.assert_array_equal(r[b, :, t].cpu().numpy(), ref.astype(np.float32))


def test_pages_shared_between_sequences(gpu_pkg):
    """Two sequences whose tables name the same pages, and one that names a page twice."""
    announce("int4 shared pages")
    B, H, D, n = 2, 4, 128, 80
    c = cache_case(gpu_pkg, 21, B, H, D, 64, n, 16)
    k, v = c.fill(gpu_pkg, [n, n])
    bt = torch.stack([c.bt[0], c.bt[0], c.bt[1], c.bt[1]]).clone()
    bt[3, 1] = bt[3, 0]
    kk, vv = [k[0], k[0], k[1], k[1].copy()], [v[0], v[0], v[1], v[1].copy()]
    for t in (kk[3], vv[3]):
        t[:, 16:32] = t[:, :16]
    q = randn(gen(2), 4, 8, 1, D)
    lens = [n, n - 5, 3, n]
    out = gpu_pkg.paged_gqa_int4_flash_decode(q, c.kc, c.vc, c.ks, c.vs, bt, lens_tensor(lens), 16)
    torch.cuda.synchronize()
    check_decode(out, q, kk, vv, lens, "shared pages", True)
    rk, _ = gpu_pkg.kv_read(c.kc, c.vc, 32, c.ks, c.vs, block_table=bt, page_size=16, dtype=FP32)
    assert torch.equal(rk[3, :, 16:], rk[3, :, :16]) and torch.equal(rk[0], rk[1])


def test_pool_past_32_bits(gpu_pkg):
    """Pages whose byte offsets in the pool need more than 32 bits."""
    announce("int4 pool beyond 4 GiB")
    P, H, page, D, group, n = 530_000, 8, 16, 128, 64, 70
    kc, vc = (torch.empty(P, H, page, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(P, H, page, 4, dtype=FP16, device=DEV) for _ in range(2))
    assert kc.numel() > 1 << 32 and ks.numel() * 2 > 1 << 29
    bt = torch.tensor([[P - 1, 3, P - 70, 525_000, P - 2]], dtype=torch.int32, device=DEV)
    g = gen(1)
    k, v = randn(g, 1, H, n, D), randn(g, 1, H, n, D)
    gpu_pkg.kv_write(k, v, kc, vc, ks, vs, block_table=bt, page_size=page)
    rk, rv = gpu_pkg.kv_read(kc, vc, n, ks, vs, block_table=bt, page_size=page, dtype=FP32)
    ref = [I4.values(*I4.quantize(t[0].float().cpu().numpy(), group)) for t in (k, v)]
    assert torch.equal(rk[0], rounded(ref[0], FP32)) and torch.equal(rv[0], rounded(ref[1], FP32))
    for q, matrix in ((randn(g, 1, 16, 1, D), True), (randn(g, 1, 16, 1, D, dtype=FP32), False)):
        out = gpu_pkg.paged_gqa_int4_flash_decode(q, kc, vc, ks, vs, bt, lens_tensor([n]), page)
        torch.cuda.synchronize()
        check_decode(out, q, [ref[0]], [ref[1]], [n], "large pool", matrix)


def test_sequence_past_32_bits(gpu_pkg):
    """One head whose row of tokens is longer than 4 GiB.  All tokens but the last 64 are zero, and those score so much
    higher that the zeros' share is below 70e6 e^-40, so the answer is the attention over the last 64."""
    announce("int4 cache row beyond 4 GiB")
    S, D, group, last = 70_000_000, 128, 128, 64
    kc, vc = (torch.zeros(1, 1, S, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(1, 1, S, 2, dtype=FP16, device=DEV) for _ in range(2))
    g = gen(8)
    q = randn(g, 1, 4, 1, D)
    k = (q[0, :1].float() * 0.5 + torch.randn(1, last, D, generator=g, device=DEV) * 0.01).to(BF16)[None]
    v = randn(g, 1, 1, last, D)
    q = q[:, :1].expand(1, 4, 1, D).contiguous()
    gpu_pkg.kv_write(k, v, kc, vc, ks, vs, start_offset=S - last)
    rk, rv = gpu_pkg.kv_read(kc, vc, last, ks, vs, start_offset=S - last, dtype=FP32)
    kx, vx = (I4.values(*I4.quantize(t[0].float().cpu().numpy(), group)) for t in (k, v))
    assert torch.equal(rk[0], rounded(kx, FP32)) and torch.equal(rv[0], rounded(vx, FP32))
    scale = 1.0
    assert (f64(q)[0, 0, 0] @ kx[0].T * scale).min() > 40
    out = gpu_pkg.attention_flash_decode_int4(q, kc, vc, ks, vs, S, scale)
    torch.cuda.synchronize()
    check_decode(out, q, [kx], [vx], [last], "long row", True, scale)


def test_refused_layouts(gpu_pkg):
    announce("int4 refused layouts")
    c = cache_case(gpu_pkg, 5, 2, 2, 128, 64, 32, 0)
    c.fill(gpu_pkg, [32, 32])
    q, kl = randn(gen(1), 2, 8, 1, 128), lens_tensor([32, 32])
    wide = torch.zeros(2, 2, 40, 64, dtype=torch.uint8, device=DEV)[:, :, :32]
    widep = torch.zeros(2, 2, 40, 4, dtype=FP16, device=DEV)[:, :, :32]
    for args in ((c.kc, wide, c.ks, c.vs), (c.kc, c.vc, c.ks, widep)):
        with pytest.raises(NotImplementedError):
            gpu_pkg.attention_flash_decode_int4(q, *args, kl)
        with pytest.raises(ValueError):
            gpu_pkg.kv_read(args[0], args[1], 4, args[2], args[3])
    for kw in (dict(start_offset=1 << 32), dict(start_offset=-(1 << 32))):
        with pytest.raises(ValueError):
            gpu_pkg.kv_read(c.kc, c.vc, 4, c.ks, c.vs, **kw)
    out = tuple(torch.empty(2, 2, 4, 128, dtype=BF16, device=DEV) for _ in range(2))
    for bad in ((out[0], None), (out[0][:, :, :3], out[1][:, :, :3]), (out[0], out[1].float()), (out[0].cpu(), out[1].cpu())):
        with pytest.raises(ValueError):
            gpu_pkg.kv_read(c.kc, c.vc, 4, c.ks, c.vs, out=bad)
    with pytest.raises(ValueError):
        gpu_pkg.kv_read(c.kc, c.vc, 4, c.ks, c.vs, out=out, dtype=FP32)
    with pytest.raises(ValueError):
        gpu_pkg.dequantize_kv_int4(c.kc, c.ks[:1])
    cache = gpu_pkg.KVCache(1, 2, 64, 2, 64, device=DEV, kv_dtype="int4")
    qk = randn(gen(2), 2, 2, 10, 64)
    for start in (-1, 60):
        with pytest.raises((AssertionError, ValueError)):
            gpu_pkg.prefill_step_attention(qk, qk, qk, cache, 0, start)


def test_two_graphs_and_eager_calls(gpu_pkg):
    """Two captured graphs (decode, read, prompt chunk) replayed in turn with eager work between, results bit-equal."""
    announce("int4 in two graphs")
    B, Hq, H, D = 2, 8, 4, 128
    g = gen(12)
    jobs = []
    for i in range(2):
        cache = gpu_pkg.KVCache(1, B, 200, H, D, device=DEV, kv_dtype="int4", group_size=32 << i)
        ctx = gpu_pkg.DecodeCtx(D, DEV)
        k0, v0 = randn(g, B, H, 90, D), randn(g, B, H, 90, D)
        cache.update(0, 0, k0, v0)
        io = [randn(g, B, n, t, D) for n, t in ((Hq, 1), (H, 1), (H, 1), (Hq, 12), (H, 12), (H, 12))]

        def step(cache=cache, ctx=ctx, io=io):
            chunk = gpu_pkg.prefill_step_attention(io[3], io[4], io[5], cache, 0, 90)
            return gpu_pkg.decode_step_attention(io[0], io[1], io[2], cache, 0, ctx), chunk, *cache.read(0, B, 70, 40)

        jobs.append((step, ctx, io))
    graphs = []
    for step, ctx, io in jobs:
        ctx.set_position(102)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for r in range(4):
        for (step, ctx, io), (graph, outs) in zip(jobs, graphs):
            for t in io:
                t.copy_(randn(g, *t.shape))
            ctx.set_position(102 + r)
        for (step, ctx, io), (graph, outs) in zip(jobs, graphs):
            graph.replay()
        got = [[t.clone() for t in outs] for _, outs in graphs]
        torch.cuda.synchronize()
        for (step, ctx, io), copies in zip(jobs, got):
            for a, b in zip(copies, step()):
                assert same(a, b), r
        torch.cuda.synchronize()


def test_prompt_of_no_tokens_and_batches_of_none(gpu_pkg):
    announce("int4 empty calls")
    cache = gpu_pkg.KVCache(1, 2, 64, 2, 64, device=DEV, kv_dtype="int4")
    e = torch.empty(2, 2, 0, 64, dtype=BF16, device=DEV)
    cache.update(0, 5, e, e)
    assert cache.read(0, 2, 0)[0].shape == (2, 2, 0, 64) and not cache.k_scale.any()
    assert cache.read(0, 0, 3)[1].shape == (0, 2, 3, 64)
    p = gpu_pkg.PagedKVCache(1, 2, 64, 2, 64, device=DEV, kv_dtype="int4")
    assert p.read(0, 0, 3)[1].shape == (0, 2, 3, 64)
    k, v = gpu_pkg.kv_read(cache.k_cache[0], None, 64, cache.k_scale[0])
    assert v is None and not k.any()
    codes, par = gpu_pkg.quantize_kv_int4(e)
    assert gpu_pkg.dequantize_kv_int4(codes, par).shape == e.shape


@pytest.mark.parametrize("B", [4200, 8192, 8193])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 24), (256, 0)])
def test_large_batches(gpu_pkg, B, D, page):
    """Thousands of short sequences: plans whose lengths, and then whose prefix, do not fit into LDS."""
    announce(f"int4 decode batch {B} D {D} page {page}")
    c = cache_case(gpu_pkg, D, B, 1, D, 32, 20, page)
    lens = [(7 * b) % 21 for b in range(B)]
    if page:
        gpu_pkg.kv_write(c.k, c.v, c.kc, c.vc, c.ks, c.vs, block_table=c.bt, page_size=page)
    else:
        gpu_pkg.kv_write(c.k, c.v, c.kc, c.vc, c.ks, c.vs)
    q = randn(gen(4), B, 2, 1, D)
    out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    some = list(range(0, B, 97)) + [B - 1]
    k, v = (I4.values(*I4.quantize(t[some].float().cpu().numpy(), 32)) for t in (c.k, c.v))
    check_decode(out[some], q[some], k, v, [lens[b] for b in some], "large batch", B <= 8192)
    assert (out[lens.index(0)::21] == 0).all()


@pytest.mark.parametrize("D,page,qdt", [(128, 0, BF16), (64, 16, FP16), (128, 24, BF16), (128, 16, FP32)])
def test_lengths_past_the_cache(gpu_pkg, D, page, qdt):
    """A kv_len beyond the capacity counts as the capacity, a negative one as none."""
    announce(f"int4 decode lengths past the cache D {D} page {page} {qdt}")
    S = 96
    c = cache_case(gpu_pkg, D, 3, 2, D, 32, S, page)
    c.fill(gpu_pkg, [S] * 3)
    q = randn(gen(4), 3, 8, 1, D, dtype=qdt)
    a = c.run(gpu_pkg, q, lens_tensor([S, 1 << 30, -5]))
    b = c.run(gpu_pkg, q, lens_tensor([S, S, 0]))
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.isfinite(a).all() and (a[2] == 0).all()
    assert torch.equal(c.run(gpu_pkg, q, 2 ** 31 - 1), c.run(gpu_pkg, q, S))


def test_strides_of_dims_of_one(gpu_pkg):
    """Dims of size 1 have no stride to compare."""
    announce("int4 dims of one")
    H, S, D = 2, 40, 128
    c = cache_case(gpu_pkg, 5, 1, H, D, 64, S, 0)
    c.fill(gpu_pkg, [S])
    other = [t.new_zeros(3, *t.shape[1:]) for t in (c.vc, c.vs)]
    for o, t in zip(other, (c.vc, c.vs)):
        o[1] = t[0]
    vc, vs = (o.as_strided(t.shape, (80, *o.stride()[1:]), o.stride(0)) for o, t in zip(other, (c.vc, c.vs)))
    q = randn(gen(4), 1, 4, 1, D)
    a = gpu_pkg.attention_flash_decode_int4(q, c.kc, vc, c.ks, vs, S)
    b = gpu_pkg.attention_flash_decode_int4(q, c.kc, c.vc, c.ks, c.vs, S)
    assert torch.equal(a, b)
    x = gpu_pkg.kv_read(c.kc, vc, S, c.ks, vs)
    y = gpu_pkg.kv_read(c.kc, c.vc, S, c.ks, c.vs)
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,group,T,table", [(16, 16, 20, FP32), (32, 32, 3, BF16), (64, 32, 33, FP32), (128, 128, 17, FP16),
                                             (256, 32, 16, FP32)])
def test_rope_write_positions(gpu_pkg, D, group, T, table, interleaved):
    """Sequences at their own positions, paged, long and short writes, tables of other types: RoPE, then the plain write.
    Positions past the table are not written."""
    announce(f"rope_kv_write int4 D {D} T {T} table {table} interleaved {interleaved}")
    B, Hq, H, page, rows = 3, 4, 2, 24, 60
    g = gen(D + T)
    dt = FP16 if table == FP16 else BF16
    q, k, v = randn(g, B, T, Hq, D, dtype=dt), randn(g, B, T, H, D, dtype=dt), randn(g, B, T, H, D, dtype=dt)
    cos, sin = gpu_pkg.RopeFrequencies(D, rows, device=torch.device(DEV)).get(rows, dtype=table)
    first = [0, 7, rows - 2]
    bt = torch.randperm(12, generator=torch.Generator().manual_seed(D))[:9].view(3, 3).to(torch.int32).to(DEV)
    (kc, ks), (vc, vs), (kc2, ks2), (vc2, vs2) = (pools(12, H, page, D, group) for _ in range(4))
    qr = gpu_pkg.rope_kv_write(q, k, v, cos, sin, kc, vc, ks, vs, block_table=bt, start_pos=lens_tensor(first),
                               page_size=page, interleaved=interleaved)
    for b, at in enumerate(first):
        n = min(T, rows - at)
        q2, k2 = gpu_pkg.rope_triton(q[b:b + 1, :n], k[b:b + 1, :n], cos[at:at + n], sin[at:at + n], interleaved=interleaved)
        assert torch.equal(qr[b:b + 1, :n], q2) and not qr[b, n:].any()
        gpu_pkg.kv_write(k2.transpose(1, 2).contiguous(), v[b:b + 1, :n].transpose(1, 2).contiguous(), kc2,
                         vc2, ks2, vs2, block_table=bt[b:b + 1], start_offset=at, page_size=page)
    torch.cuda.synchronize()
    for x, y in ((kc, kc2), (ks, ks2), (vc, vc2), (vs, vs2)):
        assert torch.equal(x, y)
