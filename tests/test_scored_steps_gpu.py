"""Scored attention and rotary frequencies as the engine's steps, caches and the transformers hook run them together."""

from __future__ import annotations

import importlib
from types import SimpleNamespace

import pytest
import torch

from helpers import announce, assert_close
from oracle import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def slopes_of(n):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / n) for h in range(n)], device=DEV)


def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


@pytest.mark.parametrize("kv_dtype", [None, torch.int8, "int4"])
def test_a_request_over_a_contiguous_cache(gpu_pkg, kv_dtype):
    """A prompt in two chunks and three decode steps: every output is the scored function's over what the cache holds."""
    B, Hq, H, D, n = 2, 8, 2, 128, 90
    o = dict(softcap=20.0, window=64, alibi_slopes=slopes_of(Hq), kv_start=i32(0, 30))
    cache = gpu_pkg.KVCache(2, B, 200, H, D, kv_dtype=kv_dtype) if kv_dtype else gpu_pkg.KVCache(2, B, 250, H, D)
    if kv_dtype is None:
        cache.is_int8 = False      # (a 16-bit cache of this length)
        cache.k_cache, cache.v_cache = (torch.zeros(2, B, H, 250, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        cache.k_scale = cache.v_scale = None
    announce(f"a request over a cache of {kv_dtype}")
    for start, T in ((0, 60), (60, n - 60)):
        q, k, v = rand(B, Hq, T, D), rand(B, H, T, D), rand(B, H, T, D)
        out = gpu_pkg.prefill_step_attention(q, k, v, cache, 1, start, **o)
        kc, vc = (torch.cat([p, x], 2) for p, x in zip(cache.read(1, B, start), (k, v))) if start else (k, v)
        want = gpu_pkg.scored_attention_flash(q, kc, vc, out_token_major=True, **o)
        assert torch.equal(out.view_as(want), want)
    ctx = gpu_pkg.DecodeCtx(D, DEV)
    rope = gpu_pkg.ScaledRope(D, rope_type="yarn", factor=4.0, original_max_seq_len=64, device=DEV)
    cos, sin = rope.tables(256)
    for step in range(3):
        ctx.set_position(n + step)
        q, k, v = rand(B, 1, Hq, D), rand(B, 1, H, D), rand(B, 1, H, D)
        if step < 2:
            out = gpu_pkg.rope_decode_step_attention(q, k, v, cos, sin, cache, 1, ctx, **o)
            qr = rope(q, None, torch.full((1,), n + step, device=DEV))[0]
            torch.testing.assert_close(gpu_pkg.rope_kv_write(q, k, v, cos, sin, cache.k_cache[1], cache.v_cache[1],
                                       None if kv_dtype is None else cache.k_scale[1], None if kv_dtype is None else cache.v_scale[1],
                                       start_offset=n + step).float(), qr.float(), rtol=2.0 ** -7, atol=1e-5)
            qh = gpu_pkg.rope_kv_write(q, k, v, cos, sin, cache.k_cache[1], cache.v_cache[1],
                                       None if kv_dtype is None else cache.k_scale[1], None if kv_dtype is None else cache.v_scale[1],
                                       start_offset=n + step).transpose(1, 2)
        else:
            qh = q.transpose(1, 2)
            out = gpu_pkg.decode_step_attention(qh, k.transpose(1, 2), v.transpose(1, 2), cache, 1, ctx, **o)
        ks, vs = (None, None) if kv_dtype is None else (cache.k_scale[1], cache.v_scale[1])
        want = gpu_pkg.scored_attention_flash_decode(qh, cache.k_cache[1], cache.v_cache[1], ctx.kv_len, ks, vs, **o)
        assert torch.equal(out, want)
        kd, vd = cache.read(1, B, n + step + 1, dtype=torch.float32)
        ref = S.scored_attention(qh.double().cpu(), kd.double().cpu(), vd.double().cpu(), softcap=20.0, window=64,
                                 slopes=slopes_of(Hq).cpu(), start=[0, 30])
        assert_close(out.transpose(1, 2), ref.numpy(), 2.0 ** -9 * float(vd.abs().max()), "decode step")


@pytest.mark.parametrize("kv_dtype", [None, torch.int8, "int4"])
def test_a_batch_over_a_paged_cache(gpu_pkg, kv_dtype):
    """Captured decode steps of a layer with a window, of requests of different lengths."""
    B, Hq, H, D = 3, 8, 2, 64
    cache = gpu_pkg.PagedKVCache(1, B, 320, H, D, kv_dtype=kv_dtype)
    cache.allocate(B, 20)
    cache.write_prefill(0, B, rand(B, H, 200, D), rand(B, H, 200, D))
    cache.seq_lens.copy_(i32(200, 17, 130))
    o = dict(window=50, softcap=30.0, kv_start=i32(0, 3, 100))
    q, k, v = rand(B, Hq, 1, D), rand(B, H, 1, D), rand(B, H, 1, D)
    announce(f"paged steps over {kv_dtype}")

    def step():
        cache.begin_decode_step(B)
        cache.write_decode(0, k, v)
        return cache.decode_attention(0, q, **o)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        q.copy_(rand(B, Hq, 1, D))
        graph.replay()
        torch.cuda.synchronize()
        kp, vp, ks, vs = cache.layer(0)
        want = gpu_pkg.paged_scored_attention_flash_decode(q, kp, vp, cache.block_tables, cache.seq_lens, 16, ks, vs, **o)
        assert torch.equal(out, want)
        n = [int(x) for x in cache.seq_lens]
        assert n == [202 + i, 19 + i, 132 + i]
        for b in range(B):
            kd, vd = (x[b:b + 1] for x in cache.read(0, B, n[b], dtype=torch.float32))
            ref = S.scored_attention(q[b:b + 1].double().cpu(), kd.double().cpu(), vd.double().cpu(), softcap=30.0, window=50,
                                     start=[int(o["kv_start"][b])])
            assert_close(out[b:b + 1].transpose(1, 2), ref.numpy(), 2.0 ** -9 * float(vd.abs().max()), "paged step")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_packed_documents_equal_each_alone(gpu_pkg, dtype):
    """Documents packed into a row, their positions restarted, give what each gives by itself."""
    Hq, H, D, R, cuts = 8, 2, 128, 64, [0, 70, 71, 200, 333]
    T = cuts[-1]
    rope = gpu_pkg.ScaledRope(D, R, rope_type="linear", factor=2.0, interleaved=True, device=DEV)
    q, k, v = rand(1, T, Hq, D, dtype=dtype), rand(1, T, H, D, dtype=dtype), rand(1, T, H, D, dtype=dtype)
    pos = torch.cat([torch.arange(b - a) for a, b in zip(cuts, cuts[1:])]).to(DEV)
    announce(f"packed documents {dtype}")
    qr, kr = rope(q, k, pos)
    o = dict(softcap=30.0, window=100, out_token_major=True)
    packed = gpu_pkg.scored_attention_flash(qr.transpose(1, 2), kr.transpose(1, 2), v.transpose(1, 2), cu_seqlens=i32(*cuts), **o)
    for a, b in zip(cuts, cuts[1:]):
        qa, ka = rope(q[:, a:b], k[:, a:b], torch.arange(b - a, device=DEV))
        assert torch.equal(qa, qr[:, a:b]) and torch.equal(ka, kr[:, a:b])
        alone = gpu_pkg.scored_attention_flash(qa.transpose(1, 2), ka.transpose(1, 2), v[:, a:b].transpose(1, 2), **o)
        # both within the weights' rounding of the same values: twice 2^-10 of the largest |v|, and two output roundings
        tol = 2.0 ** -14 if dtype == torch.float32 else 2.0 ** -9
        eps = torch.finfo(dtype).eps
        torch.testing.assert_close(packed[:, a:b].float(), alone.float(), rtol=eps, atol=tol * float(v.float().abs().max()))


def test_the_transformers_hook(gpu_pkg):
    plugins = importlib.import_module("simple-inference-autoresearch_amd.plugins")
    f, module = plugins.sia_attention_forward, SimpleNamespace(is_causal=True)
    q, k, v = rand(1, 8, 150, 64), rand(1, 2, 150, 64), rand(1, 2, 150, 64)
    q64, k64, v64 = (x.double().cpu() for x in (q, k, v))
    tol = 2.0 ** -10 * float(v.float().abs().max())
    cuts = i32(0, 40, 41, 150)
    for kw, ref in ((dict(sliding_window=33), dict(window=33)), (dict(softcap=10.0), dict(softcap=10.0)),
                    (dict(sliding_window=33, softcap=10.0), dict(window=33, softcap=10.0)),
                    (dict(cu_seq_lens_q=cuts, cu_seq_lens_k=cuts, max_length_q=109, max_length_k=109), dict(cuts=cuts.tolist())),
                    (dict(sliding_window=None, softcap=None), {})):
        announce(f"hook {list(kw)}")
        out, weights = f(module, q, k, v, None, scaling=0.125, **kw)
        assert weights is None and out.shape == (1, 150, 8, 64)
        assert_close(out.transpose(1, 2), S.scored_attention(q64, k64, v64, **ref).numpy(), tol, f"hook {list(kw)}")
    # a decode step: the query at the end of the keys
    out, _ = f(module, q[:, :, -1:], k, v, None, scaling=0.125, sliding_window=33, softcap=10.0)
    ref = S.scored_attention(q64[:, :, -1:], k64, v64, window=33, softcap=10.0)
    assert_close(out.transpose(1, 2), ref.numpy(), tol, "hook decode step")
    with pytest.raises(NotImplementedError):
        f(module, q[:, :, -1:], k, v, None, cu_seq_lens_q=cuts, cu_seq_lens_k=cuts)
    with pytest.raises(NotImplementedError):
        f(module, q.expand(2, -1, -1, -1), k, v, None, cu_seq_lens_q=cuts, cu_seq_lens_k=cuts)


def test_gqa_attention_with_options(gpu_pkg):
    q, k, v = rand(2, 8, 70, 128), rand(2, 2, 90, 128), rand(2, 2, 90, 128)
    announce("gqa_attention with options")
    want = gpu_pkg.scored_attention_flash(q, k, v, window=20, cu_seqlens=i32(0, 50), prefix_len=i32(30), out_token_major=True)
    assert torch.equal(gpu_pkg.gqa_attention(q, k, v, window=20, cu_seqlens=i32(0, 50), prefix_len=i32(30)), want.view(2, 70, -1))
    assert torch.equal(gpu_pkg.gqa_attention(q, k, v, window=None), gpu_pkg.gqa_attention(q, k, v))
