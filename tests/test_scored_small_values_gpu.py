"""Scored prompts over bfloat16 values far below fp16's range: they count as they do in a decode step.

V enters P V in fp16, which holds bfloat16 values from 2^-17 on as they are and smaller ones to within 2^-25; where
that is more than 2^-12 of the largest value that a row sees, the row is taken in fp32.

Tolerance: 2^-10 of the largest visible |v| before the output's own rounding: a weight's rounding to fp16, 2^-11, fp32
scores, 2^-14, and V's, 2^-12 (test_scored_gpu.py has the first two).
"""

from __future__ import annotations

import math

import pytest
import torch

from helpers import announce, assert_close
from oracle import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def qkv(B, heads, Tq, Tk, D, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (torch.randn(B, Tq, heads[0], D, generator=g, device=DEV) * 2).bfloat16().transpose(1, 2)
    k, v = (torch.randn(B, Tk, heads[1], D, generator=g, device=DEV).bfloat16().transpose(1, 2) for _ in range(2))
    return q, k, v


def ref_of(q, k, v, **o):
    return S.scored_attention(*(t.double().cpu() for t in (q, k, v)), **o).numpy()


def close(got, ref, v, what):
    """Within 2^-10 of the largest of v, everything in units of a power of two next to it (exact: no output is denormal)."""
    top = float(v.float().abs().max())
    unit = 2.0 ** math.floor(math.log2(top))
    assert_close((got.double() / unit).cpu().numpy(), ref / unit, 2.0 ** -10 * top / unit, what, dtype=got.dtype)


# (short and long key ranges, few rows over many keys: V converted in LDS, from images, in split runs)
SHAPES = [(16, (4, 2), 130, 130), (32, (4, 2), 130, 130), (64, (4, 2), 150, 150), (64, (4, 2), 40, 4000), (128, (8, 2), 150, 150),
          (128, (8, 2), 300, 1100), (128, (8, 2), 40, 4000), (256, (4, 1), 150, 150), (256, (4, 1), 40, 3000), (128, (8, 2), 1, 90)]


@pytest.mark.parametrize("size", [-11, -13, -16, -20, -27, -66, -100])
@pytest.mark.parametrize("D,heads,Tq,Tk", SHAPES)
def test_values_of_any_size(gpu_pkg, D, heads, Tq, Tk, size):
    q, k, v = qkv(2, heads, Tq, Tk, D, seed=2)
    v = (v.float() * 2.0 ** size).bfloat16()
    announce(f"V of 2^{size}, D={D} {Tq} over {Tk}")
    out = gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0, window=900)
    close(out, ref_of(q, k, v, softcap=30.0, window=900), v, f"V of 2^{size}")


@pytest.mark.parametrize("D,heads,Tq,Tk", SHAPES)
def test_each_row_goes_by_what_it_sees(gpu_pkg, D, heads, Tq, Tk):
    """Small values of one document beside ordinary ones of another, of one head beside another's."""
    q, k, v = qkv(2, heads, Tq, Tk, D, seed=3)
    cut = Tk - Tq // 2 - 3
    v[:, 0, :cut] = (v[:, 0, :cut].float() * 1e-7).bfloat16()
    v[1, -1] = (v[1, -1].float() * 1e-8).bfloat16()
    if heads[1] == 1:
        v[0, 0, cut:] = (v[0, 0, cut:].float() * 1e-9).bfloat16()
    announce(f"small values of a document and of a head, D={D} {Tq} over {Tk}")
    out = gpu_pkg.scored_attention_flash(q, k, v, cu_seqlens=i32(0, cut))
    ref = ref_of(q, k, v, cuts=[0, cut])
    first = max(0, cut - (Tk - Tq))                       # queries of the first document
    per = heads[0] // heads[1]
    for b in range(2):
        for h in range(heads[0]):
            x = v[b, h // per]
            for rows, keys in ((slice(0, first), slice(0, cut)), (slice(first, Tq), slice(cut, Tk))):
                if rows.stop > rows.start:
                    close(out[b, h, rows], ref[b, h, rows], x[keys], f"sequence {b} head {h}")


@pytest.mark.parametrize("D,heads,Tq,Tk", SHAPES)
def test_zeros_and_values_that_cancel(gpu_pkg, D, heads, Tq, Tk):
    q, k, v = qkv(1, heads, Tq, Tk, D, seed=4)
    announce(f"zeros and values that cancel, D={D} {Tq} over {Tk}")
    assert (gpu_pkg.scored_attention_flash(q, k, torch.zeros_like(v), softcap=30.0) == 0).all()
    # equal weights: every row of the first document is the mean of (3, -1) 2^-27, each of them under half of fp16's step
    w = torch.full_like(v, -2.0 ** -27)
    w[:, :, ::2] = 3 * 2.0 ** -27
    out = gpu_pkg.scored_attention_flash(torch.zeros_like(q), k, w, causal=False, window=1 << 20)
    even, odd = (Tk + 1) // 2, Tk // 2
    mean = (3 * even - odd) / Tk * 2.0 ** -27
    assert ((out.double() - mean).abs() <= 2.0 ** -10 * 3 * 2.0 ** -27 + 2.0 ** -9 * mean).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_captured_and_replayed(gpu_pkg, D):
    q, k, v = qkv(1, (4, 2), 140, 140, D, seed=5)
    announce(f"captured, D={D}")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0)
    for size in (1e-8, 1.0, 1e-6):
        v.copy_(torch.randn(1, 2, 140, D, device=DEV) * size)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0))
        close(out, ref_of(q, k, v, softcap=30.0), v, f"V of {size}")
