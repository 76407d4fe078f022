"""float32 queries over a 4-bit cache on the matrix cores: taken where batch x query heads x capacity is large (every case
here).  Tolerance: fp32 throughout, as derived in test_int4_gpu.py without the term for fp16 operands."""

from __future__ import annotations

import pytest
import torch

from helpers import announce
from test_int4_gpu import DEV, FP32, cache_case, check_decode, gen, randn, same

pytestmark = pytest.mark.gpu


def lens_tensor(lens):
    return torch.tensor(lens, dtype=torch.int32, device=DEV)


CASES = [
    # D, group, (Hq, Hkv), page, capacity, lengths
    (128, 64, (32, 8), 16, 1600, [700, 1, 0, 300, 1500]),
    (128, 32, (32, 8), 0, 1600, [16, 15, 17, 0, 1000]),
    (128, 128, (40, 2), 32, 2000, [33, 250, 1, 64]),
    (64, 64, (16, 8), 16, 2000, [700, 1, 0, 300, 1500, 31]),
    (64, 32, (12, 4), 0, 5000, [127, 600, 3]),
    (256, 32, (16, 4), 16, 2400, [400, 1, 0, 95]),
    (256, 64, (8, 2), 0, 10000, [1200, 700]),
    (256, 128, (64, 2), 64, 800, [77, 640, 16]),
]


@pytest.mark.parametrize("D,group,heads,page,cap,lens", CASES)
def test_parity(gpu_pkg, D, group, heads, page, cap, lens):
    announce(f"int4 fp32 D {D} group {group} heads {heads} page {page} lens {lens}")
    B, (Hq, H) = len(lens), heads
    assert B * Hq * cap >= 150000
    c = cache_case(gpu_pkg, D + group, B, H, D, group, cap, page, FP32)
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(9), B, Hq, 1, D, dtype=FP32)
    out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    assert out.dtype == FP32 and out.shape == (B, 1, Hq, D)
    check_decode(out, q, k, v, lens, "ragged", False)
    n = min(x for x in lens if x)
    live = [b for b, x in enumerate(lens) if x]
    one = c.run(gpu_pkg, q, n, 0.25)
    torch.cuda.synchronize()
    check_decode(one[live], q[live], [k[b] for b in live], [v[b] for b in live], [n] * len(live), "shared", False, 0.25)
    assert (c.run(gpu_pkg, q, 0) == 0).all()
    # the matrix and the vector-ALU kernels agree within both bounds: a call cut to one sequence is the latter's
    if Hq * min(cap, 400) < 150000 and not page:
        n0 = min(lens[0], 400)
        small = gpu_pkg.attention_flash_decode_int4(q[:1], c.kc[:1, :, :400], c.vc[:1, :, :400], c.ks[:1, :, :400],
                                                    c.vs[:1, :, :400], n0)
        check_decode(small, q[:1], k[:1], v[:1], [n0], "vector", False)


@pytest.mark.parametrize("tiles", [1, 3, 100000])
@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (256, 128)])
def test_splits_and_nan(gpu_pkg, D, group, tiles):
    """Pieces of a few tiles and the whole batch in one share; a sequence's NaN stays its own."""
    announce(f"int4 fp32 split D {D} tiles {tiles}")
    lens = [97, 1000, 0, 641, 33]
    c = cache_case(gpu_pkg, D, 5, 8, D, group, 2000, 16, FP32)
    c.k[0, :, ::3, 5] = float("nan")
    c.v[0, :, 1::3, D - 1] = float("inf")
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(4), 5, 16, 1, D, dtype=FP32)
    with gpu_pkg.decode_options(tiles_per_split=tiles):
        out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    live = [1, 2, 3, 4]
    check_decode(out[live], q[live], [k[b] for b in live], [v[b] for b in live], [lens[b] for b in live],
                 f"{tiles} tiles a piece", False)
    assert torch.isnan(out[0]).all(-1).all()


def test_strided_and_in_a_graph(gpu_pkg):
    announce("int4 fp32 strided q, graph")
    lens, D = [900, 31, 1024], 128
    c = cache_case(gpu_pkg, 7, 3, 4, D, 64, 4000, 16, FP32)
    k, v = c.fill(gpu_pkg, lens)
    kl = lens_tensor(lens)
    qkv = randn(gen(8), 3, 1, 24, D, dtype=FP32)
    q = qkv[:, :, :16].transpose(1, 2)
    eager = c.run(gpu_pkg, q, kl)
    torch.cuda.synchronize()
    check_decode(eager, q, k, v, lens, "strided", False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run(gpu_pkg, q, kl)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.run(gpu_pkg, q, kl)
    for i in range(3):
        qkv.copy_(randn(gen(20 + i), *qkv.shape, dtype=FP32))
        kl.copy_(lens_tensor([900 - i, 31 + i, 500 * i]))
        graph.replay()
        ref = c.run(gpu_pkg, q, kl)
        torch.cuda.synchronize()
        # (the second sequence's tokens 31 and 32 were never written: NaN on both sides)
        assert same(out, ref), i
