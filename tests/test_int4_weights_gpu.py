"""Softmax weights of the 4-bit decode at the ends of fp16's range, which the matrix cores take them in.

A weight w, relative to its wave's largest one, enters as p = 2^s w for some s >= 11.  Its rounding to fp16 is off by at
most 2^-11 p where p is normal and by 2^-25 where it is a denormal, that is by 2^-11 w + 2^-36.  A value's rounding is off
by 2^-11 of it.  The scores are products of few bits: their factor (twice), the product and its difference to the reference
round once each, by 2^-24 of the spread of the scores, or are exact.  Sums are in fp32.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from helpers import announce, f64, ulp
from test_int4_gpu import BF16, DEV, FP16, cache_case

pytestmark = pytest.mark.gpu


def check(out, weights, v, what, spread=0.0):
    """out (Hq, D) against ``weights`` (n,), the largest 1, over exact values v (H, n, D); ``spread`` of the scores in
    log2 units, 0 where they are exact."""
    n, G = len(weights), out.shape[0] // v.shape[0]
    got = f64(out)
    total = weights.sum()
    for h in range(v.shape[0]):
        ref, wabs = weights @ v[h] / total, weights @ np.abs(v[h]) / total
        # (scores, and sums of n weights and products in fp32: in the numerator and in the normaliser)
        bound = (2.0 ** -10 + 2 * (4 * spread + n / 4 + 74) * 2.0 ** -24) * wabs + 2.0 ** -36 * np.abs(v[h]).sum(0) / total
        allowed = bound + 0.5 * ulp(np.abs(ref) + bound, out.dtype)
        for x in got[h * G:(h + 1) * G]:
            assert np.isfinite(x).all(), f"{what}: non-finite output"
            assert (np.abs(x - ref) <= allowed).all(), f"{what}: off by {(np.abs(x - ref) / allowed).max():.2f} of the bound"


def one_share(gpu_pkg, c, q, n, scale):
    """Every head's keys in one wave: eight heads, a length per sequence (of two), no split."""
    with gpu_pkg.decode_options(tiles_per_split=100000):
        return c.run(gpu_pkg, q.expand(2, -1, -1, -1), torch.tensor([n, 1], dtype=torch.int32, device=DEV), scale)


@pytest.mark.parametrize("D,group,page", [(64, 32, 0), (128, 64, 16), (256, 128, 16), (128, 64, 24)])
@pytest.mark.parametrize("G", [4, 12])
@pytest.mark.parametrize("step", [1, 2])
def test_maxima_that_grow_at_the_end_of_fp32(gpu_pkg, D, group, page, G, step):
    """Scores of 2^27 + 16 j (log2 units), neighbours in fp32, j growing along the sequence: no weight overflows fp16."""
    announce(f"int4 decode scores of 2^27 D {D} page {page} G {G} step {step}")
    H, n = 8, 32 * 8
    c = cache_case(gpu_pkg, D, 2, H, D, group, n, page)
    j = 1 + step * (torch.arange(n, device=DEV) // 32)
    c.k[:] = 0
    c.k[..., :group] = 2.0 ** 15                                    # m of the first group
    c.k[..., group:2 * group] = (j * 2.0 ** -8).to(BF16)[:, None]   # and of the second
    _, v = c.fill(gpu_pkg, [n, 1])
    # q . k = group (2^15 + 2^-8 j); a factor of 2^7 32 / group makes it 2^27 + 16 j
    want = np.float32(2.0 ** 12 / group)
    scale = np.float32(want / math.log2(math.e))
    while np.float32(scale * np.float32(math.log2(math.e))) < want:
        scale = np.nextafter(scale, np.float32(np.inf))
    assert np.float32(scale * np.float32(math.log2(math.e))) == want
    q = torch.ones(1, G * H, 1, D, dtype=BF16, device=DEV)
    out = one_share(gpu_pkg, c, q, n, float(scale))
    torch.cuda.synchronize()
    jj = j.cpu().numpy().astype(np.float64)
    check(out[0, 0], 2.0 ** (16 * (jj - jj.max())), v[0], f"step {step}")


@pytest.mark.parametrize("D,group,page,qdt", [(64, 32, 0, FP16), (128, 64, 16, BF16), (256, 128, 16, BF16),
                                              (128, 64, 24, BF16)])
@pytest.mark.parametrize("G", [4, 12])
@pytest.mark.parametrize("gap", [13.3, 19.5, 24.4, 25.05, 30.3])
def test_attention_sink(gpu_pkg, D, group, page, qdt, G, gap):
    """The first token's weight is 2^gap times every other's, its value zero: the others' weights make the result."""
    announce(f"int4 decode sink D {D} page {page} G {G} gap {gap}")
    H, n = 8, 9000
    c = cache_case(gpu_pkg, D, 2, H, D, group, n, page)
    c.k[:] = 0
    c.k[:, :, 0] = 1
    c.v[:, :, 0] = 0
    _, v = c.fill(gpu_pkg, [n, 1])
    q = torch.ones(1, G * H, 1, D, dtype=qdt, device=DEV)
    out = one_share(gpu_pkg, c, q, n, gap * math.log(2) / D)
    torch.cuda.synchronize()
    weights = np.full(n, 2.0 ** -gap)
    weights[0] = 1
    check(out[0, 0], weights, v[0], f"gap {gap}", gap)


@pytest.mark.parametrize("D,group,page", [(64, 64, 16), (128, 32, 0), (256, 64, 16), (64, 32, 24)])
@pytest.mark.parametrize("G", [4, 12])
@pytest.mark.parametrize("growth", [0.5, 3.9375, 4.0625, 7.9375, 15.0])
def test_scores_that_grow_along_the_sequence(gpu_pkg, D, group, page, G, growth):
    """Every pair of tiles ``growth`` log2 units above the one before, values up to fp16's largest: weights above the
    running maximum stay inside fp16."""
    announce(f"int4 decode growing scores D {D} page {page} G {G} growth {growth}")
    H, n = 8, 32 * 12
    c = cache_case(gpu_pkg, D + 1, 2, H, D, group, n, page)
    # one value a row: the minimum of every group, step 0
    c.k[:] = (torch.arange(n, device=DEV) // 32).to(BF16)[:, None]
    c.v[..., ::5] = 65280.0
    _, v = c.fill(gpu_pkg, [n, 1])
    q = torch.ones(1, G * H, 1, D, dtype=BF16, device=DEV)
    out = one_share(gpu_pkg, c, q, n, growth * math.log(2) / D)
    torch.cuda.synchronize()
    pair = np.arange(n) // 32
    check(out[0, 0], 2.0 ** (growth * (pair - pair.max())), v[0], f"growth {growth}", 11 * growth)
