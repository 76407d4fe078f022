"""Decode over 4-bit pools whose pages hold no whole tiles of 16 tokens, or a number of them that is no power of two: the
kernels that look up every token.  Tolerances as in test_int4_gpu.py (16-bit queries at head_dim 64 and up: the matrix
cores)."""

from __future__ import annotations

import pytest
import torch

from helpers import announce
from test_int4_gpu import BF16, DEV, FP16, cache_case, check_decode, gen, randn

pytestmark = pytest.mark.gpu


def lens_tensor(lens):
    return torch.tensor(lens, dtype=torch.int32, device=DEV)


CASES = [
    # D, group, q dtype, (Hq, Hkv), page, lengths
    (128, 64, BF16, (32, 8), 24, [700, 1, 0, 300, 1500, 24, 25]),
    (128, 32, FP16, (8, 8), 8, [33, 250, 1, 64, 8, 0]),
    (128, 128, BF16, (40, 2), 48, [900, 63, 48]),
    (128, 64, FP16, (64, 2), 1, [513, 20, 4]),
    (64, 64, BF16, (16, 16), 2, [700, 1, 0, 300, 1500, 31]),
    (64, 32, FP16, (12, 4), 5, [127, 600, 3]),
    (64, 32, BF16, (5, 1), 100, [2000]),
    (64, 64, FP16, (24, 2), 3, [1, 2, 3, 700]),
    (256, 32, BF16, (16, 4), 80, [400, 1, 0, 95]),
    (256, 64, FP16, (8, 2), 17, [1200, 700]),
    (256, 128, BF16, (24, 2), 4, [77, 640, 16]),
    (256, 32, FP16, (40, 2), 9, [350, 31]),
]


@pytest.mark.parametrize("D,group,qdt,heads,page,lens", CASES)
def test_page_sizes(gpu_pkg, D, group, qdt, heads, page, lens):
    announce(f"int4 pages D {D} group {group} {qdt} heads {heads} page {page} lens {lens}")
    c = cache_case(gpu_pkg, D + page, len(lens), heads[1], D, group, max(lens) + 5, page)
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(9), len(lens), heads[0], 1, D, dtype=qdt)
    out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    check_decode(out, q, k, v, lens, "ragged", True)
    n = min(x for x in lens if x)
    live = [b for b, x in enumerate(lens) if x]
    one = c.run(gpu_pkg, q, n, 0.25)
    torch.cuda.synchronize()
    check_decode(one[live], q[live], [k[b] for b in live], [v[b] for b in live], [n] * len(live), "shared", True, 0.25)
    assert (c.run(gpu_pkg, q, 0) == 0).all()


@pytest.mark.parametrize("tiles", [1, 2, 3, 17, 100000])
@pytest.mark.parametrize("D,group,page", [(64, 32, 24), (128, 64, 40), (256, 128, 12)])
def test_splits(gpu_pkg, D, group, page, tiles):
    announce(f"int4 pages split D {D} page {page} tiles {tiles}")
    lens = [1000, 17, 0, 640, 33]
    c = cache_case(gpu_pkg, D, 5, 4, D, group, 1000, page)
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(4), 5, 16, 1, D)
    with gpu_pkg.decode_options(tiles_per_split=tiles):
        out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    check_decode(out, q, k, v, lens, f"{tiles} tiles a piece", True)


def test_same_bits_as_pages_of_whole_tiles(gpu_pkg):
    """The same tokens in pages of 16 and of 24 (16 tokens and 8 of the next 16 in each): one sum, one result."""
    announce("int4 pages 24 against 16")
    lens, H, D = [900, 31, 0, 333], 4, 128
    a = cache_case(gpu_pkg, 3, 4, H, D, 64, 900, 16)
    b = cache_case(gpu_pkg, 3, 4, H, D, 64, 900, 24)
    a.fill(gpu_pkg, lens)
    b.fill(gpu_pkg, lens)
    q = randn(gen(4), 4, 16, 1, D)
    x, y = a.run(gpu_pkg, q, lens_tensor(lens)), b.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    assert torch.equal(x, y)


@pytest.mark.parametrize("page", [8, 24, 48])
def test_views_nan_and_bad_pages(gpu_pkg, page):
    """A layer of a wider pool and strided queries; another sequence's NaN; ids outside the pool read page 0."""
    announce(f"int4 pages views, page {page}")
    lens, H, D, group = [90, 200, 41, 97], 2, 128, 32
    c = cache_case(gpu_pkg, 77, 4, H, D, group, 200, page)
    for name in ("kc", "vc", "ks", "vs"):
        t = getattr(c, name)
        wide = torch.zeros(t.shape[0], 2, t.shape[1] + 1, t.shape[2], t.shape[3], dtype=t.dtype, device=DEV)
        view = wide[:, 1, :t.shape[1]]
        view.copy_(t)
        setattr(c, name, view)
    table = torch.zeros(4, 2 * c.bt.shape[1], dtype=torch.int32, device=DEV)
    table[:, ::2] = c.bt
    c.bt = table[:, ::2]
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(8), 4, 1, 12, D)[:, :, :8].transpose(1, 2)
    out = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    check_decode(out, q, k, v, lens, "views", True)
    c.k[1, 0, 120] = float("nan")
    c.fill(gpu_pkg, lens)
    with gpu_pkg.decode_options(tiles_per_split=100000):
        bad = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    assert torch.isnan(bad[1, 0, :4]).all()
    live = [0, 2, 3]
    check_decode(bad[live], q[live], [k[b] for b in live], [v[b] for b in live], [lens[b] for b in live], "clean", True)
    for t in (c.kc, c.vc, c.ks, c.vs):
        t[0] = 0
    c.bt[0, 1], c.bt[0, 2] = -7, 1 << 30
    x = c.run(gpu_pkg, q, lens_tensor(lens))
    c.bt[0, 1], c.bt[0, 2] = 0, 0
    y = c.run(gpu_pkg, q, lens_tensor(lens))
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(x, nan=9.0), torch.nan_to_num(y, nan=9.0)) and torch.isfinite(x[0]).all()


def test_large_pool_takes_the_other_path(gpu_pkg):
    """Offsets in a pool of more than 4 GiB need 64 bits: the vector-ALU kernels, within their (fp32) tolerance."""
    announce("int4 pages, pool beyond 4 GiB")
    P, H, page, D, group, n = 360_000, 8, 24, 128, 64, 70
    kc, vc = (torch.empty(P, H, page, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.empty(P, H, page, 4, dtype=FP16, device=DEV) for _ in range(2))
    assert kc.numel() > 1 << 32
    bt = torch.tensor([[P - 1, 3, P - 70]], dtype=torch.int32, device=DEV)
    g = gen(1)
    k, v = randn(g, 1, H, n, D), randn(g, 1, H, n, D)
    gpu_pkg.kv_write(k, v, kc, vc, ks, vs, block_table=bt, page_size=page)
    q = randn(g, 1, 16, 1, D)
    out = gpu_pkg.paged_gqa_int4_flash_decode(q, kc, vc, ks, vs, bt, lens_tensor([n]), page)
    torch.cuda.synchronize()
    rk, rv = gpu_pkg.kv_read(kc, vc, n, ks, vs, block_table=bt, page_size=page, dtype=torch.float32)
    check_decode(out, q, [rk[0].double().cpu().numpy()], [rv[0].double().cpu().numpy()], [n], "large pool", False)
