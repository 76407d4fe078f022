"""The 4-bit KV cache on the GPU against ``oracle/int4.py``: quantising, writing, reading back, decode attention.

Codes, parameters and values read back are compared bit for bit (a value is the fp32 rounding of m + n s, rounded once
more to the output type).  Attention is compared with float64 attention over the exact values m + n s, within

* a rounding of every weight and of every value to fp16 where the matrix cores take them: 2 * 2^-11 of
  ``sum_t w_t |v_t|``;
* the fp32 roundings (unit u = 2^-24): a score's error is at most (D + 16) u of ``scale sum |q k|``, which moves a weight
  by twice that relative; sums over keys add at most (n / 4 + 64) u; both again for the normaliser;
* one rounding to the output type.
"""

from __future__ import annotations

import ctypes
import importlib

import numpy as np
import pytest
import torch

from helpers import announce, f64, ulp
from oracle import int4 as I4

pytestmark = pytest.mark.gpu
DEV = "cuda"
L = importlib.import_module("simple-inference-autoresearch_amd._lib")
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
GROUPS = [(16, 16), (32, 32), (64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale + 0.3).to(dtype)


def quant(x, group):
    """Oracle codes (packed) and parameters of a tensor."""
    codes, par = I4.quantize(x.float().cpu().numpy(), group)
    return I4.pack(codes), par


def rounded(values, dtype):
    """float64 values -> fp32 -> dtype, as a tensor on the GPU."""
    return torch.from_numpy(values.astype(np.float32)).to(DEV).to(dtype)


def vals(codes, params):
    """Exact values of packed codes and parameters (tensors)."""
    return I4.values(I4.unpack(codes.cpu().numpy()), params.cpu().numpy())


def same(a, b):
    """Equal, NaN standing for NaN."""
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(torch.nan_to_num(a, nan=12345.0),
                                                                     torch.nan_to_num(b, nan=12345.0))


def check_decode(out, q, k, v, lens, what, matrix, scale=None):
    """out (B, 1, Hq, D) against attention over exact values k, v (list per sequence of (Hkv, >= n, D))."""
    B, Hq, _, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    u = 2.0 ** -24
    got, qq = f64(out), f64(q)
    for b, n in enumerate(lens):
        ref, wabs, sabs = I4.decode(qq[b, :, 0], k[b], v[b], n, scale)
        fp32 = 2 * (D + 16) * u * sabs + (n / 4 + 74) * u
        bound = (2 * fp32 + (2.0 ** -10 if matrix else 0.0)) * wabs
        allowed = bound + 0.5 * ulp(np.abs(ref) + bound, out.dtype)
        err = np.abs(got[b, 0] - ref)
        assert np.isfinite(got[b, 0]).all(), f"{what}: non-finite output of sequence {b}"
        assert (err <= allowed).all(), f"{what}: sequence {b} off by {(err / allowed).max():.2f} of the bound"


# ------------------------------------------------------- quantise, write, read


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D,group", GROUPS)
def test_quantize_bit_exact(gpu_pkg, dtype, D, group):
    announce(f"quantize_kv_int4 {dtype} D {D} group {group}")
    x = randn(gen(D + group), 3, 5, 7, D, dtype=dtype, scale=2.0)
    rows = x.view(-1, D)
    rows[0] = 0
    rows[1] = -1.7
    rows[2, 3] = float("nan")
    rows[3, D - 1] = float("inf")
    rows[4, 0] = -float("inf")
    rows[5] *= 1e-6
    rows[6] *= 3e4 if dtype == FP16 else 1e6                      # clamped at +-65504
    rows[7] = torch.arange(D, device=DEV) % 31 * 0.5              # s = 1 and ties at n + 1/2
    rows[8, :2] = torch.tensor([60000.0, -60000.0], device=DEV)
    codes, par = gpu_pkg.quantize_kv_int4(x, group if group >= 32 else 32)
    torch.cuda.synchronize()
    rc, rp = quant(x, group)
    assert codes.dtype == torch.uint8 and par.dtype == FP16 and codes.shape == x.shape[:-1] + (D // 2,)
    np.testing.assert_array_equal(codes.cpu().numpy(), rc)
    np.testing.assert_array_equal(par.cpu().numpy(), rp)          # (NaN equals NaN, -0 equals 0)
    # (row 6 in fp16: the product itself overflows to infinities in some groups, which read back as NaN like row 3's)
    finite = torch.isfinite(x).view(-1, D // group, group).all(-1, keepdim=True).expand(-1, -1, group).reshape(x.shape)
    for out in (BF16, FP16, FP32):
        y = gpu_pkg.dequantize_kv_int4(codes, par, out)
        assert same(y, rounded(vals(codes, par), out))
        assert torch.equal(torch.isfinite(y), finite)             # no finite input overflows any output type


def test_quantize_shapes_and_refusals(gpu_pkg):
    announce("quantize_kv_int4 shapes")
    g = gen(0)
    x = randn(g, 4, 6, 128)
    for t in (x[0, 0], x[1], x.transpose(0, 1), x[:, ::2], randn(g, 5, 130)[:, 1:129], x[:0]):
        codes, par = gpu_pkg.quantize_kv_int4(t, 64)
        rc, rp = quant(t, 64) if t.numel() else (np.zeros((0, 6, 64), np.uint8), np.zeros((0, 6, 4), np.float16))
        np.testing.assert_array_equal(codes.cpu().numpy(), rc)
        np.testing.assert_array_equal(par.cpu().numpy(), rp)
        assert gpu_pkg.dequantize_kv_int4(codes, par).shape == t.shape
    for bad in (randn(g, 2, 48), randn(g, 2, 96)):
        with pytest.raises((NotImplementedError, ValueError)):
            gpu_pkg.quantize_kv_int4(bad, 32)
    with pytest.raises(ValueError):
        gpu_pkg.quantize_kv_int4(x, 16)
    with pytest.raises(ValueError):
        gpu_pkg.quantize_kv_int4(x.cpu(), 64)
    with pytest.raises(NotImplementedError):
        gpu_pkg.quantize_kv_int4(x.to(torch.int8), 64)
    codes, par = gpu_pkg.quantize_kv_int4(x, 64)
    with pytest.raises(ValueError):
        gpu_pkg.dequantize_kv_int4(codes, par[..., :3])
    with pytest.raises(ValueError):
        gpu_pkg.dequantize_kv_int4(codes, par.float())


def pools(P, H, page, D, group):
    """Codes and parameters filled with a pattern that no write leaves."""
    return (torch.full((P, H, page, D // 2), 0xA5, dtype=torch.uint8, device=DEV),
            torch.full((P, H, page, 2 * D // group), 7.0, dtype=FP16, device=DEV))


@pytest.mark.parametrize("page", [0, 16, 24])
@pytest.mark.parametrize("D,group,dtype", [(16, 16, FP32), (64, 32, FP16), (128, 64, BF16), (256, 128, BF16)])
def test_write_then_read(gpu_pkg, page, D, group, dtype):
    """Tokens land where their position says, everything else stays, and reading gives the values back."""
    announce(f"kv_write/kv_read int4 page {page} D {D} group {group} {dtype}")
    B, H, T = 3, 2, 29
    g = gen(D + page)
    x = randn(g, B, T, 2 * H, D, dtype=dtype)                     # token-major, two slices of one buffer
    k, v = x[:, :, :H].transpose(1, 2), x[:, :, H:].transpose(1, 2)
    first = [0, 5, 40]
    start = torch.tensor(first, dtype=torch.int32, device=DEV)
    if page:
        nblk = -(-(max(first) + T - 6) // page)                   # the last sequence's last tokens lie past the table
        bt = torch.randperm(B * nblk + 1, generator=torch.Generator().manual_seed(1))[:B * nblk].view(B, nblk)
        bt = bt.to(torch.int32)
        bt[1, 1] = B * nblk + 3                                   # a page id outside the pool
        bt[0, 0] = -1 if page == 16 else bt[0, 0]
        P, S, cap = B * nblk + 1, page, nblk * page
    else:
        bt, P, S, cap = None, B, max(first) + T - 6, max(first) + T - 6
    (kc, ks), (vc, vs) = pools(P, H, S, D, group), pools(P, H, S, D, group)
    want = [t.cpu().numpy().copy() for t in (kc, ks, vc, vs)]
    values = np.zeros((2, B, H, T, D))
    (rk, rkp), (rv, rvp) = quant(k, group), quant(v, group)
    for b in range(B):
        for t in range(T):
            pos = first[b] + t
            if pos >= cap:
                continue
            if page:
                slot, at = int(bt[b, pos // page]), pos % page
                if not 0 <= slot < P:
                    continue
            else:
                slot, at = b, pos
            for i, (src, dst) in enumerate(((rk, 0), (rkp, 1), (rv, 2), (rvp, 3))):
                want[dst][slot, :, at] = src[b, :, t]
            values[0, b, :, t] = I4.values(I4.unpack(rk[b, :, t]), rkp[b, :, t])
            values[1, b, :, t] = I4.values(I4.unpack(rv[b, :, t]), rvp[b, :, t])
    btd = None if bt is None else bt.to(DEV)
    gpu_pkg.kv_write(k, v, kc, vc, ks, vs, block_table=btd, start_pos=start, page_size=page)
    torch.cuda.synchronize()
    for got, ref in zip((kc, ks, vc, vs), want):
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
    for out in (BF16, FP16, FP32):
        rk, rv = gpu_pkg.kv_read(kc, vc, T, ks, vs, block_table=btd, start_pos=start, page_size=page, dtype=out)
        torch.cuda.synchronize()
        assert same(rk, rounded(values[0], out)) and same(rv, rounded(values[1], out))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32), (256, 64)])
def test_rope_write_is_rope_then_write(gpu_pkg, D, group, interleaved):
    announce(f"rope_kv_write int4 D {D} group {group} interleaved {interleaved}")
    B, T, Hq, H, S = 2, 9, 4, 2, 40
    g = gen(D)
    q, k, v = randn(g, B, T, Hq, D), randn(g, B, T, H, D), randn(g, B, T, H, D)
    cos, sin = gpu_pkg.RopeFrequencies(D, S, device=torch.device(DEV)).get(S, dtype=BF16)
    (kc, ks), (vc, vs), (kc2, ks2), (vc2, vs2) = (pools(B, H, S, D, group) for _ in range(4))
    qr = gpu_pkg.rope_kv_write(q, k, v, cos, sin, kc, vc, ks, vs, start_offset=3, interleaved=interleaved)
    q2, k2 = gpu_pkg.rope_triton(q, k, cos[3:3 + T], sin[3:3 + T], interleaved=interleaved)
    gpu_pkg.kv_write(k2.transpose(1, 2), v.transpose(1, 2), kc2, vc2, ks2, vs2, start_offset=3)
    torch.cuda.synchronize()
    assert torch.equal(qr, q2)
    for a, b in ((kc, kc2), (ks, ks2), (vc, vc2), (vs, vs2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("src", [BF16, FP16, FP32, torch.int8])
@pytest.mark.parametrize("paged", [False, True])
def test_read_other_caches(gpu_pkg, src, paged):
    """kv_read of 16-bit, fp32 and int8 caches, into strided outputs, k alone too."""
    announce(f"kv_read {src} paged {paged}")
    B, H, S, D, T, page = 2, 3, 50, 64, 21, 8
    g = gen(3)
    x = randn(g, B, H, S, D, dtype=FP32), randn(g, B, H, S, D, dtype=FP32)
    sc = (None, None)
    if src == torch.int8:
        pairs = [gpu_pkg.quantize_kv_int8(t, FP32 if paged else FP16) for t in x]
        x, sc = [p[0] for p in pairs], [p[1] for p in pairs]
        ref = [(a.double() * s.double()[..., None]) for a, s in zip(x, sc)]
    else:
        x = [t.to(src) for t in x]
        ref = [t.double() for t in x]
    bt, kw = None, {}
    if paged:
        nblk = -(-S // page)
        bt = torch.randperm(B * nblk, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(B, nblk).to(DEV)

        def pool(t):
            p = torch.zeros(B * nblk, H, page, *t.shape[3:], dtype=t.dtype, device=DEV)
            for b in range(B):
                for s in range(S):
                    p[int(bt[b, s // page]), :, s % page] = t[b, :, s]
            return p
        x = [pool(t) for t in x]
        sc = [pool(t) if t is not None else None for t in sc]
        kw = dict(block_table=bt, page_size=page)
    for out in (BF16, FP32):
        buf = torch.full((2, B, T + 2, H, D), 9.0, dtype=out, device=DEV)         # token-major, room behind
        o = tuple(buf[i, :, :T].transpose(1, 2) for i in range(2))
        k, v = gpu_pkg.kv_read(x[0], x[1], T, sc[0], sc[1], start_offset=17, out=o, **kw)
        torch.cuda.synchronize()
        assert k is o[0] and same(k.contiguous(), ref[0][:, :, 17:17 + T].float().to(out))
        assert same(v.contiguous(), ref[1][:, :, 17:17 + T].float().to(out)) and (buf[:, :, T:] == 9).all()
    k, v = gpu_pkg.kv_read(x[0], None, T, sc[0], None, start_offset=29, dtype=FP32, **kw)
    assert v is None and same(k, ref[0][:, :, 29:29 + T].float())
    k, v = gpu_pkg.kv_read(x[0], x[1], 0, sc[0], sc[1], **kw)
    assert k.shape == (B, H, 0, D)
    if not paged:
        with pytest.raises(ValueError):
            gpu_pkg.kv_read(x[0], x[1], T, sc[0], sc[1], start_offset=S - T + 1)
    with pytest.raises(ValueError):
        gpu_pkg.kv_read(x[0], x[1], -1, sc[0], sc[1], **kw)


# ------------------------------------------------------------- decode attention


def cache_case(gpu_pkg, seed, B, H, D, group, S, page, dtype=BF16):
    """A contiguous cache or pool written by kv_write, its block table, and the exact values per sequence."""
    g = gen(seed)
    k, v = randn(g, B, H, S, D, dtype=dtype), randn(g, B, H, S, D, dtype=dtype)
    if page:
        nblk = -(-S // page)
        P = B * nblk + 2
        bt = torch.randperm(P, generator=torch.Generator().manual_seed(seed))[:B * nblk].view(B, nblk).to(torch.int32)
        bt = bt.to(DEV)
        shape = (P, H, page)
    else:
        bt, shape = None, (B, H, S)
    # (parameters of NaN wherever no token is: nothing past a sequence's length may reach the result)
    kc, vc = (torch.full(shape + (D // 2,), 0xFF, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.full(shape + (2 * D // group,), float("nan"), dtype=FP16, device=DEV) for _ in range(2))
    return SimpleCase(kc, vc, ks, vs, bt, page, k, v, group)


class SimpleCase:
    def __init__(self, kc, vc, ks, vs, bt, page, k, v, group):
        self.kc, self.vc, self.ks, self.vs, self.bt, self.page = kc, vc, ks, vs, bt, page
        self.k, self.v, self.group = k, v, group

    def fill(self, gpu_pkg, lens):
        """Write the first lens[b] tokens of every sequence; returns the exact values."""
        for b, n in enumerate(lens):
            if n:
                if self.page:
                    gpu_pkg.kv_write(self.k[b:b + 1, :, :n], self.v[b:b + 1, :, :n], self.kc, self.vc, self.ks, self.vs,
                                     block_table=self.bt[b:b + 1], page_size=self.page)
                else:
                    gpu_pkg.kv_write(self.k[b:b + 1, :, :n], self.v[b:b + 1, :, :n], self.kc[b:b + 1],
                                     self.vc[b:b + 1], self.ks[b:b + 1], self.vs[b:b + 1])
        return tuple([I4.values(*I4.quantize(t[b].float().cpu().numpy(), self.group)) for b in range(len(lens))]
                     for t in (self.k, self.v))

    def run(self, gpu_pkg, q, kv_len, sm_scale=None):
        if self.page:
            return gpu_pkg.paged_gqa_int4_flash_decode(q, self.kc, self.vc, self.ks, self.vs, self.bt, kv_len,
                                                       self.page, sm_scale)
        return gpu_pkg.attention_flash_decode_int4(q, self.kc, self.vc, self.ks, self.vs, kv_len, sm_scale)


def is_matrix(qdt, D, page):
    """Whether the matrix cores take it: any page size, where a layer's pool is below 4 GiB (all pools here)."""
    return qdt != FP32 and D >= 64


DECODES = [
    # D, group, q dtype, (Hq, Hkv), page, lengths
    (128, 64, BF16, (32, 8), 16, [700, 1, 0, 300, 1500]),
    (128, 32, BF16, (32, 8), 0, [16, 15, 17, 0, 1000]),
    (128, 128, FP16, (8, 8), 32, [33, 250, 1, 64]),
    (128, 64, FP16, (40, 2), 64, [900, 63]),
    (128, 32, BF16, (64, 2), 16, [513, 20, 4]),
    (64, 64, BF16, (16, 16), 16, [700, 1, 0, 300, 1500, 31]),
    (64, 32, FP16, (12, 4), 0, [127, 600, 3]),
    (64, 32, BF16, (5, 1), 16, [2000]),
    (64, 64, FP16, (32, 8), 0, [1, 2, 3]),
    (256, 32, BF16, (16, 4), 16, [400, 1, 0, 95]),
    (256, 64, FP16, (8, 2), 0, [1200, 700]),
    (256, 128, BF16, (16, 2), 32, [77, 640, 16]),
    (32, 32, BF16, (8, 2), 16, [300, 1, 0]),
    (16, 16, FP16, (4, 4), 0, [257, 40]),
    (128, 64, BF16, (12, 4), 24, [700, 1, 0, 300]),
    (64, 32, FP16, (8, 2), 1, [100, 7]),
    (128, 32, FP32, (32, 8), 0, [500, 0, 1]),
    (64, 64, FP32, (8, 1), 16, [800, 31]),
    (256, 128, FP32, (4, 2), 16, [300]),
]


@pytest.mark.parametrize("D,group,qdt,heads,page,lens", DECODES)
def test_decode_parity(gpu_pkg, D, group, qdt, heads, page, lens):
    announce(f"int4 decode D {D} group {group} {qdt} heads {heads} page {page} lens {lens}")
    B, (Hq, H) = len(lens), heads
    c = cache_case(gpu_pkg, D + group, B, H, D, group, max(lens) + 5, page)
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(9), B, Hq, 1, D, dtype=qdt)
    out = c.run(gpu_pkg, q, torch.tensor(lens, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert out.shape == (B, 1, Hq, D) and out.dtype == qdt
    check_decode(out, q, k, v, lens, "ragged", is_matrix(qdt, D, page))
    n = min(x for x in lens if x)                                # one shared length, as a (1,) tensor and as an int
    o1 = c.run(gpu_pkg, q, torch.tensor([n], dtype=torch.int32, device=DEV), 0.25)
    live = [b for b, x in enumerate(lens) if x]
    o2 = c.run(gpu_pkg, q, n, 0.25)
    torch.cuda.synchronize()
    check_decode(o1[live], q[live], [k[b] for b in live], [v[b] for b in live], [n] * len(live), "shared",
                 is_matrix(qdt, D, page), 0.25)
    assert torch.equal(o1[live], o2[live])
    assert (c.run(gpu_pkg, q, 0) == 0).all() and (c.run(gpu_pkg, q, -3) == 0).all()
    assert c.run(gpu_pkg, q[:0], torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 1, Hq, D)


@pytest.mark.parametrize("tiles", [1, 3, 17])
@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (256, 128)])
def test_decode_split(gpu_pkg, D, group, tiles):
    """Every sequence cut into pieces of a few tiles."""
    announce(f"int4 decode split D {D} tiles {tiles}")
    lens = [1000, 17, 0, 640]
    c = cache_case(gpu_pkg, D, 4, 4, D, group, 1000, 16)
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(4), 4, 16, 1, D)
    with gpu_pkg.decode_options(tiles_per_split=tiles):
        out = c.run(gpu_pkg, q, torch.tensor(lens, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    check_decode(out, q, k, v, lens, f"{tiles} tiles a piece", True)


@pytest.mark.parametrize("D,page", [(128, 16), (64, 0), (256, 16), (32, 16), (128, 24)])
def test_decode_views_and_values(gpu_pkg, D, page):
    """Strided caches and queries, values at the ends of fp16's range, and a NaN that only its own sequence sees."""
    announce(f"int4 decode views D {D} page {page}")
    lens, H, group = [90, 200, 41], 2, 32
    c = cache_case(gpu_pkg, 77, 3, H, D, group, 200, page)
    big = torch.where(torch.rand(c.v.shape, generator=gen(5), device=DEV) < 0.01, 60000.0, 1.0)
    c.v = (c.v.float() * big).clamp(-65504, 65504).to(BF16).clamp(-65280, 65280)
    # a layer of a larger pool, heads and tokens of another stride
    for name in ("kc", "vc", "ks", "vs"):
        t = getattr(c, name)
        wide = torch.zeros(t.shape[0], 2, t.shape[1] + 1, t.shape[2], t.shape[3], dtype=t.dtype, device=DEV)
        view = wide[:, 1, :t.shape[1]]
        view.copy_(t)
        setattr(c, name, view)
    k, v = c.fill(gpu_pkg, lens)
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    qkv = randn(gen(8), 3, 1, 12, D)
    q = qkv[:, :, :8].transpose(1, 2)
    out = c.run(gpu_pkg, q, kl)
    torch.cuda.synchronize()
    check_decode(out, q, k, v, lens, "views", is_matrix(BF16, D, page))
    c.k[1, 0, 120] = float("nan")
    c.fill(gpu_pkg, lens)
    bad = c.run(gpu_pkg, q, kl)
    torch.cuda.synchronize()
    assert torch.isnan(bad[1, 0, :4]).all() and torch.equal(bad[1, 0, 4:], out[1, 0, 4:])
    assert torch.equal(bad[[0, 2]], out[[0, 2]])


def test_decode_bad_pages_stay_inside_the_pool(gpu_pkg):
    """A page id outside the pool reads page 0, as in the other decode functions."""
    announce("int4 decode bad pages")
    for page in (16, 24):
        c = cache_case(gpu_pkg, 5, 1, 2, 128, 64, 96, page)
        k, v = c.fill(gpu_pkg, [96])
        q = randn(gen(1), 1, 8, 1, 128)
        kl = torch.tensor([96], dtype=torch.int32, device=DEV)
        c.kc[0], c.vc[0], c.ks[0], c.vs[0] = 0, 0, 0, 0
        c.bt[0, 1], c.bt[0, 2] = -7, 1 << 30
        a = c.run(gpu_pkg, q, kl)
        c.bt[0, 1], c.bt[0, 2] = 0, 0
        b = c.run(gpu_pkg, q, kl)
        torch.cuda.synchronize()
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_decode_refusals(gpu_pkg):
    announce("int4 decode refusals")
    c = cache_case(gpu_pkg, 5, 2, 2, 128, 64, 32, 0)
    q = randn(gen(1), 2, 8, 1, 128)
    kl = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    f = gpu_pkg.attention_flash_decode_int4
    with pytest.raises(AssertionError):
        f(randn(gen(1), 2, 8, 2, 128), c.kc, c.vc, c.ks, c.vs, kl)
    for args in ((q, c.kc, c.vc, c.ks[..., :3], c.vs, kl), (q, c.kc, c.vc, c.ks.float(), c.vs.float(), kl),
                 (q, c.kc, c.vc, c.ks, c.vs[..., :2], kl), (q, c.kc.to(torch.int8), c.vc.to(torch.int8), c.ks, c.vs, kl),
                 (q, c.kc[..., :32], c.vc[..., :32], c.ks, c.vs, kl), (q, c.kc, c.vc, None, None, kl),
                 (q[:, :7], c.kc, c.vc, c.ks, c.vs, kl), (q, c.kc[:1], c.vc[:1], c.ks[:1], c.vs[:1], kl),
                 (q, c.kc, c.vc, c.ks, c.vs, kl.cpu()), (q, c.kc, c.vc, c.ks, c.vs, kl.long())):
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(ValueError):                              # int8 entry points refuse codes
        gpu_pkg.attention_flash_decode_int8(q, c.kc, c.vc, c.ks[..., 0], c.vs[..., 0], kl)
    p = cache_case(gpu_pkg, 5, 2, 2, 128, 64, 32, 16)
    with pytest.raises(AssertionError):
        gpu_pkg.paged_gqa_int4_flash_decode(q, p.kc, p.vc, p.ks, p.vs, p.bt, kl, 32)
    with pytest.raises(ValueError):
        gpu_pkg.paged_gqa_int4_flash_decode(q, p.kc, p.vc, p.ks, p.vs, p.bt[:1], kl, 16)


# ------------------------------------------------------ used together: the caches


def decode_reference(ks, vs, group):
    k, v = (torch.cat(t, 2) for t in (ks, vs))
    return tuple([I4.values(*I4.quantize(x.float().cpu().numpy(), group)) for x in t] for t in (k, v))


@pytest.mark.parametrize("D,group", [(128, 64), (64, 32), (32, 64)])
def test_kvcache_steps(gpu_pkg, D, group):
    """Prompt in two chunks through prefill_step_attention, then decode steps, over KVCache(kv_dtype="int4")."""
    announce(f"KVCache int4 D {D}")
    B, Hq, H, T = 2, 8, 2, 45
    gr = min(group, D)
    cache = gpu_pkg.KVCache(2, 3, 128, H, D, device=DEV, kv_dtype="int4", group_size=group)
    g = gen(D)
    k0, v0, q0 = randn(g, B, H, T, D), randn(g, B, H, T, D), randn(g, B, Hq, T, D)
    cut = 30
    o1 = gpu_pkg.prefill_step_attention(q0[:, :, :cut], k0[:, :, :cut], v0[:, :, :cut], cache, 1, 0)
    o2 = gpu_pkg.prefill_step_attention(q0[:, :, cut:], k0[:, :, cut:], v0[:, :, cut:], cache, 1, cut)
    rk, rv = cache.read(1, B, T)
    torch.cuda.synchronize()
    kx, vx = decode_reference([k0], [v0], gr)
    assert same(rk, rounded(np.stack(kx), BF16)) and same(rv, rounded(np.stack(vx), BF16))
    assert torch.equal(o1, gpu_pkg.gqa_attention(q0[:, :, :cut], k0[:, :, :cut], v0[:, :, :cut]))
    mixed = [torch.cat([a[:, :, :cut], b[:, :, cut:]], 2) for a, b in ((rk, k0), (rv, v0))]
    assert torch.equal(o2, gpu_pkg.gqa_attention(q0[:, :, cut:], *mixed, causal=True))
    ks, vs = [k0], [v0]
    ctx = gpu_pkg.DecodeCtx(D, DEV)
    for step in range(3):
        q, kn, vn = randn(g, B, Hq, 1, D), randn(g, B, H, 1, D), randn(g, B, H, 1, D)
        ctx.set_position(T + step)
        out = gpu_pkg.decode_step_attention(q, kn, vn, cache, 1, ctx)
        ks.append(kn)
        vs.append(vn)
        torch.cuda.synchronize()
        kx, vx = decode_reference(ks, vs, gr)
        check_decode(out, q, kx, vx, [T + step + 1] * B, f"step {step}", D >= 64)
    assert not cache.k_cache[0].any() and not cache.k_cache[1, B:].any()


def test_prefill_step_of_other_caches(gpu_pkg):
    """prefill_step_attention over the 16-bit cache (its own prefix) and over int8 (its values read back)."""
    announce("prefill_step_attention bf16 / int8")
    B, Hq, H, D, T, cut = 1, 4, 2, 64, 40, 25
    g = gen(2)
    q, k, v = randn(g, B, Hq, T, D), randn(g, B, H, T, D), randn(g, B, H, T, D)
    for kind in (None, torch.int8):
        cache = gpu_pkg.KVCache(1, B, 64, H, D, device=DEV, kv_dtype=kind)
        gpu_pkg.prefill_step_attention(q[:, :, :cut], k[:, :, :cut], v[:, :, :cut], cache, 0, 0)
        out = gpu_pkg.prefill_step_attention(q[:, :, cut:], k[:, :, cut:], v[:, :, cut:], cache, 0, cut)
        pk, pv = cache.read(0, B, cut)
        torch.cuda.synchronize()
        if kind is None:
            assert torch.equal(pk, k[:, :, :cut]) and torch.equal(pv, v[:, :, :cut])
        kk, vv = torch.cat([pk, k[:, :, cut:]], 2), torch.cat([pv, v[:, :, cut:]], 2)
        assert torch.equal(out, gpu_pkg.gqa_attention(q[:, :, cut:], kk, vv, causal=True))


def test_paged_cache_steps_in_a_graph(gpu_pkg):
    """A paged int4 cache: prompt, then one captured step (RoPE + write + attention) replayed, each bit-equal to eager."""
    announce("PagedKVCache int4 in a HIP graph")
    B, Hq, H, D, T0 = 3, 16, 4, 128, 37
    caches = [gpu_pkg.PagedKVCache(1, 4, 100, H, D, device=DEV, kv_dtype="int4", group_size=32) for _ in range(2)]
    g = gen(6)
    k0, v0 = randn(g, B, H, T0, D), randn(g, B, H, T0, D)
    cos, sin = gpu_pkg.RopeFrequencies(D, 128, device=torch.device(DEV)).get(128, dtype=BF16)
    for c in caches:
        c.allocate(B, c.max_blocks_per_seq)
        c.write_prefill(0, B, k0, v0)
        c.set_lengths(B, T0)
        c.seq_lens[1] = 11
    q, k, v = (torch.zeros(B, 1, n, D, dtype=BF16, device=DEV) for n in (Hq, H, H))

    def step(c):
        c.begin_decode_step(B)
        return c.decode_attention(0, c.write_decode_rope(0, q, k, v, cos, sin).transpose(1, 2))

    warm = caches[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = [t.clone() for t in (warm.k_pool, warm.v_pool, warm.k_scale_pool, warm.v_scale_pool, warm.seq_lens)]
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(warm)
    for t, s in zip((warm.k_pool, warm.v_pool, warm.k_scale_pool, warm.v_scale_pool, warm.seq_lens), saved):
        t.copy_(s)
    for i in range(4):
        for t in (q, k, v):
            t.copy_(randn(g, *t.shape))
        graph.replay()
        ref = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i
        for name in ("k_pool", "v_pool", "seq_lens"):
            assert torch.equal(getattr(warm, name), getattr(caches[1], name)), name
    n = warm.seq_lens[:B].tolist()
    assert n == [T0 + 4, 15, T0 + 4]
    rk, _ = warm.read(0, B, max(n))
    assert rk.shape == (B, H, T0 + 4, D) and torch.isfinite(rk).all()


def test_on_two_streams(gpu_pkg):
    announce("int4 on two streams")
    jobs = []
    for seed, D, page in ((1, 128, 16), (2, 64, 0)):
        lens = [3000, 500]
        c = cache_case(gpu_pkg, seed, 2, 4, D, 32, 3000, page)
        c.fill(gpu_pkg, lens)
        q = randn(gen(seed), 2, 16, 1, D)
        jobs.append((c, q, torch.tensor(lens, dtype=torch.int32, device=DEV)))
    want = [c.run(gpu_pkg, q, kl) for c, q, kl in jobs]
    reads = [gpu_pkg.kv_read(c.kc, c.vc, 100, c.ks, c.vs, block_table=c.bt, page_size=c.page) for c, _, _ in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        got = []
        for st, (c, q, kl) in zip(streams, jobs):
            with torch.cuda.stream(st):
                got.append((c.run(gpu_pkg, q, kl), gpu_pkg.kv_read(c.kc, c.vc, 100, c.ks, c.vs, block_table=c.bt,
                                                                   page_size=c.page)))
        torch.cuda.synchronize()
        for (o, r), w, rw in zip(got, want, reads):
            assert torch.equal(o, w) and same(r[0], rw[0]) and same(r[1], rw[1])


def test_plugin_builders(gpu_pkg):
    announce("int4 cache builders")
    plugins = importlib.import_module("simple-inference-autoresearch_amd.plugins")
    cfg = type("C", (), dict(num_hidden_layers=2, num_key_value_heads=2, head_dim=64))()
    a = plugins.llama_cache_builder(cfg, max_batch=1, max_seq_len=300, dtype=BF16, device=DEV, kv_dtype="int4")
    b = plugins.llama_paged_cache_builder(cfg, max_batch=1, max_seq_len=300, dtype=BF16, device=DEV, kv_dtype="int4",
                                          group_size=32)
    assert a.is_int4 and a.k_scale.shape[-1] == 2 and b.is_int4 and b.k_scale_pool.shape[-1] == 4


def test_c_abi(gpu_pkg):
    """The C entry points directly, into a NaN-filled output."""
    announce("int4 C ABI")
    h = L.require_library()
    lens = [0, 300, 0, 77]
    c = cache_case(gpu_pkg, 3, 4, 2, 128, 64, 300, 16)
    k, v = c.fill(gpu_pkg, lens)
    q = randn(gen(3), 4, 8, 1, 128)
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.full((4, 1, 8, 128), float("nan"), dtype=BF16, device=DEV)
    ws = torch.empty(gpu_pkg.decode_workspace_size(4, 8, 2, 128), dtype=torch.uint8, device=DEV)
    ds = [ctypes.byref(L.desc(t)) for t in (q, c.kc, c.vc, c.ks, c.vs, c.bt, kl)]
    rc = h.sia_paged_gqa_int4_flash_decode(*ds, 16, 128 ** -0.5, ctypes.byref(L.desc(out)), ws.data_ptr(), ws.numel(),
                                           None, L.stream_handle(q.device))
    torch.cuda.synchronize()
    assert rc == 0
    check_decode(out, q, k, v, lens, "C ABI", True)
