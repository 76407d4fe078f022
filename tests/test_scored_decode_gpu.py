"""Scored decode attention, over every cache format, against the float64 definition (``oracle/scored.py``).

Tolerances: those of the 16-bit products (2^-10 of the largest |v|: half a step of an fp16 weight is 2^-11 of it, scores are
off by up to 2^-14 of a weight) and of float32 (2^-15); int8 caches add the query's three int8 terms, 2^-17 of the largest
element each over 256 products of magnitude 8: 2^-9 of the largest |v|.
"""

from __future__ import annotations

import pytest
import torch

from helpers import announce, assert_close
from oracle import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def slopes_of(n):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / n) for h in range(n)], device=DEV)


class Case:
    """A cache of ``fmt`` ("same", "int8", "int8 fp16", "int4"), contiguous (page 0) or paged, and the values it holds."""

    def __init__(self, gpu_pkg, lens, heads, D, dtype, fmt="same", page=0, seed=1, kv_dtype=None):
        self.pkg, self.lens, self.page, self.fmt = gpu_pkg, lens, page, fmt
        B, H = len(lens), heads[1]
        g = torch.Generator(device=DEV).manual_seed(seed)
        S_ = max(max(lens), 1)
        kv_dtype = kv_dtype or dtype
        self.q = (torch.randn(B, heads[0], 1, D, generator=g, device=DEV) * 2).to(dtype)
        k, v = (torch.randn(B, H, S_, D, generator=g, device=DEV).to(kv_dtype) for _ in range(2))
        self.ks = self.vs = None
        if fmt.startswith("int8"):
            sd = torch.float16 if fmt.endswith("fp16") else torch.float32
            (k, self.ks), (v, self.vs) = gpu_pkg.quantize_kv_int8(k, sd), gpu_pkg.quantize_kv_int8(v, sd)
            self.kd, self.vd = k.double() * self.ks.double()[..., None], v.double() * self.vs.double()[..., None]
        elif fmt == "int4":
            (k, self.ks), (v, self.vs) = gpu_pkg.quantize_kv_int4(k, 32), gpu_pkg.quantize_kv_int4(v, 32)
            self.kd, self.vd = (gpu_pkg.dequantize_kv_int4(c, p, torch.float32).double() for c, p in ((k, self.ks), (v, self.vs)))
        else:
            self.kd, self.vd = k.double(), v.double()
        self.k, self.v, self.bt = k, v, None
        self.kv_len = i32(*lens)
        if page:
            self._to_pages(seed)

    def _to_pages(self, seed):
        B, page = len(self.lens), self.page
        nb = -(-self.k.shape[2] // page)
        perm = torch.randperm(B * nb + 3, generator=torch.Generator().manual_seed(seed))[:B * nb].view(B, nb)
        self.bt = perm.to(torch.int32).to(DEV)

        def pool(x):
            if x is None:
                return None
            out = torch.zeros((B * nb + 3, x.shape[1], page) + x.shape[3:], dtype=x.dtype, device=DEV)
            for b in range(B):
                for i in range(nb):
                    part = x[b, :, i * page:(i + 1) * page]
                    out[perm[b, i], :, :part.shape[1]] = part
            return out

        self.k, self.v, self.ks, self.vs = pool(self.k), pool(self.v), pool(self.ks), pool(self.vs)

    def run(self, **o):
        if self.bt is None:
            return self.pkg.scored_attention_flash_decode(self.q, self.k, self.v, self.kv_len, self.ks, self.vs, **o)
        return self.pkg.paged_scored_attention_flash_decode(self.q, self.k, self.v, self.bt, self.kv_len, self.page,
                                                            self.ks, self.vs, **o)

    def ref(self, softcap=None, alibi_slopes=None, window=None, kv_start=None, sm_scale=None):
        out = torch.zeros(len(self.lens), 1, self.q.shape[1], self.q.shape[3], dtype=torch.float64)
        for b, n in enumerate(self.lens):
            if n == 0:
                continue
            st = None if kv_start is None else [int(kv_start[b if len(kv_start) > 1 else 0])]
            o = S.scored_attention(self.q[b:b + 1].double().cpu(), self.kd[b:b + 1, :, :n].cpu(), self.vd[b:b + 1, :, :n].cpu(),
                                   softcap=softcap, slopes=None if alibi_slopes is None else alibi_slopes.cpu(),
                                   window=window, start=st, sm_scale=sm_scale)
            out[b, 0] = o[0, :, 0]
        return out.numpy()

    def atol(self):
        top = float(self.vd[torch.isfinite(self.vd)].abs().max())
        return top * (2.0 ** -15 if self.q.dtype == torch.float32 else 2.0 ** -9 if self.fmt.startswith("int8") else 2.0 ** -10)

    def check(self, what, **o):
        announce(what)
        out = self.run(**o)
        assert_close(out, self.ref(**o), self.atol(), what)
        return out


OPTIONS = {
    "cap": lambda n, B: dict(softcap=20.0),
    "alibi": lambda n, B: dict(alibi_slopes=slopes_of(n)),
    "window": lambda n, B: dict(window=100),
    "window 1": lambda n, B: dict(window=1),
    "start": lambda n, B: dict(kv_start=i32(*[(37 * b) % 300 for b in range(B)])),
    "all": lambda n, B: dict(softcap=20.0, alibi_slopes=slopes_of(n), window=333,
                             kv_start=i32(*[(37 * b) % 300 for b in range(B)])),
}


@pytest.mark.parametrize("name", list(OPTIONS))
@pytest.mark.parametrize("dtype,fmt", [(torch.bfloat16, "same"), (torch.float16, "same"), (torch.float32, "same"),
                                       (torch.bfloat16, "int8"), (torch.float16, "int8 fp16"), (torch.float32, "int8"),
                                       (torch.bfloat16, "int4")])
@pytest.mark.parametrize("D,heads", [(128, (8, 2)), (64, (6, 6)), (256, (4, 1))])
@pytest.mark.parametrize("page", [0, 16])
def test_options(gpu_pkg, name, dtype, fmt, D, heads, page):
    lens = [700, 1, 0, 333, 16, 512]
    c = Case(gpu_pkg, lens, heads, D, dtype, fmt, page)
    c.check(f"{name} {dtype} {fmt} D={D} {heads} page={page}", **OPTIONS[name](heads[0], len(lens)))


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("fmt", ["same", "int8", "int4"])
@pytest.mark.parametrize("page", [0, 1, 8, 24, 32, 64])
def test_pages_and_head_dims(gpu_pkg, D, fmt, page):
    c = Case(gpu_pkg, [200, 77, 129], (20, 1), D, torch.bfloat16, fmt, page, seed=2)
    c.check(f"pages of {page} D={D} {fmt}", **OPTIONS["all"](20, 3))


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 100, 1000, 5000])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 4096, 2 ** 31 - 1, 2 ** 40])
def test_windows_and_lengths(gpu_pkg, n, window):
    """One shared length, the window's first key anywhere in its tile."""
    for D, heads in ((128, (8, 2)), (64, (8, 8)), (256, (4, 2))):
        c = Case(gpu_pkg, [n] * 2, heads, D, torch.bfloat16, seed=n)
        c.kv_len = i32(n)
        c.check(f"n={n} window={window} D={D}", window=window, softcap=30.0)


@pytest.mark.parametrize("B", [1, 40, 70, 300])
def test_batches(gpu_pkg, B):
    """Lengths and first keys of their own, shared lengths with first keys of their own, both shared; first keys past the end."""
    lens = [(b * 97 + 5) % 400 for b in range(B)]
    c = Case(gpu_pkg, lens, (8, 2), 64, torch.float16, page=16, seed=B)
    start = i32(*[(b * 61) % 450 for b in range(B)])
    c.check(f"B={B} ragged", kv_start=start, softcap=25.0)
    c.check(f"B={B} one first key", kv_start=i32(33), alibi_slopes=slopes_of(8))
    c = Case(gpu_pkg, [350] * B, (8, 2), 128, torch.float16, seed=B)
    c.kv_len = i32(350)
    c.check(f"B={B} one length", kv_start=start, window=200)
    c.check(f"B={B} one length and first key", kv_start=i32(77))
    assert (c.run(kv_start=i32(350)) == 0).all() and (c.run(kv_start=i32(10 ** 6)) == 0).all()
    c.check(f"B={B} a first key below 0", kv_start=i32(-5))


@pytest.mark.parametrize("tiles", [1, 3, 7])
def test_split_and_merged(gpu_pkg, tiles):
    for fmt in ("same", "int8"):
        for D in (64, 128, 256):
            c = Case(gpu_pkg, [900, 33, 500], (8, 2), D, torch.bfloat16, fmt, 16, seed=3)
            with gpu_pkg.decode_options(tiles_per_split=tiles):
                c.check(f"pieces of {tiles} tiles, {fmt}, D={D}", **OPTIONS["all"](8, 3))


@pytest.mark.parametrize("fmt", ["same", "int8", "int8 fp16"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_hidden_tokens(gpu_pkg, fmt, D, dtype):
    """NaN before the window, in other pages and behind the sequence changes no bit; table entries there are not used."""
    if dtype == torch.float32 and fmt == "int8 fp16":
        fmt = "int8"
    lens = [500, 130, 64]
    args = dict(softcap=30.0, window=75, kv_start=i32(430, 0, 20))
    announce(f"hidden tokens {fmt} D={D} {dtype}")
    for page in (0, 16):
        c = Case(gpu_pkg, lens, (8, 2), D, dtype, fmt, page, seed=4)
        want = c.run(**args)
        assert_close(want, c.ref(**args), c.atol(), "hidden tokens")
        first = [430, 55, 20]
        for x in (c.k, c.v, c.ks, c.vs):
            if x is None:
                continue
            bad = NAN if x.dtype.is_floating_point else -128
            if page == 0:
                for b in range(3):
                    x[b, :, :first[b]] = bad
                    x[b, :, lens[b]:] = bad
            else:
                keep = torch.zeros(x.shape[0], page, dtype=torch.bool)
                for b in range(3):
                    for t in range(first[b], lens[b]):
                        keep[int(c.bt[b, t // page]), t % page] = True
                m = (~keep.to(DEV))[:, None].expand(-1, x.shape[1], -1)
                x.masked_fill_(m if x.dim() == 3 else m[..., None], bad)
        if page:
            for b in range(3):
                c.bt[b, :first[b] // page] = (-1, 10 ** 6, 2 ** 31 - 1)[b]
        assert torch.equal(c.run(**args), want)


def test_captured_and_replayed(gpu_pkg):
    """One graph serves every length and first key, of its own or shared."""
    for fmt, D in (("same", 128), ("int8", 64), ("same", 256), ("int4", 128)):
        c = Case(gpu_pkg, [600, 40, 300], (8, 2), D, torch.bfloat16, fmt, 16, seed=5)
        start = i32(0, 10, 20)
        args = dict(softcap=30.0, window=256, kv_start=start, alibi_slopes=slopes_of(8))
        announce(f"captured {fmt} D={D}")
        c.run(**args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.run(**args)
        for n, s in (((600, 1, 0), (599, 0, 5)), ((17, 600, 555), (0, 16, 500)), ((333, 333, 333), (0, 0, 0))):
            c.kv_len.copy_(i32(*n))
            start.copy_(i32(*s))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, c.run(**args))


def test_large_cap_and_scores(gpu_pkg):
    """Caps past the matrix kernels' limit, scores far past the cap on both sides."""
    for D in (64, 128):
        c = Case(gpu_pkg, [300, 77], (8, 2), D, torch.float16, seed=6)
        c.check("cap 5000", softcap=5000.0)
        c.check("scores past the cap", softcap=3.0, sm_scale=4.0)


def test_refusals(gpu_pkg):
    c = Case(gpu_pkg, [60, 7], (8, 2), 64, torch.bfloat16)
    for bad in (dict(softcap=0.0), dict(softcap=NAN), dict(window=0), dict(alibi_slopes=slopes_of(2)), dict(kv_start=i32(1, 2, 3)),
                dict(kv_start=torch.tensor([1.0], device=DEV)), dict(kv_start=torch.tensor([1], dtype=torch.int32)),
                dict(sm_scale=-1.0)):
        announce(f"refused {list(bad)}")
        with pytest.raises(ValueError):
            c.run(**bad)
    f = gpu_pkg.scored_attention_flash_decode
    with pytest.raises(ValueError):
        f(c.q, c.k, c.v, c.kv_len, torch.zeros(2, 2, 60, device=DEV), torch.zeros(2, 2, 60, device=DEV))   # scales of a 16-bit cache
    with pytest.raises(ValueError):
        f(c.q, c.k.to(torch.int8), c.v.to(torch.int8), c.kv_len)                                           # and none of an int8 one
    with pytest.raises(AssertionError):
        f(c.q.expand(-1, -1, 2, -1), c.k, c.v, c.kv_len)
    p = Case(gpu_pkg, [60, 7], (8, 2), 64, torch.bfloat16, page=16)
    with pytest.raises(AssertionError):
        gpu_pkg.paged_scored_attention_flash_decode(p.q, p.k, p.v, p.bt, p.kv_len, 32)
    assert f(c.q[:0], c.k[:0], c.v[:0], i32(), softcap=3.0).shape == (0, 1, 8, 64)
