"""Scored attention over prompts against the float64 definition (``oracle/scored.py``).

Tolerances.  16-bit inputs: a weight enters P V in 16 bits, off by at most half a step of fp16, 2^-11 of it (bf16 decode
splits it in two bf16 parts, 2^-16), and is what it is for scores off by up to 2^-14 of a weight (fp32 sums of 256 products
of magnitude 16, and the cap's 2^-22 c): 2^-10 of the largest |v| before the output's own rounding.  float32: scores of up
to 64 log2 units rounded at 2^-24 of it, times a few roundings: 2^-15 of the largest |v|.
"""

from __future__ import annotations

import pytest
import torch

from helpers import announce, assert_close
from oracle import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = float("nan")


def tol(v, dtype):
    top = float(v[torch.isfinite(v)].abs().max()) if v.numel() else 1.0
    return top * (2.0 ** -15 if dtype == torch.float32 else 2.0 ** -10)


def qkv(B, heads, Tq, Tk, D, dtype, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (torch.randn(B, Tq, heads[0], D, generator=g, device=DEV) * 2).to(dtype).transpose(1, 2)
    k, v = (torch.randn(B, Tk, heads[1], D, generator=g, device=DEV).to(dtype).transpose(1, 2) for _ in range(2))
    return q, k, v


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def i32cpu(*x):
    return torch.tensor(x, dtype=torch.int32)


def slopes_of(n):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / n) for h in range(n)], device=DEV)


def check(gpu_pkg, q, k, v, what, causal=True, softcap=None, slopes=None, window=None, cuts=None, prefix=None, start=None,
          length=None, hide=None):
    """One call against the definition; ``hide(k, v)`` spoils what nobody sees after the reference is taken."""
    announce(what)
    out = gpu_pkg.scored_attention_flash(
        q, k, v, causal=causal, softcap=softcap, alibi_slopes=slopes, window=window,
        cu_seqlens=None if cuts is None else torch.tensor(cuts, dtype=torch.int32, device=DEV),
        prefix_len=prefix, kv_start=start, kv_len=length)
    ref = S.scored_attention(*(t.double().cpu() for t in (q, k, v)), causal=causal, softcap=softcap,
                             slopes=None if slopes is None else slopes.cpu(), window=window, cuts=cuts, prefix=prefix,
                             start=start, length=length)
    assert_close(out, ref.numpy(), tol(v.float(), q.dtype), what)
    return out


OPTIONS = {
    "cap": dict(softcap=20.0),
    "cap full": dict(softcap=5.0, causal=False),
    "alibi": dict(slopes=True),
    "alibi full": dict(slopes=True, causal=False),
    "window": dict(window=37),
    "window full": dict(window=70, causal=False),
    "window 1": dict(window=1),
    "documents": dict(cuts=True),
    "documents full": dict(cuts=True, causal=False),
    "prefix": dict(prefix=True),
    "padded": dict(start=True, length=True),
    "padded full": dict(start=True, length=True, causal=False),
    "all": dict(softcap=20.0, slopes=True, window=90, cuts=True, prefix=True, start=True, length=True),
    "all full": dict(softcap=20.0, slopes=True, window=90, cuts=True, start=True, length=True, causal=False),
}


def options(name, B, heads, Tk):
    o = dict(OPTIONS[name])
    if o.get("slopes"):
        o["slopes"] = slopes_of(heads[0])
    if o.get("cuts"):
        o["cuts"] = [0, Tk // 5, Tk // 5 + 1, Tk // 2 + 3, Tk - 2, Tk]
    if o.get("prefix"):
        o["prefix"] = i32(*[(b * 53 + Tk // 2) % (Tk + 1) for b in range(B)])
    if o.get("start"):
        o["start"] = i32(*[(b * 31) % (Tk // 2 + 1) for b in range(B)])
    if o.get("length"):
        o["length"] = i32(*[Tk - (b * 17) % (Tk // 3 + 1) for b in range(B)])
    return o


@pytest.mark.parametrize("name", list(OPTIONS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,heads,Tq,Tk", [(128, (8, 2), 200, 200), (64, (6, 6), 131, 300), (256, (4, 1), 65, 97)])
def test_options(gpu_pkg, name, dtype, D, heads, Tq, Tk):
    q, k, v = qkv(3, heads, Tq, Tk, D, dtype)
    check(gpu_pkg, q, k, v, f"{name} {dtype} D={D} {heads} {Tq}+{Tk - Tq}", **options(name, 3, heads, Tk))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [(5, 1), (12, 4), (16, 2)])
def test_head_layouts(gpu_pkg, dtype, D, heads):
    q, k, v = qkv(2, heads, 70, 133, D, dtype, seed=2)
    check(gpu_pkg, q, k, v, f"heads {heads} D={D} {dtype}", **options("all", 2, heads, 133))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (2, 2), (1, 500), (2, 65), (31, 64), (33, 63), (64, 64), (65, 128), (257, 257),
                                   (100, 40), (5, 700), (513, 600)])
@pytest.mark.parametrize("name", ["cap", "window", "documents full", "all"])
def test_lengths(gpu_pkg, D, Tq, Tk, name):
    q, k, v = qkv(1, (8, 2), Tq, Tk, D, torch.bfloat16, seed=3)
    check(gpu_pkg, q, k, v, f"{name} Tq={Tq} Tk={Tk} D={D}", **options(name, 1, (8, 2), Tk))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf"), "lowest"])
def test_hidden_keys(gpu_pkg, dtype, D, bad):
    """Whatever stands in padding, in another document or outside the window does not reach a row."""
    bad = torch.finfo(dtype).min if bad == "lowest" else bad
    B, heads, T = 2, (4, 2), 300
    q, k, v = qkv(B, heads, T, T, D, dtype, seed=4)
    start, length = i32(10, 70), i32(290, 200)
    cuts = [0, 64, 101, 230]
    args = dict(softcap=30.0, window=50, cu_seqlens=i32(*cuts), kv_start=start, kv_len=length)
    announce(f"hidden {bad} {dtype} D={D}")
    ref = S.scored_attention(*(t.double().cpu() for t in (q, k, v)), softcap=30.0, window=50, cuts=cuts, start=start,
                             length=length).numpy()
    atol = tol(v.float(), dtype)
    for b in range(B):
        for x in (k, v):
            x[b, :, :int(start[b])] = bad
            x[b, :, int(length[b]):] = bad
    assert_close(gpu_pkg.scored_attention_flash(q, k, v, **args), ref, atol, "spoiled padding")
    # one document's keys, spoiled, reach its own rows alone
    for x in (k, v):
        x[:, :, 101:230] = bad
    out = gpu_pkg.scored_attention_flash(q, k, v, **args)
    rows = [*range(0, 101), *range(230, T)]
    assert_close(out[:, :, rows], ref[:, :, rows], atol, "another document spoiled")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(gpu_pkg, dtype, D):
    T = 200
    q, k, v = qkv(1, (4, 2), T, T, D, dtype, seed=5)
    v[:, 0, 77, 3] = float("inf")
    v[:, 1, 130, 5] = NAN
    announce(f"Inf and NaN in V {dtype} D={D}")
    out = gpu_pkg.scored_attention_flash(q, k, v, window=60)
    see = S.visible(T, T, True, 60)
    for h in range(4):
        at, dim = ((77, 3), (130, 5))[h // 2]
        col = out[0, h, :, dim].float().cpu()
        assert (torch.isposinf(col) if h < 2 else torch.isnan(col))[see[:, at]].all()
        assert torch.isfinite(col[~see[:, at]]).all()
        rest = [d for d in range(D) if d != dim]
        assert torch.isfinite(out[0, h][:, rest]).all()


def test_bf16_values_beyond_fp16(gpu_pkg):
    """bf16 keeps its range: no value is cut at fp16's."""
    q, k, v = qkv(1, (4, 2), 150, 150, 128, torch.bfloat16, seed=6)
    v[:, :, ::7] = 3e6
    check(gpu_pkg, q, k, v, "V beyond fp16", softcap=30.0)


def test_rows_without_keys_are_zero(gpu_pkg):
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v = qkv(2, (4, 2), 90, 90, 64, dtype)
        announce(f"rows without keys {dtype}")
        out = gpu_pkg.scored_attention_flash(q, k, v, softcap=10.0, kv_start=i32(0, 40), kv_len=i32(0, 90))
        assert (out[0] == 0).all() and (out[1, :, :40] == 0).all() and (out[1, :, 40:] != 0).any()
        out = gpu_pkg.scored_attention_flash(q, k, v, causal=False, kv_start=i32(90))
        assert (out == 0).all()
        out = gpu_pkg.scored_attention_flash(q, k[:, :, :0], v[:, :, :0], window=4)
        assert out.shape == q.shape and (out == 0).all()
        assert gpu_pkg.scored_attention_flash(q[:, :, :0], k, v, window=4).shape == (2, 4, 0, 64)
        assert gpu_pkg.scored_attention_flash(q[:0], k[:0], v[:0], window=4).shape == (0, 4, 90, 64)


def test_without_options_it_is_plain_attention(gpu_pkg):
    for causal in (True, False):
        q, k, v = qkv(2, (8, 2), 130, 200, 128, torch.bfloat16)
        check(gpu_pkg, q, k, v, f"no option causal={causal}", causal=causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,heads,Tq,Tk", [(128, (8, 2), 5, 4100), (128, (32, 8), 200, 6200), (64, (8, 8), 33, 3100),
                                           (256, (4, 1), 100, 2050)])
@pytest.mark.parametrize("name", ["cap", "window long", "all", "alibi full", "padded"])
def test_few_rows_over_many_keys(gpu_pkg, dtype, D, heads, Tq, Tk, name):
    """Chunks behind a long prefix, whose keys are split over work-groups and merged."""
    q, k, v = qkv(1, heads, Tq, Tk, D, dtype, seed=10)
    o = dict(window=2500) if name == "window long" else options(name, 1, heads, Tk)
    check(gpu_pkg, q, k, v, f"{name} Tq={Tq} Tk={Tk} D={D} {dtype}", **o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_hidden_keys_of_split_calls(gpu_pkg, dtype, D):
    """NaN in padding of every run of a split call; an Inf where only some rows see it."""
    Tq, Tk = 40, 4000
    q, k, v = qkv(1, (4, 2), Tq, Tk, D, dtype, seed=11)
    start, length = i32(1010), i32(3990)
    args = dict(softcap=30.0, kv_start=start, kv_len=length)
    announce(f"hidden keys of a split call {dtype} D={D}")
    ref = S.scored_attention(*(t.double().cpu() for t in (q, k, v)), softcap=30.0, start=start, length=length).numpy()
    atol = tol(v.float(), dtype)
    for x in (k, v):
        x[:, :, :1010] = NAN
        x[:, :, 3990:] = NAN
    assert_close(gpu_pkg.scored_attention_flash(q, k, v, **args), ref, atol, "spoiled padding")
    v[:, 0, 3970, 3] = float("inf")               # query 10 on sees it
    out = gpu_pkg.scored_attention_flash(q, k, v, **args)
    assert torch.isposinf(out[0, :2, 10:, 3]).all()
    rest = [d for d in range(D) if d != 3]
    assert_close(out[..., rest], ref[..., rest], atol, "another dimension")
    assert_close(out[:, :, :10], ref[:, :, :10], atol, "rows before it")
    assert_close(out[:, 2:], ref[:, 2:], atol, "other heads")


def test_documents_in_any_order_and_per_sequence(gpu_pkg):
    q, k, v = qkv(2, (8, 2), 333, 333, 128, torch.bfloat16, seed=7)
    announce("cu_seqlens in another order, with others among them")
    a = gpu_pkg.scored_attention_flash(q, k, v, cu_seqlens=i32(0, 50, 51, 200, 333))
    b = gpu_pkg.scored_attention_flash(q, k, v, cu_seqlens=i32(200, -5, 51, 50, 50, 100000, 0, -2 ** 31, 2 ** 31 - 1))
    assert torch.equal(a, b)
    rows = torch.tensor([[0, 50, 51, 200], [0, 7, 300, 333]], dtype=torch.int32, device=DEV)
    c = gpu_pkg.scored_attention_flash(q, k, v, cu_seqlens=rows)
    assert torch.equal(c[0], a[0])
    ref = S.scored_attention(*(t.double().cpu() for t in (q, k, v)), cuts=rows.tolist())
    assert_close(c, ref.numpy(), tol(v.float(), q.dtype), "cu_seqlens per sequence")
    many = torch.arange(0, 333, 2, dtype=torch.int32, device=DEV)
    check(gpu_pkg, q, k, v, "167 documents", cuts=many.tolist())


def test_views_layouts_and_streams(gpu_pkg):
    B, heads, T, D = 2, (8, 2), 140, 128
    g = torch.Generator(device=DEV).manual_seed(8)
    qkv_ = torch.randn(B, T, heads[0] + 2 * heads[1], D, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = (x.transpose(1, 2) for x in qkv_.split([heads[0], heads[1], heads[1]], dim=2))
    announce("slices of a fused projection, token-major output, another stream")
    args = dict(softcap=30.0, window=64, alibi_slopes=slopes_of(heads[0]))
    want = gpu_pkg.scored_attention_flash(q.contiguous(), k.contiguous(), v.contiguous(), **args)
    assert torch.equal(gpu_pkg.scored_attention_flash(q, k, v, **args), want)
    assert torch.equal(gpu_pkg.scored_attention_flash(q, k, v, out_token_major=True, **args).transpose(1, 2), want)
    odd = torch.randn(B, heads[1], T, D + 3, generator=g, device=DEV).to(torch.bfloat16)[..., 1:D + 1]   # rows that start anywhere
    assert torch.equal(gpu_pkg.scored_attention_flash(q, odd, v, **args),
                       gpu_pkg.scored_attention_flash(q, odd.contiguous(), v, **args))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gpu_pkg.scored_attention_flash(q, k, v, **args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_captured_and_replayed(gpu_pkg, dtype):
    """One graph serves every mask: bounds, prefixes and documents are read on the device."""
    q, k, v = qkv(2, (8, 2), 100, 160, 128, dtype, seed=9)
    start, length, prefix, cuts = i32(0, 5), i32(160, 100), i32(0, 40), i32(0, 30, 90)
    args = dict(softcap=25.0, window=80, kv_start=start, kv_len=length, prefix_len=prefix, cu_seqlens=cuts,
                alibi_slopes=slopes_of(8))
    announce(f"captured {dtype}")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu_pkg.scored_attention_flash(q, k, v, **args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu_pkg.scored_attention_flash(q, k, v, **args)
    for i in range(3):
        start.copy_(i32(i, 7 * i))
        length.copy_(i32(160 - 9 * i, 100 + i))
        prefix.copy_(i32(20 * i, 3))
        cuts.copy_(i32(0, 30 + i, 90 - 20 * i))
        q.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gpu_pkg.scored_attention_flash(q, k, v, **args))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,Tq,Tk", [(128, 100, 160), (64, 33, 3000), (256, 40, 40)])
def test_bounds_far_outside(gpu_pkg, dtype, D, Tq, Tk):
    """First keys, lengths, prefixes and windows at the ends of their types mean none or all."""
    q, k, v = qkv(1, (4, 2), Tq, Tk, D, dtype, seed=12)
    lo, hi = -2 ** 31, 2 ** 31 - 1
    announce(f"bounds far outside {dtype} D={D}")
    plain = gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0)
    for same in (dict(kv_start=i32(lo)), dict(kv_len=i32(hi)), dict(prefix_len=i32(lo)), dict(window=hi), dict(window=2 ** 40),
                 dict(kv_start=i32(lo), kv_len=i32(hi), prefix_len=i32(-1), window=hi, cu_seqlens=i32(lo, hi, 0))):
        assert torch.equal(gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0, **same), plain), same
    full = gpu_pkg.scored_attention_flash(q, k, v, causal=False, softcap=30.0)
    check(gpu_pkg, q, k, v, "a prefix of everything", softcap=30.0, prefix=i32(hi))
    assert_close(gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0, prefix_len=i32(hi)), full.double().cpu().numpy(),
                 2 * tol(v.float(), dtype), "prefix of everything, full")
    for none in (dict(kv_start=i32(hi)), dict(kv_len=i32(lo)), dict(kv_len=i32(0)), dict(kv_start=i32(Tk), prefix_len=i32(hi)),
                 dict(kv_start=i32(hi), kv_len=i32(lo), window=hi, cu_seqlens=i32(hi, lo))):
        assert (gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0, **none) == 0).all(), none


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_query_that_is_not_finite_stays_alone(gpu_pkg, dtype):
    q, k, v = qkv(2, (8, 2), 150, 150, 128, dtype, seed=13)
    announce(f"NaN in q {dtype}")
    want = gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0, window=60)
    q[1, 3, 77] = NAN
    out = gpu_pkg.scored_attention_flash(q, k, v, softcap=30.0, window=60)
    assert torch.isnan(out[1, 3, 77]).all()
    out[1, 3, 77] = want[1, 3, 77]
    assert torch.equal(out, want)


@pytest.mark.parametrize("cap", [1e-30, 1e30])
def test_caps_without_measure(gpu_pkg, cap):
    """A cap far below every score leaves equal weights, one far above every score leaves the scores."""
    q, k, v = qkv(1, (4, 2), 70, 70, 64, torch.bfloat16, seed=15)
    announce(f"cap {cap}")
    check(gpu_pkg, q, k, v, f"cap {cap}", softcap=cap)
    for none in (1e-50, 1e39):                       # no float32 holds them
        with pytest.raises(ValueError):
            gpu_pkg.scored_attention_flash(q, k, v, softcap=none)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("heads", [(4, 1), (2, 2)])
@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(softcap=30.0, window=700), dict(prefix=i32cpu(650)),
                                dict(cuts=[0, 33, 640, 1000]), dict(start=i32cpu(0, 950), length=i32cpu(560, 1055))],
                         ids=["causal", "full", "window", "prefix", "documents", "padding"])
def test_biases_over_many_blocks(gpu_pkg, dtype, D, heads, kw):
    """Slopes that raise the scores towards the last block, or (negative) towards the first, whoever sees it."""
    q, k, v = qkv(2, heads, 1055, 1055, D, dtype, seed=17)
    kw = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    slopes = torch.tensor([0.7, -0.02, 0.004, -0.3][:heads[0]], device=DEV)
    check(gpu_pkg, q, k, v, f"many blocks {dtype} {D} {heads} {list(kw)}", slopes=slopes, **kw)


def test_biases_of_a_large_call(gpu_pkg):
    q, k, v = qkv(8, (4, 1), 2100, 2100, 128, torch.bfloat16, seed=18)
    slopes = torch.tensor([0.7, 0.1, 0.004, -0.01], device=DEV)
    k[:, :, :3], v[:, :, :3] = NAN, NAN
    announce("2100 tokens in 8 rows, biased")
    out = gpu_pkg.scored_attention_flash(q, k, v, alibi_slopes=slopes, kv_start=i32(3))
    for b in (0, 7):
        ref = S.scored_attention(*(t[b:b + 1].double().cpu() for t in (q, torch.nan_to_num(k), torch.nan_to_num(v))),
                                 slopes=slopes.cpu(), start=torch.tensor([3]))
        assert_close(out[b:b + 1], ref.numpy(), tol(v.float(), q.dtype), f"row {b}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale,cap", [(1e-30, None), (0.1, 1e-30), (1e-30, 20.0)])
def test_slopes_beside_a_vanishing_unit(gpu_pkg, D, scale, cap):
    """Scores or a cap next to 0 leave the bias alone, however far the keys."""
    q, k, v = qkv(1, (4, 2), 300, 300, D, torch.bfloat16, seed=16)
    announce(f"scale {scale} cap {cap}")
    out = gpu_pkg.scored_attention_flash(q, k, v, sm_scale=scale, softcap=cap, alibi_slopes=slopes_of(4))
    ref = S.scored_attention(*(t.double().cpu() for t in (q, k, v)), sm_scale=scale, softcap=cap, slopes=slopes_of(4).cpu())
    assert_close(out, ref.numpy(), tol(v.float(), q.dtype), f"scale {scale} cap {cap}")


def test_single_queries_of_any_view(gpu_pkg):
    q, k, v = qkv(2, (8, 2), 1, 90, 128, torch.bfloat16, seed=14)
    odd = torch.zeros(2, 2, 90, 131, dtype=k.dtype, device=DEV)[..., 1:129]
    odd.copy_(k)
    announce("a single query over a view whose rows start anywhere")
    check(gpu_pkg, q, odd, v, "odd rows", softcap=30.0, window=50)


def test_refusals(gpu_pkg):
    f = gpu_pkg.scored_attention_flash
    q, k, v = qkv(2, (8, 2), 20, 20, 64, torch.bfloat16)
    for bad in (dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=NAN), dict(softcap=float("inf")), dict(window=0),
                dict(window=-3), dict(alibi_slopes=slopes_of(4)), dict(alibi_slopes=slopes_of(8).half()),
                dict(alibi_slopes=slopes_of(16)[::2]), dict(kv_start=i32(1, 2, 3)), dict(kv_len=i32(1, 2).long()),
                dict(prefix_len=i32(1, 2, 3, 4)[::2]), dict(kv_len=torch.tensor([1], dtype=torch.int32)),
                dict(cu_seqlens=torch.tensor([0, 3], device=DEV)), dict(cu_seqlens=torch.zeros(3, 2, dtype=torch.int32, device=DEV)),
                dict(cu_seqlens=torch.zeros(2, 4, dtype=torch.int32, device=DEV)[:, ::2]), dict(sm_scale=0.0),
                dict(sm_scale=NAN)):
        announce(f"refused {list(bad)}")
        with pytest.raises(ValueError):
            f(q, k, v, **bad)
    with pytest.raises(AssertionError):
        f(q[..., :48], k[..., :48], v[..., :48])
    with pytest.raises(ValueError):
        f(q, k.half(), v.half())
    with pytest.raises(ValueError):
        f(q[:, :7], k, v)
    with pytest.raises(ValueError):
        f(q.cpu(), k, v)
