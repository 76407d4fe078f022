"""CPU checks of the 4-bit K/V format (oracle/int4.py) and of the C entry points' refusals."""

from __future__ import annotations

import ctypes
import importlib

import numpy as np
import pytest
import torch  # noqa: F401  (torch's HIP runtime must be loaded before the library)

from conftest import PKG_NAME, load_pkg
from oracle import int4 as I4


@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_pack_is_a_permutation(D):
    codes = np.random.default_rng(D).integers(0, 16, (5, D)).astype(np.uint8)
    assert sorted(I4.word_place(p, D) for p in range(D // 8)) == list(range(D // 8))
    np.testing.assert_array_equal(I4.unpack(I4.pack(codes)), codes)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_k_step_stays_inside_one_group(D):
    """Word j of the 16 (D = 64: 8) bytes that each of 4 lanes loads covers 32 consecutive elements."""
    block = min(D, 128)
    per = block // 32
    word = {I4.word_place(p, D): p for p in range(D // 8)}
    for b in range(D // block):
        for j in range(per):
            p = [word[b * (block // 8) + g * per + j] for g in range(4)]
            assert p == [b * (block // 8) + 4 * j + g for g in range(4)]


@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e4])
def test_values_are_within_half_a_step(scale):
    """|x^ - x| <= s / 2 + what rounding s down costs (15 s 2^-10) + the rounding of m (2^-11 |m|) + fp32 roundings."""
    x = (np.random.default_rng(1).standard_normal((200, 128)) * scale).astype(np.float32)
    codes, par = I4.quantize(x, 32)
    v = I4.values(codes, par)
    s = np.repeat(par[:, 0::2].astype(np.float64), 32, -1)
    m = np.repeat(par[:, 1::2].astype(np.float64), 32, -1)
    # (the parameters' spacing is 2^-24 below 2^-14: m is off by at most half of it, 15 s by 15 times it)
    tiny = 15.5 * 2.0 ** -24
    xc = np.clip(x.astype(np.float64), -65504, 65504)
    assert (np.abs(v - xc) <= s / 2 + 15 * s * 2.0 ** -10 + np.abs(m) * 2.0 ** -11 + tiny + 1e-6 * np.abs(xc)).all()
    hi = xc.reshape(200, 4, 32).max(-1)
    top = par[:, 1::2].astype(np.float64) + 15 * par[:, 0::2].astype(np.float64)
    assert (top <= np.maximum(hi, par[:, 1::2].astype(np.float64)) * (1 + np.sign(hi) * 2.0 ** -22)).all()


def test_special_groups():
    x = np.zeros((6, 32), np.float32)
    x[0] = 3.0
    x[1, 5] = np.nan
    x[2, 7] = np.inf
    x[3, :2] = [1e30, -1e30]
    x[4] = np.linspace(0, 15, 32)
    codes, par = I4.quantize(x, 32)
    v = I4.values(codes, par)
    assert (v[0] == 3).all() and np.isnan(v[1]).all() and np.isnan(v[2]).all() and (v[5] == 0).all()
    assert np.isfinite(v[3]).all() and v[3, 1] == -65504 and v[3, 0] <= 65504
    assert par[4, 0] == 1 and par[4, 1] == 0


# ------------------------------------------------------------------- refusals


def _desc(lm, dtype, shape, addr=0x10000, stride=None):
    t = lm.SiaTensor()
    t.data, t.dtype, t.ndim = addr, dtype, len(shape)
    n = 1
    for i in reversed(range(len(shape))):
        t.shape[i], t.stride[i] = shape[i], n
        n *= shape[i]
    for i, s in (stride or {}).items():
        t.stride[i] = s
    return t


def _read_args(lm, **kw):
    """A valid read of 4 tokens of a contiguous int4 cache (2, 3, 40, 128), groups of 64, but for ``kw``."""
    U8, F16, BF16 = lm.SIA_U8, lm.SIA_F16, lm.SIA_BF16
    a = {"k": _desc(lm, U8, (2, 3, 40, 64)), "v": _desc(lm, U8, (2, 3, 40, 64)), "ks": _desc(lm, F16, (2, 3, 40, 4)),
         "vs": _desc(lm, F16, (2, 3, 40, 4)), "bt": None, "sp": None, "start": 36, "page": 0,
         "ko": _desc(lm, BF16, (2, 3, 4, 128)), "vo": _desc(lm, BF16, (2, 3, 4, 128))}
    a.update(kw)
    return [ctypes.byref(x) if isinstance(x, lm.SiaTensor) else x for x in a.values()]


def test_read_refusals_come_before_the_device():
    lib, lm = load_pkg().load_library(), importlib.import_module(PKG_NAME + "._lib")
    U8, F16, BF16, I32, F32 = lm.SIA_U8, lm.SIA_F16, lm.SIA_BF16, lm.SIA_I32, lm.SIA_F32
    if not torch.cuda.is_available():     # a valid call is stopped by the device check only
        assert lib.sia_kv_read(*_read_args(lm), None) == lm.SIA_ERR_DEVICE
    bad = [
        dict(start=37), dict(start=-1), dict(vo=None), dict(v=None, vo=None, k=None),
        dict(ks=None), dict(vs=None), dict(ks=_desc(lm, F32, (2, 3, 40, 4))), dict(ks=_desc(lm, F16, (2, 3, 40, 3))),
        dict(ks=_desc(lm, F16, (2, 3, 40, 6))), dict(ks=_desc(lm, F16, (2, 3, 39, 4))),
        dict(ks=_desc(lm, F16, (2, 3, 40, 4), 0x10002)), dict(vs=_desc(lm, F16, (2, 3, 40, 4), 0x10002)),
        dict(ks=_desc(lm, F16, (2, 3, 40, 4), stride={2: 5})), dict(vs=_desc(lm, F16, (2, 3, 40, 8))),
        dict(k=_desc(lm, U8, (2, 3, 40, 128))), dict(k=_desc(lm, U8, (1, 3, 40, 64))),
        dict(k=_desc(lm, U8, (2, 3, 40, 64), 0x10004)), dict(v=_desc(lm, U8, (2, 3, 40, 64), stride={0: 9600})),
        dict(ko=_desc(lm, BF16, (2, 3, 4, 128), 0x10008)), dict(sp=_desc(lm, I32, (3,))),
        dict(bt=_desc(lm, I32, (2, 3)), page=16), dict(bt=_desc(lm, I32, (1, 3)), page=40),
        dict(bt=_desc(lm, I32, (2, 1)), page=40, start=37),
    ]
    for kw in bad:
        assert lib.sia_kv_read(*_read_args(lm, **kw), None) == lm.SIA_ERR_INVALID_ARGUMENT, kw
    for kw in (dict(ks=_desc(lm, F16, (2, 3, 40, 16))),                       # groups of 16 at head_dim 128
               dict(k=_desc(lm, I32, (2, 3, 40, 64))), dict(ko=_desc(lm, U8, (2, 3, 4, 128)))):
        assert lib.sia_kv_read(*_read_args(lm, **kw), None) == lm.SIA_ERR_UNSUPPORTED, kw
    empty = dict(ko=_desc(lm, BF16, (2, 3, 0, 128)), vo=_desc(lm, BF16, (2, 3, 0, 128)))
    assert lib.sia_kv_read(*_read_args(lm, **empty), None) == lm.SIA_OK       # no tokens: nothing to do


def test_write_refusals_come_before_the_device():
    lib, lm = load_pkg().load_library(), importlib.import_module(PKG_NAME + "._lib")
    U8, F16, BF16, F32 = lm.SIA_U8, lm.SIA_F16, lm.SIA_BF16, lm.SIA_F32

    def call(**kw):
        a = {"k": _desc(lm, BF16, (2, 3, 4, 128)), "v": _desc(lm, BF16, (2, 3, 4, 128)),
             "kd": _desc(lm, U8, (2, 3, 40, 64)), "vd": _desc(lm, U8, (2, 3, 40, 64)),
             "ks": _desc(lm, F16, (2, 3, 40, 4)), "vs": _desc(lm, F16, (2, 3, 40, 4)), "bt": None, "sp": None}
        a.update(kw)
        return lib.sia_kv_write(*[ctypes.byref(x) if x is not None else None for x in a.values()], 0, 0, None)

    if not torch.cuda.is_available():
        assert call() == lm.SIA_ERR_DEVICE
    for kw in (dict(ks=None), dict(vs=None), dict(ks=_desc(lm, F32, (2, 3, 40, 4))),
               dict(kd=_desc(lm, U8, (2, 3, 40, 128))), dict(kd=_desc(lm, U8, (2, 3, 40, 64), 0x10004)),
               dict(ks=_desc(lm, F16, (2, 3, 40, 3))), dict(vs=_desc(lm, F16, (2, 3, 40, 8))),
               dict(vs=_desc(lm, F16, (2, 3, 40, 4), 0x10002))):
        assert call(**kw) == lm.SIA_ERR_INVALID_ARGUMENT, kw


def test_python_refusals():
    pkg = load_pkg()
    kv = importlib.import_module(PKG_NAME + ".kv_cache")
    for g in (0, 16, 48, 256):
        with pytest.raises(ValueError):
            kv.int4_group(128, g)
    assert kv.int4_group(16, 64) == 16 and kv.int4_group(256, 128) == 128
    with pytest.raises(ValueError):
        pkg.KVCache(1, 1, 16, 1, 64, device="cpu", kv_dtype=torch.uint8)
    with pytest.raises(ValueError):
        pkg.PagedKVCache(1, 1, 16, 1, 64, device="cpu", kv_dtype=torch.uint8)
    with pytest.raises(ValueError):
        pkg.KVCache(1, 1, 16, 1, 64, device="cpu", kv_dtype="int4", group_size=48)
    c = pkg.KVCache(2, 3, 20, 4, 128, device="cpu", kv_dtype="int4", group_size=32)
    assert c.k_cache.shape == (2, 3, 4, 20, 64) and c.v_scale.shape == (2, 3, 4, 20, 8) and c.is_quantized
    p = pkg.PagedKVCache(2, 3, 40, 4, 16, device="cpu", kv_dtype="int4")
    assert p.k_pool.shape == (2, 9, 4, 16, 8) and p.k_scale_pool.shape == (2, 9, 4, 16, 2)


def test_reciprocal_of_every_step():
    """1 / s from a reciprocal within one ulp (v_rcp_f32) and one Newton step under FMAs is correctly rounded, and x / s
    from it (three more instructions) too, for every positive fp16 s: the write kernel's arithmetic."""
    f, d = np.float32, np.float64
    s = np.arange(1, 0x7C00, dtype=np.uint16).view(np.float16).astype(f)
    want = (d(1) / s.astype(d)).astype(f)
    for off in (-1, 0, 1):
        r = (want.view(np.int32) + off).view(f)
        # (an fp32 product of two fp32 numbers is exact in fp64, and so are the sums here up to one fp64 rounding, far
        # below the fp32 rounding that follows)
        e = (d(1) - s.astype(d) * r.astype(d)).astype(f)
        inv = (e.astype(d) * r.astype(d) + r.astype(d)).astype(f)
        np.testing.assert_array_equal(inv, want)
    rng = np.random.default_rng(0)
    for _ in range(20):
        x = (rng.standard_normal(s.size) * s * 8).astype(f)
        x[::3] = (s[::3] * (rng.integers(0, 16, x[::3].size) + 0.5)).astype(f)          # ties
        q0 = (x.astype(d) * want.astype(d)).astype(f)
        r = (x.astype(d) - q0.astype(d) * s.astype(d)).astype(f)
        q = (r.astype(d) * want.astype(d) + q0.astype(d)).astype(f)
        np.testing.assert_array_equal(q, (x.astype(d) / s.astype(d)).astype(f))
