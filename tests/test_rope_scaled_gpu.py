"""Rotary positions from frequencies against the float64 definition (``oracle/scored.py``).

Tolerance: sine and cosine off by 2^-23 and, as fp32 products with the factor, by half a step more; two products and a sum
in fp32 of elements up to m: 2^-21 m scale, before the output's own rounding.  Float64 angles of the reference are off by
2^-52 of the number of radians, below that for positions up to 2^28.
"""

from __future__ import annotations

import pytest
import torch

from helpers import announce, assert_close
from oracle import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def freqs(R, theta=10000.0):
    return theta ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)


def check(got, x, pos, freq, R, interleaved, scale, what):
    ref = S.rope(x.double().cpu(), pos.cpu().expand(x.shape[0], -1), freq.cpu(), R, interleaved, scale)
    assert_close(got, ref.numpy(), 2.0 ** -21 * float(x.float().abs().max()) * max(1.0, scale), what)
    assert torch.equal(got[..., R:], x[..., R:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (128, 24), (64, 16), (256, 64), (80, 20), (64, 2), (66, 6), (128, 126)])
def test_parts_of_the_head(gpu_pkg, dtype, interleaved, D, R):
    B, T, Hq, H = 2, 37, 6, 2
    qkv = torch.randn(B, T, Hq + 2 * H, D, device=DEV).to(dtype)
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + H]
    pos = torch.randint(0, 5000, (B, T), dtype=torch.int32, device=DEV)
    announce(f"rope {dtype} D={D} R={R} interleaved={interleaved}")
    before = qkv.clone()
    qo, ko = gpu_pkg.rope_scaled(q, k, pos, freqs(R).to(DEV), rotary_dim=R, interleaved=interleaved, scale=1.25)
    assert qo.is_contiguous() and ko.is_contiguous() and torch.equal(qkv, before)
    check(qo, q, pos, freqs(R), R, interleaved, 1.25, "q")
    check(ko, k, pos, freqs(R), R, interleaved, 1.25, "k")


@pytest.mark.parametrize("first", [0, 1, 10 ** 6, 2 ** 28, -70000])
def test_far_positions(gpu_pkg, first):
    q = torch.randn(1, 300, 2, 128, device=DEV)
    announce(f"positions from {first}")
    for dt in (torch.int32, torch.int64):
        pos = torch.arange(300, dtype=dt, device=DEV) + first
        for f in (freqs(128), freqs(128).float()):
            qo, ko = gpu_pkg.rope_scaled(q, None, pos, f.to(DEV))
            assert ko is None
            check(qo, q, pos, f, 128, False, 1.0, f"positions from {first}")


def test_positions_of_64_bits(gpu_pkg):
    """Exact modulo a turn: at frequencies of whole 2^-20 turns, positions 2^20 apart turn alike."""
    f = (2 * torch.pi) * torch.arange(1, 33, dtype=torch.float64, device=DEV) * 2.0 ** -20
    q = torch.randn(1, 64, 3, 64, device=DEV)
    pos = torch.arange(64, device=DEV)
    announce("64-bit positions")
    near, _ = gpu_pkg.rope_scaled(q, None, pos, f)
    far, _ = gpu_pkg.rope_scaled(q, None, pos + (1 << 31), f)
    torch.testing.assert_close(far, near, rtol=0, atol=2e-6 * float(q.abs().max()))   # 2^31 F is off by 2^31 2^-52 f / 2 pi turns


@pytest.mark.parametrize("B,T", [(1, 1), (64, 1), (3, 2), (1, 5000), (7, 129)])
def test_shapes(gpu_pkg, B, T):
    q, k = torch.randn(B, T, 32, 128, device=DEV).bfloat16(), torch.randn(B, T, 8, 128, device=DEV).bfloat16()
    pos = torch.arange(T, device=DEV).expand(B, T) + 11 * torch.arange(B, device=DEV)[:, None]
    announce(f"rope B={B} T={T}")
    qo, ko = gpu_pkg.rope_scaled(q, k, pos, freqs(128).to(DEV))
    check(qo, q, pos, freqs(128), 128, False, 1.0, "q")
    check(ko, k, pos, freqs(128), 128, False, 1.0, "k")


def test_views_streams_and_empty(gpu_pkg):
    f = freqs(64).to(DEV)
    x = torch.randn(2, 9, 40, 4, 64, device=DEV).half()      # (B, ?, T, H, D): rows far apart
    q, k = x[:, 3], x[:, 5, :, 1:2]
    pos = torch.arange(80, dtype=torch.int32, device=DEV)[::2]
    announce("rope of views")
    qo, ko = gpu_pkg.rope_scaled(q, k, pos, f)
    a, b = gpu_pkg.rope_scaled(q.contiguous(), k.contiguous(), pos.contiguous(), f)
    assert torch.equal(qo, a) and torch.equal(ko, b)
    qt = q.transpose(2, 3).contiguous().transpose(2, 3)       # head_dim not contiguous
    odd = torch.randn(2, 40, 4, 67, device=DEV).half()[..., 1:65]
    assert torch.equal(gpu_pkg.rope_scaled(qt, odd, pos, f)[0], a)
    assert torch.equal(gpu_pkg.rope_scaled(q, odd, pos, f)[1], gpu_pkg.rope_scaled(q, odd.contiguous(), pos, f)[1])
    for e in (q[:0], q[:, :0], q[:, :, :0]):
        p = pos[:e.shape[1]]
        got, _ = gpu_pkg.rope_scaled(e, None, p, f)
        assert got.shape == e.shape
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s, _ = gpu_pkg.rope_scaled(q, None, pos, f)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(s, a)


def test_captured_step(gpu_pkg):
    q, k = torch.randn(4, 1, 8, 128, device=DEV).bfloat16(), torch.randn(4, 1, 2, 128, device=DEV).bfloat16()
    pos, f = torch.zeros(4, 1, dtype=torch.int64, device=DEV), freqs(64).to(DEV)
    announce("captured rope")
    gpu_pkg.rope_scaled(q, k, pos, f, rotary_dim=64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = gpu_pkg.rope_scaled(q, k, pos, f, rotary_dim=64)
    for i in range(3):
        pos.add_(torch.arange(4, device=DEV)[:, None] + 100 * i)
        graph.replay()
        torch.cuda.synchronize()
        a, b = gpu_pkg.rope_scaled(q, k, pos, f, rotary_dim=64)
        assert torch.equal(qo, a) and torch.equal(ko, b)


@pytest.mark.parametrize("kind", ["default", "linear", "ntk", "yarn", "llama3"])
def test_scaled_contexts(gpu_pkg, kind):
    """ScaledRope applied equals rope_triton with its tables; a llama3 one has RopeFrequencies' frequencies."""
    r = gpu_pkg.ScaledRope(128, rope_theta=500000.0, rope_type=kind, factor=8.0, original_max_seq_len=2048, device=DEV)
    q, k = torch.randn(1, 700, 4, 128, device=DEV), torch.randn(1, 700, 2, 128, device=DEV)
    announce(f"ScaledRope {kind}")
    qo, ko = r(q, k, torch.arange(700, device=DEV))
    qt, kt = gpu_pkg.rope_triton(q, k, *r.tables(700))
    atol = 2.0 ** -20 * 6 * r.scale           # both within 2^-21 of the largest element
    torch.testing.assert_close(qo, qt, rtol=0, atol=atol)
    torch.testing.assert_close(ko, kt, rtol=0, atol=atol)
    if kind == "llama3":
        old = gpu_pkg.RopeFrequencies(128, 64, 500000.0, "llama3", 8.0, original_max_seq_len=2048, device=torch.device(DEV))
        torch.testing.assert_close(r.tables(64)[0], old.cos, rtol=0, atol=64 * 2.0 ** -21)
    if kind == "yarn":
        base = gpu_pkg.ScaledRope(128, rope_theta=500000.0, device=DEV).inv_freq
        assert r.scale > 1 and torch.equal(r.inv_freq[:8], base[:8]) and torch.allclose(r.inv_freq[-4:], base[-4:] / 8)


def test_frequencies_of_any_value(gpu_pkg):
    """Negative ones turn backwards, ones next to zero not at all, and one without a value reaches its own pair alone."""
    q, pos = torch.randn(1, 9, 2, 64, device=DEV), torch.arange(9, device=DEV) * 1000
    announce("negative, vanishing and missing frequencies")
    for f in (-freqs(64), torch.full((32,), -1e-20, dtype=torch.float64), torch.zeros(32, dtype=torch.float64)):
        out, _ = gpu_pkg.rope_scaled(q, None, pos, f.to(DEV))
        check(out, q, pos, f, 64, False, 1.0, "negative frequencies")
    want, _ = gpu_pkg.rope_scaled(q, None, pos, freqs(64).to(DEV))
    for bad in (float("nan"), float("inf")):
        f = freqs(64)
        f[5] = bad
        out, _ = gpu_pkg.rope_scaled(q, None, pos, f.to(DEV))
        assert torch.isnan(out[..., [5, 37]]).all()
        out[..., [5, 37]] = want[..., [5, 37]]
        assert torch.equal(out, want)


def test_refusals(gpu_pkg):
    q, k = torch.randn(2, 5, 4, 64, device=DEV), torch.randn(2, 5, 2, 64, device=DEV)
    pos, f = torch.arange(5, device=DEV), freqs(64).to(DEV)
    g = gpu_pkg.rope_scaled
    for args, kw in (((q, k, pos, f), dict(rotary_dim=32)), ((q, k, pos, f), dict(rotary_dim=66)), ((q, k, pos, f), dict(rotary_dim=0)),
                     ((q, k, pos, f), dict(rotary_dim=63)), ((q, k, pos[:4], f), {}), ((q, k, pos.float(), f), {}),
                     ((q, k, pos, f.half()), {}), ((q, k, pos, f[:-1]), {}), ((q, k[:1], pos, f), {}),
                     ((q, k.half(), pos, f), {}), ((q, k, pos.cpu(), f), {}), ((q, k, pos, f.cpu()), {}),
                     ((q[0], k, pos, f), {}), ((q, k, pos.expand(3, 5), f), {}), ((q.cpu(), k, pos, f), {})):
        announce(f"refused {kw}")
        with pytest.raises(ValueError):
            g(*args, **kw)
    with pytest.raises(NotImplementedError):
        g(torch.randn(1, 5, 1, 65, device=DEV), None, pos, f, rotary_dim=64)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=256), dict(rope_type="other"), dict(factor=0.0)):
        with pytest.raises(ValueError):
            gpu_pkg.ScaledRope(128, **bad)
