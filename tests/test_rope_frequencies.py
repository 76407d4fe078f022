"""ScaledRope's frequencies against restatements of their rules, pair by pair in Python floats (CPU).

Tolerance: a power, a product and a blend in float64, a few 2^-53 each: 1e-13.  transformers computes its frequencies in
float32: 4e-6 for a power of an exponent rounded at 2^-24 (ln theta 2^-24 <= 8e-7 for theta up to 5e5) and what follows.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

SETTINGS = [(128, 1e4, 4096), (128, 1e4, 8192), (128, 1e4, 65536), (128, 1e4, 131072), (32, 1e4, 40000), (8, 1e4, 8192),
            (64, 5e5, 8192), (2, 1e4, 2048), (128, 1e4, 100), (16, 100.0, 1 << 20)]


def base(R, theta):
    return [theta ** (-2.0 * i / R) for i in range(R // 2)]


def yarn(R, theta, L, factor, fast, slow):
    """The blend runs over whole pairs, from the one that turns ``fast`` times in L positions to the one of ``slow``."""
    first = max(math.floor(R / 2 * math.log(L / (2 * math.pi * fast), theta)), 0)
    last = min(math.ceil(R / 2 * math.log(L / (2 * math.pi * slow), theta)), R - 1)
    out = []
    for i, f in enumerate(base(R, theta)):
        share = 0.0 if i <= first else 1.0 if i >= last else (i - first) / (last - first)   # of the interpolated frequency
        out.append(f * (1.0 - share) + f / factor * share)
    return out


def close(got, want, tol=1e-13):
    got = [float(x) for x in got]
    assert len(got) == len(want)
    worst = max(abs(a - b) / b for a, b in zip(got, want))
    assert worst <= tol, worst


@pytest.mark.parametrize("R,theta,L", SETTINGS)
@pytest.mark.parametrize("factor,fast,slow", [(8.0, 32.0, 1.0), (4.0, 16.0, 2.0), (40.0, 32.0, 1.0)])
def test_yarn(pkg, R, theta, L, factor, fast, slow):
    r = pkg.ScaledRope(R, rope_theta=theta, rope_type="yarn", factor=factor, original_max_seq_len=L, beta_fast=fast,
                       beta_slow=slow, device="cpu")
    close(r.inv_freq, yarn(R, theta, L, factor, fast, slow))
    assert r.scale == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)


@pytest.mark.parametrize("R,theta,L", [(128, 1e4, 65536), (128, 1e4, 131072), (32, 1e4, 40000), (8, 1e4, 8192)])
def test_yarn_where_the_last_pair_still_turns(pkg, R, theta, L):
    """A pair that turns more than beta_slow times is blended, not interpolated in full, the last one too."""
    f = pkg.ScaledRope(R, rope_theta=theta, rope_type="yarn", factor=8.0, original_max_seq_len=L, device="cpu").inv_freq
    plain = base(R, theta)
    assert plain[-1] * L / (2 * math.pi) > 1.0
    assert float(f[-1]) > plain[-1] / 8 * (1 + 1e-9)


@pytest.mark.parametrize("R,theta,L", [s for s in SETTINGS if s[0] > 2])
@pytest.mark.parametrize("factor", [8.0, 40.0])
def test_yarn_of_transformers(pkg, R, theta, L, factor):
    utils = pytest.importorskip("transformers.modeling_rope_utils")
    params = {"rope_type": "yarn", "rope_theta": theta, "factor": factor, "original_max_position_embeddings": L}
    config = SimpleNamespace(rope_theta=theta, rope_scaling=params, rope_parameters=params, head_dim=R, hidden_size=4 * R,
                             num_attention_heads=4, max_position_embeddings=int(L * factor), partial_rotary_factor=1.0,
                             standardize_rope_params=lambda: None)
    try:
        want, scale = utils.ROPE_INIT_FUNCTIONS["yarn"](config, "cpu")
    except (AttributeError, KeyError, TypeError) as e:      # (another version's way of reading a config)
        pytest.skip(f"transformers takes another config: {e}")
    r = pkg.ScaledRope(R, rope_theta=theta, rope_type="yarn", factor=factor, original_max_seq_len=L, device="cpu")
    close(r.inv_freq, [float(x) for x in want.double()], 4e-6)
    assert r.scale == pytest.approx(scale, rel=1e-6)


@pytest.mark.parametrize("R,theta", [(128, 1e4), (64, 5e5), (4, 1e4)])
def test_linear_and_ntk(pkg, R, theta):
    make = lambda kind: pkg.ScaledRope(R, rope_theta=theta, rope_type=kind, factor=8.0, device="cpu").inv_freq
    close(make("default"), base(R, theta))
    close(make("linear"), [f / 8.0 for f in base(R, theta)])
    # ntk: a geometric row whose first frequency stays and whose last is divided by the factor
    n, last = R // 2, base(R, theta)[-1] / 8.0
    close(make("ntk"), [last ** (i / (n - 1)) for i in range(n)])
