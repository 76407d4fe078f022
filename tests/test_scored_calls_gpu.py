"""Scored prompt calls of one query, which run as decode steps where those take them.

Tolerances as in test_scored_gpu.py.
"""

from __future__ import annotations

import pytest
import torch

from helpers import announce, assert_close
from oracle import scored as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


def tol(v):
    return 2.0 ** -10 * float(v.float().abs().max())


@pytest.mark.parametrize("B", [16384, 16385, 20000])
def test_single_queries_of_large_batches(gpu_pkg, B):
    """More sequences than a decode call takes are a prompt call like any other."""
    q, k, v = rand(B, 2, 1, 64), rand(B, 1, 5, 64), rand(B, 1, 5, 64)
    start = torch.arange(B, device=DEV, dtype=torch.int32) % 6
    announce(f"{B} single queries")
    out = gpu_pkg.scored_attention_flash(q, k, v, softcap=20.0, kv_start=start)
    some = [0, 1, 5, 6, 11, B // 2, B - 2, B - 1]
    ref = S.scored_attention(*(t[some].double().cpu() for t in (q, k, v)), softcap=20.0, start=start[some].tolist())
    assert_close(out[some], ref.numpy(), tol(v), f"{B} single queries")
    assert (out[start == 5] == 0).all()


def test_single_queries_are_checked_as_any_others(gpu_pkg):
    f = gpu_pkg.scored_attention_flash
    for Tq in (1, 2):
        q, k, v = rand(2, 4, Tq, 64), rand(2, 2, 30, 64), rand(2, 2, 30, 64)
        for args, kw in (((q, rand(3, 2, 30, 64), rand(3, 2, 30, 64)), {}), ((q, k, rand(3, 2, 30, 64)), {}),
                         ((q, k, v), dict(prefix_len=i32(1, 2, 3))), ((q, k, v), dict(prefix_len=i32(1).long())),
                         ((q, k, v), dict(prefix_len=torch.tensor([1], dtype=torch.int32)))):
            announce(f"Tq={Tq} refused {list(kw)}")
            with pytest.raises(ValueError):
                f(*args, softcap=20.0, **kw)
    q, k, v = rand(2, 4, 1, 64), rand(2, 2, 30, 64), rand(2, 2, 30, 64)
    assert torch.equal(f(q, k, v, softcap=20.0, prefix_len=i32(3, 40)), f(q, k, v, softcap=20.0))


def test_keys_far_apart(gpu_pkg):
    """A token stride that a decode call refuses: the view is copied, whether for one query or for two."""
    # 2 tokens 2^31 bytes apart of a buffer that only they touch
    base = torch.empty(2, 1 << 30, dtype=torch.bfloat16, device=DEV)
    k = base.as_strided((1, 1, 2, 64), (1 << 31, 1 << 31, 1 << 30, 1))
    k.copy_(rand(1, 1, 2, 64))
    v = rand(1, 1, 2, 64)
    announce("tokens 2 GiB apart")
    for Tq in (1, 2):
        q = rand(1, 2, Tq, 64)
        ref = S.scored_attention(*(t.double().cpu() for t in (q, k.contiguous(), v)), softcap=20.0)
        assert_close(gpu_pkg.scored_attention_flash(q, k, v, softcap=20.0), ref.numpy(), tol(v), f"Tq={Tq}")
