"""Scored decode steps over more keys than 2^30."""

from __future__ import annotations

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


@pytest.mark.parametrize("D,page", [(64, 1 << 23), (16, 1 << 23)])
def test_more_keys_than_two_to_the_30(gpu_pkg, D, page):
    """Without a window every key is seen, however many: one page of ones among 128 of zeros."""
    n = (1 << 30) + page
    kp, vp = torch.zeros(2, 1, page, D, dtype=torch.int8, device=DEV), torch.zeros(2, 1, page, D, dtype=torch.int8, device=DEV)
    vp[1] = 64
    ks, vs = torch.ones(2, 1, page, device=DEV), torch.full((2, 1, page), 2.0, device=DEV)
    table = torch.zeros(1, n // page, dtype=torch.int32, device=DEV)
    table[0, 0] = 1
    q = rand(1, 1, 1, D)
    announce(f"{n} keys, D={D}")
    args = (q, kp, vp, table, i32(n), page, ks, vs)
    out = gpu_pkg.paged_scored_attention_flash_decode(*args, softcap=20.0)
    want = 128.0 / (n // page)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want).all()
    # a window that leaves half of the page of ones: what it leaves of it over all that it leaves
    W = n - page // 2
    out = gpu_pkg.paged_scored_attention_flash_decode(*args, window=W)
    want = 128.0 * (page - page // 2) / W
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want).all()
