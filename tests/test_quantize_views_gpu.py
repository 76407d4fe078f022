"""Quantising K/V views whose rows do not start on 16 bytes."""

from __future__ import annotations

import pytest
import torch

from helpers import announce
from test_int4_gpu import BF16, DEV, FP16, FP32, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(128,), (5, 64), (2, 3, 1, 256)])
def test_contiguous_views_that_start_anywhere(gpu_pkg, dtype, shape):
    announce(f"quantize views {dtype} {shape}")
    n = torch.Size(shape).numel()
    base = randn(gen(n), n + 8, dtype=dtype)
    for first in (0, 1, 3, 7):
        x = base[first:first + n].view(shape)
        assert x.is_contiguous()
        own = x.clone()
        for f in (lambda t: gpu_pkg.quantize_kv_int4(t, 32), gpu_pkg.quantize_kv_int8):
            for a, b in zip(f(x), f(own)):
                assert a.shape == b.shape and torch.equal(a, b), first
