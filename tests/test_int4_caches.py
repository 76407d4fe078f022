"""What the Python layer of the 4-bit caches decides by itself, without a GPU."""

from __future__ import annotations

import pytest
import torch

from conftest import load_pkg


def test_read_needs_a_place_for_k():
    """A pair without k would be filled in part: nothing would reach the caller's v."""
    pkg = load_pkg()
    src = torch.zeros(1, 2, 8, 64)
    for out in ((None, torch.zeros(1, 2, 4, 64)), (None, None)):
        with pytest.raises(ValueError, match="pair"):
            pkg.kv_read(src, src, 4, out=out)


def test_footprint_counts_the_parameters():
    """Codes of half a byte and 4 bytes of parameters per group, for K and for V; the other caches as before."""
    pkg = load_pkg()
    elements = 2 * 3 * 4 * 5000 * 128
    for group, held in ((32, 0.5 + 4 / 32), (64, 0.5 + 4 / 64), (128, 0.5 + 4 / 128)):
        c = pkg.KVCache(2, 3, 5000, 4, 128, device="cpu", kv_dtype="int4", group_size=group)
        assert c.bytes() == 2 * elements * held and f"vram={2 * elements * held / 1e9:.2f} GB" in repr(c)
    assert pkg.KVCache(2, 3, 5000, 4, 128, device="cpu").bytes() == 2 * elements                     # int8
    assert pkg.KVCache(2, 3, 200, 4, 128, device="cpu").bytes() == 2 * elements // 25 * 2            # bf16
    p = pkg.PagedKVCache(2, 3, 80000, 4, 128, device="cpu", kv_dtype="int4", group_size=32)
    assert f"vram={2 * 16 * elements * 0.625 / 1e9:.2f} GB" in repr(p)
    p = pkg.PagedKVCache(2, 3, 5008, 4, 128, device="cpu", kv_dtype=torch.int8)
    assert f"vram={2 * 2 * 3 * 4 * 5008 * 128 / 1e9:.2f} GB" in repr(p)
