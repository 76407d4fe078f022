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
