"""The transformers hook where the caller passes the lengths of packed documents."""

from __future__ import annotations

import importlib
from types import SimpleNamespace

import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


def test_the_hook_with_one_document_a_row(gpu_pkg):
    """Lengths of one document in each row, as a decode step carries them on, change nothing."""
    plugins = importlib.import_module("simple-inference-autoresearch_amd.plugins")
    f, module = plugins.sia_attention_forward, SimpleNamespace(is_causal=True)
    for B, Tq, Tk in ((1, 1, 150), (1, 7, 150), (3, 1, 90), (2, 64, 64)):
        q, k, v = rand(B, 8, Tq, 64), rand(B, 2, Tk, 64), rand(B, 2, Tk, 64)
        of_q, of_k = (torch.arange(B + 1, dtype=torch.int32, device=DEV) * n for n in (Tq, Tk))
        announce(f"hook, one document in each of {B} rows, {Tq} over {Tk}")
        for kw in ({}, dict(sliding_window=33, softcap=10.0)):
            want, _ = f(module, q, k, v, None, scaling=0.125, **kw)
            for more in (dict(cu_seq_lens_q=of_q, cu_seq_lens_k=of_k), dict(cu_seq_lens_q=of_q.long(), cu_seq_lens_k=of_k.long())):
                got, _ = f(module, q, k, v, None, scaling=0.125, max_length_q=Tq, max_length_k=Tk, **more, **kw)
                assert torch.equal(got, want)
    q, k, v = rand(1, 8, 20, 64), rand(1, 2, 20, 64), rand(1, 2, 20, 64)
    for of_q, of_k in ((i32(0, 5, 20), i32(0, 20)), (i32(0, 20), i32(0, 5, 20)), (i32(0, 5, 20), None), (None, i32(0, 5, 20))):
        with pytest.raises(NotImplementedError):
            f(module, q, k, v, None, cu_seq_lens_q=of_q, cu_seq_lens_k=of_k)
