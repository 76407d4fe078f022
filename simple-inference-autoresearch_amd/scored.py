"""Attention with a score function: capped scores, a bias by distance, and masks that leave each query one run of keys.

No counterpart in the reference, whose attention has the scale and the causal mask alone.  A query at position ``p`` of its
sequence ``b`` sees key ``j``, in query head ``h``, with the score

    x = sm_scale q . k;   x = softcap tanh(x / softcap);   x -= alibi_slopes[h] |p - j|

where ``kv_start[b] <= j < kv_len[b]``, ``|p - j| < window``, ``p`` and ``j`` lie in the same document (no entry ``c`` of
``cu_seqlens`` with ``min(p, j) < c <= max(p, j)``) and, in a causal call, ``j <= p`` or ``j < prefix_len[b]``.  A query
that sees no key gives zeros, and what stands in keys that it does not see, a NaN too, does not reach it.

* :func:`scored_attention_flash` -- prompts and chunks of prompts, next to
  :func:`~.prefill.attention_flash_triton`.
* :func:`scored_attention_flash_decode`, :func:`paged_scored_attention_flash_decode` -- decode steps over every cache
  format, next to :func:`~.decode.attention_flash_decode` and its kin.

The steps of ``attention.py``, :meth:`~.paged_kv_cache.PagedKVCache.decode_attention` and the transformers hook take the
same options and run these functions where one is given.  An option left ``None`` shapes and hides nothing.
"""

from __future__ import annotations

import torch

from . import _lib
from .decode import _HEAD_DIMS, _common, _kv_len_tensor, _options
from . import decode as _decode

_DECODE_DIMS = (64, 128, 256)   # head dims of the matrix decode kernels (single-query calls)
_DECODE_BATCH = 16384           # most sequences of a decode call
_CAP_RANGE = (1e-37, 1e37)      # with room for its products in float32


def _score(softcap, window):
    """(softcap, window) as the extension takes them, 0 for none."""
    if softcap is None:
        softcap = 0.0
    elif not _CAP_RANGE[0] <= softcap <= _CAP_RANGE[1]:
        raise ValueError("softcap must be a positive finite number (1e-37 to 1e37)")
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError("window must be at least 1")
    return float(softcap), int(window)


def _in_place(t: torch.Tensor) -> bool:
    """Whether the decode kernels read a view as it is: head_dim contiguous, rows aligned to 16 bytes, tokens within 2 GiB."""
    es = t.element_size()
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * es % 16 == 0 for s in t.stride()[:-1])
            and t.stride(-2) * es < 1 << 31)


def _per_sequence(t: torch.Tensor, q: torch.Tensor) -> bool:
    """Whether the prompts' kernels take ``t`` as an option with an entry for all sequences or for each."""
    return (t.dtype == torch.int32 and t.device == q.device and t.dim() <= 1
            and (t.numel() == 1 or (t.numel() == q.shape[0] and t.stride(0) == 1)))


def _is_step(q, k, v, causal, cu_seqlens, prefix_len, kv_len) -> bool:
    """Whether a prompt call is a decode step that :func:`scored_attention_flash_decode` takes: one query row at the end
    of the keys (a causal row there sees every key, prefix or not).  What that refuses goes to the prompts' kernels."""
    B, _, Tq, D = q.shape
    return (Tq == 1 and k.shape[2] >= 1 and D in _DECODE_DIMS and B <= _DECODE_BATCH and k.shape[0] == B
            and cu_seqlens is None and kv_len is None and q.is_cuda and k.dtype == q.dtype and v.dtype == q.dtype
            and (prefix_len is None or (causal and _per_sequence(prefix_len, q)))
            and all(_in_place(t) for t in (q, k, v)))


def is_scored(softcap=None, alibi_slopes=None, window=None, kv_start=None) -> bool:
    """Whether one of a decode call's options is given."""
    return softcap is not None or alibi_slopes is not None or window is not None or kv_start is not None


def scored_attention_flash(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
                           sm_scale: float | None = None, *, softcap: float | None = None,
                           alibi_slopes: torch.Tensor | None = None, window: int | None = None,
                           cu_seqlens: torch.Tensor | None = None, prefix_len: torch.Tensor | None = None,
                           kv_start: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
                           out_token_major: bool = False) -> torch.Tensor:
    """Attention of ``q (B, Hq, Tq, D)`` over ``k, v (B, Hkv, Tk, D)`` with a score function (see the module).

    Query ``i`` sits at position ``Tk - Tq + i``.  Returns ``(B, Hq, Tq, D)``,
    or ``(B, Tq, Hq, D)`` when ``out_token_major``, in q's dtype.

    softcap: the scores' bound, a positive number.
    alibi_slopes: ``(Hq,)`` float32.
    window: keys a query sees on either side, itself among them.
    cu_seqlens: int32 ``(n,)`` or ``(B, n)``, positions at which documents start (others among them are harmless).
    prefix_len: int32, keys that every causal query sees, ``(1,)``/``()`` shared or ``(B,)``.
    kv_start, kv_len: int32 likewise, the keys of a padded row: ``[kv_start, kv_len)``.

    Tensors of options are on q's device and read there, so a call can be
    captured in a graph.  float16, bfloat16 and float32; strided views as
    :func:`~.prefill.attention_flash_triton` takes them.
    """
    B, Hq, Tq, D = q.shape
    if not (k.shape[-1] == D and v.shape[-1] == D):
        raise AssertionError()
    if D not in _HEAD_DIMS:
        raise AssertionError(f"unsupported head_dim {D}")
    if sm_scale is None:
        sm_scale = 1.0 / (D ** 0.5)
    cap, win = _score(softcap, window)
    ops = _lib.gpu_ops()
    if _is_step(q, k, v, causal, cu_seqlens, prefix_len, kv_len):
        n = torch.full((1,), k.shape[2], dtype=torch.int32, device=q.device)
        out = scored_attention_flash_decode(q, k, v, n, sm_scale=sm_scale, softcap=softcap, alibi_slopes=alibi_slopes,
                                            window=window, kv_start=kv_start)
        return out if out_token_major else out.view(B, Hq, 1, D)
    return ops.prefill_scored(q, k, v, bool(causal), float(sm_scale), cap, alibi_slopes, win, cu_seqlens, prefix_len,
                              kv_start, kv_len, bool(out_token_major))


def scored_attention_flash_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_len,
                                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                                  sm_scale: float | None = None, *, softcap: float | None = None,
                                  alibi_slopes: torch.Tensor | None = None, window: int | None = None,
                                  kv_start: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention with a score function over a contiguous cache; the query sits at position ``kv_len - 1``.

    q (B, Hq, 1, D); k, v (B, Hkv, S, D) in 16 bits or float32, or int8 with
    scales (B, Hkv, S), or uint8 codes (B, Hkv, S, D/2) with int4 parameters, as
    :func:`~.decode.attention_flash_decode` and its int8 and int4 forms take
    them; ``kv_len`` and ``kv_start`` int32, ``(1,)``/``()`` shared or ``(B,)``.
    Returns (B, 1, Hq, D) in q's dtype.
    """
    scale = _common(q, k, sm_scale)
    cap, win = _score(softcap, window)
    kl = _kv_len_tensor(kv_len, q.device)
    tps, b, e = _options() if _decode._opts_users else (0, 0, 0)
    return _lib.gpu_ops().decode_scored(q, k, v, k_scale, v_scale, None, kl, 0, scale, cap, alibi_slopes, win, kv_start,
                                        tps, b, e)


def paged_scored_attention_flash_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                                        block_table: torch.Tensor, kv_len, page_size: int,
                                        k_scale_pool: torch.Tensor | None = None,
                                        v_scale_pool: torch.Tensor | None = None, sm_scale: float | None = None, *,
                                        softcap: float | None = None, alibi_slopes: torch.Tensor | None = None,
                                        window: int | None = None,
                                        kv_start: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`scored_attention_flash_decode` over paged pools ``(num_blocks, Hkv, page_size, D)`` of any format.

    ``block_table`` (B, max_blocks) int32; table entries of pages that lie wholly
    in front of a sequence's window or first key are not used.
    """
    P = k_pool.shape[2]
    if P != page_size:
        raise AssertionError(f"k_pool page dim {P} != page_size {page_size}")
    scale = _common(q, k_pool, sm_scale)
    cap, win = _score(softcap, window)
    kl = _kv_len_tensor(kv_len, q.device)
    tps, b, e = _options() if _decode._opts_users else (0, 0, 0)
    return _lib.gpu_ops().decode_scored(q, k_pool, v_pool, k_scale_pool, v_scale_pool, block_table, kl, page_size, scale,
                                        cap, alibi_slopes, win, kv_start, tps, b, e)


def _scored_layer(q, k, v, k_scale, v_scale, layer, block_table, kv_len, page_size, sm_scale, softcap, alibi_slopes,
                  window, kv_start) -> torch.Tensor:
    """A decode call over layer ``layer`` of a cache's whole ``(L, ...)`` pools."""
    cap, win = _score(softcap, window)
    tps, b, e = _options() if _decode._opts_users else (0, 0, 0)
    return _lib.gpu_ops().decode_layer_scored(q, k, v, k_scale, v_scale, layer, block_table, kv_len, page_size, sm_scale,
                                              cap, alibi_slopes, win, kv_start, tps, b, e)
