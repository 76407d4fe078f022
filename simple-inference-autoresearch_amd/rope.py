"""Rotary position embedding with the reference's interface.

Drop-in for ``kernels/rope_kernel.py`` and ``ops/rope.py`` of the reference
engine:

* :func:`rope_triton` -- ``kernels/rope_kernel.py:261-285`` (and
  ``_check_cos_sin`` / ``_apply_qk``, 167-258): Q and K rotated in one HIP
  launch (``sia_rope_qk``), strided Q/K slices of a fused qkv buffer read
  without a copy, contiguous outputs.
* :func:`apply_rope` -- ``ops/rope.py:206-226``: the split-half rotation the
  attention module calls.
* :class:`RopeFrequencies` -- ``ops/rope.py:72-185``: the cos/sin tables
  (Llama 3 frequency scaling) and their per-dtype cast cache.

Without a counterpart in the reference:

* :func:`rope_scaled` -- a part of each head rotated, at any positions, with
  angles computed from frequencies in the kernel.
* :class:`ScaledRope` -- the frequencies of scaled contexts (linear, NTK, YaRN,
  Llama 3), applied by it or as tables for the functions that take tables.

The rotation is ``out_a = x_a cos - x_b sin``, ``out_b = x_b cos + x_a sin``
in fp32 with every product and sum rounded on its own (no fused
multiply-add), stored in the input dtype with round-to-nearest-even.  Row
``r`` of the flattened ``(B*T)`` rows takes position ``r % cos.shape[0]``,
as in the reference kernel.
"""

from __future__ import annotations

import math

import torch

from . import _lib


def _check_cos_sin(cos: torch.Tensor, sin: torch.Tensor, head_dim: int) -> int:
    """The reference's table checks (``kernels/rope_kernel.py:167-190``); returns the row stride."""
    half = head_dim // 2
    if cos.shape[-1] not in (head_dim, half):
        raise ValueError(f"cos/sin last dim must be head_dim ({head_dim}) or head_dim/2 ({half}); "
                         f"got {cos.shape[-1]}")
    if cos.shape != sin.shape:
        raise ValueError(f"cos and sin must have identical shape; got {cos.shape} vs {sin.shape}")
    if cos.stride(-1) != 1 or sin.stride(-1) != 1:
        raise ValueError("cos/sin must be unit-stride along the last dim")
    if cos.stride(0) != sin.stride(0):
        raise ValueError("cos and sin must share the same row stride")
    if cos.dim() != 2:
        raise ValueError(f"cos/sin must be (seq_len, width) tables; got {cos.dim()} dims")
    return cos.stride(0)


def rope_triton(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotate ``q (B, T, Hq, D)`` and ``k (B, T, Hkv, D)`` by the ``cos``/``sin`` tables.

    ``cos``/``sin``: ``(T', D)`` duplicated or ``(T', D/2)`` raw; only the
    first ``D/2`` columns are read.  ``interleaved=False`` pairs ``(i, i+D/2)``
    (Llama/NeoX), ``True`` pairs ``(2i, 2i+1)`` (GPT-J).  Returns contiguous
    ``(q_rot, k_rot)`` with the inputs' shapes and dtypes.
    """
    B, T, n_heads_q, head_dim = q.shape
    _check_cos_sin(cos, sin, head_dim)
    if head_dim % 2:
        raise AssertionError("head_dim must be even for RoPE")
    ks = k.shape
    if ks[0] != B or ks[1] != T or ks[3] != head_dim:
        raise AssertionError(f"k {tuple(ks)} does not match q {tuple(q.shape)} in B, T or head_dim")
    # views whose B*T rows are not one stride apart (head_dim unit-stride,
    # heads head_dim apart, stride(0) == T*stride(1) unless T == 1 or B == 1)
    # are copied by the extension op, which also allocates the outputs
    return _lib.gpu_ops().rope_qk(q, k, cos, sin, bool(interleaved))


def apply_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
    """``ops/rope.py:206``: split-half RoPE of ``q``/``k`` with ``(T, head_dim)`` tables."""
    return rope_triton(q, k, cos, sin)


class RopeFrequencies:
    """cos/sin tables for positions ``[0, max_seq_len)`` (``ops/rope.py:72-185``).

    Frequencies ``1 / theta^(2i/D)`` in fp32; with ``rope_type="llama3"`` each
    is rescaled by wavelength (kept below ``original_max_seq_len /
    high_freq_factor``, divided by ``factor`` above ``original_max_seq_len /
    low_freq_factor``, linearly blended between), the blend evaluated in
    double precision as the reference does, then stored as fp32.  Tables are
    fp32 ``(max_seq_len, head_dim)`` with each angle duplicated across the
    two halves.
    """

    def __init__(self, head_dim: int, max_seq_len: int, rope_theta: float = 500_000.0, rope_type: str = "llama3",
                 factor: float = 32.0, low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                 original_max_seq_len: int = 8192, device: torch.device | None = None):
        self.head_dim = head_dim
        self.max_seq_len = max_seq_len
        device = device or torch.device("cuda" if torch.cuda.is_available() else "cpu")
        exponent = torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim
        freqs = 1.0 / (rope_theta ** exponent)
        if rope_type == "llama3":
            freqs = self._llama3_scaled(freqs, factor, low_freq_factor, high_freq_factor, original_max_seq_len)
        angle = torch.outer(torch.arange(max_seq_len, dtype=torch.float32, device=device), freqs)
        angle = torch.cat([angle, angle], dim=-1)
        self.cos = angle.cos()
        self.sin = angle.sin()
        self._cast_cache: dict[torch.dtype, tuple[torch.Tensor, torch.Tensor]] = {}

    @staticmethod
    def _llama3_scaled(freqs: torch.Tensor, factor: float, low_freq_factor: float, high_freq_factor: float,
                       original_max_seq_len: int) -> torch.Tensor:
        f = freqs.double()
        wavelen = (2 * math.pi) / f
        smooth = (original_max_seq_len / wavelen - low_freq_factor) / (high_freq_factor - low_freq_factor)
        blended = (1 - smooth) * f / factor + smooth * f
        out = torch.where(wavelen > original_max_seq_len / low_freq_factor, f / factor, blended)
        out = torch.where(wavelen < original_max_seq_len / high_freq_factor, f, out)
        return out.to(freqs.dtype)

    def get(self, seq_len: int, start_pos: int = 0, dtype: torch.dtype | None = None):
        """``(cos, sin)`` rows ``[start_pos, start_pos + seq_len)``, cast to ``dtype`` from a cached full table."""
        if dtype is None or dtype == torch.float32:
            cos_tbl, sin_tbl = self.cos, self.sin
        else:
            cached = self._cast_cache.get(dtype)
            if cached is None:
                cached = (self.cos.to(dtype), self.sin.to(dtype))
                self._cast_cache[dtype] = cached
            cos_tbl, sin_tbl = cached
        return cos_tbl[start_pos:start_pos + seq_len], sin_tbl[start_pos:start_pos + seq_len]


def rope_scaled(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
                rotary_dim: int | None = None, interleaved: bool = False, scale: float = 1.0):
    """Rotate the first ``rotary_dim`` elements of every head of ``q (B, T, Hq, D)`` and ``k (B, T, Hkv, D)``.

    ``positions``: int32 or int64 ``(T,)`` or ``(B, T)``; ``inv_freq``: float32
    or float64 ``(rotary_dim / 2,)``, the angle per position of each pair, which
    is ``(i, i + rotary_dim / 2)`` or, ``interleaved``, ``(2i, 2i + 1)``.  The
    rotated part is multiplied by ``scale``, the rest copied.  There is no table
    and no last position: an angle is off by ``|position| 2^-64`` of a turn at
    most (2^-24 at 2^40), its sine and cosine by 2^-23.  Strided views are read
    in place; returns contiguous ``(q_rot, k_rot)``, ``k_rot`` None where ``k`` is.
    """
    if rotary_dim is None:
        rotary_dim = q.shape[-1]
    return _lib.gpu_ops().rope_scaled(q, k, positions, inv_freq, rotary_dim, bool(interleaved), float(scale))


class ScaledRope:
    """Rotary frequencies of a context scaled beyond the one a model was trained on, and their application.

    ``rotary_dim`` elements of each head of ``head_dim`` are rotated (default:
    all).  ``rope_type``:

    * ``"default"``: ``f_i = theta^(-2i/R)``;
    * ``"linear"``: ``f_i / factor``;
    * ``"ntk"``: ``theta`` times ``factor^(R / (R - 2))``;
    * ``"yarn"``: ``f_i`` for pairs that turn more than ``beta_fast`` times in
      ``original_max_seq_len`` positions, ``f_i / factor`` below ``beta_slow``
      turns, a linear blend over the pairs between (its ends are
      rounded outwards, to at least 0 and at most ``R - 1``, past the last
      pair); rotated elements are multiplied by ``attention_factor`` (default
      ``0.1 ln(factor) + 1``);
    * ``"llama3"``: :class:`RopeFrequencies`' rule.

    ``inv_freq`` is kept in float64 on ``device``.  Call the object with ``q``,
    ``k`` and positions to rotate them (:func:`rope_scaled`), or take
    :meth:`tables` for the fused calls that read tables of whole heads.
    """

    def __init__(self, head_dim: int, rotary_dim: int | None = None, rope_theta: float = 10_000.0,
                 rope_type: str = "default", factor: float = 1.0, original_max_seq_len: int = 8192,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, low_freq_factor: float = 1.0,
                 high_freq_factor: float = 4.0, attention_factor: float | None = None, interleaved: bool = False,
                 device: torch.device | str | None = None):
        R = head_dim if rotary_dim is None else rotary_dim
        if R < 2 or R % 2 or R > head_dim:
            raise ValueError(f"rotary_dim {R} must be even, at least 2 and at most head_dim {head_dim}")
        if not factor > 0:
            raise ValueError("factor must be positive")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, R, interleaved
        i = torch.arange(R // 2, dtype=torch.float64)
        theta = float(rope_theta)
        if rope_type == "ntk":
            if R == 2:
                raise ValueError('rope_type "ntk" needs a rotary_dim above 2')
            theta *= factor ** (R / (R - 2))
        freq = theta ** (-2.0 * i / R)
        self.scale = 1.0
        if rope_type == "linear":
            freq = freq / factor
        elif rope_type == "yarn":
            low, high = (R * math.log(original_max_seq_len / (turns * 2 * math.pi)) / (2 * math.log(theta))
                         for turns in (beta_fast, beta_slow))
            low, high = max(math.floor(low), 0), min(math.ceil(high), R - 1)   # (past the last pair: it is blended too)
            ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
            freq = freq / factor * ramp + freq * (1 - ramp)
            self.scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        elif rope_type == "llama3":
            freq = RopeFrequencies._llama3_scaled(freq, factor, low_freq_factor, high_freq_factor, original_max_seq_len)
        elif rope_type not in ("default", "ntk"):
            raise ValueError(f"unknown rope_type {rope_type!r}")
        if attention_factor is not None:
            self.scale = float(attention_factor)
        device = torch.device(device) if device is not None else torch.device("cuda" if torch.cuda.is_available() else "cpu")
        self.inv_freq = freq.to(device)

    def __call__(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor):
        """``q (B, T, Hq, D)``, ``k (B, T, Hkv, D)`` rotated at ``positions (T,)`` or ``(B, T)``."""
        return rope_scaled(q, k, positions, self.inv_freq, self.rotary_dim, self.interleaved, self.scale)

    def tables(self, max_seq_len: int, dtype: torch.dtype = torch.float32):
        """``(cos, sin)``, each ``(max_seq_len, head_dim)``, for the functions that rotate whole heads from tables.

        Angles in float64, each entry rounded once; the factor of the rotated elements is in the entries.
        """
        if self.rotary_dim != self.head_dim:
            raise ValueError("tables cover whole heads; a part of the head is rotated by calling the object")
        angle = torch.arange(max_seq_len, dtype=torch.float64, device=self.inv_freq.device)[:, None] * self.inv_freq
        angle = torch.cat([angle, angle], dim=-1)
        return (self.scale * angle.cos()).to(dtype), (self.scale * angle.sin()).to(dtype)
