"""Rotary positions in the forms that ``ops.rope`` (neox halves of the whole head, dense q and k; reference
``csrc/ffi/ops.cpp:13-108``) does not cover: interleaved pairs, a rotated part of the head, q and k inside a fused
projection, tables in fp32, and tables for stretched contexts built on the device."""
from __future__ import annotations

from typing import Optional, Union

import torch

import ascend910a_extras.ascend910a_extras_C as _C

Tensor = torch.Tensor

_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "dynamic": 3, "yarn": 4, "wavelength": 5, "pairs": 6}


def rotary_tables(
    max_position: int,
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: str = "none",
    factor: float = 1.0,
    original_max_position: float = 0,
    low_freq_factor: float = 1.0,
    high_freq_factor: float = 4.0,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    attention_factor: Optional[float] = None,
    pair_factors: Optional[Tensor] = None,
    dtype: torch.dtype = torch.float16,
    device: Union[torch.device, str, None] = None,
) -> tuple[Tensor, Tensor]:
    """``cos, sin``, each ``[max_position, rotary_dim/2]``, of the angles ``p * f_j`` with ``f_j = base**(-2j/rotary_dim)``,
    formed in 64 bits (positions far out are as exact as near ones) and rounded once to ``dtype`` (fp16 or fp32).
    ``ops.rope`` takes the fp16 tables of ``rotary_dim = head_dim``.

    ``scaling``: ``"linear"`` (``f_j / factor``), ``"ntk"`` (the base times ``factor**(R/(R-2))``), ``"dynamic"`` (the same,
    with the factor that ``max_position`` beyond ``original_max_position`` asks for), ``"yarn"`` (by parts, from
    ``beta_fast`` to ``beta_slow`` turns within ``original_max_position``; every entry times ``0.1 ln(factor) + 1``),
    ``"wavelength"`` (by wave length, between ``low_freq_factor`` and ``high_freq_factor`` turns), ``"pairs"``
    (``f_j / pair_factors[j]``, fp32 ``[rotary_dim/2]`` on the device; every entry times
    ``sqrt(1 + ln(factor) / ln(original_max_position))``).  ``attention_factor`` replaces the factor on the entries."""
    if scaling not in _SCALINGS:
        raise RuntimeError(f"rotary_tables: scaling must be one of {', '.join(_SCALINGS)}, got {scaling!r}")
    if dtype not in (torch.float16, torch.float32):
        raise RuntimeError(f"rotary_tables: dtype must be torch.float16 or torch.float32, got {dtype}")
    if attention_factor is not None and not attention_factor > 0:
        raise RuntimeError(f"rotary_tables: attention_factor must be positive, got {attention_factor}")
    if (pair_factors is not None) != (scaling == "pairs"):
        raise RuntimeError("rotary_tables: pair_factors belong to scaling='pairs', and it needs them")
    if device is None:
        device = pair_factors.device if pair_factors is not None else "cuda"
    low, high = (beta_fast, beta_slow) if scaling == "yarn" else (low_freq_factor, high_freq_factor)
    return _C.rotary_tables(max_position, rotary_dim, base, _SCALINGS[scaling], factor, original_max_position, low, high,
                            attention_factor or 0.0, pair_factors, dtype == torch.float32, torch.device(device))


def rotary_embedding(q: Tensor, k: Tensor, position_ids: Tensor, cos: Tensor, sin: Tensor,
                     interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """Rotates the first ``2 * cos.size(1)`` elements of every head of ``q [tokens, heads, D]`` and
    ``k [tokens, kv_heads, D]`` by the table rows ``position_ids`` (int32 ``[tokens]``; positions outside the tables take the
    nearest row) and copies the rest.  Element ``j`` is paired with ``j + R/2``, or ``2j`` with ``2j + 1`` where
    ``interleaved``.  ``q`` and ``k`` may be views into a fused projection (elements of a head next to each other, other
    strides and the start multiples of 8 elements).  ``cos``/``sin`` ``[max_position, R/2]`` are fp16 or fp32.  Returns new
    dense tensors ``(out_q, out_k)``."""
    return _C.rotary_embedding(q, k, position_ids, cos, sin, interleaved)
