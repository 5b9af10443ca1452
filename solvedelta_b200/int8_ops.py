"""Projections with 8-bit weights and activations for serving: rows of int8 with a scale for each token and each
output channel, the products exact in 32-bit integers (csrc/sd_int8.cuh).  No reverse pass, no fallback.

A row stands for ``q * scale`` with ``scale = max|x| / 127`` and ``q = 127 x / max|x|`` rounded to the nearest whole
number (ties to even); weights are quantised the same way, a scale for each output channel.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn

from . import _lib


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of the rows of ``x`` ``[..., K]`` (BF16 or FP32 CUDA): ``q`` int8 ``[..., K]``, its rows padded to
    whole groups of 16 bytes, ``scale`` FP32 ``[...]``.  A row of zeros has scale 0; a row with an infinity or a NaN has
    ``q = 0`` and scale NaN, so that everything computed from it is NaN."""
    return _lib.host().quantize_rows(x)


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, swiglu: bool = False,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``y[..., j] = scale[...] * weight_scale[j] * sum_k q[..., k] weight[j, k] + bias[j]``: ``q`` int8 ``[..., K]``
    with FP32 ``scale`` ``[...]``, ``weight`` int8 ``[N, K]`` with FP32 ``weight_scale`` ``[N]``, ``bias`` BF16 or FP32
    ``[N]``.  Sums are exact (``K`` up to 131072), the rest is FP32, rounded once to ``out_dtype`` (BF16 or FP32).  With
    ``swiglu`` the result is ``silu(y[..., :N/2]) * y[..., N/2:]``.  Rows as :func:`quantize_rows` makes them are read in
    place; others (an odd stride, an odd start) are copied first."""
    return _lib.host().int8_matmul(q, scale, weight, weight_scale, bias, swiglu, out_dtype)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                swiglu: bool = False, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`int8_matmul` of :func:`quantize_rows` of ``x`` ``[..., K]`` (BF16 or FP32): the projection of a layer whose
    weight is held in int8.  For the few rows of a cached token it is one launch."""
    return _lib.host().int8_linear(x, weight, weight_scale, bias, swiglu, out_dtype)


__all__ = ["int8_linear", "int8_matmul", "quantize_rows"]
