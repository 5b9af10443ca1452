"""Projections with 8-bit weights and activations for serving: rows of int8 with a scale for each token and each
output channel, the products exact in 32-bit integers (csrc/sd_int8.cuh).  No reverse pass, no forward-mode
derivative (both are refused), no fallback.

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
    ``q = 0`` and scale NaN, so that everything computed from it is NaN.  Neither output carries a gradient or a
    tangent."""
    return _lib.host().quantize_rows(x)


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, swiglu: bool = False,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``y[..., j] = scale[...] * weight_scale[j] * sum_k q[..., k] weight[j, k] + bias[j]``: ``q`` int8 ``[..., K]``
    with FP32 ``scale`` ``[...]``, ``weight`` int8 ``[N, K]`` with FP32 ``weight_scale`` ``[N]``, ``bias`` BF16 or FP32
    ``[N]``.  Sums are exact (``K`` up to 131072), the rest is FP32 (the sum times ``scale``, times ``weight_scale``,
    plus ``bias``: infinite where one of these leaves FP32), rounded once to ``out_dtype`` (BF16 or FP32).  With
    ``swiglu`` the result is ``silu(y[..., :N/2]) * y[..., N/2:]``.  Rows as :func:`quantize_rows` makes them are read in
    place; others (an odd stride, an odd start) are copied first."""
    return _lib.host().int8_matmul(q, scale, weight, weight_scale, bias, swiglu, out_dtype)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                swiglu: bool = False, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`int8_matmul` of :func:`quantize_rows` of ``x`` ``[..., K]`` (BF16 or FP32): the projection of a layer whose
    weight is held in int8.  For the few rows of a cached token it is one launch."""
    return _lib.host().int8_linear(x, weight, weight_scale, bias, swiglu, out_dtype)


def int8_gated_mlp(x: torch.Tensor, up: torch.Tensor, up_scale: torch.Tensor, up_bias: Optional[torch.Tensor],
                   down: torch.Tensor, down_scale: torch.Tensor, down_bias: Optional[torch.Tensor]) -> torch.Tensor:
    """``int8_linear(int8_linear(x, up, up_scale, up_bias, swiglu=True), down, down_scale, down_bias)`` in one native call,
    the 8-bit counterpart of :func:`mixer_ops.gated_mlp`: ``up`` holds gate rows and as many value rows; BF16 out."""
    return _lib.host().int8_gated_mlp(x, up, up_scale, up_bias, down, down_scale, down_bias)


class Int8Linear(nn.Module):
    """A projection for inference whose weight is held in int8 with a scale for each output channel (buffers ``weight``
    ``[out, in]``, ``weight_scale`` ``[out]`` and, where there is one, ``bias``); the rows it is given are quantised row by
    row on the way in, the result is BF16.  ``bias`` is BF16 or FP32 (``bias_dtype``).  Not trainable: with gradients
    recorded for its input it raises."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, device=None,
                 bias_dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        # rows start on 16-byte boundaries, as the kernels read them
        pitch = (in_features + 15) // 16 * 16
        weight = torch.zeros(out_features, pitch, dtype=torch.int8, device=device)[:, :in_features]
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", torch.zeros(out_features, dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=bias_dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        """The projection of a CUDA ``nn.Linear`` (BF16 or FP32), its weight quantised output channel by output channel, its
        bias as it is.  A module that does more than its product (a subclass, an adapter, a parametrisation, a hook) is
        refused: that part would be lost."""
        if (type(linear) is not nn.Linear or "forward" in linear.__dict__ or linear._forward_hooks
                or linear._forward_pre_hooks):
            raise TypeError("only a plain nn.Linear without hooks can be held in int8")
        weight = linear.weight.detach()
        made = cls(linear.in_features, linear.out_features, linear.bias is not None, weight.device,
                   torch.bfloat16 if linear.bias is None or linear.bias.dtype == torch.bfloat16 else torch.float32)
        q, scale = quantize_rows(weight)
        if not torch.isfinite(scale).all():
            raise ValueError("a weight with infinities or NaNs cannot be quantised")
        made.weight.copy_(q)
        made.weight_scale.copy_(scale)
        if linear.bias is not None:
            made.bias.copy_(linear.bias.detach())
        return made.train(linear.training)

    def _apply(self, fn, recurse: bool = True):
        # a change of the module's floating type (model.bfloat16(), model.half()) is not one of the scales
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        if self.weight.stride(0) % 16 != 0:   # moved without its padding
            pitch = (self.in_features + 15) // 16 * 16
            padded = torch.zeros(self.out_features, pitch, dtype=torch.int8, device=self.weight.device)
            self.weight = padded[:, :self.in_features].copy_(self.weight)
        if self.bias is not None and self.bias.dtype not in (torch.bfloat16, torch.float32):
            self.bias = self.bias.to(torch.bfloat16)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int8_linear(x, self.weight, self.weight_scale, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


__all__ = ["Int8Linear", "int8_gated_mlp", "int8_linear", "int8_matmul", "quantize_rows"]
