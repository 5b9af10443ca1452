"""Drawing tokens from logits on the device (csrc/sd_sampling.cuh): temperature, top-k, top-p and min-p in one launch,
from random numbers that the caller gives."""
from __future__ import annotations

from typing import Union

import torch

from . import _lib


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                  min_p: Union[float, torch.Tensor] = 0.0, empty_token: int = -1) -> torch.Tensor:
    """One token per row of ``logits`` ``[B, V]`` (BF16 or FP32 CUDA, ``V`` up to 262144) as ``torch.long`` ``[B]``,
    drawn with the FP32 numbers ``uniform`` ``[B]`` in [0, 1).

    Candidates, in the order of their logits and equal ones by index, have the weight ``exp((x - max) / temperature)``.
    ``top_k`` keeps the first k of them (0: all), ``top_p`` of those the ones before which less than ``top_p`` of their
    weight lies (1: all; the first always stays), ``min_p`` those whose weight is at least ``min_p`` times the largest.
    The token is the first index at which the running sum of the kept weights, in the order of the vocabulary, exceeds
    ``uniform`` times their sum.  ``temperature`` 0 takes the first of the order.  Each setting is a number (taken in
    FP32) or a tensor ``[B]`` on the device of the logits, one value for each row (numbers out of range are refused; in a tensor a
    temperature that is not above 1e-30 and a ``top_p`` that is not above 0 take the first of the order, a ``top_k``
    below 1, a ``top_p`` above 1 and a ``min_p`` below 0 keep all, a ``min_p`` above 1 counts as 1).  A
    temperature above 1e30 counts as 1e30.

    Logits of -inf and NaN are never drawn; those of +inf share the draw.  A row that has nothing to draw gets
    ``empty_token``.  The weights are exact to 2^-45 of the largest (smaller ones are zero) and their sums are exact, so
    a row's token does not depend on the batch it is in.  Nothing synchronises with the host: the call can be captured
    into a graph."""
    return _lib.host().sample_tokens(logits, uniform, temperature, top_k, top_p, min_p, int(empty_token))


__all__ = ["sample_tokens"]
