"""Gated linear unit: the first half of a gated feed-forward (kernel K11).

    y = silu(x Wg^T + bg) * (x Wv^T + bv)

with both projections, the activation and the product in one MFMA kernel; the
pre-activations never reach memory, forward or backward (the backward pass
computes them again). On GPU the HIP kernels run (bf16 or fp32, fp32
accumulation), on CPU the differentiable reference.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import hip_ext
from .reference import gated_linear_ref


def gated_linear(
    x: torch.Tensor,                      # [..., K]
    weight: torch.Tensor,                 # [2F, K]: the gate's rows, then the value's
    bias: Optional[torch.Tensor] = None,  # [2F]
) -> torch.Tensor:
    """silu(x Wg^T + bg) * (x Wv^T + bv), [..., F] in x's type.

    weight and bias share x's type. Differentiable once in every tensor.
    """
    if x.is_cuda:
        return hip_ext().gated_linear(x, weight, bias)
    if not x.is_floating_point():
        raise TypeError(f"x must be of a floating type, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError("x must have a last axis")
    if weight.dim() != 2 or weight.shape[0] % 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight must be [2F, {x.shape[-1]}], got {tuple(weight.shape)}")
    if bias is not None and bias.shape != (weight.shape[0],):
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    given = [t for t in (x, weight, bias) if t is not None]
    if any(t.dtype != x.dtype for t in given):
        raise TypeError(f"dtype mismatch: {[t.dtype for t in given]}")
    return gated_linear_ref(x, weight, bias)
