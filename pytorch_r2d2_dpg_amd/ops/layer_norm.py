"""Layer norm with a fused residual sum (kernel K9).

    s = x + residual;  n = (s - mean(s)) / sqrt(var(s) + eps);  y = n * weight + bias

over the last axis: one launch forward, two backward (rows, then the fixed-order
sum of the weight's and bias's gradients). Sums and statistics are in 32 bits.
On GPU the HIP kernels run (bf16 or fp32; checks and gradient are the binding's),
on CPU the differentiable reference.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import hip_ext
from .reference import layer_norm_ref


def layer_norm(
    x: torch.Tensor,                          # [..., D]
    weight: torch.Tensor,                     # [D]
    bias: Optional[torch.Tensor] = None,      # [D]
    eps: float = 1e-5,
    residual: Optional[torch.Tensor] = None,  # like x
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Normalise the last axis of ``x``, or of ``x + residual``.

    Returns y, or (y, x + residual) where a residual is given; both have x's
    shape and type, which weight, bias and residual share. Differentiable once
    in every tensor.
    """
    if x.is_cuda:
        out = hip_ext().layer_norm(x, weight, bias, eps, residual)
        return out[0] if residual is None else (out[0], out[1])
    if not x.is_floating_point():
        raise TypeError(f"x must be of a floating type, got {x.dtype}")
    D = x.shape[-1] if x.dim() else 0
    if D == 0:
        raise ValueError(f"x must have a last axis to normalise (got {tuple(x.shape)})")
    if weight.shape != (D,) or (bias is not None and bias.shape != (D,)):
        raise ValueError(f"weight and bias must be [{D}]")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must have x's shape {tuple(x.shape)}, "
                         f"got {tuple(residual.shape)}")
    given = [t for t in (x, weight, bias, residual) if t is not None]
    if any(t.dtype != x.dtype for t in given):
        raise TypeError(f"dtype mismatch: {[t.dtype for t in given]}")
    return layer_norm_ref(x, weight, bias, eps, residual)
