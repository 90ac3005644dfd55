"""Layer norm with a fused residual sum (kernel K9).

    s = x + residual;  n = (s - mean(s)) / sqrt(var(s) + eps);  y = n * weight + bias

over the last axis: one launch forward, two backward (rows, then the fixed-order
sum of the weight's and bias's gradients). Sums and statistics are in 32 bits.
On GPU the HIP kernel runs (bf16 or fp32), on CPU the differentiable reference.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import hip_ext
from .reference import layer_norm_ref


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, s = hip_ext().layer_norm_fwd(x, weight, bias, residual, eps)
        ctx.set_materialize_grads(False)
        ctx.has_bias, ctx.fused, ctx.eps = bias is not None, residual is not None, eps
        ctx.save_for_backward(x, weight, residual)
        return y if residual is None else (y, s)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds=None):
        x, weight, residual = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else dy.contiguous()
        ds = None if ds is None else ds.contiguous()
        dx, dwb = hip_ext().layer_norm_bwd(x, residual, weight, dy, ds, ctx.eps)
        return dx, dwb[0], dwb[1] if ctx.has_bias else None, dx if ctx.fused else None, None


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
    if not x.is_cuda:
        return layer_norm_ref(x, weight, bias, eps, residual)
    x, weight = x.contiguous(), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        hip_ext().check_capture(given)
        return _LayerNorm.apply(x, weight, bias, residual, float(eps))
    y, s = hip_ext().layer_norm_fwd(x, weight, bias, residual, float(eps))
    return y if residual is None else (y, s)
