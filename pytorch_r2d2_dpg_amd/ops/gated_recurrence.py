"""Gated linear recurrence over time (kernel K10).

    a = sigma(f);  h_t = a_t h_{t-1} + (1 - a_t) v_t;  y_t = h_t silu(o_t)

The gates come packed from one projection, as the LSTM's do, but none of them
depends on h: the recurrence is linear, so time scans in parallel where the
LSTM's steps form a chain. The state is held in 32 bits whatever the gates'
type. One step (T = 1) is the same call. On GPU the HIP kernels run (bf16 or
fp32), on CPU the differentiable reference.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import hip_ext
from .reference import gated_recurrence_ref


def gated_recurrence(
    gates: torch.Tensor,                     # [T, B, 3H]: forget, value, output
    h0: Optional[torch.Tensor] = None,       # [B, H] fp32; zeros where absent
    lengths: Optional[torch.Tensor] = None,  # [B] int32: real steps of each row
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Run the recurrence from ``h0``. Returns (y [T,B,H] in the gates' type,
    hT [B,H] in fp32).

    With ``lengths`` the steps at or past lengths[b] hold row b's state: their
    y is 0, their gates have no effect and no gradient. Values outside [0, T]
    count as the nearer end. Differentiable once in gates and h0.
    """
    if gates.is_cuda:
        return hip_ext().gated_recurrence(gates, h0, lengths)
    if not gates.is_floating_point():
        raise TypeError(f"gates must be of a floating type, got {gates.dtype}")
    if gates.dim() != 3 or gates.shape[2] % 3:
        raise ValueError(f"gates must be [T, B, 3H], got {tuple(gates.shape)}")
    B, H = gates.shape[1], gates.shape[2] // 3
    if h0 is not None:
        if h0.shape != (B, H):
            raise ValueError(f"h0 must be [{B}, {H}], got {tuple(h0.shape)}")
        wide = torch.promote_types(gates.dtype, torch.float32)
        if h0.dtype != wide:
            raise TypeError(f"h0 must be {wide}: the state is not rounded (got {h0.dtype})")
    if lengths is not None:
        if lengths.shape != (B,):
            raise ValueError(f"lengths must be [{B}], got {tuple(lengths.shape)}")
        if lengths.dtype != torch.int32:
            raise TypeError(f"lengths must be int32, got {lengths.dtype}")
    return gated_recurrence_ref(gates, h0, lengths)
