"""GatedCore module — residual gated-recurrence blocks in place of the LSTM.

Two pre-norm blocks at the hidden size, each of a gated linear recurrence and a
gated feed-forward:

    s = in(x);   per block:
        y, h = gated_recurrence(gates(norm(s)), h);    s = s + mix(y)
        s = s + down(gated_linear(norm(s)))

and a last norm. No gate depends on h, so an unroll is a scan and a few large
products where the LSTM's is a chain of T dependent ones. The residual sums run
inside the norms. The state is the pair (h of block one, h of block two), each
[B, H] in fp32: it fits wherever the LSTM's (h, c) does.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import nn

from ..ops.gated_linear import gated_linear
from ..ops.gated_recurrence import gated_recurrence
from ..ops.layer_norm import layer_norm
from .lstm import State


class _Norm(nn.Module):
    def __init__(self, size: int):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(size))
        self.bias = nn.Parameter(torch.zeros(size))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return layer_norm(x, self.weight, self.bias, residual=residual)


class GatedBlock(nn.Module):
    def __init__(self, hidden_size: int, width: int):
        super().__init__()
        H = hidden_size
        self.norm_in = _Norm(H)
        self.gates = nn.Linear(H, 3 * H)   # forget, value, output
        self.mix = nn.Linear(H, H)
        self.norm_ff = _Norm(H)
        self.up = nn.Linear(H, 2 * width)  # gate, value
        self.down = nn.Linear(width, H)
        with torch.no_grad():
            # forget gates that remember over 2 to 128 steps, spread by their logarithm
            steps = torch.exp(torch.empty(H).uniform_(math.log(2.0), math.log(128.0)))
            self.gates.bias[:H] = torch.log(steps - 1.0)


class GatedCore(nn.Module):
    def __init__(self, input_size: int, hidden_size: int):
        super().__init__()
        self.input_size = input_size
        self.hidden_size = hidden_size
        self.inp = nn.Linear(input_size, hidden_size)
        self.blocks = nn.ModuleList(GatedBlock(hidden_size, 2 * hidden_size) for _ in range(2))
        self.norm_out = _Norm(hidden_size)

    def zero_state(self, batch: int, device=None, dtype=None) -> State:
        """The state stays fp32 (or wider) whatever the parameters' type."""
        p = self.inp.weight
        dtype = torch.promote_types(dtype or p.dtype, torch.float32)
        z = torch.zeros(batch, self.hidden_size, device=device or p.device, dtype=dtype)
        return z, z.clone()

    def forward(self, x: torch.Tensor, state: Optional[State] = None):
        """x: [T, B, I]; returns (y [T,B,H], (h1, h2))."""
        wide = torch.promote_types(x.dtype, torch.float32)
        if state is None:
            state = self.zero_state(x.shape[1], device=x.device, dtype=x.dtype)
        s = self.inp(x)
        n = self.blocks[0].norm_in(s)
        out = []
        for i, (block, h) in enumerate(zip(self.blocks, state)):
            y, h = gated_recurrence(block.gates(n), h.to(wide))
            out.append(h)
            n, s = block.norm_ff(block.mix(y), residual=s)
            f = block.down(gated_linear(n, block.up.weight, block.up.bias))
            last = i + 1 == len(self.blocks)
            n, s = (self.norm_out if last else self.blocks[i + 1].norm_in)(f, residual=s)
        return n, (out[0], out[1])

    def step(self, x: torch.Tensor, state: Optional[State] = None):
        """x: [B, I] single step; returns (y [B,H], (h1, h2))."""
        y, st = self.forward(x.unsqueeze(0), state)
        return y[0], st
