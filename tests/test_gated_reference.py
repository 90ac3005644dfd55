"""The references of the layer norm, gated recurrence and gated linear unit at the
values where they can go wrong."""

import pytest
import torch

from pytorch_r2d2_dpg_amd.ops.gated_linear import gated_linear
from pytorch_r2d2_dpg_amd.ops.gated_recurrence import gated_recurrence
from pytorch_r2d2_dpg_amd.ops.layer_norm import layer_norm


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_recurrence_pads_have_no_effect(fill, dtype):
    """Whatever the steps past a length hold, in gates and gradients."""
    T, B, H = 9, 4, 5
    lengths = torch.tensor([0, 3, 7, 9], dtype=torch.int32)
    got = []
    for pad in (0.0, fill):
        gates, h0 = rand(T, B, 3 * H, dtype=dtype), rand(B, H, seed=1)
        dy, dh = rand(T, B, H, seed=2, dtype=dtype), rand(B, H, seed=3)
        for b, n in enumerate(lengths.tolist()):
            gates[n:, b], dy[n:, b] = pad, pad
        leaves = [gates.requires_grad_(True), h0.requires_grad_(True)]
        outs = list(gated_recurrence(gates, h0, lengths))
        got.append(outs + list(torch.autograd.grad(outs, leaves, [dy, dh])))
    for clean, other in zip(*got):
        assert torch.equal(clean, other)
    y, hT, dgates, dh0 = got[1]
    for b, n in enumerate(lengths.tolist()):
        assert not y[n:, b].any() and not dgates[n:, b].any()
    assert torch.equal(hT[0], rand(B, H, seed=1)[0]) and torch.equal(dh0[0], rand(B, H, seed=3)[0])


def ints(*shape, dtype):
    return torch.ones(*shape, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.uint8, torch.bool, torch.complex64])
def test_types_that_are_not_real_floats_are_refused(dtype):
    """Results rounded to whole numbers would be wrong without an error."""
    for call in (lambda: layer_norm(ints(2, 4, dtype=dtype), ints(4, dtype=dtype)),
                 lambda: gated_recurrence(ints(2, 2, 6, dtype=dtype)),
                 lambda: gated_linear(ints(2, 4, dtype=dtype), ints(6, 4, dtype=dtype))):
        with pytest.raises(TypeError, match="floating"):
            call()
