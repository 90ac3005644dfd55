"""Layer norm, gated recurrence and gated linear unit on CPU: the references
against the definitions in 64 bits, their gradients against differences, and
the refusals, which the GPU path shares."""

import pytest
import torch

from gated_oracles import check, linear_oracle, norm_oracle, recurrence_oracle
from pytorch_r2d2_dpg_amd.ops.gated_linear import gated_linear
from pytorch_r2d2_dpg_amd.ops.gated_recurrence import gated_recurrence
from pytorch_r2d2_dpg_amd.ops.layer_norm import layer_norm


def rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ------------------------------------------------ references against 64 bits
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_reference(residual):
    x, w, b = rand(5, 3, 9), rand(9, seed=1), rand(9, seed=2)
    r, dy, ds = (rand(5, 3, 9, seed=s) if residual else None for s in (3, 4, 5))
    dy = rand(5, 3, 9, seed=4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    out = layer_norm(x, w, b, residual=r)
    outs, seeds = (list(out), [dy, ds]) if residual else ([out], [dy])
    got = outs + list(torch.autograd.grad(outs, leaves, seeds))
    for i, (a, e) in enumerate(zip(got, norm_oracle(x, w, b, r, dy, ds))):
        check(i, a, e)


@pytest.mark.parametrize("T", [0, 1, 7])
@pytest.mark.parametrize("ragged", [False, True])
def test_gated_recurrence_reference(T, ragged):
    B, H = 4, 5
    gates, h0 = rand(T, B, 3 * H).requires_grad_(True), rand(B, H, seed=1).requires_grad_(True)
    lengths = torch.tensor([0, 1, T, T + 3], dtype=torch.int32) if ragged else None
    dy, dh = rand(T, B, H, seed=2), rand(B, H, seed=3)
    y, hT = gated_recurrence(gates, h0, lengths)
    got = [y, hT] + list(torch.autograd.grad([y, hT], [gates, h0], [dy, dh], allow_unused=True))
    got[2] = torch.zeros_like(gates) if got[2] is None else got[2]
    for i, (a, e) in enumerate(zip(got, recurrence_oracle(gates, h0, lengths, dy, dh))):
        check(i, a, e)


@pytest.mark.parametrize("bias", [False, True])
def test_gated_linear_reference(bias):
    x, w, dy = rand(2, 3, 7).requires_grad_(True), rand(10, 7, seed=1).requires_grad_(True), rand(2, 3, 5, seed=2)
    b = rand(10, seed=3).requires_grad_(True) if bias else None
    y = gated_linear(x, w, b)
    got = [y] + list(torch.autograd.grad([y], [x, w] + ([b] if bias else []), [dy]))
    for i, (a, e) in enumerate(zip(got, linear_oracle(x, w, b, dy))):
        check(i, a, e)


def test_gradients_against_differences():
    d = torch.float64
    args = [rand(4, 6, dtype=d), rand(6, seed=1, dtype=d), rand(6, seed=2, dtype=d)]
    res = rand(4, 6, seed=3, dtype=d).requires_grad_(True)
    args = [t.requires_grad_(True) for t in args]
    assert torch.autograd.gradcheck(lambda x, w, b, r: layer_norm(x, w, b, residual=r), (*args, res))
    gates = rand(5, 3, 6, seed=4, dtype=d).requires_grad_(True)
    h0 = rand(3, 2, seed=5, dtype=d).requires_grad_(True)
    lengths = torch.tensor([0, 3, 5], dtype=torch.int32)
    assert torch.autograd.gradcheck(lambda g, h: gated_recurrence(g, h, lengths), (gates, h0))
    x, w = rand(3, 4, seed=6, dtype=d).requires_grad_(True), rand(6, 4, seed=7, dtype=d).requires_grad_(True)
    b = rand(6, seed=8, dtype=d).requires_grad_(True)
    assert torch.autograd.gradcheck(gated_linear, (x, w, b))


def test_types_follow_the_input():
    x, w = rand(3, 8, dtype=torch.bfloat16), rand(8, dtype=torch.bfloat16)
    assert layer_norm(x, w).dtype == torch.bfloat16
    y, h = gated_recurrence(rand(2, 3, 6, dtype=torch.bfloat16))
    assert y.dtype == torch.bfloat16 and h.dtype == torch.float32
    assert gated_linear(x, rand(4, 8, dtype=torch.bfloat16)).dtype == torch.bfloat16


# ------------------------------------------------------------------- refusals
@pytest.mark.parametrize("call, error", [
    (lambda: layer_norm(torch.tensor(1.0), rand(1)), ValueError),
    (lambda: layer_norm(rand(3, 0), rand(0)), ValueError),
    (lambda: layer_norm(rand(3, 4), rand(5)), ValueError),
    (lambda: layer_norm(rand(3, 4), rand(4), rand(3)), ValueError),
    (lambda: layer_norm(rand(3, 4), rand(4), residual=rand(1, 4)), ValueError),
    (lambda: layer_norm(rand(3, 4), rand(4, dtype=torch.bfloat16)), TypeError),
    (lambda: gated_recurrence(rand(3, 6)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 7)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 6), rand(3, 3)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 6), rand(3, 2, dtype=torch.bfloat16)), TypeError),
    (lambda: gated_recurrence(rand(2, 3, 6), None, torch.zeros(2, dtype=torch.int32)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 6), None, torch.zeros(3)), TypeError),
    (lambda: gated_linear(torch.tensor(1.0), rand(4, 1)), ValueError),
    (lambda: gated_linear(rand(3, 4), rand(5, 4)), ValueError),
    (lambda: gated_linear(rand(3, 4), rand(6, 5)), ValueError),
    (lambda: gated_linear(rand(3, 4), rand(6, 4), rand(3)), ValueError),
    (lambda: gated_linear(rand(3, 4), rand(6, 4, dtype=torch.bfloat16)), TypeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()
