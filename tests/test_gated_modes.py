"""Ways of calling the layer norm, gated recurrence and gated linear unit that
their kernels cannot serve: each is refused, and none gives a wrong answer."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from pytorch_r2d2_dpg_amd.ops import ext_available, hip_ext
from pytorch_r2d2_dpg_amd.ops.gated_linear import gated_linear
from pytorch_r2d2_dpg_amd.ops.gated_recurrence import gated_recurrence
from pytorch_r2d2_dpg_amd.ops.layer_norm import layer_norm

built = pytest.mark.skipif(not ext_available(), reason="the extension is not built")


def args(device="cpu"):
    """For each operator a call of its binding, and of its entry point, as functions
    of its first argument, with one to call them with."""
    x, w, w2 = torch.randn(3, 8, device=device), torch.ones(8, device=device), torch.randn(6, 8, device=device)
    g = torch.randn(2, 3, 6, device=device)
    return [
        (x, lambda t: hip_ext().layer_norm(t, w, None, 1e-5, None)[0], lambda t: layer_norm(t, w)),
        (g, lambda t: hip_ext().gated_recurrence(t, None, None)[0], lambda t: gated_recurrence(t)[0]),
        (x, lambda t: hip_ext().gated_linear(t, w2, None), lambda t: gated_linear(t, w2)),
    ]


# ------------------------------------------------------- forward-mode tangents
@built
@pytest.mark.parametrize("grad", [True, False])
def test_bindings_refuse_tangents(grad):
    """no_grad does not switch forward mode off: a tangent would be lost in silence.
    Looked for before the device is, so that this shows without a GPU."""
    for x, binding, _ in args():
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            d = fwd.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                binding(d)


def test_references_carry_tangents_without_gradients():
    for x, _, op in args():
        with fwd.dual_level(), torch.no_grad():
            assert fwd.unpack_dual(op(fwd.make_dual(x, torch.ones_like(x)))).tangent is not None


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    for x, _, op in args("cuda"):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            d = fwd.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                op(d)
            with torch.inference_mode():  # torch itself carries no tangent here
                assert torch.equal(op(d), op(x))
