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


# ------------------------------------------------------------------- recording
def recorders():
    """Ways of recording a function's torch operations, by name."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def fake(f, x):
        mode = FakeTensorMode(allow_non_fake_inputs=True)
        with mode:
            return f(x)

    def functional(f, x):
        from torch._subclasses.functional_tensor import FunctionalTensorMode
        with FunctionalTensorMode():
            return f(x)

    return {
        "jit.trace": lambda f, x: torch.jit.trace(f, (x,), check_trace=False),
        "make_fx": lambda f, x: make_fx(f)(x),
        "make_fx, before dispatch": lambda f, x: make_fx(f, pre_dispatch=True)(x),
        "make_fx of fake tensors": lambda f, x: make_fx(f, tracing_mode="fake")(x),
        "fake tensors": fake,
        "functional tensors": functional,
    }


RECORDERS = ["jit.trace", "make_fx", "make_fx, before dispatch", "make_fx of fake tensors",
             "fake tensors", "functional tensors"]


@built
@pytest.mark.parametrize("way", RECORDERS)
def test_bindings_refuse_to_be_recorded(way):
    """A recording has the outputs' allocations, and not the launch that fills them.
    Looked for before the device is, so that this shows without a GPU."""
    for x, binding, _ in args():
        with pytest.raises(NotImplementedError, match="recorded"):
            recorders()[way](binding, x)


@pytest.mark.parametrize("way", ["jit.trace", "make_fx"])
def test_references_can_be_recorded(way):
    for x, _, op in args():
        other = x + 1
        assert torch.equal(recorders()[way](op, x)(other), op(other))


@pytest.mark.gpu
@pytest.mark.parametrize("way", RECORDERS)
def test_recording_is_refused(way):
    for x, _, op in args("cuda"):
        with pytest.raises(NotImplementedError, match="recorded"):
            recorders()[way](op, x)
        assert op(x).isfinite().all()  # and nothing of it stays


@pytest.mark.gpu
def test_modes_that_only_watch_are_served():
    from torch.utils.flop_counter import FlopCounterMode
    for x, _, op in args("cuda"):
        want = op(x)
        with FlopCounterMode(display=False):
            assert torch.equal(op(x), want)


# ----------------------------------------------------------- the backward pass
@pytest.mark.gpu
def test_a_gradient_with_a_tangent_is_refused():
    """Forward mode through the backward pass alone: the outputs' gradients carry the
    tangents, of either output of an operator with two."""
    for i, (x, _, op) in enumerate(args("cuda")):
        x.requires_grad_(True)
        y = op(x)
        dy = torch.ones_like(y)
        with fwd.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, x, fwd.make_dual(dy, dy), retain_graph=True)
        assert torch.autograd.grad(y, x, dy)[0].isfinite().all()
    x, g = torch.randn(3, 8, device="cuda"), torch.randn(2, 3, 6, device="cuda", requires_grad=True)
    r = torch.randn(3, 8, device="cuda", requires_grad=True)
    for second, leaf in ((layer_norm(x, torch.ones(8, device="cuda"), residual=r)[1], r),
                         (gated_recurrence(g)[1], g)):
        with fwd.dual_level():
            d = fwd.make_dual(torch.ones_like(second), torch.ones_like(second))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(second, leaf, d)


@pytest.mark.gpu
@pytest.mark.parametrize("before", [False, True])
def test_recording_the_backward_pass_is_refused(before):
    from torch.fx.experimental.proxy_tensor import make_fx
    for x, _, op in args("cuda"):
        x.requires_grad_(True)
        y = op(x)
        dy = torch.ones_like(y)
        back = make_fx(lambda g: torch.autograd.grad(y, x, g, retain_graph=True)[0], pre_dispatch=before)
        with pytest.raises(NotImplementedError, match="recorded"):
            back(dy)
        assert torch.autograd.grad(y, x, dy)[0].isfinite().all()


# -------------------------------------------------------------------- captures
@pytest.mark.gpu
def test_capture_of_an_eagerly_computed_input_is_refused():
    """Its backward pass would leave the capture for the stream of the eager one."""
    for x, _, op in args("cuda"):
        leaf = x.clone().requires_grad_(True)
        y = leaf * 2
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                op(y)
        want = torch.autograd.grad(op(y), leaf, torch.ones_like(op(x)))[0]  # eager: as ever
        assert want.isfinite().all()


@pytest.mark.gpu
def test_capture_of_inputs_computed_within_it():
    for x, _, op in args("cuda"):
        leaf = x.clone().requires_grad_(True)
        dy = torch.randn_like(op(x))

        def step():
            return torch.autograd.grad(op(leaf * 2), leaf, dy)[0]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for turn in range(3):
            with torch.no_grad():
                leaf.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, step())
        eager = x.clone().requires_grad_(True) * 2
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():  # nothing to differentiate
            y = op(eager)
        graph.replay()
        assert torch.equal(y, op(eager).detach())


@pytest.mark.gpu
def test_capture_over_an_eager_graph_of_a_side_stream():
    """A side stream joins the capture, unlike the default stream: a warm-up's graph may live."""
    for x, _, op in args("cuda"):
        leaf = x.clone().requires_grad_(True)
        dy = torch.randn_like(op(x))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            alive = op(leaf)
            torch.autograd.grad(alive, leaf, dy)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = op(leaf)
            got = torch.autograd.grad(y, leaf, dy)[0]
        y = y.detach()
        for _ in range(3):
            with torch.no_grad():
                leaf.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            fresh = leaf.detach().clone().requires_grad_(True)
            want = op(fresh)
            assert torch.equal(y, want) and torch.equal(got, torch.autograd.grad(want, fresh, dy)[0])
        del alive


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_graphed_callables(dtype):
    """torch's own capture of a module, forward and backward, whose warm-up graph lives."""
    from pytorch_r2d2_dpg_amd.models import GatedCore

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.core = GatedCore(24, 32)

        def forward(self, x):
            return self.core(x)[0]

    torch.manual_seed(6)
    net = Net().to("cuda", dtype)
    plain = Net().to("cuda", dtype)
    plain.load_state_dict(net.state_dict())
    sample = torch.randn(9, 4, 24, device="cuda", dtype=dtype, requires_grad=True)
    graphed = torch.cuda.make_graphed_callables(net, (sample,))
    for _ in range(3):
        x = torch.randn(9, 4, 24, device="cuda", dtype=dtype, requires_grad=True)
        dy = torch.randn(9, 4, 32, device="cuda", dtype=dtype)
        want = torch.autograd.grad(plain(x), [x, *plain.parameters()], dy)
        got = torch.autograd.grad(graphed(x), [x, *net.parameters()], dy)
        # Library products may sum in another order: as in test_gated_core.py either side
        # is 24 roundings of half a step off at most.
        for a, b in zip(got, want):
            assert (a - b).double().norm() <= 24 * torch.finfo(dtype).eps * b.double().norm()


# --------------------------------------------------------- tensors without memory
@built
@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_tensors_without_memory_are_refused(device):
    """Fake tensors that outlive their mode, and zeros that are only said to be: their
    pointer is null. No GPU takes part: refused before the device is looked for."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w, w2 = (torch.empty(*s, device=device) for s in ((3, 8), (8,), (6, 8)))
        g, h0 = torch.empty(2, 3, 6, device=device), torch.empty(3, 2, device=device)
        n = torch.empty(3, dtype=torch.int32, device=device)
    e = hip_ext()
    calls = [lambda: e.layer_norm(x, w, None, 1e-5, None), lambda: e.gated_recurrence(g, None, None),
             lambda: e.gated_linear(x, w2, None)]
    if device == "cuda":
        calls += [lambda: layer_norm(x, w), lambda: gated_recurrence(g), lambda: gated_linear(x, w2)]
    else:  # in any place
        real, rg, zero = torch.randn(3, 8), torch.randn(2, 3, 6), torch._efficientzerotensor((3, 8))
        calls += [lambda: e.layer_norm(real, w, None, 1e-5, None),
                  lambda: e.layer_norm(real, torch.ones(8), w, 1e-5, None),
                  lambda: e.layer_norm(real, torch.ones(8), None, 1e-5, zero),
                  lambda: e.layer_norm(zero, torch.ones(8), None, 1e-5, None),
                  lambda: e.gated_recurrence(rg, h0, None), lambda: e.gated_recurrence(rg, None, n),
                  lambda: e.gated_linear(real, w2, None), lambda: e.gated_linear(zero, torch.ones(6, 8), None)]
    for call in calls:
        with pytest.raises(NotImplementedError, match="memory"):
            call()


@pytest.mark.gpu
def test_negations_that_are_only_noted():
    """Such as the imaginary part of a conjugate: memory holds the values before the sign."""
    def neg(t):
        return torch._neg_view(t)

    x, w, g, h0, w2, r = (torch.randn(*s, device="cuda") for s in
                          ((3, 8), (8,), (2, 3, 6), (3, 2), (6, 8), (3, 8)))
    for op, ts in ((lambda a, b, c: layer_norm(a, b, b, residual=c)[0], (x, w, r)),
                   (lambda a, b: gated_recurrence(a, b)[0], (g, h0)),
                   (lambda a, b: gated_linear(a, b), (x, w2))):
        assert torch.equal(op(*map(neg, ts)), op(*(-t for t in ts)))
        leaves = [t.clone().requires_grad_(True) for t in ts]
        y = op(*map(neg, leaves))
        dy = torch.randn_like(y)
        got = torch.autograd.grad(y, leaves, neg(dy))
        plain = [(-t).detach().requires_grad_(True) for t in ts]
        for a, b in zip(got, torch.autograd.grad(op(*plain), plain, dy)):  # the signs cancel
            assert torch.equal(a, b)
    z = torch.complex(torch.randn(1, 1, device="cuda"), torch.randn(1, 1, device="cuda"))
    one, bias = torch.ones(1, device="cuda"), torch.ones(2, device="cuda")
    im = z.conj().imag
    assert im.is_neg() and im.is_contiguous()
    ww = torch.ones(2, 1, device="cuda")
    assert torch.equal(gated_linear(im, ww, bias), gated_linear(-z.imag, ww, bias))
    assert torch.equal(layer_norm(one, one, im[0]), layer_norm(one, one, -z.imag[0]))
