"""Layer norm, gated recurrence and gated linear unit kernels against their
definitions in 64 bits, at the sizes and masks where they can go wrong."""

import pytest
import torch

from gated_oracles import check, linear_oracle, norm_oracle, recurrence_oracle
from pytorch_r2d2_dpg_amd.ops.gated_linear import gated_linear
from pytorch_r2d2_dpg_amd.ops.gated_recurrence import gated_recurrence
from pytorch_r2d2_dpg_amd.ops.layer_norm import layer_norm

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def rand(*shape, seed=0, dtype=FP32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed + 1000 * len(shape))
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).cuda()


def leaves(*tensors):
    for t in tensors:
        if t is not None:
            t.requires_grad_(True)
    return [t for t in tensors if t is not None]


def check_all(got, want):
    assert len(got) == len(want)
    for i, (g, w) in enumerate(zip(got, want)):
        check(f"output {i}", g, w)


# ------------------------------------------------------------------ layer norm
def run_norm(rows, dim, dtype, residual, bias=True, seed=0, scale=1.0, shift=0.2):
    x = rand(rows, dim, seed=seed, dtype=dtype, scale=scale, shift=shift)
    w = rand(dim, seed=seed + 1, dtype=dtype, scale=0.1, shift=1.0)
    b = rand(dim, seed=seed + 2, dtype=dtype) if bias else None
    r = rand(rows, dim, seed=seed + 3, dtype=dtype) if residual else None
    dy, ds = rand(rows, dim, seed=seed + 4, dtype=dtype), rand(rows, dim, seed=seed + 5, dtype=dtype)
    ins = leaves(x, w, b, r)
    out = layer_norm(x, w, b, residual=r)
    outs, seeds = (list(out), [dy, ds]) if residual else ([out], [dy])
    grads = list(torch.autograd.grad(outs, ins, seeds))
    if residual:
        assert torch.equal(grads[0], grads.pop())  # x and the residual share one gradient
    check_all(outs + grads, norm_oracle(x, w, b, r, dy, ds if residual else None))
    with torch.no_grad():  # the same values without gradients
        again = layer_norm(x, w, b, residual=r)
    for a, o in zip(again if residual else [again], outs):
        assert torch.equal(a, o)


# each count of threads and runs a row, both sides of every border, and past registers
@pytest.mark.parametrize("dim", [1, 7, 64, 512, 513, 771, 1025, 2048, 2049, 4100, 8192, 8200, 33000])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_dims(dim, dtype, residual):
    run_norm(5, dim, dtype, residual, seed=dim)


@pytest.mark.parametrize("rows", [0, 1, 3, 4, 2049, 5000])
@pytest.mark.parametrize("dim", [40, 600])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_norm_rows(rows, dim, dtype):
    run_norm(rows, dim, dtype, True, bias=rows != 3, seed=rows)


def test_norm_far_from_zero_and_constant():
    run_norm(9, 300, FP32, False, scale=0.01, shift=1000.0)  # the variance must not cancel
    x = torch.full((3, 70), 2.5, device="cuda")
    y = layer_norm(x, rand(70), rand(70, seed=1))
    assert torch.equal(y, rand(70, seed=1).expand(3, 70))


def test_norm_keeps_rows_apart():
    x, w = rand(6, 200), rand(200, seed=1)
    clean = layer_norm(x, w)
    bad = x.clone()
    bad[1, 3], bad[4, 7] = float("nan"), float("inf")
    y = layer_norm(bad, w)
    for i in (0, 2, 3, 5):
        assert torch.equal(y[i], clean[i])
    assert y[1].isnan().all() and y[4].isnan().any()


def test_norm_strides_and_shapes():
    wide = rand(4, 6, 90, dtype=BF16)
    x, w = wide[:, ::2, 5:55], rand(100, seed=1, dtype=BF16)[::2]
    assert torch.equal(layer_norm(x, w), layer_norm(x.contiguous(), w.contiguous()))
    x0 = wide.view(-1)[1:1 + 23 * 50].view(23, 50)  # rows that start on odd elements
    dy = rand(23, 50, seed=2, dtype=BF16)
    ins = leaves(x0.detach(), w.contiguous())
    y = layer_norm(*ins)
    check_all([y] + list(torch.autograd.grad([y], ins, [dy])), norm_oracle(*ins, None, None, dy, None))


def test_norm_partial_gradients():
    x, w, r = rand(7, 33), rand(33, seed=1), rand(7, 33, seed=2)
    ins = leaves(x, w, r)
    _, s = layer_norm(x, w, residual=r)
    g = rand(7, 33, seed=3)
    gx, gw, gr = torch.autograd.grad([s], ins, [g])  # through the sum alone
    assert torch.equal(gx, g) and torch.equal(gr, g) and not gw.any()
    y, _ = layer_norm(x, w, residual=r)
    check_all([torch.autograd.grad([y], [x], [g])[0]],
              [norm_oracle(x, w, None, r, g, torch.zeros_like(g))[2]])


def test_norm_many_short_rows():
    run_norm(4_300_000, 3, BF16, False)  # more threads than a launch has, at 1024 a row


def test_norm_offsets_past_32_bits():
    few, times, dim = 1000, 1100, 2048  # 2.25e9 elements
    x, r = (rand(few, dim, seed=i, dtype=BF16).repeat(times, 1) for i in (0, 1))
    dy = rand(few, dim, seed=2, dtype=BF16).repeat(times, 1)
    w, b = rand(dim, seed=3, dtype=BF16), rand(dim, seed=4, dtype=BF16)
    ins = leaves(x)
    y, s = layer_norm(x, w, b, residual=r)
    dx = torch.autograd.grad([y], ins, [dy])[0]
    want = norm_oracle(x[:few], w, b, r[:few], dy[:few], torch.zeros_like(dy[:few]))
    for i in (0, times // 2, times - 1):
        rows = slice(i * few, (i + 1) * few)
        check_all([y[rows], s[rows], dx[rows]], want[:3])


# ------------------------------------------------------------ gated recurrence
def run_recurrence(T, B, H, dtype, lengths=None, state=True, seed=0):
    gates = rand(T, B, 3 * H, seed=seed, dtype=dtype)
    gates[:, :, :H] *= 1.5
    gates[:, :, :H] += 2
    h0 = rand(B, H, seed=seed + 1) if state else None
    dy, dh = rand(T, B, H, seed=seed + 2, dtype=dtype), rand(B, H, seed=seed + 3)
    if lengths is not None:
        lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ins = leaves(gates, h0)
    outs = list(gated_recurrence(gates, h0, lengths))
    got = outs + list(torch.autograd.grad(outs, ins, [dy, dh]))
    want = recurrence_oracle(gates, h0, lengths, dy, dh)
    check_all(got, want if state else want[:3])
    with torch.no_grad():
        for a, o in zip(gated_recurrence(gates, h0, lengths), outs):
            assert torch.equal(a, o)
    return got


# one step, borders of a wave's chunk, of a block's waves, several passes, segments
@pytest.mark.parametrize("T", [0, 1, 2, 15, 16, 17, 40, 128, 129, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_recurrence_steps(T, dtype):
    run_recurrence(T, 3, 70, dtype, seed=T)


@pytest.mark.parametrize("B, H", [(1, 1), (1, 2), (5, 3), (33, 64), (2, 129), (7, 200), (0, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_recurrence_channels(B, H, dtype):
    run_recurrence(37, B, H, dtype, state=H != 64, seed=B + H)


@pytest.mark.parametrize("B, H", [(0, 8), (3, 0), (0, 0)])
def test_recurrence_without_channels(B, H):
    for T in (0, 1, 3000):
        run_recurrence(T, B, H, FP32)


@pytest.mark.parametrize("T, B, H", [(3000, 1, 64), (2049, 2, 65), (5000, 3, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_recurrence_long(T, B, H, dtype):
    run_recurrence(T, B, H, dtype, lengths=[T - 1000, T + 5, 17][:B] if B > 1 else None, seed=T)


@pytest.mark.parametrize("T", [1, 16, 75, 400])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_recurrence_lengths(T, dtype):
    run_recurrence(T, 6, 33, dtype, lengths=[0, 1, T, T + 9, -3, T // 2], seed=T)


def test_recurrence_pads_have_no_effect():
    T, B, H = 50, 4, 48
    lengths = torch.tensor([0, 13, 32, 50], dtype=torch.int32, device="cuda")
    got = []
    for fill in (0.0, float("nan"), float("inf"), torch.finfo(FP32).min):
        gates, h0 = rand(T, B, 3 * H), rand(B, H, seed=1)
        dy, dh = rand(T, B, H, seed=2), rand(B, H, seed=3)
        for b, n in enumerate(lengths.tolist()):
            gates[n:, b], dy[n:, b] = fill, fill
        ins = leaves(gates, h0)
        outs = list(gated_recurrence(gates, h0, lengths))
        got.append(outs + list(torch.autograd.grad(outs, ins, [dy, dh])))
    y, hT, dg, dh0 = got[0]
    for b, n in enumerate(lengths.tolist()):
        assert not y[n:, b].any() and not dg[n:, b].any()
    assert torch.equal(hT[0], rand(B, H, seed=1)[0]) and torch.equal(dh0[0], rand(B, H, seed=3)[0])
    for other in got[1:]:
        for a, o in zip(other, got[0]):
            assert torch.equal(a, o)


def test_recurrence_saturated_gates():
    T, B, H = 20, 2, 32
    for f in (float("inf"), 200.0, -200.0, float("-inf")):
        gates, h0 = rand(T, B, 3 * H), rand(B, H, seed=1)
        gates[:, :, :H] = f
        ins = leaves(gates, h0)
        y, hT = gated_recurrence(gates, h0)
        assert torch.equal(hT, h0 if f > 0 else gates[-1, :, H:2 * H])
        for g in torch.autograd.grad([y, hT], ins, [torch.ones_like(y), torch.ones_like(hT)]):
            assert g.isfinite().all()


def test_recurrence_in_pieces():
    """One step a call, as a serving loop makes them, ends where one call does."""
    T, B, H = 40, 5, 72
    gates, h0 = rand(T, B, 3 * H, dtype=BF16), rand(B, H, seed=1)
    want = recurrence_oracle(gates, h0, None, None, None)
    with torch.no_grad():
        h, ys = h0, []
        for t in range(T):
            y, h = gated_recurrence(gates[t:t + 1], h)
            ys.append(y)
    check_all([torch.cat(ys), h], want[:2])


def test_recurrence_strides_and_partial_gradients():
    T, B, H = 30, 4, 20
    gates = rand(B, T, 3 * H).transpose(0, 1)
    dy = rand(B, T, H, seed=1).transpose(0, 1)
    ins = leaves(gates.detach())
    y, hT = gated_recurrence(*ins)
    want = recurrence_oracle(gates, None, None, dy, None)
    check_all([y, hT, torch.autograd.grad([y], ins, [dy])[0]], want[:3])
    dh = rand(B, H, seed=2)
    y, hT = gated_recurrence(*ins)
    check_all([torch.autograd.grad([hT], ins, [dh])[0]],
              [recurrence_oracle(gates, None, None, None, dh)[2]])


def test_recurrence_offsets_past_32_bits():
    T, B, H = 2816, 512, 512  # 2.2e9 gate values
    gates = torch.randn(T, 1, 3 * H, device="cuda", dtype=BF16).repeat(1, B, 1)
    gates[:, -1] = rand(T, 3 * H, dtype=BF16)
    ins = leaves(gates)
    dy = torch.ones(T, B, H, device="cuda", dtype=BF16)
    y, hT = gated_recurrence(gates)
    dg = torch.autograd.grad([y], ins, [dy])[0]
    want = recurrence_oracle(gates[:, -1:], None, None, dy[:, -1:], None)
    check_all([y[:, -1:], hT[-1:], dg[:, -1:]], want[:3])
    assert torch.equal(y[:, 0], y[:, -2]) and torch.equal(dg[:, 0], dg[:, -2])


def test_recurrence_steps_past_32_bits():
    """Steps whose gates lie 2^31 values on: the last of them forget the first,
    as a thousand sigmoids of normal gates multiply to less than 2^-500."""
    T, tail = 720_000_000, 1000
    gates = torch.zeros(T, 1, 3, device="cuda", dtype=BF16)
    gates[-tail:] = rand(tail, 1, 3, dtype=BF16)
    dy = torch.ones(T, 1, 1, device="cuda", dtype=BF16)
    ins = leaves(gates)
    y, hT = gated_recurrence(gates)
    dg = torch.autograd.grad([y], ins, [dy])[0]
    want = recurrence_oracle(gates[-tail:], None, None, dy[-tail:], None)
    check_all([y[-tail:], hT, dg[-tail:]], want[:3])
    assert not y[:-tail].any()


# ----------------------------------------------------------- gated linear unit
def run_linear(M, K, F, dtype, bias=True, seed=0, shape=None, oracle_on="cpu"):
    x = rand(M, K, seed=seed, dtype=dtype).reshape(shape or (M, K))
    w = rand(2 * F, K, seed=seed + 1, dtype=dtype, scale=max(K, 1) ** -0.5)
    b = rand(2 * F, seed=seed + 2, dtype=dtype, scale=0.3) if bias else None
    dy = rand(M, F, seed=seed + 3, dtype=dtype).reshape(*x.shape[:-1], F)
    ins = leaves(x, w, b)
    y = gated_linear(x, w, b)
    got = [y] + list(torch.autograd.grad([y], ins, [dy]))
    want = linear_oracle(x, w, b, dy, device=oracle_on)
    check_all(got, want)
    for g, (exact, _) in zip(got, want):
        # Errors of independent signs: the result's own rounding, and dp's, whose
        # share of a sum is half of its norm at most.
        if M * F * K and exact.numel() > 64:
            off = (g.detach().double().cpu() - exact).norm() / exact.norm()
            assert off < 2 * torch.finfo(dtype).eps / 2 + 64 * 2.0 ** -24, float(off)
    with torch.no_grad():
        assert torch.equal(gated_linear(x, w, b), y)
    return got


@pytest.mark.parametrize("M", [0, 1, 2, 15, 17, 64, 65, 129, 300])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_linear_rows(M, dtype):
    run_linear(M, 72, 80, dtype, seed=M)


@pytest.mark.parametrize("M, K, F", [(0, 8, 8), (5, 0, 8), (5, 8, 0), (0, 0, 0)])
def test_linear_empty(M, K, F):
    run_linear(M, K, F, BF16)
    run_linear(M, K, F, FP32, bias=False)


@pytest.mark.parametrize("K", [1, 7, 8, 31, 64, 203, 520])
@pytest.mark.parametrize("F", [1, 16, 33, 129, 264])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_linear_widths(K, F, dtype):
    run_linear(70, K, F, dtype, bias=F != 16, seed=K + F)


# rows shorter than a load, in loops long enough to leave their ends
@pytest.mark.parametrize("K", [1, 3, 4, 5, 9])
@pytest.mark.parametrize("F", [1, 2, 3, 5])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_linear_narrow(K, F, dtype):
    run_linear(700, K, F, dtype, seed=K + F)


@pytest.mark.parametrize("M, K, F", [(1500, 512, 1024), (5000, 96, 64), (33, 2048, 512), (8200, 136, 1032), (8195, 67, 1029)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_linear_larger(M, K, F, dtype):
    run_linear(M, K, F, dtype, seed=M)


# every tile that the four products are cut into, whole and past its edges, with
# and without splits, in 16-byte pieces and element by element
# (as far as these sizes reach: test_gated_cuts.py has one for every kernel)
@pytest.mark.parametrize("M, K, F", [
    (4096, 2048, 4096), (5000, 1048, 2056), (5001, 1043, 2055), (8200, 1032, 2056), (8201, 1029, 2054),
    (10240, 1024, 2048), (16384, 520, 136), (16380, 517, 129), (1500, 136, 2048), (1501, 203, 2045),
    (300, 1024, 2048), (4090, 67, 2041), (20480, 67, 1024), (4096, 1024, 64)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_linear_tiles(M, K, F, dtype):
    run_linear(M, K, F, dtype, seed=K, oracle_on="cuda")


def test_linear_offsets_past_32_bits():
    few, times, K, F = 64, 65600, 520, 16  # 2.2e9 elements
    x, dy = rand(few, K, dtype=BF16).repeat(times, 1), rand(few, F, seed=1, dtype=BF16).repeat(times, 1)
    w, b = rand(2 * F, K, seed=2, dtype=BF16, scale=K ** -0.5), rand(2 * F, seed=3, dtype=BF16)
    ins = leaves(x, w, b)
    y = gated_linear(x, w, b)
    dx, dw, db = torch.autograd.grad([y], ins, [dy])
    want = linear_oracle(x[:few], w, b, dy[:few])
    for i in (0, times // 2, times - 1):
        rows = slice(i * few, (i + 1) * few)
        check_all([y[rows], dx[rows]], want[:2])
    # Sums over `times` equal blocks of rows: dp is rounded alike in each, as in
    # run_linear, and the additions' roundings have independent signs.
    for got, (exact, _) in zip((dw, db), want[2:]):
        off = (got.double().cpu() / times - exact).norm() / exact.norm()
        assert off < 2 * torch.finfo(BF16).eps / 2 + (few * times) ** 0.5 * 2.0 ** -24, float(off)


def test_linear_shapes_strides_and_partial_gradients():
    run_linear(24, 40, 32, BF16, shape=(2, 3, 4, 40))
    x, w = rand(60, 9, 50, dtype=BF16)[::3, 2, 3:43], rand(40, 48, seed=1, dtype=BF16).t()
    b = rand(48, seed=2, dtype=BF16)
    assert torch.equal(gated_linear(x, w, b), gated_linear(x.contiguous(), w.contiguous(), b))
    dy = rand(20, 24, seed=3, dtype=BF16)
    want = linear_oracle(x, w, b, dy)
    for pick in ([0], [1], [2], [0, 2]):
        ins = [x.detach().contiguous(), w.detach().contiguous(), b.detach()]
        for i in pick:
            ins[i].requires_grad_(True)
        y = gated_linear(*ins)
        check_all(torch.autograd.grad([y], [ins[i] for i in pick], [dy]), [want[1 + i] for i in pick])
    # rows that start on odd elements
    flat = rand(21 * 40 + 1, dtype=BF16)
    x = flat[1:].view(21, 40)
    assert torch.equal(gated_linear(x, w), gated_linear(x.clone(), w))


def test_linear_keeps_rows_apart():
    x, w = rand(70, 96, dtype=BF16), rand(64, 96, seed=1, dtype=BF16)
    clean = gated_linear(x, w)
    bad = x.clone()
    bad[5, 3], bad[69, 0] = float("nan"), float("inf")
    y = gated_linear(bad, w)
    same = [i for i in range(70) if i not in (5, 69)]
    assert torch.equal(y[same], clean[same]) and y[5].isnan().all()


# ----------------------------------------------------- refusals, streams, graphs
def i32(*shape, device="cuda"):
    return torch.zeros(*shape, dtype=torch.int32, device=device)


@pytest.mark.parametrize("call, error", [
    (lambda: layer_norm(rand(3, 8).half(), rand(8).half()), TypeError),
    (lambda: layer_norm(rand(3, 8), rand(8, dtype=BF16)), TypeError),
    (lambda: layer_norm(rand(3, 8), rand(8).cpu()), RuntimeError),
    (lambda: layer_norm(rand(3, 8), rand(8), residual=rand(3, 8).cpu()), RuntimeError),
    (lambda: layer_norm(rand(3, 8), rand(8), residual=rand(1, 8)), ValueError),
    (lambda: layer_norm(rand(3, 8), rand(7)), ValueError),
    (lambda: layer_norm(rand(3, 8), rand(8), rand(7)), ValueError),
    (lambda: layer_norm(rand(3, 0), rand(0)), ValueError),
    (lambda: layer_norm(rand(1)[0], rand(1)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 6).half()), TypeError),
    (lambda: gated_recurrence(rand(2, 3, 6).double()), TypeError),
    (lambda: gated_recurrence(rand(2, 3, 7)), ValueError),
    (lambda: gated_recurrence(rand(3, 6)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 6), rand(3, 3)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 6), rand(3, 2, dtype=BF16)), TypeError),
    (lambda: gated_recurrence(rand(2, 3, 6), rand(3, 2).cpu()), RuntimeError),
    (lambda: gated_recurrence(rand(2, 3, 6), None, i32(2)), ValueError),
    (lambda: gated_recurrence(rand(2, 3, 6), None, i32(3).long()), TypeError),
    (lambda: gated_recurrence(rand(2, 3, 6), None, i32(3, device="cpu")), RuntimeError),
    (lambda: gated_linear(rand(3, 8), rand(4, 8).cpu()), RuntimeError),
    (lambda: gated_linear(rand(3, 8).half(), rand(4, 8).half()), TypeError),
    (lambda: gated_linear(rand(3, 8), rand(4, 8, dtype=BF16)), TypeError),
    (lambda: gated_linear(rand(3, 8), rand(5, 8)), ValueError),
    (lambda: gated_linear(rand(3, 8), rand(4, 7)), ValueError),
    (lambda: gated_linear(rand(3, 8), rand(4, 8), rand(2)), ValueError),
    (lambda: gated_linear(rand(1)[0], rand(4, 1)), ValueError),
])
def test_gpu_refusals(call, error):
    with pytest.raises(error):
        call()


def test_second_derivatives_are_refused():
    x, w = rand(3, 8).requires_grad_(True), rand(8, seed=1)
    for op in (lambda: layer_norm(x, w), lambda: gated_linear(x, rand(6, 8, seed=2)),
               lambda: gated_recurrence(x.view(1, 1, 24))[0]):
        g = torch.autograd.grad(op().square().sum(), x, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    x, w = rand(3, 8), rand(8, seed=1)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for op in (lambda: layer_norm(d, w), lambda: gated_linear(d, rand(6, 8, seed=2)),
                   lambda: gated_recurrence(d.view(1, 1, 24))):
            with pytest.raises(NotImplementedError):
                op()


def test_a_graph_is_walked_once_unless_retained():
    p = block_inputs(FP32)
    x, w, g = p["x"], p["wl"], p["wg"]
    for op in (lambda: layer_norm(x, p["w1"]), lambda: gated_linear(x, w),
               lambda: gated_recurrence(x @ g.t())[0]):
        y = op()
        first = torch.autograd.grad(y, x, p["dy"], retain_graph=True)[0]
        again = torch.autograd.grad(y, x, p["dy"])[0]
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, x, p["dy"])


def test_saved_tensors_may_live_elsewhere_or_be_computed_again():
    from torch.utils.checkpoint import checkpoint
    p = block_inputs(BF16)
    want = block(p, lambda n: n @ p["wg"].t())
    with torch.autograd.graph.save_on_cpu():
        got = block(p, lambda n: n @ p["wg"].t())
    for a, b in zip(got, want):
        assert torch.equal(a, b)

    def run(x):
        y, hT = gated_recurrence(layer_norm(x, p["w1"], p["b1"]) @ p["wg"].t(), p["h0"])
        return gated_linear(y, p["wl"], p["bl"])

    a = torch.autograd.grad(run(p["x"]), [p["x"], p["wl"]], p["dy"])
    b = torch.autograd.grad(checkpoint(run, p["x"], use_reentrant=False), [p["x"], p["wl"]], p["dy"])
    assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_saved_inputs_changed_in_place_are_noticed():
    x, w, g = rand(3, 8), rand(8, seed=1), rand(2, 3, 12, seed=2)
    lengths = torch.tensor([2, 1, 0], dtype=torch.int32, device="cuda")
    for op, change in ((lambda: layer_norm(x, w.requires_grad_(True)), x),
                       (lambda: gated_linear(x, rand(6, 8, seed=2).requires_grad_(True)), x),
                       (lambda: gated_recurrence(g.requires_grad_(True), None, lengths)[0], lengths)):
        y = op()
        change.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_one_tensor_in_two_places():
    x, w = rand(5, 40), rand(40, seed=1)
    ins = leaves(x, w)
    y, s = layer_norm(x, w, w, residual=x)
    assert torch.equal(s, 2 * x)
    dy, ds = rand(5, 40, seed=2), rand(5, 40, seed=3)
    dx, dw = torch.autograd.grad([y, s], ins, [dy, ds])
    want = norm_oracle(x, w, w, x, dy, ds)
    check_all([y, s], want[:2])
    check_all([dx, dw], [(2 * want[2][0], 2 * want[2][1]),
                         (want[3][0] + want[4][0], want[3][1] + want[4][1])])
    w1 = rand(40, seed=4)  # one axis alone
    assert torch.equal(layer_norm(x[0], w1), layer_norm(x[:1], w1)[0])
    w2 = rand(6, 40, seed=5)
    assert torch.equal(gated_linear(x[0], w2), gated_linear(x[:1], w2)[0])


def block(p, gates_of):
    """The three as a residual block uses them; returns outputs and gradients."""
    n = layer_norm(p["x"], p["w1"], p["b1"])
    y, hT = gated_recurrence(gates_of(n), p["h0"])
    n2, s = layer_norm(y, p["w2"], p["b2"], residual=p["x"])
    out = gated_linear(n2, p["wl"], p["bl"]) + s
    ins = [p[k] for k in ("x", "w1", "b1", "wg", "h0", "w2", "b2", "wl", "bl")]
    return [out, hT] + list(torch.autograd.grad([out, hT], ins, [p["dy"], p["dh"]]))


def block_inputs(dtype, T=33, B=5, H=64, seed=0):
    p = {"x": rand(T, B, H, seed=seed, dtype=dtype), "wg": rand(3 * H, H, seed=seed + 1, dtype=dtype, scale=H ** -0.5),
         "h0": rand(B, H, seed=seed + 2), "wl": rand(2 * H, H, seed=seed + 3, dtype=dtype, scale=H ** -0.5),
         "bl": rand(2 * H, seed=seed + 4, dtype=dtype)}
    for i, k in enumerate(("w1", "b1", "w2", "b2")):
        p[k] = rand(H, seed=seed + 5 + i, dtype=dtype, scale=0.1, shift=float(k[0] == "w"))
    leaves(*p.values())
    p["dy"], p["dh"] = rand(T, B, H, seed=seed + 9, dtype=dtype), rand(B, H, seed=seed + 10)
    return p


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_together_against_64_bits(dtype):
    p = block_inputs(dtype)
    got = block(p, lambda n: n @ p["wg"].t())
    q = {k: v.detach().double().cpu() for k, v in p.items()}
    leaves(*[q[k] for k in q if k not in ("dy", "dh")])
    want = block(q, lambda n: n @ q["wg"].t())
    # five roundings to the type lie on the longest path, each of half a step, and
    # the norms and gates carry them on no larger than the values' own norm
    bound = 5 * torch.finfo(dtype).eps / 2 * 2 + 256 * 2.0 ** -24
    for i, (g, w) in enumerate(zip(got, want)):
        off = (g.detach().double().cpu() - w).norm() / w.norm()
        assert off < bound, (i, float(off))


def test_streams():
    p, q = block_inputs(BF16), block_inputs(BF16, seed=50)
    want = [block(s, lambda n, s=s: n @ s["wg"].t()) for s in (p, q)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for i, s in enumerate((p, q)):
            with torch.cuda.stream(streams[i]):
                got[i] = block(s, lambda n, s=s: n @ s["wg"].t())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)


def test_two_graphs_replayed():
    cases = [block_inputs(BF16), block_inputs(BF16, T=300, B=2, seed=50)]
    graphs, outs = [], []
    for p in cases:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(p, lambda n: n @ p["wg"].t())
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(block(p, lambda n: n @ p["wg"].t()))
        graphs.append(graph)
    for turn in range(3):
        for i, p in enumerate(cases):
            with torch.no_grad():
                p["x"].copy_(rand(*p["x"].shape, seed=90 + turn, dtype=BF16))
                p["dy"].copy_(rand(*p["dy"].shape, seed=70 + turn, dtype=BF16))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for p, out in zip(cases, outs):
            for a, b in zip(out, block(p, lambda n: n @ p["wg"].t())):
                assert torch.equal(a, b)


def test_capture_over_a_live_eager_graph_is_refused():
    x, w = rand(4, 16), rand(16, seed=1).requires_grad_(True)
    alive = layer_norm(x, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            layer_norm(x, w)
    del alive
    y = layer_norm(x, w)
    assert torch.equal(torch.autograd.grad([y], [w], [torch.ones_like(y)])[0].isfinite(),
                       torch.ones(16, dtype=torch.bool, device="cuda"))
