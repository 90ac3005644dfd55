"""Workloads of the operators behind the gated recurrent core.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as the framework's kernel:

* ``norm``  layer norm over the last axis, optionally of a residual sum,
* ``rec``   gated linear recurrence over time, state carried in and out,
* ``glu``   gated linear unit: two projections, the activation and the product.

A case is a dict of an operator, its sizes, type ("bf16" or "fp32") and whether it trains: a training case runs forward and
backward and returns every gradient, the others run without gradients.
"""

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # one control step of 64 batched environments: a row each, latency alone counts
        {"name": "norm-step", "op": "norm", "rows": 64, "dim": 512, "dtype": "bf16", "residual": True, "train": False},
        # the flagship learner batch: 256 sequences of 80 steps at hidden size 512
        {"name": "norm-train", "op": "norm", "rows": 20480, "dim": 512, "dtype": "bf16", "residual": True, "train": True},
        # odd rows and an odd width in full precision
        {"name": "norm-train-odd", "op": "norm", "rows": 4099, "dim": 771, "dtype": "fp32", "residual": False, "train": True},
        # many wide rows: bandwidth alone counts
        {"name": "norm-train-wide", "op": "norm", "rows": 32768, "dim": 4096, "dtype": "bf16", "residual": True, "train": True},
        # one control step of 64 batched environments
        {"name": "rec-step", "op": "rec", "steps": 1, "batch": 64, "hidden": 512, "dtype": "bf16", "lengths": False, "train": False},
        # the flagship learner batch
        {"name": "rec-train", "op": "rec", "steps": 80, "batch": 256, "hidden": 512, "dtype": "bf16", "lengths": False, "train": True},
        # a padded batch of ragged sequences, odd everywhere
        {"name": "rec-train-odd", "op": "rec", "steps": 121, "batch": 37, "hidden": 203, "dtype": "fp32", "lengths": True, "train": True},
        # few long sequences: too few channels to fill the card without splitting time
        {"name": "rec-train-long", "op": "rec", "steps": 16384, "batch": 4, "hidden": 512, "dtype": "bf16", "lengths": False, "train": True},
        # one control step of 64 batched environments: the weights are read for a few rows
        {"name": "glu-step", "op": "glu", "rows": 64, "dim": 512, "width": 1024, "dtype": "bf16", "bias": True, "train": False},
        # the flagship learner batch
        {"name": "glu-train", "op": "glu", "rows": 20480, "dim": 512, "width": 1024, "dtype": "bf16", "bias": True, "train": True},
        # odd everywhere, full precision
        {"name": "glu-train-odd", "op": "glu", "rows": 1531, "dim": 203, "width": 333, "dtype": "fp32", "bias": True, "train": True},
        # a wide network on a large batch: the matrix cores alone count
        {"name": "glu-train-large", "op": "glu", "rows": 16384, "dim": 2048, "width": 4096, "dtype": "bf16", "bias": False, "train": True},
    ]


def _spread(rng, low, high):
    """A whole number spread over its logarithm; half of them multiples of eight where that fits."""
    n = round(low * (high / low) ** rng.random())
    return min(high, max(8, n // 8 * 8)) if n > 16 and rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["norm", "rec", "glu"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp32"]), "train": rng.random() < 0.6}
    if op == "norm":
        case["dim"] = _spread(rng, 16, 8192)
        case["rows"] = _spread(rng, 1, min(32768, (1 << 26) // case["dim"]))
        case["residual"] = rng.random() < 0.5
    elif op == "rec":
        case["hidden"] = _spread(rng, 16, 1024)
        case["batch"] = _spread(rng, 1, 512)
        case["steps"] = _spread(rng, 1, min(16384, (1 << 24) // (case["hidden"] * case["batch"])))
        case["lengths"] = rng.random() < 0.4
    else:
        case["dim"] = _spread(rng, 16, 2048)
        case["width"] = _spread(rng, 16, 4096)
        case["rows"] = _spread(rng, 1, 16384 if case["dtype"] == "bf16" else 4096)
        case["bias"] = rng.random() < 0.5
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPE[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    s = {"case": case}
    if case["op"] == "norm":
        n, d = case["rows"], case["dim"]
        s["x"] = normal(n, d, scale=0.7, shift=0.2)
        s["residual"] = normal(n, d) if case["residual"] else None
        s["weight"] = normal(d, scale=0.1, shift=1.0)
        s["bias"] = normal(d, scale=0.1)
        s["leaves"] = [s["x"], s["weight"], s["bias"]] + ([s["residual"]] if case["residual"] else [])
        s["dy"] = normal(n, d)
        s["ds"] = normal(n, d) if case["residual"] else None
    elif case["op"] == "rec":
        t, b, h = case["steps"], case["batch"], case["hidden"]
        gates = torch.randn(t, b, 3, h, generator=gen, device="cuda")
        gates[:, :, 0] = gates[:, :, 0] * 1.5 + 2.0  # forget gates that remember over tens of steps
        s["gates"] = gates.view(t, b, 3 * h).to(dt)
        s["h0"] = normal(b, h, scale=0.5, dtype=torch.float32)
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32) if case["lengths"] else None
        s["leaves"] = [s["gates"], s["h0"]]
        s["dy"] = normal(t, b, h)
        s["dh"] = normal(b, h, dtype=torch.float32)
    else:
        n, k, f = case["rows"], case["dim"], case["width"]
        s["x"] = normal(n, k)
        s["weight"] = ((torch.rand(2 * f, k, generator=gen, device="cuda") * 2 - 1) / k**0.5).to(dt)
        s["bias"] = normal(2 * f, scale=0.1) if case["bias"] else None
        s["leaves"] = [s["x"], s["weight"]] + ([s["bias"]] if case["bias"] else [])
        s["dy"] = normal(n, f)
    if case["train"]:
        for p in s["leaves"]:
            p.requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    if own:
        return OWN[case["op"]](state, case["train"])
    with torch.no_grad():
        return PLAIN[case["op"]](state, case["train"])


# ---------------------------------------------------------------- the framework's calls
def _grads(state, outputs, seeds):
    grads = torch.autograd.grad(outputs, state["leaves"], seeds)
    return [o.detach() for o in outputs] + list(grads)


def own_norm(s, train):
    from pytorch_r2d2_dpg_amd.ops.layer_norm import layer_norm

    with torch.set_grad_enabled(train):
        out = layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, residual=s["residual"])
    outputs = list(out) if s["residual"] is not None else [out]
    return _grads(s, outputs, [s["dy"], s["ds"]][: len(outputs)]) if train else outputs


def own_rec(s, train):
    from pytorch_r2d2_dpg_amd.ops.gated_recurrence import gated_recurrence

    with torch.set_grad_enabled(train):
        outputs = list(gated_recurrence(s["gates"], s["h0"], lengths=s["lengths"]))
    return _grads(s, outputs, [s["dy"], s["dh"]]) if train else outputs


def own_glu(s, train):
    from pytorch_r2d2_dpg_amd.ops.gated_linear import gated_linear

    with torch.set_grad_enabled(train):
        outputs = [gated_linear(s["x"], s["weight"], s["bias"])]
    return _grads(s, outputs, [s["dy"]]) if train else outputs


OWN = {"norm": own_norm, "rec": own_rec, "glu": own_glu}


# ---------------------------------------------------------------- the plain forms
def plain_norm(s, train):
    dt = s["x"].dtype
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    w = s["weight"].float()
    c = x - x.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = c * rstd
    out = [(n * w + s["bias"].float()).to(dt)]
    if s["residual"] is not None:
        out.append(x.to(dt))
    if train:
        dy = s["dy"].float()
        g = dy * w
        dx = (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True)) * rstd
        if s["residual"] is not None:
            dx = dx + s["ds"].float()
        out += [dx.to(dt), (dy * n).sum(0).to(dt), dy.sum(0).to(dt)]
        if s["residual"] is not None:
            out.append(dx.to(dt))
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t over the first axis, by doubling: each pass joins runs twice as long."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], a[d:] * b[:-d] + b[d:]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def plain_rec(s, train):
    dt = s["gates"].dtype
    f, v, o = s["gates"].float().chunk(3, dim=-1)
    steps = f.shape[0]
    a, keep = torch.sigmoid(f), torch.sigmoid(-f)
    gate = torch.sigmoid(o)
    if s["lengths"] is not None:
        real = (torch.arange(steps, device=f.device)[:, None] < s["lengths"][None, :])[:, :, None]
        a, keep = torch.where(real, a, 1.0), torch.where(real, keep, 0.0)
        o = torch.where(real, o, 0.0)
    b = keep * v
    b[0] += a[0] * s["h0"]
    h = _scan(a, b)
    out = [(h * o * gate).to(dt), h[-1].clone()]
    if train:
        dy = s["dy"].float()
        if s["lengths"] is not None:
            dy = torch.where(real, dy, 0.0)
        p = dy * o * gate
        p[-1] += s["dh"]
        back = torch.cat([torch.zeros_like(a[:1]), a[1:].flip(0)])
        g = _scan(back, p.flip(0)).flip(0)
        before = torch.cat([s["h0"][None], h[:-1]])
        df = g * (before - v) * a * keep
        do = dy * h * (gate + o * gate * (1 - gate))
        out += [torch.cat([df, g * keep, do], dim=-1).to(dt), a[0] * g[0]]
    return out


def plain_glu(s, train):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    p = x @ w.t()
    if s["bias"] is not None:
        p = p + s["bias"].float()
    g, u = p.chunk(2, dim=-1)
    gate = torch.sigmoid(g)
    out = [(g * gate * u).to(dt)]
    if train:
        dy = s["dy"].float()
        dp = torch.cat([dy * u * (gate + g * gate * (1 - gate)), dy * g * gate], dim=-1)
        out += [(dp @ w).to(dt), (dp.t() @ x).to(dt)]
        if s["bias"] is not None:
            out.append(dp.sum(0).to(dt))
    return out


PLAIN = {"norm": plain_norm, "rec": plain_rec, "glu": plain_glu}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        streams = 4 if case["residual"] else 2  # x, y and with a residual r and s
        flops = 8 * n
        if case["train"]:
            streams += 3 if case["residual"] else 2  # dy, dx and ds; a residual's gradient is x's own
            flops += 14 * n
        return {"bytes": streams * n * e + 4 * case["dim"] * e, "flops": flops}
    if case["op"] == "rec":
        n, state = case["steps"] * case["batch"] * case["hidden"], case["batch"] * case["hidden"]
        streams, states, flops = 4, 2, 14 * n  # gates and y; h0 and hT
        if case["train"]:
            streams, states, flops = 8, 4, 44 * n  # dy and the gates' gradients too
        return {"bytes": streams * n * e + states * state * 4, "flops": flops}
    m, k, f = case["rows"], case["dim"], case["width"]
    if case["train"]:
        return {"bytes": (2 * m * k + 2 * m * f + 4 * f * k) * e, "flops": 12.0 * m * k * f}
    return {"bytes": (m * k + m * f + 2 * f * k) * e, "flops": 4.0 * m * k * f}


# ---------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    names = [k for k in ("x", "weight", "bias", "residual", "gates", "h0") if s.get(k) is not None]
    d = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names}
    with torch.set_grad_enabled(case["train"]):
        outputs, seeds = DEFINED[case["op"]](s, d)
    if not case["train"]:
        return outputs
    leaves = [next(d[k] for k in names if s[k] is p) for p in s["leaves"]]
    grads = torch.autograd.grad(outputs, leaves, [x.double() for x in seeds])
    return [o.detach() for o in outputs] + list(grads)


def defined_norm(s, d):
    x = d["x"] + d["residual"] if "residual" in d else d["x"]
    var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * d["weight"] + d["bias"]
    return ([y, x], [s["dy"], s["ds"]]) if "residual" in d else ([y], [s["dy"]])


def defined_rec(s, d):
    f, v, o = d["gates"].chunk(3, dim=-1)
    h, ys = d["h0"], []
    lengths = s["lengths"].tolist() if s["lengths"] is not None else None
    for t in range(f.shape[0]):
        a = 1 / (1 + torch.exp(-f[t]))
        new = a * h + v[t] / (1 + torch.exp(f[t]))
        y = new * o[t] / (1 + torch.exp(-o[t]))
        if lengths is not None:
            real = torch.tensor([t < n for n in lengths], device=h.device)[:, None]
            new, y = torch.where(real, new, h), torch.where(real, y, 0.0)
        h = new
        ys.append(y)
    return [torch.stack(ys), h + 0], [s["dy"], s["dh"]]


def defined_glu(s, d):
    width = s["case"]["width"]
    g, u = d["x"] @ d["weight"][:width].t(), d["x"] @ d["weight"][width:].t()
    if "bias" in d:
        g, u = g + d["bias"][:width], u + d["bias"][width:]
    return [g / (1 + torch.exp(-g)) * u], [s["dy"]]


DEFINED = {"norm": defined_norm, "rec": defined_rec, "glu": defined_glu}
