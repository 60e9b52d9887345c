"""Layer norm, linear layers with a fused epilogue, and the gated linear recurrence.

The three operators a sequence or volume model puts around its convolutions, as
measurable cases: ``listed()`` names fixed ones, ``draw()`` gives more of the same
ranges, ``prepare()`` makes a case's inputs on the GPU, ``run()`` makes one pass (the
framework's operators where ``own`` is true, else their plain form in elementary torch
operations), ``exact()`` gives the same outputs from the definitions in float64.

* layer norm over the last dimension: y = (x - mean) / sqrt(var + eps) * w + b;
* linear: y = act(x W^T + b) + r, act one of none, gelu (exact) and silu;
* gated recurrence along one axis: f = sigmoid(g), h_t = f_t h_{t-1} + (1 - f_t) x_t.

A ``train`` pass returns the outputs and every gradient; a ``forward`` pass the outputs.
"""

import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _norm(name, rows, width, dtype, way):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "way": way}


def _linear(name, rows, inner, outer, dtype, way, act, residual):
    return {"name": name, "op": "linear", "rows": rows, "inner": inner, "outer": outer,
            "dtype": dtype, "way": way, "act": act, "residual": residual}


def _recurrence(name, batch, channels, steps, space, layout, dtype, way):
    return {"name": name, "op": "recurrence", "batch": batch, "channels": channels,
            "steps": steps, "space": space, "layout": layout, "dtype": dtype, "way": way}


def listed():
    return [
        # one decoding step of eight sequences: nothing but latency
        _norm("norm_step", 8, 1024, "bf16", "forward"),
        # the 64-channel channels-last output of the benchmark's Conv4d layer, [16, 64, 16^4]
        _norm("norm_volume", 1048576, 64, "bf16", "train"),
        # the wide rows of a large model's training step
        _norm("norm_wide", 16384, 4096, "bf16", "train"),
        # odd rows of an odd width: no 16-byte vectors, a ragged last block
        _norm("norm_odd", 4097, 771, "f32", "train"),
        # four sequences' next tokens through an expanding layer: the weights are the traffic
        _linear("linear_token", 4, 1024, 4096, "bf16", "forward", "gelu", False),
        # the pointwise expansion after the benchmark's Conv4d layer: many rows, thin matrices
        _linear("linear_volume", 1048576, 64, 256, "bf16", "train", "gelu", False),
        # the expanding layer of a model's training step
        _linear("linear_train", 16384, 1024, 4096, "bf16", "train", "gelu", False),
        # the contracting layer over a long prompt, added to the residual stream
        _linear("linear_residual", 65536, 4096, 1024, "bf16", "forward", "none", True),
        # full precision at odd sizes: rows that no bulk copy can start on
        _linear("linear_odd", 1999, 771, 1283, "f32", "train", "silu", True),
        # one decoding step of 64 sequences from their kept states
        _recurrence("recurrence_step", 64, 1024, 1, 1, "tokens", "bf16", "forward"),
        # one long sequence: few columns, so the long axis has to be shared out
        _recurrence("recurrence_long", 1, 512, 65536, 1, "tokens", "bf16", "train"),
        # the time axis of a channels-first video volume, an odd number of frames
        _recurrence("recurrence_video", 8, 64, 33, 45, "volume", "f32", "train"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], uniform in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5))))


def draw(rng):
    op = rng.choice(["norm", "linear", "recurrence"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    way = rng.choice(["forward", "train"])
    if op == "norm":
        width = _spread(rng, 16, 8192)
        if rng.random() < 0.5:
            width = max(16, width // 16 * 16)
        rows = _spread(rng, 1, max(1, min(1048576, 67108864 // width)))
        case = _norm("", rows, width, dtype, way)
    elif op == "linear":
        inner, outer = _spread(rng, 16, 8192), _spread(rng, 16, 8192)
        if rng.random() < 0.6:
            inner, outer = max(16, inner // 16 * 16), max(16, outer // 16 * 16)
        passes = 3 if way == "train" else 1
        most = min(1048576, int(400e9 / (2 * inner * outer * passes)), 335544320 // (inner + outer))
        rows = _spread(rng, 1, max(1, most))
        case = _linear("", rows, inner, outer, dtype, way, rng.choice(["none", "gelu", "silu"]),
                       rng.random() < 0.4)
    else:
        layout = rng.choice(["tokens", "tokens", "channels", "volume"])
        batch, channels = _spread(rng, 1, 64), _spread(rng, 8, 2048)
        if rng.random() < 0.5:
            channels = max(8, channels // 8 * 8)
        space = _spread(rng, 2, 64) if layout == "volume" else 1
        area = space * space
        steps = _spread(rng, 1, max(1, min(65536, 33554432 // (batch * channels * area))))
        if batch * channels * area * steps > 33554432:
            batch = max(1, 33554432 // (channels * area * steps))
        if batch * channels * area * steps > 33554432:
            channels = max(8, 33554432 // (batch * area * steps))
        case = _recurrence("", batch, channels, steps, space, layout, dtype, way)
    del case["name"]
    return case


def work(case):
    e, train = BYTES[case["dtype"]], case["way"] == "train"
    if case["op"] == "norm":
        n, c = case["rows"] * case["width"], case["width"]
        return {"bytes": (4 if train else 2) * n * e + (4 if train else 2) * c * e,
                "flops": (20 if train else 8) * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        read = m * k + n * k + n + (m * n if case["residual"] else 0) + (m * n if train else 0)
        written = m * n + (m * k + n * k + n if train else 0)
        return {"bytes": (read + written) * e, "flops": (6 if train else 2) * m * n * k}
    columns = case["batch"] * case["channels"] * case["space"] ** 2
    n = columns * case["steps"]
    return {"bytes": (6 if train else 3) * n * e + (4 if train else 2) * columns * 4,
            "flops": (24 if train else 10) * n}


def _recurrence_shape(case):
    b, c, t, s = case["batch"], case["channels"], case["steps"], case["space"]
    if case["layout"] == "tokens":
        return (b, t, c), 1
    if case["layout"] == "channels":
        return (b, c, t), 2
    return (b, c, t, s, s), 2


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, train = DTYPES[case["dtype"]], case["way"] == "train"

    def normal(shape, scale=1.0, mean=0.0, kind=dtype, grad=train):
        t = torch.randn(shape, device="cuda", generator=generator).mul_(scale).add_(mean).to(kind)
        return t.requires_grad_() if grad else t

    state = {"case": case}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        state["x"] = normal((rows, width), 1.5, 0.3)
        state["w"] = normal((width,), 0.1, 1.0)
        state["b"] = normal((width,), 0.1)
        if train:
            state["dy"] = normal((rows, width), grad=False)
    elif case["op"] == "linear":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        state["x"] = normal((rows, inner))
        state["w"] = normal((outer, inner), 1.0 / math.sqrt(inner))
        state["b"] = normal((outer,), 0.1)
        state["r"] = normal((rows, outer)) if case["residual"] else None
        if train:
            state["dy"] = normal((rows, outer), grad=False)
    else:
        shape, dim = _recurrence_shape(case)
        start = shape[:dim] + shape[dim + 1:]
        state["x"] = normal(shape)
        state["g"] = normal(shape, 1.5, 2.0)
        state["h0"] = normal(start, 0.5, kind=torch.float32)
        if train:
            state["dy"] = normal(shape, grad=False)
            state["dlast"] = normal(start, kind=torch.float32, grad=False)
    return state


# ---- the framework's operators ---------------------------------------------------------


def _package():
    root = str(Path(__file__).resolve().parent.parent / "torch-convnd_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import torch_convnd

    return torch_convnd


def _run_own(state):
    convnd = _package()
    case = state["case"]
    train = case["way"] == "train"
    if case["op"] == "norm":
        y = convnd.layer_norm(state["x"], state["w"], state["b"], EPS)
        if not train:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, (state["x"], state["w"], state["b"]), state["dy"])]
    if case["op"] == "linear":
        act = None if case["act"] == "none" else case["act"]
        y = convnd.linear(state["x"], state["w"], state["b"], activation=act, residual=state["r"])
        if not train:
            return [y]
        wanted = [state["x"], state["w"], state["b"]]
        if state["r"] is not None:
            wanted.append(state["r"])
        return [y.detach(), *torch.autograd.grad(y, wanted, state["dy"])]
    y, last = convnd.gated_recurrence(state["x"], state["g"], state["h0"],
                                      dim=_recurrence_shape(case)[1])
    if not train:
        return [y, last]
    return [y.detach(), last.detach(),
            *torch.autograd.grad((y, last), (state["x"], state["g"], state["h0"]),
                                 (state["dy"], state["dlast"]))]


# ---- plain forms: elementary operations in 32 bits, rounded once -----------------------


def _plain_norm(state):
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    out = state["x"].dtype
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    unit = centred * rstd
    y = (unit * w + b).to(out)
    if state["case"]["way"] != "train":
        return [y]
    dy = state["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return [y, dx.to(out), (dy * unit).sum(0).to(out), dy.sum(0).to(out)]


def _plain_activation(z, act):
    """(act(z), act'(z))."""
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    return z, None


def _plain_linear(state):
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    out, act = state["x"].dtype, state["case"]["act"]
    y, slope = _plain_activation(x @ w.t() + b, act)
    if state["r"] is not None:
        y = y + state["r"].float()
    y = y.to(out)
    if state["case"]["way"] != "train":
        return [y]
    dy = state["dy"].float()
    dz = dy if slope is None else dy * slope
    grads = [(dz @ w).to(out), (dz.t() @ x).to(out), dz.sum(0).to(out)]
    return [y, *grads] + ([state["dy"]] if state["r"] is not None else [])


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t (h_{-1} = 0) along dimension 1, by pairs: the states at odd
    steps are the same recurrence over half as many steps."""
    steps = a.shape[1]
    if steps == 1:
        return b
    even = 2 * (steps // 2)
    odd = _scan(a[:, 1:even:2] * a[:, 0:even:2],
                a[:, 1:even:2] * b[:, 0:even:2] + b[:, 1:even:2])
    h = torch.empty_like(b)
    h[:, 0] = b[:, 0]
    h[:, 1:even:2] = odd
    h[:, 2::2] = a[:, 2::2] * odd[:, : (steps - 1) // 2] + b[:, 2::2]
    return h


def _plain_recurrence(state):
    dim = _recurrence_shape(state["case"])[1]
    out = state["x"].dtype
    x, g = (state[k].float().movedim(dim, 1) for k in ("x", "g"))
    h0 = state["h0"].unsqueeze(1)
    f = 1.0 / (1.0 + torch.exp(-g))
    keep = 1.0 / (1.0 + torch.exp(g))
    b = keep * x
    b = torch.cat([b[:, :1] + f[:, :1] * h0, b[:, 1:]], 1)
    h = _scan(f, b)
    y, last = h.movedim(1, dim).to(out).contiguous(), h[:, -1].contiguous()
    if state["case"]["way"] != "train":
        return [y, last]
    dh = state["dy"].float().movedim(dim, 1)
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + state["dlast"].unsqueeze(1)], 1)
    after = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], 1)  # what step t passes to t + 1
    total = _scan(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([h0, h[:, :-1]], 1)
    dx = total * keep
    dg = total * (before - x) * f * keep
    return [y, last, dx.movedim(1, dim).to(out).contiguous(),
            dg.movedim(1, dim).to(out).contiguous(), (total[:, 0] * f[:, 0]).contiguous()]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "linear": _plain_linear,
                "recurrence": _plain_recurrence}[state["case"]["op"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------


def _exact_norm(state):
    x, w, b = (state[k].double() for k in ("x", "w", "b"))
    width = x.shape[1]
    variance, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    deviation = torch.sqrt(variance + EPS)
    y = torch.addcmul(b, (x - mean) / deviation, w)
    if state["case"]["way"] != "train":
        return [y]
    dy = state["dy"].double()
    z = (x - mean) / deviation
    dz = dy * w
    dx = (width * dz - dz.sum(1, keepdim=True) - z * (dz * z).sum(1, keepdim=True)) / (width * deviation)
    return [y, dx, torch.einsum("rc,rc->c", dy, z), torch.einsum("rc->c", dy)]


def _exact_linear(state):
    x, w, b = (state[k].double() for k in ("x", "w", "b"))
    act = state["case"]["act"]
    z = torch.addmm(b, x, w.t())
    if act == "gelu":
        y = torch.special.ndtr(z) * z
    elif act == "silu":
        y = torch.sigmoid(z) * z
    else:
        y = z
    if state["r"] is not None:
        y = y + state["r"].double()
    if state["case"]["way"] != "train":
        return [y]
    dz = state["dy"].double()
    if act == "gelu":
        dz = dz * (torch.special.ndtr(z) + z / math.sqrt(2 * math.pi) * torch.exp(-z.square() / 2))
    elif act == "silu":
        s = torch.sigmoid(z)
        dz = dz * (s + z * s * (1 - s))
    got = [y, torch.mm(dz, w), torch.mm(dz.t(), x), dz.sum(0)]
    return got + ([state["dy"].double()] if state["r"] is not None else [])


def _exact_recurrence(state):
    case = state["case"]
    dim = _recurrence_shape(case)[1]
    steps = case["steps"]
    x, g = (state[k].double().movedim(dim, 0).contiguous() for k in ("x", "g"))
    f = torch.sigmoid(g)
    h = torch.empty_like(x)
    carried = state["h0"].double()
    for t in range(steps):
        carried = torch.lerp(x[t], carried, f[t])
        h[t] = carried
    got = [h.movedim(0, dim).contiguous(), carried]
    if case["way"] != "train":
        return got
    dy = state["dy"].double().movedim(dim, 0)
    flow = state["dlast"].double()
    dx, dg = torch.empty_like(x), torch.empty_like(x)
    for t in reversed(range(steps)):
        flow = flow + dy[t]
        before = h[t - 1] if t else state["h0"].double()
        dx[t] = flow * (1 - f[t])
        dg[t] = flow * (before - x[t]) * f[t] * (1 - f[t])
        flow = flow * f[t]
    return got + [dx.movedim(0, dim).contiguous(), dg.movedim(0, dim).contiguous(), flow]


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "linear": _exact_linear,
                "recurrence": _exact_recurrence}[case["op"]](state)
