"""layer_norm, linear and gated_recurrence against plain float64 implementations.

Tolerances. An output of type T is one rounding of a float32 (float64) value, so it may be
off by eps(T) |ref| plus the error of that value, which is bounded per test from the number
of float32 operations behind it (unit roundoff 2^-24; the tensor core truncates, 2^-23, once
per 16 products) times the sum of the absolute terms. A gradient that goes through a value
kept in T (the pre-activation and dz of a 16-bit linear layer) adds eps(T) times the same sum.
"""

from __future__ import annotations

import math
import threading

import pytest
import torch

import torch_convnd

HALF = (torch.bfloat16, torch.float16)
DTYPES = (torch.bfloat16, torch.float16, torch.float32, torch.float64)
gpu = pytest.mark.gpu


def eps(dtype):
    return torch.finfo(dtype).eps


def unit(dtype):
    """Unit roundoff of the sums behind an output of `dtype`."""
    return 2.0**-53 if dtype == torch.float64 else 2.0**-24


def randn(shape, dtype, seed, scale=1.0, mean=0.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(shape, device="cuda", dtype=torch.float64, generator=generator)
    return (t * scale + mean).to(dtype)


def check(got, ref, slack, what):
    """|got - ref| <= eps(type) |ref| + slack, everywhere; NaN and infinities in the same
    places."""
    assert got.shape == ref.shape, what
    g, r = got.double(), ref.double()
    finite = torch.isfinite(r)
    assert torch.equal(torch.isnan(g), torch.isnan(r)), f"{what}: NaN in other places"
    assert torch.equal(g[~finite & ~torch.isnan(r)], r[~finite & ~torch.isnan(r)]), what
    slack = torch.as_tensor(slack, dtype=torch.float64, device=g.device).expand(r.shape)
    allowed = eps(got.dtype) * r.abs() + slack + torch.finfo(got.dtype).tiny
    off = (g - r).abs()[finite] - allowed[finite]
    assert off.numel() == 0 or float(off.max()) <= 0.0, (
        f"{what}: {float(off.max()):.3g} past the bound, worst reference "
        f"{float(r[finite].abs().max()):.3g}")


def double(*tensors, grad=True):
    return [None if t is None else t.detach().double().requires_grad_(grad) for t in tensors]


# ---- layer norm ------------------------------------------------------------------------


def plain_norm(x, w, b, epsilon):
    centred = x - x.mean(-1, keepdim=True)
    u = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + epsilon)
    y = u if w is None else u * w
    return (y if b is None else y + b), u


def norm_case(x, w, b, dy, epsilon=1e-5):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = torch_convnd.layer_norm(*leaves, epsilon)
    wanted = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, wanted, dy)
    xd, wd, bd = double(x, w, b)
    ref, u = plain_norm(xd, wd, bd, epsilon)
    refs = torch.autograd.grad(ref, [t for t in (xd, wd, bd) if t is not None], dy.double())
    width, rows = x.shape[-1], max(1, x.numel() // x.shape[-1])
    # sums of `width` terms in float32: at most width / 32 serial additions and 10 levels; the
    # centred values are as accurate as the mean, 2^-24 of the row's largest value
    ops = (width / 32 + 16) * unit(x.dtype)
    with torch.no_grad():
        xa = xd.abs().amax(-1, keepdim=True)
        rstd = 1 / torch.sqrt(xd.var(-1, unbiased=False, keepdim=True) + epsilon)
        wa = torch.ones((), device=x.device, dtype=torch.float64) if w is None else wd.abs().max()
        du = ops * (xa * rstd + u.abs())  # error of u
        check(y, ref, du * wa + 0, "y")
        g = dy.double().abs().amax(-1, keepdim=True) * wa
        ua = u.abs().amax(-1, keepdim=True)
        slack_dx = rstd * (4 * ops * g * (1 + ua * ua) + 4 * du.amax(-1, keepdim=True) * g * (1 + ua))
        check(grads[0], refs[0], slack_dx, "dx")
        # column sums: at most rows / 64 serial additions and 16 levels beside them
        sums = (rows / 64 + 64) * unit(x.dtype)
        flat_dy, flat_u = dy.double().reshape(-1, width), u.reshape(-1, width)
        i = 1
        if w is not None:
            terms = (flat_dy * flat_u).abs().sum(0)
            extra = (flat_dy.abs() * du.reshape(-1, width)).sum(0)
            check(grads[i], refs[i], sums * terms + extra, "dweight")
            i += 1
        if b is not None:
            check(grads[i], refs[i], sums * flat_dy.abs().sum(0), "dbias")


NORM_WIDTHS = [1, 2, 7, 8, 31, 32, 33, 64, 96, 128, 257, 500, 771, 1024, 1032, 2056, 4096, 8192]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", NORM_WIDTHS)
def test_norm_widths(width, dtype):
    rows = 37 if width > 64 else 1003
    x = randn((rows, width), dtype, 1, 1.5, 0.3)
    norm_case(x, randn((width,), dtype, 2, 0.2, 1.0), randn((width,), dtype, 3),
              randn((rows, width), dtype, 4))


@gpu
@pytest.mark.parametrize("dtype,width", [
    (torch.bfloat16, 16384), (torch.bfloat16, 16392), (torch.float16, 20001),
    (torch.float32, 8196), (torch.float32, 16385), (torch.float64, 5000)])
def test_norm_wide_rows(dtype, width):
    x = randn((9, width), dtype, 1)
    norm_case(x, randn((width,), dtype, 2, 0.2, 1.0), randn((width,), dtype, 3),
              randn((9, width), dtype, 4))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 2, 8, 63, 64, 65, 5000, 100003])
def test_norm_rows(rows, dtype):
    x = randn((rows, 48), dtype, 1)
    norm_case(x, randn((48,), dtype, 2, 0.2, 1.0), randn((48,), dtype, 3),
              randn((rows, 48), dtype, 4))


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("which", ["none", "weight", "bias", "float32"])
def test_norm_parameters(dtype, which):
    x, dy = randn((129, 260), dtype, 1), randn((129, 260), dtype, 4)
    kind = torch.float32 if which == "float32" else dtype
    w = None if which in ("none", "bias") else randn((260,), kind, 2, 0.2, 1.0)
    b = None if which in ("none", "weight") else randn((260,), kind, 3)
    norm_case(x, w, b, dy)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_strided_and_unaligned_rows(dtype):
    w, b = randn((64,), dtype, 2, 0.2, 1.0), randn((64,), dtype, 3)
    store = randn((50, 200), dtype, 1)
    dstore = randn((50, 200), dtype, 4)
    for start, stop in ((0, 64), (8, 72), (1, 65), (133, 197)):
        norm_case(store[:, start:stop], w, b, dstore[:, stop - 64:stop])
    norm_case(store[:, :64].t().contiguous().t(), w, b, dstore[:, 64:128])
    norm_case(store[::2, 8:72], w, b, dstore[:25, :64])
    norm_case(store[:1, 8:72].expand(7, 64), w, b, dstore[:7, :64])
    # channels-last volumes: a view of the channels as the last dimension
    volume = torch_convnd.channels_last(randn((2, 64, 3, 4, 5), dtype, 5)).movedim(1, -1)
    assert volume.is_contiguous()
    norm_case(volume, w, b, randn(tuple(volume.shape), dtype, 6))


@gpu
def test_norm_large_mean_and_constant_rows():
    x = randn((64, 1000), torch.float32, 1, 1.0, 4096.0)
    norm_case(x, randn((1000,), torch.float32, 2), None, randn((64, 1000), torch.float32, 3))
    x = torch.full((4, 96), 3.0, device="cuda")
    assert torch.equal(torch_convnd.layer_norm(x), torch.zeros_like(x))


@gpu
@pytest.mark.parametrize("width", [24, 64, 771, 4096])
def test_norm_nonfinite_rows_stay_alone(width):
    x = randn((70, width), torch.bfloat16, 1)
    clean = torch_convnd.layer_norm(x)
    bad = x.clone()
    bad[3, 0], bad[40, width - 1] = float("inf"), float("nan")
    y = torch_convnd.layer_norm(bad)
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[3] = keep[40] = False
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[~keep]).any(1).all()


@gpu
def test_norm_empty_and_frozen():
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = torch_convnd.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))
    x = randn((20, 16), torch.float32, 1)
    torch_convnd.launch_count(reset=True)
    y = torch_convnd.layer_norm(x.requires_grad_(), w.detach())
    y.sum().backward()
    assert torch_convnd.launch_count() == 2  # no pass over the parameters' gradients
    x = x.detach()
    y = torch_convnd.layer_norm(x, w)
    (dw,) = torch.autograd.grad(y, (w,), torch.ones_like(y))
    check(dw, plain_norm(x.double(), None, None, 1e-5)[1].sum(0), 20 * 64 * 2.0**-24, "dw alone")


# ---- linear ----------------------------------------------------------------------------


def plain_linear(x, w, b, r, act):
    z = x @ w.t()
    if b is not None:
        z = z + b
    y = z
    if act == "gelu":
        y = 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    elif act == "silu":
        y = z * torch.sigmoid(z)
    return (y if r is None else y + r), z


def linear_case(x, w, b=None, r=None, act=None, backward=True, seed=9):
    dtype = x.dtype
    leaves = [t if t is None else t.detach().requires_grad_(backward) for t in (x, w, b, r)]
    y = torch_convnd.linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    refs = double(x, w, b, r)
    ref, z = plain_linear(*refs, act)
    k = x.shape[-1]
    bound = (k / 16 + 12) * 2 * unit(dtype)
    with torch.no_grad():
        terms = refs[0].abs() @ refs[1].abs().t() + (0 if b is None else refs[2].abs())
        slack = 1.2 * bound * terms + 8 * unit(dtype) * (z.abs() + (0 if r is None else r.abs()))
        check(y, ref, slack, "y")
    if not backward:
        return
    dy = randn(tuple(y.shape), dtype, seed)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    wanted = torch.autograd.grad(ref, [t for t in refs if t is not None], dy.double())
    with torch.no_grad():
        rows, n = max(1, x.numel() // k), w.shape[0]
        dya = dy.double().reshape(-1, n).abs()
        # dz: the slope is at most 1.13 and changes by at most 0.8 per unit of z, which is
        # off by its float32 error and, where it is kept in 16 bits, by its rounding
        dz = 1.13 * dya
        off = torch.zeros_like(dz)
        if act is not None:
            off = dya * (slack.reshape(-1, n) + eps(dtype) * z.reshape(-1, n).abs()) * 0.8
            off = off + dz * (eps(dtype) + 16 * unit(dtype))
        xa, wa = refs[0].reshape(-1, k).abs(), refs[1].abs()
        def product_slack(a, da, b, length):
            return (length / 16 + 12) * 2 * unit(dtype) * (a @ b) + da @ b
        check(grads[0].reshape(-1, k), wanted[0].reshape(-1, k), product_slack(dz, off, wa, n), "dx")
        check(grads[1], wanted[1], product_slack(dz.t(), off.t(), xa, rows), "dweight")
        i = 2
        if b is not None:
            sums = (rows / 8 + 32) * unit(dtype)
            check(grads[i], wanted[i], sums * dz.sum(0) + off.sum(0), "dbias")
            i += 1
        if r is not None:
            assert torch.equal(grads[i], dy)


def linear_inputs(m, k, n, dtype, bias=True, residual=False):
    return (randn((m, k), dtype, 1), randn((n, k), dtype, 2, 1 / math.sqrt(k)),
            randn((n,), dtype, 3, 0.3) if bias else None,
            randn((m, n), dtype, 4) if residual else None)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 8, 8), (2, 7, 3), (3, 64, 100), (5, 129, 17), (16, 64, 64), (17, 72, 264),
    (64, 256, 128), (127, 100, 60), (128, 64, 256), (129, 136, 520), (257, 515, 259),
    (300, 1030, 77), (1000, 32, 16), (33, 2048, 40), (520, 1024, 1024)])
def test_linear_sizes(m, k, n, dtype):
    linear_case(*linear_inputs(m, k, n, dtype, residual=m % 2 == 1), act="gelu" if n % 3 else None)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_linear_epilogues(act, bias, residual, dtype):
    for m in (4, 200):
        linear_case(*linear_inputs(m, 96, 144, dtype, bias, residual), act=act)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_rows_and_long_sums(dtype):
    linear_case(*linear_inputs(20011, 32, 24, dtype), act="silu")
    linear_case(*linear_inputs(12, 8200, 40, dtype), act=None)
    linear_case(*linear_inputs(2, 40, 9000, dtype), act="gelu")
    linear_case(*linear_inputs(4100, 520, 264, dtype), act=None)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_strided_and_unaligned_operands(dtype):
    store = randn((40, 300), dtype, 1)
    w, b, _ = linear_inputs(1, 64, 48, dtype)[1:]
    for start in (0, 8, 1, 235):
        linear_case(store[:, start:start + 64], w, b, act="gelu")
    linear_case(store[::3, :64], w, b)
    linear_case(store[:, :64].t().contiguous().t(), w, b)
    linear_case(store[:1, :64].expand(9, 64), w, b)
    flat = randn((48 * 64 + 1,), dtype, 5, 0.1)
    linear_case(store[:, :64], flat[1:].view(48, 64), flat[1:49], act="silu")
    linear_case(store[:, :48], w.t()[:48].t().contiguous(), b, store[:, 100:148])
    linear_case(randn((2, 3, 5, 64), dtype, 6), w, b, randn((2, 3, 5, 48), dtype, 7), "gelu")
    linear_case(randn((64,), dtype, 6), w, b)


@gpu
def test_linear_empty_rows_and_frozen_parts():
    x, w, b, _ = linear_inputs(0, 24, 16, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = torch_convnd.linear(*leaves, activation="gelu")
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert dx.shape == (0, 24) and not dw.any() and not db.any()
    x, w, b, _ = linear_inputs(130, 24, 16, torch.bfloat16)
    for frozen in range(3):
        leaves = [t.detach().clone().requires_grad_(i != frozen) for i, t in enumerate((x, w, b))]
        y = torch_convnd.linear(*leaves, activation="gelu")
        dy = randn((130, 16), torch.bfloat16, 5)
        grads = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)
        full = [t.detach().clone().requires_grad_() for t in (x, w, b)]
        whole = torch.autograd.grad(torch_convnd.linear(*full, activation="gelu"), full, dy)
        for got, ref in zip(grads, [g for i, g in enumerate(whole) if i != frozen]):
            assert torch.equal(got, ref)


@gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [
    (8192, 64, 256), (8193, 64, 64), (20000, 8, 8), (37889, 40, 200), (50001, 64, 136), (8320, 16, 72)])
def test_linear_tall_and_thin(m, k, n, act, dtype):
    x, w, b, _ = linear_inputs(m, k, n, dtype)
    linear_case(x, w, b, act=act)
    wide = torch.cat([x, x.flip(0)], 1)
    linear_case(wide[:, k:], w, act=act, seed=10)  # rows twice as far apart, no bias


@gpu
@pytest.mark.parametrize("dtype", HALF)
def test_linear_nonfinite_rows_stay_alone(dtype):
    x, w, b, _ = linear_inputs(140, 72, 40, dtype)
    clean = torch_convnd.linear(x, w, b)
    bad = x.clone()
    bad[5, 3] = float("nan")
    bad[139, 71] = float("inf")
    y = torch_convnd.linear(bad, w, b)
    keep = torch.ones(140, dtype=torch.bool, device="cuda")
    keep[5] = keep[139] = False
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[5]).all() and not torch.isfinite(y[139]).any()


@gpu
def test_linear_float32_extremes():
    """The three-term split of float32 operands covers the whole exponent range."""
    x, w, _, _ = linear_inputs(130, 64, 40, torch.float32)
    for sx, sw in ((2.0**60, 2.0**-60), (2.0**-50, 2.0**40), (2.0**100, 2.0**-110)):
        linear_case(x * sx, w * sw, backward=False)


@gpu
def test_linear_autocast():
    x, w, b, _ = linear_inputs(64, 32, 48, torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = torch_convnd.linear(x, w, b, activation="gelu")
    assert y.dtype == torch.bfloat16
    assert torch.equal(y, torch_convnd.linear(x.bfloat16(), w.bfloat16(), b.bfloat16(),
                                              activation="gelu"))


# ---- gated recurrence ------------------------------------------------------------------


def plain_recurrence(x, g, h0, dim):
    """States by the definition, one step after another."""
    x, g = x.movedim(dim, 0), g.movedim(dim, 0)
    h = torch.zeros(x.shape[1:], dtype=x.dtype, device=x.device) if h0 is None else h0
    states = []
    for t in range(x.shape[0]):
        f = torch.sigmoid(g[t])
        h = f * h + torch.sigmoid(-g[t]) * x[t]
        states.append(h)
    y = torch.stack(states) if states else x
    return y.movedim(0, dim), h


def recurrence_case(x, g, h0, dim, use=("y", "last"), seed=11):
    dtype = x.dtype
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, g, h0)]
    y, last = torch_convnd.gated_recurrence(leaves[0], leaves[1], leaves[2], dim=dim)
    assert last.dtype == wide and y.dtype == dtype
    refs = double(x, g, h0)
    ref_y, ref_last = plain_recurrence(*refs, dim)
    dy, dlast = randn(tuple(y.shape), dtype, seed), randn(tuple(last.shape), wide, seed + 1)
    outs, ref_outs, given, ref_given = [], [], [], []
    for name, out, ref, grad in (("y", y, ref_y, dy), ("last", last, ref_last, dlast)):
        if name in use:
            outs.append(out)
            ref_outs.append(ref)
            given.append(grad)
            ref_given.append(grad.double())
    wanted = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(outs, wanted, given)
    ref_grads = torch.autograd.grad(ref_outs, [t for t in refs if t is not None], ref_given)
    with torch.no_grad():
        # a state is a mean of earlier values with weights that sum to at most 1: an error of
        # one step fades as the state does, so a state is off by at most the largest value
        # times the steps it remembers (at most all of them) times a few roundings
        steps = min(x.shape[dim], 4096)
        big = max([float(t.abs().max()) for t in refs[::2] if t is not None and t.numel()] + [0.0])
        slack = 8 * (steps + 2) * unit(dtype) * big
        check(y, ref_y, slack, "y")
        check(last, ref_last, slack, "last")
        # a flow is a sum of at most `steps` gradients, each off by the same count of
        # roundings; where it is long its weights fade like the states'
        flow = 8 * max([float(t.abs().max()) for t in ref_given if t.numel()] + [0.0])
        reach = max(1.0, float(1 / torch.sigmoid(-refs[1].clamp(-30, 6)).mean())) if x.numel() else 1
        flow_slack = 8 * (min(steps, 512) + 2) * unit(dtype) * flow * reach
        for name, got, ref in zip(("dx", "dgate", "dinitial"), grads, ref_grads):
            check(got, ref, flow_slack * (2 * big if name == "dgate" else 1.0) + slack * flow, name)


def recurrence_inputs(shape, dim, dtype, initial=True, mean=1.5):
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    state = shape[:dim] + shape[dim + 1:]
    return (randn(shape, dtype, 1), randn(shape, dtype, 2, 1.5, mean),
            randn(state, wide, 3) if initial else None)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps", [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 300, 1025])
def test_recurrence_steps(steps, dtype):
    recurrence_case(*recurrence_inputs((3, steps, 20), 1, dtype), 1)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,dim", [
    ((40,), 0), ((5, 40), 1), ((40, 5), 0), ((2, 7, 260), 2), ((2, 7, 261), -1), ((1, 90, 1), 1),
    ((2, 3, 50, 2), 2), ((2, 70, 129), 1), ((3, 8, 35, 4, 5), 2), ((3, 8, 4, 5, 36), 4),
    ((6, 1, 512), 1), ((1, 2000, 8), 1), ((2, 3, 1100), 2), ((300, 3, 7), 1)])
def test_recurrence_axes(shape, dim, dtype):
    x, g, h0 = recurrence_inputs(shape, dim % len(shape), dtype)
    recurrence_case(x, g, h0, dim)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_recurrence_memory_orders(dtype):
    x, g, h0 = recurrence_inputs((2, 16, 21, 6, 5), 2, dtype)
    cl = torch_convnd.channels_last
    for a, b in ((cl(x), cl(g)), (cl(x), g), (x, cl(g)), (x, g[..., :1].expand_as(x))):
        recurrence_case(a, b, h0, 2)
    y, last = torch_convnd.gated_recurrence(cl(x), cl(g), h0, dim=2)
    assert torch_convnd.is_channels_last(y)
    straight, straight_last = torch_convnd.gated_recurrence(x, g, h0, dim=2)
    assert torch.equal(y, straight) and torch.equal(last, straight_last)
    wide = randn((2, 30, 40), dtype, 5)
    recurrence_case(wide[:, ::2, 3:20], randn((2, 15, 17), dtype, 6), None, 1)
    recurrence_case(wide.transpose(1, 2), randn((2, 40, 30), dtype, 6), None, 1)
    flat = randn((3 * 20 * 8 + 1,), dtype, 7)[1:].view(3, 20, 8)
    recurrence_case(flat, randn((3, 20, 8), dtype, 8), None, 1)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("use", [("y",), ("last",)])
def test_recurrence_unused_outputs_and_no_initial(use, dtype):
    recurrence_case(*recurrence_inputs((2, 70, 24), 1, dtype, initial=False), 1, use=use)


@gpu
@pytest.mark.parametrize("shape,dim", [((2, 200, 16), 1), ((2, 16, 200), 2)])
def test_recurrence_infinite_gates_restart_and_hold(shape, dim):
    x, g, h0 = recurrence_inputs(shape, dim, torch.float32)
    gates = g.movedim(dim, 0)
    gates[40], gates[41:60], gates[150] = -math.inf, math.inf, -math.inf
    recurrence_case(x, g, h0, dim)
    y, _ = torch_convnd.gated_recurrence(x, g, h0, dim=dim)
    y, xs = y.movedim(dim, 0), x.movedim(dim, 0)
    assert torch.equal(y[40], xs[40]) and torch.equal(y[150], xs[150])
    assert torch.equal(y[59], xs[40])
    # what came before a restart does not reach past it, not even as 0 * inf
    bad = x.clone()
    bad.movedim(dim, 0)[10] = 3e38
    z, _ = torch_convnd.gated_recurrence(bad, g, h0, dim=dim)
    assert torch.equal(z.movedim(dim, 0)[40:], y[40:])


@gpu
def test_recurrence_nonfinite_columns_stay_alone():
    x, g, h0 = recurrence_inputs((2, 150, 70), 1, torch.bfloat16)
    clean, clean_last = torch_convnd.gated_recurrence(x, g, h0, dim=1)
    bad = x.clone()
    bad[0, 60, 5], bad[1, 3, 69] = float("nan"), float("inf")
    y, last = torch_convnd.gated_recurrence(bad, g, h0, dim=1)
    keep = torch.ones((2, 70), dtype=torch.bool, device="cuda")
    keep[0, 5] = keep[1, 69] = False
    assert torch.equal(y.transpose(1, 2)[keep], clean.transpose(1, 2)[keep])
    assert torch.equal(last[keep], clean_last[keep])
    assert torch.equal(y[0, :60, 5], clean[0, :60, 5]) and torch.isnan(y[0, 60:, 5]).all()
    assert torch.equal(y[1, :3, 69], clean[1, :3, 69]) and torch.isinf(y[1, 3, 69])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_recurrence_continues_from_its_last_state(dtype):
    x, g, h0 = recurrence_inputs((4, 97, 40), 1, dtype)
    whole, last = torch_convnd.gated_recurrence(x, g, h0, dim=1)
    parts, state = [], h0
    for start, stop in ((0, 1), (1, 2), (2, 40), (40, 41), (41, 97)):
        y, state = torch_convnd.gated_recurrence(x[:, start:stop], g[:, start:stop], state, dim=1)
        parts.append(y)
    bound = 97 * 8 * 2.0**-24 * float(max(x.abs().max(), h0.abs().max()))
    check(torch.cat(parts, 1), whole, bound, "states")
    check(state, last, bound, "last")


@gpu
def test_recurrence_without_steps_or_columns():
    h0 = randn((2, 8), torch.float32, 1).requires_grad_()
    x = torch.empty(2, 0, 8, device="cuda", requires_grad=True)
    y, last = torch_convnd.gated_recurrence(x, x, h0, dim=1)
    assert y.shape == (2, 0, 8) and torch.equal(last, h0)
    (d0,) = torch.autograd.grad(last, (h0,), torch.ones_like(last))
    assert torch.equal(d0, torch.ones_like(h0))
    _, last = torch_convnd.gated_recurrence(x, x, None, dim=1)
    assert torch.equal(last, torch.zeros(2, 8, device="cuda"))
    empty = torch.empty(0, 5, 8, device="cuda")
    y, last = torch_convnd.gated_recurrence(empty, empty, dim=1)
    assert y.shape == (0, 5, 8) and last.shape == (0, 8)


@gpu
@pytest.mark.parametrize("mean", [-6.0, 0.0, 6.0])
def test_recurrence_long(mean):
    recurrence_case(*recurrence_inputs((1, 9001, 33), 1, torch.float32, mean=mean), 1)


# ---- what the three share --------------------------------------------------------------


def each_operator(dtype=torch.float32):
    """(name, function of leaves, leaves) of one small call of each operator."""
    x, w, b, r = linear_inputs(70, 40, 24, dtype, residual=True)
    n = randn((40,), dtype, 5), randn((40,), dtype, 6)
    rx, rg, h0 = recurrence_inputs((2, 37, 12), 1, dtype)
    return [
        ("layer_norm", lambda *t: torch_convnd.layer_norm(*t), (x, *n)),
        ("linear", lambda a, c, d, e: torch_convnd.linear(a, c, d, activation="gelu", residual=e),
         (x, w, b, r)),
        ("gated_recurrence", lambda *t: torch_convnd.gated_recurrence(*t, dim=1), (rx, rg, h0)),
    ]


@gpu
def test_gradients_against_differences():
    w = randn((5, 7), torch.float64, 1).requires_grad_()
    x = randn((4, 7), torch.float64, 2).requires_grad_()
    n = randn((7,), torch.float64, 3).requires_grad_()
    b = randn((5,), torch.float64, 4).requires_grad_()
    r = randn((4, 5), torch.float64, 5).requires_grad_()
    c = randn((7,), torch.float64, 6).requires_grad_()
    assert torch.autograd.gradcheck(torch_convnd.layer_norm, (x, n, c))
    for act in (None, "gelu", "silu"):
        assert torch.autograd.gradcheck(
            lambda *t: torch_convnd.linear(*t[:3], activation=act, residual=t[3]), (x, w, b, r))
    for shape, dim in (((2, 19, 3), 1), ((2, 3, 35), 2)):
        rx, rg, h0 = (t.requires_grad_() for t in recurrence_inputs(shape, dim, torch.float64))
        assert torch.autograd.gradcheck(
            lambda *t: torch_convnd.gated_recurrence(*t, dim=dim), (rx, rg, h0))


@gpu
def test_repeated_calls_give_the_same_bits_on_any_stream():
    for dtype in (torch.bfloat16, torch.float32):
        for name, call, leaves in each_operator(dtype):
            def step():
                own = [t.detach().requires_grad_() for t in leaves]
                outs = call(*own)
                outs = outs if isinstance(outs, tuple) else (outs,)
                return [*outs, *torch.autograd.grad(outs, own, [torch.ones_like(o) for o in outs])]
            first = step()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                second = step()
            torch.cuda.current_stream().wait_stream(side)
            for a, c in zip(first, second):
                assert torch.equal(a, c), name
    torch_convnd.device_status()


@gpu
@pytest.mark.parametrize("rows", [256, 8192])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_in_a_new_thread(rows, act):
    """A thread that has made no CUDA call yet (an autograd worker's first backward)."""
    x, w, _, _ = linear_inputs(rows, 64, 128, torch.bfloat16)
    dy = randn((rows, 128), torch.bfloat16, 5)
    ops = torch.ops.torch_convnd
    def run():
        _, pre = ops.linear_train(x, w, None, None, act)
        return ops.linear_backward(dy, pre, x, w, act, [True, True, False])[:2]
    def backward_only():
        found.append(ops.linear_backward(dy, pre, x, w, act, [True, True, False])[:2])
    found, expected = [], run()
    _, pre = ops.linear_train(x, w, None, None, act)
    for target in (backward_only, lambda: found.append(run())):
        thread = threading.Thread(target=target)
        thread.start()
        thread.join()
    assert len(found) == 2
    for got in found:
        assert all(torch.equal(g, e) for g, e in zip(got, expected))


@gpu
def test_operators_register_completely():
    for dtype in (torch.bfloat16, torch.float32):
        x, w, b, r = linear_inputs(6, 16, 8, dtype, residual=True)
        ops = torch.ops.torch_convnd
        rx, rg, h0 = recurrence_inputs((2, 5, 6), 1, dtype)
        grads = [t.detach().requires_grad_() for t in (x, w, b, r, rx, rg, h0)]
        x, w, b, r, rx, rg, h0 = grads
        n = randn((16,), dtype, 5).requires_grad_()
        torch.library.opcheck(ops.layer_norm.default, (x, n, None, 1e-5))
        torch.library.opcheck(ops.linear.default, (x, w, b, r, "gelu"))
        torch.library.opcheck(ops.gated_recurrence.default, (rx, rg, h0, 1))
        cl = torch_convnd.channels_last(randn((2, 4, 3, 5), dtype, 7))
        torch.library.opcheck(ops.gated_recurrence_train.default, (cl, cl.clone(), None, 2),
                              test_utils=("test_schema", "test_faketensor"))
        torch.library.opcheck(ops.linear_train.default, (x.detach(), w.detach(), None, None, "none"),
                              test_utils=("test_schema", "test_faketensor"))
        torch.library.opcheck(ops.layer_norm_train.default, (x.detach(), None, None, 1e-5),
                              test_utils=("test_schema", "test_faketensor"))


@gpu
def test_steps_are_captured_in_cuda_graphs():
    for name, call, leaves in each_operator(torch.bfloat16):
        own = [t.detach().requires_grad_() for t in leaves]
        def step():
            outs = call(*own)
            outs = outs if isinstance(outs, tuple) else (outs,)
            return [*outs, *torch.autograd.grad(outs, own, [torch.ones_like(o) for o in outs])]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                expected = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, expected):
            assert torch.equal(a, c), name


@gpu
def test_second_derivatives_are_refused():
    for name, call, leaves in each_operator():
        own = [t.detach().requires_grad_() for t in leaves]
        out = call(*own)
        out = out[0] if isinstance(out, tuple) else out
        (grad,) = torch.autograd.grad(out.sum(), own[:1], create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            grad.sum().backward()


@gpu
def test_offsets_past_32_bits():
    rows, width = (1 << 31) // 512 + 3, 512
    x = torch.zeros((rows, width), device="cuda", dtype=torch.bfloat16)
    x[-1] = randn((width,), torch.bfloat16, 1)
    y = torch_convnd.layer_norm(x)
    check(y[-1:], plain_norm(x[-1:].double(), None, None, 1e-5)[0], 64 * 2.0**-24 * 8, "last row")
    assert not y[-2].any()
    del y
    g = torch.full_like(x, -math.inf)
    states, last = torch_convnd.gated_recurrence(x, g, dim=0)
    assert torch.equal(states[-1], x[-1]) and torch.equal(last, x[-1].float())
    del states, g
    w = randn((16, width), torch.bfloat16, 2)
    tail = torch_convnd.linear(x[-130:], w)
    y = torch_convnd.linear(x, w)
    assert torch.equal(y[-130:], tail)


def test_refusals():
    """Bad arguments raise on any device, before the device is looked at."""
    x = torch.zeros(4, 8)
    norm, linear, recurrence = (torch_convnd.layer_norm, torch_convnd.linear,
                                torch_convnd.gated_recurrence)
    cases = [
        (lambda: norm(x.int()), "supports float16"),
        (lambda: norm(torch.zeros(())), "last dimension"),
        (lambda: norm(torch.zeros(4, 0)), "last dimension"),
        (lambda: norm(x, torch.ones(7)), "vectors of the last dimension"),
        (lambda: norm(x, None, torch.ones(8, 1)), "vectors of the last dimension"),
        (lambda: norm(x, torch.ones(8).double()), "dtype or float32"),
        (lambda: norm(x.double(), torch.ones(8)), "dtype or float32"),
        (lambda: norm(x.half(), torch.ones(8), torch.ones(8).half()), "same dtype"),
        (lambda: norm(x.to_sparse()), "strided"),
        (lambda: linear(x, torch.ones(3, 7)), "in_features"),
        (lambda: linear(x, torch.ones(0, 8)), "in_features"),
        (lambda: linear(x, torch.ones(3, 8).double()), "device and dtype"),
        (lambda: linear(x, torch.ones(3, 8), torch.ones(4)), "out_features"),
        (lambda: linear(x, torch.ones(3, 8), residual=torch.ones(3)), "output's shape"),
        (lambda: linear(x, torch.ones(3, 8), residual=torch.ones(4, 3).half()), "device and dtype"),
        (lambda: torch.ops.torch_convnd.linear(x, torch.ones(3, 8), None, None, "relu"), "supports"),
        (lambda: recurrence(x, x[:, :7], dim=1), "input's shape"),
        (lambda: recurrence(x, x.half(), dim=1), "device and dtype"),
        (lambda: recurrence(x, x, dim=2), "dimension of the input"),
        (lambda: recurrence(x, x, torch.zeros(8), dim=1), "without dim"),
        (lambda: recurrence(x.half(), x.half(), torch.zeros(4).half(), dim=1), "without dim"),
    ]
    for call, message in cases:
        with pytest.raises((RuntimeError, NotImplementedError), match=message):
            call()
    with pytest.raises(ValueError, match="Invalid activation"):
        linear(x, torch.ones(3, 8), activation="relu")
    for call in (lambda: norm(x), lambda: linear(x, torch.ones(3, 8)), lambda: recurrence(x, x, dim=1)):
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            call()


@gpu
def test_devices_must_match():
    x = torch.zeros(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="device"):
        torch_convnd.layer_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="device"):
        torch_convnd.linear(x, torch.ones(3, 8))
    with pytest.raises(RuntimeError, match="device"):
        torch_convnd.gated_recurrence(x, torch.zeros(4, 8), dim=1)
