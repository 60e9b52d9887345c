"""The layer operators at the edges of their inputs: alignment, gaps, empty axes, tails.

Where two calls do the same arithmetic on the same values the results have to be the same
bits; elsewhere a bound is derived beside the test.
"""

from __future__ import annotations

import ctypes
import math
import threading

import pytest
import torch

import torch_convnd
from test_layers import check, eps, linear_inputs, randn, recurrence_inputs
from torch_convnd import _native

gpu = pytest.mark.gpu


def off_boundary(t):
    """The same values, shape and strides (contiguous) one element past a 16-byte boundary."""
    moved = torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)[1:].view(t.shape)
    moved.copy_(t)
    assert moved.data_ptr() % 16 != 0
    return moved


# ---- gated recurrence along the last axis: steps next to one another ---------------------


def recurrence_backward(x, g, h0, dy):
    leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
    y, _ = torch_convnd.gated_recurrence(*leaves, dim=x.ndim - 1)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("steps", [7, 301, 1001, 5003])
def test_recurrence_gradients_do_not_depend_on_alignment(steps, dtype):
    """Kept states lie where the backward looks for them, whatever starts off 16 bytes."""
    x, g, h0 = recurrence_inputs((3, 7, steps), 2, dtype)
    dy = randn((3, 7, steps), dtype, 5)
    expected = recurrence_backward(x, g, h0, dy)
    for moved in ((3,), (0,), (1,), (0, 1), (0, 1, 3)):
        inputs = [off_boundary(t) if i in moved else t for i, t in enumerate((x, g, h0, dy))]
        for name, got, ref in zip(("y", "dx", "dgate", "dinitial"), recurrence_backward(*inputs), expected):
            assert torch.equal(got, ref), f"{name}, unaligned {moved}"


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_recurrence_gradient_through_concatenation(dtype):
    """torch.cat hands its second part a gradient that starts inside a larger buffer."""
    x, g, h0 = recurrence_inputs((1, 7, 1001), 2, dtype)
    dy = randn((1, 8, 1001), dtype, 5)
    leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
    y, _ = torch_convnd.gated_recurrence(*leaves, dim=2)
    ahead = torch.zeros((1, 1, 1001), device="cuda", dtype=dtype)
    grads = torch.autograd.grad(torch.cat([ahead, y], 1), leaves, dy)
    for got, ref in zip(grads, recurrence_backward(x, g, h0, dy[:, 1:].clone())[1:]):
        assert torch.equal(got, ref)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("steps", [301, 1101])
def test_recurrence_step_layout_against_definition(steps, dtype):
    """Bounds that follow each column's own memory: a rounding of step t reaches step t + k
    times the gates between them, so the sum of those products (`reach`, the same recurrence
    over ones) times a step's roundings bounds a state's error, and likewise the flow's. A
    step rounds its gate (2^-20 with the fast exponential, four float32 roundings else),
    the two products and the sum, and composed maps round each of theirs once more: 16."""
    x, g, h0 = recurrence_inputs((2, 5, steps), 2, dtype)
    dy = off_boundary(randn((2, 5, steps), dtype, 5))
    y, dx, dgate, d0 = recurrence_backward(x, g, h0, dy)
    u = 16 * (2.0**-20 if dtype == torch.bfloat16 else 2.0**-24)
    xs, gs, ds = x.double(), g.double(), dy.double()
    f, keep = torch.sigmoid(gs), torch.sigmoid(-gs)
    before, states, reach, state, r = [], [], [], h0.double(), torch.zeros_like(h0).double()
    for t in range(steps):
        before.append(state)
        state = f[..., t] * state + keep[..., t] * xs[..., t]
        r = f[..., t] * r + 1
        states.append(state)
        reach.append(r)
    before, states, reach = (torch.stack(v, -1) for v in (before, states, reach))
    flow, total, memory, m = torch.zeros_like(state), [], [], torch.zeros_like(state)
    for t in reversed(range(steps)):
        total.append(flow + ds[..., t])
        m = m + 1
        memory.append(m)
        flow, m = f[..., t] * total[-1], f[..., t] * m
    total, memory = (torch.stack(v[::-1], -1) for v in (total, memory))
    big, largest = max(xs.abs().max(), h0.abs().max()), ds.abs().max()
    off_state, off_flow = u * big * reach, u * largest * memory
    check(y, states, off_state, "y")
    check(dx, total * keep, keep * off_flow + u * (total * keep).abs(), "dx")
    slope = f * keep
    check(dgate, total * (before - xs) * slope,
          slope * (off_flow * (before - xs).abs() + total.abs() * (off_state + u * big)) * 1.01
          + u * (total * (before - xs) * slope).abs(), "dgate")
    check(d0, flow, off_flow[..., 0], "dinitial")


@gpu
def test_recurrence_c_abi_buffers_of_any_alignment():
    """Outputs of another alignment than the inputs, in either pass."""
    library = _native.core()
    pointer, size = ctypes.c_void_p, ctypes.c_size_t
    dims = [ctypes.c_int32, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64]
    library.cnd_gated_recurrence_forward.argtypes = dims + [pointer] * 7 + [size, pointer]
    library.cnd_gated_recurrence_backward.argtypes = dims + [pointer] * 10 + [size, pointer]
    library.cnd_gated_recurrence_workspace_size.argtypes = dims
    library.cnd_gated_recurrence_workspace_size.restype = size
    columns, steps = 6, 1101
    x, g, _ = recurrence_inputs((columns, steps), 1, torch.float32, initial=False)
    dy = randn((columns, steps), torch.float32, 5)
    problem = (2, columns, steps, 1)
    blocks = library.cnd_gated_recurrence_blocks(*problem)
    bytes_ = library.cnd_gated_recurrence_workspace_size(*problem)
    workspace = torch.empty(max(bytes_, 1), device="cuda", dtype=torch.uint8)
    stream = pointer(torch.cuda.current_stream().cuda_stream)

    def step(moved):
        def output():
            t = torch.zeros_like(x)
            return off_boundary(t) if moved[0] else t
        y, last = output(), torch.empty(columns, device="cuda")
        states = torch.empty((blocks, columns), device="cuda")
        assert library.cnd_gated_recurrence_forward(
            *problem, x.data_ptr(), g.data_ptr(), None, y.data_ptr(), last.data_ptr(),
            states.data_ptr(), workspace.data_ptr(), bytes_, stream) == 0
        moved = moved[1:]
        dx, dgate, d0 = output(), output(), torch.empty(columns, device="cuda")
        mask = (ctypes.c_int32 * 3)(1, 1, 1)
        assert library.cnd_gated_recurrence_backward(
            *problem, dy.data_ptr(), None, x.data_ptr(), g.data_ptr(), states.data_ptr(),
            dx.data_ptr(), dgate.data_ptr(), d0.data_ptr(), mask, workspace.data_ptr(), bytes_,
            stream) == 0
        return y, last, dx, dgate, d0

    expected = step((False, False))
    for moved in ((True, False), (False, True), (True, True)):
        for got, ref in zip(step(moved), expected):
            assert torch.equal(got, ref), moved


# ---- linear: residual tiles that arrive ahead --------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(60001, 64, 256), (40000, 512, 520), (9000, 64, 128), (3001, 72, 64)])
def test_linear_residual_tiles_are_waited_for(m, k, n, dtype):
    """Many tiles a block, each with a residual fetched while the one before is worked on: the
    same bits call after call, those of the sum taken in float32 outside, and no expired wait."""
    x, w, b, r = linear_inputs(m, k, n, dtype, residual=True)
    plain = torch_convnd.linear(x, w, b)
    y = torch_convnd.linear(x, w, b, residual=r)
    # the rounding of `plain` is the only difference: half a unit in its last place
    check(y, plain.double() + r.double(), eps(dtype) * plain.double().abs(), "y")
    for _ in range(100):
        assert torch.equal(torch_convnd.linear(x, w, b, residual=r), y)
    torch_convnd.device_status()


# ---- fake kernels ------------------------------------------------------------------------

GAPS = {  # inputs of gated_recurrence: (make, dim)
    "rows and columns cut, transposed": (
        lambda **o: torch.empty((2, 30, 40), **o)[:, ::2, 3:20].transpose(1, 2), 1),
    "channels-last volume cut": (
        lambda **o: torch.empty((2, 6, 8, 10), **o).to(memory_format=torch.channels_last)[:, :, :6, ::2], 2),
    "expanded": (lambda **o: torch.empty((2, 1, 7), **o).expand(2, 300, 7), 1),
    "long, transposed": (lambda **o: torch.empty((2, 600, 40), **o)[:, 1:-3, ::2].transpose(1, 2), 2),
    "dense, transposed": (lambda **o: torch.empty((2, 600, 40), **o).transpose(1, 2), 2),
}


@pytest.mark.parametrize("name,strides,last", [
    ("rows and columns cut, transposed", (255, 15, 1), (15, 1)),
    ("channels-last volume cut", (180, 30, 5, 1), (30, 5, 1)),
    ("expanded", (2100, 7, 1), (7, 1)),
    ("dense, transposed", (24000, 1, 40), (40, 1))])
def test_recurrence_fake_strides_follow_the_native_rule(name, strides, last):
    """The input's own strides where it is dense, else contiguous."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    make, dim = GAPS[name]
    with FakeTensorMode():
        x = make(device="cuda")
        y, state = torch_convnd.gated_recurrence(x, x, dim=dim)
        assert y.stride() == strides and state.stride() == last
        _, _, states = torch.ops.torch_convnd.gated_recurrence_train(x, x, None, dim)
        dx, dgate, d0 = torch.ops.torch_convnd.gated_recurrence_backward(
            y, state, x, x, states, dim, [True, True, True])
        assert dx.stride() == dgate.stride() == strides and d0.stride() == last


@gpu
@pytest.mark.parametrize("name", list(GAPS))
def test_recurrence_fake_kernels_agree_with_native(name):
    make, dim = GAPS[name]
    x = make(device="cuda").normal_() if name != "expanded" else make(device="cuda")
    train = torch.ops.torch_convnd.gated_recurrence_train.default
    torch.library.opcheck(train, (x, x, None, dim), test_utils=("test_schema", "test_faketensor"))
    y, last, states = train(x, x, None, dim)
    torch.library.opcheck(
        torch.ops.torch_convnd.gated_recurrence_backward.default,
        (y, last, x, x, states, dim, [True, True, True]), test_utils=("test_schema", "test_faketensor"))


# ---- gated recurrence without steps ------------------------------------------------------

EMPTY = [lambda t: t[:, :0], lambda t: t[:, 2:2], lambda t: t.transpose(0, 2)[:, :0],
         lambda t: t.permute(2, 1, 0)[::2, :0], lambda t: t[:0]]


@gpu
@pytest.mark.parametrize("cut", EMPTY)
def test_recurrence_over_an_empty_slice(cut):
    """A slice without steps keeps the strides of its source; the state is dense all the same."""
    x = cut(randn((4, 5, 6), torch.float32, 1)).requires_grad_()
    h0 = randn((x.shape[0], x.shape[2]), torch.float32, 2).requires_grad_()
    y, last = torch_convnd.gated_recurrence(x, x, h0, dim=1)
    assert y.shape == x.shape and last.is_contiguous() and torch.equal(last, h0)
    dlast = randn(tuple(last.shape), torch.float32, 3)
    d0, dx = torch.autograd.grad(last, (h0, x), dlast)
    assert torch.equal(d0, dlast) and dx.shape == x.shape
    _, last = torch_convnd.gated_recurrence(x, x, None, dim=1)
    assert torch.equal(last, torch.zeros_like(h0))
    torch.library.opcheck(torch.ops.torch_convnd.gated_recurrence_train.default,
                          (x.detach(), x.detach(), h0.detach(), 1),
                          test_utils=("test_schema", "test_faketensor"))


# ---- activations far from zero -----------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_activation_tails_keep_their_digits(act, dtype):
    """Relative accuracy where the activation is far smaller than its argument. GELU in
    float32: v^2 / 2 rounds twice, which moves its exponential by v^2 2^-24 of itself, at most
    2^-17 for |v| = 11, beside 6 units of the tail's own form and three products. SiLU: two units
    of exp and three roundings. Values below the smallest normal number may be flushed."""
    low = -11.0 if dtype == torch.float32 else -30.0
    v = torch.linspace(low, -3, 4001, device="cuda", dtype=dtype)[:, None]
    one = torch.ones((1, 1), device="cuda", dtype=dtype)
    y = torch_convnd.linear(v, one, activation=act)
    leaf = v.clone().requires_grad_()
    (slope,) = torch.autograd.grad(torch_convnd.linear(leaf, one, activation=act), leaf,
                                   torch.ones_like(y))
    z = v.double().cpu()
    if act == "gelu":
        cdf = torch.special.erfc(-z / math.sqrt(2)) / 2
        density = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        ref, ref_slope = z * cdf, cdf + z * density
        terms = cdf + z.abs() * density
    else:
        s = torch.exp(z) / (1 + torch.exp(z))
        ref, ref_slope = z * s, s * (1 + z * (1 - s))
        terms = s * (1 + z.abs())
    u = 2.0**-24 if dtype == torch.float32 else 2.0**-53
    grow = u * (4 * low * low + 32)
    tiny = torch.finfo(dtype).tiny
    for got, want, size in ((y, ref, ref.abs()), (slope, ref_slope, terms)):
        off = (got.double().cpu() - want).abs()
        assert bool((off <= grow * size + 8 * tiny).all()), float((off / size).max())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_gelu_at_minus_infinity_is_its_limit(dtype):
    """0, also from a product whose long sum is split and joined by another kernel."""
    for k in (8, 8192):
        x = torch.zeros((3, k), device="cuda", dtype=dtype)
        b = torch.tensor([-math.inf, math.inf, 0.0], device="cuda", dtype=dtype).repeat(3)
        y = torch_convnd.linear(x, torch.zeros((9, k), device="cuda", dtype=dtype), b,
                                activation="gelu")
        assert torch.equal(y[0], torch.tensor([0.0, math.inf, 0.0], device="cuda", dtype=dtype).repeat(3))
        leaf = b.clone().requires_grad_()
        out = torch_convnd.linear(x[:1], torch.zeros((9, k), device="cuda", dtype=dtype), leaf,
                                  activation="gelu")
        (slope,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
        assert torch.equal(slope, torch.tensor([0.0, 1.0, 0.5], device="cuda", dtype=dtype).repeat(3))


@gpu
def test_linear_float64_of_many_features():
    """More features than a grid's second dimension counts 64-wide tiles (65535)."""
    n = 65535 * 64 + 70
    w = randn((n, 1), torch.float64, 1).requires_grad_()
    x = randn((3, 1), torch.float64, 2).requires_grad_()
    y = torch_convnd.linear(x, w)
    assert torch.equal(y, x * w[:, 0])
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    bound = n * 2.0**-53 * w.abs().sum()
    assert bool(((dx - w.sum()).abs() <= bound).all())
    check(dw, x.sum().expand_as(dw), 4 * 2.0**-53 * float(x.abs().sum()), "dw")
    rows = randn((2, n), torch.float64, 3).requires_grad_()
    up = randn((2, n), torch.float64, 4).requires_grad_()
    out = torch_convnd.linear(rows, up)
    dx, dw = torch.autograd.grad(out, (rows, up), torch.eye(2, device="cuda", dtype=torch.float64))
    assert torch.equal(dx, up) and torch.equal(dw, rows)


# ---- calls from several threads ----------------------------------------------------------


@gpu
def test_layer_norm_widths_in_parallel_threads():
    """Calls of one kernel that want different amounts of shared memory do not disturb one
    another."""
    cases = [(randn((64, width), torch.float32, width), []) for width in (2056, 4096)]
    for x, expected in cases:
        expected.append(torch_convnd.layer_norm(x))
    failures = []

    def work(x, expected):
        try:
            for _ in range(3000):
                y = torch_convnd.layer_norm(x)
            if not torch.equal(y, expected[0]):
                failures.append("values")
        except RuntimeError as error:
            failures.append(str(error))

    threads = [threading.Thread(target=work, args=case) for case in cases for _ in range(3)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures[:2]


# ---- waits that expired elsewhere --------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,dim", [((1, 20000, 256), 1), ((2, 60000), 1)])
def test_recurrence_after_another_kernels_expired_wait(shape, dim, dtype):
    """An error that nobody has read yet does not cut the recurrence's own waits short."""
    x, g, _ = recurrence_inputs(shape, dim, dtype, initial=False)
    dy = randn(shape, dtype, 5)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, g)]
        y, last = torch_convnd.gated_recurrence(*leaves, dim=dim)
        return [y, last, *torch.autograd.grad(y, leaves, dy)]

    torch_convnd.device_status()
    expected = step()
    library = _native.core()
    assert library.cnd_debug_stall_test(-20, None) == 0, library.cnd_last_error()
    for _ in range(5):
        for got, ref in zip(step(), expected):
            assert torch.equal(got, ref)
    with pytest.raises(RuntimeError, match="bounded wait expired"):
        torch_convnd.device_status()
    torch_convnd.device_status()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_recurrence_nan_of_all_ones_is_sent_between_chunks(dtype):
    """NaNs whose bits are those of an exchange slot not written yet, in x and in the gate."""
    bits = torch.int32 if dtype == torch.float32 else torch.int64
    for shape, dim in (((1, 4000, 40), 1), ((2, 30000), 1)):
        x, g, _ = recurrence_inputs(shape, dim, dtype, initial=False)
        clean = torch_convnd.gated_recurrence(x, g, dim=dim)[0].movedim(dim, 0)
        x.view(bits).movedim(dim, 0)[1000].flatten()[:1] = -1
        g.view(bits).movedim(dim, 0)[2000].flatten()[-1:] = -1
        y, last = torch_convnd.gated_recurrence(x, g, dim=dim)
        y = y.movedim(dim, 0).flatten(1)
        assert torch.equal(y[:1000, 0], clean.flatten(1)[:1000, 0]) and torch.isnan(y[1000:, 0]).all()
        assert torch.equal(y[:2000, -1], clean.flatten(1)[:2000, -1]) and torch.isnan(y[2000:, -1]).all()
        leaves = [t.detach().requires_grad_() for t in (x, g)]
        out = torch_convnd.gated_recurrence(*leaves, dim=dim)[0]
        dx, dgate = torch.autograd.grad(out, leaves, torch.ones_like(out))
        # the flow goes through the gates behind a step only
        flow = dx.movedim(dim, 0).flatten(1)
        assert torch.isfinite(flow[:, 0]).all() and torch.isnan(flow[:2001, -1]).all()
        assert torch.isfinite(flow[2001:, -1]).all()
    torch_convnd.device_status()


# ---- other ways of differentiating and tracing --------------------------------------------

CALLS = {
    "layer_norm": lambda t: torch_convnd.layer_norm(t),
    "layer_norm, weight": lambda t: torch_convnd.layer_norm(t.detach() * 0, t[0]),
    "linear": lambda t: torch_convnd.linear(t, t.detach()),
    "linear, residual": lambda t: torch_convnd.linear(t.detach(), t.detach()[:, :], residual=t @ t.t()),
    "gated_recurrence": lambda t: torch_convnd.gated_recurrence(t, t.detach(), dim=0)[0],
    "gated_recurrence, initial": lambda t: torch_convnd.gated_recurrence(
        t.detach(), t.detach(), t[0], dim=0)[0],
}


@pytest.mark.parametrize("name", list(CALLS))
def test_forward_mode_is_refused(name):
    """A tangent would be lost in silence; the refusal comes before the device is looked at."""
    x = torch.ones(4, 8)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(CALLS[name], (x,), (torch.ones_like(x),))
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[name](dual)


@gpu
def test_forward_mode_is_refused_on_the_device():
    x = torch.ones((4, 8), device="cuda")
    for call in CALLS.values():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))


def graphs_over(lengths, call):
    """Graphs that torch.compile makes of `call` over several lengths of a dynamic axis."""
    from torch._dynamo.testing import CompileCounter

    torch._dynamo.reset()
    counter = CompileCounter()
    compiled = torch.compile(call, backend=counter, dynamic=True, fullgraph=True)
    for length in lengths:
        compiled(torch.empty((3, length, 8), device="meta", requires_grad=True))
    torch._dynamo.reset()
    return counter.frame_count


@pytest.mark.parametrize("dim", [1, 2])
def test_recurrence_compiles_once_for_all_lengths(dim):
    def call(x):
        t = x if dim == 1 else x.transpose(1, 2).contiguous()
        return torch_convnd.gated_recurrence(t, t, dim=dim)[0]

    assert graphs_over((65, 130, 300, 777, 1200), call) == 1


def test_recurrence_fake_counts_kept_states_like_the_library():
    from torch_convnd._layers import _kept_states

    count = _native.core().cnd_gated_recurrence_blocks
    for steps in (0, 1, 2, 63, 64, 65, 128, 249, 250, 251, 256, 257, 506, 1000, 1 << 20):
        for inner in (0, 1, 2, 33):
            assert _kept_states(steps, inner) == count(2, 3, steps, inner), (steps, inner)


# ---- C ABI: addresses that no element can have ---------------------------------------------


def abi_cases():
    """(call of test_layers_capi, keyword, address, status): every buffer of every entry point,
    off its elements by half of one, and every workspace off 16 bytes."""
    import test_layers_capi as abi

    half, wide = abi.A + 1, abi.A + 2
    for name in ("x", "w", "b", "y"):
        yield abi.norm_forward, name, half, -1
    yield abi.norm_forward, "stats", wide, -1
    for name in ("dy", "x", "w", "dx", "dw", "db"):
        yield abi.norm_backward, name, half, -1
    yield abi.norm_backward, "stats", wide, -1
    for name in ("x", "w", "b", "residual", "y", "pre"):
        yield abi.linear_forward, name, half, -1
    for name in ("dy", "pre", "x", "w", "dx", "dw", "db"):
        yield abi.linear_backward, name, half, -1
    for name in ("x", "gate", "y"):
        yield abi.recurrence_forward, name, half, -1
    for name in ("initial", "last", "states"):
        yield abi.recurrence_forward, name, wide, -1
    for name in ("dy", "x", "gate", "dx", "dgate"):
        yield abi.recurrence_backward, name, half, -1
    for name in ("dlast", "states", "dinitial"):
        yield abi.recurrence_backward, name, wide, -1
    for run in (abi.norm_backward, abi.linear_backward, abi.recurrence_forward, abi.recurrence_backward):
        yield run, "workspace", abi.A + 8, -4


@pytest.mark.parametrize("run,name,address,status", [
    pytest.param(*case, id=f"{case[0].__name__}-{case[1]}") for case in abi_cases()])
def test_c_abi_refuses_misaligned_buffers(run, name, address, status):
    got, message = run(**{name: address})
    assert got == status and "aligned" in message


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_c_abi_refuses_a_misaligned_linear_workspace(dtype):
    import test_layers_capi as abi

    odd = {"dtype": dtype, "in_features": 63, "x_stride": 63}  # operands are prepared there
    got, message = abi.linear_forward(odd, workspace=abi.A + 8)
    assert got == -4 and "aligned" in message
