"""Layer norm, fused linear layers and the gated linear recurrence.

The operators that stand around convolutions in sequence and volume models, on the same
native library: ``layer_norm`` and ``linear`` work on the last dimension (for a
channels-last activation ``x`` of shape ``[N, C, d...]`` that is ``x.movedim(1, -1)``, a
view), ``gated_recurrence`` along any axis. The native shim registers their CUDA, CPU
(validation, then refusal) and autograd kernels; the schemas and fake kernels are here.
"""

from __future__ import annotations

import torch
from torch import Tensor

from ._native import is_loaded, load_native

ACTIVATIONS = (None, "gelu", "silu")

SCHEMAS = (
    "layer_norm(Tensor input, Tensor? weight, Tensor? bias, float eps) -> Tensor",
    "layer_norm_train(Tensor input, Tensor? weight, Tensor? bias, float eps) "
    "-> (Tensor, Tensor)",
    "layer_norm_backward(Tensor grad_output, Tensor input, Tensor? weight, Tensor? bias, "
    "Tensor stats, bool[3] output_mask) -> (Tensor?, Tensor?, Tensor?)",
    "linear(Tensor input, Tensor weight, Tensor? bias, Tensor? residual, str activation) "
    "-> Tensor",
    "linear_train(Tensor input, Tensor weight, Tensor? bias, Tensor? residual, "
    "str activation) -> (Tensor, Tensor)",
    "linear_backward(Tensor grad_output, Tensor pre, Tensor input, Tensor weight, "
    "str activation, bool[3] output_mask) -> (Tensor?, Tensor?, Tensor?)",
    "gated_recurrence(Tensor input, Tensor gate, Tensor? initial, int dim) "
    "-> (Tensor, Tensor)",
    "gated_recurrence_train(Tensor input, Tensor gate, Tensor? initial, int dim) "
    "-> (Tensor, Tensor, Tensor)",
    "gated_recurrence_backward(Tensor? grad_output, Tensor? grad_last, Tensor input, "
    "Tensor gate, Tensor states, int dim, bool[3] output_mask) "
    "-> (Tensor?, Tensor?, Tensor?)",
)


def layer_norm(
    input: Tensor,
    weight: Tensor | None = None,
    bias: Tensor | None = None,
    eps: float = 1e-5,
) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    Statistics and sums are float32 (float64 for a float64 input). ``weight`` and ``bias``
    are vectors of the last dimension's size, of the input's dtype or float32. The result is
    contiguous; an input whose rows have unit stride and one common distance is read in
    place. ``eps`` must not be negative. First derivatives only, in reverse mode.
    """
    if not is_loaded():
        load_native()
    return torch.ops.torch_convnd.layer_norm.default(input, weight, bias, eps)


def linear(
    input: Tensor,
    weight: Tensor,
    bias: Tensor | None = None,
    *,
    activation: str | None = None,
    residual: Tensor | None = None,
) -> Tensor:
    """``act(input @ weight.T + bias) + residual`` in one pass over the output.

    ``input`` is ``[..., in_features]``, ``weight`` ``[out_features, in_features]``,
    ``residual`` has the output's shape; all share one dtype (autocast casts them).
    ``activation`` is None, ``'gelu'`` (exact) or ``'silu'``. Products accumulate in
    float32; float32 operands keep float32 accuracy. For the backward of an activation, the
    value before it and its gradient are kept in the tensors' dtype: in 16 bits, gradients are
    about half again as far from exact as with both in float32, for half the traffic. First
    derivatives only, in reverse mode.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"Invalid activation {activation!r}; expected None, 'gelu' or 'silu'")
    if not is_loaded():
        load_native()
    return torch.ops.torch_convnd.linear.default(
        input, weight, bias, residual, "none" if activation is None else activation)


def gated_recurrence(
    input: Tensor,
    gate: Tensor,
    initial: Tensor | None = None,
    *,
    dim: int,
) -> tuple[Tensor, Tensor]:
    """``h_t = f_t * h_{t-1} + (1 - f_t) * x_t`` along ``dim``, ``f = sigmoid(gate)``.

    Returns every state (the input's shape, dtype and memory order) and the last one (the
    shape without ``dim``, float32, or float64 for a float64 input). ``initial`` is the state
    before the first step, of the last state's shape and dtype (default zeros), so a sequence
    can be continued call by call, one step at a time or many. A gate of ``-inf`` restarts its
    column, ``+inf`` holds it (of finite states and inputs). First derivatives only, in reverse
    mode.
    """
    if not is_loaded():
        load_native()
    return torch.ops.torch_convnd.gated_recurrence.default(input, gate, initial, dim)


# ---- fake kernels ----------------------------------------------------------------------


def _wide(input):
    return torch.float64 if input.dtype == torch.float64 else torch.float32


def _fake_norm(input, weight, bias, eps):
    return input.new_empty(input.shape)


def _fake_norm_train(input, weight, bias, eps):
    rows = input.numel() // input.shape[-1]
    return input.new_empty(input.shape), input.new_empty((2, rows), dtype=_wide(input))


def _fake_norm_backward(grad_output, input, weight, bias, stats, output_mask):
    params = weight if weight is not None else bias if bias is not None else input
    width = input.shape[-1]
    return (input.new_empty(input.shape) if output_mask[0] else None,
            params.new_empty((width,)) if output_mask[1] else None,
            params.new_empty((width,)) if output_mask[2] else None)


def _fake_linear(input, weight, bias, residual, activation):
    return input.new_empty((*input.shape[:-1], weight.shape[0]))


def _fake_linear_train(input, weight, bias, residual, activation):
    output = _fake_linear(input, weight, bias, residual, activation)
    return output, input.new_empty((0,)) if activation == "none" else torch.empty_like(output)


def _fake_linear_backward(grad_output, pre, input, weight, activation, output_mask):
    return (input.new_empty(input.shape) if output_mask[0] else None,
            weight.new_empty(weight.shape) if output_mask[1] else None,
            weight.new_empty((weight.shape[0],)) if output_mask[2] else None)


def _dense_like(input):
    """An empty tensor in the input's memory order, contiguous if the input is not dense."""
    like = torch.empty_like(input, memory_format=torch.preserve_format)
    # preserve_format takes a dense input's strides as they are, and packs any other's in the
    # order of its strides, where the native kernels work on a contiguous copy
    same = all(size == 1 or ours == theirs
               for size, ours, theirs in zip(input.shape, like.stride(), input.stride()))
    return like if same else input.new_empty(input.shape)


def _state_like(input, dim):
    """A state: the input without ``dim``, in the same memory order (contiguous if empty)."""
    dense = _dense_like(input)
    dim = dim % input.ndim
    if input.numel() == 0:
        return input.new_empty((*input.shape[:dim], *input.shape[dim + 1:]), dtype=_wide(input))
    steps, own = dense.shape[dim], dense.stride(dim)
    sizes, strides = [], []
    for d in range(input.ndim):
        if d != dim:
            size, stride = dense.shape[d], dense.stride(d)
            outside = steps > 1 and size > 1 and stride > own
            sizes.append(size)
            strides.append(stride // steps if outside else stride)
    return input.new_empty_strided(sizes, strides, dtype=_wide(input))


def _fake_recurrence(input, gate, initial, dim):
    return _dense_like(input), _state_like(input, dim)


def _kept_states(steps, inner):
    """cnd_gated_recurrence_blocks(), in arithmetic that sizes known only as symbols go through."""
    if steps == 0:
        return 0
    return (steps + 6) // 256 + 1 if inner == 1 and steps > 1 else (steps - 1) // 64 + 1


def _fake_recurrence_train(input, gate, initial, dim):
    last = _state_like(input, dim)
    dense = _dense_like(input)
    steps, own = dense.shape[dim], dense.stride(dim)
    inner = 1
    for d, (size, stride) in enumerate(zip(dense.shape, dense.stride())):
        if d != dim % input.ndim and not (steps > 1 and size > 1 and stride > own):
            inner *= size
    return dense, last, input.new_empty((_kept_states(steps, inner), last.numel()), dtype=_wide(input))


def _fake_recurrence_backward(grad_output, grad_last, input, gate, states, dim, output_mask):
    return (_dense_like(input) if output_mask[0] else None,
            _dense_like(input) if output_mask[1] else None,
            _state_like(input, dim) if output_mask[2] else None)


def define(library) -> None:
    """Define the schemas, first-call loaders and fake kernels on the operator library."""
    from ._operators import _first_call

    for schema in SCHEMAS:
        library.define(schema)
        name = schema.partition("(")[0]
        library.impl(name, _first_call(name), "CompositeExplicitAutograd")
    for name, fake in {
        "layer_norm": _fake_norm,
        "layer_norm_train": _fake_norm_train,
        "layer_norm_backward": _fake_norm_backward,
        "linear": _fake_linear,
        "linear_train": _fake_linear_train,
        "linear_backward": _fake_linear_backward,
        "gated_recurrence": _fake_recurrence,
        "gated_recurrence_train": _fake_recurrence_train,
        "gated_recurrence_backward": _fake_recurrence_backward,
    }.items():
        torch.library.register_fake(f"torch_convnd::{name}")(fake)
