"""A recurrent convolution block: the operators of this package together, as a model over
sequences of N-dimensional frames (video, volumes over time) uses them."""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch
from torch import Tensor, nn

from ._geometry import DEFAULT_WORKSPACE_BYTES, _tuple
from ._layers import gated_recurrence, layer_norm, linear
from .modules import ConvNd


class RecurrentConvBlock(nn.Module):
    """Mixes frames in space by a convolution and in time by a gated linear recurrence.

    For frames ``x`` of shape ``[N, T, d_1, ..., d_r, C]`` (``dimensions`` = r spatial axes,
    channels last)::

        u = layer_norm(x)
        c = conv(u)                                  # each frame by itself, 'same' size
        g = linear(u)                                # one gate per channel and position
        h, state = gated_recurrence(c, g, state)     # along T
        x = linear(h) + x
        x = linear(gelu(linear(layer_norm(x)))) + x  # `expansion` * C features inside

    ``forward(x, state=None)`` returns ``(x, state)``. No step looks ahead of its frame, so a
    sequence may be fed in pieces, down to one frame a call, with the state of one call
    passed to the next: a model is trained on whole sequences and served frame by frame.
    ``state`` is ``[N, d_1, ..., d_r, C]``, float32 (float64 for a float64 input).

    Every tensor between the operators is read in the layout it was written in: the
    convolution takes and returns channels-last activations, the other operators work on the
    last dimension or along T.
    """

    def __init__(
        self,
        channels: int,
        kernel_size: int | Sequence[int],
        *,
        dimensions: int,
        expansion: int = 4,
        eps: float = 1e-5,
        device=None,
        dtype=None,
        workspace_bytes: int = DEFAULT_WORKSPACE_BYTES,
    ):
        super().__init__()
        if not isinstance(dimensions, int) or isinstance(dimensions, bool) or not 1 <= dimensions <= 61:
            raise ValueError("dimensions must be an integer from 1 to 61")
        if channels <= 0 or expansion <= 0:
            raise ValueError("channels and expansion must be positive")
        kernel = _tuple(kernel_size, dimensions, "kernel_size")
        if any(k % 2 == 0 for k in kernel):
            raise ValueError("kernel_size must be odd")
        self.channels = channels
        self.dimensions = dimensions
        self.expansion = expansion
        self.eps = eps
        factory = {"device": device, "dtype": dtype}
        self.conv = ConvNd(channels, channels, (1, *kernel), padding=(0, *(k // 2 for k in kernel)),
                           dimensions=dimensions + 1, workspace_bytes=workspace_bytes, **factory)
        inner = expansion * channels
        for name, rows, columns in (("gate", channels, channels), ("out", channels, channels),
                                    ("up", inner, channels), ("down", channels, inner)):
            setattr(self, f"{name}_weight", nn.Parameter(torch.empty(rows, columns, **factory)))
            setattr(self, f"{name}_bias", nn.Parameter(torch.empty(rows, **factory)))
        for name in ("norm1", "norm2"):
            setattr(self, f"{name}_weight", nn.Parameter(torch.empty(channels, **factory)))
            setattr(self, f"{name}_bias", nn.Parameter(torch.empty(channels, **factory)))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        """kaiming-uniform(a=sqrt(5)) weights and U(-1/sqrt(fan_in), 1/sqrt(fan_in)) biases as
        in the convolution, identity norms, and gates that start at sigmoid(1): a memory of
        about four frames."""
        self.conv.reset_parameters()
        for name in ("gate", "out", "up", "down"):
            weight, bias = getattr(self, f"{name}_weight"), getattr(self, f"{name}_bias")
            nn.init.kaiming_uniform_(weight, a=math.sqrt(5))
            bound = 1 / math.sqrt(weight.shape[1])
            nn.init.uniform_(bias, -bound, bound)
        nn.init.ones_(self.gate_bias)
        for name in ("norm1", "norm2"):
            nn.init.ones_(getattr(self, f"{name}_weight"))
            nn.init.zeros_(getattr(self, f"{name}_bias"))

    def forward(self, input: Tensor, state: Tensor | None = None) -> tuple[Tensor, Tensor]:
        if input.ndim != self.dimensions + 3 or input.shape[-1] != self.channels:
            raise ValueError(
                f"expected [N, T, {self.dimensions} spatial axes, {self.channels} channels], "
                f"got {tuple(input.shape)}")
        u = layer_norm(input, self.norm1_weight, self.norm1_bias, self.eps)
        candidate = self.conv(u.movedim(-1, 1)).movedim(1, -1)
        gate = linear(u, self.gate_weight, self.gate_bias)
        hidden, state = gated_recurrence(candidate, gate, state, dim=1)
        x = linear(hidden, self.out_weight, self.out_bias, residual=input)
        v = layer_norm(x, self.norm2_weight, self.norm2_bias, self.eps)
        v = linear(v, self.up_weight, self.up_bias, activation="gelu")
        return linear(v, self.down_weight, self.down_bias, residual=x), state

    def extra_repr(self) -> str:
        return f"{self.channels}, dimensions={self.dimensions}, expansion={self.expansion}"
