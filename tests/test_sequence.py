"""RecurrentConvBlock against the same block of plain torch operations in float64.

Tolerances. A float64 block differs by the rounding of its sums, held to the project's 1e-9
relative bound. A bfloat16 block rounds each of its eight intermediate results to 2^-9
relative (twice that in the gradients, which also pass through rounded forward values), so
its relative L2 error stays below 8 * 2^-8, its gradients' below 16 * 2^-8.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import torch_convnd
from tolerances import relative_l2

gpu = pytest.mark.gpu

BOUNDS = {torch.float64: (1e-9, 1e-9), torch.bfloat16: (8 * 2.0**-8, 16 * 2.0**-8)}


def plain_block(block, x, state=None):
    """The block's formula, in the type of its parameters."""
    width = (block.channels,)
    u = F.layer_norm(x, width, block.norm1_weight, block.norm1_bias, block.eps)
    weight = block.conv.weight
    conv = {1: F.conv1d, 2: F.conv2d, 3: F.conv3d}[block.dimensions]
    frames = u.flatten(0, 1).movedim(-1, 1)
    c = conv(frames, weight.squeeze(2), block.conv.bias,
             padding=tuple(k // 2 for k in weight.shape[3:]))
    c = c.movedim(1, -1).reshape(u.shape)
    f = torch.sigmoid(F.linear(u, block.gate_weight, block.gate_bias))
    h = torch.zeros_like(x[:, 0]) if state is None else state
    steps = []
    for t in range(x.shape[1]):
        h = f[:, t] * h + (1 - f[:, t]) * c[:, t]
        steps.append(h)
    x = F.linear(torch.stack(steps, 1), block.out_weight, block.out_bias) + x
    v = F.layer_norm(x, width, block.norm2_weight, block.norm2_bias, block.eps)
    v = F.gelu(F.linear(v, block.up_weight, block.up_bias))
    return F.linear(v, block.down_weight, block.down_bias) + x, h


def make(channels, kernel, dimensions, dtype):
    torch.manual_seed(5)
    wide = torch_convnd.RecurrentConvBlock(
        channels, kernel, dimensions=dimensions, device="cuda", dtype=torch.float64)
    block = torch_convnd.RecurrentConvBlock(
        channels, kernel, dimensions=dimensions, device="cuda", dtype=dtype)
    block.load_state_dict(wide.state_dict())
    wide.load_state_dict(block.state_dict())  # the rounded values
    return block, wide


@gpu
@pytest.mark.parametrize("dtype", list(BOUNDS))
@pytest.mark.parametrize("shape,kernel", [
    ((2, 5, 9, 16), 3), ((1, 33, 6, 7, 32), (3, 5)), ((2, 4, 5, 6, 7, 24), 3), ((1, 1, 4, 4, 8), 1)])
def test_block(shape, kernel, dtype):
    block, wide = make(shape[-1], kernel, len(shape) - 3, dtype)
    x = torch.randn(shape, device="cuda", dtype=dtype)
    state = torch.randn(shape[:1] + shape[2:], device="cuda", dtype=torch.float32)
    state = state.double() if dtype == torch.float64 else state
    dy = torch.randn(shape, device="cuda", dtype=dtype)
    got_in = [x.clone().requires_grad_(), state.clone().requires_grad_()]
    ref_in = [x.double().requires_grad_(), state.double().requires_grad_()]
    got, got_state = block(*got_in)
    ref, ref_state = plain_block(wide, *ref_in)
    forward, backward = BOUNDS[dtype]
    assert relative_l2(got, ref) <= forward
    assert relative_l2(got_state, ref_state) <= forward
    grads = torch.autograd.grad([got, got_state], [*got_in, *block.parameters()],
                                [dy, torch.ones_like(got_state)])
    refs = torch.autograd.grad([ref, ref_state], [*ref_in, *wide.parameters()],
                               [dy.double(), torch.ones_like(ref_state)])
    names = ["input", "state", *(name for name, _ in block.named_parameters())]
    for name, g, r in zip(names, grads, refs):
        assert relative_l2(g, r) <= backward, name


@gpu
@pytest.mark.parametrize("dtype", list(BOUNDS))
@pytest.mark.parametrize("pieces", [(1, 1, 1, 1, 1, 1), (4, 2), (1, 5)])
def test_frames_served_in_pieces_match_the_sequence(pieces, dtype):
    block, _ = make(32, 3, 2, dtype)
    x = torch.randn(2, sum(pieces), 8, 9, 32, device="cuda", dtype=dtype)
    with torch.no_grad():
        whole, last = block(x)
        state, outputs = None, []
        for piece in x.split(pieces, dim=1):
            y, state = block(piece, state)
            outputs.append(y)
    assert relative_l2(torch.cat(outputs, 1), whole) <= BOUNDS[dtype][0]
    assert relative_l2(state, last) <= BOUNDS[dtype][0]


@gpu
def test_block_trains():
    block, _ = make(16, 3, 2, torch.bfloat16)
    x = torch.randn(2, 8, 6, 6, 16, device="cuda", dtype=torch.bfloat16)
    target = torch.roll(x, 1, dims=1)
    optimizer = torch.optim.Adam(block.parameters(), lr=3e-3)
    losses = []
    for _ in range(30):
        loss = F.mse_loss(block(x)[0].float(), target.float())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss))
    assert losses[-1] < 0.8 * losses[0]


def test_block_shapes_without_a_gpu():
    block = torch_convnd.RecurrentConvBlock(
        8, (3, 5), dimensions=2, expansion=2, device="meta", dtype=torch.bfloat16)
    y, state = block(torch.empty(2, 3, 6, 7, 8, device="meta", dtype=torch.bfloat16))
    assert y.shape == (2, 3, 6, 7, 8) and y.dtype == torch.bfloat16
    assert state.shape == (2, 6, 7, 8) and state.dtype == torch.float32
    assert block.conv.weight.shape == (8, 8, 1, 3, 5)
    assert block.up_weight.shape == (16, 8) and block.down_weight.shape == (8, 16)


@pytest.mark.parametrize("change,message", [
    ({"dimensions": 0}, "dimensions"), ({"dimensions": 62}, "dimensions"),
    ({"dimensions": True}, "dimensions"), ({"channels": 0}, "positive"),
    ({"expansion": 0}, "positive"), ({"kernel_size": 2}, "odd"),
    ({"kernel_size": (3,)}, "kernel_size")])
def test_block_refuses(change, message):
    arguments = {"channels": 8, "kernel_size": 3, "dimensions": 2, "device": "meta", **change}
    with pytest.raises(ValueError, match=message):
        torch_convnd.RecurrentConvBlock(**arguments)


@pytest.mark.parametrize("shape", [(2, 3, 6, 8), (2, 3, 6, 7, 9), (2, 3, 6, 7, 8, 8)])
def test_block_refuses_other_shapes(shape):
    block = torch_convnd.RecurrentConvBlock(8, 3, dimensions=2, device="meta")
    with pytest.raises(ValueError, match="expected"):
        block(torch.empty(shape, device="meta"))
