"""Refusals of the layer entry points of the C ABI: every bad argument is a status and a
message before anything is launched, so no GPU is needed."""

from __future__ import annotations

import ctypes

import pytest

from torch_convnd import _native

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4
F16, BF16, F32, F64 = range(4)
P, I32, I64, SIZE = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
MASK = (I32 * 3)(1, 1, 1)
A = 1 << 20  # an address that is never read: every call below is refused


class Linear(ctypes.Structure):
    _fields_ = [("dtype", I32), ("activation", I32), ("rows", I64), ("in_features", I64),
                ("out_features", I64), ("x_stride", I64)]


def call(name, types, *args):
    library = _native.core()
    function = getattr(library, name)
    function.argtypes, function.restype = types, ctypes.c_int
    status = function(*args)
    library.cnd_last_error.restype = ctypes.c_char_p
    return status, library.cnd_last_error().decode()


def norm_forward(dtype=BF16, param=BF16, rows=4, width=8, stride=8, eps=1e-5, x=A, w=A, b=A, y=A,
                 stats=A):
    return call("cnd_layer_norm_forward",
                [I32, I32, I64, I64, I64, ctypes.c_double, P, P, P, P, P, P],
                dtype, param, rows, width, stride, eps, x, w, b, y, stats, None)


def norm_backward(dtype=BF16, param=BF16, rows=4, width=8, dy_stride=8, x_stride=8, dy=A, x=A, w=A,
                  stats=A, dx=A, dw=A, db=A, mask=MASK, workspace=A, size=1 << 30):
    return call("cnd_layer_norm_backward",
                [I32, I32, I64, I64, I64, I64, P, P, P, P, P, P, P, P, P, SIZE, P],
                dtype, param, rows, width, dy_stride, x_stride, dy, x, w, stats, dx, dw, db, mask,
                workspace, size, None)


def linear_forward(problem=(), x=A, w=A, b=A, residual=None, y=A, pre=None, workspace=A,
                   size=1 << 40, null=False):
    fields = {"dtype": BF16, "activation": 0, "rows": 16, "in_features": 64, "out_features": 64,
              "x_stride": 64, **dict(problem)}
    p = Linear(**fields)
    return call("cnd_linear_forward", [P] * 8 + [SIZE, P], None if null else ctypes.addressof(p),
                x, w, b, residual, y, pre, workspace, size, None)


def linear_backward(problem=(), dy=A, pre=A, x=A, w=A, dx=A, dw=A, db=A, mask=MASK, workspace=A,
                    size=1 << 40):
    fields = {"dtype": BF16, "activation": 1, "rows": 16, "in_features": 64, "out_features": 64,
              "x_stride": 64, **dict(problem)}
    p = Linear(**fields)
    return call("cnd_linear_backward", [P] * 10 + [SIZE, P], ctypes.addressof(p), dy, pre, x, w, dx,
                dw, db, mask, workspace, size, None)


def recurrence_forward(dtype=BF16, outer=2, steps=4096, inner=8, x=A, gate=A, initial=None, y=A,
                       last=A, states=None, workspace=A, size=1 << 40):
    return call("cnd_gated_recurrence_forward",
                [I32, I64, I64, I64, P, P, P, P, P, P, P, SIZE, P], dtype, outer, steps, inner, x,
                gate, initial, y, last, states, workspace, size, None)


def recurrence_backward(dtype=BF16, outer=2, steps=4096, inner=8, dy=A, dlast=A, x=A, gate=A,
                        states=A, dx=A, dgate=A, dinitial=A, mask=MASK, workspace=A, size=1 << 40):
    return call("cnd_gated_recurrence_backward",
                [I32, I64, I64, I64, P, P, P, P, P, P, P, P, P, P, SIZE, P], dtype, outer, steps,
                inner, dy, dlast, x, gate, states, dx, dgate, dinitial, mask, workspace, size, None)


def refused(result, *codes):
    status, message = result
    assert status in codes and message, result


@pytest.mark.parametrize("change", [
    {"dtype": 9}, {"dtype": -1}, {"param": F64}, {"rows": -1}, {"width": 0}, {"width": -3},
    {"stride": 7}, {"eps": -1.0}, {"eps": float("nan")}, {"x": None}, {"y": None}])
def test_layer_norm_forward_refuses(change):
    refused(norm_forward(**change), INVALID, UNSUPPORTED)


@pytest.mark.parametrize("change", [
    {"dtype": 9}, {"param": F64}, {"rows": -1}, {"width": 0}, {"dy_stride": 7}, {"x_stride": 7},
    {"dy": None}, {"x": None}, {"stats": None}, {"dx": None}, {"dw": None}, {"db": None},
    {"mask": None}])
def test_layer_norm_backward_refuses(change):
    refused(norm_backward(**change), INVALID, UNSUPPORTED)


@pytest.mark.parametrize("change", [{"workspace": None}, {"size": 0}])
def test_layer_norm_backward_refuses_a_short_workspace(change):
    refused(norm_backward(**change), INVALID, WORKSPACE)


@pytest.mark.parametrize("problem,change", [
    ({"dtype": 7}, {}), ({"activation": 5}, {}), ({"rows": -1}, {}), ({"in_features": -1}, {}),
    ({"out_features": -1}, {}), ({"x_stride": 63}, {}), ({}, {"x": None}), ({}, {"w": None}),
    ({}, {"y": None}), ({}, {"x": A + 2}), ({}, {"w": A + 8}), ({}, {"null": True})])
def test_linear_forward_refuses(problem, change):
    refused(linear_forward(problem, **change), INVALID, UNSUPPORTED)


@pytest.mark.parametrize("problem,change", [
    ({"dtype": 7}, {}), ({"activation": -1}, {}), ({"rows": -1}, {}), ({"x_stride": 63}, {}),
    ({}, {"dy": None}), ({}, {"pre": None}), ({}, {"x": None}), ({}, {"w": None}),
    ({}, {"dx": None}), ({}, {"dw": None}), ({}, {"db": None}), ({}, {"mask": None}),
    ({}, {"dy": A + 2}), ({}, {"dx": A + 2}), ({}, {"w": A + 4})])
def test_linear_backward_refuses(problem, change):
    refused(linear_backward(problem, **change), INVALID, UNSUPPORTED)


def test_linear_refuses_a_short_workspace():
    odd = {"dtype": F32, "in_features": 63, "x_stride": 63}  # operands are prepared there
    refused(linear_forward(odd, size=16), INVALID, WORKSPACE)
    refused(linear_forward(odd, workspace=None), INVALID, WORKSPACE)
    refused(linear_backward(size=16), INVALID, WORKSPACE)
    refused(linear_backward(workspace=None), INVALID, WORKSPACE)


@pytest.mark.parametrize("change", [
    {"dtype": 9}, {"outer": -1}, {"steps": -1}, {"inner": -1}, {"x": None}, {"gate": None},
    {"y": None}, {"last": None}])
def test_recurrence_forward_refuses(change):
    refused(recurrence_forward(**change), INVALID, UNSUPPORTED)


@pytest.mark.parametrize("change", [
    {"dtype": 9}, {"outer": -1}, {"steps": -1}, {"inner": -1}, {"x": None}, {"gate": None},
    {"states": None}, {"dx": None}, {"dgate": None}, {"dinitial": None}, {"mask": None}])
def test_recurrence_backward_refuses(change):
    refused(recurrence_backward(**change), INVALID, UNSUPPORTED)


@pytest.mark.parametrize("run", [recurrence_forward, recurrence_backward])
@pytest.mark.parametrize("change", [{"workspace": None}, {"size": 16}])
def test_recurrence_refuses_a_short_workspace(run, change):
    refused(run(**change), INVALID, WORKSPACE)
