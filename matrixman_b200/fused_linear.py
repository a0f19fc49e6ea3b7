"""``matrixman.linear``: a linear layer with bias, activation and residual in one
call, with gradients.

The reference has ``addmm`` only (backends/opengl/ops/matmul.py:262-281), with
the activation and the residual as operators of their own.  Here one native
call computes ``act(x @ weight.T + bias) + residual`` in float32 accuracy, and
its backward pass computes the gradients of all four operands.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .tensor import MatrixManTensor, contiguous_strides, is_contiguous, numel, view_strides

ACTIVATIONS = _lib.LINEAR_ACTS


def _matrix(t: MatrixManTensor, name: str) -> MatrixManTensor:
    """[..., n] as [rows, n] without a copy where the strides allow it."""
    if t.dim() == 2:
        return t
    n = int(t.shape[-1])
    rows = numel(t.shape[:-1])
    if rows == 0 or n == 0 or is_contiguous(t.shape, t._logical_strides):
        return MatrixManTensor(t._owner, (rows, n), t._storage_offset, (n, 1))
    strides = view_strides(t.shape, t._logical_strides, (rows, n))
    if strides is None:
        t = ops.materialize(t)
        strides = (n, 1)
    return MatrixManTensor(t._owner, (rows, n), t._storage_offset, strides)


def _dense_rows(t: MatrixManTensor) -> MatrixManTensor:
    if int(t.shape[1]) > 1 and t._logical_strides[1] != 1:
        return ops.materialize(t)
    return t


def _workspace(rt, m: int, n: int, k: int, backward: bool):
    size = ctypes.c_size_t(0)
    _lib.call("mm_linear_workspace_size", m, n, k, 1 if backward else 0, ctypes.byref(size))
    return rt.new_storage(size.value, torch.uint8, _lib.POOL_SCRATCH) if size.value else None, size.value


def _ref(t):
    return ops._p(t.desc()) if t is not None else None


def _forward(x, weight, bias, residual, act: int, first: bool, keep: bool):
    """(y, z): z is what the activation was applied to (None unless kept)."""
    rt = x.runtime
    m, k = (int(v) for v in x.shape)
    n = int(weight.shape[0])
    y = ops.empty(rt, (m, n))
    z = ops.empty(rt, (m, n)) if keep else None
    work, size = _workspace(rt, m, n, k, False)
    ops._launch("mm_linear", _ref(x), _ref(weight), _ref(bias), _ref(residual), act, 1 if first else 0, _ref(y),
                _ref(z), ctypes.c_void_p(work.pointer) if work else None, size, rt.stream)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, first):
        x2 = _matrix(x, "input")
        r2 = _dense_rows(_matrix(residual, "residual")) if residual is not None else None
        # ReLU's slope can be read off its own output where nothing is added to it.
        own_output = act == ACTIVATIONS["relu"] and residual is None
        y, z = _forward(x2, weight, bias, r2, act, first, act != 0 and not own_output)
        shape = tuple(int(v) for v in x.shape[:-1]) + (int(weight.shape[0]),)
        out = y if x.dim() == 2 else MatrixManTensor(y._owner, shape, 0, contiguous_strides(shape))
        ctx.act, ctx.first, ctx.own_output = act, first, own_output
        ctx.save_for_backward(x, weight, out if own_output else z)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy = ops.require_mm(dy, "linear gradient")
        rt = dy.runtime
        g = _dense_rows(_matrix(dy, "gradient"))
        x2 = _matrix(x, "input")
        m, k = (int(v) for v in x2.shape)
        n = int(weight.shape[0])
        want_dz = need_r and ctx.first
        dx = ops.empty(rt, (m, k)) if need_x else None
        dw = ops.empty(rt, (n, k)) if need_w else None
        db = ops.empty(rt, (n,)) if need_b else None
        dz = ops.empty(rt, (m, n)) if want_dz else None
        if need_x or need_w or need_b or want_dz:
            z2 = _matrix(z, "pre-activation") if z is not None else None
            work, size = _workspace(rt, m, n, k, True)
            ops._launch("mm_linear_backward", _ref(g), _ref(x2), _ref(weight), _ref(z2), ctx.act, _ref(dx), _ref(dw),
                        _ref(db), _ref(dz), ctypes.c_void_p(work.pointer) if work else None, size, rt.stream)
        if dx is not None:
            dx = MatrixManTensor(dx._owner, tuple(x.shape), 0, contiguous_strides(tuple(x.shape)))
        dr = None
        if need_r:
            dr = dy if not ctx.first else MatrixManTensor(dz._owner, tuple(dy.shape), 0,
                                                          contiguous_strides(tuple(dy.shape)))
        return dx, dw, db, dr, None, None


def linear(x, weight, bias=None, *, activation: str | None = None, residual=None,
           residual_before_act: bool = False) -> MatrixManTensor:
    """``act(x @ weight.T + bias) + residual`` in one native call.

    x ``[..., k]``, weight ``[n, k]`` (torch.nn.Linear's layout), bias ``[n]``,
    residual ``[..., n]`` of the output's shape.  activation: None / "none",
    "relu", "silu", "sigmoid", "gelu" or "gelu_tanh".  With
    ``residual_before_act`` the residual is added before the activation.
    Differentiable once in x, weight, bias and residual.  float32 throughout;
    weight and bias may be CPU tensors (uploaded once, as for the other
    operators) when they need no gradient."""
    x = ops.require_mm(x, "linear")
    ops.require_f32(x, "linear")
    act = ACTIVATIONS.get("none" if activation is None else activation)
    if act is None:
        raise ValueError(f"MatrixMan/CUDA: linear activation must be one of {sorted(ACTIVATIONS)}, "
                         f"got {activation!r}")
    rt = x.runtime
    grad = torch.is_grad_enabled()
    operands = []
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and not isinstance(t, MatrixManTensor):
            if grad and isinstance(t, torch.Tensor) and t.requires_grad:
                raise RuntimeError(f"MatrixMan/CUDA: linear {name} needs a gradient and must be a MatrixMan tensor")
            t = ops.device_operand(rt, t, f"linear {name}")
        if t is not None:
            ops.require_f32(t, f"linear {name}")
        operands.append(t)
    weight, bias = operands
    if weight is None or weight.dim() != 2:
        raise ValueError("MatrixMan/CUDA: linear weight must be [n, k]")
    n, k = (int(v) for v in weight.shape)
    if x.dim() < 1 or int(x.shape[-1]) != k:
        raise ValueError(f"MatrixMan/CUDA: linear input {tuple(x.shape)} does not end in the weight's {k}")
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"MatrixMan/CUDA: linear bias must be [{n}], got {tuple(bias.shape)}")
    if residual is not None:
        residual = ops.require_mm(residual, "linear residual")
        ops.require_f32(residual, "linear residual")
        if tuple(residual.shape) != tuple(x.shape[:-1]) + (n,):
            raise ValueError("MatrixMan/CUDA: linear residual must have the output's shape "
                             f"{tuple(x.shape[:-1]) + (n,)}, got {tuple(residual.shape)}")
    ops._runtime_of(x, weight, bias, residual)
    if x.dim() == 1:
        out = linear(x.unsqueeze(0), weight, bias, activation=activation,
                     residual=None if residual is None else residual.unsqueeze(0),
                     residual_before_act=residual_before_act)
        return out.squeeze(0)
    if bias is not None and bias._logical_strides[0] != 1 and n > 1:
        bias = bias.contiguous() if not bias.requires_grad else bias.clone(memory_format=torch.contiguous_format)
    if grad and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _Linear.apply(x, weight, bias, residual, act, bool(residual_before_act))
    x2 = _matrix(x, "input")
    r2 = _dense_rows(_matrix(residual, "residual")) if residual is not None else None
    y, _ = _forward(x2, weight, bias, r2, act, bool(residual_before_act), False)
    if x.dim() == 2:
        return y
    shape = tuple(int(v) for v in x.shape[:-1]) + (n,)
    return MatrixManTensor(y._owner, shape, 0, contiguous_strides(shape))
