"""``matrixman.linear``: a linear layer with bias, activation and residual in one
call, with gradients.

The reference has ``addmm`` only (backends/opengl/ops/matmul.py:262-281), with
the activation and the residual as operators of their own.  Here one native
call computes ``act(x @ weight.T + bias) + residual`` in float32 accuracy, and
its backward pass computes the gradients of all four operands.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .privateuse import native_calls
from .tensor import MatrixManTensor, is_contiguous, numel, view_strides

ACTIVATIONS = _lib.LINEAR_ACTS
_RELU = ACTIVATIONS["relu"]
pointer = ops.pointer


def _matrix(t: MatrixManTensor) -> tuple[MatrixManTensor, int, tuple]:
    """[..., n] as a matrix of rows: a tensor, the number of rows, and the two
    strides; copied only where the strides force it."""
    st = t._logical_strides
    if len(st) == 2:
        return t, int(t.shape[0]), st
    shape = tuple(t.shape)
    n = shape[-1]
    rows = numel(shape[:-1])
    if rows == 0 or n == 0 or is_contiguous(shape, st):
        return t, rows, (n, 1)
    flat = view_strides(shape, st, (rows, n))
    if flat is not None:
        return t, rows, flat
    return ops.materialize(t), rows, (n, 1)


def _dense_rows(t: MatrixManTensor) -> tuple[MatrixManTensor, int]:
    """The same with dense rows: a tensor and the rows' distance."""
    m, _, st = _matrix(t)
    n = int(t.shape[-1])
    if n > 1 and st[1] != 1:
        return ops.materialize(t), n
    return m, st[0]


def _forward(x, weight, bias, residual, act: int, first: bool, keep: bool):
    """(y, z) of the output's shape: z is what the activation was applied to
    (None unless kept)."""
    done = ops.native_call("linear", "mm_linear", x, weight, bias, residual, act, first, keep)
    if done is not None:
        return done
    rt = x.runtime
    x2, m, xs = _matrix(x)
    n, k = weight.shape
    ws = weight._logical_strides
    r2, rs = (None, 0) if residual is None else _dense_rows(residual)
    shape = tuple(x.shape[:-1]) + (n,)
    y = ops.new_dense(rt, shape)
    z = ops.new_dense(rt, shape) if keep else None
    ops._launch("mm_linear", pointer(x2), xs[0], xs[1], pointer(weight), ws[0], ws[1],
                None if bias is None else pointer(bias), None if r2 is None else pointer(r2), rs, m, n, k, act,
                first, y._owner.pointer, None if z is None else z._owner.pointer, None, 0, rt.stream)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, first):
        # ReLU's slope can be read off its own output where nothing is added to it.
        own_output = act == _RELU and residual is None
        y, z = _forward(x, weight, bias, residual, act, first, act != 0 and not own_output)
        ctx.act, ctx.first = act, first
        ctx.save_for_backward(x, weight, y if own_output else z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        want_z = need_r and ctx.first
        if need_x or need_w or need_b or want_z:
            done = ops.native_call("linear_backward", "mm_linear_backward", dy, x, weight, z, ctx.act, need_x, need_w,
                                   need_b, want_z)
            if done is not None:
                dx, dw, db, dz = done
                return dx, dw, db, dz if ctx.first else (dy if need_r else None), None, None
        dy = ops.require_mm(dy, "linear gradient")
        rt = dy.runtime
        n, k = weight.shape
        dx = ops.new_dense(rt, tuple(x.shape)) if need_x else None
        dw = ops.new_dense(rt, (n, k)) if need_w else None
        db = ops.new_dense(rt, (n,)) if need_b else None
        dz = ops.new_dense(rt, tuple(dy.shape)) if want_z else None
        if need_x or need_w or need_b or dz is not None:
            g, gs = _dense_rows(dy)
            x2, m, xs = _matrix(x)
            ws = weight._logical_strides
            ops._launch("mm_linear_backward", pointer(g), gs, pointer(x2), xs[0], xs[1], pointer(weight), ws[0], ws[1],
                        None if z is None else pointer(z), m, n, k, ctx.act,
                        *(None if t is None else t._owner.pointer for t in (dx, dw, db, dz)), None, 0, rt.stream)
        dr = None
        if need_r:
            dr = dz if ctx.first else dy
        return dx, dw, db, dr, None, None


def _operand(x, t, name: str, grad: bool) -> MatrixManTensor:
    if isinstance(t, MatrixManTensor):
        if t.runtime is not x.runtime:
            raise RuntimeError(f"MatrixMan/CUDA: linear {name} is on another matrixman device")
    else:
        if grad and isinstance(t, torch.Tensor) and t.requires_grad:
            raise RuntimeError(f"MatrixMan/CUDA: linear {name} needs a gradient and must be a MatrixMan tensor")
        t = ops.device_operand(x.runtime, t, f"linear {name}")
    ops.require_f32(t, f"linear {name}")
    return t


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
    act = ACTIVATIONS.get(activation) if activation is not None else 0
    if act is None:
        raise ValueError(f"MatrixMan/CUDA: linear activation must be one of {sorted(ACTIVATIONS)}, "
                         f"got {activation!r}")
    grad = torch.is_grad_enabled()
    first = bool(residual_before_act)
    if grad:
        native = native_calls()
        if native is not None and native.linear_ready(x, weight, bias, residual):
            if x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or (
                    residual is not None and residual.requires_grad):
                return _Linear.apply(x, weight, bias, residual, act, first)
            return _forward(x, weight, bias, residual, act, first, False)[0]
    else:
        done = ops.native_call("linear", "mm_linear", x, weight, bias, residual, act, first, False)
        if done is not None:
            return done[0]
    # Everything but the ordinary case: CPU parameters, strides that take a copy, and what is refused.
    x = ops.require_mm(x, "linear")
    ops.require_f32(x, "linear")
    weight = _operand(x, weight, "weight", grad)
    if bias is not None:
        bias = _operand(x, bias, "bias", grad)
    if weight.dim() != 2:
        raise ValueError("MatrixMan/CUDA: linear weight must be [n, k]")
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"MatrixMan/CUDA: linear input {tuple(x.shape)} does not end in the weight's {k}")
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"MatrixMan/CUDA: linear bias must be [{n}], got {tuple(bias.shape)}")
        if bias._logical_strides[0] != 1 and n > 1:
            bias = bias.clone(memory_format=torch.contiguous_format)
    if residual is not None:
        residual = ops.require_mm(residual, "linear residual")
        ops.require_f32(residual, "linear residual")
        if tuple(residual.shape) != tuple(x.shape[:-1]) + (n,):
            raise ValueError("MatrixMan/CUDA: linear residual must have the output's shape "
                             f"{tuple(x.shape[:-1]) + (n,)}, got {tuple(residual.shape)}")
        if residual.runtime is not x.runtime:
            raise RuntimeError("MatrixMan/CUDA: linear residual is on another matrixman device")
    if x.dim() == 1:
        out = linear(x.unsqueeze(0), weight, bias, activation=activation,
                     residual=None if residual is None else residual.unsqueeze(0),
                     residual_before_act=residual_before_act)
        return out.squeeze(0)
    if grad and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                 (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act, first)
    return _forward(x, weight, bias, residual, act, first, False)[0]
