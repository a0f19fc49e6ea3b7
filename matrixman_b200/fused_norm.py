"""``matrixman.group_norm``: group norm with the activation that follows it, in one
call, with gradients.

The reference normalises with eval BatchNorm only (backends/cuda/batch_norm.py)
and runs the activation as an operator of its own.  Here one native call reads
the feature maps and writes ``act(group_norm(x))`` in their memory order, and its
backward pass computes the gradients of the maps and both parameters.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .tensor import MatrixManTensor, numel


aten = torch.ops.aten


def _dispatched(x, act: int) -> tuple | None:
    """The sizes that ATen's operators take, where a dispatch mode is on (counters, tracing,
    selective checkpoints): it has to see the norm, so the call goes through the dispatcher
    instead of straight to the native one.  ATen has no form with an activation."""
    if act or not torch._C._len_torch_dispatch_stack():
        return None
    shape = tuple(x.shape)
    return (*shape[:2], numel(shape[2:])) if len(shape) >= 2 else None


def _forward(x, groups, weight, bias, eps, act, keep=True):
    sizes = _dispatched(x, act)
    if sizes is not None:
        return aten.native_group_norm.default(x, weight, bias, *sizes, groups, eps)
    return ops.group_norm(x, groups, weight, bias, eps, act, keep)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, mean, rstd = _forward(x, groups, weight, bias, eps, act)
        ctx.groups, ctx.act = groups, act
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        mask = ctx.needs_input_grad[:3]
        sizes = _dispatched(x, ctx.act)
        if sizes is not None:
            got = aten.native_group_norm_backward.default(dy, x, mean, rstd, weight, *sizes, ctx.groups, mask)
        else:
            got = ops.group_norm_backward(dy, x, mean, rstd, weight, bias, ctx.groups, mask, ctx.act)
        return (*got, None, None, None)


def _torch_group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, cudnn_enabled=True):
    """torch.nn.functional.group_norm on MatrixMan tensors.  ATen's own composite
    copies channels-last maps and gradients to channels first in its backward pass."""
    ops.require_mm(x, "GroupNorm")
    if torch.is_grad_enabled():
        need = [t for t in (x, weight, bias) if t is not None and t.requires_grad]
        if not all(isinstance(t, MatrixManTensor) for t in need):
            # Parameters on the CPU: ATen's autograd knows which gradients are asked for.
            shape = tuple(x.shape)
            return torch.native_group_norm(x, weight, bias, *shape[:2], numel(shape[2:]), num_groups, eps)[0]
        if need:
            return _GroupNorm.apply(x, weight, bias, num_groups, eps, 0)
    return _forward(x, num_groups, weight, bias, eps, 0, keep=False)[0]


_library = torch.library.Library("aten", "IMPL", "AutogradPrivateUse1")
_library.impl("group_norm", _torch_group_norm)


def group_norm(x, num_groups: int, weight=None, bias=None, eps: float = 1e-5, *,
               activation: str | None = None) -> MatrixManTensor:
    """``act(torch.nn.functional.group_norm(x, num_groups, weight, bias, eps))`` in one
    native call.

    x ``[N, C, *]`` with any number of spatial dimensions, channels last in memory
    (the order of prepared models; read and written once) or first; other strides
    are copied to channels last.  The result has x's order.  activation: None /
    "none", "relu", "silu", "sigmoid", "gelu" or "gelu_tanh".  Differentiable once
    in x, weight and bias.  float32 throughout; weight and bias may be CPU tensors
    (uploaded once, as for the other operators) when they need no gradient.

    SiLU, sigmoid and tanh-GELU (and their slopes) use the device's approximations of
    2^x and 1 / x.  Relative to the exact value at z the activations are off by at most
    1.5 (|t| + 2) 2^-24 + 2^-20, where t is what the exponential is taken of (z, but for
    GELU, which has 4.5 in place of 1.5), so their last bits differ from
    `matrixman.linear`'s."""
    act = _lib.LINEAR_ACTS.get(activation) if activation is not None else 0
    if act is None:
        raise ValueError(f"MatrixMan/CUDA: group_norm activation must be one of {sorted(_lib.LINEAR_ACTS)}, "
                         f"got {activation!r}")
    ops.require_mm(x, "group_norm")
    if torch.is_grad_enabled():
        need = x.requires_grad
        for name, t in (("weight", weight), ("bias", bias)):
            if isinstance(t, torch.Tensor) and t.requires_grad:
                need = True
                if not isinstance(t, MatrixManTensor):
                    raise RuntimeError(f"MatrixMan/CUDA: group_norm {name} needs a gradient and must be a MatrixMan "
                                       "tensor")
        if need:
            return _GroupNorm.apply(x, weight, bias, int(num_groups), float(eps), act)
    return _forward(x, int(num_groups), weight, bias, float(eps), act, keep=False)[0]
