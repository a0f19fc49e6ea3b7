"""AdamW whose step runs over all tensors in one native call, with the moments
held in 32 or in 8 bits.

The reference steps Adam through element-wise operators, tensor by tensor
(backends/opengl/dispatch.py:171-179 lerp_, :264-290 addcmul_ / addcdiv_); here
``mm_adamw`` walks every parameter of a group in one pass.
"""

from __future__ import annotations

import array
import copy

import torch

from . import _lib, ops
from .tensor import MatrixManTensor, contiguous_strides, is_contiguous, is_dense, numel

BLOCK = 256  # elements that share a scale of the 8-bit states
_CODES = ("exp_avg_code", "exp_avg_scale", "exp_avg_sq_code", "exp_avg_sq_scale")


_pointer = ops.pointer


def _check_storage(t, name: str) -> MatrixManTensor:
    t = ops.require_mm(t, name)
    ops.require_f32(t, name)
    if not is_dense(t.shape, t._logical_strides):
        raise NotImplementedError(f"MatrixMan/CUDA: {name} must fill its storage span (no strided or expanded views)")
    return t


def _same_order(t: MatrixManTensor, like: MatrixManTensor) -> bool:
    """Whether two dense tensors of one shape keep their elements in one order."""
    return t._logical_strides == like._logical_strides or all(
        n == 1 or a == b for n, a, b in zip(like.shape, t._logical_strides, like._logical_strides))


def _in_order(t: MatrixManTensor, like: MatrixManTensor) -> MatrixManTensor:
    return t if _same_order(t, like) else ops.materialize(t, like._logical_strides)


def run_adamw(rt, rows: list, state_bits: int, *, lr: float, beta1: float, beta2: float, eps: float,
              weight_decay: float, decoupled: bool, maximize: bool, advance: bool) -> None:
    """One native step over ``rows`` of (param, grad, exp_avg, exp_avg_sq,
    exp_avg_scale, exp_avg_sq_scale, step, numel): addresses and a count, laid
    out as mm_adamw_tensor_t."""
    if not rows:
        return
    table = array.array("q", [v for row in rows for v in row])
    ops._launch("mm_adamw", table.buffer_info()[0], len(rows), state_bits, lr, beta1, beta2, eps, weight_decay,
                decoupled, maximize, advance, None, 0, rt.stream)


class AdamW(torch.optim.Optimizer):
    """Decoupled-weight-decay Adam (torch.optim.AdamW's update) in one pass.

    ``state_bits=32`` keeps ``exp_avg`` and ``exp_avg_sq`` as float32 tensors.
    ``state_bits=8`` keeps one byte per element for each, with one float32 scale
    per block of 256 elements: a sign and a 7-bit code for the first moment, an
    8-bit code for the square root of the second (6 % and 3 % largest rounding
    over 16 powers of two).  A non-finite gradient makes the states of its block
    NaN.  ``state_values`` / ``set_state_values`` read and set the moments as
    float32 in either form, and ``state_dict`` holds them so, so a checkpoint
    of one form loads into the other.

    Parameters and gradients are float32 MatrixMan tensors of one device per
    group; a parameter fills its storage span (any order of dimensions) and
    shares it with no other.  The step count lives on the device, so a captured
    step can be replayed; every parameter with a gradient must have its state by
    then (from a step, or set), and lr, betas, eps and weight_decay stay what
    they were at capture."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 maximize: bool = False, state_bits: int = 32):
        if isinstance(lr, torch.Tensor):
            raise NotImplementedError("MatrixMan/CUDA: AdamW takes lr as a number")
        if not lr >= 0.0:
            raise ValueError(f"MatrixMan/CUDA: AdamW lr must be non-negative, got {lr}")
        if not eps >= 0.0:
            raise ValueError(f"MatrixMan/CUDA: AdamW eps must be non-negative, got {eps}")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"MatrixMan/CUDA: AdamW betas must be two numbers in [0, 1), got {betas}")
        if not weight_decay >= 0.0:
            raise ValueError(f"MatrixMan/CUDA: AdamW weight_decay must be non-negative, got {weight_decay}")
        if state_bits not in (32, 8):
            raise ValueError(f"MatrixMan/CUDA: AdamW state_bits must be 32 or 8, got {state_bits}")
        self.state_bits = int(state_bits)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      maximize=bool(maximize)))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        try:
            self._check_params()
        except Exception:
            self.param_groups.pop()
            raise

    def _check_params(self) -> None:
        spans = []
        for group in self.param_groups:
            devices = set()
            for p in group["params"]:
                _check_storage(p, "AdamW parameter")
                devices.add(p.runtime.index)
                if numel(p.shape):
                    start = _pointer(p)
                    spans.append((start, start + 4 * numel(p.shape)))
            if len(devices) > 1:
                raise RuntimeError("MatrixMan/CUDA: AdamW needs one matrixman device per parameter group")
        spans.sort()
        for (_, end), (start, _) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError("MatrixMan/CUDA: AdamW parameters appear twice or share memory")

    # -- state ---------------------------------------------------------------
    def _new_state(self, p: MatrixManTensor) -> dict:
        rt = p.runtime
        if rt.capturing:  # the zeros would be part of the graph, and every replay a first step
            raise RuntimeError("MatrixMan/CUDA: AdamW cannot make a parameter's state during graph capture; take a "
                               "step or set the state (set_state_values, load_state_dict) before capturing")
        state = {"step": ops.full(rt, (), 0.0)}
        if self.state_bits == 32:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = ops.fill_(ops.empty(rt, p.shape, p._logical_strides, kind=_lib.POOL_PARAMETER), 0.0)
        else:
            blocks = (numel(p.shape) + BLOCK - 1) // BLOCK
            for name in ("exp_avg", "exp_avg_sq"):
                # Codes as float32 storage of four each, so that they can be zeroed.
                state[name + "_code"] = ops.fill_(
                    ops.empty(rt, (blocks * BLOCK // 4,), kind=_lib.POOL_PARAMETER), 0.0)
                state[name + "_scale"] = ops.fill_(ops.empty(rt, (blocks,), kind=_lib.POOL_PARAMETER), 0.0)
        return state

    def _state_of(self, p) -> dict:
        state = self.state[p]
        if not state:
            state.update(self._new_state(p))
        return state

    def _check_state(self, p: MatrixManTensor, state: dict) -> dict:
        """A state (the program may have set it) of the kinds and sizes that the
        kernels reach by its addresses."""
        n = numel(p.shape)
        blocks = (n + BLOCK - 1) // BLOCK
        sizes = {"step": 1}
        if self.state_bits == 8:
            sizes.update(zip(_CODES, (blocks * BLOCK // 4, blocks) * 2))
        else:
            sizes.update(exp_avg=n, exp_avg_sq=n)
        for name, size in sizes.items():
            if name not in state:
                raise RuntimeError(f"MatrixMan/CUDA: AdamW state has no {name}")
            t = ops.require_mm(state[name], f"AdamW state {name}")
            ops.require_f32(t, f"AdamW state {name}")
            if t.runtime is not p.runtime:
                raise RuntimeError(f"MatrixMan/CUDA: AdamW state {name} is on another device than its parameter")
            if name in ("exp_avg", "exp_avg_sq"):
                if tuple(t.shape) != tuple(p.shape) or not _same_order(t, p):
                    raise RuntimeError(f"MatrixMan/CUDA: AdamW state {name} must have its parameter's shape and "
                                       f"strides, {tuple(p.shape)} and {p._logical_strides}, got {tuple(t.shape)} "
                                       f"and {t._logical_strides}")
            elif numel(t.shape) != size or not is_contiguous(t.shape, t._logical_strides):
                raise RuntimeError(f"MatrixMan/CUDA: AdamW state {name} must hold {size} dense values, "
                                   f"got {tuple(t.shape)}")
        return state

    def _row(self, p: MatrixManTensor, grad: MatrixManTensor, state: dict) -> tuple:
        self._check_state(p, state)
        if self.state_bits == 8:
            m, v = state["exp_avg_code"], state["exp_avg_sq_code"]
            ms, vs = _pointer(state["exp_avg_scale"]), _pointer(state["exp_avg_sq_scale"])
        else:
            m, v = state["exp_avg"], state["exp_avg_sq"]
            ms = vs = 0
        return (_pointer(p), _pointer(grad), _pointer(m), _pointer(v), ms, vs, _pointer(state["step"]),
                numel(p.shape))

    def _step(self, params: list, states: list, factors: tuple, maximize: bool) -> None:
        """A step whose tensors need checks or copies first."""
        rt = params[0].runtime
        rows, held = [], []
        for p, state in zip(params, states):
            grad = ops.require_mm(p.grad, "AdamW gradient")
            ops.require_f32(grad, "AdamW gradient")
            _check_storage(p, "AdamW parameter")
            if grad.runtime is not rt or p.runtime is not rt:
                raise RuntimeError("MatrixMan/CUDA: AdamW parameter and gradient are on different devices")
            grad = _in_order(grad, p)
            held.append(grad)
            rows.append(self._row(p, grad, state))
        lr, beta1, beta2, eps, weight_decay = factors
        run_adamw(rt, rows, self.state_bits, lr=lr, beta1=beta1, beta2=beta2, eps=eps, weight_decay=weight_decay,
                  decoupled=True, maximize=maximize, advance=True)

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            beta1, beta2 = group["betas"]
            factors = (float(group["lr"]), beta1, beta2, group["eps"], group["weight_decay"])
            states = [self.state.get(p) or self._state_of(p) for p in params]
            if ops.native_call("adamw_step", "mm_adamw", params, states, self.state_bits, *factors,
                               group["maximize"]) is None:
                self._step(params, states, factors, group["maximize"])
            torch.autograd.graph.increment_version(params)
        return loss

    def state_values(self, p) -> tuple[MatrixManTensor, MatrixManTensor]:
        """(exp_avg, exp_avg_sq) of a parameter as new float32 tensors (8-bit
        states: the values that the codes stand for)."""
        state = self._state_of(p)
        if self.state_bits == 8:
            done = ops.native_call("adamw_values", "mm_adamw_decode", p, *(state.get(k) for k in (*_CODES, "step")))
            if done is not None:
                return done
        self._check_state(p, state)
        if self.state_bits == 32:
            return ops.clone(state["exp_avg"]), ops.clone(state["exp_avg_sq"])
        rt, n, shape = p.runtime, numel(p.shape), tuple(p.shape)
        at = (n + 63) // 64 * 64  # both in one block
        owner = rt.new_storage(at + n)
        m, v = (MatrixManTensor._wrap(owner, shape, o, p._logical_strides) for o in (0, at))
        ops._launch("mm_adamw_decode", *(_pointer(state[k]) for k in _CODES), n, _pointer(m), _pointer(v), rt.stream)
        return m, v

    @torch.no_grad()
    def set_state_values(self, p, exp_avg, exp_avg_sq, step=None) -> None:
        """Set a parameter's moments (float32, its shape; CPU or MatrixMan
        tensors) and, if given, its step count."""
        state = self._check_state(p, self._state_of(p))
        rt = p.runtime
        given = []
        for name, t in (("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)):
            if not isinstance(t, MatrixManTensor) and isinstance(t, torch.Tensor) and t.device.type == "cpu":
                t = MatrixManTensor(rt.upload(t.detach().contiguous()), tuple(t.shape), 0,
                                    contiguous_strides(tuple(t.shape)))
            t = ops.require_mm(t, f"AdamW {name}")
            ops.require_f32(t, f"AdamW {name}")
            if t.runtime is not rt:
                raise RuntimeError(f"MatrixMan/CUDA: AdamW {name} is on another matrixman device")
            if tuple(t.shape) != tuple(p.shape):
                raise ValueError(f"MatrixMan/CUDA: AdamW {name} must have its parameter's shape")
            given.append(t)
        if self.state_bits == 32:
            for name, t in zip(("exp_avg", "exp_avg_sq"), given):
                ops.copy_into(t, state[name])
        else:
            m, v = (_in_order(t, p) for t in given)
            ops._launch("mm_adamw_encode", _pointer(m), _pointer(v), numel(p.shape),
                        *(_pointer(state[k]) for k in _CODES), rt.stream)
        if step is not None:
            ops.fill_(state["step"], float(step))

    # -- checkpoints -----------------------------------------------------------
    def state_dict(self) -> dict:
        """torch's optimiser layout with float32 moments on the CPU, whatever
        ``state_bits`` is."""
        packed = super().state_dict()
        params = [p for g in self.param_groups for p in g["params"]]
        index = [i for g in packed["param_groups"] for i in g["params"]]
        packed["state"] = {}
        for i, p in zip(index, params):
            if self.state.get(p):
                m, v = self.state_values(p)
                packed["state"][i] = {"step": self.state[p]["step"].cpu(), "exp_avg": m.cpu(), "exp_avg_sq": v.cpu()}
        return packed

    def load_state_dict(self, state_dict: dict) -> None:
        """Load ``state_dict()`` of this class (either ``state_bits``) or of
        torch.optim.AdamW; what cannot be loaded leaves the optimiser as it was."""
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("MatrixMan/CUDA: AdamW state_dict has other parameter groups")
        index = [i for g in groups for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        if any(g.get("amsgrad") for g in groups):
            raise NotImplementedError("MatrixMan/CUDA: AdamW does not implement amsgrad")
        states, settings = dict(self.state), [dict(g) for g in self.param_groups]
        try:
            # Everything that a group holds, a scheduler's "initial_lr" among it.
            for group, saved in zip(self.param_groups, groups):
                group.update(copy.deepcopy({k: v for k, v in saved.items() if k != "params"}))
            self.state.clear()
            for i, p in zip(index, params):
                saved = state_dict["state"].get(i)
                if saved:
                    step = saved["step"]
                    step = step.cpu() if isinstance(step, MatrixManTensor) else step
                    self.set_state_values(p, saved["exp_avg"], saved["exp_avg_sq"], step=float(step))
        except Exception:
            self.state.clear()
            self.state.update(states)
            for group, before in zip(self.param_groups, settings):
                group.clear()
                group.update(before)
            raise
