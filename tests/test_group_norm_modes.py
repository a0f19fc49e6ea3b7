"""F.group_norm under dispatch modes, most on a runtime that has no device: the modes
see the operators that run, as they do for F.layer_norm."""

import pytest
import torch
import torch.nn.functional as F
from torch.utils._python_dispatch import TorchDispatchMode

import matrixman_b200  # noqa: F401 - registers the operators
from matrixman_b200.tensor import MatrixManTensor

from .test_adamw_states import launches, rt, tensor  # noqa: F401 - fixtures

aten = torch.ops.aten


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.calls = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.calls.append(func)
        return func(*args, **(kwargs or {}))


@pytest.fixture
def maps(rt):  # noqa: F811
    last = tensor(rt, 2, 8, 3, 5, strides=(120, 1, 40, 8))
    return last, tensor(rt, 8), tensor(rt, 8)


@pytest.mark.parametrize("grad", [False, True])
def test_a_mode_sees_the_norm(maps, launches, grad):  # noqa: F811
    x, w, b = (t.requires_grad_(grad) for t in maps)
    with Seen() as seen:
        y = F.group_norm(x, 4, w, b)
    assert aten.native_group_norm.default in seen.calls
    assert launches == ["mm_group_norm"] and isinstance(y, MatrixManTensor) and y.stride() == x.stride()


def test_what_a_mode_returns_is_taken(maps, launches):  # noqa: F811
    """A mode that answers itself, as caching checkpoints do."""
    x, w, b = maps
    other = tensor(x.runtime, 2, 8, 3, 5)

    class Answers(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func is aten.native_group_norm.default:
                return other, tensor(x.runtime, 2, 4), tensor(x.runtime, 2, 4)
            return func(*args, **(kwargs or {}))

    with Answers():
        y = F.group_norm(x, 4, w, b)
    assert y is other or y._owner is other._owner
    assert launches == []


@pytest.mark.gpu
def test_a_mode_sees_the_gradient(mm):
    from .test_group_norm_gpu import EPS, check, inputs, on_device, oracle
    x, w, b, dy = inputs(2, 8, (3, 5), 4, "none")
    want = oracle(x, 4, w, b, dy)
    leaves = [t.detach().requires_grad_(True) for t in (on_device(mm, x, True), mm.to_device(w), mm.to_device(b))]
    with Seen() as seen:
        y = F.group_norm(leaves[0], 4, *leaves[1:], EPS)
        grads = torch.autograd.grad(y, leaves, on_device(mm, dy, True))
    assert [f for f in seen.calls if "group_norm" in str(f)] == [aten.native_group_norm.default,
                                                               aten.native_group_norm_backward.default]
    assert grads[0]._logical_strides == leaves[0]._logical_strides
    for name, got in zip(("y", "dx", "dw", "db"), (y.detach(), *grads)):
        check(name, got.cpu(), want[name])


@pytest.mark.gpu
def test_parameters_on_the_cpu_under_a_mode(mm):
    from .test_group_norm_gpu import EPS, check, inputs, on_device, oracle
    x, w, b, dy = inputs(2, 8, (3, 5), 4, "none")
    want = oracle(x, 4, w, b, dy)
    leaf = on_device(mm, x, True).detach().requires_grad_(True)
    with Seen() as seen:
        y = F.group_norm(leaf, 4, w, b, EPS)
        dx, = torch.autograd.grad(y, leaf, on_device(mm, dy, True))
    assert aten.native_group_norm_backward.default in seen.calls
    check("y", y.detach().cpu(), want["y"])
    check("dx", dx.cpu(), want["dx"])


def test_without_a_mode_nothing_is_dispatched(maps, launches, monkeypatch):  # noqa: F811
    from matrixman_b200 import dispatch
    monkeypatch.delitem(dispatch._HANDLERS, aten.native_group_norm.default)
    F.group_norm(maps[0], 4, *maps[1:])
    assert launches == ["mm_group_norm"]
