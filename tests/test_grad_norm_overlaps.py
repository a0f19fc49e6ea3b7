"""Which gradients share memory, by strides (host code, on a runtime that has no
device): clipping refuses them, dense or not."""

import itertools
import random

import pytest
import torch

from matrixman_b200 import optim
from matrixman_b200.runtime import DeviceStorage
from matrixman_b200.tensor import MatrixManTensor

from .test_adamw_states import launches, rt  # noqa: F401 - fixtures


def views(rt, *specs):  # noqa: F811
    """Tensors of (shape, strides, offset) over one buffer."""
    storage = DeviceStorage(rt, 1 << 24, 4 * 100000, torch.float32, 0)
    return [MatrixManTensor(storage, shape, offset, strides) for shape, strides, offset in specs]


def clip(tensors):
    params = [torch.nn.Parameter(t.detach()) for t in tensors]
    for p, t in zip(params, tensors):
        p.grad = t
    return optim.clip_grad_norm_(params, 1.0)


SLICE = ((17, 13), (30, 1), 94)


@pytest.mark.parametrize("specs", [
    [SLICE, SLICE],                                     # the same one twice
    [SLICE, ((17, 13), (30, 1), 94 + 12)],              # one column in common
    [SLICE, ((30,), (1,), 300)],                        # a row of the buffer
    [((5, 4), (30, 2), 0), ((3,), (1,), 32)],           # a dense one between its columns
    [((5, 4), (30, 2), 0), ((4, 10), (60, 3), 0)],      # other strides
    [((8,), (1,), 0), SLICE, ((2, 2), (40, 7), 500), ((17, 13), (30, 1), 94 + 30 * 16 + 12)]])
def test_shared_memory_is_refused(rt, launches, specs):  # noqa: F811
    with pytest.raises((ValueError, RuntimeError), match="shares? memory"):
        clip(views(rt, *specs))
    assert "mm_grad_clip" not in launches


@pytest.mark.parametrize("specs", [
    [SLICE, ((17, 13), (30, 1), 94 + 13)],              # neighbouring columns
    [SLICE, ((17, 13), (30, 1), 94 + 30 * 17)],
    [((5, 4), (30, 2), 0), ((5, 4), (30, 2), 1)],       # interleaved
    [((5, 4), (30, 2), 0), ((1,), (1,), 1), ((1,), (1,), 39)],
    [((5, 0), (30, 2), 0), ((5, 4), (30, 2), 0)],
    [((64, 8), (256, 1), 8 * i) for i in range(32)]])
def test_memory_side_by_side_is_taken(rt, launches, specs):  # noqa: F811
    clip(views(rt, *specs))
    assert launches.count("mm_grad_clip") == 1


def test_against_the_addresses_themselves(rt):  # noqa: F811
    rng = random.Random(5)
    for _ in range(2000):
        specs = []
        for _ in range(2):
            shape = tuple(rng.randint(1, 5) for _ in range(rng.randint(0, 3)))
            strides, reach = [], 0
            for n in shape:  # without overlap inside
                strides.append(reach + rng.randint(1, 4))
                reach += (n - 1) * strides[-1]
            order = rng.sample(range(len(shape)), len(shape))
            specs.append((tuple(shape[i] for i in order), tuple(strides[i] for i in order), rng.randint(0, 40)))
        cells = [{o + sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, shape))}
                 for shape, strides, o in specs]
        assert optim._share_memory(*views(rt, *specs)) == bool(cells[0] & cells[1]), specs
