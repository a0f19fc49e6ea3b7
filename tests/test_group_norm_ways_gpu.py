"""Group norm's ways of dividing a call, each against the formulas in float64: maps in
one block, in clusters of any size, several images in a block, walking kernels.  The
bounds are those of test_group_norm_gpu.py."""

import pytest
import torch

from matrixman_b200 import _lib

from .test_group_norm_gpu import ACTS, check, inputs, oracle, run
from .test_group_norm_plan import plan

pytestmark = pytest.mark.gpu

NAMES = ("y", "dx", "dw", "db")


@pytest.fixture
def at_most(mm):
    """Sets the most blocks of a cluster; the default comes back afterwards."""
    rt = mm.to_device(torch.zeros(1)).runtime

    def limit(most):
        _lib.check(rt.lib.mm_debug_group_norm_ranks(rt.index, most))

    yield limit
    limit(-1)


def pixels(spatial):
    count = 1
    for s in spatial:
        count *= s
    return count


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", [(2, 48, (64, 64), 8), (1, 16, (160, 160), 4), (5, 130, (37, 41), 13)])
def test_devices_that_place_no_large_cluster(mm, at_most, n, c, spatial, groups, last):
    """Calls that would take clusters are answered without them, by smaller ones or the
    walking kernels."""
    most = max(plan(n, c, pixels(spatial), groups, last, backward)[0] for backward in (0, 1))
    assert most > 1
    act = ACTS[c % len(ACTS)]
    x, w, b, dy = inputs(n, c, spatial, groups, act)
    want = oracle(x, groups, w, b, dy, act)
    for ranks in range(most):
        at_most(ranks)
        for name, got in zip(NAMES, run(mm, x, groups, w, b, dy, act, last)):
            check(name, got, want[name])
