"""What group norm's kernels promise beyond the bounds of test_group_norm_gpu.py, of
maps held on chip and of the walking kernels alike.  u = 2^-24."""

import pytest
import torch

from .test_group_norm_gpu import EPS, on_device, randn, run
from .test_group_norm_plan import plan
from .test_group_norm_ways_gpu import pixels

pytestmark = pytest.mark.gpu

# A group beyond a cluster's memory, of vectors of four, two and one.
WALKING = [(1, 16, (300, 300), 1), (1, 18, (302, 301), 1), (1, 15, (305, 303), 1)]


@pytest.mark.parametrize("n,c,spatial,groups", WALKING)
def test_these_walk(n, c, spatial, groups):
    assert all(plan(n, c, pixels(spatial), groups, last, back)[0] == 0 for last in (0, 1) for back in (0, 1))


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", [(2, 48, (64, 64), 8), *WALKING])
@pytest.mark.parametrize("value", [0.1, 1000.1, -3.3e7, 1e34])
def test_a_constant_is_its_own_mean(mm, n, c, spatial, groups, last, value):
    """No spread: y is the bias, whatever the value's bits."""
    b = randn(c, seed=1)
    y = mm.group_norm(on_device(mm, torch.full((n, c, *spatial), value), last), groups, mm.to_device(torch.ones(c)),
                      mm.to_device(b), EPS)
    assert torch.equal(y.cpu(), b.reshape(1, c, 1, 1).expand(n, c, *spatial))


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", [(2, 48, (64, 64), 8), *WALKING])
def test_means_whose_squares_overflow(mm, n, c, spatial, groups, last):
    """Around 1e20, in steps of two of a float's there: the spread's squares are far from
    overflowing, so everything is finite."""
    x = 1e20 + 2.0 ** 44 * randn(n, c, *spatial, seed=2).round()
    assert x.unique().numel() > 5
    got = run(mm, x, groups, torch.ones(c), torch.zeros(c), randn(n, c, *spatial, seed=3), "none", last)
    assert all(torch.isfinite(t).all() for t in got)
