"""Group norm's ways of dividing a call, each against the formulas in float64: maps in
one block, in clusters of any size, several images in a block, walking kernels.  The
bounds are those of test_group_norm_gpu.py."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from matrixman_b200 import _lib

from . import test_group_norm_gpu as base
from .test_group_norm_gpu import ACTS, check, inputs, oracle, randn, run
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


def against_the_formulas(mm, n, c, spatial, groups, last, act):
    x, w, b, dy = inputs(n, c, spatial, groups, act)
    want = oracle(x, groups, w, b, dy, act)
    for name, got in zip(NAMES, run(mm, x, groups, w, b, dy, act, last)):
        check(name, got, want[name])


# Groups beyond a cluster's memory, of vectors of four, two and one, in many segments; as
# many segments as the device takes; more columns than a block has.
@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", [(1, 16, (300, 300), 1), (1, 18, (302, 301), 1), (1, 15, (305, 303), 1),
                                                (2, 32, (303, 301), 2), (1, 130, (300, 300), 2), (1, 2060, (41, 40), 1)])
def test_maps_that_only_the_walking_kernels_take(mm, n, c, spatial, groups, last):
    for backward in (0, 1):
        ranks, _, segments = plan(n, c, pixels(spatial), groups, last, backward)
        assert ranks == 0 and segments > 1
    against_the_formulas(mm, n, c, spatial, groups, last, ACTS[(c + last) % len(ACTS)])


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", base.SIZES)
def test_all_sizes_walked(mm, at_most, n, c, spatial, groups, last):
    at_most(0)
    against_the_formulas(mm, n, c, spatial, groups, last, ACTS[(n + c + groups + 1) % len(ACTS)])


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("act", ACTS)
def test_activations_walked(mm, at_most, act, last):
    at_most(0)
    base.test_activations(mm, act, last)


@pytest.mark.parametrize("last", [True, False])
def test_other_cases_walked(mm, at_most, last):
    """Non-finite groups, missing parameters, strides, single gradients, the same bits in a replayed graph."""
    at_most(0)
    base.test_constant_and_non_finite_groups(mm, last)
    for affine in ((True, False), (False, True), (False, False)):
        base.test_without_weight_or_bias(mm, affine, last)
    base.test_strides(mm)
    base.test_only_the_gradients_asked_for(mm)
    base.test_same_bits_twice_and_in_a_replayed_graph(mm, 7, 60, (17, 13), 5, last)
    base.test_torch_functional_and_module(mm, last)


@pytest.mark.parametrize("last", [True, False])
def test_non_finite_values_of_large_maps(mm, last):
    n, c, spatial, groups = 3, 16, (300, 300), 1
    assert plan(n, c, pixels(spatial), groups, last, False)[0] == 0
    x, w, b, dy = inputs(n, c, spatial, groups, "none")
    x[0, 3, 7, 250] = float("nan")
    x[1, 0, 0, 0] = float("inf")
    y, dx, dw, db = run(mm, x, groups, w, b, dy, "none", last)
    assert torch.isnan(y[:2]).all() and torch.isnan(dx[:2]).all() and torch.isnan(dw).all() and torch.isfinite(db).all()
    want = oracle(x[2:], groups, w, b, dy[2:])
    check("y", y[2:], want["y"])
    check("dx", dx[2:], want["dx"])


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", [(1301, 24, (2, 3), 4), (1301, 24, (7,), 4), (4099, 64, (), 8),
                                                (2603, 30, (3,), 5), (5001, 9, (2, 2), 3)])
def test_several_images_in_a_block(mm, n, c, spatial, groups, last):
    """The last block has fewer."""
    for backward in (0, 1):
        ranks, images, _ = plan(n, c, pixels(spatial), groups, last, backward)
        assert ranks == 1 and images > 1 and n % images
    against_the_formulas(mm, n, c, spatial, groups, last, ACTS[c % len(ACTS)])


@pytest.mark.parametrize("walking", [True, False])
@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("offset", [100.0, -1000.0])
@pytest.mark.parametrize("n,c,spatial,groups", [(2, 16, (9, 9), 4), (2, 16, (150, 150), 4), (1, 16, (300, 300), 1),
                                                (1, 15, (305, 303), 1)])
def test_small_spread_far_from_zero(mm, at_most, n, c, spatial, groups, offset, last, walking):
    """What takes the mean's scale is rounded at most 12 times on the way to the mean: a thread's
    own (1), its joins (3 of a vector, 5 of a warp, or 2 and 5 of a block) and the segments' (1), 2
    of x - mean.  So a part's mean is off by E = 12 u |mean|, and the squared distances between
    parts, which are at most the variance, by 4 E sqrt(var) + 4 E^2.  The rest is rounded at the
    spread's scale, as in the general bound."""
    if walking:
        at_most(0)
    x = 0.01 * randn(n, c, *spatial, seed=1) + offset
    y = mm.group_norm(base.on_device(mm, x, last), groups, None, None, base.EPS).cpu().double()
    t = x.double().reshape(n, groups, -1)
    mu = t.mean(2, keepdim=True)
    rstd = 1 / torch.sqrt(((t - mu) ** 2).mean(2, keepdim=True) + base.EPS)
    xh = (t - mu) * rstd
    adds = 160 + t.shape[2] / 16384
    e = 12 * base.U * mu.abs() * rstd
    bound = e + adds * base.U * xh.abs().mean(2, keepdim=True) + (2 * e + 2 * e * e + (adds / 2 + 8) * base.U) * xh.abs()
    assert bound.max() < (0.1 if offset == 100.0 else 1.0)
    check("y", y.reshape(t.shape), (xh, bound))


FIRST_CALL = """
import torch, matrixman_b200 as mm
mm.init()
x = mm.to_device(torch.randn(2, 48, 64, 64))
rt = x.runtime
rt.synchronize()
rt.capture_begin()
y = mm.group_norm(x, 8, activation="silu")
graph = rt.capture_end()
graph.replay()
got = y.cpu()
assert torch.equal(got, mm.group_norm(x, 8, activation="silu").cpu()) and torch.isfinite(got).all()
print("ok")
"""


def test_a_process_whose_first_call_is_captured():
    """Whether a cluster can be placed is asked during the capture."""
    assert plan(2, 48, 4096, 8, False, False)[0] > 1
    done = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parents[1])
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stderr
