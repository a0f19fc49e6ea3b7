"""What group norm's kernels promise beyond the bounds of test_group_norm_gpu.py, of
maps held on chip and of the walking kernels alike.  u = 2^-24."""

import pytest
import torch

from matrixman_b200 import ops

from .test_group_norm_gpu import EPS, U, check, inputs, on_device, randn, run
from .test_group_norm_plan import plan
from .test_group_norm_ways_gpu import at_most, pixels  # noqa: F401 - a fixture

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


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("walking", [True, False])
def test_relu_passes_the_gradients_of_what_it_let_through(mm, at_most, last, walking):  # noqa: F811
    """Each channel's bias cancels its first pixel to within a rounding of 0."""
    if walking:
        at_most(0)
    n, c, groups = 1, 1024, 32
    x, w, _, _ = inputs(n, c, (8, 8), groups, "none")
    first = mm.group_norm(on_device(mm, x, last), groups, mm.to_device(w), None, EPS).cpu()[0, :, 0, 0]
    dy = torch.zeros(n, c, 8, 8)
    dy[0, :, 0, 0] = 1.0
    y, _, _, db = run(mm, x, groups, w, -first, dy, "relu", last)
    let = y[0, :, 0, 0] > 0
    assert 100 < let.sum() < 924
    assert torch.equal(db > 0, let)


@pytest.mark.parametrize("act", ["silu", "sigmoid", "gelu_tanh"])
@pytest.mark.parametrize("walking", [True, False])
def test_activations_far_below_zero(mm, at_most, act, walking):  # noqa: F811
    """Relative accuracy down to the smallest sigmoid of a finite exponential, 2^-128.  The
    weight is 0, so z is the bias.  The exponent is one product and one rounding (its error is
    (|t| + 2) u, relative to the exponential), the exponential and the inverse are off by 2^-22 each,
    five roundings follow, and results below 2^-126 are multiples of 2^-149."""
    if walking:
        at_most(0)
    c = 4096
    b = torch.linspace(-88.7, 20.0, c) if act != "gelu_tanh" else torch.linspace(-10.4, 5.0, c)
    t = (2 * (2 / torch.pi) ** 0.5 * (b.double() + 0.044715 * b.double() ** 3)) if act == "gelu_tanh" else b.double()
    b, t = b[t > -88.72], t[t > -88.72]
    b, t = b[:b.numel() // 64 * 64], t[:t.numel() // 64 * 64]
    s = 1 / (1 + torch.exp(-t))
    want = s if act == "sigmoid" else b.double() * s
    x = randn(1, b.numel(), 3, seed=1)
    y = mm.group_norm(mm.to_device(x), 2, mm.to_device(torch.zeros(b.numel())), mm.to_device(b), EPS, activation=act)
    got = y.cpu()[0, :, 0].double()
    inner = 3 if act == "gelu_tanh" else 0  # roundings of t itself
    bound = want.abs() * ((1.5 + inner) * (t.abs() + 2) * U + 2 * 2.0 ** -22 + 8 * U) + 2.0 ** -148 * (1 + b.double().abs())
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() - bound).max()


# One segment per image, and a thread takes 2000 and 1000 of its values; the images are all the
# same, so that they take little memory.  A thread's sum goes through at most 128 additions,
# the block's through 13 more, and what is added behind that takes 64 bits every eight: 150 u,
# of values of one sign.
@pytest.mark.parametrize("n,c,size,last", [(230, 2, 512000, True), (19000, 1, 32001, False)])
def test_sums_of_one_sign_over_long_segments(mm, n, c, size, last):
    assert plan(n, c, size, c, last, True)[::2] == (0, 1)
    one, grad = randn(1, c, size, seed=1), torch.full((1, c, size), 0.1)
    x, dy = (on_device(mm, t, last).expand(n, c, size) for t in (one, grad))
    assert x._logical_strides[0] == 0
    m64 = one.double().mean(2, keepdim=True)
    r64 = 1 / torch.sqrt(((one.double() - m64) ** 2).mean(2, keepdim=True) + EPS)
    xh = (one.double() - m64) * r64
    exh = r64 * U * m64.abs() + 4 * U * xh.abs()  # mean and rstd are given in float32
    mean, rstd = (mm.to_device(t.float().reshape(1, c)).expand(n, c).contiguous() for t in (m64, r64))
    dx, dw, db = ops.group_norm_backward(dy, x, mean, rstd, mm.to_device(torch.ones(c)), None, c, (True, True, True))
    g = grad.double()
    check("db", db.cpu(), (n * g.sum((0, 2)), n * 150 * U * g.sum((0, 2))))
    check("dw", dw.cpu(), (n * (g * xh).sum((0, 2)), n * (151 * U * (g * xh).abs() + g * exh).sum((0, 2))))
    s1, s2 = g.mean(2, keepdim=True), (g * xh).mean(2, keepdim=True)
    es1, es2 = 151 * U * s1, (152 * U * (g * xh).abs() + g * exh).mean(2, keepdim=True)
    want = r64 * (g - s1 - xh * s2)
    bound = r64 * (4 * U * (g + s1 + (xh * s2).abs()) + es1 + xh.abs() * es2 + exh * s2.abs()) + 4 * U * want.abs()
    for image in (0, n - 1):
        check("dx", dx[image:image + 1].cpu(), (want, bound))


def test_means_of_one_sign_over_many_channels(mm):
    """A group of 262,144 channels of nine pixels: its mean is the sum of as many partial
    sums, of nine additions each, in 64 bits every four."""
    n, c, size = 1, 1 << 18, 9
    one, grad = randn(n, c, size, seed=1), torch.full((n, c, size), 0.1)
    for last in (True, False):
        assert plan(n, c, size, 1, last, True)[0] == 0
        y, dx, _, _ = run(mm, one, 1, torch.ones(c), torch.zeros(c), grad, "none", last)
        m64 = one.double().mean()
        r64 = 1 / torch.sqrt(((one.double() - m64) ** 2).mean() + EPS)
        # g is constant, so dx = rstd (g - mean(g) - xh mean(g xh)) is what sums round to, and
        # mean(g xh) is g times the mean of xh, whose own mean is off by 50 roundings at most
        xh = ((one.double() - m64) * r64).abs()
        bound = r64 * 0.1 * (24 * U + 4 * U + xh * (64 * U * xh.mean()))
        check("dx", dx.cpu(), (torch.zeros(n, c, size, dtype=torch.float64), bound))


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("far", [1e6, -3e6, 1e7])
def test_a_first_part_far_from_the_others(mm, far, last):
    """The join adds distances from the first part's mean, here of 262,144 channels around 0 of which
    the first is far.  In units of far u, a distance is rounded by 1 at most, its product with the
    part's nine values by 1 of nine, and the k-th sum of eight products by k: as independent
    roundings of up to these sizes, (1 + 1 + (4 + 9 + ... + 64) / 8) / 3 = 3.0^2 per part, and 3.0 /
    sqrt(262144) of their mean.  8 of those, and 64 u of the mean magnitude for the mean's own rounding and
    everything else."""
    n, c, size = 1, 1 << 18, 9
    assert plan(n, c, size, 1, last, False)[0] == 0
    x = randn(n, c, size, seed=1)
    x[:, 0] = far
    y = mm.group_norm(on_device(mm, x, last), 1, None, None, EPS).cpu().double()
    x = x.double()
    rstd = 1 / torch.sqrt(((x - x.mean()) ** 2).mean() + EPS)
    want = (x - x.mean()) * rstd
    shift = (24 / c ** 0.5 * abs(far) + 64 * x.abs().mean()) * U * rstd
    check("y", y, (want, shift + 200 * U * want.abs()))
