"""Group norm with an activation, forward and backward, against the formulas in
float64.

Tolerances count roundings, u = 2^-24 each.  A mean or a sum over m = S D values
of an image and group goes through at most 64 additions in a thread (a segment's
pixels), 52 in its block and 13 + m / 16384 behind that, so L = 160 + m / 16384
roundings: a mean is off by at most L u mean|x|.  That error moves every x - mean;
rstd takes half the relative error of the variance (L + 6 roundings).  Hence
|xh error| <= rstd L u mean|x| + (L / 2 + 8) u |xh|, and z = xh w + b adds two
roundings of its terms.  An activation's slope is below 1.13 and its own change
per z below 1.1 (of sigmoid: 0.25, 0.1), its evaluation takes at most 24 roundings
of |act(z)| (16 of |z| in the exponent, where |z| act'(z) <= 1.13 |z|), so
|y error| <= 1.13 |z error| + 24 u (|y| + |z|).  dx, dw and db follow by adding
up the terms of their formulas; sums of columns take L + n S / 2048 additions.

ReLU's slope jumps at 0: elements whose z is within its error of 0 may take
either, and are moved away from it in the input."""

import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

from matrixman_b200 import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
ACTS = ["none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh"]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed))


def act_of(name):
    return {"none": lambda z: z * 1, "relu": F.relu, "silu": lambda z: z * torch.sigmoid(z), "sigmoid": torch.sigmoid,
            "gelu": lambda z: z * 0.5 * torch.special.erfc(-z * math.sqrt(0.5)),
            "gelu_tanh": lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}[name]


def slopes(z, act):
    """act(z), act'(z) and act''(z)'s size."""
    z = z.detach().requires_grad_(True)
    with torch.enable_grad():
        y = act_of(act)(z)
        s, = torch.autograd.grad(y.sum(), z, create_graph=act not in ("none", "relu"))
        c = torch.autograd.grad(s.sum(), z)[0].abs() if s.requires_grad else torch.zeros_like(z)
    return y.detach(), s.detach(), c


def oracle(x, groups, w, b, dy, act="none", eps=EPS):
    """Values and error bounds in float64 of maps x [N, C, *]."""
    shape = x.shape
    n, c = shape[:2]
    x, dy = (t.double().reshape(n, groups, c // groups, -1) for t in (x, dy))
    w64 = (w.double() if w is not None else torch.ones(c, dtype=torch.float64)).reshape(1, groups, -1, 1)
    b64 = (b.double() if b is not None else torch.zeros(c, dtype=torch.float64)).reshape(1, groups, -1, 1)

    def mean(t):
        return t.mean((2, 3), keepdim=True)

    mu = mean(x)
    rstd = 1 / torch.sqrt(mean((x - mu) ** 2) + eps)
    xh = (x - mu) * rstd
    z = xh * w64 + b64
    y, slope, curve = slopes(z, act)
    dz = dy * slope
    g = dz * w64
    s1, s2 = mean(g), mean(g * xh)
    dx = rstd * (g - s1 - xh * s2)
    m = x.shape[2] * x.shape[3]
    adds = 160 + m / 16384
    cols = adds + n * x.shape[3] / 2048
    exh = rstd * adds * U * mean(x.abs()) + (adds / 2 + 8) * U * xh.abs()
    ez = w64.abs() * exh + 2 * U * (z.abs() + b64.abs())
    ey = 1.13 * ez + 24 * U * (y.abs() + z.abs() + (0 if act != "sigmoid" else 1))
    # the slope moves with z, and takes up to 32 roundings of terms up to 1 + |z|
    edz = dy.abs() * (1.1 * curve * ez + (0 if act in ("none", "relu") else 32) * U * (1 + z.abs())) + 2 * U * dz.abs()
    eg = w64.abs() * edz + U * g.abs()
    es1 = mean(eg) + (adds + 2) * U * mean(g.abs())
    es2 = (adds + 4) * U * mean((g * xh).abs()) + mean(g.abs() * exh) + mean(eg * xh.abs())
    # rstd itself is off by (adds / 2 + 8) u, relatively
    edx = rstd * (4 * U * (g.abs() + s1.abs() + (xh * s2).abs()) + eg + es1 + xh.abs() * es2 + exh * s2.abs()) \
        + (adds / 2 + 8) * U * dx.abs()

    def columns(t):
        return t.sum((0, 3)).reshape(c)

    edw = cols * U * columns((dz * xh).abs()) + columns(dz.abs() * exh + edz * xh.abs())
    edb = cols * U * columns(dz.abs()) + columns(edz)
    return {"y": (y.reshape(shape), ey.reshape(shape)), "dx": (dx.reshape(shape), edx.reshape(shape)),
            "dw": (columns(dz * xh), edw), "db": (columns(dz), edb), "z": (z.reshape(shape), ez.reshape(shape))}


def check(name, got, want):
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), name
    err = (got.double() - value).abs()
    worst = (err - bound).max().item() if err.numel() else -1.0
    assert not torch.isnan(got).any(), name
    assert worst <= 0, f"{name}: {err.max().item():.3g} off, {worst:.3g} over its bound"


def inputs(n, c, spatial, groups, act, seed=0):
    """Maps with channels of different scale and offset."""
    x = randn(n, c, *spatial, seed=seed + 1)
    ones = (1,) * len(spatial)
    x = x * (0.2 + torch.rand(c, generator=gen(seed + 2))).reshape(1, c, *ones) + randn(c, seed=seed + 3).reshape(1, c, *ones)
    w, b, dy = 1 + 0.3 * randn(c, seed=seed + 4), randn(c, seed=seed + 5), randn(n, c, *spatial, seed=seed + 6)
    if act == "relu":
        z, e = oracle(x, groups, w, b, dy)["z"]
        dy = torch.where(z.abs() > 4 * e, dy, torch.zeros(()))  # (no gradient where the slope is not settled)
    return x, w, b, dy


def last_memory(t):
    """The same values with channels last in memory."""
    order = (0, *range(2, t.dim()), 1)
    back = (0, t.dim() - 1, *range(1, t.dim() - 1))
    return t.permute(order).contiguous().permute(back)


def on_device(mm, t, last):
    if not last or t.dim() < 3:
        return mm.to_device(t.contiguous())
    order = (0, *range(2, t.dim()), 1)
    back = (0, t.dim() - 1, *range(1, t.dim() - 1))
    return mm.to_device(t.permute(order).contiguous()).permute(back)


def run(mm, x, groups, w, b, dy, act, last):
    dx = on_device(mm, x, last).detach().requires_grad_(True)
    dw = mm.to_device(w).requires_grad_(True) if w is not None else None
    db = mm.to_device(b).requires_grad_(True) if b is not None else None
    y = mm.group_norm(dx, groups, dw, db, EPS, activation=act)
    assert y._logical_strides == dx._logical_strides or 1 in x.shape
    leaves = [t for t in (dx, dw, db) if t is not None]
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, on_device(mm, dy, last))))
    return y.detach().cpu(), *(grads[id(t)].cpu() if t is not None else None for t in (dx, dw, db))


# Sizes: single values, images without and with one pixel, odd channels (single
# floats), pairs, multiples of four, groups of 1 to 1100 channels, more channels
# than a block has columns, pixel counts on both sides of a segment, wide images.
SIZES = [(1, 1, (1,), 1), (2, 2, (1,), 1), (3, 6, (), 3), (1, 64, (20, 20), 16), (5, 130, (37, 41), 13),
         (2, 15, (7, 3), 5), (33, 512, (), 8), (4, 32, (8, 8), 32), (3, 12, (5, 13), 1), (2, 20, (3, 4, 5), 2),
         (1, 7, (300,), 7), (2, 1100, (3, 3), 1), (1, 2200, (2, 1), 2), (2, 48, (64, 64), 8), (1, 16, (160, 160), 4),
         (300, 24, (2, 3), 4), (1, 36, (65,), 12), (2, 10, (129, 2), 1), (1, 3, (255, 257), 3), (1, 1, (70, 70), 1),
         (2, 1028, (9,), 257)]


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", SIZES)
def test_forward_and_backward(mm, n, c, spatial, groups, last):
    act = ACTS[(n + c + groups) % len(ACTS)]
    x, w, b, dy = inputs(n, c, spatial, groups, act)
    want = oracle(x, groups, w, b, dy, act)
    for name, got in zip(("y", "dx", "dw", "db"), run(mm, x, groups, w, b, dy, act, last)):
        check(name, got, want[name])


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("act", ACTS)
def test_activations(mm, act, last):
    x, w, b, dy = inputs(3, 40, (11, 9), 4, act, seed=10)
    b = 4 * b  # far into both tails
    if act == "relu":
        z, e = oracle(x, 4, w, b, dy)["z"]
        dy = torch.where(z.abs() > 4 * e, dy, torch.zeros(()))
    want = oracle(x, 4, w, b, dy, act)
    for name, got in zip(("y", "dx", "dw", "db"), run(mm, x, 4, w, b, dy, act, last)):
        check(name, got, want[name])


def test_gradient_against_differences(mm):
    """d/dt of sum(y dy) along a direction, by central differences in float64."""
    x, v, dy = (randn(2, 12, 3, 5, seed=s) for s in (1, 2, 3))
    w, b = randn(12, seed=4), randn(12, seed=5)
    dx = run(mm, x, 3, w, b, dy, "silu", True)[1]
    h = 1e-5

    def f(t):
        return (F.silu(F.group_norm(x.double() + t * v.double(), 3, w.double(), b.double(), EPS)) * dy.double()).sum()

    slope = ((f(h) - f(-h)) / (2 * h)).item()
    # differences: h^2 times third derivatives of order 10; ours: 360 terms of a few u each
    assert abs((dx.double() * v.double()).sum().item() - slope) <= 1e-4 * (dx.double() * v.double()).abs().sum().item()


@pytest.mark.parametrize("last", [True, False])
def test_torch_functional_and_module(mm, last):
    x, w, b, dy = inputs(4, 24, (10, 6), 6, "none")
    want = oracle(x, 6, w, b, dy)
    dx = on_device(mm, x, last).detach().requires_grad_(True)
    dw, db = (mm.to_device(t).requires_grad_(True) for t in (w, b))
    y = F.group_norm(dx, 6, dw, db, EPS)
    grads = torch.autograd.grad(y, (dx, dw, db), on_device(mm, dy, last))
    for name, got in zip(("y", "dx", "dw", "db"), (y.detach(), *grads)):
        check(name, got.cpu(), want[name])
    module = torch.nn.GroupNorm(6, 24, eps=EPS)
    with torch.no_grad():
        module.weight.copy_(w)
        module.bias.copy_(b)
        check("y", module(on_device(mm, x, last)).cpu(), want["y"])


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("affine", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(mm, affine, last):
    x, w, b, dy = inputs(3, 30, (7, 7), 5, "silu")
    w, b = w if affine[0] else None, b if affine[1] else None
    want = oracle(x, 5, w, b, dy, "silu")
    for name, got in zip(("y", "dx", "dw", "db"), run(mm, x, 5, w, b, dy, "silu", last)):
        if got is not None:
            check(name, got, want[name])


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("spatial", [(9, 9), (150, 150)])
def test_large_offset_keeps_the_variance(mm, spatial, last):
    """Maps far from zero: the distances from the mean are what is squared."""
    x, dy = randn(2, 16, *spatial, seed=1) * 0.01 + 1000.0, randn(2, 16, *spatial, seed=2)
    x[:, :, 0] = 0.0 if spatial[0] > 100 else 1000.0  # a row of padding in front
    w, b = torch.ones(16), torch.zeros(16)
    want = oracle(x, 4, w, b, dy)
    for name, got in zip(("y", "dx", "dw", "db"), run(mm, x, 4, w, b, dy, "none", last)):
        check(name, got, want[name])


@pytest.mark.parametrize("last", [True, False])
def test_constant_and_non_finite_groups(mm, last):
    x = randn(5, 16, 6, 5, seed=1)
    x[0, :4] = 3.5                      # no spread: y is the bias
    x[1, 5, 2, 3] = float("nan")
    x[2, 9, 0, 0] = float("inf")
    x[3, 13, 5, 4] = float("-inf")
    w, b, dy = randn(16, seed=2), randn(16, seed=3), randn(5, 16, 6, 5, seed=4)
    y, dx, dw, db = run(mm, x, 4, w, b, dy, "none", last)
    assert torch.equal(y[0, :4], b[:4].reshape(4, 1, 1).expand(4, 6, 5))
    clean = torch.ones(5, 4, dtype=torch.bool)
    for image, group in ((1, 1), (2, 2), (3, 3)):
        assert torch.isnan(y[image, 4 * group:4 * group + 4]).all()
        assert torch.isnan(dx[image, 4 * group:4 * group + 4]).all()
        assert torch.isnan(dw[4 * group:4 * group + 4]).all()
        clean[image, group] = False
    ok = clean.repeat_interleave(4, 1)
    want = oracle(torch.where(ok[..., None, None], x, torch.zeros(())), 4, w, b, dy)
    for name, got in (("y", y), ("dx", dx)):
        check(name, got[ok], tuple(t[ok] for t in want[name]))
    check("dw", dw[:4], tuple(t[:4] for t in want["dw"]))
    assert not torch.isnan(db).any()


def test_strides(mm):
    """Slices of channels of a concatenation, cropped images, transposed pixels,
    rows of a matrix, expanded gradients."""
    w, b = randn(12, seed=1), randn(12, seed=2)
    base = randn(3, 9, 10, 40, seed=3)  # N H W C
    dev = mm.to_device(base)
    first = randn(3, 30, 9, 10, seed=4)
    dfirst = mm.to_device(first)
    cases = [(dev.permute(0, 3, 1, 2)[:, 5:17], base.permute(0, 3, 1, 2)[:, 5:17]),
             (dev.permute(0, 3, 1, 2)[:, 8:20], base.permute(0, 3, 1, 2)[:, 8:20]),
             (dev.permute(0, 3, 1, 2)[:, 4:16, 2:7], base.permute(0, 3, 1, 2)[:, 4:16, 2:7]),
             (dev.permute(0, 3, 1, 2)[:, 4:16, :, 1:8], base.permute(0, 3, 1, 2)[:, 4:16, :, 1:8]),
             (dev.permute(0, 3, 2, 1)[::2, 4:16], base.permute(0, 3, 2, 1)[::2, 4:16]),
             (dfirst[:, 7:19], first[:, 7:19]), (dfirst[:, 3:27:2], first[:, 3:27:2]),
             (dfirst[1:, 1:13, :, 2:9], first[1:, 1:13, :, 2:9]), (dfirst.transpose(2, 3)[:, :12], first.transpose(2, 3)[:, :12]),
             (dfirst[:, :12, 3, 4], first[:, :12, 3, 4]), (dfirst[:, 0, :, 0].t()[:, :1].expand(9, 12), first[:, 0, :, 0].t()[:, :1].expand(9, 12))]
    for view, cpu in cases:
        x = view.detach().requires_grad_(True)
        dy = randn(*cpu.shape, seed=5)
        y = mm.group_norm(x, 4, mm.to_device(w), mm.to_device(b), EPS, activation="silu")
        want = oracle(cpu, 4, w, b, dy, "silu")
        check("y", y.detach().cpu(), want["y"])
        for last in (True, False):
            check("dx", torch.autograd.grad(y, x, on_device(mm, dy, last), retain_graph=True)[0].cpu(), want["dx"])
        ones = mm.to_device(torch.ones(())).expand(*cpu.shape)
        check("dx", torch.autograd.grad(y, x, ones)[0].cpu(), oracle(cpu, 4, w, b, torch.ones(cpu.shape), "silu")["dx"])
    # parameters at a stride
    x, ws = randn(2, 12, 5, seed=6), randn(12, 2, seed=7)
    dws = mm.to_device(ws)
    y = mm.group_norm(mm.to_device(x), 3, dws[:, 0], dws[:, 1], EPS)
    check("y", y.cpu(), oracle(x, 3, ws[:, 0], ws[:, 1], x)["y"])


def test_only_the_gradients_asked_for(mm):
    x, w, b, dy = inputs(4, 24, (10, 6), 6, "gelu")
    want = oracle(x, 6, w, b, dy, "gelu")
    for last in (True, False):
        g = on_device(mm, dy, last)
        dw = mm.to_device(w).requires_grad_(True)
        y = mm.group_norm(on_device(mm, x, last), 6, dw, mm.to_device(b), EPS, activation="gelu")
        check("dw", torch.autograd.grad(y, dw, g)[0].cpu(), want["dw"])
        db = mm.to_device(b).requires_grad_(True)
        y = mm.group_norm(on_device(mm, x, last), 6, w, db, EPS, activation="gelu")
        check("db", torch.autograd.grad(y, db, g)[0].cpu(), want["db"])
        dx = on_device(mm, x, last).detach().requires_grad_(True)
        y = mm.group_norm(dx, 6, w, b, EPS, activation="gelu")  # CPU parameters, uploaded
        check("dx", torch.autograd.grad(y, dx, g)[0].cpu(), want["dx"])


def test_no_images(mm):
    x = mm.to_device(torch.zeros(0, 8, 3, 3)).requires_grad_(True)
    w = mm.to_device(torch.ones(8)).requires_grad_(True)
    y = mm.group_norm(x, 2, w, None, EPS, activation="silu")
    dx, dw = torch.autograd.grad(y, (x, w), mm.to_device(torch.zeros(0, 8, 3, 3)))
    assert y.shape == (0, 8, 3, 3) and dx.shape == (0, 8, 3, 3) and torch.equal(dw.cpu(), torch.zeros(8))


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", [(7, 60, (17, 13), 5), (2, 32, (160, 160), 4)])
def test_same_bits_twice_and_in_a_replayed_graph(mm, n, c, spatial, groups, last):
    x, w, b, dy = inputs(n, c, spatial, groups, "silu")
    first, again = (run(mm, x, groups, w, b, dy, "silu", last) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    dx, g = (on_device(mm, t, last) for t in (x, dy))
    dw, db = (mm.to_device(t).requires_grad_(True) for t in (w, b))
    leaf = dx.detach().requires_grad_(True)
    rt = dx.runtime

    def call():
        y = mm.group_norm(leaf, groups, dw, db, EPS, activation="silu")
        return (y, *torch.autograd.grad(y, (leaf, dw, db), g))

    kept = call()  # an eager graph of the leaves, alive during the capture
    rt.synchronize()
    rt.capture_begin()
    out = call()
    graph = rt.capture_end()
    other = run(mm, 2 * x, groups, w, b, dy, "silu", last)  # eager work between replays
    for scale, want in ((2, other), (1, first)):
        with torch.no_grad():
            leaf.copy_(on_device(mm, scale * x, last))
        graph.replay()
        assert all(torch.equal(t.detach().cpu(), q) for t, q in zip(out, want))
    del kept


def test_refusals(mm):
    x = mm.to_device(randn(4, 8, 3, seed=1))
    with pytest.raises(RuntimeError, match="groups"):
        mm.group_norm(x, 3)
    with pytest.raises(RuntimeError, match="groups"):
        mm.group_norm(x, 0)
    with pytest.raises(ValueError, match="activation"):
        mm.group_norm(x, 2, activation="tanh")
    with pytest.raises(RuntimeError, match="MatrixManTensor"):
        mm.group_norm(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError, match="N, C"):
        mm.group_norm(mm.to_device(torch.zeros(8)), 2)
    with pytest.raises(RuntimeError, match="weight"):
        mm.group_norm(x, 2, mm.to_device(torch.ones(7)))
    with pytest.raises(RuntimeError, match="bias"):
        mm.group_norm(x, 2, None, mm.to_device(torch.ones(8, 1)))
    with pytest.raises(NotImplementedError, match="float32"):
        mm.group_norm(mm.to_device(torch.zeros(2, 8, dtype=torch.int64)), 2)
    with pytest.raises(NotImplementedError):
        mm.group_norm(mm.to_device(torch.zeros(2, 8, 0)), 2)
    with pytest.raises(NotImplementedError):
        mm.group_norm(mm.to_device(torch.zeros(2, 0, 3)), 1)
    w = torch.ones(8, requires_grad=True)  # a CPU parameter cannot take a gradient from the device
    with pytest.raises(RuntimeError, match="gradient"):
        mm.group_norm(x, 2, w)
    leaf = x.detach().requires_grad_(True)
    y = mm.group_norm(leaf, 2)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(y, leaf, mm.to_device(torch.ones(4, 8, 3)), create_graph=True)[0],
                            leaf, mm.to_device(torch.ones(4, 8, 3)))


def test_the_backward_pass_keeps_the_statistics_but_not_the_output(mm):
    x = mm.to_device(torch.ones(64, 64, 32, 32)).requires_grad_(True)
    rt = x.runtime
    live = lambda: rt.pool_stats()["live_bytes"]["activation"]
    start = live()
    y = mm.group_norm(x, 8, activation="silu")
    assert live() - start >= 4 * 64 * 64 * 32 * 32
    s = y.sum(dim=1)
    del y
    assert live() - start <= 4 * 64 * 32 * 32 + 3 * 512 + 2 * 4 * 64 * 8  # s, mean, rstd
    s.sum(dim=0).sum(dim=0).sum(dim=0).backward()
    assert x.grad.shape == x.shape


@pytest.mark.parametrize("act", ["none", "silu"])
def test_one_step_calls_and_the_python_code_agree(mm, monkeypatch, act):
    """The same bits, shapes and strides through the C++ calls and without them."""
    from matrixman_b200 import ops
    host = randn(4, 12, 6, 5, seed=1)
    nhwc = mm.to_device(host.permute(0, 2, 3, 1).contiguous())
    w, b = mm.to_device(randn(12, seed=2)), mm.to_device(randn(12, seed=3))
    wide = mm.to_device(randn(4, 6, 5, 20, seed=4)).permute(0, 3, 1, 2)
    rows = mm.to_device(randn(9, 12, seed=5))
    maps = [mm.to_device(host), nhwc.permute(0, 3, 1, 2), wide[:, 3:15], wide[:, 4:16, 1:], rows, rows[:, :, None],
            mm.to_device(randn(3, 12, 7, seed=6)), mm.to_device(randn(2, 12, 3, 2, 4, seed=7)), rows[:1].expand(5, 12),
            mm.to_device(randn(12, 9, seed=8)).t(), mm.to_device(randn(5, 12, 1, 8, seed=9)),
            mm.to_device(randn(3, 12, 4, 5, seed=10)).transpose(2, 3)]

    def all_of(x):
        x = x.detach().requires_grad_(True)
        p, q = w.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y = mm.group_norm(x, 3, p, q, EPS, activation=act)
        with torch.no_grad():
            plain = mm.group_norm(x, 3, p, q, EPS, activation=act)
        dy = mm.to_device(randn(*x.shape, seed=20))
        return (y, plain, *torch.autograd.grad(y, (x, p, q), dy))

    native = [all_of(x) for x in maps]
    monkeypatch.setattr(ops, "native_call", lambda *a: None)
    for x, got in zip(maps, native):
        for one, other in zip(got, all_of(x)):
            assert one.shape == other.shape and one._logical_strides == other._logical_strides
            assert torch.equal(one.detach().cpu(), other.detach().cpu())


def test_torch_functional_keeps_channels_last(mm):
    """No copy to another order on the way, forward or backward."""
    x, w, b, dy = inputs(2, 16, (9, 7), 4, "none")
    dx = on_device(mm, x, True).detach().requires_grad_(True)
    y = F.group_norm(dx, 4)
    grad, = torch.autograd.grad(y, dx, on_device(mm, dy, True))
    assert y._logical_strides == dx._logical_strides == grad._logical_strides
    module = torch.nn.GroupNorm(4, 16)  # parameters on the CPU: forward and dx work, their own gradients do not
    y = module(dx)
    want = oracle(x, 4, torch.ones(16), torch.zeros(16), dy)
    check("y", y.detach().cpu(), want["y"])
    check("dx", torch.autograd.grad(y, dx, on_device(mm, dy, True), retain_graph=True)[0].cpu(), want["dx"])
    for p in module.parameters():
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, p, on_device(mm, dy, True), retain_graph=True)


@pytest.mark.parametrize("last", [True, False])
def test_bounded_waits_run_out_and_recover(mm, last):
    """With the test hook each cluster's first block gives the others nothing and the limit of a wait is one try of
    1 ms, so their waits run out: the kernel leaves a code, every block goes on to its end, and the next wait of the
    host raises.  Calls after that are whole."""
    lib = _lib.load()
    x, w, b, dy = inputs(2, 48, (64, 64), 8, "silu")
    want = run(mm, x, 8, w, b, dy, "silu", last)
    dx, g = (on_device(mm, t, last) for t in (x, dy))
    leaf, dw, db = (t.detach().requires_grad_(True) for t in (dx, mm.to_device(w), mm.to_device(b)))
    rt = dx.runtime
    y = mm.group_norm(leaf, 8, dw, db, EPS, activation="silu")
    rt.synchronize()
    code = ctypes.c_int(-1)
    for call in (lambda: mm.group_norm(dx, 8, w, b, EPS, activation="silu"),
                 lambda: torch.autograd.grad(y, (leaf, dw, db), g, retain_graph=True)):
        _lib.check(lib.mm_debug_tc_fault(rt.index, 1_000_000, 1))
        try:
            call()
        finally:
            _lib.check(lib.mm_debug_tc_fault(rt.index, 0, 0))
        with pytest.raises(_lib.MatrixManNativeError, match="code 111"):
            rt.synchronize(timeout_ms=30_000)
        _lib.check(lib.mm_kernel_error(rt.index, ctypes.byref(code), 0))
        assert code.value == 0  # reported once
        assert all(torch.equal(p, q) for p, q in zip(run(mm, x, 8, w, b, dy, "silu", last), want))
