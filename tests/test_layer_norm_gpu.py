"""Layer norm's forward and backward pass against the formulas in float64.

Tolerances count roundings, u = 2^-24 each.  A sum of H terms goes through at
most 32 additions in a thread (H / 1024 in the kernel for rows too wide for
registers) and 10 in the tree over the threads: L = 42 + H / 1024 roundings, so
a mean is off by at most L u mean|x|.  That error moves every x - mean of the
row; rstd takes half the relative error of the variance (L + 6 roundings).
Hence |xh error| <= rstd L u mean|x| + (L / 2 + 8) u |xh|, and y, dx, dw, db
follow by adding up the terms of their formulas.  Column sums take at most
rows / 256 + 64 additions."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed))


def oracle(x, w, b, dy, eps=EPS):
    """Values and error bounds in float64 of rows x [R, H]."""
    x, dy = x.double(), dy.double()
    rows, h = x.shape
    w64 = w.double() if w is not None else torch.ones(h, dtype=torch.float64)
    b64 = b.double() if b is not None else torch.zeros(h, dtype=torch.float64)
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    y = xh * w64 + b64
    g = dy * w64
    s1, s2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - s1 - xh * s2)
    adds = 42 + h / 1024
    cols = 64 + rows / 256
    exh = rstd * adds * U * x.abs().mean(1, keepdim=True) + (adds / 2 + 8) * U * xh.abs()
    ey = w64.abs() * exh + 4 * U * (y.abs() + b64.abs())
    es1 = (adds + 2) * U * g.abs().mean(1, keepdim=True)
    es2 = (adds + 4) * U * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * exh).mean(1, keepdim=True)
    # rstd itself is off by (adds / 2 + 8) u, relatively
    edx = rstd * (4 * U * (g.abs() + s1.abs() + (xh * s2).abs()) + es1 + xh.abs() * es2 + exh * s2.abs()) \
        + (adds / 2 + 8) * U * dx.abs()
    edw = cols * U * (dy * xh).abs().sum(0) + (dy.abs() * exh).sum(0)
    edb = cols * U * dy.abs().sum(0)
    return {"y": (y, ey), "dx": (dx, edx), "dw": ((dy * xh).sum(0), edw), "db": (dy.sum(0), edb)}


def check(name, got, want):
    value, bound = want
    err = (got.double().reshape(value.shape) - value).abs()
    worst = (err - bound).max().item() if err.numel() else -1.0
    assert not torch.isnan(got).any(), name
    assert worst <= 0, f"{name}: {err.max().item():.3g} off, {worst:.3g} over its bound"


def run(mm, x, w, b, dy, shape=None):
    dx = mm.to_device(x).requires_grad_(True)
    dw = mm.to_device(w).requires_grad_(True) if w is not None else None
    db = mm.to_device(b).requires_grad_(True) if b is not None else None
    y = F.layer_norm(dx, shape or (x.shape[-1],), dw, db, EPS)
    leaves = [t for t in (dx, dw, db) if t is not None]
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, mm.to_device(dy))))
    return y.detach().cpu(), *(grads[id(t)].cpu() if t is not None else None for t in (dx, dw, db))


# Widths on both sides of every change of kernel: one warp per row up to 1024
# (512 backward), blocks up to 16384 (8192), the walking kernels above; odd ones
# load single floats, even ones pairs, multiples of four 16 bytes.
@pytest.mark.parametrize("rows,width", [
    (1, 1), (3, 2), (5, 31), (7, 33), (1, 64), (130, 127), (33, 128), (9, 130), (1000, 256), (65, 511), (12, 513),
    (600, 516), (4, 1023), (17, 1024), (5, 1026), (300, 1250), (3, 2047), (40, 2048), (6, 4097), (310, 4096),
    (2, 8191), (3, 8192), (5, 8194), (2, 16384), (3, 16390), (2, 40001)])
def test_forward_and_backward(mm, rows, width):
    x = randn(rows, width, seed=1) * (0.1 + 3 * torch.rand(rows, 1, generator=gen(2))) + randn(rows, 1, seed=3)
    w, b, dy = 1 + 0.3 * randn(width, seed=4), randn(width, seed=5), randn(rows, width, seed=6)
    want = oracle(x, w, b, dy)
    y, dx, dw, db = run(mm, x, w, b, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        check(name, got, want[name])


def test_gradient_against_differences(mm):
    """d/dt of sum(y dy) along a direction, by central differences in float64."""
    x, w, b, dy, v = (randn(6, 20, seed=s) if s not in (2, 3) else randn(20, seed=s) for s in (1, 2, 3, 4, 5))
    _, dx, _, _ = run(mm, x, w, b, dy)
    h = 1e-5

    def f(t):
        return (F.layer_norm(x.double() + t * v.double(), (20,), w.double(), b.double(), EPS) * dy.double()).sum()

    slope = ((f(h) - f(-h)) / (2 * h)).item()
    # differences: h^2 times third derivatives of order 10; ours: 120 terms of a few u each
    assert abs((dx.double() * v.double()).sum().item() - slope) <= 1e-4 * (dx.double() * v.double()).abs().sum().item()


@pytest.mark.parametrize("affine", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(mm, affine):
    x, dy = randn(11, 96, seed=1), randn(11, 96, seed=2)
    w = randn(96, seed=3) if affine[0] else None
    b = randn(96, seed=4) if affine[1] else None
    want = oracle(x, w, b, dy)
    y, dx, dw, db = run(mm, x, w, b, dy)
    check("y", y, want["y"])
    check("dx", dx, want["dx"])
    if w is not None:
        check("dw", dw, want["dw"])
    if b is not None:
        check("db", db, want["db"])


def test_large_offset_keeps_the_variance(mm):
    """Rows far from zero: the distances from the mean are what is squared."""
    x = randn(9, 700, seed=1) * 0.01 + 1000.0
    w, b, dy = torch.ones(700), torch.zeros(700), randn(9, 700, seed=2)
    want = oracle(x, w, b, dy)
    y, dx, dw, db = run(mm, x, w, b, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        check(name, got, want[name])


def test_constant_and_non_finite_rows(mm):
    x = randn(4, 64, seed=1)
    x[0] = 3.5                # no spread: y is the bias
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    w, b = randn(64, seed=2), randn(64, seed=3)
    y = F.layer_norm(mm.to_device(x), (64,), mm.to_device(w), mm.to_device(b), EPS).cpu()
    assert torch.equal(y[0], b)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    check("y", y[3:], oracle(x[3:], w, b, x[3:])["y"])


def test_shapes_strides_and_normalized_dims(mm):
    x = randn(4, 6, 10, 8, seed=1)
    w, b, dy = randn(10, 8, seed=2), randn(10, 8, seed=3), randn(4, 6, 10, 8, seed=4)
    want = oracle(x.reshape(24, 80), w.reshape(80), b.reshape(80), dy.reshape(24, 80))
    y, dx, dw, db = run(mm, x, w, b, dy, (10, 8))
    assert y.shape == x.shape and dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        check(name, got, want[name])
    # a transposed input, rows at a stride, an odd element offset, an expanded gradient
    base = randn(40, 101, seed=5)
    dev = mm.to_device(base)
    wv, bv = randn(37, seed=6), randn(37, seed=7)
    for view, cpu in ((dev[:, 3:40], base[:, 3:40]), (dev[:37].t(), base[:37].t()), (dev[1::3, 64:101], base[1::3, 64:101])):
        got = F.layer_norm(view, (37,), mm.to_device(wv), mm.to_device(bv), EPS).cpu()
        check("y", got, oracle(cpu, wv, bv, cpu)["y"])
    leaf = mm.to_device(base).requires_grad_(True)
    F.layer_norm(leaf, (101,), None, None, EPS).sum(dim=1).sum(dim=0).backward()
    ones = torch.ones(40, 101)
    check("dx", leaf.grad.cpu(), oracle(base, None, None, ones)["dx"])


def test_only_the_gradients_asked_for(mm):
    x, w, b, dy = randn(50, 300, seed=1), randn(300, seed=2), randn(300, seed=3), randn(50, 300, seed=4)
    want = oracle(x, w, b, dy)
    dw = mm.to_device(w).requires_grad_(True)
    y = F.layer_norm(mm.to_device(x), (300,), dw, mm.to_device(b), EPS)
    check("dw", torch.autograd.grad(y, dw, mm.to_device(dy))[0].cpu(), want["dw"])
    dx = mm.to_device(x).requires_grad_(True)
    y = F.layer_norm(dx, (300,), w, b, EPS)  # CPU parameters, uploaded
    check("dx", torch.autograd.grad(y, dx, mm.to_device(dy))[0].cpu(), want["dx"])


def test_no_rows(mm):
    x = mm.to_device(torch.zeros(0, 16)).requires_grad_(True)
    w = mm.to_device(torch.ones(16)).requires_grad_(True)
    y = F.layer_norm(x, (16,), w, None, EPS)
    dx, dw = torch.autograd.grad(y, (x, w), mm.to_device(torch.zeros(0, 16)))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and torch.equal(dw.cpu(), torch.zeros(16))


def test_same_bits_twice_and_in_a_replayed_graph(mm):
    x, w, b, dy = randn(999, 260, seed=1), randn(260, seed=2), randn(260, seed=3), randn(999, 260, seed=4)
    first, again = run(mm, x, w, b, dy), run(mm, x, w, b, dy)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    args = [mm.to_device(t) for t in (x, w, b, dy)]
    rt = args[0].runtime
    aten = torch.ops.aten

    def call():
        y, mean, rstd = aten.native_layer_norm(args[0], [260], args[1], args[2], EPS)
        return (y, *aten.native_layer_norm_backward(args[3], args[0], [260], mean, rstd, args[1], args[2],
                                                    [True, True, True]))

    call()
    rt.synchronize()
    rt.capture_begin()
    out = call()
    graph = rt.capture_end()
    other = run(mm, 2 * x, w, b, dy)  # eager work between replays
    args[0].copy_(mm.to_device(2 * x))
    graph.replay()
    assert all(torch.equal(t.cpu(), q) for t, q in zip(out, other))
    args[0].copy_(mm.to_device(x))
    graph.replay()
    assert all(torch.equal(t.cpu(), q) for t, q in zip(out, first))


def test_refusals(mm):
    x = mm.to_device(randn(4, 8, seed=1))
    with pytest.raises(RuntimeError):
        F.layer_norm(x, (7,))
    with pytest.raises(RuntimeError, match="normalized"):
        torch.ops.aten.native_layer_norm(x, [8], mm.to_device(torch.ones(4)), None, EPS)
    with pytest.raises(NotImplementedError):
        F.layer_norm(mm.to_device(torch.zeros(4, 0)), (0,))
    with pytest.raises(NotImplementedError, match="float32"):
        torch.ops.aten.native_layer_norm(mm.to_device(torch.zeros(2, 8, dtype=torch.int64)), [8], None, None, EPS)
    w = torch.ones(8, requires_grad=True)  # a CPU parameter cannot take a gradient from the device
    with pytest.raises(RuntimeError):
        y = F.layer_norm(x.requires_grad_(True), (8,), w, None, EPS)
        torch.autograd.grad(y, w, x.detach())


@pytest.mark.parametrize("native", [True, False])
def test_the_backward_pass_keeps_the_statistics_but_not_the_output(mm, monkeypatch, native):
    from matrixman_b200 import ops
    if not native:
        monkeypatch.setattr(ops, "native_call", lambda *a: None)
    x = mm.to_device(torch.ones(4096, 512)).requires_grad_(True)
    rt = x.runtime
    live = lambda: rt.pool_stats()["live_bytes"]["activation"]
    start = live()
    y = F.layer_norm(x, (512,))
    assert live() - start >= 4 * 4096 * 512
    s = y.sum(dim=1)
    del y
    assert live() - start <= 3 * 4 * 4096 + 3 * 512  # mean, rstd, s
    s.sum(dim=0).backward()
    assert x.grad.shape == x.shape
