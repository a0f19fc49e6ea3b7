"""Group norm and the gradient norm beyond 2^31 elements: zeros (one fill) but for the
last few values, whose results are compared with the formulas in float64."""

import pytest
import torch

from .test_group_norm_gpu import check, oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


@pytest.fixture
def zeros(mm):
    """zeros(*shape) on the device; memory goes back when the test ends."""
    from matrixman_b200 import ops
    from matrixman_b200.runtime import get_runtime
    rt = get_runtime()
    yield lambda *shape: ops.full(rt, shape, 0.0)
    rt.synchronize()
    rt.trim()


@pytest.mark.parametrize("last", [True, False])
def test_many_images(mm, zeros, last):
    n, c, h, w, groups = (1 << 31) // (64 * 1024) + 3, 64, 32, 32, 8
    shape, order = ((n, h, w, c), (0, 3, 1, 2)) if last else ((n, c, h, w), (0, 1, 2, 3))
    tail, dy = torch.randn(2, *shape[1:], generator=gen(1)), torch.randn(2, *shape[1:], generator=gen(2))
    g, b = torch.randn(c, generator=gen(3)), torch.randn(c, generator=gen(4))
    x, grad = zeros(*shape), zeros(*shape)
    x[n - 2:].copy_(mm.to_device(tail))
    grad[n - 2:].copy_(mm.to_device(dy))
    x = x.permute(order).detach().requires_grad_(True)
    dg, db = mm.to_device(g).requires_grad_(True), mm.to_device(b).requires_grad_(True)
    y = mm.group_norm(x, groups, dg, db, EPS, activation="silu")
    grads = torch.autograd.grad(y, (x, dg, db), grad.permute(order))
    want = oracle(tail.permute(order), groups, g, b, dy.permute(order), "silu")
    check("y", y.detach()[n - 2:].cpu(), want["y"])
    check("dx", grads[0][n - 2:].cpu(), want["dx"])
    check("dw", grads[1].cpu(), want["dw"])  # (the other images add zeros)
    check("db", grads[2].cpu(), want["db"])
    zero = mm.to_device(torch.zeros(1, c, 1, 1))
    first = mm.group_norm(zero.expand(1, c, h, w), groups, dg.detach(), db.detach(), EPS, activation="silu").cpu()
    assert torch.equal(y.detach()[n // 2:n // 2 + 1].cpu(), first)  # a constant image is its bias


@pytest.mark.parametrize("last", [True, False])
def test_large_images(mm, zeros, last):
    """Images too large for a cluster, one channel per group: mean and variance follow
    from the three pixels that are not zero."""
    n, c, pixels = 2, 1030, (1 << 20) + 3
    assert n * c * pixels > 1 << 31
    shape = (n, pixels, c) if last else (n, c, pixels)
    tail, dy = torch.randn(3, c, generator=gen(1)), torch.randn(3, c, generator=gen(2))
    g, b = 1 + 0.1 * torch.randn(c, generator=gen(3)), torch.randn(c, generator=gen(4))
    x, grad = zeros(*shape), zeros(*shape)
    if last:
        x[1, pixels - 3:].copy_(mm.to_device(tail))
        grad[1, pixels - 3:].copy_(mm.to_device(dy))
        x, grad = x.permute(0, 2, 1), grad.permute(0, 2, 1)
    else:
        x[1, :, pixels - 3:].copy_(mm.to_device(tail.t().contiguous()))
        grad[1, :, pixels - 3:].copy_(mm.to_device(dy.t().contiguous()))
    x = x.detach().requires_grad_(True)
    dg, db = mm.to_device(g).requires_grad_(True), mm.to_device(b).requires_grad_(True)
    y = mm.group_norm(x, c, dg, db, EPS)
    dx, dw, dbias = torch.autograd.grad(y, (x, dg, db), grad)
    t, d = tail.double(), dy.double()
    mean, var = t.sum(0) / pixels, (t ** 2).sum(0) / pixels - (t.sum(0) / pixels) ** 2
    rstd = 1 / torch.sqrt(var + EPS)
    xh = (t - mean) * rstd
    s1, s2 = (d * g).sum(0) / pixels, (d * g * xh).sum(0) / pixels
    wants = [(y.detach(), xh * g + b), (dx, rstd * (d * g - s1 - xh * s2))]
    for got, want in wants:
        # the variance is a sum of 2^20 terms joined by up to 2000 roundings, most of them of zeros
        assert ((got[1, :, pixels - 3:].cpu().t().double() - want).abs() <= 1e-4 * want.abs().max(0).values).all()
    assert ((dw.cpu().double() - (d * xh).sum(0)).abs() <= 1e-4 * (d * xh).abs().sum(0)).all()
    assert ((dbias.cpu().double() - d.sum(0)).abs() <= 8 * U * d.abs().sum(0)).all()


def test_gradient_norm(mm, zeros):
    n = (1 << 31) + 4099
    p = torch.nn.Parameter(zeros(1))
    big = zeros(n)
    tail = torch.randn(4097, generator=gen(1))
    big[n - 4097:].copy_(mm.to_device(tail))
    q = torch.nn.Parameter(zeros(n))
    q.grad = big
    p.grad = mm.to_device(torch.ones(1))
    want = (tail.double().square().sum() + 1).sqrt()
    norm = mm.optim.clip_grad_norm_([p, q], 1.0)
    assert abs(norm.cpu().double() - want) <= 1.02 * U * want
    coef = 1.0 / (want.item() + 1e-6)
    assert ((q.grad[n - 4097:].cpu().double() - coef * tail.double()).abs() <= 5.1 * U * tail.double().abs()).all()
    assert q.grad[:5].cpu().tolist() == [0.0] * 5
