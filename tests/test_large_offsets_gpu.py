"""Tensors of more than 2^31 elements: the last rows come out as they do alone.

The rows in front are zero (one fill), so only the last ones are compared; the
same kernel works on them with the same order of sums, so bits are equal where
the size does not change the kernel, and otherwise within the sums' roundings."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


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


def test_layer_norm(mm, zeros):
    rows, width = (1 << 31) // 4096 + 5, 4096
    tail, w, b = torch.randn(3, width, generator=gen(1)), torch.randn(width, generator=gen(2)), torch.randn(width, generator=gen(3))
    dy = torch.randn(3, width, generator=gen(4))
    x, g = zeros(rows, width), zeros(rows, width)
    x[rows - 3:].copy_(mm.to_device(tail))
    g[rows - 3:].copy_(mm.to_device(dy))
    dw, db = mm.to_device(w).requires_grad_(True), mm.to_device(b).requires_grad_(True)
    x.requires_grad_(True)
    y = F.layer_norm(x, (width,), dw, db)
    grads = torch.autograd.grad(y, (x, dw, db), g)
    leaf = mm.to_device(tail).requires_grad_(True)
    want = F.layer_norm(leaf, (width,), dw, db)
    wants = torch.autograd.grad(want, (leaf, dw, db), mm.to_device(dy))
    assert torch.equal(y.detach()[rows - 3:].cpu(), want.detach().cpu())
    assert torch.equal(grads[0][rows - 3:].cpu(), wants[0].cpu())
    for a, c in zip(grads[1:], wants[1:]):  # three terms and zeros
        assert ((a.cpu() - c.cpu()).abs() <= 4 * U * (c.cpu().abs() + dy.abs().sum(0) * 8)).all()


def test_linear(mm, zeros):
    m, n, k = (1 << 21) + 3, 1030, 8
    tail, w = torch.randn(3, k, generator=gen(1)), torch.randn(n, k, generator=gen(2))
    dy = torch.randn(3, n, generator=gen(3))
    x = zeros(m, k)
    x[m - 3:].copy_(mm.to_device(tail))
    x.requires_grad_(True)
    dw = mm.to_device(w).requires_grad_(True)
    y = mm.linear(x, dw, activation="silu")
    z = tail.double() @ w.double().t()
    size = tail.double().abs() @ w.double().abs().t()
    got = y.detach()[m - 3:].cpu().double()
    assert ((got - z * torch.sigmoid(z)).abs() <= 1.13 * 35 * U * size + 16 * U * (z.abs() + 1)).all()
    g = zeros(m, n)
    g[m - 3:].copy_(mm.to_device(dy))
    gx, gw = torch.autograd.grad(y, (x, dw), g)
    s = torch.sigmoid(z)
    dz = dy.double() * s * (1 + z * (1 - s))
    edz = dy.double().abs() * (1.13 * 35 * U * size + 24 * U * (1 + z.abs()))
    err = (gx[m - 3:].cpu().double() - dz @ w.double()).abs()
    assert (err <= 2 * (n + 11) * U * (dz.abs() @ w.double().abs()) + edz @ w.double().abs()).all()
    assert torch.equal(gx[:m - 3].sum(dim=0).cpu(), torch.zeros(k))
    err = (gw.cpu().double() - dz.t() @ tail.double()).abs()
    assert (err <= 32 * U * (dz.abs().t() @ tail.double().abs()) + edz.t() @ tail.double().abs()).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(mm, zeros, bits):
    n = (1 << 31) + 1000
    p = torch.nn.Parameter(zeros(n))
    p.grad = zeros(n)
    g = torch.randn(300, generator=gen(1))
    p.grad[n - 300:].copy_(mm.to_device(g))
    opt = mm.optim.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=bits)
    opt.step()
    got = p.detach()[n - 300:].cpu()
    # the first step moves by lr against the gradient's sign, up to about 16 roundings and eps over the gradient
    assert ((got + 0.5 * g.sign()).abs() <= 0.5 * (16 * U + 1e-8 / g.abs())).all()
    assert torch.equal(p.detach()[n - 1300:n - 300].cpu(), torch.zeros(1000))
