"""Group norm, linear layers, clipping and AdamW used together: the training step of
a block over channels-last feature maps, prepared models with group norms, and
torch's own clipping.

Gradients go through two products of k <= 96 terms and one norm over m <= 3000
values forward, and their backward passes.  Each product's error has at most
(sqrt(k) + 32) u of the norm of its terms' magnitudes, u = 2^-24, and for terms of
random sign that norm is about 0.64 sqrt(k) times the result's: 2e-5 of the result's
norm for k = 96.  The norm's statistics are off by less than 160 u of magnitudes
that are at most 3 standard deviations here: 3e-5.  Both are passed on by factors of
order one, six products and three norms in all: 3e-4 of a gradient's norm."""

import math

import pytest
import torch
import torch.nn.functional as F
from torch import nn

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KW = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def weights(c, k, classes):
    def randn(*s, i):
        return torch.randn(*s, generator=gen(i))
    return {"w1": randn(k, c, i=1) / math.sqrt(c), "b1": 0.1 * randn(k, i=2), "g": 1 + 0.1 * randn(k, i=3),
            "b": 0.1 * randn(k, i=4), "w2": randn(c, k, i=5) / math.sqrt(k), "b2": 0.1 * randn(c, i=6),
            "w3": randn(classes, c, i=7) / math.sqrt(c), "b3": 0.1 * randn(classes, i=8)}


def on_device(mm, p, x, groups):
    """x [N, H, W, C]: 1 x 1 convolutions as linear layers over the pixels."""
    h = mm.linear(x, p["w1"], p["b1"]).permute(0, 3, 1, 2)
    h = mm.group_norm(h, groups, p["g"], p["b"], activation="silu").permute(0, 2, 3, 1)
    y = mm.linear(h, p["w2"], p["b2"], residual=x)
    return mm.linear(y.mean(dim=(1, 2)), p["w3"], p["b3"])


def in_float64(p, x, groups):
    h = (x @ p["w1"].t() + p["b1"]).permute(0, 3, 1, 2)
    h = F.silu(F.group_norm(h, groups, p["g"], p["b"])).permute(0, 2, 3, 1)
    y = h @ p["w2"].t() + p["b2"] + x
    return y.mean(dim=(1, 2)) @ p["w3"].t() + p["b3"]


def loss_of(logits, t):
    return F.nll_loss(torch.log_softmax(logits, 1), t)


@pytest.mark.parametrize("n,h,w,c,k,groups", [(2, 3, 5, 24, 40, 5), (4, 17, 13, 64, 96, 8), (3, 20, 40, 32, 48, 16)])
def test_clipped_training_steps(mm, n, h, w, c, k, groups):
    host = weights(c, k, 10)
    params = {name: nn.Parameter(mm.to_device(v)) for name, v in host.items()}
    opt = mm.optim.AdamW(list(params.values()), max_grad_norm=0.05, **KW)
    for step in range(3):
        x = torch.randn(n, h, w, c, generator=gen(10 + step))
        t = torch.randint(0, 10, (n,), generator=gen(20 + step))
        ref = {name: p.detach().cpu().double().requires_grad_(True) for name, p in params.items()}
        opt.zero_grad()
        loss = loss_of(on_device(mm, params, mm.to_device(x), groups), mm.to_device(t))
        loss.backward()
        want = loss_of(in_float64(ref, x.double(), groups), t)
        want.backward()
        assert abs(loss.detach().cpu().item() - want.item()) <= 3e-4 * abs(want.item())
        for name, p in params.items():
            err = (p.grad.cpu().double() - ref[name].grad).norm() / ref[name].grad.norm()
            assert err <= 3e-4, (name, err)
        # (the norm of the device's own gradients, so that its rounding is all)
        norm = torch.cat([p.grad.cpu().double().reshape(-1) for p in params.values()]).norm()
        before = {name: p.detach().cpu() for name, p in params.items()}
        opt.step()
        assert abs(opt.grad_norm.cpu().double() - norm) <= 1.02 * U * norm and norm > 0.05
        assert all(not torch.equal(before[name], p.detach().cpu()) for name, p in params.items())


def test_captured_training_step(mm):
    """Forward, backward, clipping and step in one graph, replayed: the same bits as
    eager steps, with an eager graph of the same leaves alive meanwhile."""
    host = weights(32, 64, 10)
    x = mm.to_device(torch.randn(4, 12, 9, 32, generator=gen(1)))
    dy = mm.to_device(torch.randn(4, 10, generator=gen(2)))
    rt = x.runtime
    runs = []
    for _ in range(2):
        params = {name: nn.Parameter(mm.to_device(v)) for name, v in host.items()}
        runs.append((params, mm.optim.AdamW(list(params.values()), max_grad_norm=1.0, **KW)))

    def step(params, opt):
        y = on_device(mm, params, x, 8)
        for p, g in zip(params.values(), torch.autograd.grad(y, list(params.values()), dy)):
            p.grad = g
        total = mm.optim.clip_grad_norm_(params.values(), 2.0)
        opt.step()
        return total

    for run in runs:
        step(*run)
    kept = on_device(mm, runs[0][0], x, 8)
    rt.synchronize()
    rt.capture_begin()
    total = step(*runs[0])
    graph = rt.capture_end()
    for _ in range(3):
        graph.replay()
        want = step(*runs[1])
        assert torch.equal(total.cpu(), want.cpu())
        assert torch.equal(runs[0][1].grad_norm.cpu(), runs[1][1].grad_norm.cpu())
    for name in host:
        assert torch.equal(runs[0][0][name].detach().cpu(), runs[1][0][name].detach().cpu()), name
    del kept


@pytest.mark.parametrize("order", [2.0, 1.0, math.inf])
def test_torch_clipping(mm, order):
    """torch.nn.utils.clip_grad_norm_ on MatrixMan parameters."""
    sizes = [(40, 30), (7,), (3, 3, 5)]
    grads = [torch.randn(s, generator=gen(i)) for i, s in enumerate(sizes)]
    params = [nn.Parameter(mm.to_device(torch.zeros(s))) for s in sizes]
    ref = [nn.Parameter(torch.zeros(s, dtype=torch.float64)) for s in sizes]
    for p, q, g in zip(params, ref, grads):
        p.grad, q.grad = mm.to_device(g), g.double()
    total = nn.utils.clip_grad_norm_(params, 0.3, order)
    want = nn.utils.clip_grad_norm_(ref, 0.3, order)
    # three norms' roundings and their own; reciprocal, product, clamp, product behind it
    assert abs(total.cpu().double() - want) <= 4 * U * want
    for p, q in zip(params, ref):
        assert ((p.grad.cpu().double() - q.grad).abs() <= 10 * U * q.grad.abs()).all()
    assert abs(torch.linalg.vector_norm(params[0].grad, order, dim=(0, 1), keepdim=True).cpu().double()
               - torch.linalg.vector_norm(ref[0].grad, order)) <= 12 * U * want
    with pytest.raises(NotImplementedError):
        torch.linalg.vector_norm(params[0].grad, order, dim=1)


def model(norm_act):
    torch.manual_seed(3)
    m = nn.Sequential(nn.Conv2d(3, 32, 3, stride=2, padding=1), nn.GroupNorm(8, 32), norm_act(),
                      nn.Conv2d(32, 48, 3, padding=1), nn.GroupNorm(4, 48), norm_act(), nn.Conv2d(48, 20, 1),
                      nn.GroupNorm(5, 20, affine=False)).eval()
    with torch.no_grad():
        for layer in m:
            if isinstance(layer, nn.GroupNorm) and layer.weight is not None:
                layer.weight.add_(0.2 * torch.randn(layer.weight.shape, generator=gen(4)))
                layer.bias.add_(0.2 * torch.randn(layer.bias.shape, generator=gen(5)))
    return m


@pytest.mark.parametrize("act", [nn.SiLU, nn.ReLU, nn.GELU, nn.Sigmoid])
@pytest.mark.parametrize("batch", [1, 5])
def test_prepared_model(mm, act, batch):
    """Eager, captured and replayed, against torch on the CPU with the convolutions' bar
    (the norms' share of the error is far below it)."""
    m = model(act)
    x = torch.randn(batch, 3, 40, 52, generator=gen(6))
    with torch.no_grad():
        want = m(x)
        p = mm.prepare(m)
        for _ in range(3):
            got = p(mm.to_device(x)).cpu()
            assert (got - want).abs().max() <= 1e-4 * want.abs().max()
