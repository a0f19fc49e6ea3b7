"""Layer norm, linear layers with activation and residual, and AdamW used
together: the training step of a residual feed-forward block.

Gradients go through two products of k <= 512 terms forward and four backward.
Each product's error has at most (sqrt(k) + 32) u of the norm of its terms'
magnitudes, u = 2^-24, and for terms of random sign that norm is about 0.64
sqrt(k) times the result's: 5e-5 of the result's norm for k = 512, so 3e-4 for
all six.  Parameters are compared with AdamW's formula in float64 on the
device's own gradients, since its first steps go by the gradients' signs."""

import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KW = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def block(width, hidden, seed=0):
    def randn(*s, i):
        return torch.randn(*s, generator=gen(seed + i))
    return {"g": 1 + 0.1 * randn(width, i=1), "b": 0.1 * randn(width, i=2),
            "w1": randn(hidden, width, i=3) / math.sqrt(width), "b1": 0.1 * randn(hidden, i=4),
            "w2": randn(width, hidden, i=5) / math.sqrt(hidden), "b2": 0.1 * randn(width, i=6)}


def on_device(mm, p, x):
    h = F.layer_norm(x, (x.shape[-1],), p["g"], p["b"], 1e-5)
    u = mm.linear(h, p["w1"], p["b1"], activation="gelu")
    return mm.linear(u, p["w2"], p["b2"], residual=x)


def in_float64(p, x):
    h = F.layer_norm(x, (x.shape[-1],), p["g"], p["b"], 1e-5)
    u = F.gelu(h @ p["w1"].t() + p["b1"])
    return u @ p["w2"].t() + p["b2"] + x


def loss_of(y, t):
    return F.nll_loss(torch.log_softmax(y.reshape(-1, y.shape[-1]), 1), t)


# A few tokens (the kernels for small sizes), a ragged batch, and one that runs on the tensor cores.
@pytest.mark.parametrize("batch,length,width,hidden", [(1, 3, 40, 96), (3, 67, 130, 257), (4, 300, 256, 512)])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(mm, batch, length, width, hidden, bits):
    host = block(width, hidden)
    params = {k: torch.nn.Parameter(mm.to_device(v)) for k, v in host.items()}
    opt = mm.optim.AdamW(list(params.values()), state_bits=bits, **KW)
    for step in range(1, 4):
        x = torch.randn(batch, length, width, generator=gen(10 + step))
        t = torch.randint(0, width, (batch * length,), generator=gen(20 + step))
        t[::5] = -100  # padding
        before = {k: p.detach().cpu() for k, p in params.items()}
        moments = {k: [s.cpu().double().numpy() for s in opt.state_values(p)] for k, p in params.items()}
        opt.zero_grad()
        loss = loss_of(on_device(mm, params, mm.to_device(x)), mm.to_device(t))
        loss.backward()
        ref = {k: v.double().requires_grad_(True) for k, v in before.items()}
        want = loss_of(in_float64(ref, x.double()), t)
        want.backward()
        assert abs(loss.detach().cpu().item() - want.item()) <= 3e-4 * abs(want.item())
        for k, p in params.items():
            err = (p.grad.cpu().double() - ref[k].grad).norm() / ref[k].grad.norm()
            assert err <= 3e-4, (k, err)
        opt.step()
        for k, p in params.items():
            m, v = moments[k]
            g = p.grad.cpu().double().numpy()
            m, v = 0.9 * m + 0.1 * g, 0.99 * v + 0.01 * g * g
            upd = KW["lr"] / (1 - 0.9 ** step) * m / (np.sqrt(v / (1 - 0.99 ** step)) + 1e-8)
            p64 = before[k].double().numpy() * (1 - KW["lr"] * KW["weight_decay"]) - upd
            # roundings of the parameter and of the step; m may cancel, so the terms' own size counts
            size = KW["lr"] / (1 - 0.9 ** step) * (abs(0.9 * moments[k][0]) + abs(0.1 * g)) / (np.sqrt(v / (1 - 0.99 ** step)) + 1e-8)
            assert (abs(p.detach().cpu().double().numpy() - p64) <= U * (3 * abs(before[k].double().numpy()) + 3 * abs(p64) + 24 * size)).all(), k


def test_captured_training_step(mm):
    """Forward, backward and optimiser in one graph, replayed: the same bits as
    eager steps, with an eager graph of the same leaves alive meanwhile."""
    width, hidden = 256, 512
    host = block(width, hidden)
    x, t = torch.randn(300, width, generator=gen(1)), torch.randint(0, width, (300,), generator=gen(2))
    runs = []
    for _ in range(2):
        params = {k: torch.nn.Parameter(mm.to_device(v)) for k, v in host.items()}
        runs.append((params, mm.optim.AdamW(list(params.values()), **KW)))
    dx = mm.to_device(x)
    dy = mm.to_device(torch.randn(300, width, generator=gen(3)))
    rt = dx.runtime

    def step(params, opt):
        y = on_device(mm, params, dx)
        for p, g in zip(params.values(), torch.autograd.grad(y, list(params.values()), dy)):
            p.grad = g
        opt.step()
        return y

    for run in runs:
        step(*run)
    kept = on_device(mm, runs[0][0], dx)  # an eager graph of the leaves, alive during the capture
    rt.synchronize()
    rt.capture_begin()
    step(*runs[0])
    graph = rt.capture_end()
    for _ in range(3):
        graph.replay()
        step(*runs[1])
    for k in host:
        assert torch.equal(runs[0][0][k].detach().cpu(), runs[1][0][k].detach().cpu()), k
    del kept
