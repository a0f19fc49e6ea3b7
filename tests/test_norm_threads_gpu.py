"""Group norm, clipping and the clipped step called from several host threads at once: each thread's
results are those it gets alone."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def work(mm, seed):
    """A few forward and backward passes (kernels that hold the maps and kernels that walk them), each clipped
    in place and inside a step."""
    g = torch.Generator()
    g.manual_seed(seed)
    out = []
    for n, c, side, groups in ((3, 32, 9, 4), (2, 48, 64, 8), (1, 130, 120, 2)):
        x, dy = (mm.to_device(torch.randn(n, c, side, side, generator=g)) for _ in range(2))
        w, b = (torch.nn.Parameter(mm.to_device(torch.randn(c, generator=g))) for _ in range(2))
        leaf = x.detach().requires_grad_(True)
        y = mm.group_norm(leaf, groups, w, b, activation="silu")
        for p, grad in zip((w, b, leaf), torch.autograd.grad(y, (w, b, leaf), dy)):
            p.grad = grad
        norm = mm.optim.clip_grad_norm_([w, b, leaf], 0.5)
        opt = mm.optim.AdamW([w, b], lr=1e-2, max_grad_norm=0.25)
        opt.step()
        out += [t.detach().cpu() for t in (y, norm, w.grad, leaf.grad, w, b, opt.grad_norm)]
    return out


def test_threads_at_once(mm):
    want = [work(mm, seed) for seed in range(4)]
    got, errors = {}, []

    def run(seed):
        try:
            got[seed] = [work(mm, seed) for _ in range(5)]
        except BaseException as e:  # (shown by the main thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(seed,)) for seed in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not errors, errors
    for seed in range(4):
        for turn in got[seed]:
            assert all(torch.equal(a, b) for a, b in zip(turn, want[seed]))
