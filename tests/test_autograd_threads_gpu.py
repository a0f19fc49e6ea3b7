"""Autograd's worker threads: off around backward(), and by init only where the
process sees a single GPU."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


class Where(torch.autograd.Function):
    """Says on which thread its backward ran."""

    @staticmethod
    def forward(ctx, x, seen):
        ctx.seen = seen
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        ctx.seen.append(threading.get_ident())
        return g, None


@pytest.mark.parametrize("on", [True, False])
def test_the_setting_is_left_as_it_was(mm, on):
    with torch.autograd.set_multithreading_enabled(on):
        assert torch._C._is_multithreading_enabled() == on
        x = mm.to_device(torch.ones(4, 8)).requires_grad_(True)
        w = mm.to_device(torch.ones(6, 8)).requires_grad_(True)
        seen = []
        y = Where.apply(mm.linear(x, w), seen)
        y.backward(mm.to_device(torch.ones(4, 6)), retain_graph=True)
        assert seen.pop() == threading.get_ident()
        assert torch._C._is_multithreading_enabled() == on
        assert torch.equal(x.grad.cpu(), torch.full((4, 8), 6.0))
        gx, = torch.autograd.grad(y, x, mm.to_device(torch.ones(4, 6)))
        assert torch.equal(gx.cpu(), torch.full((4, 8), 6.0))
        assert (seen.pop() == threading.get_ident()) == (not on)
        with pytest.raises(RuntimeError):
            y.backward(mm.to_device(torch.ones(4, 7)))
        assert torch._C._is_multithreading_enabled() == on


@pytest.mark.parametrize("devices", [1, 2, 8])
def test_init_leaves_it_where_workers_could_run_side_by_side(mm, monkeypatch, devices):
    from matrixman_b200 import api, runtime
    monkeypatch.setattr(runtime, "device_count", lambda: devices)
    for on in (True, False):
        with torch.autograd.set_multithreading_enabled(on):
            monkeypatch.setattr(api, "_backend", None)
            mm.init()
            assert torch._C._is_multithreading_enabled() == (on and devices > 1)


def test_a_scalar_loss_and_another_thread(mm):
    """backward() without arguments, and from a thread that never called init."""
    x = mm.to_device(torch.ones(4, 8)).requires_grad_(True)
    w = mm.to_device(torch.ones(6, 8)).requires_grad_(True)
    mm.linear(x, w).sum(dim=1).sum(dim=0).backward()
    assert torch.equal(w.grad.cpu(), torch.full((6, 8), 4.0))
    got = []

    def work():
        try:
            seen = []
            Where.apply(mm.linear(x, w), seen).sum(dim=1).sum(dim=0).backward()
            got.append((seen[0] == threading.get_ident(), torch._C._is_multithreading_enabled()))
        except Exception as e:  # for the assertion below
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join(60)
    assert got == [(True, True)]  # (the setting is each thread's own)
    assert torch.equal(w.grad.cpu(), torch.full((6, 8), 8.0))
