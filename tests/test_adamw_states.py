"""What matrixman.optim.AdamW refuses before anything reaches a device: tensors of
made-up addresses on a runtime that has no device, and every launch recorded."""

import pytest
import torch

import matrixman_b200 as matrixman
from matrixman_b200 import ops, optim
from matrixman_b200.privateuse import register_privateuse1_backend
from matrixman_b200.runtime import DeviceStorage
from matrixman_b200.tensor import MatrixManTensor, contiguous_strides, numel


class FakeRuntime:
    closed = True  # nothing to release
    stream = 0
    capturing = False

    def __init__(self, index=0):
        self.index = index
        self.next = 1 << 20

    def new_storage(self, n, dtype=torch.float32, kind=0, stream=None):
        at = self.next
        self.next += (max(n, 1) * 8 + 511) // 512 * 512
        return DeviceStorage(self, at, max(n, 1) * (4 if dtype == torch.float32 else 8), dtype, kind)


def tensor(rt, *shape, strides=None, dtype=torch.float32):
    strides = contiguous_strides(shape) if strides is None else strides
    span = (sum((n - 1) * s for n, s in zip(shape, strides)) + 1) if numel(shape) else 1
    return MatrixManTensor(rt.new_storage(span, dtype), shape, 0, strides)


@pytest.fixture
def rt():
    register_privateuse1_backend()
    return FakeRuntime()


@pytest.fixture
def launches(monkeypatch):
    got = []
    monkeypatch.setattr(ops, "_launch", lambda name, *args: got.append(name))
    return got


def state_of(rt, shape, bits):
    n = numel(shape)
    blocks = (n + 255) // 256
    if bits == 32:
        return {"step": tensor(rt), "exp_avg": tensor(rt, *shape), "exp_avg_sq": tensor(rt, *shape)}
    return {"step": tensor(rt), "exp_avg_code": tensor(rt, 64 * blocks), "exp_avg_scale": tensor(rt, blocks),
            "exp_avg_sq_code": tensor(rt, 64 * blocks), "exp_avg_sq_scale": tensor(rt, blocks)}


def made(rt, shape, bits):
    p = torch.nn.Parameter(tensor(rt, *shape))
    opt = matrixman.optim.AdamW([p], state_bits=bits)
    p.grad = tensor(rt, *shape)
    opt.state[p] = state_of(rt, shape, bits)
    return opt, p


BAD = [(32, "exp_avg", lambda rt: tensor(rt, 10), "shape"),
       (32, "exp_avg_sq", lambda rt: tensor(rt, 10, 100), "shape"),
       (32, "exp_avg", lambda rt: tensor(rt, 1000, dtype=torch.int64), "float32"),
       (32, "exp_avg", lambda rt: tensor(rt, 1000, strides=(2,)), "strides"),
       (32, "exp_avg_sq", lambda rt: torch.zeros(1000), "CUDA-backed"),
       (32, "exp_avg", lambda rt: None, "has no"),
       (8, "exp_avg_code", lambda rt: tensor(rt, 64 * 4 - 1), "dense values"),
       (8, "exp_avg_code", lambda rt: tensor(rt, 64 * 4, strides=(2,)), "dense values"),
       (8, "exp_avg_sq_code", lambda rt: tensor(rt, 64), "dense values"),
       (8, "exp_avg_scale", lambda rt: tensor(rt, 3), "dense values"),
       (8, "exp_avg_sq_scale", lambda rt: tensor(rt, 3), "dense values"),
       (8, "exp_avg_sq_scale", lambda rt: None, "has no")]
BAD += [(bits, "step", make, words) for bits in (32, 8)
        for make, words in ((lambda rt: tensor(rt, 0), "dense values"), (lambda rt: tensor(rt, 2), "dense values"),
                            (lambda rt: tensor(rt, dtype=torch.int64), "float32"), (lambda rt: None, "has no"),
                            (lambda rt: tensor(FakeRuntime()), "device"), (lambda rt: 3.0, "CUDA-backed"))]


@pytest.mark.parametrize("bits,name,make,words", BAD)
def test_states_of_other_sizes_are_refused(rt, launches, bits, name, make, words):
    opt, p = made(rt, (1000,), bits)
    opt.step()
    assert launches == ["mm_adamw"]
    value = make(rt)
    if value is None:
        del opt.state[p][name]
    else:
        opt.state[p][name] = value
    calls = (opt.step, lambda: opt.state_values(p), opt.state_dict,
             lambda: opt.set_state_values(p, tensor(rt, 1000), tensor(rt, 1000)))
    for call in calls:
        with pytest.raises((RuntimeError, NotImplementedError), match=words):
            call()
    assert launches == ["mm_adamw"]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shape", [(1000,), (256,), (3, 5), (0, 4), ()])
def test_states_of_the_right_sizes_pass(rt, launches, bits, shape):
    opt, p = made(rt, shape, bits)
    opt.step()
    opt.set_state_values(p, tensor(rt, *shape), tensor(rt, *shape))
    assert launches[0] == "mm_adamw" and len(launches) > 1


def test_state_of_another_shape_with_as_many_values(rt, launches):
    opt, p = made(rt, (20, 50), 32)
    opt.state[p]["exp_avg"] = tensor(rt, 50, 20)
    with pytest.raises(RuntimeError, match="shape"):
        opt.step()
    opt.state[p]["exp_avg"] = tensor(rt, 20, 50, strides=(1, 20))
    with pytest.raises(RuntimeError, match="strides"):
        opt.step()
    assert launches == []


@pytest.mark.parametrize("shape", [(0,), (2,)])
def test_fused_step_of_another_size(rt, launches, shape):
    p, g, m, v = (tensor(rt, 40) for _ in range(4))
    kw = dict(lr=1e-3, beta1=0.9, beta2=0.999, weight_decay=0.0, eps=1e-8, amsgrad=False, maximize=False)
    for op in (torch.ops.aten._fused_adamw_, torch.ops.aten._fused_adam_):
        op([p], [g], [m], [v], [], [tensor(rt)], **kw)
        with pytest.raises(RuntimeError, match="one value per step"):
            op([p], [g], [m], [v], [], [tensor(rt, *shape)], **kw)
    assert launches == ["mm_adamw"] * 2


@pytest.mark.parametrize("bits", [32, 8])
def test_no_state_is_made_during_capture(rt, launches, monkeypatch, bits):
    monkeypatch.setattr(ops, "full", lambda rt, shape, value: tensor(rt, *shape))
    monkeypatch.setattr(ops, "fill_", lambda t, value: t)
    params = [torch.nn.Parameter(tensor(rt, 300)) for _ in range(2)]
    opt = matrixman.optim.AdamW(params, state_bits=bits)
    params[0].grad = tensor(rt, 300)
    opt.step()
    params[1].grad = tensor(rt, 300)
    rt.capturing = True
    for call in (opt.step, lambda: opt.state_values(params[1]),
                 lambda: opt.set_state_values(params[1], tensor(rt, 300), tensor(rt, 300))):
        with pytest.raises(RuntimeError, match="capture"):
            call()
    assert launches == ["mm_adamw"] and not opt.state.get(params[1])
    params[1].grad = None
    opt.step()
    rt.capturing = False
    params[1].grad = tensor(rt, 300)
    opt.step()
    assert launches == ["mm_adamw"] * 3


def test_loading_keeps_what_a_scheduler_left_in_the_groups(rt, launches):
    p = torch.nn.Parameter(tensor(rt, 300))
    opt = matrixman.optim.AdamW([p], lr=0.5)
    scheduler = torch.optim.lr_scheduler.StepLR(opt, step_size=2, gamma=0.1)
    saved, at = opt.state_dict(), scheduler.state_dict()
    new = matrixman.optim.AdamW([torch.nn.Parameter(tensor(rt, 300))], lr=1.0)
    new.load_state_dict(saved)
    assert new.param_groups[0]["initial_lr"] == 0.5 and len(new.param_groups[0]["params"]) == 1
    assert new.param_groups[0]["params"][0] is not p
    resumed = torch.optim.lr_scheduler.StepLR(new, step_size=2, gamma=0.1, last_epoch=at["last_epoch"])
    assert resumed.base_lrs == [0.5]
    saved["param_groups"][0]["lr"] = 7.0
    assert new.param_groups[0]["lr"] == 0.5


def test_what_cannot_be_loaded_changes_nothing(rt, launches, monkeypatch):
    monkeypatch.setattr(ops, "full", lambda rt, shape, value: tensor(rt, *shape))
    monkeypatch.setattr(ops, "fill_", lambda t, value: t)
    params = [torch.nn.Parameter(tensor(rt, 300)) for _ in range(2)]
    opt = matrixman.optim.AdamW(params, lr=0.5)
    for p in params:
        opt.state[p] = state_of(rt, (300,), 32)
    before = {p: dict(opt.state[p]) for p in params}
    right = {"step": 1.0, "exp_avg": tensor(rt, 300), "exp_avg_sq": tensor(rt, 300)}
    for wrong in ({"step": 1.0, "exp_avg": tensor(rt, 299), "exp_avg_sq": tensor(rt, 300)},
                  {"step": 1.0, "exp_avg": tensor(rt, 300)}):
        saved = {"state": {0: right, 1: wrong}, "param_groups": [{"params": [0, 1], "lr": 0.25, "other": 1}]}
        with pytest.raises((ValueError, KeyError)):
            opt.load_state_dict(saved)
        assert opt.param_groups[0]["lr"] == 0.5 and "other" not in opt.param_groups[0]
        assert opt.param_groups[0]["params"] == params
        assert all(opt.state[p][k] is v for p in params for k, v in before[p].items())
