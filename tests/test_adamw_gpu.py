"""matrixman.optim.AdamW against the update's formulas.

32-bit states against float64: u = 2^-24.  m and v take two products and a sum
with factors that are rounded themselves: 4 u (6 u for v) of their terms.  The
step lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps) adds about 12
roundings of its own value to m's and half of v's; p takes 3 u more of itself.

8-bit states against a restatement in numpy float32, whose operations are
rounded one by one as the kernel's are: the codes, the scales and p are equal
bit for bit."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(3,), (256,), (1, 255), (257,), (512, 784), (10, 256), (4096,), (4097,), (5, 7, 11), (1,), (12289,), (0, 4)]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed))


def params_of(mm, shapes, seed=1):
    host = [0.1 * randn(*s, seed=seed + i) for i, s in enumerate(shapes)]
    return host, [torch.nn.Parameter(mm.to_device(t)) for t in host]


def grads_of(shapes, step, scale=1.0):
    return [scale * randn(*s, seed=1000 * step + i) * math.exp(i % 5 - 2) for i, s in enumerate(shapes)]


def step64(p, g, m, v, t, lr, b1, b2, eps, wd):
    p, g, m, v = (np.asarray(q, dtype=np.float64) for q in (p, g, m, v))
    nm, nv = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    em = 4 * U * (abs(b1 * m) + abs((1 - b1) * g))
    ev = 6 * U * nv
    d = np.sqrt(nv / (1 - b2 ** t)) + eps
    s = lr / (1 - b1 ** t)
    np_ = p * (1 - lr * wd) - s * nm / d
    ep = 3 * U * (abs(p) + abs(np_)) + s * em / d + abs(s * nm / d) * (12 + 3) * U
    return np_, nm, nv, ep, em, ev


@pytest.mark.parametrize("maximize", [False, True])
def test_32_bit_steps(mm, maximize):
    kw = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
    host, params = params_of(mm, SHAPES)
    opt = mm.optim.AdamW(params, maximize=maximize, **kw)
    for t in range(1, 4):
        before = [(p.detach().cpu(), *(s.cpu() for s in opt.state_values(p))) for p in params]
        gs = grads_of(SHAPES, t)
        for p, g in zip(params, gs):
            p.grad = mm.to_device(g)
        opt.step()
        for p, g, (p0, m0, v0) in zip(params, gs, before):
            want = step64(p0, -g if maximize else g, m0, v0, t, kw["lr"], *kw["betas"], kw["eps"], kw["weight_decay"])
            got = [q.cpu().double().numpy() for q in (p.detach(), *opt.state_values(p))]
            for a, b, e in zip(got, want[:3], want[3:]):
                assert (abs(a - b) <= e).all()
        assert all(float(opt.state[p]["step"].cpu()) == t for p in params)


def f32(x):
    return np.float32(x)


def encode(a, shift, top, least):
    size = np.abs(a)
    scale = size.max()
    if not scale >= np.float32(2.0 ** -126):
        scale = f32(0)
    with np.errstate(all="ignore"):
        bits = (size * (f32(1) / scale)).astype(np.float32).view(np.int32).astype(np.int64)
    code = ((bits + ((1 << (shift - 1)) - 1) + ((bits >> shift) & 1)) >> shift) - (0x3F800000 >> shift) + top
    code = np.where((size > 0) & (scale > 0), np.clip(code, least, top), 0)
    return code, scale


def decode(code, scale, shift, top):
    q = ((code + (0x3F800000 >> shift) - top) << shift).astype(np.int32).view(np.float32)
    return np.where(code > 0, q, f32(0)) * scale


def stored(a, shift, top, least):
    out = np.zeros_like(a)
    for at in range(0, a.size, 256):
        part = a[at:at + 256]
        value = decode(*encode(part, shift, top, least), shift, top)
        out[at:at + 256] = np.where(part < 0, -value, value)
    return out


def step8(p, g, m, v, t, lr, b1, b2, eps, wd):
    """p, m, v after a step, in numpy float32; m and v as their codes' values."""
    p, g, m, v = (np.asarray(q, dtype=np.float32).reshape(-1) for q in (p, g, m, v))
    nm = m * f32(b1) + g * f32(1 - b1)
    nr = np.sqrt(v * f32(b2) + (g * g) * f32(1 - b2))
    step, root = f32(lr / (1 - b1 ** t)), f32(1 / math.sqrt(1 - b2 ** t))
    np_ = p * f32(1 - lr * wd) - (nm / (nr * root + f32(eps))) * step
    sr = stored(nr, 19, 255, 1)
    return np_, stored(nm, 20, 127, 0), sr * sr


def test_8_bit_steps_equal_their_restatement(mm):
    kw = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
    host, params = params_of(mm, SHAPES)
    opt = mm.optim.AdamW(params, state_bits=8, **kw)
    state = [(h.numpy().reshape(-1), np.zeros(h.numel(), np.float32), np.zeros(h.numel(), np.float32)) for h in host]
    for t in range(1, 5):
        gs = grads_of(SHAPES, t)
        for p, g in zip(params, gs):
            g.view(-1)[::7] = 0.0
            p.grad = mm.to_device(g)
        opt.step()
        for i, (p, g) in enumerate(zip(params, gs)):
            state[i] = step8(state[i][0], g, state[i][1], state[i][2], t, kw["lr"], *kw["betas"], kw["eps"],
                             kw["weight_decay"])
            got = [q.cpu().numpy().reshape(-1) for q in (p.detach(), *opt.state_values(p))]
            for name, a, b in zip(("p", "exp_avg", "exp_avg_sq"), got, state[i]):
                assert np.array_equal(a, b), (t, SHAPES[i], name)


def test_8_bit_codes_are_near_and_stable(mm):
    """Half a step: 1/16 of m, 1/32 of sqrt(v) within 16 powers of two of the
    block's largest; a second round trip changes nothing."""
    n = 1000
    m = randn(n, seed=1) * torch.logspace(-4, 0, n)
    v = (randn(n, seed=2) * torch.logspace(-4, 0, n)) ** 2
    m[5], v[6] = 0.0, 0.0
    p = torch.nn.Parameter(mm.to_device(torch.zeros(n)))
    opt = mm.optim.AdamW([p], state_bits=8)
    opt.set_state_values(p, m, v, step=3)
    gm, gv = (t.cpu() for t in opt.state_values(p))
    for at in range(0, n, 256):
        part = slice(at, at + 256)
        size, near = m[part].abs(), (gm - m)[part].abs()
        assert (near <= size / 16 * (1 + 8 * U) + size.max() * 2.0 ** -16).all()
        root, near = v[part].sqrt(), (gv.sqrt() - v.sqrt())[part].abs()
        assert (near <= root / 32 * (1 + 8 * U) + root.max() * 2.0 ** -15).all()
    assert gm[5] == 0 and gv[6] == 0 and (gv[v > 0] > 0).all()
    opt.set_state_values(p, gm, gv)
    assert all(torch.equal(a, b.cpu()) for a, b in zip((gm, gv), opt.state_values(p)))
    assert float(opt.state[p]["step"].cpu()) == 3


def test_8_bit_zero_tiny_and_non_finite_blocks(mm):
    n = 1024
    p = torch.nn.Parameter(mm.to_device(torch.ones(n)))
    opt = mm.optim.AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8)
    g = torch.zeros(n)
    g[256:512] = 1e-30           # squares vanish, m stays
    g[512:768] = 1.0
    g[600] = float("nan")
    g[768:] = -2.0
    p.grad = mm.to_device(g)
    opt.step()
    got = p.detach().cpu()
    m, v = (t.cpu() for t in opt.state_values(p))
    assert torch.equal(got[:256], torch.ones(256)) and (m[:256] == 0).all() and (v[:256] == 0).all()
    assert torch.isfinite(got[256:512]).all() and torch.isfinite(m[256:512]).all()
    assert torch.isnan(got[600]) and torch.isfinite(got[torch.arange(n) != 600]).all()
    assert torch.isnan(m[512:768]).all() and torch.isnan(v[512:768]).all()  # the block's states stay visible
    # the first step is lr in the gradient's direction: m / (1 - b1) over sqrt(v / (1 - b2)) is +-1 within 16 u
    assert ((got[768:] - 1.01).abs() <= 20 * U).all()


def test_views_strides_and_neighbours(mm):
    """Parameters inside one buffer, at odd offsets: nothing outside them moves."""
    for bits in (32, 8):
        buf = mm.to_device(torch.arange(3000.0))
        grad = mm.to_device(randn(3000, seed=1))
        a = torch.nn.Parameter(buf[1:778].detach())
        b = torch.nn.Parameter(buf[1001:2801].view(60, 30).t().detach())
        opt = mm.optim.AdamW([a, b], lr=0.5, weight_decay=0.0, state_bits=bits)
        a.grad = grad[3:780]
        b.grad = mm.to_device(randn(30, 60, seed=2))  # another order of dimensions than b's
        opt.step()
        got = buf.cpu()
        want = torch.arange(3000.0)
        inside = torch.zeros(3000, dtype=torch.bool)
        inside[1:778] = True
        inside[1001:2801] = True
        assert torch.equal(got[~inside], want[~inside])
        ga, gb = a.grad.cpu(), b.grad.cpu()
        # the first step moves by lr against the gradient's sign; numbers up to 2800 are rounded to 2^-13
        assert ((got[1:778] - want[1:778] + 0.5 * ga.sign()).abs() <= 2.0 ** -12).all()
        assert ((got[1001:2801].view(60, 30).t() - want[1001:2801].view(60, 30).t() + 0.5 * gb.sign()).abs() <= 2.0 ** -12).all()


def test_parameters_without_gradient_and_groups(mm):
    host, params = params_of(mm, [(300,), (40, 20), (7,)])
    opt = mm.optim.AdamW([{"params": params[:2], "lr": 0.1}, {"params": params[2:], "lr": 0.2, "weight_decay": 0.0}])
    params[1].grad = mm.to_device(torch.ones(40, 20))
    params[2].grad = mm.to_device(torch.ones(7))
    version = params[1]._version
    opt.step()
    assert params[1]._version > version and params[0] not in opt.state
    assert torch.equal(params[0].detach().cpu(), host[0])
    assert ((params[1].detach().cpu() - (host[1] * (1 - 0.1 * 0.01) - 0.1)).abs() <= 32 * U).all()
    assert ((params[2].detach().cpu() - (host[2] - 0.2)).abs() <= 32 * U).all()
    params[0].grad = mm.to_device(torch.ones(300))
    opt.step()
    assert [float(opt.state[p]["step"].cpu()) for p in params] == [1.0, 2.0, 2.0]


def test_many_tensors_take_several_launches(mm):
    shapes = [(i % 37 + 1,) for i in range(900)]
    host, params = params_of(mm, shapes)
    opt = mm.optim.AdamW(params, lr=0.25, weight_decay=0.0)
    for p in params:
        p.grad = mm.to_device(torch.ones(p.shape))
    opt.step()
    for h, p in zip(host, params):
        assert ((p.detach().cpu() - (h - 0.25)).abs() <= 32 * U).all()


def test_captured_step_counts_on(mm):
    for bits in (32, 8):
        host, params = params_of(mm, [(700,), (33, 9)])
        _, twins = params_of(mm, [(700,), (33, 9)])
        opts = [mm.optim.AdamW(q, lr=1e-2, state_bits=bits) for q in (params, twins)]
        gs = [mm.to_device(randn(*p.shape, seed=5)) for p in params]
        for q in (params, twins):
            for p, g in zip(q, gs):
                p.grad = g
        for o in opts:
            o.step()
        rt = params[0].runtime
        rt.synchronize()
        rt.capture_begin()
        opts[0].step()
        graph = rt.capture_end()
        for _ in range(3):
            graph.replay()
            opts[1].step()
        for p, q in zip(params, twins):
            assert torch.equal(p.detach().cpu(), q.detach().cpu())
            assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(opts[0].state_values(p), opts[1].state_values(q)))
        assert float(opts[0].state[params[0]]["step"].cpu()) == 4.0


@pytest.mark.parametrize("save,load", [(32, 32), (8, 8), (32, 8), (8, 32)])
def test_state_dict_round_trip(mm, save, load):
    shapes = [(300,), (20, 30)]
    host, params = params_of(mm, shapes)
    opt = mm.optim.AdamW(params, lr=1e-2, state_bits=save)
    for t in (1, 2):
        for p, g in zip(params, grads_of(shapes, t)):
            p.grad = mm.to_device(g)
        opt.step()
    saved = opt.state_dict()
    other = [torch.nn.Parameter(mm.to_device(p.detach().cpu())) for p in params]
    new = mm.optim.AdamW(other, lr=1.0, state_bits=load)
    new.load_state_dict(saved)
    assert new.param_groups[0]["lr"] == 1e-2
    for p, q in zip(params, other):
        assert float(new.state[q]["step"].cpu()) == 2.0
        for a, b in zip(opt.state_values(p), new.state_values(q)):
            a, b = a.cpu(), b.cpu()
            if load == 32 or save == 8:
                assert torch.equal(a, b)
            else:
                assert ((a - b).norm() / a.norm()) < 0.0625 * 2  # v's step is twice its root's


def test_torch_fused_optimisers(mm):
    """torch.optim.AdamW / Adam with fused=True run on the same kernel."""
    shapes = [(130,), (17, 40)]
    for cls, wd in ((torch.optim.AdamW, 0.1), (torch.optim.Adam, 0.1), (torch.optim.Adam, 0.0)):
        host, params = params_of(mm, shapes)
        cpu = [torch.nn.Parameter(h.double()) for h in host]
        kw = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=wd)
        dev, ref = cls(params, fused=True, **kw), cls(cpu, foreach=False, **kw)
        for t in (1, 2, 3):
            for p, q, g in zip(params, cpu, grads_of(shapes, t)):
                p.grad, q.grad = mm.to_device(g), g.double()
            dev.step()
            ref.step()
        for p, q in zip(params, cpu):
            # three steps of lr each, 40 roundings of the step's and 9 of the parameter's magnitude
            assert ((p.detach().cpu().double() - q.detach()).abs() <= U * (3 * 40 * 1e-2 * 3 + 9 * q.detach().abs())).all()


def test_refusals(mm):
    p = torch.nn.Parameter(mm.to_device(torch.zeros(8)))
    for kw in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(0.9, 1.0)), dict(weight_decay=-1.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            mm.optim.AdamW([p], **kw)
    with pytest.raises(NotImplementedError):
        mm.optim.AdamW([p], lr=torch.tensor(1e-3))
    with pytest.raises(RuntimeError, match="MatrixMan"):
        mm.optim.AdamW([torch.nn.Parameter(torch.zeros(3))])
    buf = mm.to_device(torch.zeros(64))
    with pytest.raises(ValueError, match="share"):
        mm.optim.AdamW([torch.nn.Parameter(buf[:40].detach()), torch.nn.Parameter(buf[32:].detach())])
    with pytest.raises(NotImplementedError, match="span"):
        mm.optim.AdamW([torch.nn.Parameter(buf[::2].detach())])
    opt = mm.optim.AdamW([p])
    q = torch.nn.Parameter(buf.detach())
    with pytest.raises(ValueError, match="share|twice|more than one"):
        opt.add_param_group({"params": [torch.nn.Parameter(p.detach())]})
    opt.add_param_group({"params": [q]})
    assert len(opt.param_groups) == 2
    with pytest.raises(ValueError, match="shape"):
        opt.set_state_values(p, torch.zeros(7), torch.zeros(7))
    with pytest.raises(NotImplementedError):
        o = torch.optim.AdamW([p], fused=True, amsgrad=True)
        p.grad = mm.to_device(torch.zeros(8))
        o.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_states_that_do_not_fit_their_parameter(mm, bits):
    """The C++ calls leave them to the Python code, which refuses them; nothing is launched and nothing moves."""
    from matrixman_b200 import telemetry
    from matrixman_b200.privateuse import native_calls
    names = ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg_code", "exp_avg_scale", "exp_avg_sq_code",
                                                          "exp_avg_sq_scale")
    for name in (*names, "step"):
        p = torch.nn.Parameter(mm.to_device(torch.ones(1000)))
        p.grad = mm.to_device(torch.ones(1000))
        opt = mm.optim.AdamW([p], state_bits=bits)
        opt.step()
        want = p.detach().cpu()
        right = opt.state[p][name]
        for wrong in (mm.to_device(torch.zeros(max(right.numel() - 1, 0))), mm.to_device(torch.zeros(2000))[::2]):
            if name in ("exp_avg", "exp_avg_sq") or wrong.numel() != right.numel():
                opt.state[p][name] = wrong
                assert native_calls().adamw_step([p], [opt.state[p]], bits, 1e-3, 0.9, 0.999, 1e-8, 0.0, False) is None
                before = dict(telemetry.launches)
                for call in (opt.step, lambda: opt.state_values(p)):
                    with pytest.raises(RuntimeError, match="AdamW state"):
                        call()
                assert dict(telemetry.launches) == before
        opt.state[p][name] = right
        assert torch.equal(p.detach().cpu(), want)
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_may_not_be_the_captured_one(mm, bits):
    host, params = params_of(mm, [(700,), (33, 9)])
    opt = mm.optim.AdamW(params, lr=1e-2, state_bits=bits)
    for p, g in zip(params, grads_of([(700,), (33, 9)], 1)):
        p.grad = mm.to_device(g)
    rt = params[0].runtime
    rt.synchronize()
    rt.capture_begin()
    try:
        with pytest.raises(RuntimeError, match="capture"):
            opt.step()
    finally:
        rt.capture_end().destroy()
    assert all(torch.equal(p.detach().cpu(), h) for p, h in zip(params, host))
    # states that were set take the place of a step
    for p in params:
        opt.set_state_values(p, torch.zeros(p.shape), torch.zeros(p.shape), step=0)
    rt.synchronize()
    rt.capture_begin()
    opt.step()
    graph = rt.capture_end()
    graph.replay()
    graph.replay()
    assert [float(opt.state[p]["step"].cpu()) for p in params] == [2.0, 2.0]
