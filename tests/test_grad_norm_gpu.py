"""The norm of many tensors, clipping by it, and the clipped AdamW step, against
the formulas in float64.

Tolerances, u = 2^-24: sums are held in 64 bits, where 10^7 terms are off by less
than 10^7 2^-53 < u / 50, so the norm is off by its rounding, 1.02 u.  The
coefficient takes that, the rounding of the limit, of norm + 1e-6 and of the
quotient, a clipped element one more: 5.1 u.  A result below 2^-126 is rounded to a
multiple of 2^-149, so it is off by up to 2^-150 (a clipped element twice that)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ORDERS = [1.0, 2.0, math.inf]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def tensors(sizes, seed=0):
    g = gen(seed)
    return [torch.randn(s, generator=g) * 10 ** torch.randn((), generator=g) for s in sizes]


def norm_of(grads, order):
    flat = torch.cat([g.double().reshape(-1) for g in grads] + [torch.zeros(1, dtype=torch.float64)])
    return torch.linalg.vector_norm(flat, order)


def params_of(mm, grads):
    got = []
    for g in grads:
        d = g if isinstance(g, mm.MatrixManTensor) else mm.to_device(g)
        got.append(torch.nn.Parameter(mm.to_device(torch.zeros(tuple(d.shape)))))
        got[-1].grad = d
    return got


def check_clip(mm, grads, limit, order, params=None):
    """Clips copies of the gradients and compares norm and values."""
    params = params_of(mm, grads) if params is None else params
    want = norm_of(grads, order)
    total = mm.optim.grad_norm(params, order)
    assert total.shape == () and abs(total.cpu().double() - want) <= 1.02 * U * want + 2.0 ** -150
    clipped = mm.optim.clip_grad_norm_(params, limit, order)
    assert torch.equal(clipped.cpu(), total.cpu())
    coef = min(1.0, limit / (want.item() + 1e-6))
    for p, g in zip(params, grads):
        got = p.grad.cpu().double()
        if coef == 1.0 and limit / (want.item() + 1e-6) > 1 + 4 * U:
            assert torch.equal(got, g.double())
        else:
            assert ((got - coef * g.double()).abs() <= 5.1 * U * coef * g.double().abs() + 2.0 ** -149).all()


# Sizes on both sides of a chunk, of the vectors a block takes at a time, of a table and of a launch.
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("sizes", [
    [(1,)], [(3,), (0,), (5, 7), ()], [(4095,), (4096,), (4097,)], [(8192 * 37 + 1,)],
    [(784, 512), (512,), (512, 256), (256,), (256, 10), (10,)], [(33,)] * 16, [(33,)] * 17, [(100, 1 + i % 90) for i in range(300)],
    [(1 + i % 7,) for i in range(1000)], [(1 + i % 5,) for i in range(2501)], [(3000001,), (2,), (2999999,)]],
    ids=lambda s: f"{len(s)}x{s[0]}")
def test_norm_and_clipping(mm, sizes, order):
    grads = tensors(sizes, seed=len(sizes))
    norm = norm_of(grads, order).item()
    check_clip(mm, grads, 0.37 * norm, order)
    check_clip(mm, grads, 1.5 * norm, order)


@pytest.mark.parametrize("order", ORDERS)
def test_packed_gradients_at_any_offset(mm, order):
    """Views one after the other into one buffer: no alignment beyond a value's."""
    sizes = [5, 4097, 1, 20000, 3, 1023, 50001]
    flat = torch.randn(sum(sizes) + 1, generator=gen(1))
    dev = mm.to_device(flat)
    cuts = [1 + sum(sizes[:i]) for i in range(len(sizes))]
    params = params_of(mm, [dev[a:a + n] for a, n in zip(cuts, sizes)])
    grads = [flat[a:a + n] for a, n in zip(cuts, sizes)]
    check_clip(mm, grads, 0.1, order, params)
    assert torch.equal(dev[:1].cpu(), flat[:1])  # what lies in front is untouched


def test_strided_gradients(mm):
    base = torch.randn(40, 30, generator=gen(1))
    dev = mm.to_device(base)
    maps = torch.randn(2, 5, 6, 7, generator=gen(2))
    dmaps = mm.to_device(maps)
    views = lambda b, m: [b[3:20, 4:17], b[20:40:2, 1:30:3].t(), m.permute(0, 3, 1, 2), b[0], b[2, 5:6].expand(1)]
    params = params_of(mm, views(dev, dmaps))
    grads = [g.clone() for g in views(base, maps)]
    check_clip(mm, grads, 0.2 * norm_of(grads, 2.0).item(), 2.0, params)
    rest = dev.cpu()
    keep = torch.ones(40, 30, dtype=torch.bool)
    for v in views(keep, torch.ones(2, 5, 6, 7, dtype=torch.bool)):
        v.fill_(False)
    assert torch.equal(rest[keep], base[keep])
    wide = params_of(mm, [mm.to_device(torch.full((1,), 3.0)).expand(16)])
    assert abs(mm.optim.grad_norm(wide).cpu().item() - 12.0) <= 1.02 * U * 12
    with pytest.raises(NotImplementedError, match="share no memory"):
        mm.optim.clip_grad_norm_(wide, 1.0)


@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-42])
def test_large_and_small_values(mm, scale):
    """Squares that a float32 does not hold."""
    grads = [torch.randn(1000, generator=gen(1)) * scale, torch.randn(77, 3, generator=gen(2)) * scale]
    for order in ORDERS:
        want = norm_of(grads, order)
        got = mm.optim.grad_norm(params_of(mm, grads), order).cpu().double()
        assert abs(got - want) <= 1.02 * U * want + 2.0 ** -150
    check_clip(mm, grads, 1.0 if scale > 1 else 0.0, 2.0)


@pytest.mark.parametrize("order", ORDERS)
def test_non_finite_gradients(mm, order):
    for bad, want in ((math.nan, math.nan), (math.inf, math.inf), (-math.inf, math.inf)):
        grads = tensors([(5000,), (3, 3)], seed=3)
        grads[0][4321] = bad
        params = params_of(mm, grads)
        with pytest.raises(RuntimeError, match="error_if_nonfinite"):
            mm.optim.clip_grad_norm_(params, 1.0, order, error_if_nonfinite=True)
        assert torch.equal(params[1].grad.cpu(), grads[1])
        total = mm.optim.clip_grad_norm_(params, 1.0, order).cpu().item()
        got = [p.grad.cpu() for p in params]
        if math.isnan(want):
            assert math.isnan(total) and all(torch.isnan(g).all() for g in got)
        else:
            assert total == math.inf and torch.isnan(got[0][4321])
            assert (got[0].nan_to_num(0.0) == 0).all() and (got[1] == 0).all()
    params = params_of(mm, tensors([(8,)], seed=4))
    mm.optim.clip_grad_norm_(params, 1e-3, order, error_if_nonfinite=True)  # finite: clipped as ever


def test_no_gradients(mm):
    p = torch.nn.Parameter(mm.to_device(torch.ones(3)))
    for params in ([], [p], p):
        assert mm.optim.grad_norm(params).cpu().item() == 0.0
        assert mm.optim.clip_grad_norm_(params, 1.0).cpu().item() == 0.0
    q = torch.nn.Parameter(mm.to_device(torch.ones(0)))
    q.grad = mm.to_device(torch.zeros(0))
    assert mm.optim.clip_grad_norm_([q], 1.0).cpu().item() == 0.0


def test_one_parameter_and_a_generator(mm):
    grads = tensors([(4, 5), (6,)], seed=1)
    a, b = params_of(mm, grads)
    assert abs(mm.optim.grad_norm(a).cpu() - grads[0].norm()) <= 4 * U * grads[0].norm()
    total = mm.optim.clip_grad_norm_((p for p in (a, b)), 1e-2)
    assert abs(total.cpu().double() - norm_of(grads, 2.0)) <= 1.02 * U * norm_of(grads, 2.0)


def test_clipping_is_seen_by_autograd(mm):
    """A saved gradient that clipping changed is not used again."""
    x = mm.to_device(torch.ones(4)).requires_grad_(True)
    p = torch.nn.Parameter(mm.to_device(torch.ones(4)))
    p.grad = mm.to_device(torch.full((4,), 5.0))
    y = x * p.grad
    mm.optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum(dim=0).backward()


def test_refusals(mm):
    grads = tensors([(4, 5), (6,)], seed=1)
    params = params_of(mm, grads)
    for order in (3.0, 0.0, -math.inf, 0.5):
        with pytest.raises(NotImplementedError, match="order"):
            mm.optim.grad_norm(params, order)
        with pytest.raises(NotImplementedError, match="order"):
            mm.optim.clip_grad_norm_(params, 1.0, order)
    for limit in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            mm.optim.clip_grad_norm_(params, limit)
        with pytest.raises(ValueError, match="max_grad_norm"):
            mm.optim.AdamW(params, max_grad_norm=limit)
    with pytest.raises(ValueError, match="twice"):
        mm.optim.clip_grad_norm_([params[0], params[1], params[0]], 1.0)
    flat = mm.to_device(torch.ones(10))
    with pytest.raises(ValueError, match="shares memory"):
        mm.optim.clip_grad_norm_(params_of(mm, [flat[:6], flat[5:]]), 1.0)
    both = mm.optim.grad_norm(params_of(mm, [flat[:6], flat[5:]]))  # reading them is no matter
    assert abs(both.cpu().item() - math.sqrt(11)) <= 1.02 * U * math.sqrt(11)
    cpu = torch.nn.Parameter(torch.ones(3))
    cpu.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="MatrixManTensor"):
        mm.optim.grad_norm([cpu])
    for g, p in zip(grads, params):
        assert torch.equal(p.grad.cpu(), g)


# ---------------------------------------------------------------------------
# The clipped AdamW step
# ---------------------------------------------------------------------------

KW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [(64, 33), (33,), (5, 4, 3), (300,), (1,)]


def models(mm, seed, **kw):
    params = [torch.nn.Parameter(mm.to_device(t)) for t in tensors(SIZES, seed)]
    return params, lambda **more: mm.optim.AdamW(params, **KW, **kw, **more)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("maximize", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_step_is_clipping_and_a_step(mm, monkeypatch, bits, maximize, native):
    if not native:
        from matrixman_b200 import ops
        monkeypatch.setattr(ops, "native_call", lambda *a: None)
    a, make_a = models(mm, 1, state_bits=bits, maximize=maximize)
    b, make_b = models(mm, 1, state_bits=bits, maximize=maximize)
    one, two = make_a(max_grad_norm=0.5), make_b()
    assert one.grad_norm is None
    for step, scale in enumerate((3.0, 1e-4, 1.0)):  # clipped, not clipped, clipped
        grads = [scale * g for g in tensors(SIZES, 10 + step)]
        for p, q, g in zip(a, b, grads):
            p.grad, q.grad = mm.to_device(g), mm.to_device(g)
        one.step()
        norm = mm.optim.clip_grad_norm_(b, 0.5)
        two.step()
        assert torch.equal(one.grad_norm.cpu(), norm.cpu())
        for p, q, g in zip(a, b, grads):
            assert torch.equal(p.grad.cpu(), g)
            assert torch.equal(p.detach().cpu(), q.detach().cpu())
            for s, t in zip(one.state_values(p), two.state_values(q)):
                assert torch.equal(s.cpu(), t.cpu())


def test_groups_are_clipped_together(mm):
    params = [torch.nn.Parameter(mm.to_device(t)) for t in tensors(SIZES, 1)]
    split = [torch.nn.Parameter(mm.to_device(t)) for t in tensors(SIZES, 1)]
    one = mm.optim.AdamW(params, **KW, max_grad_norm=0.1)
    two = mm.optim.AdamW([{"params": split[:2]}, {"params": split[2:], "lr": KW["lr"]}], **KW, max_grad_norm=0.1)
    for p, q, g in zip(params, split, tensors(SIZES, 2)):
        p.grad, q.grad = mm.to_device(g), mm.to_device(g)
    params[1].grad = split[1].grad = None
    one.step()
    two.step()
    assert torch.equal(one.grad_norm.cpu(), two.grad_norm.cpu())
    assert all(torch.equal(p.detach().cpu(), q.detach().cpu()) for p, q in zip(params, split))
    two.max_grad_norm = None  # from here on unclipped
    two.step()


def test_gradients_of_another_order(mm):
    """Gradients whose strides are not their parameter's, and strided ones."""
    host = torch.randn(8, 6, generator=gen(1))
    grads = [torch.randn(8, 6, generator=gen(2)), torch.randn(8, 12, generator=gen(3))]
    p = [torch.nn.Parameter(mm.to_device(host)) for _ in range(4)]
    p[0].grad, p[1].grad = mm.to_device(grads[0].t().contiguous()).t(), mm.to_device(grads[1])[:, ::2]
    p[2].grad, p[3].grad = mm.to_device(grads[0]), mm.to_device(grads[1][:, ::2].contiguous())
    one, two = (mm.optim.AdamW(q, **KW, max_grad_norm=0.3) for q in (p[:2], p[2:]))
    one.step()
    two.step()
    # (the same values in another order: sums in 64 bits round to the same float32)
    for a, b in ((p[0], p[2]), (p[1], p[3])):
        assert torch.equal(a.detach().cpu(), b.detach().cpu())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(mm, bits):
    """A clipping call and a clipped step in one graph, with new gradients before each replay."""
    a, make_a = models(mm, 1, state_bits=bits)
    b, make_b = models(mm, 1, state_bits=bits)
    one, two = make_a(max_grad_norm=0.5), make_b(max_grad_norm=0.5)
    rt = a[0].runtime

    def set_grads(params, seed, scale):
        for p, g in zip(params, tensors(SIZES, seed)):
            if p.grad is None:
                p.grad = mm.to_device(scale * g)
            else:
                p.grad.copy_(mm.to_device(scale * g))

    def call(params, opt):
        total = mm.optim.clip_grad_norm_(params, 2.0)
        opt.step()
        return total

    for params, opt in ((a, one), (b, two)):
        set_grads(params, 3, 1.0)
        call(params, opt)
    rt.synchronize()
    rt.capture_begin()
    total = call(a, one)
    graph = rt.capture_end()
    with pytest.raises(RuntimeError, match="capture"):
        rt.capture_begin()
        try:
            mm.optim.clip_grad_norm_(a, 2.0, error_if_nonfinite=True)
        finally:
            rt.capture_end()
    for seed, scale in ((4, 1.0), (5, 1e-3), (6, 30.0)):
        set_grads(a, seed, scale)
        graph.replay()
        set_grads(b, seed, scale)
        want = call(b, two)
        assert torch.equal(total.cpu(), want.cpu()) and torch.equal(one.grad_norm.cpu(), two.grad_norm.cpu())
        for p, q in zip(a, b):
            assert torch.equal(p.grad.cpu(), q.grad.cpu()) and torch.equal(p.detach().cpu(), q.detach().cpu())


def test_non_finite_norms_reach_the_parameters(mm):
    for bad in (math.nan, math.inf):
        p = torch.nn.Parameter(mm.to_device(torch.ones(10)))
        q = torch.nn.Parameter(mm.to_device(torch.ones(10)))
        g = torch.ones(10)
        g[3] = bad
        p.grad, q.grad = mm.to_device(g), mm.to_device(torch.ones(10))
        opt = mm.optim.AdamW([p, q], **KW, max_grad_norm=1.0)
        opt.step()
        assert not math.isfinite(opt.grad_norm.cpu().item())
        if math.isnan(bad):
            assert torch.isnan(p.detach().cpu()).all() and torch.isnan(q.detach().cpu()).all()
        else:  # the coefficient is 0: an infinite gradient times 0 is NaN, the others are 0
            assert torch.isnan(p.detach().cpu()[3]) and not torch.isnan(q.detach().cpu()).any()


def test_a_refused_limit_and_checkpoints(mm):
    params, make = models(mm, 1)
    opt = make(max_grad_norm=0.5)
    for p, g in zip(params, tensors(SIZES, 2)):
        p.grad = mm.to_device(g)
    opt.step()
    other, make_other = models(mm, 1)
    for p, q in zip(params, other):
        q.data.copy_(p.detach())
    loaded = make_other(max_grad_norm=0.5)
    loaded.load_state_dict(opt.state_dict())
    for p, q, g in zip(params, other, tensors(SIZES, 3)):
        p.grad, q.grad = mm.to_device(g), mm.to_device(g)
    opt.step()
    loaded.step()
    assert all(torch.equal(p.detach().cpu(), q.detach().cpu()) for p, q in zip(params, other))


@pytest.mark.parametrize("order", ORDERS)
def test_one_step_calls_and_the_python_code_agree(mm, monkeypatch, order):
    from matrixman_b200 import ops
    grads = tensors([(784, 51), (51,), (), (0, 3), (7, 3, 5)], seed=2)

    def both(params):
        first = mm.optim.grad_norm(params, order)
        return first, mm.optim.clip_grad_norm_(iter(params), 0.5, order), *(p.grad for p in params[1:])

    def fresh():  # one without a gradient in front, one whose gradient is transposed
        got = params_of(mm, grads[:1] + grads)
        got[0].grad = None
        got[1].grad = mm.to_device(grads[0].t().contiguous()).t()
        return got

    native = both(fresh())
    monkeypatch.setattr(ops, "native_call", lambda *a: None)
    assert all(torch.equal(a.cpu(), b.cpu()) and a.shape == b.shape for a, b in zip(native, both(fresh())))
