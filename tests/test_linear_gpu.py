"""matrixman.linear against its formulas in float64.

Tolerances: u = 2^-24.  A sum of k products, each product and addition rounded
(or truncated by the tensor core: 2 u), is off by at most 2 (k + 8) u times the
sum of the products' magnitudes, whatever the order; splitting an operand into
three bf16 pieces loses nothing of it and leaves out products below 2^-24 of
theirs (3 u more).  Bias and residual add 2 u of the result's terms.  The
activation passes the error on with its slope (at most 1.13 for all of them,
0.25 for the sigmoid) and adds 16 u of its own argument's and value's
magnitude (exp, erfc, division: a few units in the last place each, times the
argument's rounding).  That worst case grows with k; the norm of the whole
error grows with sqrt(k), as k roundings of either sign add up, and is held to
(sqrt(k) + 32) u of the norm of the products' magnitudes."""

import ctypes
import math

import pytest
import torch

from matrixman_b200 import _lib, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh"]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed))


def act64(z, act):
    return {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v / (1 + torch.exp(-v)),
            "sigmoid": torch.sigmoid, "gelu": lambda v: 0.5 * v * torch.special.erfc(-v / math.sqrt(2)),
            # (1 + tanh a) / 2 = sigmoid(2 a), without the sum that cancels for large negative a
            "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)),
            }[act](z)


def products(a, b):
    """a [m, k] b [n, k]^T in float64, and the error bound of its float32 sum."""
    a, b = a.double(), b.double()
    size = a.abs() @ b.abs().t()
    return a @ b.t(), (2 * (a.shape[1] + 8) + 3) * U * size, size


def close(name, got, want, bound, size=None, k=None):
    got = got.double()
    assert got.shape == want.shape, name
    err = (got - want).abs()
    if err.numel():
        over = (err - bound).max().item()
        assert over <= 0, f"{name}: {err.max().item():.3g} off, {over:.3g} over its bound"
    if size is not None and k:
        assert err.norm().item() <= (math.sqrt(k) + 32) * U * size.norm().item(), name


def check(mm, x, w, b, r, act, first=False, grad=True):
    """Forward, and all gradients with a random output gradient, of 2-D x."""
    m, k = x.shape
    n = w.shape[0]
    z, ez, size = products(x, w)
    if b is not None:
        z = z + b.double()
    if r is not None and first:
        z = z + r.double()
    ez = ez + 4 * U * (z.abs() + (b.double().abs() if b is not None else 0) + (r.double().abs() if r is not None else 0))
    a = act64(z, act)
    y = a + r.double() if r is not None and not first else a
    slope = 0.25 if act == "sigmoid" else 1.13
    ey = slope * ez + (16 * U * (z.abs() * (act != "sigmoid") + a.abs()) if act not in ("none", "relu") else 0) + 2 * U * y.abs()

    leaves = {"x": mm.to_device(x), "w": mm.to_device(w)}
    if b is not None:
        leaves["b"] = mm.to_device(b)
    if r is not None:
        leaves["r"] = mm.to_device(r)
    with torch.no_grad():
        plain = mm.linear(leaves["x"], leaves["w"], leaves.get("b"), activation=act, residual=leaves.get("r"),
                          residual_before_act=first).cpu()
    close("y", plain, y, ey, size if act in ("none", "relu") and b is None and r is None else None, k)
    if not grad:
        return
    for t in leaves.values():
        t.requires_grad_(True)
    out = mm.linear(leaves["x"], leaves["w"], leaves.get("b"), activation=act, residual=leaves.get("r"),
                    residual_before_act=first)
    assert torch.equal(out.detach().cpu(), plain)
    dy = randn(m, n, seed=99)
    grads = dict(zip(leaves, [g.cpu() for g in torch.autograd.grad(out, list(leaves.values()), mm.to_device(dy))]))
    z64 = z.clone().requires_grad_(True)
    s = torch.autograd.grad(act64(z64, act), z64, torch.ones_like(z))[0]
    # The slope is read at the computed z.  Its own slope is at most 1.13 (GELU), so it is off by 1.13 ez + 24 u;
    # where ReLU's z is within its error of 0 either slope is right: leave those out of the comparison.
    border = (z.abs() <= ez) if act == "relu" else torch.zeros_like(z, dtype=torch.bool)
    es = torch.where(border, torch.ones_like(z), torch.zeros_like(z)) if act == "relu" else \
        (1.13 * ez + 24 * U * (1 + z.abs()) if act != "none" else torch.zeros_like(z))
    dz = dy.double() * s
    edz = dy.double().abs() * es + U * dz.abs()
    dx, edx, _ = products(dz, w.t())
    close("dx", grads["x"], dx, edx + edz @ w.double().abs())
    dw, edw, _ = products(dz.t(), x.t())
    close("dw", grads["w"], dw, edw + edz.t() @ x.double().abs())
    if b is not None:
        close("db", grads["b"], dz.sum(0), (m + 8) * U * dz.abs().sum(0) + edz.sum(0))
    if r is not None:
        close("dr", grads["r"], dz if first else dy.double(), edz if first else torch.zeros_like(dz))


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 5, 3), (1, 512, 784), (1, 257, 1030), (2, 64, 64), (3, 10, 256), (7, 100, 33), (16, 130, 129),
    (17, 33, 700), (31, 65, 4096), (33, 127, 128), (64, 64, 65), (100, 300, 200), (128, 256, 512), (129, 257, 31),
    (256, 512, 784), (255, 1000, 1281), (700, 129, 40), (513, 384, 96), (2000, 40, 8),
    (5000, 7, 300), (4000, 300, 7), (9001, 10, 16), (300, 1, 600), (600, 300, 1),
    (1, 4097, 1030), (1, 40001, 64), (2, 3001, 400), (3, 2501, 260), (4, 9000, 132), (12, 1301, 700), (16, 4099, 36)])
def test_sizes(mm, m, n, k):
    check(mm, randn(m, k, seed=1), randn(n, k, seed=2), randn(n, seed=3), None, "none")


# Tiles shared by two CTAs: in whole rounds with a rest, with divided reductions,
# with operands along and across the reduction, rows that end in either half.
@pytest.mark.parametrize("m,n,k", [(511, 1300, 2049), (2570, 1001, 33), (2500, 1100, 70), (500, 380, 6000)])
def test_tiles_of_cta_pairs(mm, m, n, k):
    check(mm, randn(m, k, seed=1), randn(n, k, seed=2), randn(n, seed=3), None, "none")
    check(mm, randn(m, k, seed=4), randn(n, k, seed=5) / math.sqrt(k), randn(n, seed=6), randn(m, n, seed=7), "gelu")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("mode", ["plain", "bias", "residual", "residual first", "both"])
def test_epilogues(mm, act, mode):
    for m, n, k in ((5, 96, 50), (150, 200, 72), (300, 260, 128)):
        x, w = randn(m, k, seed=1), randn(n, k, seed=2) / math.sqrt(k)
        b = randn(n, seed=3) if mode in ("bias", "both") else None
        r = randn(m, n, seed=4) if mode not in ("plain", "bias") else None
        check(mm, x, w, b, r, act, first=mode == "residual first")


@pytest.mark.parametrize("act", ACTS)
def test_activation_over_its_range(mm, act):
    """x = 1, so z is the weight: from far below to far above, and the ends."""
    z = torch.cat([torch.linspace(-30, 30, 4001), torch.tensor([0.0, -0.0, 88.0, -88.0, -104.0, 1e30, -1e30, 1e-30])])
    got = mm.linear(mm.to_device(torch.ones(1, 1)), mm.to_device(z[:, None]), activation=act).cpu()[0].double()
    want = act64(z.double(), act)
    # Beyond 1e3 every tail is below exp(-1000), i.e. 0 even in float64 (where z^3 or z * 0 may overflow).
    far = {"none": z.double(), "sigmoid": (z > 0).double()}.get(act, z.double().clamp(min=0))
    want = torch.where(z.abs() > 1e3, far, want)
    # the argument's rounding: |z| times the relative change of the value, at most z^2 u of it for the GELUs' tails
    bound = 16 * U * (want.abs() * (1 + z.double().abs().clamp(max=40) ** 2)) + 1e-37
    assert ((got - want).abs() <= bound).all(), (got - want).abs().sub(bound).argmax()


def test_wide_range_of_magnitudes(mm):
    """Features of very different units, scaled back by their weights: float32's
    exponents are kept, so every term counts with its own precision."""
    k = 320
    scale = torch.logspace(-12, 12, k)
    for m in (4, 200):
        x, w = randn(m, k, seed=1) * scale, randn(150, k, seed=2) / scale
        z, ez, size = products(x, w)
        got = mm.linear(mm.to_device(x), mm.to_device(w)).cpu()
        close("y", got, z, ez, size, k)


def test_non_finite_inputs_reach_their_rows_only(mm):
    for m in (6, 200):
        x, w = randn(m, 96, seed=1), randn(140, 96, seed=2)
        x[1, 5] = float("nan")
        x[3, 7] = float("inf")
        got = mm.linear(mm.to_device(x), mm.to_device(w)).cpu()
        want = x @ w.t()
        assert torch.isnan(got[1]).all()
        assert torch.equal(got[3], want[3])  # infinities of the weights' signs
        rest = [i for i in range(m) if i not in (1, 3)]
        assert torch.isfinite(got[rest]).all()


@pytest.mark.parametrize("m,n,k", [(1500, 1500, 100), (511, 1300, 2049)])
def test_infinities_in_both_halves_of_a_pairs_tile(mm, m, n, k):
    x, w = randn(m, k, seed=1), randn(n, k, seed=2)
    rows, cols = (5, 200, 300, m - 1), (3, 70, 127, n - 1)
    for i, r in enumerate(rows):
        x[r, 7 * i + 3] = float("-inf") if i % 2 else float("inf")
    for i, c in enumerate(cols):
        w[c, 5 * i + 40] = float("inf")
    got, want = mm.linear(mm.to_device(x), mm.to_device(w)).cpu(), x @ w.t()
    hit = torch.zeros(m, n, dtype=torch.bool)
    hit[list(rows)] = True
    hit[:, list(cols)] = True
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and not torch.isfinite(got[hit]).any()
    same = hit & ~torch.isnan(want)
    assert torch.equal(got[same], want[same])
    assert torch.isfinite(got[~hit]).all()


def test_strides_and_leading_dimensions(mm):
    base, w, r = randn(6, 50, 90, seed=1), randn(70, 90, seed=2), randn(6, 50, 70, seed=3)
    dev, dw = mm.to_device(base), mm.to_device(w)
    want = (base.double() @ w.double().t())
    bound = 2 * 101 * U * (base.double().abs() @ w.double().abs().t())
    close("3-D", mm.linear(dev, dw).cpu(), want, bound)
    close("rows at a stride", mm.linear(dev[:, ::2], dw).cpu(), want[:, ::2], bound[:, ::2])
    close("transposed lead", mm.linear(dev.transpose(0, 1), dw).cpu(), want.transpose(0, 1), bound.transpose(0, 1))
    close("1-D", mm.linear(dev[2, 3], dw).cpu(), want[2, 3], bound[2, 3])
    xt, wt = mm.to_device(base[0].t().contiguous()).t(), mm.to_device(w.t().contiguous()).t()
    close("transposed operands", mm.linear(xt, wt).cpu(), want[0], bound[0])
    odd = mm.to_device(randn(301 * 91 + 1, seed=5))
    flat = odd.cpu()
    x1 = odd[1:].view(301, 91)[:, :90]
    x1c = flat[1:].view(301, 91)[:, :90]
    res = mm.to_device(randn(301, 80, seed=6))
    got = mm.linear(x1, dw, residual=res[:, 5:75]).cpu()
    ref = x1c.double() @ w.double().t() + res.cpu()[:, 5:75].double()
    close("unaligned rows", got, ref, 2 * 103 * U * (x1c.double().abs() @ w.double().abs().t()) + 2 * U * ref.abs())
    close("lead and residual", mm.linear(dev, dw, residual=mm.to_device(r)).cpu(), want + r.double(), bound + 4 * U * (want + r.double()).abs())


def test_gradients_of_views_and_expanded_gradients(mm):
    x, w = randn(40, 3, 60, seed=1), randn(24, 60, seed=2)
    dx, dw = mm.to_device(x).requires_grad_(True), mm.to_device(w).requires_grad_(True)
    out = mm.linear(dx.transpose(0, 1), dw, activation="none")
    out.sum(dim=2).sum(dim=1).sum(dim=0).backward()
    want = w.double().sum(0).expand(40, 3, 60)
    close("dx", dx.grad.cpu(), want, 2 * 40 * U * w.double().abs().sum(0).expand(40, 3, 60))
    close("dw", dw.grad.cpu(), x.double().sum((0, 1)).expand(24, 60), 2 * 140 * U * x.double().abs().sum((0, 1)).expand(24, 60))


def test_shared_weight_adds_its_gradients(mm):
    x, w = randn(9, 30, seed=1), randn(30, 30, seed=2) / 5
    dw = mm.to_device(w).requires_grad_(True)
    y = mm.linear(mm.linear(mm.to_device(x), dw, activation="relu"), dw)
    got = torch.autograd.grad(y, dw, mm.to_device(torch.ones(9, 30)))[0].cpu()
    w64 = w.double().requires_grad_(True)
    want = torch.autograd.grad((torch.relu(x.double() @ w64.t()) @ w64.t()).sum(), w64)[0]
    # two products of 30 terms and their sum, every term below the product of the magnitudes' sums
    bound = 200 * U * ((x.double().abs() @ w.double().abs().t()).sum() * w.double().abs().max() + x.double().abs().sum() * w.double().abs().sum(0).max())
    close("dw", got, want, bound.expand(30, 30))


def test_gradient_against_differences(mm):
    x, w, b, r, dy = randn(5, 12, seed=1), randn(7, 12, seed=2), randn(7, seed=3), randn(5, 7, seed=4), randn(5, 7, seed=5)
    for act in ACTS[2:]:
        leaves = [mm.to_device(t).requires_grad_(True) for t in (x, w, b, r)]
        y = mm.linear(*leaves[:3], activation=act, residual=leaves[3], residual_before_act=True)
        grads = [g.cpu().double() for g in torch.autograd.grad(y, leaves, mm.to_device(dy))]
        h = 1e-5
        for i, t in enumerate((x, w, b, r)):
            v = randn(*t.shape, seed=10 + i).double()

            def f(s):
                a = [q.double() + (s * v if j == i else 0) for j, q in enumerate((x, w, b, r))]
                return (act64(a[0] @ a[1].t() + a[2] + a[3], act) * dy.double()).sum()

            slope = ((f(h) - f(-h)) / (2 * h)).item()
            assert abs((grads[i] * v).sum().item() - slope) <= 1e-4 * ((grads[i] * v).abs().sum().item() + 1)


def test_empty_sizes(mm):
    for m, n, k in ((0, 4, 5), (4, 0, 5), (4, 5, 0), (0, 0, 0)):
        x, w, b = torch.zeros(m, k), torch.zeros(n, k), torch.arange(float(n))
        leaves = [mm.to_device(t).requires_grad_(True) for t in (x, w, b)]
        y = mm.linear(*leaves)
        assert torch.equal(y.detach().cpu(), b.expand(m, n))
        grads = torch.autograd.grad(y, leaves, mm.to_device(torch.ones(m, n)))
        assert [tuple(g.shape) for g in grads] == [(m, k), (n, k), (n,)]
        assert torch.equal(grads[1].cpu(), torch.zeros(n, k))
        assert torch.equal(grads[2].cpu(), torch.full((n,), float(m)))


@pytest.mark.parametrize("m,n,k", [(3, 200, 300), (300, 500, 260), (511, 1300, 2049)])
def test_same_bits_twice_and_in_replayed_graphs(mm, m, n, k):
    x, w, b, dy = randn(m, k, seed=1), randn(n, k, seed=2), randn(n, seed=3), randn(m, n, seed=4)
    args = [mm.to_device(t) for t in (x, w, b)]
    rt = args[0].runtime

    def call(first):
        leaves = [t.detach().requires_grad_(True) for t in (first, *args[1:])]
        y = mm.linear(*leaves, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, mm.to_device(dy)))

    one = [t.cpu() for t in call(args[0])]
    assert all(torch.equal(p, q.cpu()) for p, q in zip(one, call(args[0])))
    other = mm.to_device(2 * x)
    two = [t.cpu() for t in call(other)]
    grad = mm.to_device(dy)

    def captured(first):
        leaves = [t.detach().requires_grad_(True) for t in (first, *args[1:])]
        rt.synchronize()
        rt.capture_begin()
        y = mm.linear(*leaves, activation="gelu")
        out = (y.detach(), *torch.autograd.grad(y, leaves, grad))
        return rt.capture_end(), out

    ga, outa = captured(args[0])
    gb, outb = captured(other)
    ga.replay()
    gb.replay()
    ga.replay()  # the two graphs' workspaces are their own
    assert all(torch.equal(p.cpu(), q) for p, q in zip(outa, one))
    assert all(torch.equal(p.cpu(), q) for p, q in zip(outb, two))


def test_two_streams_at_once(mm):
    """Calls on two streams, each of several kernels that overlap, give the bits of calls one at a time."""
    lib = _lib.load()
    sizes = [(511, 1300, 2049), (700, 640, 900)]
    calls = []
    for i, (m, n, k) in enumerate(sizes):
        x, w, dy = (mm.to_device(randn(*s, seed=10 * i + j)) for j, s in enumerate(((m, k), (n, k), (m, n))))
        rt = x.runtime
        calls.append(((m, n, k), x, w, dy, [ops.empty(rt, s) for s in ((m, n), (m, k), (n, k), (n,))]))

    def queue(call, stream):
        (m, n, k), x, w, dy, (y, dx, dw, db) = call
        at = [t.element_ptr for t in (x, w, dy, y, dx, dw, db)]
        assert lib.mm_linear(at[0], k, 1, at[1], k, 1, None, None, 0, m, n, k, 0, 0, at[3], None, None, 0, stream) == 0
        assert lib.mm_linear_backward(at[2], n, at[0], k, 1, at[1], k, 1, None, m, n, k, 0, at[4], at[5], at[6], None,
                                      None, 0, stream) == 0

    alone = []
    for call in calls:
        queue(call, rt.stream)
        alone.append([t.cpu() for t in call[4]])
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        _lib.check(lib.mm_stream_create(rt.index, ctypes.byref(s)), "stream")
    rt.synchronize()
    for _ in range(5):
        for call, s in zip(calls, streams):
            queue(call, s)
    for s in streams:
        _lib.check(lib.mm_stream_sync(s, 20000), "stream wait")
    for call, want in zip(calls, alone):
        assert all(torch.equal(t.cpu(), v) for t, v in zip(call[4], want))
    for s in streams:
        _lib.check(lib.mm_stream_destroy(s), "stream")


def test_refusals(mm):
    x, w, b = mm.to_device(randn(4, 8, seed=1)), mm.to_device(randn(6, 8, seed=2)), mm.to_device(randn(6, seed=3))
    with pytest.raises(ValueError, match="activation"):
        mm.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="end in"):
        mm.linear(mm.to_device(randn(4, 7, seed=1)), w)
    with pytest.raises(ValueError, match="bias"):
        mm.linear(x, w, mm.to_device(randn(5, seed=1)))
    with pytest.raises(ValueError, match="residual"):
        mm.linear(x, w, b, residual=mm.to_device(randn(6, seed=1)))
    with pytest.raises(ValueError, match=r"\[n, k\]"):
        mm.linear(x, b)
    with pytest.raises(NotImplementedError, match="float32"):
        mm.linear(mm.to_device(torch.zeros(4, 8, dtype=torch.int64)), w)
    with pytest.raises(RuntimeError, match="MatrixMan"):
        mm.linear(torch.zeros(4, 8), w)
    with pytest.raises(RuntimeError, match="gradient"):
        mm.linear(x, torch.zeros(6, 8, requires_grad=True))
    leaf = mm.to_device(randn(6, 8, seed=2)).requires_grad_(True)
    g, = torch.autograd.grad(mm.linear(x, leaf), leaf, mm.to_device(randn(4, 6, seed=5)), create_graph=True)
    assert not g.requires_grad or pytest.raises(RuntimeError, lambda: torch.autograd.grad(g, leaf, leaf.detach()))


def test_cpu_weights(mm):
    x, w, b = randn(5, 40, seed=1), randn(30, 40, seed=2), randn(30, seed=3)
    got = mm.linear(mm.to_device(x), w, b).cpu()
    assert torch.equal(got, mm.linear(mm.to_device(x), mm.to_device(w), mm.to_device(b)).cpu())


def test_short_pair_products_one_behind_the_other(mm):
    """Hundreds of short products of CTA pairs, each starting on the SMs that the one before leaves: a CTA that
    left while an arrival was on its way to it would disturb the barriers of the next one there."""
    lib = _lib.load()
    m, n, k = 2500, 1100, 70
    x, w, dy = mm.to_device(randn(m, k, seed=1)), mm.to_device(randn(n, k, seed=2)), mm.to_device(randn(m, n, seed=3))
    rt = x.runtime
    dx, dw = ops.empty(rt, (m, k)), ops.empty(rt, (n, k))
    y = ops.empty(rt, (m, n))

    def queue():
        assert lib.mm_linear(x.element_ptr, k, 1, w.element_ptr, k, 1, None, None, 0, m, n, k, 0, 0, y.element_ptr, None,
                             None, 0, rt.stream) == 0
        assert lib.mm_linear_backward(dy.element_ptr, n, x.element_ptr, k, 1, w.element_ptr, k, 1, None, m, n, k, 0,
                                      dx.element_ptr, dw.element_ptr, None, None, None, 0, rt.stream) == 0

    queue()
    want = [t.cpu() for t in (y, dx, dw)]
    for _ in range(300):
        queue()
    assert all(torch.equal(t.cpu(), v) for t, v in zip((y, dx, dw), want))
    code = ctypes.c_int(-1)
    _lib.check(lib.mm_kernel_error(rt.index, ctypes.byref(code), 0))
    assert code.value == 0


@pytest.mark.parametrize("m,n,k", [(2500, 1100, 70), (511, 1300, 2049), (128, 1000, 4096)])
def test_bounded_waits_run_out_and_recover(mm, m, n, k):
    """With the test hook CTA 0 leaves its first loads out and the limit of a wait is 1 ms, so the waits for that
    stage run out: the kernel records a code, waits for its own copies and MMAs, frees tensor memory and
    returns, and the next wait of the host raises.  Calls after that are whole, and are not hurried by a code
    that nobody has read."""
    lib = _lib.load()
    x, w, dy = mm.to_device(randn(m, k, seed=1)), mm.to_device(randn(n, k, seed=2)), mm.to_device(randn(m, n, seed=3))
    rt = x.runtime
    xg, wg = x.detach().requires_grad_(True), w.detach().requires_grad_(True)

    def forward():
        with torch.no_grad():
            return mm.linear(x, w)

    def grads():
        return torch.autograd.grad(mm.linear(xg, wg), (xg, wg), dy)

    want = [t.cpu() for t in (forward(), *grads())]
    rt.synchronize()
    code = ctypes.c_int(-1)
    for call in (forward, grads):
        _lib.check(lib.mm_debug_tc_fault(rt.index, 1_000_000, 1))
        try:
            call()
        finally:
            _lib.check(lib.mm_debug_tc_fault(rt.index, 0, 0))
        with pytest.raises(_lib.MatrixManNativeError, match=r"code 10[1-5]"):
            rt.synchronize(timeout_ms=30_000)
        _lib.check(lib.mm_kernel_error(rt.index, ctypes.byref(code), 0))
        assert code.value == 0  # reported once
        assert all(torch.equal(t.cpu(), v) for t, v in zip((forward(), *grads()), want))
    # a readback and torch's own synchronisation report it too, mm_kernel_error to C callers
    for wait in (lambda y: y.cpu(), lambda y: torch.Stream(device=y.device).synchronize()):
        _lib.check(lib.mm_debug_tc_fault(rt.index, 1_000_000, 1))
        try:
            y = forward()
        finally:
            _lib.check(lib.mm_debug_tc_fault(rt.index, 0, 0))
        with pytest.raises(RuntimeError, match=r"code 10[1-5]"):
            wait(y)
    _lib.check(lib.mm_debug_tc_fault(rt.index, 1_000_000, 1))
    try:
        forward()
    finally:
        _lib.check(lib.mm_debug_tc_fault(rt.index, 0, 0))
    y = forward()  # the code stands, this call is whole
    _lib.check(lib.mm_stream_sync(rt.stream, 30_000))
    _lib.check(lib.mm_kernel_error(rt.index, ctypes.byref(code), 1))
    assert 101 <= code.value <= 105
    assert torch.equal(y.cpu(), want[0])


@pytest.mark.parametrize("m,n,k", [(5, 40, 24), (60, 96, 50), (700, 640, 300), (2500, 1100, 70)])
@pytest.mark.parametrize("mode", ["plain", "residual", "residual first"])
def test_relu_drops_non_finite_gradients_where_it_was_off(mm, m, n, k, mode):
    """As threshold_backward: the gradient is selected, not multiplied by 0, and passes where z is NaN."""
    x, w, r, dy = randn(m, k, seed=1), randn(n, k, seed=2), randn(m, n, seed=3), randn(m, n, seed=4)
    x[1, 3] = float("nan")  # z's row 1
    first = mode == "residual first"
    res = None if mode == "plain" else mm.to_device(r).requires_grad_(True)
    lx, lw, lb = (mm.to_device(t).requires_grad_(True) for t in (x, w, torch.zeros(n)))
    y = mm.linear(lx, lw, lb, activation="relu", residual=res, residual_before_act=first)
    z, ez, _ = products(x, w)
    if first:
        z, ez = z + r.double(), ez + 4 * U * r.double().abs()
    dy[z.abs() <= ez + 4 * U * z.abs()] = 0.0  # either sign of the computed z is right there
    off = (z < -1e-3).nonzero()
    hit = off[:: max(len(off) // 50, 1)]
    for i, (a, b) in enumerate(hit.tolist()):
        dy[a, b] = (float("inf"), float("-inf"), float("nan"))[i % 3]
    leaves = (lx, lw, lb) + ((res,) if res is not None else ())
    grads = [g.cpu() for g in torch.autograd.grad(y, leaves, mm.to_device(dy))]
    # What the framework's own ReLU makes of the same z and gradient, and its sums in float64.
    zt = mm.to_device(z.float()).requires_grad_(True)
    dz = torch.autograd.grad(torch.relu(zt), zt, mm.to_device(dy))[0].cpu()
    assert torch.isfinite(dz).all() and torch.equal(dz[1], dy[1]) and (dz[hit[:, 0], hit[:, 1]] == 0).all()
    want, bound, _ = products(dz, w.t())
    close("dx", grads[0], want, bound)
    got, ok = grads[1], [c for c in range(k) if c != 3]
    want, bound, _ = products(dz.t(), x[:, ok].t().nan_to_num(0.0))
    close("dw", got[:, ok], want, bound)
    close("db", grads[2], dz.double().sum(0), (m + 8) * U * dz.double().abs().sum(0))
    if res is not None:
        expect = dz if first else dy
        assert torch.equal(grads[3].nan_to_num(7.0, 8.0, 9.0), expect.nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("m,n,k", [(10, 300, 260), (100, 64, 256), (2500, 1100, 70)])
@pytest.mark.parametrize("exponent", [-100, -109, -116, -124, -140])
def test_operands_near_the_smallest_numbers(mm, m, n, k, exponent):
    """Three bf16 pieces hold a value exactly from 2^-110 on, a smaller one to within bf16's smallest step,
    2^-133 (the last piece is cut off there)."""
    x, w = torch.ldexp(randn(m, k, seed=1), torch.tensor(exponent)), torch.ldexp(randn(n, k, seed=2), torch.tensor(60))
    z, ez, _ = products(x, w)
    bound = ez + 2.0 ** -133 * w.double().abs().sum(1)
    close("x", mm.linear(mm.to_device(x), mm.to_device(w)).cpu(), z, bound)
    close("w", mm.linear(mm.to_device(w), mm.to_device(x)).cpu(), z.t(), bound.t())


def test_fault_is_recorded_without_a_runtime():
    """A C caller with streams and workspaces of its own need not call mm_init: a wait that gives up is recorded for
    it all the same (in a process of its own, on torch's memory)."""
    import subprocess
    import sys
    from .conftest import ROOT
    code = """
import ctypes, torch
from matrixman_b200 import _lib
lib = _lib.load()
m, n, k = 2500, 1100, 70
x, w, y = (torch.ones(s, device="cuda") for s in ((m, k), (n, k), (m, n)))
size, code, word = ctypes.c_size_t(), ctypes.c_int(-1), ctypes.c_void_p()
assert lib.mm_fault_word(0, ctypes.byref(word)) == _lib.MM_ERR_STATE
assert lib.mm_linear_workspace_size(m, n, k, 0, ctypes.byref(size)) == 0
work = torch.empty(size.value, dtype=torch.uint8, device="cuda")
def call():
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert lib.mm_linear(x.data_ptr(), k, 1, w.data_ptr(), k, 1, None, None, 0, m, n, k, 0, 0, y.data_ptr(), None,
                         work.data_ptr(), size.value, s.cuda_stream) == 0, _lib.last_error()
    torch.cuda.synchronize()
    assert lib.mm_kernel_error(0, ctypes.byref(code), 1) == 0
    return code.value
assert call() == 0 and torch.equal(y, torch.full_like(y, 70.0))
assert lib.mm_debug_tc_fault(0, 1_000_000, 1) == 0
got = call()
assert lib.mm_debug_tc_fault(0, 0, 0) == 0
assert 101 <= got <= 105, got
y.zero_()
assert call() == 0 and torch.equal(y, torch.full_like(y, 70.0))
print("recorded", got)
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "recorded" in run.stdout, run.stderr[-2000:]
