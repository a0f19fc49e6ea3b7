"""The C++ extension's operator calls against the Python code that they stand in
for: the same bits, the same shapes and strides, the same errors; and what is
not the ordinary case is left to the Python code."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed))


@pytest.fixture
def both(mm, monkeypatch):
    """both(f): f's results by the extension and by the Python code; says how
    many calls the extension answered."""
    from matrixman_b200 import ops
    native = ops.native_call

    def run(f):
        answered = []

        def counted(*args):
            r = native(*args)
            answered.append(r is not None)
            return r

        monkeypatch.setattr(ops, "native_call", counted)
        one = f()
        monkeypatch.setattr(ops, "native_call", lambda *a: None)
        two = f()
        assert len(one) == len(two)
        for a, b in zip(one, two):
            assert (a is None) == (b is None)
            if a is not None:
                assert a.shape == b.shape and a.stride() == b.stride() and a._logical_strides == b._logical_strides
                assert torch.equal(a.detach().cpu(), b.detach().cpu())
        return answered

    return run


@pytest.mark.parametrize("shape", [(5, 64), (2, 3, 40), (1, 1), (0, 8), (3, 4, 0, 8)])
def test_layer_norm(mm, both, shape):
    x, g = mm.to_device(randn(*shape, seed=1)).requires_grad_(True), mm.to_device(randn(*shape, seed=2))
    w = mm.to_device(randn(shape[-1], seed=3)).requires_grad_(True)
    b = mm.to_device(randn(shape[-1], seed=4)).requires_grad_(True)

    def step():
        y = F.layer_norm(x, shape[-1:], w, b)
        return (y, *torch.autograd.grad(y, (x, w, b), g))

    assert both(step) == [True, True]

    def without():
        y = F.layer_norm(x, shape[-1:])
        return (y, *torch.autograd.grad(y, (x,), g))

    assert both(without) == [True, True]


@pytest.mark.parametrize("lead", [(7,), (3, 5), (0,), (2, 0, 3)])
@pytest.mark.parametrize("first", [False, True])
def test_linear(mm, both, lead, first):
    x = mm.to_device(randn(*lead, 24, seed=1)).requires_grad_(True)
    w = mm.to_device(randn(10, 24, seed=2)).requires_grad_(True)
    b = mm.to_device(randn(10, seed=3)).requires_grad_(True)
    r = mm.to_device(randn(*lead, 10, seed=4)).requires_grad_(True)
    g = mm.to_device(randn(*lead, 10, seed=5))
    for act in ("none", "relu", "gelu"):
        for leaves in ((x, w), (x, w, b), (x, w, b, r), (w,), (x,), (r,)):
            bias = b if any(t is b for t in leaves) else None
            res = r if any(t is r for t in leaves) else None

            def step():
                y = mm.linear(x, w, bias, activation=act, residual=res, residual_before_act=first)
                return (y, *torch.autograd.grad(y, leaves, g))

            assert both(step) == [True, True]


def test_left_to_python(mm, both):
    x = mm.to_device(randn(6, 5, 16, seed=1))
    w, wn = mm.to_device(randn(12, 16, seed=2)), mm.to_device(randn(16, seed=3))
    with torch.no_grad():
        # (asked again once the checks are done and CPU parameters uploaded)
        assert both(lambda: (mm.linear(x.transpose(0, 1), w),)) == [False, False]
        assert both(lambda: (mm.linear(x, randn(12, 16, seed=4)),)) == [False, True]
        assert both(lambda: (F.layer_norm(x.transpose(1, 2), (5,)),)) == [False]
        assert both(lambda: (F.layer_norm(x, (16,), randn(16, seed=5), None),)) == [False]
        assert both(lambda: (F.layer_norm(x, (5, 16)),)) == []
        assert both(lambda: (F.layer_norm(x[0].t(), (5,)),)) == [False]
        assert both(lambda: (F.layer_norm(x[:, 2], (16,), wn),)) == [True]


def test_errors_and_counts(mm):
    from matrixman_b200 import ops, telemetry
    x, w = mm.to_device(randn(4, 8, seed=1)), mm.to_device(randn(6, 8, seed=2))
    before = telemetry.launches["mm_linear"]
    mm.linear(x, w)
    assert telemetry.launches["mm_linear"] == before + 1
    from matrixman_b200.privateuse import native_calls
    native = native_calls()
    assert native.linear(x, w, None, None, 99, False, False) == 1  # MM_ERR_INVALID, for the caller to raise
    with pytest.raises(ValueError, match="activation"):
        ops.native_call("linear", "mm_linear", x, w, None, None, 99, False, False)
    assert native.linear(x, torch.zeros(6, 8), None, None, 0, False, False) is None
    assert native.linear(torch.zeros(4, 8), w, None, None, 0, False, False) is None
    assert native.linear(x, mm.to_device(torch.zeros(6, 9)), None, None, 0, False, False) is None
    assert native.layer_norm(mm.to_device(torch.zeros(2, 8, dtype=torch.int64)), 8, None, None, 1e-5) is None
    assert native.layer_norm(None, 8, None, None, 1e-5) is None
    assert native.layer_norm(x, 7, None, None, 1e-5) is None


def test_out_of_memory_is_an_error_of_the_call(mm):
    import ctypes
    from matrixman_b200 import _lib
    x, w = mm.to_device(randn(300, 64, seed=1)), mm.to_device(randn(1 << 20, 64, seed=2))
    rt = x.runtime
    rt.trim()
    lib = _lib.load()
    assert lib.mm_debug_fail_alloc_after(rt.index, ctypes.c_int64(0)) == 0
    try:
        with pytest.raises(MemoryError):
            mm.linear(x, w)
    finally:
        assert lib.mm_debug_fail_alloc_after(rt.index, ctypes.c_int64(-1)) == 0
    assert mm.linear(x[:1], w).shape == (1, 1 << 20)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(mm, monkeypatch, bits):
    from matrixman_b200 import ops
    native = ops.native_call
    shapes = [(300,), (17, 40), (0, 3), (1,)]
    runs = []
    for call in (native, lambda *a: None):
        answered = []

        def counted(*args, call=call, answered=answered):
            r = call(*args)
            answered.append(r is not None)
            return r

        monkeypatch.setattr(ops, "native_call", counted)
        params = [torch.nn.Parameter(mm.to_device(randn(*s, seed=i))) for i, s in enumerate(shapes)]
        opt = mm.optim.AdamW(params, lr=1e-2, state_bits=bits, maximize=True)
        for step in range(3):
            for i, p in enumerate(params):
                p.grad = mm.to_device(randn(*shapes[i], seed=10 * step + i))
            opt.step()
        out = [p.detach().cpu() for p in params] + [v.cpu() for p in params for v in opt.state_values(p)]
        runs.append((out, answered))
    assert all(torch.equal(a, b) for a, b in zip(runs[0][0], runs[1][0]))
    assert all(runs[0][1]) and not any(runs[1][1])
    # a gradient in another order, and one of another kind, go through the Python code
    monkeypatch.setattr(ops, "native_call", native)
    p = torch.nn.Parameter(mm.to_device(torch.zeros(6, 4)))
    opt = mm.optim.AdamW([p], lr=1.0, weight_decay=0.0, state_bits=bits)
    p.grad = mm.to_device(torch.ones(4, 6)).t()
    opt.step()
    assert ((p.detach().cpu() + 1).abs() <= 2.0 ** -19).all()


def test_other_threads_run_while_a_call_waits_for_the_queue(mm):
    """More launches than the queue holds: the C++ call blocks, and without the interpreter's lock. (Threads are
    not switched by time here, so another one runs only where this one lets go.)"""
    import sys
    import threading
    from matrixman_b200.privateuse import native_calls
    native = native_calls()
    p = torch.nn.Parameter(mm.to_device(torch.zeros(1 << 24)))
    p.grad = mm.to_device(torch.ones(1 << 24))
    opt = mm.optim.AdamW([p], weight_decay=0.0)
    opt.step()
    params, states = [p], [opt.state[p]]
    p.runtime.synchronize()
    ticks, stop = [0], threading.Event()

    def tick():
        while not stop.is_set():
            ticks[0] += 1
            stop.wait(1e-4)

    interval = sys.getswitchinterval()
    t = threading.Thread(target=tick)
    t.start()
    while not ticks[0]:
        stop.wait(1e-3)
    sys.setswitchinterval(60)
    try:
        before = ticks[0]
        for _ in range(1500):
            native.adamw_step(params, states, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, False)
        after = ticks[0]
    finally:
        sys.setswitchinterval(interval)
        stop.set()
        t.join()
    assert after - before >= 10
    assert float(opt.state[p]["step"].cpu()) == 1501.0


def test_two_threads_at_once(mm):
    """Calls of several overlapping kernels, queued on one stream by two threads in turns of their own making."""
    import threading
    work = []
    for i, (m, n, k) in enumerate([(511, 1300, 2049), (2500, 1100, 70)]):
        x, w = (mm.to_device(randn(*s, seed=10 * i + j)).requires_grad_(True) for j, s in enumerate(((m, k), (n, k))))
        g, ln = mm.to_device(randn(m, n, seed=10 * i + 5)), mm.to_device(randn(n, seed=10 * i + 6)).requires_grad_(True)

        def step(x=x, w=w, g=g, ln=ln, n=n):
            y = F.layer_norm(mm.linear(x, w, activation="gelu"), (n,), ln)
            return [y.detach(), *torch.autograd.grad(y, (x, w, ln), g)]

        work.append((step, [t.cpu() for t in step()]))
    bad = []

    def run(step, want):
        try:
            with torch.autograd.set_multithreading_enabled(False):
                for _ in range(40):
                    got = step()
                if not all(torch.equal(t.cpu(), v) for t, v in zip(got, want)):
                    bad.append("other bits")
        except Exception as e:  # for the assertion below
            bad.append(e)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not bad and not any(t.is_alive() for t in threads)
