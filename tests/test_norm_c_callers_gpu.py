"""mm_group_norm, mm_grad_norm, mm_grad_clip and mm_adamw_scaled as a C caller uses them: on streams
of its own, with workspaces of exactly the size that is asked for, at any float's address.  Results are
those of the Python calls, whose tests hold them to the formulas; nothing around the arrays changes."""

import ctypes

import pytest
import torch

from matrixman_b200 import _lib, ops

pytestmark = pytest.mark.gpu

GUARD = 64  # floats in front of and behind every array
FILL = -77.0


class Arena:
    """Arrays of floats in device memory, each between guards, `shift` floats off 256-byte boundaries."""

    def __init__(self, mm):
        self.mm, self.held = mm, []

    def array(self, values, shift=0):
        flat = values.reshape(-1)
        whole = torch.full((flat.numel() + 2 * GUARD + shift,), FILL)
        whole[GUARD + shift:GUARD + shift + flat.numel()] = flat
        t = self.mm.to_device(whole)
        self.held.append((t, GUARD + shift, flat.numel()))
        return ops.pointer(t) + 4 * (GUARD + shift)

    def empty(self, count, shift=0):
        return self.array(torch.full((count,), FILL), shift)

    def read(self, i):
        """The values of the i-th array, after a look at its guards."""
        t, at, n = self.held[i]
        whole = t.cpu()
        assert (whole[:at] == FILL).all() and (whole[at + n:] == FILL).all(), f"array {i}: a guard changed"
        return whole[at:at + n]


@pytest.fixture
def stream(mm):
    rt = mm.to_device(torch.zeros(1)).runtime
    out = ctypes.c_void_p()
    _lib.check(rt.lib.mm_stream_create(rt.index, ctypes.byref(out)))
    yield rt, out
    rt.synchronize()
    _lib.check(rt.lib.mm_stream_destroy(out))


def size_of(call, *args):
    size = ctypes.c_size_t()
    _lib.check(call(*args, ctypes.byref(size)))
    assert size.value % 4 == 0
    return size.value


# Maps that one block, a cluster, and only the walking kernels hold; of odd channels.
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("n,c,side,groups", [(3, 16, 5, 4), (2, 48, 64, 8), (1, 130, 300, 2), (2, 15, 33, 5)])
def test_group_norm(mm, stream, n, c, side, groups, last, shift):
    rt, own = stream
    lib = rt.lib
    g = torch.Generator()
    g.manual_seed(c)
    x, dy = (torch.randn(n, c, side, side, generator=g) for _ in range(2))
    w, b = 1 + torch.rand(c, generator=g), torch.randn(c, generator=g)
    act = _lib.LINEAR_ACTS["silu"]
    pixels = side * side

    def order(t):
        return t.permute(0, 2, 3, 1).contiguous() if last else t

    def maps(t):  # as far from a boundary as the C call's arrays
        flat = mm.to_device(torch.cat([torch.zeros(shift), order(t).reshape(-1)]))[shift:]
        return flat.view(n, side, side, c).permute(0, 3, 1, 2) if last else flat.view(n, c, side, side)

    xr, gr = maps(x), maps(dy)
    y, mean, rstd = ops.group_norm(xr, groups, mm.to_device(w), mm.to_device(b), 1e-5, act)
    want = [order(y.cpu()), mean.cpu(), rstd.cpu()]
    grads = ops.group_norm_backward(gr, xr, mean, rstd, mm.to_device(w), mm.to_device(b), groups, (True,) * 3, act)
    want += [order(grads[0].cpu()), grads[1].cpu(), grads[2].cpu()]

    size = size_of(lib.mm_group_norm_workspace_size, n, c, pixels, groups)
    arena = Arena(mm)
    px, pd, pw, pb = (arena.array(t, shift) for t in (order(x), order(dy), w, b))
    py, pm, pr, pdx, pdw, pdb = (arena.empty(k, shift) for k in (x.numel(), n * groups, n * groups, x.numel(), c, c))
    work = arena.empty(size // 4)
    image, row = c * pixels, c if last else pixels
    rt.synchronize()
    for _ in range(2):  # (the second call finds the workspace as the first left it)
        _lib.check(lib.mm_group_norm(px, image, row, n, c, pixels, groups, int(last), pw, pb, 1e-5, act, py, pm, pr,
                                     work, size, own))
        _lib.check(lib.mm_group_norm_backward(pd, image, row, px, image, row, n, c, pixels, groups, int(last), pm, pr,
                                              pw, pb, act, pdx, pdw, pdb, work, size, own))
    _lib.check(lib.mm_stream_sync(own, 30_000))
    for i, v in enumerate(want):
        assert torch.equal(arena.read(4 + i), v.reshape(-1))
    for i in (0, 1, 2, 3, 10):
        arena.read(i)


@pytest.mark.parametrize("order", [_lib.NORM_ORDERS[k] for k in (1.0, 2.0, float("inf"))])
@pytest.mark.parametrize("sizes", [[1], [7, 0, 8193, 40001], [3 + i % 11 for i in range(1300)]])
def test_norm_and_clipping(mm, stream, sizes, order):
    rt, own = stream
    lib = rt.lib
    g = torch.Generator()
    g.manual_seed(len(sizes))
    grads = [torch.randn(k, generator=g) for k in sizes]
    params = [torch.nn.Parameter(mm.to_device(torch.zeros(k))) for k in sizes]
    flat, offset = mm.to_device(torch.cat([torch.zeros(1), *grads])), 1  # at the C call's distances
    for p in params:
        p.grad = flat[offset:offset + p.numel()]
        offset += p.numel()
    kind = {v: k for k, v in _lib.NORM_ORDERS.items()}[order]
    want = mm.optim.clip_grad_norm_(params, 0.5, kind).cpu()
    size = size_of(lib.mm_grad_norm_workspace_size, len(sizes))
    arena = Arena(mm)
    packed = torch.cat(grads)
    at = arena.array(packed, 1)
    pn, pc, work = arena.empty(1), arena.empty(1), arena.empty(size // 4)
    rows, offset = [], 0
    for k in sizes:
        rows += [at + 4 * offset, k]
        offset += k
    table = (ctypes.c_int64 * len(rows))(*rows)
    rt.synchronize()
    _lib.check(lib.mm_grad_norm(ctypes.addressof(table), len(sizes), order, 0.5, pn, pc, work, size, own))
    _lib.check(lib.mm_stream_sync(own, 30_000))
    norm, coef = arena.read(1)[0], arena.read(2)[0]
    assert torch.equal(arena.read(0), packed) and torch.equal(norm, want)
    assert torch.equal(coef, torch.clamp(torch.tensor(0.5) / (norm + 1e-6), max=1.0))
    _lib.check(lib.mm_grad_clip(ctypes.addressof(table), len(sizes), order, 0.5, pn, work, size, own))
    _lib.check(lib.mm_stream_sync(own, 30_000))
    assert torch.equal(arena.read(1)[0], norm) and torch.equal(arena.read(0), packed * coef)
    arena.read(3)


def test_scaled_step(mm, stream):
    """A scale of 1 gives mm_adamw's bits; one of 0.25 those of gradients that were multiplied by it."""
    rt, own = stream
    lib = rt.lib
    g = torch.Generator()
    g.manual_seed(5)
    n = 12345
    p, grad, m = (torch.randn(n, generator=g) for _ in range(3))
    v = torch.rand(n, generator=g)
    size = size_of(lib.mm_adamw_workspace_size, 1)
    got = {}
    for name, gr, scale in (("plain", grad, None), ("one", grad, 1.0), ("quarter", grad, 0.25),
                            ("scaled before", grad * 0.25, None)):
        arena = Arena(mm)
        pp, pg, pm, pv, ps = (arena.array(t) for t in (p, gr, m, v, torch.tensor([3.0])))
        work = arena.empty(size // 4)
        pscale = None if scale is None else arena.array(torch.tensor([scale]))
        row = (ctypes.c_int64 * 8)(pp, pg, pm, pv, 0, 0, ps, n)
        rt.synchronize()
        _lib.check(lib.mm_adamw_scaled(ctypes.addressof(row), 1, 32, 1e-3, 0.9, 0.999, 1e-8, 0.01, 1, 0, 1, pscale,
                                       work, size, own))
        _lib.check(lib.mm_stream_sync(own, 30_000))
        assert torch.equal(arena.read(1), gr)
        got[name] = [arena.read(i) for i in (0, 2, 3, 4)]
        arena.read(5)
    for a, b in (("plain", "one"), ("quarter", "scaled before")):
        assert all(torch.equal(s, t) for s, t in zip(got[a], got[b]))
    assert not torch.equal(got["one"][0], got["quarter"][0])
