"""Argument checks of the layer-norm, linear and AdamW entry points: every call
below is refused (or has nothing to do) before anything reaches a device, so
the pointers are never followed."""

import ctypes

from matrixman_b200 import _lib

FAKE = 1 << 20


def test_layer_norm_checks():
    f = _lib.load().mm_layer_norm
    ok = dict(x=FAKE, xs=8, rows=4, width=8, w=FAKE, b=FAKE, y=FAKE, mean=FAKE, rstd=FAKE)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["x"], a["xs"], a["rows"], a["width"], a["w"], a["b"], 1e-5, a["y"], a["mean"], a["rstd"], None)

    for name in ("x", "y", "mean", "rstd"):
        assert call(**{name: None}) == _lib.MM_ERR_INVALID
    for name in ("xs", "rows", "width"):
        assert call(**{name: -1}) == _lib.MM_ERR_INVALID
    assert call(rows=1 << 31) == _lib.MM_ERR_UNSUPPORTED
    assert call(width=1 << 31) == _lib.MM_ERR_UNSUPPORTED
    assert call(width=0) == _lib.MM_ERR_UNSUPPORTED
    assert call(rows=0) == _lib.MM_OK


def test_layer_norm_backward_checks():
    f = _lib.load().mm_layer_norm_backward
    size = ctypes.c_size_t(0)
    assert _lib.load().mm_layer_norm_backward_workspace_size(4, 8, ctypes.byref(size)) == _lib.MM_OK
    assert size.value == 2 * 4 * 8 * 4
    assert _lib.load().mm_layer_norm_backward_workspace_size(-1, 8, ctypes.byref(size)) == _lib.MM_ERR_INVALID
    ok = dict(dy=FAKE, dys=8, x=FAKE, xs=8, rows=4, width=8, mean=FAKE, rstd=FAKE, dx=FAKE, dw=FAKE, db=FAKE,
              work=FAKE, n=1 << 16)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["dy"], a["dys"], a["x"], a["xs"], a["rows"], a["width"], a["mean"], a["rstd"], FAKE, a["dx"],
                 a["dw"], a["db"], a["work"], a["n"], None)

    for name in ("dy", "x", "mean", "rstd"):
        assert call(**{name: None}) == _lib.MM_ERR_INVALID
    for name in ("dys", "xs", "rows", "width"):
        assert call(**{name: -1}) == _lib.MM_ERR_INVALID
    assert call(n=16) == _lib.MM_ERR_INVALID
    assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID
    assert call(dx=None, dw=None, db=None) == _lib.MM_OK


def test_linear_checks():
    lib = _lib.load()
    big = 1 << 30
    ok = dict(x=FAKE, xs0=8, xs1=1, w=FAKE, ws0=8, ws1=1, rs=6, m=4, n=6, k=8, act=0, y=FAKE, work=FAKE, size=big)

    def call(**kw):
        a = {**ok, **kw}
        return lib.mm_linear(a["x"], a["xs0"], a["xs1"], a["w"], a["ws0"], a["ws1"], FAKE, FAKE, a["rs"], a["m"],
                             a["n"], a["k"], a["act"], 0, a["y"], None, a["work"], a["size"], None)

    assert call(act=6) == _lib.MM_ERR_INVALID and call(act=-1) == _lib.MM_ERR_INVALID
    for name in ("m", "n", "k", "xs0", "xs1", "ws0", "ws1", "rs"):
        assert call(**{name: -1}) == _lib.MM_ERR_INVALID
    for name in ("x", "w", "y"):
        assert call(**{name: None}) == _lib.MM_ERR_INVALID
    assert call(m=1 << 31) == _lib.MM_ERR_UNSUPPORTED
    assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID
    assert call(m=4096, n=4096, k=4096, size=8) == _lib.MM_ERR_INVALID
    assert call(m=0) == _lib.MM_OK and call(n=0) == _lib.MM_OK

    ok = dict(dy=FAKE, dys=6, x=FAKE, xs0=8, xs1=1, w=FAKE, ws0=8, ws1=1, z=FAKE, m=4, n=6, k=8, act=4, dx=FAKE,
              dw=FAKE, db=FAKE, dz=None, work=FAKE, size=big)

    def back(**kw):
        a = {**ok, **kw}
        return lib.mm_linear_backward(a["dy"], a["dys"], a["x"], a["xs0"], a["xs1"], a["w"], a["ws0"], a["ws1"],
                                      a["z"], a["m"], a["n"], a["k"], a["act"], a["dx"], a["dw"], a["db"], a["dz"],
                                      a["work"], a["size"], None)

    for name in ("dy", "x", "w", "z"):
        assert back(**{name: None}) == _lib.MM_ERR_INVALID
    for name in ("m", "n", "k", "dys", "xs0", "xs1", "ws0", "ws1"):
        assert back(**{name: -1}) == _lib.MM_ERR_INVALID
    assert back(m=4096, n=4096, k=4096, dys=4096, size=8) == _lib.MM_ERR_INVALID
    assert back(work=FAKE + 8) == _lib.MM_ERR_INVALID
    assert back(act=9) == _lib.MM_ERR_INVALID
    assert back(dx=None, dw=None, db=None) == _lib.MM_OK


def test_adamw_checks():
    lib = _lib.load()
    row = (ctypes.c_int64 * 8)(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 10)

    def call(tensors=row, count=1, bits=32, b1=0.9, b2=0.99, work=FAKE, n=8):
        return lib.mm_adamw(tensors, count, bits, 1e-3, b1, b2, 1e-8, 0.0, 1, 0, 1, work, n, None)

    assert call(bits=16) == _lib.MM_ERR_UNSUPPORTED
    assert call(b1=1.0) == _lib.MM_ERR_INVALID and call(b2=-0.1) == _lib.MM_ERR_INVALID
    assert call(count=-1) == _lib.MM_ERR_INVALID and call(tensors=None) == _lib.MM_ERR_INVALID
    assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID and call(n=7) == _lib.MM_ERR_INVALID
    assert call(count=0) == _lib.MM_OK
    for i in (0, 1, 2, 3, 6):
        bad = (ctypes.c_int64 * 8)(*row)
        bad[i] = 0
        assert call(tensors=bad) == _lib.MM_ERR_INVALID
    bad = (ctypes.c_int64 * 8)(*row)
    bad[7] = -1
    assert call(tensors=bad) == _lib.MM_ERR_INVALID
    for i in (4, 5):
        bad = (ctypes.c_int64 * 8)(*row)
        bad[i] = 0
        assert call(tensors=bad, bits=8) == _lib.MM_ERR_INVALID
    bad = (ctypes.c_int64 * 8)(*row)
    bad[2] = FAKE + 4
    assert call(tensors=bad, bits=8) == _lib.MM_ERR_INVALID
    assert lib.mm_adamw_encode(FAKE, FAKE, -1, FAKE, FAKE, FAKE, FAKE, None) == _lib.MM_ERR_INVALID
    assert lib.mm_adamw_encode(None, FAKE, 5, FAKE, FAKE, FAKE, FAKE, None) == _lib.MM_ERR_INVALID
    assert lib.mm_adamw_encode(FAKE, FAKE, 5, FAKE + 1, FAKE, FAKE, FAKE, None) == _lib.MM_ERR_INVALID
    assert lib.mm_adamw_decode(FAKE, FAKE, None, FAKE, 5, FAKE, FAKE, None) == _lib.MM_ERR_INVALID
    assert lib.mm_adamw_decode(None, None, None, None, 0, None, None, None) == _lib.MM_OK


def test_adamw_refuses_the_same_memory_twice():
    """The workspace is too small, which is said only of calls whose tensors are their own."""
    lib = _lib.load()

    def call(rows, bits=32, advance=1):
        table = (ctypes.c_int64 * (8 * len(rows)))(*(v for r in rows for v in r))
        status = lib.mm_adamw(table, len(rows), bits, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, 0, advance, FAKE, 1, None)
        assert status == _lib.MM_ERR_INVALID
        return "workspace" if "workspace" in _lib.last_error() else "shares" if "shares" in _lib.last_error() else "?"

    def row(i, **kw):
        names = ("p", "g", "m", "v", "ms", "vs", "step")
        got = {k: FAKE + 4096 * (16 * i + j) for j, k in enumerate(names)} | {"n": 10} | kw
        return [got[k] for k in (*names, "n")]

    for bits in (32, 8):
        assert call([row(0), row(1), row(2)], bits) == "workspace"
        first = dict(zip(("p", "g", "m", "v", "ms", "vs", "step"), row(0)))
        for name in ("p", "m", "v", "step") + (("ms", "vs") if bits == 8 else ()):
            assert call([row(0), row(1), row(2, **{name: first[name]})], bits) == "shares"
            assert call([row(0), row(1, p=first[name])], bits) == "shares"
        assert call([row(0, v=first["m"])], bits) == "shares"
        assert call([row(0), row(1, g=first["g"])], bits) == "workspace"  # gradients are only read
        assert call([row(0), row(1, step=first["step"])], bits, advance=0) == "workspace"
        assert call([row(0), row(1, n=0, p=first["p"], m=first["m"], v=0)], bits) == "workspace"  # nothing to write
    assert call([row(i) for i in range(1000)]) == "workspace"
    assert call([row(i) for i in range(1000)] + [row(1000, m=row(3)[2])]) == "shares"


def test_workspace_sizes_of_refused_dimensions():
    """What the calls refuse has no size (products of such dimensions overflow)."""
    lib = _lib.load()
    for big in (1 << 31, 1 << 40, 1 << 62):
        for sizes in ((big, 8, 8), (8, big, 8), (8, 8, big), (big, big, big)):
            for back in (0, 1):
                size = ctypes.c_size_t(77)
                assert lib.mm_linear_workspace_size(*sizes, back, ctypes.byref(size)) == _lib.MM_ERR_UNSUPPORTED
                assert size.value == 77
            assert lib.mm_linear(FAKE, 8, 1, FAKE, 8, 1, None, None, 0, *sizes, 0, 0, FAKE, None, None, 0,
                                 None) == _lib.MM_ERR_UNSUPPORTED
            assert lib.mm_linear_backward(FAKE, 8, FAKE, 8, 1, FAKE, 8, 1, None, *sizes, 0, FAKE, FAKE, FAKE, None, None,
                                          0, None) == _lib.MM_ERR_UNSUPPORTED
        for sizes in ((big, 8), (8, big)):
            size = ctypes.c_size_t(77)
            assert lib.mm_layer_norm_backward_workspace_size(*sizes, ctypes.byref(size)) == _lib.MM_ERR_UNSUPPORTED
            assert size.value == 77
    size = ctypes.c_size_t(0)
    assert lib.mm_linear_workspace_size(-1, 8, 8, 0, ctypes.byref(size)) == _lib.MM_ERR_INVALID
    assert lib.mm_linear_workspace_size(4096, 4096, 4096, 1, ctypes.byref(size)) == _lib.MM_OK and size.value > 0
