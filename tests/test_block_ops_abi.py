"""Argument checks of the layer-norm, linear and AdamW entry points: every call
below is refused (or has nothing to do) before anything reaches a device, so
the pointers are never followed."""

import ctypes

from matrixman_b200 import _lib

FAKE = 1 << 20


def t(shape, strides=None, dtype=_lib.MM_F32, ptr=FAKE):
    if strides is None:
        strides, acc = [], 1
        for s in reversed(shape):
            strides.insert(0, acc)
            acc *= s
    return ctypes.byref(_lib.make_tensor(ptr, shape, strides, dtype))


def test_layer_norm_checks():
    f = _lib.load().mm_layer_norm
    ok = dict(x=t((4, 8)), w=t((8,)), b=t((8,)), y=t((4, 8)), mean=t((4,)), rstd=t((4,)))

    def call(**kw):
        a = {**ok, **kw}
        return f(a["x"], a["w"], a["b"], 1e-5, a["y"], a["mean"], a["rstd"], None)

    assert call(x=t((4, 8, 2))) == _lib.MM_ERR_UNSUPPORTED
    assert call(x=t((4, 8), dtype=_lib.MM_I64)) == _lib.MM_ERR_UNSUPPORTED
    assert call(x=t((4, 8), (1, 4))) == _lib.MM_ERR_UNSUPPORTED
    assert call(x=t((4, 8), ptr=0)) == _lib.MM_ERR_INVALID
    assert call(w=t((7,))) == _lib.MM_ERR_INVALID
    assert call(w=t((8,), (2,))) == _lib.MM_ERR_UNSUPPORTED
    assert call(b=t((9,))) == _lib.MM_ERR_INVALID
    assert call(y=t((4, 9))) == _lib.MM_ERR_INVALID
    assert call(y=t((4, 8), (16, 1))) == _lib.MM_ERR_UNSUPPORTED
    assert call(mean=t((5,))) == _lib.MM_ERR_INVALID
    assert call(x=None) == _lib.MM_ERR_INVALID
    assert call(x=t((0, 8)), y=t((0, 8)), mean=t((0,)), rstd=t((0,))) == _lib.MM_OK
    assert call(x=t((4, 0)), w=None, b=None, y=t((4, 0))) == _lib.MM_ERR_UNSUPPORTED


def test_layer_norm_backward_checks():
    f = _lib.load().mm_layer_norm_backward
    size = ctypes.c_size_t(0)
    assert _lib.load().mm_layer_norm_backward_workspace_size(4, 8, ctypes.byref(size)) == _lib.MM_OK
    assert size.value == 2 * 4 * 8 * 4
    assert _lib.load().mm_layer_norm_backward_workspace_size(-1, 8, ctypes.byref(size)) == _lib.MM_ERR_INVALID
    ok = dict(dy=t((4, 8)), x=t((4, 8)), mean=t((4,)), rstd=t((4,)), w=t((8,)), dx=t((4, 8)), dw=t((8,)), db=t((8,)),
              work=FAKE, n=1 << 16)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["dy"], a["x"], a["mean"], a["rstd"], a["w"], a["dx"], a["dw"], a["db"], a["work"], a["n"], None)

    assert call(dy=t((3, 8))) == _lib.MM_ERR_INVALID
    assert call(dx=t((4, 7))) == _lib.MM_ERR_INVALID
    assert call(dw=t((9,))) == _lib.MM_ERR_INVALID
    assert call(db=t((8,), (3,))) == _lib.MM_ERR_UNSUPPORTED
    assert call(work=None) == _lib.MM_ERR_INVALID
    assert call(n=16) == _lib.MM_ERR_INVALID
    assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID
    assert call(dx=None, dw=None, db=None) == _lib.MM_OK


def test_linear_checks():
    lib = _lib.load()
    big = 1 << 30
    ok = dict(x=t((4, 8)), w=t((6, 8)), b=t((6,)), r=t((4, 6)), act=0, y=t((4, 6)), z=None, work=FAKE, n=big)

    def call(**kw):
        a = {**ok, **kw}
        return lib.mm_linear(a["x"], a["w"], a["b"], a["r"], a["act"], 0, a["y"], a["z"], a["work"], a["n"], None)

    assert call(act=6) == _lib.MM_ERR_INVALID and call(act=-1) == _lib.MM_ERR_INVALID
    assert call(w=t((6, 9))) == _lib.MM_ERR_INVALID
    assert call(b=t((5,))) == _lib.MM_ERR_INVALID
    assert call(r=t((4, 7))) == _lib.MM_ERR_INVALID
    assert call(r=t((4, 6), (1, 4))) == _lib.MM_ERR_UNSUPPORTED
    assert call(y=t((4, 6), (12, 1))) == _lib.MM_ERR_UNSUPPORTED
    assert call(z=t((4, 5))) == _lib.MM_ERR_INVALID
    assert call(x=t((1 << 31, 8))) == _lib.MM_ERR_UNSUPPORTED
    assert call(x=t((4, 8), dtype=_lib.MM_I64)) == _lib.MM_ERR_UNSUPPORTED

    ok = dict(dy=t((4, 6)), x=t((4, 8)), w=t((6, 8)), z=t((4, 6)), act=4, dx=t((4, 8)), dw=t((6, 8)), db=t((6,)),
              dz=None, work=FAKE, n=big)

    def back(**kw):
        a = {**ok, **kw}
        return lib.mm_linear_backward(a["dy"], a["x"], a["w"], a["z"], a["act"], a["dx"], a["dw"], a["db"], a["dz"],
                                      a["work"], a["n"], None)

    assert back(z=None) == _lib.MM_ERR_INVALID
    assert back(dy=t((4, 5))) == _lib.MM_ERR_INVALID
    assert back(dx=t((4, 9))) == _lib.MM_ERR_INVALID
    assert back(dw=t((8, 6))) == _lib.MM_ERR_INVALID
    assert back(db=t((7,))) == _lib.MM_ERR_INVALID
    assert back(dz=t((4, 7))) == _lib.MM_ERR_INVALID
    assert back(work=None) == _lib.MM_ERR_INVALID
    assert back(n=8) == _lib.MM_ERR_INVALID
    assert back(act=9) == _lib.MM_ERR_INVALID


def test_adamw_checks():
    lib = _lib.load()
    row = (ctypes.c_int64 * 8)(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 10)

    def call(tensors=row, count=1, bits=32, b1=0.9, b2=0.99, work=FAKE, n=8):
        return lib.mm_adamw(tensors, count, bits, 1e-3, b1, b2, 1e-8, 0.0, 1, 0, 1, work, n, None)

    assert call(bits=16) == _lib.MM_ERR_UNSUPPORTED
    assert call(b1=1.0) == _lib.MM_ERR_INVALID and call(b2=-0.1) == _lib.MM_ERR_INVALID
    assert call(count=-1) == _lib.MM_ERR_INVALID and call(tensors=None) == _lib.MM_ERR_INVALID
    assert call(work=None) == _lib.MM_ERR_INVALID and call(n=7) == _lib.MM_ERR_INVALID
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
