"""Argument checks of the gradient-norm entry points: every call below is refused
before anything reaches a device, so the pointers are never followed."""

import ctypes
import math

from matrixman_b200 import _lib

FAKE = 1 << 20


def rows(*pairs):
    return (ctypes.c_int64 * (2 * len(pairs)))(*(v for p in pairs for v in p))


def test_grad_norm_checks():
    lib = _lib.load()
    two = rows((FAKE, 10), (FAKE + 4096, 20))

    def norm(grads=two, count=2, order=2, limit=1.0, out=FAKE, work=FAKE, size=1 << 20):
        return lib.mm_grad_norm(grads, count, order, limit, out, FAKE, work, size, None)

    def clip(grads=two, count=2, order=2, limit=1.0, out=FAKE, work=FAKE, size=1 << 20):
        return lib.mm_grad_clip(grads, count, order, limit, out, work, size, None)

    for call in (norm, clip):
        assert call(count=-1) == _lib.MM_ERR_INVALID and call(grads=None) == _lib.MM_ERR_INVALID
        assert call(order=3) == _lib.MM_ERR_UNSUPPORTED and call(order=-1) == _lib.MM_ERR_UNSUPPORTED
        assert call(limit=-1.0) == _lib.MM_ERR_INVALID and call(limit=math.nan) == _lib.MM_ERR_INVALID
        assert call(out=None) == _lib.MM_ERR_INVALID
        assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID and call(size=8) == _lib.MM_ERR_INVALID
        for bad in ((0, 10), (FAKE, -1), (FAKE + 2, 10), (FAKE, 1 << 62)):
            assert call(grads=rows((FAKE, 10), bad)) == _lib.MM_ERR_INVALID


def test_clipping_refuses_shared_memory():
    """The workspace is too small, which is said only of calls whose tensors are apart."""
    lib = _lib.load()

    def call(*pairs):
        status = lib.mm_grad_clip(rows(*pairs), len(pairs), 2, 1.0, FAKE, FAKE, 8, None)
        assert status == _lib.MM_ERR_INVALID
        return "workspace" if "workspace" in _lib.last_error() else "shares" if "shares" in _lib.last_error() else "?"

    assert call((FAKE, 10), (FAKE + 40, 10)) == "workspace"
    assert call((FAKE, 11), (FAKE + 40, 10)) == "shares"
    assert call((FAKE + 40, 10), (FAKE, 11)) == "shares"
    assert call((FAKE, 10), (FAKE, 10)) == "shares"
    assert call((FAKE, 1000), (FAKE + 80, 3)) == "shares"
    assert call((FAKE, 10), (FAKE, 0), (FAKE + 20, 0)) == "workspace"
    many = [(FAKE + 4096 * i, 1024) for i in range(3000)]
    assert call(*many) == "workspace"
    assert call(*many, (FAKE + 4096 * 1234 + 8, 1)) == "shares"


def test_grad_norm_workspace_size():
    lib = _lib.load()
    size = ctypes.c_size_t(0)
    assert lib.mm_grad_norm_workspace_size(0, ctypes.byref(size)) == _lib.MM_OK and size.value > 0
    few = size.value
    assert lib.mm_grad_norm_workspace_size(5000, ctypes.byref(size)) == _lib.MM_OK and size.value > few
    assert lib.mm_grad_norm_workspace_size(-1, ctypes.byref(size)) == _lib.MM_ERR_INVALID
    assert lib.mm_grad_norm_workspace_size(1, None) == _lib.MM_ERR_INVALID


def test_scaled_adamw_checks():
    lib = _lib.load()
    row = (ctypes.c_int64 * 8)(FAKE, FAKE + 64, FAKE + 128, FAKE + 192, 0, 0, FAKE + 256, 10)

    def call(bits=32, b1=0.9, work=FAKE, n=8):
        return lib.mm_adamw_scaled(row, 1, bits, 1e-3, b1, 0.99, 1e-8, 0.0, 1, 0, 1, FAKE, work, n, None)

    assert call(bits=16) == _lib.MM_ERR_UNSUPPORTED and call(b1=1.0) == _lib.MM_ERR_INVALID
    assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID and call(n=7) == _lib.MM_ERR_INVALID
