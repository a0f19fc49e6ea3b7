"""Argument checks of the group-norm entry points: every call below is refused
(or has nothing to do) before anything reaches a device, so the pointers are
never followed."""

import ctypes

from matrixman_b200 import _lib

FAKE = 1 << 20


def test_group_norm_checks():
    f = _lib.load().mm_group_norm
    ok = dict(x=FAKE, xi=96, xr=8, n=4, c=8, px=12, g=2, act=2, y=FAKE, mean=FAKE, rstd=FAKE, work=FAKE, size=1 << 20)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["x"], a["xi"], a["xr"], a["n"], a["c"], a["px"], a["g"], 1, FAKE, FAKE, 1e-5, a["act"], a["y"],
                 a["mean"], a["rstd"], a["work"], a["size"], None)

    for name in ("x", "y", "mean", "rstd"):  # (mean and rstd go together)
        assert call(**{name: None}) == _lib.MM_ERR_INVALID
    for name in ("xi", "xr", "n", "c", "px"):
        assert call(**{name: -1}) == _lib.MM_ERR_INVALID
    for groups in (0, -2, 3, 16):
        assert call(g=groups) == _lib.MM_ERR_INVALID
    for act in (-1, 6):
        assert call(act=act) == _lib.MM_ERR_INVALID
    for big in (1 << 31, 1 << 40, 1 << 62):
        for name in ("n", "c", "px"):
            assert call(**{name: big}) == _lib.MM_ERR_UNSUPPORTED
    assert call(n=1 << 20, c=1 << 12) == _lib.MM_ERR_UNSUPPORTED
    assert call(px=0) == _lib.MM_ERR_UNSUPPORTED
    assert call(n=0) == _lib.MM_OK and call(c=0) == _lib.MM_OK
    assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID
    assert call(size=8) == _lib.MM_ERR_INVALID


def test_group_norm_backward_checks():
    f = _lib.load().mm_group_norm_backward
    ok = dict(dy=FAKE, gi=96, gr=8, x=FAKE, xi=96, xr=8, n=4, c=8, px=12, g=2, mean=FAKE, rstd=FAKE, act=2, dx=FAKE,
              dw=FAKE, db=FAKE, work=FAKE, size=1 << 20)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["dy"], a["gi"], a["gr"], a["x"], a["xi"], a["xr"], a["n"], a["c"], a["px"], a["g"], 1, a["mean"],
                 a["rstd"], FAKE, FAKE, a["act"], a["dx"], a["dw"], a["db"], a["work"], a["size"], None)

    for name in ("dy", "x", "mean", "rstd"):
        assert call(**{name: None}) == _lib.MM_ERR_INVALID
    for name in ("gi", "gr", "xi", "xr", "n", "c", "px"):
        assert call(**{name: -1}) == _lib.MM_ERR_INVALID
    for groups in (0, 3):
        assert call(g=groups) == _lib.MM_ERR_INVALID
    assert call(act=6) == _lib.MM_ERR_INVALID
    assert call(n=1 << 31) == _lib.MM_ERR_UNSUPPORTED
    assert call(work=FAKE + 4) == _lib.MM_ERR_INVALID
    assert call(size=8) == _lib.MM_ERR_INVALID
    assert call(dx=None, dw=None, db=None) == _lib.MM_OK


def test_group_norm_workspace_size():
    lib = _lib.load()
    size = ctypes.c_size_t(77)
    assert lib.mm_group_norm_workspace_size(4, 8, 12, 2, ctypes.byref(size)) == _lib.MM_OK
    assert 0 < size.value < 1 << 16
    size = ctypes.c_size_t(77)
    for sizes in ((1 << 31, 8, 12, 2), (4, 1 << 40, 12, 2), (4, 8, 1 << 62, 2)):
        assert lib.mm_group_norm_workspace_size(*sizes, ctypes.byref(size)) == _lib.MM_ERR_UNSUPPORTED
    for sizes in ((-1, 8, 12, 2), (4, 8, 12, 3), (4, 8, 12, 0)):
        assert lib.mm_group_norm_workspace_size(*sizes, ctypes.byref(size)) == _lib.MM_ERR_INVALID
    assert size.value == 77
    assert lib.mm_group_norm_workspace_size(4, 8, 12, 2, None) == _lib.MM_ERR_INVALID
