"""How group norm divides its calls (host code): the hooks that show and limit it."""

import ctypes

import pytest

from matrixman_b200 import _lib


def plan(n, c, pixels, groups, last, backward):
    got = [ctypes.c_int(-1) for _ in range(3)]
    _lib.check(_lib.load().mm_debug_group_norm_plan(n, c, pixels, groups, last, backward, *map(ctypes.byref, got)))
    return tuple(v.value for v in got)  # blocks of a cluster, images of a block, segments


@pytest.mark.parametrize("last", [True, False])
@pytest.mark.parametrize("backward", [True, False])
def test_calls_of_every_kind(last, backward):
    assert plan(1, 64, 400, 16, last, backward) == (1, 1, 0)
    ranks, images, segments = plan(2, 48, 4096, 8, last, backward)
    assert 1 < ranks <= 16 and images == 1 and segments == 0
    ranks, images, segments = plan(4099, 64, 1, 8, last, backward)
    assert ranks == 1 and images > 1 and 4099 % images and segments == 0
    ranks, images, segments = plan(1, 16, 90000, 1, last, backward)
    assert ranks == 0 and images == 0 and segments > 1


def test_what_the_hooks_refuse():
    lib = _lib.load()
    out = [ctypes.byref(ctypes.c_int()) for _ in range(3)]
    call = lib.mm_debug_group_norm_plan
    assert call(2, 48, 4096, 7, 1, 0, *out) == _lib.MM_ERR_INVALID
    assert call(-1, 48, 4096, 8, 1, 0, *out) == _lib.MM_ERR_INVALID
    for empty in ((0, 48, 4096), (2, 0, 4096), (2, 48, 0)):
        assert call(*empty, 8, 1, 0, *out) == _lib.MM_ERR_INVALID
    assert call(2, 48, 4096, 8, 1, 0, None, *out[1:]) == _lib.MM_ERR_INVALID
    for device in (-1, 64):
        assert lib.mm_debug_group_norm_ranks(device, 0) == _lib.MM_ERR_INVALID
