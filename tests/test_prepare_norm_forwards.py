"""matrixman.prepare joins a group norm with the activation behind it only where the
container runs one after the other and nobody looks in between (on the host)."""

import torch
from torch import nn

import matrixman_b200 as matrixman
from matrixman_b200.preparation import PreparedGroupNorm

from .test_prepare_norm_cpu import inner


class Skip(nn.Sequential):
    def forward(self, x):
        n = self[0](x)
        return self[1](n) + n


class Plain(nn.Sequential):
    pass


def test_containers_with_their_own_forward_keep_the_activation():
    got = list(inner(matrixman.prepare(Skip(nn.GroupNorm(2, 8), nn.SiLU()).eval())))
    assert isinstance(got[0], PreparedGroupNorm) and got[0].activation == "none" and isinstance(got[1], nn.SiLU)
    got = list(inner(matrixman.prepare(Plain(nn.GroupNorm(2, 8), nn.SiLU()).eval())))
    assert got[0].activation == "silu" and isinstance(got[1], nn.Identity)


def test_modules_with_hooks_are_left():
    def model(hooked, register):
        m = nn.Sequential(nn.GroupNorm(2, 8), nn.ReLU()).eval()
        getattr(m[hooked], register)(lambda *a: None)
        return list(inner(matrixman.prepare(m)))

    for register in ("register_forward_hook", "register_forward_pre_hook"):
        got = model(0, register)
        assert [type(m) for m in got] == [nn.GroupNorm, nn.ReLU]
        got = model(1, register)
        assert got[0].activation == "none" and isinstance(got[1], nn.ReLU)
    m = nn.Sequential(nn.GroupNorm(2, 8), nn.ReLU()).eval()
    got = list(inner(matrixman.prepare(m)))
    assert got[0].activation == "relu" and torch.equal(got[0].weight, m[0].weight)
