"""What matrixman.prepare makes of group norms, on the host."""

import torch
from torch import nn

import matrixman_b200 as matrixman
from matrixman_b200.preparation import PreparedConv2d, PreparedGroupNorm


def inner(p):
    return p.module if hasattr(p, "module") and isinstance(p.module, nn.Module) else p


def test_norms_take_over_their_activation():
    act = nn.SiLU()  # shared
    model = nn.Sequential(nn.Conv2d(3, 8, 3), nn.GroupNorm(2, 8, eps=1e-3), act, nn.Conv2d(8, 8, 3), act,
                          nn.GroupNorm(4, 8, affine=False), nn.GELU(approximate="tanh"), nn.GroupNorm(8, 8), nn.Tanh(),
                          nn.GroupNorm(1, 8)).eval()
    p = matrixman.prepare(model)
    got = list(inner(p))
    assert p._matrixman_preparation_report.block_units_prepared["GroupNorm"] == 4
    norms = [m for m in got if isinstance(m, PreparedGroupNorm)]
    assert [m.activation for m in norms] == ["silu", "gelu_tanh", "none", "none"]
    assert [m.num_groups for m in norms] == [2, 4, 8, 1] and norms[0].eps == 1e-3
    assert norms[1].weight is None and torch.equal(norms[0].weight, model[1].weight)
    assert isinstance(got[2], nn.Identity) and isinstance(got[6], nn.Identity) and isinstance(got[8], nn.Tanh)
    assert isinstance(got[3], PreparedConv2d) and isinstance(got[4], nn.Identity)
    assert isinstance(model[1], nn.GroupNorm) and model[2] is act  # a copy was prepared


def test_shared_norms_are_left():
    norm = nn.GroupNorm(2, 8)
    p = matrixman.prepare(nn.Sequential(norm, nn.ReLU(), norm, nn.ReLU()).eval())
    assert [type(m) for m in inner(p)] == [nn.GroupNorm, nn.ReLU, nn.GroupNorm, nn.ReLU]
