"""torch.linalg.vector_norm on MatrixMan tensors, on a runtime that has no device."""

import pytest
import torch

from .test_adamw_states import launches, rt  # noqa: F401 - fixtures
from .test_grad_norm_overlaps import views


@pytest.mark.parametrize("dim", [(), [], None, (0, 1), (-1, 0)])
def test_vector_norm_over_all_dimensions(rt, launches, dim):  # noqa: F811
    x = views(rt, ((3, 4), (4, 1), 0))[0]
    assert torch.linalg.vector_norm(x, dim=dim).shape == () and launches == ["mm_grad_norm"]


def test_vector_norms_that_torch_refuses(rt, launches):  # noqa: F811
    x = views(rt, ((0, 4), (4, 1), 0))[0]
    with pytest.raises(RuntimeError, match="empty"):
        torch.linalg.vector_norm(x, float("inf"))
    assert launches == []
    assert torch.linalg.vector_norm(x).shape == ()
