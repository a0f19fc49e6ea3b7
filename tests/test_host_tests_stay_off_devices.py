"""Host tests step optimisers over made-up addresses and record the launches.  Where
the C++ extension is loaded (GPU tests ran before them in the same process) its calls
would hand those addresses to a device; here a recording stand-in is in its place."""

import pytest

from matrixman_b200 import optim, privateuse

from .test_adamw_states import launches, made, rt, tensor  # noqa: F401 - fixtures


class Recorder:
    """Takes every call as the extension would, and does nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args, **kwargs: self.calls.append(name) or True


@pytest.fixture(scope="module", autouse=True)
def loaded():
    """The extension, loaded before the first of these tests."""
    before, privateuse._native = privateuse._native, Recorder()
    yield privateuse._native
    privateuse._native = before


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_over_made_up_addresses(loaded, rt, launches, bits):  # noqa: F811
    opt, p = made(rt, (1000,), bits)
    opt.step()
    opt.set_state_values(p, tensor(rt, 1000), tensor(rt, 1000))
    assert loaded.calls == [] and launches[0] == "mm_adamw"


def test_a_norm_over_made_up_addresses(loaded, rt, launches):  # noqa: F811
    _, p = made(rt, (1000,), 32)
    optim.grad_norm([p])
    optim.clip_grad_norm_([p], 1.0)
    assert loaded.calls == [] and launches == ["mm_grad_norm", "mm_grad_clip"]
