import os
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

GOLDEN = ROOT / "tests" / "golden"


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (runs through libmatrixman_b200 on cuda:0)")


@pytest.fixture(autouse=True)
def no_device_behind_host_tests(request, monkeypatch):
    """Tests without the gpu marker make tensors of made-up addresses and record
    launches: the C++ extension, which GPU tests before them may have loaded, would
    hand those addresses to a device."""
    if request.node.get_closest_marker("gpu") is None:
        from matrixman_b200 import privateuse
        monkeypatch.setattr(privateuse, "_native", None)


@pytest.fixture(scope="session")
def golden():
    import numpy as np
    return dict(np.load(GOLDEN / "reference_vectors.npz"))


@pytest.fixture(scope="session")
def mm():
    """The product package with the device runtime initialised (GPU tests only)."""
    import matrixman_b200 as matrixman
    matrixman.init()
    return matrixman
