import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs through libullm_hip.so)")


@pytest.fixture(scope="session")
def dev():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("GPU test run without a visible GPU")
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _large_memory_goes_back(request):
    """A test of gigabytes leaves them in torch's allocator as one free segment, from
    which the next tests' tensors would be cut: tests that count on what is reserved
    (calls that find no scratch) would then find room in it."""
    yield
    if request.node.get_closest_marker("gpu"):
        import torch

        if torch.cuda.is_initialized() and torch.cuda.memory_reserved() > 256 << 20:
            torch.cuda.empty_cache()
