"""What a test of gigabytes allocates is given back before the next one runs (in
file order: the first test leaves it behind, the second looks for it)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gigabytes_are_used():
    assert torch.empty(3 << 30, dtype=torch.uint8, device="cuda").numel() == 3 << 30


def test_gigabytes_are_gone():
    """No free segment that a later tensor could be cut from."""
    assert torch.cuda.memory_reserved() - torch.cuda.memory_allocated() <= 256 << 20
