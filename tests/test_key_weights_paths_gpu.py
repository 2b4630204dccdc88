"""key_weights(_paged) on the GPU: calls at the ends of what it takes, on each of its ways
(scores stored, query rows in registers, keys in registers)."""
import numpy as np
import pytest
import torch

from ullm_amd import attention as A

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (32, 1, 64), (320, 1, 64), (8, 4, 256)])
def test_no_rows(dev, kv, H, Hk, D):
    """Rows of none: the weights fade, each by one rounding."""
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.empty(3, 0, H, D, dtype=kv, device=dev)
    k = torch.randn(3, 96, Hk * D, device=dev, generator=g).to(kv)
    old = torch.rand(3, Hk, 96, device=dev, generator=g)
    lens, there = i32([96, 0, 41], dev), torch.arange(96, device=dev) < torch.tensor([96, 0, 41], device=dev)[:, None, None]
    table = i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]], dev)
    for window in (0, 20):
        for decay in (0.0, 0.3, 1.0):
            want = torch.where(there, decay * old, old)
            for w in (A.key_weights(q, k, old.clone(), lens, 96, Hk, window=window, decay=decay),
                      A.key_weights_paged(q, k.view(9, 32, Hk * D), table, old.clone(), lens, 96, Hk, window=window, decay=decay)):
                assert torch.equal(w, want)
