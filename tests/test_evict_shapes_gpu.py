"""Scores of kv_evict whose dimensions are not the caches' are refused, also where they have
as many numbers."""
import numpy as np
import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


@pytest.mark.parametrize("paged", [False, True])
def test_layers_and_sequences_are_not_exchanged(dev, paged):
    NL, B, G, n, d = 2, 3, 2, 64, 32
    k = torch.randn(NL, B, n, d, device=dev).half()
    v, scores = k.clone(), torch.rand(NL, B, G, n, device=dev)
    lens, budget = i32([64, 50, 9], dev), i32([20, 20, 20], dev)
    if paged:
        table = i32([[0, 1], [2, 3], [4, 5]], dev)
        pools = [x.view(NL, B * 2, 32, d) for x in (k, v)]
        call = lambda s: A.kv_evict_paged(*pools, table, s, lens, budget, max_budget=20)  # noqa: E731
    else:
        call = lambda s: A.kv_evict(k, v, s, lens, budget, max_budget=20)  # noqa: E731
    old = k.clone()
    for shape in ((B, NL, G, n), (NL * B, G, n), (G, NL, B, n), (NL * B * G, n), (1, B, NL, G, n)):
        with pytest.raises(L.UllmHipError, match="scores"):
            call(scores.reshape(shape))
    assert torch.equal(k, old)
    kept, new = call(scores)
    assert kept.shape == (NL, B, G, 20) and new.tolist() == [20, 20, 9]


def test_dimensions_of_one(dev):
    """One layer or one sequence: with or without their dimension."""
    for NL, B, shapes in ((1, 3, ((1, 3, 2, 40), (3, 2, 40))), (3, 1, ((3, 1, 2, 40), (3, 2, 40))), (1, 1, ((1, 1, 2, 40), (1, 2, 40), (2, 40)))):
        k = torch.randn(NL, B, 40, 32, device=dev).half()
        scores, kept = torch.rand(NL, B, 2, 40, device=dev), []
        for shape in shapes:
            kept.append(A.kv_evict(k.clone(), k.clone(), scores.clone().view(shape), i32([33] * B, dev), i32([11] * B, dev), max_budget=11)[0])
        assert all(torch.equal(x, kept[0]) and x.shape == (NL, B, 2, 11) for x in kept)
