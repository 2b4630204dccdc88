"""Calls of the drafted trees and the page tables at their edges, on the GPU."""
import math

import numpy as np
import pytest
import torch

from test_tree_gpu import NAN, attend, bits, i32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,H,Hk,B,T", [(64, 64, 16, 24, 20), (64, 128, 16, 8, 64), (128, 32, 8, 16, 60), (128, 8, 4, 64, 33)])
@pytest.mark.parametrize("n", [0, 5, 30, 95])
@pytest.mark.parametrize("page", [0, 32])
def test_infinities_of_a_first_step_over_f32(dev, D, H, Hk, B, T, n, page):
    """More than 64 rows of a kv head over f32, and so few keys that the first step of a
    workgroup holds drafts: a value that is not finite reaches each node that sees it, and
    no other, whichever wave fetched it."""
    rng = np.random.default_rng(n + D)
    see = rng.random((B, T, T)) < 0.3
    at, to, what = [0, T // 2, T - 1], [3, 7, T - 2], [math.inf, NAN, -math.inf]
    see[:, :, at] = False
    for j, i in zip(at, to):
        see[:, i, j] = True
    caches, _, table = make(rng, dev, [n] * B, [T] * B, T, Hk, D, torch.float32, page, 0, n + T)
    q = torch.randn(B, T, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(D))
    args = (table, bits(see).to(dev), i32([n] * B, dev), n + T, Hk, None, i32(np.tile(n + np.arange(T), (B, 1)), dev), 0)

    def put(j, value, cols):
        t = n + j
        for b in range(B):
            caches[1][(table[b, t // page], t % page) if page else (b, t)][cols] = value

    for j in at:
        put(j, 0.0, slice(None))
    want = attend(q, caches, *args)
    for j, value in zip(at, what):
        put(j, value, slice(j % 2, None, 2))
    others = [i for i in range(T) if i not in to]
    for _ in range(20):
        out = attend(q, caches, *args)
        assert torch.equal(out[:, others], want[:, others])
        for j, i, value in zip(at, to, what):
            got = out[:, i, :, j % 2::2]
            assert got.isnan().all() if math.isnan(value) else (got == value).all(), (n, i)
            assert torch.isfinite(out[:, i, :, 1 - j % 2::2]).all()
