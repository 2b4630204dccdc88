"""The softmax weights of attn_tree over 16-bit caches on the GPU: how many of their
bits enter P.V, whatever the output's type, against the formula in 64 bits.

Weights are held in two 16-bit pieces, so a weight is off by at most 2 u(t)^2 of
itself (u(t) = eps(t)/2), and over f16 by at most 2^-25 of its row's largest one, half
of f16's least step; the other terms are those of test_tree_gpu.py, and the output's
own rounding comes on top."""
import numpy as np
import pytest
import torch

from test_tree_gpu import DT, attend, bits, i32, make, ref, trees, unit
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu


def bound(o, a, e, n_keys, t, out_t, most, v_max):
    """Of |out - o|, element by element; most: the rows' largest weights."""
    D = o.shape[-1]
    es = 2 * ((D + 4) * 2.0 ** -24 * e + 8 * 2.0 ** -24) + n_keys * 2.0 ** -24
    tol = unit(out_t) * o.abs() + (2 * unit(t) ** 2 + es) * a
    if t == torch.float16:
        tol = tol + n_keys * 2.0 ** -25 * most * v_max
    least = 2.0 ** -25 if out_t == torch.float16 else 0.0  # half of f16's least step, near 0
    return 1.01 * tol + least + 1e-30


@pytest.mark.parametrize("dt,H,Hk,D,lens,T,page,window", [
    ("f16", 8, 4, 64, [36], 1, 0, 0), ("bf16", 4, 4, 128, [9, 63], 17, 32, 0), ("f16", 12, 2, 128, [4095], 26, 0, 0),
    ("bf16", 40, 8, 128, [90, 700, 31, 1500], 7, 32, 0), ("f16", 8, 4, 256, [1500, 900], 33, 128, 1024),
    ("bf16", 8, 4, 256, [700], 5, 0, 0), ("bf16", 32, 4, 128, [9000, 5000], 64, 64, 0), ("f16", 64, 16, 64, [1111, 222], 50, 64, 0),
    ("bf16", 12, 2, 64, [30] * 40, 7, 32, 0), ("f16", 64, 16, 256, [300] * 4, 33, 64, 0),
    # workgroups of the widths and cuts that the calls of test_tree_gpu.py do not reach
    ("bf16", 64, 16, 128, [700] * 24, 20, 64, 0), ("f16", 8, 4, 256, [300] * 64, 64, 0, 0), ("bf16", 32, 8, 256, [12000], 20, 0, 0),
    ("f16", 12, 2, 64, [40] * 200, 3, 32, 0), ("bf16", 12, 2, 64, [40] * 200, 7, 0, 0), ("f16", 64, 16, 64, [700] * 24, 20, 32, 0),
    ("bf16", 64, 16, 64, [12000], 33, 64, 0)])
def test_output_is_rounded_once(dev, dt, H, Hk, D, lens, T, page, window):
    """An output in the cache's type is the f32 output rounded, nothing less exact:
    both within the bound of two pieces of every weight."""
    t, rng, B = DT[dt], np.random.default_rng(D + T), len(lens)
    n_pos = max(lens) + T
    see, depth, mask = trees(rng, B, T, "tree")
    pos = np.array(lens)[:, None] + depth
    caches, rows, table = make(rng, dev, lens, [T] * B, T, Hk, D, t, page, 0, n_pos)
    q = (2 * torch.randn(B, T, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(T))).to(t)
    outs = [attend(q, caches, table, mask.to(dev), i32(lens, dev), n_pos, Hk, None, i32(pos, dev), window, out_dtype=o)
            for o in (t, torch.float32)]
    assert outs[0].dtype == t and torch.equal(outs[0], outs[1].to(t))
    for b in range(0, B, max(B // 4, 1)):
        o, a, e = ref(q[b], rows[0][b], rows[1][b], see[b], lens[b], T, pos[b], window, D ** -0.5, D)
        for out in outs:
            tol = bound(o, a, e, lens[b] + T, t, out.dtype, 1, rows[1][b].double().abs().max())
            worst = ((out[b].double() - o).abs() / tol).max().item()
            assert worst <= 1, f"{out.dtype} b={b}: {worst:.3g} of the bound"
