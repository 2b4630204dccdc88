"""The softmax weights of attn_tree over 16-bit caches on the GPU: how many of their
bits enter P.V, whatever the output's type, against the formula in 64 bits.

Weights are held in two 16-bit pieces, so a weight is off by at most 2 u(t)^2 of
itself (u(t) = eps(t)/2), and over f16 by at most 2^-39 of its row's largest one, half
of f16's least step where the largest is 2^14 or more; the other terms are those of
test_tree_gpu.py, and the output's own rounding comes on top."""
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
        tol = tol + n_keys * 2.0 ** -39 * most * v_max
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


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D,H,Hk,B,T,n", [(64, 4, 1, 300, 2, 600), (128, 8, 2, 260, 5, 500), (256, 4, 2, 258, 9, 300), (128, 64, 8, 40, 20, 700)])
@pytest.mark.parametrize("less", [12.0, 22.3, 25.5, 30.0])
@pytest.mark.parametrize("sink", [0, 33, -1])
def test_long_tail_behind_one_large_weight(dev, dt, D, H, Hk, B, T, n, less, sink):
    """One key of value 0 that takes nearly all the weight, first, early or last, and
    many of 2^-less of it that make the result: enough sequences that none is cut."""
    t, x = DT[dt], 4.0
    g = torch.Generator(device=dev).manual_seed(int(less))
    k, v = torch.zeros(1, n + T, Hk * D, device=dev, dtype=t), (100 * torch.randn(1, n + T, Hk * D, device=dev, generator=g)).to(t)
    at = sink % n
    k[0, at, ::D], v[0, at] = x, 0
    q = torch.zeros(B, T, H, D, device=dev, dtype=t)
    q[..., 0] = x
    scale = less * np.log(2) / (x * x)
    see = np.tril(np.ones((T, T), bool))
    o, a, e = ref(q[0], k[0], v[0], see, n, T, np.arange(T) + n, 0, scale, D)
    for out_t in (t, torch.float32):
        out = A.attn_tree(q, k, v, None, i32([n] * B, dev), n + T, Hk, scale=scale, out_dtype=out_t)
        assert (out == out[0]).all()
        tol = bound(o, a, e, n + T, t, out_t, 1, v.double().abs().max())
        worst = ((out[0].double() - o).abs() / tol).max().item()
        assert worst <= 1, f"{out_t}: {worst:.3g} of the bound, {((out[0].double() - o).norm() / o.norm()).item():.2g} of the result"
