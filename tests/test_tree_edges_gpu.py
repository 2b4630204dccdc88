"""Calls of the drafted trees and the page tables at their edges, on the GPU."""
import math

import numpy as np
import pytest
import torch

from test_tree_gpu import DT, NAN, attend, bits, i32, make
from ullm_amd import _lib as L
from ullm_amd import attention as A

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


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", ["side by side", "layers in a row", "narrow"])
@pytest.mark.parametrize("P,kvd", [(32, 64), (64, 8), (2, 2056), (128, 328)])
def test_page_copies_of_views_of_wider_rows(dev, dt, form, P, kvd):
    """Pools that are columns of wider rows: a fork copies those columns of the filled
    rows, and whatever else the rows hold stays as it was."""
    t, NL, n_pages = DT[dt], 3, 9
    g = torch.Generator(device=dev).manual_seed(P)
    if form == "layers in a row":
        both = [torch.randn(n_pages, P, NL + 1, kvd, device=dev, generator=g).to(t) for _ in "kv"]
        views = [x.permute(2, 0, 1, 3)[:NL] for x in both]
        of = lambda xs: [x.permute(2, 0, 1, 3)[:NL] for x in xs]  # noqa: E731
    elif form == "side by side":
        both = [torch.randn(NL, n_pages, P, 2 * kvd, device=dev, generator=g).to(t)]
        of = lambda xs: [xs[0][..., :kvd], xs[0][..., kvd:]]  # noqa: E731
    else:
        both = [torch.randn(NL, n_pages, P, kvd + 24, device=dev, generator=g).to(t) for _ in "kv"]
        of = lambda xs: [x[..., 8:8 + kvd] for x in xs]  # noqa: E731
    views, want = of(both), [x.clone() for x in both]
    part = P // 2 + 1 if P > 2 else 1
    lens = [P + part, part]
    table, new, info = A.kv_pages_update(*views, i32([[6, 3], [8, -1]], dev), i32(lens, dev), i32([0, 0, 1, 1, 0], dev),
                                         i32([lens[0] + 1, 2 * P, P, P, lens[0]], dev))
    assert table.tolist() == [[6, 3], [6, 0], [8, -1], [1, -1], [6, 2]] and info.tolist() == [3, 3, 0]
    assert new.tolist() == [lens[0], lens[0], part, part, lens[0]]
    for x, o in zip(of(want), of([x.clone() for x in both])):
        for src, to in ((3, 0), (8, 1), (3, 2)):
            x[:, to, :part] = o[:, src, :part]
    for x, w in zip(both, want):
        assert torch.equal(x, w)
    if form != "narrow":  # one layer
        before = [x.clone() for x in both]
        A.kv_pages_update(*(x[1] for x in views), i32([[6, 3]], dev), i32([P + part], dev), i32([0, 0], dev), i32([2 * P] * 2, dev))
        for x, o in zip(of(before), of([x.clone() for x in before])):
            x[1, 0, :part] = o[1, 3, :part]
        for x, w in zip(both, before):
            assert torch.equal(x, w)


def test_pools_whose_rows_overlap_are_refused(dev):
    k = torch.zeros(1 << 14, device=dev, dtype=torch.float16)
    for sizes, strides in (((4, 32, 64), (32 * 32, 32, 1)), ((2, 4, 32, 8), (0, 32 * 8, 8, 1)), ((2, 4, 32, 8), (4, 32 * 8, 8, 1))):
        v = k.as_strided(sizes, strides)
        with pytest.raises(L.UllmHipError):
            A.kv_pages_update(v, v, i32([[0]], dev), i32([5], dev), i32([0, 0], dev), i32([6, 6], dev))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 16])
def test_strides_left_out_are_the_caches_own(dev, dt, pad):
    """Caches [B, n_ctx, kv_dim], whole or columns of wider rows, without strides: every
    sequence's rows go to its own, and are read from there."""
    t, H, Hk, D, T, n_ctx, lens = DT[dt], 8, 2, 64, 5, 90, [60, 3, 85]
    B = len(lens)
    g = torch.Generator(device=dev).manual_seed(pad)
    full = [torch.randn(B, n_ctx, Hk * D + pad, device=dev, generator=g).to(t) for _ in "kv"]
    want = [x.clone() for x in full]
    q, k, v = (torch.randn(B, T, n * D, device=dev, generator=g) for n in (H, Hk, Hk))
    cs, ln = A.rope_table(n_ctx, D, 1e4), i32(lens, dev)
    more = dict(n_head=H, n_kv_head=Hk, head_dim=D, q_dtype=t)
    qs = [A.qkv_append_tree(q[b:b + 1], k[b:b + 1], v[b:b + 1], want[0][b], want[1][b], cs, ln[b:b + 1],
                            kv_stride=Hk * D + pad, **more) for b in range(B)]
    views = [x[..., :Hk * D] for x in full]
    got = A.qkv_append_tree(q, k, v, *views, cs, ln, **more)
    assert torch.equal(got, torch.cat(qs))
    for x, w in zip(full, want):
        assert torch.equal(x, w)
    out = A.attn_tree(got.view(B, T, H, D), *views, None, ln, n_ctx, Hk)
    assert torch.equal(out, attend(got.view(B, T, H, D), full, None, None, ln, n_ctx, Hk, None, None, 0))


def test_one_cache_for_all_sequences_is_read_but_not_written(dev):
    t, H, Hk, D, T, B = torch.float16, 4, 2, 64, 3, 2
    k = torch.zeros(50, Hk * D, device=dev, dtype=t)
    ln, cs = i32([20, 30], dev), A.rope_table(50, D, 1e4)
    x = [torch.ones(B, T, n * D, device=dev) for n in (H, Hk, Hk)]
    more = dict(n_head=H, n_kv_head=Hk, head_dim=D, q_dtype=t)
    for cache, strides in ((k, {}), (k, dict(seq_stride=0)), (k.expand(B, 50, Hk * D), {}), (k[None], {})):
        with pytest.raises(L.UllmHipError) as e:
            A.qkv_append_tree(*x, cache, cache.clone(), cs, ln, **strides, **more)
        assert e.value.code == L.E_INVALID
        q = torch.ones(B, T, H, D, device=dev, dtype=t)
        assert A.attn_tree(q, cache, cache, None, ln, 40, Hk, **strides).shape == q.shape
    assert not k.any()


@pytest.mark.parametrize("strides", [
    dict(seq_stride=1 << 62), dict(seq_stride=(1 << 63) - 8), dict(kv_stride=1 << 62), dict(kv_stride=(1 << 63) - 8),
    dict(kv_stride=1 << 61, seq_stride=1 << 62), dict(kv_stride=-128), dict(seq_stride=-8), dict(kv_stride=129 * 128)])
def test_strides_past_the_caches_are_refused(dev, strides):
    """Also those whose products pass 64 bits."""
    t, H, Hk, D, T, B = torch.float16, 4, 2, 64, 3, 5
    k = torch.zeros(B, 9, Hk * D, device=dev, dtype=t)
    ln, cs = i32([2] * B, dev), A.rope_table(50, D, 1e4)
    x = [torch.ones(B, T, n * D, device=dev) for n in (H, Hk, Hk)]
    for n in (5, 9):
        for call in (lambda: A.qkv_append_tree(*x, k, k.clone(), cs, ln, n_head=H, n_kv_head=Hk, head_dim=D, q_dtype=t, n_ctx=n, **strides),
                     lambda: A.attn_tree(torch.ones(B, T, H, D, device=dev, dtype=t), k, k, None, ln, n, Hk, **strides)):
            with pytest.raises(L.UllmHipError) as e:
                call()
            assert e.value.code == L.E_INVALID
    assert not k.any()


@pytest.mark.parametrize("page", [0, 32])
@pytest.mark.parametrize("NL", [1, 5])
def test_accept_of_a_cache_that_is_both_k_and_v(dev, page, NL):
    """One tensor given as K and V moves once: twice would undo a path that turns round."""
    T, n, kvd = 40, 30, 512
    x = torch.randn(NL, 96, kvd, device=dev, generator=torch.Generator(device=dev).manual_seed(NL)).bfloat16()
    want, path = x.clone(), np.random.default_rng(NL).permutation(T)
    want[:, n:n + T] = x[:, torch.from_numpy(n + path).to(dev)]
    count, ln, p = i32([T], dev), i32([n], dev), i32(path[None], dev)
    if page:
        k = x.view(NL, 3, page, kvd)
        new = A.kv_accept_paged(k, k, i32([[0, 1, 2]], dev), p, count, ln)
    else:
        new = A.kv_accept(x, x, p, count, ln)
    assert new.tolist() == [n + T] and torch.equal(x, want)


def test_a_cache_of_heads_with_as_many_positions_as_sequences(dev):
    """[n_ctx, n_kv_head, head_dim] is one cache, also where n_ctx is the batch."""
    t, H, Hk, D, T, B = torch.float16, 4, 2, 64, 2, 40
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn(B, Hk, D, device=dev, generator=g).to(t) for _ in "kv")
    q, ln = torch.randn(B, T, H, D, device=dev, generator=g).to(t), i32([i % 38 for i in range(B)], dev)
    out = A.attn_tree(q, k, v, None, ln, B, Hk)
    assert torch.equal(out, A.attn_tree(q, k.view(B, -1), v.view(B, -1), None, ln, B, Hk, kv_stride=Hk * D, seq_stride=0))
