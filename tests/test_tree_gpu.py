"""Drafted trees over a cache on the GPU: attn_tree(_paged), qkv_append_tree(_paged)
and GpuAttention.forward_tree, against the same formulas in 64 bits.

The reference decodes one token at a time (crates/ullm-model/src/lib.rs:911-938,
windowed :1180-1208); a node of a tree attends what a token at its position
would, with the tokens of its own path behind the sequence.

Tolerances of the attention, element by element, from the roundings that the
entry point documents (u(t) = eps(t)/2):
  out's type                u(out) |o|
  weights in P.V            u(P) A, A = sum_t p_t |v_t|: P in the cache's type where
                            out has it, 2 u(t)^2 in twice its bits for an f32 out
  scores, exp and sums, in f32: the score of a key is off by at most
                            (D + 4) 2^-24 scale sum_d |q_d k_d|, which moves its
                            weight by that much relative, the normaliser too; n
                            terms are summed
No input is retried and every tolerance is this bound."""
import math

import numpy as np
import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NAN = float("nan")


def unit(t):
    return torch.finfo(t).eps / 2


def bits(see):
    """int64 mask words of a bool [B, T, T]."""
    B, T, _ = see.shape
    W = -(-T // 64)
    m = np.zeros((B, T, W), np.uint64)
    for j in range(T):
        m[:, :, j // 64] |= see[:, :, j].astype(np.uint64) << np.uint64(j % 64)
    return torch.from_numpy(m.view(np.int64))


def trees(rng, B, T, kind):
    """(see [B, T, T] bool, depth [B, T], mask int64 or None)."""
    parents = np.full((B, T), -1, np.int64)
    for b in range(B):
        for i in range(1, T):
            parents[b, i] = i - 1 if rng.random() < 0.5 else rng.integers(-1, i)
    if kind == "chain":
        return np.tril(np.ones((B, T, T), bool)), np.tile(np.arange(T), (B, 1)), None
    mask, depth = A.tree_masks(parents)
    see = (mask.numpy().view(np.uint64)[:, :, np.arange(T) // 64] >> np.arange(T, dtype=np.uint64) % np.uint64(64)) & np.uint64(1)
    see = see.astype(bool)
    if kind == "random":  # any bits, some rows without one
        see = rng.random((B, T, T)) < 0.3
        see[:, ::3] = False
    if kind == "none":
        see[:] = False
    return see, depth.numpy(), bits(see)


def ref(q, k, v, see, n, m, pos, window, scale, D):
    """One sequence: q [T,H,D], k/v [n+m, Hk*D] in any type; o, A and the bound of
    the score errors, all in 64 bits; rows that see nothing are 0."""
    q, k, v = q.double(), k.double(), v.double()
    T, H = q.shape[:2]
    Hk = k.shape[1] // D
    vis = torch.ones(m, n + m, dtype=torch.bool)
    vis[:, n:] = torch.from_numpy(see[:m, :m])
    if window:
        key = torch.cat((torch.arange(n), torch.from_numpy(pos[:m])))
        vis &= key[None] > torch.from_numpy(pos[:m])[:, None] - window
    vis = vis.to(q.device)
    o, a, e = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(T, H, 1, dtype=torch.float64, device=q.device)
    for h in range(H if m else 0):
        j = h // (H // Hk)
        kj, vj = k[:, j * D:(j + 1) * D], v[:, j * D:(j + 1) * D]
        s = (q[:m, h] @ kj.t().contiguous() * scale).masked_fill(~vis, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1), 0.0)
        # what a key holds reaches only the nodes that see it
        bad = ~torch.isfinite(vj).all(1)
        o[:m, h] = p[:, ~bad] @ vj[~bad]
        a[:m, h] = p[:, ~bad] @ vj[~bad].abs()
        for t in bad.nonzero()[:, 0].tolist():
            rows = vis[:, t]
            o[:m, h][rows] += p[rows, t, None] * vj[t]
            a[:m, h][rows] += p[rows, t, None] * vj[t].abs()
        mag = (q[:m, h].abs() @ kj.nan_to_num(0, 0, 0).abs().t().contiguous() * abs(scale)).masked_fill(~vis, 0)
        e[:m, h, 0] = mag.amax(1)
    return o, a, e


def check(out, o, a, e, n_keys, t, what):
    D, f32 = o.shape[-1], torch.float32
    up = 0.0 if t == f32 else unit(t) if out.dtype == t else 2 * unit(t) ** 2
    es = 2 * ((D + 4) * 2.0 ** -24 * e + 8 * 2.0 ** -24) + n_keys * 2.0 ** -24
    tol = 1.01 * (unit(out.dtype) * o.abs() + (up + es) * a) + 1e-30
    got = out.double()
    fin = torch.isfinite(o)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: finite where it is not, or not where it is"
    worst = ((got - o).abs() / tol)[fin]
    assert worst.numel() == 0 or worst.max().item() <= 1, f"{what}: {worst.max().item():.3g} of the bound"
    if t == f32 and fin.all() and o.norm() > 0:  # roundings of either sign: sqrt(n) 2^-24 and less
        rel = ((got - o).norm() / o.norm()).item()
        assert rel <= 1e-5, f"{what}: rel {rel:.2e}"


def make(rng, dev, lens, nodes, T, Hk, D, t, page, pad, n_pos):
    """(caches as attn_tree takes them, rows of each sequence): unused rows and
    pages hold NaN."""
    g = torch.Generator(device=dev).manual_seed(int(rng.integers(1 << 30)))
    B, kvs = len(lens), Hk * D + pad
    rows = [[torch.randn(n + m, Hk * D, device=dev, generator=g).to(t) for n, m in zip(lens, nodes)] for _ in "kv"]
    if page:
        need = [-(-(n + m) // page) for n, m in zip(lens, nodes)]
        n_pages = sum(need) + 3
        perm, at = rng.permutation(n_pages), 0
        table = np.full((B, -(-n_pos // page) + 1), -1, np.int32)
        table[:, -1] = n_pages + 5
        caches = [torch.full((n_pages, page, kvs), NAN, device=dev, dtype=t) for _ in "kv"]
        for b in range(B):
            for i in range(need[b]):
                pg = int(perm[at])
                at += 1
                table[b, i] = pg
                for c, r in zip(caches, rows):
                    part = r[b][i * page:(i + 1) * page]
                    c[pg, :len(part), :Hk * D] = part
        return caches, rows, torch.from_numpy(table).to(dev)
    caches = [torch.full((B, n_pos, kvs), NAN, device=dev, dtype=t) for _ in "kv"]
    for b in range(B):
        for c, r in zip(caches, rows):
            c[b, :len(r[b]), :Hk * D] = r[b]
    return caches, rows, None


def attend(q, caches, table, mask, lens, n_pos, Hk, n, pos, window, **more):
    if table is not None:
        return A.attn_tree_paged(q, *caches, table, mask, lens, n_pos, Hk, n_nodes=n, positions=pos, window=window, **more)
    return A.attn_tree(q, *caches, mask, lens, n_pos, Hk, n_nodes=n, positions=pos, window=window,
                       kv_stride=caches[0].stride(1), seq_stride=caches[0].stride(0), **more)


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


CASES = [
    # (type, out, H, Hk, D, lens, nodes, T, page, window, mask, pad)
    ("f32", "f32", 8, 2, 64, [0], [1], 1, 0, 0, "tree", 0),
    ("f16", "f16", 8, 2, 128, [0, 1, 31, 32], [1, 2, 3, 3], 3, 32, 0, "tree", 0),
    ("bf16", "bf16", 8, 2, 128, [33, 0, 5, 64], [5, 0, 7, 1], 7, 0, 0, "chain", 8),
    ("bf16", "f32", 12, 2, 128, [1000, 63], [26, 11], 26, 64, 0, "tree", 0),
    ("f16", "f32", 14, 2, 64, [777, 1300, 2], [40, 64, 17], 64, 32, 0, "tree", 64),
    ("f32", "f32", 12, 2, 128, [500, 129], [33, 65], 65, 64, 0, "tree", 4),
    ("f16", "f16", 8, 4, 256, [300, 2000], [29, 33], 33, 128, 0, "tree", 16),
    ("f32", "f32", 8, 4, 256, [257], [19], 19, 0, 0, "tree", 0),
    ("bf16", "bf16", 40, 8, 128, [90, 700, 31], [7, 3, 7], 7, 32, 0, "tree", 0),
    ("bf16", "bf16", 5, 5, 64, [4000], [100], 100, 256, 0, "tree", 0),
    ("f16", "f16", 32, 1, 64, [129, 4100], [9, 70], 70, 64, 0, "random", 0),
    ("bf16", "bf16", 32, 4, 128, [0, 100, 3], [64, 60, 1], 64, 32, 0, "random", 0),
    ("f32", "f32", 6, 3, 64, [0, 40], [12, 30], 30, 32, 0, "random", 0),
    ("f16", "f16", 8, 4, 128, [0, 0], [20, 7], 20, 32, 0, "none", 0),
    ("bf16", "bf16", 8, 4, 128, [2000, 30, 1030], [33, 33, 10], 33, 64, 37, "tree", 0),
    ("f16", "f16", 8, 4, 256, [1500, 900], [20, 33], 33, 0, 1024, "tree", 0),
    ("f32", "f32", 8, 2, 64, [700, 10], [50, 50], 50, 32, 3, "tree", 0),
    ("bf16", "f32", 4, 2, 128, [900, 64], [64, 64], 64, 64, 1, "tree", 0),
    ("f16", "f32", 4, 4, 64, [300], [20], 20, 0, 11, "chain", 0),
    ("bf16", "bf16", 32, 4, 128, [9000, 20000], [64, 64], 64, 64, 0, "tree", 0),
    ("f16", "f16", 16, 2, 128, [1200], [300], 300, 64, 0, "tree", 0),
    ("f32", "f32", 4, 1, 128, [3000], [130], 130, 128, 0, "random", 0),
    ("f16", "f16", 3, 1, 64, [50], [1024], 1024, 32, 0, "tree", 0),
    # enough keys and heads for workgroups of 65 rows and more, of each type and width
    ("f32", "f32", 64, 32, 64, [1100], [60], 60, 64, 0, "tree", 0),
    ("f32", "f32", 32, 16, 128, [1500, 700], [50, 41], 50, 32, 0, "random", 4),
    ("f32", "f32", 64, 16, 64, [1300, 40], [64, 50], 64, 32, 21, "tree", 0),
    ("f32", "f32", 32, 8, 256, [900, 300, 5], [30, 21, 30], 30, 64, 0, "tree", 0),
    ("bf16", "f32", 64, 16, 128, [1500, 800], [64, 33], 64, 64, 0, "tree", 0),
    ("f16", "f32", 32, 16, 256, [700, 801], [60, 59], 60, 0, 300, "tree", 8),
    ("bf16", "bf16", 64, 16, 64, [1111, 2222], [50, 64], 64, 32, 0, "random", 0),
    # and of 17 to 32 rows, whose waves share the keys of a tile over f32
    ("f32", "f32", 64, 32, 64, [1100, 1000, 900], [16, 15, 9], 16, 32, 0, "tree", 0),
    ("f32", "f32", 64, 32, 128, [1100, 950], [16, 10], 16, 0, 400, "tree", 0),
    ("f32", "f32", 32, 16, 256, [1000, 333], [15, 16], 16, 64, 7, "tree", 4),
    ("f16", "f16", 64, 32, 128, [1500, 1200], [16, 10], 16, 32, 0, "random", 0),
    # more sequences than are looked at by a wave at once, of one workgroup each and cut
    ("bf16", "bf16", 4, 2, 64, [(7 * i) % 201 for i in range(300)], [i % 4 for i in range(300)], 3, 32, 0, "tree", 0),
    ("f16", "f16", 4, 1, 64, [6000 if i % 29 == 3 else 37 * i % 90 for i in range(130)], [5 - i % 3 for i in range(130)], 5, 32, 0, "tree", 0),
    ("bf16", "bf16", 4, 2, 128, [5000 if i == 69 else 0 for i in range(70)], [1] * 70, 2, 64, 64, "chain", 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attn_tree(dev, case):
    dt, odt, H, Hk, D, lens, nodes, T, page, window, kind, pad = CASES[case]
    print(f"[tree] {CASES[case]}", flush=True)
    t, rng, B = DT[dt], np.random.default_rng(case + 1), len(lens)
    n_pos = max(n + m for n, m in zip(lens, nodes)) + case % 3
    see, depth, mask = trees(rng, B, T, kind)
    pos = np.array(lens)[:, None] + depth
    caches, rows, table = make(rng, dev, lens, nodes, T, Hk, D, t, page, pad, n_pos)
    g = torch.Generator(device=dev).manual_seed(case)
    q = (2 * torch.randn(B, T, H, D, device=dev, generator=g)).to(t)
    out = attend(q, caches, table, None if mask is None else mask.to(dev), i32(lens, dev), n_pos, Hk, i32(nodes, dev),
                 i32(pos, dev), window, out_dtype=DT[odt])
    torch.cuda.synchronize()
    assert out.dtype == DT[odt] and out.shape == q.shape
    for b in range(B):
        r = ref(q[b], rows[0][b], rows[1][b], see[b], lens[b], nodes[b], pos[b], window, 1 / math.sqrt(D), D)
        check(out[b], *r, lens[b] + nodes[b], t, f"case {case} b={b}")
        assert not out[b, nodes[b]:].any()


SHAPES = [
    # (type, out, H, Hk, D, B, T, L): a small call for each shape of a workgroup, uncut and in parts
    ("bf16", "f32", 12, 2, 128, 1, 1, 40), ("f16", "f32", 12, 2, 128, 1, 1, 700), ("bf16", "bf16", 12, 2, 128, 200, 3, 40),
    ("f16", "f16", 16, 16, 128, 1, 20, 3000), ("bf16", "f32", 12, 2, 128, 200, 7, 40), ("f16", "f32", 16, 16, 128, 6, 33, 700),
    ("bf16", "bf16", 64, 16, 128, 24, 20, 40), ("f16", "f16", 64, 16, 128, 1, 20, 12000),
    ("bf16", "f32", 64, 16, 128, 16, 33, 300), ("f16", "f32", 64, 16, 128, 1, 33, 12000),
    ("bf16", "bf16", 12, 2, 256, 1, 1, 40), ("f16", "f16", 12, 2, 256, 1, 1, 300), ("bf16", "f32", 12, 2, 256, 200, 3, 40),
    ("f16", "f32", 16, 16, 256, 6, 20, 300), ("bf16", "bf16", 12, 2, 256, 200, 7, 40), ("f16", "f16", 16, 16, 256, 2, 33, 1500),
    ("bf16", "f32", 32, 8, 256, 24, 20, 300), ("f16", "f32", 8, 4, 256, 2, 33, 12000), ("bf16", "bf16", 12, 2, 64, 1, 1, 40),
    ("f16", "f16", 12, 2, 64, 1, 1, 700), ("bf16", "f32", 128, 16, 64, 16, 3, 40), ("f16", "f32", 12, 2, 64, 24, 3, 700),
    ("bf16", "bf16", 32, 4, 64, 3, 64, 40), ("f16", "f16", 128, 16, 64, 1, 7, 700), ("bf16", "f32", 64, 16, 64, 24, 20, 40),
    ("f16", "f32", 8, 4, 64, 4, 33, 12000), ("bf16", "bf16", 64, 16, 64, 16, 33, 300), ("f16", "f16", 12, 2, 64, 2, 33, 30000),
    ("f32", "f32", 12, 2, 128, 1, 1, 40), ("f32", "f32", 12, 2, 128, 1, 1, 300), ("f32", "f32", 12, 2, 128, 200, 3, 40),
    ("f32", "f32", 16, 16, 128, 6, 20, 300), ("f32", "f32", 12, 2, 128, 200, 7, 40), ("f32", "f32", 64, 8, 128, 1, 48, 700),
    ("f32", "f32", 8, 4, 128, 64, 33, 40), ("f32", "f32", 12, 2, 128, 1, 20, 12000), ("f32", "f32", 12, 2, 256, 1, 1, 40),
    ("f32", "f32", 12, 2, 256, 1, 1, 300), ("f32", "f32", 64, 8, 256, 24, 3, 40), ("f32", "f32", 32, 4, 256, 1, 33, 300),
    ("f32", "f32", 64, 8, 256, 24, 7, 40), ("f32", "f32", 16, 16, 256, 1, 33, 1500), ("f32", "f32", 64, 16, 256, 8, 33, 40),
    ("f32", "f32", 8, 4, 256, 16, 33, 700), ("f32", "f32", 12, 2, 64, 1, 1, 40), ("f32", "f32", 12, 2, 64, 1, 1, 300),
    ("f32", "f32", 12, 2, 64, 200, 3, 40), ("f32", "f32", 16, 16, 64, 1, 20, 3000), ("f32", "f32", 12, 2, 64, 200, 7, 40),
    ("f32", "f32", 64, 8, 64, 1, 48, 700), ("f32", "f32", 64, 16, 64, 24, 20, 40), ("f32", "f32", 128, 16, 64, 1, 48, 700),
    ("f32", "f32", 128, 16, 64, 8, 64, 40), ("f32", "f32", 64, 8, 64, 1, 64, 1500),
]


@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_every_shape(dev, case):
    dt, odt, H, Hk, D, B, T, L = SHAPES[case]
    print(f"[tree] {SHAPES[case]}", flush=True)
    t, rng = DT[dt], np.random.default_rng(case + 100)
    lens = [L - (i * 11) % (L // 2) for i in range(B)]
    nodes = [T - i % min(T, 3) for i in range(B)]
    see, depth, _ = trees(rng, B, T, "random")
    pos = np.array(lens)[:, None] + depth
    page = (0, 32, 64)[case % 3]
    caches, rows, table = make(rng, dev, lens, nodes, T, Hk, D, t, page, 0, L + T)
    if T > 1:  # a key that no node of the first sequence sees
        see[0, :, 1] = False
        at = lens[0] + 1
        at = (table[0, at // page], at % page) if page else (0, at)
        for r, c, bad in ((rows[0], caches[0], NAN), (rows[1], caches[1], math.inf)):
            r[0][lens[0] + 1] = bad
            c[at] = bad
    g = torch.Generator(device=dev).manual_seed(case)
    q = (2 * torch.randn(B, T, H, D, device=dev, generator=g)).to(t)
    out = attend(q, caches, table, bits(see).to(dev), i32(lens, dev), L + T, Hk, i32(nodes, dev), i32(pos, dev), 0, out_dtype=DT[odt])
    for b in range(0, B, max(B // 6, 1)):
        r = ref(q[b], rows[0][b], rows[1][b], see[b], lens[b], nodes[b], pos[b], 0, 1 / math.sqrt(D), D)
        check(out[b], *r, lens[b] + nodes[b], t, f"case {case} b={b}")
        assert not out[b, nodes[b]:].any()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [0, 32])
def test_unseen_keys_reach_no_node(dev, dt, D, page):
    """NaN, infinities and the type's lowest value in the K and V rows of nodes
    that others do not see, and before windows: only who sees them has them."""
    t, rng, H, Hk, lens, T = DT[dt], np.random.default_rng(D), 8, 4, [70, 0, 40], 21
    B, n_pos = len(lens), 100
    see = np.zeros((B, T, T), bool)
    see[:, np.arange(T), np.arange(T)] = True       # each sees itself,
    see[:, 1::2, 0] = True                          # the odd ones the first
    see[:, 6, 6] = False                            # and one sees nothing of the draft
    pos = np.array(lens)[:, None] + np.tile(np.arange(T), (B, 1))
    for window in (0, 9):
        nodes = [T, T, T - 3]
        caches, rows, table = make(rng, dev, lens, nodes, T, Hk, D, t, page, 0, n_pos)
        low = torch.finfo(t).min
        for b in range(B):
            for r, c, bad in ((0, 2, NAN), (1, 4, NAN), (1, 5, math.inf), (1, 8, -math.inf), (0, 10, low), (1, 11, low),
                              (1, 13, math.inf), (1, 13, NAN)):
                i = lens[b] + c
                cols = slice(0, D) if c == 4 else slice(3, None, 5)
                rows[r][b][i, cols] = bad
                if page:
                    caches[r][table[b, i // page], i % page, :Hk * D] = rows[r][b][i]
                else:
                    caches[r][b, i, :Hk * D] = rows[r][b][i]
            if window and lens[b]:  # before every window
                rows[1][b][0] = NAN
                caches[1][(table[b, 0], 0) if page else (b, 0)] = NAN
        q = torch.randn(B, T, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).to(t)
        out = attend(q, caches, table, bits(see).to(dev), i32(lens, dev), n_pos, Hk, i32(nodes, dev), i32(pos, dev), window)
        for b in range(B):
            o, a, e = ref(q[b], rows[0][b], rows[1][b], see[b], lens[b], nodes[b], pos[b], window, 1 / math.sqrt(D), D)
            clean = [i for i in range(nodes[b]) if i not in (2, 4, 5, 8, 10, 11, 13)]
            check(out[b, clean], o[clean], a[clean], e[clean], lens[b] + T, t, f"window {window} b={b}")
            assert out[b, 2].isnan().all()           # a NaN score
            assert out[b, 4, :H // Hk].isnan().all()  # a NaN value
            assert not torch.isfinite(out[b, 5]).all() and torch.isfinite(out[b, 5]).any()


@pytest.mark.parametrize("dt,odt,D,T,n", [
    ("f32", "f32", 64, 60, 1000), ("f32", "f32", 128, 60, 1000), ("f32", "f32", 256, 60, 1000), ("bf16", "bf16", 128, 60, 1000),
    ("f16", "f32", 64, 60, 1000), ("f16", "f16", 256, 60, 1000), ("bf16", "f32", 256, 60, 1000),
    ("f32", "f32", 64, 45, 3200), ("f32", "f32", 64, 16, 3200), ("f32", "f32", 128, 16, 1600), ("f32", "f32", 256, 16, 1000)])
def test_unseen_keys_of_wide_trees(dev, dt, odt, D, T, n):
    """The same with workgroups of 17 rows and more, whose waves share their tiles,
    and with keys of a cut sequence: every node that does not see them is as if
    they were zeros, every other is not finite."""
    t, rng, H, Hk, last = DT[dt], np.random.default_rng(D + 1), 64, 32, T - 3
    see, depth, _ = trees(rng, 1, T, "random")
    see[0, :, 7] = see[0, :, last] = False
    see[0, 5, 7] = see[0, 12, last] = True
    pos = n + depth
    caches, rows, _ = make(rng, dev, [n], [T], T, Hk, D, t, 0, 0, n + T)
    q = torch.randn(1, T, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).to(t)
    args = (None, bits(see).to(dev), i32([n], dev), n + T, Hk, None, i32(pos, dev), 0)
    for i in (7, last):
        for c in caches:
            c[0, n + i] = 0
    want = attend(q, caches, *args, out_dtype=DT[odt])
    caches[0][0, n + 7], caches[1][0, n + 7] = NAN, math.inf
    caches[1][0, n + last, 1::2] = NAN
    caches[1][0, n + last, ::2] = -math.inf
    out = attend(q, caches, *args, out_dtype=DT[odt])
    others = [i for i in range(T) if i not in (5, 12)]
    assert torch.equal(out[0, others], want[0, others])
    assert not torch.isfinite(out[0, [5, 12]]).any()


@pytest.mark.parametrize("dt,H,Hk,D,T", [("f32", 32, 16, 128, 50), ("f32", 4, 2, 64, 5), ("f16", 8, 2, 128, 20), ("bf16", 4, 4, 256, 40)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3])
def test_any_scale(dev, dt, H, Hk, D, T, scale):
    t, n = DT[dt], 1200
    g = torch.Generator(device=dev).manual_seed(8)
    k, v = (torch.randn(1, n + T, Hk * D, device=dev, generator=g).to(t) for _ in "kv")
    q = torch.randn(1, T, H, D, device=dev, generator=g).to(t)
    out = A.attn_tree(q, k, v, None, i32([n], dev), n + T, Hk, scale=scale)
    o, a, e = ref(q[0], k[0], v[0], np.tril(np.ones((T, T), bool)), n, T, np.arange(T) + n, 0, scale, D)
    check(out[0], o, a, e, n + T, t, "scale")


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_pages_outside_the_pool_read_as_zeros(dev, dt):
    t, H, Hk, D, P, T = DT[dt], 4, 2, 64, 32, 5
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn(4, P, Hk * D, device=dev, generator=g).to(t) for _ in "kv")
    q = torch.randn(1, T, H, D, device=dev, generator=g).to(t)
    bad = i32([[2, -1, 4, 1 << 30]], dev)  # max_len of 4 pages, a pool of 4
    zero = torch.zeros(P, Hk * D, device=dev, dtype=t)
    lens, n_pos = i32([120], dev), 128
    out = A.attn_tree_paged(q, k, v, bad, None, lens, n_pos, Hk)
    kk, vv = (torch.cat((x[2], zero, zero, zero))[None].contiguous() for x in (k, v))
    want = A.attn_tree(q, kk, vv, None, lens, n_pos, Hk)
    assert torch.equal(out, want)
    # a length and node counts that the host's bounds do not allow stay inside them
    out = A.attn_tree_paged(q, k, v, bad, None, i32([1 << 30], dev), n_pos, Hk, n_nodes=i32([1 << 30], dev))
    assert torch.isfinite(out).all()
    out = A.attn_tree_paged(q, k, v, bad, None, i32([-5], dev), n_pos, Hk, n_nodes=i32([-7], dev))
    assert not out.any()


@pytest.mark.parametrize("dt,page", [("bf16", 64), ("f16", 0), ("f32", 32)])
def test_offsets_past_32_bits(dev, dt, page):
    """Pages and sequences that begin beyond 4 GiB of their pool."""
    t, H, Hk, D, T = DT[dt], 4, 2, 128, 9
    kvs, es = Hk * D, torch.finfo(DT[dt]).bits // 8
    rng = np.random.default_rng(5)
    rows = [torch.randn(300 + T, kvs, device=dev, generator=torch.Generator(device=dev).manual_seed(7 + i)).to(t) for i in range(2)]
    q = torch.randn(2, T, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(9)).to(t)
    lens, n = [300, 17], 300 + T
    far = ((1 << 32) + (1 << 28)) // (es * kvs)  # rows
    if page:
        n_pages = far // page
        k, v = (torch.empty(n_pages, page, kvs, device=dev, dtype=t) for _ in "kv")
        table = np.array([[n_pages - 1 - 2 * i for i in range(-(-n // page))]] * 2, np.int32)
        table[1] -= 40
        for b in range(2):
            for i in range(table.shape[1]):
                part = slice(i * page, min((i + 1) * page, n))
                for c, r in ((k, rows[0]), (v, rows[1])):
                    c[int(table[b, i]), :part.stop - part.start] = r[part]
        out = A.attn_tree_paged(q, k, v, torch.from_numpy(table).to(dev), None, i32(lens, dev), n, Hk)
    else:
        k, v = (torch.empty(far + n, kvs, device=dev, dtype=t) for _ in "kv")
        for c, r in ((k, rows[0]), (v, rows[1])):
            c[:n] = r
            c[far:far + n] = r
        out = A.attn_tree(q, k, v, None, i32(lens, dev), n, Hk, seq_stride=far * kvs)
    see = np.tril(np.ones((T, T), bool))
    for b in range(2):
        r = ref(q[b], rows[0][:lens[b] + T], rows[1][:lens[b] + T], see, lens[b], T, np.arange(T) + lens[b], 0, D ** -0.5, D)
        check(out[b], *r, n, t, f"b={b}")


def test_strides_and_scale(dev):
    """Rows of several caches side by side (a kv_stride over the heads' width), one
    cache for all sequences (seq_stride 0), a given scale, out and workspace."""
    t, H, Hk, D, T, n = torch.float16, 8, 2, 64, 6, 200
    g = torch.Generator(device=dev).manual_seed(2)
    both = torch.randn(n + T, 2 * Hk * D, device=dev, generator=g).to(t)
    k, v = both[:, :Hk * D], both[:, Hk * D:]
    q = torch.randn(2, T, H, D, device=dev, generator=g).to(t)
    out = torch.full((2, T, H, D), 7.0, device=dev)
    got = A.attn_tree(q, k, v, None, i32([n, n - 50], dev), n + T, Hk, scale=0.3, kv_stride=2 * Hk * D, out=out)
    assert got is out
    see = np.tril(np.ones((T, T), bool))
    for b, m in enumerate((n, n - 50)):
        r = ref(q[b], k[:m + T], v[:m + T], see, m, T, np.arange(T) + m, 0, 0.3, D)
        check(out[b], *r, n, t, f"b={b}")


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [0, 32])
def test_keys_past_max_len_and_no_positions(dev, dt, page):
    """A max_len inside the drafts cuts their keys, not their rows; without
    positions a window goes by the slots (and is refused over a mask)."""
    t, rng, H, Hk, D, T, lens = DT[dt], np.random.default_rng(4), 8, 2, 128, 11, [60, 90]
    caches, rows, table = make(rng, dev, lens, [T, T], T, Hk, D, t, page, 0, 101)
    q = torch.randn(2, T, H, D, device=dev, generator=torch.Generator(device=dev).manual_seed(6)).to(t)
    see, _, mask = trees(rng, 2, T, "tree")
    out = attend(q, caches, table, mask.to(dev), i32(lens, dev), 95, Hk, None, None, 0)
    cut = see.copy()
    cut[1, :, 5:] = False
    for b in range(2):
        r = ref(q[b], rows[0][b], rows[1][b], cut[b], lens[b], T, lens[b] + np.arange(T), 0, D ** -0.5, D)
        check(out[b], *r, 101, t, f"b={b}")
    out = attend(q, caches, table, None, i32(lens, dev), 101, Hk, None, None, 9)
    for b in range(2):
        r = ref(q[b], rows[0][b], rows[1][b], np.tril(np.ones((T, T), bool)), lens[b], T, lens[b] + np.arange(T), 9, D ** -0.5, D)
        check(out[b], *r, 101, t, f"b={b}")
    with pytest.raises(L.UllmHipError) as e:
        attend(q, caches, table, mask.to(dev), i32(lens, dev), 101, Hk, None, None, 9)
    assert e.value.code == L.E_INVALID


def test_nothing_drafted(dev):
    k = torch.zeros(1, 64, 128, device=dev, dtype=torch.float16)
    for B, T in ((0, 4), (2, 0)):
        q = torch.zeros(B, T, 4, 64, device=dev, dtype=torch.float16)
        out = A.attn_tree(q, k, k, None, i32(np.zeros(B), dev), 64, 2)
        assert out.shape == q.shape
    q = torch.ones(1, 3, 4, 64, device=dev, dtype=torch.float16)
    assert not A.attn_tree(q, k, k, None, i32([0], dev), 0, 2).any()  # max_len 0: no key is there


def test_graph_replays_follow_their_inputs(dev):
    """One graph over append and attention, replayed with other lengths, trees,
    tables and tokens, equals the eager calls each time; two graphs with the same
    workspace may run one after the other."""
    t, H, Hk, D, T, P, B = torch.bfloat16, 8, 2, 128, 20, 32, 3
    n_pos, rng = 900, np.random.default_rng(11)
    stride = -(-n_pos // P)
    g = torch.Generator(device=dev).manual_seed(4)
    kp, vp = (torch.randn(B * stride, P, Hk * D, device=dev, generator=g).to(t) for _ in "kv")
    cs = A.rope_table(n_pos, D, 1e4)
    q, k, v = (torch.zeros(B, T, n * D, device=dev) for n in (H, Hk, Hk))
    lens, nn, pos, table = i32([0] * B, dev), i32([0] * B, dev), i32(np.zeros((B, T)), dev), i32(np.zeros((B, stride)), dev)
    mask = torch.zeros(B, T, 1, dtype=torch.int64, device=dev)
    ws = torch.empty(int(L.lib().ullm_hip_tree_workspace_bytes(L.DT_BF16, B, T, n_pos, 0, H, Hk, D)) or 1,
                     dtype=torch.uint8, device=dev)

    def step():
        qr = A.qkv_append_tree_paged(q, k, v, kp, vp, cs, lens, pos, table, n_head=H, n_kv_head=Hk, head_dim=D,
                                     n_nodes=nn, q_dtype=t)
        return A.attn_tree_paged(qr.view(B, T, H, D), kp, vp, table, mask, lens, n_pos, Hk, n_nodes=nn, positions=pos, workspace=ws)

    def fill(seed):
        r = np.random.default_rng(seed)
        ln, nd = r.integers(0, n_pos - T, B), r.integers(0, T + 1, B)
        see, depth, m = trees(r, B, T, "tree")
        for x, y in ((lens, ln), (nn, nd), (pos, ln[:, None] + depth), (table, r.permutation(B * stride).reshape(B, stride))):
            x.copy_(i32(y, dev))
        mask.copy_(m.to(dev))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=dev, generator=g))

    fill(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for i in range(6):
        fill(i)
        want = step().clone()
        torch.cuda.synchronize()
        for gr, out in graphs:
            out.fill_(NAN)
            gr.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want), f"replay {i}"


def test_another_stream_and_repeats(dev):
    """The same bits on another stream (its scratch is its own) and call after call."""
    t, H, Hk, D, T = torch.float16, 8, 2, 64, 12
    g = torch.Generator(device=dev).manual_seed(6)
    k, v = (torch.randn(1, 6000, Hk * D, device=dev, generator=g).to(t) for _ in "kv")
    q = torch.randn(1, T, H, D, device=dev, generator=g).to(t)
    lens = i32([5900], dev)
    want = A.attn_tree(q, k, v, None, lens, 6000, Hk)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
    outs = [torch.empty_like(want) for _ in range(3)]
    for o in outs:
        A.attn_tree(q, k, v, None, lens, 6000, Hk, out=o, stream=s)
    for _ in range(8):  # would take the scratch if it were free
        torch.full((1 << 20,), 0xFF, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    for _ in range(5):
        assert torch.equal(A.attn_tree(q, k, v, None, lens, 6000, Hk), want)


# ---- append ----
def append_ref(x, norm, bias, cs, neox, rd, D, eps):
    """[m, n*D] f32 -> [m, n, D] f64: bias, norm and rotation by cs [m, rd/2, 2]."""
    x = x.double() + (0 if bias is None else bias.double())
    x = x.view(x.shape[0], -1, D)
    if norm is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    if cs is None:
        return x
    c, s = cs.double()[:, None, :, 0], cs.double()[:, None, :, 1]
    h = torch.arange(rd // 2, device=x.device)
    i, j = (h, h + rd // 2) if neox else (2 * h, 2 * h + 1)
    y = x.clone()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    return y


@pytest.mark.parametrize("D,H,Hk,kv,qd,neox,rd,norm,bias,page", [
    (64, 8, 2, "f32", "f32", True, 64, False, False, 32),
    (128, 12, 2, "f16", "f16", False, 128, False, True, 64),
    (128, 32, 8, "bf16", "bf16", True, 128, True, False, 0),
    (256, 8, 4, "f16", "f32", True, 256, True, True, 16),
    (64, 14, 2, "bf16", "f16", False, 32, True, True, 1),
    (128, 5, 5, "f32", "bf16", True, 64, False, False, 0),
])
def test_append_tree(dev, D, H, Hk, kv, qd, neox, rd, norm, bias, page):
    """q, and the K/V rows at their slots, against 64 bits: each value is off by its
    type's rounding and at most 8 f32 roundings of the larger of its pair (norm: one
    of the sum of squares, the square root, two products; rotation: three).  Rows
    past the nodes, positions outside the table and slots outside the cache change
    nothing, and nothing else of the cache changes."""
    t, eps, T = DT[kv], 1e-6, 11
    rng, g = np.random.default_rng(D + H), torch.Generator(device=dev).manual_seed(D + rd)
    lens, nodes, n_pos, n_ctx = [0, 37, 100, 5], [11, 0, 7, 11], 120, 104
    B, kvs = len(lens), Hk * D + 16
    q, k, v = (torch.randn(B, T, n * D, device=dev, generator=g) for n in (H, Hk, Hk))
    w = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    qn, kn = (1 + 0.1 * w(D), 1 + 0.1 * w(D)) if norm else (None, None)
    qb, kb, vb = (w(H * D), w(Hk * D), w(Hk * D)) if bias else (None, None, None)
    cs = A.rope_table(n_pos, rd, 1e4)
    pos = np.array(lens)[:, None] + rng.integers(0, 9, (B, T))
    pos[3, 2], pos[3, 4], pos[2, 1] = -1, n_pos, n_pos - 1
    old = w(B, n_ctx, kvs).to(t), w(B, n_ctx, kvs).to(t)
    more = dict(n_head=H, n_kv_head=Hk, head_dim=D, n_nodes=i32(nodes, dev), rotary_dim=rd, neox=neox, q_norm=qn,
                k_norm=kn, eps=eps, q_bias=qb, k_bias=kb, v_bias=vb, q_dtype=DT[qd])
    if page:
        cols = -(-n_ctx // page)
        table = rng.permutation(B * cols).reshape(B, cols).astype(np.int32)
        table[3, 8 // page] = -1 if page > 1 else B * cols  # slot 8 has no page
        pools = [torch.zeros(B * cols * page, kvs, device=dev, dtype=t) for _ in "kv"]
        slot = lambda b, p: -1 if p >= n_ctx or not 0 <= table[b, p // page] < B * cols else int(table[b, p // page]) * page + p % page  # noqa: E731
        for b in range(B):
            for p in range(n_ctx):
                if slot(b, p) >= 0:
                    for c, o in zip(pools, old):
                        c[slot(b, p)] = o[b, p]
        before = [c.clone() for c in pools]
        # the table ends after the last whole page of n_ctx
        got = A.qkv_append_tree_paged(q, k, v, *(c.view(-1, page, kvs) for c in pools), cs, i32(lens, dev), i32(pos, dev),
                                      i32(table[:, :n_ctx // page], dev), **more)
        n_ctx = n_ctx // page * page
    else:
        pools = [o.clone().view(-1, kvs) for o in old]
        before = [c.clone() for c in pools]
        slot = lambda b, p: b * 104 + p if p < n_ctx else -1  # noqa: E731
        got = A.qkv_append_tree(q, k, v, *(c.view(B, 104, kvs) for c in pools), cs, i32(lens, dev), i32(pos, dev),
                                kv_stride=kvs, seq_stride=104 * kvs, **more)
    want = [c.double() for c in before]
    tol = [torch.zeros_like(c) for c in want]
    wq, tq = torch.zeros(B, T, H * D, dtype=torch.float64, device=dev), torch.zeros(B, T, H * D, dtype=torch.float64, device=dev)
    f8 = 8 * 2.0 ** -24

    def pair_max(x):  # the larger magnitude of a value's pair, 0.. for those not rotated
        return x.abs().amax(-1, keepdim=True).expand_as(x)

    for b in range(B):
        for i in range(nodes[b]):
            p = int(pos[b, i])
            if not 0 <= p < n_pos:
                continue
            c = cs[p:p + 1]
            yq = append_ref(q[b, i:i + 1], qn, qb, c, neox, rd, D, eps)
            wq[b, i] = yq.flatten()
            tq[b, i] = (unit(DT[qd]) * yq.abs() + f8 * pair_max(yq)).flatten()
            at = slot(b, lens[b] + i) if lens[b] + i < n_ctx else -1
            if at < 0:
                continue
            yk = append_ref(k[b, i:i + 1], kn, kb, c, neox, rd, D, eps)
            yv = append_ref(v[b, i:i + 1], None, vb, None, neox, rd, D, eps)
            for n, y in enumerate((yk, yv)):
                want[n][at, :Hk * D] = y.flatten()
                tol[n][at, :Hk * D] = (unit(t) * y.abs() + f8 * pair_max(y)).flatten()
    tiny = 2.0 ** -25 * (kv == "f16"), 2.0 ** -25 * (qd == "f16")  # half of f16's least step, near 0
    assert got.dtype == DT[qd] and ((got.double() - wq).abs() <= 1.01 * tq + tiny[1]).all()
    for n in range(2):
        assert ((pools[n].double() - want[n]).abs() <= 1.01 * tol[n] + tiny[0] * (tol[n] > 0)).all(), "kv"[n]


# ---- the whole path, and the engine's own ----
def test_engine_tree_equals_token_by_token(dev):
    """A draft through GpuAttention.forward_tree gives each node what forward gives
    a token after the node's path, and after accept the cache goes on from there."""
    p = A.AttnParams(n_layer=7, n_head=8, n_kv_head=2, head_dim=64, n_ctx=256, sliding_window=40, kv_dtype=torch.float32)
    rng, g = np.random.default_rng(3), torch.Generator(device=dev).manual_seed(8)
    a, b = A.GpuAttention(p, dev), A.GpuAttention(p, dev)
    pos, parents = 90, [-1, 0, 0, 1, 1, 3, 2, 5, -1]
    T = len(parents)
    rows = lambda n, m: torch.randn(n, m * 64, device=dev, generator=g)  # noqa: E731
    for layer in range(p.n_layer):
        x = rows(pos, 8), rows(pos, 2), rows(pos, 2)
        a.forward_batch(layer, *x)
        b.forward_batch(layer, *x)
    mask, depth = A.tree_masks(parents)
    draft = [(rows(T, 8), rows(T, 2), rows(T, 2)) for _ in range(p.n_layer)]
    where = (pos + depth).to(dev)
    outs = [a.forward_tree(n, *draft[n], pos, mask.to(dev), where) for n in range(p.n_layer)]
    for node in range(T):
        path, i = [], node
        while i >= 0:
            path.insert(0, i)
            i = parents[i]
        for layer in range(p.n_layer):
            for d, i in enumerate(path):
                got = b.forward(layer, *(x[i] for x in draft[layer]), pos + d)
            assert torch.allclose(outs[layer][node], got, rtol=0, atol=2e-3), (layer, node)
    path = [0, 1, 3, 5, 7]
    keep = torch.full((T,), -1, dtype=torch.int32)
    keep[:5] = torch.tensor(path)
    new = a.accept(keep.to(dev), i32([5], dev), pos)
    assert new.tolist() == [pos + 5]
    for layer in range(p.n_layer):
        for d, i in enumerate(path):
            b.forward(layer, *(x[i] for x in draft[layer]), pos + d)
        # a rotation is three f32 roundings of values below 8, in another order on the two sides
        assert (a.key_cache[layer, :pos + 5] - b.key_cache[layer, :pos + 5]).abs().max() <= 2 * 3 * 8 * 2.0 ** -24
        assert torch.equal(a.val_cache[layer, :pos + 5], b.val_cache[layer, :pos + 5])
    with pytest.raises(L.UllmHipError):
        a.forward_tree(0, *draft[0], p.n_ctx - 3, None, None)


def test_serving_loop(dev):
    """Several steps as a server runs them: pages, append, attention, accept, fork,
    over two layers, against caches kept row by row on the side."""
    t, H, Hk, D, P, NL, T, S = torch.float16, 8, 2, 64, 32, 2, 7, 3
    rng, g = np.random.default_rng(21), torch.Generator(device=dev).manual_seed(1)
    n_pages, cols, n_pos = 40, 12, 12 * P
    kp, vp = (torch.full((NL, n_pages, P, Hk * D), NAN, device=dev, dtype=t) for _ in "kv")
    cs = A.rope_table(n_pos, D, 1e4)
    table, lens = i32(np.full((S, cols), -1), dev), i32([0] * S, dev)
    side = [[[] for _ in range(NL)] for _ in range(S)]  # rows (k, v) of each sequence and layer
    for step in range(14):
        n = [len(side[s][0]) for s in range(S)]
        parent = list(range(S)) if step % 4 else [int(x) for x in rng.integers(0, S, S)]
        if step == 9:
            parent[1], side[1] = -1, [[] for _ in range(NL)]
        side = [[list(rows) for rows in side[p]] if p >= 0 else [[] for _ in range(NL)] for p in parent]
        n = [len(side[s][0]) for s in range(S)]
        table, lens, info = A.kv_pages_update(kp, vp, table, lens, i32(parent, dev), i32([m + T for m in n], dev))
        assert lens.tolist() == n and info[2].item() == 0
        parents = np.stack([[-1 if i == 0 else rng.integers(-1, i) for i in range(T)] for _ in range(S)])
        mask, depth = A.tree_masks(parents)
        pos = lens[:, None] + depth.to(dev)
        see = (mask[:, :, 0, None] >> torch.arange(T) & 1).bool().numpy()
        for layer in range(NL):
            q, k, v = (torch.randn(S, T, m * D, device=dev, generator=g) for m in (H, Hk, Hk))
            qr = A.qkv_append_tree_paged(q, k, v, kp[layer], vp[layer], cs, lens, pos.int(), table, n_head=H, n_kv_head=Hk,
                                         head_dim=D, q_dtype=t)
            out = A.attn_tree_paged(qr.view(S, T, H, D), kp[layer], vp[layer], table, mask.to(dev), lens, n_pos, Hk,
                                    positions=pos.int())
            for s in range(S):
                new_k = torch.stack([append_ref(k[s, i:i + 1], None, None, cs[pos[s, i]][None], True, D, D, 0).flatten()
                                     for i in range(T)]).to(t)
                new_v = v[s].to(t)
                ks, vs = ([r[x] for r in side[s][layer]] for x in (0, 1))
                kk, vv = torch.stack(ks + list(new_k)), torch.stack(vs + list(new_v))
                o, a, e = ref(qr[s].view(T, H, D), kk, vv, see[s], n[s], T, None, 0, D ** -0.5, D)
                # K rows may differ by a rounding where the f64 value lies next to a border
                assert ((out[s].double() - o).abs() <= 4 * unit(t) * (o.abs() + a) + 2e-3).all(), (step, layer, s)
                side[s][layer] += [(new_k[i], new_v[i]) for i in range(T)]
        path = np.full((S, T), -1, np.int32)
        count = rng.integers(0, T + 1, S)
        for s in range(S):
            path[s, :count[s]] = np.sort(rng.permutation(T)[:count[s]])
            for layer in range(NL):
                rows = side[s][layer]
                side[s][layer] = rows[:n[s]] + [rows[n[s] + int(i)] for i in path[s, :count[s]]]
        lens = A.kv_accept_paged(kp, vp, table, i32(path, dev), i32(count, dev), lens)
    for s in range(S):
        for layer in range(NL):
            for x, pool in ((0, kp), (1, vp)):
                got = pool[layer][table[s].long()].flatten(0, 1)[:len(side[s][layer])]
                assert torch.allclose(got.float(), torch.stack([r[x] for r in side[s][layer]]).float(), rtol=2e-3, atol=1e-4)


@pytest.mark.parametrize("change,code", [
    (dict(q=lambda x: x.cpu()), L.E_INVALID), (dict(q=lambda x: x.float()), L.E_INVALID),
    (dict(q=lambda x: x.transpose(1, 2)), L.E_INVALID), (dict(k=lambda x: x[:, :50].clone()), L.E_INVALID),
    (dict(lens=lambda x: x.long()), L.E_INVALID), (dict(lens=lambda x: x[:0]), L.E_INVALID),
    (dict(mask=lambda x: x.int()), L.E_INVALID), (dict(mask=lambda x: x[:, :3]), L.E_INVALID),
    (dict(n=lambda x: x.float()), L.E_INVALID), (dict(pos=lambda x: x[:, :2]), L.E_INVALID),
    (dict(out=lambda x: x.double()), L.E_UNSUPPORTED), (dict(out=lambda x: x[:, :2]), L.E_INVALID),
    (dict(out=lambda x: x.bfloat16()), L.E_UNSUPPORTED), (dict(pos=lambda x: None), L.E_INVALID),
    (dict(ws=lambda x: x[:8]), L.E_WORKSPACE), (dict(ws=lambda x: x[1:]), L.E_WORKSPACE),
])
def test_refusals(dev, change, code):
    a = dict(q=torch.zeros(1, 5, 4, 64, device=dev, dtype=torch.float16), k=torch.zeros(1, 4096, 128, device=dev, dtype=torch.float16),
             lens=i32([60], dev), mask=torch.zeros(1, 5, 1, dtype=torch.int64, device=dev), n=i32([5], dev),
             pos=i32([[60] * 5], dev), out=torch.zeros(1, 5, 4, 64, device=dev), ws=torch.zeros(1 << 20, dtype=torch.uint8, device=dev))
    for n, f in change.items():
        a[n] = f(a[n])
    with pytest.raises(L.UllmHipError) as e:
        A.attn_tree(a["q"], a["k"], a["k"], a["mask"], a["lens"], 4096, 2, n_nodes=a["n"], positions=a["pos"], window=3000,
                    out=a["out"], workspace=a["ws"])
    assert e.value.code == code
