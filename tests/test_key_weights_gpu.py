"""key_weights(_paged) on the GPU against the formula in 64 bits.

The tolerance of a weight is derived, with u = 2^-24 (half a step of f32):
- a score is a sum of D products with at most 3 roundings of each operand's pieces,
  accumulated in any order: off by at most (D + 8) u S, S the largest sum of
  |q||k| scale of a key that is seen; its scaling and the exponential's argument add
  at most 4 u S + 4 u, the exponential itself 2 u: with d = (D + 12) u S + 6 u a
  weight is off by at most 2 d of itself (its own score and the denominator's),
- the denominator is a sum of at most n terms in any order: n u of itself,
- the sum over R rows and its last steps: (R + 8) u.
What an exponential rounds to zero (below 2^-126 of the largest) adds R 2^-120."""
import math

import numpy as np
import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def rule(q, k, n, r, window, scale):
    """(weights [n], their relative tolerance) of the keys of one kv head: q [rows, group, D], k [n, D]
    in 64 bits, row i at position n - r + i."""
    pos, key = torch.arange(n - r, n, device=k.device)[:, None], torch.arange(n, device=k.device)
    see = (key <= pos) & (pos >= 0)
    if window:
        see &= key > pos - window
    w, most = torch.zeros(n, dtype=torch.float64, device=k.device), 0.0
    for h in range(q.shape[1]):
        s = (q[:r, h] @ k.t().contiguous() * scale).masked_fill(~see, -math.inf)
        w += torch.nan_to_num(torch.softmax(s, -1), nan=0.0).sum(0)
        mag = (q[:r, h].abs() @ k.abs().t().contiguous() * abs(scale)).masked_fill(~see, 0)
        most = max(most, float(mag.max()) if mag.numel() else 0.0)
    rows = q.shape[1] * r
    d = (q.shape[2] + 12) * U * most + 6 * U
    return w, 2 * d + (n + rows + 8) * U, rows * 2.0 ** -120


def case(dev, kv, qt, B, rows, H, Hk, D, lens, n_rows=None, window=0, page=0, decay=1.0, seed=0, scale=None, spread=1.0,
         extra=0, given=False, stream=None, view=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    max_len = max(lens) + extra
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    q = (spread * rnd(B, rows, H, D)).to(DT[kv if qt == "kv" else "f32"])
    if page:
        cols = -(-max_len // page)
        n_pages = B * cols + 2
        table = rng.permutation(n_pages)[:B * cols].reshape(B, cols).astype(np.int32)
        k = rnd(n_pages, page, Hk * D).to(DT[kv])
        dense = k[torch.from_numpy(table).long().to(dev)].flatten(1, 2)
    else:
        k = dense = rnd(B, max_len, Hk * D).to(DT[kv])
    acc = torch.rand(B, Hk, max_len + 5, device=dev, generator=g)
    if decay == 0.0:
        acc[:] = float("nan")
    old = acc.clone()
    n_rows = [rows] * B if n_rows is None else n_rows
    scale = D ** -0.5 if scale is None else scale
    args = dict(n_rows=i32(n_rows, dev), window=window, scale=scale, decay=decay, stream=stream)
    if given:
        size = L.lib().ullm_hip_key_weights_workspace_bytes(L.DT_F32, B, rows, max_len, window, H, Hk, D)
        size = max(size, L.lib().ullm_hip_key_weights_workspace_bytes({"f32": 0, "f16": 1, "bf16": 2}[kv], B, rows, max_len, window, H, Hk, D))
        args["workspace"] = torch.full((size,), 255, dtype=torch.uint8, device=dev)
    w = acc[..., :max_len + 2] if view else acc
    if page:
        out = A.key_weights_paged(q, k, i32(table, dev), w, i32(lens, dev), max_len, Hk, **args)
    else:
        out = A.key_weights(q, k, w, i32(lens, dev), max_len, Hk, **args)
    if stream is not None:
        stream.synchronize()
    assert out.data_ptr() == acc.data_ptr()
    for b in range(B):
        n, r = min(max(lens[b], 0), max_len), min(max(n_rows[b], 0), rows)
        assert torch.equal(acc[b, :, n:].nan_to_num(), old[b, :, n:].nan_to_num()), "positions past the length"
        for j in range(Hk):
            qh = q[b, :, j * (H // Hk):(j + 1) * (H // Hk)].double()
            want, rel, low = rule(qh, dense[b, :n, j * D:(j + 1) * D].double(), n, r, window, scale)
            err = (acc[b, j, :n].double() - want - (decay * old[b, j, :n].double() if decay else 0)).abs()
            tol = want * rel + low + (4 * U * (want + old[b, j, :n].double() * decay) if decay else 0)
            worst = (err - tol).max().item() if n else 0.0
            assert worst <= 0, (b, j, err.max().item(), worst)


SHAPES = [(32, 8, 64), (12, 2, 128), (8, 4, 256), (32, 4, 128), (40, 8, 128), (14, 2, 64), (3, 3, 128), (32, 1, 64), (20, 1, 256)]


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("qt", ["f32", "kv"])
@pytest.mark.parametrize("H,Hk,D", SHAPES)
def test_one_row(dev, kv, qt, H, Hk, D):
    """A decode step over ragged lengths, contiguous and in pages."""
    case(dev, kv, qt, 5, 1, H, Hk, D, [1, 31, 64, 777, 300], page=32, seed=1)
    case(dev, kv, qt, 2, 1, H, Hk, D, [1025, 2], seed=2, extra=3)


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("qt", ["f32", "kv"])
@pytest.mark.parametrize("rows", [2, 5, 16, 33, 70])
def test_several_rows(dev, kv, qt, rows):
    H, Hk, D = SHAPES[rows % len(SHAPES)]
    case(dev, kv, qt, 3, rows, H, Hk, D, [rows, 500, 129], [rows, rows - 1, min(rows, 7)], page=64, seed=rows)
    case(dev, kv, qt, 1, rows, H, Hk, D, [900], seed=rows, decay=0.0)


@pytest.mark.parametrize("kv,qt,H,Hk,D,S", [
    ("bf16", "kv", 8, 2, 128, 700), ("f16", "f32", 14, 2, 64, 333), ("f32", "f32", 6, 2, 128, 257), ("f16", "kv", 4, 2, 256, 301),
    ("bf16", "f32", 8, 4, 256, 130), ("f32", "kv", 5, 1, 64, 511)])
def test_whole_prompts(dev, kv, qt, H, Hk, D, S):
    case(dev, kv, qt, 1, S, H, Hk, D, [S], decay=0.0, seed=S)
    case(dev, kv, qt, 2, S, H, Hk, D, [S + 40, S // 2], [S, S // 3], seed=S, page=32, decay=0.5)
    case(dev, kv, qt, 1, S, H, Hk, D, [S + 7], window=50, seed=S)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 100, 5000])
def test_windows(dev, window):
    for kv, qt in (("f16", "kv"), ("bf16", "f32"), ("f32", "f32")):
        case(dev, kv, qt, 3, 1, 8, 2, 64, [1000, 30, 77], window=window, page=32, seed=window)
        case(dev, kv, qt, 2, 40, 8, 2, 128, [1000, 60], [40, 25], window=window, seed=window)


def test_counts_and_lengths_outside_their_range(dev):
    """Lengths are cut to 0..max_len, rows to 0..max_rows; a sequence without rows only
    fades, one without positions is left alone; rows before position 0 see nothing."""
    case(dev, "f16", "kv", 6, 4, 8, 2, 64, [0, 50, 3, 50, 1 << 20, -5][:4] + [50, 0], [4, 0, 4, -3, 99, 4], decay=0.5)
    k = torch.randn(2, 60, 128, device=dev).half()
    q = torch.randn(2, 8, 64, device=dev)
    w = torch.zeros(2, 2, 60, device=dev)
    A.key_weights(q, k, w, i32([1000, -9], dev), 60, 2)
    ref = torch.zeros(2, 2, 60, device=dev)
    A.key_weights(q[:1].contiguous(), k[:1].contiguous(), ref[:1], i32([60], dev), 60, 2)
    assert torch.equal(w, ref) and (w[0].sum(-1) - 4).abs().max() < 1e-4 and (w[1] == 0).all()


@pytest.mark.parametrize("B", [63, 64, 65, 130])
def test_many_sequences(dev, B):
    """Up to 64 sequences are cut together on the device, more of them each alone."""
    lens = [1 + (b * 37) % 300 for b in range(B)]
    for rows, page in ((1, 32), (1, 0), (9, 64)):
        case(dev, "bf16", "kv", B, rows, 8, 2, 64, lens, [min(rows, n) for n in lens], page=page, seed=B)
    case(dev, "f16", "f32", B, 6, 6, 2, 64, [max(1, n // 20) for n in lens[:-1]] + [2000], [1] * (B - 1) + [6], window=700, seed=B)


@pytest.mark.parametrize("kv,qt", [("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("f16", "kv")])
def test_queries_of_zeros(dev, kv, qt):
    """Every key that is seen gets the same weight, with any scale."""
    for rows in (1, 40, 300):
        for scale in (0.125, 0.0, 1e-30):
            q = torch.zeros(1, rows, 4, 64, device=dev).to(DT[kv if qt == "kv" else "f32"])
            k = torch.randn(1, 400, 128, device=dev).to(DT[kv])
            w = torch.zeros(1, 2, 400, device=dev)
            A.key_weights(q, k, w, i32([400], dev), 400, 2, scale=scale, window=100)
            pos, key = torch.arange(400 - rows, 400)[:, None], torch.arange(400)
            see = ((key <= pos) & (key > pos - 100)).double()
            want = 2 * (see / see.sum(1, keepdim=True)).sum(0)
            assert (w[0].double().cpu() - want).abs().max() <= want.max() * (400 + rows + 20) * U


def test_all_rows_before_the_sequence(dev):
    """n_rows past the length: only the rows that stand at a position count."""
    q = torch.randn(1, 30, 4, 64, device=dev).half()
    k = torch.randn(1, 12, 64, device=dev).half()
    a, b = torch.zeros(1, 1, 12, device=dev), torch.zeros(1, 1, 12, device=dev)
    A.key_weights(q, k, a, i32([12], dev), 12, 1)
    A.key_weights(q[:, 18:].contiguous(), k, b, i32([12], dev), 12, 1)
    assert (a - b).abs().max() <= 60 * U * 48


@pytest.mark.parametrize("kv,qt", [("f32", "f32"), ("f16", "f32"), ("f16", "kv"), ("bf16", "f32"), ("bf16", "kv")])
def test_unseen_keys_may_hold_anything(dev, kv, qt):
    """NaN and infinities behind the length, and before the window, stay out."""
    H, Hk, D, n = 8, 2, 128, 200
    g = torch.Generator(device=dev).manual_seed(3)
    for rows in (1, 40):
        q = torch.randn(1, rows, H, D, device=dev, generator=g).to(DT[kv if qt == "kv" else "f32"])
        k = torch.randn(1, 300, Hk * D, device=dev, generator=g).to(DT[kv])
        bad = k.clone()
        bad[:, n:] = float("nan")
        bad[:, :n - rows - 60] = float("inf")
        bad[:, 3] = float("nan")
        a, b = torch.zeros(1, Hk, 300, device=dev), torch.zeros(1, Hk, 300, device=dev)
        A.key_weights(q, k, a, i32([n], dev), 300, Hk, window=60)
        A.key_weights(q, bad, b, i32([n], dev), 300, Hk, window=60)
        assert torch.equal(a, b) and b.isfinite().all()


def test_large_and_small_scores(dev):
    """Scores of hundreds: one key takes all; scores near 0: all alike; a negative scale
    and one of 0."""
    for kv, qt in (("f16", "kv"), ("bf16", "f32"), ("f32", "f32"), ("f16", "f32")):
        for scale, spread in ((1.0, 8.0), (1e-3, 1e-3), (-0.2, 1.0), (0.0, 1.0)):
            case(dev, kv, qt, 2, 3, 8, 2, 64, [300, 41], scale=scale, spread=spread, seed=5)


def test_pages_outside_the_pool_read_as_zeros(dev):
    H, Hk, D = 8, 2, 64
    q = torch.randn(2, 3, H, D, device=dev).half()
    k = torch.randn(5, 32, Hk * D, device=dev).half()
    table = i32([[4, -1, 2], [7, 0, 1 << 30]], dev)
    dense = torch.zeros(2, 96, Hk * D, device=dev).half()
    dense[0, :32], dense[0, 64:], dense[1, 32:64] = k[4], k[2], k[0]
    a, b = torch.zeros(2, Hk, 96, device=dev), torch.zeros(2, Hk, 96, device=dev)
    A.key_weights_paged(q, k, table, a, i32([90, 96], dev), 96, Hk)
    A.key_weights(q, dense, b, i32([90, 96], dev), 96, Hk)
    assert torch.equal(a, b) and a[0].sum() > 0


def test_strides_of_the_cache(dev):
    """Columns of wider rows, one cache for all sequences, and a slice of a buffer of
    weights of several layers."""
    H, Hk, D = 8, 2, 64
    g = torch.Generator(device=dev).manual_seed(3)
    wide = torch.randn(2, 100, 512, device=dev, generator=g).half()
    q = torch.randn(2, 5, H, D, device=dev, generator=g).half()
    k = wide[..., 128:256]
    lens = i32([100, 64], dev)
    layers = torch.zeros(3, 2, Hk, 104, device=dev)
    ref = torch.zeros(2, Hk, 100, device=dev)
    A.key_weights(q, k.contiguous(), ref, lens, 100, Hk)
    A.key_weights(q, k, layers[1], lens, 100, Hk)
    assert torch.equal(layers[1, ..., :100], ref) and (layers[0] == 0).all() and (layers[1:, ..., 100:] == 0).all()
    one = torch.zeros(2, Hk, 100, device=dev)
    A.key_weights(q, k[:1].contiguous(), one, lens, 100, Hk, seq_stride=0)
    two = torch.zeros(2, Hk, 100, device=dev)
    A.key_weights(q, k[:1].expand(2, 100, 128).contiguous(), two, lens, 100, Hk)
    assert torch.equal(one, two)


def test_given_workspace_and_stream(dev):
    st = torch.cuda.Stream()
    case(dev, "f16", "f32", 3, 1, 8, 2, 128, [700, 5, 64], given=True, view=True)
    case(dev, "bf16", "kv", 2, 40, 8, 2, 128, [700, 65], page=64, given=True)
    torch.cuda.synchronize()
    case(dev, "f32", "f32", 2, 20, 8, 2, 64, [700, 65], given=True)


def test_other_stream(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    q, k = torch.randn(1, 8, 64, device=dev, generator=g), torch.randn(1, 500, 128, device=dev, generator=g)
    a, b = torch.zeros(1, 2, 500, device=dev), torch.zeros(1, 2, 500, device=dev)
    A.key_weights(q, k, a, i32([500], dev), 500, 2)
    n = i32([500], dev)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    A.key_weights(q, k, b, n, 500, 2, stream=st)
    st.synchronize()
    assert torch.equal(a, b)


def test_same_call_same_bits(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    q, k = torch.randn(2, 300, 8, 128, device=dev, generator=g).half(), torch.randn(2, 3000, 256, device=dev, generator=g).half()
    outs = []
    for _ in range(5):
        w = torch.zeros(2, 2, 3000, device=dev)
        A.key_weights(q, k, w, i32([3000, 1234], dev), 3000, 2)
        outs.append(w)
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_front_refuses(dev):
    q, k, w, n = torch.zeros(2, 8, 64, device=dev), torch.zeros(2, 50, 128, device=dev), torch.zeros(2, 2, 50, device=dev), i32([9, 9], dev)
    good = dict(q=q, k_cache=k, weights=w, seq_lens=n, max_len=50, n_kv_head=2)
    A.key_weights(**good)
    for bad in (dict(q=q.half()), dict(q=q.double()), dict(q=q[..., ::2]), dict(k_cache=k[:, :40]), dict(weights=w[:, :1]), dict(weights=w[..., :49]),
                dict(weights=w.half()), dict(weights=torch.zeros(2, 2, 100, device=dev)[..., ::2]), dict(weights=torch.zeros(2, 4, 50, device=dev)[:, ::2][:1].expand(2, 2, 50)),
                dict(seq_lens=n.long()), dict(seq_lens=n[:1]), dict(n_rows=n[:1]), dict(max_len=51), dict(n_kv_head=3), dict(max_len=-1),
                dict(workspace=torch.empty(8, dtype=torch.uint8, device=dev))):
        with pytest.raises(L.UllmHipError):
            A.key_weights(**{**good, **bad})


@pytest.mark.parametrize("rows", [1, 50])
def test_captured_and_replayed(dev, rows):
    g = torch.Generator(device=dev).manual_seed(3)
    q, k = torch.randn(2, rows, 8, 128, device=dev, generator=g).half(), torch.randn(2, 3000, 256, device=dev, generator=g).half()
    n, w = i32([3000, 600], dev), torch.zeros(2, 2, 3000, device=dev)
    A.key_weights(q, k, w, n, 3000, 2, decay=0.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.key_weights(q, k, w, n, 3000, 2, decay=0.0)
    for r in range(4):
        q.copy_(torch.randn(q.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(r)))
        n.copy_(i32([3000 - 700 * r, 100 + r], dev))
        w.zero_()
        graph.replay()
        want = torch.zeros_like(w)
        A.key_weights(q, k, want, n, 3000, 2, decay=0.0)
        torch.cuda.synchronize()
        assert torch.equal(w, want)


@pytest.mark.parametrize("rows", [1, 20, 100])
def test_offsets_past_32_bits(dev, rows):
    """A cache whose rows lie 128 KB apart, 5.2 GB of them, against the same rows close
    together; as one sequence and as pages."""
    H, Hk, D, n = 8, 2, 64, 40000
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn(1, rows, H, D, device=dev, generator=g).half()
    k = torch.randn(1, n, Hk * D, device=dev, generator=g).half()
    wide = torch.empty(1, n, 65536, device=dev, dtype=torch.float16)
    far = wide[..., :Hk * D]
    far.copy_(k)
    ref, out, paged = (torch.zeros(1, Hk, n, device=dev) for _ in range(3))
    lens = i32([n - 3], dev)
    A.key_weights(q, k, ref, lens, n, Hk)
    A.key_weights(q, far, out, lens, n, Hk)
    A.key_weights_paged(q, wide.view(n // 32, 32, 65536), i32([list(range(n // 32))], dev), paged, lens, n, Hk)
    assert torch.equal(out, ref) and torch.equal(paged, ref) and ref[..., -100:-3].sum() > 0
