"""kv_evict(_paged) on the GPU against the same rules on the host.  Everything is
whole numbers or moved bits: equal, never near."""
import numpy as np
import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def stay(x, n, sink, recent):
    """Positions of x (its length is the sequence's) that stay, in order."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64)), np.isnan(x)
    size = len(x[0])
    first = min(sink, n)
    last = min(recent, n - first)
    mid = np.arange(first, size - last)
    order = np.lexsort((mid, x[1][mid], -x[0][mid]))  # largest, numbers before NaN, lowest
    best = mid[order[:n - first - last]]
    return np.concatenate((np.arange(first), np.sort(best), np.arange(size - last, size))).astype(np.int64)


def case(dev, dt, NL, B, G, hd, lens, budgets, sink, recent, page=0, kind="spread", n_ctx=None, seed=0, out=True, wide=False,
         shared=False):
    """One call and its check.  `wide`: the caches are columns of wider rows."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    n_ctx = n_ctx or max(lens) + 3
    kvd, pad = G * hd, 2 * hd if wide else 0
    if page:
        cols = -(-n_ctx // page)
        n_pages = B * cols + 2
        table = rng.permutation(n_pages)[:B * cols].reshape(B, cols).astype(np.int32)
        shape = (NL, n_pages, page)
    else:
        shape = (NL, B, n_ctx)
    full = [torch.randn(*shape, kvd + pad, device=dev, generator=g).to(DT[dt]) for _ in "kv"]
    if shared:
        full[1] = full[0]
    k, v = (x[..., hd:hd + kvd] if wide else x for x in full)
    sc = rng.standard_normal((NL, B, G, n_ctx)).astype(np.float32)
    if kind == "spread":
        sc = np.exp(3 * sc).astype(np.float32)
    elif kind == "ties":
        sc = np.round(sc)
    elif kind == "equal":
        sc[:] = 0.25
    elif kind == "odd":
        sc[sc > 1.2] = np.nan
        sc[sc < -1.2] = -np.inf
        sc[..., ::5] = np.inf
        sc[..., 1::5] = -0.0
        sc[..., 2::5] = 0.0
        sc[..., 3::17] = 1e-42
    scores = torch.from_numpy(sc).to(dev)
    so = torch.full_like(scores, 7.0) if out else scores
    want = [x.clone() for x in full]
    top = max(max(budgets), 0)
    kept = np.full((NL, B, G, top), -1, np.int32)
    ref = np.full_like(sc, 7.0) if out else sc.copy()
    new = []
    for b in range(B):
        n = min(lens[b], max(budgets[b], 0))
        new.append(n)
        if page:
            place = torch.tensor([int(table[b, t // page]) * page + t % page for t in range(lens[b])], dtype=torch.long, device=dev)
        for lay in range(NL):
            for j in range(G):
                x = sc[lay, b, j, :lens[b]]
                s = stay(x, n, sink, recent) if n < lens[b] else np.arange(n)
                kept[lay, b, j, :n] = s
                ref[lay, b, j, :lens[b]] = 0
                ref[lay, b, j, :n] = x[s]
                c = slice((hd if wide else 0) + j * hd, (hd if wide else 0) + (j + 1) * hd)
                for w, f in zip(want, full):
                    w = w[lay].flatten(0, 1) if page else w[lay, b]
                    f = f[lay].flatten(0, 1) if page else f[lay, b]
                    p = place if page else torch.arange(lens[b], device=dev)
                    w[p[:n], c] = f[p[torch.from_numpy(s).to(dev)], c]
    more = dict(max_budget=top, sink=sink, recent=recent, scores_out=so if out else None)
    args = (scores, i32(lens, dev), i32(budgets, dev))
    if page:
        got, out_lens = A.kv_evict_paged(k, v, i32(table, dev), *args, **more)
    else:
        got, out_lens = A.kv_evict(k, v, *args, **more)
    assert out_lens.tolist() == new
    assert np.array_equal(got.cpu().numpy(), kept)
    assert np.array_equal(so.cpu().numpy().view(np.int32), ref.view(np.int32))
    for w, f in zip(want, full):
        assert torch.equal(w.view(torch.uint8), f.view(torch.uint8))


@pytest.mark.parametrize("page", [0, 1, 32, 256])
@pytest.mark.parametrize("dt,NL,B,G,hd,lens,budgets,sink,recent", [
    ("f32", 1, 1, 1, 4, [1], [0], 0, 0), ("f32", 1, 1, 1, 4, [1], [1], 0, 0), ("f16", 2, 1, 2, 8, [7], [3], 1, 1),
    ("bf16", 3, 3, 4, 64, [300, 17, 129], [100, 30, 64], 4, 16), ("f32", 1, 2, 8, 64, [1401, 1024], [1024, 1023], 4, 128),
    ("f16", 2, 2, 3, 40, [2049, 4100], [1000, 4099], 0, 0), ("bf16", 1, 1, 2, 128, [9000], [2048], 16, 256),
    ("f16", 1, 4, 1, 256, [513, 5, 0, 64], [64, 0, 4, -2], 3, 70), ("f32", 2, 1, 1, 512, [700], [5], 9, 9)])
def test_against_the_host(dev, page, dt, NL, B, G, hd, lens, budgets, sink, recent):
    case(dev, dt, NL, B, G, hd, lens, budgets, sink, recent, page, seed=len(lens) * 7 + hd)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd"])
@pytest.mark.parametrize("out", [False, True])
def test_scores(dev, kind, out):
    for lens, budgets in (([3000, 64, 1], [700, 63, 1]), ([4096, 4097, 4095], [4095, 2048, 1])):
        case(dev, "f16", 1, 3, 2, 16, lens, budgets, 2, 5, kind=kind, out=out)


@pytest.mark.parametrize("n", [20000, 70001, 140000])
def test_long_rows(dev, n):
    """More scores than one workgroup's registers or LDS hold."""
    case(dev, "f16", 1, 1, 2, 8, [n], [n // 3], 4, 100, seed=n)
    case(dev, "f16", 1, 1, 2, 8, [n], [n - 1], 4, 100, kind="ties", seed=n, out=False)


def test_short_and_long_sequences_of_a_long_cache(dev):
    """Scores that fit a workgroup's registers beside some that do not."""
    case(dev, "f16", 1, 4, 2, 8, [5000, 39000, 32768, 32769], [4000, 30000, 100, 32768], 4, 100, n_ctx=40000)


def test_columns_of_wider_rows(dev):
    for page in (0, 32):
        case(dev, "bf16", 2, 2, 2, 32, [100, 200], [50, 60], 2, 8, page, wide=True)


def test_k_that_is_v(dev):
    case(dev, "f16", 2, 2, 2, 32, [100, 200], [50, 60], 2, 8, shared=True)


def test_forms_of_the_caches(dev):
    """The same one sequence as [n_ctx, d], [1, n_ctx, d], [layers, n_ctx, d] and
    [layers, 1, n_ctx, d]."""
    g = torch.Generator(device=dev).manual_seed(1)
    k = torch.randn(3, 60, 64, device=dev, generator=g).half()
    sc = torch.rand(3, 2, 60, device=dev, generator=g)
    lens, budget = i32([55], dev), i32([20], dev)
    k3, v3 = k.clone(), k.clone() + 1
    kept, _ = A.kv_evict(k3, v3, sc.clone(), lens, budget, max_budget=20, sink=1, recent=4)
    assert kept.shape == (3, 1, 2, 20)
    k4, v4 = k.clone()[:, None], (k.clone() + 1)[:, None]
    A.kv_evict(k4, v4, sc.clone()[:, None], lens, budget, max_budget=20, sink=1, recent=4)
    assert torch.equal(k4[:, 0], k3) and torch.equal(v4[:, 0], v3)
    for lay in range(3):
        for lead in ((), (None,)):
            k1, v1, s1 = k[lay].clone()[lead], (k[lay] + 1)[lead], sc[lay].clone()
            A.kv_evict(k1, v1, s1, lens, budget, max_budget=20, sink=1, recent=4)
            assert torch.equal(k1.view(60, 64), k3[lay]) and torch.equal(v1.view(60, 64), v3[lay])


def test_pages_outside_the_pool(dev):
    """Rows in pages that are none are neither read nor written."""
    g = torch.Generator(device=dev).manual_seed(1)
    k = torch.randn(4, 32, 16, device=dev, generator=g).half()
    v, old = k.clone(), k.clone()
    table = i32([[2, -1, 0, 9]], dev)
    sc = torch.rand(1, 1, 128, device=dev, generator=g)
    kept, lens = A.kv_evict_paged(k, v, table, sc, i32([500], dev), i32([50], dev), max_budget=50)
    assert lens.item() == 50 and torch.equal(k, v)
    kept = kept.view(-1).tolist()
    page = {0: 2, 2: 0}
    for j, t in enumerate(kept[:32]):  # page 1 of the sequence is none: rows 32 to 49 are nowhere
        assert torch.equal(k[2, j], old[page[t // 32], t % 32] if t // 32 in page else old[2, j])
    assert torch.equal(k[0], old[0]) and torch.equal(k[1], old[1]) and torch.equal(k[3], old[3])


def test_bounds_of_lengths_and_scores(dev):
    """Lengths past the cache or the scores are cut, below 0 they are 0; budgets past
    max_budget are cut."""
    k = torch.randn(3, 40, 16, device=dev).half()
    v, old = k.clone(), k.clone()
    sc = torch.rand(3, 1, 30, device=dev)
    x = sc.cpu().numpy()
    kept, lens = A.kv_evict(k, v, sc, i32([1 << 30, -7, 25], dev), i32([1 << 30, 5, 1 << 30], dev), max_budget=10)
    assert lens.tolist() == [10, 0, 10]
    for b, n in ((0, 30), (2, 25)):
        s = stay(x[b, 0, :n], 10, 0, 0)
        assert kept[0, b, 0].tolist() == s.tolist() and torch.equal(k[b, :10], old[b, s]) and torch.equal(k[b, 10:], old[b, 10:])
    assert (kept[0, 1] == -1).all() and torch.equal(k[1], old[1])


def test_nothing_is_kept(dev):
    k = torch.randn(1, 40, 16, device=dev)
    old, sc = k.clone(), torch.rand(1, 1, 40, device=dev)
    kept, lens = A.kv_evict(k, k.clone(), sc, i32([40], dev), i32([9], dev), max_budget=0)
    assert lens.item() == 0 and kept.numel() == 0 and torch.equal(k, old) and (sc == 0).all()


def test_front_refuses(dev):
    k = torch.zeros(2, 40, 16, device=dev).half()
    sc, i = torch.zeros(2, 2, 40, device=dev), i32([9, 9], dev)
    good = dict(k_cache=k, v_cache=k.clone(), scores=sc, seq_lens=i, budget=i.clone(), max_budget=9)
    A.kv_evict(**good)
    for bad in (dict(scores=sc.double()), dict(scores=sc[0]), dict(scores=sc[:, :1, ::2]), dict(seq_lens=i.long()), dict(seq_lens=i[:1]),
                dict(budget=i[:1]), dict(max_budget=-1), dict(sink=-1), dict(recent=-1), dict(scores=torch.zeros(2, 3, 40, device=dev)),
                dict(scores=torch.zeros(2, 4, 40, device=dev)), dict(v_cache=k[:, :30]), dict(v_cache=k.float()), dict(kept=i),
                dict(scores_out=sc[:, :1]), dict(lens_out=i), dict(lens_out=i[:1]), dict(k_cache=k[:1].expand(2, 40, 16), v_cache=k[:1].expand(2, 40, 16))):
        with pytest.raises(L.UllmHipError):
            A.kv_evict(**{**good, **bad})


def test_captured_and_replayed(dev):
    g = torch.Generator(device=dev).manual_seed(1)
    k0 = torch.randn(2, 2, 500, 64, device=dev, generator=g).half()
    k, v = k0.clone(), k0.clone() + 1
    sc, so = torch.rand(2, 2, 2, 500, device=dev, generator=g), torch.zeros(2, 2, 2, 500, device=dev)
    lens, budget = i32([500, 77], dev), i32([100, 70], dev)
    call = lambda k, v, so: A.kv_evict(k, v, sc, lens, budget, max_budget=100, sink=2, recent=9, scores_out=so)  # noqa: E731
    call(k, v, so)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(k, v, so)
    for r in range(4):
        sc.copy_(torch.rand(sc.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(r)))
        k.copy_(k0)
        v.copy_(k0 + 1)
        graph.replay()
        ke, ve, se = k0.clone(), k0 + 1, torch.zeros_like(so)
        want = call(ke, ve, se)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*got, k, v), (*want, ke, ve)))
        assert torch.equal(so[:, 0], se[:, 0])


@pytest.mark.parametrize("page", [0, 32])
def test_offsets_past_32_bits(dev, page):
    """Rows 128 KB apart, 5.2 GB of them, against the same rows close together."""
    n, G, hd, keep = 40000, 2, 64, 36000
    g = torch.Generator(device=dev).manual_seed(4)
    k = torch.randn(1, 1, n, G * hd, device=dev, generator=g).half()
    wide = torch.full((1, 1, n, 65536), 3.0, device=dev, dtype=torch.float16)
    far = wide[..., 65536 - G * hd:]
    far.copy_(k)
    sc = torch.rand(1, 1, G, n, device=dev, generator=g)
    lens, budget = i32([n - 3], dev), i32([keep], dev)
    more = dict(max_budget=keep, sink=4, recent=100)
    want, _ = A.kv_evict(k, k, sc.clone(), lens, budget, **more)
    if page:
        pool = far.view(1, n // page, page, G * hd)
        got, _ = A.kv_evict_paged(pool, pool, i32([list(range(n // page))], dev), sc, lens, budget, **more)
    else:
        got, _ = A.kv_evict(far, far, sc, lens, budget, **more)
    assert torch.equal(got, want) and torch.equal(far, k)
    assert (wide[0, 0, ::1000, :65536 - G * hd] == 3).all()
