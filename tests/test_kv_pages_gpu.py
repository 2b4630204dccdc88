"""Rows and pages of a cache on the GPU: kv_accept(_paged) and kv_pages_update,
against the same rules row by row on the host.  Everything is whole numbers or
moved bits: equal, never near."""
import numpy as np
import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def pool(dev, dt, *shape, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(*shape, device=dev, generator=g).to(DT[dt])


@pytest.mark.parametrize("dt,NL,B,P,kvd,T", [
    ("f32", 1, 1, 32, 4, 1), ("f16", 3, 4, 32, 64, 9), ("bf16", 28, 2, 64, 256, 26), ("f16", 2, 5, 1, 8, 17),
    ("f32", 1, 33, 128, 512, 64), ("bf16", 5, 3, 256, 1024, 300), ("f16", 1, 2, 32, 40, 1024), ("bf16", 2, 1, 64, 8192, 5),
])
def test_accept_paged(dev, dt, NL, B, P, kvd, T):
    rng = np.random.default_rng(T)
    lens = rng.integers(0, 200, B)
    cols = -(-(int(lens.max()) + T) // P)
    n_pages = B * cols + 2
    k, v = (pool(dev, dt, NL, n_pages, P, kvd, seed=s) for s in (1, 2))
    table = rng.permutation(n_pages)[:B * cols].reshape(B, cols).astype(np.int32)
    path, count = np.full((B, T), -1, np.int32), rng.integers(0, T + 1, B)
    for b in range(B):
        kind = b % 3
        nodes = rng.permutation(T)[:count[b]]
        path[b, :count[b]] = np.sort(nodes) if kind == 0 else nodes if kind == 1 else rng.integers(0, T, count[b])
        if kind == 2 and count[b] > 2:
            path[b, 1], path[b, 2] = -1, 1 << 30  # left as they are
    if B > 2:
        table[2, -1] = n_pages  # rows there are neither read nor written
    want = [x.clone().view(NL, n_pages * P, kvd) for x in (k, v)]
    row = lambda b, t: int(table[b, t // P]) * P + t % P if t < cols * P and 0 <= table[b, t // P] < n_pages else -1  # noqa: E731
    for x, y in zip(want, (k, v)):
        src = y.clone().view(NL, n_pages * P, kvd)
        pairs = [(row(b, int(lens[b]) + j), row(b, int(lens[b]) + int(path[b, j]))) for b in range(B) for j in range(count[b]) if path[b, j] >= 0]
        pairs = [(d, s) for d, s in pairs if d >= 0 and s >= 0]
        if pairs:
            d, s = (torch.tensor(z, device=dev) for z in zip(*pairs))
            x[:, d] = src[:, s]
    new = A.kv_accept_paged(k, v, i32(table, dev), i32(path, dev), i32(count, dev), i32(lens, dev))
    assert new.tolist() == (lens + count).tolist()
    assert torch.equal(k.view_as(want[0]), want[0]) and torch.equal(v.view_as(want[1]), want[1])


@pytest.mark.parametrize("shape", [(50, 64), (1, 50, 64), (3, 50, 64), (4, 1, 50, 64), (2, 3, 50, 64)])
@pytest.mark.parametrize("wide", [False, True])
def test_accept_contiguous(dev, shape, wide):
    """Every form of the caches, also as a slice of wider rows, of which only the
    slice moves."""
    B = 3 if shape == (2, 3, 50, 64) else 1
    T, lens, count = 6, [44, 10, 47][:B], [6, 3, 5][:B]
    path = [[5, 4, 3, 2, 1, 0], [2, 2, 5, -1, -1, -1], [0, 2, 9, 1, 4, -1]][:B]
    full = [pool(dev, "f16", *shape[:-1], 128 if wide else 64, seed=s) for s in (3, 4)]
    k, v = (f[..., 32:96] if wide else f for f in full)
    want = [f.clone() for f in full]
    for w, f in zip(want, full):
        w4, f4 = (x.view(-1, B, 50, x.shape[-1]) for x in (w, f.clone()))
        c = slice(32, 96) if wide else slice(None)
        for b in range(B):
            for j in range(count[b]):
                s, d = lens[b] + path[b][j], lens[b] + j
                if path[b][j] >= 0 and s < 50 and d < 50:
                    w4[:, b, d, c] = f4[:, b, s, c]
    new = A.kv_accept(k, v, i32(path, dev), i32(count, dev), i32(lens, dev))
    assert new.tolist() == [a + b for a, b in zip(lens, count)]
    for w, f in zip(want, full):
        assert torch.equal(w, f)


def test_accept_counts_outside_their_range(dev):
    k = pool(dev, "f16", 40, 64)
    old = k.clone()
    out = A.kv_accept(k, k.clone(), i32([[3, 2]], dev), i32([-4], dev), i32([7], dev))
    assert out.tolist() == [7] and torch.equal(k, old)
    out = A.kv_accept(k, k.clone(), i32([[3, 2]], dev), i32([99], dev), i32([7], dev))
    assert out.tolist() == [9] and torch.equal(k[7], old[10]) and torch.equal(k[8], old[9])
    out = A.kv_accept(k, k.clone(), i32(np.zeros((1, 0)), dev), i32([1], dev), i32([7], dev))
    assert out.tolist() == [7]


def update_ref(table, lens, parent, cap, held, n_pages, P, cols):
    """(table, lens, info, copies (source, to, positions)), sequence by sequence."""
    S, stride = table.shape
    todo, used = [], {i for i in range(n_pages) if held is not None and held[i]}
    ok = lambda pg: 0 <= pg < n_pages  # noqa: E731
    for p, c in zip(parent, cap):
        c = min(max(c, 0), cols * P)
        kept = min(max(lens[p], 0), stride * P, c) if 0 <= p < S else 0
        row = [int(x) if ok(x) else -1 for x in table[p]] if 0 <= p < S else []
        todo.append((row, kept, -(-c // P)))
        used |= {x for x in row[:kept // P] if x >= 0}
    owner = {}
    for s, (row, kept, _) in enumerate(todo):
        if kept % P and row[kept // P] >= 0 and row[kept // P] not in used:
            owner.setdefault(row[kept // P], s)
    lasts = {row[kept // P] for row, kept, _ in todo if kept % P}
    free = [i for i in range(n_pages) if i not in used and i not in lasts]
    out, new_lens, copies, asked = np.full((len(todo), cols), -1, np.int32), [], [], 0
    for s, (row, kept, need) in enumerate(todo):
        full, part = divmod(kept, P)
        out[s, :full] = row[:full]
        j, last = full, row[full] if part else -1
        if last >= 0 and owner.get(last) == s:
            out[s, j], j = last, j + 1
        elif last >= 0:
            if asked < len(free):
                copies.append((last, free[asked], part))
            else:
                kept = full * P
        for i in range(j, need):
            out[s, i] = free[asked] if asked < len(free) else -1
            asked += 1
        new_lens.append(kept)
    return out, new_lens, [len(copies), min(asked, len(free)), max(asked - len(free), 0)], copies


def run_update(dev, dt, NL, n_pages, P, kvd, table, lens, parent, cap, held, cols, stacked=True):
    k, v = (pool(dev, dt, *((NL,) if stacked else ()), n_pages, P, kvd, seed=s) for s in (5, 6))
    want = [x.clone().view(NL, n_pages, P, kvd) for x in (k, v)]
    wt, wl, wi, copies = update_ref(table, lens, parent, cap, held, n_pages, P, cols)
    for x in want:
        old = x.clone()
        for src, to, n in copies:
            x[:, to, :n] = old[:, src, :n]
    args = (k, v, i32(table, dev), i32(lens, dev), i32(parent, dev), i32(cap, dev))
    got = A.kv_pages_update(*args, held=None if held is None else torch.tensor(held, device=dev), table_stride=cols)
    assert got[2].tolist() == wi
    assert got[1].tolist() == wl
    assert torch.equal(got[0].cpu(), torch.from_numpy(wt))
    for x, y in zip(want, (k, v)):
        assert torch.equal(x.view(torch.int16 if dt != "f32" else torch.int32), y.view_as(x).view(torch.int16 if dt != "f32" else torch.int32))
    return wt, wl


@pytest.mark.parametrize("seed", range(12))
def test_update_random_steps(dev, seed):
    """Steps of forks, cuts, growth, ends and begins on one table, with invalid
    entries, held pages, tables that widen and narrow, and pools that run out."""
    rng = np.random.default_rng(seed)
    dt, P = ["f32", "f16", "bf16"][seed % 3], int(rng.choice([1, 2, 32, 64]))
    NL, kvd, S = int(rng.integers(1, 4)), int(rng.choice([8, 64, 136])), int(rng.integers(1, 40))
    cols = int(rng.integers(1, 12))
    n_pages = int(rng.integers(1, max(2, S * cols)))
    table, lens = np.full((S, cols), -1, np.int32), [0] * S
    for step in range(5):
        n, new_cols = int(rng.integers(1, 45)), int(rng.integers(1, 14))
        parent = rng.integers(-2, len(lens) + 2, n)
        if step % 2 == 0 and n <= len(lens):
            parent = np.arange(n)
        cap = rng.integers(-1, new_cols * P + 3, n)
        held = rng.random(n_pages) < 0.1 if step % 3 == 1 else None
        if step == 3:
            table[rng.random(table.shape) < 0.1] = rng.choice([-7, n_pages, 1 << 30])
        print(f"[pages] seed {seed} step {step}: {len(lens)} -> {n} sequences, {n_pages} pages of {P}", flush=True)
        table, lens = run_update(dev, dt, NL, n_pages, P, kvd, table, lens, parent, cap, held, new_cols, NL > 1)


@pytest.mark.parametrize("n_pages,S,cols", [(1 << 20, 1500, 300), (33, 3000, 1), (70000, 64, 1024)])
def test_update_large(dev, n_pages, S, cols):
    """More pages than a workgroup has threads times words, more sequences than
    threads."""
    rng = np.random.default_rng(S)
    lens = rng.integers(0, cols * 2 + 1, S)
    table = rng.permutation(max(n_pages, S * cols))[:S * cols].reshape(S, cols) % n_pages
    parent = rng.integers(-1, S, S)
    cap = np.minimum(lens[parent] + rng.integers(-3, 5, S), cols * 2)
    held = rng.random(n_pages) < 0.3
    run_update(dev, "f16", 1, n_pages, 2, 8, table.astype(np.int32), lens.tolist(), parent, cap, held, cols, False)


def test_update_forks_share_and_copy(dev):
    """Three beams from one: the whole page is shared, the first keeps the part-filled
    one, the others get copies of its filled rows only."""
    k, v = pool(dev, "bf16", 2, 8, 32, 64, seed=1), pool(dev, "bf16", 2, 8, 32, 64, seed=2)
    old = k.clone(), v.clone()
    table, lens, info = A.kv_pages_update(k, v, i32([[6, 3, -1]], dev), i32([40], dev), i32([0, 0, 0], dev), i32([41, 41, 65], dev))
    assert table.tolist() == [[6, 3, -1], [6, 0, -1], [6, 1, 2]] and lens.tolist() == [40] * 3 and info.tolist() == [2, 3, 0]
    for x, o in zip((k, v), old):
        for pg in (0, 1):
            assert torch.equal(x[:, pg, :8], o[:, 3, :8]) and torch.equal(x[:, pg, 8:], o[:, pg, 8:])
        assert torch.equal(x[:, 2:], o[:, 2:])
    # freed again, and a held part-filled page is never given away or written
    table, lens, info = A.kv_pages_update(k, v, table, lens, i32([1, -1], dev), i32([41, 0], dev))
    assert table.tolist() == [[6, 0, -1], [-1] * 3] and info.tolist() == [0, 0, 0]
    held = torch.zeros(8, dtype=torch.bool, device=dev)
    held[0] = True
    table, lens, info = A.kv_pages_update(k, v, table, lens, i32([0], dev), i32([41], dev), held=held)
    assert table.tolist() == [[6, 1, -1]] and info.tolist() == [1, 1, 0]


def test_update_nothing(dev):
    k = pool(dev, "f16", 4, 32, 64)
    none = i32([], dev)
    table, lens, info = A.kv_pages_update(k, k.clone(), i32([[0, 1]], dev), i32([40], dev), none, none)
    assert table.shape == (0, 2) and lens.numel() == 0 and info.tolist() == [0, 0, 0]
    # from no sequence at all
    table, lens, info = A.kv_pages_update(k, k.clone(), i32(np.zeros((0, 3)), dev), none, i32([-1, 0], dev), i32([33, 64], dev))
    assert table.tolist() == [[0, 1, -1], [2, 3, -1]] and lens.tolist() == [0, 0] and info.tolist() == [0, 4, 0]


def test_update_given_outputs_and_graph(dev):
    """Captured with its outputs given and the lengths updated in place, replayed on
    new tables."""
    rng = np.random.default_rng(2)
    S, cols, P, n_pages = 9, 5, 32, 60
    k, v = pool(dev, "f16", 2, n_pages, P, 64, seed=1), pool(dev, "f16", 2, n_pages, P, 64, seed=2)
    table, lens, parent, cap = i32(np.zeros((S, cols)), dev), i32([0] * S, dev), i32([0] * S, dev), i32([0] * S, dev)
    to, info = i32(np.zeros((S, cols)), dev), i32([0] * 3, dev)
    ws = torch.empty(L.lib().ullm_hip_kv_pages_workspace_bytes(S, n_pages), dtype=torch.uint8, device=dev)
    call = lambda: A.kv_pages_update(k, v, table, lens, parent, cap, table_out=to, lens_out=lens, info=info, workspace=ws)  # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = call()
    assert got[0] is to and got[1] is lens and got[2] is info
    for i in range(5):
        ln = rng.integers(0, cols * P, S)
        tb = rng.permutation(n_pages)[:S * cols].reshape(S, cols)
        par, cp = rng.integers(-1, S, S), rng.integers(0, cols * P, S)
        for x, y in ((table, tb), (lens, ln), (parent, par), (cap, cp)):
            x.copy_(i32(y, dev))
        kc, vc = k.clone(), v.clone()
        wt, wl, wi, copies = update_ref(tb, ln, par, cp, None, n_pages, P, cols)
        for src, dst, n in copies:
            for x, o in ((kc, k), (vc, v)):
                x[:, dst, :n] = o[:, src, :n]
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(to.cpu(), torch.from_numpy(wt)) and lens.tolist() == wl and info.tolist() == wi
        assert torch.equal(k, kc) and torch.equal(v, vc)


def test_offsets_past_32_bits(dev):
    """Rows and pages beyond 4 GiB of a pool of two layers."""
    n_pages, P, kvd = 70000, 32, 1024
    k, v = (torch.empty(2, n_pages, P, kvd, device=dev, dtype=torch.float16) for _ in "kv")
    last = n_pages - 1
    for i, x in enumerate((k, v)):
        x[:, last] = pool(dev, "f16", 2, P, kvd, seed=i)
    row = [x[:, last, 5].clone() for x in (k, v)]
    A.kv_accept_paged(k, v, i32([[last]], dev), i32([[3]], dev), i32([1], dev), i32([2], dev))
    for x, r in zip((k, v), row):
        assert torch.equal(x[:, last, 2], r)
    held = torch.ones(n_pages, dtype=torch.bool, device=dev)
    held[last - 1] = held[last] = False
    table, _, info = A.kv_pages_update(k, v, i32([[last]], dev), i32([9], dev), i32([0, 0], dev), i32([10, 10], dev), held=held)
    assert table.tolist() == [[last], [last - 1]] and info.tolist() == [1, 1, 0]
    for x in (k, v):
        assert torch.equal(x[:, last - 1, :9], x[:, last, :9])


def test_refusals(dev):
    k, t, n = pool(dev, "f16", 4, 32, 64), i32([[0, 1]], dev), i32([40], dev)
    one = i32([0], dev)
    for bad in (
        lambda: A.kv_pages_update(k.cpu(), k, t, n, one, one),
        lambda: A.kv_pages_update(k, k[:2], t, n, one, one),
        lambda: A.kv_pages_update(k, k, t.long(), n, one, one),
        lambda: A.kv_pages_update(k, k, t, n.long(), one, one),
        lambda: A.kv_pages_update(k, k, t, n, one, i32([0, 1], dev)),
        lambda: A.kv_pages_update(k, k, t, n, one, one, held=torch.zeros(3, dtype=torch.bool, device=dev)),
        lambda: A.kv_pages_update(k, k, t, n, one, one, table_out=t),
        lambda: A.kv_pages_update(k, k, t, n, one, one, workspace=torch.empty(16, dtype=torch.uint8, device=dev)),
        lambda: A.kv_pages_update(k[:, ::2], k[:, ::2], t, n, one, one, table_stride=0),
        lambda: A.kv_pages_update(k.transpose(0, 1), k.transpose(0, 1), t, n, one, one),
        lambda: A.kv_accept_paged(k, k, t, i32([[0]], dev), one, n, lens_out=n),
        lambda: A.kv_accept_paged(k, k, t, i32([[0]], dev), one.float(), n),
        lambda: A.kv_accept_paged(k[..., :4], k[..., :4], t, i32([[0]], dev), one, n),
        lambda: A.kv_accept_paged(k, k, t[:0], i32([[0]], dev), one, n),
        lambda: A.kv_accept(k, k, i32([[0], [0]], dev), i32([1, 1], dev), i32([1, 1], dev)),
        lambda: A.kv_accept(k[0].expand(3, 32, 64), k[0].expand(3, 32, 64), i32([[0]], dev), one, n),
        lambda: A.kv_accept(k[..., 1:33], k[..., 1:33], i32([[0]], dev), one, n),
    ):
        with pytest.raises(L.UllmHipError):
            bad()
