"""tree_verify on the GPU against the same rules in 64 bits, sequence by sequence.
Everything that comes back is whole numbers: equal, never near."""
import math

import numpy as np
import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rule(p, q, tokens, u, parents, n, distinct):
    """One sequence: (path, next token); p [T + 1, V], q [T, V] or None, in 64 bits."""
    clean = lambda x: np.where((x > 0) & (x < np.inf), x, 0.0)  # noqa: E731
    p, q = clean(p), None if q is None else clean(q)
    u = np.nan_to_num(u, nan=0.0).clip(0, 1 - 2.0 ** -24)
    path, cur = [], -1
    while True:
        rest, mass, left = p[cur + 1].copy(), 1.0, 1.0
        for i in range(cur + 1, n):
            x = tokens[i]
            if max(parents[i], -1) != cur or not 0 <= x < p.shape[1]:
                continue
            share = mass if q is None else q[cur + 1, x] / left * mass
            if rest[x] > 0 and u[i] * share < rest[x]:
                path.append(i)
                cur = i
                break
            if q is None:
                mass = max(mass - rest[x], 0.0)
                rest[x] = 0
            else:
                rest = np.maximum(rest - q[cur + 1] * (mass / left), 0)
                mass = math.fsum(rest)
                if distinct:
                    left = max(left - q[cur + 1, x], 2.0 ** -24)
        else:
            break
    if not rest.sum() > 0:
        rest = p[cur + 1]
    sums = np.cumsum(rest)
    return path, int(np.searchsorted(sums, u[-1] * sums[-1], side="right")) if sums[-1] > 0 else -1


def check(p, q, tokens, u, parents=None, n=None, distinct=False, **more):
    B, T = tokens.shape
    path, count, nxt = A.tree_verify(p, q, tokens, u, parents=parents, n_nodes=n, distinct=distinct, **more)
    assert path.shape == (B, T) and path.dtype == count.dtype == nxt.dtype == torch.int32
    chain = np.arange(T) - 1
    host = lambda x: x.double().cpu().numpy()  # noqa: E731
    for b in range(B):
        want, token = rule(host(p[b]), None if q is None else host(q[b]), tokens[b].tolist(), host(u[b]),
                           chain if parents is None else parents[b].tolist(),
                           T if n is None else min(max(int(n[b]), 0), T), distinct)
        assert path[b].tolist() == want + [-1] * (T - len(want)), b
        assert count[b].item() == len(want) and nxt[b].item() == token, (b, nxt[b].item(), token)
    return path, count, nxt


def trees(rng, B, T, fan):
    par = np.full((B, T), -1, np.int32)
    for b in range(B):
        room = [fan] * (T + 1)
        for i in range(T):
            free = [j for j in range(i + 1) if room[j]]
            j = free[-1] if rng.random() < 0.5 else rng.choice(free)
            room[j] -= 1
            par[b, i] = j - 1
    return par


def make(dev, B, T, V, dt="f32", fan=1, kind="probs", seed=0, noise=0.7, cut=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    logits = 4 * torch.randn(B, T + 1, V, device=dev, generator=g)
    p = torch.softmax(logits, -1)
    ql = logits[:, :T] + noise * torch.randn(B, T, V, device=dev, generator=g)
    q = torch.softmax(ql, -1)
    if cut:
        p, q = (torch.where(x < cut, 0.0, x) for x in (p, q))
        p, q = (x / x.sum(-1, keepdim=True).clamp(min=1e-30) for x in (p, q))
    p, q = p.to(DT[dt]), q.to(DT[dt])
    par = trees(rng, B, T, fan)
    tokens = np.zeros((B, T), np.int32)
    qh = q.double().cpu().numpy()
    for b in range(B):
        used = {}
        for i in range(T):
            row = qh[b, par[b, i] + 1].copy()
            if kind != "probs":
                row[used.setdefault(par[b, i], [])] = 0
            x = rng.choice(V, p=row / row.sum()) if kind != "lookup" and row.sum() > 0 else int(row.argmax())
            used.setdefault(par[b, i], []).append(x)
            tokens[b, i] = x
    u = torch.rand(B, T + 1, device=dev, generator=g)
    return (p, None if kind == "lookup" else q, torch.from_numpy(tokens).to(dev), u,
            torch.from_numpy(par).to(dev))


@pytest.mark.parametrize("kind", ["probs", "distinct", "lookup"])
@pytest.mark.parametrize("B,T,V,fan,dt", [
    (1, 1, 5, 1, "f32"), (3, 4, 1000, 1, "f32"), (2, 7, 32001, 1, "bf16"), (5, 9, 4099, 2, "f16"), (4, 26, 20011, 4, "f32"),
    (3, 12, 513, 7, "bf16"), (2, 40, 777, 40, "f32"), (33, 3, 100, 3, "f32"), (1, 5, 131072, 5, "f16")])
def test_against_64_bits(dev, kind, B, T, V, fan, dt):
    p, q, tok, u, par = make(dev, B, T, V, dt, fan, kind, seed=B * 100 + T)
    n = torch.tensor([T - (b % 3) for b in range(B)], dtype=torch.int32, device=dev)
    check(p, q, tok, u, par, n, kind == "distinct")


@pytest.mark.parametrize("kind", ["probs", "distinct", "lookup"])
def test_many_rejections(dev, kind):
    """A draft that is far off, probabilities with their tails cut: most nodes are
    rejected, residuals shrink to a few tokens or to nothing."""
    for seed in range(4):
        p, q, tok, u, par = make(dev, 6, 16, 300, fan=8, kind=kind, seed=seed, noise=5.0, cut=1e-3)
        check(p, q, tok, u, par, None, kind == "distinct")


def test_sequence_alone_and_whole_chains(dev):
    p, q, tok, u, par = make(dev, 4, 6, 999)
    # no nodes: a token from row 0
    _, count, _ = check(p[:, :1].contiguous(), None, tok[:, :0].contiguous(), u[:, :1].contiguous())
    assert count.tolist() == [0] * 4
    check(p, q, tok, u, None, torch.tensor([0, 6, -3, 99], dtype=torch.int32, device=dev))
    # a draft that is the target itself keeps every node
    _, count, _ = check(p, p[:, :6].contiguous(), torch.ones_like(tok), u)
    assert count.tolist() == [6] * 4


def test_longest_chain(dev):
    p = torch.full((1, 1025, 3), 1 / 3, device=dev)
    tok = torch.ones(1, 1024, dtype=torch.int32, device=dev)
    u = torch.rand(1, 1025, device=dev)
    path, count, _ = check(p, p[:, :1024].contiguous(), tok, u)
    assert count.item() == 1024 and path[0].tolist() == list(range(1024))


def test_ends_of_the_unit_interval(dev):
    """u = 0 takes the first token of any weight, the largest u the last; numbers
    outside [0, 1) count as the nearest inside, NaN as 0."""
    p = torch.zeros(6, 1, 1500, device=dev)
    p[:, 0, 700], p[:, 0, 701], p[:, 0, 1400] = 0.25, 0.5, 0.25
    u = torch.tensor([[0.0], [1 - 2.0 ** -24], [1.0], [-1.0], [float("nan")], [float("inf")]], device=dev)
    none = torch.zeros(6, 0, dtype=torch.int32, device=dev)
    _, _, nxt = check(p, None, none, u)
    assert nxt.tolist() == [700, 1400, 1400, 700, 700, 1400]


def test_equal_probabilities_fall_between_tokens(dev):
    """2^10 tokens of 2^-10: u = k 2^-10 lies on a border and takes token k."""
    k = torch.arange(0, 1024, 31, device=dev)
    p = torch.full((len(k), 1, 1024), 2.0 ** -10, device=dev)
    _, _, nxt = A.tree_verify(p, None, torch.zeros(len(k), 0, dtype=torch.int32, device=dev), (k / 1024.0)[:, None])
    assert nxt.tolist() == k.tolist()


def test_what_is_no_probability(dev):
    p, q, tok, u, par = make(dev, 5, 4, 600, fan=2)
    for x in (p, q):
        x[:, :, ::7] = float("nan")
        x[:, :, 1::11] = float("inf")
        x[:, :, 2::13] = -1.0
    check(p, q, tok, u, par)
    check(p, None, tok, u, par)
    p[1:3] = 0.0
    p[3] = float("nan")
    _, _, nxt = check(p, q, tok, u, par)
    assert nxt[1:4].tolist() == [-1] * 3


def test_odd_nodes(dev):
    """Tokens outside the vocabulary are passed over, parents at or behind their node
    are never reached, equal siblings are each drawn anew."""
    p, q, tok, u, par = make(dev, 4, 8, 50, fan=3, seed=5)
    tok[0, ::2] = torch.tensor([-1, 50, 1 << 30, -(1 << 31)], dtype=torch.int32, device=dev)
    tok[1] = tok[1, 0]
    par[2, 3:] = torch.tensor([3, 7, 8, 100, 1 << 30], dtype=torch.int32, device=dev)
    par[3] = torch.tensor([-5, -1, -(1 << 31), 0, 0, 1, 2, 2], dtype=torch.int32, device=dev)
    for distinct in (False, True):
        check(p, q, tok, u, par, None, distinct)
    check(p, None, tok, u, par)


def test_rows_at_any_stride(dev):
    """Views of wider buffers: a padded vocabulary, sequences apart, rows that begin
    at any element."""
    for dt in ("f32", "bf16"):
        p, q, tok, u, par = make(dev, 3, 5, 1003, dt, 2, seed=3)
        wide_p = torch.full((3, 9, 1031), float("nan"), dtype=DT[dt], device=dev)
        wide_q = torch.full((3, 7, 1013), float("nan"), dtype=DT[dt], device=dev)
        vp, vq = wide_p[:, 1:7, 3:1006], wide_q[:, 2:, 5:1008]
        vp.copy_(p)
        vq.copy_(q)
        check(vp, vq, tok, u, par)


def test_given_outputs_and_stream(dev):
    p, q, tok, u, par = make(dev, 3, 5, 5000, fan=2)
    path, count, nxt = (torch.full(s, 77, dtype=torch.int32, device=dev) for s in ((3, 5), (3,), (3,)))
    ws = torch.full((L.lib().ullm_hip_tree_verify_workspace_bytes(5000, 3),), 255, dtype=torch.uint8, device=dev)
    got = A.tree_verify(p, q, tok, u, parents=par)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    out = A.tree_verify(p, q, tok, u, parents=par, path=path, n_accept=count, next_token=nxt, workspace=ws, stream=st)
    st.synchronize()
    for a, b, c in zip(out, (path, count, nxt), got):
        assert a.data_ptr() == b.data_ptr() and torch.equal(a, c)


def test_front_refuses(dev):
    p, q, tok, u, par = make(dev, 2, 3, 64)
    for bad in (dict(draft=q[:, :2]), dict(draft=q.half()), dict(tokens=tok.long()), dict(tokens=tok[:, :2]), dict(uniform=u[:, :3]),
                dict(uniform=u.double()), dict(parents=par[:1]), dict(n_nodes=tok), dict(target=p.double()),
                dict(target=p.transpose(1, 2)), dict(path=tok[:, :2].contiguous()), dict(path=tok), dict(n_accept=tok),
                dict(next_token=u), dict(workspace=torch.empty(8, dtype=torch.uint8, device=dev))):
        a = {**dict(target=p, draft=q, tokens=tok, uniform=u, parents=par), **bad}
        with pytest.raises(L.UllmHipError):
            A.tree_verify(a.pop("target"), a.pop("draft"), a.pop("tokens"), a.pop("uniform"), **a)


@pytest.mark.parametrize("kind", ["probs", "distinct", "lookup"])
def test_what_comes_out_is_the_target(dev, kind):
    """The first token that comes out of a tree of 3 children is distributed as the
    target's row, whatever the draft: 2^16 independent trees over 6 tokens, each
    frequency within 5 standard deviations."""
    N, V = 1 << 16, 6
    g = torch.Generator(device=dev).manual_seed(11)
    p = torch.tensor([0.3, 0.05, 0.25, 0.1, 0.0, 0.3], device=dev)
    q = torch.tensor([0.1, 0.4, 0.2, 0.2, 0.05, 0.05], device=dev)
    if kind == "lookup":
        tok = torch.tensor([1, 0, 2], device=dev).expand(N, 3)
    else:
        tok = torch.multinomial(q.expand(N, V), 3, replacement=kind == "probs", generator=g)
    tok = tok.int().contiguous()
    u = torch.rand(N, 4, device=dev, generator=g)
    counts = torch.zeros(V, dtype=torch.float64, device=dev)
    for lo in range(0, N, 1 << 14):
        s = slice(lo, lo + (1 << 14))
        m = 1 << 14
        path, count, nxt = A.tree_verify(p.expand(m, 4, V), None if kind == "lookup" else q.expand(m, 3, V), tok[s], u[s],
                                         parents=torch.full((m, 3), -1, dtype=torch.int32, device=dev),
                                         distinct=kind == "distinct")
        first = torch.where(count > 0, torch.gather(tok[s], 1, path[:, :1].clamp(min=0).long())[:, 0], nxt)
        counts += torch.bincount(first.long(), minlength=V).double()
    e = N * p.double()
    assert ((counts - e).abs() <= 5 * (e * (1 - p.double())).sqrt()).all(), counts


def test_captured_and_replayed(dev):
    p, q, tok, u, par = make(dev, 3, 6, 9000, fan=3, seed=2)
    out = A.tree_verify(p, q, tok, u, parents=par)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A.tree_verify(p, q, tok, u, parents=par)
    for r in range(4):
        u.copy_(torch.rand(u.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(r)))
        graph.replay()
        out = A.tree_verify(p, q, tok, u, parents=par)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, out))
