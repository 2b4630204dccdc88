"""The operators that decide what a cache keeps, as a serving loop runs them: drafted
trees appended and attended over a paged cache, verified, their accepted rows moved
together, the weights of the cache collected, and the cache cut to a budget where it
has grown past it; against the same steps in 64 bits over rows kept on the host's side.

Decisions (which nodes, tokens and positions are kept) are equal.  Attention over f16:
the output's rounding is half a step, 2^-11 of its value, and a weight is off by twice
its score's error (D + 12) 2^-24 S, S the largest sum of |q||k| scale, with a sum of n
keys n 2^-24: all of it times the largest |v|.  Collected weights as in
test_key_weights_gpu.py, summed over the steps."""
import math

import numpy as np
import pytest
import torch

from ullm_amd import attention as A

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def verify_rule(p, q, tokens, u, parents, n):
    path, cur = [], -1
    while True:
        rest, mass, left, found = p[cur + 1].copy(), 1.0, 1.0, None
        for i in range(cur + 1, n):
            if parents[i] != cur:
                continue
            x = tokens[i]
            if rest[x] > 0 and u[i] * (q[cur + 1, x] / left * mass) < rest[x]:
                found = i
                break
            rest = np.maximum(rest - q[cur + 1] * (mass / left), 0)
            mass, left = math.fsum(rest), max(left - q[cur + 1, x], 2.0 ** -24)
        if found is None:
            break
        path.append(found)
        cur = found
    if not rest.sum() > 0:
        rest = p[cur + 1]
    sums = np.cumsum(rest)
    return path, int(np.searchsorted(sums, u[-1] * sums[-1], side="right"))


@pytest.mark.parametrize("budget,sink,recent", [(40, 2, 16), (64, 0, 0), (25, 4, 21)])
def test_serving_loop_with_a_budget(dev, budget, sink, recent):
    NL, B, T, H, Hk, D, P, V = 2, 3, 7, 6, 2, 64, 32, 331
    gq, cols, n_pages, limit = H // Hk, 6, 20, budget + 20
    g = torch.Generator(device=dev).manual_seed(budget)
    rng = np.random.default_rng(budget)
    kp, vp = (torch.zeros(NL, n_pages, P, Hk * D, dtype=torch.float16, device=dev) for _ in "kv")
    rope = A.rope_table(4096, D, 1e4, dev)
    lens, table = i32([0, 0, 0], dev), torch.full((B, cols), -1, dtype=torch.int32, device=dev)
    room = cols * P
    acc = torch.zeros(NL, B, Hk, room, device=dev)
    pos_true = np.zeros(B, np.int64)  # tokens so far, evicted ones too
    # the host's rows: [layer][sequence][kv head] -> list of (k, v), and their collected weights and tolerances
    rows = [[[[] for _ in range(Hk)] for _ in range(B)] for _ in range(NL)]
    got = [[[[] for _ in range(Hk)] for _ in range(B)] for _ in range(NL)]
    evictions = 0
    for step in range(100):
        # room for the drafts
        n_host = lens.tolist()
        table, lens2, info = A.kv_pages_update(kp, vp, table, lens, i32(range(B), dev), i32([n + T for n in n_host], dev))
        assert info[2].item() == 0 and lens2.tolist() == n_host
        par = np.array([[-1] + [int(rng.integers(-1, i)) for i in range(1, T)] for _ in range(B)], np.int32)
        mask, depth = A.tree_masks(par)
        positions = i32(pos_true[:, None] + depth.numpy(), dev)
        nodes = i32([T, T - 2, T], dev)
        q_rows = []
        for lay in range(NL):
            q, k, v = (torch.randn(B, T, n * D, device=dev, generator=g) for n in (H, Hk, Hk))
            qo = A.qkv_append_tree_paged(q, k, v, kp[lay], vp[lay], rope, lens, positions, table, n_head=H, n_kv_head=Hk, head_dim=D,
                                         n_nodes=nodes, q_dtype=torch.float16)
            out = A.attn_tree_paged(qo.view(B, T, H, D), kp[lay], vp[lay], table, mask.to(dev), lens, max(n_host) + T, Hk,
                                    n_nodes=nodes, positions=positions)
            q_rows.append(qo.view(B, T, H, D))
            for b in range(B):
                tab, m = table[b].tolist(), int(nodes[b])
                at = torch.tensor([tab[t // P] * P + t % P for t in range(n_host[b], n_host[b] + m)], device=dev)
                new_k, new_v = (x[lay].view(-1, Hk, D)[at].double().cpu().numpy() for x in (kp, vp))
                bits = mask[b, :, 0].tolist()
                for j in range(Hk):
                    ks = np.array([r[0] for r in rows[lay][b][j]] + list(new_k[:, j]))
                    vs = np.array([r[1] for r in rows[lay][b][j]] + list(new_v[:, j]))
                    see = np.ones((m, len(ks)), bool)
                    see[:, n_host[b]:] = [[bits[i] >> c & 1 for c in range(m)] for i in range(m)]
                    for h in range(j * gq, (j + 1) * gq):
                        qh = qo.view(B, T, H, D)[b, :m, h].double().cpu().numpy()
                        s = np.where(see, qh @ ks.T / 8, -np.inf)
                        w = np.exp(s - s.max(1, keepdims=True))
                        want = w / w.sum(1, keepdims=True) @ vs
                        err = np.abs(out[b, :m, h].double().cpu().numpy() - want)
                        most = (np.abs(qh) @ np.abs(ks).T / 8).max()
                        tol = 2.0 ** -11 * np.abs(want) + (2 * (D + 12) * most + len(ks) + 20) * U * np.abs(vs).max() + 2.0 ** -24
                        assert (err <= tol).all(), (step, lay, b, h, (err - tol).max())
        # which nodes are kept
        logits = 2 * torch.randn(B, T + 1, V, device=dev, generator=g)
        p = torch.softmax(logits, -1)
        qd = torch.softmax(logits[:, :T] + 0.5 * torch.randn(B, T, V, device=dev, generator=g), -1)
        tokens = np.zeros((B, T), np.int32)
        for b in range(B):
            used = {}
            for i in range(T):
                w = qd[b, par[b, i] + 1].double().cpu().numpy().copy()
                w[used.setdefault(par[b, i], [])] = 0
                tokens[b, i] = rng.choice(V, p=w / w.sum())
                used[par[b, i]].append(tokens[b, i])
        u = torch.rand(B, T + 1, device=dev, generator=g)
        path, count, nxt = A.tree_verify(p, qd, i32(tokens, dev), u, parents=i32(par, dev), n_nodes=nodes, distinct=True)
        for b in range(B):
            want, tok = verify_rule(p[b].double().cpu().numpy(), qd[b].double().cpu().numpy(), tokens[b], u[b].double().cpu().numpy(),
                                    par[b], int(nodes[b]))
            assert path[b].tolist() == want + [-1] * (T - len(want)) and count[b].item() == len(want) and nxt[b].item() == tok
        # their rows together; the host reads what they held
        for lay in range(NL):
            for b in range(B):
                tab = table[b].tolist()
                for i in path[b, :count[b]].tolist():
                    t = n_host[b] + i
                    r = tab[t // P] * P + t % P
                    k, v = (x[lay].view(-1, Hk, D)[r].double().cpu().numpy() for x in (kp, vp))
                    for j in range(Hk):
                        rows[lay][b][j].append((k[j], v[j]))
                        got[lay][b][j].append([0.0, 0.0])
        lens = A.kv_accept_paged(kp, vp, table, path, count, lens)
        pos_true += count.cpu().numpy()
        n_host = lens.tolist()
        # the weights that the accepted rows give
        for lay in range(NL):
            qa = torch.gather(q_rows[lay], 1, path.clamp(min=0).long()[:, :, None, None].expand(B, T, H, D))
            A.key_weights_paged(qa, kp[lay], table, acc[lay], lens, max(max(n_host), 1), Hk, n_rows=count)
            for b in range(B):
                n, r = n_host[b], count[b].item()
                for j in range(Hk):
                    if not n or not r:
                        continue
                    ks = np.array([x[0] for x in rows[lay][b][j]])
                    add = np.zeros(n)
                    most = 0.0
                    for h in range(j * gq, (j + 1) * gq):
                        qh = qa[b, :r, h].double().cpu().numpy()
                        s = qh @ ks.T / 8
                        s[np.arange(n)[None] > (n - r + np.arange(r))[:, None]] = -np.inf
                        w = np.exp(s - s.max(1, keepdims=True))
                        add += (w / w.sum(1, keepdims=True)).sum(0)
                        most = max(most, (np.abs(qh) @ np.abs(ks).T / 8).max())
                    rel = 2 * ((D + 12) * U * most + 6 * U) + (n + r * gq + 12) * U
                    for t, e in enumerate(got[lay][b][j]):
                        e[1] += add[t] * rel + (e[0] + add[t]) * 4 * U
                        e[0] += add[t]
                    have = acc[lay, b, j, :n].double().cpu().numpy()
                    assert (np.abs(have - [e[0] for e in got[lay][b][j]]) <= [e[1] + 1e-30 for e in got[lay][b][j]]).all()
        if max(n_host) <= limit:
            continue
        evictions += 1
        before = acc.cpu().numpy().copy()
        kept, new = A.kv_evict_paged(kp, vp, table, acc, lens, i32([budget] * B, dev), max_budget=budget, sink=sink, recent=recent)
        assert new.tolist() == [min(n, budget) for n in n_host]
        for lay in range(NL):
            for b in range(B):
                n, m = n_host[b], min(n_host[b], budget)
                for j in range(Hk):
                    first = min(sink, m)
                    last = min(recent, m - first)
                    x = before[lay, b, j, :n]
                    mid = np.arange(first, n - last)
                    best = mid[np.lexsort((mid, -x[mid]))][:m - first - last]
                    stay = np.concatenate((np.arange(first), np.sort(best), np.arange(n - last, n))) if m < n else np.arange(n)
                    assert kept[lay, b, j, :m].tolist() == stay.tolist() and (kept[lay, b, j, m:] == -1).all()
                    rows[lay][b][j] = [rows[lay][b][j][t] for t in stay]
                    got[lay][b][j] = [got[lay][b][j][t] for t in stay]
                    assert acc[lay, b, j, :m].tolist() == x[stay].tolist() and (acc[lay, b, j, m:n] == 0).all()
        lens = new
        if evictions == 4:
            break
    assert evictions == 4 and pos_true.min() > 5
