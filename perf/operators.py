"""Cases of the operators that decode several drafted tokens at once over a
shared cache: what a serving loop with speculative decoding and beams has
`ullm_amd.attention` do.

A case is a dict of plain values.  `op` names the call:

  attn_tree    attention of a tree of drafted tokens over the cache that holds
               their sequence and themselves (attn_tree, attn_tree_paged)
  append_tree  bias, Q/K norm and RoPE of the drafted tokens, each at its depth
               in the tree, and the store of their K and V rows behind the
               sequence (qkv_append_tree_paged)
  accept       the rows of the accepted path moved together behind the
               sequence, in every layer (kv_accept_paged)
  pages        the block table of the next step: sequences that go on, fork,
               end and begin, pages shared, copied where two would write one,
               taken and given back (kv_pages_update)

`prepare` makes the inputs on the GPU from the seed, `run` is one pass: the
operator in elementary torch operations, or where `own` is true the call.
`exact` is the same result in 64 bits, sequence by sequence.
"""
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6

# Attention shapes (n_head, n_kv_head, head_dim): those of the attention cases
# beside this file, and groups of 5 and 7 heads, which fill no power of two.
SHAPES = [(32, 8, 64), (12, 2, 128), (32, 8, 128), (8, 4, 256), (32, 4, 128), (40, 8, 128), (14, 2, 64)]


def listed():
    return [
        # The smallest call: three drafted tokens behind a short prompt, a
        # small model in the reference's own f32 cache.
        dict(name="tree_f32_3_short", op="attn_tree", kv="f32", heads=32, kv_heads=8, dim=64,
             batch=1, nodes=3, lo=37, hi=37, page=0, window=0),
        # One conversation of a small model at 4K, a tree of 26 nodes.
        dict(name="tree_f16_26_4k", op="attn_tree", kv="f16", heads=12, kv_heads=2, dim=128,
             batch=1, nodes=26, lo=4095, hi=4095, page=0, window=0),
        # A serving step: 8 ragged sequences up to 32K, 64 nodes each.
        dict(name="tree_bf16_64_b8_32k", op="attn_tree", kv="bf16", heads=32, kv_heads=4, dim=128,
             batch=8, nodes=64, lo=4096, hi=32768, page=64, window=0),
        # Many short conversations, a few drafted tokens each.
        dict(name="tree_bf16_7_b24_1k", op="attn_tree", kv="bf16", heads=40, kv_heads=8, dim=128,
             batch=24, nodes=7, lo=90, hi=1500, page=32, window=0),
        # A sliding-window layer of head_dim 256.
        dict(name="tree_f16_33_window", op="attn_tree", kv="f16", heads=8, kv_heads=4, dim=256,
             batch=4, nodes=33, lo=600, hi=7001, page=128, window=1024),
        # The f32 cache in pages.
        dict(name="tree_f32_48_8k", op="attn_tree", kv="f32", heads=32, kv_heads=8, dim=64,
             batch=2, nodes=48, lo=3000, hi=8111, page=32, window=0),
        # The append of a single short draft, biases and interleaved pairs.
        dict(name="append_f16_5", op="append_tree", kv="f16", heads=12, kv_heads=2, dim=128,
             batch=1, nodes=5, lo=700, hi=700, page=64, norm=False, bias=True, neox=False),
        # The append of a batch of trees, Q/K norms and NeoX pairs.
        dict(name="append_bf16_64_b16", op="append_tree", kv="bf16", heads=32, kv_heads=8, dim=128,
             batch=16, nodes=64, lo=100, hi=2000, page=64, norm=True, bias=False, neox=True),
        # The accepted rows of one conversation, 28 layers.
        dict(name="accept_f16_26_l28", op="accept", kv="f16", heads=12, kv_heads=2, dim=128,
             batch=1, nodes=26, accept=5, lo=500, hi=500, page=64, layers=28),
        # The accepted rows of a batch, 36 layers.
        dict(name="accept_bf16_64_b32_l36", op="accept", kv="bf16", heads=32, kv_heads=8, dim=128,
             batch=32, nodes=64, accept=12, lo=30, hi=95, page=32, layers=36),
        # The page table of 64 long sequences, some of which end or begin.
        dict(name="pages_serve_64_16k", op="pages", kv="f16", heads=2, kv_heads=2, dim=64,
             batch=64, beams=1, lo=1000, hi=16384, page=32, layers=1, grow=65),
        # Beams: 8 requests of 4 beams that fork and die, 16 layers.
        dict(name="pages_beam_32_l16", op="pages", kv="bf16", heads=32, kv_heads=8, dim=64,
             batch=32, beams=4, lo=200, hi=700, page=32, layers=16, grow=1),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(("attn_tree", "attn_tree", "attn_tree", "append_tree", "accept", "pages"))
    heads, kv_heads, dim = rng.choice(SHAPES)
    hi = _spread(rng, 2, 32768 if op == "attn_tree" else 8192)
    c = dict(op=op, kv=rng.choice(("f32", "f16", "bf16")), heads=heads, kv_heads=kv_heads, dim=dim,
             batch=_spread(rng, 1, 32), lo=rng.choice((hi, max(1, hi // 7))), hi=hi,
             page=rng.choice((32, 64, 128, 256)))
    if op == "attn_tree":
        c.update(nodes=_spread(rng, 1, 128), window=rng.choice((0, 0, 0, 1024)))
        if rng.random() < 0.3:
            c.update(batch=_spread(rng, 1, 4), page=0)
    elif op == "append_tree":
        c.update(nodes=_spread(rng, 1, 128), norm=rng.random() < 0.5, bias=rng.random() < 0.5,
                 neox=rng.random() < 0.5)
    elif op == "accept":
        nodes = _spread(rng, 2, 128)
        c.update(nodes=nodes, accept=_spread(rng, 1, nodes), layers=_spread(rng, 1, 36))
    else:
        beams = rng.choice((1, 2, 4, 5))
        c.update(batch=beams * _spread(rng, 1, 24), beams=beams, layers=_spread(rng, 1, 28),
                 grow=rng.choice((1, 1, 17, 65)))
    return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and _cache_bytes(c) <= 1 << 30:
            return c


# ---- sizes of a case ----
def _lengths(case):
    """A ragged batch's lengths, spread over [lo, hi] by its sizes alone."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(b)]


def _nodes(case):
    """Drafted tokens of each sequence: the first has all of them."""
    b, n = case["batch"], case["nodes"]
    return [n - int(0.5 * n * ((i * 0.7548776662) % 1.0)) for i in range(b)]


def _kv_dim(case):
    return case["kv_heads"] * case["dim"]


def _need(case, length):
    """Pages of a sequence with room for what the case adds to it."""
    more = case["grow"] if case["op"] == "pages" else case["nodes"]
    return -(-(length + more) // case["page"])


def _pool(case):
    """(pages of the pool, columns of the block table)."""
    need = [_need(case, n) for n in _lengths(case)]
    spare = len(need) * (2 + -(-case["grow"] // case["page"])) if case["op"] == "pages" else 3
    return sum(need) + spare, max(need) + 1


def _cache_bytes(case):
    rows = (case["batch"] * (case["hi"] + case["nodes"]) if case["page"] == 0
            else _pool(case)[0] * case["page"])
    return 2 * rows * _kv_dim(case) * SIZE[case["kv"]] * case.get("layers", 1)


def work(case):
    lens, row = _lengths(case), _kv_dim(case) * SIZE[case["kv"]]
    q_row = case["heads"] * case["dim"]
    if case["op"] == "attn_tree":
        nodes, win, size = _nodes(case), case["window"], SIZE[case["kv"]]
        seen = [min(n, win - 1) if win else n for n in lens]
        rows = sum(nodes)
        return {"bytes": sum(k + m for k, m in zip(seen, nodes)) * 2 * row + 2 * rows * q_row * size,
                "flops": 4.0 * q_row * sum(m * (k + 1) for k, m in zip(seen, nodes))}
    if case["op"] == "append_tree":
        rows = sum(_nodes(case))
        return {"bytes": rows * ((q_row + 2 * _kv_dim(case)) * 4 + 2 * row + q_row * SIZE[case["kv"]]),
                "flops": 8.0 * rows * (q_row + _kv_dim(case))}
    if case["op"] == "accept":
        moved = case["batch"] * max(1, case["accept"] - 1)
        return {"bytes": 4.0 * moved * row * case["layers"], "flops": 0.0}
    n_pages, cols = _pool(case)
    # the table read and written, and a part page copied for three beams of four
    copied = case["batch"] * (1 - 1 / case["beams"]) * 0.5 * case["page"]
    return {"bytes": 8.0 * case["batch"] * cols + 4.0 * copied * row * case["layers"], "flops": 0.0}


# ---- inputs ----
def _trees(rs, nodes, most):
    """(parent, depth) of each sequence's tree: node 0 is the root, half of the
    others go on from the node before them, half from any earlier one."""
    parent = np.full((len(nodes), most), -1, np.int64)
    depth = np.zeros((len(nodes), most), np.int64)
    for b, n in enumerate(nodes):
        for i in range(1, n):
            parent[b, i] = i - 1 if rs.rand() < 0.5 else rs.randint(0, i)
            depth[b, i] = depth[b, parent[b, i]] + 1
    return parent, depth


def _masks(parent, nodes):
    """Ancestor bits: word j // 64, bit j % 64 of row i says that node i sees node j."""
    b, t = parent.shape
    m = np.zeros((b, t, -(-t // 64)), np.uint64)
    for s in range(b):
        for i in range(nodes[s]):
            if parent[s, i] >= 0:
                m[s, i] = m[s, parent[s, i]]
            m[s, i, i // 64] |= np.uint64(1 << (i % 64))
    return m.view(np.int64)


def _on_gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator("cuda").manual_seed(seed)
    dt, kvd, op = DT[case["kv"]], _kv_dim(case), case["op"]
    lens, b = _lengths(case), case["batch"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    s = {"case": case, "lens": _on_gpu(np.array(lens, np.int32))}
    layers = (case["layers"],) if "layers" in case else ()
    if case["page"]:
        n_pages, cols = _pool(case)
        s["k"], s["v"] = (randn(*layers, n_pages, case["page"], kvd, dtype=dt) for _ in "kv")
        perm, at = rs.permutation(n_pages), 0
        table = np.full((b, cols), -1, np.int32)
        for i, n in enumerate(lens):
            need = -(-n // case["page"]) if op == "pages" else _need(case, n)
            table[i, :need] = perm[at:at + need]
            at += need
            if op == "pages" and i % case["beams"]:  # beams share their request's whole pages
                first = i - i % case["beams"]
                whole = min(n, lens[first]) // case["page"]
                table[i, :whole] = table[first, :whole]
        s["table"] = _on_gpu(table)
    else:
        s["k"], s["v"] = (randn(b, case["hi"] + case["nodes"], kvd, dtype=dt) for _ in "kv")
    if op == "pages":
        beams, parent = case["beams"], np.arange(b)
        if beams > 1:  # the next beams of a request go on from any of its present ones
            parent = parent - parent % beams + rs.randint(0, beams, b)
            cap = np.array(lens)[parent] + case["grow"]
        else:  # one sequence in eight ends, one in eight makes room for a new one
            what = rs.randint(0, 8, b)
            cap = np.where(what == 0, 0, np.array(lens) + case["grow"])
            cap = np.where(what == 1, np.minimum(cap, 1 + rs.randint(0, case["hi"], b)), cap)
            parent = np.where(what == 1, -1, parent)
        held = np.zeros(s["k"].shape[-3], np.bool_)
        held[perm[at:at + b // 8]] = True  # pages of a stored prefix that no sequence has now
        s.update(parent=_on_gpu(parent.astype(np.int32)), cap=_on_gpu(cap.astype(np.int32)),
                 held=_on_gpu(held))
        return s
    nodes = _nodes(case)
    s["n"] = _on_gpu(np.array(nodes, np.int32))
    if op == "accept":
        path = np.full((b, case["nodes"]), -1, np.int32)
        count = np.zeros(b, np.int32)
        for i, m in enumerate(nodes):
            count[i] = min(m, case["accept"])
            path[i, 1:count[i]] = 1 + np.sort(rs.permutation(m - 1)[:count[i] - 1])
            path[i, 0] = 0
        s.update(path=_on_gpu(path), count=_on_gpu(count))
        return s
    parent, depth = _trees(rs, nodes, case["nodes"])
    s["pos"] = _on_gpu((np.array(lens)[:, None] + depth).astype(np.int32))
    h, hk, d, t = case["heads"], case["kv_heads"], case["dim"], case["nodes"]
    if op == "attn_tree":
        s["q"] = 2 * randn(b, t, h, d, dtype=dt)  # scores of standard deviation 2
        s["mask"] = _on_gpu(_masks(parent, nodes))
        s["max_len"] = max(n + m for n, m in zip(lens, nodes))
        return s
    s.update(q=randn(b, t, h * d), k_in=randn(b, t, hk * d), v_in=randn(b, t, hk * d))
    s["qn"], s["kn"] = ((1 + 0.1 * randn(d) for _ in "qk") if case["norm"] else (None, None))
    s["qb"], s["kb"], s["vb"] = ((0.1 * randn(n * d) for n in (h, hk, hk)) if case["bias"]
                                 else (None, None, None))
    angle = torch.outer(torch.arange(case["hi"] + t, dtype=torch.float64),
                        1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    s["cs"] = torch.stack((angle.cos(), angle.sin()), -1).float().cuda().contiguous()
    return s


# ---- one pass ----
def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"attn_tree": _attn_tree, "append_tree": _append_tree, "accept": _accept,
            "pages": _pages}[c["op"]](s, c)


def _own(s, c):
    from ullm_amd import attention as A

    if c["op"] == "attn_tree":
        more = dict(n_nodes=s["n"], positions=s["pos"], window=c["window"])
        if c["page"]:
            return A.attn_tree_paged(s["q"], s["k"], s["v"], s["table"], s["mask"], s["lens"],
                                     s["max_len"], c["kv_heads"], **more)
        return A.attn_tree(s["q"], s["k"], s["v"], s["mask"], s["lens"], s["max_len"], c["kv_heads"],
                           seq_stride=s["k"].stride(0), **more)
    if c["op"] == "append_tree":
        q = A.qkv_append_tree_paged(s["q"], s["k_in"], s["v_in"], s["k"], s["v"], s["cs"], s["lens"],
                                    s["pos"], s["table"], n_head=c["heads"], n_kv_head=c["kv_heads"],
                                    head_dim=c["dim"], n_nodes=s["n"], neox=c["neox"],
                                    q_norm=s["qn"], k_norm=s["kn"], eps=EPS, q_bias=s["qb"],
                                    k_bias=s["kb"], v_bias=s["vb"], q_dtype=DT[c["kv"]])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if c["op"] == "accept":
        lens = A.kv_accept_paged(s["k"], s["v"], s["table"], s["path"], s["count"], s["lens"])
        return {"lens": lens, "k": s["k"], "v": s["v"]}
    table, lens, info = A.kv_pages_update(s["k"], s["v"], s["table"], s["lens"], s["parent"],
                                          s["cap"], held=s["held"])
    return {"table": table, "lens": lens, "info": info, "k": s["k"], "v": s["v"]}


def _attn_tree(s, c):
    """out[b, i, h] = softmax over the keys that node i of sequence b sees of
    q . k / sqrt(dim), times their v.  It sees the keys of the sequence, and
    node j's where its mask has bit j, those at most window - 1 positions
    before its own if there is a window."""
    h, hk, d, b, t = c["heads"], c["kv_heads"], c["dim"], c["batch"], c["nodes"]
    dev = s["q"].device
    if c["page"]:
        pages = s["table"].clamp(min=0).long()
        k, v = (s[x][pages].flatten(1, 2) for x in "kv")
    else:
        k, v = s["k"], s["v"]
    k, v = (x[:, :s["max_len"]].float().unflatten(2, (hk, d)).transpose(1, 2).contiguous() for x in (k, v))
    n_keys = k.shape[2]
    at, lens = torch.arange(n_keys, device=dev), s["lens"].long()
    node = torch.arange(t, device=dev)
    bits = (s["mask"][:, :, node // 64] >> (node % 64)) & 1  # [b, i, j]
    j = at - lens[:, None]                                   # node index of each key
    in_tree = (j >= 0) & (j < s["n"][:, None])
    jc = j.clamp(0, t - 1)
    sees = torch.gather(bits, 2, jc[:, None].expand(b, t, n_keys)) == 1
    sees = torch.where(in_tree[:, None], sees, (j < 0)[:, None])
    if c["window"]:
        key_pos = torch.where(j < 0, at, torch.gather(s["pos"].long(), 1, jc))
        sees &= key_pos[:, None] > s["pos"][:, :, None] - c["window"]
    sees &= node[:, None] < s["n"][:, None, None]
    q = s["q"].float().view(b, t, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(b * hk, -1, d)
    w = torch.bmm(q, k.flatten(0, 1).transpose(1, 2).contiguous()) / math.sqrt(d)
    w = w.view(b, hk, t, h // hk, n_keys).masked_fill_(~sees[:, None, :, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(m > -math.inf, m, 0)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(b * hk, -1, n_keys), v.flatten(0, 1)).view(b, hk, t, h // hk, d)
    o = o / torch.where(total > 0, total, 1)
    return o.permute(0, 2, 1, 3, 4).reshape(b, t, h, d).to(s["q"].dtype)


def _slots(s, c, at):
    """Rows of the pool (page * page size + slot) of positions `at` [b, n]."""
    page = torch.gather(s["table"].long(), 1, at // c["page"])
    return page * c["page"] + at % c["page"]


def _append_tree(s, c):
    """Bias, x / rms(x) * weight of each q and k head, RoPE at the token's
    position; node i's K and V rows are stored behind the sequence, at its
    length + i.  Rows that hold no token give a q of zeros."""
    b, t, d = c["batch"], c["nodes"], c["dim"]
    node = torch.arange(t, device=s["q"].device)
    there = node < s["n"][:, None]
    cos, sin = s["cs"][s["pos"].long()].unbind(-1)
    cos, sin = cos[:, :, None], sin[:, :, None]

    def heads(x, bias, norm, rope):
        x = (x if bias is None else x + bias).view(b, t, -1, d)
        if norm is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
        if not rope:
            return x
        if c["neox"]:
            lo, hi = x[..., :d // 2], x[..., d // 2:]
            return torch.cat((lo * cos - hi * sin, lo * sin + hi * cos), -1)
        lo, hi = x[..., 0::2], x[..., 1::2]
        return torch.stack((lo * cos - hi * sin, lo * sin + hi * cos), -1).flatten(-2)

    dt = DT[c["kv"]]
    q = heads(s["q"], s["qb"], s["qn"], True).flatten(2)
    q = torch.where(there[:, :, None], q, 0).to(dt)
    # a row without a token stores node 0's row once more
    node = torch.where(there, node, 0)
    dst = _slots(s, c, s["lens"].long()[:, None] + node).flatten()
    for name, x in (("k", heads(s["k_in"], s["kb"], s["kn"], True)),
                    ("v", heads(s["v_in"], s["vb"], None, False))):
        x = x.flatten(2).to(dt)
        x = torch.gather(x, 1, node[:, :, None].expand_as(x))
        s[name].flatten(0, 1)[dst] = x.flatten(0, 1)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _accept(s, c):
    """Row length + j of each sequence takes what row length + path[j] held,
    for the accepted nodes of the path; the lengths grow by as many."""
    j = torch.arange(c["nodes"], device=s["path"].device)
    count, lens = s["count"][:, None], s["lens"].long()[:, None]
    j = torch.where(j < count, j, 0)  # the others move row 0 once more
    src = torch.where(count > 0, torch.gather(s["path"].long(), 1, j), 0)
    src, dst = _slots(s, c, lens + src).flatten(), _slots(s, c, lens + j).flatten()
    for x in (s["k"].flatten(1, 2), s["v"].flatten(1, 2)):
        x[:, dst] = x[:, src]
    return {"lens": s["lens"] + s["count"], "k": s["k"], "v": s["v"]}


def _pages(s, c):
    """The next table.  Sequence s goes on from parent[s] (< 0: from nothing),
    keeps min(its length, capacity[s]) positions and has pages for capacity[s].
    Pages that are full of kept positions are shared.  The last, part-filled
    one goes to the first sequence that keeps it, if none shares it as a full
    one and it is not held; every other gets a copy in a page of its own.
    Pages are taken lowest number first, sequence by sequence, from those that
    no sequence keeps and that are not held."""
    page, dev = c["page"], s["table"].device
    table, cols = s["table"].long(), s["table"].shape[1]
    n_pages, cap = s["k"].shape[1], s["cap"].long().clamp(max=s["table"].shape[1] * page)
    parent = s["parent"].long()
    b = parent.shape[0]
    p = parent.clamp(min=0)
    kept = torch.where(parent >= 0, torch.minimum(s["lens"].long()[p], cap), 0)
    full, part, need = kept // page, kept % page, -(-cap // page)
    rows = table[p]
    col, seq = torch.arange(cols, device=dev), torch.arange(b, device=dev)
    shared = torch.zeros(n_pages + 1, dtype=torch.bool, device=dev)
    shared[torch.where(col < full[:, None], rows, n_pages).flatten()] = True
    shared[:-1] |= s["held"]
    last = torch.gather(rows, 1, full.clamp(max=cols - 1)[:, None])[:, 0]
    last = torch.where(part > 0, last, n_pages)
    owner = torch.full((n_pages + 1,), b, device=dev).scatter_reduce_(0, last, seq, "amin")
    keeps = (part > 0) & ~shared[last] & (owner[last] == seq)
    live = shared.clone()
    live[last] = True
    free = torch.argsort(live[:-1].int(), stable=True)  # free pages first, in order
    n_free = (~live[:-1]).sum()
    take = need - full - keeps.long()
    first = torch.cumsum(take, 0) - take
    nth = first[:, None] + col - full[:, None] - keeps[:, None].long()
    fresh = torch.where(nth < n_free, free[nth.clamp(0, n_pages - 1)], -1)
    new = torch.where(col < full[:, None], rows, fresh)
    new = torch.where((col == full[:, None]) & keeps[:, None], last[:, None], new)
    new = torch.where(col < need[:, None], new, -1)
    copied = (part > 0) & ~keeps
    to = torch.gather(new, 1, full.clamp(max=cols - 1)[:, None])[:, 0]
    lost = copied & (to < 0)
    copied &= to >= 0
    src, dst = last[copied], to[copied]
    there = (torch.arange(page, device=dev) < part[copied][:, None])[None, :, :, None]
    for x in (s["k"], s["v"]):
        x[:, dst] = torch.where(there, x[:, src], x[:, dst])
    lens = torch.where(lost, full * page, kept)
    asked = take.sum()
    info = torch.stack((copied.sum(), torch.minimum(asked, n_free), (asked - n_free).clamp(min=0)))
    return {"table": new.int(), "lens": lens.int(), "info": info.int(), "k": s["k"], "v": s["v"]}


# ---- in 64 bits, one sequence at a time ----
def exact(case, seed):
    s = prepare(case, seed)
    return {"attn_tree": _exact_attn, "append_tree": _exact_append, "accept": _exact_accept,
            "pages": _exact_pages}[case["op"]](s, case)


def _rows_of(s, c, b, positions):
    """Pool rows of positions of sequence b."""
    tab = s["table"][b].tolist()
    return torch.tensor([tab[t // c["page"]] * c["page"] + t % c["page"] for t in positions],
                        dtype=torch.long, device="cuda")


def _exact_attn(s, c):
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, nodes = s["lens"].tolist(), s["n"].tolist()
    for b, (n, m) in enumerate(zip(lens, nodes)):
        if c["page"]:
            rows = _rows_of(s, c, b, range(n + m))
            k, v = (s[x].flatten(0, 1)[rows].double() for x in "kv")
        else:
            k, v = (s[x][b, :n + m].double() for x in "kv")
        words = s["mask"][b].tolist()
        tree = [[words[i][j // 64] >> (j % 64) & 1 for j in range(m)] for i in range(m)]
        see = torch.ones(m, n + m, dtype=torch.bool, device="cuda")
        see[:, n:] = torch.tensor(tree, dtype=torch.bool, device="cuda")
        if c["window"]:
            pos = s["pos"][b, :m].long()
            key = torch.cat((torch.arange(n, device="cuda"), pos))
            see &= pos[:, None] - key < c["window"]
        for g in range(h):
            j = g // (h // hk)
            w = s["q"][b, :m, g].double() @ k[:, j * d:(j + 1) * d].t().contiguous() * d ** -0.5
            w = torch.softmax(w.masked_fill(~see, -math.inf), -1)
            out[b, :m, g] = w @ v[:, j * d:(j + 1) * d]
    return out


def _exact_append(s, c):
    d, dt = c["dim"], torch.float64
    k, v = s["k"].to(dt), s["v"].to(dt)
    q = torch.zeros(s["q"].shape, dtype=dt, device="cuda")
    half = torch.arange(d // 2, device="cuda")
    a, z = (half, half + d // 2) if c["neox"] else (2 * half, 2 * half + 1)
    for b, m in enumerate(s["n"].tolist()):
        cs = s["cs"][s["pos"][b, :m].long()].to(dt)[:, None]
        rows = _rows_of(s, c, b, range(int(s["lens"][b]), int(s["lens"][b]) + m))

        def turn(x, bias, norm):
            x = x[b, :m].to(dt) + (0 if bias is None else bias.to(dt))
            x = x.view(m, -1, d)
            if norm is not None:
                x = x / ((x ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * norm.to(dt)
            y = torch.empty_like(x)
            y[..., a] = x[..., a] * cs[..., 0] - x[..., z] * cs[..., 1]
            y[..., z] = x[..., a] * cs[..., 1] + x[..., z] * cs[..., 0]
            return y.reshape(m, -1)

        q[b, :m] = turn(s["q"], s["qb"], s["qn"])
        k.flatten(0, 1)[rows] = turn(s["k_in"], s["kb"], s["kn"])
        v.flatten(0, 1)[rows] = s["v_in"][b, :m].to(dt) + (0 if s["vb"] is None else s["vb"].to(dt))
    return {"q": q, "k": k, "v": v}


def _exact_accept(s, c):
    k, v = s["k"].double(), s["v"].double()
    lens = s["lens"].tolist()
    for b, m in enumerate(s["count"].tolist()):
        path = s["path"][b, :m].tolist()
        src = _rows_of(s, c, b, [lens[b] + i for i in path])
        dst = _rows_of(s, c, b, range(lens[b], lens[b] + m))
        for x, y in ((k, s["k"]), (v, s["v"])):
            x.flatten(1, 2)[:, dst] = y.flatten(1, 2)[:, src].double()
        lens[b] += m
    return {"lens": torch.tensor(lens, dtype=torch.int32), "k": k, "v": v}


def _exact_pages(s, c):
    page, n_pages = c["page"], s["k"].shape[1]
    table, lens, held = s["table"].tolist(), s["lens"].tolist(), s["held"].tolist()
    cols = len(table[0])
    todo, used = [], {i for i in range(n_pages) if held[i]}
    for par, cap in zip(s["parent"].tolist(), s["cap"].tolist()):
        cap = min(cap, cols * page)
        kept = min(lens[par], cap) if par >= 0 else 0
        todo.append((par, kept, -(-cap // page)))
        used.update(table[par][:kept // page] if par >= 0 else [])
    owner = {}
    for i, (par, kept, _) in enumerate(todo):
        if kept % page and table[par][kept // page] not in used:
            owner.setdefault(table[par][kept // page], i)
    free = iter([i for i in range(n_pages) if i not in used and i not in owner])
    k, v = s["k"].double(), s["v"].double()
    new, new_lens, info = [], [], [0, 0, 0]
    for i, (par, kept, need) in enumerate(todo):
        full, part = divmod(kept, page)
        row = table[par][:full] if full else []
        if part and owner.get(table[par][full]) == i:
            row = row + [table[par][full]]
        mine = len(row)
        for _ in range(need - mine):
            got = next(free, -1)
            info[1 if got >= 0 else 2] += 1
            row = row + [got]
        if part and mine == full:
            to = row[full]
            if to < 0:
                kept = full * page
            else:
                info[0] += 1
                for x, y in ((k, s["k"]), (v, s["v"])):
                    x[:, to, :part] = y[:, table[par][full], :part].double()
        new.append(row + [-1] * (cols - len(row)))
        new_lens.append(kept)
    return {"table": torch.tensor(new, dtype=torch.int32), "lens": torch.tensor(new_lens, dtype=torch.int32),
            "info": torch.tensor(info, dtype=torch.int32), "k": k, "v": v}
