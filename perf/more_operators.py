"""Cases of the operators that decide what a KV cache keeps: which drafted
tokens of a step, and which positions of a sequence that has grown too long.

A case is a dict of plain values.  `op` names the call:

  weights  the attention weight that each position of a cache gets from some
           rows of queries, summed over them and over the query heads of a kv
           head, added to what it had (key_weights, key_weights_paged)
  evict    a cache cut down to a budget: the first positions, the last ones and
           those of the largest collected weight stay, in order, each kv head
           by its own weights, in every layer (kv_evict, kv_evict_paged)
  verify   drafted tokens, a chain or a tree, kept or rejected by the target's
           probabilities, the draft's and given random numbers, so that what is
           kept is distributed as the target alone; and the token that follows
           (tree_verify)

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

# Attention shapes (n_head, n_kv_head, head_dim): those of the attention cases
# beside this file, and groups of 5 and 7 heads, which fill no power of two.
SHAPES = [(32, 8, 64), (12, 2, 128), (32, 8, 128), (8, 4, 256), (32, 4, 128), (40, 8, 128), (14, 2, 64)]


def listed():
    return [
        # The smallest call: the last token of a short prompt, a small model in
        # the reference's own f32 cache.
        dict(name="weights_f32_one_short", op="weights", kv="f32", q="f32", heads=32, kv_heads=8, dim=64,
             batch=1, rows=1, lo=300, hi=300, page=0, window=0, decay=1.0),
        # A decode step of 8 ragged sequences up to 32K: every step collects.
        dict(name="weights_bf16_one_b8_32k", op="weights", kv="bf16", q="f32", heads=32, kv_heads=4, dim=128,
             batch=8, rows=1, lo=4096, hi=32768, page=64, window=0, decay=1.0),
        # The last 32 rows of a 32K prompt look back over all of it, once.
        dict(name="weights_bf16_last32_32k", op="weights", kv="bf16", q="bf16", heads=32, kv_heads=8, dim=128,
             batch=1, rows=32, lo=32768, hi=32768, page=0, window=0, decay=0.0),
        # All rows of a 2048-token prompt.
        dict(name="weights_bf16_prompt_2k", op="weights", kv="bf16", q="bf16", heads=32, kv_heads=8, dim=128,
             batch=1, rows=2048, lo=2048, hi=2048, page=0, window=0, decay=0.0),
        # A few accepted tokens of 4 sequences, head_dim 256, a sliding window,
        # older weights fading.
        dict(name="weights_f16_7_window", op="weights", kv="f16", q="f16", heads=8, kv_heads=4, dim=256,
             batch=4, rows=7, lo=1500, hi=7001, page=128, window=1024, decay=0.75),
        # One layer of a short conversation, f32.
        dict(name="evict_f32_one_layer", op="evict", kv="f32", heads=32, kv_heads=8, dim=64, batch=1,
             lo=1401, hi=1401, budget=1024, sink=4, recent=128, layers=1, page=0),
        # One conversation of a small model at 4K, cut to a quarter in 28 layers.
        dict(name="evict_f16_4k_l28", op="evict", kv="f16", heads=12, kv_heads=2, dim=128, batch=1,
             lo=4096, hi=4096, budget=1024, sink=4, recent=64, layers=28, page=0),
        # A batch of ragged sequences in pages; the short ones stay whole.
        dict(name="evict_bf16_b8_l8", op="evict", kv="bf16", heads=32, kv_heads=4, dim=128, batch=8,
             lo=1500, hi=8192, budget=2048, sink=16, recent=256, layers=8, page=64),
        # Four drafted tokens of one conversation, a small vocabulary.
        dict(name="verify_chain_4_b1", op="verify", p="f32", draft="probs", batch=1, nodes=4, fan=1,
             vocab=32000, cut=False),
        # A serving step: 32 chains of 7 drafted tokens, a large vocabulary.
        dict(name="verify_chain_7_b32", op="verify", p="f32", draft="probs", batch=32, nodes=7, fan=1,
             vocab=131072, cut=False),
        # 8 trees of 26 distinct drafts each, an odd vocabulary, probabilities
        # with their tails cut off.
        dict(name="verify_tree_26_b8", op="verify", p="f32", draft="distinct", batch=8, nodes=26, fan=4,
             vocab=100003, cut=True),
        # 16 trees of tokens found by lookup, which have no probabilities of
        # their own; the target's in 16 bits.
        dict(name="verify_lookup_bf16_b16", op="verify", p="bf16", draft="none", batch=16, nodes=15, fan=2,
             vocab=50001, cut=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(("weights", "weights", "evict", "verify"))
    if op == "verify":
        nodes = _spread(rng, 1, 64)
        return dict(op=op, p=rng.choice(("f32", "f32", "f16", "bf16")),
                    draft=rng.choice(("probs", "probs", "distinct", "none")), batch=_spread(rng, 1, 32),
                    nodes=nodes, fan=rng.choice((1, 2, 4, 7)), vocab=_spread(rng, 500, 131072),
                    cut=rng.random() < 0.3)
    heads, kv_heads, dim = rng.choice(SHAPES)
    kv = rng.choice(("f32", "f16", "bf16"))
    hi = _spread(rng, 2, 32768 if op == "weights" else 12000)
    c = dict(op=op, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, batch=_spread(rng, 1, 32),
             lo=rng.choice((hi, max(1, hi // 7))), hi=hi, page=rng.choice((0, 32, 64, 128, 256)))
    if op == "weights":
        c.update(q=rng.choice(("f32", kv)), rows=rng.choice((1, _spread(rng, 1, 2048))),
                 window=rng.choice((0, 0, 0, 1024)), decay=rng.choice((0.0, 1.0, 0.5)))
        return c
    budget = _spread(rng, 1, hi)
    c.update(budget=budget, sink=min(rng.choice((0, 1, 4, 16)), budget), layers=_spread(rng, 1, 36),
             recent=rng.choice((0, budget // 8, budget // 2)))
    return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _state_bytes(case):
    if case["op"] == "verify":
        return case["batch"] * (2 * case["nodes"] + 1) * case["vocab"] * SIZE[case["p"]]
    n = (1 if case["op"] == "weights" else 2) * case.get("layers", 1)
    return n * case["batch"] * (case["hi"] + max(case["page"], 1)) * _kv_dim(case) * SIZE[case["kv"]]


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        scores = c["heads"] * c["rows"] * c["hi"] * c["batch"] if c["op"] == "weights" else 0
        if _cost(c) <= most and _state_bytes(c) <= 1 << 30 and scores <= 1 << 28:
            return c


# ---- sizes of a case ----
def _lengths(case):
    """A ragged batch's lengths, spread over [lo, hi] by its sizes alone."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(b)]


def _counts(case, most):
    """Rows or nodes of each sequence: the first has all of them."""
    return [most - int(0.5 * most * ((i * 0.7548776662) % 1.0)) for i in range(case["batch"])]


def _rows(case):
    return [min(r, n) for r, n in zip(_counts(case, case["rows"]), _lengths(case))]


def _kv_dim(case):
    return case["kv_heads"] * case["dim"]


def _need(case, n):
    return -(-n // case["page"])


def work(case):
    if case["op"] == "verify":
        # the row that the last token is drawn from, and the draft's beside it
        rows = case["batch"] * (1 if case["draft"] == "none" else 2)
        return {"bytes": float(rows * case["vocab"] * SIZE[case["p"]]), "flops": 0.0}
    lens, row = _lengths(case), _kv_dim(case) * SIZE[case["kv"]]
    if case["op"] == "weights":
        rows, win = _rows(case), case["window"]
        span = [min(n, win + r - 1) if win else n for n, r in zip(lens, rows)]
        each = [sum(min(n - i, win) if win else n - i for i in range(r)) for n, r in zip(lens, rows)]
        q = sum(rows) * case["heads"] * case["dim"] * SIZE[case["q"]]
        acc = sum(lens) * case["kv_heads"] * 4 * (2 if case["decay"] else 1)
        return {"bytes": float(sum(span) * row + q + acc),
                "flops": 2.0 * case["heads"] * case["dim"] * sum(each)}
    kept = [min(n, case["budget"]) for n in lens]
    moved = sum(k - min(case["sink"], k) for n, k in zip(lens, kept) if n > k)
    small = 4.0 * case["kv_heads"] * (sum(lens) + 2 * sum(kept))  # weights, kept ones, their positions
    return {"bytes": case["layers"] * (4.0 * moved * row + small), "flops": 0.0}


# ---- inputs ----
def _on_gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator("cuda").manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, rs, gen)
    lens, b, dt, kvd = _lengths(case), case["batch"], DT[case["kv"]], _kv_dim(case)
    hk = case["kv_heads"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    s = {"case": case, "lens": _on_gpu(np.array(lens, np.int32)), "max_len": max(lens)}
    layers = (case["layers"],) if case["op"] == "evict" else ()
    if case["page"]:
        n_pages, cols = sum(_need(case, n) for n in lens) + 2, _need(case, max(lens))
        perm, at = rs.permutation(n_pages), 0
        table = np.full((b, cols), -1, np.int32)
        for i, n in enumerate(lens):
            need = _need(case, n)
            table[i, :need] = perm[at:at + need]
            at += need
        s["table"], shape = _on_gpu(table), (n_pages, case["page"], kvd)
    else:
        shape = (b, case["hi"], kvd)
    s["k"] = randn(*layers, *shape, dtype=dt)
    if case["op"] == "weights":
        # scores of standard deviation 2: some keys get most of a row's weight
        s["q"] = (2 * randn(b, case["rows"], case["heads"], case["dim"])).to(DT[case["q"]])
        s["n"] = _on_gpu(np.array(_rows(case), np.int32))
        s["acc"] = torch.rand((b, hk, case["hi"]), generator=gen, device="cuda")
        return s
    s["v"] = randn(*layers, *shape, dtype=dt)
    # sums of softmax weights are spread over orders of magnitude; some keys never got any
    acc = torch.exp(2 * randn(*layers, b, hk, case["hi"]) - 7)
    s["acc"] = torch.where(randn(*acc.shape) > 1.5, 0.0, acc)
    s["acc_out"] = torch.zeros_like(s["acc"])
    s["budget"] = _on_gpu(np.full(b, case["budget"], np.int32))
    return s


def _tree(rs, case):
    """Parents of each sequence's nodes: node 0 goes on from the sequence, the
    others from any earlier node or the sequence, at most `fan` from each."""
    b, t, fan = case["batch"], case["nodes"], case["fan"]
    parent = np.empty((b, t), np.int32)
    for s in range(b):
        room = [fan] * (t + 1)
        for i in range(t):
            free = [j for j in range(i + 1) if room[j]]
            j = free[-1] if rs.rand() < 0.5 else free[rs.randint(len(free))]
            room[j] -= 1
            parent[s, i] = j - 1
    return parent


def _prepare_verify(case, rs, gen):
    b, t, v, dt = case["batch"], case["nodes"], case["vocab"], DT[case["p"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def probs(logits):
        p = torch.softmax(logits, -1)
        if case["cut"]:
            p = torch.where(p < 2e-5, 0.0, p)
            p = p / p.sum(-1, keepdim=True)
        return p.to(dt)

    logits = 4 * randn(b, t + 1, v)
    target = probs(logits)
    logits = logits[:, :t] + 0.7 * randn(b, t, v)  # the draft is a little off
    draft = probs(logits)
    # node i's token is drawn from the draft's row after its parent: among
    # siblings without return (distinct), with it (probs), or the likeliest ones
    most = min(case["fan"], v)
    noise = -torch.log(-torch.log(torch.rand((b, t, v), generator=gen, device="cuda").clamp(1e-30, 1 - 1e-7)))
    if case["draft"] == "probs":
        picks = torch.cat([torch.multinomial(draft[i].float(), most, replacement=True, generator=gen)[None]
                           for i in range(b)])
    else:
        picks = ((torch.log(draft.float()) + noise) if case["draft"] == "distinct" else logits).topk(most, -1)[1]
    parent = _tree(rs, case)
    nth = np.zeros((b, t), np.int64)
    for s in range(b):
        seen = {}
        for i in range(t):
            nth[s, i] = seen.get(parent[s, i], 0)
            seen[parent[s, i]] = nth[s, i] + 1
    at = _on_gpu(parent.astype(np.int64) + 1) * most + _on_gpu(nth)
    tokens = torch.gather(picks.flatten(1), 1, at).int()
    return {"case": case, "p": target, "q": None if case["draft"] == "none" else draft, "tokens": tokens,
            "parent": _on_gpu(parent), "n": _on_gpu(np.array(_counts(case, t), np.int32)),
            "u": torch.rand((b, t + 1), generator=gen, device="cuda")}


# ---- one pass ----
def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"weights": _weights, "evict": _evict, "verify": _verify}[c["op"]](s, c)


def _own(s, c):
    from ullm_amd import attention as A

    if c["op"] == "weights":
        more = dict(n_rows=s["n"], window=c["window"], decay=c["decay"])
        if c["page"]:
            return A.key_weights_paged(s["q"], s["k"], s["table"], s["acc"], s["lens"], s["max_len"],
                                       c["kv_heads"], **more)
        return A.key_weights(s["q"], s["k"], s["acc"], s["lens"], s["max_len"], c["kv_heads"], **more)
    if c["op"] == "evict":
        more = dict(max_budget=c["budget"], sink=c["sink"], recent=c["recent"], scores_out=s["acc_out"])
        if c["page"]:
            kept, lens = A.kv_evict_paged(s["k"], s["v"], s["table"], s["acc"], s["lens"], s["budget"], **more)
        else:
            kept, lens = A.kv_evict(s["k"], s["v"], s["acc"], s["lens"], s["budget"], **more)
        return {"kept": kept, "lens": lens, "acc": s["acc_out"], "k": s["k"], "v": s["v"]}
    path, count, token = A.tree_verify(s["p"], s["q"], s["tokens"], s["u"], parents=s["parent"], n_nodes=s["n"],
                                       distinct=c["draft"] == "distinct")
    return {"path": path, "count": count, "next": token}


def _weights(s, c):
    """acc = decay * acc + the sum over the rows and the query heads of a kv
    head of softmax(q . k / sqrt(dim)) over the keys that the row sees: row i of
    n stands at position length - n + i and sees the positions up to its own,
    the last `window` of them if there is a window."""
    h, hk, d, b, r = c["heads"], c["kv_heads"], c["dim"], c["batch"], c["rows"]
    k = s["k"][s["table"].clamp(min=0).long()].flatten(1, 2) if c["page"] else s["k"]
    k = k[:, :s["max_len"]].float().unflatten(2, (hk, d)).permute(0, 2, 3, 1).contiguous()
    n_keys, dev = k.shape[3], k.device
    q = s["q"].float().view(b, r, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(b * hk, -1, d)
    w = torch.bmm(q, k.flatten(0, 1)) / math.sqrt(d)
    row, key = torch.arange(r, device=dev)[:, None], torch.arange(n_keys, device=dev)
    lens, n = s["lens"].long()[:, None, None], s["n"].long()[:, None, None]
    pos = lens - n + row
    sees = (key <= pos) & (row < n)
    if c["window"]:
        sees &= key > pos - c["window"]
    w = w.view(b, hk, r, h // hk, n_keys).masked_fill_(~sees[:, None, :, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(m > -math.inf, m, 0)).exp_()
    total = w.sum(-1, keepdim=True)
    w = w.div_(torch.where(total > 0, total, 1)).sum((2, 3))
    acc = s["acc"][:, :, :n_keys]
    there = (key < s["lens"][:, None])[:, None]
    acc.copy_(torch.where(there, c["decay"] * acc + w, acc))
    return s["acc"]


def _slots(s, c, at):
    """Rows of the cache (over all sequences) of positions `at` [b, n]."""
    if not c["page"]:
        return torch.arange(c["batch"], device=at.device)[:, None] * c["hi"] + at
    page = torch.gather(s["table"].long(), 1, at // c["page"])
    return page * c["page"] + at % c["page"]


def _evict(s, c):
    """kept[l, b, g]: the min(length, budget) positions that stay, in order: the
    first `sink`, the last `recent`, then those of the largest weight, the
    lowest of equals.  Row j of group g takes position kept[j]."""
    layers, b, hk, d, top = c["layers"], c["batch"], c["kv_heads"], c["dim"], c["budget"]
    acc, dev = s["acc"], s["acc"].device
    at = torch.arange(c["hi"], device=dev)
    lens = s["lens"].long()[:, None, None]
    n = torch.minimum(lens, s["budget"].long()[:, None, None])
    first = n.clamp(max=c["sink"])
    last = (n - first).clamp(max=c["recent"])
    kind = torch.where((at < first) | (at >= lens - last), 0, 1) + 2 * (at >= lens)  # [b, 1, hi]
    order = torch.sort(acc, dim=-1, descending=True, stable=True)[1]
    kind = torch.gather(kind.expand(acc.shape), -1, order)
    order = torch.gather(order, -1, torch.sort(kind, dim=-1, stable=True)[1])[..., :top]
    j = torch.arange(top, device=dev)[:order.shape[-1]]
    order = torch.sort(torch.where(j < n, order, c["hi"]), -1)[0]
    kept = torch.full((layers, b, hk, top), -1, dtype=torch.int32, device=dev)
    kept[..., :len(j)] = torch.where(j < n, order, -1)
    src = torch.where(j < n, order, torch.minimum(j, lens - 1))  # the others stay
    out = s["acc_out"]
    out.copy_(torch.where(at < lens, 0.0, out))
    out[..., :len(j)] = torch.where(j < n, torch.gather(acc, -1, src), out[..., :len(j)])
    dst = torch.minimum(j, lens - 1).expand(src.shape)
    group = torch.arange(hk, device=dev)[:, None]
    lay = torch.arange(layers, device=dev)[:, None]
    src, dst = (_slots(s, c, x.transpose(0, 1).reshape(b, -1)).view(b, layers, hk, -1).transpose(0, 1)
                for x in (src, dst))
    for x in (s["k"], s["v"]):
        x = x.view(layers, -1, hk, d)
        lay4 = lay[:, :, None, None]
        x[lay4, dst, group] = x[lay4, src, group]
    return {"kept": kept, "lens": n.flatten().int(), "acc": out, "k": s["k"], "v": s["v"]}


def _verify(s, c):
    """The nodes in order, each a child of the last one kept.  p is the target's
    row after that one, q the draft's; c = 0, S = Z = 1 to begin with.  A child
    of token x is kept if R(x) > 0 and u q(x) / Z S < R(x), R = max(p - c q, 0).
    If not, c grows by S / Z, Z shrinks by q(x) where the children are distinct
    (to 2^-24 at least), and S = sum(R).  The next token is the first whose
    cumulative sum of R exceeds u sum(R); that of p where R is all zero.  A
    draft without probabilities: R is p without the tokens rejected so far, and
    a child is kept if u S < p(x), S = 1 - their p."""
    b, t, v = c["batch"], c["nodes"], c["vocab"]
    dev, ar = s["p"].device, torch.arange(b, device=s["p"].device)
    lookup, distinct = s["q"] is None, c["draft"] == "distinct"
    cur = torch.zeros(b, dtype=torch.long, device=dev)
    zero, one = (torch.full((b,), x, dtype=torch.float64, device=dev) for x in (0.0, 1.0))
    k, total, left = zero, one, one
    gone = torch.zeros((b, v), dtype=torch.bool, device=dev)
    path = torch.full((b, t), -1, dtype=torch.int32, device=dev)
    count = torch.zeros(b, dtype=torch.int32, device=dev)
    n, u = s["n"], s["u"].double()
    p, q = s["p"][ar, cur].double(), None if lookup else s["q"][ar, cur].double()

    def rest():
        if lookup:
            return torch.where(gone, 0.0, p)
        return (p - k[:, None] * q).clamp(min=0)

    for i in range(t):
        x = s["tokens"][:, i].long()
        mine = (s["parent"][:, i] + 1 == cur) & (i < n)
        px = p[ar, x]
        if lookup:
            r, test = torch.where(gone[ar, x], 0.0, px), u[:, i] * total
        else:
            qx = q[ar, x]
            r, test = (px - k * qx).clamp(min=0), u[:, i] * (qx / left) * total
        keep = mine & (r > 0) & (test < r)
        no = mine & ~keep
        if lookup:
            total = torch.where(no, (total - r).clamp(min=0), total)
            gone[ar, x] |= no
        else:
            k = torch.where(no, k + total / left, k)
            if distinct:
                left = torch.where(no, (left - qx).clamp(min=2.0 ** -24), left)
            total = torch.where(no, rest().sum(-1), total)
        path.scatter_(1, count.clamp(max=t - 1).long()[:, None], torch.where(
            keep, i, path[ar, count.clamp(max=t - 1).long()])[:, None].int())
        count += keep
        cur = torch.where(keep, i + 1, cur)
        k, total, left = torch.where(keep, zero, k), torch.where(keep, one, total), torch.where(keep, one, left)
        gone &= ~keep[:, None]
        p = s["p"][ar, cur].double()
        if not lookup:
            q = s["q"][ar, cur.clamp(max=t - 1)].double()
    w = rest()
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p)
    w = torch.cumsum(w, -1)
    token = (w <= u[:, t:] * w[:, -1:]).sum(-1)
    return {"path": path, "count": count, "next": torch.where(w[:, -1] > 0, token, -1).int()}


# ---- in 64 bits, one sequence at a time ----
def exact(case, seed):
    s = prepare(case, seed)
    return {"weights": _exact_weights, "evict": _exact_evict, "verify": _exact_verify}[case["op"]](s, case)


def _rows_of(s, c, b, positions):
    """Rows of the cache of positions of sequence b."""
    if not c["page"]:
        return b * c["hi"] + torch.as_tensor(positions, device="cuda")
    tab = s["table"][b].tolist()
    return torch.tensor([tab[t // c["page"]] * c["page"] + t % c["page"] for t in positions],
                        dtype=torch.long, device="cuda")


def _exact_weights(s, c):
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    acc = s["acc"].double()
    for b, (n, r) in enumerate(zip(s["lens"].tolist(), s["n"].tolist())):
        k = s["k"].flatten(0, 1)[_rows_of(s, c, b, range(n))].double()
        pos, key = torch.arange(n - r, n, device="cuda")[:, None], torch.arange(n, device="cuda")
        see = key <= pos
        if c["window"]:
            see &= pos - key < c["window"]
        acc[b, :, :n] *= c["decay"]
        for g in range(h):
            j = g // (h // hk)
            w = s["q"][b, :r, g].double() @ k[:, j * d:(j + 1) * d].t().contiguous() * d ** -0.5
            acc[b, j, :n] += torch.softmax(w.masked_fill(~see, -math.inf), -1).sum(0)
    return acc


def _exact_evict(s, c):
    layers, b, hk, d = c["layers"], c["batch"], c["kv_heads"], c["dim"]
    acc = s["acc"].double().cpu().numpy()
    kept = np.full((layers, b, hk, c["budget"]), -1, np.int32)
    out = s["acc_out"].double().cpu().numpy()
    lens, new = s["lens"].tolist(), []
    k, v = (s[x].double().view(layers, -1, hk, d) for x in "kv")
    for i, n in enumerate(lens):
        m = min(n, c["budget"])
        new.append(m)
        first = min(c["sink"], m)
        last = min(c["recent"], m - first)
        place = _rows_of(s, c, i, range(n))
        for lay in range(layers):
            for g in range(hk):
                x = acc[lay, i, g, :n]
                middle = np.arange(first, n - last)
                best = middle[np.lexsort((middle, -x[middle]))][:m - first - last]
                stay = np.concatenate((np.arange(first), np.sort(best), np.arange(n - last, n)))
                kept[lay, i, g, :m] = stay
                out[lay, i, g, :n] = 0
                out[lay, i, g, :m] = x[stay]
                at = torch.from_numpy(stay).cuda()
                for y in (k, v):
                    y[lay, place[:m], g] = y[lay, place[at], g].clone()
    return {"kept": torch.from_numpy(kept), "lens": torch.tensor(new, dtype=torch.int32),
            "acc": torch.from_numpy(out), "k": k.view(s["k"].shape), "v": v.view(s["v"].shape)}


def _exact_verify(s, c):
    b, t = c["batch"], c["nodes"]
    path = np.full((b, t), -1, np.int32)
    count, token = np.zeros(b, np.int32), np.zeros(b, np.int32)
    x, u = s["tokens"].tolist(), s["u"].double().tolist()
    parents, nodes = s["parent"].tolist(), s["n"].tolist()
    for i in range(b):
        at, kept, rows = -1, [], {}

        def row(name, r):
            if (name, r) not in rows:
                rows[name, r] = s[name][i, r].double().cpu().numpy()
            return rows[name, r]

        while True:
            children = [j for j in range(nodes[i]) if parents[i][j] == at]
            p = row("p", at + 1)
            # what is left of p and of q, each with its sum
            rest, mass, found = p.copy(), 1.0, None
            if children and s["q"] is not None:
                q, q_mass = row("q", at + 1).copy(), 1.0
            for j in children:
                y = x[i][j]
                if s["q"] is None:
                    if rest[y] > 0 and u[i][j] * mass < rest[y]:
                        found = j
                        break
                    mass = max(mass - rest[y], 0.0)
                    rest[y] = 0
                    continue
                if rest[y] > 0 and u[i][j] * q[y] / q_mass * mass < rest[y]:
                    found = j
                    break
                rest = np.maximum(rest - q * (mass / q_mass), 0)
                mass = rest.sum()
                if c["draft"] == "distinct":
                    q_mass = max(q_mass - q[y], 2.0 ** -24)
                    q[y] = 0
            if found is None:
                break
            kept.append(found)
            at = found
        if not rest.sum() > 0:
            rest = p
        sums = np.cumsum(rest)
        token[i] = int(np.searchsorted(sums, u[i][t] * sums[-1], side="right")) if sums[-1] > 0 else -1
        path[i, :len(kept)] = kept
        count[i] = len(kept)
    return {"path": torch.from_numpy(path), "count": torch.from_numpy(count), "next": torch.from_numpy(token)}
