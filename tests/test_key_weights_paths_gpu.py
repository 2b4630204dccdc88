"""key_weights(_paged) on the GPU: calls at the ends of what it takes, on each of its ways
(scores stored, query rows in registers, keys in registers)."""
import numpy as np
import pytest
import torch

from test_key_weights_gpu import rule
from ullm_amd import _lib as L
from ullm_amd import attention as A

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


@pytest.mark.parametrize("kv", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (32, 1, 64), (320, 1, 64), (8, 4, 256)])
def test_no_rows(dev, kv, H, Hk, D):
    """Rows of none: the weights fade, each by one rounding."""
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.empty(3, 0, H, D, dtype=kv, device=dev)
    k = torch.randn(3, 96, Hk * D, device=dev, generator=g).to(kv)
    old = torch.rand(3, Hk, 96, device=dev, generator=g)
    lens, there = i32([96, 0, 41], dev), torch.arange(96, device=dev) < torch.tensor([96, 0, 41], device=dev)[:, None, None]
    table = i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]], dev)
    for window in (0, 20):
        for decay in (0.0, 0.3, 1.0):
            want = torch.where(there, decay * old, old)
            for w in (A.key_weights(q, k, old.clone(), lens, 96, Hk, window=window, decay=decay),
                      A.key_weights_paged(q, k.view(9, 32, Hk * D), table, old.clone(), lens, 96, Hk, window=window, decay=decay)):
                assert torch.equal(w, want)


def against_64_bits(w, old, q, k, lens, n_rows, decay=1.0, window=0):
    """w [B, Hk, n] after a call over k [B, n, Hk * D] (old before it), by the bounds of
    test_key_weights_gpu.py."""
    B, rows, H, D = q.shape
    Hk = w.shape[1]
    G = H // Hk
    for b in range(B):
        n, r = min(max(lens[b], 0), k.shape[1]), min(max(n_rows[b], 0), rows)
        assert torch.equal(w[b, :, n:], old[b, :, n:]), "positions past the length"
        for j in range(Hk):
            want, rel, low = rule(q[b, :, j * G:(j + 1) * G].double(), k[b, :n, j * D:(j + 1) * D].double(), n, r, window, D ** -0.5)
            was = decay * old[b, j, :n].double() if decay else torch.zeros(n, dtype=torch.float64, device=w.device)
            over = (w[b, j, :n].double() - want - was).abs() - (want * rel + low + 4 * U * (want + was))
            assert n == 0 or over.max().item() <= 0, (b, j, over.max().item())


@pytest.mark.parametrize("kv,D", [(torch.float16, 64), (torch.float32, 256)])
def test_longest_that_is_always_taken(dev, kv, D):
    """2^26 - 1 positions of one kv head and 4096 rows, as far as launches and workspace go: the
    sequence itself is 5000 positions of one large page."""
    g = torch.Generator(device=dev).manual_seed(3)
    rows, n, page, max_len = 4096, 5000, 1 << 16, (1 << 26) - 1
    q = torch.randn(1, rows, 1, D, device=dev, generator=g).to(kv)
    pool = torch.randn(1, page, D, device=dev, generator=g).to(kv)
    table = torch.full((1, 1024), -1, dtype=torch.int32, device=dev)
    table[0, 0] = 0
    w = torch.full((1, 1, max_len), 0.5, device=dev)
    A.key_weights_paged(q, pool, table, w, i32([n], dev), max_len, 1)
    assert (w[0, 0, n:] == 0.5).all()
    against_64_bits(w[..., :n], torch.full((1, 1, n), 0.5, device=dev), q, pool[:, :n], [n], [rows])


# cache, f32 queries, rows, heads, kv heads, head_dim, max_len: scores stored; query rows in
# registers, shared by one, two and four waves; keys in registers, the denominators of one
# part a row block (128 keys; 32 kv heads' rows, which fill the card) and of several
F16, F32, BF16 = torch.float16, torch.float32, torch.bfloat16
WAYS = [(BF16, False, 4, 8, 2, 128, 700), (F16, True, 1, 14, 2, 64, 333), (F32, True, 3, 4, 1, 256, 260),
        (BF16, False, 12, 8, 2, 128, 700), (F16, True, 30, 8, 2, 64, 900), (BF16, True, 50, 2, 1, 128, 500),
        (F16, False, 250, 1, 1, 64, 1300), (F32, True, 60, 1, 1, 128, 300),
        (BF16, False, 300, 2, 1, 64, 128), (BF16, True, 600, 32, 8, 64, 700), (F16, True, 300, 6, 2, 128, 900),
        (F16, False, 300, 6, 2, 64, 900), (F32, True, 90, 8, 2, 256, 400)]


@pytest.mark.parametrize("fill", [255, 127, 0])
@pytest.mark.parametrize("kv,f32,rows,H,Hk,D,max_len", WAYS)
def test_odd_counts_over_a_full_workspace(dev, kv, f32, rows, H, Hk, D, max_len, fill):
    """Lengths past max_len and below 0, rows past max_rows and more than positions, over a
    workspace that holds NaN, 3.4e38 or 0, on a stream of its own; windows and pages."""
    g = torch.Generator(device=dev).manual_seed(rows + D)
    B, page = 4, 32
    lens, n_rows = [1 << 20, -5, max_len * 3 // 4, 41], [rows, rows, 1 << 20, rows]
    q = torch.randn(B, rows, H, D, device=dev, generator=g).to(F32 if f32 else kv)
    cols = -(-max_len // page)
    pool = torch.randn(B * cols, page, Hk * D, device=dev, generator=g).to(kv)
    k = pool.view(B, cols * page, Hk * D)[:, :max_len]
    table = torch.arange(B * cols, dtype=torch.int32, device=dev).view(B, cols).contiguous()
    old = torch.rand(B, Hk, max_len + 3, device=dev, generator=g)
    code = {F32: L.DT_F32, F16: L.DT_F16, BF16: L.DT_BF16}[kv]
    count, length, stream = i32(n_rows, dev), i32(lens, dev), torch.cuda.Stream()
    for window in (0, 50):
        size = L.lib().ullm_hip_key_weights_workspace_bytes(code, B, rows, max_len, window, H, Hk, D)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        for paged in (False, True):
            ws.fill_(fill)
            w = old.clone()
            more = dict(n_rows=count, window=window, decay=0.5, workspace=ws, stream=stream)
            torch.cuda.synchronize()
            if paged:
                A.key_weights_paged(q, pool, table, w, length, max_len, Hk, **more)
            else:
                A.key_weights(q, k, w, length, max_len, Hk, **more)
            stream.synchronize()
            against_64_bits(w, old, q, k, lens, n_rows, 0.5, window)
