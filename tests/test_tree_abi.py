"""The drafted trees' entry points on the CPU: bad arguments get their codes before
any device work, sizes of the workspaces, and the masks."""
import ctypes as C
import re

import numpy as np
import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A

FAKE, ODD = C.c_void_p(0x10000), C.c_void_p(0x10008)
BIG = 1 << 40


def call(name, base, **change):
    a = dict(base)
    assert not set(change) - set(a), change
    a.update(change)
    return getattr(L.lib(), "ullm_hip_" + name)(*a.values())


ATTN = dict(q=FAKE, k=FAKE, v=FAKE, dtype=L.DT_F16, kvs=256, ss=256 * 99, mask=FAKE, lens=FAKE, n=FAKE, pos=FAKE, nodes=9,
            max_len=99, window=0, batch=2, H=8, Hk=2, D=128, scale=0.1, out=FAKE, odt=L.DT_F16, ws=FAKE, wsn=BIG, st=None)
PAGED = dict(q=FAKE, k=FAKE, v=FAKE, dtype=L.DT_F16, kvs=256, P=32, pages=9, tab=FAKE, cols=4, mask=FAKE, lens=FAKE, n=FAKE,
             pos=FAKE, nodes=9, max_len=99, window=0, batch=2, H=8, Hk=2, D=128, scale=0.1, out=FAKE, odt=L.DT_F16, ws=FAKE,
             wsn=BIG, st=None)
BAD_ATTN = [
    (dict(dtype=5), L.E_UNSUPPORTED), (dict(D=96), L.E_UNSUPPORTED), (dict(odt=L.DT_BF16), L.E_UNSUPPORTED),
    (dict(odt=7), L.E_UNSUPPORTED), (dict(Hk=3), L.E_INVALID), (dict(Hk=0), L.E_INVALID), (dict(H=0), L.E_INVALID),
    (dict(nodes=1025), L.E_INVALID), (dict(nodes=-1), L.E_INVALID), (dict(batch=-1), L.E_INVALID),
    (dict(batch=65536), L.E_INVALID), (dict(max_len=-1), L.E_INVALID), (dict(window=-1), L.E_INVALID),
    (dict(kvs=255), L.E_INVALID), (dict(kvs=260), L.E_INVALID), (dict(kvs=1 << 40), L.E_INVALID),
    (dict(q=None), L.E_INVALID), (dict(k=None), L.E_INVALID), (dict(v=None), L.E_INVALID), (dict(lens=None), L.E_INVALID),
    (dict(out=None), L.E_INVALID), (dict(q=ODD), L.E_INVALID), (dict(k=ODD), L.E_INVALID), (dict(out=ODD), L.E_INVALID),
    (dict(window=5, pos=None), L.E_INVALID), (dict(nodes=1024, H=8200, Hk=2), L.E_INVALID),
    (dict(batch=65535, H=512, Hk=256, kvs=256 * 128), L.E_INVALID),
]


@pytest.mark.parametrize("change,code", BAD_ATTN + [(dict(ss=-8), L.E_INVALID), (dict(ss=4), L.E_INVALID)])
def test_attn_refuses(change, code):
    assert call("attn_tree", ATTN, **change) == code
    assert L.lib().ullm_hip_last_error()


@pytest.mark.parametrize("change,code", BAD_ATTN + [
    (dict(P=16), L.E_INVALID), (dict(P=48), L.E_INVALID), (dict(pages=0), L.E_INVALID), (dict(cols=3), L.E_INVALID),
    (dict(tab=None), L.E_INVALID)])
def test_attn_paged_refuses(change, code):
    assert call("attn_tree_paged", PAGED, **change) == code


def test_nothing_to_do():
    for change in (dict(batch=0), dict(nodes=0)):
        assert call("attn_tree", ATTN, **change, q=None, out=None) == L.OK
        assert call("attn_tree_paged", PAGED, **change, q=None, tab=None) == L.OK
        assert call("qkv_append_tree", APPEND, **change, q=None) == L.OK
    assert call("kv_accept", ACCEPT, batch=0, k=None) == L.OK
    assert call("kv_pages_update", UPDATE, n=0, k=None) == L.OK


APPEND = dict(q=FAKE, k=FAKE, v=FAKE, qb=None, kb=None, vb=None, qn=None, kn=None, eps=1e-6, cs=FAKE, n_pos=99, neox=1, rd=128,
              batch=2, nodes=9, lens=FAKE, n=None, pos=None, H=8, Hk=2, D=128, qo=FAKE, qdt=L.DT_F16, kc=FAKE, vc=FAKE,
              kdt=L.DT_F16, kvs=256, ss=256 * 99, n_ctx=99, st=None)
APPEND_P = {**{n: x for n, x in APPEND.items() if n not in ("ss", "n_ctx", "st")}, "P": 32, "pages": 9, "tab": FAKE, "cols": 4, "st": None}
BAD_APPEND = [
    (dict(qdt=4), L.E_UNSUPPORTED), (dict(kdt=4), L.E_UNSUPPORTED), (dict(D=32), L.E_UNSUPPORTED), (dict(H=7), L.E_INVALID),
    (dict(rd=130), L.E_INVALID), (dict(rd=3), L.E_INVALID), (dict(kvs=128), L.E_INVALID), (dict(n_pos=0), L.E_INVALID),
    (dict(batch=-1), L.E_INVALID), (dict(batch=1 << 20, nodes=1 << 20), L.E_INVALID), (dict(lens=None), L.E_INVALID),
    (dict(qo=None), L.E_INVALID), (dict(cs=None), L.E_INVALID), (dict(kc=ODD), L.E_INVALID), (dict(kvs=260), L.E_INVALID),
    (dict(q=ODD), L.E_INVALID), (dict(kb=ODD), L.E_INVALID),
]


@pytest.mark.parametrize("change,code", BAD_APPEND)
def test_append_refuses(change, code):
    # in-place q of another type among them: qo is q here
    assert call("qkv_append_tree", {**APPEND, "qo": C.c_void_p(0x20000)}, **change) == code
    assert call("qkv_append_tree_paged", {**APPEND_P, "qo": C.c_void_p(0x20000)}, **change) == code


def test_append_refuses_more():
    assert call("qkv_append_tree", APPEND) == L.E_INVALID  # q_out is q, of another type
    apart = {**APPEND, "qo": C.c_void_p(0x20000)}
    for change in (dict(ss=-8), dict(ss=4), dict(n_ctx=-1)):
        assert call("qkv_append_tree", apart, **change) == L.E_INVALID
    apart = {**APPEND_P, "qo": C.c_void_p(0x20000)}
    for change in (dict(P=0), dict(P=24), dict(pages=0), dict(cols=0), dict(tab=None)):
        assert call("qkv_append_tree_paged", apart, **change) == L.E_INVALID


ACCEPT = dict(k=FAKE, v=FAKE, dtype=L.DT_F16, kvs=256, ss=256 * 99, n_ctx=99, kvd=256, NL=3, ls=256 * 99 * 2, path=FAKE, T=9,
              n=FAKE, lens=FAKE, out=C.c_void_p(0x20000), batch=2, st=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), L.E_UNSUPPORTED), (dict(batch=-1), L.E_INVALID), (dict(batch=65536), L.E_INVALID), (dict(T=1025), L.E_INVALID),
    (dict(T=-1), L.E_INVALID), (dict(NL=0), L.E_INVALID), (dict(NL=40000), L.E_INVALID), (dict(kvd=0), L.E_INVALID),
    (dict(kvd=264), L.E_INVALID), (dict(kvd=4), L.E_INVALID), (dict(ss=-8), L.E_INVALID), (dict(ss=4), L.E_INVALID),
    (dict(ls=4), L.E_INVALID), (dict(ls=-8), L.E_INVALID), (dict(ls=0), L.E_INVALID), (dict(ss=0), L.E_INVALID), (dict(n_ctx=-1), L.E_INVALID), (dict(k=None), L.E_INVALID),
    (dict(path=None), L.E_INVALID), (dict(n=None), L.E_INVALID), (dict(lens=None), L.E_INVALID), (dict(k=ODD), L.E_INVALID),
    (dict(out=FAKE), L.E_INVALID), (dict(out=C.c_void_p(0x10004)), L.E_INVALID)])
def test_accept_refuses(change, code):
    assert call("kv_accept", ACCEPT, **change) == code


def test_accept_paged_refuses():
    paged = dict(k=FAKE, v=FAKE, dtype=L.DT_F16, kvs=256, P=32, pages=9, kvd=256, NL=3, ls=256 * 99 * 2, tab=FAKE, cols=3,
                 path=FAKE, T=9, n=FAKE, lens=FAKE, out=None, batch=2, st=None)
    for change in (dict(P=3), dict(pages=0), dict(cols=0), dict(tab=None), dict(T=2000), dict(k=ODD), dict(kvs=8)):
        assert call("kv_accept_paged", paged, **change) == L.E_INVALID


UPDATE = dict(k=FAKE, v=FAKE, dtype=L.DT_F16, kvs=256, P=32, pages=99, NL=2, ls=256 * 32 * 99, tab=FAKE, cols=4, lens=FAKE, S=3,
              parent=FAKE, cap=FAKE, held=None, to=C.c_void_p(0x20000), out_cols=4, lo=C.c_void_p(0x30000), n=3,
              info=C.c_void_p(0x40000), ws=C.c_void_p(0x50000), wsn=BIG, st=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), L.E_UNSUPPORTED), (dict(P=33), L.E_INVALID), (dict(pages=0), L.E_UNSUPPORTED),
    (dict(pages=(1 << 20) + 1), L.E_UNSUPPORTED), (dict(NL=-1), L.E_INVALID), (dict(S=-1), L.E_INVALID),
    (dict(n=-1), L.E_INVALID), (dict(n=65536), L.E_INVALID), (dict(cols=0), L.E_INVALID), (dict(out_cols=0), L.E_INVALID),
    (dict(out_cols=1 << 27), L.E_INVALID), (dict(n=65535, out_cols=(1 << 15) + 1), L.E_INVALID), (dict(n=3, out_cols=1 << 30, P=1), L.E_INVALID), (dict(cols=1 << 27), L.E_INVALID), (dict(kvs=0), L.E_INVALID),
    (dict(kvs=4), L.E_INVALID), (dict(ls=4), L.E_INVALID), (dict(ls=-8), L.E_INVALID), (dict(k=None), L.E_INVALID),
    (dict(tab=None), L.E_INVALID), (dict(lens=None), L.E_INVALID), (dict(parent=None), L.E_INVALID), (dict(cap=None), L.E_INVALID),
    (dict(to=None), L.E_INVALID), (dict(lo=None), L.E_INVALID), (dict(info=None), L.E_INVALID), (dict(k=ODD), L.E_INVALID),
    (dict(to=FAKE), L.E_INVALID), (dict(lo=FAKE, lens=C.c_void_p(0x60000)), L.E_INVALID),
    (dict(ws=None), L.E_WORKSPACE), (dict(wsn=64), L.E_WORKSPACE), (dict(ws=ODD), L.E_WORKSPACE)])
def test_update_refuses(change, code):
    assert call("kv_pages_update", UPDATE, **change) == code


def test_workspace_sizes():
    f = L.lib().ullm_hip_kv_pages_workspace_bytes
    assert f(0, 5) == 0 and f(5, 0) == 0 and f(1, 1) >= 8
    assert f(64, 1000) > f(32, 1000) and f(64, 2000) > f(64, 1000)
    f = L.lib().ullm_hip_tree_workspace_bytes
    assert f(L.DT_F16, 1, 4, 100, 0, 8, 3, 128) == 0 and f(L.DT_F16, 1, 4, 100, 0, 8, 2, 96) == 0
    assert f(9, 1, 4, 100, 0, 8, 2, 128) == 0 and f(L.DT_F16, 0, 4, 100, 0, 8, 2, 128) == 0


def _gpu_visible():
    return torch.cuda.device_count() > 0


@pytest.mark.parametrize("dt", [L.DT_F32, L.DT_F16, L.DT_BF16])
@pytest.mark.parametrize("H,Hk,D", [(32, 8, 64), (12, 2, 128), (8, 4, 256), (32, 1, 128), (5, 5, 64)])
def test_workspace_serves_every_smaller_call(dt, H, Hk, D):
    """The header's promise, over shapes whose workgroups change with the sizes: what
    a call needs is read from its refusal.  A call that needs none reaches a launch,
    so this runs only where there is no GPU."""
    if _gpu_visible():
        pytest.skip("launches kernels on fake pointers when a GPU is visible; runs on CPU-only hosts")
    for T in (1, 8, 17, 64, 130):
        for win in (0, 100, 1024):
            size = L.lib().ullm_hip_tree_workspace_bytes(dt, 8, T, 4096, win, H, Hk, D)
            for B in (1, 3, 8):
                for t in {1, T // 2 or 1, T}:
                    for n in (1, 31, 40, 300, 1000, 4096):
                        rc = call("attn_tree", ATTN, dtype=dt, odt=dt, kvs=Hk * D, ss=0, nodes=t, max_len=n, window=win,
                                  batch=B, H=H, Hk=Hk, D=D, ws=None, wsn=0)
                        if rc == L.E_WORKSPACE:
                            assert int(re.search(rb"workspace of (\d+)", L.lib().ullm_hip_last_error()).group(1)) <= size
                        else:
                            assert rc in (L.OK, L.E_HIP)


def test_tree_masks():
    parents = np.array([[-1, 0, 0, 2, -1], [-1, 0, 1, 2, 3]])
    mask, depth = A.tree_masks(parents)
    assert mask.shape == (2, 5, 1) and mask.dtype == torch.int64 and depth.dtype == torch.int32
    assert mask[0, :, 0].tolist() == [1, 3, 5, 13, 16] and depth[0].tolist() == [0, 1, 1, 2, 0]
    assert mask[1, :, 0].tolist() == [1, 3, 7, 15, 31] and depth[1].tolist() == [0, 1, 2, 3, 4]
    long = torch.arange(130) - 1
    mask, depth = A.tree_masks(long)
    assert mask.shape == (130, 3) and mask[129].tolist() == [-1, -1, 3] and mask[63].tolist() == [-1, 0, 0]
    assert depth.tolist() == list(range(130))
    assert A.tree_masks(np.zeros((3, 0), int))[0].shape == (3, 0, 0)
    with pytest.raises(L.UllmHipError):
        A.tree_masks([-1, 1])
