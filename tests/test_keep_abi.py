"""The entry points that decide what a cache keeps (ullm_hip_tree_verify,
ullm_hip_key_weights, ullm_hip_kv_evict), on the CPU: bad arguments get their codes
before any device work, and the sizes of the workspaces."""
import ctypes as C
import re

import pytest
import torch

from ullm_amd import _lib as L
from ullm_amd import attention as A


def at(n):
    return C.c_void_p(n << 32)


FAKE, ODD = at(1), C.c_void_p((1 << 32) + 8)
BIG = 1 << 40


def call(name, base, **change):
    a = dict(base)
    assert not set(change) - set(a), change
    a.update(change)
    return getattr(L.lib(), "ullm_hip_" + name)(*a.values())


VERIFY = dict(p=at(1), ps=5 * 99, pr=99, q=at(2), qs=4 * 99, qr=99, dtype=L.DT_F32, V=99, tok=at(3), par=at(4), n=at(5), u=at(6),
              T=4, distinct=0, B=2, path=at(7), count=at(8), next=at(9), ws=at(10), wsn=BIG, st=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), L.E_UNSUPPORTED), (dict(V=0), L.E_INVALID), (dict(V=(1 << 30) + 1), L.E_INVALID), (dict(T=-1), L.E_INVALID),
    (dict(T=1025), L.E_INVALID), (dict(B=-1), L.E_INVALID), (dict(B=65536), L.E_INVALID), (dict(ps=-1), L.E_INVALID),
    (dict(pr=-1), L.E_INVALID), (dict(qs=-1), L.E_INVALID), (dict(qr=-1), L.E_INVALID), (dict(p=None), L.E_INVALID),
    (dict(tok=None), L.E_INVALID), (dict(u=None), L.E_INVALID), (dict(path=None), L.E_INVALID), (dict(count=None), L.E_INVALID),
    (dict(next=None), L.E_INVALID), (dict(p=C.c_void_p(0x100000002)), L.E_INVALID), (dict(q=C.c_void_p(0x100000001)), L.E_INVALID),
    (dict(path=at(3)), L.E_INVALID), (dict(path=at(4)), L.E_INVALID), (dict(count=at(5)), L.E_INVALID), (dict(next=at(6)), L.E_INVALID),
    (dict(next=at(8)), L.E_INVALID), (dict(count=at(7)), L.E_INVALID), (dict(ws=None), L.E_WORKSPACE), (dict(wsn=8), L.E_WORKSPACE),
    (dict(ws=ODD), L.E_WORKSPACE)])
def test_verify_refuses(change, code):
    assert call("tree_verify", VERIFY, **change) == code
    assert L.lib().ullm_hip_last_error()


WEIGHTS = dict(q=FAKE, qdt=L.DT_F32, k=FAKE, dtype=L.DT_F16, kvs=256, ss=256 * 99, lens=FAKE, n=None, rows=9, max_len=99, window=0,
               batch=2, H=8, Hk=2, D=128, scale=0.1, decay=1.0, w=FAKE, ws_row=99, ws=FAKE, wsn=BIG, st=None)
WEIGHTS_P = dict(q=FAKE, qdt=L.DT_F32, k=FAKE, dtype=L.DT_F16, kvs=256, P=32, pages=9, tab=FAKE, cols=4, lens=FAKE, n=None, rows=9,
                 max_len=99, window=0, batch=2, H=8, Hk=2, D=128, scale=0.1, decay=1.0, w=FAKE, ws_row=99, ws=FAKE, wsn=BIG, st=None)
BAD_WEIGHTS = [
    (dict(dtype=5), L.E_UNSUPPORTED), (dict(qdt=L.DT_BF16), L.E_UNSUPPORTED), (dict(qdt=9), L.E_UNSUPPORTED),
    (dict(dtype=L.DT_F32, qdt=L.DT_F16), L.E_UNSUPPORTED), (dict(D=96), L.E_UNSUPPORTED), (dict(Hk=3), L.E_INVALID),
    (dict(Hk=0), L.E_INVALID), (dict(H=0), L.E_INVALID), (dict(rows=-1), L.E_INVALID), (dict(rows=1 << 21), L.E_INVALID),
    (dict(batch=-1), L.E_INVALID), (dict(batch=65536), L.E_INVALID), (dict(max_len=-1), L.E_INVALID), (dict(window=-1), L.E_INVALID),
    (dict(kvs=255), L.E_INVALID), (dict(kvs=260), L.E_INVALID), (dict(ws_row=98), L.E_INVALID), (dict(q=None), L.E_INVALID),
    (dict(k=None), L.E_INVALID), (dict(lens=None), L.E_INVALID), (dict(w=None), L.E_INVALID), (dict(q=ODD), L.E_INVALID),
    (dict(k=ODD), L.E_INVALID), (dict(ws=None), L.E_WORKSPACE), (dict(wsn=8), L.E_WORKSPACE), (dict(ws=ODD), L.E_WORKSPACE)]


@pytest.mark.parametrize("change,code", BAD_WEIGHTS + [(dict(ss=-8), L.E_INVALID), (dict(ss=4), L.E_INVALID)])
def test_weights_refuse(change, code):
    assert call("key_weights", WEIGHTS, **change) == code
    assert L.lib().ullm_hip_last_error()


@pytest.mark.parametrize("change,code", BAD_WEIGHTS + [
    (dict(P=16), L.E_INVALID), (dict(P=48), L.E_INVALID), (dict(pages=0), L.E_INVALID), (dict(cols=3), L.E_INVALID),
    (dict(tab=None), L.E_INVALID)])
def test_weights_paged_refuse(change, code):
    assert call("key_weights_paged", WEIGHTS_P, **change) == code


EVICT = dict(k=at(1), v=at(2), dtype=L.DT_F16, kvs=256, ss=256 * 99, n_ctx=99, kvd=256, NL=3, ls=256 * 99 * 2, s=at(3), so=at(3),
             ss_row=99, G=2, lens=at(4), budget=at(5), top=50, sink=1, recent=2, kept=at(6), out=at(7), batch=2, st=None)
BAD_EVICT = [
    (dict(dtype=3), L.E_UNSUPPORTED), (dict(batch=-1), L.E_INVALID), (dict(batch=40000), L.E_INVALID), (dict(G=0), L.E_INVALID),
    (dict(G=3), L.E_INVALID), (dict(G=64), L.E_INVALID), (dict(NL=0), L.E_INVALID), (dict(NL=40000), L.E_INVALID),
    (dict(kvd=0), L.E_INVALID), (dict(kvd=264), L.E_INVALID), (dict(ls=4), L.E_INVALID), (dict(ls=-8), L.E_INVALID),
    (dict(ls=0), L.E_INVALID), (dict(top=-1), L.E_INVALID), (dict(sink=-1), L.E_INVALID), (dict(recent=-1), L.E_INVALID),
    (dict(ss_row=-1), L.E_INVALID), (dict(k=None), L.E_INVALID), (dict(v=None), L.E_INVALID), (dict(lens=None), L.E_INVALID),
    (dict(budget=None), L.E_INVALID), (dict(s=None), L.E_INVALID), (dict(kept=None), L.E_INVALID), (dict(k=ODD), L.E_INVALID),
    (dict(out=at(4)), L.E_INVALID), (dict(out=at(5)), L.E_INVALID), (dict(kept=at(3)), L.E_INVALID), (dict(kept=at(4)), L.E_INVALID),
    (dict(kept=at(7)), L.E_INVALID), (dict(so=C.c_void_p((3 << 32) + 4)), L.E_INVALID), (dict(so=at(4)), L.E_INVALID),
    (dict(so=at(6), s=at(8)), L.E_INVALID), (dict(ss_row=(1 << 30) + 1), L.E_INVALID),
    (dict(NL=32767, batch=100, G=2), L.E_INVALID), (dict(NL=32767, kvd=16384, kvs=16384, ss=16384 * 99, ls=16384 * 99 * 2), L.E_INVALID)]


@pytest.mark.parametrize("change,code", BAD_EVICT + [
    (dict(ss=-8), L.E_INVALID), (dict(ss=4), L.E_INVALID), (dict(ss=0), L.E_INVALID), (dict(n_ctx=-1), L.E_INVALID)])
def test_evict_refuses(change, code):
    assert call("kv_evict", EVICT, **change) == code
    assert L.lib().ullm_hip_last_error()


@pytest.mark.parametrize("change,code", BAD_EVICT + [
    (dict(P=3), L.E_INVALID), (dict(pages=0), L.E_INVALID), (dict(cols=0), L.E_INVALID), (dict(tab=None), L.E_INVALID),
    (dict(kept=at(9)), L.E_INVALID), (dict(out=at(9)), L.E_INVALID), (dict(so=at(9)), L.E_INVALID)])
def test_evict_paged_refuses(change, code):
    a = {}
    for n, x in EVICT.items():
        a.update(dict(P=32, pages=9) if n == "ss" else {} if n == "n_ctx" else {n: x})
        if n == "ls":
            a.update(tab=at(9), cols=4)
    assert call("kv_evict_paged", a, **{n: x for n, x in change.items() if n != "ss"}) == code


def test_nothing_to_do():
    assert call("tree_verify", VERIFY, B=0, p=None, ws=None) == L.OK
    for change in (dict(batch=0), dict(max_len=0)):
        assert call("key_weights", WEIGHTS, **change, q=None, ws=None) == L.OK
        assert call("key_weights_paged", WEIGHTS_P, **change, q=None, ws=None) == L.OK
    assert call("kv_evict", EVICT, batch=0, k=None) == L.OK


def test_workspace_sizes():
    f = L.lib().ullm_hip_tree_verify_workspace_bytes
    assert f(0, 5) == 0 and f(5, 0) == 0 and f(1, 1) > 0
    assert all(f(v, 4) <= f(v + 1, 4) <= f(v + 1, 5) for v in range(1, 200000, 997))
    f = L.lib().ullm_hip_key_weights_workspace_bytes
    assert f(L.DT_F16, 1, 4, 100, 0, 8, 3, 128) == 0 and f(L.DT_F16, 1, 4, 100, 0, 8, 2, 96) == 0
    assert f(9, 1, 4, 100, 0, 8, 2, 128) == 0 and f(L.DT_F16, 0, 4, 100, 0, 8, 2, 128) == 0


@pytest.mark.parametrize("dt", [L.DT_F32, L.DT_F16, L.DT_BF16])
@pytest.mark.parametrize("H,Hk,D", [(32, 8, 64), (12, 2, 128), (8, 4, 256), (32, 1, 128), (5, 5, 64)])
def test_weights_workspace_serves_every_smaller_call(dt, H, Hk, D):
    """The header's promise: what a call needs is read from its refusal.  A call that
    needs none reaches a launch, so this runs only where there is no GPU."""
    if torch.cuda.device_count() > 0:
        pytest.skip("launches kernels on fake pointers when a GPU is visible; runs on CPU-only hosts")
    for rows in (1, 8, 17, 130, 700):
        for win in (0, 100, 1024):
            size = L.lib().ullm_hip_key_weights_workspace_bytes(dt, 8, rows, 4096, win, H, Hk, D)
            for B in (1, 3, 8):
                for r in {1, rows // 2 or 1, rows}:
                    for n in (1, 31, 40, 300, 1000, 4096):
                        rc = call("key_weights", WEIGHTS, dtype=dt, qdt=L.DT_F32, kvs=Hk * D, ss=0, rows=r, max_len=n, ws_row=n,
                                  window=win, batch=B, H=H, Hk=Hk, D=D, ws=None, wsn=0)
                        if rc == L.E_WORKSPACE:
                            assert int(re.search(rb"workspace of (\d+)", L.lib().ullm_hip_last_error()).group(1)) <= size
                        else:
                            assert rc in (L.OK, L.E_HIP)


def test_front_refuses_tensors_of_the_host():
    x = torch.zeros(1, 1, 8, 64)
    i = torch.ones(1, dtype=torch.int32)
    for f in (lambda: A.key_weights(x, x[0], torch.zeros(1, 8, 1), i, 1, 8),
              lambda: A.kv_evict(x[0, 0], x[0, 0], torch.zeros(1, 1, 8), i, i, max_budget=1),
              lambda: A.tree_verify(x[0], None, torch.zeros(1, 7, dtype=torch.int32), torch.zeros(1, 8))):
        with pytest.raises(L.UllmHipError, match="GPU"):
            f()
