"""Refusals of the drafted trees' and page tables' entry points at their edges, on
the CPU: codes come before any device work."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_tree_abi import ACCEPT, APPEND, FAKE, ODD, UPDATE, call
from ullm_amd import _lib as L
from ullm_amd import attention as A

ROWS = {**{n: x for n, x in UPDATE.items() if n in ("k", "v", "dtype", "kvs", "P", "pages")}, "kvd": 128,
        **{n: x for n, x in UPDATE.items() if n not in ("k", "v", "dtype", "kvs", "P", "pages")}}


@pytest.mark.parametrize("change,code", [
    (dict(kvd=0), L.E_INVALID), (dict(kvd=-8), L.E_INVALID), (dict(kvd=264), L.E_INVALID), (dict(kvd=12), L.E_INVALID),
    (dict(ls=120), L.E_INVALID), (dict(ls=0), L.E_INVALID), (dict(kvs=132), L.E_INVALID), (dict(dtype=3), L.E_UNSUPPORTED),
    (dict(k=ODD), L.E_INVALID), (dict(tab=None), L.E_INVALID), (dict(to=FAKE), L.E_INVALID), (dict(wsn=64), L.E_WORKSPACE)])
def test_update_rows_refuses(change, code):
    assert call("kv_pages_update_rows", ROWS, **change) == code


def test_update_rows_of_nothing():
    assert call("kv_pages_update_rows", ROWS, n=0, k=None) == L.OK


@pytest.mark.parametrize("kvs,ss", [(256, 0), (256, 8), (256, 248), (512, 256), (768, 256), (1024, 512)])
def test_sequences_that_share_rows_are_refused(kvs, ss):
    """Four sequences whose first rows overlap, or whose rows lie between another's."""
    apart = {**APPEND, "qo": C.c_void_p(0x20000), "batch": 4, "kvs": kvs, "ss": ss}
    assert call("qkv_append_tree", apart) == L.E_INVALID
    assert b"share rows" in L.lib().ullm_hip_last_error()
    assert call("kv_accept", {**ACCEPT, "batch": 4, "kvs": kvs, "ss": ss}) == L.E_INVALID
    assert b"share rows" in L.lib().ullm_hip_last_error()


def test_parents_of_a_tree():
    """Any number below 0 is the sequence itself; what is no whole number, or no
    earlier node, is refused."""
    for parents in ([-9, 0, 1], [-1, 0, -7], [[-100, -2], [-(1 << 40), 0]]):
        at = np.array(parents)
        mask, depth = A.tree_masks(at)
        same = A.tree_masks(np.maximum(at, -1))
        assert torch.equal(mask, same[0]) and torch.equal(depth, same[1])
    assert A.tree_masks(torch.tensor([-5, 0], dtype=torch.int8))[1].tolist() == [0, 1]
    assert A.tree_masks([])[0].shape == (0, 0) and A.tree_masks([-1.0, 0.0, 0.0])[1].tolist() == [0, 1, 1]
    for parents in ([-1.0, 0.5], np.array([(1 << 64) - 1], np.uint64), [-1, 1 << 40], [True, False], [-1, float("nan")], 3):
        with pytest.raises(L.UllmHipError):
            A.tree_masks(parents)


def test_outputs_in_what_is_still_read_are_refused():
    """lens_out inside path or the block table, and page outputs inside the old table
    or one another."""
    far = {**ACCEPT, "path": C.c_void_p(0x60000), "lens": C.c_void_p(0x70000), "n": C.c_void_p(0x80000)}
    for out in (0x60000, 0x60000 + 4 * 17, 0x60000 - 4):  # 2 x 9 entries
        assert call("kv_accept", {**far, "out": C.c_void_p(out)}) == L.E_INVALID
    paged = dict(k=FAKE, v=FAKE, dtype=L.DT_F16, kvs=256, P=32, pages=9, kvd=256, NL=3, ls=256 * 99 * 2, tab=C.c_void_p(0x90000),
                 cols=3, path=far["path"], T=9, n=far["n"], lens=far["lens"], out=None, batch=2, st=None)
    for out in (0x90000, 0x90000 + 4 * 5, 0x60000 + 4):
        assert call("kv_accept_paged", {**paged, "out": C.c_void_p(out)}) == L.E_INVALID
    far = {**ROWS, "tab": C.c_void_p(0x90000), "lens": C.c_void_p(0x70000), "parent": C.c_void_p(0x80000), "cap": C.c_void_p(0xa0000)}
    for change in (dict(info=0x90000 + 4 * 11), dict(lo=0x90000 + 4 * 11), dict(info=0x20000 + 4 * 11), dict(lo=0x20000 + 4 * 11),
                   dict(info=0x30000 + 8), dict(to=0x40000 - 4 * 11)):
        assert call("kv_pages_update_rows", far, **{n: C.c_void_p(x) for n, x in change.items()}) == L.E_INVALID
        assert b"overlap" in L.lib().ullm_hip_last_error()


def test_append_of_more_rows_than_a_launch_has():
    apart = {**APPEND, "qo": C.c_void_p(0x20000), "kvs": 256, "ss": 256 * 99}
    for batch, nodes in ((1 << 24, 1), (1, 1 << 24), (1 << 14, 1 << 10), ((1 << 29) - 1, 1), ((1 << 31) - 1, (1 << 31) - 1), (1 << 30, 1 << 26)):
        assert call("qkv_append_tree", {**apart, "batch": batch, "nodes": nodes}) == L.E_INVALID
