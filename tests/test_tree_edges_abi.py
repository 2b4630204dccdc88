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
