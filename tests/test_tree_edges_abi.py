"""Refusals of the drafted trees' and page tables' entry points at their edges, on
the CPU: codes come before any device work."""
import pytest

from test_tree_abi import FAKE, ODD, UPDATE, call
from ullm_amd import _lib as L

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
