"""The ends of what ullm_hip_key_weights(_paged) takes, on the CPU.  What a call needs is
read from its refusal of a workspace that is none, so nothing is launched."""
import ctypes as C
import re

import pytest

from ullm_amd import _lib as L

FAKE = C.c_void_p(1 << 32)


def needs(dtype=L.DT_F16, qdt=L.DT_F32, rows=9, max_len=99, window=0, batch=2, H=8, Hk=2, D=128, page=0):
    """(code, bytes of workspace) of a call without one."""
    tail = [FAKE, None, rows, max_len, window, batch, H, Hk, D, 0.1, 1.0, FAKE, max_len, None, 0, None]
    if page:
        rc = L.lib().ullm_hip_key_weights_paged(FAKE, qdt, FAKE, dtype, Hk * D, page, 9, FAKE, -(-max_len // page), *tail)
    else:
        rc = L.lib().ullm_hip_key_weights(FAKE, qdt, FAKE, dtype, Hk * D, 0, *tail)
    m = re.search(rb"workspace of (\d+)", L.lib().ullm_hip_last_error())
    return rc, int(m.group(1)) if m else None


@pytest.mark.parametrize("dt", [L.DT_F32, L.DT_F16, L.DT_BF16])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (32, 1, 64), (320, 1, 64), (8, 4, 256)])
@pytest.mark.parametrize("window", [0, 40])
def test_workspace_of_a_call_without_rows(dt, H, Hk, D, window):
    """It is planned as one of one row: the size says so, and serves it from larger ones."""
    f = L.lib().ullm_hip_key_weights_workspace_bytes
    for qdt in (dt, L.DT_F32):
        for max_len in (1, 99, 5000):
            rc, need = needs(dt, qdt, 0, max_len, window, 2, H, Hk, D)
            assert rc == L.E_WORKSPACE and 0 < need <= f(dt, 2, 0, max_len, window, H, Hk, D)
            assert f(dt, 2, 0, max_len, window, H, Hk, D) <= f(dt, 2, 1, max_len, window, H, Hk, D)
    assert f(dt, 2, -1, 99, window, H, Hk, D) == 0


@pytest.mark.parametrize("D,dt", [(64, L.DT_BF16), (256, L.DT_F32)])
@pytest.mark.parametrize("batch,H,Hk,rows,max_len", [
    (1, 1, 1, 4096, (1 << 26) - 1), (1, 1, 1, 1 << 23, (1 << 26) - 1), (2250, 8, 8, 3700, 3713), (2304, 8, 8, 3600, 3640),
    (32768, 8, 8, 255, 255), (32768, 8, 8, 255, 1), (1 << 12, 64, 64, 255, 255), (8, 8, 8, 1 << 20, (1 << 20) - 1),
    (65535, 4, 4, 255, 255), (1, 64, 64, 1 << 17, (1 << 20) - 1), (1, 64, 1, 1 << 17, (1 << 26) - 1), (1023, 256, 256, 255, 255)])
@pytest.mark.parametrize("window", [0, 1000])
def test_what_is_always_taken(batch, H, Hk, rows, max_len, D, dt, window):
    """batch * n_kv_head <= 2^18, batch * n_head * max_rows and batch * n_kv_head * max_len
    < 2^26, max_rows * n_head <= 2^23: taken, as far as its workspace, which the size covers."""
    rows = min(rows, ((1 << 26) - 1) // (batch * H))
    assert batch * Hk <= 1 << 18 and batch * Hk * max_len < 1 << 26 and rows * H <= 1 << 23
    size = L.lib().ullm_hip_key_weights_workspace_bytes(dt, batch, rows, max_len, window, H, Hk, D)
    for page in (0, 1 << 16):
        for qdt in {dt, L.DT_F32}:
            rc, need = needs(dt, qdt, rows, max_len, window, batch, H, Hk, D, page)
            assert rc == L.E_WORKSPACE and need <= size
