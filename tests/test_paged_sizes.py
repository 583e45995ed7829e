"""Operators for several requests at once: sizes that no launch takes are refused, on the host (include/wzy_paged.h)."""
import ctypes as C

import pytest

from test_paged import PTR, batch, cache, heads, pool, refused, work


@pytest.mark.parametrize("qh,kvh", [(4096, 64), (16384, 64), (2048, 8), (2048, 64)])
def test_steps_of_too_many_rows(wz, qh, kvh):
    b, w = batch(max_tokens=1 << 20), work(wz, qh=qh, kvh=kvh)
    assert wz.wzy_paged_work_bytes(C.byref(b), C.byref(w)) == 0
    assert "wzy_paged_work_bytes" in wz.wzy_last_error().decode()
    assert wz.wzy_paged_attend_workspace_bytes(C.byref(b), C.byref(w)) == 0
    refused(wz, "wzy_paged_plan", pool(), b, w, 1, None)
    refused(wz, "wzy_paged_attend", cache(kvh=kvh, ld_cell=kvh * 128), b, w, heads(), heads(2 * PTR), 0.1, PTR, 1 << 50, None)


@pytest.mark.parametrize("max_tokens,max_new,n_req,qh,kvh", [((1 << 20) - 64 - 512, 0, 1, 2048, 8), ((1 << 17) - 4096 - 8, 0, 4096, 16384, 64),
                                                             (1 << 20, 1, 4096, 64, 64), (1 << 20, 0, 4096, 256, 1)])
def test_steps_of_as_many_rows_as_a_launch_takes(wz, max_tokens, max_new, n_req, qh, kvh):
    b, w = batch(max_tokens=max_tokens, max_new=max_new, n_req=n_req), work(wz, qh=qh, kvh=kvh)
    assert max_tokens * qh + 128 * n_req * kvh <= 2 ** 31 - 2 ** 17 or max_new == 1
    assert wz.wzy_paged_work_bytes(C.byref(b), C.byref(w)) > 0
    assert wz.wzy_paged_attend_workspace_bytes(C.byref(b), C.byref(w)) > 0
