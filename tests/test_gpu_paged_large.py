"""Work lists of large steps (include/wzy_paged.h): thousands of requests, thousands of rows, several lists, against 64 bits."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
import wzy_amd
from mx_ref import BF16, F16, HALF_STEP, typed, values
from test_gpu_paged import Batch, Cache, attend_case, ref

pytestmark = pytest.mark.gpu
DA = wzy_amd.DeviceArray


def mixed(requests, seed, most):
    """cached and new cells of a step: single tokens, windows of a few rows, requests without rows, some chunks of `most`"""
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, 120, requests)
    new = rng.choice([0, 1, 1, 1, 2, 4], requests)
    at = rng.choice(requests, 8, replace=False)
    new[at[:4]] = rng.integers(most // 2, most, 4)
    cached[at[4:]] = rng.integers(700, 2500, 4)
    return cached, new


@pytest.mark.parametrize("requests", [257, 1024, 1025, 2500, 4096])
@pytest.mark.parametrize("rows", [0, 9000])
def test_attend_many_requests(wz, gpu, requests, rows):
    # rows 0: at most 4,096 of them where the requests allow it, one launch; 9,000: lists filled by workgroups of their own
    cached, new = mixed(requests, requests, 150)
    if not rows:
        while new.sum() > 4096:
            new[np.flatnonzero(new > 1)[:: 2]] = 1
            new[np.flatnonzero(new == 1)[:: 9]] = 0
    attend_case(wz, BF16, cached.tolist(), new.tolist(), 2, 1, 64, 16, seed=requests, max_tokens=rows or None)


@pytest.mark.parametrize("t,qh,kvh,hd,window", [(BF16, 4, 2, 64, 0), (F16, 12, 1, 128, 0), (F16, 2, 2, 256, 700), (BF16, 3, 1, 64, 40)])
def test_attend_prompts_past_one_launch_of_rows(wz, gpu, t, qh, kvh, hd, window):
    # prompts, a chunk behind a long cache, which is cut into parts, verify windows, single tokens, padding
    cached = [0, 9, 6000, 17, 3000, 0, 40]
    new = [2300, 1, 40, 4, 1, 1900, 0]
    attend_case(wz, t, cached, new, qh, kvh, hd, 64, window=window, seed=hd, max_tokens=4500)


def test_attend_refused_requests_in_large_steps(wz, gpu):
    # no free page: requests that need one are refused, many with rows of their own, and become zero
    rng = np.random.default_rng(7)
    cached, new = rng.integers(0, 100, 1300), rng.choice([0, 1, 2, 40], 1300)
    attend_case(wz, F16, cached.tolist(), new.tolist(), 2, 2, 64, 32, seed=3, free=60)


@pytest.mark.parametrize("requests,max_tokens", [(1200, 4096), (1200, 8000), (6, 8000)])
def test_several_lists_of_a_large_plan(wz, gpu, requests, max_tokens):
    """layers with and without a window, and with other heads, from one plan"""
    cached, new = mixed(requests, 5, 200) if requests > 8 else (np.array([0, 50, 4000, 7, 0, 3]), np.array([2500, 1, 30, 4, 1800, 1]))
    rng = np.random.default_rng(requests)
    total = cached + new
    pages = -(-total // 16)
    b = Batch(16, cached, new, int(pages.max()), int(pages.sum()) + 2, None, max_tokens=max_tokens, max_new=int(new.max()))
    kinds = [(2, 1, 64, 0), (2, 1, 64, 33), (6, 2, 128, 0)]
    works, items = (wzy_amd.PagedWork * 3)(), []
    for i, kind in enumerate(kinds):
        works[i] = b.work(wz, *kind)
        items.append(b.items)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), works, 3, None)
    table, q_start, kv_len, served = b.check()
    assert served.all()
    for w, (qh, kvh, hd, window) in zip(works, kinds):
        cache, kv = Cache(F16, b.n_pages, 16, kvh, hd), []
        for r in range(b.R):
            (kb, k), (vb, v) = (typed(rng.standard_normal((kv_len[r], kvh, hd)), F16) for _ in range(2))
            cell = np.arange(kv_len[r])
            cache.put(table[r, cell // 16] * 16 + cell % 16, kb, vb)
            kv.append((k, v))
        cache.upload()
        qb, q = typed(rng.standard_normal((max_tokens, qh, hd)), F16)
        qd, out = DA.from_numpy(qb), DA((max_tokens, qh, hd), np.uint16)
        n = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
        ws = DA(n, np.uint8)
        qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * hd, hd)
        wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.1, ws.ptr, n, None)
        got = values(out.numpy(), F16)
        for r in range(b.R):
            if new[r] == 0:
                continue
            rows = slice(q_start[r], q_start[r + 1])
            want, size, top = R.attend(q[rows], *kv[r], int(cached[r]), window, 0.1)
            # weights and outputs half a step each, scores hd steps of 2^-24 of their terms twice, sums; fp16 weights end at 2^-31
            tol = HALF_STEP[F16] * (np.abs(want) + size) * 1.01 + size * (2 * hd * 2.0 ** -24 * top + 2.0 ** -14) + 2.0 ** -28 * kv_len[r]
            assert (np.abs(got[rows] - want) <= tol).all(), r
