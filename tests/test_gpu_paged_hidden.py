"""Attention over pages (include/wzy_paged.h): a value that is not finite in a cell that a row does not see, in tiles whose waves hold
one token each and in single tokens' blocks."""
import ctypes as C
import time

import numpy as np
import pytest

import wzy_amd
from mx_ref import BF16, F16, HALF_STEP, typed, values
from test_gpu_paged import NAN, Batch, Cache, ref
from test_gpu_paged_steps import INF, attend_rows

pytestmark = pytest.mark.gpu
DA = wzy_amd.DeviceArray


def hidden_values(wz, t, qh, kvh, hd, cached, new, window, page=16, scale=0.1):
    """infinities and NaN at the ends of what the first and the last token of each request see, and one cell past them"""
    rng = np.random.default_rng(qh + hd + new[0])
    total = [c + n for c, n in zip(cached, new)]
    b = Batch(page, cached, new, max(-(-n // page) for n in total), sum(-(-n // page) for n in total) + 2, None, max_new=max(new))
    w = b.work(wz, qh, kvh, hd, window)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    table, q_start = b.check()[:2]
    cache, kv = Cache(t, b.n_pages, page, kvh, hd), []
    for r, n in enumerate(total):
        kb, vb = (typed(rng.standard_normal((n, kvh, hd)), t)[0] for _ in range(2))
        put = [(n - 1, 3, INF[t])] + ([(n - 2, 40, NAN[t])] if new[r] > 1 else [])
        if window and n > window:
            put += [(n - 1 - window, 7, NAN[t]), (n - window, 9, INF[t] | 0x8000)]
            put += [(cached[r] + 1 - window, 63, INF[t])] if cached[r] + 1 > window else []
        for cell, column, bits in put:
            vb[cell, kvh - 1, column] = bits
        cell = np.arange(n)
        cache.put(table[r, cell // page] * page + cell % page, kb, vb)
        kv.append((values(kb, t), values(vb, t)))
    cache.upload()
    qb, q = typed(rng.standard_normal((b.max_tokens, qh, hd)), t)
    qd, out = DA.from_numpy(qb), DA((b.max_tokens, qh, hd), np.uint16)
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * hd, hd)
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), scale, ws.ptr, nb, None)
    got = values(out.numpy(), t)
    for r in range(b.R):
        k, v = kv[r]
        qr, y = q[q_start[r]:q_start[r + 1]], got[q_start[r]:q_start[r + 1]]
        want = attend_rows(qr, k, v, cached[r], window, scale)
        ok = np.isfinite(want)
        np.testing.assert_array_equal(np.isfinite(y), ok)
        np.testing.assert_array_equal(y[~ok], want[~ok])
        size = np.abs(v[np.isfinite(v)]).max()
        top = scale * np.abs(qr).sum(-1).max() * np.abs(k).max()
        # weights and outputs rounded by half a step each; scores by up to hd steps of 2^-24 of their terms, twice; sums
        bound = HALF_STEP[t] * (np.abs(want[ok]) + size) * 1.01 + size * (2 * hd * 2.0 ** -24 * top + 2.0 ** -14)
        assert (np.abs(y[ok] - want[ok]) <= bound).all()


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("qh,kvh,hd,cached,new,window", [
    (32, 1, 64, [40], [2], 0), (32, 1, 256, [40], [2], 0), (32, 1, 128, [100], [2], 33), (31, 1, 64, [30, 9], [2, 1], 0),      # 64 rows
    (48, 1, 64, [40], [3], 0), (64, 1, 128, [40], [4], 0), (71, 1, 256, [10], [20], 0), (256, 1, 64, [60], [5], 0),            # 128 rows
    (24, 2, 64, [100, 0], [3, 60], 64), (24, 2, 256, [300, 5], [19, 60], 64), (128, 2, 128, [90], [6], 31)])
def test_waves_of_one_token_in_tiles_of_several(wz, gpu, t, qh, kvh, hd, cached, new, window):
    hidden_values(wz, t, qh, kvh, hd, cached, new, window)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("qh,kvh,hd", [(4, 2, 64), (24, 2, 256), (40, 1, 128), (200, 1, 64)])
@pytest.mark.parametrize("window", [0, 1, 37])
def test_single_token_that_sees_an_infinity(wz, gpu, t, qh, kvh, hd, window):
    # blocks that the token's cells do not fill repeat its last or first cell, with weights of 0
    hidden_values(wz, t, qh, kvh, hd, [40, 0, 63, 700], [1, 1, 1, 1], window)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("qh,kvh,hd,cached,new,window", [
    (4, 1, 64, [9000, 3], [40, 90], 0), (12, 1, 128, [5000], [50], 0), (2, 2, 256, [6000, 2], [100, 1], 2500),     # tiles cut into parts
    (6, 2, 256, [4000, 70], [5, 4], 1000), (8, 2, 64, [3000, 5], [3, 9], 0), (4, 2, 128, [31, 200], [70, 33], 20), (1, 1, 64, [0], [300], 5)])
def test_many_values_that_are_not_finite(wz, gpu, t, qh, kvh, hd, cached, new, window):
    """infinities of both signs and NaN all over the last blocks and where windows begin: each row has those that it sees"""
    rng = np.random.default_rng(hd + qh)
    total, page, scale = [c + n for c, n in zip(cached, new)], 32, 0.1
    b = Batch(page, cached, new, max(-(-n // page) for n in total), sum(-(-n // page) for n in total) + 2, None, max_new=max(new))
    w = b.work(wz, qh, kvh, hd, window)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    table, q_start = b.check()[:2]
    cache, kv = Cache(t, b.n_pages, page, kvh, hd), []
    for r, n in enumerate(total):
        kb, vb = (typed(rng.standard_normal((n, kvh, hd)), t)[0] for _ in range(2))
        for at in [cached[r]] + ([max(0, cached[r] + 1 - window)] if window else []):
            for _ in range(2 * new[r]):
                cell = int(rng.integers(max(at - 40, 0), min(at + new[r] + 10, n)))
                vb[cell, rng.integers(kvh), rng.integers(hd)] = rng.choice([INF[t], INF[t] | 0x8000, NAN[t]])
        cell = np.arange(n)
        cache.put(table[r, cell // page] * page + cell % page, kb, vb)
        kv.append((values(kb, t), values(vb, t)))
    cache.upload()
    qb, q = typed(rng.standard_normal((b.max_tokens, qh, hd)), t)
    qd, out = DA.from_numpy(qb), DA((b.max_tokens, qh, hd), np.uint16)
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * hd, hd)
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), scale, ws.ptr, nb, None)
    got = values(out.numpy(), t)
    for r in range(b.R):
        k, v = kv[r]
        qr, y = q[q_start[r]:q_start[r + 1]], got[q_start[r]:q_start[r + 1]]
        want = attend_rows(qr, k, v, cached[r], window, scale)
        ok = np.isfinite(want)
        assert ok.any() and not ok.all()
        np.testing.assert_array_equal(y[~ok], want[~ok])
        size = np.abs(v[np.isfinite(v)]).max()
        top = scale * np.abs(qr).sum(-1).max() * np.abs(k).max()
        bound = HALF_STEP[t] * (np.abs(want[ok]) + size) * 1.01 + size * (2 * hd * 2.0 ** -24 * top + 2.0 ** -13)
        assert (np.abs(y[ok] - want[ok]) <= bound).all()


def test_a_value_that_is_not_finite_does_not_hold_up_a_step(wz, gpu):
    # a chunk behind 20,000 cells; row by row over its parts it would take a hundred times as long
    rng = np.random.default_rng(3)
    cached, new, qh, hd, page = 20000, 512, 8, 128, 64
    n = cached + new
    b = Batch(page, [cached], [new], -(-n // page), -(-n // page) + 2, None, max_new=new)
    w = b.work(wz, qh, 1, hd)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    table = b.check()[0]
    cache = Cache(BF16, b.n_pages, page, 1, hd)
    kb, vb = (typed(rng.standard_normal((n, 1, hd)), BF16)[0] for _ in range(2))
    cell = np.arange(n)
    qd, out = DA.from_numpy(typed(rng.standard_normal((new, qh, hd)), BF16)[0]), DA((new, qh, hd), np.uint16)
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * hd, hd)

    def seconds():
        cache.put(table[0, cell // page] * page + cell % page, kb, vb)
        cache.upload()
        best = 1e9
        for _ in range(5):
            wz.wzy_device_sync()
            start = time.perf_counter()
            wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.1, ws.ptr, nb, None)
            wz.wzy_device_sync()
            best = min(best, time.perf_counter() - start)
        return best
    finite = seconds()
    vb[cached + 100, 0, 9] = INF[BF16]
    assert seconds() < 5 * finite
    y = values(out.numpy(), BF16)
    assert np.isfinite(y[:100]).all() and not np.isfinite(y[100:, :, 9]).any() and np.isfinite(np.delete(y, 9, 2)).all()
