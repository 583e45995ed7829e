"""Operators for several requests at once (include/wzy_paged.h) on the GPU against plain 64-bit formulations
(tests/paged_ref.py)."""
import ctypes as C
import math

import numpy as np
import pytest

import paged_ref as R
import wzy_amd
from mx_ref import BF16, F16, F32, HALF_STEP, typed, values

pytestmark = pytest.mark.gpu
DA = wzy_amd.DeviceArray
FILL = 0xA5
NAN = {BF16: 0x7FC1, F16: 0x7E01, F32: 0x7FC00001}


def ref(x):
    return C.byref(x)


def ints(a):
    return DA.from_numpy(np.asarray(a, np.int32))


def filled(shape, dtype):
    a = np.zeros(shape, dtype)
    a.view(np.uint8)[:] = FILL
    return a


class Batch:
    """A step's arrays on the device, with what stands behind them watched"""

    def __init__(self, page, n_cached, n_new, max_pages, n_pages, free, max_tokens=None, max_new=0, seed=0):
        rng = np.random.default_rng(seed)
        self.page, self.n_pages = page, n_pages
        self.n_cached, self.n_new = np.asarray(n_cached, np.int32), np.asarray(n_new, np.int32)
        self.R, self.max_pages = len(n_cached), max_pages
        self.max_tokens = max(1, int(self.n_new.clip(0).sum())) if max_tokens is None else max_tokens
        self.max_new = max_new
        self.table = np.full((self.R, max_pages), -7, np.int32)
        ids = rng.permutation(n_pages)
        at = 0
        for r in range(self.R):
            held = min(-(-max(int(self.n_cached[r]), 0) // page), max_pages)
            self.table[r, :held] = ids[at:at + held]
            at += held
        self.free = np.full(n_pages, -9, np.int32)
        self.n_free = min(free, n_pages - at) if free is not None else n_pages - at
        self.free[:self.n_free] = ids[at:at + self.n_free]
        self.d = dict(cached=ints(self.n_cached), new=ints(self.n_new), table=ints(self.table), free=ints(self.free),
                      n_free=ints([self.n_free, 77]), left=ints([55, 77]))
        for name, n in (("q_start", self.R + 1), ("kv_len", self.R), ("served", self.R), ("positions", self.max_tokens),
                        ("slots", self.max_tokens)):
            self.d[name] = DA.from_numpy(filled(n + 3, np.int32))
        d = self.d
        self.c = wzy_amd.PagedBatch(self.R, self.max_tokens, max_pages, d["cached"].ptr, d["new"].ptr, d["table"].ptr, d["q_start"].ptr,
                                    d["kv_len"].ptr, d["served"].ptr, d["positions"].ptr, d["slots"].ptr, max_new)
        self.pool = wzy_amd.PagedPool(d["free"].ptr, d["n_free"].ptr, d["left"].ptr, n_pages, page)

    def work(self, wz, qh, kvh, hd, window=0):
        w = wzy_amd.PagedWork(qh, kvh, hd, window, None, 0)
        w.bytes = wz.wzy_paged_work_bytes(ref(self.c), ref(w))
        self.items = DA.from_numpy(filled(w.bytes + 64, np.uint8))
        w.items = self.items.ptr
        return w

    def read(self, name, n):
        a = self.d[name].numpy()
        assert (a[n:].view(np.uint8) == FILL).all(), name
        return a[:n]

    def check(self):
        """every output against the plain form"""
        table, q_start, kv_len, served, positions, slots, left = R.plan(
            self.page, self.n_pages, self.n_free, self.free, self.n_cached, self.n_new, self.table, self.max_tokens,
            self.max_new or self.max_tokens)
        np.testing.assert_array_equal(self.d["table"].numpy().reshape(self.R, -1), table)
        np.testing.assert_array_equal(self.read("q_start", self.R + 1), q_start)
        np.testing.assert_array_equal(self.read("kv_len", self.R), kv_len)
        np.testing.assert_array_equal(self.read("served", self.R), served)
        np.testing.assert_array_equal(self.read("positions", self.max_tokens), positions)
        np.testing.assert_array_equal(self.read("slots", self.max_tokens), slots)
        np.testing.assert_array_equal(self.d["left"].numpy(), [left, 77])
        return table, q_start, kv_len, served


# ---- pages, tables, slots --------------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("requests", [1, 2, 67, 1025, 4096])
def test_plan(wz, gpu, page, requests):
    rng = np.random.default_rng(requests + page)
    cached = rng.integers(0, 5 * page, requests) * (rng.random(requests) < 0.9)
    new = rng.choice([0, 1, 1, 1, 3, page, 2 * page + 5], requests)
    cached[0], new[-1] = page, 1                                          # a full last page
    b = Batch(page, cached, new, 9, int(requests * 12 + 9), None, seed=requests)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), None, 0, None)
    assert b.check()[3].all()


def test_plan_long_prompts_and_tail(wz, gpu):
    # many rows (their own launch), padded; a prompt of thousands of rows beside single tokens
    b = Batch(32, [0, 100, 31, 0, 7], [9000, 1, 1, 0, 777], 300, 400, None, max_tokens=12345)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), None, 0, None)
    assert b.check()[3].all()


@pytest.mark.parametrize("max_tokens", [40, 5000])
def test_plan_refuses_requests(wz, gpu, max_tokens):
    # pool of 5: the third needs more than is left, the fourth needs none, the fifth would fit but comes after
    b = Batch(16, [0, 16, 5, 3, 0, 0, 90, 0], [17, 1, 30, 2, 1, 0, 20, 3], 6, 64, 4, max_tokens=max_tokens, max_new=30)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), None, 0, None)
    assert b.check()[3].tolist() == ([1, 1, 0, 0, 0, 1, 0, 0] if max_tokens == 40 else [1, 1, 0, 1, 0, 1, 0, 0])
    # too many for max_new, for the table, negative lengths, rows past the end
    b = Batch(16, [-5, 4, 80, 2 ** 31 - 1, 1], [3, 9, 17, 2 ** 31 - 1, -4], 6, 64, None, max_tokens=50, max_new=8)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), None, 0, None)
    assert b.check()[3].tolist() == [1, 0, 0, 0, 1]


@pytest.mark.parametrize("rows", [3, 4200])
def test_plan_gives_no_slot_in_bad_pages(wz, gpu, rows):
    # a held page that is none of the cache's, and bad ids in the pool: slots -1, nothing else
    b = Batch(16, [5, 20, 3], [1, rows - 2, 1], 300, 400, None)
    b.table[0, 0] = -1
    b.free[b.n_free - 1] = 400
    b.d["table"], b.d["free"] = ints(b.table), ints(b.free)
    b.c.table, b.pool.free_pages = b.d["table"].ptr, b.d["free"].ptr
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), None, 0, None)
    want = R.plan(16, 400, b.n_free, b.free, b.n_cached, b.n_new, b.table, b.max_tokens, b.max_tokens)
    table, slots = want[0], want[5]
    np.testing.assert_array_equal(b.d["table"].numpy().reshape(3, -1), table)
    slots = np.where((slots < 0) | (slots >= 6400), -1, slots)
    assert slots[0] == -1 and (rows == 3 or (slots == -1).sum() == 17)
    np.testing.assert_array_equal(b.read("slots", rows), slots)


def test_plan_in_place_then_release(wz, gpu):
    b = Batch(16, [20, 0, 33, 1], [13, 1, 15, 0], 4, 20, None)
    b.pool.n_free_out = b.pool.n_free
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), None, 0, None)
    want = R.plan(16, 20, b.n_free, b.free, b.n_cached, b.n_new, b.table, b.max_tokens, b.max_tokens)
    assert b.d["n_free"].numpy()[0] == want[-1]
    table = want[0]
    cells = ints(want[2])
    b.c.n_cached = cells.ptr
    ended = ints([0, 1, 1, 0])
    wz.wzy_paged_release(ref(b.pool), ref(b.c), ended.ptr, None)
    back = [table[1, 0]] + table[2, :3].tolist()
    assert b.d["n_free"].numpy().tolist() == [want[-1] + 4, 77]
    np.testing.assert_array_equal(b.d["free"].numpy()[want[-1]:want[-1] + 4], back)
    table[1, 0] = table[2, :3] = -1
    np.testing.assert_array_equal(b.d["table"].numpy().reshape(4, 4), table)


def test_release_leaves_bad_entries_out_and_ends_at_a_full_pool(wz, gpu):
    n = 3000
    b = Batch(16, [16 * 2] * n, [0] * n, 2, 2 * n, None)
    table = b.table.copy()
    table[5, 1], table[9, 0] = -1, 2 * n
    b.d["table"] = ints(table)
    b.c.table = b.d["table"].ptr
    b.d["n_free"] = ints([10])
    b.pool.n_free = b.d["n_free"].ptr
    ended = np.ones(n, np.int32)
    ended[7] = 0
    e = ints(ended)
    wz.wzy_paged_release(ref(b.pool), ref(b.c), e.ptr, None)
    back = [i for r in range(n) if ended[r] for i in table[r] if 0 <= i < 2 * n]
    assert len(back) == 2 * n - 4
    assert b.d["left"].numpy()[0] == 2 * n
    np.testing.assert_array_equal(b.d["free"].numpy()[10:], back[:2 * n - 10])
    left = b.d["table"].numpy().reshape(n, 2)
    assert (np.delete(left, 7, 0) == -1).all() and (left[7] == table[7]).all()


# ---- rotary positions ------------------------------------------------------------------------------------
def freqs(wz, n_rot, scaling=0, theta=1e4, factor=1.0, low=1.0, high=32.0, ctx=4096, amplitude=1.0):
    d = DA(n_rot // 2 + 2, np.float64, zero=True)
    cfg = wzy_amd.RopeCfg(theta, factor, low, high, amplitude, ctx, n_rot, scaling)
    wz.wzy_rope_freqs(ref(cfg), d.ptr, None)
    return d


@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
@pytest.mark.parametrize("n_rot,theta,ctx,low,high", [(64, 1e7, 32768, 1.0, 32.0), (2, 1e4, 4096, 1.0, 4.0), (512, 5e5, 8192, 1.0, 4.0),
                                                      (34, 1.5, 7, 0.5, 100.0)])
def test_rope_freqs(wz, gpu, scaling, n_rot, theta, ctx, low, high):
    d = freqs(wz, n_rot, scaling, theta, 8.0, low, high, ctx, 1.25 if scaling else 0.0).numpy()
    want = R.frequencies(n_rot, theta, scaling, 8.0, low, high, ctx) / (2 * math.pi)
    # a power, a logarithm, a division: a few steps of 2^-53, more where the ramp's slope is steep
    np.testing.assert_allclose(d[:-2], want, rtol=1e-12, atol=0)
    assert d[-2] == (1.25 if scaling else 1.0) and d[-1] == 0.0


def rope_bound(x, want, t):
    """the turned pair's two products and sum in fp32 (coefficients rounded too): at most 2^-24 * 4 of the pair's length; then
    one rounding to the type"""
    return HALF_STEP[t] * np.abs(want) + 2.0 ** -22 * np.abs(x).max(-1, keepdims=True) * 2 + 2.0 ** -25


@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,heads,hd,n_rot,gap", [(1, 24, 256, 64, 0), (5, 3, 64, 64, 8), (700, 2, 128, 32, 0), (33, 1, 40, 24, 0),
                                                     (7, 5, 17, 6, 3), (129, 4, 512, 512, 0), (2, 1, 2, 2, 1)])
def test_rope(wz, gpu, pairs, t, rows, heads, hd, n_rot, gap):
    rng = np.random.default_rng(rows + hd)
    bits, x = typed(rng.standard_normal((rows, heads, hd)), t)
    wide = filled((rows, heads, hd + gap), bits.dtype)
    wide[:, :, :hd] = bits
    pos = rng.integers(0, 2 ** 20, rows).astype(np.int32)
    pos[0] = rng.choice([0, 2 ** 31 - 1, -5])
    f = freqs(wz, n_rot, 0, 1e4, amplitude=1.5)
    tab = wzy_amd.RopeTab(f.ptr, n_rot, pairs)
    xd, yd, pd = DA.from_numpy(wide), DA.from_numpy(filled(wide.shape, bits.dtype)), ints(pos)
    xs = wzy_amd.Heads(xd.ptr, heads * (hd + gap), hd + gap)
    ys = wzy_amd.Heads(yd.ptr, heads * (hd + gap), hd + gap)
    wz.wzy_rope(ref(tab), ref(xs), t, rows, heads, hd, pd.ptr, ref(ys), None)
    got = yd.numpy()
    assert (np.ascontiguousarray(got[:, :, hd:]).view(np.uint8) == FILL).all()
    want = R.rope(x, R.frequencies(n_rot, 1e4), n_rot, pairs, pos, 1.5)
    y = values(np.ascontiguousarray(got[:, :, :hd]), t)
    assert (np.abs(y - want) <= rope_bound(x, want, t)).all()
    np.testing.assert_array_equal(y[..., n_rot:], x[..., n_rot:])
    wz.wzy_rope(ref(tab), ref(xs), t, rows, heads, hd, pd.ptr, ref(xs), None)          # in place: the same bits
    np.testing.assert_array_equal(xd.numpy(), got)


@pytest.mark.parametrize("pairs", [0, 1])
@pytest.mark.parametrize("t,rows", [(F32, 2100), (BF16, 4201), (F16, 4201)])
def test_rope_large_call_equals_small_ones(wz, gpu, t, rows, pairs):
    # more than 32 MB of output: the same bits as calls of 1,000 rows, in place too
    rng = np.random.default_rng(rows)
    heads, hd, n_rot = 32, 128, 96
    bits = typed(rng.standard_normal((rows, heads, hd)), t)[0]
    size, pd = bits.itemsize, ints(rng.integers(0, 2 ** 20, rows))
    f = freqs(wz, n_rot)
    tab = wzy_amd.RopeTab(f.ptr, n_rot, pairs)
    xd, one, many = DA.from_numpy(bits), DA.from_numpy(filled(bits.shape, bits.dtype)), DA.from_numpy(filled(bits.shape, bits.dtype))

    def rows_of(d, r):
        return wzy_amd.Heads(d.ptr + r * heads * hd * size, heads * hd, hd)
    assert rows * heads * hd * size > 32 << 20
    for r in range(0, rows, 1000):
        wz.wzy_rope(ref(tab), ref(rows_of(xd, r)), t, min(1000, rows - r), heads, hd, pd.ptr + 4 * r, ref(rows_of(many, r)), None)
    wz.wzy_rope(ref(tab), ref(rows_of(xd, 0)), t, rows, heads, hd, pd.ptr, ref(rows_of(one, 0)), None)
    wz.wzy_rope(ref(tab), ref(rows_of(xd, 0)), t, rows, heads, hd, pd.ptr, ref(rows_of(xd, 0)), None)
    np.testing.assert_array_equal(one.numpy(), many.numpy())
    np.testing.assert_array_equal(xd.numpy(), many.numpy())


class Cache:
    """K and V of [page][cell][head] or [page][head][cell], gaps between, all NaN to begin with"""

    def __init__(self, t, n_pages, page, kvh, hd, by_head=False, gap=0):
        self.t, self.shape, self.by_head, self.hd = t, (n_pages, page, kvh), by_head, hd
        inner = hd + gap
        dims = (n_pages, kvh, page, inner) if by_head else (n_pages, page, kvh, inner)
        self.k, self.v = (np.full(dims, NAN[t], np.uint16) for _ in range(2))
        self.ld = (dims[1] * dims[2] * inner, inner if by_head else kvh * inner, page * inner if by_head else inner)
        self.page, self.kvh = page, kvh

    def rows(self, a):
        """[n_pages * page, kvh, hd] view"""
        a = a.transpose(0, 2, 1, 3) if self.by_head else a
        return a[..., :self.hd]

    def put(self, slots, k, v):
        for a, x in ((self.k, k), (self.v, v)):
            self.rows(a)[slots // self.page, slots % self.page] = x

    def upload(self):
        self.dk, self.dv = DA.from_numpy(self.k), DA.from_numpy(self.v)
        self.c = wzy_amd.PagedCache(self.dk.ptr, self.dv.ptr, *self.ld, self.shape[0], self.page, self.kvh, self.hd, self.t)
        return self


@pytest.mark.parametrize("ct", [BF16, F16])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,qh,kvh,hd,n_rot,pairs,by_head", [(1, 24, 2, 256, 64, 0, False), (37, 6, 3, 64, 64, 1, True),
                                                                (300, 0, 1, 128, 96, 0, False), (9, 8, 8, 128, 22, 0, True),
                                                                (1500, 2, 2, 64, 0, 0, False)])
def test_append(wz, gpu, ct, t, rows, qh, kvh, hd, n_rot, pairs, by_head):
    rng = np.random.default_rng(rows + qh)
    page, n_pages = 16, rows // 16 + 5
    bits, x = typed(rng.standard_normal((rows, qh + 2 * kvh, hd)), t)
    pos = rng.integers(0, 300000, rows).astype(np.int32)
    slots = rng.permutation(n_pages * page)[:rows].astype(np.int32)
    drop = rng.random(rows) < (0.2 if rows > 1 else 0)
    bad = np.where(drop, rng.choice([-1, -2 ** 31, n_pages * page, 2 ** 31 - 1], rows), slots).astype(np.int32)
    c = Cache(ct, n_pages, page, kvh, hd, by_head, gap=8).upload()
    xd, pd, sd = DA.from_numpy(bits), ints(pos), ints(bad)
    ld = (qh + 2 * kvh) * hd
    size = bits.itemsize
    q, k, v = (wzy_amd.Heads(xd.ptr + at * hd * size, ld, hd) for at in (0, qh, qh + kvh))
    qo = DA.from_numpy(filled((rows, max(qh, 1), hd), np.uint16))
    qs = wzy_amd.Heads(qo.ptr, max(qh, 1) * hd, hd)
    f = freqs(wz, n_rot, 0, 1e6) if n_rot else None
    tab = wzy_amd.RopeTab(f.ptr, n_rot, pairs) if n_rot else None
    wz.wzy_paged_append(ref(c.c), ref(tab) if n_rot else None, ref(q) if qh else None, qh, ref(qs) if qh else None, ref(k), ref(v),
                        t, rows, pd.ptr, sd.ptr, None)
    turned = R.rope(x, R.frequencies(n_rot, 1e6), n_rot, pairs, pos) if n_rot else x
    bound = rope_bound(x, turned, ct) if n_rot else HALF_STEP[ct] * np.abs(x) + 2.0 ** -25
    if qh:
        y = values(qo.numpy(), ct)
        assert (np.abs(y - turned[:, :qh]) <= bound[:, :qh]).all()
    else:
        assert (qo.numpy().view(np.uint8) == FILL).all()
    at = slots[~drop]
    gk, gv = c.dk.numpy(), c.dv.numpy()
    k2 = values(np.ascontiguousarray(c.rows(gk)[at // page, at % page]), ct)
    v2 = values(np.ascontiguousarray(c.rows(gv)[at // page, at % page]), ct)
    assert (np.abs(k2 - turned[~drop, qh:qh + kvh]) <= bound[~drop, qh:qh + kvh]).all()
    want = values(typed(x[:, qh + kvh:], ct)[0], ct) if t == F32 else x[:, qh + kvh:]
    assert (np.abs(v2 - want[~drop]) <= HALF_STEP[ct] * np.abs(want[~drop]) + 2.0 ** -25).all()
    for g in (gk, gv):                                                    # nothing else is touched
        c.rows(g)[at // page, at % page] = NAN[ct]
        assert (g == NAN[ct]).all()


@pytest.mark.parametrize("t,ct", [(F32, BF16), (BF16, BF16), (F16, F16)])
def test_append_large_call_equals_small_ones(wz, gpu, t, ct):
    rng = np.random.default_rng(t)
    rows, qh, kvh, hd, n_rot, page = 3001, 24, 2, 256, 64, 64
    n_pages, ld = 50, (qh + 2 * kvh) * hd
    bits = typed(rng.standard_normal((rows, qh + 2 * kvh, hd)), t)[0]
    size, xd, pd = bits.itemsize, DA.from_numpy(bits), ints(rng.integers(0, 300000, rows))
    sd = ints(rng.permutation(n_pages * page)[:rows])
    f = freqs(wz, n_rot, 0, 1e6)
    tab = wzy_amd.RopeTab(f.ptr, n_rot, 0)
    assert rows * ld * 2 > 32 << 20
    got = []
    for step in (rows, 500):
        c, qo = Cache(ct, n_pages, page, kvh, hd).upload(), DA.from_numpy(filled((rows, qh, hd), np.uint16))
        for r in range(0, rows, step):
            q, k, v = (wzy_amd.Heads(xd.ptr + (r * ld + at * hd) * size, ld, hd) for at in (0, qh, qh + kvh))
            qs = wzy_amd.Heads(qo.ptr + 2 * r * qh * hd, qh * hd, hd)
            wz.wzy_paged_append(ref(c.c), ref(tab), ref(q), qh, ref(qs), ref(k), ref(v), t, min(step, rows - r), pd.ptr + 4 * r, sd.ptr + 4 * r, None)
        got.append((qo.numpy(), c.dk.numpy(), c.dv.numpy()))
    for x, y in zip(*got):
        np.testing.assert_array_equal(x, y)


# ---- attention -------------------------------------------------------------------------------------------
def attend_case(wz, t, cached, new, qh, kvh, hd, page, window=0, by_head=False, seed=0, spread=1.0, max_tokens=None, free=None,
                scale=None, max_new=None, special=None, space=FILL):
    """plan, append through numpy, attend; returns (got, want, bound) a request"""
    rng = np.random.default_rng(seed)
    n_pages = sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 3
    max_pages = max(-(-(c + n) // page) for c, n in zip(cached, new)) + 1
    b = Batch(page, cached, new, max_pages, n_pages, free, max_tokens=max_tokens, max_new=max(new) if max_new is None else max_new, seed=seed)
    w = b.work(wz, qh, kvh, hd, window)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    table, q_start, kv_len, served = b.check()
    assert (b.items.numpy()[w.bytes:] == FILL).all()
    cache = Cache(t, n_pages, page, kvh, hd, by_head, gap=8 if by_head else 0)
    kv = []
    for r in range(b.R):
        n = int(kv_len[r])
        k = rng.standard_normal((n, kvh, hd)) * np.exp(rng.standard_normal((n, 1, 1)) * 0.3)
        v = rng.standard_normal((n, kvh, hd)) + rng.standard_normal((kvh, hd)) * 0.5
        (kb, k), (vb, v) = typed(k, t), typed(v, t)
        if special:
            special(r, kb, vb)
            k, v = values(kb, t), values(vb, t)
        cell = np.arange(n)
        lo = max(0, int(b.n_cached[r]) + 1 - window) if window else 0      # cells that no token sees stay NaN
        cell = cell[lo:]
        cache.put(table[r, cell // page] * page + cell % page, kb[lo:], vb[lo:])
        kv.append((k, v))
    cache.upload()
    qb, q = typed(rng.standard_normal((b.max_tokens, qh, hd)) * spread, t)
    qd = DA.from_numpy(qb)
    out = DA.from_numpy(filled((b.max_tokens + 1, qh, hd + 8), np.uint16))
    scale = hd ** -0.5 if scale is None else scale
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = filled(nb + 64, np.uint8)
    ws[:nb] = space
    ws = DA.from_numpy(ws)
    qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * (hd + 8), hd + 8)
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), scale, ws.ptr, nb, None)
    got = out.numpy()
    assert (ws.numpy()[nb:] == FILL).all()
    assert (np.ascontiguousarray(got[:, :, hd:]).view(np.uint8) == FILL).all()
    assert (got[q_start[-1]:].view(np.uint8) == FILL).all()                # rows behind the last, as they were
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), scale, ws.ptr, nb, None)
    np.testing.assert_array_equal(out.numpy(), got)                        # and the same bits again
    res = []
    for r in range(b.R):
        y = values(np.ascontiguousarray(got[q_start[r]:q_start[r + 1], :, :hd]), t)
        if not served[r]:
            assert (y == 0).all()
            continue
        if q_start[r] == q_start[r + 1]:
            continue
        want, size, top = R.attend(q[q_start[r]:q_start[r + 1]], *kv[r], int(b.n_cached[r]), window, scale)
        h, n = HALF_STEP[t], kv_len[r]
        # weights and outputs are rounded by half a step each; scores by up to hd steps of 2^-24 of their terms, twice (a weight and
        # the sum); sums by n 2^-24; fp16 weights, of 2^6 and more at the largest, end at 2^-25 of a step
        bound = h * (np.abs(want) + size) * 1.01 + size * (2 * hd * 2.0 ** -24 * top + n * 2.0 ** -23 + 2.0 ** -20) + n * 2.0 ** -31 * 8
        res.append((y, want, bound))
        assert (np.abs(y - want) <= bound).all(), (r, np.abs(y - want).max(), (np.abs(y - want) / bound).max())
    return res


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_attend_single_tokens(wz, gpu, t, hd, page):
    # one token of each request: the first cell, block and page borders, long ones that are cut into parts
    cached = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 100, 257, 1000, 4097]
    attend_case(wz, t, cached, [1] * len(cached), 6, 2, hd, page, seed=hd)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("qh,kvh,hd", [(24, 2, 256), (1, 1, 64), (5, 5, 128), (32, 1, 64), (33, 1, 128), (14, 2, 64)])
def test_attend_groups(wz, gpu, t, qh, kvh, hd):
    # verify windows of 1 to 5 rows: narrow and wide tiles in one step
    attend_case(wz, t, [40, 0, 300, 7, 129], [1, 2, 5, 3, 4], qh, kvh, hd, 32, seed=qh, by_head=True)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("hd,page", [(64, 128), (128, 16), (256, 32)])
def test_attend_chunks(wz, gpu, t, hd, page):
    # prompts and chunks, whole tiles and ragged ones, beside single tokens and a request that has no row
    attend_case(wz, t, [0, 70, 513, 5, 9], [200, 64, 33, 1, 0], 4, 2, hd, page, seed=page, max_tokens=333)


@pytest.mark.parametrize("window", [1, 17, 32, 100, 5000])
@pytest.mark.parametrize("hd", [64, 256])
def test_attend_window(wz, gpu, window, hd):
    attend_case(wz, BF16, [0, 200, 1030, 3], [150, 1, 40, 1], 4, 2, hd, 16, window=window, seed=window)


@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 64, 65])
@pytest.mark.parametrize("qh,kvh,max_new", [(1, 1, 1), (3, 3, 40), (2, 1, 20)])
def test_attend_short_window(wz, gpu, window, qh, kvh, max_new):
    # windows of a block or two, of requests long enough for parts; what parts do not write would be a NaN in the workspace
    cached = [0, 31, 32, 63, 95, 96, 100, 127, 128, 500, 1000]
    attend_case(wz, BF16, cached, [1] * len(cached), qh, kvh, 64, 16, window=window, seed=window, max_new=max_new, space=255)
    attend_case(wz, F16, cached, [2, 1, 3] * 3 + [1, 2], qh, kvh, 256, 32, window=window, seed=window, max_new=max_new + 2, space=255)


def test_attend_parts_write_all_that_is_joined(wz, gpu):
    # first tiles of a prompt have fewer blocks than its tiles have parts
    attend_case(wz, BF16, [0, 3], [1500, 200], 1, 1, 64, 16, seed=1, space=255)
    attend_case(wz, F16, [0, 3], [1500, 1], 2, 1, 128, 64, window=700, seed=2, space=255)


def test_attend_refused_request_of_most_rows(wz, gpu):
    # 2^31 pieces of 16 bytes to clear; all tokens' rows in one place, so that they fit
    b = Batch(16, [3], [1 << 20], 1, 4, None)
    w = b.work(wz, 256, 1, 64)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    assert b.read("served", 1)[0] == 0
    cache = Cache(BF16, 4, 16, 1, 64).upload()
    qd, out = DA(256 * 64, np.uint16, zero=True), DA.from_numpy(filled(257 * 64, np.uint16))
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    qs, os_ = wzy_amd.Heads(qd.ptr, 0, 64), wzy_amd.Heads(out.ptr, 0, 64)
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.125, ws.ptr, nb, None)
    got = out.numpy()
    assert (got[:256 * 64] == 0).all() and (got[256 * 64:].view(np.uint8) == FILL).all()


def test_attend_long_chunk_in_parts(wz, gpu):
    # few tiles over many cells: the wide kernel's parts are joined; scores so far apart that parts weigh nothing
    attend_case(wz, BF16, [9000], [40], 4, 1, 128, 64, seed=5)
    attend_case(wz, F16, [9000, 2], [11, 40], 12, 1, 256, 64, seed=6, spread=30.0)


@pytest.mark.parametrize("t", [BF16, F16])
def test_attend_large_and_small_scores(wz, gpu, t):
    attend_case(wz, t, [700, 20], [1, 90], 4, 2, 64, 16, seed=1, spread=40.0)
    attend_case(wz, t, [700, 20], [1, 90], 4, 2, 64, 16, seed=2, spread=1e-3)
    attend_case(wz, t, [700], [1], 4, 2, 128, 16, seed=3, scale=5.0)


def test_attend_refused_requests_become_zero(wz, gpu):
    # one free page: the second request, of 60 rows, is not served; its neighbours are
    attend_case(wz, BF16, [3, 16, 40], [1, 60, 1], 4, 2, 64, 16, seed=9, free=1)


def test_attend_not_a_number_stays_where_it_is_seen(wz, gpu):
    # a cell's NaN key reaches every later row of its head and no earlier one
    t, at = BF16, 50

    def special(r, kb, vb):
        kb[at, 0, 3] = NAN[t]
    rng = np.random.default_rng(0)
    cached, new, qh, kvh, hd, page = [40], [30], 2, 2, 64, 16
    b = Batch(page, cached, new, 6, 9, None, max_new=30)
    w = b.work(wz, qh, kvh, hd)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    table = b.check()[0]
    cache = Cache(t, 9, page, kvh, hd)
    kb, vb = (typed(rng.standard_normal((70, kvh, hd)), t)[0] for _ in range(2))
    special(0, kb, vb)
    cell = np.arange(70)
    cache.put(table[0, cell // page] * page + cell % page, kb, vb)
    cache.upload()
    qd, out = DA.from_numpy(typed(rng.standard_normal((30, qh, hd)), t)[0]), DA(30 * qh * hd, np.uint16)
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * hd, hd)
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.125, ws.ptr, nb, None)
    y = values(out.numpy().reshape(30, qh, hd), t)
    assert np.isfinite(y[:, 1]).all() and np.isfinite(y[:at - 40, 0]).all() and np.isnan(y[at - 40:, 0]).all()


def test_attend_bad_pages_read_the_cache(wz, gpu):
    # ids outside the cache count as page 0
    cache = Cache(BF16, 4, 16, 1, 64)
    rng = np.random.default_rng(4)
    kb, vb = (typed(rng.standard_normal((16, 1, 64)), BF16)[0] for _ in range(2))
    cache.put(np.arange(16), kb, vb)
    cache.upload()
    b = Batch(16, [15], [1], 2, 4, None)
    w = b.work(wz, 1, 1, 64)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    outs = []
    for page in (0, -1, 4, 2 ** 31 - 1, -2 ** 31):
        b.d["table"] = ints([[page, page]])
        b.c.table = b.d["table"].ptr
        qd, out = DA.from_numpy(typed(np.ones((1, 1, 64)), BF16)[0]), DA(64, np.uint16, zero=True)
        nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
        ws = DA(nb, np.uint8)
        qs, os_ = wzy_amd.Heads(qd.ptr, 64, 64), wzy_amd.Heads(out.ptr, 64, 64)
        wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.125, ws.ptr, nb, None)
        outs.append(out.numpy())
    assert all((o == outs[0]).all() for o in outs) and outs[0].any()


def test_attend_list_of_another_kind_writes_nothing(wz, gpu):
    # a list that was not planned, or for other heads, has no work
    b = Batch(16, [5], [1], 2, 4, None)
    w = b.work(wz, 4, 2, 64)
    cache = Cache(BF16, 4, 16, 2, 64).upload()
    qd, out = DA(4 * 64, np.uint16, zero=True), DA.from_numpy(filled(4 * 64, np.uint16))
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    qs, os_ = wzy_amd.Heads(qd.ptr, 256, 64), wzy_amd.Heads(out.ptr, 256, 64)
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.125, ws.ptr, nb, None)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    w.window = 9
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.125, ws.ptr, nb, None)
    assert (out.numpy().view(np.uint8) == FILL).all()


# ---- sampling --------------------------------------------------------------------------------------------
def run_sample(wz, bits, t, rows, vocab, gap, **p):
    wide = filled((rows, vocab + gap), bits.dtype)
    wide[:, :vocab] = bits
    d = dict(x=DA.from_numpy(wide), ids=DA.from_numpy(filled(rows + 2, np.int32)), probs=DA.from_numpy(filled(rows + 2, np.float32)))
    for k, dt in (("temp", np.float32), ("top_k", np.int32), ("top_p", np.float32), ("min_p", np.float32), ("u", np.float32)):
        d[k] = DA.from_numpy(np.asarray(p[k], dt)) if p.get(k) is not None else None
    nb = wz.wzy_sample_workspace_bytes(rows, vocab)
    ws = DA.from_numpy(filled(nb + 64, np.uint8))
    at = [d[k].ptr if d[k] is not None else None for k in ("temp", "top_k", "top_p", "min_p", "u")]
    for _ in range(2):
        wz.wzy_sample(d["x"].ptr, t, vocab + gap, rows, vocab, *at, d["ids"].ptr, d["probs"].ptr, ws.ptr, nb, None)
        ids, probs = d["ids"].numpy(), d["probs"].numpy()
    assert (ws.numpy()[nb:] == FILL).all() and (ids[rows:].view(np.uint8) == FILL).all() and (probs[rows:].view(np.uint8) == FILL).all()
    return ids[:rows], probs[:rows]


def check_sample(wz, x, t, gap=0, **p):
    rows, vocab = x.shape
    bits, v = typed(x, t)
    ids, probs = run_sample(wz, bits, t, rows, vocab, gap, **p)
    for r in range(rows):
        one = {k: a[r] if k == "top_k" else float(np.float32(a[r])) for k, a in p.items() if a is not None}
        i, q, near = R.sample(v[r], **one)
        if near < 1e-11:                                                   # a border that 64 bits do not decide
            continue
        assert ids[r] == i, (r, ids[r], i, one, near)
        assert abs(probs[r] - q) <= 2.0 ** -23 * q + 1e-30, (r, probs[r], q)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab,gap", [(1, 1, 0), (2, 2, 1), (9, 100, 0), (5, 8193, 3), (4, 33333, 7), (3, 151936, 0)])
def test_sample(wz, gpu, t, rows, vocab, gap):
    rng = np.random.default_rng(rows + vocab)
    for filters in ("", "k", "p", "m", "kp", "kpm", "pm"):
        x = rng.standard_normal((rows, vocab)) * rng.choice([0.01, 1.0, 4.0], (rows, 1))
        p = dict(temp=rng.uniform(0.2, 1.5, rows), u=rng.random(rows).astype(np.float32))
        if "k" in filters:
            p["top_k"] = rng.choice([0, 1, 2, 40, vocab, 2 * vocab, 3000], rows)
        if "p" in filters:
            p["top_p"] = rng.choice([0.0, 1e-6, 0.3, 0.9, 0.999, 1.0], rows)
        if "m" in filters:
            p["min_p"] = rng.choice([0.0, 1e-4, 0.05, 0.9, 1.0], rows)
        check_sample(wz, x, t, gap, **p)


def test_sample_ends_of_u(wz, gpu):
    rng = np.random.default_rng(3)
    x = np.tile(rng.standard_normal(500), (6, 1))
    u = np.array([0.0, 1.0, -3.0, 7.0, np.nan, 1.0 - 2.0 ** -24], np.float32)
    ids, _ = run_sample(wz, typed(x, F32)[0], F32, 6, 500, 0, u=u)
    v = typed(x, F32)[1][0]
    order = np.lexsort((np.arange(500), -v))
    assert ids.tolist() == [order[0], order[-1], order[0], order[-1], order[0], R.sample(v, u=float(u[-1]))[0]]


@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_sample_ties_and_specials(wz, gpu, t):
    # equal logits by the thousands (more than are gathered), a few values only, infinities, NaN, empty rows
    rng = np.random.default_rng(11)
    n = 20000
    x = np.zeros((10, n))
    x[1, 5000:] = -1.0
    x[2] = rng.integers(0, 3, n)
    x[3] = -np.inf
    x[3, [7, 4000]] = [1.0, 2.0]
    x[4] = -np.inf
    x[5] = np.nan
    x[6, [3, 900]] = np.inf
    x[7, ::2] = np.nan
    x[8] = rng.integers(0, 2, n) * 1e-3 + rng.integers(0, 2, n) * 0.02
    x[9] = np.where(rng.random(n) < 0.5, 0.0, -0.0)
    for k, tp, mp in ((0, 1.0, 0.0), (7001, 1.0, 0.0), (0, 0.7, 0.0), (15000, 0.5, 0.0), (0, 1.0, 0.5), (9000, 0.9, 0.98)):
        u = rng.random(10).astype(np.float32)
        check_sample(wz, x, t, temp=np.full(10, 0.8), top_k=np.full(10, k), top_p=np.full(10, tp), min_p=np.full(10, mp), u=u)


def test_sample_greedy_and_extreme_temperatures(wz, gpu):
    rng = np.random.default_rng(12)
    x = rng.standard_normal((8, 3001)) * 3
    x[2, [10, 20]] = 50.0                                                  # a tie at the top: the lower id
    x[3] *= 1e30
    x[4, 5] = 3e38
    check_sample(wz, x, F32, temp=np.array([0.0, 1e-5, -1.0, 1.0, 1.0, 2e-5, 1e4, 1e30]), u=rng.random(8).astype(np.float32),
                 top_k=np.array([0, 5, 9, 50, 0, 0, 0, 2000]))
    check_sample(wz, x, F32, temp=np.full(8, 0.7), u=rng.random(8).astype(np.float32), min_p=np.array([2.0, 1.0, 1.5, 0.1, 0.1, 0.0, -1.0, 1e-30]))


def test_sample_as_the_host_sampler(wz, gpu):
    """the engine's sampler on the same logits: the same cuts, apart from its fp32 sums"""
    rng = np.random.default_rng(13)
    rows, vocab = 40, 5000
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    cfg = wzy_amd.GenCfg()
    wz.wzy_engine_cfg_default(ref(cfg))
    cfg.temp, cfg.top_k, cfg.top_p, cfg.min_p = 0.7, 50, 0.9, 0.02
    ids, probs = run_sample(wz, x, F32, rows, vocab, 0, temp=[0.7] * rows, top_k=[50] * rows, top_p=[0.9] * rows, min_p=[0.02] * rows, u=u)
    for r in range(rows):
        hi, hp = np.zeros(128, np.int32), np.zeros(128, np.float32)
        n = wz.wzy_engine_target_dist(x[r].ctypes.data, vocab, ref(cfg), None, 0, hi.ctypes.data, hp.ctypes.data, 128)
        at = np.flatnonzero(hi[:n] == ids[r])
        assert len(at) == 1
        assert abs(hp[at[0]] - probs[r]) <= 1e-5 * probs[r] + 1e-7
        c = np.cumsum(hp[:n].astype(np.float64))
        near = np.abs(c - u[r]).min()
        if near > 1e-5:
            tok = C.c_int(-1)
            wz.wzy_engine_verify_full(x[r].ctypes.data, vocab, ref(cfg), None, 0, -1, float(u[r]), ref(tok))
            assert tok.value == ids[r]
