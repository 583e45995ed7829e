"""Operators for several requests at once (include/wzy_paged.h) used together: serving steps, streams, graphs, large caches,
values that are not finite."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
import wzy_amd
from mx_ref import BF16, F16, F32, HALF_STEP, typed, values
from test_gpu_paged import FILL, NAN, Batch, Cache, filled, freqs, ints, ref, rope_bound

pytestmark = pytest.mark.gpu
DA = wzy_amd.DeviceArray
INF = {BF16: 0x7F80, F16: 0x7C00}


class Serving:
    """a batch's device state: what a serving program keeps"""

    def __init__(self, wz, slots, max_tokens, max_pages, n_pages, page, qh, kvh, hd, t=BF16, vocab=1000, window=0, seed=0):
        self.wz, self.R, self.max_tokens, self.t, self.vocab = wz, slots, max_tokens, t, vocab
        self.qh, self.kvh, self.hd, self.page, self.n_pages, self.window = qh, kvh, hd, page, n_pages, window
        self.d = dict(cached=ints([0] * slots), new=ints([0] * slots), table=ints([[-1] * max_pages] * slots),
                      free=ints(np.random.default_rng(seed).permutation(n_pages)), n_free=ints([n_pages]), q_start=ints([0] * (slots + 1)),
                      kv_len=ints([0] * slots), served=ints([0] * slots), positions=ints([0] * max_tokens), slots=ints([0] * max_tokens))
        d = self.d
        self.b = wzy_amd.PagedBatch(slots, max_tokens, max_pages, d["cached"].ptr, d["new"].ptr, d["table"].ptr, d["q_start"].ptr,
                                    d["kv_len"].ptr, d["served"].ptr, d["positions"].ptr, d["slots"].ptr, 0)
        self.pool = wzy_amd.PagedPool(d["free"].ptr, d["n_free"].ptr, d["n_free"].ptr, n_pages, page)
        self.w = wzy_amd.PagedWork(qh, kvh, hd, window, None, 0)
        self.w.bytes = wz.wzy_paged_work_bytes(ref(self.b), ref(self.w))
        self.items = DA(self.w.bytes, np.uint8)
        self.w.items = self.items.ptr
        self.cache = Cache(t, n_pages, page, kvh, hd).upload()
        self.n_space = wz.wzy_paged_attend_workspace_bytes(ref(self.b), ref(self.w))
        self.space = DA(self.n_space, np.uint8)
        self.freqs = freqs(wz, hd // 2, 0, 1e4)
        self.tab = wzy_amd.RopeTab(self.freqs.ptr, hd // 2, 0)
        self.x = DA((max_tokens, qh + 2 * kvh, hd), np.float32, zero=True)
        self.q, self.out = (DA((max_tokens, qh, hd), np.uint16, zero=True) for _ in range(2))
        self.logits, self.u = DA((slots, vocab), np.float32, zero=True), DA(slots, np.float32, zero=True)
        self.ids, self.probs = DA(slots, np.int32), DA(slots, np.float32)
        self.top_k, self.top_p = ints([40, 0, 3, 0, 500][:slots]), DA.from_numpy(np.array([1.0, 0.8, 0.5, 1.0, 0.9][:slots], np.float32))
        self.n_sample = wz.wzy_sample_workspace_bytes(slots, vocab)
        self.sample_space = DA(self.n_sample, np.uint8)

    def heads(self, a, at=0):
        return wzy_amd.Heads(a.ptr + at * self.hd * a.dtype.itemsize, a.shape[1] * self.hd, self.hd)

    def enqueue(self, s):
        """one step of one layer on stream s"""
        wz = self.wz
        wz.wzy_paged_plan(ref(self.pool), ref(self.b), ref(self.w), 1, s)
        q, k, v, qo, o = self.heads(self.x), self.heads(self.x, self.qh), self.heads(self.x, self.qh + self.kvh), self.heads(self.q), self.heads(self.out)
        wz.wzy_paged_append(ref(self.cache.c), ref(self.tab), ref(q), self.qh, ref(qo), ref(k), ref(v), F32, self.max_tokens,
                            self.d["positions"].ptr, self.d["slots"].ptr, s)
        wz.wzy_paged_attend(ref(self.cache.c), ref(self.b), ref(self.w), ref(qo), ref(o), self.hd ** -0.5, self.space.ptr, self.n_space, s)
        wz.wzy_sample(self.logits.ptr, F32, self.vocab, self.R, self.vocab, None, self.top_k.ptr, self.top_p.ptr, None, self.u.ptr, self.ids.ptr,
                      self.probs.ptr, self.sample_space.ptr, self.n_sample, s)

    def put(self, name, a):
        a = np.ascontiguousarray(a)
        d = self.d[name] if name in self.d else getattr(self, name)
        assert a.nbytes == d.nbytes and a.dtype == d.dtype
        self.wz.wzy_memcpy_h2d(d.ptr, a.ctypes.data, d.nbytes, None)


def attend_rows(q, k, v, cached, window, scale):
    """as paged_ref.attend, but cells that a row does not see stay out of its sums whatever they hold"""
    out = np.zeros_like(q)
    g = q.shape[1] // k.shape[1]
    for t in range(q.shape[0]):
        lo = max(0, cached + t - window + 1) if window else 0
        for h in range(q.shape[1]):
            s = k[lo:cached + t + 1, h // g] @ q[t, h] * scale
            w = np.exp(s - s.max())
            with np.errstate(invalid="ignore"):
                out[t, h] = w / w.sum() @ v[lo:cached + t + 1, h // g]
    return out


@pytest.mark.parametrize("t", [BF16, F16])
def test_serving_steps(wz, gpu, t):
    """prompts, verify windows and single tokens over a dozen steps; requests end and others take their place"""
    rng = np.random.default_rng(1)
    R5, hd, qh, kvh, page = 5, 64, 6, 2, 16
    s = Serving(wz, R5, 300, 12, 50, page, qh, kvh, hd, t)
    cached = np.zeros(R5, np.int32)
    for step in range(12):
        new = rng.choice([0, 1, 1, 4], R5).astype(np.int32)
        if step == 0:
            new[:] = [100, 7, 0, 33, 1]
        if step == 5:                                       # two requests end, a long prompt comes instead
            ended = np.array([1, 0, 0, 1, 0], np.int32)
            e = ints(ended)
            before = int(s.d["n_free"].numpy()[0])
            wz.wzy_paged_release(ref(s.pool), ref(s.b), e.ptr, None)
            assert s.d["n_free"].numpy()[0] == before + sum(-(-int(cached[r]) // page) for r in (0, 3))
            cached[ended == 1] = 0
            new[0], new[3] = 150, 1
        x = rng.standard_normal((s.max_tokens, qh + 2 * kvh, hd)).astype(np.float32)
        logits, u = rng.standard_normal((R5, s.vocab)).astype(np.float32) * 2, rng.random(R5).astype(np.float32)
        for name, a in (("cached", cached), ("new", new), ("x", x), ("logits", logits), ("u", u)):
            s.put(name, a)
        out0 = s.out.numpy()
        s.enqueue(None)
        assert s.d["served"].numpy().all()
        q_start, table = s.d["q_start"].numpy(), s.d["table"].numpy().reshape(R5, -1)
        held = [i for r in range(R5) for i in table[r, :-(-int(cached[r] + new[r]) // page)]]
        assert len(set(held)) == len(held) and 0 <= min(held) and max(held) < s.n_pages       # nobody shares a page
        kc, vc, q, out = s.cache.dk.numpy(), s.cache.dv.numpy(), values(s.q.numpy(), t), s.out.numpy()
        np.testing.assert_array_equal(out[q_start[-1]:], out0[q_start[-1]:])
        f = R.frequencies(hd // 2, 1e4)
        for r in range(R5):
            n, a = int(new[r]), int(q_start[r])
            if n == 0:
                continue
            cell = np.arange(cached[r] + n)
            page_of = table[r, cell // page]
            k, v = (values(np.ascontiguousarray(c[page_of, cell % page]), t) for c in (kc, vc))
            xr = x[a:a + n].astype(np.float64)
            turned = R.rope(xr, f, hd // 2, 0, cached[r] + np.arange(n))
            bound = rope_bound(xr, turned, t)
            assert (np.abs(q[a:a + n] - turned[:, :qh]) <= bound[:, :qh]).all()
            assert (np.abs(k[cached[r]:] - turned[:, qh:qh + kvh]) <= bound[:, qh:qh + kvh]).all()
            assert (np.abs(v[cached[r]:] - xr[:, qh + kvh:]) <= HALF_STEP[t] * np.abs(xr[:, qh + kvh:]) + 2.0 ** -25).all()
            want, size, top = R.attend(q[a:a + n], k, v, int(cached[r]), 0, hd ** -0.5)
            tol = HALF_STEP[t] * (np.abs(want) + size) * 1.01 + size * (2 * hd * 2.0 ** -24 * top + 2.0 ** -14) + 2.0 ** -20
            assert (np.abs(values(out[a:a + n], t) - want) <= tol).all()
        ids, probs, top_k, top_p = s.ids.numpy(), s.probs.numpy(), s.top_k.numpy(), s.top_p.numpy()
        for r in range(R5):
            i, p, near = R.sample(logits[r].astype(np.float64), 1.0, int(top_k[r]), float(top_p[r]), 0.0, float(u[r]))
            if near > 1e-11:
                assert ids[r] == i and abs(probs[r] - p) <= 2.0 ** -23 * p + 1e-30
        cached += new


def test_two_streams_and_graph_replays(wz, gpu):
    """two batches on two streams at once, then a captured step replayed with other lengths, eager work between: the same bits"""
    hip = C.CDLL("libamdhip64.so")
    rng = np.random.default_rng(2)
    R5, T = 5, 64
    lens = [([0, 40, 3, 100, 17], [30, 1, 4, 1, 9]), ([5, 0, 77, 31, 130], [1, 1, 1, 1, 1]), ([16, 15, 0, 64, 1], [2, 20, 33, 0, 1])]
    x = rng.standard_normal((T, 10, 64)).astype(np.float32)
    logits, u = rng.standard_normal((R5, 1000)).astype(np.float32), rng.random(R5).astype(np.float32)
    pages = rng.permutation(90).astype(np.int32)            # the pool holds those that no request has
    table, free = pages[:60].reshape(R5, 12), np.concatenate([pages[60:], pages[:60]])
    k, v = (typed(rng.standard_normal((90, 16, 2, 64)), BF16)[0] for _ in range(2))

    def fresh():
        s = Serving(wz, R5, T, 12, 90, 16, 6, 2, 64)
        for name, a in (("x", x), ("logits", logits), ("u", u)):
            s.put(name, a)
        s.put("free", free)
        s.put("n_free", np.int32([30]))
        s.left = ints([0])
        s.pool.n_free_out = s.left.ptr                      # the pool stays as it is: the same step again takes the same pages
        return s

    def reset(s, which):
        for name, a in (("table", table), ("cached", np.int32(lens[which][0])), ("new", np.int32(lens[which][1]))):
            s.put(name, a)
        wz.wzy_memcpy_h2d(s.cache.dk.ptr, k.ctypes.data, k.nbytes, None)
        wz.wzy_memcpy_h2d(s.cache.dv.ptr, v.ctypes.data, v.nbytes, None)
        wz.wzy_memset(s.out.ptr, 0x5A, s.out.nbytes, None)
        wz.wzy_device_sync()

    def bits(s):
        return [s.out.numpy(), s.q.numpy()[:s.d["q_start"].numpy()[-1]], s.cache.dk.numpy(), s.cache.dv.numpy(), s.ids.numpy(), s.probs.numpy(),
                s.d["slots"].numpy(), s.d["table"].numpy(), s.left.numpy()]

    one, two, three = fresh(), fresh(), fresh()
    want = []
    for which in range(3):
        reset(one, which)
        one.enqueue(None)
        wz.wzy_device_sync()
        want.append(bits(one))
    st = [C.c_void_p(), C.c_void_p()]
    for s in st:
        wz.wzy_stream_create(C.byref(s))
    reset(one, 0)
    reset(two, 1)
    for _ in range(5):
        one.enqueue(st[0].value)
        two.enqueue(st[1].value)
    wz.wzy_device_sync()
    for s, w in ((one, want[0]), (two, want[1])):
        for a, b in zip(bits(s), w):
            np.testing.assert_array_equal(a, b)
    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(st[0], 2) == 0
    three.enqueue(st[0].value)
    assert hip.hipStreamEndCapture(st[0], C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for which in (0, 1, 2, 1, 0, 2):
        reset(three, which)
        assert hip.hipGraphLaunch(run, st[0]) == 0
        wz.wzy_device_sync()
        for a, b in zip(bits(three), want[which]):
            np.testing.assert_array_equal(a, b)
        reset(one, 2)
        one.enqueue(None)
        wz.wzy_device_sync()
        for a, b in zip(bits(one), want[2]):
            np.testing.assert_array_equal(a, b)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    for s in st:
        wz.wzy_stream_destroy(s.value)


def test_two_lists_of_one_plan(wz, gpu):
    """layers with and without a window, and with other heads, from one plan"""
    rng = np.random.default_rng(4)
    cached, new = [60, 0, 200], [3, 40, 1]
    b = Batch(16, cached, new, 14, 40, None, max_new=40)
    kinds = [(4, 2, 64, 0), (4, 2, 64, 20), (3, 1, 128, 0)]
    works = (wzy_amd.PagedWork * 3)()
    items = []
    for i, kind in enumerate(kinds):
        works[i] = b.work(wz, *kind)
        items.append(b.items)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), works, 3, None)
    table = b.check()[0]
    for w, (qh, kvh, hd, window) in zip(works, kinds):
        cache = Cache(F16, 40, 16, kvh, hd)
        kv = []
        for r in range(3):
            (kb, k), (vb, v) = (typed(rng.standard_normal((cached[r] + new[r], kvh, hd)), F16) for _ in range(2))
            cell = np.arange(cached[r] + new[r])
            cache.put(table[r, cell // 16] * 16 + cell % 16, kb, vb)
            kv.append((k, v))
        cache.upload()
        qb, q = typed(rng.standard_normal((44, qh, hd)), F16)
        qd, out = DA.from_numpy(qb), DA((44, qh, hd), np.uint16)
        n = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
        ws = DA(n, np.uint8)
        qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * hd, hd)
        wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.1, ws.ptr, n, None)
        got, at = values(out.numpy(), F16), 0
        for r in range(3):
            want, size, top = R.attend(q[at:at + new[r]], *kv[r], cached[r], window, 0.1)
            tol = HALF_STEP[F16] * (np.abs(want) + size) * 1.01 + size * (2 * hd * 2.0 ** -24 * top + 2.0 ** -15) + 2.0 ** -20
            assert (np.abs(got[at:at + new[r]] - want) <= tol).all()
            at += new[r]


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("qh,hd,cached,new,window", [(2, 64, 40, 4, 0), (24, 256, 40, 4, 0), (12, 128, 300, 5, 0), (4, 64, 70, 90, 0),
                                                     (8, 256, 30, 60, 25), (2, 128, 5000, 6, 3000)])
def test_values_that_are_not_finite(wz, gpu, t, qh, hd, cached, new, window):
    """an infinity or a NaN in V reaches the rows that see its cell, in its column, and no others"""
    rng = np.random.default_rng(hd + new)
    kvh, page, n = 2 if qh > 2 else 1, 16, cached + new
    b = Batch(page, [cached], [new], -(-n // page), -(-n // page) + 2, None, max_new=new)
    w = b.work(wz, qh, kvh, hd, window)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    table = b.check()[0]
    kb, vb = (typed(rng.standard_normal((n, kvh, hd)), t)[0] for _ in range(2))
    for cell, column, bits in ((cached + new // 2, 3, INF[t]), (cached + new - 1, 40, NAN[t]), (cached + 1, 63, INF[t] | 0x8000)):
        vb[cell, kvh - 1, column] = bits
    if window:                                              # out of the window of the later rows
        vb[cached + new // 2 - window, 0, 7] = NAN[t]
    k, v = values(kb, t), values(vb, t)
    cache = Cache(t, b.n_pages, page, kvh, hd)
    cell = np.arange(n)
    cache.put(table[0, cell // page] * page + cell % page, kb, vb)
    cache.upload()
    qb, q = typed(rng.standard_normal((new, qh, hd)), t)
    qd, out = DA.from_numpy(qb), DA((new, qh, hd), np.uint16)
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    qs, os_ = wzy_amd.Heads(qd.ptr, qh * hd, hd), wzy_amd.Heads(out.ptr, qh * hd, hd)
    wz.wzy_paged_attend(ref(cache.c), ref(b.c), ref(w), ref(qs), ref(os_), 0.1, ws.ptr, nb, None)
    got, want = values(out.numpy(), t), attend_rows(q, k, v, cached, window, 0.1)
    ok = np.isfinite(want)
    np.testing.assert_array_equal(np.isfinite(got), ok)
    np.testing.assert_array_equal(got[~ok], want[~ok])
    size = np.abs(v[np.isfinite(v)]).max()
    assert (np.abs(got[ok] - want[ok]) <= HALF_STEP[t] * (np.abs(want[ok]) + size) + 2.0 ** -12 * size).all()


def test_cache_past_four_gib(wz, gpu):
    """pages 4 GiB apart: every product of a page's number and its stride passes 32 bits"""
    rng = np.random.default_rng(8)
    page, hd, n, t = 32, 64, 70, BF16
    ld_page = 1 << 31                                       # elements
    k, v = (DA(2 * (2 * ld_page + page * hd), np.uint8) for _ in range(2))
    c = wzy_amd.PagedCache(k.ptr, v.ptr, ld_page, hd, hd, 3, page, 1, hd, t)
    b = Batch(page, [0], [n], 3, 3, None, max_new=n)
    w = b.work(wz, 2, 1, hd)
    wz.wzy_paged_plan(ref(b.pool), ref(b.c), ref(w), 1, None)
    b.check()
    bits, x = typed(rng.standard_normal((n, 4, hd)), t)
    xd, qd, out = DA.from_numpy(bits), DA((n, 2, hd), np.uint16), DA((n, 2, hd), np.uint16)
    q, kk, vv = (wzy_amd.Heads(xd.ptr + 2 * hd * at, 4 * hd, hd) for at in (0, 2, 3))
    qo, o = wzy_amd.Heads(qd.ptr, 2 * hd, hd), wzy_amd.Heads(out.ptr, 2 * hd, hd)
    wz.wzy_paged_append(ref(c), None, ref(q), 2, ref(qo), ref(kk), ref(vv), t, n, None, b.d["slots"].ptr, None)
    nb = wz.wzy_paged_attend_workspace_bytes(ref(b.c), ref(w))
    ws = DA(nb, np.uint8)
    wz.wzy_paged_attend(ref(c), ref(b.c), ref(w), ref(qo), ref(o), 0.125, ws.ptr, nb, None)
    np.testing.assert_array_equal(qd.numpy(), bits[:, :2])
    want, size, top = R.attend(x[:, :2], x[:, 2:3], x[:, 3:4], 0, 0, 0.125)
    tol = HALF_STEP[t] * (np.abs(want) + size) * 1.01 + size * (2 * hd * 2.0 ** -24 * top + 2.0 ** -15)
    assert (np.abs(values(out.numpy(), t) - want) <= tol).all()
