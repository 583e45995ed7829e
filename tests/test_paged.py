"""Operators for several requests at once: refusals and sizes, on the host (include/wzy_paged.h)."""
import ctypes as C

import pytest

import wzy_amd
from wzy_amd import TYPE_BF16, TYPE_F16, TYPE_F32

EINVAL = -1
PTR = 4096                                                                 # never dereferenced: checks come first


def batch(**over):
    a = dict(n_req=4, max_tokens=8, max_pages=16, n_cached=PTR, n_new=PTR, table=PTR, q_start=PTR, kv_len=PTR, served=PTR, positions=PTR,
             slots=PTR, max_new=0)
    a.update(over)
    return wzy_amd.PagedBatch(*a.values())


def work(wz, b=None, **over):
    a = dict(qh=8, kvh=2, hd=128, window=0, items=PTR, bytes=1 << 30)
    a.update(over)
    return wzy_amd.PagedWork(*a.values())


def pool(**over):
    a = dict(free_pages=PTR, n_free=PTR, n_free_out=PTR, n_pages=64, page=16)
    a.update(over)
    return wzy_amd.PagedPool(*a.values())


def cache(**over):
    a = dict(k=PTR, v=PTR, ld_page=16 * 2 * 128, ld_cell=2 * 128, ld_head=128, n_pages=64, page=16, kvh=2, hd=128, type=TYPE_BF16)
    a.update(over)
    return wzy_amd.PagedCache(*a.values())


def heads(p=PTR, ld=8 * 128, ld_head=128):
    return wzy_amd.Heads(p, ld, ld_head)


def refused(wz, fn, *args):
    rc = getattr(wz.dll, fn)(*[C.byref(a) if isinstance(a, C.Structure) else a for a in args])
    assert rc == EINVAL
    assert fn in wz.wzy_last_error().decode()


@pytest.mark.parametrize("over", [dict(n_req=0), dict(n_req=4097), dict(max_tokens=0), dict(max_tokens=(1 << 20) + 1), dict(max_pages=0),
                                  dict(max_pages=1 << 21), dict(max_new=-1), dict(n_cached=None), dict(n_new=None), dict(table=None),
                                  dict(q_start=None), dict(kv_len=None), dict(served=None), dict(positions=None), dict(slots=None)])
def test_plan_refuses_batches(wz, over):
    refused(wz, "wzy_paged_plan", pool(), batch(**over), None, 0, None)


@pytest.mark.parametrize("over", [dict(page=8), dict(page=24), dict(page=8192), dict(n_pages=0), dict(n_pages=1 << 27), dict(free_pages=None),
                                  dict(n_free=None), dict(n_free_out=None)])
def test_plan_and_release_refuse_pools(wz, over):
    refused(wz, "wzy_paged_plan", pool(**over), batch(), None, 0, None)
    refused(wz, "wzy_paged_release", pool(**over), batch(), PTR, None)


@pytest.mark.parametrize("over", [dict(qh=0), dict(kvh=0), dict(kvh=65, qh=65), dict(qh=9), dict(qh=600), dict(hd=96), dict(window=-1), dict(items=None),
                                  dict(items=PTR + 8), dict(bytes=100)])
def test_plan_refuses_work_lists(wz, over):
    refused(wz, "wzy_paged_plan", pool(), batch(), work(wz, **over), 1, None)


def test_plan_refuses_counts_of_lists(wz):
    refused(wz, "wzy_paged_plan", pool(), batch(), None, 1, None)
    refused(wz, "wzy_paged_plan", pool(), batch(), work(wz), 9, None)
    two = (wzy_amd.PagedWork * 2)(work(wz), work(wz))                       # one memory for two
    assert wz.dll.wzy_paged_plan(C.byref(pool()), C.byref(batch()), two, 2, None) == EINVAL
    refused(wz, "wzy_paged_release", pool(), batch(), None, None)


def test_sizes(wz):
    b, w = batch(), work(wz)
    n = wz.wzy_paged_work_bytes(C.byref(b), C.byref(w))
    assert 64 < n < 1 << 20
    assert wz.wzy_paged_work_bytes(C.byref(batch(max_tokens=4096)), C.byref(w)) > n
    assert wz.wzy_paged_work_bytes(C.byref(batch(n_req=0)), C.byref(w)) == 0
    assert wz.wzy_paged_work_bytes(C.byref(b), C.byref(work(wz, hd=100))) == 0
    assert wz.wzy_paged_attend_workspace_bytes(C.byref(b), C.byref(work(wz, kvh=0))) == 0
    # single tokens of 4 heads a key head need no wide tiles' room
    small = wz.wzy_paged_attend_workspace_bytes(C.byref(batch(max_new=1)), C.byref(w))
    assert 0 < small < wz.wzy_paged_attend_workspace_bytes(C.byref(batch(max_tokens=4096)), C.byref(w))
    assert wz.wzy_sample_workspace_bytes(0, 10) == wz.wzy_sample_workspace_bytes(1, 0) == wz.wzy_sample_workspace_bytes(1, (1 << 22) + 1) == 0
    assert wz.wzy_sample_workspace_bytes(2, 1000) > wz.wzy_sample_workspace_bytes(1, 1000) > 0


@pytest.mark.parametrize("over", [dict(theta=1.0), dict(theta=float("nan")), dict(n_rot=0), dict(n_rot=3), dict(n_rot=514), dict(scaling=4), dict(scaling=-1),
                                  dict(scaling=1, factor=0.5), dict(scaling=2, low=0.0), dict(scaling=2, low=4.0, high=4.0), dict(scaling=3, ctx=0),
                                  dict(amplitude=float("inf"))])
def test_rope_freqs_refuses(wz, over):
    a = dict(theta=1e4, factor=2.0, low=1.0, high=32.0, amplitude=1.0, ctx=4096, n_rot=64, scaling=0)
    a.update(over)
    refused(wz, "wzy_rope_freqs", wzy_amd.RopeCfg(*a.values()), PTR, None)


def test_rope_refuses(wz):
    tab, x = wzy_amd.RopeTab(PTR, 64, 0), heads()

    def no(tab=tab, x=x, t=TYPE_BF16, rows=1, n=8, hd=128, pos=PTR, y=x):
        refused(wz, "wzy_rope", tab, x, t, rows, n, hd, pos, y, None)
    no(tab=None)
    no(tab=wzy_amd.RopeTab(None, 64, 0))
    no(tab=wzy_amd.RopeTab(PTR, 65, 0))
    no(tab=wzy_amd.RopeTab(PTR, 130, 0))
    no(tab=wzy_amd.RopeTab(PTR, 64, 2))
    no(t=3)
    no(rows=-1)
    no(n=0)
    no(n=1025)
    no(hd=513)
    no(pos=None)
    no(x=heads(None))
    no(y=heads(None))
    no(x=heads(PTR + 1))
    no(x=heads(ld_head=100))
    no(y=heads(ld=-8))
    no(y=heads(ld=2048))                                                   # in place with another stride
    assert wz.dll.wzy_rope(C.byref(tab), C.byref(x), TYPE_BF16, 0, 8, 128, PTR, C.byref(x), None) == 0


@pytest.mark.parametrize("over", [dict(k=None), dict(v=None), dict(k=PTR + 8), dict(ld_page=4), dict(ld_cell=100), dict(ld_cell=1 << 24), dict(ld_head=64),
                                  dict(kvh=0), dict(kvh=65), dict(hd=96), dict(type=TYPE_F32), dict(page=17), dict(n_pages=0)])
def test_append_and_attend_refuse_caches(wz, over):
    q = heads()
    refused(wz, "wzy_paged_append", cache(**over), None, q, 8, heads(2 * PTR), q, q, TYPE_F16, 1, PTR, PTR, None)
    refused(wz, "wzy_paged_attend", cache(**over), batch(), work(wz), q, heads(2 * PTR), 0.1, PTR, 1 << 40, None)


def test_append_refuses(wz):
    tab, q, o = wzy_amd.RopeTab(PTR, 64, 0), heads(), heads(2 * PTR)

    def no(tab=tab, q=q, qh=8, o=o, k=q, v=q, t=TYPE_BF16, rows=1, pos=PTR, slots=PTR):
        refused(wz, "wzy_paged_append", cache(), tab, q, qh, o, k, v, t, rows, pos, slots, None)
    no(tab=wzy_amd.RopeTab(PTR, 256, 0))
    no(q=None)
    no(o=None)
    no(qh=0)
    no(qh=1025)
    no(k=None)
    no(v=None)
    no(t=9)
    no(rows=-1)
    no(pos=None)
    no(slots=None)
    no(o=q, t=TYPE_F16)                                                     # in place, another type
    no(o=heads(ld=4096))
    assert wz.dll.wzy_paged_append(C.byref(cache()), None, None, 0, None, C.byref(q), C.byref(q), TYPE_F32, 0, None, None, None) == 0


def test_attend_refuses(wz):
    q, o = heads(), heads(2 * PTR)
    space = wz.wzy_paged_attend_workspace_bytes(C.byref(batch()), C.byref(work(wz)))

    def no(b=batch(), w=None, q=q, o=o, scale=0.1, ws=PTR, n=space, c=cache()):
        refused(wz, "wzy_paged_attend", c, b, w or work(wz), q, o, scale, ws, n, None)
    no(b=batch(n_req=0))
    no(b=batch(table=None))
    no(w=work(wz, hd=64))
    no(w=work(wz, kvh=4))
    no(w=work(wz, bytes=64))
    no(w=work(wz, items=None))
    no(q=heads(None))
    no(q=heads(PTR + 2))
    no(q=heads(ld=1028))
    no(o=heads(2 * PTR, ld_head=132))
    no(o=q)
    no(scale=0.0)
    no(scale=-1.0)
    no(scale=float("nan"))
    no(scale=float("inf"))
    no(ws=None)
    no(ws=PTR + 4)
    no(n=space - 1)


def test_sample_refuses(wz):
    n = wz.wzy_sample_workspace_bytes(2, 100)

    def no(x=PTR, t=TYPE_F32, ld=100, rows=2, vocab=100, u=PTR, ids=PTR, ws=PTR, n=n):
        refused(wz, "wzy_sample", x, t, ld, rows, vocab, None, None, None, None, u, ids, None, ws, n, None)
    no(x=None)
    no(x=PTR + 2)
    no(t=5)
    no(ld=99)
    no(rows=-1)
    no(rows=65536)
    no(vocab=0)
    no(vocab=(1 << 22) + 1)
    no(u=None)
    no(ids=None)
    no(ws=None)
    no(ws=PTR + 8)
    no(n=n - 1)
    assert wz.dll.wzy_sample(None, TYPE_F32, 100, 0, 100, None, None, None, None, None, None, None, None, 0, None) == 0
