"""Plain 64-bit formulations of the operators for several requests at once (test infrastructure)."""
import math

import numpy as np


def plan(page, n_pages, n_free, free, n_cached, n_new, table, max_tokens, max_new):
    """one request after another: (table, q_start, kv_len, served, positions, slots, n_free)"""
    table = table.copy()
    R, max_pages = table.shape
    q_start, kv_len, served = np.zeros(R + 1, np.int32), np.zeros(R, np.int32), np.zeros(R, np.int32)
    positions, slots = np.zeros(max_tokens, np.int32), np.full(max_tokens, -1, np.int32)
    at, wanted, taken = 0, 0, 0
    for r in range(R):
        c, n = max(int(n_cached[r]), 0), max(int(n_new[r]), 0)
        ok = c + n <= max_pages * page and n <= max_new and (n == 0 or at + n <= max_tokens)
        held = -(-c // page)
        need = -(-(c + n) // page) - held if ok else 0
        wanted += need
        if need and wanted > n_free:
            ok = False
        if ok:
            for i in range(need):
                table[r, held + i] = free[n_free - 1 - taken]
                taken += 1
        served[r], kv_len[r] = ok, c + n if ok else 0
        for i in range(n if ok else 0):
            p = c + i
            positions[at + i], slots[at + i] = p, table[r, p // page] * page + p % page
        at += n
        q_start[r + 1] = min(at, max_tokens)
    return table, q_start, kv_len, served, positions, slots, n_free - taken


def frequencies(n_rot, theta, scaling=0, factor=1.0, low=1.0, high=32.0, ctx=0):
    """0 plain, 1 linear, 2 by rotations, 3 by pair numbers"""
    out = []
    for i in range(n_rot // 2):
        f = theta ** (-2.0 * i / n_rot)
        keep = 1.0
        if scaling == 1:
            keep = 0.0
        if scaling == 2:
            keep = (ctx * f / (2 * math.pi) - low) / (high - low)
        if scaling == 3:
            a, b = (n_rot * math.log(ctx / (2 * math.pi * x)) / (2 * math.log(theta)) for x in (high, low))
            a, b = max(math.floor(a), 0), min(math.ceil(b), n_rot - 1)
            keep = 1 - (i - a) / (b - a) if b > a else float(i <= a)
        keep = min(max(keep, 0.0), 1.0)
        out.append(keep * f + (1 - keep) * f / factor)
    return np.array(out)


def rope(x, f, n_rot, pairs, positions, amplitude=1.0):
    """x [rows, heads, hd] float64"""
    a = positions.astype(np.float64)[:, None] * f
    c, s = (np.cos(a) * amplitude)[:, None, :], (np.sin(a) * amplitude)[:, None, :]
    y = x.copy()
    i, j = (slice(0, n_rot, 2), slice(1, n_rot, 2)) if pairs else (slice(0, n_rot // 2), slice(n_rot // 2, n_rot))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def attend(q, k, v, n_cached, window, scale):
    """q [new, qh, hd], k and v [cells, kvh, hd] float64 -> (out, sum of |p v|, the largest sum of |q k|)"""
    new, qh, hd = q.shape
    cells, g = k.shape[0], qh // k.shape[1]
    out, size, top = np.zeros_like(q), np.zeros_like(q), 0.0
    p = n_cached + np.arange(new)[:, None]
    see = (np.arange(cells) <= p) & ((np.arange(cells) > p - window) if window else True)
    for h in range(qh):
        kh, vh = k[:, h // g], v[:, h // g]
        s = np.where(see, q[:, h] @ kh.T * scale, -np.inf)
        top = max(top, (np.abs(q[:, h]) @ np.abs(kh).T).max() * scale)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[:, h], size[:, h] = w @ vh, w @ np.abs(vh)
    return out, size, top


def sample(logits, temp=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """one row of float64 logits -> (id, prob, how near the draw and the cuts come to another answer)"""
    x = np.where(np.isnan(logits), -np.inf, logits)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return -1, 0.0, 1.0
    if not temp > 1e-5:
        return int(order[0]), 1.0, 1.0
    if 1 <= top_k < len(order):
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(x[order] == top, 0.0, (x[order] - top) / temp))
    cum = np.cumsum(w.astype(np.longdouble))
    n, near = len(w), 1.0
    if min_p > 0:
        m = int((w >= min_p).sum()) if min_p <= 1 else 1
        near = min(near, np.abs(w / min_p - 1)[1:].min(initial=1.0))
        n = max(m, 1)
    if 0 < top_p < 1:
        t = top_p * cum[-1]
        n = min(n, int((cum < t).sum()) + 1)
        near = min(near, float(np.abs(cum - t).min() / cum[-1]))
    t = min(max(u, 0.0), 1.0) * cum[n - 1]
    i = min(int((cum[:n] < t).sum()), n - 1)
    if 0 < u < 1:
        near = min(near, float(np.abs(cum[:n] - t).min() / cum[n - 1]))
    return int(order[i]), float(w[i] / cum[n - 1]), near
