"""Measured cases of the operators that serve several requests at once from a paged key-value cache.

The operators, as a program that serves a batch of requests with this library calls them in each step:

  plan     pages for the step's new tokens from the pool of free ones; block tables, row starts, positions and
           cache slots of the packed rows, from the requests' lengths on the GPU
  rope     rotary positions on rows of heads
  append   rotary positions on new queries and keys, keys and values to their slots of the paged cache
  attend   attention of the new tokens over the paged cache: single tokens, verify windows, prompt chunks
  sample   next tokens by temperature, top-k, min-p and top-p from given uniform numbers

With `own` false the operators run in plain torch arithmetic, with `own` true through the library's C ABI.
"""
import ctypes as C
import math
import os
import statistics
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
THETA = 1e7


def listed():
    return [
        # eight requests decode one token each: latency
        dict(name="plan_8", op="plan", requests=8, page=16, most_cached=32768, new="one"),
        # a large step: single tokens of most requests, prompt chunks of the others
        dict(name="plan_1000", op="plan", requests=1000, page=64, most_cached=20000, new="mixed"),
        # one token's heads of the 24-head model, fp32 activations, into a bf16 cache
        dict(name="append_t1", op="append", type="f32", cache="bf16", rows=1, qh=24, kvh=2, hd=256, n_rot=64, page=64,
             layout="halves", scaling="none", far=32768),
        # a prompt chunk of the same model
        dict(name="append_8192", op="append", type="bf16", cache="bf16", rows=8192, qh=24, kvh=2, hd=256, n_rot=64, page=64,
             layout="halves", scaling="none", far=262144),
        # rows of a model with interleaved pairs whose context was stretched eight times, an odd number of rows
        dict(name="rope_4097", op="rope", type="f16", rows=4097, heads=32, hd=128, n_rot=128, layout="pairs",
             scaling="rotations", far=1000000),
        # one request's next token over 32k cells
        dict(name="attend_t1_32k", op="attend", type="bf16", qh=24, kvh=2, hd=256, page=64, requests=1, new=1, cached=32767,
             spread=0.0, window=0),
        # decode of 64 requests of very different lengths
        dict(name="attend_64", op="attend", type="bf16", qh=32, kvh=8, hd=128, page=16, requests=64, new=1, cached=6000,
             spread=1.0, window=0),
        # verify windows of 4 rows of 16 requests, layers that see the last 4096 cells
        dict(name="attend_verify", op="attend", type="f16", qh=24, kvh=2, hd=256, page=64, requests=16, new=4, cached=9001,
             spread=0.5, window=4096),
        # a prompt's last chunk over what earlier chunks left
        dict(name="attend_chunk", op="attend", type="bf16", qh=24, kvh=2, hd=256, page=64, requests=1, new=2047, cached=30001,
             spread=0.0, window=0),
        # whole prompts of several requests
        dict(name="attend_prompts", op="attend", type="f16", qh=32, kvh=8, hd=128, page=128, requests=4, new=5000, cached=0,
             spread=0.5, window=0),
        # a verify window's rows, filtered as the engine's requests are by default
        dict(name="sample_t4", op="sample", type="f32", rows=4, vocab=151936, filters="k"),
        # a full batch over the whole vocabulary
        dict(name="sample_256", op="sample", type="f32", rows=256, vocab=151936, filters="p"),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "append", "append", "attend", "attend", "attend", "sample", "sample"])
    if op == "plan":
        return dict(op=op, requests=log_int(rng, 1, 1000), page=2 ** rng.randint(4, 8), most_cached=log_int(rng, 1, 20000),
                    new=rng.choice(["one", "few", "mixed"]))
    if op in ("rope", "append"):
        kvh = rng.choice([1, 2, 3, 4, 8])
        case = dict(op=op, type=rng.choice(sorted(TYPES)), rows=log_int(rng, 1, 8000), hd=rng.choice([64, 128, 256]),
                    layout=rng.choice(["halves", "pairs"]), scaling=rng.choice(["none", "linear", "rotations", "index"]),
                    far=log_int(rng, 1000, 1000000))
        case["n_rot"] = rng.choice([case["hd"], case["hd"] // 2, case["hd"] // 4, 2 * rng.randint(1, case["hd"] // 2)])
        if op == "rope":
            return dict(case, heads=rng.randint(1, 24))
        return dict(case, qh=kvh * rng.randint(1, 24 // kvh), kvh=kvh, page=2 ** rng.randint(4, 8),
                    cache=rng.choice(["bf16", "f16"]))
    if op == "sample":
        rows = log_int(rng, 1, 256)
        return dict(op=op, type=rng.choice(sorted(TYPES)), rows=rows, vocab=log_int(rng, 100, 151936),
                    filters=rng.choice(["none", "k", "p", "m", "kpm", "kpm"]))
    kvh, hd = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256])
    case = dict(op=op, type=rng.choice(["bf16", "f16"]), qh=kvh * rng.randint(1, 32 // kvh), kvh=kvh, hd=hd,
                page=2 ** rng.randint(4, 8), requests=log_int(rng, 1, 64), spread=rng.choice([0.0, 0.5, 1.0]),
                window=rng.choice([0, 0, log_int(rng, 1, 8000)]))
    cells = min(250000, 10 ** 9 // (4 * kvh * hd)) // case["requests"]     # cells and pairs stay below the largest's
    case["cached"] = log_int(rng, 1, min(40000, cells))
    pairs = 10 ** 11 // (case["qh"] * hd * case["requests"] * (case["cached"] + 2000))
    case["new"] = rng.choice([1, 1, log_int(rng, 1, 9), log_int(rng, 1, max(2, min(3000, pairs, 20000 // case["requests"])))])
    return case


# ---- inputs ------------------------------------------------------------------------------------------
def lengths(case):
    """cached and new cells of a step's requests: the same lengths for every seed, which decides who has which"""
    R = case["requests"]
    at = [(i + 0.5) / R for i in range(R)]
    if case["op"] == "plan":
        few, many = [i % 9 for i in range(R)], [1 if i % 4 else int(500.0 ** u) for i, u in enumerate(at)]
        return [int(u * u * (case["most_cached"] + 0.999)) for u in at], {"one": [1] * R, "few": few, "mixed": many}[case["new"]]
    like = [math.exp(case["spread"] * (statistics.NormalDist().inv_cdf(u) - case["spread"] / 2)) for u in at]
    new = [max(1, round(case["new"] * v)) for v in like] if case["new"] > 8 else [case["new"]] * R
    return [round(case["cached"] * v) for v in like], new


class Gen:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, mean=0.0, sd=1.0):
        return torch.empty(shape, device=DEV).normal_(mean, sd, generator=self.g)

    def uniform(self, *shape):
        return torch.rand(shape, device=DEV, generator=self.g)

    def ints(self, lo, hi, *shape):
        """lo .. hi inclusive"""
        return torch.randint(lo, hi + 1, shape, device=DEV, generator=self.g, dtype=torch.int32)

    def perm(self, n):
        return torch.randperm(n, device=DEV, generator=self.g).int()


def int32(*shape):
    return torch.zeros(shape, device=DEV, dtype=torch.int32)


def stretched(case):
    """how a rotary table is made: theta, scaling and its numbers (the context was trained to 1/8 of the farthest)"""
    return dict(theta=THETA, factor=1.0 if case["scaling"] == "none" else 8.0, ctx=max(case["far"] // 8, 64), low=1.0, high=32.0,
                amplitude=1.0 if case["scaling"] in ("none", "linear") else 0.1 * math.log(8.0) + 1.0)


def prepare(case, seed):
    g, op = Gen(seed), case["op"]
    s = dict(case=case)
    if op == "plan":
        R, P = case["requests"], case["page"]
        s["n_cached"], s["n_new"] = (torch.tensor(v, device=DEV, dtype=torch.int32)[g.perm(R).long()] for v in lengths(case))
        held = -(-s["n_cached"] // P)
        s["max_pages"] = -(-(case["most_cached"] + 512) // P)
        need = int((-(-(s["n_cached"] + s["n_new"]) // P) - held).sum())
        s["max_tokens"] = max(1, int(s["n_new"].sum()))
        n_pages = int(held.sum()) + need + need // 8 + 4
        ids = g.perm(n_pages)
        s["table"] = torch.full((R, s["max_pages"]), -1, device=DEV, dtype=torch.int32)
        at = torch.arange(s["max_pages"], device=DEV)[None, :] < held[:, None]
        s["table"][at] = ids[:int(held.sum())]
        s["n_pages"], s["free"] = n_pages, ids.clone()
        s["free"][:n_pages - int(held.sum())] = ids[int(held.sum()):]
        s["n_free"] = torch.full((1,), n_pages - int(held.sum()), device=DEV, dtype=torch.int32)
        return s
    if op in ("rope", "append"):
        rows, hd, t = case["rows"], case["hd"], TYPES[case["type"]]
        s["rope"] = stretched(case)
        # stretches of neighbouring positions, as requests have them
        s["positions"] = ((torch.arange(rows, device=DEV) + int(g.ints(0, case["far"] - 1, 1))) % case["far"]).int()
        if op == "rope":
            s["x"] = g.normal(rows, case["heads"], hd).to(t)
            s["out"] = torch.empty_like(s["x"])
            return s
        qh, kvh, P = case["qh"], case["kvh"], case["page"]
        row = g.normal(rows, qh + 2 * kvh, hd).to(t)        # one projection's row: queries, keys, values
        s["q"], s["k"], s["v"] = row[:, :qh], row[:, qh:qh + kvh], row[:, qh + kvh:]
        n_pages = rows // P + 8
        pages = g.perm(n_pages)
        cell = torch.arange(rows, device=DEV) + P // 2      # the first page is half full
        s["slots"] = pages[cell // P] * P + (cell % P).int()
        ct = TYPES[case["cache"]]
        s["kc"], s["vc"] = (g.normal(n_pages, P, kvh, hd).to(ct) for _ in range(2))
        s["q_out"] = torch.empty(rows, qh, hd, device=DEV, dtype=ct)
        return s
    if op == "attend":
        R, P, t = case["requests"], case["page"], TYPES[case["type"]]
        qh, kvh, hd = case["qh"], case["kvh"], case["hd"]
        cached, new = ([v[i] for i in g.perm(R).tolist()] for v in lengths(case))
        s["cached"], s["new"] = cached, new
        s["n_cached"], s["n_new"] = (torch.tensor(v, device=DEV, dtype=torch.int32) for v in (cached, new))
        held = [-(-(c + n) // P) for c, n in zip(cached, new)]
        n_pages = sum(held) + 3
        s["max_pages"], s["n_pages"], s["max_tokens"] = max(held) + 1, n_pages, sum(new)
        s["table"] = torch.full((R, s["max_pages"]), -1, device=DEV, dtype=torch.int32)
        ids, at, taken = g.perm(n_pages), 0, []             # pages of new tokens are the pool's next
        for r, h in enumerate(held):
            s["table"][r, :h] = ids[at:at + h]
            taken.append(ids[at - (-cached[r] // P):at + h])
            at += h
        taken = torch.cat(taken + [ids[:0]]).flip(0)
        s["free"] = torch.cat([taken, ids[:n_pages - len(taken)]])
        s["n_free"] = torch.full((1,), len(taken), device=DEV, dtype=torch.int32)
        s["kc"], s["vc"] = (torch.empty(n_pages, P, kvh, hd, device=DEV, dtype=t) for _ in range(2))
        for a in range(0, n_pages, 8192):                   # cells of different size, channels with a mean
            part = s["kc"][a:a + 8192]
            part.copy_(g.normal(*part.shape) * torch.exp(g.normal(part.shape[0], P, 1, 1, sd=0.3)))
            s["vc"][a:a + 8192].copy_(g.normal(*part.shape) + g.normal(1, 1, kvh, hd, sd=0.5))
        s["q"] = g.normal(s["max_tokens"], qh, hd, sd=1.5).to(t)
        s["out"] = torch.empty_like(s["q"])
        return s
    rows, vocab, f = case["rows"], case["vocab"], case["filters"]
    logits = g.normal(rows, vocab, sd=2.5)
    for _ in range(3):                                      # a few likely tokens
        at = torch.randint(0, vocab, (rows, 1), device=DEV, generator=g.g)
        logits.scatter_(1, at, g.normal(rows, 1, mean=11.0, sd=1.5))
    s["logits"] = logits.to(TYPES[case["type"]])
    s["temp"] = 0.3 + 0.9 * g.uniform(rows)
    s["top_k"] = g.ints(1, 100, rows) if "k" in f else None
    s["top_p"] = 0.5 + 0.48 * g.uniform(rows) if "p" in f else None
    s["min_p"] = 0.1 * g.uniform(rows) if "m" in f else None
    s["u"] = g.uniform(rows)
    s["ids"], s["probs"] = int32(rows), torch.zeros(rows, device=DEV)
    return s


# ---- the plain form ----------------------------------------------------------------------------------
def angles(rope, scaling, n_rot, positions):
    """[rows, n_rot / 2] in 64 bits"""
    i = torch.arange(n_rot // 2, device=DEV, dtype=torch.float64)
    f = rope["theta"] ** (-2.0 * i / n_rot)
    if scaling == "linear":
        f = f / rope["factor"]
    elif scaling != "none":
        if scaling == "rotations":                          # rotations of a pair over the trained context
            keep = (rope["ctx"] * f / (2 * math.pi) - rope["low"]) / (rope["high"] - rope["low"])
        else:                                               # the same ends as pair numbers
            at = [n_rot * math.log(rope["ctx"] / (2 * math.pi * b)) / (2 * math.log(rope["theta"])) for b in (rope["high"], rope["low"])]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n_rot - 1)
            keep = 1 - (i - lo) / max(hi - lo, 0.001)
        keep = keep.clamp(0, 1)
        f = keep * f + (1 - keep) * f / rope["factor"]
    return positions.double()[:, None] * f


def rotate(x, rope, case, positions, dtype=torch.float32):
    """x [rows, heads, hd] with its first n_rot columns rotated"""
    n, a = case["n_rot"], angles(rope, case["scaling"], case["n_rot"], positions)
    c, s = ((f(a) * rope["amplitude"]).to(dtype)[:, None, :] for f in (torch.cos, torch.sin))
    x = x.to(dtype)
    if case["layout"] == "halves":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., n:]], -1)


def plain_plan(s):
    P, n_cached, n_new = s["case"]["page"], s["n_cached"].long(), s["n_new"].long()
    held, total = -(-n_cached // P), -(-(n_cached + n_new) // P)
    need = total - held
    before = need.cumsum(0) - need
    table, columns = s["table"].clone(), torch.arange(s["max_pages"], device=DEV)[None, :]
    order = s["n_free"].long() - 1 - before[:, None] - (columns - held[:, None])
    table = torch.where((columns >= held[:, None]) & (columns < total[:, None]), s["free"][order.clamp(0, s["n_pages"] - 1)], table)
    q_start = torch.cat([torch.zeros(1, device=DEV, dtype=torch.int64), n_new.cumsum(0)])
    t = torch.arange(s["max_tokens"], device=DEV)
    r = torch.searchsorted(q_start[1:], t, right=True).clamp_max(len(n_new) - 1)
    live = t < q_start[-1]
    position = torch.where(live, n_cached[r] + t - q_start[r], 0)
    slots = torch.where(live, table[r, position // P] * P + position % P, -1)
    return dict(table=table, q_start=q_start.int(), kv_len=(n_cached + n_new).int(), served=torch.ones_like(s["n_new"]),
                positions=position.int(), slots=slots.int(), n_free=s["n_free"] - need.sum().int())


def plain_attend(s):
    c, out, at = s["case"], [], 0
    qh, kvh, hd, P = c["qh"], c["kvh"], c["hd"], c["page"]
    for r, (cached, new) in enumerate(zip(s["cached"], s["new"])):
        n = cached + new
        pages = s["table"][r, :-(-n // P)].long()
        k, v = (x[pages].flatten(0, 1)[:n].float().permute(1, 0, 2).contiguous() for x in (s["kc"], s["vc"]))
        q = s["q"][at:at + new].float().view(new, kvh, qh // kvh, hd).permute(1, 2, 0, 3).reshape(kvh, -1, hd)
        p = torch.bmm(q, k.transpose(1, 2).contiguous()).view(kvh, qh // kvh, new, n) * hd ** -0.5
        behind = torch.arange(cached, n, device=DEV)[:, None] - torch.arange(n, device=DEV)[None, :]
        hidden = behind < 0
        if c["window"]:
            hidden |= behind >= c["window"]
        p = p.masked_fill_(hidden, float("-inf"))
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out.append(torch.bmm(p.view(kvh, -1, n), v).view(kvh, qh // kvh, new, hd).permute(2, 0, 1, 3).reshape(new, qh, hd).to(s["q"].dtype))
        at += new
    return dict(out=torch.cat(out))


def plain_sample(s):
    v, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    w = torch.exp((v.double() - v[:, :1].double()) / s["temp"].double()[:, None])
    rank = torch.arange(v.shape[1], device=DEV)[None, :]
    if s["top_k"] is not None:
        w = torch.where(rank < s["top_k"][:, None], w, 0.0)
    cum = w.cumsum(1)
    keep = w > 0
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
    if s["top_p"] is not None:
        keep &= cum - w < s["top_p"].double()[:, None] * cum[:, -1:]
    w = torch.where(keep, w, 0.0)
    cum = w.cumsum(1)
    at = (cum < s["u"].double()[:, None] * cum[:, -1:]).sum(1, keepdim=True)
    at = torch.minimum(at, keep.sum(1, keepdim=True) - 1)
    return dict(ids=order.gather(1, at)[:, 0].int(), probs=(w.gather(1, at) / cum[:, -1:])[:, 0].float())


def plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "plan":
        return plain_plan(s)
    if op == "rope":
        return dict(out=rotate(s["x"], s["rope"], c, s["positions"]).to(s["x"].dtype))
    if op == "append":
        q, k = (rotate(s[n], s["rope"], c, s["positions"]).to(s["kc"].dtype) for n in "qk")
        at = s["slots"].long()
        s["kc"].flatten(0, 1)[at] = k
        s["vc"].flatten(0, 1)[at] = s["v"].to(s["vc"].dtype)
        return dict(q=q, k=s["kc"], v=s["vc"])
    return plain_attend(s) if op == "attend" else plain_sample(s)


# ---- the library's calls -------------------------------------------------------------------------------
def library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wzy-flash-serve_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import wzy_amd
    return wzy_amd


def calls(s):
    """the calls of one pass with their arguments, and what they leave: a serving program keeps these structures"""
    W = library()
    lib, c, op = W.lib(), s["case"], s["case"]["op"]
    types = {torch.float32: W.TYPE_F32, torch.bfloat16: W.TYPE_BF16, torch.float16: W.TYPE_F16}
    st = torch.cuda.current_stream().cuda_stream or None

    def at(t):
        return None if t is None else t.data_ptr()

    def heads(t):
        return W.Heads(t.data_ptr(), t.stride(0), t.stride(1))

    def batch(requests):
        s["q_start"], s["kv_len"], s["served"] = int32(requests + 1), int32(requests), int32(requests)
        s["row_positions"], s["row_slots"] = int32(s["max_tokens"]), int32(s["max_tokens"])
        return W.PagedBatch(requests, s["max_tokens"], s["max_pages"], at(s["n_cached"]), at(s["n_new"]), at(s["table"]),
                            at(s["q_start"]), at(s["kv_len"]), at(s["served"]), at(s["row_positions"]), at(s["row_slots"]),
                            max(lengths(c)[1]))

    def work(b, qh, kvh, hd, window):
        w = W.PagedWork(qh, kvh, hd, window, None, 0)
        w.bytes = lib.wzy_paged_work_bytes(C.byref(b), C.byref(w))
        s["work"] = torch.empty(w.bytes, device=DEV, dtype=torch.uint8)
        w.items = at(s["work"])
        return w

    def cache():
        return W.PagedCache(at(s["kc"]), at(s["vc"]), s["kc"].stride(0), s["kc"].stride(1), s["kc"].stride(2), s["kc"].shape[0],
                            c["page"], c["kvh"], c["hd"], types[s["kc"].dtype])

    if op == "plan":
        s["left"] = int32(1)
        pool = W.PagedPool(at(s["free"]), at(s["n_free"]), at(s["left"]), s["n_pages"], c["page"])
        b = batch(c["requests"])
        w = work(b, 24, 2, 256, 0)                          # the step's attention layers are all alike
        out = dict(table=s["table"], q_start=s["q_start"], kv_len=s["kv_len"], served=s["served"], positions=s["row_positions"],
                   slots=s["row_slots"], n_free=s["left"])
        return [(lib.wzy_paged_plan, (C.byref(pool), C.byref(b), C.byref(w), 1, st))], out, (pool, b, w)
    if op in ("rope", "append"):
        m = s["rope"]
        kind = dict(none=W.ROPE_PLAIN, linear=W.ROPE_LINEAR, rotations=W.ROPE_ROTATIONS, index=W.ROPE_INDEX)[c["scaling"]]
        cfg = W.RopeCfg(m["theta"], m["factor"], m["low"], m["high"], m["amplitude"], m["ctx"], c["n_rot"], kind)
        s["freqs"] = torch.empty(c["n_rot"] // 2 + 1, device=DEV, dtype=torch.float64)
        lib.wzy_rope_freqs(C.byref(cfg), at(s["freqs"]), st)
        r = W.RopeTab(at(s["freqs"]), c["n_rot"], W.ROPE_PAIRS if c["layout"] == "pairs" else W.ROPE_HALVES)
        if op == "rope":
            x, y = heads(s["x"]), heads(s["out"])
            todo = [(lib.wzy_rope, (C.byref(r), C.byref(x), types[s["x"].dtype], c["rows"], c["heads"], c["hd"], at(s["positions"]),
                                    C.byref(y), st))]
            return todo, dict(out=s["out"]), (r, x, y)
        kv, q, k, v, qo = cache(), heads(s["q"]), heads(s["k"]), heads(s["v"]), heads(s["q_out"])
        todo = [(lib.wzy_paged_append, (C.byref(kv), C.byref(r), C.byref(q), c["qh"], C.byref(qo), C.byref(k), C.byref(v),
                                        types[s["q"].dtype], c["rows"], at(s["positions"]), at(s["slots"]), st))]
        return todo, dict(q=s["q_out"], k=s["kc"], v=s["vc"]), (r, kv, q, k, v, qo)
    if op == "attend":
        s["left"] = int32(1)                                # the step's plan serves all its layers
        pool = W.PagedPool(at(s["free"]), at(s["n_free"]), at(s["left"]), s["n_pages"], c["page"])
        b = batch(c["requests"])
        w = work(b, c["qh"], c["kvh"], c["hd"], c["window"])
        lib.wzy_paged_plan(C.byref(pool), C.byref(b), C.byref(w), 1, st)
        kv, q, o = cache(), heads(s["q"]), heads(s["out"])
        n = lib.wzy_paged_attend_workspace_bytes(C.byref(b), C.byref(w))
        s["space"] = torch.empty(n, device=DEV, dtype=torch.uint8)
        todo = [(lib.wzy_paged_attend, (C.byref(kv), C.byref(b), C.byref(w), C.byref(q), C.byref(o), c["hd"] ** -0.5, at(s["space"]), n,
                                        st))]
        return todo, dict(out=s["out"]), (pool, b, w, kv, q, o)
    n = lib.wzy_sample_workspace_bytes(c["rows"], c["vocab"])
    s["space"] = torch.empty(n, device=DEV, dtype=torch.uint8)
    todo = [(lib.wzy_sample, (at(s["logits"]), types[s["logits"].dtype], s["logits"].stride(0), c["rows"], c["vocab"], at(s["temp"]),
                              at(s["top_k"]), at(s["top_p"]), at(s["min_p"]), at(s["u"]), at(s["ids"]), at(s["probs"]),
                              at(s["space"]), n, st))]
    return todo, dict(ids=s["ids"], probs=s["probs"]), None


def run(state):
    if not own:
        return plain(state)
    if "calls" not in state:
        state["calls"] = calls(state)
    for fn, args in state["calls"][0]:
        fn(*args)
    return state["calls"][1]


# ---- work and exact values -----------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "plan":
        new = sum(lengths(case)[1])
        return dict(bytes=new * (8 + 8 / case["page"]) + 20 * case["requests"], flops=0)
    if op == "rope":
        n = case["rows"] * case["heads"] * case["hd"]
        return dict(bytes=2 * n * TYPES[case["type"]].itemsize + 4 * case["rows"], flops=0)
    if op == "append":
        n = case["rows"] * (case["qh"] + 2 * case["kvh"]) * case["hd"]
        return dict(bytes=n * (TYPES[case["type"]].itemsize + 2) + 8 * case["rows"], flops=0)
    if op == "attend":
        (cached, new), hd, most = lengths(case), case["hd"], case["window"] or 10 ** 9
        cells = sum(min(c + n, most + n) for c, n in zip(cached, new))
        pairs = sum(n * sum(min(c + (n + 1) / 2, most) for c in cached) / len(cached) for n in new)     # whoever has which
        return dict(bytes=4 * hd * (case["kvh"] * cells + case["qh"] * sum(new)), flops=4 * pairs * case["qh"] * hd)
    return dict(bytes=case["rows"] * case["vocab"] * TYPES[case["type"]].itemsize, flops=0)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "plan":
        return exact_plan(s)
    if op == "attend":
        return exact_attend(s)
    if op == "sample":
        return exact_sample(s)
    n, m = case["n_rot"], s["rope"]

    def turned(x):
        """as a product of complex numbers"""
        f = []
        for i in range(n // 2):
            base = m["theta"] ** (-2.0 * i / n)
            keep = {"none": 1.0, "linear": 0.0}.get(case["scaling"])
            if keep is None and case["scaling"] == "rotations":
                keep = (m["ctx"] / (2 * math.pi / base) - m["low"]) / (m["high"] - m["low"])
            elif keep is None:
                first, last = (math.log(m["ctx"] / (b * 2 * math.pi)) / math.log(m["theta"]) * n / 2 for b in (m["high"], m["low"]))
                first, last = max(math.floor(first), 0), min(math.ceil(last), n - 1)
                keep = (last - i) / (last - first) if last > first else float(i <= first)
            keep = min(max(keep, 0.0), 1.0)
            f.append(base * (keep + (1.0 - keep) / m["factor"]))
        a = s["positions"].double()[:, None] * torch.tensor(f, device=DEV, dtype=torch.float64)
        z = torch.polar(torch.full_like(a, m["amplitude"]), a)[:, None, :]
        y = x.double().clone()
        first, second = (slice(0, n // 2), slice(n // 2, n)) if case["layout"] == "halves" else (slice(0, n, 2), slice(1, n, 2))
        r = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z
        y[..., first], y[..., second] = r.real, r.imag
        return y
    if op == "rope":
        return dict(out=turned(s["x"]))
    kc, vc = s["kc"].double(), s["vc"].double()
    page, cell = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    kc[page, cell], vc[page, cell] = turned(s["k"]), s["v"].double()
    return dict(q=turned(s["q"]), k=kc, v=vc)


def exact_plan(s):
    """one request after another, on the host"""
    P, table, free = s["case"]["page"], s["table"].tolist(), s["free"].tolist()[:int(s["n_free"])]
    q_start, kv_len, positions, slots = [0], [], [], []
    for r, (c, n) in enumerate(zip(s["n_cached"].tolist(), s["n_new"].tolist())):
        for p in range(c, c + n):
            if p % P == 0:
                table[r][p // P] = free.pop()
            positions.append(p)
            slots.append(table[r][p // P] * P + p % P)
        q_start.append(q_start[-1] + n)
        kv_len.append(c + n)
    pad = s["max_tokens"] - len(slots)

    def ints(v):
        return torch.tensor(v, device=DEV, dtype=torch.int32)
    return dict(table=ints(table), q_start=ints(q_start), kv_len=ints(kv_len), served=ints([1] * len(kv_len)),
                positions=ints(positions + [0] * pad), slots=ints(slots + [-1] * pad), n_free=ints([len(free)]))


def exact_attend(s):
    c = s["case"]
    group, out, at = c["qh"] // c["kvh"], torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64), 0
    for r, (cached, new) in enumerate(zip(s["cached"], s["new"])):
        cell = torch.arange(cached + new, device=DEV)
        page = s["table"][r].long()[cell // c["page"]]
        for h in range(c["qh"]):
            k, v = (x[page, cell % c["page"], h // group].double() for x in (s["kc"], s["vc"]))
            for a in range(0, new, 1024):
                b = min(a + 1024, new)
                position = torch.arange(cached + a, cached + b, device=DEV)[:, None]
                seen = (cell <= position) & ((position - cell < c["window"]) if c["window"] else True)
                x = s["q"][at + a:at + b, h].double() @ k.T / math.sqrt(c["hd"])
                out[at + a:at + b, h] = torch.softmax(torch.where(seen, x, -math.inf), 1) @ v
        at += new
    return dict(out=out)


def exact_sample(s):
    """rank by rank: cuts as ranks, the draw by a search in the sums"""
    x = s["logits"].double()
    ids, probs = [], []
    for r in range(x.shape[0]):
        order = torch.argsort(-x[r], stable=True)
        n = int(s["top_k"][r]) if s["top_k"] is not None else x.shape[1]
        order = order[:min(n, x.shape[1])]
        w = torch.exp((x[r][order] - x[r].max()) / float(s["temp"][r]))
        total = w.cumsum(0)
        n = len(w)
        if s["min_p"] is not None:
            n = int((w >= float(s["min_p"][r])).sum())
        if s["top_p"] is not None:
            n = min(n, int(torch.searchsorted(total, float(s["top_p"][r]) * total[-1])) + 1)
        i = min(int(torch.searchsorted(total[:n].contiguous(), float(s["u"][r]) * total[n - 1])), n - 1)
        ids.append(order[i])
        probs.append(w[i] / total[n - 1])
    return dict(ids=torch.stack(ids).int(), probs=torch.stack(probs))
