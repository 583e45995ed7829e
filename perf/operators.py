"""Measured cases of the microscaled (MX) operators: 4- and 8-bit rows with one power-of-two scale per 32 values.

The operators, as a program that serves a model with this library calls them:

  quant    rows to MX codes and scales: activations to 8 bits (e4m3), weights or activations to 4 bits (e2m1;
           4-bit codes come back as the values they stand for, through the inverse operator)
  norm     residual addition and root-mean-square norm: the new residual rows, the normed rows and their 8-bit form
  swiglu   silu(gate) * up to 8 bits, between an expert's two products
  gemm     MX activations by 4-bit MX weights: the decode form (a few rows) and prefill chunks
  grouped  the same with one weight matrix per expert and ragged groups of rows, gathered by token

With `own` false the operators run in plain torch arithmetic, with `own` true through the library's C ABI.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
EMAX = {"e2m1": 2, "e4m3": 8}


def listed():
    return [
        # a verify window's rows on their way into a product: latency
        dict(name="quant_e4m3_t4", op="quant", fmt="e4m3", type="f32", rows=4, cols=2048, pad=0),
        # an LM head's weights at load time, out and back: 311 M values
        dict(name="quant_e2m1_head", op="quant", fmt="e2m1", type="bf16", rows=151936, cols=2048, pad=0),
        # one decoded token between two half-layers
        dict(name="norm_t1", op="norm", type="bf16", rows=1, cols=2048, pad=0, res=True),
        # a prefill chunk of the wide model, one row short
        dict(name="norm_8191", op="norm", type="bf16", rows=8191, cols=2560, pad=0, res=True),
        # four tokens' ten experts each
        dict(name="swiglu_t4", op="swiglu", type="f32", rows=40, cols=512, pad=0),
        # a prefill chunk's expert entries
        dict(name="swiglu_81920", op="swiglu", type="bf16", rows=81920, cols=512, pad=0),
        # one decoded token through the sparse-attention query projection
        dict(name="gemm_t1", op="gemm", fmt="e4m3", M=1, N=12288, K=2048, out="f32"),
        # a verify window through the LM head
        dict(name="gemm_head_t4", op="gemm", fmt="e4m3", M=4, N=151936, K=2048, out="f32"),
        # a short prompt through the attention output projection
        dict(name="gemm_250", op="gemm", fmt="e4m3", M=250, N=2048, K=6144, out="bf16"),
        # a prefill chunk through the delta-rule input projection, activations in 4 bits
        dict(name="gemm_8192", op="gemm", fmt="e2m1", M=8192, N=6144, K=2048, out="bf16"),
        # gate and up of the experts of a verify window: most groups empty, the others of one or two rows
        dict(name="grouped_t4", op="grouped", fmt="e4m3", tokens=4, top_k=10, groups=512, N=1024, K=2048, out="f32"),
        # gate and up of a prefill chunk: about 160 rows an expert
        dict(name="grouped_8192", op="grouped", fmt="e4m3", tokens=8192, top_k=10, groups=512, N=1024, K=2048, out="bf16"),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "norm", "swiglu", "gemm", "gemm", "gemm", "grouped", "grouped"])
    kind, fmt = rng.choice(sorted(TYPES)), rng.choice(["e2m1", "e4m3"])
    if op in ("quant", "norm", "swiglu"):
        cols = 32 * log_int(rng, 1, 256)
        rows = log_int(rng, 1, min(100000, 40000000 // cols))
        case = dict(op=op, type=kind, rows=rows, cols=cols, pad=rng.choice([0, 0, 8, 40, 512]))
        if op == "quant":
            case["fmt"] = fmt
        if op == "norm":
            case["res"] = rng.random() < 0.75
        return case
    if op == "gemm":
        M, K = log_int(rng, 1, 12000), 32 * log_int(rng, 1, 256)
        N = log_int(rng, 1, max(1, min(160000, 10 ** 11 // (M * K), 50000000 // M)))
        return dict(op=op, fmt=fmt, M=M, N=N, K=K, out=kind)
    groups = log_int(rng, 1, 512)
    top_k, K, N = rng.randint(1, min(12, groups)), 32 * log_int(rng, 4, 80), log_int(rng, 100, 2560)
    tokens = log_int(rng, 1, 8192)
    return dict(op=op, fmt=fmt, tokens=tokens, top_k=top_k, groups=groups, N=N, K=K, out=kind)


# ---- the plain form ----------------------------------------------------------------------------------
def to_mx(v, fmt):
    """[rows, cols] values -> (fp32 element values or e2m1 code numbers, scale bytes)"""
    x = v.float().unflatten(1, (-1, 32))
    top = x.abs().amax(2).view(torch.int32) >> 23            # biased exponent of the block's largest value
    bad = top == 255                                          # a NaN or an infinity: the scale is NaN, the codes 0
    byte = torch.where(bad, 255, (top - EMAX[fmt]).clamp_min(0))
    x = x * ((254 - byte.clamp_max(253)) << 23).view(torch.float32)[..., None]
    x = torch.where(bad[..., None], 0.0, x)
    if fmt == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).flatten(1), byte.to(torch.uint8)
    m = x.abs()                                               # a tie goes to the even code
    code = ((m > 0.25).byte() + (m >= 0.75).byte() + (m > 1.25).byte() + (m >= 1.75).byte() + (m > 2.5).byte()
            + (m >= 3.5).byte() + (m > 5.0).byte())
    return (code | (x.signbit().byte() << 3)).flatten(1), byte.to(torch.uint8)


def from_mx(codes, scales, dtype=torch.float32):
    """what codes (e4m3 values, or e2m1 pairs in bytes) and scale bytes stand for"""
    if codes.dtype == torch.uint8:
        table = torch.tensor(E2M1 + [-t for t in E2M1], device=codes.device, dtype=dtype)
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(1)
        codes = table[codes.int()]
    s = torch.exp2(scales.to(dtype) - 127.0)
    s = torch.where(scales == 255, float("nan"), s)
    return (codes.to(dtype).unflatten(1, (-1, 32)) * s[..., None]).flatten(1)


def pack(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def mx_rows(v, fmt):
    """a stored MX matrix: codes as the library lays them out (bytes of two e2m1, or e4m3) and scale bytes"""
    c, s = to_mx(v, fmt)
    return (pack(c) if fmt == "e2m1" else c), s


def e8m0(scales):
    return scales.view(torch.float8_e8m0fnu)


def plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "quant":
        codes, scales = to_mx(s["x"], c["fmt"])
        if c["fmt"] == "e4m3":
            return dict(codes=codes, scales=e8m0(scales))
        return dict(values=from_mx(pack(codes), scales).to(torch.bfloat16), scales=e8m0(scales))
    if op == "norm":
        h = s["x"].float() if s["res"] is None else s["x"].float() + s["res"].float()
        h = h.to(s["x"].dtype)
        v = h.float()
        v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * s["gamma"]
        codes, scales = to_mx(v, "e4m3")
        return dict(sum=h, y=v.to(h.dtype), codes=codes, scales=e8m0(scales))
    if op == "swiglu":
        g, u = s["x"][:, :c["cols"]].float(), s["x"][:, c["cols"]:2 * c["cols"]].float()
        codes, scales = to_mx(g * u / (1.0 + torch.exp(-g)), "e4m3")
        return dict(codes=codes, scales=e8m0(scales))
    if op == "gemm":
        return dict(y=(from_mx(*s["a"]) @ from_mx(*s["w"]).T).to(s["y"].dtype))
    # every group's rows in a slot of their own, padded to the largest group
    G, N, K = c["groups"], c["N"], c["K"]
    a = from_mx(*s["a"])[s["row_ids"].long()]
    off = s["offsets"].long()
    e = torch.arange(a.shape[0], device=DEV)
    g = torch.searchsorted(off[1:], e, right=True)
    slots = torch.zeros(G, s["largest"], K, device=DEV)
    slots[g, e - off[g]] = a
    y = torch.bmm(slots, from_mx(*s["w"]).view(G, N, K).transpose(1, 2).contiguous())
    return dict(y=y[g, e - off[g]].to(s["y"].dtype))


# ---- inputs ------------------------------------------------------------------------------------------
class Gen:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, mean=0.0, sd=1.0):
        return torch.empty(shape, device=DEV).normal_(mean, sd, generator=self.g)

    def rows(self, rows, cols):
        """activations: N(0, 1) with a few channels ten times as large, rows of different size"""
        x = self.normal(rows, cols)
        x[:, torch.randperm(cols, device=DEV, generator=self.g)[:max(1, cols // 256)]] *= 10.0
        return x.mul_(torch.exp(self.normal(rows, 1, sd=0.5)))


def prepare(case, seed):
    g, op = Gen(seed), case["op"]
    u8 = dict(device=DEV, dtype=torch.uint8)
    s = dict(case=case)
    if op in ("quant", "norm", "swiglu"):
        rows, cols, t = case["rows"], case["cols"], TYPES[case["type"]]
        ld = cols * (2 if op == "swiglu" else 1) + case["pad"]
        wide = (g.normal(rows, ld, sd=cols ** -0.5) if case.get("fmt") == "e2m1" else g.rows(rows, ld)).to(t)
        s["x"] = wide[:, :ld - case["pad"]]
        per = 2 if case.get("fmt") == "e2m1" else 1
        s["codes"] = torch.empty(rows, cols // per, **u8)
        s["scales"] = torch.empty(rows, cols // 32, **u8)
        if op == "quant" and per == 2:
            s["values"] = torch.empty(rows, cols, device=DEV, dtype=torch.bfloat16)
        if op == "norm":
            s["res"] = g.rows(rows, ld).to(t)[:, :cols] if case["res"] else None
            s["gamma"] = g.normal(cols, mean=1.0, sd=0.1)
            s["sum"], s["y"] = (torch.empty(rows, ld, device=DEV, dtype=t)[:, :cols] for _ in range(2))
        return s
    N, K = case["N"], case["K"]
    if op == "gemm":
        M = case["M"]
        s["a"] = mx_rows(g.rows(M, K), case["fmt"])
        s["w"] = mx_rows(g.normal(N, K, sd=K ** -0.5), "e2m1")
    else:
        # tokens choose top_k different experts; some experts are chosen more often
        T, G, k = case["tokens"], case["groups"], case["top_k"]
        like = torch.exp(g.normal(G, sd=0.5))
        ids = torch.multinomial(like.expand(T, G), k, generator=g.g).flatten()
        order = torch.argsort(ids, stable=True)
        counts = torch.bincount(ids, minlength=G)
        s["row_ids"] = (order // k).int()
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), counts.cumsum(0)]).int()
        s["largest"] = int(counts.max())
        s["live"] = int((counts > 0).sum())
        M = T * k
        s["a"] = mx_rows(g.rows(T, K), case["fmt"])
        s["w"] = mx_rows(g.normal(G * N, K, sd=K ** -0.5), "e2m1")
    s["y"] = torch.empty(M, N, device=DEV, dtype=TYPES[case["out"]])
    return s


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

    def mat(codes, scales, fmt):
        return W.MxMat(codes.data_ptr(), scales.data_ptr(), 0, 0, W.MX_E2M1 if fmt == "e2m1" else W.MX_E4M3)

    def at(t):
        return None if t is None else t.data_ptr()

    if op in ("quant", "norm", "swiglu"):
        x, rows, cols = s["x"], c["rows"], c["cols"]
        q, t, ld = mat(s["codes"], s["scales"], c.get("fmt", "e4m3")), types[x.dtype], x.stride(0)
        out = dict(codes=s["codes"].view(torch.float8_e4m3fn), scales=e8m0(s["scales"]))
        if op == "norm":
            out.update(sum=s["sum"], y=s["y"])
            todo = [(lib.wzy_mx_add_rmsnorm, (at(x), at(s["res"]), t, ld, at(s["gamma"]), EPS, rows, cols, at(s["sum"]),
                                              at(s["y"]), C.byref(q), st))]
        elif op == "swiglu":
            todo = [(lib.wzy_mx_swiglu, (at(x), at(x) + cols * x.element_size(), t, ld, rows, cols, C.byref(q), st))]
        else:
            todo = [(lib.wzy_mx_quantize, (at(x), t, ld, rows, cols, C.byref(q), st))]
            if c["fmt"] == "e2m1":
                out = dict(values=s["values"], scales=e8m0(s["scales"]))
                todo.append((lib.wzy_mx_dequantize, (C.byref(q), rows, cols, at(s["values"]), W.TYPE_BF16, cols, st)))
        return todo, out, q
    a, w, y = mat(*s["a"], c["fmt"]), mat(*s["w"], "e2m1"), s["y"]
    if op == "gemm":
        todo = [(lib.wzy_mx_gemm, (C.byref(a), C.byref(w), c["M"], c["N"], c["K"], at(y), types[y.dtype], c["N"], st))]
    else:
        todo = [(lib.wzy_mx_grouped_gemm, (C.byref(a), c["tokens"], at(s["row_ids"]), C.byref(w), at(s["offsets"]),
                                           c["groups"], y.shape[0], c["N"], c["K"], at(y), types[y.dtype], c["N"], st))]
    return todo, dict(y=y), (a, w)


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
    if op in ("quant", "norm", "swiglu"):
        n, size = case["rows"] * case["cols"], TYPES[case["type"]].itemsize
        if op == "quant":
            return dict(bytes=n * (size + 1 / 32 + (2.5 if case["fmt"] == "e2m1" else 1)), flops=0)
        if op == "swiglu":
            return dict(bytes=n * (2 * size + 1 + 1 / 32), flops=0)
        return dict(bytes=n * (size * (4 if case["res"] else 3) + 1 + 1 / 32) + 4 * case["cols"], flops=0)
    N, K, out = case["N"], case["K"], TYPES[case["out"]].itemsize
    a, w = K * ((1 if case["fmt"] == "e4m3" else 0.5) + 1 / 32), N * K * (0.5 + 1 / 32)
    if op == "gemm":
        M = case["M"]
        return dict(bytes=M * a + w + M * N * out, flops=2 * M * N * K)
    T, G, M = case["tokens"], case["groups"], case["tokens"] * case["top_k"]
    live = G * (1 - (1 - case["top_k"] / G) ** T)             # groups that have entries, where all are alike
    return dict(bytes=T * a + live * w + M * N * out + 4 * (M + G + 1), flops=2 * M * N * K)


def exact_mx(v, fmt):
    """elements and scales of float64 rows: the exponent by frexp, the element rounded on its own grid"""
    x = v.unflatten(1, (-1, 32))
    amax = x.abs().amax(2)
    low = torch.full_like(amax, -127.0)
    e = torch.where(amax > 0, torch.frexp(amax)[1].double() - 1 - EMAX[fmt], low).clamp_min(-127.0)
    x = torch.ldexp(x, -e[..., None])
    first, bits, most = (0, 1, 6.0) if fmt == "e2m1" else (-6, 3, 448.0)
    step = torch.exp2((torch.frexp(x)[1].double() - 1).clamp_min(first) - bits)
    return ((x / step).round() * step).clamp(-most, most).flatten(1), e


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("quant", "norm", "swiglu"):
        if case["rows"] * case["cols"] > 4e8:
            return None
        x = s["x"].double()
        if op == "quant":
            v, e = exact_mx(x, case["fmt"])
            if case["fmt"] == "e4m3":
                return dict(codes=v, scales=torch.exp2(e))
            return dict(values=(v.unflatten(1, (-1, 32)) * torch.exp2(e)[..., None]).flatten(1), scales=torch.exp2(e))
        if op == "swiglu":
            g, u = x[:, :case["cols"]], x[:, case["cols"]:2 * case["cols"]]
            v, e = exact_mx(g * torch.sigmoid(g) * u, "e4m3")
            return dict(codes=v, scales=torch.exp2(e))
        h = (x if s["res"] is None else x + s["res"].double()).to(s["x"].dtype).double()
        n = h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * s["gamma"].double()
        v, e = exact_mx(n, "e4m3")
        return dict(sum=h, y=n, codes=v, scales=torch.exp2(e))
    a, w = (from_mx(*s[k], dtype=torch.float64) for k in ("a", "w"))
    if op == "gemm":
        return dict(y=a @ w.T)
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device=DEV)
    off, w = s["offsets"].tolist(), w.view(case["groups"], case["N"], case["K"])
    for i in range(case["groups"]):
        if off[i] < off[i + 1]:
            y[off[i]:off[i + 1]] = a[s["row_ids"][off[i]:off[i + 1]].long()] @ w[i].T
    return dict(y=y)
