"""Microscaled (MX) operators on the GPU against plain 64-bit formulations (tests/mx_ref.py)."""
import ctypes as C

import numpy as np
import pytest

import mx_ref as R
import wzy_amd
from mx_ref import BF16, E2M1, E4M3, F16, F32

pytestmark = pytest.mark.gpu
DA = wzy_amd.DeviceArray
FILL = 0xA5


class Mat:
    """An MX matrix on the device, its rows with gaps that must keep their bytes"""

    def __init__(self, rows, cols, fmt, gap=0, sgap=0, codes=None, scales=None):
        self.rows, self.cols, self.fmt = rows, cols, fmt
        self.nb = cols // 2 if fmt == E2M1 else cols
        c = np.full((rows, self.nb + gap), FILL, np.uint8)
        s = np.full((rows, cols // 32 + sgap), FILL, np.uint8)
        if codes is not None:
            c[:, :self.nb], s[:, :cols // 32] = R.pack(codes, fmt), scales
        self.c, self.s = DA.from_numpy(c), DA.from_numpy(s)
        self.m = wzy_amd.MxMat(self.c.ptr, self.s.ptr, self.nb + gap, cols // 32 + sgap, fmt)

    def ref(self):
        return C.byref(self.m)

    def read(self):
        c, s = self.c.numpy(), self.s.numpy()
        assert (c[:, self.nb:] == FILL).all() and (s[:, self.cols // 32:] == FILL).all()
        return R.unpack(c[:, :self.nb], self.fmt), s[:, :self.cols // 32]


def wide(bits, gap):
    """rows with `gap` more elements each, filled with a bit pattern"""
    a = np.zeros((bits.shape[0], bits.shape[1] + gap), bits.dtype)
    a.view(np.uint8)[:] = FILL
    a[:, :bits.shape[1]] = bits
    return a


def out_rows(rows, cols, t, gap=0):
    return DA.from_numpy(wide(np.zeros((rows, cols), np.float32 if t == F32 else np.uint16), gap))


def read_rows(d, cols, t):
    a = d.numpy()
    assert (np.ascontiguousarray(a[:, cols:]).view(np.uint8) == FILL).all()
    return R.values(np.ascontiguousarray(a[:, :cols]), t)


def activations(rng, rows, cols):
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[:, rng.integers(0, cols, max(1, cols // 128))] *= 10
    return x * np.exp(rng.standard_normal((rows, 1)) * 0.5).astype(np.float32)


def borders(fmt):
    """values on and next to every rounding border of a block whose scale is 1, ties among them, and its limits"""
    t = R.element_values(fmt)[:8 if fmt == E2M1 else 127]
    mid = (t[1:] + t[:-1]) / 2
    v = np.concatenate([t, mid, mid * (1 - 2.0 ** -20), mid * (1 + 2.0 ** -20), [R.MOST[fmt] * 1.1]])
    return np.concatenate([v, -v])


def special_rows(fmt, cols):
    """32-value blocks: borders under scale 1 (led by the block's largest), zeros, denormals, the type's ends, NaN, inf"""
    b = borders(fmt)
    lead = 2.0 ** R.EMAX[fmt] * 1.25
    blocks = [np.concatenate([[lead], b[i:i + 31], np.zeros(31)])[:32] for i in range(0, len(b), 31)]
    z = np.zeros(32)

    def one(*at):
        a = z.copy()
        for i, v in at:
            a[i] = v
        return a
    blocks += [z, -z, one((3, 1e-40)), one((3, -1e-38), (9, 2e-45)), one((0, 2.0 ** -126)), one((5, 3.4e38), (6, -1e30)),
               one((31, np.nan)), one((0, np.inf), (1, 1.0)), one((7, -np.inf)), np.full(32, 1.0), np.full(32, 0.75),
               np.full(32, 7.999), np.arange(32) / 31 * 6.5 - 3]
    while len(blocks) % (cols // 32):
        blocks.append(z)
    return np.array(blocks, np.float64).reshape(-1, cols)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols,gap", [(1, 32, 0), (1, 2048, 8), (3, 96, 40), (77, 320, 0), (513, 2560, 16)])
def test_quantize_bit_exact(wz, gpu, fmt, t, rows, cols, gap):
    rng = np.random.default_rng(rows * 7 + cols + t)
    bits, x = R.typed(activations(rng, rows, cols) * 2.0 ** rng.integers(-9, 9, (rows, 1)), t)
    d = DA.from_numpy(wide(bits, gap))
    q = Mat(rows, cols, fmt, gap=16 if gap else 0, sgap=3 if gap else 0)
    wz.wzy_mx_quantize(d.ptr, t, cols + gap, rows, cols, q.ref(), None)
    codes, scales = q.read()
    wc, ws = R.quantize(x, fmt)
    np.testing.assert_array_equal(scales, ws)
    np.testing.assert_array_equal(codes, wc)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_quantize_borders_and_specials(wz, gpu, fmt, t):
    bits, x = R.typed(special_rows(fmt, 96), t)
    rows = x.shape[0]
    d = DA.from_numpy(bits)
    q = Mat(rows, 96, fmt)
    wz.wzy_mx_quantize(d.ptr, t, 96, rows, 96, q.ref(), None)
    codes, scales = q.read()
    wc, ws = R.quantize(x, fmt)
    np.testing.assert_array_equal(scales, ws)
    np.testing.assert_array_equal(codes, wc)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_dequantize_every_code_and_scale(wz, gpu, fmt, t):
    # every code under scale bytes from end to end, NaN among both
    n = 16 if fmt == E2M1 else 256
    scales = np.array([0, 1, 2, 9, 60, 100, 112, 120, 126, 127, 128, 135, 141, 200, 230, 245, 254, 255], np.uint8)
    codes = np.tile(np.arange(n, dtype=np.uint8), (len(scales), 256 // n))
    sc = np.repeat(scales[:, None], 8, 1)
    q = Mat(len(scales), 256, fmt, gap=32, sgap=1, codes=codes, scales=sc)
    y = out_rows(len(scales), 256, t, 8)
    wz.wzy_mx_dequantize(q.ref(), len(scales), 256, y.ptr, t, 264, None)
    got = read_rows(y, 256, t)
    with np.errstate(over="ignore"):
        want = R.typed(R.dequantize(codes, sc, fmt).astype(np.float32), t)[1]
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 2560), (1000, 64)])
def test_dequantize_inverts_quantize(wz, gpu, rows, cols):
    rng = np.random.default_rng(rows)
    for fmt in (E2M1, E4M3):
        x = DA.from_numpy(activations(rng, rows, cols))
        q, y = Mat(rows, cols, fmt), DA(rows * cols, np.float32)
        wz.wzy_mx_quantize(x.ptr, F32, cols, rows, cols, q.ref(), None)
        wz.wzy_mx_dequantize(q.ref(), rows, cols, y.ptr, F32, cols, None)
        q2 = Mat(rows, cols, fmt)
        wz.wzy_mx_quantize(y.ptr, F32, cols, rows, cols, q2.ref(), None)       # a fixed point
        np.testing.assert_array_equal(y.numpy().reshape(rows, cols), R.dequantize(*q.read(), fmt).astype(np.float32))
        y2 = R.dequantize(*q2.read(), fmt)
        np.testing.assert_array_equal(y2, R.dequantize(*q.read(), fmt))


def assert_quantized_near(codes, scales, v, rel):
    """codes and scales are those of some values within rel (an array, relative) of v: each lies between the quantised
    lower and upper ends.  A block whose scale could be either of two is checked under the scale it took."""
    lo, hi = v - np.abs(v) * rel - 1e-36, v + np.abs(v) * rel + 1e-36
    small, large = np.where(v > 0, lo, hi), np.where(v > 0, hi, lo)      # towards and away from zero
    small = np.where(np.sign(small) != np.sign(v), 0.0, small)
    s0, s1 = R.quantize(small, E4M3)[1], R.quantize(large, E4M3)[1]
    assert ((scales >= s0) & (scales <= s1)).all()
    got = R.element_values(E4M3)[codes]
    up = np.exp2(127.0 - scales.astype(np.float64)).repeat(32, 1)
    grid = R.element_values(E4M3)[:127]

    def rounded(x):
        x = np.clip(x, -448, 448)
        step = np.exp2(np.maximum(np.frexp(x)[1] - 1, -6) - 3.0)
        return np.rint(x / step) * step
    assert np.isin(np.abs(got), grid).all()
    assert (got >= rounded(lo * up)).all() and (got <= rounded(hi * up)).all()


# the sum of squares: at most 32 terms a lane, 6 + 3 levels, every add off by 2^-24: 41 x 2^-24 of the sum, half of that
# of its root, then mean, eps, root, reciprocal and two products at most 2^-23 each
NORM_REL = 41 * 2.0 ** -25 + 6 * 2.0 ** -23


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols,gap,res", [(1, 32, 0, True), (1, 2048, 0, True), (3, 96, 8, False), (9, 2560, 0, True),
                                               (5, 4128, 24, True), (2, 8192, 0, False), (3, 16384, 0, True), (2100, 320, 0, True)])
def test_add_rmsnorm(wz, gpu, t, rows, cols, gap, res):
    rng = np.random.default_rng(rows + cols + t)
    xb, x = R.typed(activations(rng, rows, cols), t)
    rb, r = R.typed(activations(rng, rows, cols), t)
    gamma = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    h = R.typed((x.astype(np.float32) + r.astype(np.float32)) if res else x, t)[1]
    n = h / np.sqrt((h * h).mean(1, keepdims=True) + np.float64(np.float32(1e-6))) * gamma
    dx, dr, dg = DA.from_numpy(wide(xb, gap)), DA.from_numpy(wide(rb, gap)), DA.from_numpy(gamma)
    s, y = out_rows(rows, cols, t, gap), out_rows(rows, cols, t, gap)
    q = Mat(rows, cols, E4M3, gap=16, sgap=1)
    wz.wzy_mx_add_rmsnorm(dx.ptr, dr.ptr if res else None, t, cols + gap, dg.ptr, 1e-6, rows, cols, s.ptr, y.ptr, q.ref(), None)
    np.testing.assert_array_equal(read_rows(s, cols, t), h)
    got = read_rows(y, cols, t)
    assert (np.abs(got - n) <= np.abs(n) * (NORM_REL + R.HALF_STEP[t] * (1 + NORM_REL)) + 2.0 ** -25).all()
    assert_quantized_near(*q.read(), n, NORM_REL)
    # each output alone, and the sum in place of the residual or of x
    s2, q2 = out_rows(rows, cols, t, gap), Mat(rows, cols, E4M3)
    wz.wzy_mx_add_rmsnorm(dx.ptr, dr.ptr if res else None, t, cols + gap, dg.ptr, 1e-6, rows, cols, None, s2.ptr, None, None)
    np.testing.assert_array_equal(s2.numpy(), y.numpy())
    into = dr if res else dx
    wz.wzy_mx_add_rmsnorm(dx.ptr, dr.ptr if res else None, t, cols + gap, dg.ptr, 1e-6, rows, cols, into.ptr, None, q2.ref(), None)
    np.testing.assert_array_equal(into.numpy(), s.numpy())
    for a, b in zip(q2.read(), q.read()):
        np.testing.assert_array_equal(a, b)


def test_add_rmsnorm_zero_and_nan_rows(wz, gpu):
    x = np.ones((4, 64), np.float32)
    x[0] = 0
    x[2, 5] = np.nan
    g = np.ones(64, np.float32)
    dx, dg, y, q = DA.from_numpy(x), DA.from_numpy(g), out_rows(4, 64, F32), Mat(4, 64, E4M3)
    wz.wzy_mx_add_rmsnorm(dx.ptr, None, F32, 64, dg.ptr, 1e-6, 4, 64, None, y.ptr, q.ref(), None)
    got = read_rows(y, 64, F32)
    assert (got[0] == 0).all() and np.isnan(got[2]).all() and np.isfinite(got[[1, 3]]).all()
    codes, scales = q.read()
    assert (scales[0] == 0).all() and (codes[0] == 0).all() and (scales[2] == 255).all() and (codes[2] == 0).all()
    wz.wzy_mx_add_rmsnorm(dx.ptr, None, F32, 64, dg.ptr, 0.0, 4, 64, None, y.ptr, q.ref(), None)
    assert np.isnan(read_rows(y, 64, F32)[0]).all() and (q.read()[1][0] == 255).all()


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols,gap", [(1, 32, 0), (40, 512, 0), (7, 640, 8), (300, 96, 24)])
def test_swiglu(wz, gpu, t, rows, cols, gap):
    rng = np.random.default_rng(rows + cols + t)
    bits, x = R.typed(np.clip(activations(rng, rows, 2 * cols) * 3, -60, 60), t)
    g, u = x[:, :cols], x[:, cols:]
    d = DA.from_numpy(wide(bits, gap))
    q = Mat(rows, cols, E4M3, gap=16, sgap=2)
    wz.wzy_mx_swiglu(d.ptr, d.ptr + cols * (4 if t == F32 else 2), t, 2 * cols + gap, rows, cols, q.ref(), None)
    # the exponent's argument is off by |g| 2^-23 at most, exp, the sum, the quotient and the product by 2^-22 each
    assert_quantized_near(*q.read(), g * u / (1 + np.exp(-g)), (np.abs(g) + 8) * 2.0 ** -22)


def test_swiglu_far_gates(wz, gpu):
    """gates far below zero give zeros, not NaN; infinities and NaN spoil their block alone"""
    x = np.ones((1, 128), np.float32)
    x[0, :32] = -200.0
    x[0, 33], x[0, 100] = np.inf, 0.0                             # inf * 0
    d, q = DA.from_numpy(x), Mat(1, 64, E4M3)
    x[0, 97] = 0.0
    d = DA.from_numpy(x)
    wz.wzy_mx_swiglu(d.ptr, d.ptr + 256, F32, 128, 1, 64, q.ref(), None)
    codes, scales = q.read()
    assert (R.element_values(E4M3)[codes[0, :32]] * R.scale_values(scales[0, :1]) == 0).all()
    assert scales[0, 0] != 255 and scales[0, 1] == 255


def test_swiglu_product_of_large_factors(wz, gpu):
    """gate * up is past fp32's range, the result is not"""
    x = np.ones((1, 128), np.float32)
    x[0, :32], x[0, 64:96] = -80.0, np.float32(1e37) * (1 + np.arange(32) / 32)
    x[0, 32:64], x[0, 96:] = 30 + np.arange(32) / 4, np.float32(4e36)
    d, q = DA.from_numpy(x), Mat(1, 64, E4M3)
    wz.wzy_mx_swiglu(d.ptr, d.ptr + 256, F32, 128, 1, 64, q.ref(), None)
    g, u = x[:, :64].astype(np.float64), x[:, 64:].astype(np.float64)
    assert_quantized_near(*q.read(), g / (1 + np.exp(-g)) * u, (np.abs(g) + 8) * 2.0 ** -22)


# ---- products -----------------------------------------------------------------------------------------
def random_mx(rng, rows, cols, fmt, gap=0, sgap=0, spread=2):
    codes = rng.integers(0, 16 if fmt == E2M1 else 256, (rows, cols)).astype(np.uint8)
    if fmt == E4M3:
        codes[(codes & 127) == 127] -= 1
    scales = rng.integers(127 - spread, 128 + spread, (rows, cols // 32)).astype(np.uint8)
    m = Mat(rows, cols, fmt, gap, sgap, codes, scales)
    return m, R.dequantize(codes, scales, fmt)


def quantized_mx(rng, rows, cols, fmt, gap=0, sgap=0):
    codes, scales = R.quantize(activations(rng, rows, cols).astype(np.float64), fmt)
    return Mat(rows, cols, fmt, gap, sgap, codes, scales), R.dequantize(codes, scales, fmt)


def check_product(got, a, w, fmt, t):
    want, tol = R.product(a, w, fmt, t)
    off = np.abs(got - want) - tol
    assert np.isfinite(got).all() and (off <= 0).all(), "off by %g past %g at %s" % (
        np.abs(got - want).max(), tol.ravel()[off.argmax()], np.unravel_index(off.argmax(), off.shape))


GEMM_SHAPES = [(1, 1, 32), (1, 16, 2048), (1, 257, 320), (2, 33, 96), (4, 100, 512), (5, 48, 2560), (8, 31, 544), (15, 17, 640),
               (16, 130, 160), (17, 128, 128), (31, 65, 352), (64, 300, 96), (100, 129, 1056), (129, 127, 640), (257, 50, 160),
               (130, 260, 64)]


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("M,N,K", GEMM_SHAPES)
def test_gemm(wz, gpu, fmt, t, M, N, K):
    rng = np.random.default_rng(M * 1000 + N + K)
    pad = (M + N) % 3
    a, av = quantized_mx(rng, M, K, fmt, 16 * pad, pad)
    w, wv = quantized_mx(rng, N, K, E2M1, 32 * pad, 2 * pad)
    y = out_rows(M, N, t, pad)
    wz.wzy_mx_gemm(a.ref(), w.ref(), M, N, K, y.ptr, t, N + pad, None)
    check_product(read_rows(y, N, t), av, wv, fmt, t)


# K in whole steps of 128 and scale rows aligned to 4 bytes: the direct-to-LDS tiles, from one step to more than the buffers hold
@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(17, 20, 512), (40, 50, 256), (33, 70, 1280), (64, 64, 896), (100, 513, 512), (128, 256, 640), (130, 260, 1152),
                                   (257, 300, 640), (300, 97, 2048), (70, 90, 768)])
def test_gemm_whole_steps(wz, gpu, fmt, t, M, N, K):
    rng = np.random.default_rng(M * 1000 + N + K)
    pad = M % 2
    a, av = quantized_mx(rng, M, K, fmt, 16 * pad, 4 * pad)
    w, wv = quantized_mx(rng, N, K, E2M1, 32 * pad, 8 * pad)
    y = out_rows(M, N, t, pad)
    wz.wzy_mx_gemm(a.ref(), w.ref(), M, N, K, y.ptr, t, N + pad, None)
    got = read_rows(y, N, t)
    step = max(1, M * N * K // 20000000)          # the bound needs every product: rows in a stride that meets every tile
    rows = np.unique(np.concatenate([np.arange(0, M, step), [M - 1]]))
    check_product(got[rows], av[rows], wv, fmt, t)
    want, off = av @ wv.T, 1e-2
    assert (np.abs(got - want) <= off * (np.abs(av) @ np.abs(wv).T)).all()      # and all rows in rough


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("M", [3, 40])
def test_gemm_every_code(wz, gpu, fmt, M):
    """codes and scales drawn evenly: the whole range of an element inside every block"""
    rng = np.random.default_rng(M)
    a, av = random_mx(rng, M, 288, fmt)
    w, wv = random_mx(rng, 70, 288, E2M1)
    for t in (F32, BF16):
        y = out_rows(M, 70, t)
        wz.wzy_mx_gemm(a.ref(), w.ref(), M, 70, 288, y.ptr, t, 70, None)
        check_product(read_rows(y, 70, t), av, wv, fmt, t)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("M", [2, 33])
def test_gemm_scales_belong_to_their_block(wz, gpu, fmt, M):
    """one element set in a and w at every k in turn, scales different in every block: powers of two come back exactly"""
    K, N = 256, 256
    a = np.zeros((M, K), np.uint8)
    a[M - 1] = 2 if fmt == E2M1 else 0x38                         # ones
    w = np.zeros((N, K), np.uint8)
    w[np.arange(N), np.arange(K)] = 2
    sa = (120 + np.arange(M * K // 32).reshape(M, -1) % 8).astype(np.uint8)
    sw = (100 + np.arange(N * K // 32).reshape(N, -1) % 50).astype(np.uint8)
    da, dw, y = Mat(M, K, fmt, codes=a, scales=sa), Mat(N, K, E2M1, codes=w, scales=sw), out_rows(M, N, F32)
    wz.wzy_mx_gemm(da.ref(), dw.ref(), M, N, K, y.ptr, F32, N, None)
    want = R.dequantize(a, sa, fmt) @ R.dequantize(w, sw, E2M1).T
    np.testing.assert_array_equal(read_rows(y, N, F32), want)


@pytest.mark.parametrize("M", [4, 50])
def test_gemm_nan_stays_in_its_row_and_column(wz, gpu, M):
    rng = np.random.default_rng(M)
    codes, scales = R.quantize(activations(rng, M, 160).astype(np.float64), E4M3)
    codes[1, 70] = 0x7F
    scales[2, 4] = 255
    a = Mat(M, 160, E4M3, codes=codes, scales=scales)
    wc, ws = R.quantize(activations(rng, 40, 160).astype(np.float64), E2M1)
    ws[7, 0] = 255
    w = Mat(40, 160, E2M1, codes=wc, scales=ws)
    for t in (F32, BF16):
        y = out_rows(M, 40, t)
        wz.wzy_mx_gemm(a.ref(), w.ref(), M, 40, 160, y.ptr, t, 40, None)
        got = read_rows(y, 40, t)
        want = np.zeros((M, 40), bool)
        want[[1, 2]] = True
        want[:, 7] = True
        np.testing.assert_array_equal(np.isnan(got), want)


def grouped(wz, rng, sizes, M, N, K, fmt, t, a_rows=None, ids=None, pad=0, stream=None):
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    a, av = quantized_mx(rng, M if a_rows is None else a_rows, K, fmt, 16 * pad, pad)
    w, wv = quantized_mx(rng, len(sizes) * N, K, E2M1)
    y = out_rows(M, N, t, pad)
    before = y.numpy()
    do, di = DA.from_numpy(off), None if ids is None else DA.from_numpy(np.asarray(ids, np.int32))
    wz.wzy_mx_grouped_gemm(a.ref(), a.rows, None if ids is None else di.ptr, w.ref(), do.ptr, len(sizes), M, N, K, y.ptr, t,
                           N + pad, stream)
    got = read_rows(y, N, t)
    rows = np.arange(M) if ids is None else np.asarray(ids)
    for g in range(len(sizes)):
        sel = rows[off[g]:off[g + 1]]
        if len(sel):
            x = np.zeros((len(sel), K))
            ok = (sel >= 0) & (sel < av.shape[0])
            x[ok] = av[sel[ok]]
            check_product(got[off[g]:off[g + 1]], x, wv[g * N:(g + 1) * N], fmt, t)
    np.testing.assert_array_equal(y.numpy()[off[-1]:], before[off[-1]:])


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("sizes,N,K", [
    ([1], 16, 32), ([0, 0, 3, 0], 40, 320), ([2, 1, 0, 5, 16, 17], 33, 160), ([300], 50, 96), ([0, 200, 1, 0, 128, 129], 130, 160),
    ([40] * 7, 64, 640), ([33, 0, 31], 257, 64)])
def test_grouped(wz, gpu, fmt, t, sizes, N, K):
    rng = np.random.default_rng(sum(sizes) + N + K)
    M = sum(sizes)
    grouped(wz, rng, sizes, M, N, K, fmt, t)
    # gathered from fewer rows, some twice; three rows behind the last group
    grouped(wz, rng, sizes, M + 3, N, K, fmt, t, a_rows=M // 2 + 1, ids=rng.integers(0, M // 2 + 1, M + 3), pad=1)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("sizes,N,K", [([300], 50, 128), ([0, 200, 1, 0, 128, 129], 130, 512), ([40] * 7, 64, 640), ([33, 0, 31], 257, 896)])
def test_grouped_whole_steps(wz, gpu, fmt, t, sizes, N, K):
    rng = np.random.default_rng(sum(sizes) + N + K)
    M = sum(sizes)
    grouped(wz, rng, sizes, M, N, K, fmt, t)
    ids = rng.integers(0, M // 2 + 1, M + 3)
    ids[rng.integers(0, M, 5)] = [-1, M // 2 + 1, 2 ** 31 - 1, -2 ** 31, 0]
    grouped(wz, rng, sizes, M + 3, N, K, fmt, t, a_rows=M // 2 + 1, ids=ids)


def test_grouped_many_groups(wz, gpu):
    """more groups than one pass of the tile search holds, and nearly all empty"""
    rng = np.random.default_rng(5)
    sizes = np.zeros(1500, int)
    sizes[[0, 511, 512, 513, 700, 1499]] = [1, 2, 20, 1, 3, 17]
    grouped(wz, rng, list(sizes), int(sizes.sum()), 20, 64, E4M3, F32)
    sizes[512] = 40000                                            # one group far larger than the average
    grouped(wz, rng, list(sizes[:520]), int(sizes[:520].sum()), 3, 32, E2M1, F32)


@pytest.mark.parametrize("M", [6, 90])
def test_grouped_ids_out_of_range_read_zeros(wz, gpu, M):
    rng = np.random.default_rng(M)
    ids = rng.integers(0, 10, M)
    ids[[0, 3]], ids[5] = [-1, 10], 2 ** 31 - 1
    grouped(wz, rng, [M // 2, M - M // 2], M, 24, 96, E4M3, F32, a_rows=10, ids=ids)
    grouped(wz, rng, [M], M, 24, 96, E2M1, BF16, a_rows=10, ids=ids)


@pytest.mark.parametrize("off", [[0, 9, 4, 12], [-5, 3, 1000, 2], [12, 12, 0, 0], [2 ** 31 - 1, -2 ** 31, 5, 12]])
@pytest.mark.parametrize("M", [12, 120])
def test_grouped_broken_offsets_stay_in_y(wz, gpu, off, M):
    rng = np.random.default_rng(1)
    a, _ = quantized_mx(rng, M, 64, E4M3)
    w, _ = quantized_mx(rng, 3 * 20, 64, E2M1)
    y = DA.from_numpy(np.full((M + 300, 20), 7.0, np.float32))
    do = DA.from_numpy(np.asarray(off, np.int64).astype(np.int32))
    wz.wzy_mx_grouped_gemm(a.ref(), M, None, w.ref(), do.ptr, 3, M, 20, 64, y.ptr, F32, 20, None)
    assert (y.numpy()[M:] == 7.0).all()


# ---- as they are used together -------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 4, 40])
def test_expert_block_run(wz, gpu, T):
    """norm -> gathered gate|up per expert -> SwiGLU -> down per expert, each step checked on what the GPU handed it"""
    rng = np.random.default_rng(T)
    D, F, E, K = 256, 96, 6, 3
    xb, x = R.typed(activations(rng, T, D), BF16)
    rb, r = R.typed(activations(rng, T, D), BF16)
    gamma = np.ones(D, np.float32)
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)])
    order = np.argsort(ids.ravel(), kind="stable")
    off = np.concatenate([[0], np.cumsum(np.bincount(ids.ravel(), minlength=E))]).astype(np.int32)
    M = T * K
    w1, w1v = quantized_mx(rng, E * 2 * F, D, E2M1)
    w2, w2v = quantized_mx(rng, E * D, F, E2M1)
    dx, dr, dg, do = DA.from_numpy(xb), DA.from_numpy(rb), DA.from_numpy(gamma), DA.from_numpy(off)
    dids = DA.from_numpy((order // K).astype(np.int32))
    q1, q2 = Mat(T, D, E4M3), Mat(M, F, E4M3)
    gu, y, sm = out_rows(M, 2 * F, BF16), out_rows(M, D, F32), out_rows(T, D, BF16)
    st = C.c_void_p()
    wz.wzy_stream_create(C.byref(st))
    s = st.value
    wz.wzy_mx_add_rmsnorm(dx.ptr, dr.ptr, BF16, D, dg.ptr, 1e-6, T, D, sm.ptr, None, q1.ref(), s)
    wz.wzy_mx_grouped_gemm(q1.ref(), T, dids.ptr, w1.ref(), do.ptr, E, M, 2 * F, D, gu.ptr, BF16, 2 * F, s)
    wz.wzy_mx_swiglu(gu.ptr, gu.ptr + 2 * F, BF16, 2 * F, M, F, q2.ref(), s)
    wz.wzy_mx_grouped_gemm(q2.ref(), M, None, w2.ref(), do.ptr, E, M, D, F, y.ptr, F32, D, s)
    wz.wzy_stream_sync(s)
    wz.wzy_stream_destroy(s)
    h = R.typed(x.astype(np.float32) + r.astype(np.float32), BF16)[1]
    np.testing.assert_array_equal(read_rows(sm, D, BF16), h)
    n = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6)
    assert_quantized_near(*q1.read(), n, NORM_REL)
    a1, guv, a2, yv = R.dequantize(*q1.read(), E4M3), read_rows(gu, 2 * F, BF16), R.dequantize(*q2.read(), E4M3), read_rows(y, D, F32)
    for e in range(E):
        o = slice(off[e], off[e + 1])
        if off[e] < off[e + 1]:
            check_product(guv[o], a1[order[o] // K], w1v[e * 2 * F:(e + 1) * 2 * F], E4M3, BF16)
            check_product(yv[o], a2[o], w2v[e * D:(e + 1) * D], E4M3, F32)
    g, u = guv[:, :F], guv[:, F:]
    assert_quantized_near(*q2.read(), g * u / (1 + np.exp(-g)), (np.abs(g) + 8) * 2.0 ** -22)


def test_two_streams_and_graph_replays(wz, gpu):
    """the same calls on two streams at once, then captured and replayed between eager calls: the same bits"""
    hip = C.CDLL("libamdhip64.so")
    rng = np.random.default_rng(9)
    T, D, N, E = 24, 512, 320, 5
    sizes = [3, 0, 11, 9, 1]
    off = DA.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32))
    x, g = DA.from_numpy(activations(rng, T, D)), DA.from_numpy(np.ones(D, np.float32))
    w, _ = quantized_mx(rng, E * N, D, E2M1)

    def outputs():
        return dict(q=Mat(T, D, E4M3), y=out_rows(T, N, F32), z=out_rows(T, N, BF16), q2=Mat(T, N, E2M1))

    def enqueue(o, s):
        wz.wzy_mx_add_rmsnorm(x.ptr, None, F32, D, g.ptr, 1e-6, T, D, None, None, o["q"].ref(), s)
        wz.wzy_mx_gemm(o["q"].ref(), w.ref(), T, N, D, o["y"].ptr, F32, N, s)
        wz.wzy_mx_grouped_gemm(o["q"].ref(), T, None, w.ref(), off.ptr, E, T, N, D, o["z"].ptr, BF16, N, s)
        wz.wzy_mx_quantize(o["y"].ptr, F32, N, T, N, o["q2"].ref(), s)

    def bits(o):
        return [o["y"].numpy(), o["z"].numpy(), *o["q"].read(), *o["q2"].read()]

    one, two = outputs(), outputs()
    enqueue(one, None)
    wz.wzy_device_sync()
    want = bits(one)
    st = [C.c_void_p(), C.c_void_p()]
    for s in st:
        wz.wzy_stream_create(C.byref(s))
    o1, o2 = outputs(), outputs()
    for _ in range(5):
        enqueue(o1, st[0].value)
        enqueue(o2, st[1].value)
    wz.wzy_device_sync()
    for o in (o1, o2):
        for a, b in zip(bits(o), want):
            np.testing.assert_array_equal(a, b)
    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(st[0], 2) == 0
    enqueue(two, st[0].value)
    assert hip.hipStreamEndCapture(st[0], C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(4):
        for d in (two["y"], two["z"]):
            wz.wzy_memset(d.ptr, 0, d.nbytes, None)
        wz.wzy_device_sync()
        assert hip.hipGraphLaunch(run, st[0]) == 0
        wz.wzy_device_sync()
        for a, b in zip(bits(two), want):
            np.testing.assert_array_equal(a, b)
        enqueue(one, None)
        wz.wzy_device_sync()
        for a, b in zip(bits(one), want):
            np.testing.assert_array_equal(a, b)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    for s in st:
        wz.wzy_stream_destroy(s.value)


def test_no_rows_launch_nothing(wz, gpu):
    q = Mat(1, 64, E4M3)
    wz.wzy_mx_quantize(None, F32, 64, 0, 64, None, None)
    wz.wzy_mx_dequantize(None, 0, 64, None, F32, 64, None)
    wz.wzy_mx_add_rmsnorm(None, None, F32, 64, None, 1e-6, 0, 64, None, None, q.ref(), None)
    wz.wzy_mx_swiglu(None, None, BF16, 64, 0, 64, None, None)
    wz.wzy_mx_gemm(None, None, 0, 5, 64, None, F32, 5, None)
    wz.wzy_mx_gemm(None, None, 5, 0, 64, None, F32, 5, None)
    wz.wzy_mx_grouped_gemm(None, 0, None, None, None, 4, 0, 5, 64, None, F32, 5, None)
    wz.wzy_device_sync()
    assert (q.read()[0] == FILL).all()


# ---- every tile, whole units of K and any K ---------------------------------------------------------------
def check_in_rough(got, a, w, t):
    """all of y: 8 products are cut at 13 bits below the largest of them, so by 8 * 2^-12 of it at most; each of the sums of eights
    rounds to 24 bits; the output to its type"""
    want, s = a @ w.T, np.abs(a) @ np.abs(w).T
    assert (np.abs(got - want) <= (2.0 ** -9 + a.shape[1] / 8 * 2.0 ** -23) * s + {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}[t] * np.abs(want)
            + 2.0 ** -24).all()


def check_large(got, a, w, fmt, t):
    """the exact bound at rows and columns in strides that meet every place of a tile in turn, the rough one everywhere"""
    m, n = max(1, a.shape[0] // 50), max(1, w.shape[0] // 60)
    i, j = np.unique(np.r_[0:len(a):m, len(a) - 1]), np.unique(np.r_[0:len(w):n, len(w) - 1])
    check_product(got[np.ix_(i, j)], a[i], w[j], fmt, t)
    check_in_rough(got, a, w, t)


TILE_SHAPES = [(5, 4100, 32), (16, 4200, 768), (1, 5000, 544), (9, 4097, 1056), (250, 600, 672), (250, 600, 512), (700, 1300, 608),
               (700, 1300, 1024), (1030, 2060, 96), (1030, 2060, 768), (2050, 2100, 544), (2050, 2100, 512), (4100, 4090, 512)]


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("M,N,K", TILE_SHAPES)
def test_gemm_every_tile(wz, gpu, fmt, t, M, N, K):
    rng = np.random.default_rng(M + N + K)
    a, av = random_mx(rng, M, K, fmt)
    w, wv = random_mx(rng, N, K, E2M1)
    y = out_rows(M, N, t)
    wz.wzy_mx_gemm(a.ref(), w.ref(), M, N, K, y.ptr, t, N, None)
    check_large(read_rows(y, N, t), av, wv, fmt, t)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("K", list(range(32, 33 * 32, 32)))
def test_gemm_every_tail(wz, gpu, fmt, K):
    """every number of blocks up to two groups of scales: a skinny call, small tiles, 16 x 64 tiles; unaligned scale rows"""
    rng = np.random.default_rng(K)
    for M, N, sgap in [(3, 40, 1), (33, 65, 3), (40, 70, 0), (7, 4112, 0)]:
        cols = np.r_[0:N:max(1, N // 20), N - 1]
        a, av = random_mx(rng, M, K, fmt, sgap=sgap)
        w, wv = random_mx(rng, N, K, E2M1, sgap=sgap)
        for t in (F32, BF16):
            y = out_rows(M, N, t)
            wz.wzy_mx_gemm(a.ref(), w.ref(), M, N, K, y.ptr, t, N, None)
            check_product(read_rows(y, N, t)[:, cols], av, wv[cols], fmt, t)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("K", [512, 544, 768, 1120])
def test_gemm_neighbours_of_a_row_do_not_show(wz, gpu, fmt, K):
    """what lies behind a row's codes and scales, NaN codes and scales of 255, is not multiplied"""
    rng = np.random.default_rng(K)
    for M, N in [(3, 30), (9, 4100), (40, 70), (300, 520), (1100, 2100)]:
        m, mv = random_mx(rng, M, K, fmt)
        w, wv = random_mx(rng, N, K, E2M1)
        for x in (m, w):
            c, s = x.c.numpy(), x.s.numpy()
            c, s = np.pad(c, ((0, 0), (0, 32)), constant_values=0xFF), np.pad(s, ((0, 0), (0, 5 if K % 256 else 4)), constant_values=0xFF)
            x.c, x.s = DA.from_numpy(c), DA.from_numpy(s)
            x.m = wzy_amd.MxMat(x.c.ptr, x.s.ptr, c.shape[1], s.shape[1], x.fmt)
        y = out_rows(M, N, BF16)
        wz.wzy_mx_gemm(m.ref(), w.ref(), M, N, K, y.ptr, BF16, N, None)
        check_large(read_rows(y, N, BF16), mv, wv, fmt, BF16)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("per,groups,N,K", [(5, 9, 130, 512), (5, 9, 130, 288), (20, 7, 260, 768), (20, 7, 260, 1056), (50, 5, 200, 512),
                                            (50, 5, 200, 608), (90, 4, 300, 1024), (90, 4, 300, 96), (300, 3, 90, 544)])
def test_grouped_every_tile(wz, gpu, fmt, t, per, groups, N, K):
    rng = np.random.default_rng(per + N + K)
    sizes = rng.multinomial(per * groups, np.arange(groups) / np.arange(groups).sum())    # an empty one first
    M = int(sizes.sum())
    grouped(wz, rng, list(sizes), M, N, K, fmt, t)
    ids = rng.integers(-2, M // 2 + 3, M + 5)
    grouped(wz, rng, list(sizes), M + 5, N, K, fmt, t, a_rows=M // 2 + 1, ids=ids, pad=1)


@pytest.mark.parametrize("K", [512, 544])
def test_grouped_largest_tiles(wz, gpu, K):
    """enough rows and tiles for 256 x 256 (E2M1); a group's weights are the first one's, rolled by its number"""
    rng = np.random.default_rng(K)
    G, N, per = 64, 2048, 130
    codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
    scales = rng.integers(125, 130, (N, K // 32)).astype(np.uint8)
    wv = R.dequantize(codes, scales, E2M1)
    w = Mat(G * N, K, E2M1, codes=np.concatenate([np.roll(codes, g, 0) for g in range(G)]),
            scales=np.concatenate([np.roll(scales, g, 0) for g in range(G)]))
    sizes = rng.multinomial(G * per, np.ones(G) / G)
    M = int(sizes.sum())
    off = np.r_[0, np.cumsum(sizes)].astype(np.int32)
    a, av = random_mx(rng, M, K, E2M1)
    y, do = out_rows(M, N, BF16), DA.from_numpy(off)
    wz.wzy_mx_grouped_gemm(a.ref(), M, None, w.ref(), do.ptr, G, M, N, K, y.ptr, BF16, N, None)
    got = read_rows(y, N, BF16)
    for g in range(G):
        i = slice(off[g], off[g + 1])
        check_large(got[i], av[i], np.roll(wv, g, 0), E2M1, BF16)


class FarRows:
    """rows of a matrix `stride` bytes apart: only the rows themselves are written"""

    def __init__(self, wz, codes, scales, fmt, stride):
        p = R.pack(codes, fmt)
        self.rows = len(p)
        self.c, self.s = DA(((self.rows - 1) * stride + p.shape[1],), np.uint8), DA.from_numpy(scales)
        for i, row in enumerate(np.ascontiguousarray(p)):
            wz.wzy_memcpy_h2d(self.c.ptr + i * stride, row.ctypes.data, row.nbytes, None)
        self.m = wzy_amd.MxMat(self.c.ptr, self.s.ptr, stride, scales.shape[1], fmt)

    def ref(self):
        return C.byref(self.m)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("K", [512, 544])
def test_rows_far_apart(wz, gpu, fmt, K):
    """the widest rows allowed: offsets past 2^31 inside a tile, past 2^32 between tiles and among gathered rows"""
    rng = np.random.default_rng(K)
    stride, M, N = 2 ** 23 - 16, 600, 90
    codes = rng.integers(0, 16 if fmt == E2M1 else 126, (M, K)).astype(np.uint8)
    scales = rng.integers(125, 130, (M, K // 32)).astype(np.uint8)
    a, av = FarRows(wz, codes, scales, fmt, stride), R.dequantize(codes, scales, fmt)
    w, wv = random_mx(rng, 2 * N, K, E2M1)
    far, farv = FarRows(wz, codes[:N] & 15, scales[:N], E2M1, stride), R.dequantize(codes[:N] & 15, scales[:N], E2M1)
    for t in (F32, BF16):
        y = out_rows(M, N, t)
        wz.wzy_mx_gemm(a.ref(), far.ref(), M, N, K, y.ptr, t, N, None)
        check_large(read_rows(y, N, t), av, farv, fmt, t)
        ids = rng.integers(0, M, M)
        ids[[0, 7]] = [-1, M]
        y, di = out_rows(M, N, t), DA.from_numpy(ids.astype(np.int32))
        do = DA.from_numpy(np.array([0, M // 3, M], np.int32))
        wz.wzy_mx_grouped_gemm(a.ref(), M, di.ptr, w.ref(), do.ptr, 2, M, N, K, y.ptr, t, N, None)
        got, x = read_rows(y, N, t), av[ids.clip(0, M - 1)]
        x[[0, 7]] = 0
        check_large(got[:M // 3], x[:M // 3], wv[:N], fmt, t)
        check_large(got[M // 3:], x[M // 3:], wv[N:], fmt, t)
        y = out_rows(300, N, t)                                   # not gathered: the second group's rows begin past 2^30
        do = DA.from_numpy(np.array([0, 40, 300], np.int32))
        wz.wzy_mx_grouped_gemm(a.ref(), M, None, w.ref(), do.ptr, 2, 300, N, K, y.ptr, t, N, None)
        got = read_rows(y, N, t)
        check_large(got[:40], av[:40], wv[:N], fmt, t)
        check_large(got[40:], av[40:300], wv[N:], fmt, t)
    for m in (a, far):
        m.c.free()


@pytest.mark.parametrize("M,N", [(3, 40), (40, 70), (7, 4112), (300, 200)])
@pytest.mark.parametrize("K", [512, 288])
def test_gemm_fp16_sums_that_cancel(wz, gpu, M, N, K):
    """a small rest of large products, of E4M3 rows: the bound of fp32 sums and one rounding"""
    rng = np.random.default_rng(M + K)
    small = rng.integers(0, 24, (M, K)) | rng.integers(0, 2, (M, K)) << 7       # up to 2^-4
    codes = small.astype(np.uint8)
    codes[:, 0::16] = codes[:, 1::16] = 0x7E                      # 448 twice in an eight, by weights that cancel
    wc = rng.integers(0, 16, (N, K)).astype(np.uint8)
    wc[:, 1::16] = wc[:, 0::16] ^ 8
    scales = np.full((M, K // 32), 127, np.uint8)
    wsc = np.full((N, K // 32), 127, np.uint8)
    a, w = Mat(M, K, E4M3, codes=codes, scales=scales), Mat(N, K, E2M1, codes=wc, scales=wsc)
    at = np.r_[0:N:max(1, N // 20), N - 1]
    av, wv = R.dequantize(codes, scales, E4M3), R.dequantize(wc, wsc, E2M1)[at]
    y, z, off = out_rows(M, N, F16), out_rows(M, N, F16), DA.from_numpy(np.array([0, M], np.int32))
    wz.wzy_mx_gemm(a.ref(), w.ref(), M, N, K, y.ptr, F16, N, None)
    wz.wzy_mx_grouped_gemm(a.ref(), M, None, w.ref(), off.ptr, 1, M, N, K, z.ptr, F16, N, None)
    for d in (y, z):                              # (E2M1 names the bound without cut products)
        check_product(read_rows(d, N, F16)[:, at], av, wv, E2M1, F16)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(24, 2048), (24, 96), (24, 8192)])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
def test_add_rmsnorm_rows_whose_squares_leave_fp32(wz, gpu, t, rows, cols, eps):
    rng = np.random.default_rng(cols)
    size = np.array([1e37, 1e30, 1e25, 2e20, 1e19, 3e18, 1e17, 1.0, 1e-10, 1e-13, 1e-17, 1e-20, 1e-22, 1e-25, 1e-30, 1e-36])
    x = rng.standard_normal((rows, cols))
    x[:len(size)] *= size[:, None]
    x[16] = 1.0
    x[16, 5] = 3e38                                               # one value far above the others
    x[17] = 1e-18
    x[17, 7] = 2e19
    x[18] = 0.0
    x[18, 9] = 1e-30
    x[19:] *= 10.0 ** rng.uniform(-36, 36, (5, 1))
    bits, h = R.typed(x, t)
    gamma = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    n = h / np.sqrt((h * h).mean(1, keepdims=True) + np.float64(np.float32(eps))) * gamma
    d, g = DA.from_numpy(bits), DA.from_numpy(gamma)
    s, y, q = out_rows(rows, cols, t), out_rows(rows, cols, t), Mat(rows, cols, E4M3)
    wz.wzy_mx_add_rmsnorm(d.ptr, None, t, cols, g.ptr, eps, rows, cols, s.ptr, y.ptr, q.ref(), None)
    np.testing.assert_array_equal(read_rows(s, cols, t), h)
    got = read_rows(y, cols, t)
    # below 2^-126 steps are 2^-149 (fp32) or 2^-133 (bf16)
    assert (np.abs(got - n) <= np.abs(n) * (NORM_REL + R.HALF_STEP[t] * (1 + NORM_REL)) + (2.0 ** -149 if t == F32 else 2.0 ** -134)).all()
    assert_quantized_near(*q.read(), n, NORM_REL)


def test_swiglu_small_gates_times_large_factors(wz, gpu):
    """exp(-gate) is past fp32's range from gates of -88.8 on; the products come out down to the format's smallest element"""
    rng = np.random.default_rng(3)
    x = np.empty((64, 128), np.float32)
    x[:, :64] = -np.linspace(80, 187, 64, dtype=np.float32)[:, None] - rng.random((64, 64), np.float32) * 0.5
    g = x[:, :64].astype(np.float64)
    x[:, 64:] = np.sign(rng.standard_normal((64, 64))) * np.minimum(2.0 ** rng.integers(-20, 8, (64, 64)) / (-g * np.exp(g)), 3e38)
    u = x[:, 64:].astype(np.float64)
    d, q = DA.from_numpy(x), Mat(64, 64, E4M3)
    wz.wzy_mx_swiglu(d.ptr, d.ptr + 256, F32, 128, 64, 64, q.ref(), None)
    codes, scales = q.read()
    v = g * u / (1 + np.exp(-g))
    # the bound of test_swiglu, and of a product that passes through fp32's denormals half a step of those, 2^-150, before a factor
    # exp(gate / 2) of 2^-57 at most takes the rest of its way: nothing beside the 1e-36 of assert_quantized_near, nor that beside 2^-9
    # of the smallest scale 2^-127
    assert_quantized_near(codes, scales, v, (np.abs(g) + 8) * 2.0 ** -22)
    big = np.abs(v).reshape(64, 2, 32).max(2) > 1e-30
    assert big.sum() > 60 and (scales[big] > 8).all()


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("M", [2, 33])
def test_gemm_scales_from_end_to_end(wz, gpu, fmt, M):
    """every scale byte of a against the one of w that brings the product back near 1; a block that is NaN as the quantiser writes it"""
    K, N = 256, 256
    a = np.zeros((M, K), np.uint8)
    a[:, 3::32] = 2 if fmt == E2M1 else 0x38                      # a one in each block
    w = np.zeros((N, K), np.uint8)
    w[np.arange(N), np.arange(N) % 8 * 32 + 3] = 2
    sw = (np.arange(N)[:, None] * np.ones(K // 32, int)).clip(0, 254).astype(np.uint8)
    for sa in (0, 1, 120, 253, 254):
        s = np.full((M, K // 32), sa, np.uint8)
        da, dw, y = Mat(M, K, fmt, codes=a, scales=s), Mat(N, K, E2M1, codes=w, scales=sw), out_rows(M, N, F32)
        wz.wzy_mx_gemm(da.ref(), dw.ref(), M, N, K, y.ptr, F32, N, None)
        want = np.exp2(sa + sw[:, 0].astype(np.float64) - 254)[None].repeat(M, 0)
        got, inside = read_rows(y, N, F32), (want >= 2.0 ** -126) & (want < 2.0 ** 128)
        np.testing.assert_array_equal(got[inside], want[inside])
        assert (got[want >= 2.0 ** 128] == np.inf).all() and (got[want < 2.0 ** -126] <= 2.0 ** -126).all()
    codes, scales = np.zeros((M, K), np.uint8), np.full((M, K // 32), 127, np.uint8)
    scales[1, 5] = 255
    ws = np.full((N, K // 32), 127, np.uint8)
    ws[9, 2] = 255
    wc = w.copy()
    wc[9] = 0
    for t in (F32, BF16, F16):
        da, dw, y = Mat(M, K, fmt, codes=codes, scales=scales), Mat(N, K, E2M1, codes=wc, scales=ws), out_rows(M, N, t)
        wz.wzy_mx_gemm(da.ref(), dw.ref(), M, N, K, y.ptr, t, N, None)
        want = np.zeros((M, N), bool)
        want[1], want[:, 9] = True, True
        np.testing.assert_array_equal(np.isnan(read_rows(y, N, t)), want)


def within_fp16(got, a, w, t):
    """got with the infinities that fp16 rounds to from 65,520 on, halfway past its last value, in place of what they stand for; none elsewhere"""
    if t == F16:
        want, most = a @ w.T, 2.0 ** -9 * (np.abs(a) @ np.abs(w).T)   # (check_in_rough bounds a sum's error by that and less than as much again)
        assert not (np.isinf(got) & (np.abs(want) + 2 * most < 65520)).any() and np.isinf(got[np.abs(want) - 2 * most > 65520]).all()
        inf = np.isinf(got)
        assert (np.sign(got[inf]) == np.sign(want[inf])).all()
        got = np.where(inf, want, got)
    return got


# Tiles that the shapes take:   E4M3 to bf16   E2M1             E4M3 to fp32   E4M3 to fp16   (256 x 256: whole units of K; otherwise in brackets)
#   200 x 320                   32x64          32x64            32x64          32x64
#   10 x 4,224                  16x64          16x64            16x64          16x64
#   4,100 x 80                  64x64          64x64            32x64          32x64
#   4,100 x 200                 64x128         64x128           64x64          64x64
#   900 x 4,104                 64x128         64x128           64x128         64x128
#   4,100 x 464                 64x128         128x128          128x128        128x128
#   3,800 x 1,552               128x128        128x128          128x128        128x128
#   3,100 x 3,848               256x256 (64x128)  256x256 (128x128)  64x128    256x256 (128x128)
@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("M,N", [(200, 320), (10, 4224), (4100, 80), (4100, 200), (900, 4104), (4100, 464), (3800, 1552), (3100, 3848)])
def test_gemm_tiles_whole_and_any(wz, gpu, fmt, t, M, N):
    """whole units and any K; rows of y aligned (whole lines stored) and not"""
    rng = np.random.default_rng(M + N)
    for n, K in [(N, 768), (N + 1, 512), (N, 608), (N + 1, 544)]:
        a, av = random_mx(rng, M, K, fmt)
        w, wv = random_mx(rng, n, K, E2M1)
        y = out_rows(M, n, t)
        wz.wzy_mx_gemm(a.ref(), w.ref(), M, n, K, y.ptr, t, n, None)
        check_large(within_fp16(read_rows(y, n, t), av, wv, t), av, wv, fmt, t)


# rows per group: 16x64, 32x128, 64x128, 128x128 tiles
@pytest.mark.parametrize("fmt", [E2M1, E4M3])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("per,groups", [(2, 12), (7, 9), (20, 7), (50, 5), (90, 4)])
def test_grouped_gathered_tiles(wz, gpu, fmt, t, per, groups):
    """whole units and any K, rows gathered, ids outside a among them, whole lines of y stored and not; the same not gathered"""
    rng = np.random.default_rng(per + groups)
    sizes = rng.multinomial(per * groups, np.arange(groups) / np.arange(groups).sum())
    M = int(sizes.sum())
    for N, K in [(256, 512), (264, 768), (129, 768), (256, 608)]:
        ids = rng.integers(-1, M // 2 + 2, M)
        ids[rng.integers(0, M, 2)] = [2 ** 31 - 1, -2 ** 31]
        grouped(wz, rng, list(sizes), M, N, K, fmt, t, a_rows=M // 2 + 1, ids=ids)
        grouped(wz, rng, list(sizes), M, N, K, fmt, t)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("K", [512, 768])
def test_grouped_largest_tiles_gathered(wz, gpu, t, K):
    """256 x 256 tiles of gathered rows, ids outside a among them; a group's weights are the first one's, rolled by its number"""
    rng = np.random.default_rng(K)
    G, N, per, T = 64, 2048, 130, 900
    codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
    scales = rng.integers(125, 130, (N, K // 32)).astype(np.uint8)
    wv = R.dequantize(codes, scales, E2M1)
    w = Mat(G * N, K, E2M1, codes=np.concatenate([np.roll(codes, g, 0) for g in range(G)]),
            scales=np.concatenate([np.roll(scales, g, 0) for g in range(G)]))
    sizes = rng.multinomial(G * per, np.ones(G) / G)
    M = int(sizes.sum())
    off = np.r_[0, np.cumsum(sizes)].astype(np.int32)
    ids = rng.integers(-5, T + 5, M)
    ids[[0, M - 1]] = [-2 ** 31, 2 ** 31 - 1]
    a, av = random_mx(rng, T, K, E2M1)
    x = np.where(((ids >= 0) & (ids < T))[:, None], av[ids.clip(0, T - 1)], 0.0)
    y, do, di = out_rows(M, N, t), DA.from_numpy(off), DA.from_numpy(ids.astype(np.int32))
    wz.wzy_mx_grouped_gemm(a.ref(), T, di.ptr, w.ref(), do.ptr, G, M, N, K, y.ptr, t, N, None)
    got = read_rows(y, N, t)
    for g in range(G):
        i = slice(off[g], off[g + 1])
        check_large(got[i], x[i], np.roll(wv, g, 0), E2M1, t)


@pytest.mark.parametrize("fmt", [E2M1, E4M3])
def test_rows_gathered_from_far_fp16(wz, gpu, fmt):
    """rows gathered from more than 4 GiB to fp16, ids outside a among them, rows of y aligned and not"""
    rng = np.random.default_rng(fmt)
    stride, T, M, K = 2 ** 23 - 16, 520, 150, 544
    codes = rng.integers(0, 16 if fmt == E2M1 else 126, (T, K)).astype(np.uint8)
    scales = rng.integers(118, 122, (T, K // 32)).astype(np.uint8)
    a, av = FarRows(wz, codes, scales, fmt, stride), R.dequantize(codes, scales, fmt)
    ids = rng.integers(0, T, M)
    ids[[0, 9, M - 1]] = [-1, T, T - 1]
    x = np.where(((ids >= 0) & (ids < T))[:, None], av[ids.clip(0, T - 1)], 0.0)
    do, di = DA.from_numpy(np.array([0, 70, M], np.int32)), DA.from_numpy(ids.astype(np.int32))
    for N in (128, 75):
        w, wv = random_mx(rng, 2 * N, K, E2M1)
        y = out_rows(M, N, F16)
        wz.wzy_mx_grouped_gemm(a.ref(), T, di.ptr, w.ref(), do.ptr, 2, M, N, K, y.ptr, F16, N, None)
        got = read_rows(y, N, F16)
        check_product(got[:70], x[:70], wv[:N], fmt, F16)
        check_product(got[70:], x[70:], wv[N:], fmt, F16)
    a.c.free()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(300, 2048), (40, 16384), (2000, 96)])
def test_add_rmsnorm_sums_in_64_bits(wz, gpu, t, rows, cols):
    """n is right to one rounding: the sum of squares, its root and the product keep more than fp32"""
    rng = np.random.default_rng(rows)
    xb, x = R.typed(activations(rng, rows, cols), t)
    gamma = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    n = x / np.sqrt((x * x).mean(1, keepdims=True) + np.float64(np.float32(1e-6))) * gamma
    dx, dg, y, q = DA.from_numpy(xb), DA.from_numpy(gamma), out_rows(rows, cols, t), Mat(rows, cols, E4M3)
    wz.wzy_mx_add_rmsnorm(dx.ptr, None, t, cols, dg.ptr, 1e-6, rows, cols, None, y.ptr, q.ref(), None)
    # 64-bit steps: at most 16,384 additions and a Newton step from 22 bits on, 2^-38 together; then fp32's half step, and bf16's of that
    rel = 2.0 ** -24 * (1 + 2.0 ** -13)
    half = np.exp2(np.frexp(n)[1] - (24.0 if t == F32 else 8.0) - 1) if t == F32 else R.HALF_STEP[t] * np.abs(n)
    assert (np.abs(read_rows(y, cols, t) - n) <= (half * (1 + 2.0 ** -13) if t == F32 else half + rel * np.abs(n))).all()
    assert_quantized_near(*q.read(), n, rel)


@pytest.mark.parametrize("low,high", [(-60, 0), (-6, 6), (-185, -40)])
def test_swiglu_right_to_few_last_bits(wz, gpu, low, high):
    """the exponential keeps fp32's bits at every gate: p and the reciprocal are off by one last bit, five roundings by half of one, and
    (rounded up) what f = -|g| log2(e) - n loses to its own rounding, 2^-26, which 2^f turns into as much"""
    rng = np.random.default_rng(max(high, 0))
    rows, cols = 2000, 256
    x = rng.uniform(low, high, (rows, 2 * cols)).astype(np.float32)
    g = x[:, :cols].astype(np.float64)
    x[:, cols:] = (rng.uniform(0.5, 2, (rows, cols)) * np.minimum(np.exp(np.maximum(-g, 0)), 1e38) / np.maximum(np.abs(g), 1e-3)).astype(np.float32)
    u = x[:, cols:].astype(np.float64)
    d, q = DA.from_numpy(x), Mat(rows, cols, E4M3)
    wz.wzy_mx_swiglu(d.ptr, d.ptr + 4 * cols, F32, 2 * cols, rows, cols, q.ref(), None)
    assert_quantized_near(*q.read(), g / (1 + np.exp(-g)) * u, 5 * 2.0 ** -23)
