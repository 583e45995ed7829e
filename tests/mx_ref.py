"""Plain 64-bit formulations of the microscaled (MX) operators and their error bounds (test infrastructure).

Written from the format: a block of 32 values has the scale 2^(floor(log2 max) - emax), at least 2^-127; elements
are rounded to nearest on their own grid (ties to even) and limited to the largest element.
"""
import numpy as np

E2M1, E4M3 = 0, 1
EMAX = {E2M1: 2, E4M3: 8}
MOST = {E2M1: 6.0, E4M3: 448.0}
GRID = {E2M1: (0, 1), E4M3: (-6, 3)}            # exponent of the smallest normal, fraction bits
F32, BF16, F16 = 0, 1, 2
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}     # of a value, at most


def f32_to_bf16_bits(x):
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def typed(x, t):
    """x rounded to type t: (array to upload, float64 values)"""
    x = np.asarray(x, np.float32)
    if t == F32:
        return x, x.astype(np.float64)
    if t == F16:
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float64)
    b = f32_to_bf16_bits(x)
    b = np.where(np.isnan(x), np.uint16(0x7FC0), b)
    return b, (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def values(bits, t):
    """float64 values of downloaded rows of type t"""
    if t == F32:
        return bits.astype(np.float64)
    if t == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def element_values(fmt):
    """value of every code"""
    if fmt == E2M1:
        m = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
        return np.concatenate([m, -m])
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def quantize(x, fmt):
    """float64 rows -> (codes one per element, scale bytes)"""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[0], -1, 32)
    amax = np.abs(b).max(2)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], 0.0, b)
    amax = np.where(bad, 0.0, amax)
    e = np.where(amax > 0, np.frexp(amax)[1] - 1 - EMAX[fmt], -127)
    e = np.maximum(e, -127)
    v = b * np.exp2(-e.astype(np.float64))[:, :, None]
    low, frac = GRID[fmt]
    step = np.exp2(np.maximum(np.frexp(v)[1] - 1, low) - frac)
    r = np.minimum(np.abs(np.rint(v / step) * step), MOST[fmt])
    table = element_values(fmt)[:8 if fmt == E2M1 else 127]
    codes = np.searchsorted(table, r)
    assert (table[codes] == r).all()
    codes = codes + np.where(np.signbit(v), 8 if fmt == E2M1 else 128, 0)
    codes = np.where(bad[:, :, None], 0, codes)
    return codes.reshape(x.shape).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def pack(codes, fmt):
    return codes if fmt == E4M3 else codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(rows, fmt):
    if fmt == E4M3:
        return rows
    return np.stack([rows & 15, rows >> 4], -1).reshape(rows.shape[0], -1)


def scale_values(s):
    return np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127.0))


def dequantize(codes, scales, fmt):
    v = element_values(fmt)[codes].reshape(codes.shape[0], -1, 32)
    return (v * scale_values(scales)[:, :, None]).reshape(codes.shape)


def product(a, w, fmt, y_type):
    """(a . w^T, bound of |y - a . w^T|) of float64 values, K in instructions of 64 or 128.

    fp32 addition: the matrix unit adds the sums of eights to the accumulator, cutting each addend below 2^-24 of
    the largest: with K / 8 sums, K / 64 accumulator updates and three joins of partial results, every cut at
    most 2^-23 of the largest running sum or block.  E4M3 with a 16-bit result: each of the seven smaller products of
    an eight loses at most 2^-13 of the largest.  Rounding the result: half a step of its type (fp16: half of its
    smallest step, 2^-25, at least)."""
    K = a.shape[1]
    p = a[:, None, :] * w[None]
    blocks = p.reshape(p.shape[0], p.shape[1], -1, 32)
    y = p.sum(2)
    largest = np.abs(np.cumsum(blocks.sum(3), 2)).max(2) + np.abs(blocks).sum(3).max(2)
    # a wave of a split product starts at any batch: its partial sums are differences of running sums
    tol = 2.0 ** -23 * (K / 8 + K / 32 + 4) * 2 * largest
    if fmt == E4M3 and y_type != F32:
        tol = tol + 7 * 2.0 ** -13 * np.abs(p).reshape(p.shape[0], p.shape[1], -1, 8).max(3).sum(2)
    tol = tol + HALF_STEP[y_type] * (np.abs(y) + tol)
    if y_type == F16:
        tol = tol + 2.0 ** -25
    return y, tol + 1e-37
