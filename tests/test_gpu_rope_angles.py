"""Angles of the rotary operator (include/wzy_paged.h) to what 64 bits give: sines next to a border of fp32's rounding."""
import math

import numpy as np
import pytest

import wzy_amd
from test_gpu_paged import F32, ints, ref

pytestmark = pytest.mark.gpu
DA = wzy_amd.DeviceArray


@pytest.mark.parametrize("degrees", [30, 44, 46, 50, 60, 66])
def test_rope_turns_are_rounded_as_the_sine_is(wz, gpu, degrees):
    # sin t lies 2e-12 below the middle of two neighbouring fp32 numbers, so it rounds to the lower one where it is known to better
    # than that: 64-bit angles give 1e-16, series of 8 terms over an eighth of a turn 2e-14
    lower = np.float32(math.sin(math.radians(degrees))) + np.arange(64, dtype=np.float32) * np.float32(2.0 ** -20)
    middle = (lower.astype(np.float64) + np.nextafter(lower, np.float32(2)).astype(np.float64)) / 2
    t = np.arcsin(middle - 2e-12) / (2 * math.pi)                       # turns
    table = np.concatenate([t + 0.25 * quarter for quarter in range(4)] + [[1.0]])
    f, pos = DA.from_numpy(table), ints([1])
    x = np.zeros((1, 512), np.float32)
    x[0, :256] = 1.0                                                    # a pair (1, 0) becomes (cos, sin)
    d = DA.from_numpy(x)
    h = wzy_amd.Heads(d.ptr, 512, 512)
    wz.wzy_rope(ref(wzy_amd.RopeTab(f.ptr, 512, 0)), ref(h), F32, 1, 1, 512, pos.ptr, ref(h), None)
    c, s = d.numpy()[0].reshape(2, 4, 64)
    for got in (s[0], -c[1], -s[2], c[3]):
        np.testing.assert_array_equal(got, lower)


def test_rope_of_more_rows_than_one_launch_takes(wz, gpu):
    # 2^25 rows and a few, two a workgroup: rows at the ends and around the borders of launches equal small calls' rows
    rows, hd = (1 << 25) + 5, 512
    rng = np.random.default_rng(1)
    xd = DA.from_numpy(rng.integers(0x3F00, 0x4100, hd).astype(np.uint16))            # every row the same, in bf16
    pd = DA.from_numpy(np.arange(rows, dtype=np.int32))
    f = DA(hd // 2 + 1, np.float64)
    wz.wzy_rope_freqs(ref(wzy_amd.RopeCfg(1e4, 1.0, 1.0, 32.0, 1.0, 4096, hd, 0)), f.ptr, None)
    tab, x = wzy_amd.RopeTab(f.ptr, hd, 0), wzy_amd.Heads(xd.ptr, 0, hd)
    out = DA((rows + 1) * hd * 2, np.uint8)                                           # 34 GB
    wz.wzy_memset(out.ptr + rows * hd * 2, 0xA5, hd * 2, None)
    wz.wzy_rope(ref(tab), ref(x), wzy_amd.TYPE_BF16, rows, 1, hd, pd.ptr, ref(wzy_amd.Heads(out.ptr, hd, hd)), None)
    small = DA(3 * hd, np.uint16)
    got = np.zeros(3 * hd, np.uint16)
    for at in (0, (1 << 23) - 1, (1 << 24) - 1, (1 << 25) - 1, rows - 3):
        wz.wzy_rope(ref(tab), ref(x), wzy_amd.TYPE_BF16, 3, 1, hd, pd.ptr + 4 * at, ref(wzy_amd.Heads(small.ptr, hd, hd)), None)
        wz.wzy_memcpy_d2h(got.ctypes.data, out.ptr + at * hd * 2, got.nbytes, None)
        np.testing.assert_array_equal(got, small.numpy())
    wz.wzy_memcpy_d2h(got.ctypes.data, out.ptr + rows * hd * 2, hd * 2, None)
    assert (got[:hd].view(np.uint8) == 0xA5).all()
