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
