"""Microscaled (MX) operators on the CPU: refusals, and the 64-bit formulation the GPU tests use against torch's
own 8-bit types."""
import ctypes as C

import numpy as np
import pytest

import mx_ref as R
import wzy_amd
from mx_ref import BF16, E2M1, E4M3, F16, F32

EINVAL = -1
A = 4096                                          # an aligned address that is never read: sizes are checked first


def mat(fmt=E4M3, codes=A, scales=A, ldc=0, lds=0):
    return C.byref(wzy_amd.MxMat(codes, scales, ldc, lds, fmt))


def refused(wz, name, *args):
    rc = getattr(wz.dll, name)(*args)
    assert rc == EINVAL, (name, args, rc)
    assert name in wz.wzy_last_error().decode()


BAD_MATS = [dict(codes=None), dict(scales=None), dict(fmt=2), dict(fmt=-1), dict(codes=A + 8), dict(ldc=32), dict(ldc=72),
            dict(ldc=-64), dict(ldc=1 << 23), dict(lds=1), dict(lds=-2)]


@pytest.mark.parametrize("bad", BAD_MATS, ids=str)
def test_bad_matrices_are_refused(wz, bad):
    q = mat(**bad)
    refused(wz, "wzy_mx_quantize", A, F32, 64, 4, 64, q, None)
    refused(wz, "wzy_mx_dequantize", q, 4, 64, A, F32, 64, None)
    refused(wz, "wzy_mx_add_rmsnorm", A, None, F32, 64, A, 1e-6, 4, 64, None, None, q, None)
    refused(wz, "wzy_mx_swiglu", A, A, F32, 64, 4, 64, q, None)
    refused(wz, "wzy_mx_gemm", q, mat(E2M1), 4, 8, 64, A, F32, 8, None)
    refused(wz, "wzy_mx_grouped_gemm", q, 4, None, mat(E2M1), A, 2, 4, 8, 64, A, F32, 8, None)
    if bad.get("ldc") != 32:                      # 32 bytes hold a row of 4-bit codes
        q = mat(**{"fmt": E2M1, **bad})
        refused(wz, "wzy_mx_gemm", mat(), q, 4, 8, 64, A, F32, 8, None)
        refused(wz, "wzy_mx_grouped_gemm", mat(), 4, None, q, A, 2, 4, 8, 64, A, F32, 8, None)


@pytest.mark.parametrize("rows,cols", [(-1, 64), (4, 0), (4, 48), (4, -32), (2 ** 31 - 1, 64)])
def test_bad_row_shapes_are_refused(wz, rows, cols):
    refused(wz, "wzy_mx_quantize", A, F32, 64, rows, cols, mat(), None)
    refused(wz, "wzy_mx_dequantize", mat(), rows, cols, A, F32, 64, None)
    refused(wz, "wzy_mx_add_rmsnorm", A, None, F32, 64, A, 1e-6, rows, cols, None, None, mat(), None)
    refused(wz, "wzy_mx_swiglu", A, A, F32, 64, rows, cols, mat(), None)


def test_bad_rows_types_and_options_are_refused(wz):
    for x, t, ld in [(None, F32, 64), (A + 4, F32, 64), (A, F32, 63), (A, F32, 66), (A, BF16, 68), (A, 3, 64), (A, -1, 64)]:
        refused(wz, "wzy_mx_quantize", x, t, ld, 4, 64, mat(), None)
        refused(wz, "wzy_mx_dequantize", mat(), 4, 64, x, t, ld, None)
        refused(wz, "wzy_mx_add_rmsnorm", x, None, t, ld, A, 1e-6, 4, 64, None, None, mat(), None)
        refused(wz, "wzy_mx_swiglu", x, A, t, ld, 4, 64, mat(), None)
        refused(wz, "wzy_mx_swiglu", A, x, t, ld, 4, 64, mat(), None)
    n = ("wzy_mx_add_rmsnorm", A, None, F32)
    refused(wz, *n, 64, A, 1e-6, 4, 64, None, None, None, None)            # no output
    refused(wz, *n, 64, None, 1e-6, 4, 64, None, A, None, None)            # no gamma
    refused(wz, *n, 64, A + 8, 1e-6, 4, 64, None, A, None, None)
    refused(wz, *n, 64, A, -1e-6, 4, 64, None, A, None, None)
    refused(wz, *n, 64, A, float("nan"), 4, 64, None, A, None, None)
    refused(wz, *n, 16416, A, 1e-6, 4, 16416, None, A, None, None)         # too wide
    refused(wz, *n, 32, A, 1e-6, 2 ** 26, 32, None, A, None, None)         # more rows than a launch holds
    refused(wz, *n, 16384, A, 1e-6, 2 ** 23, 16384, None, A, None, None)
    refused(wz, *n, 64, A, 1e-6, 4, 64, A, A, None, None)                  # sum and y in one buffer
    refused(wz, *n, 64, A, 1e-6, 4, 64, None, None, mat(E2M1), None)
    refused(wz, "wzy_mx_add_rmsnorm", A, A + 8, F32, 64, A, 1e-6, 4, 64, None, A, None, None)
    refused(wz, "wzy_mx_swiglu", A, A, F32, 64, 4, 64, mat(E2M1), None)


def test_bad_products_are_refused(wz):
    w = mat(E2M1)
    for M, N, K, y, t, ldy in [(-1, 8, 64, A, F32, 8), (4, -8, 64, A, F32, 8), (4, 8, 0, A, F32, 8), (4, 8, 40, A, F32, 8),
                               (4, 8, 2 ** 20 + 32, A, F32, 8), (4, 8, 64, None, F32, 8), (4, 8, 64, A + 2, F32, 8),
                               (4, 8, 64, A + 1, BF16, 8), (4, 8, 64, A, 3, 8), (4, 8, 64, A, F16, 7)]:
        refused(wz, "wzy_mx_gemm", mat(), w, M, N, K, y, t, ldy, None)
        refused(wz, "wzy_mx_grouped_gemm", mat(), 4, None, w, A, 2, M, N, K, y, t, ldy, None)
    refused(wz, "wzy_mx_gemm", mat(), mat(E4M3), 4, 8, 64, A, F32, 8, None)
    refused(wz, "wzy_mx_gemm", None, w, 4, 8, 64, A, F32, 8, None)
    refused(wz, "wzy_mx_gemm", mat(), None, 4, 8, 64, A, F32, 8, None)
    g = ("wzy_mx_grouped_gemm", mat())
    refused(wz, *g, 4, None, w, None, 2, 4, 8, 64, A, F32, 8, None)        # no offsets
    refused(wz, *g, 3, None, w, A, 2, 4, 8, 64, A, F32, 8, None)           # fewer rows than entries, not gathered
    refused(wz, *g, -1, A, w, A, 2, 4, 8, 64, A, F32, 8, None)
    refused(wz, *g, 0, A, w, A, 2, 4, 8, 64, A, F32, 8, None)
    refused(wz, *g, 4, None, w, A, 0, 4, 8, 64, A, F32, 8, None)
    refused(wz, *g, 4, None, w, A, 65537, 4, 8, 64, A, F32, 8, None)


def test_formulation_against_torch_types():
    import torch
    assert np.array_equal(R.element_values(E4M3), torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy(),
                          equal_nan=True)
    s = np.arange(256, dtype=np.uint8)
    assert np.array_equal(R.scale_values(s), torch.from_numpy(s).view(torch.float8_e8m0fnu).double().numpy(), equal_nan=True)
    x = np.random.default_rng(0).standard_normal((64, 256)) * 3
    x[:, ::32] = 300.0                            # scale 1 in every block
    codes, scales = R.quantize(x, E4M3)
    assert (scales == 127).all()
    t = torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert (codes == t).mean() > 0.999 and (codes == R.quantize(x.astype(np.float32), E4M3)[0]).mean() > 0.999
    b, v = R.typed(x.astype(np.float32), BF16)
    assert np.array_equal(b, torch.from_numpy(x).float().to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16))


def test_formulation_of_small_cases():
    x = np.zeros((1, 64))
    x[0, :9] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25]
    x[0, 32:36] = [7.9, 6.1, -0.0, -7.0]
    c, s = R.quantize(x, E2M1)
    assert s.tolist() == [[127, 127]]
    assert c[0, :9].tolist() == [6, 0, 2, 2, 4, 4, 6, 6, 8] and c[0, 32:36].tolist() == [7, 7, 8, 15]
    c, s = R.quantize(np.full((1, 32), 2.0 ** -140), E2M1)
    assert s[0, 0] == 0 and (c == 0).all()
    assert (R.quantize(np.zeros((1, 32)), E4M3)[1] == 0).all()
    r, tol = R.product(np.ones((1, 32)), np.ones((1, 32)), E2M1, F32)
    assert r[0, 0] == 32 and 0 < tol[0, 0] < 1e-2
