/* wzy_mx.h -- microscaled (MX) operators of the MI355X (gfx950) library: 4- and 8-bit rows with one
 * power-of-two scale per 32 values (the OCP Microscaling formats MXFP4 and MXFP8), the steps that produce
 * them and the matrix products that take them.
 *
 * Conventions are those of wzy_kernels.h: device pointers, `stream` is a hipStream_t of the current device
 * passed as void* (NULL = the null stream), a status code comes back and wzy_last_error() says why a call was
 * refused.  Nothing here synchronizes, allocates, uses a workspace or keeps state between calls: calls on
 * several streams may overlap, and every call can be captured into a graph.  A refused call launches nothing.
 * An output shares no byte with an input or another output, but where its operator says so.
 * A call with no rows (rows, M or N of 0) is valid and launches nothing.
 *
 * Together: wzy_mx_add_rmsnorm hands its rows in 8 bits to wzy_mx_gemm (projections, LM head) or, gathered by
 * token, to wzy_mx_grouped_gemm (an expert's gate|up); wzy_mx_swiglu turns that product into the 8-bit rows of
 * the second grouped product.  The reference has no such formats: its 4-bit weights are the experts' NVFP4.
 */
#ifndef WZY_MX_H
#define WZY_MX_H

#include <stddef.h>
#include <stdint.h>

#include "wzy_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element formats of an MX matrix */
#define WZY_MX_E2M1 0     /* 4 bits: 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives; two per byte, even column in the low nibble */
#define WZY_MX_E4M3 1     /* 8 bits: up to 448, no infinities, code 0x7F / 0xFF = NaN */

/* types of rows that are not quantised */
#define WZY_F32 0
#define WZY_BF16 1
#define WZY_F16 2

/* rows x cols elements, cols a multiple of 32.  Row r's codes start at codes + r * ld_codes (cols / 2 bytes
 * of E2M1, cols bytes of E4M3), its cols / 32 scale bytes at scales + r * ld_scales.  A scale byte b stands
 * for 2^(b - 127), 255 for NaN (every value of its block is NaN).  ld_* in bytes, 0 = rows without gaps;
 * codes and ld_codes are multiples of 16, ld_codes below 2^23; scales have no alignment. */
typedef struct wzy_mx_mat {
    uint8_t* codes;
    uint8_t* scales;
    int64_t ld_codes, ld_scales;
    int fmt;
} wzy_mx_mat;

/* x [rows x cols] (x_type, row stride ldx elements) to MX: per block the scale 2^(floor(log2 max|x|) - emax),
 * emax = 2 (E2M1) or 8 (E4M3), at least 2^-127 (a block of zeros takes 2^-127); each element x / scale rounded to
 * nearest, ties to the even code, and limited to +-6 or +-448; the sign of zero is kept.  A block that holds a NaN or an
 * infinity becomes NaN: scale byte 255, codes 0.  Bit-exact: no step of it is rounded but the last.
 * x and its rows are aligned to 16 bytes; rows * cols / 32 below 2^31. */
int wzy_mx_quantize(const void* x, int x_type, int64_t ldx, int rows, int cols, const wzy_mx_mat* q, void* stream);

/* The values q stands for, y [rows x cols] (y_type, row stride ldy).  Exact in fp32 and, down to 2^-126, in bf16;
 * fp16 rounds to nearest (to an infinity past 65,504).  y and its rows are aligned to 16 bytes;
 * rows * cols / 32 below 2^31. */
int wzy_mx_dequantize(const wzy_mx_mat* q, int rows, int cols, void* y, int y_type, int64_t ldy, void* stream);

/* h = x + residual (added in fp32, rounded to `type`; residual NULL: h = x),
 * n = h * 1 / sqrt(mean(h^2) + eps) * gamma   (the mean over the row's cols; in 64 bits, rounded to fp32 once),
 * sum = h, y = n rounded to `type`, q = n as MX E4M3 (from fp32, as wzy_mx_quantize quantises).
 * x, residual, sum and y are [rows x cols] of `type` with one row stride ld (elements); gamma [cols] fp32.
 * Any of sum, y, q may be NULL, not all three; sum may be x or residual, and so may y where sum is NULL or another buffer.
 * Rows aligned to 16 bytes, gamma too; cols at most 16,384; at most 8,388,607 rows, and up to 2^26 - 1 of them where cols <= 512; eps >= 0 (a row of zeros with eps 0 is NaN). */
int wzy_mx_add_rmsnorm(const void* x, const void* residual, int type, int64_t ld, const float* gamma, float eps,
                       int rows, int cols, void* sum, void* y, const wzy_mx_mat* q, void* stream);

/* q = MX E4M3 of gate / (1 + exp(-gate)) * up, computed in fp32; gate and up [rows x cols] of `type` with row
 * stride ld (elements), for instance the halves of one gate|up row (up = gate + cols).  Rows aligned to 16 bytes;
 * rows * cols / 32 below 2^31. */
int wzy_mx_swiglu(const void* gate, const void* up, int type, int64_t ld, int rows, int cols, const wzy_mx_mat* q,
                  void* stream);

/* y [M x N] (y_type, row stride ldy >= N) = a [M x K] . w [N x K]^T, a of either format, w E2M1, K a multiple of
 * 32.  Sums are fp32, on the scaled MFMA instructions; products are whole, but for E4M3 rows with bf16 output: of each eight
 * consecutive k the seven smaller products lose up to 2^-13 of the largest (1e-5 of a sum of the usual size, below the output's
 * rounding unless the sum cancels).  E4M3 rows to fp32 and fp16 take up to twice that one's time for it.  A NaN scale or code makes its
 * row of y (a) or its column (w) NaN.
 * M = 1 .. 16 is the decode form: the weights stream once, at memory speed.  y is aligned to its element.
 * K at most 2^20. */
int wzy_mx_gemm(const wzy_mx_mat* a, const wzy_mx_mat* w, int M, int N, int K, void* y, int y_type, int64_t ldy,
                void* stream);

/* One product per group of entries: for offsets[g] <= e < offsets[g + 1],
 *   y[e] = a[row_ids[e]] . w_g^T,   w_g = rows g * N .. g * N + N - 1 of w (E2M1).
 * offsets [groups + 1] and row_ids [M] are device memory.  Groups may be empty; M is the number of rows of y and
 * at least offsets[groups], and rows of y in no group keep what they hold.  row_ids NULL: entry e reads row e.
 * a has a_rows >= 1 rows; an id outside 0 .. a_rows - 1 gives a row of zeros.  offsets are taken as they are but limited to 0 .. M;
 * where they decrease or overlap, which rows are computed is not specified (nothing outside y [M x N] is written).
 * 1 <= groups <= 65,536; shapes otherwise as wzy_mx_gemm. */
int wzy_mx_grouped_gemm(const wzy_mx_mat* a, int a_rows, const int* row_ids, const wzy_mx_mat* w, const int* offsets,
                        int groups, int M, int N, int K, void* y, int y_type, int64_t ldy, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* WZY_MX_H */
