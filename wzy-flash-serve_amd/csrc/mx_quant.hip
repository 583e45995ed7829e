// mx_quant.hip -- rows to and from the microscaled (MX) formats: quantise, dequantise, residual addition +
// RMSNorm, SwiGLU.  All are bound by memory: each value is read and written once.
//
// A block of 32 values sits on the four lanes of a DPP quad, 8 consecutive values a lane: 16- or 32-byte loads, the
// block's maximum by two quad permutations, 4 or 8 bytes of codes stored per lane.  (A large copy on this card reads and
// writes 5.0 TB/s.)
#include "wzy_mx.h"

using namespace wzy;

namespace {

constexpr int QT = 256;                       // threads of the flat kernels: 64 blocks at a time
constexpr int QU = 4;                         // blocks a quad holds at once: their loads are in flight together

// SwiGLU, g / (1 + exp(-g)) * u.  exp(x) = 2^n * p: x * log2(e) = n + f taken to 48 bits, p = 2^f by the hardware's instruction.  Right to 4 * 2^-23
// (p and the reciprocal one last bit each, half of one for each of three roundings); __expf alone is off by |g| * 2^-24.
WZY_DEV float exp_parts(float x, int& n) {
    const float r = rintf(x * 0x1.715476p+0f);
    n = (int) r;
    return __builtin_amdgcn_exp2f(fmaf(x, 0x1.4ae0cp-26f, fmaf(x, 0x1.715476p+0f, -r)));
}
WZY_DEV float swiglu(float g, float u) {                          // g >= -87
    int n;
    const float p = exp_parts(fmaxf(-g, -100.0f), n);             // (a NaN of g comes back below)
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_ldexpf(p, n)) * u;
}
// g < -87, as g * exp(g) / (1 + exp(g)) * u: exp(-g) is past fp32's range from -88.8 on, where a large u still makes values that E4M3 under a
// scale of 2^-127 holds.  2^n multiplies half before u and half after it, so that no step leaves the range before the result does.
WZY_DEV float swiglu_far(float g, float u) {
    int n;
    const float p = exp_parts(fmaxf(g, -400.0f), n);              // the product is 0 long before; 1 + exp(g) is 1
    return __builtin_ldexpf(__builtin_ldexpf(g * p, n >> 1) * u, n - (n >> 1));
}

// ---- quantise and SwiGLU: blocks in flat order over rows x cols / 32 ------------------------------------
// Flat, so that any shape fills the chip: a row is a division, no workgroup belongs to one.  151,936 x 2,048 bf16 to E2M1 164 us
// (4.8 TB/s); SwiGLU of 81,920 x 512 bf16 41 us (5.1 TB/s); 4 x 2,048 fp32 2.1 us on the GPU, 3.6 a call.
template <int TYPE, int FMT, bool GLU>
__global__ void __launch_bounds__(QT) mx_quant_kernel(const void* __restrict__ x, const void* __restrict__ up, int64_t ld,
                                                      uint32_t blocks, FastDiv per_row, MxView q) {
    const int sub = threadIdx.x & 3;
    const uint32_t b0 = blockIdx.x * (uint32_t) (QT / 4 * QU) + (threadIdx.x >> 2);
    float v[QU][8], u[GLU ? QU : 1][8];
    uint32_t row[QU], col[QU];
#pragma unroll
    for (int i = 0; i < QU; ++i) {
        const uint32_t b = min(b0 + i * (QT / 4), blocks - 1);
        row[i] = fast_div(b, per_row);
        col[i] = b - row[i] * per_row.d;
        const size_t at = (size_t) row[i] * ld + 32 * (size_t) col[i] + 8 * sub;
        load8<TYPE>(x, at, v[i]);
        if constexpr (GLU) load8<TYPE>(up, at, u[i]);
    }
#pragma unroll
    for (int i = 0; i < QU; ++i) {
        if constexpr (GLU) {
            float low = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) low = fminf(low, v[i][j]);
            if (low >= -87.0f) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = swiglu(v[i][j], u[i][j]);
            } else {                                              // rare: not worth the common path's time
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] < -87.0f ? swiglu_far(v[i][j], u[i][j]) : swiglu(v[i][j], u[i][j]);
            }
        }
        const int byte = mx_block_scale<FMT>(v[i]);
        const uint2 c = mx_block_codes<FMT>(v[i], byte);
        if (b0 + i * (QT / 4) < blocks) mx_block_store<FMT>(q, row[i], col[i], sub, c, byte);
    }
}

// ---- dequantise ------------------------------------------------------------------------------------------
// The same walk the other way.  E2M1 to 151,936 x 2,048 bf16 120 us (6.6 TB/s).
template <int TYPE, int FMT>
__global__ void __launch_bounds__(QT) mx_dequant_kernel(MxView q, uint32_t blocks, FastDiv per_row, void* __restrict__ y, int64_t ld) {
    const int sub = threadIdx.x & 3;
    const uint32_t b0 = blockIdx.x * (uint32_t) (QT / 4 * QU) + (threadIdx.x >> 2);
    uint2 c[QU];
    uint32_t s[QU], row[QU], col[QU];
#pragma unroll
    for (int i = 0; i < QU; ++i) {
        const uint32_t b = min(b0 + i * (QT / 4), blocks - 1);
        row[i] = fast_div(b, per_row);
        col[i] = b - row[i] * per_row.d;
        const uint8_t* const p = q.codes + (size_t) row[i] * q.ldc;
        if constexpr (FMT == WZY_MX_E2M1) c[i] = make_uint2(*(const uint32_t*) (p + 16 * (size_t) col[i] + 4 * sub), 0);
        else c[i] = *(const uint2*) (p + 32 * (size_t) col[i] + 8 * sub);
        s[i] = q.scales[(size_t) row[i] * q.lds + col[i]];
    }
#pragma unroll
    for (int i = 0; i < QU; ++i) {
        mx_f32x2 p[4];
        if constexpr (FMT == WZY_MX_E2M1) {
            p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i].x, 1.0f, 0);
            p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i].x, 1.0f, 1);
            p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i].x, 1.0f, 2);
            p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i].x, 1.0f, 3);
        } else {
            p[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int) c[i].x, false);
            p[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int) c[i].x, true);
            p[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int) c[i].y, false);
            p[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int) c[i].y, true);
        }
        const float sc = mx_scale_value(s[i]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p[j >> 1][j & 1] * sc;
        if (b0 + i * (QT / 4) < blocks) store8<TYPE>(y, (size_t) row[i] * ld + 32 * (size_t) col[i] + 8 * sub, v);
    }
}

// ---- residual addition + RMSNorm: one workgroup a row -------------------------------------------------------
// Thread t holds the 8-value pieces t, t + threads, ... of the row in registers: one read, the sum of squares over the
// workgroup, one write.  NV pieces a thread, 64 .. 512 threads.  The sum and what follows are in 64 bits: squares of fp32 values are exact
// there and in range, and a normed value is rounded once before it becomes a code; beside the memory traffic the operations are free
// (fp32 sums: the same times).  8,191 x 2,560 bf16 with residual, sum, y and E4M3 out 37 us (5.1 TB/s); one row of 2,048 2.1 us on the GPU,
// 4.3 a call.
constexpr int NORM_MAX = 16384;
struct NormArgs {
    const void* x; const void* res; const float* gamma;
    void* sum; void* y;
    MxView q;
    int64_t ld;
    double inv_cols;
    float eps;
    int cols;
};
template <int CTRL>
WZY_DEV double add_dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t) dpp_i<CTRL>((int) b), hi = (uint32_t) dpp_i<CTRL>((int) (b >> 32));
    return v + __builtin_bit_cast(double, (uint64_t) hi << 32 | lo);
}
WZY_DEV double lane64(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t) (uint32_t) __builtin_amdgcn_readlane((int) (b >> 32), lane) << 32 |
                                          (uint32_t) __builtin_amdgcn_readlane((int) b, lane));
}
WZY_DEV double wave_sum64(double v) {
    v = add_dpp64<DPP_XOR1>(v);
    v = add_dpp64<DPP_XOR2>(v);
    v = add_dpp64<DPP_HALF_MIRROR>(v);
    v = add_dpp64<DPP_MIRROR>(v);
    return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}
template <int TYPE, int NV>
__global__ void __launch_bounds__(512) mx_norm_kernel(NormArgs a) {
    __shared__ double s_red[8];
    const size_t at0 = (size_t) blockIdx.x * a.ld;
    const int tid = threadIdx.x, nt = blockDim.x, pieces = a.cols / 8;
    float v[NV][8];
    double ss = 0.;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = tid + i * nt;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (p < pieces) {
            load8<TYPE>(a.x, at0 + 8 * (size_t) p, v[i]);
            if (a.res) {
                float r[8];
                load8<TYPE>(a.res, at0 + 8 * (size_t) p, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = round_to<TYPE>(v[i][j] + r[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fma((double) v[i][j], (double) v[i][j], ss);
    }
    ss = wave_sum64(ss);
    if ((tid & 63) == 0) s_red[tid >> 6] = ss;
    __syncthreads();
    double tot = 0.;
    for (int w = 0; w < nt / 64; ++w) tot += s_red[w];
    // one Newton step from the instruction's approximation, but where that is 0, infinite or NaN
    const double m = fma(tot, a.inv_cols, (double) a.eps), r0 = __builtin_amdgcn_rsq(m);
    const double r = m > 0. && m < __builtin_inf() ? fma(0.5 * r0, fma(-m * r0, r0, 1.0), r0) : r0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = tid + i * nt;
        if (p >= pieces) continue;                 // whole quads: pieces is a multiple of 4
        if (a.sum) store8<TYPE>(a.sum, at0 + 8 * (size_t) p, v[i]);
        float g[8];
        load8<WZY_F32>(a.gamma, 8 * (size_t) p, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = (float) ((double) v[i][j] * r * (double) g[j]);
        if (a.y) store8<TYPE>(a.y, at0 + 8 * (size_t) p, g);
        if (a.q.codes) {
            const int byte = mx_block_scale<WZY_MX_E4M3>(g);
            mx_block_store<WZY_MX_E4M3>(a.q, blockIdx.x, (uint32_t) p >> 2, p & 3, mx_block_codes<WZY_MX_E4M3>(g, byte), byte);
        }
    }
}

int check_shape(const char* who, int rows, int cols) {
    WZY_REQUIRE(rows >= 0 && cols >= 32 && cols % 32 == 0 && (int64_t) rows * (cols / 32) < (int64_t) 1 << 31,
                "%s: %d rows of %d (cols a multiple of 32, rows * cols / 32 below 2^31)", who, rows, cols);
    return WZY_OK;
}
uint32_t flat_grid(uint32_t blocks) { return (blocks + QT / 4 * QU - 1) / (QT / 4 * QU); }

}  // namespace

extern "C" int wzy_mx_quantize(const void* x, int x_type, int64_t ldx, int rows, int cols, const wzy_mx_mat* q, void* stream) {
    const char* const who = "wzy_mx_quantize";
    MxView v;
    WZY_TRY(check_shape(who, rows, cols));
    WZY_TRY(mx_check_type(who, x_type));
    if (rows == 0) return WZY_OK;
    WZY_TRY(mx_check_rows(who, "x", x, x_type, ldx, cols));
    WZY_TRY(mx_check_mat(who, "q", q, cols, v));
    const uint32_t blocks = (uint32_t) rows * (uint32_t) (cols / 32);
    return mx_with_type(x_type, [&](auto t) {
        if (q->fmt == WZY_MX_E2M1)
            mx_quant_kernel<t(), WZY_MX_E2M1, false><<<flat_grid(blocks), QT, 0, as_stream(stream)>>>(x, nullptr, ldx, blocks, FastDiv(cols / 32), v);
        else
            mx_quant_kernel<t(), WZY_MX_E4M3, false><<<flat_grid(blocks), QT, 0, as_stream(stream)>>>(x, nullptr, ldx, blocks, FastDiv(cols / 32), v);
        WZY_LAUNCH_CHECK();
        return WZY_OK;
    });
}

extern "C" int wzy_mx_swiglu(const void* gate, const void* up, int type, int64_t ld, int rows, int cols, const wzy_mx_mat* q,
                             void* stream) {
    const char* const who = "wzy_mx_swiglu";
    MxView v;
    WZY_TRY(check_shape(who, rows, cols));
    WZY_TRY(mx_check_type(who, type));
    if (rows == 0) return WZY_OK;
    WZY_TRY(mx_check_rows(who, "gate", gate, type, ld, cols));
    WZY_TRY(mx_check_rows(who, "up", up, type, ld, cols));
    WZY_TRY(mx_check_mat(who, "q", q, cols, v));
    WZY_REQUIRE(q->fmt == WZY_MX_E4M3, "%s: q is E4M3", who);
    const uint32_t blocks = (uint32_t) rows * (uint32_t) (cols / 32);
    return mx_with_type(type, [&](auto t) {
        mx_quant_kernel<t(), WZY_MX_E4M3, true><<<flat_grid(blocks), QT, 0, as_stream(stream)>>>(gate, up, ld, blocks, FastDiv(cols / 32), v);
        WZY_LAUNCH_CHECK();
        return WZY_OK;
    });
}

extern "C" int wzy_mx_dequantize(const wzy_mx_mat* q, int rows, int cols, void* y, int y_type, int64_t ldy, void* stream) {
    const char* const who = "wzy_mx_dequantize";
    MxView v;
    WZY_TRY(check_shape(who, rows, cols));
    WZY_TRY(mx_check_type(who, y_type));
    if (rows == 0) return WZY_OK;
    WZY_TRY(mx_check_mat(who, "q", q, cols, v));
    WZY_TRY(mx_check_rows(who, "y", y, y_type, ldy, cols));
    const uint32_t blocks = (uint32_t) rows * (uint32_t) (cols / 32);
    return mx_with_type(y_type, [&](auto t) {
        if (q->fmt == WZY_MX_E2M1)
            mx_dequant_kernel<t(), WZY_MX_E2M1><<<flat_grid(blocks), QT, 0, as_stream(stream)>>>(v, blocks, FastDiv(cols / 32), y, ldy);
        else
            mx_dequant_kernel<t(), WZY_MX_E4M3><<<flat_grid(blocks), QT, 0, as_stream(stream)>>>(v, blocks, FastDiv(cols / 32), y, ldy);
        WZY_LAUNCH_CHECK();
        return WZY_OK;
    });
}

extern "C" int wzy_mx_add_rmsnorm(const void* x, const void* residual, int type, int64_t ld, const float* gamma, float eps,
                                  int rows, int cols, void* sum, void* y, const wzy_mx_mat* q, void* stream) {
    const char* const who = "wzy_mx_add_rmsnorm";
    NormArgs a{};
    WZY_TRY(check_shape(who, rows, cols));
    WZY_TRY(mx_check_type(who, type));
    WZY_REQUIRE(cols <= NORM_MAX, "%s: %d columns (at most %d)", who, cols, NORM_MAX);
    WZY_REQUIRE(eps >= 0.f, "%s: eps %g", who, (double) eps);
    WZY_REQUIRE(sum || y || q, "%s: no output", who);
    if (rows == 0) return WZY_OK;
    WZY_TRY(mx_check_rows(who, "x", x, type, ld, cols));
    if (residual) WZY_TRY(mx_check_rows(who, "residual", residual, type, ld, cols));
    if (sum) WZY_TRY(mx_check_rows(who, "sum", sum, type, ld, cols));
    if (y) WZY_TRY(mx_check_rows(who, "y", y, type, ld, cols));
    WZY_REQUIRE(gamma && (uintptr_t) gamma % 16 == 0, "%s: gamma at %p (16-byte aligned)", who, (const void*) gamma);
    WZY_REQUIRE(!y || y != sum, "%s: y and sum are one buffer", who);
    if (q) {
        WZY_TRY(mx_check_mat(who, "q", q, cols, a.q));
        WZY_REQUIRE(q->fmt == WZY_MX_E4M3, "%s: q is E4M3", who);
    }
    a.x = x; a.res = residual; a.gamma = gamma; a.sum = sum; a.y = y; a.ld = ld; a.inv_cols = 1.0 / cols; a.eps = eps; a.cols = cols;
    const int pieces = cols / 8, nv = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : 4;
    const int threads = (int) align_up((size_t) (pieces + nv - 1) / nv, 64);
    WZY_REQUIRE((int64_t) rows * threads < (int64_t) 1 << 32, "%s: %d rows of %d (at most %lld in a call)", who, rows, cols,
                ((1LL << 32) - 1) / threads);
    return mx_with_type(type, [&](auto t) {
        if (nv == 1) mx_norm_kernel<t(), 1><<<rows, threads, 0, as_stream(stream)>>>(a);
        else if (nv == 2) mx_norm_kernel<t(), 2><<<rows, threads, 0, as_stream(stream)>>>(a);
        else mx_norm_kernel<t(), 4><<<rows, threads, 0, as_stream(stream)>>>(a);
        WZY_LAUNCH_CHECK();
        return WZY_OK;
    });
}
