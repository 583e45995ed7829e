// wzy_mx.h -- shared by the microscaled (MX) kernels: element types, scales, block quantisation, host checks.
#pragma once
#include <type_traits>

#include "../../include/wzy_mx.h"
#include "wzy_device.h"
#include "wzy_host.h"

namespace wzy {

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 mx_f16x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));

// An MX matrix as kernels take it (row strides in bytes).
struct MxView {
    uint8_t* codes;
    uint8_t* scales;
    int64_t ldc, lds;
};

constexpr int mx_emax(int fmt) { return fmt == WZY_MX_E2M1 ? 2 : 8; }
inline int64_t mx_row_bytes(int fmt, int cols) { return fmt == WZY_MX_E2M1 ? cols / 2 : cols; }
inline int mx_type_bytes(int type) { return type == WZY_F32 ? 4 : 2; }

// Host checks of an MX operand; fills the view.
inline int mx_check_mat(const char* who, const char* what, const wzy_mx_mat* q, int cols, MxView& v) {
    WZY_REQUIRE(q && q->codes && q->scales, "%s: %s is null", who, what);
    WZY_REQUIRE(q->fmt == WZY_MX_E2M1 || q->fmt == WZY_MX_E4M3, "%s: %s has format %d", who, what, q->fmt);
    v.codes = q->codes;
    v.scales = q->scales;
    v.ldc = q->ld_codes ? q->ld_codes : mx_row_bytes(q->fmt, cols);
    v.lds = q->ld_scales ? q->ld_scales : cols / 32;
    WZY_REQUIRE(v.ldc >= mx_row_bytes(q->fmt, cols) && v.ldc < (1 << 23) && v.ldc % 16 == 0 && (uintptr_t) q->codes % 16 == 0,
                "%s: codes of %s: rows of %lld bytes at %p (16-byte aligned, at least %lld, below 2^23)", who, what,
                (long long) v.ldc, (void*) q->codes, (long long) mx_row_bytes(q->fmt, cols));
    WZY_REQUIRE(v.lds >= cols / 32 && v.lds < (1 << 23), "%s: scales of %s: rows of %lld bytes (at least %d, below 2^23)", who,
                what, (long long) v.lds, cols / 32);
    return WZY_OK;
}
inline int mx_check_type(const char* who, int type) {
    WZY_REQUIRE(type == WZY_F32 || type == WZY_BF16 || type == WZY_F16, "%s: type %d", who, type);
    return WZY_OK;
}
// rows of 8-element accesses: 16-byte aligned base and stride
inline int mx_check_rows(const char* who, const char* what, const void* p, int type, int64_t ld, int cols) {
    WZY_REQUIRE(p, "%s: %s is null", who, what);
    WZY_REQUIRE(ld >= cols && ld <= (int64_t) 1 << 40 && ld * mx_type_bytes(type) % 16 == 0 && (uintptr_t) p % 16 == 0,
                "%s: rows of %s: stride %lld at %p (16-byte aligned, at least %d elements)", who, what, (long long) ld, p, cols);
    return WZY_OK;
}

// n / d for n < 2^31 by one multiplication (d >= 1): q = (n + mulhi(n, m)) >> s, s = ceil(log2 d),
// m = floor(2^32 (2^s - d) / d) + 1.
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div), s(0) {
        while ((1ull << s) < d) ++s;
        m = (uint32_t) ((((1ull << s) - d) << 32) / d + 1);
    }
};
WZY_DEV uint32_t fast_div(uint32_t n, const FastDiv& f) { return (n + __umulhi(n, f.m)) >> f.s; }

// ---- rows of fp32 / bf16 / fp16: 8 consecutive elements per lane --------------------------------------
template <int TYPE>
WZY_DEV void load8(const void* p, size_t i, float (&v)[8]) {
    if constexpr (TYPE == WZY_F32) {
        const float4 a = ((const float4*) ((const float*) p + i))[0], b = ((const float4*) ((const float*) p + i))[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *(const uint4*) ((const uint16_t*) p + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (TYPE == WZY_BF16) {
                v[2 * j] = bf16_lo(w[j]);
                v[2 * j + 1] = bf16_hi(w[j]);
            } else {
                v[2 * j] = h16_to_f((uint16_t) w[j]);
                v[2 * j + 1] = h16_to_f((uint16_t) (w[j] >> 16));
            }
        }
    }
}
// two values rounded to nearest even and packed
template <int TYPE>
WZY_DEV uint32_t pack2(float a, float b) {
    if constexpr (TYPE == WZY_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_f32x2{a, b}, mx_bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_f32x2{a, b}, mx_f16x2));
}
template <int TYPE>
WZY_DEV void store8(void* p, size_t i, const float (&v)[8]) {
    if constexpr (TYPE == WZY_F32) {
        ((float4*) ((float*) p + i))[0] = make_float4(v[0], v[1], v[2], v[3]);
        ((float4*) ((float*) p + i))[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *(uint4*) ((uint16_t*) p + i) = make_uint4(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]), pack2<TYPE>(v[4], v[5]),
                                                   pack2<TYPE>(v[6], v[7]));
    }
}
template <int TYPE>
WZY_DEV float round_to(float v) {
    if constexpr (TYPE == WZY_F32) return v;
    else if constexpr (TYPE == WZY_BF16) return (float) (__bf16) v;
    else return round_h16(v);
}

// ---- one block of 32 values on the four lanes of a quad, 8 consecutive values each ---------------------
// Scale byte of the block (the same in all four lanes).  The maximum is taken over the magnitudes' bits, so a NaN
// or an infinity (exponent 255) wins it; the exponent of a denormal is 0 and its byte 0, 2^-127, as the format's
// lowest scale wants.
template <int FMT>
WZY_DEV int mx_block_scale(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    m = max(m, (uint32_t) dpp_i<DPP_XOR1>((int) m));
    m = max(m, (uint32_t) dpp_i<DPP_XOR2>((int) m));
    const int e = (int) (m >> 23);
    return e == 255 ? 255 : max(e - mx_emax(FMT), 0);
}
// The lane's 8 codes under that scale: x * 2^(127 - byte) is exact (or, far below the smallest element, rounds to
// zero either way); the conversion instructions round to nearest even; E2M1's saturates by itself, E4M3's turns
// values past 464 into NaN and is limited before.  E2M1: 4 bytes in .x.
template <int FMT>
WZY_DEV uint2 mx_block_codes(const float (&v)[8], int byte) {
    const float up = __builtin_bit_cast(float, (uint32_t) (254 - min(byte, 253)) << 23);
    uint32_t lo = 0, hi = 0;
    if constexpr (FMT == WZY_MX_E2M1) {
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, v[0] * up, v[1] * up, 1.0f, 0);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, v[2] * up, v[3] * up, 1.0f, 1);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, v[4] * up, v[5] * up, 1.0f, 2);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, v[6] * up, v[7] * up, 1.0f, 3);
    } else {
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = __builtin_amdgcn_fmed3f(v[i] * up, -448.0f, 448.0f);
        lo = (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        lo = (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], (int) lo, true);
        hi = (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
        hi = (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], (int) hi, true);
    }
    return byte == 255 ? make_uint2(0, 0) : make_uint2(lo, hi);
}
// block b (of cols / 32) of row r: the lane's codes, and the scale by the quad's first lane
template <int FMT>
WZY_DEV void mx_block_store(const MxView& q, size_t r, uint32_t b, int sub, uint2 codes, int byte) {
    uint8_t* const c = q.codes + r * q.ldc;
    if constexpr (FMT == WZY_MX_E2M1) *(uint32_t*) (c + 16 * (size_t) b + 4 * sub) = codes.x;
    else *(uint2*) (c + 32 * (size_t) b + 8 * sub) = codes;
    if (sub == 0) q.scales[r * q.lds + b] = (uint8_t) byte;
}
// what a scale byte stands for (2^-127 is an fp32 denormal)
WZY_DEV float mx_scale_value(uint32_t byte) {
    return __builtin_bit_cast(float, byte == 255 ? 0x7FC00000u : byte == 0 ? 0x00400000u : byte << 23);
}

// run f with the compile-time value of a runtime type
template <class F>
int mx_with_type(int type, F&& f) {
    switch (type) {
        case WZY_F32: return f(std::integral_constant<int, WZY_F32>());
        case WZY_BF16: return f(std::integral_constant<int, WZY_BF16>());
        default: return f(std::integral_constant<int, WZY_F16>());
    }
}

}  // namespace wzy
