// mx_gemm.hip -- products of microscaled (MX) rows on the scaled MFMA instructions of gfx950.
//
//   y[m, n] = sum over blocks b of 32:  2^(sa[m, b] + sw[n, b] - 254) * sum_i a[m, 32 b + i] * w[n, 32 b + i]
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies E2M1 by E2M1 or E4M3 codes as they lie in memory and applies the two
// scale bytes of each block of 32, with fp32 accumulators; nothing is dequantised.  Operand layout (measured): lane
// (q = lane / 16, r = lane % 16) holds row r and block q of 128 k.  E2M1: the block's 32 codes in order, 16 bytes.  E4M3: two
// 16-byte pieces, piece j holding the 16 k from 16 q + 64 j; the scale byte of lane group q still belongs to block q.  D:
// register i of lane (q, r) is row 4 q + i of the first operand, column r of the second.  w comes first, so a lane holds
// consecutive columns of y.  (32x32x64 does as much per cycle, and on data that is not zeros draws more power: registers
// alone, random codes, 6,770 against 8,130 TFLOP/s in E2M1, 4,350 against 4,700 with E4M3.)
//
// Precision (measured): an instruction adds the products of 8 consecutive k after cutting each to 13 bits below the
// largest of the eight, and the sums of eights in fp32.  E2M1 products span 9 bits: nothing is lost.  An E4M3 operand
// spans 19 bits.  For fp32 and fp16 outputs it is taken in two parts, codes with exponent bit 3 set and the others: each
// part spans 11 bits, so both products are whole, at twice the MFMA work.  For bf16 outputs the cuts stay: over activations they come to
// 1e-5 of a sum's size, 1/200 of the output's rounding, and show where a sum cancels (1 output in 200 is off by more than half a step, K
// 2,048); two parts would cost up to 100 % (8,192 x 6,144 x 2,048 89 -> 165 us, 250 x 2,048 x 6,144 9.6 -> 14.8, 4 x 151,936 x 2,048 33.2 -> 33.5,
// per group 81,920 x 1,024 x 2,048 280 -> 400).  An fp16 step is 8 times finer: of cut sums 1 in 35 is off by more than half of one.
//
// Three kernels, chosen in launch():
//   mx_dma     tiles of 16 x 64 to 256 x 256 through LDS, filled by direct-to-LDS loads several steps ahead
//   mx_skinny  up to 16 rows and few columns: operands straight from memory, K split over a workgroup's waves
//   mx_far     rows gathered from more than 4 GiB: 64 x 64 tiles through registers, with 64-bit addresses
// mx_dma and mx_far serve the product per group: a workgroup finds its group's tile from the offsets by itself, so there is no
// preparing launch, no workspace and nothing for the host to know.
#include <algorithm>

#include "wzy_mx.h"

using namespace wzy;

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef uint32_t v4u_t __attribute__((ext_vector_type(4)));
typedef float v4f_t __attribute__((ext_vector_type(4)));

namespace {

struct MxGemm {
    MxView a, w;
    const int* row_ids;
    const int* offsets;               // null: one dense product
    void* y;
    int64_t ldy;
    int a_rows, groups, M, N, K, y_type;
    int mt, nt;                       // row and column tiles
};

// 4 bytes at any address
struct __attribute__((packed, aligned(1))) Bytes4 { uint32_t x; };
// up to 4 scale bytes at p, n of them inside the row; bytes past it read as 0 (2^-127: not NaN)
WZY_DEV uint32_t load_scales4(const uint8_t* p, int n) {
    if (n >= 4) return ((const Bytes4*) p)->x;
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < n) v |= (uint32_t) p[i] << (8 * i);
    return v;
}
WZY_DEV uint4 load16(const uint8_t* p, bool ok) { return ok ? *(const uint4*) p : make_uint4(0, 0, 0, 0); }

// codes of an E4M3 dword whose exponent bit 3 is set (magnitudes from 2 up), the others as +0
WZY_DEV uint32_t e4m3_large(uint32_t x) {
    const uint32_t m = x & 0x40404040u;
    return x & ((m << 2) - (m >> 6));
}
WZY_DEV v8i_t operand4(uint4 v) { return v8i_t{(int) v.x, (int) v.y, (int) v.z, (int) v.w, 0, 0, 0, 0}; }
WZY_DEV v8i_t operand8(uint4 a, uint4 b) {
    return v8i_t{(int) a.x, (int) a.y, (int) a.z, (int) a.w, (int) b.x, (int) b.y, (int) b.z, (int) b.w};
}
template <int FMT>
WZY_DEV v8i_t operand_of(const uint4 (&v)[FMT == WZY_MX_E4M3 ? 2 : 1]) {
    if constexpr (FMT == WZY_MX_E4M3) return operand8(v[0], v[1]);
    else return operand4(v[0]);
}
// products taken in two parts, none cut
constexpr bool two_parts(int fmt, int out) { return fmt == WZY_MX_E4M3 && out != WZY_BF16; }
template <int FMT>
struct Code;                                                     // the instructions' format numbers
template <> struct Code<WZY_MX_E4M3> { static constexpr int v = 0; };
template <> struct Code<WZY_MX_E2M1> { static constexpr int v = 4; };

// w (E2M1) by a: D's rows are w's, its columns a's.  OW, OA: the scale's byte in its dword.
template <int FMT, int OUT, int OW, int OA>
WZY_DEV v4f_t mfma16(v8i_t w, v8i_t a, v4f_t c, int sw, int sa) {
    if constexpr (two_parts(FMT, OUT)) {
        v8i_t hi, lo;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hi[i] = (int) e4m3_large((uint32_t) a[i]);
            lo[i] = a[i] ^ hi[i];
        }
        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, lo, c, 4, 0, OW, sw, OA, sa);
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, hi, c, 4, 0, OW, sw, OA, sa);
    } else {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 4, Code<FMT>::v, OW, sw, OA, sa);
    }
}
template <int OUT>
WZY_DEV void put(void* y, size_t i, float v) {
    if constexpr (OUT == WZY_F32) ((float*) y)[i] = v;
    else if constexpr (OUT == WZY_BF16) ((uint16_t*) y)[i] = (uint16_t) pack2<WZY_BF16>(v, v);
    else ((uint16_t*) y)[i] = f_to_h16(v);
}

// ---- the tile of a group ---------------------------------------------------------------------------------
// Tiles of up to TM rows are numbered through the groups in order; the wave finds tile t: 64 lanes x 8 groups a
// pass, a prefix sum over the lanes.  False where there are fewer tiles.  Offsets are limited to 0 .. M, so a
// tile never leaves y.
struct __attribute__((packed, aligned(4))) Ints4 { int x, y, z, w; };
template <int CTRL, int ROWMASK>
WZY_DEV int add_dpp(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWMASK, 0xF, true); }
// sums of lanes 0 .. l: within 16-lane rows by shifts, then the rows' last lanes on to the next rows
WZY_DEV int prefix_sum(int v) {
    v = add_dpp<0x111, 0xF>(v);                                    // row_shr 1, 2, 4, 8
    v = add_dpp<0x112, 0xF>(v);
    v = add_dpp<0x114, 0xF>(v);
    v = add_dpp<0x118, 0xF>(v);
    v = add_dpp<DPP_ROW_BCAST15, 0xA>(v);
    return add_dpp<DPP_ROW_BCAST31, 0xC>(v);
}
WZY_DEV int clamp_off(int o, int M) { return min(max(o, 0), M); }
template <int TM>
WZY_DEV bool find_tile(const MxGemm& g, int t, int& group, int& row0, int& rows) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < g.groups; base += 512) {
        const int g0 = base + 8 * lane;
        int off[9], cnt[8], sum = 0;
        if (g0 + 8 <= g.groups) {
            const Ints4 a = *(const Ints4*) (g.offsets + g0), b = *(const Ints4*) (g.offsets + g0 + 4);
            off[0] = a.x; off[1] = a.y; off[2] = a.z; off[3] = a.w;
            off[4] = b.x; off[5] = b.y; off[6] = b.z; off[7] = b.w;
            off[8] = g.offsets[g0 + 8];
        } else {
#pragma unroll
            for (int i = 0; i < 9; ++i) off[i] = g.offsets[min(g0 + i, g.groups)];
        }
#pragma unroll
        for (int i = 0; i < 9; ++i) off[i] = clamp_off(off[i], g.M);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            cnt[i] = (max(off[i + 1] - off[i], 0) + TM - 1) / TM;
            sum += cnt[i];
        }
        const int pre = prefix_sum(sum);                          // over the lanes, its own included
        const int first = before + pre - sum;
        const uint64_t hit = __ballot(t >= first && t < first + sum);
        if (hit) {
            const int src = __ffsll((unsigned long long) hit) - 1;
            int at = first, gg = 0, r0 = 0, n = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (t >= at && t < at + cnt[i]) {
                    gg = g0 + i;
                    r0 = off[i] + (t - at) * TM;
                    n = min(off[i + 1] - r0, TM);
                }
                at += cnt[i];
            }
            group = __builtin_amdgcn_readlane(gg, src);
            row0 = __builtin_amdgcn_readlane(r0, src);
            rows = __builtin_amdgcn_readlane(n, src);
            return rows > 0;                                       // (0: only where offsets that fall make the counts wrap)
        }
        before = __builtin_amdgcn_readlane(before + pre, 63);
    }
    return false;
}

// Tile of this workgroup.  Consecutive workgroups go to the 8 XCDs in turn, each with an L2 of its own.  Dense: the tiles are
// numbered in bands of four row tiles, down the band and then along it, and XCD x takes the x-th eighth of them: the 32 or 64
// tiles it works on at a time share 4 panels of a and 8 or 16 of w.  Grouped: the number of tiles is not known here, so an
// XCD takes every eighth row tile and runs its column tiles one after another.  (Bands of four there, so that tiles of one group
// share their weights: 3 % slower at 8,192 tokens of 10 of 512 experts, the row tiles being as many bytes.)
template <bool GROUPED>
WZY_DEV bool tile_of(const MxGemm& g, int& mi, int& ni) {
    const int x = (int) blockIdx.x & 7, s = (int) blockIdx.x >> 3;
    if constexpr (GROUPED) {
        mi = (s / g.nt) * 8 + x;
        ni = s % g.nt;
    } else {
        const int t = x * ((int) gridDim.x >> 3) + s, band = t / (4 * g.nt), r = t - band * 4 * g.nt, h = min(g.mt - 4 * band, 4);
        if (h <= 0) return false;
        ni = r / h;
        mi = 4 * band + r % h;
    }
    mi = __builtin_amdgcn_readfirstlane(mi);                       // the divisions leave them in vector registers
    ni = __builtin_amdgcn_readfirstlane(ni);
    return ni < g.nt;
}

// row of a that entry e reads; -1: zeros
WZY_DEV int entry_row(const MxGemm& g, int e) {
    const int r = g.row_ids[e];
    return (unsigned) r < (unsigned) g.a_rows ? r : -1;
}

// ---- up to 16 rows -----------------------------------------------------------------------------------------
// A workgroup of up to 8 waves takes 16 weight rows; wave w the batches w, w + waves, ... of 512 k, so neighbouring waves read
// neighbouring pieces of the same rows, and the waves' sums meet in LDS.  Of a batch's 16 blocks lane group q takes 4 q .. 4 q + 3 in
// its four instructions: its scales are one dword a row, its weights 64 bytes.
template <int FMT, int OUT>
__global__ void __launch_bounds__(512) mx_skinny_kernel(MxGemm g) {
    constexpr bool E8 = FMT == WZY_MX_E4M3;
    __shared__ v4f_t s_acc[7][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ks = blockDim.x >> 6;
    const int q = lane >> 4, lr = lane & 15, n0 = (int) blockIdx.x * 16;
    const size_t ar = min(lr, g.M - 1), wr = min(n0 + lr, g.N - 1);
    const uint8_t* const ap = g.a.codes + ar * g.a.ldc;
    const uint8_t* const asp = g.a.scales + ar * g.a.lds;
    const uint8_t* const wp = g.w.codes + wr * g.w.ldc;
    const uint8_t* const wsp = g.w.scales + wr * g.w.lds;
    const int nblk = g.K / 32;
    v4f_t acc = {0.f, 0.f, 0.f, 0.f};
    struct Batch { uint4 w[4], a[4][E8 ? 2 : 1]; uint32_t sw, sa; };
    // E4M3: piece j of lane group q holds half q % 2 of the block of lane group q / 2 + 2 j
    auto a_off = [&](int b, int s, int j) { return E8 ? 32 * (b + 4 * ((q >> 1) + 2 * j) + s) + 16 * (q & 1) : 16 * (b + 4 * q + s); };
    auto load = [&](int b) {                                       // b: first block of the batch
        Batch t;
        if (b + 16 <= nblk) {                                      // wave-uniform
#pragma unroll
            for (int s = 0; s < 4; ++s) t.w[s] = ld_stream_u4(wp + 16 * (b + 4 * q + s));
            t.sw = ((const Bytes4*) (wsp + b + 4 * q))->x;
            t.sa = ((const Bytes4*) (asp + b + 4 * q))->x;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < (E8 ? 2 : 1); ++j) t.a[s][j] = *(const uint4*) (ap + a_off(b, s, j));
        } else {
            const int left = nblk - b - 4 * q;                     // blocks of this lane group inside the row
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                t.w[s] = load16(wp + 16 * (b + 4 * q + s), s < left);
#pragma unroll
                for (int j = 0; j < (E8 ? 2 : 1); ++j) t.a[s][j] = load16(ap + a_off(b, s, j), E8 ? b + 4 * ((q >> 1) + 2 * j) + s < nblk : s < left);
            }
            t.sw = load_scales4(wsp + b + 4 * q, left);
            t.sa = load_scales4(asp + b + 4 * q, left);
        }
        return t;
    };
    auto multiply = [&](const Batch& t) {
        acc = mfma16<FMT, OUT, 0, 0>(operand4(t.w[0]), operand_of<FMT>(t.a[0]), acc, (int) t.sw, (int) t.sa);
        acc = mfma16<FMT, OUT, 1, 1>(operand4(t.w[1]), operand_of<FMT>(t.a[1]), acc, (int) t.sw, (int) t.sa);
        acc = mfma16<FMT, OUT, 2, 2>(operand4(t.w[2]), operand_of<FMT>(t.a[2]), acc, (int) t.sw, (int) t.sa);
        acc = mfma16<FMT, OUT, 3, 3>(operand4(t.w[3]), operand_of<FMT>(t.a[3]), acc, (int) t.sw, (int) t.sa);
    };
    int b = 16 * wave;
    if (b < nblk) {
        Batch t = load(b);
        for (b += 16 * ks; b < nblk; b += 16 * ks) {               // the next batch's loads leave before this one is used
            const Batch n = load(b);
            multiply(t);
            t = n;
        }
        multiply(t);
    }
    if (wave) s_acc[wave - 1][lane] = acc;
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < ks; ++w) acc += s_acc[w - 1][lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int n = n0 + 4 * q + r;
        if (lr < g.M && n < g.N) put<OUT>(g.y, (size_t) lr * g.ldy + n, acc[r]);
    }
}

// ---- tiles in LDS --------------------------------------------------------------------------------------------
// Row of w behind row lr of column block j of a wave.  16-bit y: the four registers of blocks j and j + 1 of a lane are eight
// columns in a row, one 16-byte store (PAIR); otherwise those of a block are four.
template <bool PAIR>
WZY_DEV int w_row(int j, int lr) { return PAIR ? 32 * (j / 2) + 8 * (lr >> 2) + 4 * (j % 2) + (lr & 3) : 16 * j + lr; }
// A row of P 16-byte pieces keeps them exchanged by the bits of the row's number that differ among the 16 rows that 16 lanes
// read one piece of at a time (16 i .. of a, w_row of w), so that these touch all 64 banks once.  Conflict cycles counted, of the LDS's active ones:
// 16 x 64 tiles none, 256 x 256 E2M1 to bf16 0.07, 32 x 64 E4M3 to bf16 0.10, 128 x 128 the same per group 0.27.
template <int P>
WZY_DEV int swz_a(int r) { return P == 16 ? r & 15 : P == 8 ? (r >> 1) & 7 : (r >> 2) & 3; }
template <int P, bool PAIR>
WZY_DEV int swz_w(int r) {
    if constexpr (PAIR) return P == 8 ? ((r >> 1) & 1) | ((r >> 3) & 3) << 1 : (r >> 3) & 3;
    else return swz_a<P>(r);
}
// A wave's part of y: lane (q4, lr) holds rows wr + 16 i + lr, columns n + 16 j + 4 q4 .. + 3, or n + 16 j + 8 q4 .. + 7 of a pair
// of blocks.  whole: no column of the tile lies past N and y's rows are aligned to 16 bytes.
template <int OUT, int NI, int CB, bool PAIR>
WZY_DEV void store_tile(const MxGemm& g, bool gather, bool whole, int row0, int rows, int wr, int n, const v4f_t (&acc)[NI][CB]) {
    constexpr int NV = PAIR ? 8 : 4;
    const int q4 = (threadIdx.x & 63) >> 4, lr = threadIdx.x & 15;
    // Whole cache lines: a lane has two 16-byte pieces of its row 64 bytes apart.  Lanes lr and lr + 8 exchange one of theirs, and a store writes
    // 8 rows of 128 bytes, past the caches (half lines stored so cost up to 18 %, whole ones through the caches nothing).  us, before and
    // after: 8,192 x 6,144 x 2,048 E2M1 to bf16 68 and 65, to fp32 101 and 82, E4M3 to fp32 207 and 182; 8,192 x 12,288 x 2,048 E2M1 142 and 127,
    // 220 and 158; per group, gathered, 81,920 x 2,048 x 512, E4M3 to bf16 257 and 234; but 8,192 x 8,192 x 320 to bf16 50 and 52.
    constexpr int LINE = OUT == WZY_F32 ? 2 : 4;                      // column blocks of 128 bytes
    if constexpr (CB % LINE == 0) {
        if (whole) {
            const bool up = lr >= 8;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r0 = wr + 16 * i;
                const bool zero = gather && r0 + lr < rows && (unsigned) g.row_ids[row0 + r0 + lr] >= (unsigned) g.a_rows;
#pragma unroll
                for (int j = 0; j < CB; j += LINE) {
                    v4u_t p[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if constexpr (OUT == WZY_F32) p[h][r] = zero ? 0u : __float_as_uint(acc[i][j + h][r]);
                            else p[h][r] = zero ? 0u : pack2<OUT>(acc[i][j + 2 * h + (r >> 1)][2 * (r & 1)], acc[i][j + 2 * h + (r >> 1)][2 * (r & 1) + 1]);
                        }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t t = (uint32_t) __builtin_amdgcn_update_dpp(0, (int) (up ? p[0][r] : p[1][r]), 0x128, 0xF, 0xF, true);   // row_ror 8
                        if (up) p[0][r] = t;
                        else p[1][r] = t;
                    }
                    uint8_t* const at = (uint8_t*) g.y + ((size_t) (row0 + r0 + (lr & 7)) * g.ldy + n + 16 * j) * (OUT == WZY_F32 ? 4 : 2) + (up ? 64 : 0) + 16 * q4;
                    if (r0 + (lr & 7) < rows) __builtin_nontemporal_store(p[0], (v4u_t*) at);
                    if (r0 + (lr & 7) + 8 < rows) __builtin_nontemporal_store(p[1], (v4u_t*) (at + 8 * g.ldy * (OUT == WZY_F32 ? 4 : 2)));
                }
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int m = wr + 16 * i + lr;
        if (m >= rows) continue;
        const bool zero = gather && (unsigned) g.row_ids[row0 + m] >= (unsigned) g.a_rows;
        const size_t row = (size_t) (row0 + m) * g.ldy;
#pragma unroll
        for (int j = 0; j < CB; j += PAIR ? 2 : 1) {
            const int c = n + 16 * j + NV * q4;
            float v[8];
#pragma unroll
            for (int r = 0; r < NV; ++r) v[r] = zero ? 0.f : acc[i][j + (r >> 2)][r & 3];
            if (whole) {
                if constexpr (PAIR) store8<OUT>(g.y, row + c, v);
                else if constexpr (OUT == WZY_F32) *(float4*) ((float*) g.y + row + c) = make_float4(v[0], v[1], v[2], v[3]);
                else *(uint2*) ((uint16_t*) g.y + row + c) = make_uint2(pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3]));
            } else {
#pragma unroll
                for (int r = 0; r < NV; ++r)
                    if (c + r < g.N) put<OUT>(g.y, row + c + r, v[r]);
            }
        }
    }
}
template <int OUT>
WZY_DEV bool whole_tile(const MxGemm& g, int n0, int tn) {
    return n0 + tn <= g.N && (((uintptr_t) g.y | (uintptr_t) g.ldy * (OUT == WZY_F32 ? 4 : 2)) & 15) == 0;
}

// Product per group with rows gathered from more than 4 GiB.  Each wave holds 32 rows by 32 columns of the tile.  K goes in steps of 128
// through two LDS buffers and two register sets: step k + 2 loads while step k multiplies.
template <int FMT, int OUT>
__global__ void __launch_bounds__(256, 2) mx_far_kernel(MxGemm g) {
    constexpr int TM = 64, TN = 64, WM = 2, WN = 2;
    constexpr bool E8 = FMT == WZY_MX_E4M3, PAIR = OUT != WZY_F32;
    constexpr int T = 64 * WM * WN, RB = TM / 16 / WM, CB = TN / 16 / WN;
    constexpr int AP = E8 ? 8 : 4, WP = 4;                         // 16-byte pieces of a row per step
    constexpr int NA = (TM * AP + T - 1) / T, NW = (TN * WP + T - 1) / T, NS = (TM + TN + T - 1) / T;
    __shared__ uint4 s_a[2][TM * AP];
    __shared__ uint4 s_w[2][TN * WP];
    __shared__ uint32_t s_sc[2][TM + TN];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q4 = lane >> 4, lr = lane & 15;
    int mi, ni, group, row0, rows;
    if (!tile_of<true>(g, mi, ni) || !find_tile<TM>(g, mi, group, row0, rows)) return;
    const int n0 = ni * TN;
    const int nblk = g.K / 32, steps = (nblk + 3) / 4;
    const uint8_t* const wbase = g.w.codes + ((size_t) group * g.N + n0) * g.w.ldc;
    const uint8_t* const wsbase = g.w.scales + ((size_t) group * g.N + n0) * g.w.lds;
    const uint8_t* ap[NA];
    const uint8_t* sp[NS];
    uint32_t wo[NW];
    bool aok[NA], sok[NS];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int p = tid + T * i, ar = entry_row(g, row0 + min(p / AP, rows - 1));
        aok[i] = ar >= 0;
        ap[i] = g.a.codes + (size_t) max(ar, 0) * g.a.ldc + 16 * (p % AP);
    }
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int p = tid + T * i;
        wo[i] = (uint32_t) min(p / WP, g.N - 1 - n0) * (uint32_t) g.w.ldc + 16 * (p % WP);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int r = tid + T * i;
        const int ar = entry_row(g, row0 + min(min(r, TM - 1), rows - 1));
        sok[i] = r < TM ? ar >= 0 : r < TM + TN;
        sp[i] = r < TM ? g.a.scales + (size_t) max(ar, 0) * g.a.lds : wsbase + (size_t) min(r - TM, g.N - 1 - n0) * g.w.lds;
    }
    struct Regs { uint4 a[NA], w[NW]; uint32_t s[NS]; };
    auto load = [&](int k) {
        Regs t;
        const int left = nblk - 4 * k;                             // blocks from this step on; none past the end
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int c = (tid + T * i) % AP;
            t.a[i] = load16(ap[i] + (size_t) k * (16 * AP), aok[i] && (E8 ? c < 2 * left : c < left));
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) t.w[i] = load16(wbase + wo[i] + (size_t) k * 64, (tid + T * i) % WP < left);
#pragma unroll
        for (int i = 0; i < NS; ++i) t.s[i] = sok[i] ? load_scales4(sp[i] + 4 * (size_t) k, left) : 0;
        return t;
    };
    auto store = [&](int b, const Regs& t) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int p = tid + T * i;
            s_a[b][p / AP * AP + ((p % AP) ^ swz_a<AP>(p / AP))] = t.a[i];
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int p = tid + T * i;
            s_w[b][p / WP * WP + ((p % WP) ^ swz_w<WP, PAIR>(p / WP))] = t.w[i];
        }
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (tid + T * i < TM + TN) s_sc[b][tid + T * i] = t.s[i];
    };
    v4f_t acc[RB][CB];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j) acc[i][j] = v4f_t{0.f, 0.f, 0.f, 0.f};
    const int wr = (wave / WN) * (TM / WM), wc = (wave % WN) * (TN / WN), wl = w_row<PAIR>(0, lr);
    const int nrb = (rows - wr + 15) / 16;                         // row blocks of this wave that hold rows
    const int asw = swz_a<AP>(lr), wsw = swz_w<WP, PAIR>(wl);
    auto multiply = [&](int b) {
        uint4 wv[CB];
        int sw[CB];
#pragma unroll
        for (int j = 0; j < CB; ++j) {
            const int r = wc + w_row<PAIR>(j, 0) + wl;
            wv[j] = s_w[b][r * WP + (q4 ^ wsw)];
            sw[j] = (int) (s_sc[b][TM + r] >> (8 * q4));
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            if (i >= nrb) break;                                   // wave-uniform
            const int r = wr + 16 * i + lr, sa = (int) (s_sc[b][r] >> (8 * q4));
            uint4 av[E8 ? 2 : 1];
#pragma unroll
            for (int j = 0; j < (E8 ? 2 : 1); ++j) av[j] = s_a[b][r * AP + ((q4 + 4 * j) ^ asw)];
#pragma unroll
            for (int j = 0; j < CB; ++j) acc[i][j] = mfma16<FMT, OUT, 0, 0>(operand4(wv[j]), operand_of<FMT>(av), acc[i][j], sw[j], sa);
        }
    };
    Regs t0 = load(0), t1 = load(1);
    store(0, t0);
    __syncthreads();
    for (int k = 0; k < steps; k += 2) {
        t0 = load(k + 2);
        multiply(0);
        if (k + 1 >= steps) break;                                 // workgroup-uniform
        store(1, t1);
        __syncthreads();
        t1 = load(k + 3);
        multiply(1);
        store(0, t0);
        __syncthreads();
    }
    store_tile<OUT, RB, CB, PAIR>(g, true, whole_tile<OUT>(g, n0, TN), row0, rows, wr, n0 + wc, acc);
}

// ---- tiles fed by direct-to-LDS loads -----------------------------------------------------------------------
// Codes and scales go from memory to LDS without registers, in
// units of UK k through ST buffers.  The loads are counted, so a wave waits for the unit it needs and leaves the later ones
// in flight, and one barrier a unit tells every wave that all parts of the next unit have landed and that this unit's
// buffer is free.  (Inline assembly: the compiler would have every LDS read wait for every such load.  The loads have no
// register result.)  Scales come 16 bytes a row, for 512 k: 4 bytes a row took as many cache requests as the codes (8,192 x 8,192 x
// 8,192 in E2M1, 377 -> 342 us).  UK 256 makes a weight row's piece a whole cache line of 128 bytes (342 -> 314); E4M3 tiles of
// 128 x 128 and more take 128, for want of LDS.
//
// Every operand is read from LDS one row block before it is used, across units too: before the last row block of a unit a wave
// waits for the next unit's loads and meets the others; all its reads of this unit are done then, so the buffer takes the
// loads of unit u + ST, and the next unit's first operands are read under the last row block's MFMAs (314 -> 303; tiles in
// bands, tile_of: 285; 16x16x128 instructions: 271).
//
// Two forms.  Where K is whole units, every row's scales begin at a dword and there are at least 16 bytes of them, nothing is checked.
// ANY takes every K and alignment: loads are kept inside the matrix, blocks past a row's end count as zeros, and scales come a
// dword a lane and are shifted into place on the way out of LDS.  (That form for aligned calls too: 5 to 10 % slower, up to 60 % where
// its registers spill, 256 x 256, so it has no such tile.  ANY against 64 x 64 and 128 x 128 tiles through registers, E4M3 to bf16, K 2,080, us:
// 4 x 151,936 45, 89; 100 x 2,048 5.9, 7.2; 300 x 2,048 x 6,176 15, 28; 8,192 x 6,144 129, 142; per group, 512 groups, 6,000 rows 157, 192.)
//
// WM x WN waves hold TM / WM rows by TN / WN columns each; KW 2: two such sets, one for each 128 of a unit, whose sums meet
// at the end (16 x 64 tiles, where a unit's chain of LDS reads and MFMAs is what takes the time: 1 x 12,288 x 2,048 to fp32 6.8 ->
// 5.7 us).
//
// What bounds it: 8,192 x 8,192 x 8,192 to bf16, E2M1 263 us (4,180 TFLOP/s), E4M3 405 (2,710).  The same launch without its MFMAs
// took 224 (313), without its loads 231 (335): loads into LDS run at 10 TB/s over the chip whatever the tile, and the MFMAs with
// their LDS reads at 5 PFLOP/s (3.3).  Bigger tiles than 256 x 256 do not fit the LDS; a fourth buffer for 32 x 64 tiles, where the
// loads are all there is (250 x 2,048 x 6,144 9.6 us), changes nothing.
WZY_DEV uint32_t lds_offset(const void* p) { return (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) char*) p; }
// 64 lanes x 16 bytes from base + off (per lane) to LDS lds .. lds + 1023, lane order; lds and base wave-uniform.  The LDS address is in m0,
// an output of the statement, so that the compiler knows it changed (it is a register of the compiler's own: a clobber of it means nothing; as an
// input, E4M3 tiles of 256 x 256 spilled inside their loop, 8,192 x 8,192 x 8,192 to bf16 398 -> 422 us).
WZY_DEV void dma16(uint32_t lds, uint32_t off, const uint8_t* base) {
    const uint64_t b = (uint64_t) (uintptr_t) base;
    lds = (uint32_t) __builtin_amdgcn_readfirstlane((int) lds);      // nothing where they are in scalar registers already
    base = (const uint8_t*) (uintptr_t) ((uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (b >> 32)) << 32 |
                                         (uint32_t) __builtin_amdgcn_readfirstlane((int) b));
    uint32_t m0;
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %2, %3" : "={m0}"(m0) : "s"(lds), "v"(off), "s"(base) : "memory");
}
// 64 lanes x 4 bytes, likewise
WZY_DEV void dma4(uint32_t lds, uint32_t off, const uint8_t* base) {
    const uint64_t b = (uint64_t) (uintptr_t) base;
    lds = (uint32_t) __builtin_amdgcn_readfirstlane((int) lds);
    base = (const uint8_t*) (uintptr_t) ((uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (b >> 32)) << 32 |
                                         (uint32_t) __builtin_amdgcn_readfirstlane((int) b));
    uint32_t m0;
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dword %2, %3" : "={m0}"(m0) : "s"(lds), "v"(off), "s"(base) : "memory");
}
// this wave's loads but the last N have landed and its LDS reads are done; then all waves meet
template <int N>
WZY_DEV void dma_wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int FMT, int OUT, int TM, int TN, int WM, int WN, int KW, int UK, int ST, int OCC, bool GROUPED, bool ANY>
__global__ void __launch_bounds__(64 * WM * WN * KW, OCC) mx_dma_kernel(MxGemm g) {
    constexpr bool E8 = FMT == WZY_MX_E4M3;
    // waves; a wave's row blocks of RH x 16 rows, column blocks of 16
    constexpr int NWV = WM * WN * KW, RH = TM / WM >= 32 ? 2 : 1, RB = TM / WM / (16 * RH), CB = TN / 16 / WN;
    constexpr int AP = UK / (E8 ? 16 : 32), WP = UK / 32;            // 16-byte pieces of a row of a and of w per unit
    constexpr int A_B = TM * AP * 16, W_B = TN * WP * 16, S_B = (TN + (ANY ? TM : (TM + 63) / 64 * 64)) * 16;
    // wave-wide loads of a step; where they do not divide by the waves, some are issued twice (same bytes, same place), so
    // that every wave has the same number in flight
    constexpr int LA = A_B / 1024, LW = W_B / 1024, LS = S_B / (ANY ? 256 : 1024);
    constexpr int NA = (LA + NWV - 1) / NWV, NW = (LW + NWV - 1) / NWV, NS = (LS + NWV - 1) / NWV, NI = NA + NW;
    static_assert(TM % 16 == 0 && TN % 64 == 0 && A_B % 1024 == 0 && RB >= 1 && CB >= 1 && ST >= 2, "tile");
    static_assert((ST - 2) * NI + NS < 64, "loads in flight are counted in six bits");
    static_assert(KW == 1 || (KW == 2 && UK == 256 && RB == 1 && (KW - 1) * WM * WN * RH * CB * 1024 <= ST * (A_B + W_B)), "waves along k");
    static_assert(ST - 2 < 512 / UK, "the count of scales in flight holds from the first unit on");
    // ANY: a group of scales also takes the next one's first dwords: two buffers will do where those are older than the codes waited
    // for with them
    constexpr int SB = !ANY || ST - 2 < 512 / UK - 1 ? 2 : 3;
    static_assert(ST * (A_B + W_B) + SB * S_B <= 160 * 1024, "LDS");
    __shared__ __align__(1024) uint8_t s_buf[ST * (A_B + W_B) + SB * S_B];
    constexpr bool PAIR = OUT != WZY_F32 && CB % 2 == 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q4 = lane >> 4, lr = lane & 15;
    int mi, ni;
    if (!tile_of<GROUPED>(g, mi, ni)) return;
    const int n0 = ni * TN;
    int row0 = mi * TM, rows = min(g.M - row0, TM), group = 0;
    if constexpr (GROUPED) {
        if (!find_tile<TM>(g, mi, group, row0, rows)) return;
    } else if (rows <= 0) return;
    const bool gather = GROUPED && g.row_ids;
    const uint8_t* const abase = g.a.codes + (gather ? 0 : (size_t) row0 * g.a.ldc);
    const uint8_t* const asbase = g.a.scales + (gather ? 0 : (size_t) row0 * g.a.lds);
    const size_t wrow0 = (size_t) group * g.N + n0;
    const uint8_t* const wbase = g.w.codes + wrow0 * g.w.ldc;
    const uint8_t* const wsbase = g.w.scales + wrow0 * g.w.lds;
    auto a_row = [&](int r) {                                        // row r of the tile, counted from abase
        r = min(r, rows - 1);
        if (!gather) return (uint32_t) r;
        const int id = g.row_ids[row0 + r];
        return (unsigned) id < (unsigned) g.a_rows ? (uint32_t) id : 0u;
    };
    // ANY: loads that pass the end of a row read on in the matrix, up to its end, and what they bring is replaced by zeros.  Offsets from the bases of the last 16 bytes of codes and the last dword
    // that holds a scale:
    const int nblk = g.K / 32;
    const size_t a_left = (size_t) (g.a_rows - 1 - (gather ? 0 : row0)), w_left = (size_t) (GROUPED ? g.groups : 1) * g.N - 1 - wrow0;
    const uint32_t as0 = (uint32_t) (uintptr_t) asbase & 3u, ws0 = (uint32_t) (uintptr_t) wsbase & 3u;
    auto low32 = [](size_t x) { return (uint32_t) min(x, (size_t) 0xFFFFFFF0u); };
    const uint32_t a_end = low32(a_left * g.a.ldc + (size_t) nblk * (E8 ? 32 : 16) - 16), w_end = low32(w_left * g.w.ldc + (size_t) nblk * 16 - 16);
    const uint32_t as_end = low32(a_left * g.a.lds + as0 + nblk - 1) & ~3u, ws_end = low32(w_left * g.w.lds + ws0 + nblk - 1) & ~3u;
    constexpr int UH = UK / 128, GU = 4 / UH;                        // units have UH halves of 128 k, groups of scales GU units
    const uint32_t lds0 = lds_offset(s_buf);
    // LDS position p (16 bytes) of a buffer: row p / pieces, its piece p % pieces permuted by the row
    uint32_t ao[NA], wo[NW], so[NS];
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int p = ((wave * NW + i) % LW) * 64 + lane, r = p / WP;
        wo[i] = (uint32_t) min(r, g.N - 1 - n0) * (uint32_t) g.w.ldc + 16 * ((p % WP) ^ swz_w<WP, PAIR>(r));
    }
    const int units = (nblk + 4 * UH - 1) / (4 * UH);
    auto dma_codes = [&](uint32_t at, uint32_t off, int u, int bytes, uint32_t end, const uint8_t* base) {
        const uint32_t k = (uint32_t) min(u, units - 1) * bytes;     // past the end the last unit again
        dma16(at, ANY ? min(off, end - k) : off, base + k);
    };
    auto issue_w = [&](int u, int buf) {                             // w's codes of unit u
#pragma unroll
        for (int i = 0; i < NW; ++i)
            dma_codes(lds0 + ST * A_B + buf * W_B + ((wave * NW + i) % LW) * 1024, wo[i], u, 64 * UH, w_end, wbase);
    };
    // The weights' first loads leave before the row ids, which a's addresses wait for, are there.
    if constexpr (GROUPED) {
#pragma unroll
        for (int u = 0; u < ST; ++u) issue_w(u, u);
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int p = ((wave * NA + i) % LA) * 64 + lane, r = p / AP;
        ao[i] = a_row(r) * (uint32_t) g.a.ldc + 16 * ((p % AP) ^ swz_a<AP>(r));
    }
    // Scales.  Aligned rows: a row a lane, 16 bytes for the four halves of a group, the row's last 16 where fewer are left.  ANY: 16 rows
    // a load, a dword a lane, 4 in a row; a row may begin at any byte, so dwords are counted from the one with its first scale.
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int r = ((wave * NS + i) % LS) * (ANY ? 16 : 64) + (ANY ? lane >> 2 : lane);
        uint32_t t;
        if (r < TN) t = (uint32_t) min(r, g.N - 1 - n0) * (uint32_t) g.w.lds + (ANY ? ws0 : 0);
        else t = a_row(r - TN) * (uint32_t) g.a.lds + (ANY ? as0 : 0);   // (only here: a_row reads row_ids)
        so[i] = ANY ? (t & ~3u) + 4 * (lane & 3) : t;
    }
    auto scale_at = [&](int q) { return min(16 * q, nblk - 16); };   // byte in an aligned row
    auto issue_a = [&](int u, int buf) {
#pragma unroll
        for (int i = 0; i < NA; ++i)
            dma_codes(lds0 + buf * A_B + ((wave * NA + i) % LA) * 1024, ao[i], u, (E8 ? 128 : 64) * UH, a_end, abase);
    };
    auto scales_at = [&](int q) { return ST * (A_B + W_B) + (SB == 2 ? q & 1 : q % 3) * S_B; };
    auto issue_scales = [&](int q) {                                 // of group q
        const uint32_t at = lds0 + scales_at(q);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int r = ((wave * NS + i) % LS) * (ANY ? 16 : 64);
            const bool w = r < TN;                                   // wave-uniform
            if constexpr (ANY) dma4(at + r * 16, min(so[i] + 16u * (uint32_t) min(q, nblk / 16 + 1), w ? ws_end : as_end), w ? wsbase - ws0 : asbase - as0);
            else dma16(at + r * 16, so[i], (w ? wsbase : asbase) + scale_at(q));
        }
    };
    v4f_t acc[RH * RB][CB];
#pragma unroll
    for (int i = 0; i < RH * RB; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j) acc[i][j] = v4f_t{0.f, 0.f, 0.f, 0.f};
    const int kg = wave / (WM * WN), wt = wave % (WM * WN);          // the wave's half of a unit (KW 2), its part of the tile
    const int wr = (wt / WN) * (TM / WM), wc = (wt % WN) * (TN / WN);
    const int nrb = (rows - wr + 16 * RH - 1) / (16 * RH);           // row blocks of this wave that hold rows
    // lane (q4, lr) reads piece q4 of row 16 i + lr of a and of row w_row(j, lr) = w_row(j, 0) + wl of w
    const int wl = w_row<PAIR>(0, lr), asw = swz_a<AP>(lr), wsw = swz_w<WP, PAIR>(wl);
    const uint8_t* const la = s_buf + (wr + lr) * (AP * 16);
    const uint8_t* const lw = s_buf + ST * A_B + (wc + wl) * (WP * 16);
    const int lsw = (wc + wl) * 16, lsa = (TN + wr + lr) * 16;      // rows of scales
    struct Wf { uint4 v[CB]; };                                      // a half's operands
    struct Af { uint4 v[RH][E8 ? 2 : 1]; };                          // of one row block
    struct Sf { int a[RH * RB], w[CB]; };                            // the scales of the lane's block in four halves, a byte each
    auto load_w = [&](int buf, int half) {
        Wf f;
#pragma unroll
        for (int j = 0; j < CB; ++j)
            f.v[j] = *(const uint4*) (lw + buf * W_B + w_row<PAIR>(j, 0) * (WP * 16) + 16 * ((4 * half + q4) ^ wsw));
        return f;
    };
    auto load_a = [&](int buf, int half, int i) {
        Af f;
#pragma unroll
        for (int e = 0; e < RH; ++e) {
            const uint8_t* const ra = la + buf * A_B + (AP * 16) * 16 * (RH * i + e);
            if constexpr (E8) {
                f.v[e][0] = *(const uint4*) (ra + 16 * ((8 * half + q4) ^ asw));
                f.v[e][1] = *(const uint4*) (ra + 16 * ((8 * half + 4 + q4) ^ asw));
            } else {
                f.v[e][0] = *(const uint4*) (ra + 16 * ((4 * half + q4) ^ asw));
            }
        }
        return f;
    };
    // first byte in its dword of each row of scales that the lane reads, 2 bits each
    uint32_t first = 0;
    if constexpr (ANY) {
#pragma unroll
        for (int j = 0; j < CB; ++j) first |= ((ws0 + (uint32_t) min(wc + w_row<PAIR>(j, 0) + wl, g.N - 1 - n0) * (uint32_t) g.w.lds) & 3u) << (2 * j);
#pragma unroll
        for (int i = 0; i < RH * RB; ++i) first |= ((as0 + a_row(wr + 16 * i + lr) * (uint32_t) g.a.lds) & 3u) << (2 * (CB + i));
    }
    static_assert(CB + RH * RB <= 16, "two bits a row");
    const uint32_t pick = 0x0C0C0400u + 0x0101u * (uint32_t) q4;     // byte q4 of one dword, then of another
    struct Reader { const uint8_t *here, *next; bool skip; uint32_t in; };   // of a group of scales
    auto scales_of = [&](int q) {
        const int n = min(max(nblk - 16 * q - q4 + 3, 0) >> 2, 4);    // the lane's blocks inside the row; the others' scales are 0
        // skip: the row's last 16 bytes begin two dwords before the group
        return Reader{s_buf + scales_at(q), s_buf + scales_at(q + 1), scale_at(q) < 16 * q, n == 4 ? ~0u : (1u << (8 * n)) - 1};
    };
    auto load_s = [&](const Reader& s, int at, int i) {              // scales of the lane's block in four halves
        uint4 d = *(const uint4*) (s.here + at);
        uint32_t in = ~0u;
        if constexpr (ANY) {
            const uint32_t e = *(const uint32_t*) (s.next + at), f = first >> (2 * i);   // (its low two bits count)
            d.x = __builtin_amdgcn_alignbyte(d.y, d.x, f);
            d.y = __builtin_amdgcn_alignbyte(d.z, d.y, f);
            d.z = __builtin_amdgcn_alignbyte(d.w, d.z, f);
            d.w = __builtin_amdgcn_alignbyte(e, d.w, f);
            in = s.in;
        } else {
            if (s.skip) { d.x = d.z; d.y = d.w; }
        }
        return (int) (((__builtin_amdgcn_perm(d.y, d.x, pick) | __builtin_amdgcn_perm(d.w, d.z, pick) << 16) & in) >> (KW == 2 ? 8 * kg : 0));
    };
    auto load_sw = [&](const Reader& s, Sf& f) {
#pragma unroll
        for (int j = 0; j < CB; ++j) f.w[j] = load_s(s, lsw + w_row<PAIR>(j, 0) * 16, j);
    };
    auto load_sa = [&](const Reader& s, Sf& f, int i) {               // of row block i
#pragma unroll
        for (int e = 0; e < RH; ++e) f.a[RH * i + e] = load_s(s, lsa + 16 * 16 * (RH * i + e), CB + RH * i + e);
    };
#pragma unroll
    for (int q = 0; q < SB; ++q) issue_scales(q);
#pragma unroll
    for (int u = 0; u < ST; ++u) {
        issue_a(u, u);
        if (!GROUPED) issue_w(u, u);
    }
    dma_wait_barrier<(ST - 1) * (GROUPED ? NA : NI)>();
    Sf sc;
    load_sw(scales_of(0), sc);
    load_sa(scales_of(0), sc, 0);
    Wf wf = load_w(0, kg);                                           // kg: 0 unless KW 2
    Af af = load_a(0, kg, 0);
    int buf = 0;                                                     // of unit u
    auto unit = [&](int u, auto p_, auto tail_, auto one_) {         // tail: the row may end in it; one: in its first half
        constexpr int P = p_();                                      // u % GU
        if (GU % ST == 0) buf = P % ST;                              // known here then
        const int next = buf + 1 == ST ? 0 : buf + 1;
        // younger than the codes of unit u + 1: those of ST - 2 units and the scales issued with them (after units of P 0)
        constexpr int scales = [] { int n = 0; for (int j = 1; j <= ST - 2; ++j) n += (P + 2 * GU - j) % GU == 0; return n; }();
        constexpr int young = (ST - 2) * NI + scales * NS;
        auto block = [&](auto last_, int half, auto d_) {            // half: of the unit; d: of the group of scales
            constexpr bool LAST = last_();
            constexpr int D = d_();
            Wf wn;
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                Af an;
                Sf sn;
                if (i + 1 < RB) {
                    an = load_a(buf, half, i + 1);
                    if (D == 0) load_sa(scales_of(u / GU), sc, i + 1);
                    if (!LAST && i == RB - 2) wn = load_w(buf, 1);
                } else if (!LAST) {
                    if (RB == 1) wn = load_w(buf, 1);
                    an = load_a(buf, 1, 0);
                } else {
                    // (grouped: the first units' weights are older than they are counted here)
                    if (GROUPED && ST > 2 && u < ST - 2) dma_wait_barrier<0>();
                    else dma_wait_barrier<young>();
                    if (P == 0) issue_scales(u / GU + SB);
                    issue_a(u + ST, buf);
                    issue_w(u + ST, buf);
                    wn = load_w(next, kg);
                    an = load_a(next, kg, 0);
                    if (P == GU - 1) {
                        load_sw(scales_of(u / GU + 1), sn);
                        load_sa(scales_of(u / GU + 1), sn, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (ANY && tail_()) {                             // codes past the row's end are zeros
                    const int in = nblk - 4 * (UH * u + half);       // blocks of this half inside the row
#pragma unroll
                    for (int e = 0; e < RH; ++e)
#pragma unroll
                        for (int j = 0; j < (E8 ? 2 : 1); ++j)
                            if ((E8 ? (q4 >> 1) + 2 * j : q4) >= in) af.v[e][j] = make_uint4(0, 0, 0, 0);
                }
                if (!GROUPED || i < nrb) {                           // wave-uniform
#pragma unroll
                    for (int e = 0; e < RH; ++e)
#pragma unroll
                        for (int j = 0; j < CB; ++j)
                            acc[RH * i + e][j] = mfma16<FMT, OUT, D, D>(operand4(wf.v[j]), operand_of<FMT>(af.v[e]), acc[RH * i + e][j], sc.w[j],
                                                                       sc.a[RH * i + e]);
                }
                af = an;
                if (LAST && P == GU - 1 && i == RB - 1) {
#pragma unroll
                    for (int j = 0; j < CB; ++j) sc.w[j] = sn.w[j];
#pragma unroll
                    for (int e = 0; e < RH; ++e) sc.a[e] = sn.a[e];
                }
            }
            wf = wn;
        };
        if constexpr (UH == 1) block(std::true_type(), 0, p_);
        else if constexpr (KW == 2) block(std::true_type(), kg, std::integral_constant<int, 2 * P>());   // (its scales are shifted to this byte)
        else if constexpr (one_()) block(std::true_type(), 0, std::integral_constant<int, 2 * P>());
        else {
            block(std::false_type(), 0, std::integral_constant<int, 2 * P>());
            block(std::true_type(), 1, std::integral_constant<int, 2 * P + 1>());
        }
        buf = next;
    };
    // Whole groups of four halves, then what is left (branches inside the loop would cost copies of the accumulators).
    constexpr std::integral_constant<int, 0> p0{};
    constexpr std::integral_constant<int, 1> p1{};
    constexpr std::integral_constant<int, 2> p2{};
    constexpr std::integral_constant<int, 3> p3{};
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    int u = 0;
    const int left = ((nblk & 15) + 3) >> 2;                           // halves
    for (int n = nblk >> 4; n > 0; --n, u += GU) {
        unit(u, p0, no, no);
        unit(u + 1, p1, no, no);
        if constexpr (UH == 1) {
            unit(u + 2, p2, no, no);
            unit(u + 3, p3, no, no);
        }
    }
    if constexpr (UH == 1) {
        if (left > 0) unit(u, p0, yes, no);
        if (left > 1) unit(u + 1, p1, yes, no);
        if constexpr (ANY) {
            if (left > 2) unit(u + 2, p2, yes, no);
            if (left > 3) unit(u + 3, p3, yes, no);
        }
    } else if constexpr (!ANY) {
        if (left > 0) unit(u, p0, yes, no);
    } else if constexpr (KW == 2) {
        if (left > 0) unit(u, p0, yes, no);
        if (left > 2) unit(u + 1, p1, yes, no);
    } else {
        if (left == 1) unit(u, p0, yes, yes);
        if (left > 1) unit(u, p0, yes, no);
        if (left == 3) unit(u + 1, p1, yes, yes);
        if (left > 3) unit(u + 1, p1, yes, no);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                 // no load outlives the workgroup's LDS
    if constexpr (KW == 2) {                                         // the two halves' sums meet
        __syncthreads();
        v4f_t* const part = (v4f_t*) s_buf + wt * (RH * CB * 64) + lane;
        if (kg == 1) {
#pragma unroll
            for (int i = 0; i < RH; ++i)
#pragma unroll
                for (int j = 0; j < CB; ++j) part[(i * CB + j) * 64] = acc[i][j];
        }
        __syncthreads();
        if (kg == 1) return;
#pragma unroll
        for (int i = 0; i < RH; ++i)
#pragma unroll
            for (int j = 0; j < CB; ++j) acc[i][j] += part[(i * CB + j) * 64];
    }
    store_tile<OUT, RH * RB, CB, PAIR>(g, gather, whole_tile<OUT>(g, n0, TN), row0, rows, wr, n0 + wc, acc);
}

constexpr int CUS = 256;

// mx_dma has 32-bit offsets from its bases: rows gathered (and what a row's loads may pass its end by) lie in 4 GiB
bool far_rows(const MxGemm& g) {
    return g.row_ids && (int64_t) g.a_rows * std::max(g.a.ldc, g.a.lds) >= ((int64_t) 1 << 32) - 4096;
}
// whole units of 256 k, a scale row of 16 bytes at least, dwords of scales aligned; otherwise the form ANY
bool whole_steps(const MxGemm& g) {
    return g.K % 256 == 0 && g.K >= 512 && (g.a.lds | g.w.lds) % 4 == 0 && ((uintptr_t) g.a.scales | (uintptr_t) g.w.scales) % 4 == 0;
}

enum Tile { T256x256, T128x128, T64x128, T64x64, T32x128, T32x64, T16x64 };
constexpr int TILE_M[] = {256, 128, 64, 64, 32, 32, 16}, TILE_N[] = {256, 128, 128, 64, 128, 64, 64};

// Tiles of a dense product: a CU's time for n tiles is that of n / 2 pairs beside each other and of an odd one (256 x 256
// tiles have a CU to themselves); the least of them is taken.  Measured, us for 128 k, {alone, a pair}.  What it decides, for instance
// (E4M3 to bf16, us): 250 x 2,048 x 6,144 32x64 9.6, 64x64 12.7, 64x128 18.6; 1,024 x 2,048 x 2,048 64x128 8.9, 64x64 9.2, 128x128 12.8;
// 2,048 x 12,288 x 2,048 128x128 51, 256x256 61, 64x128 60; 8,192 x 6,144 x 2,048 256x256 93, 128x128 100.
Tile dense_tile(const MxGemm& g, bool e8, bool whole) {
    constexpr Tile kind[] = {T256x256, T128x128, T64x128, T64x64, T32x64};
    constexpr float cost[4][5][2] = {{{1.62f, 3.24f}, {0.62f, 0.96f}, {0.36f, 0.58f}, {0.24f, 0.40f}, {0.17f, 0.28f}},   // E4M3
                                     {{1.06f, 2.12f}, {0.40f, 0.67f}, {0.27f, 0.46f}, {0.19f, 0.29f}, {0.14f, 0.24f}},   // E2M1
                                     {{9.00f, 9.00f}, {0.95f, 1.70f}, {0.65f, 1.10f}, {0.38f, 0.62f}, {0.25f, 0.37f}},    // E4M3 to fp32
                                     {{3.15f, 6.30f}, {1.15f, 1.80f}, {0.85f, 1.25f}, {0.55f, 0.70f}, {0.38f, 0.45f}}};  // E4M3 to fp16
    const bool f32 = g.y_type == WZY_F32;
    const auto& c = cost[!e8 ? 1 : f32 ? 2 : g.y_type == WZY_F16 ? 3 : 0];
    Tile best = T32x64;
    float least = 0.f;
    for (int i = (e8 && f32) || !whole ? 1 : 0; i < 5; ++i) {      // E4M3 to fp32 and ANY have no 256 x 256: their registers spill inside the loop (E4M3 to 16 bits spills 4 or 5, before and after it)
        const int64_t t = ((int64_t) g.M + TILE_M[kind[i]] - 1) / TILE_M[kind[i]] * (((int64_t) g.N + TILE_N[kind[i]] - 1) / TILE_N[kind[i]]);
        const int64_t n = (t + CUS - 1) / CUS;
        const float us = (float) (n / 2) * c[i][1] + (float) (n % 2) * c[i][0];
        if (least == 0.f || us < least) least = us, best = kind[i];
    }
    return best;
}
// Tiles of a product per group, by the rows of a group that has any.  Measured at 512 groups, N 1,024, K 2,048, E4M3 to bf16, us: 6 rows
// 16x64 106, 32x128 108 (to fp32 117, 134); 12 rows 128, 118, 64x128 132; 20 rows 32x128 126, 64x128 134; 40 rows 168, 149, 128x128 164; 80
// rows 64x128 213, 128x128 192; 160 rows 128x128 304, 256x256 367, but E2M1 253, 218.  (Which groups have entries is not known here: where a few of
// many hold all rows, tiles are smaller than they would best be, 8,192 rows in 4 of 512 groups 35.5 us, in 4 of 4 27.5.)
Tile grouped_tile(const MxGemm& g, bool e8, bool whole) {
    const int rows = g.M / std::min(g.M, g.groups);
    if (rows <= 8) return T16x64;
    if (rows <= 25) return T32x128;
    if (rows <= 56) return T64x128;
    const bool many = (int64_t) g.groups * ((g.N + 255) / 256) >= 2 * CUS;
    return whole && !e8 && rows >= 128 && many ? T256x256 : T128x128;
}

template <int FMT, int OUT, bool GROUPED>
int launch(MxGemm g, hipStream_t st) {
    constexpr bool E8 = FMT == WZY_MX_E4M3;
    auto go = [&](auto kernel, int tm, int tn, int threads) {
        // every group may end in a part tile, so rows / tile + groups tiles cover any split (and no more than there are rows)
        const int64_t mt = GROUPED ? std::min<int64_t>(g.M, (int64_t) g.M / tm + g.groups) : ((int64_t) g.M + tm - 1) / tm;
        const int64_t nt = ((int64_t) g.N + tn - 1) / tn;
        const int64_t grid = GROUPED ? (mt + 7) / 8 * 8 * nt : (mt * nt + 7) / 8 * 8;
        WZY_REQUIRE(grid * threads < (int64_t) 1 << 32, "wzy_mx_%sgemm: %lld tiles", GROUPED ? "grouped_" : "", (long long) grid);
        g.mt = (int) mt;
        g.nt = (int) nt;
        kernel<<<(uint32_t) grid, threads, 0, st>>>(g);
        WZY_LAUNCH_CHECK();
        return WZY_OK;
    };
    if constexpr (GROUPED) {
        if (far_rows(g)) return go(mx_far_kernel<FMT, OUT>, 64, 64, 256);
    } else {
        // Up to 16 rows: 16 x 64 tiles where there are enough of them, or K split over the waves.  1 row, E4M3 to fp32, us: N 2,048, K
        // 2,048 5.0 against 4.8; N 2,048, K 6,144 9.1, 5.9; N 12,288, K 2,048 5.7, 6.6; 4 x 151,936 x 2,048 35, 56.
        if (g.M <= 16 && g.N <= 4096) {
            mx_skinny_kernel<FMT, OUT><<<(g.N + 15) / 16, 64 * std::min(8, (g.K + 511) / 512), 0, st>>>(g);
            WZY_LAUNCH_CHECK();
            return WZY_OK;
        }
    }
    auto tiles = [&](auto any_) {
        constexpr bool ANY = any_();
        const Tile t = GROUPED ? grouped_tile(g, E8, !ANY) : g.M <= 16 ? T16x64 : dense_tile(g, E8, !ANY);
        if (t == T16x64) return go(mx_dma_kernel<FMT, OUT, 16, 64, 1, 2, 2, 256, 3, 2, GROUPED, ANY>, 16, 64, 256);
        if (t == T64x128) return go(mx_dma_kernel<FMT, OUT, 64, 128, 1, 4, 1, 256, 2, 2, GROUPED, ANY>, 64, 128, 256);
        if constexpr (GROUPED) {
            if (t == T32x128) return go(mx_dma_kernel<FMT, OUT, 32, 128, 1, 4, 1, 256, 3, 2, GROUPED, ANY>, 32, 128, 256);
        } else {
            // Products in two parts, at most a tile a CU: both halves of a unit at once.  To fp32, 32 x 2,048 x 6,144 13.9 -> 12.1 us, 250 x 2,048 x
            // 2,048 7.1 -> 6.7; the other types 4 to 15 % slower, ANY no faster.
            if constexpr (!ANY && two_parts(FMT, OUT)) {
                if (t == T32x64 && ((int64_t) g.M + 31) / 32 * (((int64_t) g.N + 63) / 64) <= CUS)
                    return go(mx_dma_kernel<FMT, OUT, 32, 64, 2, 2, 2, 256, 3, 2, GROUPED, ANY>, 32, 64, 512);
            }
            if (t == T32x64) return go(mx_dma_kernel<FMT, OUT, 32, 64, 2, 2, 1, 256, 3, 2, GROUPED, ANY>, 32, 64, 256);
            if (t == T64x64) return go(mx_dma_kernel<FMT, OUT, 64, 64, 2, 2, 1, 256, 3, 2, GROUPED, ANY>, 64, 64, 256);
        }
        if constexpr (!ANY && (!E8 || (!GROUPED && OUT != WZY_F32))) {
            if (t == T256x256) return go(mx_dma_kernel<FMT, OUT, 256, 256, 2, 4, 1, E8 ? 128 : 256, E8 ? 3 : 2, 2, GROUPED, ANY>, 256, 256, 512);
        }
        return go(mx_dma_kernel<FMT, OUT, 128, 128, 2, 2, 1, E8 ? 128 : 256, 2, 2, GROUPED, ANY>, 128, 128, 256);
    };
    return whole_steps(g) ? tiles(std::false_type()) : tiles(std::true_type());
}
template <bool GROUPED>
int dispatch(const MxGemm& g, int fmt, hipStream_t st) {
    return mx_with_type(g.y_type, [&](auto t) {
        return fmt == WZY_MX_E4M3 ? launch<WZY_MX_E4M3, t(), GROUPED>(g, st) : launch<WZY_MX_E2M1, t(), GROUPED>(g, st);
    });
}

int check_gemm(const char* who, const wzy_mx_mat* a, const wzy_mx_mat* w, MxGemm& g) {
    WZY_REQUIRE(g.M >= 0 && g.N >= 0 && g.K >= 32 && g.K % 32 == 0 && g.K <= 1 << 20, "%s: %d x %d x %d (K a multiple of 32 up to 2^20)",
                who, g.M, g.N, g.K);
    WZY_TRY(mx_check_type(who, g.y_type));
    if (g.M == 0 || g.N == 0) return WZY_OK;
    WZY_TRY(mx_check_mat(who, "a", a, g.K, g.a));
    WZY_TRY(mx_check_mat(who, "w", w, g.K, g.w));
    WZY_REQUIRE(w->fmt == WZY_MX_E2M1, "%s: w is E2M1", who);
    WZY_REQUIRE(g.y && (uintptr_t) g.y % mx_type_bytes(g.y_type) == 0 && g.ldy >= g.N, "%s: y at %p, row stride %lld (at least %d)", who,
                g.y, (long long) g.ldy, g.N);
    return WZY_OK;
}

}  // namespace

extern "C" int wzy_mx_gemm(const wzy_mx_mat* a, const wzy_mx_mat* w, int M, int N, int K, void* y, int y_type, int64_t ldy,
                           void* stream) {
    MxGemm g{};
    g.y = y; g.ldy = ldy; g.M = M; g.N = N; g.K = K; g.y_type = y_type; g.a_rows = M;
    WZY_TRY(check_gemm("wzy_mx_gemm", a, w, g));
    if (M == 0 || N == 0) return WZY_OK;
    return dispatch<false>(g, a->fmt, as_stream(stream));
}

extern "C" int wzy_mx_grouped_gemm(const wzy_mx_mat* a, int a_rows, const int* row_ids, const wzy_mx_mat* w, const int* offsets,
                                   int groups, int M, int N, int K, void* y, int y_type, int64_t ldy, void* stream) {
    const char* const who = "wzy_mx_grouped_gemm";
    MxGemm g{};
    g.y = y; g.ldy = ldy; g.M = M; g.N = N; g.K = K; g.y_type = y_type; g.a_rows = a_rows;
    g.row_ids = row_ids; g.offsets = offsets; g.groups = groups;
    WZY_REQUIRE(groups >= 1 && groups <= 65536, "%s: %d groups (1 .. 65,536)", who, groups);
    WZY_TRY(check_gemm(who, a, w, g));
    if (M == 0 || N == 0) return WZY_OK;
    WZY_REQUIRE(a_rows >= 1, "%s: %d rows of a", who, a_rows);
    WZY_REQUIRE(offsets, "%s: offsets is null", who);
    WZY_REQUIRE(row_ids || a_rows >= M, "%s: %d rows of a for %d entries without row_ids", who, a_rows, M);
    return dispatch<true>(g, a->fmt, as_stream(stream));
}
