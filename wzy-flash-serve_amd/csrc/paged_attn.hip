// paged_attn.hip -- attention of new tokens over a paged key-value cache.
//
//   o = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m),   t_j = scale log2(e) q . k_j,   m the running maximum of t
//
// One pass over the keys, 32 at a time, on v_mfma_f32_32x32x16: S^T = K Q^T, then O^T += V^T P^T.  The products are taken
// transposed so that a lane holds one query row throughout: of S^T it has 16 keys' scores (the other 16 are in the lane 32
// away), so maximum and sum cost one exchange between the halves, rescaling is by a lane's own factor, and the accumulator
// registers of S^T, rounded, are P^T's operand as they stand: register i of lane half h is key 8 (i / 4) + 4 h + i % 4, which
// is the order in which V^T's operand then takes its keys (the product's sum may run over them in any order).  V lies in LDS
// as in memory, a row a key, and ds_read_b64_tr_b16 hands each lane four keys of one column.
//
// Rows are (token, head of the group) pairs of one key head, so a group's heads share every byte of K and V.
//   narrow  up to 32 rows: the waves of a workgroup take every fourth block of 32 keys each, through buffers of their own,
//           with no barrier until their results are joined.  Bound by memory: 64 single tokens of requests of up to 6,000 cells,
//           8 key heads of 128, 280 us (5.5 TB/s).  One of 32,768 cells, 2 heads of 256, 17 us and 6 for the merge of its 256 parts:
//           67 MB in one wave of workgroups, whose first loads and joins are half of it
//   middle  up to 64 rows, where no request of the step has more (verify windows): two waves share a block, the two pairs take
//           every other one.  16 windows of 4 tokens x 12 heads of 256 over 4,096 cells: 30 us and 7 for the merge (with the wide form,
//           whose tiles would hold 80 empty rows, 47 for both before it was there and 40 after).  Bound by memory and the start of
//           each part
//   wide    128 rows, 32 a wave: the workgroup's waves share each block.  2,047 tokens x 12 heads of 256 behind 30,001 cells:
//           1,420 us with 36 for the merge, 1,100 TFLOP/s (a library's 8,192^3 product: 1,184); prompts, heads of 128: 940 us, 945
//           TFLOP/s (cards differ by 5 % in both).  Bound by the matrix cores and the vector units' exponentials in turn: neither
//           fewer operations a block nor fewer LDS reads (64 rows a wave, in twice the registers: 1,255 us for the prompts) make it
//           faster.  256 rows on 8 waves: 1,185
// The maximum follows the scores only when one has come 2^8 above it, so most blocks leave the accumulators alone; weights
// then reach 2^8, and in fp16, whose numbers end at 2^-24, all are taken 2^6 larger.
#include <algorithm>

#include "wzy_paged.h"

using namespace wzy;

typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef __bf16 v8b_t __attribute__((ext_vector_type(8)));
typedef _Float16 v8h_t __attribute__((ext_vector_type(8)));
typedef float v16f_t __attribute__((ext_vector_type(16)));
typedef uint32_t v4w_t __attribute__((ext_vector_type(4)));

namespace {

struct AttnArgs {
    const char* k;
    const char* v;
    int64_t ld_page, ld_cell, ld_head;       // bytes
    const int* table;
    const char* q;
    char* out;
    int64_t ldq, ldq_head, ldo, ldo_head;    // bytes
    const PgHead* head;
    float* part_o;                           // [part][kvh][tile rows][hd]
    float2* part_ml;                         // [part][kvh][tile rows]: maximum, sum
    FastDiv div_g;
    float c;                                 // scale * log2(e)
    int n_pages, lp, max_pages, n_req, max_tokens;
    int g, kvh, window, geometry;
    int item_at, cap_parts;
};

template <int T> struct Half;                // of the cache's type
template <> struct Half<WZY_BF16> {
    static constexpr float SHIFT = 0.0f;
    static constexpr uint32_t EXP = 0x7F80;             // of what is not finite
    static WZY_DEV float value(uint32_t b) { return bf16_lo(b); }
    static WZY_DEV v16f_t mfma(v4w_t a, v4w_t b, v16f_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b_t, a), __builtin_bit_cast(v8b_t, b), c, 0, 0, 0);
    }
};
template <> struct Half<WZY_F16> {
    static constexpr float SHIFT = 6.0f;
    static constexpr uint32_t EXP = 0x7C00;
    static WZY_DEV float value(uint32_t b) { return h16_to_f((uint16_t) b); }
    static WZY_DEV v16f_t mfma(v4w_t a, v4w_t b, v16f_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h_t, a), __builtin_bit_cast(v8h_t, b), c, 0, 0, 0);
    }
};
constexpr float RISE = 8.0f;
constexpr int MERGE_THREADS = 256, MERGE_LOADS = 8;       // of a part's row, under way at once
constexpr unsigned MERGE_SHARED = 1024;                   // workgroups of a merge, up to which they share rows

WZY_DEV uint32_t lds_offset(const void* p) { return (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) char*) p; }
// 64 lanes x 16 bytes to LDS lds .. lds + 1023 in lane order, from a wave-uniform base + off, or from an address a lane
WZY_DEV void dma16(uint32_t lds, uint32_t off, const char* base) {
    uint32_t m0;
    lds = (uint32_t) __builtin_amdgcn_readfirstlane((int) lds);          // nothing where it is in a scalar register already
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %2, %3" : "={m0}"(m0) : "s"(lds), "v"(off), "s"(base) : "memory");
}
WZY_DEV void dma16(uint32_t lds, const char* p) {
    uint32_t m0;
    lds = (uint32_t) __builtin_amdgcn_readfirstlane((int) lds);          // nothing where it is in a scalar register already
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %2, off" : "={m0}"(m0) : "s"(lds), "v"(p) : "memory");
}
// this wave's loads but the last N have landed
template <int N>
WZY_DEV void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
WZY_DEV void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// this wave's loads have landed and its LDS reads are done; then all waves meet
WZY_DEV void wait_all_and_meet() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// this wave's loads but the last N have landed; then all waves meet
template <int N>
WZY_DEV void wait_loads_and_meet() { asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory"); }
WZY_DEV void wait_lds_and_meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
WZY_DEV const char* uniform(const char* p) {
    const uint64_t b = (uint64_t) (uintptr_t) p;
    return (const char*) (uintptr_t) ((uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (b >> 32)) << 32 |
                                      (uint32_t) __builtin_amdgcn_readfirstlane((int) b));
}
// lane l's value and lane l ^ 32's, in either order
WZY_DEV float2 both_halves(float v) {
    uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
    return make_float2(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
WZY_DEV float half_max(float v) { const float2 b = both_halves(v); return fmaxf(b.x, b.y); }
WZY_DEV float half_sum(float v) { const float2 b = both_halves(v); return b.x + b.y; }

// K or V of 32 keys in LDS: a row a key, as the loads leave them, 1 KiB (ROWS keys) each.  Within those the 16-byte pieces of
// a row change places by its number (an exclusive or), and the loads lie PAD apart, so that the lanes that read at once find
// all banks: K is read as 32 rows' same piece, V as 4 rows x 64 bytes.  Both permutations leave all but a few bits of a piece's
// number alone: a lane needs SETS addresses, the rest are offsets in the instructions.
template <int HD, bool V>
struct Block {
    static constexpr int PIECES = HD / 8, ROW = HD * 2, LOADS = 32 * ROW / 1024, ROWS = 64 / PIECES;
    static constexpr int PAD = V && HD == 256 ? 64 : 16, STEP = 1024 + PAD, BYTES = LOADS * STEP;
    // pieces change places in units of 1 << SHIFT pieces
    static constexpr int SHIFT = HD == 256 ? 3 : HD == 128 || V ? 2 : 1, SETS = HD == 256 || (HD == 64 && V) ? 2 : 4;
    static WZY_DEV int swap(int row) { return HD == 64 ? (row >> 1) & (SETS - 1) : row & (SETS - 1); }
    static WZY_DEV int row_at(int row) { return row / ROWS * STEP + row % ROWS * ROW; }
    // addresses of a lane: set j for pieces whose bits at SHIFT are j
    static WZY_DEV void addresses(uint32_t (&at)[SETS], int lane) {
        const int i = lane & 15, row = V ? 4 * (lane >> 5) + (i >> 2) : lane & 31;
        const int low = V ? (2 * (lane >> 4 & 1) + (i >> 1 & 1)) * 16 + 8 * (i & 1) : (lane >> 5) * 16;
#pragma unroll
        for (int j = 0; j < SETS; ++j) at[j] = (uint32_t) (row_at(row) + low + ((j ^ swap(row)) << (SHIFT + 4)));
    }
    // K's operand of columns 16 s ..: row l % 32, piece 2 s + l / 32
    static WZY_DEV v4w_t k_operand(const char* lds, const uint32_t (&at)[SETS], int s) {
        constexpr int M = (SETS - 1) << SHIFT;
        const int piece = 2 * s;
        return *(const v4w_t*) (lds + at[(piece & M) >> SHIFT] + (piece & ~M) * 16);
    }
    // V^T's operand of columns 32 d + l % 32: keys 16 s + 4 h + 0 .. 3 and 8 more than those, h = l / 32
    static WZY_DEV v4w_t v_operand(const char* lds, const uint32_t (&at)[SETS], int s, int d) {
        constexpr int M = (SETS - 1) << SHIFT;
        const int piece = 4 * d;
        v4w_t r;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const char* const from = lds + at[(piece & M) >> SHIFT] + (piece & ~M) * 16 + row_at(16 * s + 8 * p);
            const uint2 w = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s_t*) from));
            r[2 * p] = w.x;
            r[2 * p + 1] = w.y;
        }
        return r;
    }
};

// A tile's place in the step
struct TileCtx {
    PgItem it;
    int head;                                // key head
    const int* pages;                        // the request's row of the table
};

// Loads of one block's K or V.  Rows of a block are 32 neighbouring cells from a multiple of 32, so a page holds all of them or
// (16 cells a page) a half.  Blocks that reach past the part's cells repeat its first or last: what lies there in memory may be
// anything, a NaN too, and a weight of 0 does not silence it.
template <int HD>
struct Loader {
    using BK = Block<HD, false>;
    using BV = Block<HD, true>;
    const AttnArgs& a;
    const TileCtx& t;
    int r0;                                  // the lane's row of a load
    int piece_k, piece_v;                    // and the bytes of that row it takes
    const char* base[2];                     // of K's halves; V's are as far off
    int64_t to_v;
    bool whole;
    int first, last;                         // rows that are there, where not all are
    WZY_DEV Loader(const AttnArgs& a_, const TileCtx& t_, int lane) : a(a_), t(t_), to_v(a_.v - a_.k) {
        r0 = lane / BK::PIECES;
        const int piece = lane % BK::PIECES;
        piece_k = (piece ^ (BK::swap(r0) << BK::SHIFT)) * 16;
        piece_v = (piece ^ (BV::swap(r0) << BV::SHIFT)) * 16;
    }
    WZY_DEV const char* cell(int c) const {
        // through the scalar cache: a vector load would be waited for together with the keys and values on their way
        int id = ((const __attribute__((address_space(4))) int*) t.pages)[__builtin_amdgcn_readfirstlane(c >> a.lp)];
        id = (unsigned) id < (unsigned) a.n_pages ? id : 0;
        return a.k + (int64_t) id * a.ld_page + (int64_t) (c & ((1 << a.lp) - 1)) * a.ld_cell + (int64_t) t.head * a.ld_head;
    }
    // the block of cells 32 b .. 32 b + 31, at least one of them the part's
    WZY_DEV void at(int b) {
        const int c = 32 * b;
        whole = c >= t.it.lo && c + 32 <= t.it.hi;
        first = max(t.it.lo - c, 0);
        last = min(t.it.hi - c, 32) - 1;
        // cells of a half that has none of the part are not looked up
        const int h0 = first < 16 ? 0 : 16, h1 = last >= 16 ? 16 : 0;
        base[0] = uniform(cell(c + h0));
        base[1] = uniform(h1 == h0 ? base[0] : cell(c + h1));
    }
    // loads start .. start + N - 1 of the block's into lds
    template <bool V, int N>
    WZY_DEV void issue(uint32_t lds, int start) const {
        using B = Block<HD, V>;
        const int piece = V ? piece_v : piece_k;
        const int64_t add = V ? to_v : 0;
        if (whole) {
            const uint32_t off = (uint32_t) r0 * (uint32_t) a.ld_cell + (uint32_t) piece;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = (start + i) * B::ROWS;
                dma16(lds + (uint32_t) ((start + i) * B::STEP), off, uniform((row < 16 ? base[0] : base[1]) + add + (int64_t) (row & 15) * a.ld_cell));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int from = min(max((start + i) * B::ROWS + r0, first), last);
                dma16(lds + (uint32_t) ((start + i) * B::STEP), (from < 16 ? base[0] : base[1]) + add + (int64_t) (from & 15) * a.ld_cell + piece);
            }
        }
    }
};

// A wave's 32 query rows
template <int HD, int T>
struct Wave {
    static constexpr int KS = HD / 16, DT = HD / 32;
    using BK = Block<HD, false>;
    using BV = Block<HD, true>;
    uint32_t at_k[BK::SETS], at_v[BV::SETS];
    v4w_t q[KS];
    v16f_t o[DT];
    float m, l;
    int pos, pos_min, pos_max;               // of the lane's row; of the wave's
    int row, rows;                           // the lane's row of the request's; how many those are

    WZY_DEV void start(const AttnArgs& a, const TileCtx& t, int row0, int lane) {
        BK::addresses(at_k, lane);
        BV::addresses(at_v, lane);
        rows = t.it.n_new * a.g;
        row = row0 + (lane & 31);
        pos_min = t.it.n_cached + (int) fast_div((uint32_t) min(row0, rows - 1), a.div_g);
        pos_max = t.it.n_cached + (int) fast_div((uint32_t) min(row0 + 31, rows - 1), a.div_g);
        const int r = min(row, rows - 1), token = (int) fast_div((uint32_t) r, a.div_g), h = r - token * a.g;
        pos = t.it.n_cached + token;
        const char* const p = a.q + (int64_t) (t.it.q0 + token) * a.ldq + (int64_t) (t.head * a.g + h) * a.ldq_head + (lane >> 5) * 16;
#pragma unroll
        for (int s = 0; s < KS; ++s) q[s] = row < rows ? *(const v4w_t*) (p + 32 * s) : v4w_t{0, 0, 0, 0};
        // taken here: else the compiler waits for them in the loop, each time, and for the keys on their way with them
#pragma unroll
        for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[s]));
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = v16f_t{};
        m = -INFINITY;
        l = 0.0f;
    }
    // are there cells of block b that some row does not see?
    WZY_DEV bool masked(const AttnArgs& a, int b) const {
        return 32 * b + 31 > pos_min || (a.window != 0 && 32 * b <= pos_max - a.window);
    }
    // Operands are read AHEAD steps before their product, and the order is held: left alone, the compiler reads them all first, into
    // registers that there are not.
    static constexpr int AHEAD = 3;
    WZY_DEV v16f_t scores(const char* kb) const {
        v4w_t k[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) k[i] = BK::k_operand(kb, at_k, i);
        v16f_t s = v16f_t{};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            s = Half<T>::mfma(k[i % AHEAD], q[i], s);
            if (i + AHEAD < KS) k[i % AHEAD] = BK::k_operand(kb, at_k, i + AHEAD);
        }
        __builtin_amdgcn_sched_barrier(0);
        return s;
    }
    // Scores to weights, rounded to the cache's type and packed, as the product takes them: the sum has them unrounded, so an output is off
    // by half a step of its weights' at most.  (A second product of what the rounding left off would take that away, for half as many
    // matrix instructions again in the wide form; but an infinity that a row sees would meet remainders that are 0 or negative, and
    // the sum would not be a number.)
    WZY_DEV void weights(const AttnArgs& a, int b, int lane, v16f_t s, v4w_t (&p)[2]) {
        if (masked(a, b)) {
            const int low = a.window ? pos - a.window : -1;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = 32 * b + 8 * (i / 4) + 4 * (lane >> 5) + i % 4;
                s[i] = key <= pos && key > low ? s[i] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        mx = half_max(mx) * a.c;
        if (__any(mx > m + RISE)) {
            const float to = fmaxf(m, mx), f = to > -INFINITY ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
            m = to;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= f;
        }
        const float less = m > -INFINITY ? Half<T>::SHIFT - m : 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c, less));
            l += s[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i / 4][i % 4] = pack2<T>(s[2 * i], s[2 * i + 1]);
    }
    WZY_DEV void add(const char* vb, const v4w_t (&p)[2]) {
        v4w_t v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = BV::v_operand(vb, at_v, i % 2, i / 2);
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            o[i / 2] = Half<T>::mfma(v[i % AHEAD], p[i % 2], o[i / 2]);
            if (i + AHEAD < 2 * DT) v[i % AHEAD] = BV::v_operand(vb, at_v, (i + AHEAD) % 2, (i + AHEAD) / 2);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
};

// The blocks from .. to - 1 that every token at pos_min .. pos_max sees whole.
struct Seen {
    int from, to;
    WZY_DEV Seen(const AttnArgs& a, int pos_min, int pos_max)
        : from(a.window != 0 && pos_max >= a.window ? ((pos_max - a.window) >> 5) + 1 : 0), to((pos_min + 1) >> 5) {}
    WZY_DEV bool all(int b) const { return b >= from && b < to; }
};
// A weight of 0 does not silence a value that is not finite.  So where some row of a tile does not see all of a block (or the block
// repeats a cell at the part's ends), such values of V become 0 in LDS before the products, and add_hidden brings them to the rows that
// see their cells afterwards.  (Leaving them out of the operands costs registers that there are not: 1.7 times the time.  Doing the
// rows again one by one over the whole part: a chunk of 2,047 tokens behind 30,001 cells 240 ms.)  Loads start .. start + N - 1 of V's,
// which have landed; was there one?
template <int HD, int T, int N>
WZY_DEV bool hide(char* vb, int start, int lane) {
    constexpr uint32_t EXP2 = Half<T>::EXP * 0x10001u, ONE2 = (0x8000u - Half<T>::EXP) * 0x10001u;
    using BV = Block<HD, true>;
    bool found = false;
#pragma unroll 4
    for (int i = 0; i < N; ++i) {
        v4w_t* const p = (v4w_t*) (vb + (start + i) * BV::STEP + 16 * lane);
        v4w_t x = *p;
        uint32_t hot[4], any = 0;                                       // an exponent of all ones and one more: the half's top bit
#pragma unroll
        for (int j = 0; j < 4; ++j) any |= hot[j] = ((x[j] & EXP2) + ONE2) & 0x80008000u;
        if (any) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] &= ~((hot[j] >> 15) * 0xFFFFu);
            *p = x;
            found = true;
        }
    }
    wave_lds_sync();
    return __any(found);
}
// the workgroup's item and key head; false where there is none, or the list is not one of this step
WZY_DEV bool tile_ctx(const AttnArgs& a, int kind, TileCtx& t) {
    const int at = (int) (blockIdx.x / (unsigned) a.kvh);
    t.head = (int) (blockIdx.x - (unsigned) at * (unsigned) a.kvh);
    const PgHead h = *a.head;                                           // both loads at once: the list has room for every workgroup
    t.it = ((const PgItem*) (a.head + 1))[a.item_at + at];
    const PgItem& i = t.it;
    if (h.magic != PG_MAGIC || h.geometry != a.geometry || at >= h.n_items[kind]) return false;
    if ((unsigned) i.req >= (unsigned) a.n_req || i.q0 < 0 || i.n_new < 1 || i.q0 > a.max_tokens - i.n_new || i.row0 < 0 || i.row0 >= i.n_new * a.g ||
        i.lo < 0 || i.hi > a.max_pages << a.lp || i.part >= a.cap_parts)
        return false;
    t.pages = a.table + (size_t) i.req * a.max_pages;
    return true;
}
WZY_DEV char* out_row(const AttnArgs& a, const TileCtx& t, int row) {
    const int token = (int) fast_div((uint32_t) row, a.div_g);
    return a.out + (int64_t) (t.it.q0 + token) * a.ldo + (int64_t) (t.head * a.g + row - token * a.g) * a.ldo_head;
}

// is there such a value in the first or the last row of lo .. hi - 1 that a block holds?
template <int HD, int T>
WZY_DEV bool hot_ends(const char* vb, int lo, int hi, int lane) {
    using BV = Block<HD, true>;
    const int row = lane < 32 ? max(lo, 0) : min(hi, 32) - 1;
    const v4w_t x = *(const v4w_t*) (vb + BV::row_at(row) + 16 * (lane % BV::PIECES));
    bool hot = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) hot |= (x[j] & Half<T>::EXP) == Half<T>::EXP || (x[j] >> 16 & Half<T>::EXP) == Half<T>::EXP;
    return __any(hot);
}
// Results of rows from .. to - 1, which are out, get what hide() took from V: whatever its weight, a value that is not finite makes the
// sum infinite, or with another not a number.  A wave reads the cells of all blocks outside `seen`, E columns a lane, CELLS at once.
// (What was there already may come again: the sum is the same.)
template <int HD, int T>
WZY_DEV void add_hidden(const AttnArgs& a, const TileCtx& t, const Seen& seen, int from, int to, int lane, int tile_rows) {
    constexpr int E = HD / 64, CELLS = 8;
    const int split = max(seen.from, seen.to) == seen.to ? 32 * seen.from : t.it.hi;         // no block is seen whole: all cells
    for (int k = 0; k < 2; ++k) {                                       // before the blocks that are seen whole, behind them
        const int c0 = k ? max(t.it.lo, max(split, 32 * seen.to)) : t.it.lo, c1 = k ? t.it.hi : min(t.it.hi, split);
        for (int c = c0; c < c1; c += CELLS) {
            float v[CELLS][E];                                          // what is not finite
            bool hot = false;
#pragma unroll
            for (int j = 0; j < CELLS; ++j) {
                const int cell = min(c + j, c1 - 1);
                int id = t.pages[cell >> a.lp];
                id = (unsigned) id < (unsigned) a.n_pages ? id : 0;
                const uint16_t* const p = (const uint16_t*) (a.v + (int64_t) id * a.ld_page + (int64_t) (cell & ((1 << a.lp) - 1)) * a.ld_cell +
                                                             (int64_t) t.head * a.ld_head) + E * lane;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = Half<T>::value(p[e]);
                    v[j][e] = fabsf(x) < INFINITY ? 0.0f : x;
                    hot |= !(fabsf(x) < INFINITY);
                }
            }
            if (!__any(hot)) continue;
            for (int row = from; row < to; ++row) {
                const int pos = t.it.n_cached + (int) fast_div((uint32_t) row, a.div_g);
                const int lo = a.window != 0 ? pos - a.window + 1 : 0, hi = min(pos + 1, c1);
                float x[E] = {};
#pragma unroll
                for (int j = 0; j < CELLS; ++j)
                    if (c + j >= lo && c + j < hi)
#pragma unroll
                        for (int e = 0; e < E; ++e) x[e] += v[j][e];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (x[e] == 0.0f) continue;
                    const int column = E * lane + e;
                    if (t.it.part < 0) {
                        uint16_t* const out = (uint16_t*) out_row(a, t, row) + column;
                        const float y = Half<T>::value(*out) + x[e];
                        *out = (uint16_t) pack2<T>(y, y);
                    } else a.part_o[(((size_t) t.it.part * a.kvh + t.head) * tile_rows + (row - t.it.row0)) * HD + column] += x[e];
                }
            }
        }
    }
}
// A request that is not served: all its rows become 0.
template <int HD>
WZY_DEV void zero_rows(const AttnArgs& a, const TileCtx& t) {
    constexpr int L = HD / 8;                                           // threads a row
    for (int row = threadIdx.x / L; row < t.it.n_new * a.g; row += 256 / L)
        *(v4w_t*) (out_row(a, t, row) + 16 * (threadIdx.x % L)) = v4w_t{0, 0, 0, 0};
}
// A lane's results: its row's columns in 16-byte (a part: fp32) or 8-byte pieces
template <int HD, int T>
WZY_DEV void put_row(const AttnArgs& a, const TileCtx& t, const Wave<HD, T>& w, float l, int lane, int tile_rows) {
    if (w.row >= w.rows) return;
    if (t.it.part < 0) {
        const float n = l != 0.0f ? 1.0f / l : 0.0f;
        char* const p = out_row(a, t, w.row) + 8 * (lane >> 5);
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(uint2*) (p + 64 * d + 16 * i) = make_uint2(pack2<T>(w.o[d][4 * i] * n, w.o[d][4 * i + 1] * n),
                                                             pack2<T>(w.o[d][4 * i + 2] * n, w.o[d][4 * i + 3] * n));
    } else {
        const size_t at = ((size_t) t.it.part * a.kvh + t.head) * tile_rows + (w.row - t.it.row0);
        float4* const p = (float4*) (a.part_o + at * HD) + (lane >> 5);
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[8 * d + 2 * i] = make_float4(w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]);
        if (lane < 32) a.part_ml[at] = make_float2(w.m, l);
    }
}

template <int HD, int T>
__global__ void __launch_bounds__(256) paged_narrow_kernel(AttnArgs a) {
    using BK = Block<HD, false>;
    using BV = Block<HD, true>;
    constexpr int MINE = BK::BYTES + BV::BYTES;
    __shared__ __align__(1024) char s_buf[4][MINE];                     // a wave's K and V; then its results in fp32
    __shared__ float s_m[4][32], s_l[4][32];
    __shared__ int s_hidden[4];
    static_assert(MINE >= 32 * HD * 4 && MINE % 16 == 0, "a wave's results take its buffers");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    TileCtx t;
    if (!tile_ctx(a, 0, t)) return;
    if (t.it.part < 0 && t.it.lo >= t.it.hi) {
        zero_rows<HD>(a, t);
        return;
    }
    Wave<HD, T> w;
    Loader<HD> ld(a, t, lane);
    char* const kb = s_buf[wave];
    char* const vb = kb + BK::BYTES;
    const uint32_t lk = lds_offset(kb), lv = lds_offset(vb);
    const int end = (t.it.hi + 31) >> 5;
    int b = (t.it.lo >> 5) + wave;
    if (lane == 0) s_hidden[wave] = 0;
    // the first block's loads before those of q, which the compiler counts as the only ones: it waits for all of them
    if (b < end) {
        ld.at(b);
        ld.template issue<false, BK::LOADS>(lk, 0);
        ld.template issue<true, BV::LOADS>(lv, 0);
    }
    w.start(a, t, 0, lane);
    const Seen seen(a, w.pos_min, w.pos_max);
    if (b < end) {
        wait_loads<0>();
        for (;; b += 4) {
            const bool more = b + 4 < end;
            wait_loads<BV::LOADS>();                                    // K is there
            const v16f_t s = w.scores(kb);
            wait_lds();                                                 // and read
            if (more) {
                ld.at(b + 4);
                ld.template issue<false, BK::LOADS>(lk, 0);
            }
            v4w_t p[2];
            w.weights(a, b, lane, s, p);
            if (more) wait_loads<BK::LOADS>();
            else wait_loads<0>();
            if (!seen.all(b)) {
                // of a single token, which is common, only the ends, which are repeated (over 2,000 cells, 12.6 us: all of V 0.5 us more)
                bool look = t.it.n_new > 1;
                if (!look) look = hot_ends<HD, T>(vb, t.it.lo - 32 * b, t.it.hi - 32 * b, lane);
                if (look && hide<HD, T, BV::LOADS>(vb, 0, lane) && lane == 0) s_hidden[wave] = 1;
            }
            w.add(vb, p);
            if (!more) break;
            wait_lds();
            ld.template issue<true, BV::LOADS>(lv, 0);
        }
    }
    w.l = half_sum(w.l);
    if (lane < 32) {
        s_m[wave][lane] = w.m;
        s_l[wave][lane] = w.l;
    }
    // results as [column / 4][row][4]: neighbouring lanes side by side
    wait_lds();
    float4* const r = (float4*) s_buf[wave];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[(8 * d + 2 * i + (lane >> 5)) * 32 + (lane & 31)] =
                make_float4(w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]);
    __syncthreads();
    const int rows = w.rows;
    for (int i = tid; i < rows * (HD / 4); i += 256) {
        const int row = i / (HD / 4), col = i % (HD / 4);
        float m = s_m[0][row], l = 0.0f;
#pragma unroll
        for (int k = 1; k < 4; ++k) m = fmaxf(m, s_m[k][row]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = s_l[k][row] != 0.0f ? __builtin_amdgcn_exp2f(s_m[k][row] - m) : 0.0f;
            const float4 x = ((const float4*) s_buf[k])[col * 32 + row];
            l += f * s_l[k][row];
            o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
        }
        if (t.it.part < 0) {
            const float n = l != 0.0f ? 1.0f / l : 0.0f;
            *(uint2*) (out_row(a, t, row) + 8 * col) = make_uint2(pack2<T>(o.x * n, o.y * n), pack2<T>(o.z * n, o.w * n));
        } else {
            const size_t at = ((size_t) t.it.part * a.kvh + t.head) * 32 + row;
            ((float4*) (a.part_o + at * HD))[col] = o;
            if (col == 0) a.part_ml[at] = make_float2(m, l);
        }
    }
    if (s_hidden[0] | s_hidden[1] | s_hidden[2] | s_hidden[3]) {
        __syncthreads();
        add_hidden<HD, T>(a, t, seen, 8 * wave, min(8 * wave + 8, rows), lane, 32);
    }
}

// Three times a block all waves meet: when K is there; when it has been read and V is there (the next K's loads start); when V has been
// read (its next loads start), but after the last block.  Both pairs meet as often, so a pair without a block in the first's last round
// meets twice more.
template <int HD, int T>
__global__ void __launch_bounds__(256, 2) paged_middle_kernel(AttnArgs a) {
    using BK = Block<HD, false>;
    using BV = Block<HD, true>;
    constexpr int BOTH = BK::BYTES + BV::BYTES, MINE = BK::LOADS / 2;
    __shared__ __align__(1024) char s_buf[2][BOTH];                     // a pair's K and V; then the second pair's results in fp32
    __shared__ float s_m[64], s_l[64];
    __shared__ int s_hidden[4];
    static_assert(2 * BOTH >= 64 * HD * 4, "a pair's results take the buffers");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave & 1, pair = wave >> 1;
    TileCtx t;
    if (!tile_ctx(a, 0, t)) return;
    if (t.it.part < 0 && t.it.lo >= t.it.hi) {
        zero_rows<HD>(a, t);
        return;
    }
    Wave<HD, T> w;
    Loader<HD> ld(a, t, lane);
    const char* const kb = s_buf[pair];
    char* const vb = s_buf[pair] + BK::BYTES;
    const uint32_t lk = lds_offset(kb), lv = lk + BK::BYTES;
    const int first = t.it.lo >> 5, end = (t.it.hi + 31) >> 5;
    int b = first + pair;
    if (b < end) {
        ld.at(b);
        ld.template issue<false, MINE>(lk, half * MINE);
        ld.template issue<true, MINE>(lv, half * MINE);
    }
    w.start(a, t, 32 * half, lane);
    if (lane == 0) s_hidden[wave] = 0;
    const Seen seen(a, t.it.n_cached, t.it.n_cached + t.it.n_new - 1);  // of all of the tile's rows, which are the request's
    wait_loads<0>();
    // both pairs go round as often as the first has blocks; where the second has one fewer, it meets the first's last time
    const int rounds = (end - first + 1) / 2, mine = (end - first + 1 - pair) / 2;
    for (int n = rounds - mine; n < rounds; ++n, b += 2) {
        const bool more = b + 2 < end;
        wait_loads_and_meet<MINE>();                                    // K is there; V, whose loads are younger, may be on its way
        const v16f_t s = w.scores(kb);
        if (!seen.all(b)) {                                             // what this wave loaded
            wait_loads<0>();
            if (hide<HD, T, MINE>(vb, half * MINE, lane) && lane == 0) s_hidden[wave] = 1;
        }
        wait_all_and_meet();
        if (more) {
            ld.at(b + 2);
            ld.template issue<false, MINE>(lk, half * MINE);
        }
        v4w_t p[2];
        w.weights(a, b, lane, s, p);
        w.add(vb, p);
        if (n + 1 < rounds || mine < rounds) wait_lds_and_meet();
        if (more) ld.template issue<true, MINE>(lv, half * MINE);
    }
    if (mine < rounds) {
        wait_all_and_meet();
        wait_all_and_meet();
    }
    w.l = half_sum(w.l);
    wait_all_and_meet();                                                // the buffers have been read
    float4* const r = (float4*) (&s_buf[0][0] + half * 32 * HD * 4);
    if (pair == 1) {
        if (lane < 32) {
            s_m[32 * half + lane] = w.m;
            s_l[32 * half + lane] = w.l;
        }
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) r[(4 * d + i) * 64 + lane] = make_float4(w.o[d][4 * i], w.o[d][4 * i + 1], w.o[d][4 * i + 2], w.o[d][4 * i + 3]);
    }
    __syncthreads();
    if (pair == 1) return;
    const float m1 = s_m[32 * half + (lane & 31)], l1 = s_l[32 * half + (lane & 31)], m = fmaxf(w.m, m1);
    const float f0 = w.l != 0.0f ? __builtin_amdgcn_exp2f(w.m - m) : 0.0f, f1 = l1 != 0.0f ? __builtin_amdgcn_exp2f(m1 - m) : 0.0f;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 x = r[(4 * d + i) * 64 + lane];
            w.o[d][4 * i] = w.o[d][4 * i] * f0 + x.x * f1;
            w.o[d][4 * i + 1] = w.o[d][4 * i + 1] * f0 + x.y * f1;
            w.o[d][4 * i + 2] = w.o[d][4 * i + 2] * f0 + x.z * f1;
            w.o[d][4 * i + 3] = w.o[d][4 * i + 3] * f0 + x.w * f1;
        }
    w.m = m;
    put_row<HD, T>(a, t, w, w.l * f0 + l1 * f1, lane, 64);
    if (s_hidden[0] | s_hidden[1] | s_hidden[2] | s_hidden[3]) {
        __threadfence_block();
        add_hidden<HD, T>(a, t, seen, 32 * half, min(32 * half + 32, w.rows), lane, 64);
    }
}

template <int HD, int T>
__global__ void __launch_bounds__(256, 2) paged_wide_kernel(AttnArgs a) {
    using BK = Block<HD, false>;
    using BV = Block<HD, true>;
    constexpr int BOTH = BK::BYTES + BV::BYTES;
    __shared__ __align__(1024) char s_buf[2][BOTH];                     // two blocks' K and V
    __shared__ int s_hidden[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    TileCtx t;
    if (!tile_ctx(a, 1, t)) return;
    Wave<HD, T> w;
    Loader<HD> ld(a, t, lane);
    const uint32_t lk = lds_offset(s_buf);
    const int end = (t.it.hi + 31) >> 5;
    int b = t.it.lo >> 5, buf = 0;
    const bool any = b < end;
    constexpr int MINE = BK::LOADS / 4;                                 // of each matrix, a wave
    auto load = [&](int block, int into) {
        const uint32_t at = lk + (uint32_t) (into * BOTH);
        ld.at(block);
        ld.template issue<false, MINE>(at, wave * MINE);
        ld.template issue<true, MINE>(at + BK::BYTES, wave * MINE);
    };
    if (b < end) load(b, 0);
    w.start(a, t, t.it.row0 + 32 * wave, lane);
    wait_loads<0>();                                                    // q too, which the compiler counts without the others
    // the blocks that the wave's rows see: others' it helps to load and waits for.  (A loop each: a branch around the work in one loop
    // costs a second set of accumulators.)
    const int from = a.window ? max(b, (max(w.pos_min - a.window + 1, 0)) >> 5) : b, to = min(end, (w.pos_max >> 5) + 1);
    // of all of the tile's rows
    const Seen seen(a, t.it.n_cached + (int) fast_div((uint32_t) t.it.row0, a.div_g),
                    t.it.n_cached + (int) fast_div((uint32_t) min(t.it.row0 + PG_WIDE, w.rows) - 1u, a.div_g));
    if (lane == 0) s_hidden[wave] = 0;
    auto next = [&] {
        if (!seen.all(b)) {                                             // what this wave loaded
            wait_loads<0>();
            if (hide<HD, T, MINE>(s_buf[buf] + BK::BYTES, wave * MINE, lane) && lane == 0) s_hidden[wave] = 1;
        }
        wait_all_and_meet();                                            // the block is there; the other buffer has been read
        if (b + 1 < end) load(b + 1, buf ^ 1);
    };
    for (; b < from && b < end; ++b, buf ^= 1) next();
    for (; b < to; ++b, buf ^= 1) {
        next();
        const v16f_t s = w.scores(s_buf[buf]);
        v4w_t p[2];
        w.weights(a, b, lane, s, p);
        w.add(s_buf[buf] + BK::BYTES, p);
    }
    for (; b < end; ++b, buf ^= 1) next();
    put_row<HD, T>(a, t, w, half_sum(w.l), lane, PG_WIDE);
    if (any && (s_hidden[0] | s_hidden[1] | s_hidden[2] | s_hidden[3])) {
        __threadfence_block();
        const int row0 = t.it.row0 + 32 * wave;
        add_hidden<HD, T>(a, t, seen, row0, min(row0 + 32, w.rows), lane, PG_WIDE);
    }
}

// Parts of a tile joined.  COLS / 4 lanes hold COLS columns of a row; of a workgroup's groups of lanes, several take one row's parts in
// turn where there are many, so that all of a row's loads are under way at once.  Where all workgroups run at once, a row is shared by
// HD / 64 of them (one token's 12 rows of 128 parts in each of 2 heads: 7 -> 5.5 us; 16 verify windows, which would have 6,144
// workgroups: 7 -> 9), else it is one's.  Bound by latency: the list's entry, then a round of loads.
struct MergeArgs {
    unsigned blocks;                         // of narrow tiles
    int narrow;                              // rows of a narrow tile
    int rows_y[2], at[2], parts[2];          // workgroups a tile, first entry, parts: narrow, wide
    const float* wide_o;
    const float2* wide_ml;
};
template <int HD, int T, int COLS>
__global__ void __launch_bounds__(MERGE_THREADS) paged_merge_kernel(AttnArgs a, MergeArgs g) {
    constexpr int L = COLS / 4, GROUPS = MERGE_THREADS / L, SLICES = HD / COLS;
    __shared__ float4 s_o[MERGE_THREADS];
    __shared__ float2 s_ml[GROUPS];
    // narrow tiles' workgroups first, by rows_y of them a tile; then wide ones'
    const int kind = blockIdx.x >= g.blocks ? 1 : 0, rows_y = g.rows_y[kind], ROWS = kind ? PG_WIDE : g.narrow;
    const unsigned in = (blockIdx.x - (kind ? g.blocks : 0)) / SLICES, tile = in / (unsigned) rows_y, y = in - tile * (unsigned) rows_y;
    const int at = (int) (tile / (unsigned) a.kvh), head = (int) (tile - (unsigned) at * (unsigned) a.kvh);
    const PgHead h = *a.head;
    const PgMerge e = ((const PgMerge*) (a.head + 1))[g.at[kind] + at];
    if (h.magic != PG_MAGIC || h.geometry != a.geometry || at >= h.n_merges[kind]) return;
    if (e.part < 0 || e.n < 1 || e.part > g.parts[kind] - e.n || e.rows < 1 || e.rows > ROWS || e.row0 < 0 || e.row0 >= a.max_tokens * a.g || e.q0 < 0 ||
        e.q0 >= a.max_tokens)
        return;
    const float* const part_o = kind ? g.wide_o : a.part_o;
    const float2* const part_ml = kind ? g.wide_ml : a.part_ml;
    int per = 1;                                                        // groups a row
    while (per < GROUPS && per * MERGE_LOADS < e.n) per *= 2;
    const int rows_here = GROUPS / per, group = threadIdx.x / L, sub = group & (per - 1);
    const int col = (int) (blockIdx.x % SLICES) * L + (int) (threadIdx.x % L);
    for (int r0 = (int) y * rows_here; r0 < e.rows; r0 += rows_y * rows_here) {
        const int r = min(r0 + group / per, e.rows - 1);
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = sub; i < e.n; i += MERGE_LOADS * per) {
            float2 ml[MERGE_LOADS];
            float4 x[MERGE_LOADS];
            float to = m;
#pragma unroll
            for (int j = 0; j < MERGE_LOADS; ++j) {
                const int k = i + j * per;
                const size_t p = ((size_t) (e.part + min(k, e.n - 1)) * a.kvh + head) * ROWS + r;
                ml[j] = part_ml[p];
                x[j] = ((const float4*) (part_o + p * HD))[col];
                if (k >= e.n) {                          // not a part: a weight of 0 would not silence an infinity
                    ml[j].y = 0.0f;
                    x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
#pragma unroll
            for (int j = 0; j < MERGE_LOADS; ++j) to = ml[j].y != 0.0f ? fmaxf(to, ml[j].x) : to;
            const float f = l != 0.0f ? __builtin_amdgcn_exp2f(m - to) : 0.0f;
            m = to;
            l *= f;
            o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
            for (int j = 0; j < MERGE_LOADS; ++j) {
                const float h8 = ml[j].y != 0.0f ? __builtin_amdgcn_exp2f(ml[j].x - m) : 0.0f;
                l += ml[j].y * h8;
                o.x += x[j].x * h8; o.y += x[j].y * h8; o.z += x[j].z * h8; o.w += x[j].w * h8;
            }
        }
        if (per > 1) {
            s_o[threadIdx.x] = o;
            if (threadIdx.x % L == 0) s_ml[group] = make_float2(m, l);
            __syncthreads();
            if (sub == 0) {
                float to = m;
                for (int j = 1; j < per; ++j) to = s_ml[group + j].y != 0.0f ? fmaxf(to, s_ml[group + j].x) : to;
                float f = l != 0.0f ? __builtin_amdgcn_exp2f(m - to) : 0.0f;
                m = to;
                l *= f;
                o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll 4
                for (int j = 1; j < per; ++j) {
                    const float2 ml = s_ml[group + j];
                    const float4 x = s_o[threadIdx.x + j * L];
                    f = ml.y != 0.0f ? __builtin_amdgcn_exp2f(ml.x - m) : 0.0f;
                    l += ml.y * f;
                    o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
                }
            }
            __syncthreads();
        }
        if (sub == 0 && r0 + group / per < e.rows) {
            const float n = l != 0.0f ? 1.0f / l : 0.0f;
            const int row = e.row0 + r, token = (int) fast_div((uint32_t) row, a.div_g);
            if (e.q0 + token < a.max_tokens)
                *(uint2*) (a.out + (int64_t) (e.q0 + token) * a.ldo + (int64_t) (head * a.g + row - token * a.g) * a.ldo_head + 8 * col) =
                    make_uint2(pack2<T>(o.x * n, o.y * n), pack2<T>(o.z * n, o.w * n));
        }
    }
}

// narrow tiles' partial results, then wide ones'
struct Space { size_t o[2], ml[2], total; };
Space space_of(const PgLayout& l, const wzy_paged_work* w) {
    Space s;
    s.total = 0;
    for (int k = 0; k < 2; ++k) {
        const size_t rows = (size_t) l.parts[k] * (k ? PG_WIDE : l.narrow) * w->kvh;
        s.o[k] = s.total;
        s.ml[k] = s.o[k] + align_up(rows * w->hd * 4, 256);
        s.total = s.ml[k] + align_up(rows * sizeof(float2), 256);
    }
    return s;
}

template <int HD, int T>
int launch(AttnArgs a, const PgLayout& l, const Space& s, char* space, int max_rows, void* stream) {
    const auto st = as_stream(stream);
    MergeArgs g{};
    g.narrow = l.narrow;
    unsigned blocks[2] = {0, 0};
    for (int kind = 0; kind < 2; ++kind) {
        if (l.items[kind] == 0) continue;
        a.item_at = l.item_at[kind]; a.cap_parts = l.parts[kind];
        a.part_o = (float*) (space + s.o[kind]);
        a.part_ml = (float2*) (space + s.ml[kind]);
        const unsigned grid = (unsigned) l.items[kind] * (unsigned) a.kvh;
        if (kind == 0 && l.narrow == 32) paged_narrow_kernel<HD, T><<<grid, 256, 0, st>>>(a);
        else if (kind == 0) paged_middle_kernel<HD, T><<<grid, 256, 0, st>>>(a);
        else paged_wide_kernel<HD, T><<<grid, 256, 0, st>>>(a);
        WZY_LAUNCH_CHECK();
        g.rows_y[kind] = kind ? 16 : std::min(l.narrow, max_rows);
        g.at[kind] = l.merge_at[kind];
        g.parts[kind] = l.parts[kind];
        blocks[kind] = (unsigned) l.merges[kind] * (unsigned) a.kvh * (unsigned) g.rows_y[kind];
    }
    if (blocks[0] + blocks[1] == 0) return WZY_OK;
    a.part_o = (float*) (space + s.o[0]);
    a.part_ml = (float2*) (space + s.ml[0]);
    g.wide_o = (const float*) (space + s.o[1]);
    g.wide_ml = (const float2*) (space + s.ml[1]);
    const unsigned all = blocks[0] + blocks[1];
    if (HD > 64 && all * (HD / 64) <= MERGE_SHARED) {
        g.blocks = blocks[0] * (HD / 64);
        paged_merge_kernel<HD, T, 64><<<all * (HD / 64), MERGE_THREADS, 0, st>>>(a, g);
    } else {
        g.blocks = blocks[0];
        paged_merge_kernel<HD, T, HD><<<all, MERGE_THREADS, 0, st>>>(a, g);
    }
    WZY_LAUNCH_CHECK();
    return WZY_OK;
}
}  // namespace

extern "C" size_t wzy_paged_attend_workspace_bytes(const wzy_paged_batch* b, const wzy_paged_work* w) {
    const char* const who = "wzy_paged_attend_workspace_bytes";
    if (pg_check_batch(who, b, 1) != WZY_OK || pg_check_work(who, w) != WZY_OK) return 0;
    const PgLayout l = pg_layout_of(b, w);
    return pg_check_launch(who, b, w, l) == WZY_OK ? space_of(l, w).total : 0;
}

extern "C" int wzy_paged_attend(const wzy_paged_cache* c, const wzy_paged_batch* b, const wzy_paged_work* w, const wzy_heads* q,
                                const wzy_heads* out, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* const who = "wzy_paged_attend";
    WZY_TRY(pg_check_cache(who, c));
    WZY_TRY(pg_check_batch(who, b, c->page));
    WZY_TRY(pg_check_work(who, w));
    WZY_REQUIRE(w->kvh == c->kvh && w->hd == c->hd, "%s: work list of %d heads of %d, cache of %d of %d", who, w->kvh, w->hd, c->kvh, c->hd);
    WZY_REQUIRE(b->table, "%s: table is null", who);
    const PgLayout l = pg_layout_of(b, w);
    WZY_TRY(pg_check_launch(who, b, w, l));
    WZY_REQUIRE(w->items && (uintptr_t) w->items % 16 == 0 && w->bytes >= sizeof(PgHead) + sizeof(PgItem) * (size_t) l.total,
                "%s: work list of %zu bytes at %p", who, w->bytes, w->items);
    WZY_TRY(pg_check_heads(who, "q", q, c->type, w->qh, c->hd));
    WZY_TRY(pg_check_heads(who, "out", out, c->type, w->qh, c->hd));
    for (const wzy_heads* h : {q, out})
        WZY_REQUIRE((uintptr_t) h->p % 16 == 0 && h->ld % 8 == 0 && h->ld_head % 8 == 0, "%s: %s has rows without 16-byte alignment", who,
                    h == q ? "q" : "out");
    WZY_REQUIRE(q->p != out->p, "%s: out is q", who);
    WZY_REQUIRE(scale > 0.0f && scale < 1e30f, "%s: scale %g", who, (double) scale);
    const Space s = space_of(l, w);
    WZY_REQUIRE(workspace && (uintptr_t) workspace % 16 == 0 && workspace_bytes >= s.total, "%s: workspace of %zu bytes at %p (%zu, 16-byte aligned)",
                who, workspace_bytes, workspace, s.total);
    AttnArgs a{};
    a.k = (const char*) c->k; a.v = (const char*) c->v;
    a.ld_page = 2 * c->ld_page; a.ld_cell = 2 * c->ld_cell; a.ld_head = 2 * c->ld_head;
    a.table = b->table;
    a.q = (const char*) q->p; a.ldq = 2 * q->ld; a.ldq_head = 2 * q->ld_head;
    a.out = (char*) out->p; a.ldo = 2 * out->ld; a.ldo_head = 2 * out->ld_head;
    a.head = (const PgHead*) w->items;
    a.g = w->qh / w->kvh; a.kvh = w->kvh; a.window = pg_window(w); a.geometry = pg_geometry(w, l);
    a.div_g = FastDiv((uint32_t) a.g);
    a.c = scale * 1.44269504088896340736f;
    a.n_pages = c->n_pages; a.lp = pg_log2(c->page); a.max_pages = b->max_pages; a.n_req = b->n_req; a.max_tokens = b->max_tokens;
    const bool bf = c->type == WZY_BF16;
    const int max_rows = (int) std::min<int64_t>((int64_t) pg_max_new(b) * a.g, 1 << 20);
    char* const sp = (char*) workspace;
    switch (c->hd) {
        case 64: return bf ? launch<64, WZY_BF16>(a, l, s, sp, max_rows, stream) : launch<64, WZY_F16>(a, l, s, sp, max_rows, stream);
        case 128: return bf ? launch<128, WZY_BF16>(a, l, s, sp, max_rows, stream) : launch<128, WZY_F16>(a, l, s, sp, max_rows, stream);
        default: return bf ? launch<256, WZY_BF16>(a, l, s, sp, max_rows, stream) : launch<256, WZY_F16>(a, l, s, sp, max_rows, stream);
    }
}
