// rope.hip -- rotary positions: frequencies, rows of heads, and rows on their way into a paged cache.
//
//   (a, b) -> A (a cos t - b sin t, b cos t + a sin t),   t = 2 pi * frac(position * f_i / 2 pi)
//
// Angles: position * (f / 2 pi) in 64 bits, less the nearest multiple of a quarter turn; what is left, at most pi / 4 either
// way, goes into the Taylor polynomials of sine and cosine in 64 bits (to x^13 and x^14: 2e-14).  They are made once a row, by
// one thread an angle, and kept in LDS for all heads of the row: at far positions fp32 angles would be off by whole turns.
// The rows are read and written once, 8 elements (and their partners) a thread where alignment allows 16-byte accesses, a pair
// a thread elsewhere.  Bound by memory at large sizes, by the launch at one row: a row of 24 + 2 + 2 heads of 256 from fp32 2.7 us,
// 8,192 of them in bf16 42 us where part of them is still in a cache and 64 where none is (235 MB; a copy of as much: 45), 4,097 rows
// of 32 heads of 128 in fp16 12.3 us (67 MB, 5.5 TB/s).  A pair a thread: the same rows in bf16 with 120 of their elements turned 36 to
// 38 us (1.8 TB/s), with 22 of them 50 to 53; 8,192 rows of 28 heads of 256, 60 turned, 140.
#include <algorithm>

#include "wzy_paged.h"

using namespace wzy;

typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef uint32_t v4w_t __attribute__((ext_vector_type(4)));

namespace {
constexpr int RT = 256, ROPE_MAX = 512, MOST_BLOCKS = 1 << 23;

struct View { const void* p; int64_t ld, ldh; };
struct RopeArgs {
    // three sets of heads: q (or the only one), k, v; the last two go to the cache's slots
    View in[3], out[3];
    int heads[3];                         // 0: absent
    const double* freqs;                  // null: nothing is turned
    const int* positions;
    const int* slots;
    int rows, hd, n_rot, n_sets;
    int per_row, per_head;                // pieces of work: of all heads of a row, of a head
    FastDiv div_row, div_head;
    int64_t ld_page, n_cells;
    int lp, rows_block, first;            // first: row of the launch's first workgroup
    bool stream;                          // stores past the caches
};

// cos and sin of 2 pi x, amplitude in
WZY_DEV float2 turn(double x, double amplitude) {
    x -= floor(x);                                             // 0 .. 1
    const int near = (int) (x * 4.0 + 0.5);                    // quarter turns, the nearest
    const double y = (x - (double) near * 0.25) * 6.283185307179586476925, z = y * y;
    double c = -1.0 / 87178291200.0, s = 1.0 / 6227020800.0;
    c = fma(c, z, 1.0 / 479001600.0); s = fma(s, z, -1.0 / 39916800.0);
    c = fma(c, z, -1.0 / 3628800.0);  s = fma(s, z, 1.0 / 362880.0);
    c = fma(c, z, 1.0 / 40320.0);     s = fma(s, z, -1.0 / 5040.0);
    c = fma(c, z, -1.0 / 720.0);      s = fma(s, z, 1.0 / 120.0);
    c = fma(c, z, 1.0 / 24.0);        s = fma(s, z, -1.0 / 6.0);
    c = fma(c, z, -0.5);              s = fma(s, z, 1.0) * y;
    c = fma(c, z, 1.0);
    const int q = near & 3;
    const double cc = q & 1 ? s : c, ss = q & 1 ? c : s;
    return make_float2((float) (amplitude * (q == 1 || q == 2 ? -cc : cc)), (float) (amplitude * (q >= 2 ? -ss : ss)));
}

template <int T>
WZY_DEV float load1(const void* p, size_t i) {
    if constexpr (T == WZY_F32) return ((const float*) p)[i];
    else if constexpr (T == WZY_BF16) return bf16_to_f(((const uint16_t*) p)[i]);
    else return h16_to_f(((const uint16_t*) p)[i]);
}
template <int T>
WZY_DEV void store1(void* p, size_t i, float v) {
    if constexpr (T == WZY_F32) ((float*) p)[i] = v;
    else if constexpr (T == WZY_BF16) ((uint16_t*) p)[i] = (uint16_t) pack2<WZY_BF16>(v, v);
    else ((uint16_t*) p)[i] = f_to_h16(v);
}

// 8 elements; stream: past the caches, which hold less than the call writes (8,192 rows of 24 + 2 + 2 heads of 256 in bf16, buffers
// changing from call to call: 68 -> 65 us, 4,097 of 32 of 128 17.4 -> 12.8; the loads likewise: no faster, and 20 us slower where the
// rows are still in a cache)
template <int T>
WZY_DEV void store_wide(void* p, size_t i, const float (&v)[8], bool stream) {
    if (!stream) {
        store8<T>(p, i, v);
        return;
    }
    if constexpr (T == WZY_F32) {
        __builtin_nontemporal_store(v4f_t{v[0], v[1], v[2], v[3]}, (v4f_t*) ((float*) p + i));
        __builtin_nontemporal_store(v4f_t{v[4], v[5], v[6], v[7]}, (v4f_t*) ((float*) p + i) + 1);
    } else
        __builtin_nontemporal_store(v4w_t{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])},
                                    (v4w_t*) ((uint16_t*) p + i));
}

// A piece of a row: WIDE, 8 elements and, in rotated halves, the 8 they pair with; else a pair or one element.
template <int TI, int TO, bool PAIRS, bool WIDE>
struct Piece {
    static constexpr int N = WIDE ? 8 : 1;
    float u[N], v[N];
    int row, set, e0, e1, turned;              // first element; its partner's (-1: none); its pair (-1: not turned)
    int h;
    WZY_DEV void locate(const RopeArgs& a, int row0, int i) {
        const int half = a.n_rot >> 1, r = (int) fast_div((uint32_t) i, a.div_row), x = i - r * a.per_row;
        h = (int) fast_div((uint32_t) x, a.div_head);
        const int piece = x - h * a.per_head;
        row = row0 + r;
        set = 0;
        if (a.n_sets > 1) {
            if (h >= a.heads[0]) { h -= a.heads[0]; set = 1; }
            if (set == 1 && h >= a.heads[1]) { h -= a.heads[1]; set = 2; }
        }
        const bool turn = set < 2 && a.freqs;                  // values are not turned
        e1 = -1;
        if constexpr (WIDE && PAIRS) {
            e0 = 8 * piece;
            turned = turn && e0 < a.n_rot ? 4 * piece : -1;
        } else if (piece * N < half) {
            e0 = WIDE ? 8 * piece : PAIRS ? 2 * piece : piece;
            e1 = PAIRS ? e0 + 1 : e0 + half;
            turned = turn ? N * piece : -1;
        } else {                                               // behind the pairs
            e0 = a.n_rot + N * piece - half;
            turned = -1;
        }
    }
    WZY_DEV void load(const RopeArgs& a) {
        const View& in = set == 0 ? a.in[0] : set == 1 ? a.in[1] : a.in[2];
        const size_t at = (size_t) row * in.ld + (size_t) h * in.ldh;
        if constexpr (WIDE) {
            load8<TI>(in.p, at + e0, u);
            if (!PAIRS && e1 >= 0) load8<TI>(in.p, at + e1, v);
        } else {
            u[0] = load1<TI>(in.p, at + e0);
            if (e1 >= 0) v[0] = load1<TI>(in.p, at + e1);
        }
    }
    static WZY_DEV void turn(float& x, float& y, float2 t) {
        const float p = x * t.x - y * t.y;
        y = y * t.x + x * t.y;
        x = p;
    }
    WZY_DEV void store(const RopeArgs& a, const float2* cs) {
        if (turned >= 0) {
            if constexpr (WIDE && PAIRS) {
#pragma unroll
                for (int j = 0; j < 4; ++j) turn(u[2 * j], u[2 * j + 1], cs[turned + j]);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) turn(u[j], v[j], cs[turned + j]);
            }
        }
        void* const dst = (void*) (set == 0 ? a.out[0].p : set == 1 ? a.out[1].p : a.out[2].p);
        size_t to;
        if (set == 0) to = (size_t) row * a.out[0].ld + (size_t) h * a.out[0].ldh;
        else {
            const int slot = a.slots[row];
            if (slot < 0 || slot >= a.n_cells) return;
            to = (size_t) (slot >> a.lp) * a.ld_page + (size_t) (slot & ((1 << a.lp) - 1)) * a.out[1].ld + (size_t) h * a.out[1].ldh;
        }
        if constexpr (WIDE) {
            store_wide<TO>(dst, to + e0, u, a.stream);
            if (!PAIRS && e1 >= 0) store_wide<TO>(dst, to + e1, v, a.stream);
        } else {
            store1<TO>(dst, to + e0, u[0]);
            if (e1 >= 0) store1<TO>(dst, to + e1, v[0]);
        }
    }
};

// One workgroup does rows_block rows, or blockIdx.y's share of one: a thread's first piece is on its way while the angles are made.
template <int TI, int TO, bool PAIRS, bool WIDE>
__global__ void __launch_bounds__(RT) rope_kernel(RopeArgs a) {
    __shared__ float2 s_cs[ROPE_MAX];
    const int tid = threadIdx.x, row0 = a.first + (int) blockIdx.x * a.rows_block, rows = min(a.rows - row0, a.rows_block);
    const int half = a.n_rot >> 1, pieces = rows * a.per_row, step = RT * (int) gridDim.y;
    Piece<TI, TO, PAIRS, WIDE> p;
    int i = (int) blockIdx.y * RT + tid;
    const bool any = i < pieces;
    if (any) {
        p.locate(a, row0, i);
        p.load(a);
    }
    if (a.freqs) {
        for (int k = tid; k < rows * half; k += RT) {
            const int r = k / half, j = k - r * half;
            s_cs[k] = turn((double) a.positions[row0 + r] * a.freqs[j], a.freqs[half]);
        }
        __syncthreads();
    }
    if (!any) return;
    for (i += step; i < pieces; i += step) {                   // the next piece loads before this one is stored
        Piece<TI, TO, PAIRS, WIDE> next;
        next.locate(a, row0, i);
        next.load(a);
        p.store(a, s_cs + (p.row - row0) * half);
        p = next;
    }
    p.store(a, s_cs + (p.row - row0) * half);
}

__global__ void rope_freqs_kernel(wzy_rope_cfg c, double* __restrict__ f) {
    const int i = threadIdx.x, half = c.n_rot / 2;
    const double two_pi = 6.283185307179586476925, ln = log(c.theta);
    if (i < half) {
        const double base = exp(-2.0 * (double) i / (double) c.n_rot * ln);
        double keep = 1.0;
        if (c.scaling == WZY_ROPE_LINEAR) keep = 0.0;
        if (c.scaling == WZY_ROPE_ROTATIONS) keep = ((double) c.ctx * base / two_pi - c.low) / (c.high - c.low);
        if (c.scaling == WZY_ROPE_INDEX) {
            const double at_high = (double) c.n_rot * log((double) c.ctx / (two_pi * c.high)) / (2.0 * ln);
            const double at_low = (double) c.n_rot * log((double) c.ctx / (two_pi * c.low)) / (2.0 * ln);
            const double a = fmax(floor(at_high), 0.0), b = fmin(ceil(at_low), (double) c.n_rot - 1.0);
            // both ends on one pair: it and those below keep their frequency
            keep = b > a ? 1.0 - ((double) i - a) / (b - a) : (double) i <= a ? 1.0 : 0.0;
        }
        keep = fmin(fmax(keep, 0.0), 1.0);
        f[i] = base * (keep + (1.0 - keep) / c.factor) / two_pi;
    }
    if (i == half) f[half] = c.amplitude == 0.0 ? 1.0 : c.amplitude;
}

int check_tab(const char* who, const wzy_rope_tab* t, int hd) {
    WZY_REQUIRE(t && t->freqs && (uintptr_t) t->freqs % 8 == 0, "%s: the rotary table is null", who);
    WZY_REQUIRE(t->n_rot >= 2 && t->n_rot % 2 == 0 && t->n_rot <= hd, "%s: n_rot %d of heads of %d", who, t->n_rot, hd);
    WZY_REQUIRE(t->layout == WZY_ROPE_HALVES || t->layout == WZY_ROPE_PAIRS, "%s: layout %d", who, t->layout);
    return WZY_OK;
}
bool rows16(const void* p, int64_t ld, int64_t ldh, int type) {
    const int n = mx_type_bytes(type);
    return (uintptr_t) p % 16 == 0 && ld * n % 16 == 0 && ldh * n % 16 == 0;
}

// Rows a workgroup takes: enough pieces for its 256 threads, while there are rows for all CUs, as far as the angles' room goes.
template <int TI, int TO>
int launch(RopeArgs a, bool pairs, bool wide, void* stream) {
    const int heads = a.heads[0] + a.heads[1] + a.heads[2], half = a.n_rot / 2;
    a.per_head = !wide ? half + a.hd - a.n_rot : pairs ? a.hd / 8 : half / 8 + (a.hd - a.n_rot) / 8;
    a.per_row = heads * a.per_head;
    a.div_row = FastDiv((uint32_t) a.per_row);
    a.div_head = FastDiv((uint32_t) a.per_head);
    int rb = 1;
    while (rb * a.per_row < 2 * RT && 2 * rb * half <= ROPE_MAX && a.rows / (2 * rb) >= 512) rb *= 2;
    a.rows_block = rb;
    a.stream = (int64_t) a.rows * heads * a.hd * mx_type_bytes(TO) > 32 << 20;
    // few rows: a row's pieces to several workgroups, each with angles of its own
    const int blocks = pg_div_up(a.rows, rb), share = blocks >= 512 ? 1 : std::min((a.per_row * rb + RT - 1) / RT, 512 / blocks);
    const auto st = as_stream(stream);
    for (int64_t at = 0; at < blocks; at += MOST_BLOCKS) {     // a launch has fewer than 2^32 threads
        const dim3 grid((unsigned) std::min<int64_t>(blocks - at, MOST_BLOCKS), (unsigned) share);
        a.first = (int) (at * rb);
        if (pairs && wide) rope_kernel<TI, TO, true, true><<<grid, RT, 0, st>>>(a);
        else if (pairs) rope_kernel<TI, TO, true, false><<<grid, RT, 0, st>>>(a);
        else if (wide) rope_kernel<TI, TO, false, true><<<grid, RT, 0, st>>>(a);
        else rope_kernel<TI, TO, false, false><<<grid, RT, 0, st>>>(a);
        WZY_LAUNCH_CHECK();
    }
    return WZY_OK;
}
}  // namespace

extern "C" int wzy_rope_freqs(const wzy_rope_cfg* c, double* freqs, void* stream) {
    const char* const who = "wzy_rope_freqs";
    WZY_REQUIRE(c && freqs && (uintptr_t) freqs % 8 == 0, "%s: null", who);
    WZY_REQUIRE(c->n_rot >= 2 && c->n_rot <= ROPE_MAX && c->n_rot % 2 == 0, "%s: n_rot %d (even, 2 .. %d)", who, c->n_rot, ROPE_MAX);
    WZY_REQUIRE(c->theta > 1.0 && c->theta <= 1e300, "%s: theta %g (above 1)", who, c->theta);
    WZY_REQUIRE(c->scaling >= WZY_ROPE_PLAIN && c->scaling <= WZY_ROPE_INDEX, "%s: scaling %d", who, c->scaling);
    WZY_REQUIRE(c->amplitude > -1e30 && c->amplitude < 1e30, "%s: amplitude %g", who, c->amplitude);
    if (c->scaling != WZY_ROPE_PLAIN) WZY_REQUIRE(c->factor >= 1.0 && c->factor <= 1e300, "%s: factor %g (at least 1)", who, c->factor);
    if (c->scaling >= WZY_ROPE_ROTATIONS)
        WZY_REQUIRE(c->low > 0.0 && c->high > c->low && c->high <= 1e300 && c->ctx >= 1, "%s: low %g, high %g, ctx %d", who, c->low, c->high, c->ctx);
    rope_freqs_kernel<<<1, ROPE_MAX / 2 + 64, 0, as_stream(stream)>>>(*c, freqs);
    WZY_LAUNCH_CHECK();
    return WZY_OK;
}

extern "C" int wzy_rope(const wzy_rope_tab* t, const wzy_heads* x, int type, int rows, int heads, int hd, const int* positions,
                        const wzy_heads* out, void* stream) {
    const char* const who = "wzy_rope";
    WZY_TRY(mx_check_type(who, type));
    WZY_REQUIRE(rows >= 0 && heads >= 1 && heads <= 1024 && hd >= 2 && hd <= ROPE_MAX, "%s: %d rows of %d heads of %d", who, rows, heads, hd);
    WZY_TRY(check_tab(who, t, hd));
    if (rows == 0) return WZY_OK;
    WZY_TRY(pg_check_heads(who, "x", x, type, heads, hd));
    WZY_TRY(pg_check_heads(who, "out", out, type, heads, hd));
    WZY_REQUIRE(positions, "%s: positions is null", who);
    WZY_REQUIRE(x->p != out->p || (x->ld == out->ld && x->ld_head == out->ld_head), "%s: in place with other strides", who);
    RopeArgs a{};
    a.in[0] = View{x->p, x->ld, x->ld_head};
    a.out[0] = View{out->p, out->ld, out->ld_head};
    a.heads[0] = heads;
    a.n_sets = 1;
    a.freqs = t->freqs; a.positions = positions; a.rows = rows; a.hd = hd; a.n_rot = t->n_rot;
    const bool wide = hd % 8 == 0 && t->n_rot % 16 == 0 && rows16(x->p, x->ld, x->ld_head, type) && rows16(out->p, out->ld, out->ld_head, type);
    return mx_with_type(type, [&](auto ti) { return launch<ti(), ti()>(a, t->layout == WZY_ROPE_PAIRS, wide, stream); });
}

extern "C" int wzy_paged_append(const wzy_paged_cache* c, const wzy_rope_tab* t, const wzy_heads* q, int qh, const wzy_heads* q_out,
                                const wzy_heads* k, const wzy_heads* v, int type, int rows, const int* positions, const int* slots,
                                void* stream) {
    const char* const who = "wzy_paged_append";
    WZY_TRY(mx_check_type(who, type));
    WZY_TRY(pg_check_cache(who, c));
    WZY_REQUIRE(rows >= 0 && qh >= 0 && qh <= 1024, "%s: %d rows, %d query heads", who, rows, qh);
    WZY_REQUIRE((qh == 0) == (q == nullptr) && (qh == 0) == (q_out == nullptr), "%s: %d query heads with q %p, q_out %p", who, qh,
                (const void*) q, (const void*) q_out);
    if (t) WZY_TRY(check_tab(who, t, c->hd));
    if (rows == 0) return WZY_OK;
    WZY_REQUIRE(slots && (positions || !t), "%s: positions or slots are null", who);
    WZY_TRY(pg_check_heads(who, "k", k, type, c->kvh, c->hd));
    WZY_TRY(pg_check_heads(who, "v", v, type, c->kvh, c->hd));
    RopeArgs a{};
    if (q) {
        WZY_TRY(pg_check_heads(who, "q", q, type, qh, c->hd));
        WZY_TRY(pg_check_heads(who, "q_out", q_out, c->type, qh, c->hd));
        WZY_REQUIRE(q->p != q_out->p || (type == c->type && q->ld == q_out->ld && q->ld_head == q_out->ld_head), "%s: q in place with other rows", who);
        a.in[0] = View{q->p, q->ld, q->ld_head};
        a.out[0] = View{q_out->p, q_out->ld, q_out->ld_head};
    }
    a.in[1] = View{k->p, k->ld, k->ld_head};
    a.in[2] = View{v->p, v->ld, v->ld_head};
    a.out[1] = View{c->k, c->ld_cell, c->ld_head};
    a.out[2] = View{c->v, c->ld_cell, c->ld_head};
    a.heads[0] = qh; a.heads[1] = a.heads[2] = c->kvh;
    a.n_sets = 3;
    a.freqs = t ? t->freqs : nullptr;
    a.positions = positions; a.slots = slots; a.rows = rows; a.hd = c->hd; a.n_rot = t ? t->n_rot : 0;
    a.ld_page = c->ld_page; a.n_cells = (int64_t) c->n_pages * c->page; a.lp = pg_log2(c->page);
    const bool wide = a.n_rot % 16 == 0 && rows16(k->p, k->ld, k->ld_head, type) && rows16(v->p, v->ld, v->ld_head, type) &&
                      (!q || (rows16(q->p, q->ld, q->ld_head, type) && rows16(q_out->p, q_out->ld, q_out->ld_head, c->type)));
    const bool pairs = t && t->layout == WZY_ROPE_PAIRS;
    return mx_with_type(type, [&](auto ti) {
        return c->type == WZY_BF16 ? launch<ti(), WZY_BF16>(a, pairs, wide, stream) : launch<ti(), WZY_F16>(a, pairs, wide, stream);
    });
}
