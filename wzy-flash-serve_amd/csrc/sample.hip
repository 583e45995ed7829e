// sample.hip -- one token a row of logits, by temperature, top-k, min-p and top-p, from given uniform numbers.
//
// The order of a row is (logit descending, id ascending).  Every cut keeps a prefix of it, and the draw takes the first
// token whose running sum of w = 2^-x, x = (max - l) log2(e) / temp, reaches a target; so all that is needed are places in
// that order: by count (top-k), by sum (top-p, the draw), by value (min-p).  No sort of the row: a histogram over x in bins of
// 1/16 (count and sum of w) says in which few bins the places lie, and only those bins' tokens are gathered and sorted.
//   sample_max     a slice of a row a workgroup: its best token
//   sample_hist    the same slices: x against the row's best, histogram in LDS, added to the row's
//   sample_plan    a workgroup a row: which bins are wanted.  (The row's last workgroup of sample_hist, told by a counter, could do it:
//                  the fences between their atomics and its loads took 200 us at 256 rows.)  Rows with a small top-k need no
//                  histogram: sample_max left the largest token of every 32, whose k-th largest bounds the row's, and the few
//                  groups above it are all that has to be read again; they get their token here
//   sample_gather  the slices again: tokens of those bins to the row's list
//   sample_pick    a workgroup a row: the list sorted, sums, places
// Rows of at most SHORT logits are sorted whole, by one launch.  Rows whose bins hold more than CAP tokens are done by sample_pick alone,
// from the row: thousands of equal logits, and flat rows too (a bin of 1/16 octave has about 1,000 x temp tokens of 151,936 normal
// logits of deviation 2.5).  With top-p 0.95, 4 of those rows take 30 us at temp 1 and 183 at temp 2, 256 of them 110 and 267; of
// deviation 0.5 at temp 1, 290 and 418.
// Few rows: 1 of 151,936 with top-k 40 19 us, top-k 500 29, top-p 27, no filter 25; 8 of them 21, 33, 32, 30 (bf16 within 3 us).
// 256 rows of 151,936 fp32 logits with top-p: 25 + 42 + 8 + 28 + 10 us; the first and fourth are bound by memory (6 TB/s), the second
// by its 64-bit operations and LDS atomics.  4 rows with top-k: 4 + 2 + 10 + 1 + 1, bound by latencies.
// w is taken in 64 bits (fp32's 1e-7 would move one draw in a thousand of a flat row) and summed as integers of 2^-F, F = 62 -
// log2(vocab), at most 51: sums do not depend on their order, so LDS and memory atomics may add them as they come.  Where top-k is
// small, everything it leaves is gathered, and the histogram counts only.
#include <algorithm>
#include <type_traits>

#include "wzy_paged.h"

using namespace wzy;

namespace {
constexpr int ST = 256, PER = 32, SLICE = ST * PER;      // sample_max, sample_hist
constexpr int PT = 1024, CAP = 4096;                     // sample_pick; tokens gathered at most
constexpr int SHORT = 2048;                              // rows of up to so many logits are sorted whole
constexpr int GROUP_K = CAP / PER;                       // top-k up to which the groups' largest tokens say what to gather
constexpr int SMALL_K = 2048;                            // top-k up to which all that it leaves is gathered
constexpr int BINS = 1024;                               // 64 octaves of w
constexpr float BIN_OCT = 16.0f;                         // bins an octave; a bin's tokens are within 1/32 of a bin of its ends
constexpr float BIN_SLACK = 1.0f / 32;
constexpr float GREEDY = 1e-5f;
constexpr uint32_t KEY_NONE = 0x007FFFFFu;               // order key of -infinity

// a row's parameters, made harmless
struct Params {
    float temp, top_p, min_p;
    double u;
    int k;
    bool first;                                          // the best token, whatever u
    WZY_DEV bool cut_p() const { return top_p > 0.0f && top_p < 1.0f; }
    WZY_DEV bool cut_m() const { return min_p > 0.0f; }
    WZY_DEV bool counts_only() const { return k >= 1 && k <= SMALL_K; }
    WZY_DEV bool counts() const { return k >= 1; }
    WZY_DEV bool from_groups() const { return k >= 1 && k <= GROUP_K; }
};

// What sample_plan leaves to the next kernels.
enum { ROW_DONE, ROW_LIST, ROW_ALONE };
struct RowPlan {
    int mode;                                            // the row has its token; a list; neither
    int n, lo[4], hi[4];                                 // intervals of bins that are gathered, in order
    float most[4], least[4];                             // the logits at their ends
    uint64_t before_mass[4], list_mass[4];               // sums before each, of the row and of the list
    uint32_t before_count[4], count;                     // tokens before each; of the row (where top-k wants them)
    uint64_t mass;                                       // of the row
    int m0, m1;                                          // bins in which min-p ends; -1: it does not matter
    uint64_t m_mass;                                     // sum before bin m0
    uint64_t best;                                       // the row's best token
    Params q;
};

struct SampleArgs {
    const void* logits;
    int64_t ld;
    int rows, vocab, slices, units, F;                   // slices of `units` x SLICE logits
    const float* temp;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int* ids;
    float* probs;
    uint64_t* best;                                      // [rows x slices]
    uint64_t* mass;                                      // [rows x BINS]
    uint32_t* count;                                     // [rows x BINS]
    RowPlan* plan;                                       // [rows]
    uint32_t* listed;                                    // [rows] tokens in the list
    uint64_t* list;                                      // [rows x CAP]
    uint32_t* group;                                     // [rows x groups] each thread's largest key of a unit (null: no row wants them)
    int groups;
};

// a logit's bits in numeric order (both zeros alike); a NaN as -infinity
WZY_DEV uint32_t order_key(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v != v ? -INFINITY : v + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
WZY_DEV float key_value(uint32_t k) {
    return __builtin_bit_cast(float, (k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}
WZY_DEV uint64_t order_u64(float v, int i) { return (uint64_t) order_key(v) << 32 | (uint32_t) ~i; }

// 2^(-j / STEPS)
constexpr int LSTEPS = 8, STEPS = 1 << LSTEPS, BIN_STEPS_LOG2 = LSTEPS - 4;
WZY_DEV void fill_table(double* s) {
    for (int i = threadIdx.x; i < STEPS; i += blockDim.x) s[i] = exp2(-(double) i / STEPS);
}
// A row's weights: m its largest logit, c = log2(e) / temp.  A token's 256 x, rounded, gives its bin and its weight.
struct Weight {
    static constexpr double MAGIC = 6755399441055744.0;  // 1.5 2^52: adding it rounds to an integer and leaves it in the low bits
    float m, cf;
    double cs;                                           // STEPS log2(e) / temp
    int F;
    const double* table;
    // 256 x, at most 1,000 octaves, and that for what is not a number.  ANY: m may be infinite
    template <bool ANY = true>
    WZY_DEV double steps(float l) const {
        const double t = ((double) m - (double) l) * cs;
        return fmin(ANY && l == m ? 0.0 : t, 1000.0 * STEPS);
    }
    static WZY_DEV int rounded(double n) { return (int) (uint32_t) __builtin_bit_cast(uint64_t, n); }
    static WZY_DEV int bin_at(double t) { return min(rounded(t + MAGIC) >> BIN_STEPS_LOG2, BINS - 1); }
    WZY_DEV int bin(float l) const { return bin_at(steps(l)); }
    // 2^-x as an integer of 2^-F: 256 x = k + r, |r| <= 1/2; 2^(-r / 256) by its series, whose fourth term is 2e-13 at most; 2^-(k / 256)
    // from the table and the exponent field.
    WZY_DEV uint64_t fixed_at(double t) const {
        return __builtin_bit_cast(uint64_t, scaled_at(t, F) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    }
    WZY_DEV uint64_t fixed(float l) const { return fixed_at(steps(l)); }
    WZY_DEV double w(float l) const { return scaled(l, 0); }
    WZY_DEV double scaled(float l, int f) const { return scaled_at(steps(l), f); }
    WZY_DEV double scaled_at(double t, int f) const {
        constexpr double A = -0.6931471805599453094 / STEPS;
        const double n = t + MAGIC, r = t - (n - MAGIC);
        const int i = rounded(n);
        double p = __builtin_fma(r, A * A * A / 6.0, A * A / 2.0);
        p = __builtin_fma(p, r, A);
        const uint64_t b = __builtin_bit_cast(uint64_t, table[i & (STEPS - 1)]) + ((uint64_t) (uint32_t) ((f - (i >> LSTEPS)) << 20) << 32);
        const double base = __builtin_bit_cast(double, b);                   // 2^-1000 at least: no denormal
        return __builtin_fma(base * r, p, base);
    }
};
WZY_DEV Params params_of(const SampleArgs& a, int row) {
    Params p;
    const float v = a.u[row];
    p.temp = a.temp ? a.temp[row] : 1.0f;
    p.k = a.top_k ? a.top_k[row] : 0;
    p.top_p = a.top_p ? a.top_p[row] : 1.0f;
    p.min_p = a.min_p ? a.min_p[row] : 0.0f;
    p.u = v > 0.0f ? fmin((double) v, 1.0) : 0.0;
    p.first = !(p.temp > GREEDY) || p.min_p > 1.0f || p.k == 1;
    return p;
}

// N elements a thread of the row's from .. (16 bytes at a time where the row allows), -infinity past end; which they are
template <int T, bool VEC>
WZY_DEV int element(int from, int j) {
    constexpr int E = !VEC ? 1 : T == WZY_F32 ? 4 : 8;
    return from + ((j / E) * (int) blockDim.x + (int) threadIdx.x) * E + j % E;
}
template <int T>
WZY_DEV float load_logit(const void* row, int i) {
    if constexpr (T == WZY_F32) return ((const float*) row)[i];
    else if constexpr (T == WZY_BF16) return bf16_to_f(((const uint16_t*) row)[i]);
    else return h16_to_f(((const uint16_t*) row)[i]);
}
template <int T, bool VEC, int N>
WZY_DEV void load_elements(const void* row, int from, int end, float (&x)[N]) {
    if constexpr (VEC) {
        constexpr int E = T == WZY_F32 ? 4 : 8;
        uint4 v[N / E];
#pragma unroll
        for (int i = 0; i < N / E; ++i) {
            const int e = element<T, true>(from, i * E);
            if (e + E <= end) v[i] = *(const uint4*) ((const char*) row + (size_t) e * (16 / E));
            else v[i] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < N / E; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < E; ++j) {
                if constexpr (T == WZY_F32) x[i * E + j] = __builtin_bit_cast(float, w[j]);
                else if constexpr (T == WZY_BF16) x[i * E + j] = j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]);
                else x[i * E + j] = h16_to_f((uint16_t) (w[j / 2] >> (16 * (j & 1))));
            }
        }
        if (from + N * (int) blockDim.x > end) {                // the row's end
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int e = element<T, true>(from, j);
                if (e - j % E + E > end) x[j] = e < end ? load_logit<T>(row, e) : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = load_logit<T>(row, min(element<T, false>(from, j), end - 1));
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = element<T, false>(from, j) < end ? x[j] : -INFINITY;
    }
}
template <int T>
WZY_DEV const void* row_of(const SampleArgs& a, int row) {
    return (const char*) a.logits + (size_t) row * a.ld * (T == WZY_F32 ? 4 : 2);
}

// f(values, first) over the slice's elements, PER a thread at a time.  (With the next ones' loads ahead, in twice the registers and
// two thirds of the waves, the histogram of 256 rows took 55 us instead of 50.)
template <int T, bool VEC, class F>
WZY_DEV void each_unit(const SampleArgs& a, int row, int slice, F&& f) {
    const void* const r = row_of<T>(a, row);
    for (int u = 0; u < a.units; ++u) {
        const int from = (slice * a.units + u) * SLICE;
        if (from >= a.vocab) break;
        float x[PER];
        load_elements<T, VEC>(r, from, min(from + SLICE, a.vocab), x);
        f(x, from);
    }
}

template <int T, bool VEC>
__global__ void __launch_bounds__(ST) sample_max_kernel(SampleArgs a) {
    __shared__ uint64_t s_best[ST / 64];
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    // the row's histogram starts empty
    for (int i = slice * ST + tid; i < BINS; i += a.slices * ST) {
        a.mass[(size_t) row * BINS + i] = 0;
        a.count[(size_t) row * BINS + i] = 0;
    }
    if (slice == 0 && tid == 0) a.listed[row] = 0;
    uint64_t b = 0;
    each_unit<T, VEC>(a, row, slice, [&](const float (&x)[PER], int from) {
        uint64_t g = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) g = max_u64(g, order_u64(x[j], element<T, VEC>(from, j)));
        if (a.group) a.group[(size_t) row * a.groups + from / PER + tid] = (uint32_t) (g >> 32);
        b = max_u64(b, g);
    });
    b = wave_max_u64(b);
    if ((tid & 63) == 0) s_best[tid >> 6] = b;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int i = 1; i < ST / 64; ++i) b = max_u64(b, s_best[i]);
        a.best[(size_t) row * a.slices + slice] = b;
    }
}

// the row's best token, to every thread
template <int NT>
WZY_DEV uint64_t row_best(const SampleArgs& a, int row, uint64_t* s) {
    uint64_t b = 0;
    for (int i = threadIdx.x; i < a.slices; i += NT) b = max_u64(b, a.best[(size_t) row * a.slices + i]);
    b = wave_max_u64(b);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = b;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) b = max_u64(b, s[i]);
    __syncthreads();
    return b;
}
WZY_DEV Weight weight_of(const SampleArgs& a, uint64_t best, float t, const double* table) {
    Weight w;
    w.m = key_value((uint32_t) (best >> 32));
    const double c = 1.44269504088896340736 / (double) t;
    w.cs = c * STEPS;
    w.cf = (float) c;
    w.F = a.F;
    w.table = table;
    return w;
}

// inclusive sums of (mass, count) over the workgroup's threads
struct Sum { uint64_t mass; uint32_t count; };
template <int CTRL, int ROWMASK>
WZY_DEV void add_lanes(Sum& v) {
    const uint32_t lo = dpp_u32<CTRL, ROWMASK>((uint32_t) v.mass), hi = dpp_u32<CTRL, ROWMASK>((uint32_t) (v.mass >> 32));
    v.mass += (uint64_t) hi << 32 | lo;
    v.count += dpp_u32<CTRL, ROWMASK>(v.count);
}
WZY_DEV void add_before(Sum& v) {                          // sums of lanes 0 .. l
    add_lanes<0x111, 0xF>(v);                            // row_shr 1, 2, 4, 8, then the rows' last lanes on to the next rows
    add_lanes<0x112, 0xF>(v);
    add_lanes<0x114, 0xF>(v);
    add_lanes<0x118, 0xF>(v);
    add_lanes<DPP_ROW_BCAST15, 0xA>(v);
    add_lanes<DPP_ROW_BCAST31, 0xC>(v);
}
WZY_DEV Sum block_sums(Sum v, Sum* s_part) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = (int) blockDim.x >> 6;
    add_before(v);
    if (lane == 63) s_part[w] = v;
    __syncthreads();
    Sum b = lane < nw ? s_part[lane] : Sum{0, 0};
    add_before(b);
    if (w > 0) {
        const uint32_t lo = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) b.mass, w - 1);
        const uint32_t hi = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (b.mass >> 32), w - 1);
        v.mass += (uint64_t) hi << 32 | lo;
        v.count += (uint32_t) __builtin_amdgcn_readlane((int) b.count, w - 1);
    }
    __syncthreads();
    return v;
}
// the first integer at or above f * sum, 1 .. sum
WZY_DEV uint64_t share(double f, uint64_t sum) {
    const double x = ceil(f * (double) sum);
    const uint64_t v = x >= (double) sum ? sum : (uint64_t) x;
    return v < 1 ? (uint64_t) 1 : v;
}
// The first bin whose inclusive sum reaches t (the last bin, if none does): a wave's lanes look at 64 of them, then at the 16 between.
template <class S>
WZY_DEV int find_bin(const S* sum, S t) {
    static_assert(BINS == 1024, "64 x 16");
    const int lane = threadIdx.x & 63;
    const uint64_t far = __ballot(sum[16 * lane + 15] >= t);
    const int at = far ? 16 * (__ffsll((unsigned long long) far) - 1) : BINS - 16;
    const uint64_t near = __ballot(sum[at + (lane & 15)] >= t) & 0xFFFF;
    return near ? at + __ffsll((unsigned long long) near) - 1 : BINS - 1;
}

// The bins that the places may lie in.  A place that hangs on one inside a bin is bracketed by the bin's ends.  One wave, all lanes
// the same.  mass, count: inclusive sums (count where top-k wants it).
WZY_DEV void plan_row(const Params& q, const uint64_t* mass, const uint32_t* count, RowPlan& out) {
    auto before = [&](int b) { return b > 0 ? mass[b - 1] : 0; };
    // intervals of top-k, top-p, min-p, the draw
    int lo[4] = {BINS, BINS, BINS, BINS}, hi[4] = {-1, -1, -1, -1};
    const uint32_t all = count[BINS - 1];
    const bool cut_k = q.k >= 1 && (uint32_t) q.k < all;
    int kb = BINS - 1, m0 = -1, m1 = -1;
    if (q.counts()) kb = find_bin(count, cut_k ? (uint32_t) q.k : all);
    if (q.counts_only()) {
        lo[0] = 0;
        hi[0] = kb;
    } else {
        // what is left lies between these sums
        uint64_t least = mass[BINS - 1], most = least;
        int last = BINS - 1;
        if (cut_k) {
            least = before(kb);
            most = mass[kb];
            lo[0] = hi[0] = last = kb;
        }
        auto within = [&](int b0, int b1) {              // the next place lies in bins b0 .. b1
            const uint64_t x = before(b0), y = mass[b1];
            least = x < least ? x : least;
            most = y < most ? y : most;
        };
        if (q.cut_p()) {
            lo[1] = find_bin(mass, share((double) q.top_p, least));
            hi[1] = find_bin(mass, share((double) q.top_p, most));
            last = min(last, hi[1]);
            within(lo[1], hi[1]);
        }
        if (q.cut_m()) {
            // log2f in fp32: to 1e-3 of a bin
            const float x = -log2f(q.min_p) * BIN_OCT;
            const int b0 = (int) fmaxf(x - BIN_SLACK - 0.01f, 0.0f), b1 = (int) (x + BIN_SLACK + 0.01f);
            if (b1 < BINS - 1 && b0 <= last) {
                lo[2] = m0 = b0;
                hi[2] = m1 = b1;
                within(b0, b1);
            }
        }
        lo[3] = find_bin(mass, share(q.u, least));
        hi[3] = find_bin(mass, share(q.u, most));
    }
    auto order = [&](int i, int j) {
        const bool sw = lo[j] < lo[i];
        const int x = sw ? lo[j] : lo[i], y = sw ? hi[j] : hi[i];
        lo[j] = sw ? lo[i] : lo[j];
        hi[j] = sw ? hi[i] : hi[j];
        lo[i] = x;
        hi[i] = y;
    };
    order(0, 1); order(2, 3); order(0, 2); order(1, 3); order(1, 2);
    // one where they touch
    if (threadIdx.x & 63) return;
    int n = 0;
    uint32_t tokens = 0;
    uint64_t sum = 0;
    int from = lo[0], to = hi[0];
    auto close = [&] {
        out.lo[n] = from;
        out.hi[n] = to;
        out.before_count[n] = from > 0 ? count[from - 1] : 0;
        out.before_mass[n] = before(from);
        out.list_mass[n] = sum;
        tokens += count[to] - out.before_count[n];
        sum += mass[to] - before(from);
        ++n;
    };
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        if (lo[i] == BINS) continue;
        if (lo[i] <= to + 1) to = max(to, hi[i]);
        else {
            close();
            from = lo[i];
            to = hi[i];
        }
    }
    close();
    out.n = n;
    out.mode = tokens > CAP ? ROW_ALONE : ROW_LIST;      // not counted: the list will tell
    out.mass = mass[BINS - 1];
    out.count = all;
    out.m0 = m0;
    out.m1 = m1;
    out.m_mass = m0 > 0 ? before(m0) : 0;
}

template <int T, bool VEC>
__global__ void __launch_bounds__(ST) sample_hist_kernel(SampleArgs a) {
    __shared__ unsigned long long s_mass[BINS + 64];
    __shared__ uint32_t s_count[BINS + 64];
    __shared__ double s_table[STEPS];
    __shared__ uint64_t s_best[ST / 64];
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const Params q = params_of(a, row);
    const bool masses = !q.counts_only(), counts = q.counts();      // top-k wants counts, the others sums
    if (masses) fill_table(s_table);
    for (int i = tid; i < BINS; i += ST) {
        s_mass[i] = 0;
        s_count[i] = 0;
    }
    const uint64_t best = row_best<ST>(a, row, s_best);          // its barriers cover what was stored before
    if (q.first || q.from_groups() || (uint32_t) (best >> 32) == KEY_NONE) return;
    const Weight w = weight_of(a, best, q.temp, s_table);
    // Tokens of the last bin (w 0, and many of a row may be there) and what is not a number go to slots that are not looked at, a lane
    // one: no branch an element.
    const int lane = tid & 63;
    uint32_t far = 0;
    auto add_masses = [&](auto any) {
        each_unit<T, VEC>(a, row, slice, [&](const float (&x)[PER], int) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const double t = w.template steps<any()>(x[j]);
                const int b = Weight::bin_at(t);
                atomicAdd(&s_mass[b == BINS - 1 ? BINS + lane : b], (unsigned long long) w.fixed_at(t));
            }
        });
    };
    if (masses && w.m < INFINITY) add_masses(std::false_type{});
    else if (masses) add_masses(std::true_type{});
    if (counts)
        each_unit<T, VEC>(a, row, slice, [&](const float (&x)[PER], int) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = w.bin(x[j]);
                atomicAdd(&s_count[b == BINS - 1 ? BINS + lane : b], 1u);
                far += b == BINS - 1 && x[j] > -INFINITY ? 1 : 0;
            }
        });
    if (far) atomicAdd(&s_count[BINS - 1], far);
    __syncthreads();
    for (int i = tid; i < BINS; i += ST) {
        if (s_mass[i]) atomicAdd((unsigned long long*) a.mass + (size_t) row * BINS + i, s_mass[i]);
        if (s_count[i]) atomicAdd(a.count + (size_t) row * BINS + i, s_count[i]);
    }
}

template <int T, bool VEC>
__global__ void __launch_bounds__(ST) sample_gather_kernel(SampleArgs a) {
    constexpr int BUF = 1024;
    __shared__ uint64_t s_token[BUF];
    __shared__ uint32_t s_n, s_at;
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const RowPlan& p = a.plan[row];
    const int mode = p.mode, n = p.n;
    if (mode != ROW_LIST) return;
    float most[4], least[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        most[i] = i < n ? p.most[i] : -INFINITY;
        least[i] = i < n ? p.least[i] : INFINITY;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    auto put = [&](uint32_t at, uint64_t token) {
        if (at < CAP) a.list[(size_t) row * CAP + at] = token;
    };
    // a bit an element, then the few that are set: no branch an element
    const void* const r = row_of<T>(a, row);
    static_assert(PER == 32, "a bit an element");
    each_unit<T, VEC>(a, row, slice, [&](const float (&x)[PER], int from) {
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) hits |= (x[j] >= least[0] && x[j] <= most[0]) || (x[j] >= least[1] && x[j] <= most[1]) ? 1u << j : 0u;
        if (n > 2)
#pragma unroll
            for (int j = 0; j < PER; ++j) hits |= (x[j] >= least[2] && x[j] <= most[2]) || (x[j] >= least[3] && x[j] <= most[3]) ? 1u << j : 0u;
        while (hits) {
            const int i = element<T, VEC>(from, __builtin_ctz(hits));
            hits &= hits - 1;
            const uint64_t token = order_u64(load_logit<T>(r, i), i);
            const uint32_t at = atomicAdd(&s_n, 1u);
            if (at < BUF) s_token[at] = token;
            else put(atomicAdd(a.listed + row, 1u), token);
        }
    });
    __syncthreads();
    const uint32_t here = min(s_n, (uint32_t) BUF);
    if (here == 0) return;
    if (tid == 0) s_at = atomicAdd(a.listed + row, here);
    __syncthreads();
    for (uint32_t i = tid; i < here; i += ST) put(s_at + i, s_token[i]);
}

// ---- sample_pick ----------------------------------------------------------------------------------------
enum Mode { BY_COUNT, BY_MASS, BY_KEY };
// a place in the order: sums up to it, itself included, and the token there
struct Place { uint64_t mass; uint32_t count; uint64_t token; };

struct PickShared {
    uint64_t token[CAP];                                 // gathered, sorted: largest first
    union {
        uint64_t token_mass[CAP];                        // sums up to each
        uint64_t unsorted[CAP];
    };
    uint32_t bucket[CAP];
    uint64_t bin_mass[BINS];                             // sums up to each bin, itself included
    uint32_t bin_count[BINS];
    double table[STEPS];
    Sum part[PT / 64];
    uint64_t best[PT / 64];
    unsigned n;
    int found;
    unsigned long long h_mass[256];
    uint32_t h_count[256];
};

template <int T, bool VEC>
struct Picker {
    const SampleArgs& a;
    PickShared& s;
    const void* row;
    Weight w;
    int b0 = 0, b1 = -1;                                 // bins that are gathered

    static constexpr int STEP = 16;
    template <class F>
    WZY_DEV void scan(F&& f) const {
        for (int from = 0; from < a.vocab; from += PT * STEP) {
            float x[STEP];
            load_elements<T, VEC>(row, from, min(from + PT * STEP, a.vocab), x);
#pragma unroll
            for (int j = 0; j < STEP; ++j) f(x[j], element<T, VEC>(from, j));
        }
    }
    WZY_DEV Sum before_bin(int b) const { return b > 0 ? Sum{s.bin_mass[b - 1], s.bin_count[b - 1]} : Sum{0, 0}; }

    // s.token[0 .. n - 1], largest first
    WZY_DEV void sort(int n) {
        const int tid = threadIdx.x;
        int n2 = 64;
        while (n2 < n) n2 <<= 1;
        for (int i = n + tid; i < n2; i += PT) s.token[i] = 0;
        for (int k = 2; k <= n2; k <<= 1)                        // bitonic
            for (int j = k >> 1; j > 0; j >>= 1) {
                __syncthreads();
                for (int i = tid; i < n2 / 2; i += PT) {
                    const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                    const uint64_t x = s.token[lo], y = s.token[hi];
                    if ((x < y) == ((lo & k) == 0)) {
                        s.token[lo] = y;
                        s.token[hi] = x;
                    }
                }
            }
        __syncthreads();
    }
    // s.token[0 .. n - 1] of at most PT / 4, by counting: four threads a token
    WZY_DEV void sort_few(int n) {
        const int i = threadIdx.x >> 2;
        const uint64_t mine = i < n ? s.token[i] : 0;
        int before = 0;
        for (int j = threadIdx.x & 3; j < n; j += 4) before += s.token[j] > mine ? 1 : 0;
        before += dpp_i<DPP_XOR1>(before);
        before += dpp_i<DPP_XOR2>(before);
        __syncthreads();
        if (i < n && (threadIdx.x & 3) == 0) s.token[before] = mine;
        __syncthreads();
    }
    // s.token = the threads' tokens (0: none), largest first: counted, summed and put by bucket (smaller buckets first), in its bucket a
    // token counts those before it.  starts() is called while s.bucket holds the buckets' first places.
    template <class F, class G>
    WZY_DEV void sort_buckets(const uint64_t (&mine)[CAP / PT], F&& bucket_of, G&& starts) {
        constexpr int E = CAP / PT;
        const int tid = threadIdx.x;
        for (int i = tid; i < CAP; i += PT) s.bucket[i] = 0;
        __syncthreads();
        int to[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            to[j] = mine[j] ? bucket_of(mine[j]) : 0;
            if (mine[j]) atomicAdd(&s.bucket[to[j]], 1u);
        }
        __syncthreads();
        uint32_t size[E], own = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            size[j] = s.bucket[E * tid + j];
            own += size[j];
        }
        uint32_t start = block_sums(Sum{0, own}, s.part).count - own;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            s.bucket[E * tid + j] = start;               // of the bucket; then, as tokens come, its end
            start += size[j];
        }
        __syncthreads();
        starts();
        __syncthreads();
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (mine[j]) s.unsorted[atomicAdd(&s.bucket[to[j]], 1u)] = mine[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (mine[j]) {
                const int first = to[j] > 0 ? (int) s.bucket[to[j] - 1] : 0, last = (int) s.bucket[to[j]];
                int place = first;
#pragma unroll 4
                for (int i = first; i < last; ++i) place += s.unsorted[i] > mine[j] ? 1 : 0;
                s.token[place] = mine[j];
            }
        __syncthreads();
    }
    // the tokens for which take(logit) holds, at most CAP of them, sorted, with their sums from `sum_before` on
    template <class F>
    WZY_DEV void gather(F&& take, Sum sum_before) {
        const int tid = threadIdx.x;
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        scan([&](float l, int i) {
            if (l > -INFINITY && take(l)) {
                const unsigned at = atomicAdd(&s.n, 1u);
                if (at < CAP) s.token[at] = order_u64(l, i);
            }
        });
        __syncthreads();
        const int n = min((int) s.n, CAP);
        sort(n);
        // CAP / PT neighbours a thread
        constexpr int Q = CAP / PT;
        uint64_t m[Q], sum = 0;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int i = Q * tid + q;
            m[q] = i < n ? w.fixed(key_value((uint32_t) (s.token[i] >> 32))) : 0;
            sum += m[q];
        }
        uint64_t at = block_sums(Sum{sum, 0}, s.part).mass - sum + sum_before.mass;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            at += m[q];
            if (Q * tid + q < n) s.token_mass[Q * tid + q] = at;
        }
        __syncthreads();
        gathered = n;
        before = Place{sum_before.mass, sum_before.count, 0};
    }
    int gathered = 0;
    Place before{0, 0, 0};                               // the sums before the gathered tokens

    // s.found = the least i of those that have one, i rising with the lanes: one atomic a wave (from all lanes they queue up at one
    // address: 6,000 cycles)
    WZY_DEV void lowest(bool have, int i) {
        const uint64_t b = __ballot(have);
        if (b && (int) (threadIdx.x & 63) == __ffsll((unsigned long long) b) - 1) atomicMin(&s.found, i);
    }
    // the first gathered token at which the target is reached (the last with key >= target, BY_KEY); the last one, if none
    WZY_DEV Place among(Mode mode, uint64_t target) {
        if (threadIdx.x == 0) s.found = gathered - 1;
        __syncthreads();
        // a bin whose tokens all fail ends before its first
        if (mode == BY_KEY && (s.token[0] >> 32) < target) return before;
        for (int i = threadIdx.x; i < gathered; i += PT) {
            bool here;
            if (mode == BY_COUNT) here = before.count + i + 1 >= target;
            else if (mode == BY_MASS) here = s.token_mass[i] >= target;
            else here = i + 1 < gathered && (s.token[i + 1] >> 32) < target;
            lowest(here, i);
        }
        __syncthreads();
        const int i = s.found;
        const Place p{s.token_mass[i], before.count + (uint32_t) i + 1, s.token[i]};
        __syncthreads();
        return p;
    }
    // a bin of more tokens than are gathered: by 8 bits of the key at a time until few enough share them, or all bits; then by id
    WZY_DEV Place descend(int b, Mode mode, uint64_t target) {
        const int tid = threadIdx.x;
        Sum so_far = before_bin(b);
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            for (int i = tid; i < 256; i += PT) { s.h_mass[i] = 0; s.h_count[i] = 0; }
            __syncthreads();
            scan([&](float l, int) {
                const uint32_t k = order_key(l);
                if (l > -INFINITY && w.bin(l) == b && (shift == 24 || (k >> (shift + 8)) == prefix)) {
                    const int d = 255 - (int) (k >> shift & 255);
                    atomicAdd(&s.h_mass[d], (unsigned long long) w.fixed(l));
                    atomicAdd(&s.h_count[d], 1u);
                }
            });
            __syncthreads();
            Sum up = so_far;
            int d = 0;
            for (; d < 256; ++d) {                       // every thread the same
                const uint32_t k = prefix << 8 | (uint32_t) (255 - d);
                const Sum next{up.mass + s.h_mass[d], up.count + s.h_count[d]};
                if (s.h_count[d]) {
                    const bool here = mode == BY_COUNT ? next.count >= target : mode == BY_MASS ? next.mass >= target : k <= (uint32_t) (target >> shift);
                    if (here) break;
                }
                up = next;
            }
            if (d == 256) {                              // not reached: the last that there is
                for (d = 255; d > 0 && !s.h_count[d]; --d) {}
                up.mass -= s.h_mass[d];
                up.count -= s.h_count[d];
            }
            so_far = up;
            // all from here on fail
            if (mode == BY_KEY && (prefix << 8 | (uint32_t) (255 - d)) < (uint32_t) (target >> shift)) return Place{up.mass, up.count, 0};
            prefix = prefix << 8 | (uint32_t) (255 - d);
            const uint32_t n = s.h_count[d];
            if (n <= CAP) {
                gather([&](float l) { return w.bin(l) == b && (order_key(l) >> shift) == prefix; }, so_far);
                b0 = 0; b1 = -1;
                return among(mode, target);
            }
        }
        // equal logits: the j-th of them by id
        __syncthreads();
        const float l = key_value(prefix);
        const uint64_t each_w = w.fixed(l);
        const uint32_t all = s.h_count[255 - (int) (prefix & 255)];
        uint64_t j = all;
        if (mode == BY_COUNT && target > so_far.count) j = target - so_far.count;
        if (mode == BY_MASS) j = each_w == 0 ? all : target > so_far.mass ? (target - so_far.mass + each_w - 1) / each_w : 1;
        if (j > all) j = all;
        if (j < 1) j = 1;
        uint32_t seen = 0;
        for (int from = 0; from < a.vocab; from += PT) {
            const int i = from + tid;
            bool hit = false;
            if (i < a.vocab) {
                float v;
                if constexpr (T == WZY_F32) v = ((const float*) row)[i];
                else if constexpr (T == WZY_BF16) v = bf16_to_f(((const uint16_t*) row)[i]);
                else v = h16_to_f(((const uint16_t*) row)[i]);
                hit = order_key(v) == prefix;
            }
            const Sum x = block_sums(Sum{0, hit ? 1u : 0u}, s.part);
            if (hit && seen + x.count == j) s.found = i;
            if (tid == PT - 1) s.n = x.count;
            __syncthreads();
            seen += s.n;
            __syncthreads();
            if (seen >= j) break;
        }
        return Place{so_far.mass + j * each_w, so_far.count + (uint32_t) j, (uint64_t) prefix << 32 | (uint32_t) ~s.found};
    }
    // the place where the target is reached
    WZY_DEV Place locate(Mode mode, uint64_t target) {
        const int tid = threadIdx.x;
        __syncthreads();
        if (tid == 0) s.found = -1;
        __syncthreads();
        int b;
        if (mode == BY_KEY) b = w.bin(key_value((uint32_t) target));
        else {
            const Sum t{s.bin_mass[tid], s.bin_count[tid]}, p = before_bin(tid);
            if (t.count > p.count && (mode == BY_COUNT ? t.count >= target && p.count < target : t.mass >= target && p.mass < target)) s.found = tid;
            __syncthreads();
            b = s.found;
        }
        if (mode != BY_KEY && b < 0) b = BINS - 1;
        while (b > 0 && s.bin_count[b] == before_bin(b).count) --b;          // an empty bin: the tokens before it
        __syncthreads();
        if (b < b0 || b > b1) {
            if (s.bin_count[b] <= CAP) {
                gather([&](float l) { return w.bin(l) <= b; }, Sum{0, 0});
                b0 = 0;
                b1 = b;
            } else if (s.bin_count[b] - before_bin(b).count <= CAP) {
                gather([&](float l) { return w.bin(l) == b; }, before_bin(b));
                b0 = b1 = b;
            } else return descend(b, mode, target);
        }
        return among(mode, target);
    }
    // The places in s.token[0 .. n - 1], sorted, and the answer.  plan: whole bins, where the sums before an interval are the row's;
    // null: the row's first tokens, all that top-k leaves among them.
    WZY_DEV void finish(const Params& q, int r, int n, const RowPlan* plan, const int (&in_list)[4]) {
        if (n <= PT) finish_with<1>(q, r, n, plan, in_list);
        else finish_with<CAP / PT>(q, r, n, plan, in_list);
    }
    template <int Q>
    WZY_DEV void finish_with(const Params& q, int r, int n, const RowPlan* plan, const int (&in_list)[4]) {
        const int tid = threadIdx.x;
        const bool all = !plan || q.counts_only();
        uint64_t m[Q], sum = 0;
#pragma unroll
        for (int j = 0; j < Q; ++j) {
            const int i = Q * tid + j;
            m[j] = i < n ? w.fixed(key_value((uint32_t) (s.token[i] >> 32))) : 0;
            sum += m[j];
        }
        uint64_t at = block_sums(Sum{sum, 0}, s.part).mass - sum;
        uint32_t count[Q];
#pragma unroll
        for (int j = 0; j < Q; ++j) {
            const int i = Q * tid + j;
            at += m[j];
            count[j] = (uint32_t) i + 1;
            m[j] = at;
            if (plan) {
                int v = 0;                               // the token's interval: the last that starts at or before it
#pragma unroll
                for (int k = 1; k < 4; ++k) v = i >= in_list[k] ? k : v;
                count[j] = (uint32_t) (i + 1 - (v == 0 ? in_list[0] : v == 1 ? in_list[1] : v == 2 ? in_list[2] : in_list[3])) + plan->before_count[v];
                m[j] = at - plan->list_mass[v] + plan->before_mass[v];
            }
            if (i < n) s.token_mass[i] = m[j];
        }
        // the first of the list for which here(sum, count) holds; the last, if none
        auto first = [&](auto&& here) {
            if (tid == 0) s.found = n - 1;
            __syncthreads();
            int f = n;
#pragma unroll
            for (int j = Q - 1; j >= 0; --j)
                if (Q * tid + j < n && here(m[j], count[j])) f = Q * tid + j;
            lowest(f < n, f);
            __syncthreads();
            const int i = s.found;
            __syncthreads();
            return i;
        };
        // What is left, as a sum: of two places the one with the smaller sum comes first.
        __syncthreads();
        uint64_t end = all ? s.token_mass[n - 1] : plan->mass;
        if (!plan) end = s.token_mass[(q.k >= 1 ? min(q.k, n) : n) - 1];
        else if (q.k >= 1 && (uint32_t) q.k < plan->count) end = s.token_mass[first([&](uint64_t, uint32_t c) { return c >= (uint32_t) q.k; })];
        const uint64_t of_k = end;
        if (q.cut_p()) {
            const uint64_t t = share((double) q.top_p, of_k), x = s.token_mass[first([&](uint64_t y, uint32_t) { return y >= t; })];
            end = x < end ? x : end;
        }
        if (q.cut_m() && (all || plan->m0 >= 0)) {
            // of the bins in which min-p ends, those that pass; the bins before pass, the bins behind do not
            const int m0 = all ? 0 : plan->m0, m1 = all ? BINS - 1 : plan->m1;
            Sum pass{0, 0};
#pragma unroll
            for (int j = 0; j < Q; ++j) {
                if (Q * tid + j >= n) continue;
                const float l = key_value((uint32_t) (s.token[Q * tid + j] >> 32));
                const int b = w.bin(l);
                if (b >= m0 && b <= m1 && w.w(l) >= (double) q.min_p) pass.mass += w.fixed(l);
            }
            pass = block_sums(pass, s.part);
            if (tid == PT - 1) s.part[0] = pass;
            __syncthreads();
            const uint64_t x = s.part[0].mass + (all ? 0 : plan->m_mass);
            __syncthreads();
            end = x < end ? x : end;
        }
        const uint64_t t = share(q.u, end);
        const int i = first([&](uint64_t x, uint32_t) { return x >= t; });
        if (tid == 0) {
            a.ids[r] = (int) ~(uint32_t) s.token[i];
            if (a.probs) a.probs[r] = (float) (w.scaled(key_value((uint32_t) (s.token[i] >> 32)), a.F) / (double) end);
        }
    }
};

// a row by itself: its histogram, then the places, with a pass over the row for each range that is gathered
template <int T, bool VEC>
WZY_DEV void pick_alone(const SampleArgs& a, int row, const Params& q, uint64_t best, PickShared& s, Picker<T, VEC>& p) {
    const int tid = threadIdx.x;
    unsigned long long* const h = (unsigned long long*) s.bin_mass;
    h[tid] = 0;
    s.bin_count[tid] = 0;
    __syncthreads();
    p.scan([&](float l, int) {
        if (!(l > -INFINITY)) return;
        const int b = p.w.bin(l);
        if (b < BINS - 1) atomicAdd(&h[b], (unsigned long long) p.w.fixed(l));
        atomicAdd(&s.bin_count[b], 1u);
    });
    __syncthreads();
    const Sum own{s.bin_mass[tid], s.bin_count[tid]}, sum = block_sums(own, s.part);
    s.bin_mass[tid] = sum.mass;
    s.bin_count[tid] = sum.count;
    __syncthreads();
    Place end{s.bin_mass[BINS - 1], s.bin_count[BINS - 1], 0};
    if (q.k >= 1 && (uint32_t) q.k < end.count) end = p.locate(BY_COUNT, (uint64_t) q.k);
    if (q.cut_p()) {
        const Place x = p.locate(BY_MASS, share((double) q.top_p, end.mass));
        if (x.count < end.count) end = x;
    }
    if (q.cut_m()) {
        // the lowest key whose weight is min_p or more: halving, every thread the same
        uint32_t hi = (uint32_t) (best >> 32), lo = KEY_NONE;             // hi passes, lo does not
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (p.w.w(key_value(mid)) >= (double) q.min_p) hi = mid;
            else lo = mid;
        }
        // where the last token kept so far passes, nothing is cut
        if (end.token == 0 || (uint32_t) (end.token >> 32) < hi) {
            const Place x = p.locate(BY_KEY, hi);
            if (x.count < end.count) end = x;
        }
    }
    const Place x = p.locate(BY_MASS, share(q.u, end.mass));
    if (tid == 0) {
        a.ids[row] = (int) ~(uint32_t) x.token;
        if (a.probs) a.probs[row] = (float) (p.w.scaled(key_value((uint32_t) (x.token >> 32)), a.F) / (double) end.mass);
    }
}

// Rows with a small top-k, from the groups' largest keys: the k-th largest of those is at most the row's k-th largest, so the tokens
// at or above it are k or more, and they lie in the groups whose largest is.  Which groups: a histogram of the keys' distance from
// the best one, 64 bins an octave (keys themselves would all fall into a few), up to the bin that holds the k-th.  False: too
// many (ties).
WZY_DEV uint32_t distance_bin(uint32_t best, uint32_t key) {
    const uint32_t d = best - key;
    const int top = 31 - __builtin_clz(d | 1);
    return d < 64 ? d : (uint32_t) (top - 5) * 64 + (d >> (top - 6) & 63);   // up to 27 * 64 - 1
}
template <int T, bool VEC>
WZY_DEV bool pick_from_groups(const SampleArgs& a, int row, const Params& q, uint64_t best, PickShared& s, Picker<T, VEC>& p) {
    const int tid = threadIdx.x;
    const uint32_t* const g = a.group + (size_t) row * a.groups;
    const uint32_t top = (uint32_t) (best >> 32);
    constexpr int HOLD = 8;                              // keys a thread keeps; more are read twice
    uint32_t mine[HOLD];
#pragma unroll
    for (int j = 0; j < HOLD; ++j) mine[j] = tid + j * PT < a.groups ? g[tid + j * PT] : 0;
    for (int i = tid; i < 2 * PT; i += PT) s.bucket[i] = 0;
    if (tid == 0) {
        s.found = 2 * PT - 1;
        s.n = 0;
    }
    __syncthreads();
    auto each_group = [&](auto&& f) {                    // groups with a token
#pragma unroll
        for (int j = 0; j < HOLD; ++j)
            if (mine[j] > KEY_NONE) f(mine[j], tid + j * PT);
        for (int i = tid + HOLD * PT; i < a.groups; i += PT)
            if (g[i] > KEY_NONE) f(g[i], i);
    };
    each_group([&](uint32_t key, int) { atomicAdd(&s.bucket[distance_bin(top, key)], 1u); });
    __syncthreads();
    const uint32_t c0 = s.bucket[2 * tid], c1 = s.bucket[2 * tid + 1], k = (uint32_t) q.k;
    const uint32_t up = block_sums(Sum{0, c0 + c1}, s.part).count, b = up - c0 - c1;
    if (b < k && up >= k) s.found = b + c0 >= k ? 2 * tid : 2 * tid + 1;       // fewer groups than k: all of them
    __syncthreads();
    const uint32_t last = (uint32_t) s.found;
    // the groups, then their tokens, a thread a token at a time
    each_group([&](uint32_t key, int i) {
        if (distance_bin(top, key) <= last) {
            const unsigned at = atomicAdd(&s.n, 1u);
            if (at < CAP) s.bucket[at] = (uint32_t) i;
        }
    });
    __syncthreads();
    const int groups = (int) s.n;
    __syncthreads();
    if (groups > CAP) return false;
    if (tid == 0) s.n = 0;
    __syncthreads();
    constexpr int E = !VEC ? 1 : T == WZY_F32 ? 4 : 8;
    for (int i = tid; i < groups * PER; i += PT) {
        const int group = (int) s.bucket[i / PER], j = i % PER, e = group / ST * SLICE + ((j / E) * ST + group % ST) * E + j % E;
        if (e < a.vocab) {
            const float l = load_logit<T>(p.row, e);
            if (l > -INFINITY && distance_bin(top, order_key(l)) <= last) {
                const unsigned at = atomicAdd(&s.n, 1u);
                if (at < CAP) s.token[at] = order_u64(l, e);
            }
        }
    }
    __syncthreads();
    const int n = (int) s.n;
    __syncthreads();
    if (n > CAP) return false;
    if (n <= PT / 4) p.sort_few(n);
    else p.sort(n);
    const int none[4] = {0, 0, 0, 0};
    p.finish(q, row, n, nullptr, none);
    return true;
}

// Rows that need no list get their token here; for the others, which bins are wanted
template <int T, bool VEC>
__global__ void __launch_bounds__(PT) sample_plan_kernel(SampleArgs a) {
    __shared__ PickShared s;
    __shared__ RowPlan s_plan;
    static_assert(BINS == PT, "a thread a bin");
    const int row = blockIdx.x, tid = threadIdx.x;
    const Params q = params_of(a, row);
    const Sum own{a.mass[(size_t) row * BINS + tid], a.count[(size_t) row * BINS + tid]};
    fill_table(s.table);
    const uint64_t best = row_best<PT>(a, row, s.best);
    if (q.first || (uint32_t) (best >> 32) == KEY_NONE) {
        const bool none = (uint32_t) (best >> 32) == KEY_NONE;
        if (tid == 0) {
            a.plan[row].mode = ROW_DONE;
            a.ids[row] = none ? -1 : (int) ~(uint32_t) best;
            if (a.probs) a.probs[row] = none ? 0.0f : 1.0f;
        }
        return;
    }
    if (q.from_groups()) {
        Picker<T, VEC> p{a, s, row_of<T>(a, row), weight_of(a, best, q.temp, s.table)};
        const bool done = pick_from_groups<T, VEC>(a, row, q, best, s, p);
        if (tid == 0) {
            a.plan[row].best = best;
            a.plan[row].q = q;
            a.plan[row].mode = done ? ROW_DONE : ROW_ALONE;
        }
        return;
    }
    const Sum at = block_sums(own, s.part);
    s.bin_mass[tid] = at.mass;
    s.bin_count[tid] = at.count;
    __syncthreads();
    if (tid >= 64) return;
    plan_row(q, s.bin_mass, s.bin_count, s_plan);
    wave_lds_sync();
    // The intervals' ends as logits, a lane an end: the lowest key whose bin is at most b (hi, or lo - 1 and the key before).  The bin falls
    // as the key rises; where it reaches b is known to a few keys.
    if (tid < 2 * s_plan.n) {
        const Weight w = weight_of(a, best, q.temp, nullptr);
        const int j = tid >> 1, b = tid & 1 ? s_plan.lo[j] - 1 : s_plan.hi[j];
        auto at_most = [&](uint32_t k) { return w.bin(key_value(k)) <= b; };
        uint32_t lo = KEY_NONE, hi = (uint32_t) (best >> 32) + 1;             // lo is not, hi is (or past the best one)
        constexpr uint32_t NEAR = 4;
        const uint32_t at = order_key((float) ((double) w.m - ((double) ((b + 1) << BIN_STEPS_LOG2) - 0.5) / w.cs));
        const uint32_t from = at > lo + NEAR ? at - NEAR : lo, to = at + NEAR < hi && at + NEAR > at ? at + NEAR : hi;
        if (from > lo && from < hi && !at_most(from)) lo = from;
        if (to > lo && to < hi && at_most(to)) hi = to;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (at_most(mid)) hi = mid;
            else lo = mid;
        }
        if (tid & 1) s_plan.most[j] = key_value(hi - 1);
        else s_plan.least[j] = key_value(hi);
    }
    if (tid == 63) {
        s_plan.best = best;
        s_plan.q = q;
    }
    wave_lds_sync();
    const uint32_t* const from = (const uint32_t*) &s_plan;
    uint32_t* const to = (uint32_t*) (a.plan + row);
    for (int i = tid; i < (int) (sizeof(RowPlan) / 4); i += 64) to[i] = from[i];
}

template <int T, bool VEC>
__global__ void __launch_bounds__(PT) sample_pick_kernel(SampleArgs a) {
    __shared__ PickShared s;
    __shared__ RowPlan plan;
    const int row = blockIdx.x, tid = threadIdx.x;
    const int mode = a.plan[row].mode;
    const uint32_t all_listed = a.listed[row];
    if (tid < (int) (sizeof(RowPlan) / 4)) ((uint32_t*) &plan)[tid] = ((const uint32_t*) (a.plan + row))[tid];
    if (mode == ROW_DONE) return;
    fill_table(s.table);
    __syncthreads();
    const Params q = plan.q;
    const uint64_t best = plan.best;
    Picker<T, VEC> p{a, s, row_of<T>(a, row), weight_of(a, best, q.temp, s.table)};
    const uint32_t listed = mode == ROW_LIST ? all_listed : 0;
    if (mode == ROW_ALONE || listed > CAP) {
        pick_alone<T, VEC>(a, row, q, best, s, p);
        return;
    }
    // The list: whole bins, so a token's place is its place in the list and what lies before its interval and is not in the list.
    // Sorted by CAP buckets, as many for each bin: in its bucket a token counts those before it.
    const int n = (int) listed;
    int lo[4], skip[4], bins = 0;                        // skip: bins of the intervals before
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool is = k < plan.n;
        lo[k] = is ? plan.lo[k] : BINS;
        skip[k] = bins;
        bins += is ? plan.hi[k] - plan.lo[k] + 1 : 0;
    }
    int in_list[4];                                      // tokens of the list before each interval
    if (n <= PT / 4) {
        if (tid < 4) s.h_count[tid] = 0;
        if (tid < n) s.token[tid] = a.list[(size_t) row * CAP + tid];
        __syncthreads();
        if (tid < n) {
            const int b = p.w.bin(key_value((uint32_t) (s.token[tid] >> 32)));
#pragma unroll
            for (int k = 1; k < 4; ++k)
                if (lo[k] < BINS && b < lo[k]) atomicAdd(&s.h_count[k], 1u);
        }
        p.sort_few(n);
#pragma unroll
        for (int k = 0; k < 4; ++k) in_list[k] = lo[k] < BINS ? (int) s.h_count[k] : CAP;
    } else {
        const int per = CAP / bins;
        const float scale = p.w.cf * BIN_OCT;
        auto bucket_of = [&](uint64_t token) {
            const float l = key_value((uint32_t) (token >> 32));
            const int b = p.w.bin(l);
            int v = 0;
#pragma unroll
            for (int k = 1; k < 4; ++k) v = b >= lo[k] ? k : v;
            const float in = l == p.w.m ? 0.0f : fminf((p.w.m - l) * scale, (float) (BINS - 1)) + BIN_SLACK - (float) b;
            const int at = b - (v == 0 ? lo[0] : v == 1 ? lo[1] : v == 2 ? lo[2] : lo[3]) + (v == 0 ? skip[0] : v == 1 ? skip[1] : v == 2 ? skip[2] : skip[3]);
            return min(at * per + min((int) (fmaxf(in, 0.0f) * (float) per), per - 1), CAP - 1);
        };
        uint64_t mine[CAP / PT];
#pragma unroll
        for (int j = 0; j < CAP / PT; ++j) mine[j] = tid + j * PT < n ? a.list[(size_t) row * CAP + tid + j * PT] : 0;
        p.sort_buckets(mine, bucket_of, [&] {
#pragma unroll
            for (int k = 0; k < 4; ++k) in_list[k] = lo[k] < BINS ? (int) s.bucket[skip[k] * per] : CAP;
        });
    }
    p.finish(q, row, n, &plan, in_list);
}

// Rows of at most SHORT logits: all of them sorted, one launch (14 rows of 2,042: 11 to 13 us against 25 in five launches, 100
// logits 6 to 7; 64 rows of 4,096 take 26 to 28 either way)
template <int T>
__global__ void __launch_bounds__(PT) sample_short_kernel(SampleArgs a) {
    __shared__ PickShared s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const void* const from = row_of<T>(a, row);
    uint64_t mine[CAP / PT], best = 0;
#pragma unroll
    for (int j = 0; j < CAP / PT; ++j) {                 // places past SHORT stay empty
        const int i = tid + j * PT;
        const float l = i < a.vocab ? load_logit<T>(from, i) : -INFINITY;
        mine[j] = l > -INFINITY ? order_u64(l, i) : 0;
        best = max_u64(best, mine[j]);
    }
    const Params q = params_of(a, row);
    if (tid == 0) s.n = 0;
    fill_table(s.table);
    best = wave_max_u64(best);
    if (lane == 0) s.best[tid >> 6] = best;
    __syncthreads();
    best = wave_max_u64(lane < PT / 64 ? s.best[lane] : 0);
    if (q.first || best == 0) {
        if (tid == 0) {
            a.ids[row] = best == 0 ? -1 : (int) ~(uint32_t) best;
            if (a.probs) a.probs[row] = best == 0 ? 0.0f : 1.0f;
        }
        return;
    }
    unsigned own = 0;                                    // the wave's
#pragma unroll
    for (int j = 0; j < CAP / PT; ++j) own += (unsigned) __popcll(__ballot(mine[j] != 0));
    if (lane == 0 && own) atomicAdd(&s.n, own);
    Picker<T, false> p{a, s, from, weight_of(a, best, q.temp, s.table)};
    const float m = p.w.m;
    if (a.vocab <= PT / 4) {
        if (tid < PT / 4) s.token[tid] = mine[0];        // none at all is smaller than any
        __syncthreads();
        p.sort_few(a.vocab);
    } else p.sort_buckets(mine, [&](uint64_t token) {                   // by the distance from the best logit, 128 buckets an octave from 2^-8 on
        const float l = key_value((uint32_t) (token >> 32)), d = l == m ? 0.0f : m - l;
        return min(max((__builtin_bit_cast(int, d) >> 16) - ((127 - 8) << 7), 0), CAP - 1);
    }, [] {});
    const int none[4] = {0, 0, 0, 0};
    p.finish(q, row, (int) s.n, nullptr, none);
}

template <int T, bool VEC>
int launch(const SampleArgs& a, void* stream) {
    const dim3 grid((unsigned) a.slices, (unsigned) a.rows);
    sample_max_kernel<T, VEC><<<grid, ST, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    sample_hist_kernel<T, VEC><<<grid, ST, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    sample_plan_kernel<T, VEC><<<a.rows, PT, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    sample_gather_kernel<T, VEC><<<grid, ST, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    sample_pick_kernel<T, VEC><<<a.rows, PT, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    return WZY_OK;
}
constexpr int MAX_VOCAB = 1 << 22, MAX_ROWS = 65535;
// slices: enough of them for all CUs, and where there are many rows larger ones, with fewer histograms to add
size_t space(int rows, int vocab, SampleArgs* a, void* base, size_t cap) {
    const int units = pg_div_up(vocab, SLICE), most = std::max(1, 2048 / rows), per = pg_div_up(units, std::min(units, most));
    const int slices = pg_div_up(units, per);
    Arena w(base, cap);
    uint64_t* const best = w.take<uint64_t>((size_t) rows * slices);
    uint64_t* const mass = w.take<uint64_t>((size_t) rows * BINS);
    uint32_t* const count = w.take<uint32_t>((size_t) rows * BINS);
    RowPlan* const plan = w.take<RowPlan>((size_t) rows);
    uint32_t* const listed = w.take<uint32_t>((size_t) rows);
    uint64_t* const list = w.take<uint64_t>((size_t) rows * CAP);
    uint32_t* const group = w.take<uint32_t>((size_t) rows * units * ST);
    if (a) {
        a->best = best; a->mass = mass; a->count = count; a->plan = plan; a->listed = listed; a->list = list;
        a->group = group;
        a->groups = units * ST;
        a->slices = slices;
        a->units = per;
    }
    return w.off;
}
}  // namespace

extern "C" size_t wzy_sample_workspace_bytes(int rows, int vocab) {
    if (rows < 1 || rows > MAX_ROWS || vocab < 1 || vocab > MAX_VOCAB) return 0;
    return space(rows, vocab, nullptr, nullptr, 0);
}

extern "C" int wzy_sample(const void* logits, int type, int64_t ld, int rows, int vocab, const float* temp, const int* top_k,
                          const float* top_p, const float* min_p, const float* u, int* ids, float* probs, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const char* const who = "wzy_sample";
    WZY_TRY(mx_check_type(who, type));
    WZY_REQUIRE(rows >= 0 && rows <= MAX_ROWS && vocab >= 1 && vocab <= MAX_VOCAB, "%s: %d rows of %d logits (at most %d of %d)", who, rows,
                vocab, MAX_ROWS, MAX_VOCAB);
    if (rows == 0) return WZY_OK;
    WZY_REQUIRE(logits && u && ids, "%s: logits, u or ids are null", who);
    const int n = mx_type_bytes(type);
    WZY_REQUIRE(ld >= vocab && ld <= (int64_t) 1 << 40 && (uintptr_t) logits % n == 0, "%s: rows of %d logits, stride %lld at %p", who, vocab,
                (long long) ld, logits);
    SampleArgs a{};
    const size_t want = space(rows, vocab, &a, workspace, workspace_bytes);
    WZY_REQUIRE(workspace && workspace_bytes >= want && (uintptr_t) workspace % 16 == 0, "%s: workspace of %zu bytes at %p (%zu, 16-byte aligned)", who,
                workspace_bytes, workspace, want);
    a.logits = logits; a.ld = ld; a.rows = rows; a.vocab = vocab;
    a.temp = temp; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.u = u; a.ids = ids; a.probs = probs;
    if (!top_k) a.group = nullptr;
    a.F = 51;
    while (a.F > 40 && (int64_t) vocab > (1ll << (62 - a.F))) --a.F;
    if (vocab <= SHORT)
        return mx_with_type(type, [&](auto t) {
            sample_short_kernel<t()><<<rows, PT, 0, as_stream(stream)>>>(a);
            WZY_LAUNCH_CHECK();
            return WZY_OK;
        });
    const bool vec = (uintptr_t) logits % 16 == 0 && ld * n % 16 == 0;
    return mx_with_type(type, [&](auto t) { return vec ? launch<t(), true>(a, stream) : launch<t(), false>(a, stream); });
}
