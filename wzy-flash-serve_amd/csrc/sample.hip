// sample.hip -- one token a row of logits, by temperature, top-k, min-p and top-p, from given uniform numbers.
//
// The order of a row is (logit descending, id ascending).  Every cut keeps a prefix of it, and the draw takes the first
// token whose running sum of w = 2^-x, x = (max - l) log2(e) / temp, reaches a target; so all that is needed are places in
// that order: by count (top-k), by sum (top-p, the draw), by value (min-p).  No sort of the row: a histogram over x in bins of
// 1/16 (count and sum of w) says in which bin a place lies, and only the tokens of that bin, or of all up to it where they are
// few, are gathered and sorted.  Three launches:
//   sample_max   a slice of a row a workgroup: its best token
//   sample_hist  the same slices: x against the row's best, histogram in LDS, then added to the row's
//   sample_pick  a workgroup a row: the places, with a pass over the row for each gathered range (one for top-k and small
//                nuclei, two for large ones)
// w is taken in 64 bits (fp32's 1e-7 would move one draw in a thousand of a flat row) and summed as integers of 2^-F, F = 62 -
// log2(vocab): sums do not depend on their order, so LDS and memory atomics may add them as they come.
#include "wzy_paged.h"

using namespace wzy;

namespace {
constexpr int ST = 256, PER = 32, SLICE = ST * PER;      // sample_max, sample_hist
constexpr int PT = 1024, CAP = 4096;                     // sample_pick; tokens gathered at most
constexpr int BINS = 1024;                               // 64 octaves of w
constexpr float BIN_OCT = 16.0f;
constexpr float GREEDY = 1e-5f;
constexpr uint32_t KEY_NONE = 0x007FFFFFu;               // order key of -infinity

struct SampleArgs {
    const void* logits;
    int64_t ld;
    int rows, vocab, slices, F;
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

// 2^(-j / 64)
WZY_DEV void fill_table(double* s) {
    for (int i = threadIdx.x; i < 64; i += blockDim.x) s[i] = exp2(-(double) i / 64.0);
}
// A row's weights: m its largest logit, c = log2(e) / temp.  The bin is taken in fp32, which is monotone too.
struct Weight {
    float m, cf;
    double c;
    int F;
    const double* table;
    WZY_DEV int bin(float l) const {
        const float x = l == m ? 0.0f : (m - l) * cf * BIN_OCT;
        return (int) fminf(x, (float) (BINS - 1));
    }
    WZY_DEV double x(float l) const { return l == m ? 0.0 : ((double) m - (double) l) * c; }
    // 2^-x: x = n + j / 64 + r / 64, |r| <= 1/2; the series of 2^(-r / 64) to the fifth power leaves 2e-18
    WZY_DEV double w(float l) const {
        const double v = x(l);
        if (!(v < 1000.0)) return 0.0;
        const double t = v * 64.0, k = rint(t), r = (t - k) * (-0.6931471805599453094 / 64.0);
        const int i = (int) k;
        double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
        p = fma(p, r, 1.0 / 6.0);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        return ldexp(p * table[i & 63], -(i >> 6));
    }
    WZY_DEV uint64_t fixed(float l) const { return (uint64_t) rint(ldexp(w(l), F)); }
};
WZY_DEV float temp_of(const SampleArgs& a, int row) { return a.temp ? a.temp[row] : 1.0f; }
WZY_DEV bool greedy(float t) { return !(t > GREEDY); }

// f(value, id) over elements from .. from + n * threads - 1 (limited to end) of a row: 16 bytes a thread where the row allows
template <int T, bool VEC, int N, class F>
WZY_DEV void each(const void* row, int from, int end, F&& f) {
    constexpr int E = T == WZY_F32 ? 4 : 8;
    if constexpr (VEC) {
        // loads first, then their use
        uint4 v[N / E];
#pragma unroll
        for (int i = 0; i < N / E; ++i) {
            const int e = from + (i * (int) blockDim.x + (int) threadIdx.x) * E;
            v[i] = e + E <= end ? *(const uint4*) ((const char*) row + (size_t) e * (16 / E)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < N / E; ++i) {
            const int e = from + (i * (int) blockDim.x + (int) threadIdx.x) * E;
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            if (e + E <= end) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    float x;
                    if constexpr (T == WZY_F32) x = __builtin_bit_cast(float, w[j]);
                    else if constexpr (T == WZY_BF16) x = j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]);
                    else x = h16_to_f((uint16_t) (w[j / 2] >> (16 * (j & 1))));
                    f(x, e + j);
                }
            } else {
                for (int j = e; j < end; ++j) {
                    float x;
                    if constexpr (T == WZY_F32) x = ((const float*) row)[j];
                    else if constexpr (T == WZY_BF16) x = bf16_to_f(((const uint16_t*) row)[j]);
                    else x = h16_to_f(((const uint16_t*) row)[j]);
                    f(x, j);
                }
            }
        }
    } else {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = min(from + i * (int) blockDim.x + (int) threadIdx.x, end - 1);
            if constexpr (T == WZY_F32) v[i] = ((const float*) row)[e];
            else if constexpr (T == WZY_BF16) v[i] = bf16_to_f(((const uint16_t*) row)[e]);
            else v[i] = h16_to_f(((const uint16_t*) row)[e]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = from + i * (int) blockDim.x + (int) threadIdx.x;
            if (e < end) f(v[i], e);
        }
    }
}
template <int T>
WZY_DEV const void* row_of(const SampleArgs& a, int row) {
    return (const char*) a.logits + (size_t) row * a.ld * (T == WZY_F32 ? 4 : 2);
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
    uint64_t b = 0;
    const int from = slice * SLICE;
    each<T, VEC, PER>(row_of<T>(a, row), from, min(from + SLICE, a.vocab), [&](float v, int i) { b = max_u64(b, order_u64(v, i)); });
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
    w.c = 1.44269504088896340736 / (double) t;
    w.cf = (float) w.c;
    w.F = a.F;
    w.table = table;
    return w;
}

template <int T, bool VEC>
__global__ void __launch_bounds__(ST) sample_hist_kernel(SampleArgs a) {
    __shared__ unsigned long long s_mass[BINS];
    __shared__ uint32_t s_count[BINS];
    __shared__ double s_table[64];
    __shared__ uint64_t s_best[ST / 64];
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const float t = temp_of(a, row);
    if (greedy(t)) return;
    fill_table(s_table);
    for (int i = tid; i < BINS; i += ST) {
        s_mass[i] = 0;
        s_count[i] = 0;
    }
    const uint64_t best = row_best<ST>(a, row, s_best);          // its barriers cover what was stored before
    if ((uint32_t) (best >> 32) == KEY_NONE) return;
    const Weight w = weight_of(a, best, t, s_table);
    uint32_t far = 0;
    uint64_t far_mass = 0;
    const int from = slice * SLICE;
    each<T, VEC, PER>(row_of<T>(a, row), from, min(from + SLICE, a.vocab), [&](float l, int) {
        if (!(l > -INFINITY)) return;
        const int b = w.bin(l);
        const uint64_t f = w.fixed(l);
        if (b == BINS - 1) {                                    // many of a row may be here: one add a thread
            ++far;
            far_mass += f;
        } else {
            atomicAdd(&s_mass[b], (unsigned long long) f);
            atomicAdd(&s_count[b], 1u);
        }
    });
    if (far) {
        atomicAdd(&s_mass[BINS - 1], (unsigned long long) far_mass);
        atomicAdd(&s_count[BINS - 1], far);
    }
    __syncthreads();
    for (int i = tid; i < BINS; i += ST)
        if (s_count[i]) {
            atomicAdd((unsigned long long*) a.mass + (size_t) row * BINS + i, s_mass[i]);
            atomicAdd(a.count + (size_t) row * BINS + i, s_count[i]);
        }
}

// ---- sample_pick ----------------------------------------------------------------------------------------
// inclusive sums of (mass, count) over the workgroup's threads
struct Sum { uint64_t mass; uint32_t count; };
WZY_DEV Sum block_sums(Sum v, Sum* s_part) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t m = (uint64_t) __shfl_up((unsigned long long) v.mass, d);
        const uint32_t c = __shfl_up(v.count, d);
        if (lane >= d) { v.mass += m; v.count += c; }
    }
    if (lane == 63) s_part[wv] = v;
    __syncthreads();
    for (int i = 0; i < wv; ++i) {
        v.mass += s_part[i].mass;
        v.count += s_part[i].count;
    }
    __syncthreads();
    return v;
}

enum Mode { BY_COUNT, BY_MASS, BY_KEY };
// a place in the order: sums up to it, itself included, and the token there
struct Place { uint64_t mass; uint32_t count; uint64_t token; };

struct PickShared {
    uint64_t token[CAP];                                 // gathered, sorted: largest first
    uint64_t token_mass[CAP];                            // sums up to each
    uint64_t bin_mass[BINS];                             // sums up to each bin, itself included
    uint32_t bin_count[BINS];
    double table[64];
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
        for (int from = 0; from < a.vocab; from += PT * STEP) each<T, VEC, STEP>(row, from, min(from + PT * STEP, a.vocab), f);
    }
    WZY_DEV Sum before_bin(int b) const { return b > 0 ? Sum{s.bin_mass[b - 1], s.bin_count[b - 1]} : Sum{0, 0}; }

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
        int n2 = 64;
        while (n2 < n) n2 <<= 1;
        for (int i = n + tid; i < n2; i += PT) s.token[i] = 0;
        // bitonic, largest first
        for (int k = 2; k <= n2; k <<= 1)
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
            if (here) atomicMin(&s.found, i);
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
};

template <int T, bool VEC>
__global__ void __launch_bounds__(PT) sample_pick_kernel(SampleArgs a) {
    __shared__ PickShared s;
    const int row = blockIdx.x, tid = threadIdx.x;
    const float t = temp_of(a, row);
    fill_table(s.table);
    const uint64_t best = row_best<PT>(a, row, s.best);
    const bool none = (uint32_t) (best >> 32) == KEY_NONE;
    if (none || greedy(t)) {
        if (tid == 0) {
            a.ids[row] = none ? -1 : (int) ~(uint32_t) best;
            if (a.probs) a.probs[row] = none ? 0.0f : 1.0f;
        }
        return;
    }
    const Sum h = block_sums(Sum{a.mass[(size_t) row * BINS + tid], a.count[(size_t) row * BINS + tid]}, s.part);
    s.bin_mass[tid] = h.mass;
    s.bin_count[tid] = h.count;
    __syncthreads();
    Picker<T, VEC> p{a, s, row_of<T>(a, row), weight_of(a, best, t, s.table)};
    Place end{s.bin_mass[BINS - 1], s.bin_count[BINS - 1], 0};
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k >= 1 && (uint32_t) k < end.count) end = p.locate(BY_COUNT, (uint64_t) k);
    const uint64_t of_k = end.mass;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f;
    // targets: the first integer at or above share * sum; the sum itself at most
    auto share = [](double f, uint64_t sum) {
        const double x = ceil(f * (double) sum);
        const uint64_t v = x >= (double) sum ? sum : (uint64_t) x;
        return v < 1 ? (uint64_t) 1 : v;
    };
    if (top_p > 0.0f && top_p < 1.0f) {
        const Place q = p.locate(BY_MASS, share((double) top_p, of_k));
        if (q.count < end.count) end = q;
    }
    if (min_p > 1.0f) end = Place{p.w.fixed(p.w.m), 1, best};            // the first alone
    else if (min_p > 0.0f) {
        // the lowest key whose weight is min_p or more (the largest logit's, if none is): halving, every thread the same
        uint32_t hi = (uint32_t) (best >> 32), lo = KEY_NONE;             // hi passes or is the largest, lo does not
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (p.w.w(key_value(mid)) >= (double) min_p) hi = mid;
            else lo = mid;
        }
        // where the last token kept so far passes, nothing is cut
        const bool binds = end.token == 0 || (uint32_t) (end.token >> 32) < hi;
        if (binds) {
            const Place q = p.locate(BY_KEY, hi);
            if (q.count < end.count) end = q;
        }
    }
    const float u = a.u[row];
    const Place q = p.locate(BY_MASS, share(u > 0.0f ? fmin((double) u, 1.0) : 0.0, end.mass));
    if (tid == 0) {
        a.ids[row] = (int) ~(uint32_t) q.token;
        if (a.probs) a.probs[row] = (float) (ldexp(p.w.w(key_value((uint32_t) (q.token >> 32))), a.F) / (double) end.mass);
    }
}

template <int T, bool VEC>
int launch(const SampleArgs& a, void* stream) {
    const dim3 grid((unsigned) a.slices, (unsigned) a.rows);
    sample_max_kernel<T, VEC><<<grid, ST, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    sample_hist_kernel<T, VEC><<<grid, ST, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    sample_pick_kernel<T, VEC><<<a.rows, PT, 0, as_stream(stream)>>>(a);
    WZY_LAUNCH_CHECK();
    return WZY_OK;
}
constexpr int MAX_VOCAB = 1 << 22, MAX_ROWS = 65535;
size_t space(int rows, int vocab, SampleArgs* a, void* base, size_t cap) {
    const int slices = pg_div_up(vocab, SLICE);
    Arena w(base, cap);
    uint64_t* const best = w.take<uint64_t>((size_t) rows * slices);
    uint64_t* const mass = w.take<uint64_t>((size_t) rows * BINS);
    uint32_t* const count = w.take<uint32_t>((size_t) rows * BINS);
    if (a) { a->best = best; a->mass = mass; a->count = count; a->slices = slices; }
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
    a.F = 62;
    while (a.F > 40 && (int64_t) vocab > (1ll << (62 - a.F))) --a.F;
    const bool vec = (uintptr_t) logits % 16 == 0 && ld * n % 16 == 0;
    return mx_with_type(type, [&](auto t) { return vec ? launch<t(), true>(a, stream) : launch<t(), false>(a, stream); });
}
