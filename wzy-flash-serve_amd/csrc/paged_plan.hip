// paged_plan.hip -- pages, block tables, slots and attention work lists of a step of several requests.
//
//   need_r = ceil((c_r + n_r) / P) - ceil(c_r / P),   page j of them = free[n_free - 1 - (sum of need before r) - j]
//   slot of row t of request r = table[r][(c_r + i) / P] * P + (c_r + i) % P,   i = t - q_start[r]
//
// A few integers a request and a row: what bounds it is the chain from the lengths to the last slot, not bytes.  One workgroup
// of 16 waves does requests, tables and work lists: the prefix sums over requests (4 a thread: wave shifts, then the 16 waves'
// sums) stay in LDS, and everything that is counted in pages, tiles or rows is numbered through and dealt to the threads, each
// finding its request by a search in those sums, so that one long prompt does not make one thread's loop long.  Up to PLAN_ROWS
// rows the same launch fills positions and slots; more rows take a second one with a workgroup per 256 of them.
#include "wzy_paged.h"

using namespace wzy;

namespace {
constexpr int PT = 1024, PLAN_ROWS = 4096, PER = PG_MAX_REQ / PT;

struct PlanArgs {
    int* free_pages;
    const int* n_free;
    int* n_free_out;
    const int* n_cached;
    const int* n_new;
    int* table;
    int* q_start;
    int* kv_len;
    int* served;
    int* positions;
    int* slots;
    int n_pages, lp, n_req, max_tokens, max_pages, max_new;   // lp: log2(page)
    int n_works, fill_rows;
};
struct PlanWork {
    PgHead* head;
    PgLayout l;
    int g, window, geometry, per_head[2], more;
};
struct PlanWorks { PlanWork w[8]; };

WZY_DEV int div_up_log2(int v, int l) { return (int) (((uint32_t) v + (1u << l) - 1) >> l); }

// exclusive prefix sums over the workgroup's threads; total to all.  s: 17 words; a barrier before the next use is the function's own.
WZY_DEV uint64_t block_scan(uint64_t v, uint64_t* s, uint64_t& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint64_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = (uint64_t) __shfl_up((unsigned long long) x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) s[w] = x;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < PT / 64; ++i) {
        const uint64_t t = s[i];
        before += i < w ? t : 0;
        all += t;
    }
    __syncthreads();
    total = all;
    return before + x - v;
}
// the last r of 0 .. n - 1 with a[r] <= v (a ascending, a[0] = 0)
WZY_DEV int find_last(const int* a, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// a tile's cells: of its first token's window, to its last token's own
struct Tile { int row0, lo, hi; };
WZY_DEV Tile tile_of(const PlanWork& w, int kind, int j, int c, int n, bool served) {
    Tile t;
    const int rows = n * w.g;
    t.row0 = kind ? PG_WIDE * j : 0;
    const int first = (int) ((uint32_t) t.row0 / (uint32_t) w.g);
    const int last = (int) ((uint32_t) (min(t.row0 + (kind ? PG_WIDE : PG_NARROW), rows) - 1) / (uint32_t) w.g);
    t.hi = served ? c + last + 1 : 0;
    t.lo = served && w.window > 0 ? max(c + first + 1 - w.window, 0) : 0;
    return t;
}

// positions and slots of row t, from the sums in LDS
template <class F>
WZY_DEV void put_row(const PlanArgs& a, int t, const int* s_start, const int* s_cached, int total, F&& page_of) {
    int pos = 0, slot = -1;
    if (t < total) {
        const int r = find_last(s_start, a.n_req, t), c = s_cached[r];
        if (c >= 0) {                                          // served
            pos = c + t - s_start[r];
            slot = (page_of(r, pos >> a.lp) << a.lp) | (pos & ((1 << a.lp) - 1));
        }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
}

__global__ void __launch_bounds__(PT) paged_plan_kernel(PlanArgs a, PlanWorks works) {
    // by request: cached cells (top bit: not served), first row, pages taken before it, tiles before it (one list's)
    __shared__ int s_cached[PG_MAX_REQ], s_start[PG_MAX_REQ + 1], s_pages[PG_MAX_REQ], s_tiles[PG_MAX_REQ];
    __shared__ int s_item[PT], s_part[PT];                     // by tile of a pass: items and parts before it
    __shared__ uint64_t s_scan[PT / 64 + 1];
    const int tid = threadIdx.x;
    const int n_free = min(max(*a.n_free, 0), a.n_pages);
    // requests PER * tid .. : rows, then pages
    int c[PER], n[PER], need[PER];
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        c[i] = r < a.n_req ? max(a.n_cached[r], 0) : 0;
        n[i] = r < a.n_req ? max(a.n_new[r], 0) : 0;
        sum += n[i];
    }
    uint64_t total;
    int64_t start = (int64_t) block_scan((uint64_t) sum, s_scan, total);
    const int rows_total = (int) min((int64_t) total, (int64_t) a.max_tokens);
    int64_t pages = 0;
    bool ok[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        const int64_t cells = (int64_t) c[i] + n[i];
        // c and n below 2^24 where the request fits; the others are not served, and their cells are not counted
        ok[i] = r < a.n_req && cells <= (int64_t) a.max_pages << a.lp && n[i] <= a.max_new && (n[i] == 0 || start + n[i] <= a.max_tokens);
        need[i] = ok[i] ? div_up_log2((int) cells, a.lp) - div_up_log2(c[i], a.lp) : 0;
        if (r < a.n_req) s_start[r] = (int) min(start, (int64_t) a.max_tokens);
        start += n[i];
        pages += need[i];
    }
    int64_t before = (int64_t) block_scan((uint64_t) pages, s_scan, total);
    int64_t taken = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        const bool fits = need[i] == 0 || before + need[i] <= n_free;
        ok[i] = ok[i] && fits;
        if (r < a.n_req) {
            s_pages[r] = (int) min(before, (int64_t) n_free);
            s_cached[r] = ok[i] ? c[i] : (int) ((uint32_t) c[i] | 0x80000000u);
            a.served[r] = ok[i] ? 1 : 0;
            a.kv_len[r] = ok[i] ? c[i] + n[i] : 0;
            a.q_start[r] = s_start[r];
        }
        before += need[i];
        taken += ok[i] ? need[i] : 0;
    }
    block_scan((uint64_t) taken, s_scan, total);               // those served are the first that need any
    const int n_taken = (int) total;
    if (tid == 0) {
        s_start[a.n_req] = rows_total;
        a.q_start[a.n_req] = rows_total;
        *a.n_free_out = n_free - n_taken;
    }
    __syncthreads();
    // pages into the table.  Page ids are limited, so that a slot is always one of the cache's.
    auto pool = [&](int i) { return min(max(a.free_pages[n_free - 1 - i], 0), a.n_pages - 1); };
    for (int i = tid; i < n_taken; i += PT) {
        const int r = find_last(s_pages, a.n_req, i);
        a.table[(size_t) r * a.max_pages + div_up_log2(s_cached[r], a.lp) + i - s_pages[r]] = pool(i);
    }
    if (a.fill_rows)
        for (int t = tid; t < a.max_tokens; t += PT)
            put_row(a, t, s_start, s_cached, rows_total, [&](int r, int p) {
                const int held = div_up_log2(s_cached[r], a.lp);
                return p < held ? min(max(a.table[(size_t) r * a.max_pages + p], 0), a.n_pages - 1) : pool(s_pages[r] + p - held);
            });

    for (int i = 0; i < a.n_works; ++i) {
        const PlanWork& w = works.w[i];
        PgItem* const items = (PgItem*) (w.head + 1);
        for (int kind = 0; kind < 2; ++kind) {
            // tiles before each request.  A request that is not served has one narrow tile without cells, whatever its rows:
            // they become 0.
            int tiles[PER], mine = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int r = PER * tid + j;
                // its rows, as far as there are any
                const int rows = r < a.n_req ? (s_start[r + 1] - s_start[r]) * w.g : 0;
                const bool narrow = rows <= PG_NARROW || !ok[j];
                tiles[j] = rows == 0 ? 0 : kind == 0 ? (narrow ? 1 : 0) : narrow ? 0 : (rows + PG_WIDE - 1) / PG_WIDE;
                mine += tiles[j];
            }
            int at = (int) block_scan((uint64_t) mine, s_scan, total);
            const int n_tiles = (int) total;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int r = PER * tid + j;
                if (r < a.n_req) s_tiles[r] = at;
                at += tiles[j];
            }
            __syncthreads();
            // a request's last tile sees the most cells and comes first
            auto tile_at = [&](int t, int& r) {
                r = find_last(s_tiles, a.n_req, t);
                const int end = r + 1 < a.n_req ? s_tiles[r + 1] : n_tiles;
                const int cc = s_cached[r];
                return tile_of(w, kind, end - 1 - t, cc & 0x7FFFFFFF, s_start[r + 1] - s_start[r], cc >= 0);
            };
            uint64_t cells = 0;
            for (int t = tid; t < n_tiles; t += PT) {
                int r;
                const Tile x = tile_at(t, r);
                cells += (uint64_t) (x.hi - (x.lo & ~31));
            }
            block_scan(cells, s_scan, total);
            // parts of at most len cells (a multiple of 32): at most per_head of them, and one more a tile
            // few tiles: together with a tile's own last part they are what the chip holds at once
            const int slots = w.per_head[kind];
            const uint32_t per_head = (uint32_t) (4 * n_tiles <= slots ? slots - n_tiles : slots + (kind ? 0 : min(n_tiles, w.more)));
            uint64_t len = (total + per_head - 1) / per_head;
            len = (len + 31) & ~(uint64_t) 31;
            const int part = (int) max(len, (uint64_t) w.l.min_len[kind]);
            int n_items = 0, n_parts = 0, n_merges = 0;
            for (int base = 0; base < n_tiles; base += PT) {
                const int t = base + tid, here = min(n_tiles - base, PT);
                int r = 0, k = 0;
                Tile x{};
                if (t < n_tiles) {
                    x = tile_at(t, r);
                    k = max(1, (x.hi - (x.lo & ~31) + part - 1) / part);
                }
                const uint64_t v = (uint64_t) k | (uint64_t) (k > 1 ? k : 0) << 24 | (uint64_t) (k > 1 ? 1 : 0) << 48;
                const uint64_t p = block_scan(v, s_scan, total);
                const int pt = n_parts + (int) (p >> 24 & 0xFFFFFF), me = n_merges + (int) (p >> 48);
                s_item[tid] = (int) (p & 0xFFFFFF);
                s_part[tid] = k > 1 ? pt : -1;
                if (k > 1 && me < w.l.merges[kind])
                    ((PgMerge*) items)[w.l.merge_at[kind] + me] =
                        PgMerge{pt, k, s_start[r], x.row0, min((s_start[r + 1] - s_start[r]) * w.g - x.row0, kind ? PG_WIDE : PG_NARROW), {0, 0, 0}};
                __syncthreads();
                const int n = (int) (total & 0xFFFFFF);
                for (int i = tid; i < n && n_items + i < w.l.items[kind]; i += PT) {
                    const int o = find_last(s_item, here, i), j = i - s_item[o];
                    const Tile y = tile_at(base + o, r);
                    // a tile's parts are of one length, but for the blocks of 32 cells
                    const int parts = (o + 1 < here ? s_item[o + 1] : n) - s_item[o], first = y.lo >> 5, blocks = ((y.hi + 31) >> 5) - first;
                    const int from = 32 * (first + (int) ((int64_t) blocks * j / parts)), to = 32 * (first + (int) ((int64_t) blocks * (j + 1) / parts));
                    items[w.l.item_at[kind] + n_items + i] = PgItem{r, y.row0, max(y.lo, from), min(y.hi, to), s_part[o] < 0 ? -1 : s_part[o] + j,
                                                                    s_start[r], s_start[r + 1] - s_start[r], s_cached[r] & 0x7FFFFFFF};
                }
                n_items += n;
                n_parts += (int) (total >> 24 & 0xFFFFFF);
                n_merges += (int) (total >> 48);
            }
            if (tid == 0) {
                w.head->n_items[kind] = min(n_items, w.l.items[kind]);
                w.head->n_merges[kind] = min(n_merges, w.l.merges[kind]);
                if (kind == 0) {
                    w.head->magic = PG_MAGIC;
                    w.head->geometry = w.geometry;
                }
            }
        }
    }
}

// rows of larger steps: the table and q_start are as the plan left them
__global__ void __launch_bounds__(256) paged_rows_kernel(PlanArgs a) {
    __shared__ int s_start[PG_MAX_REQ + 1], s_cached[PG_MAX_REQ];
    for (int r = threadIdx.x; r < a.n_req; r += 256) {
        const int c = max(a.n_cached[r], 0);
        s_start[r] = a.q_start[r];
        s_cached[r] = a.served[r] ? c : (int) ((uint32_t) c | 0x80000000u);
    }
    __syncthreads();
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.max_tokens) return;
    put_row(a, t, s_start, s_cached, a.q_start[a.n_req],
            [&](int r, int p) { return min(max(a.table[(size_t) r * a.max_pages + p], 0), a.n_pages - 1); });
}

// One workgroup: pages to push are counted a request, summed over requests, and numbered through.
__global__ void __launch_bounds__(PT) paged_release_kernel(PlanArgs a, const int* __restrict__ ended) {
    __shared__ int s_pages[PG_MAX_REQ + 1];
    __shared__ uint64_t s_scan[PT / 64 + 1];
    const int tid = threadIdx.x, n_free = min(max(*a.n_free, 0), a.n_pages);
    int held[PER];
    uint64_t sum = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        held[i] = 0;
        if (r < a.n_req && ended[r]) held[i] = min(div_up_log2(max(a.n_cached[r], 0), a.lp), a.max_pages);
        sum += (uint64_t) held[i];
    }
    uint64_t at = block_scan(sum, s_scan, total);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        if (r < a.n_req) s_pages[r] = (int) at;
        at += (uint64_t) held[i];
    }
    __syncthreads();
    const int n = (int) total;
    int n_out = n_free;
    for (int base = 0; base < n; base += PT) {
        const int i = base + tid;
        int id = -1;
        if (i < n) {
            const int r = find_last(s_pages, a.n_req, i);
            int* const e = a.table + (size_t) r * a.max_pages + i - s_pages[r];
            id = *e;
            *e = -1;
        }
        const bool ok = id >= 0 && id < a.n_pages;
        const int to = n_out + (int) block_scan(ok ? 1 : 0, s_scan, total);
        if (ok && to < a.n_pages) a.free_pages[to] = id;
        n_out = (int) min((int64_t) n_out + (int64_t) total, (int64_t) a.n_pages);
    }
    if (tid == 0) *a.n_free_out = n_out;
}

int check_pool(const char* who, const wzy_paged_pool* p) {
    WZY_REQUIRE(p && p->free_pages && p->n_free && p->n_free_out, "%s: pool is null", who);
    WZY_REQUIRE(pg_page_ok(p->n_pages, p->page), "%s: %d pages of %d cells", who, p->n_pages, p->page);
    return WZY_OK;
}
}  // namespace

// The list's room does not depend on the page: any table has at most PG_MAX_CELLS cells, and a smaller one's bound is not
// needed where the parts are limited by their number.
static PgLayout layout_of(const wzy_paged_batch* b, const wzy_paged_work* w) {
    return pg_layout(b->n_req, b->max_tokens, pg_max_new(b), PG_MAX_CELLS, w);
}
namespace wzy {
PgLayout pg_layout_of(const wzy_paged_batch* b, const wzy_paged_work* w) { return layout_of(b, w); }
}

extern "C" size_t wzy_paged_work_bytes(const wzy_paged_batch* b, const wzy_paged_work* w) {
    if (pg_check_batch("wzy_paged_work_bytes", b, 1) != WZY_OK || pg_check_work("wzy_paged_work_bytes", w) != WZY_OK) return 0;
    return sizeof(PgHead) + sizeof(PgItem) * (size_t) layout_of(b, w).total;
}

extern "C" int wzy_paged_plan(const wzy_paged_pool* pool, const wzy_paged_batch* b, const wzy_paged_work* works, int n_works,
                              void* stream) {
    const char* const who = "wzy_paged_plan";
    WZY_TRY(check_pool(who, pool));
    WZY_TRY(pg_check_batch(who, b, pool->page));
    WZY_REQUIRE(b->n_cached && b->n_new && b->table && b->q_start && b->kv_len && b->served && b->positions && b->slots,
                "%s: an array of the batch is null", who);
    WZY_REQUIRE(n_works >= 0 && n_works <= 8 && (n_works == 0 || works), "%s: %d work lists (0 .. 8)", who, n_works);
    PlanWorks pw{};
    for (int i = 0; i < n_works; ++i) {
        const wzy_paged_work* const w = works + i;
        WZY_TRY(pg_check_work(who, w));
        const PgLayout l = layout_of(b, w);
        const size_t want = sizeof(PgHead) + sizeof(PgItem) * (size_t) l.total;
        WZY_REQUIRE(w->items && (uintptr_t) w->items % 16 == 0 && w->bytes >= want, "%s: work list %d: %zu bytes at %p (%zu, 16-byte aligned)",
                    who, i, w->bytes, w->items, want);
        for (int j = 0; j < i; ++j) WZY_REQUIRE(works[j].items != w->items, "%s: work lists %d and %d are one", who, j, i);
        pw.w[i] = PlanWork{(PgHead*) w->items, l, w->qh / w->kvh, w->window, pg_geometry(w),
                           {pg_div_up(pg_parts(0, w->hd), w->kvh), pg_div_up(pg_parts(1, w->hd), w->kvh)}, PG_MORE / w->kvh};
    }
    PlanArgs a{pool->free_pages, pool->n_free, pool->n_free_out, b->n_cached, b->n_new, b->table, b->q_start, b->kv_len, b->served,
               b->positions, b->slots, pool->n_pages, pg_log2(pool->page), b->n_req, b->max_tokens, b->max_pages, pg_max_new(b), n_works,
               b->max_tokens <= PLAN_ROWS};
    paged_plan_kernel<<<1, PT, 0, as_stream(stream)>>>(a, pw);
    WZY_LAUNCH_CHECK();
    if (!a.fill_rows) {
        paged_rows_kernel<<<pg_div_up(b->max_tokens, 256), 256, 0, as_stream(stream)>>>(a);
        WZY_LAUNCH_CHECK();
    }
    return WZY_OK;
}

extern "C" int wzy_paged_release(const wzy_paged_pool* pool, const wzy_paged_batch* b, const int* ended, void* stream) {
    const char* const who = "wzy_paged_release";
    WZY_TRY(check_pool(who, pool));
    WZY_REQUIRE(b && b->n_req >= 1 && b->n_req <= PG_MAX_REQ, "%s: requests (1 .. %d)", who, PG_MAX_REQ);
    WZY_REQUIRE(b->max_pages >= 1 && (int64_t) b->max_pages * pool->page <= PG_MAX_CELLS, "%s: max_pages %d", who, b->max_pages);
    WZY_REQUIRE(b->n_cached && b->table && ended, "%s: an array is null", who);
    PlanArgs a{};
    a.free_pages = pool->free_pages; a.n_free = pool->n_free; a.n_free_out = pool->n_free_out; a.n_cached = b->n_cached; a.table = b->table;
    a.n_pages = pool->n_pages; a.lp = pg_log2(pool->page); a.n_req = b->n_req; a.max_pages = b->max_pages;
    paged_release_kernel<<<1, PT, 0, as_stream(stream)>>>(a, ended);
    WZY_LAUNCH_CHECK();
    return WZY_OK;
}
