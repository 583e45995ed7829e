// paged_plan.hip -- pages, block tables, slots and attention work lists of a step of several requests.
//
//   need_r = ceil((c_r + n_r) / P) - ceil(c_r / P),   page j of them = free[n_free - 1 - (sum of need before r) - j]
//   slot of row t of request r = table[r][(c_r + i) / P] * P + (c_r + i) % P,   i = t - q_start[r]
//
// A few integers a request and a row: what bounds it is the chain from the lengths to the last slot, not bytes.  One workgroup
// of 16 waves (4 for up to 256 requests and rows) does requests, tables and work lists: the prefix sums over requests (4 a thread: wave shifts, then the 16 waves'
// sums) stay in LDS, and everything that is counted in pages, parts or rows is numbered through and dealt to the threads, each
// finding its request by a search in those sums, so that one long prompt does not make one thread's loop long.  Up to PLAN_ROWS
// rows the same launch fills positions, slots and work lists; more rows take a second one with a workgroup per 256 of them.
// 8 requests' next tokens, one list: 6.6 us.  1,000 requests with 24,000 rows of prompts: 6.8 us and 6.1 us.  Release is one workgroup
// too, its pages numbered through: 8 requests of 512 pages each 4 us, 125 of 300 pages (of 1,000 requests) 51, all 1,000 of them 390.
#include "wzy_paged.h"

using namespace wzy;

namespace {
constexpr int PT = 1024, PLAN_ROWS = 4096;

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

// sums of lanes 0 .. l: within 16-lane rows by shifts, then the rows' last lanes on to the next rows
template <int CTRL, int ROWMASK>
WZY_DEV int add_dpp(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWMASK, 0xF, true); }
WZY_DEV int prefix_sum(int v) {
    v = add_dpp<0x111, 0xF>(v);                                    // row_shr 1, 2, 4, 8
    v = add_dpp<0x112, 0xF>(v);
    v = add_dpp<0x114, 0xF>(v);
    v = add_dpp<0x118, 0xF>(v);
    v = add_dpp<DPP_ROW_BCAST15, 0xA>(v);
    return add_dpp<DPP_ROW_BCAST31, 0xC>(v);
}
// N exclusive prefix sums over the workgroup's NT threads at once, v in and out; the totals to all.  Sums below 2^31.
template <int NT, int N>
WZY_DEV void block_scan(int (&v)[N], int (*s)[NT / 64], int (&total)[N]) {
    constexpr int NW = NT / 64;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = prefix_sum(v[i]);
        if (lane == 63) s[i][w] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int t = prefix_sum(lane < NW ? s[i][lane & (NW - 1)] : 0);
        total[i] = __builtin_amdgcn_readlane(t, NW - 1);
        v[i] = x[i] - v[i] + (w > 0 ? __builtin_amdgcn_readlane(t, w > 0 ? w - 1 : 0) : 0);
    }
    __syncthreads();
}
// the last r of 0 .. n - 1 with a(r) <= v (a ascending, a(0) = 0)
template <class F>
WZY_DEV int find_last_of(int n, int v, F&& a) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a(mid) <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}
WZY_DEV int find_last(const int* a, int n, int v) {
    return find_last_of(n, v, [&](int r) { return a[r]; });
}

// A request in one list: its tiles, and the parts each is cut into.  A request that is not served has one narrow tile without
// cells, whatever its rows: they become 0.
struct Cut { int kind, tiles, parts, blocks; };
WZY_DEV Cut cut_of(const PlanWork& w, int c, int n, bool served, const int (&part)[2]) {
    Cut x;
    const int rows = n * w.g;
    x.kind = rows <= w.l.narrow || !served ? 0 : 1;
    x.tiles = rows == 0 ? 0 : x.kind ? (rows + PG_WIDE - 1) / PG_WIDE : 1;
    // blocks of 32 cells that a tile sees: of a narrow one, which is its request's only one, just so many; of a wide one at most, the
    // last one's end or as many as its tokens' windows span
    x.blocks = served ? (c + n + 31) >> 5 : 0;
    if (w.window > 0 && served)
        x.blocks = x.kind ? min(x.blocks, ((w.window + (int) ((uint32_t) PG_WIDE / (uint32_t) w.g)) >> 5) + 2) : x.blocks - (max(c + 1 - w.window, 0) >> 5);
    const int p = part[x.kind];
    x.parts = p > 0 && x.blocks > p ? (x.blocks + p - 1) / p : 1;
    return x;
}
// item i of a kind, which is the request's i - before.items[kind]-th, and with a tile's first part its merge entry
WZY_DEV void put_item(const PlanWork& w, int kind, int i, int r, const PgBefore& before, int c, int n, bool served, int q0, const int (&part)[2]) {
    const Cut x = cut_of(w, c, n, served, part);
    const int j = i - before.items[kind], tile = (int) ((uint32_t) j / (uint32_t) x.parts), k = j - tile * x.parts, rows = n * w.g;
    // a request's last tile sees the most cells and comes first
    const int row0 = kind ? PG_WIDE * (x.tiles - 1 - tile) : 0, row1 = min(row0 + (kind ? PG_WIDE : w.l.narrow), rows);
    const int hi = served ? c + (int) ((uint32_t) (row1 - 1) / (uint32_t) w.g) + 1 : 0;
    const int lo = served && w.window > 0 ? max(c + (int) ((uint32_t) row0 / (uint32_t) w.g) + 1 - w.window, 0) : 0;
    // parts of one length, but for the blocks of 32 cells
    const int first = lo >> 5, blocks = ((hi + 31) >> 5) - first;
    // (below 2^32: 2^19 blocks, and parts are at most pg_parts() + PG_MORE)
    const uint32_t nb = (uint32_t) blocks, np = (uint32_t) x.parts;
    const int from = 32 * (first + (int) (nb * (uint32_t) k / np)), to = 32 * (first + (int) (nb * (uint32_t) (k + 1) / np));
    const int pt = before.parts + tile * x.parts;
    PgItem* const items = (PgItem*) (w.head + 1);
    if (i >= w.l.items[kind] || (x.parts > 1 && pt + x.parts > w.l.parts[kind])) return;
    items[w.l.item_at[kind] + i] = PgItem{r, row0, max(lo, from), min(hi, to), x.parts > 1 ? pt + k : -1, q0, n, c};
    if (x.parts > 1 && k == 0 && before.merges + tile < w.l.merges[kind])
        ((PgMerge*) items)[w.l.merge_at[kind] + before.merges + tile] = PgMerge{pt, x.parts, q0, row0, row1 - row0, {0, 0, 0}};
}

// positions and slots of row t, from the sums in LDS
template <class F>
WZY_DEV void put_row(const PlanArgs& a, int t, const int* s_start, const int* s_cached, int total, F&& page_of) {
    int pos = 0, slot = -1;
    if (t < total) {
        const int r = find_last(s_start, a.n_req, t), c = s_cached[r];
        if (c >= 0) {                                          // served
            pos = c + t - s_start[r];
            const int page = page_of(r, pos >> a.lp);
            if ((unsigned) page < (unsigned) a.n_pages) slot = (page << a.lp) | (pos & ((1 << a.lp) - 1));
        }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
}

template <int NT, int PER>
__global__ void __launch_bounds__(NT) paged_plan_kernel(PlanArgs a, PlanWorks works) {
    constexpr int REQ = NT * PER;
    // by request: cached cells (top bit: not served), first row, pages taken before it, what is before it in a list
    __shared__ int s_cached[REQ], s_start[REQ + 1], s_pages[REQ];
    __shared__ PgBefore s_before[REQ];
    __shared__ int s_scan[6][NT / 64];
    const int tid = threadIdx.x;
    const int n_free = min(max(*a.n_free, 0), a.n_pages);
    // requests PER * tid .. : rows.  A thread's are counted up to one more than there is room for, so that sums stay in 32 bits.
    int c[PER], n[PER], sum = 0, v1[1], t1[1];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        c[i] = r < a.n_req ? max(a.n_cached[r], 0) : 0;
        n[i] = r < a.n_req ? min(max(a.n_new[r], 0), a.max_tokens + 1) : 0;
        sum = min(sum + n[i], a.max_tokens + 1);
    }
    v1[0] = sum;
    block_scan<NT>(v1, s_scan, t1);
    const int rows_total = min(t1[0], a.max_tokens);
    int start = v1[0], need[PER];
    bool ok[PER];
    v1[0] = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        // where the request fits, its cells are at most 2^24
        ok[i] = r < a.n_req && (int64_t) c[i] + n[i] <= (int64_t) a.max_pages << a.lp && n[i] <= a.max_new && (n[i] == 0 || start + n[i] <= a.max_tokens);
        need[i] = ok[i] ? div_up_log2(c[i] + n[i], a.lp) - div_up_log2(c[i], a.lp) : 0;
        if (r < a.n_req) s_start[r] = min(start, a.max_tokens);
        start = min(start + n[i], 1 << 30);
        v1[0] += need[i];
    }
    block_scan<NT>(v1, s_scan, t1);
    int before = v1[0], taken[1] = {0}, n_taken[1];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        ok[i] = ok[i] && (need[i] == 0 || before + need[i] <= n_free);
        if (r < a.n_req) {
            s_pages[r] = min(before, n_free);
            s_cached[r] = ok[i] ? c[i] : (int) ((uint32_t) c[i] | 0x80000000u);
            a.served[r] = ok[i] ? 1 : 0;
            a.kv_len[r] = ok[i] ? c[i] + n[i] : 0;
            a.q_start[r] = s_start[r];
        }
        before += need[i];
        taken[0] += ok[i] ? need[i] : 0;
    }
    if (tid == 0) {
        s_start[a.n_req] = rows_total;
        a.q_start[a.n_req] = rows_total;
    }
    block_scan<NT>(taken, s_scan, n_taken);                    // those served are the first that need any
    if (tid == 0) *a.n_free_out = n_free - n_taken[0];
    // pages into the table
    auto pool = [&](int i) { return a.free_pages[n_free - 1 - i]; };
    for (int i = tid; i < n_taken[0]; i += NT) {
        const int r = find_last(s_pages, a.n_req, i);
        a.table[(size_t) r * a.max_pages + div_up_log2(s_cached[r], a.lp) + i - s_pages[r]] = pool(i);
    }
    if (a.fill_rows)
        for (int t = tid; t < a.max_tokens; t += NT)
            put_row(a, t, s_start, s_cached, rows_total, [&](int r, int p) {
                const int held = div_up_log2(s_cached[r], a.lp);
                return p < held ? a.table[(size_t) r * a.max_pages + p] : pool(s_pages[r] + p - held);
            });

    for (int i = 0; i < a.n_works; ++i) {
        const PlanWork& w = works.w[i];
        // the longest parts: tiles, and blocks of all tiles (in two halves, so that sums stay in 32 bits)
        int part[2] = {0, 0}, v[6] = {0, 0, 0, 0, 0, 0}, sums[6];
        int64_t blocks[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = PER * tid + j;
            if (r < a.n_req) {
                const Cut x = cut_of(w, c[j], s_start[r + 1] - s_start[r], ok[j], part);
                v[x.kind] += x.tiles;
                blocks[x.kind] += (int64_t) x.tiles * x.blocks;
            }
        }
        v[2] = (int) (blocks[0] >> 16); v[3] = (int) (blocks[0] & 0xFFFF);
        v[4] = (int) (blocks[1] >> 16); v[5] = (int) (blocks[1] & 0xFFFF);
        block_scan<NT>(v, s_scan, sums);
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            // at most per_head parts of that length, and one more a tile; few tiles: together with a tile's own last part they are what
            // the chip holds at once
            const int64_t all = ((int64_t) sums[2 + 2 * kind] << 16) + sums[3 + 2 * kind];
            const int slots = w.per_head[kind], nt = sums[kind];
            const int per_head = 4 * nt <= slots ? slots - nt : slots + (kind ? 0 : min(nt, w.more));
            // (at most all blocks of the longest request: the quotient may pass 31 bits)
            part[kind] = max((int) fmin(ceil((double) all / (double) per_head), PG_MAX_CELLS / 32), w.l.min_len[kind] / 32);
        }
        // items, parts and merges before each request
        Cut x[PER];
#pragma unroll
        for (int j = 0; j < 6; ++j) v[j] = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = PER * tid + j;
            x[j] = r < a.n_req ? cut_of(w, c[j], s_start[r + 1] - s_start[r], ok[j], part) : Cut{0, 0, 1, 0};
            const int k = x[j].kind, its = x[j].tiles * x[j].parts;
            v[k] += its;
            if (x[j].parts > 1) {
                v[2 + 2 * k] += its;
                v[3 + 2 * k] += x[j].tiles;
            }
        }
        block_scan<NT>(v, s_scan, sums);
        PgBefore* const out = (PgBefore*) ((PgItem*) (w.head + 1) + w.l.before_at);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = PER * tid + j, k = x[j].kind, its = x[j].tiles * x[j].parts;
            if (r < a.n_req) {
                const PgBefore b{{v[0], v[1]}, v[2 + 2 * k], v[3 + 2 * k]};
                if (a.fill_rows) s_before[r] = b;
                else out[r] = b;
            }
            v[k] += its;
            if (x[j].parts > 1) {
                v[2 + 2 * k] += its;
                v[3 + 2 * k] += x[j].tiles;
            }
        }
        if (tid == 0) *w.head = PgHead{PG_MAGIC, w.geometry, {min(sums[0], w.l.items[0]), min(sums[1], w.l.items[1])},
                                       {min(sums[3], w.l.merges[0]), min(sums[5], w.l.merges[1])}, {part[0], part[1]}, {}};
        if (!a.fill_rows) continue;
        __syncthreads();
        for (int j = tid; j < sums[0] + sums[1]; j += NT) {
            const int kind = j < sums[0] ? 0 : 1, it = j - (kind ? sums[0] : 0);
            const int r = find_last_of(a.n_req, it, [&](int q) { return s_before[q].items[kind]; });
            const int cc = s_cached[r];
            put_item(w, kind, it, r, s_before[r], cc & 0x7FFFFFFF, s_start[r + 1] - s_start[r], cc >= 0, s_start[r], part);
        }
        __syncthreads();
    }
}

// Rows and work lists of larger steps, a workgroup per 256 of them: the table, q_start and the sums are as the plan left them.
struct RowBlocks { int at[9]; };                               // first workgroup of each list; those before are rows'
__global__ void __launch_bounds__(256) paged_rows_kernel(PlanArgs a, PlanWorks works, RowBlocks blocks) {
    __shared__ int s_start[PG_MAX_REQ + 1], s_cached[PG_MAX_REQ], s_items[2][PG_MAX_REQ];
    const int block = blockIdx.x;
    int list = -1;
    while (list + 1 < a.n_works && block >= blocks.at[list + 1]) ++list;
    const PgBefore* before = nullptr;
    if (list >= 0) before = (const PgBefore*) ((const PgItem*) (works.w[list].head + 1) + works.w[list].l.before_at);
    for (int r = threadIdx.x; r < a.n_req; r += 256) {
        const int c = max(a.n_cached[r], 0);
        s_start[r] = a.q_start[r];
        s_cached[r] = a.served[r] ? c : (int) ((uint32_t) c | 0x80000000u);
        if (list >= 0) {
            const PgBefore b = before[r];
            s_items[0][r] = b.items[0];
            s_items[1][r] = b.items[1];
        }
    }
    if (threadIdx.x == 0) s_start[a.n_req] = a.q_start[a.n_req];
    __syncthreads();
    if (list < 0) {
        const int t = block * 256 + threadIdx.x;
        if (t < a.max_tokens)
            put_row(a, t, s_start, s_cached, s_start[a.n_req],
                    [&](int r, int p) { return a.table[(size_t) r * a.max_pages + p]; });
        return;
    }
    const PlanWork& w = works.w[list];
    const PgHead h = *w.head;
    const int part[2] = {h.part[0], h.part[1]}, j = (block - blocks.at[list]) * 256 + (int) threadIdx.x;
    if (j >= h.n_items[0] + h.n_items[1]) return;
    const int kind = j < h.n_items[0] ? 0 : 1, it = j - (kind ? h.n_items[0] : 0), r = find_last(s_items[kind], a.n_req, it), cc = s_cached[r];
    put_item(w, kind, it, r, before[r], cc & 0x7FFFFFFF, s_start[r + 1] - s_start[r], cc >= 0, s_start[r], part);
}

// One workgroup: pages to push are counted a request, summed over requests, and numbered through.
__global__ void __launch_bounds__(PT) paged_release_kernel(PlanArgs a, const int* __restrict__ ended) {
    constexpr int PER = PG_MAX_REQ / PT;
    __shared__ int s_pages[PG_MAX_REQ];
    __shared__ int s_scan[1][PT / 64];
    const int tid = threadIdx.x, n_free = min(max(*a.n_free, 0), a.n_pages);
    int held[PER], at[1] = {0}, n[1];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        held[i] = r < a.n_req && ended[r] ? min(div_up_log2(max(a.n_cached[r], 0), a.lp), a.max_pages) : 0;
        at[0] += held[i];                                      // the table has fewer than 2^31 entries
    }
    block_scan<PT>(at, s_scan, n);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = PER * tid + i;
        if (r < a.n_req) s_pages[r] = at[0];
        at[0] += held[i];
    }
    __syncthreads();
    int n_out = n_free;
    for (int base = 0; base < n[0]; base += PT) {
        const int i = base + tid;
        int id = -1;
        if (i < n[0]) {
            const int r = find_last(s_pages, a.n_req, i);
            int* const e = a.table + (size_t) r * a.max_pages + i - s_pages[r];
            id = *e;
            *e = -1;
        }
        const bool ok = id >= 0 && id < a.n_pages;
        int v[1] = {ok ? 1 : 0}, all[1];
        block_scan<PT>(v, s_scan, all);
        const int to = n_out + v[0];
        if (ok && to < a.n_pages) a.free_pages[to] = id;
        n_out = min(n_out + all[0], a.n_pages);
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
    const char* const who = "wzy_paged_work_bytes";
    if (pg_check_batch(who, b, 1) != WZY_OK || pg_check_work(who, w) != WZY_OK) return 0;
    const PgLayout l = layout_of(b, w);
    return pg_check_launch(who, b, w, l) == WZY_OK ? sizeof(PgHead) + sizeof(PgItem) * (size_t) l.total : 0;
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
        WZY_TRY(pg_check_launch(who, b, w, l));
        const size_t want = sizeof(PgHead) + sizeof(PgItem) * (size_t) l.total;
        WZY_REQUIRE(w->items && (uintptr_t) w->items % 16 == 0 && w->bytes >= want, "%s: work list %d: %zu bytes at %p (%zu, 16-byte aligned)",
                    who, i, w->bytes, w->items, want);
        for (int j = 0; j < i; ++j) WZY_REQUIRE(works[j].items != w->items, "%s: work lists %d and %d are one", who, j, i);
        pw.w[i] = PlanWork{(PgHead*) w->items, l, w->qh / w->kvh, pg_window(w), pg_geometry(w, l),
                           {pg_div_up(pg_parts(0, l.narrow, w->hd), w->kvh), pg_div_up(pg_parts(1, l.narrow, w->hd), w->kvh)}, PG_MORE / w->kvh};
    }
    PlanArgs a{pool->free_pages, pool->n_free, pool->n_free_out, b->n_cached, b->n_new, b->table, b->q_start, b->kv_len, b->served,
               b->positions, b->slots, pool->n_pages, pg_log2(pool->page), b->n_req, b->max_tokens, b->max_pages, pg_max_new(b), n_works,
               b->max_tokens <= PLAN_ROWS};
    // few requests and rows: fewer waves to bring together
    const auto st = as_stream(stream);
    if (b->n_req <= 256 && b->max_tokens <= 256) paged_plan_kernel<256, 1><<<1, 256, 0, st>>>(a, pw);
    else if (b->n_req <= 1024) paged_plan_kernel<1024, 1><<<1, 1024, 0, st>>>(a, pw);
    else paged_plan_kernel<1024, 4><<<1, 1024, 0, st>>>(a, pw);
    WZY_LAUNCH_CHECK();
    if (!a.fill_rows) {
        RowBlocks rb{};
        int at = pg_div_up(b->max_tokens, 256);
        for (int i = 0; i < n_works; ++i) {
            rb.at[i] = at;
            at += pg_div_up((int64_t) pw.w[i].l.items[0] + pw.w[i].l.items[1], 256);
        }
        paged_rows_kernel<<<at, 256, 0, st>>>(a, pw, rb);
        WZY_LAUNCH_CHECK();
    }
    return WZY_OK;
}

extern "C" int wzy_paged_release(const wzy_paged_pool* pool, const wzy_paged_batch* b, const int* ended, void* stream) {
    const char* const who = "wzy_paged_release";
    WZY_TRY(check_pool(who, pool));
    WZY_REQUIRE(b && b->n_req >= 1 && b->n_req <= PG_MAX_REQ, "%s: requests (1 .. %d)", who, PG_MAX_REQ);
    WZY_REQUIRE(b->max_pages >= 1 && (int64_t) b->max_pages * pool->page <= PG_MAX_CELLS && (int64_t) b->max_pages * b->n_req < 1ll << 31,
                "%s: max_pages %d", who, b->max_pages);
    WZY_REQUIRE(b->n_cached && b->table && ended, "%s: an array is null", who);
    PlanArgs a{};
    a.free_pages = pool->free_pages; a.n_free = pool->n_free; a.n_free_out = pool->n_free_out; a.n_cached = b->n_cached; a.table = b->table;
    a.n_pages = pool->n_pages; a.lp = pg_log2(pool->page); a.n_req = b->n_req; a.max_pages = b->max_pages;
    paged_release_kernel<<<1, PT, 0, as_stream(stream)>>>(a, ended);
    WZY_LAUNCH_CHECK();
    return WZY_OK;
}
