// wzy_paged.h -- shared by the paged-cache kernels: the work lists of an attention layer, host checks.
#pragma once
#include "../../include/wzy_paged.h"
#include "wzy_device.h"
#include "wzy_host.h"
#include "wzy_mx.h"

namespace wzy {

// ---- work lists ---------------------------------------------------------------------------------------
// The rows of one request and key head are its (token, head of the group) pairs, token-major: row m is token m / g, head
// m % g, g = qh / kvh.  They are cut into tiles: requests of up to 32 rows are one narrow tile (of up to 64, in steps where
// no request has more), others have wide tiles of PG_WIDE rows.  A tile's cells (from the first that its first token sees to
// its last token's own) are cut into parts of equal length where the tiles alone do not fill the chip, all tiles of a request
// into as many as its longest needs; parts leave partial results in the workspace, and a merge entry says which belong
// together.  The same list serves every key head.
constexpr int PG_WIDE = 128;
constexpr int PG_MAX_REQ = 4096, PG_MAX_TOKENS = 1 << 20, PG_MAX_CELLS = 1 << 24;
// Parts that a step is cut into, over all key heads, and of narrow tiles one more a tile, as far as PG_MORE, so that requests of
// different lengths come out even.  Narrow: as many workgroups as the chip holds at once by their LDS, 4, 2 or 1 a CU.  Middle: 3 a CU, of
// heads of 256 the 2 that their registers allow (4 x 12 tokens over 20,000 cells, 32 heads on 8: heads of 64 36 us, with 1,024 parts 37;
// of 128 74, with 512 70; of 256 135, with 768 142).  Wide: 2 a CU, all that heads of 256 have registers for (a chunk of 2,047: 1,425 us,
// with 1,024 parts 1,510).  Smaller heads have them for more, and few tiles over many cells would gain by it: 512 tokens behind 30,000
// cells, 32 heads on 8, of 64 275 us (with 1,024 parts 196), of 128 355 (with 768 301).
constexpr int pg_parts(int kind, int narrow, int hd) {
    return kind ? 512 : narrow == 64 ? (hd == 256 ? 512 : 768) : hd == 64 ? 1024 : hd == 128 ? 512 : 256;
}
constexpr int PG_MORE = 512;
constexpr int PG_MAGIC = 0x70616765;

struct PgItem {
    int req, row0;                              // request, first row of the tile
    int lo, hi;                                 // the part's cells
    int part;                                   // place in the workspace; -1: the tile is whole, results go out
    int q0, n_new, n_cached;                    // the request's first packed row, its tokens
};
struct PgMerge {
    int part, n;                                // the tile's parts
    int q0, row0, rows, pad[3];
};
struct PgHead {
    int magic, geometry;
    int n_items[2], n_merges[2];                // narrow, wide
    int part[2];                                // longest part, blocks of 32 cells
    int pad[8];
};
struct PgBefore { int items[2], parts, merges; };   // what the requests before one have; parts and merges of its own kind
static_assert(sizeof(PgItem) == 32 && sizeof(PgMerge) == 32 && sizeof(PgHead) == 64 && sizeof(PgBefore) == 16, "work list");

// What one list holds at most, and where (in entries of 32 bytes behind the head; the requests' sums come last).
struct PgLayout {
    int narrow;                                 // rows of a narrow tile: 32 or 64
    int items[2], parts[2], merges[2];          // capacities: narrow, wide
    int min_len[2];                             // shortest part, cells
    int item_at[2], merge_at[2], before_at, total;
};

inline int pg_div_up(int64_t a, int64_t b) { return (int) ((a + b - 1) / b); }
inline int pg_max_new(const wzy_paged_batch* b) { return b->max_new > 0 && b->max_new < b->max_tokens ? b->max_new : b->max_tokens; }

// A part is long enough to be worth its partial results: a narrow tile's take 4 * hd bytes a row to write and read against the
// 4 * hd bytes of each cell's key and value; a wide tile's as much a row, for 128 rows.
inline PgLayout pg_layout(int n_req, int max_tokens, int max_new, int max_cells, const wzy_paged_work* w) {
    PgLayout l{};
    const int g = w->qh / w->kvh;
    const int64_t rows = (int64_t) max_new * g;
    l.narrow = rows > 32 && rows <= 64 ? 64 : 32;
    const bool any_wide = rows > l.narrow;
    const int64_t tiles[2] = {n_req, any_wide ? (int64_t) max_tokens * g / PG_WIDE + n_req : 0};
    l.min_len[0] = 64;
    l.min_len[1] = 512;
    int at = 0;
    for (int k = 0; k < 2; ++k) {
        // n = ceil(span / len) with the sum of span / len at most per_head: all tiles' parts, and those of tiles that have several
        const int64_t more = k ? 0 : n_req < PG_MORE / w->kvh ? n_req : PG_MORE / w->kvh;
        const int64_t per_head = pg_div_up(pg_parts(k, l.narrow, w->hd), w->kvh) + more;
        const int64_t most = tiles[k] * pg_div_up(max_cells, l.min_len[k]);
        l.items[k] = (int) (most < tiles[k] + per_head ? most : tiles[k] + per_head);
        l.parts[k] = (int) (most < 2 * per_head ? most : 2 * per_head);
        l.merges[k] = (int) (tiles[k] < l.parts[k] / 2 ? tiles[k] : l.parts[k] / 2);
        l.item_at[k] = at;
        at += l.items[k];
    }
    for (int k = 0; k < 2; ++k) {
        l.merge_at[k] = at;
        at += l.merges[k];
    }
    l.before_at = at;
    l.total = at + (n_req + 1) / 2;
    return l;
}
PgLayout pg_layout_of(const wzy_paged_batch* b, const wzy_paged_work* w);
// what a list was built for: a call whose numbers give another layout finds no work in it
inline int pg_geometry(const wzy_paged_work* w, const PgLayout& l) {
    uint32_t h = 2166136261u;
    for (int v : {w->hd, w->qh, w->kvh, w->window, l.narrow, l.items[0], l.items[1], l.parts[0], l.parts[1], l.merges[0], l.merges[1], l.total})
        h = (h ^ (uint32_t) v) * 16777619u;
    return (int) h;
}
// no request has more cells than that
inline int pg_window(const wzy_paged_work* w) { return w->window < PG_MAX_CELLS ? w->window : 0; }

// ---- host checks ----------------------------------------------------------------------------------------
inline bool pg_page_ok(int n_pages, int page) {
    return page >= 16 && page <= 4096 && (page & (page - 1)) == 0 && n_pages >= 1 && (int64_t) n_pages * page < (1ll << 31);
}
inline int pg_check_batch(const char* who, const wzy_paged_batch* b, int page) {
    WZY_REQUIRE(b, "%s: batch is null", who);
    WZY_REQUIRE(b->n_req >= 1 && b->n_req <= PG_MAX_REQ, "%s: %d requests (1 .. %d)", who, b->n_req, PG_MAX_REQ);
    WZY_REQUIRE(b->max_tokens >= 1 && b->max_tokens <= PG_MAX_TOKENS, "%s: max_tokens %d (1 .. %d)", who, b->max_tokens, PG_MAX_TOKENS);
    WZY_REQUIRE(b->max_new >= 0, "%s: max_new %d", who, b->max_new);
    WZY_REQUIRE(b->max_pages >= 1 && (int64_t) b->max_pages * page <= PG_MAX_CELLS && (int64_t) b->max_pages * b->n_req < 1ll << 31,
                "%s: max_pages %d (at most %d cells, fewer than 2^31 entries)", who, b->max_pages, PG_MAX_CELLS);
    return WZY_OK;
}
inline int pg_check_work(const char* who, const wzy_paged_work* w) {
    WZY_REQUIRE(w, "%s: work is null", who);
    WZY_REQUIRE(w->kvh >= 1 && w->kvh <= 64 && w->qh >= w->kvh && w->qh % w->kvh == 0 && w->qh / w->kvh <= 256,
                "%s: %d query heads, %d key heads", who, w->qh, w->kvh);
    WZY_REQUIRE(w->hd == 64 || w->hd == 128 || w->hd == 256, "%s: head size %d (64, 128 or 256)", who, w->hd);
    WZY_REQUIRE(w->window >= 0, "%s: window %d", who, w->window);
    return WZY_OK;
}
// a list's workgroups fit one launch, which has fewer than 2^32 threads
inline int pg_check_launch(const char* who, const wzy_paged_batch* b, const wzy_paged_work* w, const PgLayout& l) {
    for (int items : l.items)
        WZY_REQUIRE((int64_t) items * w->kvh < 1 << 24, "%s: %d rows of %d query heads (their product below 2^31)", who, b->max_tokens, w->qh);
    return WZY_OK;
}
// rows of heads at any alignment of an element
inline int pg_check_heads(const char* who, const char* what, const wzy_heads* h, int type, int heads, int hd) {
    WZY_REQUIRE(h && h->p, "%s: %s is null", who, what);
    WZY_REQUIRE((uintptr_t) h->p % mx_type_bytes(type) == 0 && h->ld >= 0 && h->ld <= (int64_t) 1 << 40 && h->ld_head >= 0 &&
                    h->ld_head <= (int64_t) 1 << 40 && (heads == 1 || h->ld_head >= hd),
                "%s: %s: row stride %lld, head stride %lld, %d heads of %d at %p", who, what, (long long) h->ld,
                (long long) h->ld_head, heads, hd, h->p);
    return WZY_OK;
}
inline int pg_check_cache(const char* who, const wzy_paged_cache* c) {
    WZY_REQUIRE(c && c->k && c->v, "%s: cache is null", who);
    WZY_REQUIRE(c->type == WZY_BF16 || c->type == WZY_F16, "%s: cache of type %d", who, c->type);
    WZY_REQUIRE(c->kvh >= 1 && c->kvh <= 64 && (c->hd == 64 || c->hd == 128 || c->hd == 256), "%s: cache of %d heads of %d", who, c->kvh, c->hd);
    WZY_REQUIRE(pg_page_ok(c->n_pages, c->page), "%s: %d pages of %d cells", who, c->n_pages, c->page);
    WZY_REQUIRE((uintptr_t) c->k % 16 == 0 && (uintptr_t) c->v % 16 == 0 && c->ld_page % 8 == 0 && c->ld_cell % 8 == 0 && c->ld_head % 8 == 0 &&
                    c->ld_page >= 0 && c->ld_page <= (int64_t) 1 << 40 && c->ld_cell >= c->hd && c->ld_cell < (1 << 24) && c->ld_head >= 0 &&
                    c->ld_head <= (int64_t) 1 << 40 && (c->kvh == 1 || c->ld_head >= c->hd) && (c->n_pages == 1 || c->ld_page >= c->hd),
                "%s: cache strides %lld, %lld, %lld (multiples of 8, at least a head's size)", who, (long long) c->ld_page,
                (long long) c->ld_cell, (long long) c->ld_head);
    return WZY_OK;
}
inline int pg_log2(int v) { return 31 - __builtin_clz((unsigned) v); }

}  // namespace wzy
