/* wzy_paged.h -- operators of the MI355X (gfx950) library for several requests at once: a paged key-value cache,
 * rotary positions, attention of new tokens over the pages, sampling of the next tokens.
 *
 * Conventions are those of wzy_kernels.h: device pointers, `stream` is a hipStream_t of the current device passed as
 * void* (NULL = the null stream), a status code comes back and wzy_last_error() says why a call was refused.  Structures
 * are host memory and read before the call returns; the pointers in them are device memory.  Nothing here synchronizes,
 * allocates or keeps state between calls, and every call can be captured into a graph.  A refused call launches nothing.
 * Work lists and workspaces belong to the caller: calls that share one must not overlap in time, others may.
 * An output shares no byte with an input or another output, but where its operator says so.  Row types are WZY_F32,
 * WZY_BF16, WZY_F16 (wzy_mx.h).
 *
 * A step of a batch: wzy_paged_plan gives the new tokens pages, positions and cache slots; each attention layer calls
 * wzy_paged_append and wzy_paged_attend; wzy_sample draws the next tokens; wzy_paged_release takes back the pages of
 * requests that ended.  No length has to be known on the host.  The reference serves one sequence from a contiguous
 * store and samples on the host (src/wzy_engine_v2.cu:36-179); it has no counterpart of these calls.
 */
#ifndef WZY_PAGED_H
#define WZY_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "wzy_kernels.h"
#include "wzy_mx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------------------------
 * Pages, block tables, slots
 * ------------------------------------------------------------------------------------------- */

/* Pool of free pages: ids free_pages[0 .. *n_free - 1], taken from the end.  A call reads *n_free and writes the new
 * number to *n_free_out, which may be n_free itself. */
typedef struct wzy_paged_pool {
    int* free_pages;             /* [n_pages] */
    const int* n_free;
    int* n_free_out;
    int n_pages;                 /* pages of the cache */
    int page;                    /* cells a page: a power of two, 16 .. 4,096; n_pages * page below 2^31 */
} wzy_paged_pool;

/* One step of a batch.  Request r holds n_cached[r] cells, in the pages table[r * max_pages ..] (page i holds its cells
 * i * page ..), and brings n_new[r] new ones; the step's new tokens are packed rows, request after request. */
typedef struct wzy_paged_batch {
    int n_req;                   /* 1 .. 4,096 */
    int max_tokens;              /* rows of the packed arrays, 1 .. 1,048,576 */
    int max_pages;               /* columns of the table; max_pages * page at most 2^24 cells, n_req * max_pages below 2^31 */
    const int* n_cached;         /* [n_req]; negative counts as 0 */
    const int* n_new;            /* [n_req]; negative counts as 0 */
    int* table;                  /* [n_req x max_pages] page ids, in and out */
    int* q_start;                /* [n_req + 1] out: request r's rows are q_start[r] .. q_start[r + 1] - 1 */
    int* kv_len;                 /* [n_req] out: n_cached + n_new; 0 for a request that is not served */
    int* served;                 /* [n_req] out: 1, or 0 */
    int* positions;              /* [max_tokens] out: n_cached + place in the request */
    int* slots;                  /* [max_tokens] out: table[position / page] * page + position % page.  Rows behind the last, and
                                    rows of a request that is not served: position 0, slot -1.  A page id
                                    outside 0 .. n_pages - 1: slot -1 */
    int max_new;                 /* the largest n_new; 0: max_tokens */
} wzy_paged_batch;

/* How the attention layers of one kind split a step among workgroups.  A list is built by wzy_paged_plan and read by every
 * wzy_paged_attend of that step; layers that differ in these numbers need lists of their own. */
typedef struct wzy_paged_work {
    int qh, kvh, hd;             /* query heads (a multiple of kvh, at most 256 of them a key head), key heads (1 .. 64),
                                    head size: 64, 128 or 256; max_tokens * qh + 128 * n_req * kvh at most 2^31 - 2^17 */
    int window;                  /* a token sees itself and the window - 1 cells before it; 0: all */
    void* items;                 /* device memory of wzy_paged_work_bytes() bytes, 16-byte aligned */
    size_t bytes;
} wzy_paged_work;
/* 0 where the structures are not valid. */
size_t wzy_paged_work_bytes(const wzy_paged_batch* batch, const wzy_paged_work* work);

/* Pages, tables, slots and work lists of one step.  Request r takes ceil((n_cached + n_new) / page) - ceil(n_cached / page)
 * pages, requests in order, a request's in order of its cells.  Not served, and left as it was, is a request that
 *   does not fit the table, or brings more than max_new tokens, or
 *   has rows past max_tokens (q_start is limited to max_tokens), or
 *   needs pages where those before it and it need more than are free (whoever comes after and needs pages too, likewise).
 * works [n_works], 0 .. 8 of them.  A request with n_new = 0 keeps its pages and has no rows. */
int wzy_paged_plan(const wzy_paged_pool* pool, const wzy_paged_batch* batch, const wzy_paged_work* works, int n_works,
                   void* stream);

/* Pages of requests that ended (ended[r] != 0; [n_req]) go back to the pool, in order of requests and cells:
 * ceil(n_cached / page) each.  Their table entries become -1.  Entries outside 0 .. n_pages - 1 are left out, and what a full
 * pool has no room for.  Of the batch, only n_req, max_pages, n_cached and table are read. */
int wzy_paged_release(const wzy_paged_pool* pool, const wzy_paged_batch* batch, const int* ended, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Rotary positions
 * ------------------------------------------------------------------------------------------- */

/* Rows of heads: head h of row r starts at p + r * ld + h * ld_head (elements). */
typedef struct wzy_heads {
    void* p;
    int64_t ld, ld_head;
} wzy_heads;

#define WZY_ROPE_HALVES 0        /* pair i = elements i and i + n_rot / 2 */
#define WZY_ROPE_PAIRS 1         /* pair i = elements 2 i and 2 i + 1 */

#define WZY_ROPE_PLAIN 0         /* f_i = theta^(-2 i / n_rot) */
#define WZY_ROPE_LINEAR 1        /* f_i / factor: positions divided by factor */
#define WZY_ROPE_ROTATIONS 2     /* r_i f_i + (1 - r_i) f_i / factor, r_i = (ctx f_i / 2 pi - low) / (high - low) limited to 0 .. 1 */
#define WZY_ROPE_INDEX 3         /* the same with r_i = 1 - (i - a) / (b - a), a = max(floor(at(high)), 0),
                                    b = min(ceil(at(low)), n_rot - 1), at(x) = n_rot ln(ctx / (2 pi x)) / (2 ln theta) */
typedef struct wzy_rope_cfg {
    double theta;                /* above 1 */
    double factor;               /* at least 1 */
    double low, high;            /* 0 < low < high: rotations over the trained context (ROTATIONS, INDEX) */
    double amplitude;            /* of the rotated pairs; 0 counts as 1 */
    int ctx;                     /* trained context (ROTATIONS, INDEX) */
    int n_rot;                   /* even, 2 .. 512 */
    int scaling;                 /* WZY_ROPE_PLAIN .. WZY_ROPE_INDEX */
} wzy_rope_cfg;
/* freqs [n_rot / 2 + 1]: f_i / 2 pi (turns a position), then the amplitude; made once and kept. */
int wzy_rope_freqs(const wzy_rope_cfg* cfg, double* freqs, void* stream);

typedef struct wzy_rope_tab {
    const double* freqs;
    int n_rot;                   /* elements 0 .. n_rot - 1 of each head are rotated, the others copied */
    int layout;                  /* WZY_ROPE_HALVES or WZY_ROPE_PAIRS */
} wzy_rope_tab;

/* out = x with its pairs (a, b) turned: A (a cos t - b sin t), A (b cos t + a sin t), t = positions[row] f_i, A the amplitude.
 * Angles in 64 bits, the rotation in fp32, one rounding to `type`.  x and out [rows x heads x hd] of `type`; out may be x
 * (same strides).  positions [rows], any int.  n_rot <= hd <= 512; heads 1 .. 1,024; addresses and strides have the
 * alignment of an element (multiples of 16 bytes, and n_rot of 16, run faster). */
int wzy_rope(const wzy_rope_tab* rope, const wzy_heads* x, int type, int rows, int heads, int hd, const int* positions,
             const wzy_heads* out, void* stream);

/* Cell c of page p, head h: k + p * ld_page + c * ld_cell + h * ld_head (elements), v likewise. */
typedef struct wzy_paged_cache {
    void* k;
    void* v;
    int64_t ld_page, ld_cell, ld_head;   /* multiples of 8; k and v 16-byte aligned; ld_cell below 2^24 */
    int n_pages, page;                   /* as in the pool */
    int kvh, hd;                         /* 1 .. 64; 64, 128 or 256 */
    int type;                            /* WZY_BF16 or WZY_F16 */
} wzy_paged_cache;

/* q (qh heads) and k turned as by wzy_rope and rounded once to the cache's type: q to q_out, k to the cells slots[row];
 * v to the same cells.  q, k, v of `type`, rows of hd elements a head, for instance parts of one projection's rows; rope NULL:
 * nothing is turned; q and q_out NULL (qh 0): keys and values only.  q_out may be q (same type and strides).  Rows whose slot is
 * outside 0 .. n_pages * page - 1 leave the cache alone.  Slots are different from each other. */
int wzy_paged_append(const wzy_paged_cache* cache, const wzy_rope_tab* rope, const wzy_heads* q, int qh, const wzy_heads* q_out,
                     const wzy_heads* k, const wzy_heads* v, int type, int rows, const int* positions, const int* slots,
                     void* stream);

/* ---------------------------------------------------------------------------------------------
 * Attention over pages
 * ------------------------------------------------------------------------------------------- */

/* out[t, h] = sum_j p_j v_j,  p = softmax over j of scale * q[t, h] . k_j, for each new token t of each request: j runs over the
 * request's cells up to t's own position, the last `window` of them, key head h / (qh / kvh).  q, out [max_tokens x qh x hd]
 * of the cache's type, 16-byte aligned, strides multiples of 8; rows of a request that is not served become 0, rows behind the last
 * request's keep what they hold.  The batch is as wzy_paged_plan left it, `work` one of its lists (a list
 * that was built for other numbers has no work: nothing is written).
 * Sums are fp32; the softmax weights are rounded to the cache's type for the second product (half a step of a weight, so of
 * an output at most as much; fp16 weights are taken 2^6 larger, so that small ones are not lost).  A value that is not finite
 * reaches only the rows that see its cell: of V, its column of those rows becomes infinite or not a number (not a number also where
 * the weight is too small for its type, or rounds to 0 beside the largest).  A row whose scores are all -infinity becomes 0, but for
 * such columns.
 * Page ids outside 0 .. n_pages - 1 count as page 0.  scale is finite and above 0. */
size_t wzy_paged_attend_workspace_bytes(const wzy_paged_batch* batch, const wzy_paged_work* work);
int wzy_paged_attend(const wzy_paged_cache* cache, const wzy_paged_batch* batch, const wzy_paged_work* work, const wzy_heads* q,
                     const wzy_heads* out, float scale, void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Sampling
 * ------------------------------------------------------------------------------------------- */

/* One token a row of logits [rows x vocab] (type, row stride ld elements), by given numbers:
 *   order        larger logit first, ties to the lower id; a NaN counts as -infinity
 *   top_k        only the first top_k of that order remain (top_k < 1: all)
 *   w_i          exp((l_i - l_0) / temp), Z their sum
 *   min_p        of those, w_i >= min_p * w_0
 *   top_p        of those, the first until their sum reaches top_p * Z, that one included (top_p <= 0 or >= 1: all)
 *   id           the first whose running sum reaches u * (the sum of what is left); prob = its share of that sum
 * as the host sampler of wzy_engine.h does, but for its repetition penalty, over any number of logits.  temp at or below 1e-5: the first of the order,
 * prob 1.  A row without a logit above -infinity gives id -1, prob 0; +infinity takes all there is, shared by those that
 * have it.  Sums are integers of 2^-40 to 2^-51 of w_0, so results do not depend on the order of additions.
 * temp, top_k, top_p, min_p [rows] may each be NULL: 1, all, all, all; u [rows] in 0 .. 1 (below 0 counts as 0, above 1 as 1,
 * NaN as 0).  probs may be NULL.  1 <= vocab <= 2^22, rows at most 65,535; any alignment of an element. */
size_t wzy_sample_workspace_bytes(int rows, int vocab);
int wzy_sample(const void* logits, int type, int64_t ld, int rows, int vocab, const float* temp, const int* top_k,
               const float* top_p, const float* min_p, const float* u, int* ids, float* probs, void* workspace,
               size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* WZY_PAGED_H */
