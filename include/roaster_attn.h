/*
 * roaster_attn.h -- softmax attention over a paged key/value cache, for the
 * full-attention layers between the projections of roaster_moe.h: a step's
 * plan (block tables, row positions, cache slots), the query/key norms with
 * the position rotation and the store into the cache, and attention over the
 * cached pages (model.c:755-863 for one token, 1536-1602 for a prompt's chunk).
 *
 * Conventions as in roaster_moe.h: row-major, device pointers, calls ordered
 * on the library's stream (roaster_stream), ROASTER_OK or a negative ROASTER_E*
 * with the message in roaster_last_error().  Argument structures are host
 * memory, read within the call.  Sizes, alignments and overlaps are checked
 * by the call (ROASTER_EINVAL, nothing launched); what only the device can see
 * (lengths, page numbers, slots) is checked by the kernels, which neither read
 * nor write out of bounds for any value, and reported by roaster_sync:
 * ROASTER_ENOMEM for a plan without enough free pages, ROASTER_EINVAL for the
 * others, each in a call of its own where there are several.  No call
 * allocates, copies to the host or waits: after roaster_init all of them can be
 * captured into a HIP graph on roaster_stream, the rows that a replay does not
 * use being marked by -1.  Two calls, or two captured
 * graphs, that may run at the same time need output buffers, a page ring and
 * workspaces of their own.
 */
#ifndef ROASTER_ATTN_H
#define ROASTER_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of a cache. */
#define ROASTER_KV_F32 0      /* as the reference keeps it */
#define ROASTER_KV_F16 1      /* half the bytes; keys and values rounded to nearest even, infinite past 65504 */

/* One layer's cache: keys and values, each [n_pages][kv_heads][page_size][head_dim].
 * Slot s of a layer is token s % page_size of page s / page_size.  One plan
 * (block table, slots) serves every layer whose cache has its n_pages and
 * page_size. */
typedef struct {
    void *k, *v;              /* 16-byte aligned */
    int   type;               /* ROASTER_KV_* */
    int   n_pages;            /* n_pages * page_size <= 2^31 - 1 */
    int   page_size;          /* a power of two, 16 .. 4096 */
    int   kv_heads;           /* 1 .. 1024 */
    int   head_dim;           /* 64, 128 or 256 */
} RoasterKvCache;

/* ---- plan: block tables and slot maps from request lengths ---------------- */
/* One step of n_req requests.  Request r holds len[r] tokens in the first
 * ceil(len[r] / page_size) pages of its table row and adds add[r] new ones (0: none;
 * -1: the request has ended, its pages go back to the ring).  The free pages
 * are ring[i % n_pages] for i in [ctl[0], ctl[1]); new pages are taken from the
 * front in the order of requests, freed ones put behind the end in that order.
 *   len_out[r] = len[r] + add[r], 0 for an ended request
 *   table      the new pages entered; other entries stay as they were
 *   ctl_out    the ring's front and end after the step
 *   first      [n_req + 1] exclusive sums of the new tokens, or NULL
 *   row_*      one row per new token, requests in order, a request's tokens in
 *              order: its request, its position in it and its cache slot; -1 in
 *              the rows behind the last, up to max_rows
 * len_out may be len, and ctl_out may be ctl; no other two may overlap.
 * A step that does not fit (free pages, table width, max_rows, a length out of
 * range, a ring that is not one) is refused as a whole: len_out = len, ctl_out =
 * ctl, table and ring untouched, first all 0, every row -1, and roaster_sync
 * reports it.  A page number out of range in the ring or in a table row gives
 * its rows slot -1 (a new one is entered as -1) and is reported; one that an ended
 * request gives back is reported, stands in the ring as -1, and counts as a free page
 * until it is taken. */
typedef struct {
    int n_req;                /* 1 .. 2048 */
    int page_size;            /* a power of two, 16 .. 4096 */
    int n_pages;              /* of the caches, and entries of the ring */
    int max_pages;            /* entries of a table row; max_pages * page_size <= 2^30 */
    int max_rows;             /* 1 .. 262144 */
    const int *len, *add;     /* [n_req] */
    int *len_out;             /* [n_req] */
    int *table;               /* [n_req][max_pages] */
    int *ring;                /* [n_pages] */
    const int64_t *ctl;       /* [2]: front, end */
    int64_t *ctl_out;         /* [2] */
    int *first;               /* [n_req + 1] or NULL */
    int *row_req, *row_pos, *row_slot;   /* [max_rows] */
} RoasterKvPlan;

int roaster_kv_plan(const RoasterKvPlan *plan);

/* ---- norms of queries and keys, rotation, store into the cache ------------- */
/* For every row t with row_slot[t] >= 0, per head:
 *   x = x * rsqrt(mean(x^2) + eps) * norm     (queries q_norm, keys k_norm; NULL: x as it is)
 *   the first rot_dim elements rotated by position: angle_i = row_pos[t] * theta^(-2 i / rot_dim),
 *   pairs (x_i, x_{i + rot_dim/2}), or (x_2i, x_2i+1) with pair_adjacent
 *   q_out[t][head] = x for queries; cache slot row_slot[t] = keys so treated, and values as they are.
 * Rows with slot -1 are skipped, q_out included; a slot past the cache is
 * skipped and reported.  Angles are computed in 64 bits.  The slots of one call
 * must differ from each other (of two rows with one slot either's elements
 * remain).  q, k, v: element d of head h of row t at [t * row + h * head + d], the
 * strides in floats, multiples of 4, bases 16-byte aligned (a projection that
 * holds each head's gate behind its query has q_head = 2 head_dim).  q_out:
 * [rows][q_heads][head_dim], apart from the inputs, or q itself where that has
 * this layout.  rows = 0 does nothing. */
typedef struct {
    int rows;                 /* 0 .. 2^20 */
    int q_heads;              /* 1 .. 1024 */
    const float *q;
    size_t q_row, q_head;
    const float *k;
    size_t k_row, k_head;
    const float *v;
    size_t v_row, v_head;
    const float *q_norm, *k_norm;        /* [head_dim], 16-byte aligned, or NULL */
    float eps;
    int rot_dim;              /* a multiple of 8, 0 .. head_dim */
    int pair_adjacent;
    double theta;             /* 1 .. 1e30 */
    const int *row_pos, *row_slot;       /* [rows] */
    float *q_out;
} RoasterQkRope;

int roaster_qk_rope_store(const RoasterQkRope *rope, const RoasterKvCache *cache);

/* ---- attention over the cached pages ---------------------------------------- */
/* Row t of request r = row_req[t] attends to positions 0 .. row_pos[t] of r (its own
 * key and value having been stored): for each head h, on key/value head
 * h / (q_heads / kv_heads),
 *   out[t][h] = sum_j softmax_j(scale * q[t][h] . K_j) V_j   (* sigmoid(gate) with a gate)
 * One row per request is a decode step; several consecutive rows of a request
 * are a draft or a prompt's chunk.  row_pos[t] = -1: no position, out is 0.
 * row_req[t] = -1: the row is skipped, out untouched.  A request, position or
 * page number out of range gives that row NaN outputs and is reported.
 * Keys and values behind a row's position are never used, whatever they hold.
 * Infinite or NaN keys and values in use make the elements that they reach
 * infinite or NaN; so does a scale * log2(e) * q past f32's range.  Sums and softmax
 * are in 32 bits; with an fp16 cache the queries enter the products with 22 bits (two
 * fp16 parts, relative to a head's largest element), and probabilities off by at
 * most 2^-22 of themselves or 2^-24 of the largest in their tile (up to 32 positions one
 * behind the other).  Where a position outweighs all before it, those in its tile are
 * off by up to 2^-38 of its probability, and tiles below 2^-70 of it may be left out.
 * How a call's work is split goes by all its rows: the last bits of a row's output depend on
 * them, and are the same for the same call.
 * An fp16 call of 16 rows or more, and of more rows for each of the n_req requests than
 * 16 / (q_heads / kv_heads), two at least, takes the rows of a request that stand
 * together together (8 query heads on one: 8 or 16 rows at a time); it is right, but slow,
 * where most of its rows are one to a request.
 * gate: element d of head h of row t at [t * gate_row + h * gate_head + d].
 * out and ws must not overlap the inputs.  rows = 0 does nothing. */
typedef struct {
    int rows;                 /* 0 .. 2^20 */
    int q_heads;              /* a multiple of kv_heads, at most 1024 */
    const float *q;           /* [rows][q_heads][head_dim], 16-byte aligned */
    const int *row_req, *row_pos;        /* [rows] */
    const int *table;         /* [n_req][max_pages] */
    int n_req, max_pages;     /* max_pages * page_size <= 2^30 */
    float scale;              /* at most 2e38 in size */
    const float *gate;        /* or NULL; 16-byte aligned, strides multiples of 4 */
    size_t gate_row, gate_head;
    float *out;               /* [rows][q_heads][head_dim], 16-byte aligned */
    void *ws;                 /* 16-byte aligned, at least roaster_attn_ws_bytes */
    size_t ws_bytes;
} RoasterAttnPaged;

/* Workspace of a call with so many rows (a larger one serves as well); host
 * only.  0 for bad arguments. */
size_t roaster_attn_ws_bytes(int rows, int q_heads, const RoasterKvCache *cache);
int roaster_attn_paged(const RoasterAttnPaged *attn, const RoasterKvCache *cache);

#ifdef __cplusplus
}
#endif
#endif
