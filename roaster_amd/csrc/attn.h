/*
 * attn.h -- what the attention operators (kv_plan.hip, qk_rope.hip, attn.hip)
 * share: their error word and the host-side checks of their arguments.
 */
#ifndef ROASTER_ATTN_INTERNAL_H
#define ROASTER_ATTN_INTERNAL_H

#include "internal.h"
#include "../../include/roaster_attn.h"
#include "attn_index.h"

/* Error bits of the attention operators' device word (rt_attn_err). */
#define ATTN_ERR_PAGES 1      /* a plan found too few free pages */
#define ATTN_ERR_PLAN 2       /* a plan's lengths, sizes or ring out of range */
#define ATTN_ERR_INDEX 4      /* a request, position, page or slot out of range */

/* Makes the library's device current for the calls of one entry point and
 * gives the caller's back: the library's stream belongs to that device. */
struct AttnDevice {
    int prev = -1;
    AttnDevice()
    {
        if (hipGetDevice(&prev) != hipSuccess || prev == rt().device) prev = -1;
        else (void)hipSetDevice(rt().device);
    }
    ~AttnDevice()
    {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

static inline bool attn_aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

/* Whether [a, a + na) and [b, b + nb) share a byte (either may be absent). */
static inline bool attn_overlap(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && x < y + nb && y < x + na;
}

static inline bool attn_page_ok(int page_size) { return page_size >= 16 && page_size <= 4096 && !(page_size & (page_size - 1)); }

static inline bool attn_cache_ok(const RoasterKvCache *c)
{
    return c && c->k && c->v && attn_aligned(c->k, 16) && attn_aligned(c->v, 16) &&
           (c->type == ROASTER_KV_F32 || c->type == ROASTER_KV_F16) && attn_page_ok(c->page_size) && c->n_pages >= 1 &&
           (int64_t)c->n_pages * c->page_size <= INT32_MAX && c->kv_heads >= 1 && c->kv_heads <= 1024 &&
           (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256);
}

static inline KvShape attn_shape(const RoasterKvCache *c)
{
    KvShape s = { 0, c->n_pages, c->kv_heads, c->head_dim };
    while ((1 << s.shift) < c->page_size) s.shift++;
    return s;
}

static inline size_t attn_cache_bytes(const RoasterKvCache *c)
{
    return (size_t)c->n_pages * c->page_size * c->kv_heads * c->head_dim * (c->type == ROASTER_KV_F16 ? 2 : 4);
}

#endif
