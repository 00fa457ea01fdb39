/*
 * attn_index.h -- where a row's tokens lie in a paged cache, and which values
 * of device-side indices are in range: the attention kernels index by these
 * functions alone.
 */
#ifndef ROASTER_ATTN_INDEX_H
#define ROASTER_ATTN_INDEX_H

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define ATTN_FN __host__ __device__ __forceinline__
#else
#define ATTN_FN inline
#endif

struct KvShape {
    int shift;                /* log2 of the page size */
    int n_pages, kv, dim;

    ATTN_FN bool page_ok(int p) const { return p >= 0 && p < n_pages; }
    ATTN_FN bool slot_ok(int s) const { return s >= 0 && (s >> shift) < n_pages; }
    /* Element 0 of token `in` (0 .. page size - 1) of head h in page p.  A page has at most
     * 1024 heads of 4096 tokens of 256 elements: 2^30. */
    ATTN_FN unsigned page_elements() const { return (unsigned)(kv << shift) * dim; }
    ATTN_FN size_t at(int p, int h, int in) const { return (uint64_t)(unsigned)p * page_elements() + (unsigned)(((h << shift) + in) * dim); }
    ATTN_FN size_t at_slot(int s, int h) const { return at(s >> shift, h, s & ((1 << shift) - 1)); }
    ATTN_FN size_t elements() const { return (size_t)n_pages * page_elements(); }
};

/* Block tables of n_req requests, max_pages entries each. */
struct KvTable {
    int n_req, max_pages;

    /* Tokens a row attends to, 0 for position -1; -1 if its request or position is out of range. */
    ATTN_FN int tokens(int req, int pos, int shift) const
    {
        if (req < 0 || req >= n_req || pos < -1 || pos >= ((int64_t)max_pages << shift)) return -1;
        return pos + 1;
    }
    ATTN_FN size_t entry(int req, int token, int shift) const { return (size_t)req * max_pages + (token >> shift); }
};

#endif
