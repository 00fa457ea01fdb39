/*
 * kv_plan.hip -- one serving step's block tables, row positions and cache
 * slots, built on the GPU from the requests' lengths (roaster_kv_plan).
 */
#include "attn.h"

#define KVP_MAX_REQ 2048
#define KVP_MAX_ROWS (1 << 18)
#define KVP_CAP (1 << 30)     /* sums saturate here: past every limit, and two of them still fit an int */
#define KVP_T 256

/* Inclusive saturating sum over the workgroup, KVP_T threads; `tot` gets the
 * whole.  min(a + b, KVP_CAP) is associative for values in [0, KVP_CAP]. */
__device__ __forceinline__ int kvp_add(int a, int b) { return min(a + b, KVP_CAP); }

__device__ __forceinline__ int kvp_scan(int v, int *s_wave, int &tot)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v = kvp_add(v, u);
    }
    if (lane == 63) s_wave[w] = v;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < KVP_T / 64; i++) {
        if (i == w) before = all;
        all = kvp_add(all, s_wave[i]);
    }
    tot = all;
    return kvp_add(v, before);
}

/* The request r with c[r] <= i < c[r + 1], for i < c[n]. */
__device__ __forceinline__ int kvp_find(const int *c, int n, int i)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (c[m] <= i) lo = m;
        else hi = m;
    }
    return lo;
}

/* Every workgroup sums all requests by itself (three scans of up to eight
 * values a thread) and then writes its share of the rows, new table entries
 * and freed pages, each found by binary search in the sums: no workgroup waits
 * for another.  Nothing is read that the same launch writes -- table entries
 * at and past ceil(len / page) are written, those before are read; ring entries
 * [front, front + taken) are read, [end, end + freed) written, apart because
 * end + freed <= front + n_pages is checked -- but len and ctl where the caller
 * gives the same memory for len_out and ctl_out: then one workgroup, which has
 * read both before its first barrier, does all, or a second launch of one
 * workgroup writes them (`what`: bit 0 rows, table and ring, bit 1 len_out,
 * ctl_out, first and the error word).  What bounds it: latency, a chain of the
 * lengths' load, three scans, a search and a page's load; 8 requests of one row 4.5
 * us, 512 requests with 22700 rows 6.9; in place, a call by itself, 5.8 in one workgroup
 * and 13.6 in two launches. */
__global__ __launch_bounds__(KVP_T) void kv_plan_kernel(RoasterKvPlan A, int shift, int what, int *err)
{
    __shared__ int c_row[KVP_MAX_REQ + 1], c_new[KVP_MAX_REQ + 1], c_old[KVP_MAX_REQ + 1], s_len[KVP_MAX_REQ];
    __shared__ int s_wave[3][KVP_T / 64];
    const int tid = threadIdx.x, n = A.n_req, per = (n + KVP_T - 1) / KVP_T, P = A.page_size, N = A.n_pages;
    const int64_t cap = (int64_t)A.max_pages << shift;
    const int64_t front = A.ctl[0], end = A.ctl[1];
    int bad = !(front >= 0 && end >= front && end - front <= N && end < ((int64_t)1 << 62));
    int rows = 0, fresh = 0, freed = 0;
    for (int i = 0; i < per; i++) {
        const int r = tid * per + i;
        if (r >= n) break;
        const int l = A.len[r], a = A.add[r];
        const bool ok = l >= 0 && l <= cap && a >= -1 && a <= A.max_rows && (int64_t)l + a <= cap;
        bad |= !ok;
        const int have = ok ? (int)(((int64_t)l + P - 1) >> shift) : 0, na = ok && a > 0 ? a : 0;
        const int need = na ? (int)(((int64_t)l + na + P - 1) >> shift) - have : 0;
        /* this thread's own running sums; the threads' before it are added below */
        s_len[r] = ok ? l : 0;
        c_row[r + 1] = rows = kvp_add(rows, na);
        c_new[r + 1] = fresh = kvp_add(fresh, need);
        c_old[r + 1] = freed = kvp_add(freed, ok && a < 0 ? min(have, KVP_CAP) : 0);
    }
    int t_row, t_new, t_old;
    const int i_row = kvp_scan(rows, s_wave[0], t_row), i_new = kvp_scan(fresh, s_wave[1], t_new),
              i_old = kvp_scan(freed, s_wave[2], t_old);
    /* what stands before this thread's requests (sums that saturate are refused below) */
    const int b_row = i_row - rows, b_new = i_new - fresh, b_old = i_old - freed;
    for (int i = 0; i < per; i++) {
        const int r = tid * per + i;
        if (r >= n) break;
        c_row[r + 1] = kvp_add(c_row[r + 1], max(b_row, 0));
        c_new[r + 1] = kvp_add(c_new[r + 1], max(b_new, 0));
        c_old[r + 1] = kvp_add(c_old[r + 1], max(b_old, 0));
    }
    if (tid == 0) c_row[0] = c_new[0] = c_old[0] = 0;
    bad = __syncthreads_or(bad);
    bad |= t_row > A.max_rows || t_old > N || (!bad && end - front + t_old > N);
    const bool few = !bad && t_new > end - front;
    const bool go = !bad && !few;
    const int gt = blockIdx.x * KVP_T + tid, gn = gridDim.x * KVP_T;

    if ((what & 2) && blockIdx.x == 0) {
        /* each thread writes the requests that it read itself */
        for (int i = 0; i < per; i++) {
            const int r = tid * per + i;
            if (r >= n) break;
            const int l = A.len[r], a = A.add[r];
            A.len_out[r] = !go ? l : a < 0 ? 0 : l + a;
        }
        for (int r = tid; A.first && r <= n; r += KVP_T) A.first[r] = go ? c_row[r] : 0;
        if (tid == 0) {
            A.ctl_out[0] = go ? front + t_new : front;
            A.ctl_out[1] = go ? end + t_old : end;
            if (!go) atomicOr(err, few ? ATTN_ERR_PAGES : ATTN_ERR_PLAN);
        }
    }
    if (!(what & 1)) return;
    const int f0 = go ? (int)(front % N) : 0, e0 = go ? (int)(end % N) : 0;
    int lost = 0;
    auto free_page = [&](int i) {                       /* the i-th page taken, -1 if the ring holds no page there */
        const int at = f0 + i - (f0 + i >= N ? N : 0), p = A.ring[at];
        if ((unsigned)p < (unsigned)N) return p;
        lost = 1;
        return -1;
    };
    for (int t = gt; t < A.max_rows; t += gn) {
        int r = -1, pos = -1, slot = -1;
        if (go && t < t_row) {
            r = kvp_find(c_row, n, t);
            const int l = s_len[r];
            pos = l + t - c_row[r];
            const int have = (int)(((int64_t)l + P - 1) >> shift), j = pos >> shift;
            int p;
            if (j >= have) p = free_page(c_new[r] + j - have);
            else {
                p = A.table[(size_t)r * A.max_pages + j];
                if ((unsigned)p >= (unsigned)N) { p = -1; lost = 1; }
            }
            slot = p < 0 ? -1 : (p << shift) + (pos & (P - 1));
        }
        A.row_req[t] = r;
        A.row_pos[t] = pos;
        A.row_slot[t] = slot;
    }
    if (!go) return;
    for (int i = gt; i < t_new; i += gn) {
        const int r = kvp_find(c_new, n, i), have = (int)(((int64_t)s_len[r] + P - 1) >> shift);
        A.table[(size_t)r * A.max_pages + have + i - c_new[r]] = free_page(i);
    }
    for (int i = gt; i < t_old; i += gn) {
        const int r = kvp_find(c_old, n, i);
        const int at = e0 + i, p = A.table[(size_t)r * A.max_pages + i - c_old[r]];
        const bool in = (unsigned)p < (unsigned)N;
        if (!in) lost = 1;
        A.ring[at - (at >= N ? N : 0)] = in ? p : -1;
    }
    if (lost) atomicOr(err, ATTN_ERR_INDEX);
}

extern "C" int roaster_kv_plan(const RoasterKvPlan *p)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!p || p->n_req < 1 || p->n_req > KVP_MAX_REQ || !attn_page_ok(p->page_size) || p->n_pages < 1 ||
        (int64_t)p->n_pages * p->page_size > INT32_MAX || p->max_pages < 1 ||
        (int64_t)p->max_pages * p->page_size > (1 << 30) || p->max_rows < 1 || p->max_rows > KVP_MAX_ROWS)
        return rt_fail(ROASTER_EINVAL, "roaster_kv_plan: need 1 <= n_req <= %d, 1 <= max_rows <= %d, page_size a power of two "
                       "in 16..4096, page_size * n_pages below 2^31, page_size * max_pages at most 2^30", KVP_MAX_REQ, KVP_MAX_ROWS);
    const void *at[] = { p->len, p->add, p->len_out, p->table, p->ring, p->ctl, p->ctl_out,
                         p->row_req, p->row_pos, p->row_slot, p->first };
    const size_t n4 = 4 * (size_t)p->n_req, r4 = 4 * (size_t)p->max_rows;
    const size_t bytes[] = { n4, n4, n4, n4 * p->max_pages, 4 * (size_t)p->n_pages, 16, 16, r4, r4, r4, n4 + 4 };
    for (int i = 0; i < 11; i++) {
        if ((i < 10 && !at[i]) || !attn_aligned(at[i], i == 5 || i == 6 ? 8 : 4))
            return rt_fail(ROASTER_EINVAL, "roaster_kv_plan: argument %d is missing or not aligned", i);
        for (int j = 0; j < i; j++) {
            const bool same = at[i] == at[j] && ((j == 0 && i == 2) || (j == 5 && i == 6));
            if (!same && attn_overlap(at[i], bytes[i], at[j], bytes[j]))
                return rt_fail(ROASTER_EINVAL, "roaster_kv_plan: arguments %d and %d overlap", j, i);
        }
    }
    if (rt_init_locked()) return ROASTER_EDEVICE;
    const AttnDevice dev;
    int *err = rt_attn_err();
    if (!err) return ROASTER_EDEVICE;
    /* a row a thread: a row's search and its page's load are one chain of waits (22700 rows of
     * 512 requests 9.7 us with four rows a thread, 6.9 with one); where the outputs replace
     * inputs that every workgroup reads, one workgroup, or for many rows a second launch for
     * those outputs */
    int blocks = (p->max_rows + KVP_T - 1) / KVP_T;
    if (blocks > 1024) blocks = 1024;
    const bool in_place = p->len_out == p->len || p->ctl_out == p->ctl, two = in_place && blocks > 8;
    if (in_place && !two) blocks = 1;
    int shift = 0;
    while ((1 << shift) < p->page_size) shift++;
    hipLaunchKernelGGL(kv_plan_kernel, dim3(blocks), dim3(KVP_T), 0, rt().stream, *p, shift, two ? 1 : 3, err);
    if (two) hipLaunchKernelGGL(kv_plan_kernel, dim3(1), dim3(KVP_T), 0, rt().stream, *p, shift, 2, err);
    return rt_check(hipGetLastError(), "kv_plan launch") ? ROASTER_EDEVICE : 0;
}
