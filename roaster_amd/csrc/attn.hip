/*
 * attn.hip -- softmax attention of new rows over a paged key/value cache
 * (roaster_attn_paged; model.c:755-863, 1536-1602).
 */
#include "attn.h"
#include "qdot.h"

#define ATT_T 256

struct AttArgs {
    RoasterAttnPaged a;
    const void *kc, *vc;
    KvShape s;
};

template <bool F16>
__device__ __forceinline__ float att_at(const void *c, size_t i)
{
    return F16 ? (float)((const _Float16 *)c)[i] : ((const float *)c)[i];
}

/* One workgroup per row and query head; its waves take the row's positions in
 * turn, each with its own running maximum and sum, and join them at the end. */
template <int D, bool F16>
__global__ __launch_bounds__(ATT_T) void attn_kernel(AttArgs A, int *err)
{
    constexpr int N = D / 64, W = ATT_T / 64;
    __shared__ float s_m[W], s_l[W], s_o[W][D];
    __shared__ bool s_bad[W];
    const RoasterAttnPaged &a = A.a;
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int r = a.row_req[t];
    if (r == -1) return;
    const KvTable T = { a.n_req, a.max_pages };
    const int n = T.tokens(r, a.row_pos[t], A.s.shift), kh = h / (a.q_heads / A.s.kv);
    bool bad = n < 0;
    const float *q = a.q + ((size_t)t * a.q_heads + h) * D + lane * N;
    float qv[N], o[N] = {}, m = -INFINITY, sum = 0;
    for (int i = 0; i < N; i++) qv[i] = q[i] * a.scale;
    for (int j = w; j < n; j += W) {
        const int p = a.table[T.entry(r, j, A.s.shift)];
        if (!A.s.page_ok(p)) { bad = true; break; }
        const size_t at = A.s.at(p, kh, j & ((1 << A.s.shift) - 1)) + lane * N;
        float s = 0;
        for (int i = 0; i < N; i++) s = fmaf(qv[i], att_at<F16>(A.kc, at + i), s);
        s = group_sum<64>(s);
        const float mn = s == s ? fmaxf(m, s) : s;             /* a NaN score stays one */
        const float c = mn == -INFINITY ? 1.0f : expf(m - mn), e = mn == -INFINITY ? 0.0f : expf(s - mn);
        sum = sum * c + e;
        for (int i = 0; i < N; i++) o[i] = fmaf(e, att_at<F16>(A.vc, at + i), o[i] * c);
        m = mn;
    }
    if (lane == 0) { s_m[w] = m; s_l[w] = sum; s_bad[w] = bad; }
    for (int i = 0; i < N; i++) s_o[w][lane * N + i] = o[i];
    __syncthreads();
    float mx = -INFINITY, l = 0;
    bool any = false;                                       /* some wave met an index out of range */
    for (int i = 0; i < W; i++) any |= s_bad[i];
    for (int i = 0; i < W; i++) mx = fmaxf(mx, s_m[i]);
    for (int i = 0; i < W; i++) l += s_m[i] == -INFINITY ? 0.0f : s_l[i] * expf(s_m[i] - mx);
    if (any && threadIdx.x == 0) atomicOr(err, ATTN_ERR_INDEX);
    for (int d = threadIdx.x; d < D; d += ATT_T) {
        float y = 0;
        for (int i = 0; i < W; i++) y += s_m[i] == -INFINITY ? 0.0f : s_o[i][d] * expf(s_m[i] - mx);
        y = any ? NAN : l == 0 ? 0.0f : y / l;
        if (a.gate) y /= 1.0f + expf(-a.gate[t * a.gate_row + h * a.gate_head + d]);
        a.out[((size_t)t * a.q_heads + h) * D + d] = y;
    }
}

extern "C" size_t roaster_attn_ws_bytes(int rows, int q_heads, const RoasterKvCache *c)
{
    if (!attn_cache_ok(c) || rows < 0 || rows > (1 << 20) || q_heads < 1 || q_heads > 1024 || q_heads % c->kv_heads) return 0;
    return 256;
}

extern "C" int roaster_attn_paged(const RoasterAttnPaged *p, const RoasterKvCache *c)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!attn_cache_ok(c)) return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: bad cache description");
    if (!p || p->rows < 0 || p->rows > (1 << 20) || p->q_heads < 1 || p->q_heads > 1024 || p->q_heads % c->kv_heads ||
        p->n_req < 1 || p->max_pages < 1 || (int64_t)p->max_pages * c->page_size > INT32_MAX || !(fabsf(p->scale) < INFINITY))
        return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: need 0 <= rows <= 2^20, q_heads a multiple of kv_heads up to 1024, "
                       "n_req >= 1, max_pages * page_size below 2^31, a finite scale");
    if (!p->rows) return 0;
    if (!p->q || !p->out || !p->row_req || !p->row_pos || !p->table || !attn_aligned(p->q, 16) || !attn_aligned(p->out, 16) ||
        !attn_aligned(p->row_req, 4) || !attn_aligned(p->row_pos, 4) || !attn_aligned(p->table, 4) ||
        !attn_aligned(p->gate, 16) || (p->gate && (p->gate_row % 4 || p->gate_head % 4 ||
        p->gate_row > ((size_t)1 << 32) || p->gate_head > ((size_t)1 << 32))))
        return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: q, out, rows and table must be given; q, out and gate 16-byte "
                       "aligned, gate strides multiples of 4 floats");
    const size_t need = roaster_attn_ws_bytes(p->rows, p->q_heads, c), D = c->head_dim;
    if (!p->ws || !attn_aligned(p->ws, 16) || p->ws_bytes < need)
        return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: the workspace needs %zu bytes, 16-byte aligned", need);
    const size_t rows = p->rows, nq = 4 * rows * p->q_heads * D, nc = attn_cache_bytes(c);
    const void *in[] = { p->q, p->row_req, p->row_pos, p->table, p->gate, c->k, c->v };
    const size_t ni[] = { nq, 4 * rows, 4 * rows, 4 * (size_t)p->n_req * p->max_pages,
                          4 * ((rows - 1) * p->gate_row + (p->q_heads - 1) * p->gate_head + D), nc, nc };
    for (int i = 0; i < 7; i++)
        if (attn_overlap(p->out, nq, in[i], ni[i]) || attn_overlap(p->ws, need, in[i], ni[i]))
            return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: out or the workspace overlaps an input");
    if (attn_overlap(p->out, nq, p->ws, need)) return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: out overlaps the workspace");
    if (rt_init_locked()) return ROASTER_EDEVICE;
    const AttnDevice dev;
    int *err = rt_attn_err();
    if (!err) return ROASTER_EDEVICE;
    const AttArgs A = { *p, c->k, c->v, attn_shape(c) };
    const dim3 gd(p->rows, p->q_heads), bd(ATT_T);
#define ATT(DD, H) hipLaunchKernelGGL((attn_kernel<DD, H>), gd, bd, 0, rt().stream, A, err)
    if (c->type == ROASTER_KV_F16) {
        if (D == 256) ATT(256, true);
        else if (D == 128) ATT(128, true);
        else ATT(64, true);
    } else {
        if (D == 256) ATT(256, false);
        else if (D == 128) ATT(128, false);
        else ATT(64, false);
    }
#undef ATT
    return rt_check(hipGetLastError(), "attention launch") ? ROASTER_EDEVICE : 0;
}
