/*
 * qk_rope.hip -- per-head norms of queries and keys, the position rotation and
 * the store of keys and values into the cache pages, in one pass
 * (roaster_qk_rope_store; model.c:755-863, 1536-1602 do these steps per head).
 */
#include "attn.h"
#include "qdot.h"

#define QKR_T 256

struct QkrArgs {
    RoasterQkRope a;
    void *kc, *vc;
    KvShape s;
    double dec;                     /* log2 of theta^(2 / rot_dim): frequency i is 2^(-i dec) */
};

/* cos and sin of pos * 2^(-i dec).  The angle is formed and reduced to
 * [-pi/4, pi/4] in 64 bits (in 32 it would be off by 2^-24 of pos radians),
 * the Taylor sums of the reduced angle in 32: their next terms are below
 * 7e-9 (r^11 / 11!, r^12 / 12!). */
__device__ __forceinline__ float2 qkr_turn(int pos, int i, double dec)
{
    const double a = (double)pos * exp2(-(double)i * dec);
    const double k = rint(a * 0.63661977236758134308);             /* 2 / pi */
    double rd = fma(-k, 1.57079632679489655800, a);                 /* pi / 2 in two parts */
    rd = fma(-k, 6.12323399573676603587e-17, rd);
    const int quad = (int)((long long)k & 3);
    const float r = (float)rd, z = r * r;
    const float s = r + r * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const float cc = quad & 1 ? s : c, ss = quad & 1 ? c : s;
    return make_float2(quad == 1 || quad == 2 ? -cc : cc, quad & 2 ? -ss : ss);
}

/* A head of D elements is D/4 lanes with four elements each, a workgroup takes
 * one row's heads 4 waves at a time, queries first, then keys, then values; the
 * next heads are loaded while these are worked on.  What bounds it: a row's launch and
 * one wait for its slot, elements and weights up to some hundred rows (4 us), then
 * memory: 2048 rows of 20 heads of 256 15.7 us, 5.1 TB/s of a copy's 4.8 (the caches
 * take part), 4000 rows of 24 heads of 128 14.7 us, 5.6 TB/s. */
template <int D, bool F16>
__global__ __launch_bounds__(QKR_T) void qk_rope_kernel(QkrArgs A, int per, int *err)
{
    __shared__ float s_cos[D / 2], s_sin[D / 2];
    constexpr int L = D / 4, HPW = QKR_T / L;              /* lanes of a head, heads at a time */
    const RoasterQkRope &a = A.a;
    const int t = blockIdx.x, tid = threadIdx.x, l = tid % L, rot = a.rot_dim, half = rot / 2;
    const int slot = a.row_slot[t];
    if (slot < 0) return;
    if (!A.s.slot_ok(slot)) {
        if (tid == 0 && blockIdx.y == 0) atomicOr(err, ATTN_ERR_INDEX);
        return;
    }
    const int nq = a.q_heads, nqk = nq + A.s.kv, nh = nqk + A.s.kv;
    const int h0 = blockIdx.y * per * HPW + tid / L, h1 = min(nh, (int)(blockIdx.y + 1) * per * HPW);
    auto src = [&](int h) {
        const float *p = h < nq ? a.q + t * a.q_row + h * a.q_head
                       : h < nqk ? a.k + t * a.k_row + (h - nq) * a.k_head
                                 : a.v + t * a.v_row + (h - nqk) * a.v_head;
        return *(const float4 *)(p + 4 * l);
    };
    float4 x = h0 < h1 ? src(h0) : make_float4(0, 0, 0, 0);
    if ((int)blockIdx.y * per * HPW < nqk) {
        for (int i = tid; i < half; i += QKR_T) {
            const float2 cs = qkr_turn(a.row_pos[t], i, A.dec);
            s_cos[i] = cs.x;
            s_sin[i] = cs.y;
        }
    }
    __syncthreads();
    for (int h = h0; h < h1; h += HPW) {
        const float4 y = x;
        if (h + HPW < h1) x = src(h + HPW);
        float v[4] = { y.x, y.y, y.z, y.w };
        if (h < nqk) {                                     /* a wave may hold heads of both kinds: the lane exchanges stay within a head */
            const float *w = h < nq ? a.q_norm : a.k_norm;
            if (w) {
                float ss = v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3];
                for (int o = 1; o < L; o <<= 1) ss += __shfl_xor(ss, o);
                const float inv = 1.0f / sqrtf(ss / D + a.eps);
                const float4 g = *(const float4 *)(w + 4 * l);
                v[0] *= inv * g.x; v[1] *= inv * g.y; v[2] *= inv * g.z; v[3] *= inv * g.w;
            }
            if (a.pair_adjacent) {
                if (4 * l < rot)
                    for (int j = 0; j < 2; j++) {
                        const float c = s_cos[2 * l + j], s = s_sin[2 * l + j], p = v[2 * j], q = v[2 * j + 1];
                        v[2 * j] = p * c - q * s;
                        v[2 * j + 1] = q * c + p * s;
                    }
            } else {
                const int d = rot / 8, other = l < d ? l + d : l - d;     /* the lane with the pair's other elements */
                float o[4];
                for (int j = 0; j < 4; j++) o[j] = __shfl(v[j], other, L);
                if (l < 2 * d)
                    for (int j = 0; j < 4; j++) {
                        const int i = 4 * (l < d ? l : other) + j;
                        const float c = s_cos[i], s = s_sin[i];
                        v[j] = l < d ? v[j] * c - o[j] * s : v[j] * c + o[j] * s;
                    }
            }
        }
        if (h < nq) *(float4 *)(a.q_out + ((size_t)t * nq + h) * D + 4 * l) = make_float4(v[0], v[1], v[2], v[3]);
        else {
            const int kh = h < nqk ? h - nq : h - nqk;
            const size_t at = A.s.at_slot(slot, kh) + 4 * l;
            void *to = h < nqk ? A.kc : A.vc;
            if (F16) {
                _Float16 r[4];
                for (int j = 0; j < 4; j++) r[j] = (_Float16)v[j];
                *(uint2 *)((_Float16 *)to + at) = __builtin_bit_cast(uint2, *(gu32x2 *)r);
            } else *(float4 *)((float *)to + at) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

extern "C" int roaster_qk_rope_store(const RoasterQkRope *p, const RoasterKvCache *c)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!attn_cache_ok(c)) return rt_fail(ROASTER_EINVAL, "roaster_qk_rope_store: bad cache description");
    const int D = c->head_dim;
    if (!p || p->rows < 0 || p->rows > (1 << 20) || p->q_heads < 1 || p->q_heads > 1024 || p->rot_dim < 0 ||
        p->rot_dim > D || p->rot_dim % 8 || !(p->theta >= 1) || !(p->theta <= 1e30))
        return rt_fail(ROASTER_EINVAL, "roaster_qk_rope_store: need 0 <= rows <= 2^20, 1 <= q_heads <= 1024, rot_dim a multiple "
                       "of 8 up to head_dim, 1 <= theta <= 1e30");
    if (!p->rows) return 0;
    const void *at[] = { p->q, p->k, p->v, p->q_out };
    const size_t str[] = { p->q_row, p->q_head, p->k_row, p->k_head, p->v_row, p->v_head };
    for (int i = 0; i < 4; i++)
        if (!at[i] || !attn_aligned(at[i], 16))
            return rt_fail(ROASTER_EINVAL, "roaster_qk_rope_store: q, k, v and q_out must be given and 16-byte aligned");
    for (int i = 0; i < 6; i++)
        if (str[i] % 4 || str[i] > ((size_t)1 << 32))
            return rt_fail(ROASTER_EINVAL, "roaster_qk_rope_store: strides are multiples of 4 floats");
    if (!p->row_pos || !p->row_slot || !attn_aligned(p->row_pos, 4) || !attn_aligned(p->row_slot, 4) ||
        !attn_aligned(p->q_norm, 16) || !attn_aligned(p->k_norm, 16))
        return rt_fail(ROASTER_EINVAL, "roaster_qk_rope_store: row_pos and row_slot must be given, the norms 16-byte aligned");
    const size_t rows = p->rows, qh = p->q_heads, kh = c->kv_heads, nq = 4 * rows * qh * D, nc = attn_cache_bytes(c);
    auto span = [&](size_t row, size_t head, size_t heads) { return 4 * ((rows - 1) * row + (heads - 1) * head + D); };
    const void *in[] = { p->q, p->k, p->v, p->q_norm, p->k_norm, p->row_pos, p->row_slot };
    const size_t ni[] = { span(p->q_row, p->q_head, qh), span(p->k_row, p->k_head, kh), span(p->v_row, p->v_head, kh),
                          4 * (size_t)D, 4 * (size_t)D, 4 * rows, 4 * rows };
    const bool in_place = p->q_out == p->q && p->q_head == (size_t)D && p->q_row == qh * D;
    for (int i = 0; i < 7; i++)
        if (attn_overlap(c->k, nc, in[i], ni[i]) || attn_overlap(c->v, nc, in[i], ni[i]) ||
            (!(i == 0 && in_place) && attn_overlap(p->q_out, nq, in[i], ni[i])))
            return rt_fail(ROASTER_EINVAL, "roaster_qk_rope_store: outputs overlap inputs");
    if (attn_overlap(c->k, nc, c->v, nc) || attn_overlap(c->k, nc, p->q_out, nq) || attn_overlap(c->v, nc, p->q_out, nq))
        return rt_fail(ROASTER_EINVAL, "roaster_qk_rope_store: outputs overlap");
    if (rt_init_locked()) return ROASTER_EDEVICE;
    const AttnDevice dev;
    int *err = rt_attn_err();
    if (!err) return ROASTER_EDEVICE;
    QkrArgs A;
    A.a = *p;
    A.kc = c->k;
    A.vc = c->v;
    A.s = attn_shape(c);
    A.dec = p->rot_dim ? 2.0 * log2(p->theta) / p->rot_dim : 0.0;
    const int hpw = QKR_T / (D / 4), nh = p->q_heads + 2 * c->kv_heads, waves = (nh + hpw - 1) / hpw;
    /* many rows: a row's heads by one workgroup, which turns its angles once; few: every
     * four waves' heads by their own (20 heads of 256, 1 row 3.4 us against 5.9 in one workgroup,
     * 512 rows 7.3 against 8.3, 1024 rows 10.7 against 10.1, 2048 17.4 against 15.7) */
    const int per = p->rows >= 768 ? waves : 1;
    const dim3 gd(p->rows, (waves + per - 1) / per), bd(QKR_T);
#define QKR(DD, H) hipLaunchKernelGGL((qk_rope_kernel<DD, H>), gd, bd, 0, rt().stream, A, per, err)
    if (c->type == ROASTER_KV_F16) {
        if (D == 256) QKR(256, true);
        else if (D == 128) QKR(128, true);
        else QKR(64, true);
    } else {
        if (D == 256) QKR(256, false);
        else if (D == 128) QKR(128, false);
        else QKR(64, false);
    }
#undef QKR
    return rt_check(hipGetLastError(), "qk_rope launch") ? ROASTER_EDEVICE : 0;
}
