/*
 * ssm.hip -- selective state space scan with its short causal convolution
 * (roaster_ssm_scan), the recurrent mixer between its projections (model.c:252-323,
 * 1282-1347 one token, 1604-1660 a prompt's chunk).
 *
 * Per value head h, with its key head's unit queries q and keys k, S of [v_dim][k_dim]:
 *   S' = d S,  w = beta (v - S' k),  S = S' + w k^T,  out = scale S q
 * (STATE: w = dt v).  Value elements do not see each other, so any block of them is a
 * scan of its own.
 */
#include "mixer.h"
#include "qdot.h"

#define SSM_T 256

struct SsmArgs {
    RoasterSsmScan a;
    RoasterSsmState s;
    int rep, channels;           /* value heads to a key head; channels of a row */
};

/* A request's rows and first position. */
struct SsmReq { int f0, n, pos; };

/* Whether request r has rows to work on; a bad one's are filled with NaN (`width` elements from `col` on). */
__device__ __forceinline__ bool ssm_request(const SsmArgs &A, int r, int col, int width, SsmReq &q, int *err)
{
    const RoasterSsmScan &a = A.a;
    const int f0 = a.first[r], f1 = a.first[r + 1];
    if (f0 == f1) return false;
    q.f0 = f0;
    q.n = f1 - f0;
    q.pos = -1;
    if (f0 >= 0 && f1 > f0 && f1 <= a.rows && f1 - f0 <= a.most) {
        q.pos = a.row_pos[f0];
        if (q.pos >= 0) return true;
    }
    if (err) {
        if (threadIdx.x == 0) atomicOr(err, ATTN_ERR_SCAN);
        for (int t = max(f0, 0); t < min(f1, a.rows); t++)
            for (int i = threadIdx.x; i < width; i += blockDim.x) a.out[t * a.out_row + col + i] = __uint_as_float(0x7FC00000u);
    }
    return false;
}

__device__ __forceinline__ float ssm_silu(float x) { return x / (1.0f + expf(-x)); }
__device__ __forceinline__ float ssm_softplus(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

/* One channel of the convolution, row by row: the last taps - 1 inputs and the weights. */
struct SsmChannel {
    float h[3], w[4], bias;      /* h[2] the newest; unused taps have weight 0 */

    __device__ __forceinline__ void start(const SsmArgs &A, int r, int pos, int c)
    {
        const int taps = A.s.taps;
        bias = A.a.conv_b ? A.a.conv_b[c] : 0.0f;
        const float *hist = A.s.conv + (size_t)r * taps * A.channels + c;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int back = 3 - j;                    /* positions behind the row */
            w[j] = back < taps ? A.a.conv_w[(size_t)c * taps + taps - 1 - back] : 0.0f;
            if (j < 3) h[j] = back < taps && pos >= back ? hist[(size_t)((unsigned)(pos - back) % taps) * A.channels] : 0.0f;
        }
    }
    __device__ __forceinline__ float next(float x, int taps)
    {
        float c = bias;
        if (taps > 3) c = fmaf(w[0], h[0], c);
        if (taps > 2) c = fmaf(w[1], h[1], c);
        c = fmaf(w[2], h[2], c);
        c = fmaf(w[3], x, c);
        h[0] = h[1];
        h[1] = h[2];
        h[2] = x;
        return ssm_silu(c);
    }
};

/* Token by token: a workgroup has one request's block of VB value elements of one head, its state in
 * registers (KD / 16 lanes a row, 16 elements each).  The queries' and keys' channels are convolved by every
 * workgroup of the head: 2 KD inputs next to VB * KD states.
 * ONE: no request has more than one row, so the entry of `conv` that it fills is none that it reads, and the workgroup writes
 * it; else ssm_conv_kernel does behind this kernel. */
template <int KD, int VB, bool DELTA, bool ONE>
__global__ __launch_bounds__(SSM_T) void ssm_token_kernel(SsmArgs A, int blocks, int *err)
{
    constexpr int P = KD / 16, RP = SSM_T / P, NR = VB / RP;
    __shared__ float s_qk[2][2 * KD], s_v[2][VB], s_sum[2][3][SSM_T / 64];
    const RoasterSsmScan &a = A.a;
    const int tid = threadIdx.x, r = blockIdx.y, h = blockIdx.x / blocks, v0 = blockIdx.x % blocks * VB;
    const int VD = A.s.v_dim, taps = A.s.taps, nk = A.s.k_heads * KD, kh = h / A.rep;
    SsmReq q;
    if (!ssm_request(A, r, h * VD + v0, VB, q, err)) return;
    const bool qk = tid < 2 * KD, val = tid < VB;
    const int cq = tid < KD ? kh * KD + tid : nk + kh * KD + tid - KD, cv = 2 * nk + h * VD + v0 + tid;
    const float *x = a.x + (size_t)q.f0 * a.x_row;
    float xq = qk ? x[cq] : 0.0f, xv = val ? x[cv] : 0.0f;
    float av = a.a[(size_t)q.f0 * a.a_row + h], bv = DELTA ? a.b[(size_t)q.f0 * a.b_row + h] : 0.0f;
    SsmChannel chq, chv;
    if (qk) chq.start(A, r, q.pos, cq);
    if (val) chv.start(A, r, q.pos, cv);
    const int p = tid % P, row = tid / P;
    float *state = A.s.state + (((size_t)r * A.s.v_heads + h) * VD + v0 + row) * KD + 4 * p;
    float4 S[NR][4];
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            S[i][j] = q.pos ? gld_f4(state + (size_t)i * RP * KD + 4 * P * j) : make_float4(0, 0, 0, 0);
    const float coef = a.a_coef[h], dtb = a.dt_bias ? a.dt_bias[h] : 0.0f, skip = a.skip ? a.skip[h] : 0.0f;
    if (ONE) {
        float *to = A.s.conv + ((size_t)r * taps + (unsigned)q.pos % taps) * A.channels;
        if (qk && v0 == 0 && h % A.rep == 0) to[cq] = xq;
        if (val) to[cv] = xv;
    }
    for (int t = 0; t < q.n; t++) {
        const int b = t & 1;
        const float dt = ssm_softplus(av + dtb), decay = expf(coef * dt), gain = DELTA ? 1.0f / (1.0f + expf(-bv)) : dt;
        float cqv = 0.0f;
        if (qk) s_qk[b][tid] = cqv = chq.next(xq, taps);
        if (val) s_v[b][tid] = chv.next(xv, taps);
        if (DELTA) {                                   /* sums of squares; KD is one or two waves' channels */
            float ss = cqv * cqv;
            for (int o = 1; o < 64; o <<= 1) ss += __shfl_xor(ss, o);
            if (tid % 64 == 0) s_sum[b][0][tid / 64] = ss;
        }
        if (!ONE && t + 1 < q.n) {
            const float *xn = x + (size_t)(t + 1) * a.x_row;
            if (qk) xq = xn[cq];
            if (val) xv = xn[cv];
            av = a.a[(size_t)(q.f0 + t + 1) * a.a_row + h];
            if (DELTA) bv = a.b[(size_t)(q.f0 + t + 1) * a.b_row + h];
        }
        __syncthreads();
        float rq = a.scale, rk = 1.0f;
        if (DELTA) {
            const float *s = s_sum[b][0];
            rq = a.scale / sqrtf((KD == 128 ? s[0] + s[1] : s[0]) + a.eps);
            rk = 1.0f / sqrtf((KD == 128 ? s[2] + s[3] : s[1]) + a.eps);
        }
        float4 qf[4], kf[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            qf[j] = *(const float4 *)(s_qk[b] + 4 * (p + P * j));
            kf[j] = *(const float4 *)(s_qk[b] + KD + 4 * (p + P * j));
            qf[j].x *= rq; qf[j].y *= rq; qf[j].z *= rq; qf[j].w *= rq;
            kf[j].x *= rk; kf[j].y *= rk; kf[j].z *= rk; kf[j].w *= rk;
        }
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const float v = s_v[b][row + i * RP];
            float w = gain * v;
            if (DELTA) {
                float sk = 0;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    sk += S[i][j].x * kf[j].x + S[i][j].y * kf[j].y + S[i][j].z * kf[j].z + S[i][j].w * kf[j].w;
                for (int o = 1; o < P; o <<= 1) sk += __shfl_xor(sk, o);
                w = gain * (v - decay * sk);
            }
            float o = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                S[i][j].x = fmaf(w, kf[j].x, decay * S[i][j].x);
                S[i][j].y = fmaf(w, kf[j].y, decay * S[i][j].y);
                S[i][j].z = fmaf(w, kf[j].z, decay * S[i][j].z);
                S[i][j].w = fmaf(w, kf[j].w, decay * S[i][j].w);
                o += S[i][j].x * qf[j].x + S[i][j].y * qf[j].y + S[i][j].z * qf[j].z + S[i][j].w * qf[j].w;
            }
            for (int u = 1; u < P; u <<= 1) o += __shfl_xor(o, u);
            if (p == 0) a.out[(size_t)(q.f0 + t) * a.out_row + h * VD + v0 + row + i * RP] = a.skip ? fmaf(skip, v, o) : o;
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) *(float4 *)(state + (size_t)i * RP * KD + 4 * P * j) = S[i][j];
}

/* The inputs of each request's last positions into its entries of `conv`. */
__global__ __launch_bounds__(SSM_T) void ssm_conv_kernel(SsmArgs A)
{
    SsmReq q;
    const int r = blockIdx.y, c = 4 * (blockIdx.x * SSM_T + threadIdx.x), taps = A.s.taps;
    if (!ssm_request(A, r, 0, 0, q, nullptr) || c >= A.channels) return;
    for (int t = max(0, q.n - taps); t < q.n; t++)
        *(float4 *)(A.s.conv + ((size_t)r * taps + ((unsigned)q.pos + t) % taps) * A.channels + c) =
            gld_f4(A.a.x + (size_t)(q.f0 + t) * A.a.x_row + c);
}

static bool ssm_state_ok(const RoasterSsmState *s)
{
    return s && s->n_req >= 1 && s->n_req <= 2048 && s->k_heads >= 1 && s->v_heads >= s->k_heads && s->v_heads <= 256 &&
           s->v_heads % s->k_heads == 0 && (s->k_dim == 64 || s->k_dim == 128) && (s->v_dim == 64 || s->v_dim == 128) &&
           s->taps >= 2 && s->taps <= 4;
}

static inline int ssm_channels(const RoasterSsmState *s) { return 2 * s->k_heads * s->k_dim + s->v_heads * s->v_dim; }

extern "C" size_t roaster_ssm_ws_bytes(int rows, int most, const RoasterSsmState *s)
{
    if (!ssm_state_ok(s) || rows < 0 || rows > (1 << 18) || most < 1 || (rows && most > rows)) return 0;
    return 16;
}

extern "C" int roaster_ssm_scan(const RoasterSsmScan *p, const RoasterSsmState *s)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!ssm_state_ok(s) || !s->conv || !s->state || !attn_aligned(s->conv, 16) || !attn_aligned(s->state, 16))
        return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: bad state description (1 <= n_req <= 2048, v_heads a multiple of k_heads up to "
                       "256, k_dim and v_dim 64 or 128, 2 to 4 taps, conv and state 16-byte aligned)");
    if (!p || p->rows < 0 || p->rows > (1 << 18) || p->most < 1 || (p->rows && p->most > p->rows) ||
        (p->mode != ROASTER_SCAN_DELTA && p->mode != ROASTER_SCAN_STATE))
        return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: need 0 <= rows <= 262144, 1 <= most <= rows, mode ROASTER_SCAN_DELTA or _STATE");
    if (!p->rows) return 0;
    const bool delta = p->mode == ROASTER_SCAN_DELTA;
    const size_t rows = p->rows, vh = s->v_heads, ch = ssm_channels(s), ov = vh * s->v_dim, n = s->n_req;
    if (!p->x || !p->a || (delta && !p->b) || !p->conv_w || !p->a_coef || !p->first || !p->row_pos || !p->out || !p->ws)
        return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: x, a, b (DELTA), conv_w, a_coef, first, row_pos, out and ws must be given");
    const float *b = delta ? p->b : NULL;
    const void *four[] = { p->a, b, p->conv_b, p->a_coef, p->dt_bias, p->skip, p->first, p->row_pos };
    for (const void *q : four)
        if (!attn_aligned(q, 4)) return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: tensors are 4-byte aligned");
    if (!attn_aligned(p->x, 16) || !attn_aligned(p->conv_w, 16) || !attn_aligned(p->out, 16) || !attn_aligned(p->ws, 16))
        return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: x, conv_w, out and ws are 16-byte aligned");
    if (!stride_ok(p->x_row, 4) || !stride_ok(p->a_row, 1) || (delta && !stride_ok(p->b_row, 1)) || !stride_ok(p->out_row, 4) ||
        p->out_row < ov)
        return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: strides are at most 2^32, of x and out multiples of 4, of out at least "
                       "v_heads * v_dim");
    const size_t need = roaster_ssm_ws_bytes(p->rows, p->most, s);
    if (p->ws_bytes < need) return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: workspace of %zu bytes, %zu needed", p->ws_bytes, need);
    const void *out[] = { p->out, s->conv, s->state, p->ws };
    const size_t no[] = { rows_span(rows, ov, p->out_row, 4), 4 * n * s->taps * ch, 4 * n * ov * s->k_dim, need };
    const void *in[] = { p->x, p->a, b, p->conv_w, p->conv_b, p->a_coef, p->dt_bias, p->skip, p->first, p->row_pos };
    const size_t ni[] = { rows_span(rows, ch, p->x_row, 4), rows_span(rows, vh, p->a_row, 4), rows_span(rows, vh, p->b_row, 4),
                          4 * ch * s->taps, 4 * ch, 4 * vh, 4 * vh, 4 * vh, 4 * (n + 1), 4 * rows };
    for (int i = 0; i < 4; i++) {
        for (int j = 0; j < 10; j++)
            if (attn_overlap(out[i], no[i], in[j], ni[j])) return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: outputs overlap inputs");
        for (int j = 0; j < i; j++)
            if (attn_overlap(out[i], no[i], out[j], no[j])) return rt_fail(ROASTER_EINVAL, "roaster_ssm_scan: outputs overlap");
    }
    if (rt_init_locked()) return ROASTER_EDEVICE;
    const AttnDevice dev;
    int *err = rt_attn_err();
    if (!err) return ROASTER_EDEVICE;
    SsmArgs A = { *p, *s, s->v_heads / s->k_heads, (int)ch };
    A.a.b = b;
    const bool one = p->most == 1;
#define TOKEN3(KD, VB, D, O)                                                                                              \
    hipLaunchKernelGGL((ssm_token_kernel<KD, VB, D, O>), dim3(vh * (s->v_dim / VB), n), dim3(SSM_T), 0, rt().stream, A,    \
                       s->v_dim / VB, err)
#define TOKEN2(KD, VB, D) do { if (one) TOKEN3(KD, VB, D, true); else TOKEN3(KD, VB, D, false); } while (0)
#define TOKEN(KD, VB) do { if (delta) TOKEN2(KD, VB, true); else TOKEN2(KD, VB, false); } while (0)
    if (s->k_dim == 128) TOKEN(128, 32);
    else TOKEN(64, 64);
#undef TOKEN
#undef TOKEN2
#undef TOKEN3
    if (rt_check(hipGetLastError(), "ssm_token launch")) return ROASTER_EDEVICE;
    if (!one) {
        hipLaunchKernelGGL(ssm_conv_kernel, dim3((ch / 4 + SSM_T - 1) / SSM_T, n), dim3(SSM_T), 0, rt().stream, A);
        if (rt_check(hipGetLastError(), "ssm_conv launch")) return ROASTER_EDEVICE;
    }
    return 0;
}
