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

/* ---- prompts: 64 tokens at a time -------------------------------------------------
 *
 * Within a chunk, G_i = sum of a_coef dt up to token i and D_ij = exp(G_i - G_j) for j <= i:
 *   A_ij = beta_i D_ij k_i.k_j (j < i),   T = (1 + A)^-1 diag(beta)
 *   W = T (V - exp(G) K S)                the w of all tokens
 *   out = exp(G) Q S + (D o Q K^T) W,     S = exp(G_63) S + K^T (exp(G_63 - G) W)
 * (STATE: W = dt V).  ssm_prep_kernel makes what does not need S for all chunks at once, ssm_chunk_kernel
 * goes through a request's chunks with a block of 16 value elements.  Both multiply on
 * v_mfma_f32_16x16x4_f32:
 *   A[m][k]: lane l holds m = l%16, k = l/16     B[k][n]: k = l/16, n = l%16
 *   D[m][n]: lane l holds m = 4*(l/16) + i, n = l%16, i = 0..3
 * four of them over 16 columns, the lane's four being 4*(l/16) .. + 3, so that an operand is
 * one 16-byte piece of a lane and a kilobyte of a wave; the workspace holds all operands so.
 * Tokens behind a request's last are zeros with gain 0 and the decay of the last. */
#define SSM_C 64                 /* tokens of a chunk */
#define SSM_HG 2                 /* value heads of a workgroup of ssm_prep_kernel */

typedef float f32x4 __attribute__((ext_vector_type(4)));

/* Workspace, in floats: of a chunk and key head the operands of Q and K (tokens as rows) and K^T, of a chunk and value
 * head those of T and D o Q K^T, then exp(G), exp(G_63 - G), gain and a_coef dt of its tokens, and a
 * word that tells whether some of it is infinite or NaN. */
struct SsmWs {
    float *p;
    int kd, kh, vh;

    __host__ __device__ size_t key_floats() const { return 3 * (size_t)SSM_C * kd; }
    __host__ __device__ size_t head_floats() const { return 2 * SSM_C * SSM_C + 5 * SSM_C; }
    __host__ __device__ size_t chunk_floats() const { return kh * key_floats() + vh * head_floats(); }
    __device__ float *key(int c, int h) const { return p + c * chunk_floats() + h * key_floats(); }
    __device__ float *head(int c, int h) const { return p + c * chunk_floats() + kh * key_floats() + h * head_floats(); }
};

/* Chunks of request r, 0 for one that is idle or left out. */
__device__ __forceinline__ int ssm_chunks(const SsmArgs &A, int r)
{
    if (r >= A.s.n_req) return 0;
    const int f0 = A.a.first[r], f1 = A.a.first[r + 1];
    if (f0 < 0 || f1 <= f0 || f1 > A.a.rows || f1 - f0 > A.a.most || A.a.row_pos[f0] < 0) return 0;
    return (f1 - f0 + SSM_C - 1) / SSM_C;
}

/* The request of chunk c and the chunk's number in it; a wave's lanes together.  -1 behind the last chunk. */
__device__ __forceinline__ int ssm_find(const SsmArgs &A, int c, int &of)
{
    const int l = threadIdx.x % 64;
    int base = 0;
    for (int r0 = 0; r0 < A.s.n_req; r0 += 64) {
        const int n = ssm_chunks(A, r0 + l);
        int end = n;
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(end, o);
            if (l >= o) end += v;
        }
        const unsigned long long hit = __ballot(c >= base + end - n && c < base + end);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            of = c - base - __shfl(end - n, at);
            return r0 + at;
        }
        base += __shfl(end, 63);
    }
    return -1;
}

/* Chunks of the requests before r. */
__device__ __forceinline__ int ssm_base(const SsmArgs &A, int r)
{
    int base = 0;
    for (int r0 = threadIdx.x % 64; r0 < r; r0 += 64) base += ssm_chunks(A, r0);
    for (int o = 1; o < 64; o <<= 1) base += __shfl_xor(base, o);
    return base;
}

__device__ __forceinline__ f32x4 ssm_mfma4(float4 a, float4 b, f32x4 c)
{
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
}

__device__ __forceinline__ float4 f4(f32x4 v) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ bool ssm_finite(float x) { return fabsf(x) < INFINITY; }

/* A chunk's tokens of one key head: convolution, norms, the products among tokens, and of SSM_HG of its value
 * heads the decays and T.  Waves 0 and 1 make a head's T each, by forward substitution with a column a lane,
 * waves 2 and 3 its D o Q K^T. */
template <int KD, bool DELTA>
__global__ __launch_bounds__(SSM_T) void ssm_prep_kernel(SsmArgs A, SsmWs W, int groups)
{
    constexpr int LD = KD + 4, LG = SSM_C + 4, G16 = KD / 16;
    constexpr int F0 = 2 * SSM_C * LD, F1 = (2 + SSM_HG) * SSM_C * LG;
    __shared__ __attribute__((aligned(16))) float s_buf[F0 > F1 ? F0 : F1];
    __shared__ double s_G[4][SSM_C];
    __shared__ int s_bad;
    const RoasterSsmScan &a = A.a;
    const int tid = threadIdx.x, l = tid % 64, w = tid / 64, taps = A.s.taps;
    const int kh = blockIdx.y / groups, hg = blockIdx.y % groups, nk = A.s.k_heads * KD;
    int of;
    const int r = ssm_find(A, blockIdx.x, of);
    if (r < 0) return;
    const int f0 = a.first[r], n = a.first[r + 1] - f0, pos = a.row_pos[f0], i0 = of * SSM_C, width = min(SSM_C, n - i0);
    float *s_q = s_buf, *s_k = s_buf + SSM_C * LD;
    if (tid == 0) s_bad = 0;

    {   /* convolution: a channel a thread, all its rows (KD 64: half of them) in order */
        constexpr int RG = SSM_C * 2 * KD / SSM_T;
        const int ch = tid % (2 * KD), j0 = tid / (2 * KD) * RG, c = ch < KD ? kh * KD + ch : nk + kh * KD + ch - KD;
        const float *x = a.x + (size_t)(f0 + i0) * a.x_row + c;
        SsmChannel cv;
        cv.start(A, r, pos, c);
        if (i0 + j0) {                                  /* rows before: at least 32 */
#pragma unroll
            for (int j = 0; j < 3; j++) cv.h[j] = j0 - 3 + j < width ? x[((ptrdiff_t)j0 - 3 + j) * (ptrdiff_t)a.x_row] : 0.0f;
        }
        float *to = (ch < KD ? s_q + ch : s_k + ch - KD) + j0 * LD;
        for (int j = 0; j < RG; j += 16) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = j0 + j + i < width ? x[(size_t)(j0 + j + i) * a.x_row] : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float y = cv.next(v[i], taps);
                to[(j + i) * LD] = j0 + j + i < width ? y : 0.0f;
            }
        }
    }
    __syncthreads();
    {   /* norms: four threads a row */
        const int row = tid / 4;
        float sq = 0, sk = 0;
        float4 q[KD / 16], k[KD / 16];
#pragma unroll
        for (int j = 0; j < KD / 16; j++) {
            q[j] = *(const float4 *)(s_q + row * LD + 4 * (tid % 4 + 4 * j));
            k[j] = *(const float4 *)(s_k + row * LD + 4 * (tid % 4 + 4 * j));
            sq += q[j].x * q[j].x + q[j].y * q[j].y + q[j].z * q[j].z + q[j].w * q[j].w;
            sk += k[j].x * k[j].x + k[j].y * k[j].y + k[j].z * k[j].z + k[j].w * k[j].w;
        }
        for (int o = 1; o < 4; o <<= 1) { sq += __shfl_xor(sq, o); sk += __shfl_xor(sk, o); }
        if (!ssm_finite(sq) || !ssm_finite(sk)) s_bad = 1;
        const float rq = DELTA ? a.scale / sqrtf(sq + a.eps) : a.scale, rk = DELTA ? 1.0f / sqrtf(sk + a.eps) : 1.0f;
#pragma unroll
        for (int j = 0; j < KD / 16; j++) {
            *(float4 *)(s_q + row * LD + 4 * (tid % 4 + 4 * j)) = make_float4(q[j].x * rq, q[j].y * rq, q[j].z * rq, q[j].w * rq);
            *(float4 *)(s_k + row * LD + 4 * (tid % 4 + 4 * j)) = make_float4(k[j].x * rk, k[j].y * rk, k[j].z * rk, k[j].w * rk);
        }
    }
    __syncthreads();
    if (hg == 0) {
        float4 *q = (float4 *)W.key(blockIdx.x, kh), *k = q + SSM_C * KD / 4, *kt = k + SSM_C * KD / 4;
        for (int f = tid; f < SSM_C * KD / 4; f += SSM_T) {
            const int g = f / 64 % G16, m = f / 64 / G16 * 16 + f % 16, at = m * LD + 16 * g + 4 * (f % 64 / 16);
            q[f] = *(const float4 *)(s_q + at);
            k[f] = *(const float4 *)(s_k + at);
        }
        for (int f = tid; f < SSM_C * KD / 4; f += SSM_T) {
            const float *at = s_k + (f / 64 % 4 * 16 + 4 * (f % 64 / 16)) * LD + f / 256 * 16 + f % 16;
            kt[f] = make_float4(at[0], at[LD], at[2 * LD], at[3 * LD]);
        }
    }
    /* products of tokens, lower blocks alone: wave w has rows 16 w of K K^T and rows 16 (3 - w) of Q K^T */
    f32x4 kk[4] = {}, qk[4] = {};
    const int wq = 3 - w;
    for (int g = 0; g < G16; g++) {
        const int col = 16 * g + 4 * (l / 16);
        const float4 ak = *(const float4 *)(s_k + (16 * w + l % 16) * LD + col), aq = *(const float4 *)(s_q + (16 * wq + l % 16) * LD + col);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            if (b > w && b > wq) continue;
            const float4 bk = *(const float4 *)(s_k + (16 * b + l % 16) * LD + col);
            if (DELTA && b <= w) kk[b] = ssm_mfma4(ak, bk, kk[b]);
            if (b <= wq) qk[b] = ssm_mfma4(aq, bk, qk[b]);
        }
    }
    __syncthreads();
    float *s_kk = s_buf, *s_qk = s_buf + SSM_C * LG;
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (DELTA && b <= w) s_kk[(16 * w + 4 * (l / 16) + i) * LG + 16 * b + l % 16] = kk[b][i];
            if (b <= wq) s_qk[(16 * wq + 4 * (l / 16) + i) * LG + 16 * b + l % 16] = qk[b][i];
        }
    __syncthreads();
    const int hh = hg * SSM_HG + w % SSM_HG, h = kh * A.rep + hh;
    if (hh >= A.rep) return;
    /* a token a lane */
    const bool in = l < width;
    const size_t row = (size_t)(f0 + i0 + l);
    const float dt = in ? ssm_softplus(a.a[row * a.a_row + h] + (a.dt_bias ? a.dt_bias[h] : 0.0f)) : 0.0f;
    const float gl = in ? a.a_coef[h] * dt : 0.0f;
    const float gain = !in ? 0.0f : DELTA ? 1.0f / (1.0f + expf(-a.b[row * a.b_row + h])) : dt;
    double G = gl;
    for (int o = 1; o < 64; o <<= 1) {
        const double v = __shfl_up(G, o);
        if (l >= o) G += v;
    }
    s_G[w][l] = G;
    const double last = __shfl(G, 63);
    float *out = W.head(blockIdx.x, h);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (w >= SSM_HG) {                                  /* D o Q K^T, in the operands' order */
        for (int m = 0; m < 4; m++)
            for (int g = 0; g <= m; g++) {
                const int i = 16 * m + l % 16, j = 16 * g + 4 * (l / 16);
                const float4 p = *(const float4 *)(s_qk + i * LG + j);
                const float v[4] = { p.x, p.y, p.z, p.w };
                f32x4 d;
#pragma unroll
                for (int c = 0; c < 4; c++) d[c] = j + c <= i ? v[c] * expf((float)(s_G[w][i] - s_G[w][j + c])) : 0.0f;
                *(f32x4 *)(out + SSM_C * SSM_C + ((m * 4 + g) * 64 + l) * 4) = d;
            }
        float *vec = out + 2 * SSM_C * SSM_C;
        vec[l] = expf((float)G);
        vec[SSM_C + l] = expf((float)(last - G));
        vec[2 * SSM_C + l] = gain;
        vec[3 * SSM_C + l] = gl;
        const bool bad = __any(!ssm_finite(gl) || !ssm_finite(gain)) || s_bad;
        if (l == 0) vec[4 * SSM_C] = bad ? 1.0f : 0.0f;
    } else if (DELTA) {
        float *s_A = s_buf + (2 + w) * SSM_C * LG;
        for (int m = 0; m < 4; m++)
            for (int g = 0; g <= m; g++) {
                const int i = 16 * m + l % 16, j = 16 * g + 4 * (l / 16);
                const float4 p = *(const float4 *)(s_kk + i * LG + j);
                const float v[4] = { p.x, p.y, p.z, p.w };
                const float beta = __shfl(gain, i);
                f32x4 d;
#pragma unroll
                for (int c = 0; c < 4; c++) d[c] = j + c < i ? beta * v[c] * expf((float)(s_G[w][i] - s_G[w][j + c])) : 0.0f;
                *(f32x4 *)(s_A + i * LG + j) = d;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float x[SSM_C];
#pragma unroll
        for (int i = 0; i < SSM_C; i++) {
            float s0 = i == l ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const f32x4 v = *(const f32x4 *)(s_A + i * LG + j);
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (j + c < i) {
                        if (c & 1) s1 = fmaf(-v[c], x[j + c], s1);
                        else s0 = fmaf(-v[c], x[j + c], s0);
                    }
            }
            x[i] = s0 + s1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < SSM_C; i++) s_A[i * LG + l] = x[i] * gain;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int m = 0; m < 4; m++)
            for (int g = 0; g <= m; g++)
                *(f32x4 *)(out + ((m * 4 + g) * 64 + l) * 4) = *(const f32x4 *)(s_A + (16 * m + l % 16) * LG + 16 * g + 4 * (l / 16));
    }
}

/* A request's chunks in order, for 16 value elements of one head; S stays in registers as the products leave it (lane:
 * value element l%16, key elements 16 (KB w + b) + 4 (l/16) + i) and in LDS as they take it.  Wave w has tokens
 * 16 w .. of every product with tokens as rows.  Operands of the next chunk are loaded while this one is worked on. */
template <int KD, bool DELTA>
__global__ __launch_bounds__(SSM_T, 1) void ssm_chunk_kernel(SsmArgs A, SsmWs W, int blocks, int max_chunks, int *err)
{
    constexpr int KB = KD / 64, G16 = KD / 16, LS = KD + 4, LT = SSM_C + 4;
    __shared__ __attribute__((aligned(16))) float s_S[16 * LS], s_R[16 * LT], s_W[16 * LT], s_We[16 * LT];
    __shared__ float s_part[2][4][16];
    __shared__ int s_bad;
    const RoasterSsmScan &a = A.a;
    const int tid = threadIdx.x, l = tid % 64, w = tid / 64, taps = A.s.taps, VD = A.s.v_dim, VH = A.s.v_heads;
    /* with a multiple of 8 heads, those of one key head and their blocks on one XCD (workgroup b runs on b % 8) */
    int h = blockIdx.x / blocks, vb = blockIdx.x % blocks;
    if (VH % 8 == 0) {
        const int j = blockIdx.x / 8;
        h = blockIdx.x % 8 * (VH / 8) + j / blocks;
        vb = j % blocks;
    }
    const int r = blockIdx.y, kh = h / A.rep, nk = A.s.k_heads * KD, v0 = h * VD + vb * 16;
    SsmReq q;
    if (!ssm_request(A, r, v0, 16, q, err)) return;
    const int base = ssm_base(A, r), chunks = (q.n + SSM_C - 1) / SSM_C;
    if (base + chunks > max_chunks) {                   /* requests that share rows, so that `first` is none of a plan */
        if (tid == 0) atomicOr(err, ATTN_ERR_SCAN);
        for (int t = tid; t < q.n * 16; t += SSM_T) a.out[(size_t)(q.f0 + t / 16) * a.out_row + v0 + t % 16] = __uint_as_float(0x7FC00000u);
        return;
    }
    const int v = l % 16, t4 = 16 * w + 4 * (l / 16), cv = 2 * nk + v0 + v;
    float *state = A.s.state + ((size_t)r * VH * VD + v0 + v) * KD + 4 * (l / 16);
    f32x4 S[KB];
#pragma unroll
    for (int b = 0; b < KB; b++) {
        S[b] = q.pos ? *(const f32x4 *)(state + 16 * (KB * w + b)) : (f32x4){ 0, 0, 0, 0 };
        *(f32x4 *)(s_S + v * LS + 16 * (KB * w + b) + 4 * (l / 16)) = S[b];
    }
    if (tid == 0) s_bad = 0;
    SsmChannel conv;                                    /* its history is that of the request's first row */
    conv.start(A, r, q.pos, cv);
    const float skip = a.skip ? a.skip[h] : 0.0f;
    const float *x = a.x + (size_t)q.f0 * a.x_row + cv;

    struct Ops {
        float4 k[G16], q[G16], t[4], a[4], kt[KB][4];
        float x[7];
        f32x4 eg, ec, gain;
        float last, bad;
    };
    auto load = [&](int c, Ops &o) {
        const float4 *key = (const float4 *)W.key(base + c, kh), *head = (const float4 *)W.head(base + c, h);
        const float *vec = (const float *)(head + 2 * SSM_C * SSM_C / 4);
#pragma unroll
        for (int g = 0; g < G16; g++) {
            if (DELTA) o.k[g] = gld_f4(key + SSM_C * KD / 4 + (w * G16 + g) * 64 + l);
            o.q[g] = gld_f4(key + (w * G16 + g) * 64 + l);
        }
#pragma unroll
        for (int j = 0; j < 7; j++) {
            const int i = c * SSM_C + t4 - 3 + j;
            o.x[j] = i >= 0 && i < q.n ? x[(size_t)i * a.x_row] : 0.0f;
        }
        o.eg = *(const f32x4 *)(vec + t4);
        o.ec = *(const f32x4 *)(vec + SSM_C + t4);
        o.gain = *(const f32x4 *)(vec + 2 * SSM_C + t4);
        o.last = vec[SSM_C - 1];
        o.bad = vec[4 * SSM_C];
#pragma unroll
        for (int g = 0; g < 4; g++)
            if (g <= w) {
                if (DELTA) o.t[g] = gld_f4(head + (w * 4 + g) * 64 + l);
                o.a[g] = gld_f4(head + SSM_C * SSM_C / 4 + (w * 4 + g) * 64 + l);
            }
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
            for (int g = 0; g < 4; g++) o.kt[b][g] = gld_f4(key + 2 * SSM_C * KD / 4 + ((KB * w + b) * 4 + g) * 64 + l);
    };
    auto chunk = [&](int c, const Ops &o) {
        const int width = min(SSM_C, q.n - c * SSM_C);
        /* values of tokens t4 .. t4 + 3 */
        float xx[7];
#pragma unroll
        for (int j = 0; j < 7; j++) xx[j] = o.x[j];
        if (c == 0 && t4 == 0) {
#pragma unroll
            for (int j = 0; j < 3; j++) xx[j] = conv.h[j];
        }
        f32x4 V;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            SsmChannel cc = conv;
            cc.h[0] = xx[i]; cc.h[1] = xx[i + 1]; cc.h[2] = xx[i + 2];
            V[i] = t4 + i < width ? cc.next(xx[i + 3], taps) : 0.0f;
            odd |= !ssm_finite(V[i]);
        }
        if (odd || o.bad != 0.0f) s_bad = c + 1;
        f32x4 P = {}, Q = {};
#pragma unroll
        for (int g = 0; g < G16; g++) {
            const float4 b = *(const float4 *)(s_S + v * LS + 16 * g + 4 * (l / 16));
            if (DELTA) P = ssm_mfma4(o.k[g], b, P);
            Q = ssm_mfma4(o.q[g], b, Q);
        }
        if (DELTA) {
            f32x4 R;
#pragma unroll
            for (int i = 0; i < 4; i++) R[i] = V[i] - o.eg[i] * P[i];
            *(f32x4 *)(s_R + v * LT + t4) = R;
            __syncthreads();
        }
        f32x4 Wv = {};
        if (DELTA) {
#pragma unroll
            for (int g = 0; g < 4; g++)
                if (g <= w) Wv = ssm_mfma4(o.t[g], *(const float4 *)(s_R + v * LT + 16 * g + 4 * (l / 16)), Wv);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) Wv[i] = o.gain[i] * V[i];
        }
        f32x4 We;
#pragma unroll
        for (int i = 0; i < 4; i++) We[i] = o.ec[i] * Wv[i];
        *(f32x4 *)(s_W + v * LT + t4) = Wv;
        *(f32x4 *)(s_We + v * LT + t4) = We;
        __syncthreads();
        float *out = a.out + (size_t)(q.f0 + c * SSM_C) * a.out_row + v0 + v;
        if (s_bad != c + 1) {
            f32x4 O;
#pragma unroll
            for (int i = 0; i < 4; i++) O[i] = o.eg[i] * Q[i];
#pragma unroll
            for (int g = 0; g < 4; g++)
                if (g <= w) O = ssm_mfma4(o.a[g], *(const float4 *)(s_W + v * LT + 16 * g + 4 * (l / 16)), O);
#pragma unroll
            for (int b = 0; b < KB; b++) {
#pragma unroll
                for (int i = 0; i < 4; i++) S[b][i] *= o.last;
#pragma unroll
                for (int g = 0; g < 4; g++) S[b] = ssm_mfma4(o.kt[b][g], *(const float4 *)(s_We + v * LT + 16 * g + 4 * (l / 16)), S[b]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (t4 + i < width) out[(size_t)(t4 + i) * a.out_row] = a.skip ? fmaf(skip, V[i], O[i]) : O[i];
        } else {
            /* an infinite or NaN input: token by token, so that it does not reach those before it */
            const float *key = W.key(base + c, kh), *vec = W.head(base + c, h) + 2 * SSM_C * SSM_C;
            *(f32x4 *)(s_R + v * LT + t4) = V;
            __syncthreads();
            for (int t = 0; t < width; t++) {
                const float decay = expf(vec[3 * SSM_C + t]), gain = vec[2 * SSM_C + t], val = s_R[v * LT + t];
                f32x4 kf[KB], qf[KB];
                float sk = 0, so = 0;
#pragma unroll
                for (int b = 0; b < KB; b++) {
                    const int at = ((t / 16 * G16 + KB * w + b) * 64 + t % 16 + l / 16 * 16) * 4;
                    qf[b] = *(const f32x4 *)(key + at);
                    kf[b] = *(const f32x4 *)(key + SSM_C * KD + at);
#pragma unroll
                    for (int i = 0; i < 4; i++) sk = fmaf(S[b][i], kf[b][i], sk);
                }
                float wt = gain * val;
                if (DELTA) {
                    sk += __shfl_xor(sk, 16);
                    sk += __shfl_xor(sk, 32);
                    if (l < 16) s_part[0][w][l] = sk;
                    __syncthreads();
                    wt = gain * (val - decay * (s_part[0][0][v] + s_part[0][1][v] + s_part[0][2][v] + s_part[0][3][v]));
                }
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        S[b][i] = fmaf(wt, kf[b][i], decay * S[b][i]);
                        so = fmaf(S[b][i], qf[b][i], so);
                    }
                so += __shfl_xor(so, 16);
                so += __shfl_xor(so, 32);
                if (l < 16) s_part[1][w][l] = so;
                __syncthreads();
                if (tid < 16) {
                    const float o4 = s_part[1][0][v] + s_part[1][1][v] + s_part[1][2][v] + s_part[1][3][v];
                    out[(size_t)t * a.out_row] = a.skip ? fmaf(skip, val, o4) : o4;
                }
                __syncthreads();
            }
        }
#pragma unroll
        for (int b = 0; b < KB; b++) *(f32x4 *)(s_S + v * LS + 16 * (KB * w + b) + 4 * (l / 16)) = S[b];
        __syncthreads();
    };
    Ops o0, o1;
    load(0, o0);
    __syncthreads();
    for (int c = 0; c < chunks; c += 2) {
        if (c + 1 < chunks) load(c + 1, o1);
        chunk(c, o0);
        if (c + 1 == chunks) break;
        if (c + 2 < chunks) load(c + 2, o0);
        chunk(c + 1, o1);
    }
#pragma unroll
    for (int b = 0; b < KB; b++) *(f32x4 *)(state + 16 * (KB * w + b)) = S[b];
    /* the inputs of the last positions: these value channels, and by one workgroup of a key head its own */
    for (int i = max(0, q.n - taps); i < q.n; i++) {
        float *to = A.s.conv + ((size_t)r * taps + ((unsigned)q.pos + i) % taps) * A.channels;
        const float *from = a.x + (size_t)(q.f0 + i) * a.x_row;
        if (tid < 16) to[2 * nk + v0 + tid] = from[2 * nk + v0 + tid];
        if (vb == 0 && h % A.rep == 0)
            for (int j = tid; j < 2 * KD; j += SSM_T) {
                const int ch = j < KD ? kh * KD + j : nk + kh * KD + j - KD;
                to[ch] = from[ch];
            }
    }
}

static bool ssm_state_ok(const RoasterSsmState *s)
{
    return s && s->n_req >= 1 && s->n_req <= 2048 && s->k_heads >= 1 && s->v_heads >= s->k_heads && s->v_heads <= 256 &&
           s->v_heads % s->k_heads == 0 && (s->k_dim == 64 || s->k_dim == 128) && (s->v_dim == 64 || s->v_dim == 128) &&
           s->taps >= 2 && s->taps <= 4;
}

static inline int ssm_channels(const RoasterSsmState *s) { return 2 * s->k_heads * s->k_dim + s->v_heads * s->v_dim; }

/* From so many new tokens of a request on a call goes by chunks. */
#define SSM_CHUNK_MIN 32

/* Chunks of a step at most: the last of each request may be short. */
static inline int ssm_max_chunks(int rows, const RoasterSsmState *s) { return rows / SSM_C + (rows < s->n_req ? rows : s->n_req); }

extern "C" size_t roaster_ssm_ws_bytes(int rows, int most, const RoasterSsmState *s)
{
    if (!ssm_state_ok(s) || rows < 0 || rows > (1 << 18) || most < 1 || (rows && most > rows)) return 0;
    if (most < SSM_CHUNK_MIN) return 16;
    const SsmWs w = { NULL, s->k_dim, s->k_heads, s->v_heads };
    return (size_t)ssm_max_chunks(rows, s) * w.chunk_floats() * sizeof(float);
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
    if (p->most >= SSM_CHUNK_MIN) {
        const SsmWs W = { (float *)p->ws, s->k_dim, s->k_heads, s->v_heads };
        const int chunks = ssm_max_chunks(p->rows, s), groups = (A.rep + SSM_HG - 1) / SSM_HG, blocks = s->v_dim / 16;
#define CHUNK(KD, D)                                                                                                          \
    do {                                                                                                                    \
        hipLaunchKernelGGL((ssm_prep_kernel<KD, D>), dim3(chunks, s->k_heads * groups), dim3(SSM_T), 0, rt().stream, A, W,    \
                           groups);                                                                                          \
        hipLaunchKernelGGL((ssm_chunk_kernel<KD, D>), dim3(vh * blocks, n), dim3(SSM_T), 0, rt().stream, A, W, blocks,        \
                           chunks, err);                                                                                    \
    } while (0)
        if (s->k_dim == 128) { if (delta) CHUNK(128, true); else CHUNK(128, false); }
        else { if (delta) CHUNK(64, true); else CHUNK(64, false); }
#undef CHUNK
        return rt_check(hipGetLastError(), "ssm_chunk launch") ? ROASTER_EDEVICE : 0;
    }
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
