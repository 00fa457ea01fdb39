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

#include <climits>
#include <type_traits>

#define SSM_T 256

struct SsmArgs {
    RoasterSsmScan a;
    RoasterSsmState s;
    int rep, channels;           /* value heads to a key head; channels of a row */
    int lim;                     /* requests of so many rows and more go by chunks */
};

/* A request's rows and first position. */
struct SsmReq { int f0, n, pos; };

/* Rows f0 .. f1 - 1 left out: NaN in `width` elements from `col` on, and a report. */
__device__ __forceinline__ void ssm_leave(const SsmArgs &A, int f0, int f1, int col, int width, int *err)
{
    if (threadIdx.x == 0) atomicOr(err, ATTN_ERR_SCAN);
    for (int t = max(f0, 0); t < min(f1, A.a.rows); t++)
        for (int i = threadIdx.x; i < width; i += blockDim.x) A.a.out[t * A.a.out_row + col + i] = __uint_as_float(0x7FC00000u);
}

/* Whether request r has rows to work on; a bad one's are filled with NaN (`width` elements from `col` on). */
__device__ __forceinline__ bool ssm_request(const SsmArgs &A, int r, int col, int width, SsmReq &q, int *err)
{
    const RoasterSsmScan &a = A.a;
    const int f0 = a.first[r], f1 = a.first[r + 1];
    if (f0 == f1) return false;
    /* differences only of numbers that are known to be rows: of others they can leave an int's range */
    if (f0 >= 0 && f1 > f0 && f1 <= a.rows && f1 - f0 <= a.most) {
        q = { f0, f1 - f0, a.row_pos[f0] };
        if (q.pos >= 0) return true;
    }
    if (err) ssm_leave(A, f0, f1, col, width, err);
    return false;
}

/* e^x as 2^(x log2 e): off by 2^-23 and |x| 2^-24 of it, which is |x| e^x 2^-24 at most 2^-25 for the decays (x <= 0), and
 * in a sigmoid at most 2^-25 too. */
__device__ __forceinline__ float ssm_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float ssm_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + ssm_exp(-x)); }
__device__ __forceinline__ float ssm_silu(float x) { return x * ssm_sigmoid(x); }
__device__ __forceinline__ float ssm_softplus(float x) { return fmaxf(x, 0.0f) + log1pf(ssm_exp(-fabsf(x))); }

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

/* States past the caches: a step's other layers lie between two uses. */
__device__ __forceinline__ float4 ssm_ldnt(const float *p)
{
    const gf32x4 v = __builtin_nontemporal_load((const GAS gf32x4 *)p);
    return make_float4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void ssm_stnt(float *p, float4 v) { __builtin_nontemporal_store((gf32x4){ v.x, v.y, v.z, v.w }, (GAS gf32x4 *)p); }

/* Token by token: a workgroup has one request's block of VB value elements of one head, its state in
 * registers (KD / 16 lanes a row, 16 elements each).  The queries' and keys' channels are convolved by every
 * workgroup of the head: 2 KD inputs next to VB * KD states.
 * ONE: no request has more than one row, so the entry of `conv` that it fills is none that it reads, and the workgroup writes
 * it; else ssm_conv_kernel or ssm_chunk_kernel does behind this kernel.
 * What bounds it: with one request of 32 heads of 128 x 128 (5.0 .. 5.6 us) a launch and the chain position, inputs, sums, state,
 * with 58 of them (42 us) memory, 254 MB at 6.0 TB/s.  Of several tokens each costs 1.3 us, the chain of the exchange in LDS,
 * the two dot products and their sums over lanes. */
template <int KD, int VB, bool DELTA, bool ONE>
__global__ __launch_bounds__(SSM_T) void ssm_token_kernel(SsmArgs A, int blocks, int *err)
{
    constexpr int P = KD / 16, RP = SSM_T / P, NR = VB / RP;
    __shared__ float s_qk[2][2 * KD], s_v[2][VB], s_sum[2][3][SSM_T / 64];
    const RoasterSsmScan &a = A.a;
    const int tid = threadIdx.x, r = blockIdx.y, h = blockIdx.x / blocks, v0 = blockIdx.x % blocks * VB;
    const int VD = A.s.v_dim, taps = A.s.taps, nk = A.s.k_heads * KD, kh = h / A.rep;
    SsmReq q;
    if (!ssm_request(A, r, h * VD + v0, VB, q, err) || q.n >= A.lim) return;
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
            S[i][j] = q.pos ? ssm_ldnt(state + (size_t)i * RP * KD + 4 * P * j) : make_float4(0, 0, 0, 0);
    const float coef = a.a_coef[h], dtb = a.dt_bias ? a.dt_bias[h] : 0.0f, skip = a.skip ? a.skip[h] : 0.0f;
    if (ONE) {
        float *to = A.s.conv + ((size_t)r * taps + (unsigned)q.pos % taps) * A.channels;
        if (qk && v0 == 0 && h % A.rep == 0) to[cq] = xq;
        if (val) to[cv] = xv;
    }
    for (int t = 0; t < q.n; t++) {
        const int b = t & 1;
        const float dt = ssm_softplus(av + dtb), decay = ssm_exp(coef * dt), gain = DELTA ? ssm_sigmoid(bv) : dt;
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
        for (int j = 0; j < 4; j++) ssm_stnt(state + (size_t)i * RP * KD + 4 * P * j, S[i][j]);
}

/* The inputs of a request's last positions into its entries of `conv`, four channels; of requests that go token by token. */
__device__ __forceinline__ void ssm_conv_put(const SsmArgs &A, int r, int c)
{
    SsmReq q;
    const int taps = A.s.taps;
    if (!ssm_request(A, r, 0, 0, q, nullptr) || q.n >= A.lim) return;
    for (int t = max(0, q.n - taps); t < q.n; t++)
        *(float4 *)(A.s.conv + ((size_t)r * taps + ((unsigned)q.pos + t) % taps) * A.channels + c) =
            gld_f4(A.a.x + (size_t)(q.f0 + t) * A.a.x_row + c);
}

__global__ __launch_bounds__(SSM_T) void ssm_conv_kernel(SsmArgs A)
{
    const int c = 4 * (blockIdx.x * SSM_T + threadIdx.x);
    if (c < A.channels) ssm_conv_put(A, blockIdx.y, c);
}

/* ---- prompts: 64 tokens at a time -------------------------------------------------
 *
 * Within a chunk, G_i = sum of a_coef dt up to token i and D_ij = exp(G_i - G_j) for j <= i:
 *   A_ij = beta_i D_ij k_i.k_j (j < i),   T = (1 + A)^-1 diag(beta)
 *   R = V - exp(G) K S,   W = T R         the w of all tokens (STATE: W = dt V)
 *   out = scale (exp(G) Q S + (D o Q K^T) W),     S = exp(G_63) S + K^T (exp(G_63 - G) W)
 * ssm_prep_kernel makes what does not need S for all chunks at once, ssm_chunk_kernel goes through a
 * request's chunks with a block of 16 value elements.
 *
 * Products run on v_mfma_f32_16x16x32_f16 with both operands in two fp16 parts (x = hi + lo, 22 bits),
 * hi hi + hi lo + lo hi, since f32 MFMAs have a sixteenth of the rate:
 *   A[m][k]: lane l holds m = l%16, k = 8*(l/16) + i, i = 0..7     (B[k][n] likewise)
 *   D[m][n]: lane l holds m = 4*(l/16) + i, n = l%16, i = 0..3
 * Q and K are unit vectors (STATE: powers of two bring their largest element to 1/16 .. 1/8, their norms so below 1.5, K's
 * going into dt and Q's into the output), so they, D o Q K^T and T are at most 4 in size and enter times 2^8.  S, R and W enter
 * times a power of two for each value element, from bounds that no product waits for: the norm of an element's
 * row of S is at most b, which a chunk makes of the norm before it (summed while the chunk runs: a bound carried from the
 * request's first chunk on keeps what the correction takes out of S again) and the sum of gain |v| |k|; |R| <= |v| + b, |w| <= |v| + |S|.
 * fp16's range below the bound (2^-38 of it) leaves 22 bits where the bound is 2^15 too large; the bounds are at most
 * 130 times the largest |v| and row of S among the chunk's and the 64 tokens before.  That takes decays
 * of at most 1: a chunk with a positive a_coef dt, or with an infinite or NaN input, goes token by token.
 * Tokens behind a request's last are zeros with gain 0 and the decay of the last. */
#define SSM_C 64                 /* tokens of a chunk */
#define SSM_HG 2                 /* value heads of a workgroup of ssm_prep_kernel */
#define SSM_UP 256.0f            /* Q, K, T and D o Q K^T as operands */
/* A token's: exp(G) * qf, qf (scale, and Q's power of two), exp(G), exp(G_63 - G), gain, a_coef dt; then 1 where the chunk has
 * to go token by token. */
enum { SSM_EQ = 0, SSM_QF = 64, SSM_EG = 128, SSM_EC = 192, SSM_GAIN = 256, SSM_GL = 320, SSM_BAD = 384, SSM_VEC = 448 };

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

/* Workspace, in bytes: of a chunk and key head the operands of Q and K (tokens as rows), of a chunk and value head those of
 * T and D o Q K^T, and the vectors below.  An operand of 16 rows by 32 columns is a kilobyte of high and one of low
 * parts in lane order.  (K^T comes from K's operands, values from x: with both here too 2048 tokens took 138 us.) */
struct SsmWs {
    char *p;
    int kd, kh, vh;

    __host__ __device__ size_t key_bytes() const { return 2 * (size_t)SSM_C * kd * 4; }
    __host__ __device__ size_t head_bytes() const { return 2 * SSM_C * SSM_C * 4 + SSM_VEC * 4; }
    __host__ __device__ size_t chunk_bytes() const { return kh * key_bytes() + vh * head_bytes(); }
    __device__ char *key(int c, int h) const { return p + c * chunk_bytes() + h * key_bytes(); }
    __device__ char *head(int c, int h) const { return p + c * chunk_bytes() + kh * key_bytes() + h * head_bytes(); }
    __device__ static float *vec(char *head) { return (float *)(head + 2 * SSM_C * SSM_C * 4); }
};

/* Chunks of request r, 0 for one that is idle, left out or short. */
__device__ __forceinline__ int ssm_chunks(const SsmArgs &A, int r)
{
    if (r >= A.s.n_req) return 0;
    const int f0 = A.a.first[r], f1 = A.a.first[r + 1];
    if (f0 < 0 || f1 <= f0 || f1 > A.a.rows || f1 - f0 > A.a.most || f1 - f0 < A.lim || A.a.row_pos[f0] < 0) return 0;
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

/* The request that is number j of those with chunks, and the chunks of those before it; likewise. */
__device__ __forceinline__ int ssm_nth(const SsmArgs &A, int j, int &base)
{
    const int l = threadIdx.x % 64;
    base = 0;
    for (int r0 = 0; r0 < A.s.n_req; r0 += 64) {
        const int n = ssm_chunks(A, r0 + l);
        const unsigned long long some = __ballot(n > 0);
        const unsigned long long hit = __ballot(n > 0 && __popcll(some & ((1ull << l) - 1)) == j);
        const int at = hit ? __ffsll(hit) - 1 : 64;
        int sum = l < at ? n : 0;
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
        base += sum;
        if (hit) return r0 + at;
        j -= __popcll(some);
    }
    return -1;
}

__device__ __forceinline__ bool ssm_finite(float x) { return fabsf(x) < INFINITY; }
/* 2^e of a finite x, 2^e <= |x| < 2^(e + 1), e within lo - 127 .. hi - 127; 1 for others. */
__device__ __forceinline__ float ssm_pow2(float x, int lo = 27, int hi = 250)
{
    const int e = (int)(__float_as_uint(x) >> 23 & 255);
    return e == 255 ? 1.0f : __uint_as_float((unsigned)min(max(e, lo), hi) << 23);
}
/* The larger of top and |x|, NaN being larger than all. */
__device__ __forceinline__ float ssm_top(float top, float x) { return __uint_as_float(max(__float_as_uint(top), __float_as_uint(x) & 0x7FFFFFFFu)); }
__device__ __forceinline__ float ssm_inv2(float p) { return __uint_as_float((254u << 23) - __float_as_uint(p)); }   /* 1 / 2^e */

/* Rounded to nearest, so that the low parts are as often negative and no larger than half a step of the high ones: the
 * product of two of them, which is left out, is at most 2^-22 of the whole and on average nothing.  (Cut off, which is as fast, it is
 * up to 2^-20 and always of the whole's sign.) */
__device__ __forceinline__ h16x2 ssm_half2(float x, float y)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector((f32x2){ x, y }, h16x2);
}
struct SsmOp { h16x8 hi, lo; };                         /* one lane's of an operand */
__device__ __forceinline__ SsmOp ssm_split(const float (&v)[8])
{
    SsmOp o;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {                    /* two at a time; what the high part leaves is exact in f32 */
        const h16x2 h = ssm_half2(v[i], v[i + 1]), r = ssm_half2(v[i] - (float)h[0], v[i + 1] - (float)h[1]);
        o.hi[i] = h[0];
        o.hi[i + 1] = h[1];
        o.lo[i] = r[0];
        o.lo[i + 1] = r[1];
    }
    return o;
}
__device__ __forceinline__ void ssm_split4(f32x4 v, float by, _Float16 *hi, _Float16 *lo)
{
    h16x4 h, r;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const float x = v[i] * by, y = v[i + 1] * by;
        const h16x2 p = ssm_half2(x, y), q = ssm_half2(x - (float)p[0], y - (float)p[1]);
        h[i] = p[0];
        h[i + 1] = p[1];
        r[i] = q[0];
        r[i + 1] = q[1];
    }
    *(h16x4 *)hi = h;
    *(h16x4 *)lo = r;
}
__device__ __forceinline__ SsmOp ssm_ld(const char *at, int l)
{
    const unsigned off = 16 * l;                        /* the base is scalar */
    return { *(const h16x8 *)(at + off), *(const h16x8 *)(at + 1024 + off) };
}
__device__ __forceinline__ void ssm_st(char *at, int l, const SsmOp &o)
{
    *(h16x8 *)(at + 16 * l) = o.hi;
    *(h16x8 *)(at + 1024 + 16 * l) = o.lo;
}
__device__ __forceinline__ h16x4 ssm_lds_cols(const char *at)
{
    typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)at));
}
/* The three products of the parts, a chain each. */
struct SsmSum {
    f32x4 hh = {}, hl = {}, lh = {};
    __device__ __forceinline__ void add(const SsmOp &a, const SsmOp &b)
    {
        lh = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo, b.hi, lh, 0, 0, 0);
        hh = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.hi, hh, 0, 0, 0);
        hl = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.lo, hl, 0, 0, 0);
    }
    __device__ __forceinline__ f32x4 get() const { return hh + (hl + lh); }
};

/* Four channels of the convolution over RG rows, from row j0 of a chunk of `width` rows at x on (x[0]: row i0 of its request). */
template <int RG>
struct SsmConv4 {
    float4 w[4], bias, x[RG + 3];                       /* the last three are the rows before */

    __device__ __forceinline__ void load(const SsmArgs &A, int r, int pos, int c, const float *rows, int i0, int j0, int width)
    {
        const size_t stride = A.a.x_row;
        const int taps = A.s.taps;
#pragma unroll
        for (int i = 0; i < RG; i++) x[i] = gld_f4(rows + (size_t)min(j0 + i, width - 1) * stride + (unsigned)c);
        const float *hist = A.s.conv + (size_t)r * taps * A.channels + c;
#pragma unroll
        for (int j = 0; j < 3; j++) {
            const int back = 3 - j;                     /* positions behind the first of them; a request's rows are RG or more apart */
            if (i0 + j0) x[RG + j] = gld_f4(rows + (ptrdiff_t)min(j0 - back, width - 1) * (ptrdiff_t)stride + (unsigned)c);
            else x[RG + j] = back < taps && pos >= back ? gld_f4(hist + (size_t)((unsigned)(pos - back) % taps) * A.channels) : make_float4(0, 0, 0, 0);
        }
        bias = make_float4(0, 0, 0, 0);
        if (A.a.conv_b) bias = make_float4(A.a.conv_b[c], A.a.conv_b[c + 1], A.a.conv_b[c + 2], A.a.conv_b[c + 3]);
        const float *at = A.a.conv_w + (size_t)c * taps;          /* 4 * taps in a row */
        const float4 zero = make_float4(0, 0, 0, 0), f0 = gld_f4(at), f1 = gld_f4(at + 4);
        if (taps == 2) {
            w[0] = w[1] = zero;
            w[2] = make_float4(f0.x, f0.z, f1.x, f1.z);
            w[3] = make_float4(f0.y, f0.w, f1.y, f1.w);
            return;
        }
        const float4 f2 = gld_f4(at + 8);
        if (taps == 3) {
            w[0] = zero;
            w[1] = make_float4(f0.x, f0.w, f1.z, f2.y);
            w[2] = make_float4(f0.y, f1.x, f1.w, f2.z);
            w[3] = make_float4(f0.z, f1.y, f2.x, f2.w);
            return;
        }
        const float4 f3 = gld_f4(at + 12);
        w[0] = make_float4(f0.x, f1.x, f2.x, f3.x);
        w[1] = make_float4(f0.y, f1.y, f2.y, f3.y);
        w[2] = make_float4(f0.z, f1.z, f2.z, f3.z);
        w[3] = make_float4(f0.w, f1.w, f2.w, f3.w);
    }
    __device__ __forceinline__ static float4 mad(float4 u, float4 v, float4 c)
    {
        return make_float4(fmaf(u.x, v.x, c.x), fmaf(u.y, v.y, c.y), fmaf(u.z, v.z, c.z), fmaf(u.w, v.w, c.w));
    }
    /* row i; inputs of unused taps are not touched, since they may be infinite or NaN */
    __device__ __forceinline__ float4 row(int i, int taps) const
    {
        auto in = [&](int k) { return k < 0 ? x[RG + 3 + k] : x[k]; };
        float4 c = bias;
        if (taps > 3) c = mad(w[0], in(i - 3), c);
        if (taps > 2) c = mad(w[1], in(i - 2), c);
        c = mad(w[2], in(i - 1), c);
        c = mad(w[3], in(i), c);
        return make_float4(ssm_silu(c.x), ssm_silu(c.y), ssm_silu(c.z), ssm_silu(c.w));
    }
};

/* A chunk's tokens of one key head: convolution, norms, the products among tokens, and of SSM_HG of its value
 * heads the decays and T, whose 16 x 16 blocks on the diagonal are inverted by substitution, a column a lane,
 * and joined by products in f32 (T_rc = - T_rr sum_k A_rk T_kc), a wave having a block c of columns.  What bounds it: of 30 us for 2048 tokens
 * and 16 key heads (two workgroups a CU, all at once) about 9 are its 94 MB beyond what one workgroup alone needs, 20 us: inputs
 * 6, the solve 5, decays 4, outputs 3, products and silu 2 each, a chain of waits with few waves to fill them. */
template <int KD, bool DELTA>
__global__ __launch_bounds__(2 * SSM_T, 4) void ssm_prep_kernel(SsmArgs A, SsmWs W, int groups)
{
    constexpr int LD = KD + 4, LG = SSM_C + 4, KS = KD / 32, OPS = 4 * KS;           /* operands of Q, and of K */
    constexpr int F0 = 2 * SSM_C * LD, F1 = (2 + SSM_HG) * SSM_C * LG, RQ = SSM_C * (KD / 2) / (2 * SSM_T);
    __shared__ __attribute__((aligned(16))) float s_buf[F0 > F1 ? F0 : F1];
    __shared__ double s_G[SSM_HG][SSM_C];
    __shared__ float s_gain[SSM_HG][SSM_C], s_gl[SSM_HG][SSM_C], s_rq[SSM_C], s_rk[SSM_C], s_qf[SSM_C], s_kf[SSM_C];
    __shared__ int s_bad;
    const RoasterSsmScan &a = A.a;
    const int tid = threadIdx.x, l = tid % 64, w = __builtin_amdgcn_readfirstlane(tid / 64), taps = A.s.taps;
    const int kh = blockIdx.y / groups, hg = blockIdx.y % groups, nk = A.s.k_heads * KD;
    int of;
    const int r = __builtin_amdgcn_readfirstlane(ssm_find(A, blockIdx.x, of));
    of = __builtin_amdgcn_readfirstlane(of);
    if (r < 0) return;
    const int f0 = a.first[r], n = a.first[r + 1] - f0, pos = a.row_pos[f0], i0 = of * SSM_C, width = min(SSM_C, n - i0);
    const int heads = min(SSM_HG, A.rep - hg * SSM_HG), h0 = kh * A.rep + hg * SSM_HG;
    const float *x = a.x + (size_t)(f0 + i0) * a.x_row;
    float *s_q = s_buf, *s_k = s_buf + SSM_C * LD;
    if (tid == 0) s_bad = 0;

    /* four channels a thread and RQ rows of them */
    const int ch = 4 * (tid % (KD / 2)), j0 = (KD == 128 ? w : tid / (KD / 2)) * RQ;
    SsmConv4<RQ> cq;
    cq.load(A, r, pos, ch < KD ? kh * KD + ch : nk + kh * KD + ch - KD, x, i0, j0, width);
    if (w < heads) {                                    /* a token a lane */
        const bool in = l < width;
        const size_t row = (size_t)(f0 + i0 + min(l, width - 1));
        const int h = h0 + w;
        const float dt = ssm_softplus(a.a[row * a.a_row + h] + (a.dt_bias ? a.dt_bias[h] : 0.0f));
        const float gl = in ? a.a_coef[h] * dt : 0.0f;
        /* e^-256 is 0 in f32 as is all below it, and a sum that holds such a token alone would lose the decays behind it: of 64
         * tokens no more than 2^14, so that their differences keep 38 bits behind the point */
        double G = fmaxf(gl, -256.0f);
        for (int o = 1; o < 64; o <<= 1) {
            const double v = __shfl_up(G, o);
            if (l >= o) G += v;
        }
        s_G[w][l] = G;
        s_gl[w][l] = gl;
        s_gain[w][l] = !in ? 0.0f : DELTA ? ssm_sigmoid(a.b[row * a.b_row + h]) : dt;
    }
    {
        float *to = (ch < KD ? s_q + ch : s_k + ch - KD) + j0 * LD;
#pragma unroll
        for (int i = 0; i < RQ; i++) {
            const float4 y = cq.row(i, taps);
            *(float4 *)(to + i * LD) = j0 + i < width ? y : make_float4(0, 0, 0, 0);
        }
    }
    __syncthreads();
    {   /* norms: eight threads a row */
        const int row = tid / 8;
        float sq = 0, sk = 0;
#pragma unroll
        for (int j = 0; j < KD / 32; j++) {
            const float4 q = *(const float4 *)(s_q + row * LD + 4 * (tid % 8 + 8 * j)), k = *(const float4 *)(s_k + row * LD + 4 * (tid % 8 + 8 * j));
            if (DELTA) {
                sq += q.x * q.x + q.y * q.y + q.z * q.z + q.w * q.w;
                sk += k.x * k.x + k.y * k.y + k.z * k.z + k.w * k.w;
            } else {                                    /* the largest, NaN being larger than all */
                sq = ssm_top(ssm_top(ssm_top(ssm_top(sq, q.x), q.y), q.z), q.w);
                sk = ssm_top(ssm_top(ssm_top(ssm_top(sk, k.x), k.y), k.z), k.w);
            }
        }
        for (int o = 1; o < 8; o <<= 1) {
            const float oq = __shfl_xor(sq, o), ok = __shfl_xor(sk, o);
            sq = DELTA ? sq + oq : ssm_top(sq, oq);
            sk = DELTA ? sk + ok : ssm_top(sk, ok);
        }
        if (tid % 8 == 0) {
            /* not from sums of squares, which leave f32's range where the vectors do not */
            const float pq = DELTA ? 1.0f : 16.0f * ssm_pow2(sq, 8, 249), pk = DELTA ? 1.0f : 16.0f * ssm_pow2(sk, 8, 249);
            const float rq = DELTA ? 1.0f / sqrtf(sq + a.eps) : ssm_inv2(pq), rk = DELTA ? 1.0f / sqrtf(sk + a.eps) : ssm_inv2(pk);
            /* without eps a sum of squares near f32's smallest makes no unit vector */
            const bool fine = sq < 0x1p120f && sk < 0x1p120f && (!DELTA || (rq < 0x1p60f && rk < 0x1p60f)) && ssm_finite(a.scale * pq);
            if (row < width && !fine) s_bad = 1;
            s_rq[row] = row < width ? rq : 0.0f;
            s_rk[row] = row < width ? rk : 0.0f;
            s_qf[row] = a.scale * pq;
            s_kf[row] = pk;
        }
    }
    __syncthreads();
    SsmOp ops[OPS / 4];                                 /* of 2 OPS, wave w's: Q's first, then K's */
    char *key = W.key(blockIdx.x, kh), *sop = (char *)s_buf;
#pragma unroll
    for (int f = 0; f < OPS / 4; f++) {
        const int g = w * (OPS / 4) + f, row = g % OPS / KS * 16 + l % 16, col = g % KS * 32 + l / 16 * 8;
        const float *at = (g < OPS ? s_q : s_k) + row * LD + col, by = SSM_UP * (g < OPS ? s_rq : s_rk)[row];
        const float4 u = *(const float4 *)at, v = *(const float4 *)(at + 4);
        ops[f] = ssm_split({ u.x * by, u.y * by, u.z * by, u.w * by, v.x * by, v.y * by, v.z * by, v.w * by });
        if (hg == 0) ssm_st(key + g * 2048, l, ops[f]);
    }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < OPS / 4; f++) ssm_st(sop + (w * (OPS / 4) + f) * 2048, l, ops[f]);
    __syncthreads();
    /* products of tokens, lower blocks alone: waves 0 .. 3 have rows 16 w of Q K^T, waves 4 .. 7 of K K^T */
    SsmSum kk[4];
    const int m4 = w % 4;
    const bool keys = w >= 4;
    auto op = [&](int g) { return SsmOp{ *(const h16x8 *)(sop + g * 2048 + 16 * l), *(const h16x8 *)(sop + g * 2048 + 1024 + 16 * l) }; };
    if (DELTA || !keys)
        for (int s = 0; s < KS; s++) {
            const SsmOp u = op((keys ? OPS : 0) + m4 * KS + s);
#pragma unroll
            for (int b = 0; b < 4; b++)
                if (b <= m4) kk[b].add(u, op(OPS + b * KS + s));
        }
    __syncthreads();
    float *s_qk = s_buf, *s_kk = s_buf + SSM_C * LG;
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if ((DELTA || !keys) && b <= m4)
                (keys ? s_kk : s_qk)[(16 * m4 + 4 * (l / 16) + i) * LG + 16 * b + l % 16] =
                    kk[b].get()[i] * (keys ? 1 / (SSM_UP * SSM_UP) : 1 / SSM_UP);
    __syncthreads();
    /* decays, four waves a head: row block w / 2 of D o Q K^T as an operand, and of A */
    const int hh = w % SSM_HG, m = w / SSM_HG, h = h0 + hh;
    float *const s_A = s_buf + (2 + hh) * SSM_C * LG, *const s_T = s_buf + hh * SSM_C * LG;    /* A; later T, with its columns as rows */
    if (hh < heads) {
        char *out = W.head(blockIdx.x, h);
        const int i = 16 * m + l % 16;
        const double Gi = s_G[hh][i];
        const float beta = s_gain[hh][i];
        for (int s = 0; s <= m / 2; s++) {
            const int j = 32 * s + 8 * (l / 16);
            float v[8], d[8];
#pragma unroll
            for (int c = 0; c < 8; c++) {
                d[c] = j + c <= i ? ssm_exp((float)(Gi - s_G[hh][j + c])) : 0.0f;
                v[c] = j + c <= i ? s_qk[i * LG + j + c] * d[c] : 0.0f;
            }
            ssm_st(out + (8 + m * 2 + s) * 2048, l, ssm_split(v));
            if (DELTA) {
#pragma unroll
                for (int c = 0; c < 8; c++) v[c] = j + c < i ? beta * s_kk[i * LG + j + c] * d[c] : 0.0f;
                *(f32x4 *)(s_A + i * LG + j) = (f32x4){ v[0], v[1], v[2], v[3] };
                *(f32x4 *)(s_A + i * LG + j + 4) = (f32x4){ v[4], v[5], v[6], v[7] };
            }
        }
        if (m == 0) {
            float *vec = W.vec(out);
            const double G = s_G[hh][l];
            const float gl = s_gl[hh][l], eg = ssm_exp((float)G), qf = s_qf[l], gain = s_gain[hh][l] * (DELTA ? 1.0f : s_kf[l]);
            vec[SSM_EQ + l] = eg * qf;
            vec[SSM_QF + l] = qf;
            vec[SSM_EG + l] = eg;
            vec[SSM_EC + l] = ssm_exp((float)(s_G[hh][SSM_C - 1] - G));
            vec[SSM_GAIN + l] = gain;
            vec[SSM_GL + l] = gl;
            const bool bad = __any(!ssm_finite(gl) || gl > 0.0f || !ssm_finite(gain)) || s_bad;
            if (l == 0) vec[SSM_BAD] = bad ? 1.0f : 0.0f;
        }
    }
    __syncthreads();
    if (!DELTA) return;
    /* T by blocks of 16 columns, one to a wave */
    if (hh < heads) {                                   /* the block on the diagonal, a column a lane, four times over */
        const int c = l % 16;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float s0 = i == c ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const f32x4 v = *(const f32x4 *)(s_A + (16 * m + i) * LG + 16 * m + j);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (j + k < i) {
                        if (k & 1) s1 = fmaf(-v[k], y[j + k], s1);
                        else s0 = fmaf(-v[k], y[j + k], s0);
                    }
            }
            y[i] = s0 + s1;
        }
        if (l < 16) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) *(f32x4 *)(s_T + (16 * m + c) * LG + 16 * m + i) = (f32x4){ y[i], y[i + 1], y[i + 2], y[i + 3] };
            /* its rows over A's own, which are not needed any more */
#pragma unroll
            for (int i = 0; i < 16; i++) s_A[(16 * m + i) * LG + 16 * m + c] = y[i];
        }
    }
    __syncthreads();
    if (hh < heads) {
        /* v_mfma_f32_16x16x4_f32, its lanes' four columns of 16 being 4*(l/16) .. + 3: results are operands of the next product as they come */
        auto mul = [&](const f32x4 &u, const f32x4 &v, f32x4 c) {
#pragma unroll
            for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(u[i], v[i], c, 0, 0, 0);
            return c;
        };
        const int at = 4 * (l / 16);
        f32x4 T[4];                                     /* T_kb, k = 0 .. */
        for (int k = 0; k < 4; k++) T[k] = (f32x4){};
        T[0] = *(const f32x4 *)(s_T + (16 * m + l % 16) * LG + 16 * m + at);
#pragma unroll
        for (int d = 1; d < 4; d++)                     /* block row m + d */
            if (m + d < 4) {
                f32x4 s = {};
                const float *A = s_A + (16 * (m + d) + l % 16) * LG + 16 * m + at;
#pragma unroll
                for (int k = 0; k < d; k++) s = mul(*(const f32x4 *)(A + 16 * k), T[k], s);
                T[d] = mul(*(const f32x4 *)(A + 16 * d), -s, (f32x4){ 0, 0, 0, 0 });
                *(f32x4 *)(s_T + (16 * m + l % 16) * LG + 16 * (m + d) + at) = T[d];
            }
    }
    __syncthreads();
    if (hh < heads)
        for (int s = 0; s <= m / 2; s++) {
            const int i = 16 * m + l % 16, j = 32 * s + 8 * (l / 16);
            float v[8];
#pragma unroll
            for (int c = 0; c < 8; c++) v[c] = j + c <= i ? s_T[(j + c) * LG + i] * (s_gain[hh][j + c] * SSM_UP) : 0.0f;
            ssm_st(W.head(blockIdx.x, h0 + hh) + (m * 2 + s) * 2048, l, ssm_split(v));
        }
}

/* A request's chunks in order, for 16 value elements of one head (v = l%16), with two groups of four waves: the first goes
 * from S to W, the second makes the outputs and the next chunk's values; token rows 16 (w % 4) .. each, and each wave has 16
 * key elements of S.  S stays in registers as the products leave it (key elements 16 w + 4 (l/16) + i) and
 * in LDS as they take it.  Operands of the next chunk are loaded while this one is worked on, without conditions, so that
 * waits count those under way exactly.  The second group is a step behind: it makes the next chunk's values before the first
 * barrier and finishes the last chunk's outputs before the second, so that neither barrier waits for it (82 -> 77 us).
 * What bounds it: 2048 tokens of 32 heads of 128 x 128 take 78 us, 32 chunks of 2.4 us one after another (2.0 if nothing
 * comes from memory): K S, T R and K^T W wait for each other, with a split into parts, LDS and a barrier between, and LDS
 * passes 200 KB a chunk, some 1600 cycles of 128 bytes.  Two workgroups a CU would need 128 registers a wave, which spills (prompt 99 -> 211 us). */
template <int KD, bool DELTA>
__global__ __launch_bounds__(2 * SSM_T, 2) void ssm_chunk_kernel(SsmArgs A, SsmWs W, int blocks, int max_chunks, int *err)
{
    constexpr int KS = KD / 32, OPS = 4 * KS, LS = KD + 8, LT = SSM_C + 8, LV = SSM_C + 4;
    __shared__ __attribute__((aligned(16))) _Float16 s_S[2][16 * LS], s_R[2][16 * LT], s_W[2][2][16 * LT], s_We[2][16 * LT];
    __shared__ __attribute__((aligned(16))) float s_V[2][16 * LV], s_top[2][16][4];
    __shared__ __attribute__((aligned(16))) char s_K[OPS * 2048];                /* K's operands as they are, read as K^T's */
    __shared__ float s_part[2][8][16];
    __shared__ __attribute__((aligned(16))) float s_norm[2][16][8];              /* squares of an element's row of S, a wave's part each; of even and of odd chunks */
    const RoasterSsmScan &a = A.a;
    /* the wave's number from the first lane, so that operands' addresses are scalar */
    const int tid = threadIdx.x, l = tid % 64, w8 = __builtin_amdgcn_readfirstlane(tid / 64), w = w8 % 4;
    const int taps = A.s.taps, VD = A.s.v_dim, VH = A.s.v_heads;
    /* with a multiple of 8 heads, those of one key head and their blocks on one XCD (workgroup b runs on b % 8) */
    int h = blockIdx.x / blocks, vb = blockIdx.x % blocks;
    if (VH % 8 == 0) {
        const int j = blockIdx.x / 8;
        h = blockIdx.x % 8 * (VH / 8) + j / blocks;
        vb = j % blocks;
    }
    const int kh = h / A.rep, nk = A.s.k_heads * KD, v0 = h * VD + vb * 16;
    int r = 0, base = 0;
    if (A.s.n_req > 1) {
        if (blockIdx.y == gridDim.y - 1) {              /* the short requests' `conv`, which ssm_token_kernel in front of this has read */
            const int pieces = A.channels / 4;
            for (int i = blockIdx.x * 2 * SSM_T + tid; i < A.s.n_req * pieces; i += gridDim.x * 2 * SSM_T)
                ssm_conv_put(A, i / pieces, 4 * (i % pieces));
            /* more long requests than rows would hold, so that some share them */
            if (blockIdx.x == 0)
                for (int j = gridDim.y - 1; (r = ssm_nth(A, j, base)) >= 0; j++) ssm_leave(A, A.a.first[r], A.a.first[r + 1], 0, VH * VD, err);
            return;
        }
        r = __builtin_amdgcn_readfirstlane(ssm_nth(A, blockIdx.y, base));
        base = __builtin_amdgcn_readfirstlane(base);
        if (r < 0) return;
    }
    SsmReq q;
    if (!ssm_request(A, r, v0, 16, q, err)) return;
    const int chunks = (q.n + SSM_C - 1) / SSM_C;
    if (base + chunks > max_chunks) {                   /* requests that share rows, so that `first` is none of a plan */
        ssm_leave(A, q.f0, q.f0 + q.n, v0, 16, err);
        return;
    }
    const int v = l % 16, t4 = 16 * w + 4 * (l / 16);
    /* a loop for each group, so that its waits count its own loads */
    auto run = [&](auto group) {
        constexpr bool first = decltype(group)::value, holds = KD == 128 || first;
        float *state = A.s.state + ((size_t)r * VH * VD + v0 + v) * KD + 16 * w8 + 4 * (l / 16);
        f32x4 S = {};
        if (holds && q.pos) S = *(const f32x4 *)state;
        const float skip = a.skip ? a.skip[h] : 0.0f;
        SsmChannel conv = {};                               /* the second group's; its history is that of the request's first row */
        if (!first) conv.start(A, r, q.pos, 2 * nk + v0 + v);
        const float *x0 = a.x + (size_t)q.f0 * a.x_row + 2 * nk + v0 + v, *x4 = x0 + 4 * (l / 16) * a.x_row;

        SsmOp one[KS], two[2];                              /* the first group's K and T, the second's Q and D o Q K^T */
        struct Head {
            f32x4 f, g;                                     /* exp(G) and exp(G_63 - G), or the outputs' factors */
            f32x4 gain;
            float last, bad;
        };
        auto load_head = [&](int c, Head &o) {
            char *head = W.head(base + c, h);
            const float *vec = W.vec(head);
            o.f = *(const f32x4 *)(vec + (first ? SSM_EG : SSM_EQ) + t4);
            o.g = *(const f32x4 *)(vec + (first ? SSM_EC : SSM_QF) + t4);
            if (!DELTA) o.gain = *(const f32x4 *)(vec + SSM_GAIN + t4);
            const __attribute__((address_space(4))) float *same = (const __attribute__((address_space(4))) float *)vec;      /* scalar loads */
            o.last = same[SSM_EG + SSM_C - 1];
            o.bad = same[SSM_BAD];
        };
        auto load_one = [&](int c) {
            const char *at = W.key(base + c, kh) + ((first ? OPS : 0) + w * KS) * 2048;
#pragma unroll
            for (int s = 0; s < KS; s++) one[s] = ssm_ld(at + s * 2048, l);
        };
        auto load_two = [&](int c) {
            const char *head = W.head(base + c, h) + (DELTA && first ? 0 : 8) * 2048;
#pragma unroll
            for (int s = 0; s < 2; s++) two[s] = ssm_ld(head + (w * 2 + min(s, w / 2)) * 2048, l);      /* tokens 32 .. have no part in rows below */
        };
        /* This wave's 16 key elements of K^T, tokens 32 s ..: the transposing read takes 4 tokens of 16 elements from 16 lanes (lane
         * 4 i + j: elements 4 j .. of token i) and gives lane c the four of element c. */
        auto key_cols = [&](int s) {
            const int j = l % 4, at = (l / 4 % 4 + 8 * (l / 16 % 2) + 16 * (w8 % 2 * 2 + j / 2)) * 16 + j % 2 * 8;
            const char *base = s_K + ((2 * s + l / 32) * KS + w8 / 2) * 2048 + at;
            SsmOp o;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const h16x4 hi = ssm_lds_cols(base + 64 * i), lo = ssm_lds_cols(base + 1024 + 64 * i);
#pragma unroll
                for (int e = 0; e < 4; e++) { o.hi[4 * i + e] = hi[e]; o.lo[4 * i + e] = lo[e]; }
            }
            return o;
        };
        /* the inputs of this lane's four tokens of chunk c and the three before; STATE: their gains, for the largest gain |v| */
        f32x4 gains = {};
        auto load_x = [&](int c, float (&xs)[7]) {
            if (!DELTA) gains = *(const f32x4 *)(W.vec(W.head(base + c, h)) + SSM_GAIN + t4);
            const int i0 = c * SSM_C + 16 * w - 3;
            if (i0 >= 0 && i0 + 19 <= q.n) {
#pragma unroll
                for (int j = 0; j < 7; j++) xs[j] = x4[(size_t)(i0 + j) * a.x_row];
            } else {
#pragma unroll
                for (int j = 0; j < 7; j++)                  /* rows before the first and behind the last are not used */
                    xs[j] = x0[(size_t)min(max(i0 + 4 * (l / 16) + j, 0), q.n - 1) * a.x_row];
            }
        };
        /* their values to LDS, and the largest of each element (STATE: of a token's gain times its value, since the largest of both
         * can be those of different tokens): infinite where one is infinite or NaN */
        auto values = [&](int c, const float (&xs)[7]) {
            float xx[7];
#pragma unroll
            for (int j = 0; j < 7; j++) xx[j] = xs[j];
            if (c == 0 && t4 == 0) {
#pragma unroll
                for (int j = 0; j < 3; j++) xx[j] = conv.h[j];
            }
            f32x4 V;
#pragma unroll
            for (int i = 0; i < 4; i++) V[i] = fmaf(conv.w[3], xx[i + 3], fmaf(conv.w[2], xx[i + 2], conv.bias));
            if (taps > 2) {
#pragma unroll
                for (int i = 0; i < 4; i++) V[i] = fmaf(conv.w[1], xx[i + 1], V[i]);
            }
            if (taps > 3) {
#pragma unroll
                for (int i = 0; i < 4; i++) V[i] = fmaf(conv.w[0], xx[i], V[i]);
            }
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                V[i] = c * SSM_C + t4 + i < q.n ? ssm_silu(V[i]) : 0.0f;
                top = max(top, __float_as_uint(DELTA ? V[i] : gains[i] * V[i]) & 0x7FFFFFFFu);
            }
            const auto far = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            top = max(far[0], far[1]);
            const auto near = __builtin_amdgcn_permlane16_swap(top, top, false, false);
            top = max(near[0], near[1]);
            *(f32x4 *)(s_V[c & 1] + v * LV + t4) = V;
            if (l < 16) s_top[c & 1][v][w] = __uint_as_float(min(top, 0x7F800000u));
        };
        auto op = [&](const _Float16 *p, int ld, int s) {
            const _Float16 *at = p + v * ld + 32 * s + 8 * (l / 16);
            return SsmOp{ *(const h16x8 *)at, *(const h16x8 *)(at + 16 * ld) };
        };
        /* chunk c's S as an operand, and the sum of its squares as such */
        auto put_S = [&](int c, float by) {
            if (!holds) return;
            ssm_split4(S, by, s_S[0] + v * LS + 16 * w8 + 4 * (l / 16), s_S[1] + v * LS + 16 * w8 + 4 * (l / 16));
            const f32x4 U = S * by;
            float sum = U[0] * U[0] + U[1] * U[1] + U[2] * U[2] + U[3] * U[3];
            const auto far = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
            sum = __uint_as_float(far[0]) + __uint_as_float(far[1]);
            const auto near = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
            sum = __uint_as_float(near[0]) + __uint_as_float(near[1]);
            if (l < 16) s_norm[c & 1][l][w8] = sum;
        };
        /* The norm of the element's row of the S that put_S had with 8192 / p, no less (squares below f32's range are less than 2^-56
         * p together); p's own bound may be far above it.  Roundings are written out, see below.  It is read where it is used, while
         * other waves put the next chunk's: read at the chunk's beginning, which would spare the second buffer, it holds up the loads
         * under way (2048 tokens 109 us instead of 99). */
        auto norm_S = [&](int c, float p) {
            f32x4 sum = *(const f32x4 *)s_norm[c & 1][v];
            if (KD == 128) sum += *(const f32x4 *)(s_norm[c & 1][v] + 4);
            return fmaf(__builtin_amdgcn_sqrtf((sum[0] + sum[1]) + (sum[2] + sum[3])), p * (1.0001f / 8192.0f), p * 0x1p-56f);
        };

        /* The norm of the element's row of S, no less; squares of small states would leave f32's range. */
        auto row_norm = [&] {
            const f32x4 U = S * 0x1p64f;
            float one = S[0] * S[0] + S[1] * S[1] + S[2] * S[2] + S[3] * S[3], up = U[0] * U[0] + U[1] * U[1] + U[2] * U[2] + U[3] * U[3];
            one += __shfl_xor(one, 16);
            up += __shfl_xor(up, 16);
            one += __shfl_xor(one, 32);
            up += __shfl_xor(up, 32);
            if (l < 16) {
                s_part[0][w8][l] = one;
                s_part[1][w8][l] = up;
            }
            __syncthreads();
            one = up = 0;
            for (int i = 0; i < 8; i++) {
                one += s_part[0][i][v];
                up += s_part[1][i][v];
            }
            return (one >= 0x1p-60f ? sqrtf(one) : sqrtf(up) * 0x1p-64f) * 1.0001f;
        };

        Head o, next;
        float xs[7];
        load_head(0, o);
        if (!first) {
            load_x(0, xs);
            values(0, xs);
            load_x(min(1, chunks - 1), xs);
        }
        load_one(0);
        if (first) load_two(0);
        float b = row_norm();
        float pS = ssm_pow2(b);                              /* |S| < 2 pS; as an operand times 2^13 / pS, so below 2^14 */
        put_S(0, 8192.0f * ssm_inv2(pS));
        __syncthreads();

        float *out = a.out + (size_t)(q.f0 + t4) * a.out_row + v0 + v;               /* this lane's four tokens in turn */
        /* A chunk's outputs are finished while the first group works on the next W: what does not need W, and the factors of D W */
        f32x4 part = {}, by = {};
        bool open = false;
        auto close = [&](int c, int n) {
            SsmSum sum;
#pragma unroll
            for (int s = 0; s < 2; s++)
                if (s <= w / 2) sum.add(two[s], op(s_W[c & 1][0], LT, s));
            const f32x4 O = part + by * sum.get();
            float *at = out + (ptrdiff_t)c * SSM_C * (ptrdiff_t)a.out_row;
            if (n >= SSM_C) {
#pragma unroll
                for (int i = 0; i < 4; i++) __builtin_nontemporal_store(O[i], at + i * a.out_row);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (t4 + i < n) at[i * a.out_row] = O[i];
            }
            open = false;
        };
        if (first) __builtin_amdgcn_s_setprio(1);            /* the other group waits for it */
        for (int c = 0; c < chunks; c++) {
            const int c1 = min(c + 1, chunks - 1);
            const f32x4 tops = *(const f32x4 *)s_top[c & 1][v], V = *(const f32x4 *)(s_V[c & 1] + v * LV + t4);
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            /* the wave's lanes have all 16 elements.  Both groups have to come to the same bounds, bit by bit, so their roundings are
             * written out and not left to the compiler */
            const float all = fmaf(128.0f, top, b);
            const bool bad = __any(o.bad != 0.0f || !(all < 0x1p120f));
            const float last = o.last;
            if (!bad) {
                /* bounds: of R, of W, and of the next S */
                const float bR = top + b, bW = DELTA ? fmaf(65.0f, top, b) : top, pR = ssm_pow2(bR), pW = ssm_pow2(bW);
                const float back = pW * (1 / (8192.0f * SSM_UP));
                f32x4 X = {};
                if (DELTA || !first) {
                    SsmSum sum;
#pragma unroll
                    for (int s = 0; s < KS; s++) sum.add(one[s], op(s_S[0], LS, s));
                    X = sum.get() * (pS * (1 / (8192.0f * SSM_UP)));
                }
                if (first) {
#pragma unroll
                    for (int s = 0; s < KS; s++) ssm_st(s_K + (w * KS + s) * 2048, l, one[s]);
                }
                load_one(c1);
                if (!first && c + 1 < chunks) values(c + 1, xs);
                if (DELTA) {
                    if (first) ssm_split4(V - o.f * X, 8192.0f * ssm_inv2(pR), s_R[0] + v * LT + t4, s_R[1] + v * LT + t4);
                    __syncthreads();
                }
                if (first) {
                    f32x4 w4 = {};
                    if (DELTA) {
                        SsmSum sum;
#pragma unroll
                        for (int s = 0; s < 2; s++)
                            if (s <= w / 2) sum.add(two[s], op(s_R[0], LT, s));
                        w4 = sum.get() * (pR * (1 / (8192.0f * SSM_UP)));
                    } else w4 = o.gain * V;
                    ssm_split4(w4, 8192.0f * ssm_inv2(pW), s_W[c & 1][0] + v * LT + t4, s_W[c & 1][1] + v * LT + t4);
                    ssm_split4(o.g * w4, 8192.0f * ssm_inv2(pW), s_We[0] + v * LT + t4, s_We[1] + v * LT + t4);
                } else {
                    load_x(min(c + 2, chunks - 1), xs);
                    if (open) close(c - 1, SSM_C);
                    load_two(c);
                    part = o.f * X;
                    if (a.skip) part = part + skip * V;
                    by = o.g * back;
                    open = true;
                }
                __syncthreads();
                if (holds) {
                    SsmSum sum;
#pragma unroll
                    for (int s = 0; s < 2; s++) sum.add(key_cols(s), op(s_We[0], LT, s));
                    S = S * last + sum.get() * back;
                }
                b = fmaf(last, fminf(b, norm_S(c, pS)), (DELTA ? 1.0f : 1.5f) * 64.0f * 1.0001f * top);
                pS = ssm_pow2(b);
                put_S(c + 1, 8192.0f * ssm_inv2(pS));
                if (first) load_two(c1);
                load_head(c1, next);
            } else {
                if (!first && open) close(c - 1, SSM_C);
                /* token by token in f32 (q and k from their operands), so that an infinite or NaN input does not reach those before it */
                const char *key = W.key(base + c, kh);
                const float *vec = W.vec(W.head(base + c, h));
                for (int t = 0; t < min(SSM_C, q.n - c * SSM_C); t++) {
                    const float decay = ssm_exp(vec[SSM_GL + t]), gain = vec[SSM_GAIN + t], val = s_V[c & 1][v * LV + t];
                    f32x4 kf = {}, qf = {};
                    if (holds) {
                        const int k = 16 * w8 + 4 * (l / 16);
                        const char *at = key + (t / 16 * KS + k / 32) * 2048 + (t % 16 + 16 * (k % 32 / 8)) * 16 + k % 8 * 2;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const _Float16 *aq = (const _Float16 *)at + i, *ak = (const _Float16 *)(at + OPS * 2048) + i;
                            qf[i] = ((float)aq[0] + (float)aq[512]) * (1 / SSM_UP);
                            kf[i] = ((float)ak[0] + (float)ak[512]) * (1 / SSM_UP);
                        }
                    }
                    float wt = gain * val;
                    if (DELTA) {
                        float sk = S[0] * kf[0] + S[1] * kf[1] + S[2] * kf[2] + S[3] * kf[3];
                        sk += __shfl_xor(sk, 16);
                        sk += __shfl_xor(sk, 32);
                        if (l < 16) s_part[0][w8][l] = sk;
                        __syncthreads();
                        sk = 0;
                        for (int i = 0; i < KD / 16; i++) sk += s_part[0][i][v];
                        wt = gain * (val - decay * sk);
                    }
                    S = decay * S + wt * kf;
                    float so = S[0] * qf[0] + S[1] * qf[1] + S[2] * qf[2] + S[3] * qf[3];
                    so += __shfl_xor(so, 16);
                    so += __shfl_xor(so, 32);
                    if (l < 16) s_part[1][w8][l] = so;
                    __syncthreads();
                    if (tid < 16) {
                        so = 0;
                        for (int i = 0; i < KD / 16; i++) so += s_part[1][i][v];
                        so *= vec[SSM_QF + t];
                        out[(size_t)(c * SSM_C + t) * a.out_row] = a.skip ? fmaf(skip, val, so) : so;     /* threads 0 .. 15: t4 = 0 */
                    }
                    __syncthreads();
                }
                b = row_norm();
                pS = ssm_pow2(b);
                put_S(c + 1, 8192.0f * ssm_inv2(pS));
                if (!first) {
                    if (c + 1 < chunks) values(c + 1, xs);
                    load_x(min(c + 2, chunks - 1), xs);
                }
                load_head(c1, next);
                load_one(c1);
                if (first) load_two(c1);
            }
            o = next;
            __syncthreads();
        }
        if (!first && open) close(chunks - 1, q.n - (chunks - 1) * SSM_C);
        if (holds) *(f32x4 *)state = S;
    };
    if (w8 < 4) run(std::true_type());
    else run(std::false_type());
    /* the inputs of the last positions: these value channels, and by one workgroup of a key head its own */
    for (int i = max(0, q.n - taps); i < q.n; i++) {
        float *to = A.s.conv + ((size_t)r * taps + ((unsigned)q.pos + i) % taps) * A.channels;
        const float *from = a.x + (size_t)(q.f0 + i) * a.x_row;
        if (tid < 16) to[2 * nk + v0 + tid] = from[2 * nk + v0 + tid];
        if (vb == 0 && h % A.rep == 0)
            for (int j = tid; j < 2 * KD; j += 2 * SSM_T) {
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

/* Of a call with long requests those of fewer tokens go token by token, in a kernel in front, us with 24 / 32 / 2 here and 32
 * heads of 128 x 128: 63 requests of one token and one of 256 100 / 91 / 146, 15 of four and one of 128 62 / 60 / 143; of 30, 300,
 * 700, 60 and 40 tokens 93 / 131 / 93.  (All by chunks, single tokens too, 487, 136 and 92.) */
#define SSM_SHORT 24
/* A call goes by chunks if a request may have so many new tokens, us by chunks / by tokens: one request of 12 tokens 23 / 22,
 * of 16 23 / 28; 4 of 20 49 / 42, of 24 50 / 48; 8 of 32 78 / 73; 16 of 32 144 / 131; 32 of 24 279 / 160, of 32 277 / 207.  A
 * token's chain of waits is long where its workgroups leave most of the GPU idle, and chunks of few tokens do the work of 64
 * where it is full.  That is with 32 heads of 128 x 128; the lines hold within an eighth for the others: 64 x 64 (keys x values)
 * one request of 12 20 / 22, 4 of 20 31 / 34, of 24 31 / 39, 8 of 28 46 / 45, of 32 46 / 50; 64 x 128 one of 16 26 / 28, 4 of 24 43 /
 * 40, 8 of 32 68 / 60; 128 x 64 one of 12 23 / 23, 4 of 20 37 / 34, of 24 36 / 40, 8 of 28 52 / 54, 16 of 40 88 / 88, 32 of 40 157 / 159.
 * But where it is full, tokens of 64 keys are shorter: 64 x 64 16 requests of 40 73 / 74, of 48 73 / 87, 32 of 40 127 / 98, of 48 124 /
 * 115; 64 x 128 16 of 40 120 / 98, of 48 119 / 115, 32 of 40 224 / 178, of 48 227 / 211. */
static inline int ssm_limit(const RoasterSsmState *s)
{
    const int blocks = s->n_req * s->v_heads;
    if (s->n_req == 1 && blocks <= 64) return 16;
    return blocks <= 128 ? SSM_SHORT : blocks <= 256 ? 32 : s->k_dim == 64 ? 48 : 40;
}

/* Chunks of a step at most: the last of each long request may be short. */
static inline int ssm_max_long(int rows, const RoasterSsmState *s) { return s->n_req == 1 ? 1 : min(s->n_req, rows / SSM_SHORT); }
static inline int ssm_max_chunks(int rows, const RoasterSsmState *s) { return rows / SSM_C + ssm_max_long(rows, s); }

extern "C" size_t roaster_ssm_ws_bytes(int rows, int most, const RoasterSsmState *s)
{
    if (!ssm_state_ok(s) || rows < 0 || rows > (1 << 18) || most < 1 || (rows && most > rows)) return 0;
    if (!rows || most < ssm_limit(s)) return 16;
    const SsmWs w = { NULL, s->k_dim, s->k_heads, s->v_heads };
    return (size_t)ssm_max_chunks(rows, s) * w.chunk_bytes();
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
    const bool chunked = p->most >= ssm_limit(s);
    SsmArgs A = { *p, *s, s->v_heads / s->k_heads, (int)ch, !chunked ? INT_MAX : n == 1 ? 1 : SSM_SHORT };
    A.a.b = b;
    const bool one = p->most == 1;
#define TOKEN3(KD, VB, D, O)                                                                                              \
    hipLaunchKernelGGL((ssm_token_kernel<KD, VB, D, O>), dim3(vh * (s->v_dim / VB), n), dim3(SSM_T), 0, rt().stream, A,    \
                       s->v_dim / VB, err)
#define TOKEN2(KD, VB, D) do { if (one) TOKEN3(KD, VB, D, true); else TOKEN3(KD, VB, D, false); } while (0)
#define TOKEN(KD, VB) do { if (delta) TOKEN2(KD, VB, true); else TOKEN2(KD, VB, false); } while (0)
    /* 32 value elements a workgroup while that fills the GPU no more than four times, else 64, for fewer reads of the queries' and
     * keys' channels (32 / 64: one request 5.6 / 6.2 us, 4 7.1 / 7.1, 8 8.5 / 8.4, 16 15.4 / 12.4, 64 52.8 / 46.1) */
    if (!chunked || n > 1) {
        if (s->k_dim == 64) TOKEN(64, 64);
        else if (n * ov / 32 >= 1024) TOKEN(128, 64);
        else TOKEN(128, 32);
    }
#undef TOKEN
#undef TOKEN2
#undef TOKEN3
    if (rt_check(hipGetLastError(), "ssm_token launch")) return ROASTER_EDEVICE;
    if (chunked) {
        const SsmWs W = { (char *)p->ws, s->k_dim, s->k_heads, s->v_heads };
        const int chunks = ssm_max_chunks(p->rows, s), groups = (A.rep + SSM_HG - 1) / SSM_HG, blocks = s->v_dim / 16;
#define CHUNK(KD, D)                                                                                                          \
    do {                                                                                                                    \
        hipLaunchKernelGGL((ssm_prep_kernel<KD, D>), dim3(chunks, s->k_heads * groups), dim3(2 * SSM_T), 0, rt().stream, A, W, \
                           groups);                                                                                          \
        hipLaunchKernelGGL((ssm_chunk_kernel<KD, D>), dim3(vh * blocks, ssm_max_long(p->rows, s) + (n > 1)), dim3(2 * SSM_T), 0,    \
                           rt().stream, A, W, blocks, chunks, err);                                                          \
    } while (0)
        if (s->k_dim == 128) { if (delta) CHUNK(128, true); else CHUNK(128, false); }
        else { if (delta) CHUNK(64, true); else CHUNK(64, false); }
#undef CHUNK
        return rt_check(hipGetLastError(), "ssm_chunk launch") ? ROASTER_EDEVICE : 0;
    }
    if (!one) {
        hipLaunchKernelGGL(ssm_conv_kernel, dim3((ch / 4 + SSM_T - 1) / SSM_T, n), dim3(SSM_T), 0, rt().stream, A);
        if (rt_check(hipGetLastError(), "ssm_conv launch")) return ROASTER_EDEVICE;
    }
    return 0;
}
