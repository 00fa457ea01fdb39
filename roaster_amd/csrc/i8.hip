/*
 * i8.hip -- matrix product in 8-bit integers with scales for each token and each
 * channel (roaster_matmul_i8), and the layout of its weights (roaster_i8_pack):
 * the projections on either side of the mixers (model.c:1284-1290, 1344-1347 one
 * token, 1604-1660 a prompt's chunk) for any number of rows.
 *
 * v_mfma_i32_32x32x32_i8, channels as its rows and tokens as its columns.  Lane layout:
 *   A[m][k]: lane l holds m = l%32, k = 16*(l/32) + i, i = 0..15      (B[k][n] likewise)
 *   D[m][n]: lane l holds m = 8*(i/4) + 4*(l/32) + i%4, n = l%32, i = 0..15
 * Weights lie as [rows/32][cols/16][32 rows][16 columns], so that an operand of 32
 * channels by 32 columns is a kilobyte in lane order.
 */
#include "mixer.h"
#include "qdot.h"

#define I8_T 256

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4_a16 __attribute__((ext_vector_type(4)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

static inline size_t i8_rows(int rows) { return ((size_t)rows + 31) & ~(size_t)31; }
static inline size_t i8_cols(int cols) { return ((size_t)cols + 127) & ~(size_t)127; }

/* ---- weights -------------------------------------------------------------------- */
/* Weight i of a super-block (kernels.c:1839-1874). */
__device__ __forceinline__ float q4k_weight(const uint8_t *blk, int i)
{
    const float d = f16_bits_to_f32(gld_u16(blk)), dmin = f16_bits_to_f32(gld_u16(blk + 2));
    const uint8_t *s = blk + 4;
    const int j = i / 32, q = blk[16 + 32 * (i / 64) + i % 32] >> (j & 1) * 4 & 15;
    const int sc = j < 4 ? s[j] & 63 : (s[j + 4] & 15) | (s[j - 4] >> 6) << 4;
    const int mn = j < 4 ? s[j + 4] & 63 : s[j + 4] >> 4 | (s[j] >> 6) << 4;
    return fmaf(d * sc, (float)q, -(dmin * mn));
}

__device__ __forceinline__ float q6k_weight(const uint8_t *blk, int i)
{
    const int n = i / 128, s = i % 128 / 32, l = i % 32;
    const int lo = blk[64 * n + 32 * (s & 1) + l] >> (s >> 1) * 4 & 15, hi = blk[128 + 32 * n + l] >> 2 * s & 3;
    const int8_t sc = (int8_t)blk[192 + 8 * n + 2 * s + l / 16];
    return f16_bits_to_f32(gld_u16(blk + 208)) * sc * (float)((lo | hi << 4) - 32);
}

/* One workgroup a row of the padded matrix; 16 columns a thread at a time.  Once a matrix, so left simple: 12288 x 2048 from
 * f32 40 us, Q4_K 80, Q6_K 46, int8 23; 2048 x 4096 from Q4_K 31. */
template <int FROM>
__global__ __launch_bounds__(I8_T) void i8_pack_kernel(const uint8_t *W, RoasterI8 to, int padded)
{
    __shared__ unsigned s_top[I8_T / 64];
    const int r = blockIdx.x, tid = threadIdx.x, n16 = to.cols / 16;
    auto weight = [&](int c) {
        if (FROM == ROASTER_I8_FROM_F32) return ((const float *)W)[(size_t)r * to.cols + c];
        const int bytes = FROM == ROASTER_I8_FROM_Q6K ? RQ6K_BYTES : RQ4K_BYTES;
        const uint8_t *blk = W + ((size_t)r * (to.cols / RQK) + c / RQK) * bytes;
        return FROM == ROASTER_I8_FROM_Q6K ? q6k_weight(blk, c % RQK) : q4k_weight(blk, c % RQK);
    };
    float mul = 0;
    if (FROM != ROASTER_I8_FROM_I8 && r < to.rows) {
        unsigned top = 0;
        for (int c = tid; c < to.cols; c += I8_T) top = max(top, __float_as_uint(weight(c)) & 0x7FFFFFFFu);
        for (int o = 1; o < 64; o <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
        if (tid % 64 == 0) s_top[tid / 64] = top;
        __syncthreads();
        for (int w = 0; w < I8_T / 64; w++) top = max(top, s_top[w]);
        const I8Scale s = i8_scale(top);
        mul = s.mul;
        if (tid == 0) to.scale[r] = s.scale;
    }
    for (int c = tid; c < padded / 16; c += I8_T) {
        int v[4] = { 0, 0, 0, 0 };
        if (r < to.rows && c < n16) {
            if (FROM == ROASTER_I8_FROM_I8) {
                const uint4 u = gld_u4(W + (size_t)r * to.cols + 16 * c);
                v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
            } else
                for (int j = 0; j < 16; j++) v[j / 4] |= (i8_round(weight(16 * c + j), mul) & 255) << 8 * (j % 4);
        }
        int8_t *at = (int8_t *)to.data + (((size_t)(r / 32) * (padded / 16) + c) * 32 + r % 32) * 16;
        *(i32x4 *)at = (i32x4){ v[0], v[1], v[2], v[3] };
    }
}

/* ---- product -------------------------------------------------------------------- */
struct I8Args {
    const int8_t *w, *x;
    const float *ws, *xs;
    float *y;
    size_t x_row, y_row;
    int T, N, n16, k32;          /* tokens, channels, 16-byte pieces of a token, blocks of 32 padded columns */
};

__device__ __forceinline__ i32x4 i8_ld(const void *p) { return *(const GAS i32x4 *)p; }

/* Few results: a workgroup takes 16 channels of up to 32 tokens, its waves a part of the columns each and join in LDS
 * (integers, so in any order).  Weights go from memory straight into v_mfma_i32_16x16x64_i8 (lane l: row l%16, columns
 * 16*(l/16) ..; results 4*(l/16) + i, i = 0..3, of token l%16), tokens too, from the L2; eight steps' loads are issued together.
 * Padded columns of the weights are zeros, so any byte of the token may stand there.
 * What bounds it: a launch and one chain of loads for a small matrix (2048 x 4096 3.8 us), memory for a large one (12288 x 2048
 * 6.1 us, 4.2 TB/s all in all, of which a launch is 2 us). */
template <int TT>
__global__ __launch_bounds__(1024) void i8_few_kernel(I8Args a)
{
    __shared__ int s_sum[TT * 16 * 16];                /* [token][channel] */
    const int tid = threadIdx.x, l = tid % 64, w = __builtin_amdgcn_readfirstlane(tid / 64), W = blockDim.x / 64;
    const int k0 = a.k32 / 2 * w / W, k1 = a.k32 / 2 * (w + 1) / W, n16 = a.n16, t0 = 16 * TT * blockIdx.y;
    const int8_t *wp = a.w + (size_t)(blockIdx.x / 2) * a.k32 * 1024 + blockIdx.x % 2 * 256;
    const unsigned off = l / 16 * 512 + l % 16 * 16;
    const int8_t *xp[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) xp[t] = a.x + min(t0 + 16 * t + l % 16, a.T - 1) * a.x_row;
    const int tok = t0 + tid / 16, ch = blockIdx.x * 16 + tid % 16;
    const float ws = a.ws[min(ch, a.N - 1)];
    float xs[TT];                                      /* of the first 256 threads' tokens tok + 16 t */
#pragma unroll
    for (int t = 0; t < TT; t++) xs[t] = a.xs[min(tok + 16 * t, a.T - 1)];
    for (int i = tid; i < TT * 256; i += blockDim.x) s_sum[i] = 0;
    i32x4 acc[TT] = {};
    for (int k = k0; k < k1; k += 8) {
        i32x4 A[8], B[TT][8];
#pragma unroll
        for (int i = 0; i < 8; i++) A[i] = *(const i32x4 *)(wp + (size_t)min(k + i, k1 - 1) * 2048 + off);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int t = 0; t < TT; t++) B[t][i] = i8_ld(xp[t] + 16 * min(4 * (k + i) + l / 16, n16 - 1));
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (k + i < k1) {
#pragma unroll
                for (int t = 0; t < TT; t++) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[i], B[t][i], acc[t], 0, 0, 0);
            }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) atomicAdd(&s_sum[(16 * t + l % 16) * 16 + 4 * (l / 16) + i], acc[t][i]);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; t++)
        if (tid < 256 && tok + 16 * t < a.T && ch < a.N) a.y[(tok + 16 * t) * a.y_row + ch] = (float)s_sum[tid + 256 * t] * (xs[t] * ws);
}

__device__ __forceinline__ void i8_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }   /* loads stay in flight */

/* Four outputs of a token from channel ch on; STREAM: past the caches. */
template <bool STREAM>
__device__ __forceinline__ void i8_put(const I8Args &a, int tok, int ch, f32x4_a16 v)
{
    if (tok >= a.T) return;
    float *y = a.y + tok * a.y_row + ch;
    if (ch + 4 <= a.N) {
        if (STREAM) __builtin_nontemporal_store((f32x4_a4)v, (f32x4_a4 *)y);
        else *(f32x4_a4 *)y = v;
    } else
        for (int k = 0; k < 4; k++)
            if (ch + k < a.N) y[k] = v[k];
}

/* More tokens: a workgroup's tile is 32 TB tokens by 128 CB channels, a wave's all its tokens by 32 CB channels.  So no
 * two waves read the same weights, which go from the L2 straight into registers, and only the tokens pass through LDS, a
 * step of U times 64 columns at a time, doubly buffered; both are loaded two steps ahead.  Pieces of 16 bytes of a token
 * are exchanged by (token / 2) % 4, so that eight lanes' reads fall on different banks.  Outputs of the larger tiles are
 * not kept in the caches, whatever their size: 2048 tokens of 12288 x 2048 by themselves 60 us, kept 70, 256 tokens 14.6 / 15.1,
 * 200 of 8192 x 2048 9.9 / 10.4; with the scan and the norm that read them behind it, a whole recurrent layer, 2048 tokens
 * 247 / 249, 256 tokens 76 / 76.
 * What bounds it: 2048 tokens of 12288 x 2048 run at 1720 TOPS (60 us; the library's product of 8192^3 at 2105), 100 MB of
 * outputs among them; 256 tokens (12 .. 14.6 us) are 384 tiles for 256 CUs, each with its first loads and its outputs at the ends. */
template <int TB, int CB, int U>
__global__ __launch_bounds__(I8_T, 2) void i8_tile_kernel(I8Args a, int tiles, int per, int tblocks)
{
    constexpr int TM = 32 * TB, XN = TM * 4 * U, XL = (XN + I8_T - 1) / I8_T;
    constexpr int LY = 32 * CB + 4, YB = 4 * 32 * LY * 4, XB = 2 * U * TM * 64;      /* outputs of a wave's 32 tokens; buffers */
    __shared__ __attribute__((aligned(16))) int8_t s_lds[XB > YB ? XB : YB];
    /* workgroup b runs on XCD b % 8: each has a run of tiles, tokens' blocks of one channel block in turn */
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= tiles) return;
    const int tid = threadIdx.x, l = tid % 64, w = __builtin_amdgcn_readfirstlane(tid / 64);
    const int t0 = id % tblocks * TM, c0 = id / tblocks * (128 * CB) + 32 * CB * w, all = a.k32 / 2, steps = (all + U - 1) / U;
    int8_t *const s_x[2] = { s_lds, s_lds + U * TM * 64 };
    const int8_t *wp[CB];
    for (int c = 0; c < CB; c++) {
        const int cb = min(c0 / 32 + c, (a.N + 31) / 32 - 1);
        wp[c] = a.w + (size_t)cb * a.k32 * 1024;
    }
    const int8_t *xp[XL];
    int xc[XL], xd[XL];
    for (int i = 0; i < XL; i++) {
        const int q = min(tid + i * I8_T, XN - 1), t = q % (TM * 4) / 4, u = q / (TM * 4);
        xp[i] = a.x + min(t0 + t, a.T - 1) * a.x_row;
        xc[i] = 4 * u + q % 4;
        xd[i] = (u * TM + t) * 64 + ((q % 4 ^ (t >> 1 & 3)) << 4);
    }
    i32x4 W[2][2 * CB * U], X[2][XL];
    auto load_w = [&](int s, i32x4 (&r)[2 * CB * U]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t at = (size_t)min(s * U + u, all - 1) * 2048;
#pragma unroll
            for (int c = 0; c < CB; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) r[(2 * u + h) * CB + c] = *(const i32x4 *)(wp[c] + at + 1024 * h + 16u * l);
        }
    };
    auto load_x = [&](int s, i32x4 (&r)[XL]) {
#pragma unroll
        for (int i = 0; i < XL; i++) r[i] = i8_ld(xp[i] + 16 * min(4 * s * U + xc[i], a.n16 - 1));
    };
    auto store_x = [&](int b, const i32x4 (&r)[XL]) {
#pragma unroll
        for (int i = 0; i < XL; i++)
            if (XN % I8_T == 0 || tid + i * I8_T < XN) *(i32x4 *)(s_x[b] + xd[i]) = r[i];
    };
    i32x16 acc[CB][TB];
    for (int c = 0; c < CB; c++)
        for (int t = 0; t < TB; t++) acc[c][t] = (i32x16){};
    auto step = [&](int s, int b) {
        store_x(b ^ 1, X[b ^ 1]);                       /* step s + 1, whose buffer no wave reads any more */
        load_x(s + 2, X[b]);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (U <= 2 || s * U + u < all) {            /* columns are padded to 128: a step of 256 may be short */
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int t = 0; t < TB; t++) {
                        const int tok = 32 * t + l % 32, c16 = 2 * h + l / 32;
                        const i32x4 B = *(const i32x4 *)(s_x[b] + (u * TM + tok) * 64 + ((c16 ^ (tok >> 1 & 3)) << 4));
#pragma unroll
                        for (int c = 0; c < CB; c++)
                            acc[c][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(W[b][(2 * u + h) * CB + c], B, acc[c][t], 0, 0, 0);
                    }
            }
        load_w(s + 2, W[b]);
        i8_barrier();
    };
    load_x(0, X[0]);
    load_w(0, W[0]);
    load_x(1, X[1]);
    load_w(1, W[1]);
    store_x(0, X[0]);
    i8_barrier();
    int s = 0;
    for (; s + 2 <= steps; s += 2) {
        step(s, 0);
        step(s + 1, 1);
    }
    if (s < steps) step(s, 0);
    /* through the wave's own LDS, so that a store's lanes hold whole rows of 32 CB channels (the products leave
     * four channels of 32 tokens); the barrier at the loop's end freed the tokens' buffers */
    float xs[TB], ws[CB][16];
#pragma unroll
    for (int t = 0; t < TB; t++) xs[t] = a.xs[min(t0 + 32 * t + l % 32, a.T - 1)];
#pragma unroll
    for (int c = 0; c < CB; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) ws[c][i] = a.ws[min(c0 + 32 * c + 8 * (i / 4) + 4 * (l / 32) + i % 4, a.N - 1)];
    float *out = (float *)s_lds + w * 32 * LY;
    for (int t = 0; t < TB; t++) {
#pragma unroll
        for (int c = 0; c < CB; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                f32x4_a16 v;
                for (int i = 0; i < 4; i++) v[i] = (float)acc[c][t][4 * j + i] * (xs[t] * ws[c][4 * j + i]);
                *(f32x4_a16 *)(out + l % 32 * LY + 32 * c + 8 * j + 4 * (l / 32)) = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 4 * CB; i++) {
            const int row = l / (8 * CB) + i * (8 / CB), ch = 4 * (l % (8 * CB)), tok = t0 + 32 * t + row;
            i8_put<(TB > 1)>(a, tok, c0 + ch, *(const f32x4_a16 *)(out + row * LY + ch));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

/* ---- entry points --------------------------------------------------------------- */
static bool i8_sizes_ok(int rows, int cols)
{
    return rows >= 1 && rows <= (1 << 20) && cols >= 16 && cols <= 65536 && cols % 16 == 0;
}

static bool i8_ok(const RoasterI8 *w)
{
    return w && i8_sizes_ok(w->rows, w->cols) && w->data && w->scale && attn_aligned(w->data, 16) && attn_aligned(w->scale, 4);
}

extern "C" size_t roaster_i8_bytes(int rows, int cols) { return i8_sizes_ok(rows, cols) ? i8_rows(rows) * i8_cols(cols) : 0; }

extern "C" int roaster_i8_pack(const void *W, int from, const RoasterI8 *to)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!i8_ok(to))
        return rt_fail(ROASTER_EINVAL, "roaster_i8_pack: need 1 <= rows <= 2^20, cols a multiple of 16 up to 65536, data (16-byte "
                       "aligned) and scale");
    const bool quant = from == ROASTER_I8_FROM_Q4K || from == ROASTER_I8_FROM_Q6K;
    if (from < ROASTER_I8_FROM_F32 || from > ROASTER_I8_FROM_I8 || (quant && to->cols % RQK))
        return rt_fail(ROASTER_EINVAL, "roaster_i8_pack: bad source type, or Q4_K / Q6_K with cols no multiple of 256");
    if (!W || !attn_aligned(W, quant ? 2 : 16))
        return rt_fail(ROASTER_EINVAL, "roaster_i8_pack: W must be given and aligned (f32 and int8 to 16 bytes)");
    const size_t rows = to->rows, cols = to->cols, nd = i8_rows(to->rows) * i8_cols(to->cols);
    const size_t nw = from == ROASTER_I8_FROM_F32 ? 4 * rows * cols : from == ROASTER_I8_FROM_I8 ? rows * cols
                                                                  : rq_mat_bytes(from == ROASTER_I8_FROM_Q6K, rows, cols);
    if (attn_overlap(W, nw, to->data, nd) || attn_overlap(W, nw, to->scale, 4 * rows) || attn_overlap(to->data, nd, to->scale, 4 * rows))
        return rt_fail(ROASTER_EINVAL, "roaster_i8_pack: W, data and scale overlap");
    if (rt_init_locked()) return ROASTER_EDEVICE;
    const AttnDevice dev;
#define PACK(F)                                                                                                            \
    hipLaunchKernelGGL((i8_pack_kernel<F>), dim3(i8_rows(to->rows)), dim3(I8_T), 0, rt().stream, (const uint8_t *)W, *to,  \
                       (int)i8_cols(to->cols))
    if (from == ROASTER_I8_FROM_F32) PACK(ROASTER_I8_FROM_F32);
    else if (from == ROASTER_I8_FROM_Q4K) PACK(ROASTER_I8_FROM_Q4K);
    else if (from == ROASTER_I8_FROM_Q6K) PACK(ROASTER_I8_FROM_Q6K);
    else PACK(ROASTER_I8_FROM_I8);
#undef PACK
    return rt_check(hipGetLastError(), "i8_pack launch") ? ROASTER_EDEVICE : 0;
}

extern "C" int roaster_matmul_i8(const RoasterMatmulI8 *p, const RoasterI8 *w)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!i8_ok(w))
        return rt_fail(ROASTER_EINVAL, "roaster_matmul_i8: bad weights (1 <= rows <= 2^20, cols a multiple of 16 up to 65536, "
                       "data 16-byte aligned)");
    if (!p || p->rows < 0 || p->rows > (1 << 20)) return rt_fail(ROASTER_EINVAL, "roaster_matmul_i8: need 0 <= rows <= 2^20");
    if (!p->rows) return 0;
    const size_t T = p->rows, N = w->rows, K = w->cols;
    if (!p->x || !p->x_scale || !p->y || !attn_aligned(p->x, 16) || !attn_aligned(p->x_scale, 4) || !attn_aligned(p->y, 4) ||
        !stride_ok(p->x_row, 16) || !stride_ok(p->y_row, 1) || p->y_row < N)
        return rt_fail(ROASTER_EINVAL, "roaster_matmul_i8: x (16-byte aligned, stride a multiple of 16 up to 2^32), x_scale and y "
                       "(stride from w->rows up to 2^32) must be given");
    const size_t ny = rows_span(T, N, p->y_row, 4);
    if (attn_overlap(p->y, ny, p->x, rows_span(T, K, p->x_row, 1)) || attn_overlap(p->y, ny, p->x_scale, 4 * T) ||
        attn_overlap(p->y, ny, w->data, i8_rows(w->rows) * i8_cols(w->cols)) || attn_overlap(p->y, ny, w->scale, 4 * N))
        return rt_fail(ROASTER_EINVAL, "roaster_matmul_i8: y overlaps inputs");
    if (rt_init_locked()) return ROASTER_EDEVICE;
    const AttnDevice dev;
    I8Args a = { (const int8_t *)w->data, p->x, w->scale, p->x_scale, p->y, p->x_row, p->y_row, p->rows, w->rows, w->cols / 16,
                 (int)(i8_cols(w->cols) / 32) };
    /* Up to 256 workgroups of 32 tokens by 16 channels go by those, whose columns four waves share, and not by tiles, which have
     * a longer chain of steps (33 tokens, 2048 x 2048 5.0 us, by tiles 6.7; 64 of 2048 x 4096 7.1 / 10.3; 256 of 512 x 2048 5.0 /
     * 6.8, of 300 x 512 4.5 / 4.4); with more of them a CU has two in turn (333 of 512 x 2048 6.6 / 6.8, of 1111 x 2064 9.9 / 7.4) */
    const size_t blocks = ((T + 31) / 32) * ((N + 15) / 16);
    if (T <= 32 || blocks <= 256) {
        /* four waves to 16 channels (8 tokens, 12288 x 2048: 6.1 us, with eight 7.4, sixteen 14.6), eight for long
         * columns (one token, 256 x 16384: 6.1 us, with four 7.2) */
        const int waves = K <= 8192 ? 4 : 8;
        if (T <= 16) hipLaunchKernelGGL(i8_few_kernel<1>, dim3((N + 15) / 16), dim3(64 * waves), 0, rt().stream, a);
        else hipLaunchKernelGGL(i8_few_kernel<2>, dim3((N + 15) / 16, (T + 31) / 32), dim3(64 * waves), 0, rt().stream, a);
    } else {
        auto tiles = [&](int tb, int cb) { return ((T + 32 * tb - 1) / (32 * tb)) * ((N + 128 * cb - 1) / (128 * cb)); };
#define TILE(TB, CB, U)                                                                                                    \
    do {                                                                                                                   \
        const int n = (int)tiles(TB, CB), per = (n + 7) / 8;                                                               \
        hipLaunchKernelGGL((i8_tile_kernel<TB, CB, U>), dim3(8 * per), dim3(I8_T), 0, rt().stream, a, n, per,       \
                           (int)((T + 32 * TB - 1) / (32 * TB)));                                                          \
    } while (0)
        /* The largest tiles read least from the L2, which bounds the others (8 .. 9 TB/s), but need enough of them:
         * us with 4 x 2 / 2 x 1 / 1 x 1, and how many there are:
         *   12288 x 2048: 2048 tokens 60 / 75 / 116 (768), 1200 37 / 44 / 62 (480), 700 31 / 29 / 39 (288 / 1056)
         *   8192 x 2048:  100 tokens 19 / 9.5 / 7.8 (.. / 256), 200 19 / 10.1 / 11.3 (.. / 448)
         * 4 x 1 and 2 x 2, and two or four groups of waves that share the columns, never came first by more than a tenth. */
        if (tiles(4, 2) >= 384) TILE(4, 2, 1);
        else if (tiles(1, 1) <= 256) TILE(1, 1, 4);
        else TILE(2, 1, 2);
#undef TILE
    }
    return rt_check(hipGetLastError(), "matmul_i8 launch") ? ROASTER_EDEVICE : 0;
}
