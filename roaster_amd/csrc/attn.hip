/*
 * attn.hip -- softmax attention of new rows over a paged key/value cache
 * (roaster_attn_paged; model.c:755-863, 1536-1602).
 *
 * A unit of work is one row, or a few of one request, and up to 8 or 16 query heads
 * of one key/value head; it goes over the row's positions in tiles of 16 tokens.
 * Every workgroup sums the rows' tiles by itself and takes an even share of all
 * units' tiles laid end to end, whatever the rows' lengths; its waves take a unit's
 * tiles in turn, each with its own running maximum and sums, and join them in LDS.
 * A unit that lies within one share is finished there.  Of one that a share's end
 * cuts, the parts go to the workspace and attn_join_kernel joins them.
 *
 * Both products are MFMAs whose sixteen columns are heads (of one row or several):
 *   S^T = K Q^T   rows: 16 tokens; keys come a kilobyte to a load and go through a
 *                 wave's own LDS into the operands' order;
 *   O^T = V^T P^T rows: 16 elements; a lane holds 16 bytes of each of its tokens'
 *                 values, transposed among its own registers, and its scores are
 *                 the very probabilities that its operand needs, so P never moves
 *                 between lanes.
 * fp16 cache: a query row is scaled by a power of two and split into two fp16
 * parts, the probabilities likewise, so that products are exact up to 2^-22 of an
 * operand.  For one row of up to eight heads the parts are the columns h and h + 8:
 * one product does both.  For more heads or rows (WIDE) the columns are sixteen of
 * them, and each operand read is multiplied by high and low parts in turn.
 * f32 cache: f32 MFMAs, always WIDE.
 *
 * What bounds it: the cache's bytes.  A large read reaches 7.2 TB/s here; 64
 * requests of 300..16000 tokens come to 5.65 (94 us; of four times the lengths to 6.4), one
 * of 200001 to 5.7 (72 us, 5 of them for the join), an f32 cache's 12 of 500..5000 to 4.9 (41 us;
 * of ten times the lengths to 6.5): what is missing are the units' beginnings and the
 * join.  437 tokens take 12 us: two launches and a chain of waits for a row, its page,
 * keys and values.
 */
#include "attn.h"
#include "qdot.h"
#include <type_traits>

#define ATT_T 256
#define ATT_W (ATT_T / 64)
#define ATT_G 512             /* workgroups at most: two per CU */
#define ATT_MIN 4             /* tiles of a share at least: one a wave */
/* A column's terms are 2^(score - m) with a base m that follows its scores, its sums keeping the base's
 * scale.  fp16: a term is kept times 2^13 and may reach 2^15; its two parts hold 22 bits of it down to 2^-3
 * and are off by 2^-25 below.  So the base goes up when a score passes it by LATE octaves, and down when
 * all of a tile stays M_DOWN below it: a term is then off by at most 2^-22 of itself or 2^-24 of its
 * tile's largest, also behind a position that outweighs the rest by 2^20 and whose value is nothing;
 * only in that position's own tile it is 2^-38 of the position's term.  (With a base that only rises
 * and LATE 8, a first position 2^22 above 700 others, its value 0, left outputs off by
 * 1.5e-4; so 1.4e-6.  It costs a prompt's rows 3 to 5%, single tokens nothing.)
 * f32: terms stay below 2^-14, so that 2^14 values of any size can be added up. */
#define LATE 2.0f
template <bool F16>
struct Soft {
    static constexpr float UP = F16 ? 13.0f : -16.0f;
};
#define M_DOWN 14.0f
#define M_MID 6.0f            /* a base that goes down stays this much above the tile's largest, for the next ones */

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

/* A unit whose parts are to be joined: first row and rows, head block, the share that began
 * it, and its shares (0: none to join). */
struct AttCut {
    int row, n, hb, g0, k;
};

struct AttArgs {
    RoasterAttnPaged a;
    const char *kc, *vc;
    KvShape s;
    int group, blocks, hpb;   /* query heads of a key/value head, their blocks, heads of a block */
    int R;                    /* rows of a unit at most */
    int by_unit;              /* the join's table goes by unit (else by the share that began the unit) */
    int grid;                 /* workgroups */
    int few;                  /* attn_few_kernel's parts: one a workgroup */
    AttCut *cut;              /* [units] or [grid] */
    float *pm, *pl, *po;      /* parts [2 ATT_G][COLS], [..][COLS], [..][COLS][D]: slot g with `few`, else 2g + 1 the unit
                                 that share g began and did not finish, 2g the one that it found begun */
};

template <int D, bool F16, bool WIDE>
struct AttCfg {
    static constexpr int COLS = WIDE ? 16 : 8;                       /* columns with sums of their own */
    static constexpr int TT = 16, SZ = F16 ? 2 : 4;                  /* tokens of a tile */
    static constexpr int VE = F16 ? (D >= 128 ? 8 : 4) : 4;       /* elements of a value load */
    static constexpr int NB = D / (16 * VE);                        /* value loads of a token */
    static constexpr int NCH = D * SZ / 16;                          /* 16-byte pieces of a token's key */
    static constexpr int KS = NCH / 4;                               /* key loads of a tile, and operands of a score */
    static constexpr int SW = NCH < 16 ? NCH : 16;
    static constexpr int VT = 4;                                     /* tokens of a lane's value operand */
};

__device__ __forceinline__ float max_g(float v)       /* over the four lanes of a column */
{
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_g(float v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ f16x2 to_half(float x, float y) { return __builtin_convertvector((f32x2){ x, y }, f16x2); }
/* What `to_half` left of x and y, times f (0 or 1). */
__device__ __forceinline__ f16x2 rest_half(f16x2 h, float f, float x, float y)
{
    return to_half(fmaf(-(float)h.x, f, x), fmaf(-(float)h.y, f, y));
}
__device__ __forceinline__ f16x8 join8(const f16x2 *h)
{
    return (f16x8){ h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y };
}

/* N elements of a query column (a lane's quarter of them) as hi + lo fp16 parts of
 * 2^e times themselves (without BOTH only the one that `low`, 0 or 1, says, in
 * hi); gives back 2^-e.  2^e times the column's largest element lies in [2^13,
 * 2^14), e within what a float's exponent holds. */
template <int N, bool BOTH>
__device__ __forceinline__ float split_q(const float4 *x, f16x8 *hi, f16x8 *lo, float low)
{
    float top = 0;
#pragma unroll
    for (int i = 0; i < N / 4; i++)
        top = fmaxf(fmaxf(fmaxf(top, fabsf(x[i].x)), fmaxf(fabsf(x[i].y), fabsf(x[i].z))), fabsf(x[i].w));
    top = max_g(top);
    const int b = (__builtin_bit_cast(int, top) >> 23) & 255, e = b == 255 ? 0 : min(13 + 127 - b, 120);
    const float up = __builtin_bit_cast(float, (127 + e) << 23);
#pragma unroll
    for (int i = 0; i < N / 8; i++) {
        f16x2 h[4], r[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 f = x[2 * i + j / 2];
            const float a = (j & 1 ? f.z : f.x) * up, c = (j & 1 ? f.w : f.y) * up;
            h[j] = to_half(a, c);
            r[j] = rest_half(h[j], BOTH ? 1.0f : low, a, c);
        }
        hi[i] = join8(BOTH ? h : r);
        if constexpr (BOTH) lo[i] = join8(r);
    }
    return __builtin_bit_cast(float, (127 - e) << 23);
}

/* Moves the bases of a wave's columns for a tile where one has to, mx being a lane's largest score, and
 * the sums l along; w is what a column's other sums are to be multiplied by, if it says so.  Bases are
 * whole, so that this rounds nothing.  Down only while the sums stay below 2^80 (values: 2^96). */
template <bool F16>
__device__ __forceinline__ bool base_moves(float mx, float &m, float &l, float &w)
{
    bool down = false;
    if (F16) {
        const unsigned long long near = __ballot(!(mx < m - M_DOWN));
        const unsigned c = (unsigned)near | (unsigned)(near >> 32);
        down = ((c | c >> 16) & 0xffff) != 0xffff;
    }
    if (!down && !__any(mx > m + LATE)) return false;
    const float top = floorf(max_g(mx));
    float to = fmaxf(m, top);
    if (down) {
        const float sum = max_g(l) * __builtin_amdgcn_exp2f(m - (top + M_MID));
        if (top < m - M_DOWN && top > -INFINITY && sum <= 0x1p80f) to = top + M_MID;       /* -inf: no position in the tile */
    }
    w = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
    l *= w;
    m = to;
    return true;
}

/* Not 0 if one of two fp16 values is infinite or NaN. */
__device__ __forceinline__ unsigned odd_half(unsigned x) { return (x & 0x7c007c00u) + 0x04000400u & 0x80008000u; }

/* One wave's state of a unit: lane (c = lane % 16, g = lane / 16) holds column c. */
template <int D, bool F16, bool WIDE>
struct AttWave {
    using C = AttCfg<D, F16, WIDE>;
    f16x8 qh[F16 ? C::KS : 1], ql[F16 && WIDE ? C::KS : 1];
    f32x4 qf[F16 ? 1 : C::KS];
    float fac;                      /* log2 score of a product, a power of two */
    float m, l;
    f32x4 o[C::NB * C::VE];
    gu32x4 k[C::KS];
    gu32x4 v[C::VT][C::NB];

    /* Column c's query as it lies, from q (a column without one computes another's and is
     * never stored). */
    static constexpr int QE = F16 ? 8 : 4;          /* elements of a product operand */
    struct Raw {
        float4 x[QE * C::KS / 4];
    };
    __device__ static void load_q(Raw &r, const float *q, int g)
    {
#pragma unroll
        for (int s = 0; s < C::KS; s++)
#pragma unroll
            for (int j = 0; j < QE / 4; j++) r.x[QE / 4 * s + j] = *(const float4 *)(q + QE * g + 4 * QE * s + 4 * j);
    }
    __device__ void clear()
    {
        m = -INFINITY;
        l = 0;
#pragma unroll
        for (int i = 0; i < C::NB * C::VE; i++) o[i] = (f32x4){};
    }
    __device__ void begin(Raw &r, int c, float scale)
    {
        const float f = scale * 1.44269504088896341f;
#pragma unroll
        for (int i = 0; i < QE * C::KS / 4; i++) { r.x[i].x *= f; r.x[i].y *= f; r.x[i].z *= f; r.x[i].w *= f; }
        fac = 1.0f;
        if constexpr (F16) fac = split_q<8 * C::KS, WIDE>(r.x, qh, ql, c < 8 ? 0.0f : 1.0f);
        else {
#pragma unroll
            for (int s = 0; s < C::KS; s++) qf[s] = (f32x4){ r.x[s].x, r.x[s].y, r.x[s].z, r.x[s].w };
        }
    }
    /* Keys of the tile that begins at byte `at`, a kilobyte to a load: with 64 bytes of each
     * of 16 tokens to a load, as the products take them, a read of nothing else comes at 5.9 TB/s, so
     * at 6.8. */
    __device__ void load_k(const char *kc, size_t at, int lane)
    {
#pragma unroll
        for (int i = 0; i < C::KS; i++) k[i] = __builtin_nontemporal_load((const GAS gu32x4 *)(kc + at + (i * 64 + lane) * 16));
    }
    /* The keys through this wave's own LDS into the products' order: piece x of token r lies
     * at x ^ (r % SW). */
    __device__ void store_k(gu32x4 *t, int lane)
    {
#pragma unroll
        for (int i = 0; i < C::KS; i++) {
            const int r = (i * 64 + lane) / C::NCH, x = lane % C::NCH;
            t[r * C::NCH + (x ^ r % C::SW)] = k[i];
        }
    }
    __device__ void load_v(const char *vc, size_t at, int c, int g)
    {
#pragma unroll
        for (int j = 0; j < C::VT; j++) {
            const char *b = vc + at;
            const unsigned off = ((4 * g + j) * D + C::VE * c) * C::SZ;
#pragma unroll
            for (int n = 0; n < C::NB; n++) {
                const GAS char *p = (const GAS char *)(b + off + 16 * C::VE * C::SZ * n);
                if (C::VE * C::SZ == 16) v[j][n] = __builtin_nontemporal_load((const GAS gu32x4 *)p);
                else {
                    const gu32x2 h = __builtin_nontemporal_load((const GAS gu32x2 *)p);
                    v[j][n] = (gu32x4){ h.x, h.y, 0, 0 };
                }
            }
        }
    }
    /* Scores of the tile in t, over fac: a lane gets its column's for tokens 4 g ..  In N sums
     * of their own (WIDE: high and low parts'), which wait less for each other and round less: of one
     * sum of 256 f32 products the outputs were off by 1.65e-6 (6 requests of 2700 tokens)
     * where those of four are by 0.54e-6. */
    template <int N>
    __device__ void scores(float *s, const gu32x4 *t, int c, int g)
    {
        f32x4 a[N] = {};
#pragma unroll
        for (int i = 0; i < C::KS; i++) {
            const gu32x4 x = t[c * C::NCH + ((4 * i + g) ^ c % C::SW)];
            if constexpr (F16) {
                f32x4 &to = a[WIDE ? 0 : i % N];
                to = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), qh[i], to, 0, 0, 0);
                if constexpr (WIDE) a[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), ql[i], a[1], 0, 0, 0);
            } else
#pragma unroll
                for (int j = 0; j < 4; j++)
                    a[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, x)[j], qf[i][j], a[j], 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j] = N == 2 ? a[0][j] + a[1][j] : (a[0][j] + a[1][j]) + (a[N - 2][j] + a[N - 1][j]);
            if (F16 && !WIDE) s[j] += dpp_f<0x128>(s[j]);              /* row_ror:8: the other part's column */
        }
    }
    /* The tile's softmax terms, p in place of the scores; `left` tokens of the tile count for
     * this column, all of them for every column unless `some`. */
    __device__ void soften(float *s, int left, bool some, int g)
    {
        float mx = -INFINITY;
        if (some)
            for (int j = 0; j < C::VT; j++)
                if (4 * g + j >= left) s[j] = -INFINITY;
        for (int j = 0; j < C::VT; j++) mx = fmaxf(mx, s[j]);
        mx *= fac;
        float w;
        if (base_moves<F16>(mx, m, l, w))
            for (int i = 0; i < C::NB * C::VE; i++) o[i] *= w;
        /* a column that has met no position yet keeps its terms 0 */
        const float base = m == -INFINITY ? 0.0f : Soft<F16>::UP - m;
        for (int j = 0; j < C::VT; j++) {
            s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], fac, base));
            l += s[j];
        }
    }
    /* Whether the tile's first `left` tokens have infinite or NaN values. */
    __device__ bool odd(int left, int g)
    {
        unsigned x = 0;
#pragma unroll
        for (int j = 0; j < C::VT; j++) {
            unsigned y = 0;
#pragma unroll
            for (int n = 0; n < C::NB; n++)
#pragma unroll
                for (int i = 0; i < C::VE * C::SZ / 4; i++)
                    y |= F16 ? odd_half(v[j][n][i]) : (v[j][n][i] & 0x7f800000u) + 0x00800000u & 0x80000000u;
            x |= 4 * g + j < left ? y : 0;
        }
        return __any(x != 0);
    }
    __device__ void values(const float *p, int left, int c, int g)
    {
        if (left < C::TT)                              /* what lies behind the rows or a bad page may be anything: 0 * NaN is NaN */
            for (int j = 0; j < C::VT; j++)
                if (4 * g + j >= left)
                    for (int n = 0; n < C::NB; n++) v[j][n] = (gu32x4){};
        if (F16) {
            const float low = WIDE || c >= 8 ? 1.0f : 0.0f;
            const f16x2 h0 = to_half(p[0], p[1]), h1 = to_half(p[2], p[3]);
            const f16x2 r0 = rest_half(h0, low, p[0], p[1]), r1 = rest_half(h1, low, p[2], p[3]);
            const f16x4 hi = { h0.x, h0.y, h1.x, h1.y }, lo = { r0.x, r0.y, r1.x, r1.y };      /* not WIDE: lo is this column's part */
#pragma unroll
            for (int n = 0; n < C::NB; n++)
#pragma unroll
                for (int e = 0; e < C::VE; e++) {
                    gu32x2 a;
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        a[j] = __builtin_amdgcn_perm(v[2 * j + 1][n][e / 2], v[2 * j][n][e / 2], e & 1 ? 0x07060302 : 0x05040100);
                    f32x4 &to = o[n * C::VE + e];
                    if constexpr (WIDE) to = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), hi, to, 0, 0, 0);
                    to = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), lo, to, 0, 0, 0);
                }
        } else {
            for (int n = 0; n < C::NB; n++)
                for (int e = 0; e < 4; e++)
                    for (int j = 0; j < 4; j++)
                        o[n * 4 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, v[j][n])[e], p[j],
                                                                            o[n * 4 + e], 0, 0, 0);
        }
    }
    /* The high parts' columns get the low parts' sums.  Where an infinite value made a
     * high sum infinite it stands for itself: the low one is NaN, or infinite the
     * other way. */
    __device__ void add_parts()
    {
        float top = 0;
#pragma unroll
        for (int i = 0; i < C::NB * C::VE; i++)
            top = fmaxf(fmaxf(fmaxf(top, fabsf(o[i][0])), fmaxf(fabsf(o[i][1]), fabsf(o[i][2]))), fabsf(o[i][3]));
        if (__any(top == INFINITY)) {
#pragma unroll
            for (int i = 0; i < C::NB * C::VE; i++)
                for (int j = 0; j < 4; j++) {
                    const float lo = dpp_f<0x128>(o[i][j]);
                    o[i][j] = fabsf(o[i][j]) == INFINITY ? o[i][j] : o[i][j] + lo;
                }
        } else {
#pragma unroll
            for (int i = 0; i < C::NB * C::VE; i++)
                for (int j = 0; j < 4; j++) o[i][j] += dpp_f<0x128>(o[i][j]);
        }
    }
};

/* Inclusive sums over the workgroup of 64-bit values; `tot` gets the whole. */
template <int W>
__device__ __forceinline__ long long att_scan(long long v, long long *s_wave, long long &tot)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    _Pragma("unroll")
    for (int o = 1; o < 64; o <<= 1) {
        const long long u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    if (lane == 63) s_wave[w] = v;
    __syncthreads();
    long long before = 0, all = 0;
    for (int i = 0; i < W; i++) {
        if (i == w) before = all;
        all += s_wave[i];
    }
    tot = all;
    return v + before;
}

/* What beginning a unit costs, in tiles, where shares are made equal: its row, page and
 * queries have to come before its first keys, and its sums go through LDS (700 requests of 1
 * to 500 tokens 84 us without it, 48 with it).  A unit of n tiles lies on LEAD + n
 * places, its tiles on the last n. */
#define ATT_LEAD 8
#define ROWS_LEAD 12          /* of 32 tokens; 4 requests of 1000 rows: 415 us with 4, 301 with 12, 313 with 24 */

/* Row t's request and tokens, and whether it goes on with the unit of row t - 1: runs of up to
 * R rows of one request, one behind the other with positions that do not fall, between
 * multiples of R. */
struct RowsAt {
    int req, n;
    bool joined;
};
__device__ __forceinline__ RowsAt rows_at(const RoasterAttnPaged &a, const KvTable &T, int shift, int R, int t)
{
    RowsAt x = { a.row_req[t], 0, false };
    x.n = T.tokens(x.req, a.row_pos[t], shift);            /* -1 for a row that is skipped, too */
    const int b = max(t - 1, 0), r = a.row_req[b], n = T.tokens(r, a.row_pos[b], shift);
    x.joined = t % R && r == x.req && n >= 0 && n <= x.n;
    return x;
}
/* Tiles of TT tokens of the unit that ends with row x, at least one for rows that have an
 * output to write; 0 if none ends there: its request is none or it goes on. */
template <int TT>
__device__ __forceinline__ int rows_tiles(const RowsAt &x, bool goes_on)
{
    if (x.req == -1 || goes_on) return 0;
    return x.n <= TT ? 1 : (int)(((long long)x.n + TT - 1) / TT);
}
template <int TT>
__device__ __forceinline__ int rows_tiles(const RoasterAttnPaged &a, const KvTable &T, int shift, int R, int t)
{
    const RowsAt x = rows_at(a, T, shift, R, t);
    return rows_tiles<TT>(x, R > 1 && t + 1 < a.rows && rows_at(a, T, shift, R, min(t + 1, a.rows - 1)).joined);
}
/* The first row of the unit that ends with row t1 (R at most 64), by a whole wave. */
__device__ __forceinline__ int rows_first(const RoasterAttnPaged &a, const KvTable &T, int shift, int R, int t1)
{
    if (R == 1) return t1;
    const int t = max(t1 - ((int)threadIdx.x & 63), 0);    /* row 0 goes on with none */
    return t1 - __builtin_ctzll(~__ballot(rows_at(a, T, shift, R, t).joined));
}

/* A wave's share holds its tile's keys, after its last tile its sums [COLS][D + 4]. */
template <int D, bool F16, bool WIDE>
struct AttLds {
    static constexpr int COLS = WIDE ? 16 : 8, KEYS = 16 * D * (F16 ? 2 : 4), SUMS = COLS * (D + 4) * 4;
    gu32x4 own[ATT_W][(KEYS > SUMS ? KEYS : SUMS) / 16];
    float m[ATT_W][COLS], l[ATT_W][COLS];
    int n[COLS], good[ATT_W], odd[ATT_W];
    __device__ float *sums(int w, int h) { return (float *)own[w] + h * (D + 4); }
};

/* out of one row's head from the sums y and l, four elements at d; 0, whatever the gate holds,
 * for a row without positions (`none`).  The reciprocals are off by one step, the
 * exponential by |gate| 2^-24 more: as little as the sums themselves. */
__device__ __forceinline__ void att_store(const RoasterAttnPaged &a, int D, int t, int h, int d, f32x4 y, float l, bool none)
{
    y = none ? (f32x4){} : y * __builtin_amdgcn_rcpf(l);
    if (a.gate && !none) {
        const f32x4 gt = *(const f32x4 *)(a.gate + t * a.gate_row + h * a.gate_head + d);
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(gt[i] * -1.44269504088896341f));
    }
    *(f32x4 *)(a.out + ((size_t)t * a.q_heads + h) * D + d) = y;
}

/* Tiles [first, last) of the unit of rows t0 .. t0 + nr - 1 and head block hb by one
 * workgroup: to out if that is all of them, else to part `slot` from column `off` on.  n: tokens
 * of its last row.  Gives back whether it found infinite or NaN values that some of the rows use and
 * others must not (0 * NaN is NaN): then it has written nothing, and the rows go one by one. */
template <int D, bool F16, bool WIDE, int N>
__device__ __forceinline__ bool att_part(const AttArgs &A, AttLds<D, F16, WIDE> &S, int *err, int t0, int nr, int req, int n, int hb,
                                         int first, int last, bool whole, int slot, int off)
{
    using C = AttCfg<D, F16, WIDE>;
    const RoasterAttnPaged &a = A.a;
    const KvTable T = { a.n_req, a.max_pages };
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), c = lane & 15, g = lane >> 4, shift = A.s.shift;
    const int kh = A.blocks == 1 ? hb : hb / A.blocks, bk = hb - kh * A.blocks, nh = min(A.hpb, A.group - bk * A.hpb);
    const int h0 = kh * A.group + bk * A.hpb;
    /* this lane's column: its row and head, and the tokens that count for it */
    const int cr = WIDE ? c / A.hpb : 0, ch = WIDE ? c - cr * A.hpb : c & 7;
    const bool on = cr < nr && ch < nh;
    int nc = n;
    if (WIDE && nr > 1) nc = on ? T.tokens(req, a.row_pos[t0 + cr], shift) : 0;
    int good = n < 0 ? -2 : n;     /* tokens before the first bad page: rows of more are NaN, all if the row itself is bad */
    int odd = 0;
    AttWave<D, F16, WIDE> wv;
    typename AttWave<D, F16, WIDE>::Raw raw;
    /* the page of tile i, then the byte at which the tile begins */
    auto page = [&](int i) { return a.table[T.entry(req, i * 16, shift)]; };
    auto where = [&](int i, int p) {
        int pg = uni(p);
        if (!A.s.page_ok(pg)) { good = min(good, i * 16); pg = 0; }
        return A.s.at(pg, kh, i * 16 & ((1 << shift) - 1)) * C::SZ;
    };
    wv.clear();
    int i = first + w;
    if (n > 0 && i < last) {
        int p = page(i), i2 = i + ATT_W;
        wv.load_q(raw, a.q + ((size_t)(t0 + (on ? cr : 0)) * a.q_heads + h0 + (on ? ch : 0)) * D, g);
        size_t b = where(i, p);
        wv.load_k(A.kc, b, lane);
        if (i2 < last) p = page(i2);
        wv.load_v(A.vc, b, c, g);
        wv.begin(raw, c, a.scale);
        int least = n;                                 /* over the columns in use */
        if (WIDE && nr > 1) {
            least = on ? nc : n;
            for (int x = 1; x < 16; x <<= 1) least = min(least, __shfl_xor(least, x));
            least = uni(least);
        }
        while (1) {
            const bool more = i2 < last;
            float s[C::VT];
            wv.store_k(S.own[w], lane);
            if (more) {
                b = where(i2, p);
                wv.load_k(A.kc, b, lane);
                if (i2 + ATT_W < last) p = page(i2 + ATT_W);
            }
            wv.template scores<N>(s, S.own[w], c, g);
            wv.soften(s, nc - i * 16, least < (i + 1) * 16, g);
            if (WIDE && nr > 1 && least < (i + 1) * 16 && wv.odd(good - i * 16, g)) odd = 1;
            wv.values(s, good - i * 16, c, g);
            if (!more) break;
            wv.load_v(A.vc, b, c, g);
            i = i2;
            i2 += ATT_W;
        }
    }
    const float l = sum_g(wv.l);
    if (g == 0 && c < C::COLS) {
        S.m[w][c] = wv.m;
        S.l[w][c] = l;
        if (w == 0) S.n[c] = nc;
    }
    if (lane == 0) { S.good[w] = good; S.odd[w] = odd; }
    if constexpr (F16 && !WIDE) wv.add_parts();
#pragma unroll
    for (int b = 0; b < C::NB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (c < C::COLS)
#pragma unroll
                for (int e = 0; e < C::VE; e += 4)
                    *(float4 *)(S.sums(w, c) + 16 * C::VE * b + C::VE * (4 * g + i) + e) =
                        make_float4(wv.o[b * C::VE + e][i], wv.o[b * C::VE + e + 1][i], wv.o[b * C::VE + e + 2][i],
                                    wv.o[b * C::VE + e + 3][i]);
    __syncthreads();
    for (int i = 0; i < ATT_W; i++) good = min(good, S.good[i]);
    if (WIDE && nr > 1) {
        for (int i = 0; i < ATT_W; i++) odd |= S.odd[i];
        if (odd) return true;
    }
    if (good < n && tid == 0) atomicOr(err, ATTN_ERR_INDEX);
    for (int idx = tid * 4; idx < C::COLS * D; idx += ATT_T * 4) {
        const int h = idx / D, d = idx % D, row = WIDE ? h / A.hpb : 0, head = h - row * A.hpb;
        if (row >= nr || head >= nh) continue;
        float mx = -INFINITY, sum = 0;
        f32x4 y = {};
#pragma unroll
        for (int i = 0; i < ATT_W; i++) mx = fmaxf(mx, S.m[i][h]);
#pragma unroll
        for (int i = 0; i < ATT_W; i++) {
            const float f = S.m[i][h] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(S.m[i][h] - mx);
            sum += S.l[i][h] * f;
            y += *(const f32x4 *)(S.sums(i, h) + d) * f;
        }
        if (S.n[h] > good) { y = (f32x4){ NAN, NAN, NAN, NAN }; sum = NAN; }
        if (whole) att_store(a, D, t0 + row, h0 + head, d, y, sum, S.n[h] == 0);
        else {
            *(f32x4 *)(A.po + ((size_t)slot * C::COLS + off + h) * D + d) = y;
            if (d == 0) {
                A.pm[slot * C::COLS + off + h] = mx;
                A.pl[slot * C::COLS + off + h] = sum;
            }
        }
    }
    return false;
}

/* Few units (at most an eighth of the workgroups, of at most 128 rows): every workgroup
 * takes one unit's part.  All tiles over (workgroups - units) is a part's size that gives
 * no more parts than workgroups, since a unit of n tiles has ceil(n / size); a unit's
 * parts are equal.  Each wave finds its part from the rows by itself, without a barrier.
 * 8 requests of 100..8000 tokens, 2 key/value heads: 19 us, with even shares 27; 32 of them,
 * the most there may be: 33, with even shares 32; 64 of them 54 and 50. */
template <int D, bool F16, bool WIDE>
__global__ __launch_bounds__(ATT_T, D == 256 && !F16 ? 1 : 2) void attn_few_kernel(AttArgs A, int *err)
{
    using C = AttCfg<D, F16, WIDE>;
    __shared__ AttLds<D, F16, WIDE> S;
    const RoasterAttnPaged &a = A.a;
    const KvTable T = { a.n_req, a.max_pages };
    const int lane = threadIdx.x & 63, shift = A.s.shift, rows = a.rows, per_row = A.s.kv * A.blocks;
    int req[2], tok[2], tl[2] = { 0, 0 };
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int t = min(lane + 64 * k, rows - 1);
        const RowsAt x = rows_at(a, T, shift, 1, t);
        req[k] = x.req;
        tok[k] = x.n;
        if (lane + 64 * k < rows) {
            tl[k] = rows_tiles<C::TT>(x, false);
            if (tl[k] == 0 && blockIdx.x == 0 && threadIdx.x < 64)       /* no unit: nothing to join */
                for (int u = 0; u < per_row; u++) A.cut[t * per_row + u].k = 0;
        }
    }
    /* the sum in f32, a little too large if anything */
    const float all = group_sum<64>((float)tl[0] + (float)tl[1]) * per_row;
    const int size = max(ATT_MIN, (int)(all * (1.0001f / ((int)gridDim.x - rows * per_row))) + 1);
    int ch[2], in[2];
    ch[0] = in[0] = (tl[0] + size - 1) / size;
    ch[1] = in[1] = (tl[1] + size - 1) / size;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u0 = __shfl_up(in[0], o), u1 = rows > 64 ? __shfl_up(in[1], o) : 0;
        if (lane >= o) { in[0] += u0; in[1] += u1; }
    }
    in[1] += __builtin_amdgcn_readlane(in[0], 63);
    const int me = blockIdx.x, r0 = __popcll(__ballot(in[0] * per_row <= me)),
              r1 = r0 < 64 ? 0 : __popcll(__ballot(in[1] * per_row <= me)), t = r0 + r1;
    if (t >= rows) return;
    const int src = t & 63;
    auto pick = [&](const int *v) { return t < 64 ? __builtin_amdgcn_readlane(v[0], src) : __builtin_amdgcn_readlane(v[1], src); };
    const int chunks = pick(ch), tiles = pick(tl), at = me - (pick(in) - chunks) * per_row;
    const int hb = uni(at / chunks), k = at - hb * chunks, base = uni(tiles / chunks), rem = tiles - base * chunks;
    const int first = k * base + min(k, rem), last = first + base + (k < rem);
    att_part<D, F16, WIDE, F16 && WIDE ? 2 : 4>(A, S, err, t, 1, pick(req), pick(tok), hb, first, last, chunks == 1, me, 0);
    if (k == 0 && threadIdx.x == 0) A.cut[t * per_row + hb] = (AttCut){ t, 1, hb, me, chunks == 1 ? 0 : chunks };
}

template <int D, bool F16, bool WIDE>
__global__ __launch_bounds__(ATT_T, D == 256 && !F16 ? 1 : 2) void attn_kernel(AttArgs A, int *err)
{
    using C = AttCfg<D, F16, WIDE>;
    __shared__ AttLds<D, F16, WIDE> S;
    __shared__ long long s_wave[ATT_W], s_at;
    __shared__ int s_row;
    const RoasterAttnPaged &a = A.a;
    const KvTable T = { a.n_req, a.max_pages };
    const int tid = threadIdx.x, shift = A.s.shift, per_row = A.s.kv * A.blocks, rows = a.rows, R = WIDE ? A.R : 1;

    /* this share: the places [at, end) of all units' laid end to end */
    const int each = (rows + ATT_T - 1) / ATT_T;
    auto places = [&](int t) {
        const int k = rows_tiles<C::TT>(a, T, shift, R, t);
        return k ? ATT_LEAD + k : 0;
    };
    long long mine = 0, tot;
    for (int i = 0; i < each; i++) {
        const int t = tid * each + i;
        if (t >= rows) break;
        const int k = places(t);
        mine += k;
        if (k == 0 && A.by_unit && blockIdx.x == 0)    /* no unit: nothing to join */
            for (int u = 0; u < per_row; u++) A.cut[t * per_row + u].k = 0;
    }
    const long long upto = att_scan<ATT_W>(mine, s_wave, tot);
    const long long all = tot * per_row, share = max((long long)ATT_MIN, (all + gridDim.x - 1) / gridDim.x);
    long long at = blockIdx.x * share;
    const long long end = min(all, at + share);
    if (at >= end) {
        if (!A.by_unit && tid == 0) A.cut[blockIdx.x].k = 0;
        return;
    }
    if (at < upto * per_row && at >= (upto - mine) * per_row) {        /* one thread's rows hold it */
        long long b = (upto - mine) * per_row;
        int t = tid * each, n;
        while (at >= b + (n = places(t)) * (long long)per_row) {
            b += n * (long long)per_row;
            t++;
        }
        s_row = t;
        s_at = b;
    }
    __syncthreads();
    int t = uni(s_row), req = uni(a.row_req[t]), n = uni(T.tokens(req, a.row_pos[t], shift));
    int tiles = rows_tiles<C::TT>((RowsAt){ req, n, false }, false);
    int hb = uni((int)((at - s_at) / (ATT_LEAD + tiles))), x0 = uni((int)((at - s_at) % (ATT_LEAD + tiles)));
    while (1) {
        /* places [x0, x1) and tiles [first, last) of unit (t, hb) */
        const int x1 = uni((int)min((long long)ATT_LEAD + tiles, x0 + (end - at)));
        const int first = max(0, x0 - ATT_LEAD), last = max(0, x1 - ATT_LEAD);
        const bool cuts = first == 0 && last > 0 && last < tiles, over = at + (x1 - x0) == end;
        const bool step = !over && hb + 1 == per_row;
        int req1 = -1, pos1 = 0;
        if (step && R == 1) {                          /* the next row, while this one is worked on */
            req1 = a.row_req[t + 1];
            pos1 = a.row_pos[t + 1];
        }
        const int t0 = uni(rows_first(a, T, shift, R, t)), nr = t - t0 + 1;
        if (last > first) {
            int t = t0, rows_n = nr, row_n = n;        /* the unit's rows together, or one by one */
            while (1) {
                /* at dim 256 four sums of scores would spill: 102 us instead of 94 (64 requests) */
                const bool odd = att_part<D, F16, WIDE, F16 && (WIDE || D == 256) ? 2 : 4>(
                    A, S, err, t, rows_n, req, row_n, hb, first, last, first == 0 && last == tiles, 2 * blockIdx.x + (first == 0),
                    (t - t0) * A.hpb);
                if (!WIDE || (rows_n == nr && !odd) || (rows_n != nr && t == t0 + nr - 1)) break;
                t = rows_n == nr ? t0 : t + 1;
                rows_n = 1;
                row_n = uni(T.tokens(req, a.row_pos[t], shift));
                __syncthreads();                       /* S is free again */
            }
        }
        if (tid == 0) {                                /* for the join: the shares of a unit begun and cut here */
            const int k = cuts ? (int)((at - x0 + ATT_LEAD + tiles - 1) / share) - (int)blockIdx.x + 1 : 0;
            const AttCut x = { t0, nr, hb, (int)blockIdx.x, k };
            if (A.by_unit && first == 0 && last > 0) A.cut[t * per_row + hb] = x;
            if (!A.by_unit && over) A.cut[blockIdx.x] = x;
        }
        if (over) break;
        at += x1 - x0;
        x0 = 0;
        hb++;
        if (step) {
            hb = 0;
            t++;
            if (R == 1 && uni(req1) != -1) {
                req = uni(req1);
                n = uni(T.tokens(req, pos1, shift));
            } else
                for (bool on = true; on;) {            /* the next row that ends a unit, 64 rows at a time */
                    const int u = t + (tid & 63), k = u < rows ? rows_tiles<C::TT>(a, T, shift, R, u) : 0;
                    const unsigned long long j = __ballot(k > 0);
                    on = j == 0;
                    t += on ? 64 : __builtin_ctzll(j);
                    if (!on) {
                        req = uni(a.row_req[t]);
                        n = uni(T.tokens(req, a.row_pos[t], shift));
                    }
                }
            tiles = rows_tiles<C::TT>((RowsAt){ req, n, false }, false);
        }
        __syncthreads();                               /* S is free again */
    }
}

/* ---- several rows of a request together (fp16 cache) ------------------------
 * A run is up to R rows of one request, one behind the other with positions that
 * do not fall: a prompt's chunk.  The workgroup brings each tile of 32 tokens into LDS
 * once, straight from memory, for its eight waves of 16 columns (row, head), which
 * multiply every operand they read by their columns' high and low parts.  Shares, cuts
 * and the join go as in attn_kernel, a unit being a run and a block of heads.
 * With HALVES 2 a run has half as many columns, and two waves share theirs, taking
 * the tiles in turn and joining in LDS: half the bytes of parts, twice the tiles to bring.
 * What bounds it: a tile is 64 MFMAs, 200 other vector instructions and 32 KB of LDS reads a
 * wave, about 2 us of the two waves on a SIMD, a third of the matrix cores' rate (each wave a
 * chain of reads, products and softmax, which 256 registers let no third wave fill); before a
 * unit's first tile lie 9 to 12 us (rows, page, queries and tile, each a wait), behind its last 1 to
 * 2, and the join takes 8 to 20.  256 rows behind 2048 tokens 45 us, 512 rows 65, a prompt of 1024
 * 62, of 2000 120, four prompts' 1000 rows behind 0..3000 tokens 301. */
#define ROWS_G 256            /* workgroups: one per CU */
#define ROWS_T 512
#define ROWS_W (ROWS_T / 64)
#define ROWS_COLS 128         /* columns of a unit: 16 a wave; half as many where two waves share theirs */
#define ROWS_PART(D, COLS) ((COLS) * (D) / 4 + 80)       /* a part in units of four sums, off a power of two: its unit's parts are read together */

/* s_waitcnt's operand for no load and no store under way, LDS and exports not waited for. */
#define ROWS_ALL_CAME ((7 << 4) | (15 << 8))
#define CAS __attribute__((address_space(4)))

/* Pieces of 16 bytes from LDS bytes a0..a3, further O0 and further O1
 * for the second four.  In one block with their wait: a read that the compiler sees
 * would wait for every tile under way into LDS. */
template <int O0, int O1>
__device__ __forceinline__ void lds_read8(gu32x4 *r, int a0, int a1, int a2, int a3)
{
    asm volatile("ds_read_b128 %0, %8 offset:%12\n\tds_read_b128 %1, %9 offset:%12\n\t"
                 "ds_read_b128 %2, %10 offset:%12\n\tds_read_b128 %3, %11 offset:%12\n\t"
                 "ds_read_b128 %4, %8 offset:%13\n\tds_read_b128 %5, %9 offset:%13\n\t"
                 "ds_read_b128 %6, %10 offset:%13\n\tds_read_b128 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                 : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(O0), "n"(O1) : "memory");
}
__device__ __forceinline__ void lds_read4(gu32x4 *r, int a0, int a1, int a2, int a3)
{
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]) : "v"(a0), "v"(a1), "v"(a2), "v"(a3) : "memory");
}
/* Eight operands of 16 elements' values each from the addresses a[], tokens of the first
 * half at O0 and of the second at O1: the transposing read takes 4 rows of 16 elements
 * from 16 lanes (lane 4 r + q: elements 4 q .. of row r) and gives lane c the four
 * elements of column c. */
template <int O0, int O1>
__device__ __forceinline__ void lds_cols8(gu32x2 (*r)[2], const int *a)
{
    asm volatile("ds_read_b64_tr_b16 %0, %16 offset:%24\n\tds_read_b64_tr_b16 %1, %16 offset:%25\n\t"
                 "ds_read_b64_tr_b16 %2, %17 offset:%24\n\tds_read_b64_tr_b16 %3, %17 offset:%25\n\t"
                 "ds_read_b64_tr_b16 %4, %18 offset:%24\n\tds_read_b64_tr_b16 %5, %18 offset:%25\n\t"
                 "ds_read_b64_tr_b16 %6, %19 offset:%24\n\tds_read_b64_tr_b16 %7, %19 offset:%25\n\t"
                 "ds_read_b64_tr_b16 %8, %20 offset:%24\n\tds_read_b64_tr_b16 %9, %20 offset:%25\n\t"
                 "ds_read_b64_tr_b16 %10, %21 offset:%24\n\tds_read_b64_tr_b16 %11, %21 offset:%25\n\t"
                 "ds_read_b64_tr_b16 %12, %22 offset:%24\n\tds_read_b64_tr_b16 %13, %22 offset:%25\n\t"
                 "ds_read_b64_tr_b16 %14, %23 offset:%24\n\tds_read_b64_tr_b16 %15, %23 offset:%25\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[2][0]), "=&v"(r[2][1]),
                   "=&v"(r[3][0]), "=&v"(r[3][1]), "=&v"(r[4][0]), "=&v"(r[4][1]), "=&v"(r[5][0]), "=&v"(r[5][1]),
                   "=&v"(r[6][0]), "=&v"(r[6][1]), "=&v"(r[7][0]), "=&v"(r[7][1])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "n"(O0), "n"(O1)
                 : "memory");
}
template <int O0, int O1>
__device__ __forceinline__ void lds_cols4(gu32x2 (*r)[2], const int *a)
{
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0][0]), "=&v"(r[0][1]), "=&v"(r[1][0]), "=&v"(r[1][1]), "=&v"(r[2][0]), "=&v"(r[2][1]),
                   "=&v"(r[3][0]), "=&v"(r[3][1])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(O0), "n"(O1) : "memory");
}

struct RowsCut {
    int row, n, hb, k;        /* first row, rows and head block of a unit, and its number of shares (0: not to be joined) */
};

struct RowsArgs {
    RoasterAttnPaged a;
    const char *kc, *vc;
    KvShape s;
    int group, blocks, hpb;   /* query heads of a key/value head, their blocks, heads of a block */
    int rpg, R;               /* rows of a column group, of a run */
    RowsCut *cut;             /* [ROWS_G] by the share that began a unit and did not finish it */
    float *pm, *pl, *po;      /* parts [2 ROWS_G][waves][16 columns], and [..][waves][D / 16][64 lanes][4]; slots as in AttArgs */
};

/* What the pieces' numbers in row r of 16 are turned by: keys' reads take one piece of
 * each row, values' two neighbours of eight rows (0..7 or 8..15), each all over the banks, 16
 * pieces wide.  A row of 64 elements is half as wide. */
template <int SW>
__device__ __forceinline__ int rows_turn(int r)
{
    return SW == 16 ? (r & 7) << 1 | r >> 3 : (r & 6) | r >> 3;
}

template <int D, int HALVES>
__global__ __launch_bounds__(ROWS_T, 2) void attn_rows_kernel(RowsArgs A, int *err)
{
    constexpr int CH = D / 8, KS = D / 32, NO = D / 16;   /* 16-byte pieces of a token; steps of a score; sums of a lane */
    constexpr int SW = CH < 16 ? CH : 16, KJ = SW / 4, VJ = SW / 2;
    constexpr int GROUPS = ROWS_W / HALVES;        /* of 16 columns: HALVES waves each, taking its tiles in turn */
    __shared__ gu32x4 s_t[4][2][32 * CH];          /* tiles of keys and values: two in use, two under way */
    __shared__ long long s_wave[ROWS_W], s_at;
    __shared__ int s_row, s_tiles, s_np, s_req, s_n, s_runs[ROWS_W];
    __shared__ int s_parts[ROWS_W];
    __shared__ float4 s_try[ROWS_W];
    __shared__ unsigned long long s_join[ROWS_W];          /* the rows that go on with a run, a bit each */
    __shared__ float s_sum[ROWS_W];
    const RoasterAttnPaged &a = A.a;
    const KvTable T = { a.n_req, a.max_pages };
    const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6), c = lane & 15, g = lane >> 4, shift = A.s.shift;
    const int per_row = A.s.kv * A.blocks, rows = a.rows, R = A.R;
    __builtin_assume(R > 1);

    /* this share: the places [at, end) of all units' laid end to end, or with few units one of
     * np equal parts of one unit (a share that two units meet in begins twice) */
    const int each = (rows + ROWS_T - 1) / ROWS_T;
    long long mine = 0, at = 0, end = 0, share = 1;
    int tl = 0, np = 0, hb, x0, req = 0, n = 0;
    auto places = [](int k) { return k ? ROWS_LEAD + k : 0; };
    if (each == 1) {                                   /* at most 512 runs, one a thread */
        const int G = gridDim.x, t = min(tid, rows - 1);
        const RowsAt x = rows_at(a, T, shift, R, t), y = rows_at(a, T, shift, R, min(t + 1, rows - 1));
        if (tid < rows) tl = rows_tiles<32>(x, t + 1 < rows && y.joined);
        req = x.req;
        n = x.n;
        mine = places(tl);
        const float some = group_sum<64>((float)tl);
        const unsigned long long on = __ballot(x.joined), runs = __ballot(tl > 0);
        if (lane == 0) {
            s_sum[w] = some;
            s_runs[w] = __popcll(runs);
            s_join[w] = on;
        }
        __syncthreads();
        float W = 0;
        int units = 0;
#pragma unroll
        for (int i = 0; i < ROWS_W; i++) { W += s_sum[i]; units += s_runs[i]; }
        W *= per_row;
        units *= per_row;
        /* Equal parts of S tiles, S the least of five with no more parts than workgroups, a unit
         * of n tiles having ceil(n / S): from all tiles over all workgroups to where there cannot
         * be too many (the quotients in f32: `hi` is a little too large).  Worth it while its
         * excess is less than a second beginning. */
        const bool parts = units > 0 && units <= G - G / 4;
        const unsigned lo = max(ATT_MIN, (int)ceilf(W / G)), hi = max(lo, (unsigned)(W * 1.0001f / max(G - units, G / 4)) + 1);
        unsigned S = hi;
        if (parts && hi > lo) {
            const unsigned d = (hi - lo) / 8;
            const unsigned at[4] = { lo, min(lo + max(1u, d), hi), min(lo + max(2u, 2 * d), hi), min(lo + max(3u, 4 * d), hi) };
            float4 f;
            f.x = group_sum<64>((float)((tl + at[0] - 1) / at[0]));
            f.y = group_sum<64>((float)((tl + at[1] - 1) / at[1]));
            f.z = group_sum<64>((float)((tl + at[2] - 1) / at[2]));
            f.w = group_sum<64>((float)((tl + at[3] - 1) / at[3]));
            if (lane == 0) s_try[w] = f;
            __syncthreads();
            f = s_try[0];
#pragma unroll
            for (int i = 1; i < ROWS_W; i++) { f.x += s_try[i].x; f.y += s_try[i].y; f.z += s_try[i].z; f.w += s_try[i].w; }
            const float most = G / per_row;
            S = f.x <= most ? at[0] : f.y <= most ? at[1] : f.z <= most ? at[2] : f.w <= most ? at[3] : hi;
        }
        if (parts && S <= lo + ROWS_LEAD) {
            const int me = blockIdx.x, mp = (tl + S - 1) / S;
            int upto = mp, all = 0;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int u = __shfl_up(upto, o);
                if (lane >= o) upto += u;
            }
            if (lane == 63) s_parts[w] = upto;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ROWS_W; i++) {
                if (i == w) upto += all;
                all += s_parts[i];
            }
            if (me >= all * per_row) {
                if (tid == 0) A.cut[me].k = 0;
                return;
            }
            if (me < upto * per_row && me >= (upto - mp) * per_row) {
                s_row = tid;
                s_tiles = tl;
                s_np = mp;
                s_req = req;
                s_n = n;
                s_at = (upto - mp) * per_row;
            }
            __syncthreads();
            np = uni(s_np);
            const int tiles = uni(s_tiles), k0 = me - (int)s_at;
            hb = uni(k0 / np);
            const int k = k0 - hb * np, base = uni(tiles / np), rem = tiles - base * np;
            x0 = ROWS_LEAD + k * base + min(k, rem);
            end = base + (k < rem);
        }
    } else
        for (int i = 0; i < each; i++) {
            const int t = tid * each + i;
            if (t < rows) mine += places(tl = rows_tiles<32>(a, T, shift, R, t));
        }
    if (np == 0) {
        long long tot;
        const long long upto = att_scan<ROWS_W>(mine, s_wave, tot);
        const long long all = tot * per_row;
        share = max((long long)ATT_MIN, (all + gridDim.x - 1) / gridDim.x);
        at = blockIdx.x * share;
        end = min(all, at + share);
        if (at >= end) {
            if (tid == 0) A.cut[blockIdx.x].k = 0;
            return;
        }
        if (at < upto * per_row && at >= (upto - mine) * per_row) {
            long long b = (upto - mine) * per_row;
            int t = tid * each;
            if (each > 1)
                while (at >= b + places(tl = rows_tiles<32>(a, T, shift, R, t)) * (long long)per_row) {
                    b += places(tl) * (long long)per_row;
                    t++;
                }
            if (each > 1) {
                req = a.row_req[t];
                n = T.tokens(req, a.row_pos[t], shift);
            }
            s_row = t;
            s_tiles = tl;
            s_at = b;
            s_req = req;
            s_n = n;
        }
        __syncthreads();
        hb = uni((int)((at - s_at) / (ROWS_LEAD + s_tiles)));
        x0 = uni((int)((at - s_at) % (ROWS_LEAD + s_tiles)));
    }
    int t1 = uni(s_row), tiles = uni(s_tiles);
    req = uni(s_req);
    n = uni(s_n);
    /* Where this lane's operands lie in a tile, in bytes: its key's piece 4 s + g at kb[s % KJ]
     * + 64 (s - s % KJ), its share of the values' 16 elements j at vb[j % VJ] + 32 (j - j % VJ):
     * four elements of token 4 g + c / 4.  (4 s + g) ^ r = 4 (s ^ r / 4) + (g ^ r % 4), and
     * alike for the pieces 2 j + (c & 2) / 2. */
    int kb[KJ], vb[VJ];
    const int t0_at = (int)(uintptr_t)(__attribute__((address_space(3))) void *)&s_t[0][0][0], vr = 4 * g + c / 4,
              fk = rows_turn<SW>(c), fv = rows_turn<SW>(vr);
#pragma unroll
    for (int k = 0; k < KJ; k++) kb[k] = t0_at + (c * CH + 4 * (k ^ fk / 4) + (g ^ fk % 4)) * 16;
#pragma unroll
    for (int k = 0; k < VJ; k++)
        vb[k] = t0_at + (vr * CH + 2 * (k ^ fv / 2) + ((c >> 1 & 1) ^ (fv & 1))) * 16 + 8 * (c & 1);
    const int cr = c / A.hpb, ch = c - cr * A.hpb;                      /* this lane's column: its row and head within the group */
    while (1) {
        /* places [x0, x1) and tiles [first, last) of this unit */
        const int x1 = uni((int)min((long long)ROWS_LEAD + tiles, x0 + (end - at)));
        const int first = max(0, x0 - ROWS_LEAD), last = max(0, x1 - ROWS_LEAD);
        if (last == 0) {                               /* the next share begins it */
            if (tid == 0) A.cut[blockIdx.x].k = 0;
            break;
        }
        const bool whole = first == 0 && last == tiles, cuts = first == 0 && !whole;
        /* the run's first row: the last one up to t1 that does not go on with the one before it */
        int t0 = t1;
        if (each == 1) {
            int k = t1 >> 6;
            unsigned long long j = ~s_join[k] & (~0ull >> (63 - (t1 & 63)));
            while (!j) j = ~s_join[--k];               /* row 0 goes on with none */
            t0 = uni(64 * k + 63 - __builtin_clzll(j));
        } else
            for (bool on = true; on;) {                /* 64 rows at a time */
                const int t = t0 - lane;
                const unsigned long long j = __ballot(t > 0 && rows_at(a, T, shift, R, t).joined);
                on = j == ~0ull;
                t0 -= on ? 64 : __builtin_ctzll(~j);
            }
        const int nr = t1 - t0 + 1;
        const int kh = A.blocks == 1 ? hb : hb / A.blocks, bk = hb - kh * A.blocks, nh = min(A.hpb, A.group - bk * A.hpb);
        const int h0 = kh * A.group + bk * A.hpb;
        bool bad = n < 0;

        /* page numbers of tile i's two 16-token parts (a part past the run's end repeats
         * the first), then the bytes at which the parts begin */
        auto pages = [&](int i, int *p) {
            const CAS int *t = (const CAS int *)a.table;              /* scalar loads: they stay out of the tiles' count */
            p[0] = t[T.entry(req, i * 32, shift)];
            p[1] = i * 32 + 16 < n ? t[T.entry(req, i * 32 + 16, shift)] : p[0];
        };
        auto where = [&](int i, const int *p, size_t *b) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int tok = i * 32 + 16 * u;
                int pg = p[u], in = (u && tok >= n ? tok - 16 : tok) & ((1 << shift) - 1);
                if (__builtin_expect(!A.s.page_ok(pg), 0)) {                /* the first part's page in its place, whose values rows may meet times 0 */
                    bad = true;
                    pg = ((const CAS int *)a.table)[T.entry(req, 0, shift)];
                    if (!A.s.page_ok(pg)) pg = 0;
                    in = 0;
                }
                b[u] = A.s.at(pg, kh, in) * 2;
            }
        };
        /* The tile's 64 CH pieces straight into LDS, 64 to a wave and load, in the order
         * they lie there: piece x of a token's row lies at x ^ rows_turn(row), so that what
         * an operand read takes falls on different banks.  A load's rows lie in one
         * 16-token part. */
        auto fetch = [&](int buf, const size_t *b) {
#pragma unroll
            for (int i = 0; i < CH / ROWS_W; i++) {
                const int q = i * ROWS_W + w, v = q >= CH / 2, at = (q - v * (CH / 2)) * 64, row = (at + lane) / CH;
                const char *from = (v ? A.vc : A.kc) + (at / CH < 16 ? b[0] : b[1]);
                const unsigned off = ((row & 15) * CH + ((at + lane) % CH ^ rows_turn<SW>(row & 15))) * 16;
                __builtin_amdgcn_global_load_lds((const GAS void *)(from + off),
                                                 (__attribute__((address_space(3))) void *)&s_t[buf][v][at], 16, 0, 0);
            }
        };
        size_t b[2];
        int pg[2][2];
        if (n > 0) {
            pages(first, pg[0]);
            pages(min(first + 1, last - 1), pg[1]);
        }
        /* this lane's column */
        const int grp = HALVES == 1 ? w : w % GROUPS, half = HALVES == 1 ? 0 : w / GROUPS, ri = grp * A.rpg + cr;
        const bool on = cr < A.rpg && ri < nr && ch < nh;
        f16x8 qh[KS], ql[KS];
        f32x4 o[NO];
        float m = -INFINITY, l = 0, fac;
        const int nc = on ? T.tokens(req, a.row_pos[t0 + ri], shift) : 0;
        float4 qx[2 * KS];
        {
            const float *q = a.q + ((size_t)(t0 + (on ? ri : 0)) * a.q_heads + h0 + (on ? ch : 0)) * D + 8 * g;
#pragma unroll
            for (int s = 0; s < 2 * KS; s++) qx[s] = *(const float4 *)(q + 32 * (s / 2) + 4 * (s % 2));
        }
        /* tiles i and i + 1, and the page numbers of the two behind them */
        auto bring = [&](int i, int buf) {
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (i + k < last) {
                    where(i + k, pg[k], b);
                    fetch(buf + k, b);
                }
        };
        if (n > 0) {
            bring(first, 0);
            pages(min(first + 2, last - 1), pg[0]);
            pages(min(first + 3, last - 1), pg[1]);
        }
        #pragma unroll
        for (int s = 0; s < 2 * KS; s++) {
            const float f = a.scale * 1.44269504088896341f;
            qx[s].x *= f; qx[s].y *= f; qx[s].z *= f; qx[s].w *= f;
        }
        fac = split_q<8 * KS, true>(qx, qh, ql, 1.0f);
#pragma unroll
        for (int k = 0; k < NO; k++) o[k] = (f32x4){};
        if (n > 0) {
            int most = nc, least = on ? nc : INT32_MAX;                /* over the wave's columns in use */
            for (int x = 32; x; x >>= 1) {
                most = max(most, __shfl_xor(most, x));
                least = min(least, __shfl_xor(least, x));
            }
            most = uni(most);
            least = uni(least);
            /* this wave's own rows may end before the run does: then it only brings tiles */
            const int mine = min(last, (int)(((long long)most + 31) / 32));
            for (int i0 = first; i0 < last; i0 += 2) {
                /* both tiles have come, to this wave and the others, and the two before are done
                 * with; a barrier for two tiles lets a SIMD's two waves drift apart, so that
                 * one's MFMAs run beside the other's softmax */
                const int buf = (i0 - first) & 2;
                __builtin_amdgcn_s_waitcnt(ROWS_ALL_CAME);
                __syncthreads();
                bring(i0 + 2, buf ^ 2);
                const int to = min(i0 + 2, mine);
#pragma unroll 1
                for (int i = i0 + half; i < to; i += HALVES) {
                const int at = (buf + i - i0) * (int)sizeof(s_t[0]);
                int kt[4], vt[VJ];                     /* this tile's operands */
#pragma unroll
                for (int k = 0; k < 4; k++) kt[k] = at + (KJ == 4 ? kb[k % KJ] : kb[k % 2] + k / 2 * CH * 256);
#pragma unroll
                for (int k = 0; k < VJ; k++) vt[k] = at + (int)sizeof(s_t[0][0]) + vb[k];
                {
                    /* a block's low parts first, whose small sums round little, and blocks apart: outputs
                     * off by 0.5e-6, in one sum by 1.1e-6 */
                    f32x4 acc[D == 256 ? 2 : 1][2] = {};
#pragma unroll
                    for (int q = 0; q < (D == 256 ? 2 : 1); q++) {
                        constexpr int S = D == 64 ? 2 : 4;             /* products of a chain that one block's reads feed */
                        gu32x4 kf[8];
                        if constexpr (D == 64) lds_read4(kf, kt[0], kt[1], kt[2], kt[3]);
                        else if (q == 0) lds_read8<0, CH * 256>(kf, kt[0], kt[1], kt[2], kt[3]);
                        else lds_read8<256, CH * 256 + 256>(kf, kt[0], kt[1], kt[2], kt[3]);
#pragma unroll
                        for (int s = 0; s < S; s++)
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const f16x8 x = __builtin_bit_cast(f16x8, kf[u * S + s]);
                                acc[q][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql[q * S + s], acc[q][u], 0, 0, 0);
                            }
#pragma unroll
                        for (int s = 0; s < S; s++)
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const f16x8 x = __builtin_bit_cast(f16x8, kf[u * S + s]);
                                acc[q][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh[q * S + s], acc[q][u], 0, 0, 0);
                            }
                    }
                    float p[8], mx = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 8; k++) p[k] = D == 256 ? acc[0][k / 4][k & 3] + acc[D == 256][k / 4][k & 3] : acc[0][k / 4][k & 3];
                    if ((i + 1) * 32 > least) {
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            if (i * 32 + 16 * (k / 4) + 4 * g + (k & 3) >= nc) p[k] = -INFINITY;
                    }
#pragma unroll
                    for (int k = 0; k < 8; k++) mx = fmaxf(mx, p[k]);
                    mx *= fac;
                    float f;
                    if (base_moves<true>(mx, m, l, f))
#pragma unroll
                        for (int k = 0; k < NO; k++) o[k] *= f;
                    /* a column that has met no position yet keeps its terms 0 */
                    const float base = m == -INFINITY ? 0.0f : Soft<true>::UP - m;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        p[k] = __builtin_amdgcn_exp2f(fmaf(p[k], fac, base));
                        l += p[k];
                    }
                    f16x2 hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        hi[k] = to_half(p[2 * k], p[2 * k + 1]);
                        lo[k] = rest_half(hi[k], 1.0f, p[2 * k], p[2 * k + 1]);
                    }
                    const f16x8 ph = join8(hi), pl = join8(lo);
                    const int left = n - i * 32;
#pragma unroll
                    for (int q = 0; q < (NO + 7) / 8; q++) {
                        constexpr int NV = NO < 8 ? NO : 8;
                        gu32x2 v[NV][2];
                        if constexpr (NO < 8) lds_cols4<0, CH * 256>(v, vt);
                        else if (q == 0) lds_cols8<0, CH * 256>(v, vt);
                        else lds_cols8<256, CH * 256 + 256>(v, vt);
                        if (left < 32) {                 /* behind the run: may be anything */
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const int in = left - 16 * u - 4 * g;
                                const unsigned m0 = in >= 2 ? ~0u : in == 1 ? 0xffffu : 0u, m1 = in >= 4 ? ~0u : in == 3 ? 0xffffu : 0u;
#pragma unroll
                                for (int z = 0; z < NV; z++) { v[z][u].x &= m0; v[z][u].y &= m1; }
                            }
                        }
                        if ((i + 1) * 32 > least) {    /* tokens that some of the wave's rows use and others must not */
                            unsigned odd = 0;
#pragma unroll
                            for (int z = 0; z < NV; z++)
                                odd |= odd_half(v[z][0].x) | odd_half(v[z][0].y) | odd_half(v[z][1].x) | odd_half(v[z][1].y);
                            if (__any(odd != 0)) {     /* 0 * NaN is NaN: row by row, each with its own tokens' values alone */
#pragma unroll 1
                                for (int r = 0; r < A.rpg; r++) {
                                    const int in = __builtin_amdgcn_readlane(nc, r * A.hpb) - i * 32 - 4 * g;
#pragma unroll
                                    for (int z = 0; z < NV; z++) {
                                        gu32x4 x;
#pragma unroll
                                        for (int u = 0; u < 2; u++) {
                                            const int k = in - 16 * u;
                                            x[2 * u] = v[z][u].x & (k >= 2 ? ~0u : k == 1 ? 0xffffu : 0u);
                                            x[2 * u + 1] = v[z][u].y & (k >= 4 ? ~0u : k == 3 ? 0xffffu : 0u);
                                        }
                                        f32x4 y = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), ph, (f32x4){}, 0, 0, 0);
                                        y = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), pl, y, 0, 0, 0);
                                        if (cr == r) o[8 * q + z] += y;
                                    }
                                }
                                continue;
                            }
                        }
#pragma unroll
                        for (int z = 0; z < NV; z += 4) {
                            f32x4 *to = o + 8 * q + z;
                            f16x8 vf[4];
#pragma unroll
                            for (int y = 0; y < 4; y++)
                                vf[y] = __builtin_bit_cast(f16x8, (gu32x4){ v[z + y][0].x, v[z + y][0].y, v[z + y][1].x, v[z + y][1].y });
#pragma unroll
                            for (int y = 0; y < 4; y++) to[y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[y], ph, to[y], 0, 0, 0);
#pragma unroll
                            for (int y = 0; y < 4; y++) to[y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[y], pl, to[y], 0, 0, 0);
                        }
                    }
                }
                }
                pages(min(i0 + 4, last - 1), pg[0]);
                pages(min(i0 + 5, last - 1), pg[1]);
            }
        }
        const size_t slot = 2 * blockIdx.x + (first == 0);
        float sum = sum_g(l);
        if constexpr (HALVES == 2) {                   /* the second half's sums to the first's waves */
            f32x4 *t = (f32x4 *)s_t + grp * (NO + 1) * 64 + lane;
            __syncthreads();                           /* the tiles in LDS are done with */
            if (half) {
#pragma unroll
                for (int k = 0; k < NO; k++) t[k * 64] = o[k];
                t[NO * 64] = (f32x4){ m, sum, 0, 0 };
            }
            __syncthreads();
            if (!half) {
                const f32x4 ml = t[NO * 64];
                const float mn = fmaxf(m, ml[0]), f0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn),
                            f1 = ml[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[0] - mn);
                sum = sum * f0 + ml[1] * f1;
                m = mn;
#pragma unroll
                for (int k = 0; k < NO; k++) o[k] = o[k] * f0 + t[k * 64] * f1;
            }
        }
        if (__builtin_expect(bad, 0)) {
            /* NaN for rows of more tokens than there are before the first bad page, or if the row itself is bad */
            if (tid == 0) atomicOr(err, ATTN_ERR_INDEX);
            int good = n < 0 ? -2 : first * 32;
            while (good >= 0 && good < n && A.s.page_ok(a.table[T.entry(req, good, shift)])) good += 16;
            if (nc > good) sum = NAN;
            else if (nc <= 32 * first)                 /* met nothing but, maybe, a bad page's substitute */
                for (int k = 0; k < NO; k++) o[k] = (f32x4){};
        }
        if (half) {
        } else if (whole) {
            if (on)
#pragma unroll
                for (int k = 0; k < NO; k++) att_store(a, D, t0 + ri, h0 + ch, 16 * k + 4 * g, o[k], sum, nc == 0);
        } else {                                       /* as the registers lie: the join needs no other order */
            const size_t at = slot * GROUPS + grp;
            if (g == 0) {
                A.pm[at * 16 + c] = m;
                A.pl[at * 16 + c] = sum;
            }
#pragma unroll
            for (int k = 0; k < NO; k++) ((f32x4 *)A.po)[slot * ROWS_PART(D, 16 * GROUPS) + (grp * NO + k) * 64 + lane] = o[k];
        }
        at += x1 - x0;
        if (tid == 0 && at == end) {
            const RowsCut x = { t0, nr, hb, !cuts ? 0 : np ? np : (int)((at - x1 + ROWS_LEAD + tiles - 1) / share) - (int)blockIdx.x + 1 };
            A.cut[blockIdx.x] = x;
        }
        if (at >= end) break;
        __syncthreads();                               /* the tiles in LDS are done with */
        x0 = 0;
        if (++hb == per_row) {
            hb = 0;
            for (bool on = true; on;) {                /* the next row that ends a run, 64 rows at a time */
                const int t = t1 + 1 + lane, k = t < rows ? rows_tiles<32>(a, T, shift, R, t) : 0;
                const unsigned long long j = __ballot(k > 0);
                on = j == 0;
                const int i = on ? 0 : __builtin_ctzll(j);
                t1 += on ? 64 : 1 + i;
                tiles = __builtin_amdgcn_readlane(k, i);
            }
            req = uni(a.row_req[t1]);
            n = uni(T.tokens(req, a.row_pos[t1], shift));
        }
    }
}

/* The parts of a cut run, four sums of one wave's lanes to a workgroup of one wave: a
 * thread joins what one lane held, its column's elements 16 j + 4 g .. for four j.  The waves
 * come first in the grid: with equal parts every eighth share, say, begins a unit, and
 * the workgroups of those would all be on one XCD (the join of 256 rows' parts 38 us
 * instead of 14). */
template <int D, int HALVES>
__global__ __launch_bounds__(64) void attn_rows_join_kernel(RowsArgs A)
{
    constexpr int NO = D / 16, GROUPS = ROWS_W / HALVES;
    const RowsCut x = A.cut[blockIdx.y];
    const int w = blockIdx.x / (NO / 4), q = blockIdx.x % (NO / 4), lane = threadIdx.x, c = lane & 15, g = lane >> 4, g0 = blockIdx.y;
    const int cr = c / A.hpb, ch = c - cr * A.hpb, ri = w * A.rpg + cr;
    const int kh = x.hb / A.blocks, bk = x.hb - kh * A.blocks;
    if (x.k == 0 || cr >= A.rpg || ri >= x.n || ch >= A.group - bk * A.hpb) return;
    float m = -INFINITY, l = 0;
    f32x4 y[4] = {};
    auto join = [&](auto N) {                          /* N parts at a time */
        for (int k0 = 0; k0 < x.k; k0 += N()) {
            float pm[N()], pl[N()];
            f32x4 po[N()][4];
#pragma unroll
            for (int j = 0; j < N(); j++) {
                const int k = min(k0 + j, x.k - 1);
                const size_t sl = k ? 2 * (g0 + k) : 2 * g0 + 1, at = sl * GROUPS + w;
                pm[j] = k0 + j < x.k ? A.pm[at * 16 + c] : -INFINITY;
                pl[j] = A.pl[at * 16 + c];
#pragma unroll
                for (int z = 0; z < 4; z++) po[j][z] = ((const f32x4 *)A.po)[sl * ROWS_PART(D, 16 * GROUPS) + (w * NO + 4 * q + z) * 64 + lane];
            }
            float mn = m;
#pragma unroll
            for (int j = 0; j < N(); j++) mn = fmaxf(mn, pm[j]);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= f;
#pragma unroll
            for (int z = 0; z < 4; z++) y[z] *= f;
#pragma unroll
            for (int j = 0; j < N(); j++) {
                if (k0 + j >= x.k) continue;
                const float p = pm[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[j] - mn);
                l += pl[j] * p;
#pragma unroll
                for (int z = 0; z < 4; z++) y[z] += po[j][z] * p;
            }
            m = mn;
        }
    };
    if (x.k == 2) join(std::integral_constant<int, 2>());
    else if (x.k <= 4) join(std::integral_constant<int, 4>());
    else join(std::integral_constant<int, 8>());
    const int t = x.row + ri;
    const bool none = A.a.row_pos[t] == -1;
#pragma unroll
    for (int z = 0; z < 4; z++) att_store(A.a, D, t, kh * A.group + bk * A.hpb + ch, 16 * (4 * q + z) + 4 * g, y[z], l, none);
}

/* The parts of one cut unit's column, L lanes with four elements each to a part:
 * each group of lanes joins its parts as a running softmax does, the groups
 * join in LDS. */
template <int D, int COLS, int L, int JT>
__global__ __launch_bounds__(JT) void attn_join_kernel(AttArgs A)
{
    constexpr int N = JT / L;
    __shared__ float s_m[N], s_l[N];
    __shared__ f32x4 s_o[N][L];
    const RoasterAttnPaged &a = A.a;
    const int tid = threadIdx.x, col = blockIdx.y, row = col / A.hpb, head = col - row * A.hpb;
    const AttCut e = A.cut[blockIdx.x];
    const int n = e.k, g0 = e.g0;
    if (n == 0) return;
    const int kh = e.hb / A.blocks, bk = e.hb - kh * A.blocks;
    if (row >= e.n || head >= A.group - bk * A.hpb) return;
    const int sub = tid / L, d = blockIdx.z * 4 * L + tid % L * 4;
    float m = -INFINITY, l = 0;
    f32x4 y = {};
    for (int k0 = sub; k0 < n; k0 += 4 * N) {
        float pm[4], pl[4];
        f32x4 po[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int k = k0 + j * N, q = k < n ? k : k0;
            const size_t at = (size_t)(A.few ? g0 + q : q ? 2 * (g0 + q) : 2 * g0 + 1) * COLS + col;
            pm[j] = k < n ? A.pm[at] : -INFINITY;
            pl[j] = A.pl[at];
            po[j] = *(const f32x4 *)(A.po + at * D + d);
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < 4; j++) mn = fmaxf(mn, pm[j]);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        y *= f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (k0 + j * N >= n) continue;
            const float w = pm[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[j] - mn);
            l += pl[j] * w;
            y += po[j] * w;
        }
        m = mn;
    }
    if (tid % L == 0) { s_m[sub] = m; s_l[sub] = l; }
    s_o[sub][tid % L] = y;
    __syncthreads();
    if (tid >= L) return;
    float mx = -INFINITY, sum = 0;
    y = (f32x4){};
    for (int i = 0; i < N; i++) mx = fmaxf(mx, s_m[i]);
#pragma unroll 8
    for (int i = 0; i < N; i++) {
        const float w = s_m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[i] - mx);
        sum += s_l[i] * w;
        y += s_o[i][tid] * w;
    }
    const int t = e.row + row;
    att_store(a, D, t, kh * A.group + bk * A.hpb + head, d, y, sum, a.row_pos[t] == -1);
}

/* Workspace: the cut table, then m and l of the parts, then the parts (16 columns). */
static const size_t ATT_CUT = (size_t)ATT_G * sizeof(AttCut), ATT_ML = (size_t)2 * ATT_G * 16 * 4;

/* The same of attn_rows_kernel. */
static const size_t ROWS_CUT = (size_t)ROWS_G * sizeof(RowsCut), ROWS_ML = (size_t)2 * ROWS_G * ROWS_COLS * 4;

/* Calls that may go by runs of rows.  With fewer rows there is little to share, with short contexts too: of
 * one request behind 2048 tokens 8 rows take 24 us so and 18 apart, 16 take 25 and 20, 32 take 27
 * and 25, but behind 16000 tokens 16 take 39 and 69.  The host sees no lengths, so this is a
 * compromise: it loses a quarter on 16 rows behind a short context, and would lose more behind a long one. */
static bool rows_may(int rows, int type) { return type == ROASTER_KV_F16 && rows >= 16; }

extern "C" size_t roaster_attn_ws_bytes(int rows, int q_heads, const RoasterKvCache *c)
{
    if (!attn_cache_ok(c) || rows < 0 || rows > (1 << 20) || q_heads < 1 || q_heads > 1024 || q_heads % c->kv_heads) return 0;
    const size_t one = ATT_CUT + 2 * ATT_ML + (size_t)2 * ATT_G * 16 * c->head_dim * 4,
                 run = ROWS_CUT + 2 * ROWS_ML + (size_t)2 * ROWS_G * ROWS_PART(c->head_dim, ROWS_COLS) * 16;
    return rows_may(rows, c->type) && run > one ? run : one;
}

template <int D, int HALVES>
static void rows_launch(RowsArgs &A, int *err)
{
    A.R = ROWS_W / HALVES * A.rpg;
    hipLaunchKernelGGL((attn_rows_kernel<D, HALVES>), dim3(ROWS_G), dim3(ROWS_T), 0, rt().stream, A, err);
    hipLaunchKernelGGL((attn_rows_join_kernel<D, HALVES>), dim3(ROWS_W / HALVES * D / 64, ROWS_G), dim3(64), 0, rt().stream, A);
}

template <int D, bool F16, bool WIDE>
static void att_launch(const AttArgs &A, int *err)
{
    constexpr int COLS = AttCfg<D, F16, WIDE>::COLS;
    const int units = A.by_unit ? A.a.rows * A.s.kv * A.blocks : A.grid, cols = A.hpb * A.R;
    if (A.few) hipLaunchKernelGGL((attn_few_kernel<D, F16, WIDE>), dim3(A.grid), dim3(ATT_T), 0, rt().stream, A, err);
    else hipLaunchKernelGGL((attn_kernel<D, F16, WIDE>), dim3(A.grid), dim3(ATT_T), 0, rt().stream, A, err);
    /* few units have many parts each: 64 elements of a column to a workgroup, 32 parts at a time */
    if (A.few) hipLaunchKernelGGL((attn_join_kernel<D, COLS, 16, 512>), dim3(units, cols, D / 64), dim3(512), 0, rt().stream, A);
    else hipLaunchKernelGGL((attn_join_kernel<D, COLS, D / 4, 128>), dim3(units, cols), dim3(128), 0, rt().stream, A);
}

extern "C" int roaster_attn_paged(const RoasterAttnPaged *p, const RoasterKvCache *c)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!attn_cache_ok(c)) return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: bad cache description");
    if (!p || p->rows < 0 || p->rows > (1 << 20) || p->q_heads < 1 || p->q_heads > 1024 || p->q_heads % c->kv_heads ||
        p->n_req < 1 || p->max_pages < 1 || (int64_t)p->max_pages * c->page_size > (1 << 30) || !(fabsf(p->scale) <= 2e38f))
        return rt_fail(ROASTER_EINVAL, "roaster_attn_paged: need 0 <= rows <= 2^20, q_heads a multiple of kv_heads up to 1024, "
                       "n_req >= 1, max_pages * page_size at most 2^30, a scale within 2e38");
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
    /* Runs of rows pay where requests have more rows each than sixteen columns hold, which
     * the two counts tell on average (the host sees neither lengths nor which request a row is of; a
     * call of other rows is right as well, only slower): 256 rows behind 2048 tokens take 45 us so, 107
     * otherwise, a prompt of 2000 120 and 444; 16 requests of 300..16000 tokens and 8 heads (two
     * rows fill the columns) with three rows 57 and 75, with 16 heads two rows 36.5 and 38; with 4
     * heads (four rows do) and 75..4000 tokens six rows 39 and 39, four 32 and 28.  Two rows of 8
     * heads are on the slower side, 45 and 53 (32 requests: 70 and 75).  One request's 256 rows with 63
     * requests' single rows in one call take 159, in two calls 136. */
    const int per16 = 16 / std::min(p->q_heads / c->kv_heads, 16);
    if (rows_may(p->rows, c->type) && p->rows >= std::max(2, per16 + 1) * (long long)p->n_req) {
        RowsArgs A;
        A.a = *p;
        A.kc = (const char *)c->k;
        A.vc = (const char *)c->v;
        A.s = attn_shape(c);
        A.group = p->q_heads / c->kv_heads;
        A.hpb = A.group < 16 ? A.group : 16;
        A.blocks = (A.group + A.hpb - 1) / A.hpb;
        A.rpg = per16;
        A.cut = (RowsCut *)p->ws;
        A.pm = (float *)((char *)p->ws + ROWS_CUT);
        A.pl = (float *)((char *)p->ws + ROWS_CUT + ROWS_ML);
        A.po = (float *)((char *)p->ws + ROWS_CUT + 2 * ROWS_ML);
        /* Few units are cut into many parts: 16 rows behind 2048 tokens take 25 us in halves and 26
         * without, 8 requests of six rows 40 and 45, 256 rows 45 and 46, but 512 rows 70 and 66. */
        const bool halves = (long long)p->rows * A.hpb * A.blocks * c->kv_heads <= ROWS_G / 8 * ROWS_COLS;
#define ROWS(DD) (halves ? rows_launch<DD, 2>(A, err) : rows_launch<DD, 1>(A, err))
        if (D == 256) ROWS(256);
        else if (D == 128) ROWS(128);
        else ROWS(64);
#undef ROWS
        return rt_check(hipGetLastError(), "attention launch") ? ROASTER_EDEVICE : 0;
    }
    AttArgs A;
    A.a = *p;
    A.kc = (const char *)c->k;
    A.vc = (const char *)c->v;
    A.s = attn_shape(c);
    A.group = p->q_heads / c->kv_heads;
    /* Sixteen columns of their own for more than eight heads (32 requests of
     * 300..16000 tokens, 16 heads on one: 38 us, with two blocks of eight 53) and for several rows of a
     * request (32 requests of two rows: 76 us, row by row 93; f32, 256 rows: 153 instead of 270).  With one
     * row of few heads the high and low parts fill them: half the MFMAs. */
    const bool f16 = c->type == ROASTER_KV_F16;
    bool wide = !f16 || A.group > 8;
    A.hpb = std::min(A.group, wide ? 16 : 8);
    A.blocks = (A.group + A.hpb - 1) / A.hpb;
    /* two workgroups a CU, but for the f32 cache's registers at dim 256 */
    A.grid = D == 256 && !f16 ? ATT_G / 2 : ATT_G;
    const long long units = (long long)p->rows * c->kv_heads * A.blocks;
    A.by_unit = units <= A.grid;
    /* With few units the rows of a request stay apart: what they share comes from the caches,
     * and there are more parts (three rows behind 437 tokens: 12.7 us, together in even shares 18.5). */
    A.few = units <= A.grid / 8 && p->rows <= 128;
    A.R = A.few || p->rows < 2 * (long long)p->n_req ? 1 : 16 / A.hpb;
    wide |= A.R > 1;
    A.cut = (AttCut *)p->ws;
    A.pm = (float *)((char *)p->ws + ATT_CUT);
    A.pl = (float *)((char *)p->ws + ATT_CUT + ATT_ML);
    A.po = (float *)((char *)p->ws + ATT_CUT + 2 * ATT_ML);
#define ATT(DD) (f16 ? wide ? att_launch<DD, true, true>(A, err) : att_launch<DD, true, false>(A, err) : att_launch<DD, false, true>(A, err))
    if (D == 256) ATT(256);
    else if (D == 128) ATT(128);
    else ATT(64);
#undef ATT
    return rt_check(hipGetLastError(), "attention launch") ? ROASTER_EDEVICE : 0;
}
