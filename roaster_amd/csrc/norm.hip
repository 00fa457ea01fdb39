/*
 * norm.hip -- root-mean-square norm with the residual's addition, over rows or
 * over heads with a gate, in f32 and in 8 bits (roaster_norm; kernels.c:584-605,
 * model.c:1349-1358 and the mixer's output norm, model.c:1282-1347).
 */
#include "mixer.h"
#include "qdot.h"

#define NORM_T 256

/* A row is a workgroup's, V times four elements a thread, all of it in registers between the sum and the
 * outputs: x, res and gate are read once.  Heads of 16 .. 256 elements lie in 4 .. 64 neighbouring lanes of one wave.
 * What bounds it: a launch up to some hundred rows (one row of 2048 3.7 us a call, 2.5 of them the kernel), then memory: 2048
 * rows of 32 heads of 128 with a gate 18.1 us, 5.6 TB/s, where a copy past the caches makes 6.0 .. 6.3.  STREAM: y past the
 * caches (22.7 us without). */
template <int V, bool STREAM>
__global__ __launch_bounds__(NORM_T) void norm_kernel(RoasterNorm a)
{
    constexpr int L = NORM_T;
    __shared__ float s_sum[NORM_T / 64];
    __shared__ unsigned s_top[NORM_T / 64];
    const int tid = threadIdx.x, row = blockIdx.x;
    const float *x = a.x + row * a.x_row;
    float4 v[V], g[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = 4 * (tid + i * L);
        v[i] = e < a.cols ? gld_f4(x + e) : make_float4(0, 0, 0, 0);
    }
    if (a.gate) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = 4 * (tid + i * L);
            g[i] = e < a.cols ? gld_f4(a.gate + row * a.gate_row + e) : make_float4(0, 0, 0, 0);
        }
    }
    if (a.res) {
        float *r = a.res + row * a.res_row;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = 4 * (tid + i * L);
            if (e < a.cols) {
                const float4 o = gld_f4(r + e);
                v[i].x += o.x; v[i].y += o.y; v[i].z += o.z; v[i].w += o.w;
                *(float4 *)(r + e) = v[i];
            }
        }
    }
    float inv[V];
    if (a.group == a.cols) {
        float ss = 0;
#pragma unroll
        for (int i = 0; i < V; i++) ss += v[i].x * v[i].x + v[i].y * v[i].y + v[i].z * v[i].z + v[i].w * v[i].w;
        for (int o = 1; o < 64; o <<= 1) ss += __shfl_xor(ss, o);
        if (tid % 64 == 0) s_sum[tid / 64] = ss;
        __syncthreads();
        ss = 0;
        for (int w = 0; w < L / 64; w++) ss += s_sum[w];
        const float r = 1.0f / sqrtf(ss / a.cols + a.eps);
#pragma unroll
        for (int i = 0; i < V; i++) inv[i] = r;
    } else if (a.group) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            float ss = v[i].x * v[i].x + v[i].y * v[i].y + v[i].z * v[i].z + v[i].w * v[i].w;
            for (int o = 1; o < a.group / 4; o <<= 1) ss += __shfl_xor(ss, o);
            inv[i] = 1.0f / sqrtf(ss / a.group + a.eps);
        }
    }
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = 4 * (tid + i * L);
        if (e >= a.cols) continue;
        if (a.group) {
            const float4 w = a.weight ? gld_f4(a.weight + (a.group == a.cols ? e : e & (a.group - 1))) : make_float4(1, 1, 1, 1);
            v[i].x *= inv[i] * w.x; v[i].y *= inv[i] * w.y; v[i].z *= inv[i] * w.z; v[i].w *= inv[i] * w.w;
        }
        if (a.gate) {
            v[i].x *= g[i].x / (1.0f + expf(-g[i].x));
            v[i].y *= g[i].y / (1.0f + expf(-g[i].y));
            v[i].z *= g[i].z / (1.0f + expf(-g[i].z));
            v[i].w *= g[i].w / (1.0f + expf(-g[i].w));
        }
        if (a.y) {
            float *y = a.y + row * a.y_row + e;
            if (STREAM) __builtin_nontemporal_store((gf32x4){ v[i].x, v[i].y, v[i].z, v[i].w }, (GAS gf32x4 *)y);
            else *(float4 *)y = v[i];
        }
        const float m[4] = { v[i].x, v[i].y, v[i].z, v[i].w };
        for (int j = 0; j < 4; j++) top = max(top, __float_as_uint(m[j]) & 0x7FFFFFFFu);
    }
    if (!a.q) return;
    for (int o = 1; o < 64; o <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    if (tid % 64 == 0) s_top[tid / 64] = top;
    __syncthreads();
    for (int w = 0; w < L / 64; w++) top = max(top, s_top[w]);
    const I8Scale s = i8_scale(top);
    if (tid == 0) a.q_scale[row] = s.scale;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = 4 * (tid + i * L);
        if (e >= a.cols) continue;
        const int p = (i8_round(v[i].x, s.mul) & 255) | (i8_round(v[i].y, s.mul) & 255) << 8 |
                      (i8_round(v[i].z, s.mul) & 255) << 16 | i8_round(v[i].w, s.mul) << 24;
        *(int *)(a.q + row * a.q_row + e) = p;
    }
}

extern "C" int roaster_norm(const RoasterNorm *p)
{
    std::lock_guard<std::recursive_mutex> g(rt_lock());
    if (!p || p->rows < 0 || p->rows > (1 << 20) || p->cols < 4 || p->cols > 16384 || p->cols % 4)
        return rt_fail(ROASTER_EINVAL, "roaster_norm: need 0 <= rows <= 2^20, cols a multiple of 4 up to 16384");
    const int gr = p->group;
    if (gr && gr != p->cols && (gr < 16 || gr > 256 || (gr & (gr - 1)) || p->cols % gr))
        return rt_fail(ROASTER_EINVAL, "roaster_norm: group is cols, a power of two from 16 to 256 that divides cols, or 0");
    if (!p->rows) return 0;
    const size_t rows = p->rows, cols = p->cols;
    if (!p->x || (!p->y && !p->q) || (p->q && !p->q_scale))
        return rt_fail(ROASTER_EINVAL, "roaster_norm: x and an output must be given, q_scale with q");
    if (!attn_aligned(p->x, 16) || !attn_aligned(p->res, 16) || !attn_aligned(p->weight, 16) || !attn_aligned(p->gate, 16) ||
        !attn_aligned(p->y, 16) || !attn_aligned(p->q, 4) || !attn_aligned(p->q_scale, 4))
        return rt_fail(ROASTER_EINVAL, "roaster_norm: f32 tensors are 16-byte aligned, q and q_scale 4-byte");
    if (!stride_ok(p->x_row, 4) || (p->gate && !stride_ok(p->gate_row, 4)) ||
        (p->res && (!stride_ok(p->res_row, 4) || p->res_row < cols)) || (p->y && (!stride_ok(p->y_row, 4) || p->y_row < cols)) ||
        (p->q && (!stride_ok(p->q_row, 4) || p->q_row < cols)))
        return rt_fail(ROASTER_EINVAL, "roaster_norm: strides are multiples of 4 up to 2^32, those of res, y and q at least cols");
    /* absent tensors are NULL and overlap nothing */
    const void *out[] = { p->res, p->y, p->q, p->q ? p->q_scale : NULL };
    const size_t no[] = { rows_span(rows, cols, p->res_row, 4), rows_span(rows, cols, p->y_row, 4),
                          rows_span(rows, cols, p->q_row, 1), 4 * rows };
    const void *in[] = { p->x, p->gate, gr ? p->weight : NULL };
    const size_t ni[] = { rows_span(rows, cols, p->x_row, 4), rows_span(rows, cols, p->gate_row, 4), 4 * (size_t)gr };
    for (int i = 0; i < 4; i++) {
        for (int j = 0; j < 3; j++)
            if (attn_overlap(out[i], no[i], in[j], ni[j]) && !(i == 1 && j == 0 && p->y == p->x && p->y_row == p->x_row))
                return rt_fail(ROASTER_EINVAL, "roaster_norm: outputs overlap inputs");
        for (int j = 0; j < i; j++)
            if (attn_overlap(out[i], no[i], out[j], no[j])) return rt_fail(ROASTER_EINVAL, "roaster_norm: outputs overlap");
    }
    if (rt_init_locked()) return ROASTER_EDEVICE;
    const AttnDevice dev;
    const int v = (int)(cols / 4 + NORM_T - 1) / NORM_T;
    /* An output that the L2s (32 MB) would not hold anyway goes past them; the residual, which the next norm reads, never
     * does (2048 rows of 2048 into 8 bits 24.5 us with torch's conversion behind it, past the caches 24.8). */
    const bool stream = p->y && 4 * rows * cols >= ((size_t)24 << 20);
#define NORM2(V, S) hipLaunchKernelGGL((norm_kernel<V, S>), dim3(rows), dim3(NORM_T), 0, rt().stream, *p)
#define NORM(V) do { if (stream) NORM2(V, true); else NORM2(V, false); } while (0)
    if (v <= 1) NORM(1);
    else if (v <= 2) NORM(2);
    else if (v <= 4) NORM(4);
    else if (v <= 8) NORM(8);
    else NORM(16);
#undef NORM
#undef NORM2
    return rt_check(hipGetLastError(), "norm launch") ? ROASTER_EDEVICE : 0;
}
