/*
 * mixer.h -- what the operators of a recurrent layer (norm.hip, i8.hip, ssm.hip)
 * share: checks of their arguments and the scale of a row in 8 bits.
 */
#ifndef ROASTER_MIXER_INTERNAL_H
#define ROASTER_MIXER_INTERNAL_H

#include "attn.h"
#include "../../include/roaster_mixer.h"

/* Bytes from the first element to the last of `rows` rows of `cols` elements at `stride`. */
static inline size_t rows_span(size_t rows, size_t cols, size_t stride, size_t size)
{
    return ((rows - 1) * stride + cols) * size;
}

static inline bool stride_ok(size_t stride, size_t multiple) { return stride % multiple == 0 && stride <= ((size_t)1 << 32); }

#ifdef __HIPCC__
/* What takes a row whose largest size has the bits `top` (those of a NaN are above all others)
 * to 8 bits, and back: x = y * mul, y ~ x * scale.  127 / top is finite from 2^-119 on. */
struct I8Scale { float mul, scale; };
__device__ __forceinline__ I8Scale i8_scale(unsigned top)
{
    const float s = __uint_as_float(top);
    if (top >= 0x7F800000u) return { 0.0f, __uint_as_float(0x7FC00000u) };
    if (s < 0x1p-119f) return { 0.0f, 0.0f };
    return { 127.0f / s, s / 127.0f };
}
/* Rounded to nearest even, within -127 .. 127 since |y * 127 / max| is at most 127 (1 + 2^-23). */
__device__ __forceinline__ int i8_round(float y, float mul) { return mul == 0.0f ? 0 : (int)rintf(y * mul); }
#endif

#endif
