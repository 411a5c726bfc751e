/* SPDX-License-Identifier: Unlicense */

/* Symmetric 8-bit rows: the codes and the scale of a row of float32 values,
 * shared by every kernel that makes them so that they agree to the bit.
 *
 * With a the row's largest magnitude, s = a / 127 and r = 127 / a (float32
 * quotients), the code of x is the float32 product x r rounded to the nearest
 * integer, ties to even: |code| <= 127, x = code s within s / 2. A row with
 * a < 2^-100 counts as zero (s = 0, codes 0): 127 / a stays finite and s
 * normal. A row with a value that is not finite has s = NaN and codes 0, so
 * that whatever is computed from it is NaN. */

#ifndef ICOREG_Q8_H
#define ICOREG_Q8_H

#include <hip/hip_runtime.h>

#include "reduce.h"

#define Q8_PITCH 64 /* rows of codes are padded with zeros to this */
#define Q8_TINY 0x1p-100f

static inline __host__ __device__ long long q8_pitch(int C)
{
    return ((long long)C + Q8_PITCH - 1) / Q8_PITCH * Q8_PITCH;
}

/* The bits of |x|: as whole numbers they order like the magnitudes, with
 * infinity and NaN (which a float maximum would drop) above all others. */
static __device__ __forceinline__ unsigned q8_mag(float x)
{
    return __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
}

struct q8_scale {
    float s, r;
};

static __device__ __forceinline__ q8_scale q8_scale_of(unsigned mag)
{
    const float a = __builtin_bit_cast(float, mag);
    q8_scale q;

    if (mag >= 0x7f800000u) {
        q.s = __builtin_nanf("");
        q.r = 0.0f;
    }
    else if (a < Q8_TINY) {
        q.s = q.r = 0.0f;
    }
    else {
        q.s = a / 127.0f;
        q.r = 127.0f / a;
    }
    return q;
}

/* Code of x in the low byte. Adding 1.5 2^23 rounds to the nearest integer,
 * ties to even, and leaves it in the low bits; the product is rounded
 * first, as the definition says, so the two must not become one fma. r = 0:
 * every code is 0, also of infinities and NaN. */
static __device__ __forceinline__ unsigned q8_code(float x, float r)
{
#pragma clang fp contract(off)
    const float p = x * r;

    return r != 0.0f ? __builtin_bit_cast(unsigned, p + 12582912.0f) & 0xffu : 0u;
}

static __device__ __forceinline__ unsigned q8_code4(float a, float b, float c, float d, float r)
{
    return q8_code(a, r) | q8_code(b, r) << 8 | q8_code(c, r) << 16 | q8_code(d, r) << 24;
}

static __device__ __forceinline__ unsigned wave_umax(unsigned v)
{
    const int ctl[4] = {0xB1, 0x4E, 0x141, 0x140};

#pragma unroll
    for (int k = 0; k < 4; k++)
        v = max(v, (unsigned)dpp_i((int)v, ctl[k]));
    return max(max((unsigned)__builtin_amdgcn_readlane((int)v, 0),
                   (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
               max((unsigned)__builtin_amdgcn_readlane((int)v, 32),
                   (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}

#endif /* ICOREG_Q8_H */
