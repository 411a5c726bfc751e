/* SPDX-License-Identifier: Unlicense */

/* Four consecutive floats by one 16-byte access at any float's address (the
 * memory unit splits what crosses a line), so that rows of odd length take
 * the same path as aligned ones. */

#ifndef ICOREG_LOAD4_H
#define ICOREG_LOAD4_H

#include <hip/hip_runtime.h>

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));

static __device__ __forceinline__ void load4(const float *p, float (&x)[4])
{
    const float4u v = *(const float4u *)p;

    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
}

static __device__ __forceinline__ void store4(float *p, float a, float b, float c, float d)
{
    const float4u v = {a, b, c, d};

    *(float4u *)p = v;
}

/* Floats c .. c + 3 of a row of n, zeros past its end. */
static __device__ __forceinline__ void load4_row(const float *row, int c, int n, float (&x)[4])
{
    if (c + 4 <= n)
        load4(row + c, x);
    else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            x[j] = c + j < n ? row[c + j] : 0.0f;
    }
}

#endif /* ICOREG_LOAD4_H */
