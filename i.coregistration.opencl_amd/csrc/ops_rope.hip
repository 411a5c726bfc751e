/* SPDX-License-Identifier: Unlicense */

/* Rotary positions computed from the tokens' coordinates: pair p of a head's
 * first rot channels turns by the angle pos[row][p % axes] freq[p],
 *
 *   y0 = m (x0 cos a - x1 sin a),  y1 = m (x0 sin a + x1 cos a),
 *
 * the channels behind them are copied. A block computes the cosines and sines
 * of its rows once, into LDS, and every head of both tensors takes them from
 * there. */

#include <hip/hip_runtime.h>

#include <math.h>

#include "act.h"
#include "common.h"
#include "ops.h"

using namespace icoreg;

#define ROPE_PAIRS 1024 /* LDS table entries of a block */

struct rope_side {
    const float *x;
    float *y;
    long long ldx, ldy;
    int nh;
};

struct rope_args {
    rope_side s[2];
    const int *pos;
    const double *freq;
    long long rows;
    int d, rot, axes, block_rows, units; /* units of a head, see below */
    float mult, sign;
};

/* cos and sin of pos freq, times m. The angle is formed in 64 bits and
 * reduced there to an eighth of a turn either way, so that far positions keep
 * their bits (2^31 radians: 2^-22 of the last one's 64-bit place); within
 * that the Taylor sums of degree 9 and 10 are good to 2^-29. */
__device__ __forceinline__ float2 rope_turn(double angle, float m, float sign)
{
    const double q = rint(angle * 0.63661977236758134308); /* quarter turns */
    const double e = fma(-q, 1.57079632679489655800, angle);
    const float y = (float)fma(-q, 6.12323399573676603587e-17, e), z = y * y;
    const int k = (int)(long long)q & 3;
    float s = fmaf(z, 2.75573192e-6f, -1.98412698e-4f), c = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);

    s = fmaf(z, s, 8.33333333e-3f);
    s = fmaf(z, s, -1.66666667e-1f);
    s = fmaf(y * z, s, y);
    c = fmaf(z, c, -1.38888889e-3f);
    c = fmaf(z, c, 4.16666667e-2f);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.0f);
    const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;

    return make_float2((k == 1 || k == 2 ? -cc : cc) * m, (k >= 2 ? -ss : ss) * m * sign);
}

template <int V> struct rope_vec {
    float v[V];
};

template <int V> __device__ __forceinline__ rope_vec<V> rope_load(const float *p)
{
    rope_vec<V> r;

    if constexpr (V == 4) {
        const float4 a = *(const float4 *)p;

        r.v[0] = a.x, r.v[1] = a.y, r.v[2] = a.z, r.v[3] = a.w;
    }
    else if constexpr (V == 2) {
        const float2 a = *(const float2 *)p;

        r.v[0] = a.x, r.v[1] = a.y;
    }
    else
        r.v[0] = *p;
    return r;
}

template <int V> __device__ __forceinline__ void rope_store(float *p, const rope_vec<V> &r)
{
    if constexpr (V == 4)
        *(float4 *)p = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    else if constexpr (V == 2)
        *(float2 *)p = make_float2(r.v[0], r.v[1]);
    else
        *p = r.v[0];
}

/* A unit is 2 V channels of a head: V pairs among the first rot channels (2 V
 * neighbours interleaved, V of either half otherwise), or 2 V channels to
 * copy. With V = 1 the last unit of an odd head is one channel. Bound by
 * memory: 65533 rows of 20 heads of 128, 64 of them turned, 671 MB in and out
 * each, 268 us, 5.0 TB/s (a large copy 4.8); 6400 rows of 16 heads of 32, 26 MB,
 * 7.4 us. A table read instead of the cosines would add its bytes and hold
 * only the positions that it was made for. */
template <int V, bool INTER>
__global__ void __launch_bounds__(256) rope_pos_kernel(const rope_args a)
{
    __shared__ float2 table[ROPE_PAIRS];
    const int tid = threadIdx.x, np = a.rot / 2, per_row = (a.s[0].nh + a.s[1].nh) * a.units;
    const long long r0 = (long long)blockIdx.x * a.block_rows;
    const int n = (int)min((long long)a.block_rows, a.rows - r0);

    for (int e = tid; e < n * np; e += 256) {
        const int r = e / np, p = e - r * np;

        table[e] = rope_turn(a.pos[(r0 + r) * a.axes + p % a.axes] * a.freq[p], a.mult, a.sign);
    }
    __syncthreads();
    for (int e = tid; e < n * per_row; e += 256) {
        const int r = e / per_row, rem = e - r * per_row, hh = rem / a.units;
        const int u = rem - hh * a.units, c = 2 * V * u;
        const bool second = hh >= a.s[0].nh;
        const rope_side &s = a.s[second];
        const int h = second ? hh - a.s[0].nh : hh;
        const float *x = s.x + (r0 + r) * s.ldx + (long long)h * a.d;
        float *y = s.y + (r0 + r) * s.ldy + (long long)h * a.d;

        if (c < a.rot) {
            const float2 *t = table + r * np + u * V;
            const int i0 = INTER ? c : u * V, i1 = INTER ? c + V : u * V + np;
            const rope_vec<V> p = rope_load<V>(x + i0), q = rope_load<V>(x + i1);
            rope_vec<V> v, w;

#pragma unroll
            for (int j = 0; j < V; j++) {
                if constexpr (INTER) {
                    /* The 2 V values in order: pair j is 2 j, 2 j + 1. */
                    const float x0 = 2 * j < V ? p.v[2 * j] : q.v[2 * j - V];
                    const float x1 = 2 * j + 1 < V ? p.v[2 * j + 1] : q.v[2 * j + 1 - V];
                    float &y0 = 2 * j < V ? v.v[2 * j] : w.v[2 * j - V];
                    float &y1 = 2 * j + 1 < V ? v.v[2 * j + 1] : w.v[2 * j + 1 - V];

                    icoreg_rope_pair(x0, x1, t[j], y0, y1);
                }
                else
                    icoreg_rope_pair(p.v[j], q.v[j], t[j], v.v[j], w.v[j]);
            }
            rope_store<V>(y + i0, v);
            rope_store<V>(y + i1, w);
        }
        else if (V > 1 || c + 1 < a.d) {
            const rope_vec<V> p = rope_load<V>(x + c), q = rope_load<V>(x + c + V);

            rope_store<V>(y + c, p);
            rope_store<V>(y + c + V, q);
        }
        else
            y[c] = x[c];
    }
}

static rope_side rope_make(const char *op, long rows, int d, int nh, struct opnd X, struct opnd Y,
                           const char *names)
{
    rope_side s = {};
    const long long w = (long long)nh * d;

    if (nh == 0)
        return s;
    if (nh < 0 || w > 0x7fffffffLL || X.ld < w || Y.ld < w || X.off < 0 || Y.off < 0)
        icoreg_fatal("%s: invalid sizes of %s: nh=%d d=%d ld=%d, %d", op, names, nh, d, X.ld, Y.ld);
    need_floats(X.buf, X.off, (rows - 1) * (long long)X.ld + w, op, names);
    need_floats(Y.buf, Y.off, (rows - 1) * (long long)Y.ld + w, op, names);
    s.x = cfptr(X.buf) + X.off;
    s.y = fptr(Y.buf) + Y.off;
    /* One row's stride means nothing. */
    s.ldx = rows > 1 ? X.ld : w;
    s.ldy = rows > 1 ? Y.ld : w;
    s.nh = nh;
    return s;
}

static bool rope_vec_ok(const rope_side &s, int v)
{
    const uintptr_t m = 4 * v - 1;

    return s.nh == 0 || (!((uintptr_t)s.x & m) && !((uintptr_t)s.y & m) && s.ldx % v == 0 &&
                         s.ldy % v == 0);
}

extern "C" void ops_rope_pos(struct ops *o, long rows, int d, int rot, int axes, cl_mem pos,
                             cl_mem freq, float mult, int flags, struct opnd X1, struct opnd Y1,
                             int nh1, struct opnd X2, struct opnd Y2, int nh2)
{
    ICOREG_API_BEGIN
    const char *op = "ops_rope_pos";
    rope_args a = {};

    if (rows < 0 || d < 1 || rot < 0 || rot % 2 || rot > d || rot > 2 * ROPE_PAIRS || axes < 1 ||
        axes > 4 || nh1 < 0 || nh2 < 0 || flags & ~(ROPE_INTERLEAVED | ROPE_INVERSE))
        icoreg_fatal("%s: invalid sizes rows=%ld d=%d rot=%d axes=%d nh=%d, %d flags=%d", op, rows,
                     d, rot, axes, nh1, nh2, flags);
    if (rows == 0 || (nh1 == 0 && nh2 == 0))
        return;
    if (rot) {
        need_bytes(pos, 0, (long long)rows * axes * 4, op, "pos");
        need_bytes(freq, 0, rot / 2 * 8LL, op, "freq");
        need_aligned(freq, 8, op, "freq");
    }
    a.s[0] = rope_make(op, rows, d, nh1, X1, Y1, "X1 or Y1");
    a.s[1] = rope_make(op, rows, d, nh2, X2, Y2, "X2 or Y2");
    for (const rope_side &p : a.s) {
        const long long span = (rows - 1) * p.ldy + (long long)p.nh * d;

        if (!p.nh || !rot)
            continue;
        need_rows_apart(p.y, span, span, 1, (const float *)pos->ptr, rows * (long long)axes,
                        rows * (long long)axes, 1, op, "an output and pos");
        need_rows_apart(p.y, span, span, 1, (const float *)freq->ptr, rot, rot, 1, op,
                        "an output and freq");
    }
    for (int i = 0; i < 2; i++)
        for (int j = 0; j < 2; j++) {
            const rope_side &p = a.s[i], &q = a.s[j];

            if (!p.nh || !q.nh)
                continue;
            if (i != j || p.x != p.y || p.ldx != p.ldy)
                need_rows_apart(p.y, p.ldy, (long long)p.nh * d, rows, q.x, q.ldx,
                                (long long)q.nh * d, rows, op,
                                "an output and an input (unless the same rows)");
            if (i < j)
                need_rows_apart(p.y, p.ldy, (long long)p.nh * d, rows, q.y, q.ldy,
                                (long long)q.nh * d, rows, op, "Y1 and Y2");
        }
    {
        const bool inter = flags & ROPE_INTERLEAVED;
        const bool in_place = (!nh1 || a.s[0].x == a.s[0].y) && (!nh2 || a.s[1].x == a.s[1].y);
        int v = 4;

        while (v > 1 && (rot % (2 * v) || d % (2 * v) || !rope_vec_ok(a.s[0], v) ||
                         !rope_vec_ok(a.s[1], v)))
            v /= 2;
        /* Rows that stay where they are have nothing to copy. */
        a.units = in_place ? rot / (2 * v) : (d + 2 * v - 1) / (2 * v);
        if (a.units == 0)
            return;
        const long long per_row = ((long long)nh1 + nh2) * a.units;
        long long n = (2048 + per_row - 1) / per_row;

        if (rot)
            n = min(n, 2LL * ROPE_PAIRS / rot);
        n = min(n, (long long)rows);
        count32(n * per_row + 256, "rope units"); /* counted past the end */
        a.pos = pos ? (const int *)pos->ptr : nullptr;
        a.freq = freq ? (const double *)freq->ptr : nullptr;
        a.rows = rows;
        a.d = d;
        a.rot = rot;
        a.axes = axes;
        a.block_rows = (int)n;
        a.mult = mult;
        a.sign = flags & ROPE_INVERSE ? -1.0f : 1.0f;
        const dim3 grid(grid_of((rows + n - 1) / n, 256, "rope blocks")), block(256);
        const hipStream_t s = stream_of(o->ocl);

        prof_scope ps(o->ocl, "rope_pos");
#define ROPE_LAUNCH(V_)                                                                  \
    if (inter)                                                                           \
        hipLaunchKernelGGL((rope_pos_kernel<V_, true>), grid, block, 0, s, a);           \
    else                                                                                 \
        hipLaunchKernelGGL((rope_pos_kernel<V_, false>), grid, block, 0, s, a)
        if (v == 4) {
            ROPE_LAUNCH(4);
        }
        else if (v == 2) {
            ROPE_LAUNCH(2);
        }
        else {
            ROPE_LAUNCH(1);
        }
#undef ROPE_LAUNCH
        launch_check("rope_pos");
    }
    ICOREG_API_END
}

extern "C" void ops_rope_freqs(double *freq, int rot, int axes, double base, int kind,
                               double factor, double trained, double slow, double fast)
{
    ICOREG_API_BEGIN
    const char *op = "ops_rope_freqs";

    if (!freq || rot < 2 || axes < 1 || rot % (2 * axes) || kind < ROPE_TRAINED ||
        kind > ROPE_PARTS || !(base > 0.0) || !(factor > 0.0))
        icoreg_fatal("%s: invalid arguments rot=%d axes=%d kind=%d base=%g factor=%g", op, rot,
                     axes, kind, base, factor);
    if (kind == ROPE_PARTS && !(trained > 0.0 && fast > slow))
        icoreg_fatal("%s: invalid range: trained=%g slow=%g fast=%g", op, trained, slow, fast);
    {
        const double n = rot / axes;

        if (kind == ROPE_REBASE && n > 2)
            base *= pow(factor, n / (n - 2));
        for (int p = 0; p < rot / 2; p++) {
            const double w = pow(base, -2.0 * (p / axes) / n);
            double g = 1.0;

            if (kind == ROPE_LINEAR)
                g = 0.0;
            else if (kind == ROPE_PARTS)
                g = fmin(fmax((trained * w / (2 * M_PI) - slow) / (fast - slow), 0.0), 1.0);
            freq[p] = w * (g + (1.0 - g) / factor);
        }
    }
    ICOREG_API_END
}
