/* SPDX-License-Identifier: Unlicense */

/* The norm between two layers of a transformer: the residual's addition, the
 * division by the row's root mean square, and the 8-bit codes of the result,
 *
 *   h = x + r,  i = 1 / sqrt(mean(h^2) + eps),  y = (h i) g,
 *
 * in one pass over the row. The mean is a 64-bit sum and i its root's
 * reciprocal rounded to float32 once: float32 sums would depend on the order,
 * and with them the codes next to a border. */

#include <hip/hip_runtime.h>

#include <math.h>

#include "common.h"
#include "load4.h"
#include "ops.h"
#include "q8.h"

using namespace icoreg;

#define NORM_MAX_C (1 << 30)   /* channels are counted in int, past the last too */
#define NORM_ROWS (1L << 21)   /* rows of a launch: 2^32 threads are too many */

struct norm_args {
    const float *X, *R, *g;
    float *H, *Y, *S;
    unsigned *Q;
    long long ldx, ldr, ldh, ldy;
    long rows;
    int C;
    double eps;
};

__device__ __forceinline__ double dpp_d(double v, int ctrl)
{
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = dpp_i((int)b, ctrl), hi = dpp_i((int)(b >> 32), ctrl);

    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

__device__ __forceinline__ double lane_d(double v, int l)
{
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_readlane((int)b, l);
    const unsigned hi = __builtin_amdgcn_readlane((int)(b >> 32), l);

    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

/* Sum over a wave whose lanes are all active; every lane gets it. */
__device__ __forceinline__ double wave_dsum(double v)
{
    v += dpp_d(v, 0xB1);
    v += dpp_d(v, 0x4E);
    v += dpp_d(v, 0x141);
    v += dpp_d(v, 0x140);
    return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}

__device__ __forceinline__ void store4_row(float *row, int c, int n, const float (&x)[4])
{
    if (c + 4 <= n)
        store4(row + c, x[0], x[1], x[2], x[3]);
    else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (c + j < n)
                row[c + j] = x[j];
    }
}

/* W waves a row, four channels a lane and step. Rows of up to 256 NV W channels
 * stay in registers between the sum, the maximum and the codes; longer ones
 * (NV = 0) are read again: h, where it is kept, from there, as it may lie over
 * x or r. Bound by memory, which each value passes once: 12805 x 4096 with the
 * residual, to h and codes (682 MB), 128 us, 5.3 TB/s (a large copy 4.8); 3202 x
 * 1024 to h and y (52 MB, some of it still in the last cache) 9 us. The 64-bit
 * products and sums run beside the loads. */
template <int NV, int W>
__global__ void __launch_bounds__(W > 4 ? 64 * W : 256) rms_norm_kernel(const norm_args a)
{
#pragma clang fp contract(off)
    constexpr int RB = W > 4 ? 1 : 4 / W; /* rows of a block */
    /* Two kernels share the rows of 257 to 1024 channels, and of up to 4096, by how
     * many there are, and a row is the same from both: each 256 channels, a step
     * of a wave, have sums of their own, added in their order, by lanes and then
     * over the lanes (up to 1024: the other way takes norms of 3202 rows 2 %
     * longer), or over the lanes first. */
    constexpr int NB = NV && NV * W <= 16 ? NV : 1;
    constexpr bool LANES = NV * W == 4;
    __shared__ double sums[W > 1 ? NB * W : 1][LANES && W > 1 ? 64 : 1];
    __shared__ unsigned tops[W > 1 ? W : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = wave % W, C = a.C;
    const long row = (long)blockIdx.x * RB + wave / W;
    const int steps = NV ? NV : (C + 256 * W - 1) / (256 * W);
    const long long words = q8_pitch(C) / 4;
    float v[NV ? NV : 1][4];
    double part[NB] = {}, sum = 0;

    if (row >= a.rows)
        return;
    const float *X = a.X + row * a.ldx, *R = a.R ? a.R + row * a.ldr : nullptr;
    float *H = a.H ? a.H + row * a.ldh : nullptr, *Y = a.Y ? a.Y + row * a.ldy : nullptr;
    unsigned *Q = a.Q ? a.Q + row * words : nullptr;
    auto at = [&](int k) { return 256 * (W * k + sub) + 4 * lane; };
    auto load = [&](int k, float (&x)[4]) {
        load4_row(X, at(k), C, x);
        if (R) {
            float r[4];

            load4_row(R, at(k), C, r);
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] += r[j];
        }
    };
#pragma unroll NV ? NV : 1
    for (int k = 0; k < steps; k++) {
        float(&x)[4] = v[NV ? k : 0];

        load(k, x);
#pragma unroll
        for (int j = 0; j < 4; j++)
            part[NB > 1 ? k : 0] += (double)x[j] * x[j];
        if (H)
            store4_row(H, at(k), C, x);
    }
    if constexpr (!LANES) {
#pragma unroll
        for (int k = 0; k < NB; k++)
            part[k] = wave_dsum(part[k]);
    }
    if constexpr (W > 1) {
        if (LANES || lane == 0) {
#pragma unroll
            for (int k = 0; k < NB; k++)
                sums[W * k + sub][LANES ? lane : 0] = part[k];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < NB * W; e++)
            sum += sums[e][LANES ? lane : 0];
    }
    else {
#pragma unroll
        for (int k = 0; k < NB; k++)
            sum += part[k];
    }
    if constexpr (LANES)
        sum = wave_dsum(sum);
    const float inv = (float)(1.0 / sqrt(sum / C + a.eps));
    unsigned mag = 0;

    /* Channels behind the last have y = 0, or NaN where the row has one, whose
     * codes are all 0: inv is never infinite, as eps is above 0. */
    auto scale = [&](int k, float (&x)[4]) {
        if (!NV) {
            if (H)
                load4_row(H, at(k), C, x);
            else
                load(k, x);
        }
        if (a.g) {
            float g[4];

            load4_row(a.g, at(k), C, g);
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] = x[j] * inv * g[j];
        }
        else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] *= inv;
        }
    };
    if (NV || Q) {
#pragma unroll NV ? NV : 1
        for (int k = 0; k < steps; k++) {
            float(&x)[4] = v[NV ? k : 0];

            scale(k, x);
#pragma unroll
            for (int j = 0; j < 4; j++)
                mag = max(mag, q8_mag(x[j]));
        }
    }
    q8_scale q = {};

    if (Q) {
        mag = wave_umax(mag);
        if constexpr (W > 1) {
            if (lane == 0)
                tops[sub] = mag;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < W; e++)
                mag = max(mag, tops[e]);
        }
        q = q8_scale_of(mag);
        if (lane == 0 && sub == 0)
            a.S[row] = q.s;
    }
#pragma unroll NV ? NV : 1
    for (int k = 0; k < steps; k++) {
        const int w = 64 * (W * k + sub) + lane;
        float(&x)[4] = v[NV ? k : 0];

        if (!NV)
            scale(k, x);
        if (Y)
            store4_row(Y, at(k), C, x);
        if (Q && w < words)
            Q[w] = q8_code4(x[0], x[1], x[2], x[3], q.r);
    }
}

/* An operand of `rows` rows of C floats, or NULL where it has no buffer. */
static float *norm_rows(const struct opnd &x, long rows, int C, long long &ld, const char *op,
                        const char *name)
{
    ld = C;
    if (!x.buf)
        return nullptr;
    if (x.off < 0 || x.ld < C)
        icoreg_fatal("%s: negative offset or short row of %s: ld %d", op, name, x.ld);
    need_floats(x.buf, x.off, (rows - 1) * (long long)x.ld + C, op, name);
    /* One row's stride means nothing. */
    ld = rows > 1 ? x.ld : C;
    return fptr(x.buf) + x.off;
}

extern "C" void ops_rms_norm(struct ops *o, long rows, int C, struct opnd X, struct opnd R, cl_mem g,
                             float eps, struct opnd H, struct opnd Y, cl_mem Q, cl_mem S)
{
    ICOREG_API_BEGIN
    const char *op = "ops_rms_norm";
    norm_args a = {};

    if (rows < 0 || rows > 0x7fffffffL || C < 1 || C > NORM_MAX_C)
        icoreg_fatal("%s: invalid sizes rows=%ld C=%d", op, rows, C);
    if (!(eps > 0.0f) || !isfinite(eps))
        icoreg_fatal("%s: eps %g is not above 0 and finite", op, eps);
    if (!H.buf && !Y.buf && !Q)
        icoreg_fatal("%s: no output", op);
    if (!Q != !S)
        icoreg_fatal("%s: codes without scales, or scales without codes", op);
    if (rows == 0)
        return;
    if (!X.buf)
        icoreg_fatal("%s: X is NULL", op);
    a.X = norm_rows(X, rows, C, a.ldx, op, "X");
    a.R = norm_rows(R, rows, C, a.ldr, op, "R");
    a.H = norm_rows(H, rows, C, a.ldh, op, "H");
    a.Y = norm_rows(Y, rows, C, a.ldy, op, "Y");
    {
        const long long qbytes = rows * q8_pitch(C);
        const struct {
            float *p;
            long long ld;
            const char *in, *q, *s, *gain;
        } out[2] = {{a.H, a.ldh, "H and an input (unless the same rows)", "H and Q", "H and S", "H and g"},
                    {a.Y, a.ldy, "Y and an input (unless the same rows)", "Y and Q", "Y and S", "Y and g"}};
        const struct {
            const float *p;
            long long ld;
            const char *q, *s;
        } in[2] = {{a.X, a.ldx, "X and Q", "X and S"}, {a.R, a.ldr, "R and Q", "R and S"}};

        if (g)
            need_floats(g, 0, C, op, "g");
        if (Q) {
            need_bytes(Q, 0, qbytes, op, "Q");
            need_aligned(Q, 16, op, "Q");
            need_floats(S, 0, rows, op, "S");
            need_apart(Q, 0, qbytes, S, 0, rows * 4, op, "Q and S");
            need_apart(g, 0, C * 4LL, Q, 0, qbytes, op, "g and Q");
            need_apart(g, 0, C * 4LL, S, 0, rows * 4, op, "g and S");
        }
        /* Codes and scales as rows of floats, for the overlaps with rows. */
        auto flat = [&](const float *p, long long ld, const void *b, long long bytes, const char *what) {
            if (p && b && bytes)
                need_rows_apart(p, ld, C, rows, (const float *)b, bytes / 4, bytes / 4, 1, op, what);
        };
        for (const auto &w : out) {
            if (!w.p)
                continue;
            for (const auto &r : in)
                if (r.p && (w.p != r.p || w.ld != r.ld))
                    need_rows_apart(w.p, w.ld, C, rows, r.p, r.ld, C, rows, op, w.in);
            flat(w.p, w.ld, Q ? Q->ptr : nullptr, qbytes, w.q);
            flat(w.p, w.ld, S ? S->ptr : nullptr, rows * 4, w.s);
            flat(w.p, w.ld, g ? g->ptr : nullptr, C * 4LL, w.gain);
        }
        for (const auto &r : in) {
            flat(r.p, r.ld, Q ? Q->ptr : nullptr, qbytes, r.q);
            flat(r.p, r.ld, S ? S->ptr : nullptr, rows * 4, r.s);
        }
        if (a.H && a.Y)
            need_rows_apart(a.H, a.ldh, C, rows, a.Y, a.ldy, C, rows, op, "H and Y");
    }
    a.g = cfptr(g);
    a.S = fptr(S);
    a.Q = Q ? (unsigned *)Q->ptr : nullptr;
    a.C = C;
    a.eps = eps;
    {
        const device_scope on(o->ocl);
        const hipStream_t s = stream_of(o->ocl);

        prof_scope ps(o->ocl, "rms_norm");
        for (long r = 0; r < rows; r += NORM_ROWS) {
            const long n = rows - r < NORM_ROWS ? rows - r : NORM_ROWS;
            norm_args b = a;

            b.X += r * a.ldx;
            if (b.R)
                b.R += r * a.ldr;
            if (b.H)
                b.H += r * a.ldh;
            if (b.Y)
                b.Y += r * a.ldy;
            if (b.Q) {
                b.Q += r * (q8_pitch(C) / 4);
                b.S += r;
            }
            b.rows = n;
            /* Few rows, several waves each, us: of 1024 channels 1 row 4.2 -> 2.9,
             * 512 rows 5.0 -> 3.5, 2048 6.3 -> 6.0, 3202 9.2 -> 9.4; of 4096, 16 waves
             * for 4, 1 row 4.6 -> 3.8, 256 rows 5.6 -> 4.8, 512 6.3 -> 6.5. */
#define NORM_LAUNCH(NV_, W_)                                                                          \
    do {                                                                                              \
        constexpr int threads = W_ > 4 ? 64 * W_ : 256;                                               \
        static_assert(W_ * 64LL * NORM_ROWS < 1LL << 32, "threads of a launch");                      \
        hipLaunchKernelGGL((rms_norm_kernel<NV_, W_>), dim3(grid_of(W_ > 1 ? n : (n + 3) / 4, threads, op)), \
                           dim3(threads), 0, s, b);                                                   \
    } while (0)
            if (C <= 256)
                NORM_LAUNCH(1, 1);
            else if (C <= 1024 && n < 2560)
                NORM_LAUNCH(1, 4);
            else if (C <= 1024)
                NORM_LAUNCH(4, 1);
            else if (C <= 4096 && n < 384)
                NORM_LAUNCH(1, 16);
            else if (C <= 4096)
                NORM_LAUNCH(4, 4);
            else if (C <= 16384)
                NORM_LAUNCH(4, 16);
            else
                NORM_LAUNCH(0, 16);
#undef NORM_LAUNCH
            launch_check("rms_norm");
        }
    }
    ICOREG_API_END
}
