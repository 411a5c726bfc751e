/* SPDX-License-Identifier: Unlicense */

/* Linear layers in 8-bit integers, a scale per token and per output channel:
 *
 *   y[i][j] = act(sx[i] sw[j] sum_k cx[i][k] cw[j][k] + b[j]) + r[i][j]
 *
 * with the codes and scales of q8.h. The sum of at most 2^17 products of
 * magnitude 127^2 fits 32-bit integers, so it is exact in every order; it is
 * converted to float32 and multiplied by the float32 product of the two
 * scales. */

#include <hip/hip_runtime.h>

#include <type_traits>

#include "act.h"
#include "common.h"
#include "gemm_dev.h"
#include "load4.h"
#include "ops.h"
#include "q8.h"

using namespace icoreg;

#define Q8_MAX_IN (1 << 17)
#define Q8_MAX_C (1 << 30)        /* channels are counted in int, past the last too */
#define Q8_ROWS (1L << 23)        /* rows of a launch: 2^32 threads are too many */
#define Q8_MAX_SIDE 0x7ffffe00    /* tokens and channels of a product, counted past the last too */

typedef int q8_i4 __attribute__((ext_vector_type(4)));
typedef int q8_i16 __attribute__((ext_vector_type(16)));

/* ---- codes of rows --------------------------------------------------------- */

/* W waves a row (1 or 4), four channels a lane and step: the largest
 * magnitude, then the codes. Rows of up to 256 NV W channels stay in registers
 * between the two; longer ones (NV = 0) are read again. Bound by memory, which
 * is why a row is read once: 12805 x 4096 (210 MB in, 52 out) 55.7 us, 4.7
 * TB/s, a large copy's rate; 3202 x 4096 10.9 us, 6.0 TB/s, its input partly
 * still in the last cache. */
template <int NV, int W>
__global__ void __launch_bounds__(256)
    quant_rows_kernel(const float *__restrict__ X, long long ldx, long rows, int C,
                      unsigned *__restrict__ Q, float *__restrict__ S)
{
    __shared__ unsigned tops[W > 1 ? W : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = wave % W;
    const long row = (long)blockIdx.x * (4 / W) + wave / W;
    const int steps = NV ? NV : (C + 256 * W - 1) / (256 * W);
    const long long words = q8_pitch(C) / 4;
    float v[NV ? NV : 1][4];
    unsigned mag = 0;

    if (row >= rows)
        return;
    X += row * ldx;
    Q += row * words;
    auto load = [&](int k, float (&x)[4]) {
        load4_row(X, 256 * (W * k + sub) + 4 * lane, C, x);
    };
#pragma unroll NV ? NV : 1
    for (int k = 0; k < steps; k++) {
        float(&x)[4] = v[NV ? k : 0];

        load(k, x);
#pragma unroll
        for (int j = 0; j < 4; j++)
            mag = max(mag, q8_mag(x[j]));
    }
    mag = wave_umax(mag);
    if constexpr (W > 1) {
        if (lane == 0)
            tops[sub] = mag;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < W; e++)
            mag = max(mag, tops[e]);
    }
    const q8_scale q = q8_scale_of(mag);

    if (lane == 0 && sub == 0)
        S[row] = q.s;
#pragma unroll NV ? NV : 1
    for (int k = 0; k < steps; k++) {
        const int w = 64 * (W * k + sub) + lane;
        float(&x)[4] = v[NV ? k : 0];

        if (!NV)
            load(k, x);
        if (w < words)
            Q[w] = q8_code4(x[0], x[1], x[2], x[3], q.r);
    }
}

static void quant_rows(struct ops *o, long rows, int C, const float *X, long long ldx, void *Q,
                       float *S)
{
    /* Long rows, a block each: 4096 channels, 16 rows 4.2 -> 2.7 us, 785 rows 6.5
     * -> 3.7. */
    const bool wide = C > 1024;
    const hipStream_t s = stream_of(o->ocl);

    prof_scope ps(o->ocl, "quant_rows");
    for (long r = 0; r < rows; r += Q8_ROWS) {
        const long n = rows - r < Q8_ROWS ? rows - r : Q8_ROWS;
        const dim3 grid((unsigned)(wide ? n : (n + 3) / 4)), block(256);

#define QUANT_LAUNCH(NV_, W_)                                                                 \
    hipLaunchKernelGGL((quant_rows_kernel<NV_, W_>), grid, block, 0, s, X + r * ldx, ldx, n, C, \
                       (unsigned *)((char *)Q + r * q8_pitch(C)), S + r)
        if (C <= 256)
            QUANT_LAUNCH(1, 1);
        else if (C <= 1024)
            QUANT_LAUNCH(4, 1);
        else if (C <= 4096)
            QUANT_LAUNCH(4, 4);
        else if (C <= 16384)
            QUANT_LAUNCH(16, 4);
        else
            QUANT_LAUNCH(0, 4);
#undef QUANT_LAUNCH
        launch_check("quant_rows");
    }
}

extern "C" int ops_q8_pitch(int C)
{
    return C < 1 || C > Q8_MAX_C ? 0 : (int)q8_pitch(C);
}

extern "C" void ops_quant_rows(struct ops *o, long rows, int C, cl_mem X, long xoff, int ldx,
                               cl_mem Q, cl_mem S)
{
    ICOREG_API_BEGIN
    const char *op = "ops_quant_rows";

    if (rows < 0 || rows > 0x7fffffffL || C < 1 || C > Q8_MAX_C || ldx < C || xoff < 0)
        icoreg_fatal("%s: invalid sizes rows=%ld C=%d ldx=%d", op, rows, C, ldx);
    if (rows == 0)
        return;
    need_floats(X, xoff, (long long)(rows - 1) * ldx + C, op, "X");
    need_bytes(Q, 0, rows * q8_pitch(C), op, "Q");
    need_aligned(Q, 16, op, "Q");
    need_floats(S, 0, rows, op, "S");
    need_apart(X, xoff * 4, ((rows - 1) * (long long)ldx + C) * 4, Q, 0, rows * q8_pitch(C), op,
               "X and Q");
    need_apart(S, 0, rows * 4, X, xoff * 4, ((rows - 1) * (long long)ldx + C) * 4, op, "S and X");
    need_apart(S, 0, rows * 4, Q, 0, rows * q8_pitch(C), op, "S and Q");
    quant_rows(o, rows, C, cfptr(X) + xoff, ldx, Q->ptr, fptr(S));
    ICOREG_API_END
}

/* ---- the product -------------------------------------------------------------- */

struct q8_args {
    int M, N;
    long long pitch; /* bytes of a row of codes, both operands */
    const signed char *A, *B;
    const float *sa, *sb, *bias, *R;
    float *C;
    long long ldc;
    int act;
    float slope;
};

/* v times the normal distribution's integral to v: max(v, 0) - |v| g(|v|), g(z)
 * = erfc(z / sqrt 2) / 2 = exp(-z^2 / 2) f(1 / (1 + 0.4 z / sqrt 2)), f a
 * polynomial of degree 6 fitted to exp(x^2) erfc(x) / 2 (its error times
 * exp(-x^2) at most 2e-8): within 4 2^-24 |v|, 16 instructions and no branch, where
 * erff takes both sides of one (64 outputs a lane are the layer's epilogue). */
__device__ __forceinline__ float q8_gelu(float v)
{
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(v), 0.282842712f, 1.0f));
    const float e = __builtin_amdgcn_exp2f(v * -0.72134752f * v);
    float p = fmaf(t, -1.036704183e-01f, 3.702977300e-01f);

    p = fmaf(t, p, -2.139942795e-01f);
    p = fmaf(t, p, 2.611404359e-01f);
    p = fmaf(t, p, 6.693785638e-02f);
    p = fmaf(t, p, 1.196817234e-01f);
    p = fmaf(t, p, -3.930720559e-04f);
    /* Infinity stays what it is, where the second term would be infinity times
     * 0 (3202 x 1024 x 4096 34.3 us without the minimum, 34.6, 34.8 with a select). */
    return fmaf(-fabsf(fminf(v, 0x1p64f)), e * p, fmaxf(v, 0.0f));
}

/* The tanh form: 0.5 v (1 + tanh w) = v / (1 + exp(-2 w)). */
__device__ __forceinline__ float q8_gelu_tanh(float v)
{
    const float w = 0.79788456080286536f * fmaf(0.044715f * v * v, v, v);

    return v / (1.0f + __builtin_amdgcn_exp2f(w * -2.88539008f));
}

/* act(sa sb sum + bias), the sum converted once. ReLU is not the leaky one with
 * slope 0, which makes NaN of minus infinity; a NaN stays one in both. */
template <int ACT>
__device__ __forceinline__ float q8_out(int sum, float sa, float sb, float b, float slope)
{
    const float v = fmaf(sa * sb, (float)sum, b);

    if (ACT == ACT_GELU)
        return q8_gelu(v);
    if (ACT == ACT_GELU_TANH)
        return q8_gelu_tanh(v);
    if (ACT == ACT_RELU)
        return v < 0.0f ? 0.0f : v;
    if (ACT == ACT_LEAKY)
        return v >= 0.0f ? v : slope * v;
    return v;
}

/* gfx9 s_waitcnt immediate: at most n vector memory operations outstanding,
 * every LDS read done. */
constexpr int q8_wait(int n) { return 0x0070 | (n & 15) | (n >> 4) << 14; }

/* Blocks of BM tokens x BN channels, WM x WN waves (KS groups of them, each
 * on its part of every step). BK bytes of both panels a step by LDS DMA, ST
 * buffers, one barrier a step, in front of its last products: there the loads
 * of the next step have arrived (those of ST - 2 more may be on their way), all
 * waves have read the last operands of this one, and its buffer takes the
 * loads of step k + ST. Steps past the last load zeros, so that the count of
 * loads stays the same. 128 bytes a row, a whole line, come from L2 at twice
 * the rate of 64 (25 TB/s, 13.7). Rows hold their 16-byte chunks in the order
 * chunk ^ row, which spreads the rows that a matrix instruction reads over the
 * banks (no conflicts counted).
 * v_mfma_i32_32x32x32_i8 with the channels as rows and the tokens as columns:
 * lane half h takes bytes 16 h .. of 32 of row lane % 32 of either operand, and
 * a lane's sums are four runs of four neighbouring channels of one token,
 * stored 16 bytes at a time. Operands of the next 32 bytes are read while
 * this one's products run. Rows past M and N are outside the panels' windows
 * and read as zeros.
 *
 * 12288 x 4096 x 4096 on blocks of 256 x 256: 206 us, 2000 TOP/s (224 on
 * another card), the matrix cores busy 54 % of it (a library's plain int8 product, nothing scaled and 32
 * bits out: 1860 at 4096 cubed, 2370 at 8192); what is left is the three rounds'
 * epilogues, 201 MB of outputs written while no product runs. 3202 x 1024 x
 * 4096 with GELU 31.6 us: one round, 8 steps and 52 MB to write. Two buffers of
 * 128 KB in all, one block a CU: a second one would hide the epilogue and does
 * not fit. */
template <int BM, int BN, int WM, int WN, int BK, int KS, int ST, int ACT>
__global__ void __launch_bounds__(64 * WM * WN * KS) q8_gemm(const q8_args g)
{
    constexpr int NT = 64 * WM * WN * KS, CH = BK / 16, KK = BK / 32 / KS;
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int ASZ = BM * BK, BSZ = BN * BK, SZ = ASZ + BSZ;
    constexpr int AL = ASZ / 16 / NT, BL = BSZ / 16 / NT;
    static_assert(AL >= 1 && BL >= 1 && ASZ % (16 * NT) == 0 && BSZ % (16 * NT) == 0, "tile shape");
    static_assert(ST == 2 || ST == 3, "buffers");
    __shared__ __align__(16) signed char s0[SZ], s1[SZ], s2[ST > 2 ? SZ : 16];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kg = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
    const int h = lane >> 5, r32 = lane & 31;
    /* Bands of 4 rows of tiles, so that the tiles in flight on an XCD share
     * rows of both operands. */
    const int tiles_n = (g.N + BN - 1) / BN, tiles_m = (g.M + BM - 1) / BM;
    const int tile = xcd_tile(blockIdx.x, gridDim.x), band = tile / (4 * tiles_n);
    const int in_band = tile - band * 4 * tiles_n, high = min(4, tiles_m - 4 * band);
    const int m0 = (4 * band + in_band % high) * BM, n0 = in_band / high * BN;
    const int pitch = (int)g.pitch;
    const signed char *A = g.A + m0 * g.pitch, *B = g.B + n0 * g.pitch;
    const long long abytes = min(BM, g.M - m0) * g.pitch, bbytes = min(BN, g.N - n0) * g.pitch;
    int aoff[AL], boff[BL], ak[AL], bk[BL];
    q8_i16 acc[TN][TM];

#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                acc[i][j][r] = 0;
#pragma unroll
    for (int q = 0; q < AL; q++) {
        const int sl = tid + NT * q, row = sl / CH;

        ak[q] = 16 * ((sl % CH) ^ (row / (16 / CH) % CH));
        aoff[q] = row * pitch + ak[q];
    }
#pragma unroll
    for (int q = 0; q < BL; q++) {
        const int sl = tid + NT * q, row = sl / CH;

        bk[q] = 16 * ((sl % CH) ^ (row / (16 / CH) % CH));
        boff[q] = row * pitch + bk[q];
    }
    auto load = [&](int k0, signed char *s) {
        const __amdgpu_buffer_rsrc_t ra = gemm_rsrc((const float *)A, abytes);
        const __amdgpu_buffer_rsrc_t rb = gemm_rsrc((const float *)B, bbytes);

#pragma unroll
        for (int q = 0; q < AL; q++) {
            const unsigned off = k0 + ak[q] < pitch ? (unsigned)(aoff[q] + k0) : GEMM_OOB;

            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                ra, (__attribute__((address_space(3))) void *)(s + 16 * (NT * q + 64 * wave)), 16,
                (int)off, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < BL; q++) {
            const unsigned off = k0 + bk[q] < pitch ? (unsigned)(boff[q] + k0) : GEMM_OOB;

            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rb, (__attribute__((address_space(3))) void *)(s + ASZ + 16 * (NT * q + 64 * wave)), 16,
                (int)off, 0, 0, 0);
        }
    };
    auto read = [&](const signed char *s, int kk, q8_i4 (&a)[TM], q8_i4 (&b)[TN]) {
#pragma unroll
        for (int j = 0; j < TM; j++) {
            const int row = wm * (BM / WM) + j * 32 + r32;

            a[j] = *(const q8_i4 *)(s + row * BK + 16 * ((2 * (KK * kg + kk) + h) ^ (row / (16 / CH) % CH)));
        }
#pragma unroll
        for (int i = 0; i < TN; i++) {
            const int row = wn * (BN / WN) + i * 32 + r32;

            b[i] = *(const q8_i4 *)(s + ASZ + row * BK + 16 * ((2 * (KK * kg + kk) + h) ^ (row / (16 / CH) % CH)));
        }
    };
    auto multiply = [&](const q8_i4 (&a)[TM], const q8_i4 (&b)[TN]) {
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[i], a[j], acc[i][j], 0, 0, 0);
    };
    const int nk = (pitch + BK - 1) / BK;
    q8_i4 a[2][TM], b[2][TN];
    /* One operand read, one product, and so on; the loads behind them. */
    auto mix = [&]() {
#pragma unroll
        for (int e = 0; e < TM + TN; e++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if (e < TM * TN)
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
    };
    auto meet = [&](auto n) {
        __builtin_amdgcn_s_waitcnt(q8_wait(decltype(n)::value * (AL + BL)));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto step = [&](int kt, signed char *now, const signed char *next) {
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (kk + 1 < KK)
                read(now, kk + 1, a[(kk + 1) & 1], b[(kk + 1) & 1]);
            else {
                meet(std::integral_constant<int, ST - 2>());
                load((kt + ST) * BK, now);
                read(next, 0, a[0], b[0]);
            }
            multiply(a[kk & 1], b[kk & 1]);
            mix();
        }
    };
    static_assert(KK % 2 == 0, "operands alternate");

    load(0, s0);
    load(BK, s1);
    if (ST > 2)
        load(2 * BK, s2);
    meet(std::integral_constant<int, ST - 1>());
    read(s0, 0, a[0], b[0]);
    for (int kt = 0; kt < nk; kt += ST) {
        step(kt, s0, s1);
        if (kt + 1 < nk)
            step(kt + 1, s1, ST > 2 ? s2 : s0);
        if (ST > 2 && kt + 2 < nk)
            step(kt + 2, s2, s0);
    }
    __builtin_amdgcn_s_waitcnt(q8_wait(0));
    if constexpr (KS > 1) {
        /* Two groups of waves have summed halves of every step: each takes
         * the other's sums of half its channels and finishes those. */
        static_assert(KS == 2 && TN % 2 == 0 && WM * WN * (TN / 2) * TM * 4096 <= SZ, "exchange");
        const int w = (wm * WN + wn) * (TN / 2) * TM;
        q8_i4 *out = (q8_i4 *)(kg ? s0 : s1) + w * 256 + lane;
        const q8_i4 *in = (const q8_i4 *)(kg ? s1 : s0) + w * 256 + lane;

        __syncthreads();
#pragma unroll
        for (int i = 0; i < TN / 2; i++)
#pragma unroll
            for (int j = 0; j < TM; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const q8_i16 &x = kg ? acc[i][j] : acc[i + TN / 2][j];

                    out[((i * TM + j) * 4 + q) * 64] =
                        q8_i4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
                }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TN / 2; i++)
#pragma unroll
            for (int j = 0; j < TM; j++) {
                if (kg)
                    acc[i][j] = acc[i + TN / 2][j];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const q8_i4 y = in[((i * TM + j) * 4 + q) * 64];

#pragma unroll
                    for (int r = 0; r < 4; r++)
                        acc[i][j][4 * q + r] += y[r];
                }
            }
    }

    /* Register r of a tile: channel (r / 4) * 8 + 4 h + r % 4, token lane % 32.
     * Loads before stores: C may be R. */
#pragma unroll
    for (int i = 0; i < TN / KS; i++) {
        const int n = n0 + wn * (BN / WN) + (i + kg * (TN / 2)) * 32 + 4 * h;
        float sb[16], b[16];

#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int at = min(n + (r >> 2) * 8 + (r & 3), g.N - 1);

            sb[r] = g.sb[at];
            b[r] = g.bias ? g.bias[at] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < TM; j++) {
            const int m = m0 + wm * (BM / WM) + j * 32 + r32;
            const float sa = g.sa[min(m, g.M - 1)];
            float *c = g.C + m * g.ldc + n;
            const float *x = g.R + m * g.ldc + n;
            float v[16];

#pragma unroll
            for (int r = 0; r < 16; r++)
                v[r] = q8_out<ACT>(acc[i][j][r], sa, sb[r], b[r], g.slope);
            if (m >= g.M)
                continue;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int left = g.N - n - 8 * q;
                float *y = v + 4 * q;

                if (left >= 4) {
                    float old[4] = {0, 0, 0, 0};

                    if (g.R)
                        load4(x + 8 * q, old);
                    store4(c + 8 * q, y[0] + old[0], y[1] + old[1], y[2] + old[2], y[3] + old[3]);
                }
                else
                    for (int r = 0; r < left; r++)
                        c[8 * q + r] = g.R ? y[r] + x[8 * q + r] : y[r];
            }
        }
    }
}

/* Few tokens: what counts is the weights' bytes and the latency. Blocks of 16
 * channels x 16 TT tokens, 64 bytes of the sum (one matrix instruction) a wave
 * and turn, the 8 waves' sums joined in LDS. Both operands come straight from
 * memory: 4 lanes read 64 bytes of a row. FUSED: every block codes its tokens
 * itself, into LDS (rows 16 bytes further apart, so that 16 of them spread
 * over the banks), while its first weights are on their way. A token of 1024
 * channels to 4096, 4.2 MB of weights: 5.1 us, of which a launch of nothing
 * takes 2.4; 400 x 256 x 256 5.8 us a call. Latency: two passes over the
 * tokens, the sums' exchange. */
#define Q8_SW 8              /* waves */
#define Q8_FUSED_BYTES 40960 /* codes in LDS */

template <int TT, bool FUSED, int ACT>
__global__ void __launch_bounds__(64 * Q8_SW)
    q8_skinny(const q8_args g, const float *__restrict__ X, long long ldx, int in)
{
    constexpr int AHEAD = 4;
    __shared__ __align__(16) signed char xs[FUSED ? Q8_FUSED_BYTES : 16];
    __shared__ q8_i4 sums[Q8_SW][TT][64];
    __shared__ unsigned tops[16 * TT];
    __shared__ float scales[16 * TT];
    const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, part = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles_n = (g.N + 15) / 16, pitch = (int)g.pitch, nk = pitch / 64;
    const int n0 = blockIdx.x % tiles_n * 16, m0 = blockIdx.x / tiles_n * 16 * TT;
    const signed char *w = g.B + (long long)min(n0 + c16, g.N - 1) * pitch + 16 * part;
    /* This thread's output: a run of 16 channels a token, in memory's order.
     * What it needs is read at the start too. */
    const int n = n0 + tid % 16, tok = tid / 16, m = m0 + tok;
    const bool mine = tok < 16 * TT && n < g.N && m < g.M;
    const float sb = mine ? g.sb[n] : 0.0f, bias = mine && g.bias ? g.bias[n] : 0.0f;
    const float res = mine && g.R ? g.R[m * g.ldc + n] : 0.0f;
    q8_i4 a[AHEAD], acc[TT];

    static_assert(16 * TT * 16 <= 64 * Q8_SW, "an output a thread");
#pragma unroll
    for (int t = 0; t < TT; t++)
        acc[t] = q8_i4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < AHEAD; e++)
        a[e] = *(const q8_i4 *)(w + 64 * min(wave + Q8_SW * e, nk - 1));
    if constexpr (FUSED) {
        /* Pieces of 256 channels of a token, dealt to the waves; the first
         * HOLD of a wave's stay in registers from the maximum to the codes. */
        constexpr int HOLD = 8;
        const int tokens = min(16 * TT, g.M - m0), pieces = (pitch + 255) / 256;
        const int all = tokens * pieces;
        float v[HOLD][4];
        auto fetch = [&](int e, float (&x)[4]) {
            const int t = e / pieces, c = 256 * (e - t * pieces) + 4 * lane;

            load4_row(X + (m0 + t) * ldx, c, in, x);
            return t;
        };

#pragma unroll
        for (int e = 0; e < HOLD; e++)
            if (wave + Q8_SW * e < all)
                fetch(wave + Q8_SW * e, v[e]);
        if (tid < 16 * TT)
            tops[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < HOLD; e++)
            if (wave + Q8_SW * e < all) {
                const unsigned top = wave_umax(max(max(q8_mag(v[e][0]), q8_mag(v[e][1])),
                                                   max(q8_mag(v[e][2]), q8_mag(v[e][3]))));

                if (lane == 0)
                    atomicMax(&tops[(wave + Q8_SW * e) / pieces], top);
            }
        for (int e = wave + Q8_SW * HOLD; e < all; e += Q8_SW) {
            float x[4];
            const int t = fetch(e, x);
            const unsigned top =
                wave_umax(max(max(q8_mag(x[0]), q8_mag(x[1])), max(q8_mag(x[2]), q8_mag(x[3]))));

            if (lane == 0)
                atomicMax(&tops[t], top);
        }
        __syncthreads();
        auto code = [&](int e, const float (&x)[4]) {
            const int t = e / pieces, c = 64 * (e - t * pieces) + lane;
            const q8_scale q = q8_scale_of(tops[t]);

            if (4 * c < pitch)
                ((unsigned *)(xs + t * (pitch + 16)))[c] = q8_code4(x[0], x[1], x[2], x[3], q.r);
        };

#pragma unroll
        for (int e = 0; e < HOLD; e++)
            if (wave + Q8_SW * e < all)
                code(wave + Q8_SW * e, v[e]);
        for (int e = wave + Q8_SW * HOLD; e < all; e += Q8_SW) {
            float x[4];

            fetch(e, x);
            code(e, x);
        }
        if (tid < tokens)
            scales[tid] = q8_scale_of(tops[tid]).s;
        __syncthreads();
    }
    for (int k = wave; k < nk; k += Q8_SW * AHEAD) {
        q8_i4 now[AHEAD];

#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            now[e] = a[e];
            a[e] = *(const q8_i4 *)(w + 64 * min(k + Q8_SW * (AHEAD + e), nk - 1));
        }
#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            const int kk = k + Q8_SW * e;

            if (kk < nk) {
#pragma unroll
                for (int t = 0; t < TT; t++) {
                    const int m = min(16 * t + c16, g.M - 1 - m0);
                    const signed char *x = FUSED ? xs + m * (pitch + 16)
                                                 : g.A + (long long)(m0 + m) * pitch;
                    const q8_i4 b = *(const q8_i4 *)(x + 64 * kk + 16 * part);

                    acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now[e], b, acc[t], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TT; t++)
        sums[wave][t][lane] = acc[t];
    __syncthreads();
    /* Sum r of lane l: channel 4 (l / 16) + r, token l % 16. */
    if (mine) {
        const int l = tid % 16 / 4 * 16 + tok % 16;
        int v = 0;

#pragma unroll
        for (int q = 0; q < Q8_SW; q++)
            v += ((const int *)&sums[q][tok / 16][l])[tid % 4];
        const float y = q8_out<ACT>(v, FUSED ? scales[tok] : g.sa[m], sb, bias, g.slope);

        g.C[m * g.ldc + n] = g.R ? y + res : y;
    }
}

template <int TT, bool FUSED>
static void q8_skinny_launch(const q8_args &g, const float *X, long long ldx, int in, hipStream_t s)
{
    const long long tiles = (long long)((g.N + 15) / 16) * ((g.M + 16 * TT - 1) / (16 * TT));
    const dim3 grid(grid_of(tiles, 64 * Q8_SW, "q8 tiles")), block(64 * Q8_SW);

    switch (g.act) {
    case ACT_GELU:
        hipLaunchKernelGGL((q8_skinny<TT, FUSED, ACT_GELU>), grid, block, 0, s, g, X, ldx, in);
        break;
    case ACT_GELU_TANH:
        hipLaunchKernelGGL((q8_skinny<TT, FUSED, ACT_GELU_TANH>), grid, block, 0, s, g, X, ldx, in);
        break;
    case ACT_RELU:
        hipLaunchKernelGGL((q8_skinny<TT, FUSED, ACT_RELU>), grid, block, 0, s, g, X, ldx, in);
        break;
    case ACT_LEAKY:
        hipLaunchKernelGGL((q8_skinny<TT, FUSED, ACT_LEAKY>), grid, block, 0, s, g, X, ldx, in);
        break;
    default:
        hipLaunchKernelGGL((q8_skinny<TT, FUSED, ACT_NONE>), grid, block, 0, s, g, X, ldx, in);
    }
}

template <int BM, int BN, int WM, int WN, int BK, int KS, int ST>
static void q8_launch(const q8_args &g, hipStream_t s)
{
    const long long tiles = (long long)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    const dim3 grid(grid_of(tiles, 64 * WM * WN * KS, "q8 tiles")), block(64 * WM * WN * KS);

    switch (g.act) {
    case ACT_GELU:
        hipLaunchKernelGGL((q8_gemm<BM, BN, WM, WN, BK, KS, ST, ACT_GELU>), grid, block, 0, s, g);
        break;
    case ACT_GELU_TANH:
        hipLaunchKernelGGL((q8_gemm<BM, BN, WM, WN, BK, KS, ST, ACT_GELU_TANH>), grid, block, 0, s, g);
        break;
    case ACT_RELU:
        hipLaunchKernelGGL((q8_gemm<BM, BN, WM, WN, BK, KS, ST, ACT_RELU>), grid, block, 0, s, g);
        break;
    case ACT_LEAKY:
        hipLaunchKernelGGL((q8_gemm<BM, BN, WM, WN, BK, KS, ST, ACT_LEAKY>), grid, block, 0, s, g);
        break;
    default:
        hipLaunchKernelGGL((q8_gemm<BM, BN, WM, WN, BK, KS, ST, ACT_NONE>), grid, block, 0, s, g);
    }
}

/* The kernels, and what a launch takes on 256 CUs: us = fixed + c (tile +
 * sum in / 1024), c the tiles of a CU (its rounds where a CU holds one), from
 * times of 8 .. 12805 tokens on 256 .. 4096 channels of either side. Both
 * sides of some borders, us: 400 x 256 x 256 skinny 3.4, 64 x 64 tiles 4.7;
 * 64 x 1024 x 4096 7.9, 6.5; 785 x 1024 x 1024 64 x 64 7.1, 128 x 128 10.2;
 * 3202 x 1024 x 1024 15.5, 12.5; 6400 x 1024 x 1024 128 x 128 21.1, 256 x 128
 * 18.3; 3202 x 1024 x 4096 256 x 128 33.6, 256 x 256 27.8; 3202 x 4096 x 4096
 * 72.8, 65.4. */
enum { Q8_256, Q8_256_128, Q8_128, Q8_64, Q8_SKINNY2, Q8_SKINNY1, Q8_FORMS };

static const struct q8_form {
    int bm, bn;
    float fixed, tile, sum;
} q8_forms[Q8_FORMS] = {{256, 256, 2.0f, 12.0f, 12.3f}, {256, 128, 2.0f, 9.5f, 6.5f},
                        {128, 128, 2.0f, 6.5f, 3.9f},   {64, 64, 4.4f, 1.4f, 1.9f},
                        {32, 16, 2.2f, 1.7f, 1.25f},    {16, 16, 2.2f, 1.4f, 0.95f}};

static float q8_cost(int form, int M, int N, int pitch, int cus)
{
    const q8_form &f = q8_forms[form];
    const long long tiles = (long long)((M + f.bm - 1) / f.bm) * ((N + f.bn - 1) / f.bn);

    return f.fixed + (float)((tiles + cus - 1) / cus) * (f.tile + f.sum * pitch / 1024.0f);
}

static int q8_best(int M, int N, int pitch, int cus, float &cost)
{
    int best = 0;

    for (int i = 0; i < Q8_FORMS; i++) {
        const float c = q8_cost(i, M, N, pitch, cus);

        if (i == 0 || c < cost) {
            best = i;
            cost = c;
        }
    }
    return best;
}

/* The kernel of M tokens, and how many of them it takes: a last round of few
 * large tiles leaves most CUs waiting (12805 x 4096 x 4096: 816 tiles of 256 x
 * 256, 48 of them alone in a fourth round, 244 us), so its tokens may go to
 * another kernel (12288 tokens, then 517 in tiles of 128 x 128: 234 us). */
static int q8_choose(int M, int N, int pitch, int cus, int &rows)
{
    float cost = 0.0f;
    int best = q8_best(M, N, pitch, cus, cost);

    rows = M;
    for (int i = Q8_256; i <= Q8_256_128; i++) {
        const long long tn = (N + q8_forms[i].bn - 1) / q8_forms[i].bn;
        const long long rounds = ((M + q8_forms[i].bm - 1) / q8_forms[i].bm) * tn / cus;
        const long long m = rounds * cus / tn * q8_forms[i].bm;
        float rest = 0.0f;

        if (m <= 0 || m >= M)
            continue;
        (void)q8_best(M - (int)m, N, pitch, cus, rest);
        rest += q8_cost(i, (int)m, N, pitch, cus);
        if (rest < cost) {
            cost = rest;
            best = i;
            rows = (int)m;
        }
    }
    return best;
}

static void q8_product(struct ops *o, q8_args g)
{
    const hipStream_t s = stream_of(o->ocl);
    const int M = g.M;

    prof_scope ps(o->ocl, "gemm_q8");
    for (int m = 0; m < M; m += g.M) {
        const int form = q8_choose(M - m, g.N, (int)g.pitch, o->ocl->cu_count, g.M);

        switch (form) {
        case Q8_256:
            q8_launch<256, 256, 2, 4, 128, 1, 2>(g, s);
            break;
        case Q8_256_128:
            q8_launch<256, 128, 4, 2, 128, 1, 3>(g, s);
            break;
        case Q8_128:
            q8_launch<128, 128, 2, 2, 128, 2, 3>(g, s);
            break;
        case Q8_64:
            q8_launch<64, 64, 2, 2, 128, 1, 3>(g, s);
            break;
        case Q8_SKINNY2:
            q8_skinny_launch<2, false>(g, nullptr, 0, 0, s);
            break;
        default:
            q8_skinny_launch<1, false>(g, nullptr, 0, 0, s);
        }
        launch_check("gemm_q8");
        g.A += g.M * g.pitch;
        g.sa += g.M;
        g.C += g.M * g.ldc;
        if (g.R)
            g.R += g.M * g.ldc;
    }
}

extern "C" int icoreg_q8_choice(struct ops *o, int rows, int in, int out, int *first)
{
    int n = 0, form;

    if (rows < 1 || rows > Q8_MAX_SIDE || in < 1 || in > Q8_MAX_IN || out < 1 || out > Q8_MAX_SIDE)
        return -1;
    form = q8_choose(rows, out, (int)q8_pitch(in), o->ocl->cu_count, n);
    if (first)
        *first = n;
    return form;
}

/* The checks of both calls and the arguments of the product, its first
 * operand left out. */
static q8_args q8_make(const char *op, int rows, int in, int out, cl_mem WQ, cl_mem WS, cl_mem b,
                       cl_mem R, long roff, cl_mem Y, long yoff, int ldy, int act, float slope)
{
    q8_args g = {};
    const long long span = (long long)(rows - 1) * ldy + out;

    if (rows < 0 || rows > Q8_MAX_SIDE || in < 1 || in > Q8_MAX_IN || out < 0 || out > Q8_MAX_SIDE ||
        ldy < out || yoff < 0 || roff < 0)
        icoreg_fatal("%s: invalid sizes rows=%d in=%d out=%d ldy=%d", op, rows, in, out, ldy);
    if (act < ACT_NONE || act > ACT_GELU_TANH)
        icoreg_fatal("%s: invalid activation %d", op, act);
    if (rows == 0 || out == 0)
        return g;
    need_bytes(WQ, 0, out * q8_pitch(in), op, "WQ");
    need_aligned(WQ, 16, op, "WQ");
    need_floats(WS, 0, out, op, "WS");
    if (b)
        need_floats(b, 0, out, op, "bias");
    need_floats(Y, yoff, span, op, "Y");
    if (R)
        need_floats(R, roff, span, op, "R");
    need_apart(Y, yoff * 4, span * 4, WQ, 0, out * q8_pitch(in), op, "Y and WQ");
    need_apart(Y, yoff * 4, span * 4, WS, 0, out * 4LL, op, "Y and WS");
    need_apart(Y, yoff * 4, span * 4, b, 0, out * 4LL, op, "Y and bias");
    if (R && cfptr(R) + roff != cfptr(Y) + yoff)
        need_rows_apart(cfptr(Y) + yoff, ldy, out, rows, cfptr(R) + roff, ldy, out, rows, op,
                        "Y and R (unless the same)");
    g.M = rows;
    g.N = out;
    g.pitch = q8_pitch(in);
    g.B = (const signed char *)WQ->ptr;
    g.sb = cfptr(WS);
    g.bias = cfptr(b);
    g.R = R ? cfptr(R) + roff : nullptr;
    g.C = fptr(Y) + yoff;
    g.ldc = ldy;
    g.act = act;
    g.slope = slope;
    return g;
}

extern "C" void ops_linear_qq(struct ops *o, int rows, int in, int out, cl_mem XQ, cl_mem XS,
                              cl_mem WQ, cl_mem WS, cl_mem b, cl_mem R, long roff, cl_mem Y,
                              long yoff, int ldy, int act, float slope)
{
    ICOREG_API_BEGIN
    const char *op = "ops_linear_qq";
    q8_args g = q8_make(op, rows, in, out, WQ, WS, b, R, roff, Y, yoff, ldy, act, slope);

    if (rows == 0 || out == 0)
        return;
    need_bytes(XQ, 0, rows * q8_pitch(in), op, "XQ");
    need_aligned(XQ, 16, op, "XQ");
    need_floats(XS, 0, rows, op, "XS");
    need_apart(Y, yoff * 4, ((rows - 1) * (long long)ldy + out) * 4, XQ, 0, rows * q8_pitch(in), op,
               "Y and XQ");
    need_apart(Y, yoff * 4, ((rows - 1) * (long long)ldy + out) * 4, XS, 0, rows * 4LL, op,
               "Y and XS");
    g.A = (const signed char *)XQ->ptr;
    g.sa = cfptr(XS);
    q8_product(o, g);
    ICOREG_API_END
}

/* Work of ops_linear_q8: the tokens' codes, then their scales. */
extern "C" size_t ops_linear_q8_work_bytes(int rows, int in)
{
    if (rows < 1 || rows > Q8_MAX_SIDE || in < 1 || in > Q8_MAX_IN)
        return 0;
    return (size_t)rows * q8_pitch(in) + (size_t)rows * 4;
}

extern "C" void ops_linear_q8(struct ops *o, int rows, int in, int out, cl_mem X, long xoff,
                              int ldx, cl_mem WQ, cl_mem WS, cl_mem b, cl_mem R, long roff,
                              cl_mem Y, long yoff, int ldy, int act, float slope, cl_mem work)
{
    ICOREG_API_BEGIN
    const char *op = "ops_linear_q8";
    q8_args g = q8_make(op, rows, in, out, WQ, WS, b, R, roff, Y, yoff, ldy, act, slope);
    const long long codes = rows * q8_pitch(in), ybytes = ((rows - 1) * (long long)ldy + out) * 4;
    const long long xbytes = ((rows - 1) * (long long)ldx + in) * 4, wbytes = codes + rows * 4LL;

    if (ldx < in || xoff < 0)
        icoreg_fatal("%s: invalid sizes in=%d ldx=%d", op, in, ldx);
    if (rows == 0 || out == 0)
        return;
    need_bytes(X, xoff * 4, xbytes, op, "X");
    need_bytes(work, 0, (long long)ops_linear_q8_work_bytes(rows, in), op, "work");
    need_aligned(work, 16, op, "work");
    need_apart(X, xoff * 4, xbytes, work, 0, wbytes, op, "X and work");
    need_apart(Y, yoff * 4, ybytes, work, 0, wbytes, op, "Y and work");
    need_apart(WQ, 0, out * q8_pitch(in), work, 0, wbytes, op, "WQ and work");
    need_apart(WS, 0, out * 4LL, work, 0, wbytes, op, "WS and work");
    need_apart(b, 0, out * 4LL, work, 0, wbytes, op, "bias and work");
    need_apart(R, roff * 4, ybytes, work, 0, wbytes, op, "R and work");
    need_rows_apart(cfptr(Y) + yoff, ldy, out, rows, cfptr(X) + xoff, ldx, in, rows, op, "Y and X");
    g.A = (const signed char *)work->ptr;
    g.sa = (const float *)((const char *)work->ptr + codes);
    {
        /* One launch where coding its tokens costs a block little: against
         * two, us a call, 1 x 1024 x 4096 4.9, 7.4; 32 x 256 x 256 4.9, 7.3;
         * 16 x 1024 x 1024 7.2, 7.4; 400 x 256 x 512 (two blocks a CU) 8.6, 7.3;
         * 16 x 2048 x 1024 9.9, 8.2; a few tokens 4 x 8192 x 1024 14.3, 24.7. */
        int n = 0;
        const int form = q8_choose(rows, out, (int)g.pitch, o->ocl->cu_count, n);
        const int tokens = min(rows, form == Q8_SKINNY2 ? 32 : 16);
        const long long blocks = (out + 15) / 16 * ((rows + tokens - 1LL) / tokens);

        if (form >= Q8_SKINNY2 && tokens * (g.pitch + 16) <= Q8_FUSED_BYTES &&
            (rows <= 4 || (tokens * in <= 16384 && blocks <= o->ocl->cu_count))) {
            prof_scope ps(o->ocl, "linear_q8");
            if (form == Q8_SKINNY2)
                q8_skinny_launch<2, true>(g, cfptr(X) + xoff, ldx, in, stream_of(o->ocl));
            else
                q8_skinny_launch<1, true>(g, cfptr(X) + xoff, ldx, in, stream_of(o->ocl));
            launch_check("linear_q8");
            return;
        }
    }
    quant_rows(o, rows, in, cfptr(X) + xoff, ldx, work->ptr, (float *)g.sa);
    q8_product(o, g);
    ICOREG_API_END
}
