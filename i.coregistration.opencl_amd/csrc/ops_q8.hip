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

#include "act.h"
#include "common.h"
#include "gemm_dev.h"
#include "ops.h"
#include "q8.h"

using namespace icoreg;

#define Q8_MAX_IN (1 << 17)

typedef int q8_i4 __attribute__((ext_vector_type(4)));
typedef int q8_i16 __attribute__((ext_vector_type(16)));

/* ---- codes of rows --------------------------------------------------------- */

/* One wave a row, four channels a lane and step: the largest magnitude, then
 * the codes. Rows of up to 256 NV channels stay in registers between the two;
 * longer ones (NV = 0) are read again. */
template <int NV, bool VEC>
__global__ void __launch_bounds__(256)
    quant_rows_kernel(const float *__restrict__ X, long long ldx, long rows, int C,
                      unsigned *__restrict__ Q, float *__restrict__ S)
{
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = NV ? NV : (C + 255) / 256;
    const long long words = q8_pitch(C) / 4;
    float v[NV ? NV : 1][4];
    unsigned mag = 0;

    if (row >= rows)
        return;
    X += row * ldx;
    Q += row * words;
    auto load = [&](int k, float (&x)[4]) {
        const int c = 256 * k + 4 * lane;

        if (VEC) {
            const float4 a = *(const float4 *)(X + min(c, C - 4));
            const bool in = c < C;

            x[0] = in ? a.x : 0.0f;
            x[1] = in ? a.y : 0.0f;
            x[2] = in ? a.z : 0.0f;
            x[3] = in ? a.w : 0.0f;
        }
        else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] = c + j < C ? X[c + j] : 0.0f;
        }
    };
#pragma unroll NV ? NV : 1
    for (int k = 0; k < steps; k++) {
        float(&x)[4] = v[NV ? k : 0];

        load(k, x);
#pragma unroll
        for (int j = 0; j < 4; j++)
            mag = max(mag, q8_mag(x[j]));
    }
    const q8_scale q = q8_scale_of(wave_umax(mag));

    if (lane == 0)
        S[row] = q.s;
#pragma unroll NV ? NV : 1
    for (int k = 0; k < steps; k++) {
        const int w = 64 * k + lane;
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
    const bool vec = ((uintptr_t)X & 15) == 0 && ldx % 4 == 0 && C % 4 == 0;
    const dim3 grid((unsigned)((rows + 3) / 4)), block(256);
    const hipStream_t s = stream_of(o->ocl);

    prof_scope ps(o->ocl, "quant_rows");
#define QUANT_LAUNCH(NV_, VEC_)                                                          \
    hipLaunchKernelGGL((quant_rows_kernel<NV_, VEC_>), grid, block, 0, s, X, ldx, rows, C, \
                       (unsigned *)Q, S)
    if (!vec)
        QUANT_LAUNCH(0, false);
    else if (C <= 256)
        QUANT_LAUNCH(1, true);
    else if (C <= 1024)
        QUANT_LAUNCH(4, true);
    else if (C <= 4096)
        QUANT_LAUNCH(16, true);
    else
        QUANT_LAUNCH(0, true);
#undef QUANT_LAUNCH
    launch_check("quant_rows");
}

extern "C" int ops_q8_pitch(int C)
{
    return C < 1 || C > 0x7fffffff - Q8_PITCH ? 0 : (int)q8_pitch(C);
}

extern "C" void ops_quant_rows(struct ops *o, long rows, int C, cl_mem X, long xoff, int ldx,
                               cl_mem Q, cl_mem S)
{
    ICOREG_API_BEGIN
    const char *op = "ops_quant_rows";

    if (rows < 0 || rows > 0x7fffffffL || C < 1 || C > 0x7fffffff - Q8_PITCH || ldx < C || xoff < 0)
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

/* act(sa sb sum + bias) + r, the sum converted once. */
__device__ __forceinline__ float q8_out(const q8_args &g, int sum, float sa, float sb, float b,
                                        float r)
{
#pragma clang fp contract(off)
    const float v = icoreg_act((sa * sb) * (float)sum + b, g.act, g.slope);

    return g.R ? v + r : v;
}

/* Blocks of BM x BN outputs, WM x WN waves, 128 bytes of both panels a step
 * by LDS DMA, two steps in flight, one barrier a step; rows hold their eight
 * 16-byte chunks in the order chunk ^ (row / 2 % 8), which spreads the rows
 * that a matrix instruction reads over the banks. v_mfma_i32_32x32x32_i8: lane
 * half h takes bytes 16 h .. of 32 of row lane % 32 of either operand. Columns
 * past a row's pitch, rows past M and N are outside the panels' windows and
 * read as zeros. */
template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) q8_gemm(const q8_args g)
{
    constexpr int NT = 64 * WM * WN, BK = 128;
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int ASZ = BM * BK, BSZ = BN * BK;
    constexpr int AL = ASZ / 16 / NT, BL = BSZ / 16 / NT;
    static_assert(AL >= 1 && BL >= 1 && ASZ % (16 * NT) == 0 && BSZ % (16 * NT) == 0, "tile shape");
    __shared__ __align__(16) signed char lds[2 * (ASZ + BSZ)];
    signed char *const A0 = lds, *const B0 = lds + ASZ, *const A1 = lds + ASZ + BSZ,
                      *const B1 = lds + 2 * ASZ + BSZ;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, h = lane >> 5, r32 = lane & 31;
    const int tiles_n = (g.N + BN - 1) / BN;
    const int tile = xcd_tile(blockIdx.x, gridDim.x);
    const int m0 = (tile / tiles_n) * BM, n0 = (tile % tiles_n) * BN;
    const int pitch = (int)g.pitch;
    const signed char *A = g.A + m0 * g.pitch, *B = g.B + n0 * g.pitch;
    const long long abytes = min(BM, g.M - m0) * g.pitch, bbytes = min(BN, g.N - n0) * g.pitch;
    int aoff[AL], boff[BL], ak[AL], bk[BL];
    q8_i16 acc[TM][TN];

#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                acc[i][j][r] = 0;
#pragma unroll
    for (int q = 0; q < AL; q++) {
        const int sl = tid + NT * q, row = sl / 8;

        ak[q] = 16 * ((sl % 8) ^ ((row >> 1) & 7));
        aoff[q] = row * pitch + ak[q];
    }
#pragma unroll
    for (int q = 0; q < BL; q++) {
        const int sl = tid + NT * q, row = sl / 8;

        bk[q] = 16 * ((sl % 8) ^ ((row >> 1) & 7));
        boff[q] = row * pitch + bk[q];
    }
    auto load = [&](int k0, signed char *__restrict__ As, signed char *__restrict__ Bs) {
        const __amdgpu_buffer_rsrc_t ra = gemm_rsrc((const float *)A, abytes);
        const __amdgpu_buffer_rsrc_t rb = gemm_rsrc((const float *)B, bbytes);

#pragma unroll
        for (int q = 0; q < AL; q++) {
            const unsigned off = k0 + ak[q] < pitch ? (unsigned)(aoff[q] + k0) : GEMM_OOB;

            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                ra, (__attribute__((address_space(3))) void *)(As + 16 * (NT * q + 64 * wave)), 16,
                (int)off, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < BL; q++) {
            const unsigned off = k0 + bk[q] < pitch ? (unsigned)(boff[q] + k0) : GEMM_OOB;

            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rb, (__attribute__((address_space(3))) void *)(Bs + 16 * (NT * q + 64 * wave)), 16,
                (int)off, 0, 0, 0);
        }
    };
    auto compute = [&](const signed char *__restrict__ As, const signed char *__restrict__ Bs) {
#pragma unroll
        for (int kk = 0; kk < BK / 32; kk++) {
            q8_i4 a[TM], b[TN];

#pragma unroll
            for (int i = 0; i < TM; i++) {
                const int row = wm * (BM / WM) + i * 32 + r32;

                a[i] = *(const q8_i4 *)(As + row * BK + 16 * ((2 * kk + h) ^ ((row >> 1) & 7)));
            }
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const int row = wn * (BN / WN) + j * 32 + r32;

                b[j] = *(const q8_i4 *)(Bs + row * BK + 16 * ((2 * kk + h) ^ ((row >> 1) & 7)));
            }
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++)
                    acc[i][j] =
                        __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    };
    const int nk = (pitch + BK - 1) / BK;
    auto step = [&](int kt, const signed char *__restrict__ Ac, const signed char *__restrict__ Bc,
                    signed char *__restrict__ An, signed char *__restrict__ Bn) {
        if (kt + 1 < nk)
            load((kt + 1) * BK, An, Bn);
        compute(Ac, Bc);
        __builtin_amdgcn_s_waitcnt(GEMM_WAIT_VM0);
        __syncthreads();
    };

    load(0, A0, B0);
    __builtin_amdgcn_s_waitcnt(GEMM_WAIT_VM0);
    __syncthreads();
    for (int kt = 0; kt < nk; kt += 2) {
        step(kt, A0, B0, A1, B1);
        if (kt + 1 < nk)
            step(kt + 1, A1, B1, A0, B0);
    }

    /* Register r of a 32 x 32 tile: row (r / 4) * 8 + 4 h + r % 4, column
     * lane % 32. Loads before stores: C may be R. */
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int n = n0 + wn * (BN / WN) + j * 32 + r32;
        const float sb = g.sb[min(n, g.N - 1)];
        const float b = g.bias ? g.bias[min(n, g.N - 1)] : 0.0f;

#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int ri = m0 + wm * (BM / WM) + i * 32 + 4 * h;
            float sa[16], x[16];

#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int m = min(ri + (r >> 2) * 8 + (r & 3), g.M - 1);

                sa[r] = g.sa[m];
                x[r] = g.R && n < g.N ? g.R[m * g.ldc + n] : 0.0f;
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int m = ri + (r >> 2) * 8 + (r & 3);

                if (m < g.M && n < g.N)
                    g.C[m * g.ldc + n] = q8_out(g, acc[i][j][r], sa[r], sb, b, x[r]);
            }
        }
    }
}

template <int BM, int BN, int WM, int WN> static void q8_launch(const q8_args &g, hipStream_t s)
{
    const long long tiles = (long long)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);

    hipLaunchKernelGGL((q8_gemm<BM, BN, WM, WN>), dim3((unsigned)count32(tiles, "q8 tiles")),
                       dim3(64 * WM * WN), 0, s, g);
}

static void q8_product(struct ops *o, const q8_args &g)
{
    const hipStream_t s = stream_of(o->ocl);
    const long long cus = o->ocl->cu_count;
    auto tiles = [&](int bm, int bn) {
        return (long long)((g.M + bm - 1) / bm) * ((g.N + bn - 1) / bn);
    };

    prof_scope ps(o->ocl, "gemm_q8");
    if (tiles(256, 256) >= 2 * cus)
        q8_launch<256, 256, 2, 4>(g, s);
    else if (tiles(128, 128) >= cus / 2)
        q8_launch<128, 128, 2, 2>(g, s);
    else
        q8_launch<64, 64, 2, 2>(g, s);
    launch_check("gemm_q8");
}

/* The checks of both calls and the arguments of the product, its first
 * operand left out. */
static q8_args q8_make(const char *op, int rows, int in, int out, cl_mem WQ, cl_mem WS, cl_mem b,
                       cl_mem R, long roff, cl_mem Y, long yoff, int ldy, int act, float slope)
{
    q8_args g = {};
    const long long span = (long long)(rows - 1) * ldy + out;

    if (rows < 0 || in < 1 || in > Q8_MAX_IN || out < 0 || ldy < out || yoff < 0 || roff < 0)
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
    if (R && cfptr(R) + roff != cfptr(Y) + yoff)
        need_apart(Y, yoff * 4, span * 4, R, roff * 4, span * 4, op, "Y and R (unless the same)");
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
    g.A = (const signed char *)XQ->ptr;
    g.sa = cfptr(XS);
    q8_product(o, g);
    ICOREG_API_END
}

/* Work of ops_linear_q8: the tokens' codes, then their scales. */
extern "C" size_t ops_linear_q8_work_bytes(int rows, int in)
{
    if (rows < 1 || in < 1 || in > Q8_MAX_IN)
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
    const long long xbytes = ((rows - 1) * (long long)ldx + in) * 4;

    if (ldx < in || xoff < 0)
        icoreg_fatal("%s: invalid sizes in=%d ldx=%d", op, in, ldx);
    if (rows == 0 || out == 0)
        return;
    need_bytes(X, xoff * 4, xbytes, op, "X");
    need_bytes(work, 0, (long long)ops_linear_q8_work_bytes(rows, in), op, "work");
    need_aligned(work, 16, op, "work");
    need_apart(X, xoff * 4, xbytes, work, 0, codes + rows * 4LL, op, "X and work");
    need_apart(Y, yoff * 4, ybytes, work, 0, codes + rows * 4LL, op, "Y and work");
    need_apart(Y, yoff * 4, ybytes, X, xoff * 4, xbytes, op, "Y and X");
    g.A = (const signed char *)work->ptr;
    g.sa = (const float *)((const char *)work->ptr + codes);
    quant_rows(o, rows, in, cfptr(X) + xoff, ldx, work->ptr, (float *)g.sa);
    q8_product(o, g);
    ICOREG_API_END
}
