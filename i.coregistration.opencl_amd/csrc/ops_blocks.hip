/* SPDX-License-Identifier: Unlicense */

/* Attention over blocks of keys that a cheap score selects for each query and
 * head.
 *
 * Index: a block of bs keys is represented by the mean of its kept keys, a
 * 64-bit sum rounded to float32, in 8-bit codes with a scale (q8.h); scale -1
 * marks a block that keeps no key.
 *
 * Selection: the score of a query's codes cq with a block's (c, s) is the
 * float32 product s (cq . c). The sum is a whole number and exact, so that
 * the selection is the same in every order of summation; the query's own
 * scale would not change an order and is left out. The `top` largest are
 * listed, largest first, ties to the lower block, NaN above all numbers.
 *
 * Attention: softmax(scale q K^T) V over the kept keys of the listed blocks,
 * in float32 as ops_attention does it. A listed block is a unit of at most 64
 * keys (two for blocks of 128); units are computed on their own, maximum,
 * sum and unnormalised output to the work buffer, and merged row by row in
 * the order of the list, so that results do not depend on the schedule. */

#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm_dev.h"
#include "load4.h"
#include "ops.h"
#include "q8.h"
#include "split.h"

using namespace icoreg;

#define BLK_MAX_TOP 64
#define BLK_LOG2E 1.4426950408889634f
#define BLK_QUP 0x1p32f /* scale of the queries split into bf16 parts */

/* Keys are counted in int, a block past the last one included. */
#define BLK_MAX_KEYS 0x7fffff00

static int blk_sub(int bs) { return bs > 64 ? bs / 64 : 1; }

static bool blk_size_ok(int bs) { return bs == 16 || bs == 32 || bs == 64 || bs == 128; }

/* ---- the index of the blocks -------------------------------------------------- */

/* A block of threads makes the code of one key block and head: L lanes of
 * four channels a key, 256 / L keys at a time, sums in 64 bits (float32 sums
 * would depend on the order, and with them the codes next to a border). 16380
 * keys of 2 heads of 64, 8.4 MB: 7.3 us; one block 5.4: loads, two barriers and
 * the rounding behind each other. */
template <int L>
__global__ void __launch_bounds__(256)
    block_index_kernel(const float *__restrict__ K, long long ldk, int Nk, int nhk, int d, int bs,
                       const unsigned char *__restrict__ kmask, int b0,
                       signed char *__restrict__ KC, float *__restrict__ KS)
{
    constexpr int G = 256 / L; /* keys at a time */
    constexpr int U = L / 4;   /* times that: 64 keys on their way at once */
    __shared__ double part[G][4 * L];
    __shared__ int kept[G];
    __shared__ unsigned top;
    const int tid = threadIdx.x, g = tid / L, c = 4 * (tid % L);
    const int b = b0 + blockIdx.x / nhk, h = blockIdx.x % nhk;
    const int k0 = b * bs, k1 = min(Nk, k0 + bs);
    const long long pitch = q8_pitch(d);
    double s[4] = {0, 0, 0, 0};
    int n = 0;

    if (tid == 0)
        top = 0;
    for (int k = k0 + g; k < k1; k += U * G) {
        float x[U][4];
        bool in[U];

#pragma unroll
        for (int u = 0; u < U; u++) {
            const int kk = min(k + u * G, k1 - 1);

            load4_row(K + kk * ldk + (long long)h * d, c, d, x[u]);
            in[u] = k + u * G < k1 && (!kmask || kmask[kk]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            n += in[u];
#pragma unroll
            for (int j = 0; j < 4; j++)
                s[j] += in[u] ? x[u][j] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        part[g][c + j] = s[j];
    if (tid % L == 0)
        kept[g] = n;
    __syncthreads();
    float m = 0.0f;

    n = 0;
    for (int i = 0; i < G; i++)
        n += kept[i];
    if (tid < d) {
        double t = 0;

        for (int i = 0; i < G; i++)
            t += part[i][tid];
        m = n ? (float)(t / n) : 0.0f;
        atomicMax(&top, q8_mag(m));
    }
    __syncthreads();
    const q8_scale q = q8_scale_of(top);
    const long long at = (long long)b * nhk + h;

    if (tid < pitch)
        KC[at * pitch + tid] = (signed char)(tid < d ? q8_code(m, q.r) : 0);
    if (tid == 0)
        KS[at] = n ? q.s : -1.0f;
}

extern "C" int ops_key_blocks(int Nk, int bs)
{
    return Nk < 1 || Nk > BLK_MAX_KEYS || !blk_size_ok(bs) ? 0 : (Nk - 1) / bs + 1;
}

extern "C" void ops_block_index(struct ops *o, struct opnd K, int Nk, int nhk, int d, int bs,
                                cl_mem kmask, int b0, int nb, cl_mem KC, cl_mem KS)
{
    ICOREG_API_BEGIN
    const char *op = "ops_block_index";
    const int nblk = ops_key_blocks(Nk, bs);

    if (!blk_size_ok(bs))
        icoreg_fatal("%s: block size %d is not 16, 32, 64 or 128", op, bs);
    if (d < 1 || d > OPS_MAX_HEAD_DIM)
        icoreg_fatal("%s: head dimension %d is not 1 .. %d", op, d, OPS_MAX_HEAD_DIM);
    if (Nk < 0 || Nk > BLK_MAX_KEYS || nhk < 1 || b0 < 0 || nb < 0 ||
        (long long)b0 + nb > nblk || K.off < 0 || K.ld < (long long)nhk * d)
        icoreg_fatal("%s: invalid sizes Nk=%d nhk=%d d=%d ld=%d, blocks %d + %d of %d", op, Nk, nhk,
                     d, K.ld, b0, nb, nblk);
    if (nb == 0)
        return;
    {
        const long long cells = (long long)(b0 + nb) * nhk;

        need_floats(K.buf, K.off, (Nk - 1) * (long long)K.ld + (long long)nhk * d, op, "K");
        if (kmask)
            need_bytes(kmask, 0, Nk, op, "kmask");
        need_bytes(KC, 0, cells * q8_pitch(d), op, "KC");
        need_aligned(KC, 16, op, "KC");
        need_floats(KS, 0, cells, op, "KS");
        const long long kbytes = ((Nk - 1) * (long long)K.ld + (long long)nhk * d) * 4;

        need_apart(KC, 0, cells * q8_pitch(d), K.buf, K.off * 4, kbytes, op, "KC and K");
        need_apart(KS, 0, cells * 4, K.buf, K.off * 4, kbytes, op, "KS and K");
        need_apart(KC, 0, cells * q8_pitch(d), KS, 0, cells * 4, op, "KC and KS");
        need_apart(KC, 0, cells * q8_pitch(d), kmask, 0, Nk, op, "KC and kmask");
        need_apart(KS, 0, cells * 4, kmask, 0, Nk, op, "KS and kmask");
    }
    const unsigned grid = grid_of((long long)nb * nhk, 256, "block index");

    prof_scope ps(o->ocl, "block_index");
#define INDEX_LAUNCH(L_)                                                                       \
    hipLaunchKernelGGL((block_index_kernel<L_>), dim3(grid), dim3(256), 0, stream_of(o->ocl),  \
                       cfptr(K.buf) + K.off, (long long)K.ld, Nk, nhk, d, bs,                  \
                       kmask ? (const unsigned char *)kmask->ptr : nullptr, b0,                \
                       (signed char *)KC->ptr, fptr(KS))
    if (d <= 32)
        INDEX_LAUNCH(8);
    else if (d <= 64)
        INDEX_LAUNCH(16);
    else
        INDEX_LAUNCH(32);
#undef INDEX_LAUNCH
    launch_check("block_index");
    ICOREG_API_END
}

/* ---- the selection -------------------------------------------------------------- */

/* Scores as whole numbers in the same order: NaN above infinity, no block
 * (SEL_NONE) below minus infinity. */
#define SEL_NONE ((int)0x80000000)
#define SEL_NAN 0x7ffffffe

__device__ __forceinline__ int sel_key(float s)
{
    const int b = __builtin_bit_cast(int, s + 0.0f); /* -0 is 0 */

    return s != s ? SEL_NAN : b ^ ((b >> 31) & 0x7fffffff);
}

__device__ __forceinline__ float sel_value(int k)
{
    return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff));
}

/* Wave maximum or minimum of whole numbers, all lanes active. */
template <class F> __device__ __forceinline__ int wave_fold(int v, F f)
{
    const int ctl[4] = {0xB1, 0x4E, 0x141, 0x140};

#pragma unroll
    for (int c = 0; c < 4; c++)
        v = f(v, dpp_i(v, ctl[c]));
    return f(f(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             f(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

/* The top `top` of a wave's candidates, slot j of lane l before slot j of
 * lane l + 1 before slot j + 1, equal keys in that order: returned sorted,
 * candidate i in lane i of (key, idx), SEL_NONE behind the last. A threshold
 * that between top and top + 8 of them reach is found (or 64, where equal ones
 * allow no other), and those are ranked; it starts at the smallest of at least
 * top maxima of groups of lanes, a few halvings away. list: 2 x 64 words of LDS of this wave. */
template <int N>
__device__ __forceinline__ void sel_top(const int (&k)[N], const int (&i)[N], int top, int *list,
                                        int &key, int &idx)
{
    const int lane = threadIdx.x & 63;
    auto larger = [](int x, int y) { return max(x, y); };
    auto smaller = [](int x, int y) { return min(x, y); };
    auto count = [&](int t) {
        int n = 0;

#pragma unroll
        for (int j = 0; j < N; j++)
            n += __popcll(__ballot(k[j] >= t));
        return n;
    };
    int most = k[0];

#pragma unroll
    for (int j = 1; j < N; j++)
        most = max(most, k[j]);
    /* 64, 32 or 16 groups. */
    if (top <= 32)
        most = max(most, dpp_i(most, 0xB1));
    if (top <= 16)
        most = max(most, dpp_i(most, 0x4E));
    /* lo: at least top candidates (or all there are), hi: fewer; halved by
     * value first, which parts scores of one size in a few steps, by bits where
     * that stalls. */
    int lo = wave_fold(most, smaller), hi = wave_fold(most, larger) + 1;

    if (lo == SEL_NONE) {
        /* Groups of none: the smallest there is. */
        lo = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < N; j++)
            lo = k[j] == SEL_NONE ? lo : min(lo, k[j]);
        lo = wave_fold(lo, smaller);
    }
    int nlo = count(lo), nhi = 0;

    const int most_wanted = min(64, top + 8);

    for (int step = 0; nlo > most_wanted && (unsigned)hi - (unsigned)lo > 1; step++) {
        int mid = (int)((unsigned)lo + ((unsigned)hi - (unsigned)lo) / 2);

        if (step < 16) {
            const float a = fmaxf(sel_value(lo), -3e38f), z = fminf(sel_value(hi), 3e38f);
            const int v = sel_key(0.5f * a + 0.5f * z);

            if (v > lo && v < hi)
                mid = v;
        }
        const int n = count(mid);

        if (n >= top) {
            lo = mid;
            nlo = n;
        }
        else {
            hi = mid;
            nhi = n;
        }
    }
    if (nlo <= 64)
        nhi = nlo, hi = lo;
    /* Every candidate from hi on, and the first of those equal to lo. */
    int at = 0, rest = nlo <= 64 ? 0 : top - nhi;

    key = SEL_NONE;
    idx = -1;
    list[lane] = SEL_NONE;
    list[64 + lane] = -1;
#pragma unroll
    for (int j = 0; j < N; j++) {
        const unsigned long long eq = __ballot(k[j] == lo && k[j] < hi);
        const unsigned long long below = (1ull << lane) - 1;
        const bool in = k[j] >= hi || (k[j] == lo && k[j] < hi && __popcll(eq & below) < rest);
        const unsigned long long all = __ballot(in);

        if (in) {
            const int p = at + __popcll(all & below);

            list[p] = k[j];
            list[64 + p] = i[j];
        }
        at += __popcll(all);
        rest -= min(rest, (int)__popcll(eq));
    }
    __builtin_amdgcn_wave_barrier();
    const int mine = list[lane], who = list[64 + lane];
    int rank = 0;

    /* Four at a time; behind the last there is SEL_NONE. */
    for (int j0 = 0; j0 < at; j0 += 4) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int other = __builtin_amdgcn_readlane(mine, j0 + e);

            rank += other + (j0 + e < lane) > mine;
        }
    }
    __builtin_amdgcn_wave_barrier();
    if (lane < at) {
        list[rank] = mine;
        list[64 + rank] = who;
    }
    __builtin_amdgcn_wave_barrier();
    key = lane < top ? list[lane] : SEL_NONE;
    idx = list[64 + lane];
    __builtin_amdgcn_wave_barrier();
}

/* What a selection reads, and where it writes. */
struct sel_args {
    const float *Q;
    const signed char *KC;
    const float *KS;
    int *SEL;
    long long ldq;
    int Nq, nh, nhk, d, nblk, top;
};

/* A wave selects the best of the blocks b0 .. b1 - 1 for one query and head,
 * 64 SLOTS at a time, the best so far kept beside the next ones. The PL = 4 or 8
 * lanes of a code row read 16 bytes each, neighbours of one line (a row a lane
 * fetches every line PL times: a step from 25 to 20 us for 16 rows of 2047
 * blocks of 128 channels, 10.4 now: the codes' way from memory, then about
 * fifteen counts of the threshold and the ranks, twice), and add their sums;
 * lane l keeps the score of block l of 64. Sorted results in the lanes, as
 * sel_top leaves them. codes, list: 128 bytes and words of LDS of this wave. */
template <int PL>
__device__ __forceinline__ void sel_row(const sel_args &a, int query, int h, int b0, int b1,
                                        unsigned char *codes, int *list, int &key, int &idx)
{
    constexpr int SLOTS = 16 / PL;
    const int lane = threadIdx.x & 63, kvh = h / (a.nh / a.nhk), c = 2 * lane;
    const float *q = a.Q + query * a.ldq + (long long)h * a.d;
    const float x = c < a.d ? q[c] : 0.0f, y = c + 1 < a.d ? q[c + 1] : 0.0f;
    const q8_scale s = q8_scale_of(wave_umax(max(q8_mag(x), q8_mag(y))));
    const bool bad = s.s != s.s; /* not finite: NaN everywhere */
    const int part = lane % PL, group = lane / PL * PL;

    codes[c] = (unsigned char)q8_code(x, s.r);
    codes[c + 1] = (unsigned char)q8_code(y, s.r);
    __builtin_amdgcn_wave_barrier();
    const uint4 qc = ((const uint4 *)codes)[part];

    key = SEL_NONE;
    idx = -1;
    for (; b0 < b1; b0 += 64 * SLOTS) {
        int k[SLOTS + 1], i[SLOTS + 1];
        uint4 w[SLOTS][PL];
        float ks[SLOTS];

        k[0] = key;
        i[0] = idx;
#pragma unroll
        for (int j = 0; j < SLOTS; j++) {
            ks[j] = a.KS[(long long)min(b0 + 64 * j + lane, b1 - 1) * a.nhk + kvh];
#pragma unroll
            for (int e = 0; e < PL; e++) {
                const long long b = min(b0 + 64 * j + group + e, b1 - 1);

                w[j][e] = ((const uint4 *)a.KC)[(b * a.nhk + kvh) * PL + part];
            }
        }
#pragma unroll
        for (int j = 0; j < SLOTS; j++) {
            const int b = b0 + 64 * j + lane;
            int mine = 0;

#pragma unroll
            for (int e = 0; e < PL; e++) {
                int dot = __builtin_amdgcn_sdot4((int)w[j][e].x, (int)qc.x, 0, false);

                dot = __builtin_amdgcn_sdot4((int)w[j][e].y, (int)qc.y, dot, false);
                dot = __builtin_amdgcn_sdot4((int)w[j][e].z, (int)qc.z, dot, false);
                dot = __builtin_amdgcn_sdot4((int)w[j][e].w, (int)qc.w, dot, false);
                dot += dpp_i(dot, 0xB1);
                dot += dpp_i(dot, 0x4E);
                if (PL == 8)
                    dot += dpp_i(dot, 0x141);
                mine = part == e ? dot : mine;
            }
            i[j + 1] = b;
            k[j + 1] = b >= b1 || ks[j] < 0.0f ? SEL_NONE
                                               : bad ? SEL_NAN : sel_key(ks[j] * (float)mine);
        }
        sel_top(k, i, a.top, list, key, idx);
    }
}

/* A block of W waves for one query and head, each on its share of the key
 * blocks; wave 0 selects among the waves' best. */
template <int W, int PL>
__global__ void __launch_bounds__(64 * W) block_select_kernel(const sel_args a)
{
    __shared__ int lists[W][128];
    __shared__ __align__(16) unsigned char codes[W][128];
    __shared__ int best[W > 1 ? W * 128 : 1];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x, share = ((a.nblk + W - 1) / W + 63) / 64 * 64;
    int key, idx;

    sel_row<PL>(a, row / a.nh, row % a.nh, wave * share, min(a.nblk, (wave + 1) * share),
                codes[wave], lists[wave], key, idx);
    if constexpr (W > 1) {
        if (lane < a.top) {
            best[wave * a.top + lane] = key;
            best[W * 64 + wave * a.top + lane] = idx;
        }
        __syncthreads();
        if (wave)
            return;
        auto join = [&](auto n) {
            constexpr int N = decltype(n)::value;
            int k[N], i[N];

#pragma unroll
            for (int w = 0; w < N; w++) {
                const int at = 64 * w + lane;

                k[w] = at < W * a.top ? best[at] : SEL_NONE;
                i[w] = at < W * a.top ? best[W * 64 + at] : -1;
            }
            sel_top(k, i, a.top, lists[0], key, idx);
        };

        if (a.top <= 16)
            join(std::integral_constant<int, W / 4>());
        else
            join(std::integral_constant<int, W>());
    }
    if (lane < a.top)
        a.SEL[(long long)row * a.top + lane] = key == SEL_NONE ? -1 : idx;
}

/* Many queries on at most 16 T key blocks: a wave takes 16 rows (a query and
 * head each, of one key head; row r of a key head is query r / g, query head r
 * % g of its g). v_mfma_i32_16x16x64_i8 with the blocks' codes as rows and the
 * queries' as columns leaves a row's scores in 4 lanes, 4 T in each, where they
 * stay. The smallest of the maxima of 16 G / 4 groups, at least top of them, is
 * reached by top scores; from there the range is halved until no more than CAP
 * reach the threshold (8 instructions a row and step, where a wave a row
 * takes 16 and more; mostly 2 or 3 steps). Those go to LDS and are ranked
 * against each other, ties by their numbers. A query, scale or score that is
 * not finite, or more equal scores than CAP, sends the wave's rows to sel_row
 * one by one. 65536 rows of 256 blocks 40 us (a wave a row 197), vector
 * instructions in 41 % of it, mostly the counts; the products 2 %. */
#define SEL_TW 4 /* waves */

template <int T, int KCH, int CAP>
__global__ void __launch_bounds__(64 * SEL_TW, T > 16 ? 2 : T > 8 ? 3 : 4)
    block_select_tile(const sel_args a)
{
    constexpr int OWN = CAP / 4, G = CAP > 24 ? 8 : 4; /* groups of a lane */
    typedef int i4 __attribute__((ext_vector_type(4)));
    typedef unsigned long long u64;
    __shared__ __align__(16) float scale[16 * T], none[16 * T];
    __shared__ u64 cand[SEL_TW][16][CAP + 1];
    __shared__ int lists[SEL_TW][128];
    __shared__ __align__(16) unsigned char codes[SEL_TW][128];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, part = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.y, g = a.nh / a.nhk, rows = a.Nq * g;
    const int r0 = (blockIdx.x * SEL_TW + wave) * 16, r = min(r0 + col, rows - 1);
    const int query = r / g, h = kvh * g + r % g;
    const long long pitch = 64 * KCH, row = (long long)query * a.nh + h;
    i4 q[KCH];
    bool odd = false;

    /* Scores s (cq . c) + 0, minus infinity for what is no block. */
    for (int b = tid; b < 16 * T; b += 64 * SEL_TW) {
        const float k = b < a.nblk ? a.KS[(long long)b * a.nhk + kvh] : -1.0f;

        scale[b] = fmaxf(k, 0.0f);
        none[b] = k < 0.0f ? -INFINITY : 0.0f;
        odd = odd || !(k < 1e32f);
    }
    odd = __syncthreads_or(odd);
    if (r0 >= rows)
        return;
    /* The query's codes: channels 64 c + 16 part .. + 15 in this lane. */
    {
        const float *p = a.Q + query * a.ldq + (long long)h * a.d;
        float x[KCH][4][4];
        unsigned top = 0;

#pragma unroll
        for (int c = 0; c < KCH; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                load4_row(p, 64 * c + 16 * part + 4 * e, a.d, x[c][e]);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    top = max(top, q8_mag(x[c][e][j]));
            }
        top = max(top, (unsigned)__shfl_xor((int)top, 16, 64));
        top = max(top, (unsigned)__shfl_xor((int)top, 32, 64));
        const q8_scale s = q8_scale_of(top);

        odd = odd || s.s != s.s;
#pragma unroll
        for (int c = 0; c < KCH; c++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                q[c][e] = (int)q8_code4(x[c][e][0], x[c][e][1], x[c][e][2], x[c][e][3], s.r);
    }
    /* Register 4 t + e: block 16 t + 4 part + e. */
    float s[4 * T], most[G];

#pragma unroll
    for (int e = 0; e < G; e++)
        most[e] = -INFINITY;
#pragma unroll
    for (int t0 = 0; t0 < T; t0 += 4) {
        i4 w[4][KCH];

        /* Four tiles' codes on their way at once, and no more: the scores
         * fill the registers. */
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < KCH; c++) {
                const int b = min(16 * (t0 + t) + col, a.nblk - 1);

                w[t][c] = *(const i4 *)(a.KC + ((long long)b * a.nhk + kvh) * pitch + 64 * c +
                                        16 * part);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int at = 16 * (t0 + t) + 4 * part;
            const float4 k = *(const float4 *)(scale + at), n = *(const float4 *)(none + at);
            const float kk[4] = {k.x, k.y, k.z, k.w}, nn[4] = {n.x, n.y, n.z, n.w};
            i4 dot = {0, 0, 0, 0};

#pragma unroll
            for (int c = 0; c < KCH; c++)
                dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t][c], q[c], dot, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = 4 * (t0 + t) + e;

                s[i] = fmaf((float)dot[e], kk[e], nn[e]);
                most[i % G] = fmaxf(most[i % G], s[i]);
            }
        }
    }
    auto over4 = [](float v, auto f) {
        v = f(v, __shfl_xor(v, 16, 64));
        return f(v, __shfl_xor(v, 32, 64));
    };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto smaller = [](float x, float y) { return fminf(x, y); };
    auto count = [&](float v) {
        int n = 0;

#pragma unroll
        for (int e = 0; e < 4 * T; e++)
            n += s[e] >= v;
        n += __shfl_xor(n, 16, 64);
        return n + __shfl_xor(n, 32, 64);
    };
    float hi, lo;

    /* 4, 8, 16 or 32 groups a row. */
#pragma unroll
    for (int n = G / 2; n >= 1; n /= 2)
        if (a.top <= 4 * n) {
#pragma unroll
            for (int e = 0; e < n; e++)
                most[e] = fmaxf(most[e], most[e + n]);
#pragma unroll
            for (int e = n; e < G; e++)
                most[e] = most[e % n];
        }
    hi = most[0];
    lo = most[0];
#pragma unroll
    for (int e = 1; e < G; e++) {
        hi = fmaxf(hi, most[e]);
        lo = fminf(lo, most[e]);
    }
    hi = over4(hi, larger);
    lo = over4(lo, smaller);
    if (__any(lo == -INFINITY)) {
        /* Groups of no block: the smallest score there is. */
        float v = INFINITY;

#pragma unroll
        for (int e = 0; e < 4 * T; e++)
            v = fminf(v, s[e] == -INFINITY ? INFINITY : s[e]);
        v = over4(v, smaller);
        lo = lo == -INFINITY ? v : lo;
    }
    int n = count(lo);
    bool done = n <= CAP;

    for (int step = 0; step < 48 && !__any(odd) && !__all(done); step++) {
        /* Values of very different size: by bits. */
        const float mid = step == 0   ? 0.75f * lo + 0.25f * hi
                          : step < 12 ? 0.5f * lo + 0.5f * hi
                                      : sel_value((int)(((long long)sel_key(lo) + sel_key(hi)) >> 1));
        const int m = count(mid);

        if (!done) {
            if (m >= a.top) {
                lo = mid;
                done = m <= CAP;
            }
            else
                hi = mid;
        }
    }
    if (__any(odd || !done)) {
        for (int e = 0; e < min(16, rows - r0); e++) {
            const int rr = r0 + e;
            int key, idx;

            sel_row<4 * KCH>(a, rr / g, kvh * g + rr % g, 0, a.nblk, codes[wave], lists[wave], key,
                              idx);
            if (lane < a.top)
                a.SEL[((long long)(rr / g) * a.nh + kvh * g + rr % g) * a.top + lane] =
                    key == SEL_NONE ? -1 : idx;
        }
        return;
    }
    /* The candidates into LDS, lane by lane of the row, as whole numbers that
     * order like the scores and, where those are equal, against their own. */
    n = 0;
#pragma unroll
    for (int e = 0; e < 4 * T; e++)
        n += s[e] >= lo;
    const int n16 = __shfl_xor(n, 16, 64), pair = n + n16, other = __shfl_xor(pair, 32, 64);
    const int total = pair + other;
    u64 *c = cand[wave][col];
    u64 *at = c + (part & 1 ? n16 : 0) + (part & 2 ? other : 0);

#pragma unroll
    for (int e = 0; e < 4 * T; e++)
        if (s[e] >= lo) {
            *at++ = (u64)((unsigned)sel_key(s[e]) ^ 0x80000000u) << 32 |
                    (unsigned)~(16 * (e / 4) + 4 * part + e % 4);
        }
    __builtin_amdgcn_wave_barrier();
    /* Candidate 4 o + part of the row is this lane's. */
    u64 mine[OWN];
    int rank[OWN];

#pragma unroll
    for (int o = 0; o < OWN; o++) {
        mine[o] = 4 * o + part < total ? c[4 * o + part] : ~0ull;
        rank[o] = 0;
    }
    for (int j = 0; __any(j < total); j++) {
        const u64 x = j < total ? c[j] : 0;

#pragma unroll
        for (int o = 0; o < OWN; o++)
            rank[o] += x > mine[o];
    }
    if (r0 + col >= rows)
        return;
    int *out = a.SEL + row * a.top;

#pragma unroll
    for (int o = 0; o < OWN; o++)
        if (4 * o + part < total && rank[o] < a.top)
            out[rank[o]] = ~(int)(unsigned)mine[o];
    for (int e = total + part; e < a.top; e += 4)
        out[e] = -1;
}

/* The kernel of a selection. us, a wave a row and tiles of 16 rows: 4096 rows of
 * 256 blocks 9.7, 17.4; 8192 15.5, 17.0; 16384 26, 16.8; 8192 rows of 500 24.9,
 * 25.4; of 51 blocks, 4096 rows 8.5, 9.4; 8192 14.5, 9.4. One wave and 16 a row: 16
 * rows of 2047 blocks 42, 10.6; 1024 rows 48, 36; 2048 rows 59, 60; of 256 blocks,
 * 16 rows 5.2, 7.3. */
enum { SEL_WAVE, SEL_WAVES, SEL_TILE };

static int sel_choose(long long rows, int nhk, int nblk, int top, int cus)
{
    if (nblk >= 1 && nblk <= 512 && top <= 32 && nhk <= 65535 &&
        rows >= (nblk <= 128 ? 20LL : 36LL) * cus)
        return SEL_TILE;
    return nblk > rows + 256 ? SEL_WAVES : SEL_WAVE;
}

extern "C" int icoreg_select_choice(struct ops *o, int Nq, int nh, int nhk, int nblk, int top)
{
    return sel_choose((long long)Nq * nh, nhk, nblk, top, o->ocl->cu_count);
}

extern "C" size_t ops_block_select_work_bytes(int Nq, int nh, int nblk, int top)
{
    (void)Nq, (void)nh, (void)nblk, (void)top;
    return 0;
}

extern "C" void ops_block_select(struct ops *o, struct opnd Q, int Nq, int nh, int nhk, int d,
                                 cl_mem KC, cl_mem KS, int nblk, int top, cl_mem SEL, cl_mem work)
{
    ICOREG_API_BEGIN
    const char *op = "ops_block_select";

    (void)work;
    if (d < 1 || d > OPS_MAX_HEAD_DIM)
        icoreg_fatal("%s: head dimension %d is not 1 .. %d", op, d, OPS_MAX_HEAD_DIM);
    if (top < 1 || top > BLK_MAX_TOP)
        icoreg_fatal("%s: %d blocks a query are not 1 .. %d", op, top, BLK_MAX_TOP);
    if (Nq < 0 || nh < 1 || nhk < 1 || nh % nhk || nblk < 0 || nblk > BLK_MAX_KEYS / 16 + 1 ||
        Q.off < 0 || Q.ld < (long long)nh * d)
        icoreg_fatal("%s: invalid sizes Nq=%d nh=%d nhk=%d d=%d ld=%d blocks=%d", op, Nq, nh, nhk,
                     d, Q.ld, nblk);
    if (Nq == 0)
        return;
    const long long rows = (long long)Nq * nh;

    need_floats(Q.buf, Q.off, (Nq - 1) * (long long)Q.ld + (long long)nh * d, op, "Q");
    need_bytes(KC, 0, (long long)nblk * nhk * q8_pitch(d), op, "KC");
    need_aligned(KC, 16, op, "KC");
    need_floats(KS, 0, (long long)nblk * nhk, op, "KS");
    need_bytes(SEL, 0, rows * top * 4, op, "SEL");
    need_apart(SEL, 0, rows * top * 4, Q.buf, Q.off * 4,
               ((Nq - 1) * (long long)Q.ld + (long long)nh * d) * 4, op, "SEL and Q");
    need_apart(SEL, 0, rows * top * 4, KC, 0, (long long)nblk * nhk * q8_pitch(d), op, "SEL and KC");
    need_apart(SEL, 0, rows * top * 4, KS, 0, (long long)nblk * nhk * 4, op, "SEL and KS");
    const int form = sel_choose(rows, nhk, nblk, top, o->ocl->cu_count), g = nh / nhk;
    const unsigned grid =
        form == SEL_TILE ? 0 : grid_of(rows, form == SEL_WAVES ? 1024 : 64, "selection rows");
    const unsigned tiles = grid_of(((long long)Nq * g + 16 * SEL_TW - 1) / (16 * SEL_TW), 64 * SEL_TW,
                                   "selection tiles");

    count32(rows + 64, "selection rows"); /* counted past the last */
    const hipStream_t s = stream_of(o->ocl);
    const sel_args a = {cfptr(Q.buf) + Q.off, (const signed char *)(KC ? KC->ptr : nullptr), cfptr(KS),
                        (int *)SEL->ptr, Q.ld, Nq, nh, nhk, d, nblk, top};

    prof_scope ps(o->ocl, "block_select");
#define SELECT_LAUNCH(W_, P_) \
    hipLaunchKernelGGL((block_select_kernel<W_, P_>), dim3(grid), dim3(64 * W_), 0, s, a)
#define SELECT_WIDTH(W_)          \
    do {                          \
        if (d <= 64)              \
            SELECT_LAUNCH(W_, 4); \
        else                      \
            SELECT_LAUNCH(W_, 8); \
    } while (0)
#define TILE_LAUNCH(T_, K_, C_) \
    hipLaunchKernelGGL((block_select_tile<T_, K_, C_>), dim3(tiles, nhk), dim3(64 * SEL_TW), 0, s, a)
#define TILE_WIDTH(T_)             \
    do {                           \
        if (top <= 16 && d <= 64)  \
            TILE_LAUNCH(T_, 1, 24); \
        else if (top <= 16)        \
            TILE_LAUNCH(T_, 2, 24); \
        else if (d <= 64)          \
            TILE_LAUNCH(T_, 1, 40); \
        else                       \
            TILE_LAUNCH(T_, 2, 40); \
    } while (0)
    if (form == SEL_TILE) {
        if (nblk <= 64)
            TILE_WIDTH(4);
        else if (nblk <= 128)
            TILE_WIDTH(8);
        else if (nblk <= 256)
            TILE_WIDTH(16);
        else
            TILE_WIDTH(32);
    }
    else if (form == SEL_WAVES)
        SELECT_WIDTH(16);
    else
        SELECT_WIDTH(1);
#undef TILE_WIDTH
#undef TILE_LAUNCH
#undef SELECT_WIDTH
#undef SELECT_LAUNCH
    launch_check("block_select");
    ICOREG_API_END
}

/* ---- attention over the selected blocks -------------------------------------------- */

struct blk_args {
    const float *Q, *K, *V;
    float *O;
    const int *SEL;
    const unsigned char *kmask;
    long long ldq, ldk, ldv, ldo;
    int q0, Nq; /* the queries of this pass: q0 .. q0 + Nq - 1 */
    int Nk, nh, nhk, d, bs, sub, nblk, top;
    float scale;
    /* Work: units' outputs (DP floats each) and (maximum, sum), rows of this
     * pass x top x sub; bits[head][block][tile of 64 rows]. */
    float *part;
    float2 *ml;
    unsigned long long *bits;
    int tiles, pieces; /* tiles of 64 rows of a kv head; splits of a list */
};

/* Unit `u` of row (query qi, head h): a wave's work in float32. Four lanes a
 * key for the scores, all lanes on channels for the output; sc holds 64
 * words of LDS of this wave. NaN among the kept scores makes the sum NaN. */
__device__ __forceinline__ void blk_unit_f32(const blk_args &a, int qi, int h, int k0, int k1,
                                             float *part, float2 *ml, float *sc)
{
    const int lane = threadIdx.x & 63, d = a.d, kvh = h / (a.nh / a.nhk);
    const float *q = a.Q + qi * a.ldq + (long long)h * d;
    const float *K = a.K + (long long)kvh * d, *V = a.V + (long long)kvh * d;
    const int n = k1 - k0;

    sc[lane] = -INFINITY;
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < n; j += 16) {
        const int key = j + (lane >> 2), part4 = lane & 3;
        const int kk = k0 + min(key, n - 1);
        const float *kp = K + kk * a.ldk;
        float s = 0.0f;

        for (int c = 4 * part4; c < d; c += 16) {
            float x[4], y[4];

            load4_row(kp, c, d, x);
            load4_row(q, c, d, y);
#pragma unroll
            for (int e = 0; e < 4; e++)
                s = fmaf(x[e], y[e], s);
        }
        s += dpp_f(s, 0xB1);
        s += dpp_f(s, 0x4E);
        if (part4 == 0 && key < n && (!a.kmask || a.kmask[kk]))
            sc[key] = s * (a.scale * BLK_LOG2E);
    }
    __builtin_amdgcn_wave_barrier();
    const float s = sc[lane];
    const bool nan = __any(s != s);
    const float m = wave_max_full(s);
    const float p = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - m);
    const float l = nan ? __builtin_nanf("") : wave_sum_full(p);

    sc[lane] = p;
    __builtin_amdgcn_wave_barrier();
    for (int c = lane; c < d; c += 64) {
        float acc = 0.0f;

        for (int j = 0; j < n; j++)
            if (!a.kmask || a.kmask[k0 + j])
                acc = fmaf(sc[j], V[(k0 + j) * a.ldv + c], acc);
        part[c] = nan ? __builtin_nanf("") : acc;
    }
    if (lane == 0)
        *ml = make_float2(nan ? 0.0f : m, l);
    __builtin_amdgcn_wave_barrier();
}

/* Few queries: a block of threads a unit, everything that it reads on its way
 * at once. Scores: 4 lanes a key, DP / 16 times 4 channels each. Output: DP / 4
 * lanes a key, KV keys each, joined in LDS. 256 units of 64 keys of 128 channels,
 * 16.8 MB: 4.7 us, 3.6 TB/s. */
template <int DP> __global__ void __launch_bounds__(256) blk_direct_kernel(const blk_args a)
{
    constexpr int NK = DP / 16, LV = DP / 4, GV = 256 / LV, KV = 64 / GV;
    __shared__ float sc[64];
    __shared__ float out[GV][DP];
    const int tid = threadIdx.x, lane = tid & 63, d = a.d;
    const long long u = blockIdx.x;
    const int sub = (int)(u % a.sub), slot = (int)(u / a.sub % a.top);
    const int row = (int)(u / a.sub / a.top), h = row % a.nh, kvh = h / (a.nh / a.nhk);
    const int *sel = a.SEL + ((long long)a.q0 * a.nh + row) * a.top;
    const int b = sel[slot];
    const bool twice = __any(lane < slot && sel[min(lane, a.top - 1)] == b);
    const int ss = a.bs / a.sub;
    const bool is = b >= 0 && b < a.nblk && !twice && b * a.bs + sub * ss < a.Nk;

    if (!is) {
        if (tid == 0)
            a.ml[u] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const int k0 = b * a.bs + sub * ss, n = min(a.Nk - k0, ss);
    const float *q = a.Q + (a.q0 + row / a.nh) * a.ldq + (long long)h * d;
    const float *K = a.K + k0 * a.ldk + (long long)kvh * d;
    const float *V = a.V + k0 * a.ldv + (long long)kvh * d;
    const int key = tid >> 2, part = tid & 3, cv = 4 * (tid % LV), gv = tid / LV;
    const bool in = key < n && (!a.kmask || a.kmask[k0 + key]);
    float x[NK][4], y[NK][4], v[KV][4];
    bool keep[KV];

#pragma unroll
    for (int i = 0; i < NK; i++) {
        load4_row(K + min(key, n - 1) * a.ldk, 16 * i + 4 * part, d, x[i]);
        load4_row(q, 16 * i + 4 * part, d, y[i]);
    }
#pragma unroll
    for (int i = 0; i < KV; i++) {
        const int k = gv + GV * i;

        load4_row(V + min(k, n - 1) * a.ldv, cv, d, v[i]);
        keep[i] = k < n && (!a.kmask || a.kmask[k0 + k]);
    }
    float s = 0.0f;

#pragma unroll
    for (int i = 0; i < NK; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            s = fmaf(x[i][j], y[i][j], s);
    s += dpp_f(s, 0xB1);
    s += dpp_f(s, 0x4E);
    if (part == 0)
        sc[key] = in ? s * (a.scale * BLK_LOG2E) : -INFINITY;
    __syncthreads();
    /* Every wave for itself: lane k holds key k. */
    const float t = sc[lane];
    const bool nan = __any(t != t);
    const float m = wave_max_full(t);
    const float p = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(t - m);
    const float l = nan ? __builtin_nanf("") : wave_sum_full(p);
    float o[4] = {0, 0, 0, 0};

#pragma unroll
    for (int i = 0; i < KV; i++) {
        const float w = __shfl(p, gv + GV * i, 64);

#pragma unroll
        for (int j = 0; j < 4; j++)
            o[j] = keep[i] ? fmaf(w, v[i][j], o[j]) : o[j];
    }
    *(float4 *)&out[gv][cv] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (tid < DP) {
        float r = 0.0f;

#pragma unroll
        for (int i = 0; i < GV; i++)
            r += out[i][tid];
        a.part[u * DP + tid] = nan ? __builtin_nanf("") : r;
    }
    if (tid == 0)
        a.ml[u] = make_float2(nan ? 0.0f : m, l);
}

/* Many queries, first step: bit r of bits[kvh][b][t] says that row 64 t + r
 * (of the kv head's rows: query-major, its query heads within) lists block
 * b. A wave a tile, eight tiles a block of threads, so that a block's words
 * leave in runs of 64 bytes; entries that are no block or a repeated one get an
 * empty unit. Or of bits in LDS has no order that matters. 65536 rows of 16:
 * 8.6 us. */
#define BLK_TW 8
#define BLK_RANGE 1024 /* key blocks at a time */

__global__ void __launch_bounds__(64 * BLK_TW) blk_bits_kernel(const blk_args a)
{
    __shared__ unsigned long long m[BLK_RANGE][BLK_TW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kvh = blockIdx.y, g = a.nh / a.nhk, t0 = blockIdx.x * BLK_TW;
    const int r = (t0 + wave) * 64 + lane, rows = a.Nq * g;
    const long long row = r < rows ? (long long)(r / g) * a.nh + kvh * g + r % g : 0;
    const int *sel = a.SEL + ((long long)a.q0 * a.nh + row) * a.top;

    for (int c0 = 0; c0 < a.nblk; c0 += BLK_RANGE) {
        const int c1 = min(a.nblk, c0 + BLK_RANGE);

        for (int e = threadIdx.x; e < (c1 - c0) * BLK_TW; e += 64 * BLK_TW)
            (&m[0][0])[e] = 0;
        __syncthreads();
        for (int s0 = 0; s0 < a.top && r < rows; s0 += 8) {
            int v[8];

#pragma unroll
            for (int i = 0; i < 8; i++)
                v[i] = sel[min(s0 + i, a.top - 1)];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int s = s0 + i, b = v[i];
                const bool is = b >= 0 && b < a.nblk;
                bool empty = !is && c0 == 0;

                if (s >= a.top)
                    break;
                if (is && b >= c0 && b < c1)
                    empty = atomicOr(&m[b - c0][wave], 1ull << lane) >> lane & 1;
                if (empty)
                    for (int j = 0; j < a.sub; j++)
                        a.ml[(row * a.top + s) * a.sub + j] = make_float2(-INFINITY, 0.0f);
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < (c1 - c0) * BLK_TW; e += 64 * BLK_TW) {
            const int b = c0 + e / BLK_TW, t = t0 + e % BLK_TW;

            if (t < a.tiles)
                a.bits[((long long)kvh * a.nblk + b) * a.tiles + t] = (&m[0][0])[e];
        }
        __syncthreads();
    }
}

/* The value of a lane of every four, as CTRL says. */
template <int CTRL> __device__ __forceinline__ int quad_i(int v)
{
    return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, false);
}

/* Second step: a block of threads holds a unit's keys and values in LDS, both
 * split in three bf16 parts (split.h: float32 products without loss), and
 * computes them for the rows that list it, 32 a wave and turn. A key block is
 * read once for all of them, where a row on its own would read its 16 blocks
 * of keys and values again, 512 KB. Each wave collects its own rows and meets the
 * others at the start and at the end only (with barriers in between 184 us, without
 * 180, by 8 waves 172). Outputs leave as the products give them, values and
 * probabilities scaled by SPLIT_UP each, marked by a negative sum; the merge
 * unscales them.
 *
 * 65536 rows of 16 units of 64 keys of 64 channels: 167 us, 617 TFLOP/s of bf16
 * products. The matrix cores are busy 28 % of it, vector instructions (splits
 * of queries and probabilities, exponentials, the exchange before the stores)
 * 45 %, and half of the waves' time goes to waits: loads of queries and lists at the
 * start of a turn, one product's sum into the next. No stores: 168 of 184 us
 * then; no look at the lists: 165; one query for all: 176. */
#define BLK_RING 128   /* rows of a wave's list at most */
#define BLK_TILES 1024 /* tiles of 64 rows a block of threads takes at most */
#define BLK_VMAX 0x1p73f /* 64 values times 2^48 stay finite below */

/* Waves of a block of threads, and of a SIMD. LDS holds two blocks of threads of
 * 64 keys of 64 channels in 48 KB and some, one of 128 channels in 96: of 8 waves
 * each where there is so little room. 4 and 8 waves, us: 4096 x 8 rows of 16
 * units of 64 keys of 128 channels 190, 151; 8 of 100 channels 124, 96; of 2 x
 * 64 keys of 48 channels 85, 71. Smaller units: 32 keys of 64 channels 33, 37; of
 * 128 68, 75; 64 keys of 32 channels 49, 53. */
constexpr int blk_waves(int nd, int nb) { return nd * nb >= 4 && nb == 2 ? 8 : 4; }
constexpr int blk_simd(int nd, int nb) { return nd < 4 ? 4 : nb == 1 ? 3 : 2; }

template <int ND, int NB, bool FULL>
__global__ void __launch_bounds__(64 * blk_waves(ND, NB), blk_simd(ND, NB))
    blk_unit_kernel(const blk_args a)
{
    constexpr int W = blk_waves(ND, NB), NT = 64 * W;
    constexpr int DP = 32 * ND, CH = DP / 8, SB = 32 * NB, KC = SB / 8;
    constexpr int RW = 16 / CH < 1 ? 1 : 16 / CH;  /* K rows in 256 bytes */
    constexpr int RV = 16 / KC < 1 ? 1 : 16 / KC;  /* V rows */
    constexpr int PK = SB * CH;                    /* 16-byte chunks of a part */
    __shared__ split_u4 ks[3 * PK], vs[3 * PK];
    __shared__ unsigned short list[W][BLK_RING];
    __shared__ float sc[W][64];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = a.nh / a.nhk, d = FULL ? DP : a.d;
    /* An XCD takes a band of them: few key heads, whose queries stay in its
     * L2. */
    const int job = xcd_tile(blockIdx.x, gridDim.x);
    const int unit = job / a.pieces, piece = job % a.pieces;
    const int sub = unit % a.sub, b = unit / a.sub % a.nblk, kvh = unit / a.sub / a.nblk;
    const int ss = a.bs / a.sub, k0 = b * a.bs + sub * ss, n = min(a.Nk - k0, ss);
    const unsigned long long *bits = a.bits + ((long long)kvh * a.nblk + b) * a.tiles;
    const int c0 = (int)((long long)a.tiles * piece / a.pieces);
    const int c1 = (int)((long long)a.tiles * (piece + 1) / a.pieces);
    const int base = c0 * 64; /* rows in the list count from here */

    if (c0 >= c1)
        return;
    /* The last block's second unit may lie past the keys. */
    const bool nothing = n <= 0;
    const unsigned long long keep =
        __ballot(lane < n && (!a.kmask || a.kmask[k0 + min(lane, n - 1)]));
    bool wild = false; /* values that the split's sums cannot hold */

    /* Keys and values that are left out are zero here: what they hold meets
     * probabilities of zero. */
    if (!nothing) {
        constexpr int NL = (PK + NT - 1) / NT;
        const float *K = a.K + k0 * a.ldk + (long long)kvh * d;
        const float *V = a.V + k0 * a.ldv + (long long)kvh * d;
        float x[NL][8], y[NL][8];
        split_u4 h, m, l;

        /* Chunk e of K: key e / CH, channels 8 (e % CH) ..; of V: row dd = e %
         * DP of the transposed values, slot 8 c + j of it the key that register
         * 8 (c / 2 % 2) + j of the scores' tile c / 4 holds in lane half c % 2. */
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int e = min(tid + NT * i, PK - 1), key = min(e / CH, n - 1), dd = e % CH * 8;
            const float *p = K + (long long)key * a.ldk;
            float u[4], v[4];

            if (FULL) {
                load4(p + dd, u);
                load4(p + dd + 4, v);
            }
            else {
                load4_row(p, dd, d, u);
                load4_row(p, dd + 4, d, v);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[i][j] = u[j];
                x[i][4 + j] = v[j];
            }
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int e = min(tid + NT * i, PK - 1), dd = min(e % DP, d - 1), c = e / DP;

#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = (c >> 1) * 16 + (j >> 2) * 8 + (c & 1) * 4 + (j & 3);

                y[i][j] = V[(long long)min(key, n - 1) * a.ldv + dd];
            }
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int e = tid + NT * i;

            if (e < PK) {
                const int key = e / CH, at = key * CH + ((e % CH) ^ (key / RW % CH));
                const bool in = keep >> key & 1;

#pragma unroll
                for (int j = 0; j < 8; j++)
                    x[i][j] = in ? x[i][j] : 0.0f;
                split8(x[i], 1.0f, h, m, l);
                ks[at] = h;
                ks[PK + at] = m;
                ks[2 * PK + at] = l;
            }
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int e = tid + NT * i;

            if (e < PK) {
                const int dd = e % DP, c = e / DP, at = dd * KC + (c ^ (dd / RV % KC));
                const unsigned k = (unsigned)(keep >> ((c >> 1) * 16 + (c & 1) * 4));

#pragma unroll
                for (int j = 0; j < 8; j++) {
                    y[i][j] = (k >> ((j >> 2) * 8 + (j & 3)) & 1) && dd < d ? y[i][j] : 0.0f;
                    wild = wild || !(fabsf(y[i][j]) < BLK_VMAX);
                }
                split8(y[i], SPLIT_UP, h, m, l);
                vs[at] = h;
                vs[PK + at] = m;
                vs[2 * PK + at] = l;
            }
        }
    }
    wild = __syncthreads_or(wild);

    auto row_of = [&](int r) { return (long long)(r / g) * a.nh + kvh * g + r % g; };
    /* The place of b in a row's list, each lane half looking through its
     * part; the row lists b. */
    auto slot_of = [&](long long row) {
        const int *sel = a.SEL + ((long long)a.q0 * a.nh + row) * a.top;
        const int from = half * ((a.top + 1) / 2), to = half ? a.top : (a.top + 1) / 2;
        int slot = BLK_MAX_TOP;

        for (int s = from; s < to; s += 4) {
            int v[4];

            if (a.top % 8 == 0) {
                const int4u x = *(const int4u *)(sel + s);

                v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
            }
            else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v[j] = sel[min(s + j, a.top - 1)];
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                slot = v[j] == b ? min(slot, min(s + j, a.top - 1)) : slot;
        }
        return min(slot, __shfl_xor(slot, 32, 64));
    };
    auto tile = [&](const unsigned short *rows, int first, int count) {
        const bool live = col < count;
        const int r = base + rows[first + (live ? col : 0) & BLK_RING - 1];
        const int qi = g == 1 ? r : r / g, h = kvh * g + r - qi * g;
        const long long row = (long long)qi * a.nh + h;
        const float up = a.scale * BLK_LOG2E * BLK_QUP;
        split_u4 q[2 * ND][3];
        split_f16x s[NB];
        constexpr int pa[6] = {0, 2, 1, 0, 1, 0}, pb[6] = {2, 0, 1, 1, 0, 0};

        {
            const float *p = a.Q + (a.q0 + qi) * a.ldq + (long long)h * d;
            float x[2 * ND][2][4];

            if constexpr (FULL) {
#pragma unroll
                for (int st = 0; st < 2 * ND; st++) {
                    load4(p + st * 16 + half * 8, x[st][0]);
                    load4(p + st * 16 + half * 8 + 4, x[st][1]);
                }
            }
            else {
#pragma unroll
                for (int st = 0; st < 2 * ND; st++) {
                    load4_row(p, st * 16 + half * 8, d, x[st][0]);
                    load4_row(p, st * 16 + half * 8 + 4, d, x[st][1]);
                }
            }
#pragma unroll
            for (int st = 0; st < 2 * ND; st++) {
                float y[8];

#pragma unroll
                for (int j = 0; j < 8; j++)
                    y[j] = x[st][j / 4][j % 4];
                split8(y, up, q[st][0], q[st][1], q[st][2]);
            }
        }
        auto key = [&](int p, int t, int st) {
            const int kk = 32 * t + col;

            return __builtin_bit_cast(split_b8,
                                      ks[p * PK + kk * CH + ((2 * st + half) ^ (kk / RW % CH))]);
        };
#pragma unroll
        for (int t = 0; t < NB; t++) {
#pragma unroll
            for (int e = 0; e < 16; e++)
                s[t][e] = 0.0f;
            /* The small products first, then the large ones. */
#pragma unroll
            for (int st = 0; st < 2 * ND; st++) {
                const split_b8 kf[3] = {key(0, t, st), key(1, t, st), key(2, t, st)};

#pragma unroll
                for (int w = 0; w < 5; w++)
                    s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        kf[pa[w]], __builtin_bit_cast(split_b8, q[st][pb[w]]), s[t], 0, 0, 0);
            }
#pragma unroll
            for (int st = 0; st < 2 * ND; st++)
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    key(0, t, st), __builtin_bit_cast(split_b8, q[st][0]), s[t], 0, 0, 0);
        }
        float mx = -INFINITY, l = 0.0f, p[NB][16];

        if (keep != (SB == 64 ? ~0ull : 0xffffffffull)) {
#pragma unroll
            for (int t = 0; t < NB; t++) {
                unsigned k = (unsigned)(keep >> (32 * t)) >> (4 * half);

                /* Tested here: as 16 conditions kept over all tiles they
                 * fill the scalar registers. */
                asm volatile("" : "+v"(k));
#pragma unroll
                for (int e = 0; e < 16; e++)
                    s[t][e] = k >> ((e >> 2) * 8 + (e & 3)) & 1 ? s[t][e] : -INFINITY;
            }
        }
#pragma unroll
        for (int t = 0; t < NB; t++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                mx = fmaxf(mx, s[t][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * (1.0f / BLK_QUP);
        const float ref = mx == -INFINITY ? 0.0f : mx;

#pragma unroll
        for (int t = 0; t < NB; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                p[t][e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], 1.0f / BLK_QUP, -ref));
                l += p[t][e];
            }
        l += __shfl_xor(l, 32, 64);

        const int slot = slot_of(row);
        const long long at = (row * a.top + slot) * a.sub + sub;
        split_f16x o[ND];
        split_u4 high[2 * NB];

        /* Again the small products first. Probabilities are scaled as values
         * are: those under 2^-110 would lose bits (2^-124: all but ten), which
         * counts beside values 2^100 times the largest probability's. */
#pragma unroll
        for (int tt = 0; tt < ND; tt++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                o[tt][e] = 0.0f;
        auto value = [&](int k, int tt, int u) {
            const int dd = tt * 32 + col;

            return __builtin_bit_cast(split_b8,
                                      vs[k * PK + dd * KC + ((2 * u + half) ^ (dd / RV % KC))]);
        };
#pragma unroll
        for (int u = 0; u < 2 * NB; u++) {
            float x[8];
            split_u4 pp[3];

#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = p[u / 2][8 * (u % 2) + j];
            split8(x, SPLIT_UP, pp[0], pp[1], pp[2]);
            high[u] = pp[0];
#pragma unroll
            for (int tt = 0; tt < ND; tt++) {
                const split_b8 vf[3] = {value(0, tt, u), value(1, tt, u), value(2, tt, u)};

#pragma unroll
                for (int w = 0; w < 5; w++)
                    o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        vf[pa[w]], __builtin_bit_cast(split_b8, pp[pb[w]]), o[tt], 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < 2 * NB; u++)
#pragma unroll
            for (int tt = 0; tt < ND; tt++)
                o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    value(0, tt, u), __builtin_bit_cast(split_b8, high[u]), o[tt], 0, 0, 0);
        /* Scores that are not finite or below the range of the split (no
         * probability at all for keys that are kept), and wild values: again in
         * float32. */
        const bool again = wild || !(l < INFINITY) || (l == 0.0f && keep);
        const unsigned long long redo = __ballot(again && live);

        /* A lane holds, for its row, runs of 4 channels 8 apart. Four lanes
         * exchange theirs, so that lane i of them has run i of all four rows,
         * and a store writes whole 128-byte lines (8 rows) instead of 32 bytes
         * of 32 rows. */
        const int to = live && !again ? (int)at : -1;
        const bool whole = __all(to >= 0);

        if (half == 0 && to >= 0)
            a.ml[to] = make_float2(mx, -l);
#pragma unroll
        for (int tt = 0; tt < ND; tt++) {
            float x[4][4];

#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    x[e][j] = o[tt][4 * e + j];
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float u = dpp_f(x[e][j], 0xB1), v = dpp_f(x[e + 1][j], 0xB1);

                    x[e][j] = lane & 1 ? v : x[e][j];
                    x[e + 1][j] = lane & 1 ? x[e + 1][j] : u;
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float u = dpp_f(x[e][j], 0x4E), v = dpp_f(x[e + 2][j], 0x4E);

                    x[e][j] = lane & 2 ? v : x[e][j];
                    x[e + 2][j] = lane & 2 ? x[e + 2][j] : u;
                }
            }
            const int there[4] = {quad_i<0x00>(to), quad_i<0x55>(to), quad_i<0xAA>(to),
                                  quad_i<0xFF>(to)};
            const unsigned run = tt * 32 + (lane & 3) * 8 + half * 4;

#pragma unroll
            for (int e = 0; e < 4; e++)
                if (whole || there[e] >= 0)
                    *(float4 *)((char *)a.part + 4u * ((unsigned)there[e] * DP + run)) =
                        make_float4(x[e][0], x[e][1], x[e][2], x[e][3]);
        }
        if (redo)
            for (int e = 0; e < count; e++)
                if (redo >> e & 1) {
                    const int rr = base + rows[first + e & BLK_RING - 1], sl = __builtin_amdgcn_readlane(slot, e);
                    const long long to = (row_of(rr) * a.top + sl) * a.sub + sub;

                    blk_unit_f32(a, a.q0 + rr / g, kvh * g + rr % g, k0, k0 + n,
                                 a.part + to * DP, a.ml + to, sc[wave]);
                }
    };

    auto turn = [&](const unsigned short *rows, int first, int count) {
        __builtin_amdgcn_wave_barrier();
        if (nothing) {
            const long long row = row_of(base + rows[first + (col < count ? col : 0) & BLK_RING - 1]);
            const int slot = slot_of(row);

            if (lane < count)
                a.ml[(row * a.top + slot) * a.sub + sub] = make_float2(-INFINITY, 0.0f);
        }
        else
            tile(rows, first, count);
        __builtin_amdgcn_wave_barrier();
    };
    unsigned short *mine = list[wave];
    int first = 0, have = 0;

    /* Tiles of 64 rows, every W-th one this wave's, the bits of 64 of them
     * read at once. */
    for (int t0 = c0 + wave; t0 < c1; t0 += W * 64) {
        const int mt = t0 + W * lane;
        const unsigned long long word = mt < c1 ? bits[mt] : 0;
        const int n64 = min(64, (c1 - t0 + W - 1) / W);

        for (int i = 0; i < n64; i++) {
            const unsigned low = __builtin_amdgcn_readlane((int)word, i);
            const unsigned high = __builtin_amdgcn_readlane((int)(word >> 32), i);
            const int before = __builtin_amdgcn_mbcnt_hi(high, __builtin_amdgcn_mbcnt_lo(low, 0));

            if ((half ? high : low) >> col & 1)
                mine[first + have + before & BLK_RING - 1] =
                    (unsigned short)((t0 + W * i) * 64 + lane - base);
            have += __popc(low) + __popc(high);
            for (; have >= 32; have -= 32, first += 32)
                turn(mine, first, 32);
        }
    }
    /* What is left of the waves, fewer than 32 rows each, together. */
    __shared__ unsigned short rest[32 * W];
    __shared__ int left[W];

    if (lane == 0)
        left[wave] = have;
    __syncthreads();
    int at = 0, all = 0;

#pragma unroll
    for (int i = 0; i < W; i++) {
        at += i < wave ? left[i] : 0;
        all += left[i];
    }
    if (lane < have)
        rest[at + lane] = mine[first + lane & BLK_RING - 1];

    __syncthreads();
    if (32 * wave < all)
        turn(rest + 32 * wave, 0, min(32, all - 32 * wave));
}

/* A unit's weight as the merge's lanes hand it round: negative (-0 too) where
 * the outputs are scaled, BLK_NO_UNIT where there are none. */
#define BLK_NO_UNIT 2.0f /* weights are at most 1, or NaN */

__device__ __forceinline__ float blk_weight(float w, float sum)
{
    return sum < 0.0f ? -w : sum != 0.0f ? w : BLK_NO_UNIT;
}

__device__ __forceinline__ void blk_add(const float4 &p, float w, float (&o)[4])
{
    const float down = __builtin_signbitf(w) ? SPLIT_DOWN : 1.0f;

    w = fabsf(w);
    o[0] = fmaf(p.x * down, w, o[0]);
    o[1] = fmaf(p.y * down, w, o[1]);
    o[2] = fmaf(p.z * down, w, o[2]);
    o[3] = fmaf(p.w * down, w, o[3]);
}

/* Units of a row merged: softmax over all of them from their maxima and sums.
 * A wave a row: lane u has unit u's weight (and unit 64 + u's), then DP / 4
 * lanes a unit add the outputs, 256 / DP units at a time. A negative sum: the
 * outputs are scaled, and the weight goes round with a minus;
 * the outputs are unscaled, not the weight, whose last bits would be lost from
 * 2^-78 on, with values large enough to count. Bound by memory: 65536 rows of
 * 16 units of 64 channels, 285 MB, 46 us, 6.2 TB/s. */
template <int DP> __global__ void __launch_bounds__(256) blk_merge_kernel(const blk_args a)
{
    constexpr int LV = DP / 4, GV = 64 / LV;
    const int units = a.top * a.sub, lane = threadIdx.x & 63, c = 4 * (lane % LV), gv = lane / LV;
    const long long row =
        (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    if (row >= (long long)a.Nq * a.nh)
        return;
    const float2 none = make_float2(-INFINITY, 0.0f);
    const float2 *ml = a.ml + row * units;
    const float *part = a.part + row * units * DP + c;
    const float2 x = lane < units ? ml[lane] : none;
    const float2 y = 64 + lane < units ? ml[64 + lane] : none;
    const float m = wave_max_full(fmaxf(x.y != 0.0f ? x.x : -INFINITY, y.y != 0.0f ? y.x : -INFINITY));
    const float wx = x.y != 0.0f ? __builtin_amdgcn_exp2f(x.x - m) : 0.0f;
    const float wy = y.y != 0.0f ? __builtin_amdgcn_exp2f(y.x - m) : 0.0f;
    const float l = wave_sum_full(fabsf(x.y) * wx + fabsf(y.y) * wy);
    const float vx = blk_weight(wx, x.y), vy = blk_weight(wy, y.y);
    float o[4] = {0, 0, 0, 0};

    /* Four loads on their way at once; units with no key hold nothing. */
    for (int u0 = gv; u0 < units + gv; u0 += 4 * GV) {
        float4 p[4];
        float w[4];

#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int u = u0 + i * GV, at = min(u, units - 1);
            const float wu = __shfl(u < 64 ? vx : vy, u & 63, 64);

            p[i] = *(const float4 *)(part + (long long)at * DP);
            w[i] = u < units ? wu : BLK_NO_UNIT;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (w[i] != BLK_NO_UNIT)
                blk_add(p[i], w[i], o);
    }
#pragma unroll
    for (int s = LV; s < 64; s *= 2)
#pragma unroll
        for (int j = 0; j < 4; j++)
            o[j] += __shfl_xor(o[j], s, 64);
    if (gv == 0) {
        float *out = a.O + (a.q0 + row / a.nh) * a.ldo + (row % a.nh) * a.d;

#pragma unroll
        for (int j = 0; j < 4; j++)
            o[j] = l == 0.0f ? 0.0f : o[j] / l;
        if (c + 4 <= a.d)
            store4(out + c, o[0], o[1], o[2], o[3]);
        else
            for (int j = 0; c + j < a.d; j++)
                out[c + j] = o[j];
    }
}

/* The same for few units a row (at most 16): 16 lanes a row, lane u with unit
 * u's weight, then DP / 4 lanes a unit (all 16, or 8 and 8 on two units at a time;
 * of 128 channels two runs a lane). */
template <int DP> __global__ void __launch_bounds__(256) blk_merge16_kernel(const blk_args a)
{
    constexpr int LV = DP / 4 < 16 ? DP / 4 : 16, GV = 16 / LV, RUNS = DP / 4 / LV;
    const int units = a.top * a.sub, lane = threadIdx.x & 63, l16 = lane & 15;
    const int c = 4 * (l16 % LV), gv = l16 / LV;
    const long long rows = (long long)a.Nq * a.nh;
    const long long want = (long long)blockIdx.x * 16 + threadIdx.x / 16;
    const long long row = min(want, rows - 1);
    const float *part = a.part + row * units * DP + c;
    const float2 x = l16 < units ? a.ml[row * units + l16] : make_float2(-INFINITY, 0.0f);
    float m = x.y != 0.0f ? x.x : -INFINITY, o[RUNS][4] = {};

    m = fmaxf(m, dpp_f(m, 0xB1));
    m = fmaxf(m, dpp_f(m, 0x4E));
    m = fmaxf(m, dpp_f(m, 0x141));
    m = fmaxf(m, dpp_f(m, 0x140));
    const float w = x.y != 0.0f ? __builtin_amdgcn_exp2f(x.x - m) : 0.0f;
    float l = fabsf(x.y) * w;
    const float wv = blk_weight(w, x.y);

    l += dpp_f(l, 0xB1);
    l += dpp_f(l, 0x4E);
    l += dpp_f(l, 0x141);
    l += dpp_f(l, 0x140);
    for (int u0 = 0; u0 < units; u0 += 4 * GV) {
        float4 p[4][RUNS];
        float wu[4];

#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int u = u0 + i * GV + gv, at = min(u, units - 1);
            const float v = __shfl(wv, (lane & 48) | at, 64);

            wu[i] = u < units ? v : BLK_NO_UNIT;
#pragma unroll
            for (int r = 0; r < RUNS; r++)
                p[i][r] = *(const float4 *)(part + (long long)at * DP + 64 * r);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (wu[i] != BLK_NO_UNIT) {
#pragma unroll
                for (int r = 0; r < RUNS; r++)
                    blk_add(p[i][r], wu[i], o[r]);
            }
    }
    if (GV == 2)
#pragma unroll
        for (int j = 0; j < 4; j++)
            o[0][j] += __shfl_xor(o[0][j], 8, 64);
    if (want < rows && gv == 0) {
        float *out = a.O + (a.q0 + row / a.nh) * a.ldo + (row % a.nh) * a.d;

#pragma unroll
        for (int r = 0; r < RUNS; r++) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                o[r][j] = l == 0.0f ? 0.0f : o[r][j] / l;
            if (c + 64 * r + 4 <= a.d)
                store4(out + c + 64 * r, o[r][0], o[r][1], o[r][2], o[r][3]);
            else
                for (int j = 0; c + 64 * r + j < a.d; j++)
                    out[c + 64 * r + j] = o[r][j];
        }
    }
}

/* The passes of a call: queries a pass, and what one needs of the work
 * buffer. */
struct blk_plan {
    bool direct;
    int pass, passes, tiles, dp, sub, nblk;
    long long part, ml, bits; /* bytes */
};

/* Units that lists pay for, see below. */
#define BLK_LIST_UNITS 400000 /* units times (channels + 32), more than that */
#define BLK_LIST_ROWS 5       /* rows that list a block, on average */

static int blk_width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

/* Bytes of a query's units: outputs, maxima and sums. */
static long long blk_query_bytes(int nh, int d, int bs, int top)
{
    return (long long)nh * top * blk_sub(bs) * (blk_width(d) + 2) * 4;
}

/* Units of a pass: 8192 x 8 rows of 16 units of 64 channels 294 us in two
 * passes of 256 MiB, 270 in one; 350 in three. */
#define BLK_PART_BYTES (512LL << 20)

static long long g_blk_budget = BLK_PART_BYTES;

extern "C" void icoreg_blocks_budget(long bytes)
{
    g_blk_budget = bytes > 0 ? bytes : BLK_PART_BYTES;
}

static blk_plan blk_plan_of(int Nq, int Nk, int nh, int nhk, int d, int bs, int top)
{
    blk_plan p;
    const int g = nh / nhk;

    p.nblk = ops_key_blocks(Nk, bs);
    p.sub = blk_sub(bs);
    p.dp = blk_width(d);
    /* A query's units and bits. */
    const long long most = max(1LL, g_blk_budget / (blk_query_bytes(nh, d, bs, top) +
                                                    (long long)nh * p.nblk / 8 + 1));

    p.passes = (int)((Nq + most - 1) / most);
    p.pass = (Nq - 1) / p.passes + 1;
    /* Units one by one or by lists, us: 8 heads of 64 on 256 blocks of 64 keys,
     * 16 listed, 32 queries 22, 22; 48 queries 28, 22; 1024 queries 435, 49. 8 heads
     * of 128, 8 of 64 blocks, 32 queries 24, 31; 64 queries 40, 32; of 32, 8 of 100
     * blocks, 64 queries 15, 19; 128 queries 24, 19. Lists of a few rows stage a
     * block's keys for nothing: 2 key heads of 128, 16 of 2047 blocks, 4 rows a list
     * 152, 192; 8 rows 299, 199. */
    const long long units = (long long)p.pass * nh * top * p.sub;

    /* Lists place their outputs by 32 bits (a query of very many heads passes them). */
    p.direct = p.nblk == 0 || nhk > 65535 || units * p.dp * 4 > 1LL << 32 ||
               units * (p.dp + 32) <= BLK_LIST_UNITS ||
               (long long)p.pass * g * top < (long long)BLK_LIST_ROWS * p.nblk;
    p.tiles = ((p.pass * g + 63) / 64 + BLK_TW - 1) / BLK_TW * BLK_TW;
    p.part = (long long)p.pass * nh * top * p.sub * p.dp * 4;
    p.ml = (long long)p.pass * nh * top * p.sub * 8;
    p.bits = p.direct ? 0 : (long long)nhk * p.nblk * p.tiles * 8;
    return p;
}

/* Bytes that cover this call and every one of fewer queries, keys or listed
 * blocks, whatever their passes and kernels: the sizes of blk_plan's parts fall
 * where a pass more or another kernel begins. Units of all queries and their
 * bits, or, where passes end that, what blk_plan_of holds a pass to: q queries
 * of u bytes have bits of at most q nh / 8 + 64 nhk bytes a key block (whole runs
 * of tiles), and q (u + nh nblk / 8) is within the budget or q = 1. Lists need so many
 * units, and are taken on at most so many blocks. */
static size_t blk_work_bytes(int Nq, int Nk, int nh, int nhk, int d, int bs, int top)
{
    typedef __int128 wide; /* products of any sizes */
    const int g = nh / nhk;
    const wide u = blk_query_bytes(nh, d, bs, top), rows = (wide)Nq * g;
    const bool lists = nhk <= 65535 &&
                       (wide)Nq * nh * top * blk_sub(bs) * (blk_width(d) + 32) > BLK_LIST_UNITS;
    const wide nblk = lists ? std::min<wide>(ops_key_blocks(Nk, bs), rows * top / BLK_LIST_ROWS) : 0;
    const wide tiles = ((rows + 63) / 64 + BLK_TW - 1) / BLK_TW * BLK_TW;
    const wide all = Nq * u + nhk * nblk * tiles * 8;
    const wide held = std::max<wide>(g_blk_budget, u + nh * nblk / 8) + 64 * nhk * nblk;

    return (size_t)std::min(all, held);
}

static bool blk_sizes_ok(int Nq, int Nk, int nh, int nhk, int d, int bs, int top)
{
    return Nq >= 0 && Nk >= 0 && Nk <= BLK_MAX_KEYS && nh >= 1 && nhk >= 1 && nh % nhk == 0 && d >= 1 &&
           d <= OPS_MAX_HEAD_DIM && blk_size_ok(bs) && top >= 1 && top <= BLK_MAX_TOP;
}

extern "C" size_t ops_attention_blocks_work_bytes(int Nq, int Nk, int nh, int nhk, int d, int bs,
                                                  int top)
{
    if (!blk_sizes_ok(Nq, Nk, nh, nhk, d, bs, top) || Nq == 0)
        return 0;
    return blk_work_bytes(Nq, Nk, nh, nhk, d, bs, top);
}

extern "C" int icoreg_blocks_passes(int Nq, int Nk, int nh, int nhk, int d, int bs, int top,
                                    size_t *work)
{
    if (!blk_sizes_ok(Nq, Nk, nh, nhk, d, bs, top) || Nq == 0)
        return -1;
    const blk_plan p = blk_plan_of(Nq, Nk, nh, nhk, d, bs, top);

    if (work)
        *work = (size_t)(p.part + p.ml + p.bits);
    return p.passes;
}

extern "C" int icoreg_blocks_choice(int Nq, int Nk, int nh, int nhk, int d, int bs, int top)
{
    if (!blk_sizes_ok(Nq, Nk, nh, nhk, d, bs, top) || Nq == 0)
        return -1;
    return !blk_plan_of(Nq, Nk, nh, nhk, d, bs, top).direct;
}

extern "C" void ops_attention_blocks(struct ops *o, struct opnd Q, struct opnd K, struct opnd V,
                                     struct opnd O, int Nq, int Nk, int nh, int nhk, int d, int bs,
                                     int top, cl_mem SEL, float scale, cl_mem kmask, cl_mem work)
{
    ICOREG_API_BEGIN
    const char *op = "ops_attention_blocks";
    const long long qw = (long long)nh * d, kw = (long long)nhk * d;

    if (!blk_sizes_ok(Nq, Nk, nh, nhk, d, bs, top))
        icoreg_fatal("%s: invalid sizes Nq=%d Nk=%d nh=%d nhk=%d d=%d bs=%d top=%d", op, Nq, Nk, nh,
                     nhk, d, bs, top);
    if (Q.ld < qw || K.ld < kw || V.ld < kw || O.ld < qw || Q.off < 0 || K.off < 0 || V.off < 0 ||
        O.off < 0)
        icoreg_fatal("%s: negative offset or short row: ld %d, %d, %d, %d", op, Q.ld, K.ld, V.ld,
                     O.ld);
    if (Nq == 0)
        return;
    const blk_plan p = blk_plan_of(Nq, Nk, nh, nhk, d, bs, top);
    const long long obytes = ((Nq - 1) * (long long)O.ld + qw) * 4;
    const long long wbytes = p.part + p.ml + p.bits;

    need_floats(Q.buf, Q.off, (Nq - 1) * (long long)Q.ld + qw, op, "Q");
    if (Nk) {
        need_floats(K.buf, K.off, (Nk - 1) * (long long)K.ld + kw, op, "K");
        need_floats(V.buf, V.off, (Nk - 1) * (long long)V.ld + kw, op, "V");
    }
    need_floats(O.buf, O.off, obytes / 4, op, "O");
    need_bytes(SEL, 0, (long long)Nq * nh * top * 4, op, "SEL");
    if (kmask)
        need_bytes(kmask, 0, Nk, op, "kmask");
    need_bytes(work, 0, wbytes, op, "work");
    need_aligned(work, 16, op, "work");
    if (cfptr(O.buf) + O.off != cfptr(Q.buf) + Q.off || O.ld != Q.ld)
        need_rows_apart(cfptr(O.buf) + O.off, O.ld, qw, Nq, cfptr(Q.buf) + Q.off, Q.ld, qw, Nq, op,
                        "O and Q (unless the same)");
    if (Nk) {
        need_rows_apart(cfptr(O.buf) + O.off, O.ld, qw, Nq, cfptr(K.buf) + K.off, K.ld, kw, Nk, op,
                        "O and K");
        need_rows_apart(cfptr(O.buf) + O.off, O.ld, qw, Nq, cfptr(V.buf) + V.off, V.ld, kw, Nk, op,
                        "O and V");
    }
    need_apart(O.buf, O.off * 4, obytes, work, 0, wbytes, op, "O and work");
    need_apart(Q.buf, Q.off * 4, ((Nq - 1) * (long long)Q.ld + qw) * 4, work, 0, wbytes, op,
               "Q and work");
    if (Nk) {
        need_apart(K.buf, K.off * 4, ((Nk - 1) * (long long)K.ld + kw) * 4, work, 0, wbytes, op,
                   "K and work");
        need_apart(V.buf, V.off * 4, ((Nk - 1) * (long long)V.ld + kw) * 4, work, 0, wbytes, op,
                   "V and work");
    }
    need_apart(kmask, 0, Nk, work, 0, wbytes, op, "kmask and work");
    need_apart(SEL, 0, (long long)Nq * nh * top * 4, O.buf, O.off * 4, obytes, op, "SEL and O");
    if (kmask)
        need_apart(kmask, 0, Nk, O.buf, O.off * 4, obytes, op, "kmask and O");
    need_apart(SEL, 0, (long long)Nq * nh * top * 4, work, 0, wbytes, op, "SEL and work");
    count32((long long)p.pass * nh * top * p.sub, "units of a pass");

    blk_args a = {};

    a.Q = cfptr(Q.buf) + Q.off;
    a.K = Nk ? cfptr(K.buf) + K.off : nullptr;
    a.V = Nk ? cfptr(V.buf) + V.off : nullptr;
    a.O = fptr(O.buf) + O.off;
    a.SEL = (const int *)SEL->ptr;
    a.kmask = kmask ? (const unsigned char *)kmask->ptr : nullptr;
    a.ldq = Q.ld;
    a.ldk = K.ld;
    a.ldv = V.ld;
    a.ldo = O.ld;
    a.Nk = Nk;
    a.nh = nh;
    a.nhk = nhk;
    a.d = d;
    a.bs = bs;
    a.sub = p.sub;
    a.nblk = p.nblk;
    a.top = top;
    a.scale = scale;
    a.part = fptr(work);
    a.ml = (float2 *)((char *)work->ptr + p.part);
    a.bits = (unsigned long long *)((char *)work->ptr + p.part + p.ml);
    const hipStream_t s = stream_of(o->ocl);
    const int g = nh / nhk;

    prof_scope ps(o->ocl, "attention_blocks");
    for (int q0 = 0; q0 < Nq; q0 += p.pass) {
        a.q0 = q0;
        a.Nq = min(p.pass, Nq - q0);
        const long long rows = (long long)a.Nq * nh, units = rows * top * p.sub;

        a.tiles = ((a.Nq * g + 63) / 64 + BLK_TW - 1) / BLK_TW * BLK_TW;
        if (p.direct) {
            const dim3 grid(grid_of(units, 256, "units"));

            if (p.dp == 32)
                hipLaunchKernelGGL(blk_direct_kernel<32>, grid, dim3(256), 0, s, a);
            else if (p.dp == 64)
                hipLaunchKernelGGL(blk_direct_kernel<64>, grid, dim3(256), 0, s, a);
            else
                hipLaunchKernelGGL(blk_direct_kernel<128>, grid, dim3(256), 0, s, a);
            launch_check("attention_blocks direct");
        }
        else {
            const int lists = count32((long long)nhk * p.nblk * p.sub, "units of keys");
            /* Splits of a list: twice the blocks of threads that a CU holds, if
             * each wave has some 64 rows to compute. Units of 64 keys, us: of 64
             * channels (2 held), 2, 4, 8 a CU 184, 170, 181; of 128 (1 held) 151,
             * 169, 215. 32, 64 rows a wave: 400 x 100 blocks of 32 channels 51.7,
             * 48.7; 128 blocks of 128 channels the same. */
            const int nd = p.dp / 32, nb = bs / p.sub <= 32 ? 1 : 2;
            const int held = 4 * blk_simd(nd, nb) / blk_waves(nd, nb);
            const long long each = max(1LL, (long long)a.Nq * g * top / p.nblk / (64 * blk_waves(nd, nb)));

            a.pieces = (int)max((a.tiles + BLK_TILES - 1LL) / BLK_TILES,
                                min(min(each, (long long)a.tiles),
                                    (2LL * held * o->ocl->cu_count + lists - 1LL) / lists));
            hipLaunchKernelGGL(blk_bits_kernel, dim3(a.tiles / BLK_TW, nhk), dim3(64 * BLK_TW), 0, s,
                               a);
            launch_check("attention_blocks bits");
            const dim3 grid(grid_of((long long)lists * a.pieces, 64 * blk_waves(nd, nb), "lists"));

#define UNIT_LAUNCH(ND_, NB_)                                                                 \
    do {                                                                                      \
        const dim3 block(64 * blk_waves(ND_, NB_));                                           \
                                                                                              \
        if (d == 32 * ND_)                                                                    \
            hipLaunchKernelGGL((blk_unit_kernel<ND_, NB_, true>), grid, block, 0, s, a);      \
        else                                                                                  \
            hipLaunchKernelGGL((blk_unit_kernel<ND_, NB_, false>), grid, block, 0, s, a);     \
    } while (0)
#define UNIT_KEYS(ND_)          \
    do {                        \
        if (nb == 1)            \
            UNIT_LAUNCH(ND_, 1); \
        else                    \
            UNIT_LAUNCH(ND_, 2); \
    } while (0)
            if (p.dp == 32)
                UNIT_KEYS(1);
            else if (p.dp == 64)
                UNIT_KEYS(2);
            else
                UNIT_KEYS(4);
#undef UNIT_KEYS
#undef UNIT_LAUNCH
            launch_check("attention_blocks units");
        }
        /* Both, us: 51200 rows of 8 units of 32 channels 21.1, 10.8; 25616 of 8 of
         * 64 12.6, 10.5; 65536 of 16 of 64 43.4, 52.0. */
        const bool few = top * p.sub <= 8;
        const dim3 grid(grid_of(few ? (rows + 15) / 16 : (rows + 3) / 4, 256, "merge"));

#define MERGE_LAUNCH(DP_)                                                           \
    do {                                                                            \
        if (few)                                                                    \
            hipLaunchKernelGGL(blk_merge16_kernel<DP_>, grid, dim3(256), 0, s, a);  \
        else                                                                        \
            hipLaunchKernelGGL(blk_merge_kernel<DP_>, grid, dim3(256), 0, s, a);    \
    } while (0)
        if (p.dp == 32)
            MERGE_LAUNCH(32);
        else if (p.dp == 64)
            MERGE_LAUNCH(64);
        else
            MERGE_LAUNCH(128);
#undef MERGE_LAUNCH
        launch_check("attention_blocks merge");
    }
    ICOREG_API_END
}
