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

#include "common.h"
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
 * four channels a key, 256 / L keys at a time, sums in 64 bits. */
template <int L, bool VEC>
__global__ void __launch_bounds__(256)
    block_index_kernel(const float *__restrict__ K, long long ldk, int Nk, int nhk, int d, int bs,
                       const unsigned char *__restrict__ kmask, int b0,
                       signed char *__restrict__ KC, float *__restrict__ KS)
{
    constexpr int G = 256 / L; /* keys at a time */
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
    for (int k = k0 + g; k < k1; k += G) {
        if (kmask && !kmask[k])
            continue;
        const float *p = K + k * ldk + (long long)h * d;

        n++;
        if (VEC) {
            if (c < d) {
                const float4 x = *(const float4 *)(p + c);

                s[0] += x.x;
                s[1] += x.y;
                s[2] += x.z;
                s[3] += x.w;
            }
        }
        else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c + j < d)
                    s[j] += p[c + j];
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
    if (Nk < 0 || Nk > BLK_MAX_KEYS || nhk < 1 || b0 < 0 || nb < 0 || (long long)b0 + nb > nblk || K.off < 0 ||
        K.ld < (long long)nhk * d)
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
    }
    const int grid = count32((long long)nb * nhk, "block index");
    const bool vec = ((uintptr_t)(cfptr(K.buf) + K.off) & 15) == 0 && K.ld % 4 == 0 && d % 4 == 0;

    prof_scope ps(o->ocl, "block_index");
#define INDEX_LAUNCH(L_, V_)                                                                   \
    hipLaunchKernelGGL((block_index_kernel<L_, V_>), dim3(grid), dim3(256), 0, stream_of(o->ocl), \
                       cfptr(K.buf) + K.off, (long long)K.ld, Nk, nhk, d, bs,                   \
                       kmask ? (const unsigned char *)kmask->ptr : nullptr, b0,                \
                       (signed char *)KC->ptr, fptr(KS))
#define INDEX_LANES(L_)        \
    do {                       \
        if (vec)               \
            INDEX_LAUNCH(L_, true);  \
        else                   \
            INDEX_LAUNCH(L_, false); \
    } while (0)
    if (d <= 32)
        INDEX_LANES(8);
    else if (d <= 64)
        INDEX_LANES(16);
    else
        INDEX_LANES(32);
#undef INDEX_LANES
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

/* The top `top` of a wave's candidates, slot j of lane l before slot j of
 * lane l + 1 before slot j + 1, equal keys in that order: returned sorted,
 * candidate i in lane i of (key, idx), SEL_NONE behind the last. list: 2 x 64
 * words of LDS of this wave. */
template <int N>
__device__ __forceinline__ void sel_top(const int (&k)[N], const int (&i)[N], int top, int *list,
                                        int &key, int &idx)
{
    const int lane = threadIdx.x & 63;
    int have = 0, most = SEL_NONE;

    auto count = [&](int t) {
        int n = 0;

#pragma unroll
        for (int j = 0; j < N; j++)
            n += __popcll(__ballot(k[j] >= t));
        return n;
    };
#pragma unroll
    for (int j = 0; j < N; j++)
        most = max(most, k[j]);
    {
        const int ctl[4] = {0xB1, 0x4E, 0x141, 0x140};

#pragma unroll
        for (int c = 0; c < 4; c++)
            most = max(most, dpp_i(most, ctl[c]));
        most = max(max(__builtin_amdgcn_readlane(most, 0), __builtin_amdgcn_readlane(most, 16)),
                   max(__builtin_amdgcn_readlane(most, 32), __builtin_amdgcn_readlane(most, 48)));
    }
    have = count(SEL_NONE + 1);
    /* lo: at least top candidates, hi: fewer; halved by value first, which
     * parts scores of one size in a few steps, by bits where that stalls. */
    int lo = SEL_NONE + 1, hi = most + 1, nlo = have, nhi = 0;

    if (have > top) {
        for (int step = 0; nlo > top && (unsigned)hi - (unsigned)lo > 1; step++) {
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
        if (nlo == top)
            nhi = top, hi = lo; /* exactly the candidates from lo on */
    }
    else
        nhi = have, hi = lo;
    /* Every candidate from hi on, and the first of those equal to lo. */
    int at = 0, rest = min(have, top) - nhi;

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

    for (int j = 0; j < at; j++) {
        const int other = __builtin_amdgcn_readlane(mine, j);

        rank += other + (j < lane) > mine;
    }
    __builtin_amdgcn_wave_barrier();
    if (lane < at) {
        list[rank] = mine;
        list[64 + rank] = who;
    }
    __builtin_amdgcn_wave_barrier();
    key = list[lane];
    idx = list[64 + lane];
    __builtin_amdgcn_wave_barrier();
}

#define SEL_SLOTS 8 /* scores a lane holds at a time */

/* A block of W waves selects for one query and head: every wave scores its
 * share of the key blocks, lane by lane, SEL_SLOTS x 64 at a time, and keeps
 * the best so far beside the next ones; wave 0 selects among the waves'. */
template <int W, int DW> /* DW: words of a code row that are not padding */
__global__ void __launch_bounds__(64 * W)
    block_select_kernel(const float *__restrict__ Q, long long ldq, int Nq, int nh, int nhk, int d,
                        const signed char *__restrict__ KC, const float *__restrict__ KS, int nblk,
                        int top, int *__restrict__ SEL)
{
    __shared__ int lists[W][128];
    __shared__ __align__(16) unsigned char codes[W][128];
    __shared__ int best[W > 1 ? W * 128 : 1];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x, h = row % nh, kvh = h / (nh / nhk);
    const float *q = Q + (long long)(row / nh) * ldq + (long long)h * d;
    const long long pitch = q8_pitch(d);
    int *list = lists[wave];
    unsigned qc[DW];
    int key = SEL_NONE, idx = -1;

    {
        const int c = 2 * lane;
        const float a = c < d ? q[c] : 0.0f, b = c + 1 < d ? q[c + 1] : 0.0f;
        const q8_scale s = q8_scale_of(wave_umax(max(q8_mag(a), q8_mag(b))));

        codes[wave][c] = (unsigned char)q8_code(a, s.r);
        codes[wave][c + 1] = (unsigned char)q8_code(b, s.r);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < DW; j++)
            qc[j] = __builtin_amdgcn_readfirstlane(((const unsigned *)codes[wave])[j]);
        /* A query that is not finite scores NaN everywhere. */
        if (s.s != s.s)
            key = SEL_NAN;
    }
    const bool bad = key == SEL_NAN;
    const int share = ((nblk + W - 1) / W + 63) / 64 * 64;
    const int b1 = min(nblk, (wave + 1) * share);

    key = SEL_NONE;
    for (int b0 = wave * share; b0 < b1; b0 += 64 * SEL_SLOTS) {
        int k[SEL_SLOTS + 1], i[SEL_SLOTS + 1];

        k[0] = key;
        i[0] = idx;
#pragma unroll
        for (int j = 0; j < SEL_SLOTS; j++) {
            const int b = b0 + 64 * j + lane;

            k[j + 1] = SEL_NONE;
            i[j + 1] = b;
            if (b < b1) {
                const long long at = (long long)b * nhk + kvh;
                const uint4 *p = (const uint4 *)(KC + at * pitch);
                const float s = KS[at];
                int dot = 0;

#pragma unroll
                for (int w = 0; w < DW / 4; w++) {
                    const uint4 x = p[w];

                    dot = __builtin_amdgcn_sdot4((int)x.x, (int)qc[4 * w], dot, false);
                    dot = __builtin_amdgcn_sdot4((int)x.y, (int)qc[4 * w + 1], dot, false);
                    dot = __builtin_amdgcn_sdot4((int)x.z, (int)qc[4 * w + 2], dot, false);
                    dot = __builtin_amdgcn_sdot4((int)x.w, (int)qc[4 * w + 3], dot, false);
                }
                if (!(s < 0.0f))
                    k[j + 1] = bad ? SEL_NAN : sel_key(s * (float)dot);
            }
        }
        sel_top(k, i, top, list, key, idx);
    }
    if (W > 1) {
        best[wave * 64 + lane] = key;
        best[(W + wave) * 64 + lane] = idx;
        __syncthreads();
        if (wave)
            return;
        int k[W], i[W];

#pragma unroll
        for (int w = 0; w < W; w++) {
            k[w] = best[w * 64 + lane];
            i[w] = best[(W + w) * 64 + lane];
        }
        sel_top(k, i, top, list, key, idx);
    }
    if (lane < top)
        SEL[(long long)row * top + lane] = key == SEL_NONE ? -1 : idx;
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
    if (Nq < 0 || nh < 1 || nhk < 1 || nh % nhk || nblk < 0 || Q.off < 0 ||
        Q.ld < (long long)nh * d)
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
    const int grid = count32(rows, "selection rows");

    prof_scope ps(o->ocl, "block_select");
#define SELECT_LAUNCH(W_, D_)                                                                   \
    hipLaunchKernelGGL((block_select_kernel<W_, D_>), dim3(grid), dim3(64 * W_), 0,             \
                       stream_of(o->ocl), cfptr(Q.buf) + Q.off, (long long)Q.ld, Nq, nh, nhk, d, \
                       (const signed char *)(KC ? KC->ptr : nullptr), cfptr(KS), nblk, top,     \
                       (int *)SEL->ptr)
#define SELECT_WIDTH(W_)        \
    do {                        \
        if (d <= 32)            \
            SELECT_LAUNCH(W_, 8);  \
        else if (d <= 64)       \
            SELECT_LAUNCH(W_, 16); \
        else                    \
            SELECT_LAUNCH(W_, 32); \
    } while (0)
    if (nblk > 128 && rows < 4 * o->ocl->cu_count)
        SELECT_WIDTH(8);
    else
        SELECT_WIDTH(1);
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
    int Nk, nh, nhk, d, bs, sub, nblk, top, vec;
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

        if (a.vec) {
            for (int c = 4 * part4; c < d; c += 16) {
                const float4 x = *(const float4 *)(kp + c), y = *(const float4 *)(q + c);

                s = fmaf(x.x, y.x, s);
                s = fmaf(x.y, y.y, s);
                s = fmaf(x.z, y.z, s);
                s = fmaf(x.w, y.w, s);
            }
        }
        else {
            for (int c = part4; c < d; c += 4)
                s = fmaf(kp[c], q[c], s);
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

/* Few queries: a wave a unit. */
template <int DP> __global__ void __launch_bounds__(256) blk_direct_kernel(const blk_args a)
{
    __shared__ float sc[4][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long units = (long long)a.Nq * a.nh * a.top * a.sub;
    const long long u = (long long)blockIdx.x * 4 + wave;

    if (u >= units)
        return;
    const int sub = (int)(u % a.sub), slot = (int)(u / a.sub % a.top);
    const int row = (int)(u / a.sub / a.top), h = row % a.nh;
    const int *sel = a.SEL + ((long long)a.q0 * a.nh + row) * a.top;
    const int b = sel[slot];
    const bool twice = __any(lane < slot && sel[min(lane, a.top - 1)] == b);
    const int ss = a.bs / a.sub, k0 = b * a.bs + sub * ss;

    if (b < 0 || b >= a.nblk || twice || k0 >= a.Nk) {
        if (lane == 0)
            a.ml[u] = make_float2(-INFINITY, 0.0f);
        return;
    }
    blk_unit_f32(a, a.q0 + row / a.nh, h, k0, min(a.Nk, k0 + ss), a.part + u * DP, a.ml + u,
                 sc[wave]);
}

/* Many queries, first step: bit r of bits[kvh][b][t] says that row 64 t + r
 * (of the kv head's rows: query-major, its query heads within) lists block
 * b. A wave a tile, eight tiles a block of threads; entries that are no block
 * or a repeated one get an empty unit. */
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
        if (r < rows)
            for (int s = 0; s < a.top; s++) {
                const int b = sel[s];
                const bool is = b >= 0 && b < a.nblk;
                bool empty = !is && c0 == 0;

                if (is && b >= c0 && b < c1)
                    empty = atomicOr(&m[b - c0][wave], 1ull << lane) >> lane & 1;
                if (empty)
                    for (int j = 0; j < a.sub; j++)
                        a.ml[(row * a.top + s) * a.sub + j] = make_float2(-INFINITY, 0.0f);
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

/* Second step: a block of threads holds a unit's keys and values in LDS, both
 * split in three bf16 parts (split.h), and computes them for the rows that
 * list it, 32 a wave and turn. */
#define BLK_PIECE 2048 /* rows whose bits are read at a time */

template <int ND, int NB>
__global__ void __launch_bounds__(256, ND == 4 ? 1 : 2) blk_unit_kernel(const blk_args a)
{
    constexpr int DP = 32 * ND, CH = DP / 8, SB = 32 * NB, KC = SB / 8;
    constexpr int RW = 16 / CH < 1 ? 1 : 16 / CH;  /* K rows in 256 bytes */
    constexpr int RV = 16 / KC < 1 ? 1 : 16 / KC;  /* V rows */
    constexpr int PK = SB * CH;                    /* 16-byte chunks of a part */
    __shared__ split_u4 ks[3 * PK], vs[3 * PK];
    __shared__ int list[BLK_PIECE + 128];
    __shared__ int wsum[4];
    __shared__ float sc[4][64];
    __shared__ unsigned long long keep_s;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = a.nh / a.nhk, d = a.d;
    const int unit = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
    const int sub = unit % a.sub, b = unit / a.sub % a.nblk, kvh = unit / a.sub / a.nblk;
    const int ss = a.bs / a.sub, k0 = b * a.bs + sub * ss, n = min(a.Nk - k0, ss);
    const unsigned *bits = (const unsigned *)(a.bits + ((long long)kvh * a.nblk + b) * a.tiles);
    const int words = 2 * a.tiles; /* of 32 rows */
    const int nchunk = (words * 32 + BLK_PIECE - 1) / BLK_PIECE;
    const int c0 = (int)((long long)nchunk * piece / a.pieces);
    const int c1 = (int)((long long)nchunk * (piece + 1) / a.pieces);

    if (c0 >= c1)
        return;
    /* The last block's second unit may lie past the keys. */
    const bool nothing = n <= 0;

    if (tid < 64) {
        const bool in = tid < n && (!a.kmask || a.kmask[k0 + min(tid, n - 1)]);
        const unsigned long long k = __ballot(in);

        if (tid == 0)
            keep_s = k;
    }
    __syncthreads();
    const unsigned long long keep = keep_s;

    /* Keys and values that are left out are zero here: what they hold meets
     * probabilities of zero. */
    if (!nothing) {
        const float *K = a.K + k0 * a.ldk + (long long)kvh * d;
        const float *V = a.V + k0 * a.ldv + (long long)kvh * d;

        for (int e = tid; e < PK; e += 256) {
            const int key = e / CH, dd = e % CH * 8;
            const bool in = keep >> key & 1;
            const float *p = K + (long long)min(key, n - 1) * a.ldk;
            float x[8];
            split_u4 h, m, l;

#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = in && dd + j < d ? p[min(dd + j, d - 1)] : 0.0f;
            split8(x, 1.0f, h, m, l);
            const int at = key * CH + ((e % CH) ^ (key / RW % CH));

            ks[at] = h;
            ks[PK + at] = m;
            ks[2 * PK + at] = l;
        }
        /* Row dd of the transposed values: slot 8 c + j of it is the key that
         * register 8 (c / 2 % 2) + j of the scores' tile c / 4 holds in lane
         * half c % 2. */
        for (int e = tid; e < PK; e += 256) {
            const int dd = e % DP, c = e / DP;
            float x[8];
            split_u4 h, m, l;

#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = (c >> 1) * 16 + (j >> 2) * 8 + (c & 1) * 4 + (j & 3);
                const bool in = keep >> key & 1;

                x[j] = in && dd < d ? V[(long long)min(key, n - 1) * a.ldv + min(dd, d - 1)] : 0.0f;
            }
            split8(x, SPLIT_UP, h, m, l);
            const int at = dd * KC + (c ^ (dd / RV % KC));

            vs[at] = h;
            vs[PK + at] = m;
            vs[2 * PK + at] = l;
        }
    }

    auto tile = [&](const int *rows, int count) {
        const bool live = col < count;
        const int r = rows[live ? col : 0], qi = r / g, h = kvh * g + r % g;
        const long long row = (long long)qi * a.nh + h;
        const float *qp = a.Q + (a.q0 + qi) * a.ldq + (long long)h * d;
        const int *sel = a.SEL + ((long long)a.q0 * a.nh + row) * a.top;
        const float up = a.scale * BLK_LOG2E * BLK_QUP;
        split_u4 q[2 * ND][3];
        split_f16x s[NB], o[ND], low[ND];
        constexpr int pa[6] = {0, 2, 1, 0, 1, 0}, pb[6] = {2, 0, 1, 1, 0, 0};
        int slot = 0;

        while (slot < a.top - 1 && sel[slot] != b)
            slot++;
#pragma unroll
        for (int st = 0; st < 2 * ND; st++) {
            const int dd = st * 16 + half * 8;
            float x[8];

            if (a.vec) {
                const float4 u = *(const float4 *)(qp + min(dd, d - 4));
                const float4 v = *(const float4 *)(qp + min(dd + 4, d - 4));

                x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
                x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
            }
            else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    x[j] = qp[min(dd + j, d - 1)];
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = dd + j < d ? x[j] * up : 0.0f;
            split8(x, 1.0f, q[st][0], q[st][1], q[st][2]);
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

#pragma unroll
        for (int t = 0; t < NB; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int kk = 32 * t + (e >> 2) * 8 + half * 4 + (e & 3);

                p[t][e] = keep >> kk & 1 ? s[t][e] * (1.0f / BLK_QUP) : -INFINITY;
                mx = fmaxf(mx, p[t][e]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float ref = mx == -INFINITY ? 0.0f : mx;

#pragma unroll
        for (int t = 0; t < NB; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                p[t][e] = __builtin_amdgcn_exp2f(p[t][e] - ref);
                l += p[t][e];
            }
        l += __shfl_xor(l, 32, 64);
#pragma unroll
        for (int tt = 0; tt < ND; tt++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                o[tt][e] = low[tt][e] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2 * NB; u++) {
            float x[8];
            split_u4 pp[3];

#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = p[u / 2][8 * (u % 2) + j];
            split8(x, SPLIT_UP, pp[0], pp[1], pp[2]);
#pragma unroll
            for (int tt = 0; tt < ND; tt++) {
                const int dd = tt * 32 + col;
                split_b8 vf[3];

#pragma unroll
                for (int k = 0; k < 3; k++)
                    vf[k] = __builtin_bit_cast(
                        split_b8, vs[k * PK + dd * KC + ((2 * u + half) ^ (dd / RV % KC))]);
#pragma unroll
                for (int w = 0; w < 6; w++) {
                    split_f16x &c = w == 5 ? o[tt] : low[tt];

                    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        vf[pa[w]], __builtin_bit_cast(split_b8, pp[pb[w]]), c, 0, 0, 0);
                }
            }
        }
        float z = l * 0.0f;

#pragma unroll
        for (int tt = 0; tt < ND; tt++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                o[tt][e] += low[tt][e];
                z = fmaf(o[tt][e], 0.0f, z);
            }
        const long long at = (row * a.top + slot) * a.sub + sub;
        /* Infinities, NaN and values that have no split: again in float32. So
         * are scores below the range of the split. */
        const bool again = z != 0.0f || (l == 0.0f && keep);
        const unsigned long long redo = __ballot(again && live);

        if (live && !(redo >> col & 1) && !(redo >> (col + 32) & 1)) {
            float *out = a.part + at * DP;

#pragma unroll
            for (int tt = 0; tt < ND; tt++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    *(float4 *)(out + tt * 32 + e * 8 + half * 4) =
                        make_float4(o[tt][4 * e] * SPLIT_DOWN, o[tt][4 * e + 1] * SPLIT_DOWN,
                                    o[tt][4 * e + 2] * SPLIT_DOWN, o[tt][4 * e + 3] * SPLIT_DOWN);
            if (half == 0)
                a.ml[at] = make_float2(mx, l);
        }
        if (redo)
            for (int e = 0; e < count; e++)
                if ((redo >> e | redo >> (e + 32)) & 1) {
                    const int rr = rows[e], qq = rr / g;
                    const long long to =
                        (long long)(unsigned)__builtin_amdgcn_readlane((int)(at & 0xffffffff), e) |
                        (long long)__builtin_amdgcn_readlane((int)(at >> 32), e) << 32;

                    blk_unit_f32(a, a.q0 + qq, kvh * g + rr % g, k0, k0 + n, a.part + to * DP,
                                 a.ml + to, sc[wave]);
                }
    };

    int have = 0;

    for (int c = c0; c < c1; c++) {
        /* 8 rows a thread: their bits, the place of the first of them. */
        const int r0 = c * BLK_PIECE + 8 * tid, w = r0 >> 5;
        unsigned m = w < words ? bits[w] >> (r0 & 31) & 0xffu : 0u;
        int p = __popc(m), before = 0;

#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int v = __shfl_up(p, s, 64);

            p += lane >= s ? v : 0;
        }
        if (lane == 63)
            wsum[wave] = p;
        __syncthreads();
        for (int i = 0; i < wave; i++)
            before += wsum[i];
        const int added = wsum[0] + wsum[1] + wsum[2] + wsum[3];
        int at = have + before + p - __popc(m);

        while (m) {
            list[at++] = r0 + __ffs(m) - 1;
            m &= m - 1;
        }
        have += added;
        __syncthreads();
        /* Whole turns of 4 waves, the rest with the next rows. */
        const int todo = c + 1 == c1 ? have : have / 128 * 128;

        for (int e = wave * 32; e < todo; e += 128) {
            if (nothing) {
                if (lane < min(32, todo - e)) {
                    const int r = list[e + lane], h = kvh * g + r % g;
                    const long long row = (long long)(r / g) * a.nh + h;
                    const int *sel = a.SEL + ((long long)a.q0 * a.nh + row) * a.top;
                    int slot = 0;

                    while (slot < a.top - 1 && sel[slot] != b)
                        slot++;
                    a.ml[(row * a.top + slot) * a.sub + sub] = make_float2(-INFINITY, 0.0f);
                }
            }
            else
                tile(list + e, min(32, todo - e));
        }
        __syncthreads();
        const int rest = have - todo, keepv = tid < rest ? list[todo + tid] : 0;

        __syncthreads();
        if (tid < rest)
            list[tid] = keepv;
        have = rest;
    }
}

/* Units of a row merged: softmax over all of them from their maxima and
 * sums, in the order of the list. Four channels a thread. */
template <int DP> __global__ void __launch_bounds__(256) blk_merge_kernel(const blk_args a)
{
    const int units = a.top * a.sub;
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = e / (DP / 4);
    const int c = (int)(e % (DP / 4)) * 4, d = a.d;

    if (row >= (long long)a.Nq * a.nh || c >= d)
        return;
    const float2 *ml = a.ml + row * units;
    const float *part = a.part + row * units * DP + c;
    float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};

    for (int u = 0; u < units; u++)
        if (ml[u].y != 0.0f)
            m = fmaxf(m, ml[u].x);
    for (int u = 0; u < units; u++) {
        const float2 x = ml[u];

        if (x.y == 0.0f)
            continue;
        const float w = __builtin_amdgcn_exp2f(x.x - m);
        const float4 p = *(const float4 *)(part + (long long)u * DP);

        l = fmaf(x.y, w, l);
        o[0] = fmaf(p.x, w, o[0]);
        o[1] = fmaf(p.y, w, o[1]);
        o[2] = fmaf(p.z, w, o[2]);
        o[3] = fmaf(p.w, w, o[3]);
    }
    float *out = a.O + (a.q0 + row / a.nh) * a.ldo + (row % a.nh) * d + c;

#pragma unroll
    for (int j = 0; j < 4; j++)
        if (c + j < d)
            out[j] = l == 0.0f ? 0.0f : o[j] / l;
}

/* The passes of a call: queries a pass, and what one needs of the work
 * buffer. */
struct blk_plan {
    bool direct;
    int pass, tiles, dp, sub, nblk;
    long long part, ml, bits; /* bytes */
};

#define BLK_PART_BYTES (256LL << 20)

static blk_plan blk_plan_of(int Nq, int Nk, int nh, int nhk, int d, int bs, int top)
{
    blk_plan p;
    const int g = nh / nhk;

    p.nblk = ops_key_blocks(Nk, bs);
    p.sub = blk_sub(bs);
    p.dp = d <= 32 ? 32 : d <= 64 ? 64 : 128;
    const long long row = (long long)top * p.sub * (p.dp + 2) * 4; /* bytes a row */
    const long long most = max(1LL, BLK_PART_BYTES / (row * nh));

    p.pass = (int)min((long long)Nq, max(most, 512LL));
    p.direct = p.nblk == 0 || (long long)p.pass * g * top < 16LL * max(p.nblk, 1) ||
               (long long)Nq * nh * top <= 4096;
    p.tiles = ((p.pass * g + 63) / 64 + BLK_TW - 1) / BLK_TW * BLK_TW;
    p.part = (long long)p.pass * nh * top * p.sub * p.dp * 4;
    p.ml = (long long)p.pass * nh * top * p.sub * 8;
    p.bits = p.direct ? 0 : (long long)nhk * p.nblk * p.tiles * 8;
    return p;
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
    const blk_plan p = blk_plan_of(Nq, Nk, nh, nhk, d, bs, top);

    return (size_t)(p.part + p.ml + p.bits);
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
    need_apart(SEL, 0, (long long)Nq * nh * top * 4, work, 0, wbytes, op, "SEL and work");
    count32((long long)p.pass * nh * top * p.sub, "units of a pass");

    blk_args a = {};
    auto al = [](const float *q, int ld) { return ((uintptr_t)q & 15) == 0 && ld % 4 == 0; };

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
    a.vec = d % 4 == 0 && al(a.Q, Q.ld) && (!Nk || (al(a.K, K.ld) && al(a.V, V.ld)));
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
            const dim3 grid((unsigned)count32((units + 3) / 4, "units"));

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
            /* Splits of a list: enough blocks of threads, each of which has
             * some 256 rows to compute. */
            const long long each = max(1LL, (long long)a.Nq * g * top / p.nblk / 256);
            const int chunks = (a.tiles * 64 + BLK_PIECE - 1) / BLK_PIECE;

            a.pieces = (int)max(1LL, min(min(each, (long long)chunks),
                                         (4LL * o->ocl->cu_count + lists - 1) / lists));
            hipLaunchKernelGGL(blk_bits_kernel, dim3(a.tiles / BLK_TW, nhk), dim3(64 * BLK_TW), 0, s,
                               a);
            launch_check("attention_blocks bits");
            const dim3 grid((unsigned)count32((long long)lists * a.pieces, "lists"));

#define UNIT_LAUNCH(ND_)                                                                  \
    do {                                                                                  \
        if (bs / p.sub <= 32)                                                             \
            hipLaunchKernelGGL((blk_unit_kernel<ND_, 1>), grid, dim3(256), 0, s, a);      \
        else                                                                              \
            hipLaunchKernelGGL((blk_unit_kernel<ND_, 2>), grid, dim3(256), 0, s, a);      \
    } while (0)
            if (p.dp == 32)
                UNIT_LAUNCH(1);
            else if (p.dp == 64)
                UNIT_LAUNCH(2);
            else
                UNIT_LAUNCH(4);
#undef UNIT_LAUNCH
            launch_check("attention_blocks units");
        }
        const dim3 grid((unsigned)count32((rows * (p.dp / 4) + 255) / 256, "merge"));

        if (p.dp == 32)
            hipLaunchKernelGGL(blk_merge_kernel<32>, grid, dim3(256), 0, s, a);
        else if (p.dp == 64)
            hipLaunchKernelGGL(blk_merge_kernel<64>, grid, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL(blk_merge_kernel<128>, grid, dim3(256), 0, s, a);
        launch_check("attention_blocks merge");
    }
    ICOREG_API_END
}
