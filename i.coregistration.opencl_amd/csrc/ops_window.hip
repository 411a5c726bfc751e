/* SPDX-License-Identifier: Unlicense */

/* Attention within a window and over the first keys: a query at position p
 * sees the keys p - left .. p + right and those of the first `sinks` that are
 * not behind p + right; of float32 keys and values, or of the 8-bit ones of a
 * cache (seqs.h, q8.h), there with right = 0 and the queries of several
 * sequences in one call.
 *
 * One pass over the keys: with the running maximum m of a row's scores s
 * (scale and log2 e in the query), the sum l of 2^(s - m) and the output o of
 * 2^(s - m) v, a larger maximum m' multiplies l and o by 2^(m - m') and the
 * result is o / l. Any m serves that keeps the powers in range, so it is
 * raised only when a score passes it by WIN_TAU.
 *
 * A cache's value is scale times code: the scale goes with the weight, and the
 * products take codes, which are exact in 16 bits. float32 operands are sums of
 * parts of 16 bits, as the matrix instructions of float32 have a 16th of the
 * rate: three bf16 parts for few rows (all 24 bits, split.h; memory bounds
 * them), two f16 parts for tiles of many (22 bits, a row and head brought to
 * 2^14 .. 2^15 by a power of two; three products instead of six).
 *
 * The keys that any row of a tile of rows sees are one or two runs of tiles of
 * keys (win_span); no others are read. Where rows do not fill the CUs, the
 * tiles of keys are split over blocks of threads, maximum, sum and unnormalised
 * output of each to the work buffer, and a second kernel joins them. */

#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "load4.h"
#include "ops.h"
#include "reduce.h"
#include "seqs.h"
#include "split.h"

using namespace icoreg;

#define WIN_LOG2E 1.4426950408889634f
#define WIN_MAX_KEYS 0x7fffff00 /* keys are counted in int, a tile past the last too */
#define WIN_MAX_SPLITS 256
#define WIN_PART_ROWS (1LL << 17) /* rows of partial results at most */
#define WIN_WRITTEN (-1.0f)       /* a sum of this: the output is in its place */

struct win_args {
    const float *Q;
    float *O;
    const float *K, *V; /* float32 keys and values, or the cache c */
    const unsigned char *kmask;
    cache_view c;
    long long ldq, ldk, ldv, ldo;
    int Nk, q0, rows, nh, nhk, d, left, right, sinks, splits;
    float scale;
    float *part; /* (row nh + head) splits + split, DP floats each */
    float2 *ml;
};

/* A row's sequence and position, and the keys of its sequence. */
struct win_row {
    int b, p, nk;
};

/* Tiles of KT keys that positions p_lo .. p_hi see any key of: tiles 0 .. st -
 * 1 and wt .. wt + n - st - 1, n in all. */
struct win_tiles {
    int st, wt, n;
    __device__ __forceinline__ int tile(int i) const { return i < st ? i : wt + i - st; }
};

/* The last and the first key of the window of position p; hi < 0 or lo > hi:
 * none. */
static __device__ __forceinline__ int win_hi(const win_args &a, int p, int nk)
{
    return a.right < 0 || p > nk - 1 - a.right ? nk - 1 : p + a.right;
}

static __device__ __forceinline__ int win_lo(const win_args &a, int p)
{
    return a.left < 0 || p <= a.left ? 0 : p - a.left;
}

/* The lowest n of 32 bits (n < 0: none). */
static __device__ __forceinline__ unsigned win_below(int n)
{
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
}

/* x where bit `bit` of see is set, else minus infinity: a field and a bitwise
 * choice, where 16 conditions would fill the scalar registers. */
static __device__ __forceinline__ float win_if(unsigned see, int bit, float x)
{
    const unsigned on = (unsigned)__builtin_amdgcn_sbfe((int)see, bit, 1);

    return __builtin_bit_cast(float, (on & __builtin_bit_cast(unsigned, x)) | (~on & 0xff800000u));
}

/* Bit i: a row of window lo .. hi sees key k0 + i, if it is kept. */
static __device__ __forceinline__ unsigned win_sees(const win_args &a, int lo, int hi, int k0)
{
    return win_below(hi - k0 + 1) & (~win_below(lo - k0) | win_below(a.sinks - k0));
}

template <int KT>
static __device__ __forceinline__ win_tiles win_span(const win_args &a, int p_lo, int p_hi, int nk)
{
    const int hi = win_hi(a, p_hi, nk), lo = win_lo(a, p_lo);
    win_tiles t = {0, 0, 0};

    if (hi < 0)
        return t;
    t.st = (min(a.sinks, hi + 1) + KT - 1) / KT;
    if (lo > hi) {
        t.n = t.st;
        return t;
    }
    t.wt = lo / KT;
    if (t.st >= t.wt && t.st > 0)
        t.st = t.wt = 0;
    t.n = t.st + hi / KT - t.wt + 1;
    return t;
}

/* One row and head over the tiles t0 .. t1 - 1 of KT <= 64 keys, in float32, by a
 * wave: lane k has key k's score, then every 64th channel. Seen keys alone are
 * read for the output, whatever the others hold. p: 64 floats of LDS of this
 * wave. Output unnormalised, o[j] channel lane + 64 j. */
template <bool CACHE, int KT>
static __device__ __forceinline__ void win_row_f32(const win_args &a, const win_row &r, int row, int h,
                                                   const win_tiles &t, int t0, int t1, float *ps,
                                                   float (&o)[2], float &m, float &l)
{
    const int lane = threadIdx.x & 63, kvh = h / (a.nh / a.nhk), d = a.d;
    const float *q = a.Q + row * a.ldq + (long long)h * d;
    const int hi = win_hi(a, r.p, r.nk), lo = win_lo(a, r.p);

    m = -INFINITY;
    l = o[0] = o[1] = 0.0f;
    for (int i = t0; i < t1; i++) {
        const int k0 = t.tile(i) * KT, k = k0 + lane;
        bool see = lane < KT && k <= hi && (k >= lo || k < a.sinks);
        long long at = 0;

        if (CACHE) {
            const int page = see ? seq_page(a.c, r.b, k) : -1;

            see = page >= 0;
            at = see ? cache_row(a.c, page, kvh, k) : 0;
        }
        else if (a.kmask)
            see = see && a.kmask[k];
        const unsigned long long seen = __ballot(see);

        if (!seen)
            continue;
        float s = 0.0f;

        if (see) {
            if (CACHE) {
                for (int c = 0; c < d; c += 4) {
                    const int w = *(const int *)(a.c.kc + at * a.c.pitch + c);
                    float x[4];

                    load4_row(q, c, d, x);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s = fmaf(x[j], (float)(w << (24 - 8 * j) >> 24), s);
                }
                s *= a.c.ks[at];
            }
            else {
                const float *kp = a.K + k * a.ldk + (long long)kvh * d;

                for (int c = 0; c < d; c += 4) {
                    float x[4], y[4];

                    load4_row(q, c, d, x);
                    load4_row(kp, c, d, y);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s = fmaf(x[j], y[j], s);
                }
            }
        }
        s = see ? s * (a.scale * WIN_LOG2E) : -INFINITY;
        const bool nan = __any(s != s);
        const float mn = fmaxf(m, wave_max_full(s));
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float corr = __builtin_amdgcn_exp2f(m - ref);
        const float p = __builtin_amdgcn_exp2f(s - ref);

        m = mn;
        l = nan ? __builtin_nanf("") : fmaf(l, corr, wave_sum_full(p));
        o[0] *= corr;
        o[1] *= corr;
        /* A cache's value is code times scale: the scale goes with the weight. */
        ps[lane] = CACHE && see ? p * a.c.vs[at] : p;
        __builtin_amdgcn_wave_barrier();
        for (unsigned long long left = seen; left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            const float w = ps[j];

            if (CACHE) {
                const long long to = (long long)__builtin_amdgcn_readlane((int)(at >> 32), j) << 32 |
                                     (unsigned)__builtin_amdgcn_readlane((int)at, j);
                const signed char *v = a.c.vc + to * a.c.pitch;

#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (lane + 64 * e < d)
                        o[e] = fmaf(w, (float)v[lane + 64 * e], o[e]);
            }
            else {
                const float *v = a.V + (k0 + j) * a.ldv + (long long)kvh * d;

#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (lane + 64 * e < d)
                        o[e] = fmaf(w, v[lane + 64 * e], o[e]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (l != l)
        m = 0.0f; /* NaN, whatever the other parts are */
}

/* What win_row_f32 leaves, to its place: the output, or a part of it. */
static __device__ __forceinline__ void win_put(const win_args &a, long long row, int h, int split, int parts,
                                               const float (&o)[2], float m, float l)
{
    const int lane = threadIdx.x & 63, dp = a.d <= 32 ? 32 : a.d <= 64 ? 64 : 128;
    const long long u = (row * a.nh + h) * a.splits + split;
    float *to = parts == 1 ? a.O + row * a.ldo + (long long)h * a.d : a.part + u * dp;

#pragma unroll
    for (int e = 0; e < 2; e++)
        if (lane + 64 * e < a.d)
            to[lane + 64 * e] = parts > 1 ? o[e] : l == 0.0f ? 0.0f : o[e] / l;
    if (lane == 0 && a.splits > 1)
        a.ml[u] = parts == 1 ? make_float2(0.0f, WIN_WRITTEN) : make_float2(m, l);
}

/* Parts that the tiles of keys are split into, of at most `splits`: at least
 * two tiles each. */
static __device__ __forceinline__ int win_parts(int tiles, int splits)
{
    return min(splits, max(1, tiles / 2));
}

/* ---- a tile of rows ---------------------------------------------------------------- */

typedef _Float16 win_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 win_h8 __attribute__((ext_vector_type(8)));
typedef float win_f2 __attribute__((ext_vector_type(2)));
typedef float win_f16x __attribute__((ext_vector_type(16)));
typedef unsigned win_u4 __attribute__((ext_vector_type(4)));

#define WIN_KT 64       /* keys of a tile; 32 of float32 ones of 128 channels, whose parts fill LDS */
#define WIN_AHEAD 2     /* operands on their way from LDS; 3 and 4 measured the same */
#define WIN_TAU 4.0f    /* the running maximum is raised when a score passes it by this (base 2) */
#define WIN_VEXP 10     /* exponent of the largest value scale: weights up to 2^TAU stay below 2^16 */
#define WIN_VMIN 0.125f /* smaller ones lose bits: 2^13 below the largest */
/* Biased exponents of the largest key whose products with a query of 2^14 ..
 * 2^15 stay finite when the key's power of two is put back, the query's own
 * not yet: 128 products of 2^31 (2^22 of codes) times 2^(WIN_KEXP - 141), or a
 * cache's scale of 2^(WIN_SEXP - 126). Above that a sum might be infinite
 * below, a weight of 0, where the score is not. */
#define WIN_KEXP 229
#define WIN_SEXP 223
/* A query's or key's parts are off by 2^-22 of each channel's value or, of those
 * far below the largest (2^14 .. 2^15 as they are scaled), by 2^-25: of d
 * channels, with f and s the powers of two of query and key, a score by no more
 * than d f s 2^15 2^-25 for each of the two, or, of codes, which are exact and
 * below 2^7 s, d f s 2^7 2^-25 for the query's. Rows for which that passes
 * WIN_LOST with the largest key of the tiles they look at are done again: 128
 * normally distributed channels have 2^-29, and 2^-20 where the largest query
 * times the largest key is 2^9 times as much beside the others. */
#define WIN_LOST 0x1p-20f

/* Codes of 8 bits in f16, exactly: a byte u = code + 128 behind 0x64 is the
 * f16 value 1024 + u. */
static __device__ __forceinline__ unsigned win_codes(unsigned bytes)
{
    const win_h2 x = __builtin_bit_cast(win_h2, bytes), off = {(_Float16)-1152.0f, (_Float16)-1152.0f};

    return __builtin_bit_cast(unsigned, x + off);
}

/* The power of two of biased exponent e, 1 .. 254. */
static __device__ __forceinline__ float win_power(int e) { return __builtin_bit_cast(float, (unsigned)e << 23); }

/* Two floats as the sum of two f16 values each, 11 bits and 11 more. */
static __device__ __forceinline__ void win_split(float a, float b, unsigned &hi, unsigned &lo)
{
    const win_f2 v = {a, b};
    const win_h2 h = __builtin_convertvector(v, win_h2);
    const win_f2 r = {__builtin_fmaf((float)h[0], -1.0f, a), __builtin_fmaf((float)h[1], -1.0f, b)};

    hi = __builtin_bit_cast(unsigned, h);
    lo = __builtin_bit_cast(unsigned, __builtin_convertvector(r, win_h2));
}

/* What a block of threads computes: rows r0 .. r0 + n - 1 (query-major, the g
 * heads of key head kvh within) of a sequence of nk keys whose first row of
 * the operands is `first`, at position p0. n = 0: none. */
struct win_job {
    int b, kvh, r0, n, first, p0, nk;
};

template <bool CACHE, int TR>
static __device__ __forceinline__ win_job win_job_of(const win_args &a, int tile, int kvh)
{
    const int g = a.nh / a.nhk;
    win_job j = {0, kvh, 0, 0, 0, 0, 0};

    if (!CACHE) {
        j.r0 = tile * TR;
        j.n = (int)min((long long)a.rows * g - j.r0, (long long)TR);
        j.p0 = a.q0;
        j.nk = a.Nk;
        return j;
    }
    /* Sequence b has the tiles of TR rows from start[b] g / TR + b on, one more than
     * it can need; the last that starts at or before this one: of 64 places of
     * what is left of the sequences, until that is 64 of them, each lane with
     * all that is known of one. None: the tile is of rows before the first
     * sequence. */
    const int lane = threadIdx.x & 63;
    int b0 = 0, left = a.c.n;

    while (left > 64) {
        const int step = (left + 63) / 64, b = b0 + lane * step;
        const bool in = lane * step < left;
        const int n = __popcll(__ballot(in && (long long)seq_start(a.c, in ? b : b0) * g / TR + b <= tile));

        if (n == 0)
            return j;
        b0 += (n - 1) * step;
        left = min(step, left - (n - 1) * step);
    }
    const int b = b0 + min(lane, left - 1), s0 = seq_start(a.c, b), s1 = seq_start(a.c, b + 1), l = a.c.len[b];
    const int n = __popcll(__ballot(lane < left && (long long)s0 * g / TR + b <= tile));

    if (n == 0)
        return j;
    j.b = b0 + n - 1;
    j.first = __builtin_amdgcn_readlane(s0, n - 1);
    const int end = __builtin_amdgcn_readlane(s1, n - 1), len = max(__builtin_amdgcn_readlane(l, n - 1), 0);
    const long long from = (long long)j.first * g / TR + j.b;
    const int rows = max(end - j.first, 0);

    j.r0 = (int)(tile - from) * TR;
    j.n = (int)min((long long)rows * g - j.r0, (long long)TR);
    j.p0 = len - rows;
    j.nk = (int)min((long long)len, (long long)a.c.ldt << a.c.page_log);
    return j;
}

/* A wave's 32 rows to their places, `down` times the accumulators; rows to do
 * again (a sum that is not finite, values that the matrix instructions' parts
 * cannot hold) in float32. */
template <int ND, bool CACHE, int KT>
static __device__ __forceinline__ void win_finish(const win_args &a, const win_job &jb, const win_tiles &span, int t0,
                                                  int t1, int parts, int split, const win_f16x (&o)[ND], float down,
                                                  float m, float l, bool again, float *ps, int d)
{
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, g = a.nh / a.nhk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), last = jb.r0 + jb.n - 1;
    const int wr = jb.r0 + 32 * wave, r = min(wr + col, last), qi = r / g, h = jb.kvh * g + r - qi * g;
    const bool mine = wr + col <= last, direct = parts == 1;
    const long long row = jb.first + qi, out = (row * a.nh + h) * a.splits + split;
    unsigned long long redo = __ballot(again && mine);

    redo = (redo | redo >> 32) & 0xffffffffull;
    if (mine && !(redo >> col & 1)) {
        const float inv = direct ? (l > 0.0f ? down / l : 0.0f) : down;
        float *to = direct ? a.O + row * a.ldo + (long long)h * d : a.part + out * (32 * ND);

#pragma unroll
        for (int tt = 0; tt < ND; tt++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int c = 32 * tt + 2 * e + 4 * half;

                if (c + 4 <= d)
                    store4(to + c, o[tt][e] * inv, o[tt][e + 1] * inv, o[tt][e + 2] * inv, o[tt][e + 3] * inv);
                else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (c + j < d)
                            to[c + j] = o[tt][e + j] * inv;
                }
            }
        if (half == 0 && a.splits > 1)
            a.ml[out] = direct ? make_float2(0.0f, WIN_WRITTEN) : make_float2(m, l);
    }
    for (; redo; redo &= redo - 1) {
        const int rr = wr + __builtin_ctzll(redo), q1 = rr / g, h1 = jb.kvh * g + rr - q1 * g;
        const win_row wrow = {jb.b, jb.p0 + q1, jb.nk};
        float y[2], m1, l1;

        win_row_f32<CACHE, KT>(a, wrow, jb.first + q1, h1, span, t0, t1, ps, y, m1, l1);
        win_put(a, jb.first + q1, h1, split, parts, y, m1, l1);
    }
}

/* A block's split, key head and tile of `tiles`: tiles from the last one down,
 * which where later rows see more are the longest, so that the short ones fill
 * the CUs' gaps at the end; key heads within, so that an XCD (blocks are dealt
 * to the 8 in turn) has few of them in its L2 where their number has a factor
 * in common with 8. */
static __device__ __forceinline__ int win_unit(const win_args &a, int tiles, int &split, int &kvh)
{
    const int per = a.nhk * a.splits, u = blockIdx.x % per;

    split = u / a.nhk;
    kvh = u % a.nhk;
    return tiles - 1 - blockIdx.x / per;
}

/* Channels of a head: any number (a load a float), a multiple of 4, or all
 * that the kernel has room for. */
enum { WIN_ANY, WIN_FOUR, WIN_FULL };

/* Floats c .. c + 3 of a row of d; behind the last channel some of them again,
 * for products with zeros and sums that are not stored. */
template <int CHANNELS>
static __device__ __forceinline__ void win_load4(const float *p, int c, int d, float (&x)[4])
{
    if (CHANNELS == WIN_FULL)
        load4(p + c, x);
    else if (CHANNELS == WIN_FOUR)
        load4(p + min(c, d - 4), x);
    else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            x[j] = p[min(c + j, d - 1)];
    }
}

#define WIN_NONE 0   /* exponent of the value scales before the first */
#define WIN_LAG 12   /* a row's scale is at most 2^12 below the largest so far, its values smaller instead */
#define WIN_DEEP 14  /* float32 values keep 22 bits 2^14 below that */
#define WIN_CODES 24 /* codes keep all 2^24 below */

typedef short win_s4 __attribute__((ext_vector_type(4)));
typedef _Float16 win_h4 __attribute__((ext_vector_type(4)));

typedef unsigned short win_us2 __attribute__((ext_vector_type(2)));

/* Largest of a wave's upper and of its lower 16 bits, each. */
static __device__ __forceinline__ unsigned win_wave_max2(unsigned v)
{
    auto larger = [](unsigned x, unsigned y) {
        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(win_us2, x),
                                                                      __builtin_bit_cast(win_us2, y)));
    };

    v = larger(v, (unsigned)dpp_i((int)v, 0xB1));
    v = larger(v, (unsigned)dpp_i((int)v, 0x4E));
    v = larger(v, (unsigned)dpp_i((int)v, 0x141));
    v = larger(v, (unsigned)dpp_i((int)v, 0x140));
    return larger(larger((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
                  larger((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}

/* The larger of lane l's and lane l ^ 32's: the halves swapped between two
 * copies, which leaves both values in every lane. */
static __device__ __forceinline__ float win_halves(float v)
{
    const unsigned b = __builtin_bit_cast(unsigned, v);
    const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    /* Copies: a bit cast of a vector's element takes the first one. */
    const unsigned x = s[0], y = s[1];

    return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

/* Largest of the L lanes of a row, L = 4, 8 or 16. */
template <int L> static __device__ __forceinline__ unsigned win_row_max(unsigned v)
{
    v = max(v, (unsigned)dpp_i((int)v, 0xB1));
    v = max(v, (unsigned)dpp_i((int)v, 0x4E));
    if (L > 4)
        v = max(v, (unsigned)dpp_i((int)v, 0x141));
    if (L > 8)
        v = max(v, (unsigned)dpp_i((int)v, 0x140));
    return v;
}

/* NW / KG waves of 32 rows, KT keys at a time. KG = 2: half of the waves takes
 * the first 32 of them and half the others, joined at the end.
 *
 * v_mfma_f32_32x32x16_f16 with the keys as rows and the queries as columns: a
 * lane has 16 scores of one query, its maximum and sum need one exchange with
 * lane ^ 32, and the weights are the second product's operand as they lie;
 * values come to it transposed by the LDS read. Keys and values are made f16
 * once for all rows of the block, as they go from registers to one of two LDS
 * tiles, while the next tile's loads are on their way: one barrier a tile.
 * PW > 0: by waves that do nothing else, beside the others' products. Us:
 *
 *   channels, call                                  without   with
 *   64, 1601 tokens of 16 heads, window 321            27.1   24.3
 *   64, 16000 tokens of 4 heads, window 201              39     35
 *   64, 16000 tokens of 4 heads, window 2001            142    124
 *   64, cache, 2 x 4096 new tokens of 8192              309    270
 *   32, 6400 tokens of 8 heads, window 641               39     61
 *
 * With 32 channels they take the place of a second block on a CU; with 128 the
 * registers (168 of a wave) do not suffice. Rows are query-major, the heads of a
 * key head within, so that these share its keys.
 *
 * Weights are two f16 parts, p times the value scale relative to the largest
 * one so far (exponent vexp, to 2^WIN_VEXP): 22 bits of those over 2^-13 of it,
 * 2^-35 of it else. Sums, maxima and outputs are float32. Rows for which that
 * is not enough (win_finish's `again`) are computed by win_row_f32.
 *
 * Bound by the instructions that two waves a SIMD issue: 3 sequences of up to 4096
 * new tokens of 8192, 16 heads on 4 of 128 channels: 785 us, 1020
 * TFLOP/s of f16 products, matrix instructions 44 % and vector ones 42 % of
 * the cycles; a large matrix product of f16 has 1309 TFLOP/s. 16380 float32
 * tokens, window 2048: 870 us, 890 TFLOP/s. 1601 tokens of 16 heads of 64,
 * window 321: 24 us, of which prologue, join and stores 6. A tile's phases held
 * apart between the halves of the waves by barriers: 837 us for the first, 775 then
 * without.
 */
template <int ND, bool CACHE, int CHANNELS, int NW, int KG, int KT, int PW>
__global__ void __launch_bounds__(64 * (NW + PW), PW ? 3 : ND == 1 ? 4 : 2) win_tile_kernel(const win_args a)
{
    constexpr int DP = 32 * ND, CH = DP / 8, P = CACHE ? 1 : 2; /* channels, 16-byte chunks of a key, f16 parts */
    /* Chunks between keys in LDS: 16 neighbouring keys' chunks of one place, as
     * the scores' operands are read, and 4 neighbouring keys' 64 bytes, as the
     * outputs' are, lie in banks of their own. */
    constexpr int KS = CH + 1, VS = ND == 1 ? 4 : CH + 4;
    constexpr int HT = 32 * NW;                  /* threads that stage keys, and values */
    static_assert(PW == 0 || 64 * PW == HT, "a unit's thread");
    constexpr int UC = CACHE ? CH / 2 : CH;      /* units of a key: 16 codes, or 8 floats */
    constexpr int U = KT * UC, NU = (U + HT - 1) / HT, RW = CACHE ? 4 : 8;
    constexpr bool SAME = 64 / UC <= 16;         /* a wave's units lie in one run of 16 keys */
    struct tile_lds {
        win_u4 k[P * KT * KS], v[P * KT * VS];
        float ks[KT], vs[KT];
        unsigned long long keep;
        /* Largest and smallest scale of a wave's values, exponents; zero: some
         * are zeros alone. */
        int top[NW / 2], low[NW / 2], zero[NW / 2], wild, lag;
    };
    constexpr int RG = NW / KG, TR = 32 * RG;    /* waves of rows, rows */
    static_assert((KT == 64 || !CACHE) && KT >= 32 * KG, "a lane a key, 32 keys a wave");
    __shared__ tile_lds lds[2];
    __shared__ float ps[NW][64];
    __shared__ unsigned most_k[NW][64]; /* largest key scale of the tiles that a wave looked at, as bits */
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool mover = wave >= NW; /* one of PW */
    const int g = a.nh / a.nhk, d = CHANNELS == WIN_FULL ? DP : a.d, pitch = a.c.pitch;
    const long long rows = (long long)a.rows * g;
    const int tiles = (int)(CACHE ? rows / TR + a.c.n : (rows + TR - 1) / TR);
    int split, kvh;
    const int tile = win_unit(a, tiles, split, kvh);
    const win_job jb = win_job_of<CACHE, TR>(a, tile, kvh);

    if (jb.n <= 0)
        return;
    const int last = jb.r0 + jb.n - 1;
    const win_tiles span = win_span<KT>(a, jb.p0 + jb.r0 / g, jb.p0 + last / g, jb.nk);
    const int parts = win_parts(span.n, a.splits);
    /* This lane's row; lanes without one take the last. */
    const int rg = wave % RG, kg = wave / RG;
    const int wr = jb.r0 + 32 * rg, r = min(wr + col, last), qi = r / g, h = jb.kvh * g + r - qi * g;
    const long long row = jb.first + qi;

    if (split >= parts) {
        if (wr + col <= last && half == 0 && kg == 0)
            a.ml[(row * a.nh + h) * a.splits + split] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const int t0 = (int)((long long)span.n * split / parts), t1 = (int)((long long)span.n * (split + 1) / parts);
    const int p = jb.p0 + qi, hi = win_hi(a, p, jb.nk), lo = win_lo(a, p);
    /* Those of the wave's first and last row, and whether it has any. */
    const bool live = wr <= last && !mover;
    const int pa = jb.p0 + min(wr, last) / g, pb = jb.p0 + min(wr + 31, last) / g;
    const int hi0 = win_hi(a, pa, jb.nk), hi1 = win_hi(a, pb, jb.nk), lo0 = win_lo(a, pa), lo1 = win_lo(a, pb);
    bool wild = false, lag = false;

    /* PW waves stage keys and values, or the first half of the waves values and
     * the other keys: unit e is key e / UC, 16 codes or 8 floats from channel 16
     * (e % UC) or 8 (e % UC) on. */
    const bool values = wave < NW / 2;
    const int ht = tid % HT, hw = wave % (NW / 2);
    struct staged {
        unsigned reg[NU][RW];
        float sc1[NU];    /* a cache's value scales, of the units */
        bool kept[NU], kept1; /* of the units; of key `lane` */
        float sr;         /* a cache's scale of key `lane` */
        unsigned byte[NU]; /* of the mask, as kept; looked at when they have come */
    } mine, other;
    int pg = -1, pg0 = t0;
    int vexp = WIN_NONE; /* exponent of the largest value scale so far; o counts in 2^(vexp - 127 - WIN_VEXP) */

    /* Pages of 16 tiles from t on, a run of 16 keys a lane. */
    auto pages = [&](int t) {
        const int key = span.tile(min(t + (lane >> 2), t1 - 1)) * WIN_KT + 16 * (lane & 3);

        pg0 = t;
        pg = key < jb.nk ? seq_page(a.c, jb.b, key) : -1;
    };
    auto page_of = [&](int t, int run) { return __shfl(pg, 4 * (t - pg0) + run, 64); };
    /* Tile t into registers. Where there is no key or page, and behind a row's
     * channels, something else is read that counts nothing: no lane has a
     * branch. */
    auto fetch = [&](int t, const auto values, staged &r) {
        const int k0 = span.tile(t) * KT;

        if constexpr (CACHE) {
            const signed char *codes = values ? a.c.vc : a.c.kc;

#pragma unroll
            for (int i = 0; i < NU; i++) {
                const int e = min(ht + HT * i, U - 1), key = e / UC, at = e % UC * 16;
                uint4 x;

                /* The address is a scalar one and an offset that never changes
                 * where a wave's lanes lie in one run. */
                if constexpr (SAME) {
                    const int run = __builtin_amdgcn_readfirstlane(key >> 4);
                    const int page = __builtin_amdgcn_readlane(pg, 4 * (t - pg0) + run);
                    const long long first = cache_row(a.c, max(page, 0), jb.kvh, k0 + 16 * run);

                    x = *(const uint4 *)(codes + first * pitch + (unsigned)((key & 15) * pitch + min(at, pitch - 16)));
                    if (values) {
                        r.kept[i] = page >= 0 && k0 + key < jb.nk;
                        r.sc1[i] = (a.c.vs + first)[key & 15];
                    }
                }
                else {
                    const int page = page_of(t, key >> 4);
                    const long long cell = cache_row(a.c, max(page, 0), jb.kvh, k0 + key);

                    x = *(const uint4 *)(codes + cell * pitch + min(at, pitch - 16));
                    if (values) {
                        r.kept[i] = page >= 0 && k0 + key < jb.nk;
                        r.sc1[i] = a.c.vs[cell];
                    }
                }
                r.reg[i][0] = x.x, r.reg[i][1] = x.y, r.reg[i][2] = x.z, r.reg[i][3] = x.w;
            }
            if (hw == 0) {
                const int page = page_of(t, lane >> 4);

                r.kept1 = page >= 0 && k0 + lane < jb.nk;
                r.sr = (values ? a.c.vs : a.c.ks)[cache_row(a.c, max(page, 0), jb.kvh, k0 + lane)];
            }
        }
        else {
            const int end = jb.nk - 1 - k0;
            const float *from = (values ? a.V : a.K) + (long long)jb.kvh * d;
            const long long ld = values ? a.ldv : a.ldk;

#pragma unroll
            for (int i = 0; i < NU; i++) {
                const int e = min(ht + HT * i, U - 1), key = e / UC, at = e % UC * 8;
                const float *x = from + (k0 + min(key, end)) * ld;
                float u[4], v[4];

                win_load4<CHANNELS>(x, at, d, u);
                win_load4<CHANNELS>(x, at + 4, d, v);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    r.reg[i][j] = __builtin_bit_cast(unsigned, u[j]);
                    r.reg[i][4 + j] = __builtin_bit_cast(unsigned, v[j]);
                }
                r.kept[i] = key <= end;
                if (a.kmask && values)
                    r.byte[i] = a.kmask[k0 + min(key, end)];
            }
            if (hw == 0 && !values) {
                r.kept1 = lane <= end && lane < KT;
                if (a.kmask)
                    r.byte[0] = a.kmask[k0 + min(lane, end)];
            }
        }
    };
    auto stash = [&](tile_lds &s, const auto values, const staged &r) {
        win_u4 *to = values ? s.v : s.k;
        const int stride = values ? VS : KS;

        if constexpr (CACHE) {
#pragma unroll
            for (int i = 0; i < NU; i++) {
                const int e = ht + HT * i, key = e / UC;
                win_u4 x[2];

                if (U % HT && e >= U)
                    continue;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const unsigned w = r.reg[i][j] ^ 0x80808080u;

                    x[j / 2][2 * j % 4] = win_codes(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
                    x[j / 2][2 * j % 4 + 1] = win_codes(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
                }
                if (values) {
                    /* Codes of a scale far below the largest: smaller, exactly. */
                    const int k = vexp - WIN_LAG - (int)(q8_mag(r.sc1[i]) >> 23);

                    if (__any(k > 0 && r.kept[i])) {
                        const int n = min(max(k, 0), WIN_CODES);
                        const unsigned short f = n <= 14 ? (unsigned short)((15 - n) << 10) : (unsigned short)(1 << (WIN_CODES - n));
                        const _Float16 down = __builtin_bit_cast(_Float16, f);
                        const win_h2 two = {down, down};

#pragma unroll
                        for (int j = 0; j < 8; j++)
                            x[j / 4][j % 4] = __builtin_bit_cast(unsigned, __builtin_bit_cast(win_h2, (unsigned)x[j / 4][j % 4]) * two);
                    }
                }
                to[key * stride + e % UC * 2] = x[0];
                to[key * stride + e % UC * 2 + 1] = x[1];
            }
            if (hw == 0 && !values) {
                const unsigned long long keep = __ballot(r.kept1);

                /* NaN: rows that see the key are done again. */
                s.ks[lane] = q8_mag(r.sr) >> 23 > WIN_SEXP ? __builtin_nanf("") : r.sr;
                if (lane == 0)
                    s.keep = keep;
            }
            else if (hw == 0) {
                /* Value scales times a power of two that brings the largest so
                 * far to 2^WIN_VEXP; a scale of NaN, and one too far below the
                 * largest, is for the float32 path. */
                const float x = r.kept1 ? r.sr : 0.0f;
                const bool bad = !(q8_mag(x) < 0x7f800000u);
                const int e = bad ? 0 : (int)(q8_mag(x) >> 23), n = max(vexp - WIN_LAG - e, 0);
                const int top = max(max(vexp, WIN_VEXP), min((int)wave_umax(e), 253));
                /* Twice, as one power may pass the range. */
                const float y = bad || n > WIN_CODES ? 0.0f : x * win_power(127 + n) * win_power(254 + WIN_VEXP - top);
                const bool w = __any(bad || (x != 0.0f && y < WIN_VMIN));
                const bool lags = __any(r.kept1 && e < top - WIN_LAG);

                s.vs[lane] = y;
                if (lane == 0) {
                    s.top[0] = top;
                    s.wild = w;
                    s.lag = lags;
                }
            }
        }
        else {
            int top = 0, low = 255; /* exponents */
            bool zero = false;
            /* What a value's scale counts in now; other tiles' largest one may
             * change that. */
            const float vup = vexp == WIN_NONE ? 1.0f : win_power(254 + WIN_VEXP - vexp);

#pragma unroll
            for (int i = 0; i < NU; i++) {
                const int e = ht + HT * i, key = e / UC;
                float f[8];
                win_u4 x, y;

#pragma unroll
                for (int j = 0; j < 8; j++)
                    f[j] = __builtin_bit_cast(float, r.reg[i][j]);
                /* Values of keys that are left out are zeros, whatever they
                 * hold. */
                const bool in = r.kept[i] && (!a.kmask || r.byte[i]);

                if (values && __any(!in)) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        f[j] = in ? f[j] : 0.0f;
                }
                const float most = fmaxf(fmaxf(fmaxf(fabsf(f[0]), fabsf(f[1])), fmaxf(fabsf(f[2]), fabsf(f[3]))),
                                         fmaxf(fmaxf(fabsf(f[4]), fabsf(f[5])), fmaxf(fabsf(f[6]), fabsf(f[7]))));
                /* Infinities and NaN make the parts NaN, as larger keys than
                 * WIN_KEXP do that pass f16's range, and the rows that meet
                 * them are done again. */
                const unsigned mag = win_row_max<UC>(__builtin_bit_cast(unsigned, most));
                int ex = min(max((int)(mag >> 23), 15), values ? 254 : WIN_KEXP);

                if (values) {
                    if (mag) {
                        top = max(top, ex - 14);
                        low = min(low, ex - 14);
                    }
                    zero = zero || (in && !mag);
                    ex = max(ex, vexp - WIN_LAG + 14);
                }
                const float up = win_power(268 - ex);

#pragma unroll
                for (int j = 0; j < 4; j++) {
                    unsigned b, c;

                    win_split(f[2 * j] * up, f[2 * j + 1] * up, b, c);
                    x[j] = b;
                    y[j] = c;
                }
                if (U % HT && e >= U)
                    continue;
                to[key * stride + e % UC] = x;
                to[(KT + key) * stride + e % UC] = y;
                if (e % UC == 0)
                    (values ? s.vs : s.ks)[key] = win_power(ex - 14) * (values ? vup : 1.0f);
            }
            if (values) {
                const unsigned both = win_wave_max2((unsigned)top << 16 | (255u - low));
                const bool zeros = __any(zero);

                if (lane == 0) {
                    s.top[hw] = (int)(both >> 16);
                    s.low[hw] = 255 - (int)(both & 0xffffu);
                    s.zero[hw] = zeros;
                }
            }
            else if (hw == 0) {
                const unsigned long long keep = __ballot(r.kept1 && (!a.kmask || r.byte[0]));

                if (lane == 0)
                    s.keep = keep;
            }
        }
    };
    auto take = [&](int t) {
        if constexpr (PW > 0) {
            fetch(t, std::false_type(), mine);
            fetch(t, std::true_type(), other);
        }
        else
            fetch(t, values, mine);
    };
    auto put = [&](tile_lds &s) {
        if constexpr (PW > 0) {
            stash(s, std::false_type(), mine);
            stash(s, std::true_type(), other);
        }
        else
            stash(s, values, mine);
    };
    auto begin = [&]() {
        if (t0 < t1) {
            if (CACHE)
                pages(t0);
            take(t0);
            put(lds[0]);
            if (t0 + 1 < t1)
                take(t0 + 1);
        }
    };
    /* The tile behind t into the other buffer, which was last read a tile ago,
     * before the barrier; then its successor's loads. */
    auto next = [&](int t) {
        if (t + 1 < t1) {
            put(lds[(t + 1 - t0) & 1]);
            if (t + 2 < t1) {
                if (CACHE && t + 2 - pg0 >= 16)
                    pages(t + 2);
                take(t + 2);
            }
        }
    };

    /* The largest value scale with tile t's, and what else its values say. */
    auto scales = [&](const tile_lds &s) {
        int top = s.top[0];

        if constexpr (!CACHE) {
            int low = s.low[0], zero = s.zero[0];

#pragma unroll
            for (int w = 1; w < NW / 2; w++) {
                low = min(low, s.low[w]);
                top = max(top, s.top[w]);
                zero |= s.zero[w];
            }
            /* From where its power of two has one that undoes it. */
            top = max(top > WIN_NONE ? max(top, WIN_VEXP + 2) : WIN_NONE, vexp);
            /* Too far below the largest before this tile or, as they were
             * staged without it, in it; values from 2^127 on may be infinite. */
            wild = wild || low < vexp - WIN_LAG - WIN_DEEP || max(low, vexp - WIN_LAG) < top - WIN_VEXP - 3 || top >= 240;
            lag = lag || zero || low < top - WIN_LAG;
        }
        else {
            wild = wild || s.wild;
            lag = lag || s.lag;
        }
        return __builtin_amdgcn_readfirstlane(top);
    };

    if constexpr (PW > 0) {
        if (mover) {
            /* Where the others have half of a tile's keys each, they wait for
             * the next one: 1000 rows of 16 heads on 8000 keys 153 us without,
             * 147 with; 16000 rows in tiles of 256 123 and 129. */
            if (KG > 1)
                __builtin_amdgcn_s_setprio(2);
            begin();
            __syncthreads();
            for (int t = t0; t < t1; t++) {
                vexp = scales(lds[(t - t0) & 1]);
                next(t);
                __syncthreads();
            }
            return;
        }
    }

    win_u4 qh[2 * ND], ql[2 * ND];
    win_f16x o[ND];
    float m = -INFINITY, l = 0.0f, qf;

    /* The query times scale and log2 e, times a power of two that brings its
     * largest magnitude to 2^14 .. 2^15; qf takes it back. */
    {
        const float *q = a.Q + row * a.ldq + (long long)h * d;
        float x[2 * ND][8];
        unsigned mag = 0;

#pragma unroll
        for (int st = 0; st < 2 * ND; st++) {
            float u[4], v[4];

            load4_row(q, st * 16 + half * 8, d, u);
            load4_row(q, st * 16 + half * 8 + 4, d, v);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[st][j] = (j < 4 ? u[j & 3] : v[j & 3]) * (a.scale * WIN_LOG2E);
                mag = max(mag, q8_mag(x[st][j]));
            }
        }
        mag = max(mag, (unsigned)__shfl_xor((int)mag, 32, 64));
        const int e = min(max((int)(mag >> 23), 15), 254);
        const float up = win_power(268 - e);

        qf = win_power(e - 14);
        most_k[wave][lane] = 0;
#pragma unroll
        for (int st = 0; st < 2 * ND; st++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                unsigned u, v;

                win_split(x[st][2 * j] * up, x[st][2 * j + 1] * up, u, v);
                qh[st][j] = u;
                ql[st][j] = v;
            }
    }
#pragma unroll
    for (int tt = 0; tt < ND; tt++)
#pragma unroll
        for (int e = 0; e < 16; e++)
            o[tt][e] = 0.0f;

    if (PW == 0)
        begin();
    __syncthreads();
    for (int t = t0; t < t1; t++) {
        const tile_lds &s = lds[(t - t0) & 1];
        const int base = span.tile(t) * KT;
        /* This lane's places: a key's chunks; of the values, which come
         * transposed by 4 x 16, 4 channels of a key. */
        const win_u4 *kp = s.k + col * KS + half;
        const char *vp = (const char *)(s.v + (4 * half + (lane & 15) / 4) * VS + 2 * (lane >> 4 & 1)) + 8 * (lane & 3);
        /* Half of a SIMD's waves at the start of a tile and half at its end, so
         * that one's products run beside the other's vector instructions. */
        if (PW == 0 && !values)
            next(t);
        const int top = scales(s);

        /* Every NW-th tile's keys, a lane each. */
        if (((t - t0) & (NW - 1)) == wave) {
            const int keep = ((const int *)&s.keep)[lane >> 5];

            most_k[wave][lane] = max(most_k[wave][lane], __builtin_bit_cast(unsigned, s.ks[lane % KT]) &
                                                             (unsigned)__builtin_amdgcn_sbfe(keep, col, 1));
        }
        /* A tile's float32 scales count in the exponent before it: its weights
         * are 2^vshift of what they are in the sums. The first ones count in
         * none. */
        const bool first = !CACHE && vexp == WIN_NONE && top > WIN_NONE;
        int vshift = 0;

        if (top != vexp) {
            const float down = win_power(max(127 + vexp - top, 1));

            if (vexp > WIN_NONE) {
                if (!CACHE)
                    vshift = max(vexp - top, -64);
                /* Sums that would pass the range below. */
                wild = wild || top - vexp > 64;
            }
            vexp = top;
#pragma unroll
            for (int tt = 0; tt < ND; tt++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    o[tt][e] *= down;
        }
        const float unshift = win_power(127 - vshift);

#pragma unroll
        for (int half_tile = 0; half_tile < KT / 32 / KG; half_tile++) {
            const int part = KG > 1 ? kg : half_tile;
            const int k0 = base + 32 * part;
            /* Some row of the wave sees some key; all see all. */
            const bool some = live && k0 <= hi1 && (k0 + 32 > lo0 || k0 < a.sinks);
            const unsigned keep = (unsigned)(s.keep >> 32 * part);

            if (some) {
                win_f16x sc;
                win_u4 ph[2], pl[2];
                float x[16], mx = -INFINITY, sum = 0.0f;
                /* Operands are read WIN_AHEAD steps before their products. */
                win_h8 kf[WIN_AHEAD][P];
                auto key = [&](int st, int part2) {
                    return __builtin_bit_cast(win_h8, kp[(32 * part + KT * part2) * KS + 2 * st]);
                };

#pragma unroll
                for (int e = 0; e < 16; e++)
                    sc[e] = 0.0f;
#pragma unroll
                for (int st = 0; st < WIN_AHEAD && st < 2 * ND; st++)
#pragma unroll
                    for (int i = 0; i < P; i++)
                        kf[st][i] = key(st, i);
#pragma unroll
                for (int st = 0; st < 2 * ND; st++) {
                    win_h8(&k)[P] = kf[st % WIN_AHEAD];

                    sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[0], __builtin_bit_cast(win_h8, ql[st]), sc, 0, 0, 0);
                    if constexpr (P > 1)
                        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[1], __builtin_bit_cast(win_h8, qh[st]), sc, 0, 0, 0);
                    sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[0], __builtin_bit_cast(win_h8, qh[st]), sc, 0, 0, 0);
                    if (st + WIN_AHEAD < 2 * ND)
#pragma unroll
                        for (int i = 0; i < P; i++)
                            k[i] = key(st + WIN_AHEAD, i);
                    __builtin_amdgcn_sched_barrier(0);
                }
                /* Register e is key 8 (e / 4) + 4 half + e % 4. */
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 k = *(const float4 *)&s.ks[32 * part + 2 * e + 4 * half];

                    x[e] = sc[e] * k.x;
                    x[e + 1] = sc[e + 1] * k.y;
                    x[e + 2] = sc[e + 2] * k.z;
                    x[e + 3] = sc[e + 3] * k.w;
                }
                if (keep != ~0u || k0 + 31 > hi0 || !(k0 >= lo1 || k0 + 32 <= a.sinks)) {
                    const unsigned see = (keep & win_sees(a, lo, hi, k0)) >> 4 * half;

#pragma unroll
                    for (int e = 0; e < 16; e++)
                        x[e] = win_if(see, 8 * (e >> 2) + (e & 3), x[e]);
                }
#pragma unroll
                for (int e = 0; e < 16; e++)
                    mx = fmaxf(mx, x[e]);
                mx = win_halves(mx) * qf;
                const bool need = mx > m + WIN_TAU;

                if (__any(need)) {
                    const float mn = need ? mx : m;
                    const float corr = need ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;

                    m = mn;
                    l *= corr;
#pragma unroll
                    for (int tt = 0; tt < ND; tt++)
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            o[tt][e] *= corr;
                }
                const float ref = (m == -INFINITY ? 0.0f : m) - (float)vshift;
                win_h8 vf[WIN_AHEAD][P];
                /* Step i: keys 16 (i / ND) .., channels 32 (i % ND) ..; slot j of a
                 * lane half is the key that register 8 (i / ND) + j of the
                 * scores is. */
                auto value = [&](int i, int part2) {
                    win_h4 y[2];

#pragma unroll
                    for (int r8 = 0; r8 < 2; r8++) {
                        const char *at = vp + 16 * ((KT * part2 + 32 * part + 16 * (i / ND) + 8 * r8) * VS + 4 * (i % ND));

                        y[r8] = __builtin_bit_cast(win_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                               (__attribute__((address_space(3))) win_s4 *)at));
                    }
                    return __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7);
                };

#pragma unroll
                for (int i = 0; i < WIN_AHEAD && i < 2 * ND; i++)
#pragma unroll
                    for (int k = 0; k < P; k++)
                        vf[i][k] = value(i, k);
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    float4 v = *(const float4 *)&s.vs[32 * part + 2 * e + 4 * half];
                    unsigned u0, u1, v0, v1;

                    if (first) {
                        const float up = win_power(254 + WIN_VEXP - vexp);

                        v = make_float4(v.x * up, v.y * up, v.z * up, v.w * up);
                        asm volatile(""); /* a branch, no products with 1 */
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        x[e + j] = __builtin_amdgcn_exp2f(fmaf(x[e + j], qf, -ref));
                        sum += x[e + j];
                    }
                    win_split(x[e] * v.x, x[e + 1] * v.y, u0, v0);
                    win_split(x[e + 2] * v.z, x[e + 3] * v.w, u1, v1);
                    ph[e / 8][e / 2 % 4] = u0;
                    ph[e / 8][e / 2 % 4 + 1] = u1;
                    pl[e / 8][e / 2 % 4] = v0;
                    pl[e / 8][e / 2 % 4 + 1] = v1;
                }
                l = fmaf(sum, unshift, l);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 2 * ND; i++) {
                    const int u = i / ND, tt = i % ND;
                    win_h8(&v)[P] = vf[i % WIN_AHEAD];

                    o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[0], __builtin_bit_cast(win_h8, pl[u]), o[tt], 0, 0, 0);
                    if constexpr (P > 1)
                        o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[1], __builtin_bit_cast(win_h8, ph[u]), o[tt], 0, 0, 0);
                    o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[0], __builtin_bit_cast(win_h8, ph[u]), o[tt], 0, 0, 0);
                    if (i + WIN_AHEAD < 2 * ND)
#pragma unroll
                        for (int k = 0; k < P; k++)
                            v[k] = value(i + WIN_AHEAD, k);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (PW == 0 && values)
            next(t);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);
    /* Channels far below a query's or key's largest may have lost bits that
     * count: see WIN_LOST. */
    {
        unsigned k = most_k[0][lane];

#pragma unroll
        for (int w = 1; w < NW; w++)
            k = max(k, most_k[w][lane]);
        if (!(__builtin_bit_cast(float, wave_umax(k)) * qf * (d * (CACHE ? 0x1p-18f : 0x1p-9f)) <= WIN_LOST))
            l = __builtin_nanf("");
    }
    if constexpr (KG > 1) {
        /* The other keys' sums, through LDS: a lane's registers as they are. */
        static_assert(sizeof(lds) >= RG * 64 * (16 * ND + 2) * 4, "room for the sums");
        float *to = (float *)lds + rg * 64 + lane;

        if (kg) {
            to[0] = m;
            to[RG * 64] = wild ? __builtin_nanf("") : l;
#pragma unroll
            for (int tt = 0; tt < ND; tt++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    to[(2 + 16 * tt + e) * RG * 64] = o[tt][e];
        }
        __syncthreads();
        if (kg)
            return;
        const float m2 = to[0], top = fmaxf(m, m2), ref = top == -INFINITY ? 0.0f : top;
        const float c1 = __builtin_amdgcn_exp2f(m - ref), c2 = __builtin_amdgcn_exp2f(m2 - ref);

        m = top;
        l = l * c1 + to[RG * 64] * c2;
#pragma unroll
        for (int tt = 0; tt < ND; tt++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                o[tt][e] = o[tt][e] * c1 + to[(2 + 16 * tt + e) * RG * 64] * c2;
    }
    float z = l * 0.0f, most = 0.0f;

#pragma unroll
    for (int tt = 0; tt < ND; tt++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            z = fmaf(o[tt][e], 0.0f, z);
            most = fmaxf(most, fabsf(o[tt][e]));
        }
    /* A weight times scale is off by up to 2^-25, which times the largest value
     * is 2^-35 of that: where values are far smaller, or zeros, and the output
     * is so too (2^-14), that may be many units of the output. Zeros alone are
     * exact. */
    if (lag && vexp > WIN_NONE && win_halves(most) < l * (CACHE ? 0x1p3f : 0x1p11f))
        wild = true;
    win_finish<ND, CACHE, KT>(a, jb, span, t0, t1, parts, split, o, win_power(max(vexp - WIN_VEXP, 1)), m, l,
                              wild || z != 0.0f, ps[wave], d);
}

#define WIN_FTAU 8.0f         /* as WIN_TAU: bf16 parts have float32's range */
#define WIN_QUP 0x1p32f       /* scale of the queries split into bf16 parts */

/* ---- few rows ---------------------------------------------------------------------- */

#define WIN_FEW 16  /* rows of a tile */
#define WIN_STEP 32 /* keys of a step of a wave */

typedef float win_f4 __attribute__((ext_vector_type(4)));

/* At most 16 rows, as a decoding step has: nothing is shared by rows of other
 * waves, so each wave goes through steps of keys of its own, from memory to
 * registers to the matrix instructions without LDS or barriers; the block's
 * four join their outputs at the end. v_mfma_f32_16x16x32_bf16: scores have
 * the keys as rows (lane % 16 of either 16) and the queries as columns, and
 * leave a lane with the keys 16 t + 4 (lane / 16) + r of its query lane % 16,
 * which slot 4 t + r of the second product takes as they are. Queries and
 * weights are three bf16 parts each (split.h), codes are bf16 values: exact.
 * Bound by the cache's bytes: one query of 16 heads on 131005 keys of 4 heads
 * of 128, 139 MB in 31 us; 64 sequences of up to 16384 keys, 278 MB in 60. A
 * step's keys are asked for a step before, its values at its start. */
template <int ND, bool CACHE, int CHANNELS>
__global__ void __launch_bounds__(256, CACHE && ND == 4 ? 3 : 2) win_few_kernel(const win_args a)
{
    constexpr int DP = 32 * ND, NT = 2 * ND;  /* channels, tiles of 16 of them */
    constexpr int VL = DP / 16;               /* channels of a lane */
    constexpr int KW = CACHE ? (ND == 1 ? 2 : 4) : 8; /* words of a load of K: 8 or 16 bytes, 8 floats */
    constexpr int KL = CACHE ? (ND == 4 ? 2 : 1) : ND; /* loads of a key */
    constexpr int VW = CACHE ? (ND == 4 ? 2 : 1) : VL; /* words of a key's channels of V */
    __shared__ float os[4][WIN_FEW][DP + 4];
    __shared__ float ms[4][WIN_FEW], lsum[4][WIN_FEW], ps[4][64];
    __shared__ int redo[WIN_FEW];
    const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = a.nh / a.nhk, d = CHANNELS == WIN_FULL ? DP : a.d, pitch = a.c.pitch;
    const int tiles = CACHE ? (int)((long long)a.rows * g / WIN_FEW) + a.c.n
                            : (int)(((long long)a.rows * g + WIN_FEW - 1) / WIN_FEW);
    int split, kvh;
    const int tile = win_unit(a, tiles, split, kvh);
    const win_job jb = win_job_of<CACHE, WIN_FEW>(a, tile, kvh);

    if (jb.n <= 0)
        return;
    const int last = jb.r0 + jb.n - 1;
    const win_tiles span = win_span<WIN_STEP>(a, jb.p0 + jb.r0 / g, jb.p0 + last / g, jb.nk);
    const int parts = win_parts(span.n, a.splits);
    /* This lane's row; lanes without one take the last. */
    const int r = min(jb.r0 + col, last), qi = r / g, h = jb.kvh * g + r - qi * g;
    const bool mine = jb.r0 + col <= last;
    const long long row = jb.first + qi;

    if (split >= parts) {
        if (mine && tid < WIN_FEW)
            a.ml[(row * a.nh + h) * a.splits + split] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const int t0 = (int)((long long)span.n * split / parts), t1 = (int)((long long)span.n * (split + 1) / parts);
    /* This wave's steps. */
    const int s0 = t0 + (int)((long long)(t1 - t0) * wave / 4), s1 = t0 + (int)((long long)(t1 - t0) * (wave + 1) / 4);
    const int p0 = jb.p0 + qi, hi = win_hi(a, p0, jb.nk), lo = win_lo(a, p0);
    /* What every row sees. */
    const int hi0 = win_hi(a, jb.p0 + jb.r0 / g, jb.nk), lo1 = win_lo(a, jb.p0 + last / g);
    const float *K = CACHE ? nullptr : a.K + (long long)jb.kvh * d, *V = CACHE ? nullptr : a.V + (long long)jb.kvh * d;
    split_u4 q[ND][3];
    win_f4 o[NT];
    float m = -INFINITY, l = 0.0f;
    unsigned seen = 0;

    if (tid < WIN_FEW)
        redo[tid] = 0;
    /* Slot j of a lane's 8 of step s of the first product: this channel. */
    auto channel = [&](int s) {
        return CACHE && ND > 1 ? 64 * (s / 2) + 16 * grp + 8 * (s % 2) : 32 * s + 8 * grp;
    };
    {
        const float *qp = a.Q + row * a.ldq + (long long)h * d;

#pragma unroll
        for (int s = 0; s < ND; s++) {
            float u[4], v[4], x[8];

            load4_row(qp, channel(s), d, u);
            load4_row(qp, channel(s) + 4, d, v);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[j] = u[j];
                x[4 + j] = v[j];
            }
            split8(x, a.scale * WIN_LOG2E * WIN_QUP, q[s][0], q[s][1], q[s][2]);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            o[i][e] = 0.0f;

    unsigned kr[2][KL][KW], vr[8][VW], next = ~0u;
    float kscale[2][4], vscale[2][4];
    int pg = -1, pg0 = s0;

    /* Pages of 32 steps from i on, two runs of 16 keys a step, one a lane. */
    auto pages = [&](int i) {
        const int key = 32 * span.tile(min(i + (lane >> 1), s1 - 1)) + 16 * (lane & 1);

        pg0 = i;
        pg = key < jb.nk ? seq_page(a.c, jb.b, key) : -1;
    };
    auto page_of = [&](int i, int t) { return __builtin_amdgcn_readlane(pg, 2 * (i - pg0) + t); };
    auto fetch_k = [&](int i) {
        const int k0 = 32 * span.tile(i);

        if constexpr (CACHE) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int page = page_of(i, t);

#pragma unroll
                for (int c = 0; c < KL; c++)
#pragma unroll
                    for (int w = 0; w < KW; w++)
                        kr[t][c][w] = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    kscale[t][e] = 0.0f;
                if (page < 0)
                    continue;
                const signed char *k = a.c.kc + cache_row(a.c, page, jb.kvh, k0 + 16 * t + col) * pitch;

                load4(a.c.ks + cache_row(a.c, page, jb.kvh, k0 + 16 * t + 4 * grp), kscale[t]);
#pragma unroll
                for (int c = 0; c < KL; c++) {
                    const int at = 64 * c + 4 * KW * grp;

                    if (at < pitch) {
                        if constexpr (KW == 4) {
                            const uint4 x = *(const uint4 *)(k + at);

                            kr[t][c][0] = x.x, kr[t][c][1] = x.y, kr[t][c][2] = x.z, kr[t][c][3] = x.w;
                        }
                        else {
                            const uint2 x = *(const uint2 *)(k + at);

                            kr[t][c][0] = x.x, kr[t][c][1] = x.y;
                        }
                    }
                }
            }
        }
        else {
            const int end = jb.nk - 1 - k0;

#pragma unroll
            for (int t = 0; t < 2; t++) {
                const float *k = K + (k0 + min(16 * t + col, end)) * a.ldk;

#pragma unroll
                for (int s = 0; s < ND; s++) {
                    float u[4], v[4];

                    win_load4<CHANNELS>(k, channel(s), d, u);
                    win_load4<CHANNELS>(k, channel(s) + 4, d, v);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        kr[t][s][j] = __builtin_bit_cast(unsigned, u[j]);
                        kr[t][s][4 + j] = __builtin_bit_cast(unsigned, v[j]);
                    }
                }
            }
            if (a.kmask)
                next = lane <= end && lane < 32 && a.kmask[k0 + lane];
        }
    };
    /* Slot j is key 16 (j / 4) + 4 grp + j % 4. */
    auto fetch_v = [&](int i) {
        const int k0 = 32 * span.tile(i);

        if constexpr (CACHE) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int page = page_of(i, t);

#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int w = 0; w < VW; w++)
                        vr[4 * t + j][w] = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    vscale[t][e] = 0.0f;
                if (page < 0)
                    continue;
                const long long at = cache_row(a.c, page, jb.kvh, k0 + 16 * t + 4 * grp);
                const signed char *v = a.c.vc + at * pitch + VL * col;

                load4(a.c.vs + at, vscale[t]);
                if (VL * col < pitch) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if constexpr (VL == 8) {
                            const uint2 x = *(const uint2 *)(v + j * pitch);

                            vr[4 * t + j][0] = x.x, vr[4 * t + j][1] = x.y;
                        }
                        else if constexpr (VL == 4)
                            vr[4 * t + j][0] = *(const unsigned *)(v + j * pitch);
                        else
                            vr[4 * t + j][0] = *(const unsigned short *)(v + j * pitch);
                    }
                }
            }
        }
        else {
            const int end = jb.nk - 1 - k0;

#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float *v = V + (k0 + min(16 * (j >> 2) + 4 * grp + (j & 3), end)) * a.ldv;

                /* Channels 64 c + 4 col .., or 2 col .. of 32. */
                if constexpr (ND == 1) {
                    vr[j][0] = __builtin_bit_cast(unsigned, v[min(2 * col, d - 1)]);
                    vr[j][1] = __builtin_bit_cast(unsigned, v[min(2 * col + 1, d - 1)]);
                }
                else {
#pragma unroll
                    for (int c = 0; c < ND / 2; c++) {
                        float u[4];

                        win_load4<CHANNELS>(v, 64 * c + 4 * col, d, u);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            vr[j][4 * c + e] = __builtin_bit_cast(unsigned, u[e]);
                    }
                }
            }
        }
    };
    auto code = [](unsigned w, int k) { return (float)((int)(w << (24 - 8 * k)) >> 24); };
    constexpr int pa6[6] = {0, 2, 1, 0, 1, 0}, pb6[6] = {2, 0, 1, 1, 0, 0};

    if (s0 < s1) {
        if (CACHE)
            pages(s0);
        fetch_k(s0);
    }
    for (int i = s0; i < s1; i++) {
        const int k0 = 32 * span.tile(i);
        win_f4 s[2];
        float x[8], mx = -INFINITY;
        unsigned keep = ~0u;

        fetch_v(i);
        if constexpr (CACHE) {
            if (page_of(i, 0) < 0)
                keep &= 0xffff0000u;
            if (page_of(i, 1) < 0)
                keep &= 0x0000ffffu;
        }
        else if (a.kmask)
            keep = (unsigned)__ballot(next);
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                s[t][e] = 0.0f;
            if constexpr (CACHE) {
#pragma unroll
                for (int st = 0; st < ND; st++) {
                    split_u4 k;

#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const unsigned y = kr[t][ND == 1 ? 0 : st / 2][ND == 1 ? w / 2 : 2 * (st % 2) + w / 2];

                        k[w] = split_pk(code(y, 2 * (w % 2)), code(y, 2 * (w % 2) + 1));
                    }
#pragma unroll
                    for (int w = 2; w >= 0; w--)
                        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            __builtin_bit_cast(split_b8, k), __builtin_bit_cast(split_b8, q[st][w]), s[t], 0, 0, 0);
                }
            }
            else {
#pragma unroll
                for (int st = 0; st < ND; st++) {
                    split_u4 k[3];
                    float y[8];

#pragma unroll
                    for (int j = 0; j < 8; j++)
                        y[j] = __builtin_bit_cast(float, kr[t][st][j]);
                    split8(y, 1.0f, k[0], k[1], k[2]);
#pragma unroll
                    for (int w = 0; w < 6; w++)
                        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(split_b8, k[pa6[w]]),
                                                                       __builtin_bit_cast(split_b8, q[st][pb6[w]]), s[t],
                                                                       0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            x[j] = CACHE ? s[j / 4][j % 4] * kscale[j / 4][j % 4] : s[j / 4][j % 4];
        unsigned see = ~0u;

        if (keep != ~0u || k0 + 31 > hi0 || !(k0 >= lo1 || k0 + 32 <= a.sinks)) {
            see = keep & win_sees(a, lo, hi, k0);
            seen |= see;
            see >>= 4 * grp;
            asm volatile("" : "+v"(see));
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = see >> (16 * (j / 4) + j % 4) & 1 ? x[j] : -INFINITY;
        }
        else
            seen = 1;
        if (i + 1 < s1) {
            if (CACHE && i + 1 - pg0 >= 32)
                pages(i + 1);
            fetch_k(i + 1);
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            mx = fmaxf(mx, x[j]);
        if (__any(mx * (1.0f / WIN_QUP) > m + WIN_FTAU)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * (1.0f / WIN_QUP);
            const float mn = mx > m + WIN_FTAU ? mx : m;
            const float corr = mx > m + WIN_FTAU ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;

            m = mn;
            l *= corr;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[t][e] *= corr;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        split_u4 pp[3];

#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], 1.0f / WIN_QUP, -ref));
            l += x[j];
            /* What is not seen counts nothing, whatever its value is. */
            if (CACHE)
                x[j] = see >> (16 * (j / 4) + j % 4) & 1 ? x[j] * vscale[j / 4][j % 4] : 0.0f;
        }
        split8(x, SPLIT_UP, pp[0], pp[1], pp[2]);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if constexpr (CACHE) {
                split_u4 v;

#pragma unroll
                for (int w = 0; w < 4; w++)
                    v[w] = split_pk(code(vr[2 * w][t / 4], t % 4), code(vr[2 * w + 1][t / 4], t % 4));
#pragma unroll
                for (int w = 2; w >= 0; w--)
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(split_b8, v), __builtin_bit_cast(split_b8, pp[w]), o[t], 0, 0, 0);
            }
            else {
                split_u4 v[3];
                float y[8];

#pragma unroll
                for (int j = 0; j < 8; j++) {
                    y[j] = __builtin_bit_cast(float, vr[j][t]);
                    if (keep != ~0u)
                        y[j] = keep >> (16 * (j / 4) + 4 * grp + j % 4) & 1 ? y[j] : 0.0f;
                }
                split8(y, SPLIT_UP, v[0], v[1], v[2]);
#pragma unroll
                for (int w = 0; w < 6; w++)
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(split_b8, v[pa6[w]]),
                                                                   __builtin_bit_cast(split_b8, pp[pb6[w]]), o[t], 0, 0,
                                                                   0);
            }
        }
    }
    /* A lane has channels of rows 4 grp + e of the tiles. */
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (grp == 0) {
        ms[wave][col] = m;
        lsum[wave][col] = l;
    }
    float z = l * 0.0f;
    /* Codes are not scaled, float32 values are; taken back before the waves'
     * sums are added, which might pass the range with it. */
    const float down = CACHE ? 1.0f / SPLIT_UP : SPLIT_DOWN;

#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int w = 4 * grp + e;
            const int c = CACHE || ND == 1 ? VL * w + t : 64 * (t / 4) + 4 * w + t % 4;

            os[wave][col][c] = o[t][e] * down;
            z = fmaf(o[t][e], 0.0f, z);
        }
    __syncthreads();
    if (z != 0.0f || (l == 0.0f && seen))
        redo[col] = 1;
    __syncthreads();
    const int qr = tid >> 4, c0 = VL * (tid & 15), rr = jb.r0 + qr;

    if (rr <= last && !redo[qr]) {
        const int q1 = rr / g, h1 = jb.kvh * g + rr - q1 * g;
        const long long row1 = jb.first + q1, out = (row1 * a.nh + h1) * a.splits + split;
        const float top = fmaxf(fmaxf(ms[0][qr], ms[1][qr]), fmaxf(ms[2][qr], ms[3][qr]));
        float y[VL] = {}, sum = 0.0f;

#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = ms[w][qr] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms[w][qr] - top);

            sum = fmaf(f, lsum[w][qr], sum);
#pragma unroll
            for (int e = 0; e < VL; e++)
                y[e] = fmaf(f, os[w][qr][c0 + e], y[e]);
        }
        const float inv = parts > 1 ? 1.0f : sum > 0.0f ? 1.0f / sum : 0.0f;
        float *to = parts > 1 ? a.part + out * DP : a.O + row1 * a.ldo + (long long)h1 * d;

#pragma unroll
        for (int e = 0; e < VL; e++)
            if (c0 + e < d)
                to[c0 + e] = y[e] * inv;
        if ((tid & 15) == 0 && a.splits > 1)
            a.ml[out] = parts > 1 ? make_float2(top, sum) : make_float2(0.0f, WIN_WRITTEN);
    }
    for (int e = wave; e < jb.n; e += 4)
        if (redo[e]) {
            const int r1 = jb.r0 + e, q1 = r1 / g, h1 = jb.kvh * g + r1 - q1 * g;
            const win_row wrow = {jb.b, jb.p0 + q1, jb.nk};
            float y[2], m1, l1;

            win_row_f32<CACHE, WIN_STEP>(a, wrow, jb.first + q1, h1, span, t0, t1, ps[wave], y, m1, l1);
            win_put(a, jb.first + q1, h1, split, parts, y, m1, l1);
        }
}

/* Parts of a row and head joined, by W waves: softmax over all of them from
 * their maxima and sums, then LV lanes of four channels a part, GV parts at a
 * time, the first of them on their way before the maxima have come. W = 4: 32
 * channels a block. Bound by the latency of two dependent loads: 16 rows of 128
 * parts 4 us, 5.9 with all channels in one block and the parts asked for last. */
template <int DP, int W> __global__ void __launch_bounds__(256) win_merge_kernel(const win_args a)
{
    constexpr int RB = 4 / W, CB = W > 1 ? DP / 32 : 1; /* rows of a block, blocks of a row */
    constexpr int LV = DP / CB / 4, GV = 64 * W / LV;
    __shared__ float ws[RB][WIN_MAX_SPLITS];
    __shared__ float red[2][4];
    __shared__ float4 sums[W > 1 ? 4 : 1][LV];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = wave % W, mine = wave / W, t = 64 * sub + lane, n = a.splits;
    const long long u = (long long)(blockIdx.x / CB) * RB + mine;

    if (u >= (long long)a.rows * a.nh)
        return;
    const int row = (int)(u / a.nh), h = (int)(u % a.nh), c = DP / CB * (blockIdx.x % CB) + 4 * (t % LV);
    const float2 *ml = a.ml + u * n;
    const float *part = a.part + u * n * DP + c;
    /* At most WIN_MAX_SPLITS = 256 parts: 4 a lane of a wave. */
    constexpr int NS = WIN_MAX_SPLITS / 64 / W;
    float2 x[NS];
    float4 p[4];
    float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
    auto fetch = [&](int s0) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            p[i] = *(const float4 *)(part + (long long)min(s0 + i * GV, n - 1) * DP);
    };

#pragma unroll
    for (int i = 0; i < NS; i++)
        x[i] = ml[min(t + 64 * W * i, n - 1)];
    const float written = ml[0].y;

    fetch(t / LV);
    if (written == WIN_WRITTEN || (a.c.n && (row < seq_start(a.c, 0) || row >= seq_start(a.c, a.c.n))))
        return;
#pragma unroll
    for (int i = 0; i < NS; i++) {
        if (t + 64 * W * i >= n)
            x[i] = make_float2(-INFINITY, 0.0f);
        m = fmaxf(m, x[i].x);
    }
    m = wave_max_full(m);
    if constexpr (W > 1) {
        if (lane == 0)
            red[0][wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    }
#pragma unroll
    for (int i = 0; i < NS; i++) {
        const float w = x[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[i].x - m);

        if (t + 64 * W * i < n)
            ws[mine][t + 64 * W * i] = w;
        l += w * x[i].y;
    }
    l = wave_sum_full(l);
    if constexpr (W > 1) {
        if (lane == 0)
            red[1][wave] = l;
        __syncthreads();
        l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    }
    else
        __builtin_amdgcn_wave_barrier();
    /* Parts of no weight hold nothing, or what does not count. */
    for (int s0 = t / LV; s0 < n; s0 += 4 * GV) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = s0 + i * GV;
            const float w = s < n ? ws[mine][s] : 0.0f;

            o[0] = w != 0.0f ? fmaf(w, p[i].x, o[0]) : o[0];
            o[1] = w != 0.0f ? fmaf(w, p[i].y, o[1]) : o[1];
            o[2] = w != 0.0f ? fmaf(w, p[i].z, o[2]) : o[2];
            o[3] = w != 0.0f ? fmaf(w, p[i].w, o[3]) : o[3];
        }
        if (s0 + 4 * GV < n)
            fetch(s0 + 4 * GV);
    }
#pragma unroll
    for (int s = LV; s < 64; s *= 2)
#pragma unroll
        for (int j = 0; j < 4; j++)
            o[j] += __shfl_xor(o[j], s, 64);
    if constexpr (W > 1) {
        if (lane < LV)
            sums[wave][lane] = make_float4(o[0], o[1], o[2], o[3]);
        __syncthreads();
        if (t >= LV)
            return;
#pragma unroll
        for (int j = 0; j < 4; j++)
            o[j] = (((const float *)&sums[0][t])[j] + ((const float *)&sums[1][t])[j]) +
                   (((const float *)&sums[2][t])[j] + ((const float *)&sums[3][t])[j]);
    }
    if (t < LV) {
        float *out = a.O + row * a.ldo + (long long)h * a.d;

#pragma unroll
        for (int j = 0; j < 4; j++)
            if (c + j < a.d)
                out[c + j] = l == 0.0f ? 0.0f : o[j] / l;
    }
}

/* ---- on the host -------------------------------------------------------------- */

static int win_width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

/* Bytes of the parts of a call of so many rows and heads, whatever its keys. */
static size_t win_work_bytes(long long rows, int nh, int d)
{
    const __int128 most = (__int128)rows * nh * WIN_MAX_SPLITS;

    return (size_t)std::min<__int128>(most, WIN_PART_ROWS) * (win_width(d) + 2) * 4;
}

extern "C" size_t ops_attention_window_work_bytes(int Nq, int nh, int d)
{
    return Nq < 1 || nh < 1 || d < 1 || d > OPS_MAX_HEAD_DIM ? 0 : win_work_bytes(Nq, nh, d);
}

extern "C" size_t ops_attention_cache_work_bytes(int rows, int nh, int d)
{
    return ops_attention_window_work_bytes(rows, nh, d);
}

/* The kernel of a call and its blocks of threads. */
struct win_plan {
    bool few;
    int groups;            /* of a tile's keys, as KG of win_tile_kernel */
    int tile, splits;      /* rows, parts of the keys */
    long long blocks;      /* without the splits */
};

/* Rows see at most `keys` each of `most`. One block of tiles is held by a CU (32 channels:
 * two); more of them than that, splits included, take a second round. A block
 * has 256 rows, or 128 with the keys shared by two groups of waves where that
 * leaves all blocks in one round. Us:
 *
 *   rows, heads (key heads), channels, window       256 rows      128 rows
 *   1601, 16, 64, 321                                     40            24  (112 blocks of 256)
 *   6400, 8, 32, 641                                      38            36
 *   4096, 16 (4), 128, 1025, cache                       117           145  (256 blocks, 512)
 *
 * Keys are split until the blocks fill that round. Us by the number of parts:
 *
 *   2000 rows, 4 heads (1) of 128, window 2048, 32 blocks   1: 188   2: 107   4: 65   8: 54   12: 69
 *   1 row, 4 heads of 128, 131005 keys of a cache           64: 40   96: 40   128: 35   192: 37   256: 39
 *   1 row, 4 heads of 128, 4096 float32 keys                16: 19   32: 16   48 and more: 13
 *   1 row each of 64 sequences of a cache, window 4096      2: 68   4: 62   6: 59   8: 64   12: 69
 *
 * Sequences of unlike lengths, the last line, make parts of unlike length and
 * want more of them than fill one round; the limits there, 6 blocks a CU and
 * 640 keys a part, were measured on that call alone.
 *
 * Parts have two tiles or more, and there is one part where the second launch
 * costs more than it saves. Us in one part and in several:
 *
 *   1 row, 4 heads of 64, 256 keys            7.4    8.0
 *   1 row, 4 heads of 64, 512 keys           10.8    8.0
 *   1 row, 4 heads of 128, 256 keys          11.9    9.8
 *   100 rows of 64 channels, 256 keys        14.2   13.8
 *   100 rows of 32 channels, 256 keys        11.2   11.6
 *   3 sequences of 200 in a cache            13.3   15.9
 *   100 rows of 64 channels, 400 keys        19.2   15.4
 *   100 rows of 64 channels, 2048 keys: parts of four tiles 17.7, of two 14.7, of one 14.7
 *
 * One kernel and one number of parts serve all sequences of a call: a single
 * token beside a prompt of many rows is computed like a row of the prompt. */
static win_plan win_plan_of(const win_args &a, bool cache, long long keys, long long most, int cus)
{
    const long long heads = (long long)a.rows * a.nh, rows = heads / a.nhk; /* of a key head */
    win_plan p;

    p.few = rows <= (long long)WIN_FEW * (cache ? a.c.n : 1);
    p.groups = 1;
    p.tile = p.few ? WIN_FEW : 256;
    auto blocks = [&](int tile) { return (cache ? rows / tile + a.c.n : (rows + tile - 1) / tile) * a.nhk; };
    /* Half of the sequences have the tile more that they may need. */
    auto filled = [&](int tile) {
        return cache ? std::max((rows / tile + (a.c.n + 1) / 2) * a.nhk, (long long)a.nhk) : blocks(tile);
    };
    const long long held = (p.few || a.d <= 32 ? 2LL : 1LL) * cus;

    if (!p.few && (cache || a.d <= 64) && filled(128) <= held) {
        p.groups = 2;
        p.tile = 128;
    }
    p.blocks = blocks(p.tile);
    long long n = held / filled(p.tile);

    if (p.few && cache && a.c.n > 1)
        n = std::max(n, std::min(6LL * cus / filled(p.tile), keys / 640));
    const long long seen = p.few ? keys : std::min(most, keys + p.tile / (a.nh / a.nhk));
    const bool wide = !cache && a.d > 64;

    const long long whole = !wide ? 256 : p.few ? 128 : 64; /* keys that stay in one part */

    n = seen <= whole ? 1 : std::min(n, seen / (p.few || wide ? 64 : 128));
    n = std::min(n, WIN_PART_ROWS / heads);
    p.splits = (int)std::max(1LL, std::min(n, (long long)WIN_MAX_SPLITS));
    return p;
}

template <bool CACHE> static void win_launch(struct ops *o, win_args &a, long long keys, long long most, cl_mem work)
{
    const int cus = o->ocl->cu_count > 0 ? o->ocl->cu_count : 256;
    const win_plan p = win_plan_of(a, CACHE, keys, most, cus);
    const long long heads = (long long)a.rows * a.nh;

    a.splits = p.splits;
    if (a.splits > 1) {
        a.part = fptr(work);
        a.ml = (float2 *)(a.part + heads * a.splits * win_width(a.d));
    }
    const device_scope on(o->ocl);
    const hipStream_t s = stream_of(o->ocl);

    prof_scope ps(o->ocl, CACHE ? "attention_cache" : "attention_window");
    const dim3 grid(grid_of(p.blocks * a.splits, p.few ? 256 : 768, "attention tiles")), block(256);

#define WIN_KERNEL(ND_, CH_, KG_, KT_)                                                               \
    hipLaunchKernelGGL((win_tile_kernel<ND_, CACHE, CH_, 8, KG_, KT_, ND_ == 2 ? 4 : 0>), grid,      \
                       dim3(ND_ == 2 ? 768 : 512), 0, s, a)
#define WIN_CHANNELS(ND_, CH_)                                                           \
    do {                                                                                 \
        if (p.few)                                                                       \
            hipLaunchKernelGGL((win_few_kernel<ND_, CACHE, CH_>), grid, block, 0, s, a); \
        else if constexpr (!CACHE && ND_ == 4)                                           \
            WIN_KERNEL(ND_, CH_, 1, 32);                                                 \
        else if (p.groups == 2)                                                          \
            WIN_KERNEL(ND_, CH_, 2, 64);                                                 \
        else                                                                             \
            WIN_KERNEL(ND_, CH_, 1, 64);                                                 \
    } while (0)
#define WIN_LAUNCH(ND_)                   \
    do {                                  \
        if constexpr (CACHE)              \
            WIN_CHANNELS(ND_, WIN_ANY);   \
        else if (a.d == 32 * ND_)         \
            WIN_CHANNELS(ND_, WIN_FULL);  \
        else if (a.d % 4 == 0)            \
            WIN_CHANNELS(ND_, WIN_FOUR);  \
        else                              \
            WIN_CHANNELS(ND_, WIN_ANY);   \
    } while (0)
    if (a.d <= 32)
        WIN_LAUNCH(1);
    else if (a.d <= 64)
        WIN_LAUNCH(2);
    else
        WIN_LAUNCH(4);
#undef WIN_LAUNCH
#undef WIN_CHANNELS
#undef WIN_KERNEL
    launch_check("attention tiles");
    if (a.splits > 1) {
        const bool wide = a.splits > 16;
        const dim3 mgrid(grid_of(wide ? heads * (win_width(a.d) / 32) : (heads + 3) / 4, 256, "attention merge"));

#define MERGE_LAUNCH(DP_)                                                                \
    do {                                                                                 \
        if (wide)                                                                        \
            hipLaunchKernelGGL((win_merge_kernel<DP_, 4>), mgrid, block, 0, s, a);       \
        else                                                                             \
            hipLaunchKernelGGL((win_merge_kernel<DP_, 1>), mgrid, block, 0, s, a);       \
    } while (0)
        if (a.d <= 32)
            MERGE_LAUNCH(32);
        else if (a.d <= 64)
            MERGE_LAUNCH(64);
        else
            MERGE_LAUNCH(128);
#undef MERGE_LAUNCH
        launch_check("attention merge");
    }
}

/* Queries and outputs, and the work buffer, of either call. */
static void win_check(win_args &a, const char *op, struct opnd Q, struct opnd O, cl_mem work)
{
    const long long w = (long long)a.nh * a.d, n = win_work_bytes(a.rows, a.nh, a.d);

    if (Q.ld < w || O.ld < w || Q.off < 0 || O.off < 0)
        icoreg_fatal("%s: negative offset or short row: ld %d, %d", op, Q.ld, O.ld);
    need_floats(Q.buf, Q.off, (a.rows - 1) * (long long)Q.ld + w, op, "Q");
    need_floats(O.buf, O.off, (a.rows - 1) * (long long)O.ld + w, op, "O");
    need_bytes(work, 0, n, op, "work");
    need_aligned(work, 16, op, "work");
    a.Q = cfptr(Q.buf) + Q.off;
    a.O = fptr(O.buf) + O.off;
    a.ldq = Q.ld;
    a.ldo = O.ld;
    if (a.O != a.Q || (a.rows > 1 && a.ldo != a.ldq))
        need_rows_apart(a.O, a.ldo, w, a.rows, a.Q, a.ldq, w, a.rows, op, "O and Q (unless the same)");
    need_apart(O.buf, O.off * 4, ((a.rows - 1) * a.ldo + w) * 4, work, 0, n, op, "O and work");
    need_apart(Q.buf, Q.off * 4, ((a.rows - 1) * a.ldq + w) * 4, work, 0, n, op, "Q and work");
}

extern "C" void ops_attention_window(struct ops *o, struct opnd Q, struct opnd K, struct opnd V,
                                     struct opnd O, int Nq, int Nk, int nh, int nhk, int d, int q0,
                                     int left, int right, int sinks, float scale, cl_mem kmask,
                                     cl_mem work)
{
    ICOREG_API_BEGIN
    const char *op = "ops_attention_window";
    const long long kw = (long long)nhk * d;
    win_args a = {};

    if (d < 1 || d > OPS_MAX_HEAD_DIM)
        icoreg_fatal("%s: head dimension %d is not 1 .. %d", op, d, OPS_MAX_HEAD_DIM);
    if (Nq < 0 || Nk < 0 || Nk > WIN_MAX_KEYS || nh < 1 || nhk < 1 || nh % nhk || sinks < 0 ||
        q0 < -WIN_MAX_KEYS || (long long)q0 + Nq > WIN_MAX_KEYS)
        icoreg_fatal("%s: invalid sizes Nq=%d Nk=%d nh=%d nhk=%d q0=%d sinks=%d", op, Nq, Nk, nh, nhk,
                     q0, sinks);
    if (Nq == 0)
        return;
    a.Nk = Nk;
    a.q0 = q0;
    a.rows = Nq;
    a.nh = nh;
    a.nhk = nhk;
    a.d = d;
    a.left = left;
    a.right = right;
    a.sinks = sinks;
    a.scale = scale;
    win_check(a, op, Q, O, work);
    if (Nk) {
        const long long qw = (long long)nh * d, n = win_work_bytes(Nq, nh, d);

        if (K.ld < kw || V.ld < kw || K.off < 0 || V.off < 0)
            icoreg_fatal("%s: negative offset or short row of K or V: ld %d, %d", op, K.ld, V.ld);
        need_floats(K.buf, K.off, (Nk - 1) * (long long)K.ld + kw, op, "K");
        need_floats(V.buf, V.off, (Nk - 1) * (long long)V.ld + kw, op, "V");
        if (kmask)
            need_bytes(kmask, 0, Nk, op, "kmask");
        a.K = cfptr(K.buf) + K.off;
        a.V = cfptr(V.buf) + V.off;
        a.ldk = K.ld;
        a.ldv = V.ld;
        a.kmask = kmask ? (const unsigned char *)kmask->ptr : nullptr;
        need_rows_apart(a.O, a.ldo, qw, Nq, a.K, a.ldk, kw, Nk, op, "O and K");
        need_rows_apart(a.O, a.ldo, qw, Nq, a.V, a.ldv, kw, Nk, op, "O and V");
        need_apart(kmask, 0, Nk, O.buf, O.off * 4, ((Nq - 1) * a.ldo + qw) * 4, op, "kmask and O");
        need_apart(K.buf, K.off * 4, ((Nk - 1) * a.ldk + kw) * 4, work, 0, n, op, "K and work");
        need_apart(V.buf, V.off * 4, ((Nk - 1) * a.ldv + kw) * 4, work, 0, n, op, "V and work");
        need_apart(kmask, 0, Nk, work, 0, n, op, "kmask and work");
    }
    const long long span = left < 0 || right < 0 ? Nk : (long long)left + right + 1 + sinks;

    win_launch<false>(o, a, std::min<long long>(Nk, span), Nk, work);
    ICOREG_API_END
}

extern "C" void ops_attention_cache(struct ops *o, const struct ops_cache *c, const struct ops_seqs *s,
                                    int rows, struct opnd Q, struct opnd O, int nh, int left, int sinks,
                                    float scale, cl_mem work)
{
    ICOREG_API_BEGIN
    const char *op = "ops_attention_cache";
    win_args a = {};

    a.c = cache_check(c, s, rows, op);
    if (a.c.pages == 0)
        a.c.ldt = 0; /* no keys */
    if (nh < 1 || nh % c->nhk || sinks < 0)
        icoreg_fatal("%s: invalid sizes nh=%d nhk=%d sinks=%d", op, nh, c->nhk, sinks);
    if (rows == 0 || s->n == 0)
        return;
    a.rows = rows;
    a.nh = nh;
    a.nhk = c->nhk;
    a.d = c->d;
    a.left = left;
    a.right = 0;
    a.sinks = sinks;
    a.scale = scale;
    win_check(a, op, Q, O, work);
    const long long w = (long long)nh * a.d;

    cache_apart(c, s, a.O, ((rows - 1) * a.ldo + w) * 4, true, false, op, "O");
    cache_apart(c, s, work->ptr, win_work_bytes(rows, nh, a.d), true, false, op, "work");
    const long long most = (long long)s->ldt * c->page;

    win_launch<true>(o, a, left < 0 ? most : std::min(most, (long long)left + 1 + sinks), most, work);
    ICOREG_API_END
}
