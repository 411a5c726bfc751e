/* SPDX-License-Identifier: Unlicense */

/* Attention within a window and over the first keys: a query at position p
 * sees the keys p - left .. p + right and those of the first `sinks` that are
 * not behind p + right; of float32 keys and values, or of the 8-bit ones of a
 * cache (seqs.h, q8.h), there with right = 0 and the queries of several
 * sequences in one call.
 *
 * The keys that any row of a tile of rows sees are one or two runs of tiles of
 * keys (win_span). Where there are few rows, the tiles of keys are split over
 * blocks of threads, maximum, sum and unnormalised output of each to the work
 * buffer, and a second kernel joins them. */

#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

#include "common.h"
#include "load4.h"
#include "ops.h"
#include "reduce.h"
#include "seqs.h"

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

/* A row's sequence and position; keys of its sequence. */
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

template <bool CACHE>
static __device__ __forceinline__ win_row win_row_of(const win_args &a, int row)
{
    if (!CACHE)
        return {0, a.q0 + row, a.Nk};
    const int b = seq_of(a.c, row);

    if (b < 0)
        return {-1, 0, 0};
    return {b, (int)(max(a.c.len[b], 0) - (long long)(seq_start(a.c, b + 1) - row)), seq_len(a.c, b)};
}

/* One row and head over the tiles t0 .. t1 - 1 of 64 keys, in float32, by a
 * wave: lane k has key k's score, then every 64th channel. Seen keys alone are
 * read for the output, whatever the others hold. p: 64 floats of LDS of this
 * wave. Output unnormalised, o[j] channel lane + 64 j. */
template <bool CACHE>
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
        const int k0 = t.tile(i) * 64, k = k0 + lane;
        bool see = k <= hi && (k >= lo || k < a.sinks);
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

/* Parts that t tiles of keys are split into, of at most `splits`: at least 4
 * tiles each. */
static __device__ __forceinline__ int win_parts(int tiles, int splits)
{
    return min(splits, max(1, tiles / 4));
}

/* A wave a row, head and split. */
template <bool CACHE> __global__ void __launch_bounds__(256) win_row_kernel(const win_args a)
{
    __shared__ float ps[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long u = (long long)blockIdx.x * 4 + wave;

    if (u >= (long long)a.rows * a.nh * a.splits)
        return;
    const int split = (int)(u % a.splits), h = (int)(u / a.splits % a.nh);
    const int row = (int)(u / a.splits / a.nh);
    const win_row r = win_row_of<CACHE>(a, row);

    if (r.b < 0) {
        /* Nothing to write, and nothing to join. */
        if (a.splits > 1 && lane == 0)
            a.ml[u] = make_float2(0.0f, WIN_WRITTEN);
        return;
    }
    const win_tiles t = win_span<64>(a, r.p, r.p, r.nk);
    const int parts = win_parts(t.n, a.splits);

    if (split >= parts) {
        if (lane == 0)
            a.ml[u] = make_float2(-INFINITY, 0.0f);
        return;
    }
    float o[2], m, l;

    win_row_f32<CACHE>(a, r, row, h, t, (int)((long long)t.n * split / parts),
                       (int)((long long)t.n * (split + 1) / parts), ps[wave], o, m, l);
    if (parts == 1) {
        float *out = a.O + row * a.ldo + (long long)h * a.d;

#pragma unroll
        for (int e = 0; e < 2; e++)
            if (lane + 64 * e < a.d)
                out[lane + 64 * e] = l == 0.0f ? 0.0f : o[e] / l;
        if (a.splits > 1 && lane == 0)
            a.ml[u] = make_float2(0.0f, WIN_WRITTEN);
        return;
    }
    const int dp = a.d <= 32 ? 32 : a.d <= 64 ? 64 : 128;

#pragma unroll
    for (int e = 0; e < 2; e++)
        if (lane + 64 * e < a.d)
            a.part[u * dp + lane + 64 * e] = o[e];
    if (lane == 0)
        a.ml[u] = make_float2(m, l);
}

/* Parts of a row and head joined: a wave each, lane s with split s, s + 64, ..
 */
__global__ void __launch_bounds__(256) win_merge_kernel(const win_args a)
{
    __shared__ float ws[4][WIN_MAX_SPLITS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long u = (long long)blockIdx.x * 4 + wave;
    const int dp = a.d <= 32 ? 32 : a.d <= 64 ? 64 : 128;

    if (u >= (long long)a.rows * a.nh)
        return;
    const float2 *ml = a.ml + u * a.splits;

    if (ml[0].y == WIN_WRITTEN)
        return;
    const int row = (int)(u / a.nh), h = (int)(u % a.nh);
    float m = -INFINITY, l = 0.0f, o[2] = {0, 0};

    for (int s = lane; s < a.splits; s += 64)
        m = fmaxf(m, ml[s].x);
    m = wave_max_full(m);
    for (int s = lane; s < a.splits; s += 64) {
        const float2 x = ml[s];
        const float w = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - m);

        ws[wave][s] = w;
        l += w * x.y;
    }
    l = wave_sum_full(l);
    __builtin_amdgcn_wave_barrier();
    for (int s = 0; s < a.splits; s++) {
        const float w = ws[wave][s];

        if (w != 0.0f)
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (lane + 64 * e < a.d)
                    o[e] = fmaf(w, a.part[(u * a.splits + s) * dp + lane + 64 * e], o[e]);
    }
    float *out = a.O + row * a.ldo + (long long)h * a.d;

#pragma unroll
    for (int e = 0; e < 2; e++)
        if (lane + 64 * e < a.d)
            out[lane + 64 * e] = l == 0.0f ? 0.0f : o[e] / l;
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

/* Splits of keys of a call whose rows see at most `keys` each. */
static int win_splits(const win_args &a, long long keys, int cus)
{
    const long long waves = (long long)a.rows * a.nh, want = 16LL * cus;
    long long n = std::min((want + waves - 1) / waves, keys / 256);

    n = std::min(n, WIN_PART_ROWS / waves);
    return (int)std::max(1LL, std::min(n, (long long)WIN_MAX_SPLITS));
}

template <bool CACHE> static void win_launch(struct ops *o, win_args &a, long long keys, cl_mem work)
{
    const long long heads = (long long)a.rows * a.nh;

    a.splits = win_splits(a, keys, o->ocl->cu_count > 0 ? o->ocl->cu_count : 256);
    if (a.splits > 1) {
        a.part = fptr(work);
        a.ml = (float2 *)(a.part + heads * a.splits * win_width(a.d));
    }
    const dim3 grid(grid_of((heads * a.splits + 3) / 4, 256, "attention rows"));
    const device_scope on(o->ocl);
    const hipStream_t s = stream_of(o->ocl);

    prof_scope ps(o->ocl, CACHE ? "attention_cache" : "attention_window");
    hipLaunchKernelGGL(win_row_kernel<CACHE>, grid, dim3(256), 0, s, a);
    launch_check("attention rows");
    if (a.splits > 1) {
        hipLaunchKernelGGL(win_merge_kernel, dim3((unsigned)((heads + 3) / 4)), dim3(256), 0, s, a);
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

    win_launch<false>(o, a, std::min<long long>(Nk, span), work);
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

    win_launch<true>(o, a, left < 0 ? most : std::min(most, (long long)left + 1 + sinks), work);
    ICOREG_API_END
}
