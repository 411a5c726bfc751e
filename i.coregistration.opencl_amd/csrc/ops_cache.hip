/* SPDX-License-Identifier: Unlicense */

/* Keys and values kept in 8 bits: codes and scale of each token and head
 * (q8.h) in the pages of a cache, written from float32 rows and read back. */

#include <hip/hip_runtime.h>

#include "common.h"
#include "load4.h"
#include "ops.h"
#include "q8.h"
#include "seqs.h"

using namespace icoreg;

extern "C" int ops_cache_pitch(int d)
{
    return d < 1 || d > OPS_MAX_HEAD_DIM ? 0 : cache_pitch(d);
}

namespace icoreg {

static long long cache_cells(const struct ops_cache *c)
{
    return (long long)c->pages * c->nhk * c->page;
}

cache_view cache_check(const struct ops_cache *c, const struct ops_seqs *s, int rows, const char *op)
{
    cache_view v = {};

    if (!c || !s)
        icoreg_fatal("%s: no cache or no sequences", op);
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        icoreg_fatal("%s: page of %d tokens is not 16, 32, 64 or 128", op, c->page);
    if (c->d < 1 || c->d > OPS_MAX_HEAD_DIM)
        icoreg_fatal("%s: head dimension %d is not 1 .. %d", op, c->d, OPS_MAX_HEAD_DIM);
    if (c->pages < 0 || c->nhk < 1 || (__int128)c->pages * c->nhk * c->page > 1LL << 53)
        icoreg_fatal("%s: invalid cache of %d pages of %d heads", op, c->pages, c->nhk);
    if (rows < 0 || s->n < 0 || s->n > SEQ_MAX_POS || s->ldt < 0 ||
        (long long)s->ldt * c->page > SEQ_MAX_POS)
        icoreg_fatal("%s: invalid sizes rows=%d, %d sequences of %d pages", op, rows, s->n, s->ldt);
    v.n = s->n;
    if (rows == 0 || s->n == 0)
        return v;

    const long long cells = cache_cells(c), pitch = cache_pitch(c->d);

    need_bytes(c->kc, 0, cells * pitch, op, "kc");
    need_bytes(c->vc, 0, cells * pitch, op, "vc");
    need_aligned(c->kc, 16, op, "kc");
    need_aligned(c->vc, 16, op, "vc");
    need_floats(c->ks, 0, cells, op, "ks");
    need_floats(c->vs, 0, cells, op, "vs");
    need_bytes(s->start, 0, (s->n + 1LL) * 4, op, "start");
    need_bytes(s->len, 0, s->n * 4LL, op, "len");
    need_bytes(s->table, 0, (long long)s->n * s->ldt * 4, op, "table");
    if (cells) {
        v.kc = (signed char *)c->kc->ptr;
        v.vc = (signed char *)c->vc->ptr;
        v.ks = fptr(c->ks);
        v.vs = fptr(c->vs);
    }
    v.start = (const int *)s->start->ptr;
    v.len = (const int *)s->len->ptr;
    v.table = s->ldt ? (const int *)s->table->ptr : nullptr;
    v.ldt = s->ldt;
    v.rows = rows;
    v.pages = c->pages;
    v.page_log = __builtin_ctz(c->page);
    v.nhk = c->nhk;
    v.d = c->d;
    v.pitch = (int)pitch;
    return v;
}

void cache_apart(const struct ops_cache *c, const struct ops_seqs *s, const void *p, long long n,
                 bool output, bool writes, const char *op, const char *name)
{
    const long long cells = cache_cells(c), codes = cells * cache_pitch(c->d);
    const struct {
        cl_mem m;
        long long n;
        bool cache;
        const char *name;
    } all[] = {{c->kc, codes, true, "kc"},
               {c->vc, codes, true, "vc"},
               {c->ks, cells * 4, true, "ks"},
               {c->vs, cells * 4, true, "vs"},
               {s->start, (s->n + 1LL) * 4, false, "start"},
               {s->len, s->n * 4LL, false, "len"},
               {s->table, (long long)s->n * s->ldt * 4, false, "table"}};

    for (const auto &b : all) {
        if (!b.m || b.n <= 0 || n <= 0 || !(b.cache ? output || writes : output))
            continue;
        const uintptr_t x = (uintptr_t)p, y = (uintptr_t)b.m->ptr;

        if (x < y + b.n && y < x + n)
            icoreg_fatal("%s: %s and %s must not overlap", op, name, b.name);
    }
}

} // namespace icoreg

/* Fatal if two of the cache's buffers, or one and the sequences', overlap. */
static void cache_own_apart(const struct ops_cache *c, const struct ops_seqs *s, const char *op)
{
    const long long cells = cache_cells(c), codes = cells * cache_pitch(c->d);

    need_apart(c->kc, 0, codes, c->vc, 0, codes, op, "kc and vc");
    need_apart(c->kc, 0, codes, c->ks, 0, cells * 4, op, "kc and ks");
    need_apart(c->kc, 0, codes, c->vs, 0, cells * 4, op, "kc and vs");
    need_apart(c->vc, 0, codes, c->ks, 0, cells * 4, op, "vc and ks");
    need_apart(c->vc, 0, codes, c->vs, 0, cells * 4, op, "vc and vs");
    need_apart(c->ks, 0, cells * 4, c->vs, 0, cells * 4, op, "ks and vs");
    const struct {
        cl_mem m;
        long long n;
        const char *names;
    } seqs[] = {{s->start, (s->n + 1LL) * 4, "the cache and start"},
                {s->len, s->n * 4LL, "the cache and len"},
                {s->table, (long long)s->n * s->ldt * 4, "the cache and table"}};

    for (const auto &x : seqs) {
        need_apart(x.m, 0, x.n, c->kc, 0, codes, op, x.names);
        need_apart(x.m, 0, x.n, c->vc, 0, codes, op, x.names);
        need_apart(x.m, 0, x.n, c->ks, 0, cells * 4, op, x.names);
        need_apart(x.m, 0, x.n, c->vs, 0, cells * 4, op, x.names);
    }
}

struct cache_args {
    cache_view c;
    float *K, *V;
    long long ldk, ldv;
};

/* A row's R key heads from h on: L lanes of four channels, 256 / L groups of
 * them a block of threads; blockIdx.y 0 is keys, 1 values. */
struct cache_item {
    int row, h, ch, p, page;
    bool in; /* of a sequence */
};

/* The item of this group of lanes, `in` clear behind the last. */
template <int L, int R> __device__ __forceinline__ cache_item cache_first(const cache_view &c)
{
    const int per = (c.nhk + R - 1) / R;
    const long long i = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;

    return {(int)min(i / per, (long long)c.rows - 1), (int)(i % per) * R, 4 * (int)(threadIdx.x % L), 0, -1,
            i < (long long)c.rows * per};
}

/* Its place. The row's sequence is the last of those that start at or before
 * it, looked for by L lanes at L places of what is left of the sequences, at
 * last each lane with all that is known of one. */
template <int L, int R> __device__ __forceinline__ void cache_look_up(const cache_view &c, cache_item &it)
{
    const int sub = threadIdx.x % L, at = threadIdx.x & 63 & ~(L - 1);
    int b0 = 0, left = c.n;
    auto before = [&](bool yes) { return __popcll(__ballot(yes) >> at & ((1ull << L) - 1)); };

    while (left > L) {
        const int step = (left + L - 1) / L, to = sub * step;
        const int n = before(to < left && seq_start(c, b0 + (to < left ? to : 0)) <= it.row);

        if (n == 0) {
            it.in = false;
            return;
        }
        b0 += (n - 1) * step;
        left = min(step, left - (n - 1) * step);
    }
    const int b = b0 + min(sub, left - 1), s0 = seq_start(c, b), s1 = seq_start(c, b + 1), l = c.len[b];
    const int n = before(sub < left && s0 <= it.row), mine = at + max(n - 1, 0);
    const int end = __shfl(s1, mine, 64), len = max(__shfl(l, mine, 64), 0);
    const long long p = (long long)len - (end - it.row);

    it.in = it.in && n > 0 && it.row < end;
    if (it.in && p >= 0 && p < (long long)c.ldt << c.page_log) {
        it.p = (int)p;
        it.page = seq_page(c, b0 + n - 1, it.p);
    }
}

/* Both kernels are bound by memory, and ask for R heads' lines before they
 * use the first: some 21000 tokens of 8 heads of 64, 86 MB of float32 and 23 of codes
 * and scales, 22 us written and 20 read; one head at a time 32 and 33. */
template <int L, int R> __global__ void __launch_bounds__(256) cache_write_kernel(const cache_args a)
{
    const bool values = blockIdx.y;
    const cache_view &c = a.c;
    cache_item it = cache_first<L, R>(c);
    const float *x = values ? a.V + it.row * a.ldv : a.K + it.row * a.ldk;
    float v[R][4];

    /* On their way while the place is looked up. */
#pragma unroll
    for (int i = 0; i < R; i++)
        load4_row(x + (long long)min(it.h + i, c.nhk - 1) * c.d, it.ch, c.d, v[i]);
    cache_look_up<L, R>(c, it);

#pragma unroll
    for (int i = 0; i < R; i++) {
        unsigned mag = 0;

#pragma unroll
        for (int j = 0; j < 4; j++)
            mag = max(mag, q8_mag(v[i][j]));
        mag = max(mag, (unsigned)dpp_i((int)mag, 0xB1));
        mag = max(mag, (unsigned)dpp_i((int)mag, 0x4E));
        mag = max(mag, (unsigned)dpp_i((int)mag, 0x141));
        if (L > 8)
            mag = max(mag, (unsigned)dpp_i((int)mag, 0x140));
        if (L > 16)
            mag = max(mag, (unsigned)__shfl_xor((int)mag, 16, 64));
        const q8_scale q = q8_scale_of(mag);

        if (it.page < 0 || it.h + i >= c.nhk)
            continue;
        const long long at = cache_row(c, it.page, it.h + i, it.p);

        if (it.ch < c.pitch)
            *(unsigned *)((values ? c.vc : c.kc) + at * c.pitch + it.ch) =
                q8_code4(v[i][0], v[i][1], v[i][2], v[i][3], q.r);
        if (it.ch == 0)
            (values ? c.vs : c.ks)[at] = q.s;
    }
}

template <int L, int R> __global__ void __launch_bounds__(256) cache_read_kernel(const cache_args a)
{
    const bool values = blockIdx.y;
    const cache_view &c = a.c;
    float *to = values ? a.V : a.K;
    cache_item it = cache_first<L, R>(c);
    int w[R];
    float s[R];

    if (!to)
        return;
    cache_look_up<L, R>(c, it);
    if (!it.in)
        return;
#pragma unroll
    for (int i = 0; i < R; i++) {
        w[i] = 0;
        s[i] = 0.0f;
        if (it.page >= 0 && it.ch < c.pitch) {
            const long long at = cache_row(c, it.page, min(it.h + i, c.nhk - 1), it.p);

            w[i] = *(const int *)((values ? c.vc : c.kc) + at * c.pitch + it.ch);
            s[i] = (values ? c.vs : c.ks)[at];
        }
    }
    float *y = to + it.row * (values ? a.ldv : a.ldk) + it.ch;

#pragma unroll
    for (int i = 0; i < R; i++) {
        float v[4];

        if (it.h + i >= c.nhk)
            continue;
#pragma unroll
        for (int j = 0; j < 4; j++)
            v[j] = (float)(w[i] << (24 - 8 * j) >> 24) * s[i];
        float *z = y + (long long)(it.h + i) * c.d;

        if (it.ch + 4 <= c.d)
            store4(z, v[0], v[1], v[2], v[3]);
        else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (it.ch + j < c.d)
                    z[j] = v[j];
        }
    }
}

/* Rows of nhk heads of an operand: their bytes, 0 where it has no buffer. */
static long long cache_rows(const struct opnd &x, const struct ops_cache *c, int rows, const char *op,
                            const char *name)
{
    const long long w = (long long)c->nhk * c->d;

    if (!x.buf)
        return 0;
    if (x.off < 0 || x.ld < w)
        icoreg_fatal("%s: negative offset or short row of %s: ld %d", op, name, x.ld);
    need_floats(x.buf, x.off, (rows - 1) * (long long)x.ld + w, op, name);
    return ((rows - 1) * (long long)x.ld + w) * 4;
}

static void cache_move(struct ops *o, const struct ops_cache *c, const struct ops_seqs *s, int rows,
                       struct opnd K, struct opnd V, bool write, const char *op)
{
    cache_args a = {};

    a.c = cache_check(c, s, rows, op);
    if (rows == 0 || s->n == 0)
        return;
    if (write ? !K.buf || !V.buf : !K.buf && !V.buf)
        icoreg_fatal("%s: K or V has no buffer", op);
    cache_own_apart(c, s, op);
    const long long kbytes = cache_rows(K, c, rows, op, "K"), vbytes = cache_rows(V, c, rows, op, "V");
    const long long w = (long long)c->nhk * c->d;

    if (K.buf) {
        a.K = fptr(K.buf) + K.off;
        a.ldk = K.ld;
        cache_apart(c, s, a.K, kbytes, !write, write, op, "K");
    }
    if (V.buf) {
        a.V = fptr(V.buf) + V.off;
        a.ldv = V.ld;
        cache_apart(c, s, a.V, vbytes, !write, write, op, "V");
    }
    if (!write && K.buf && V.buf)
        need_rows_apart(a.K, a.ldk, w, rows, a.V, a.ldv, w, rows, op, "K and V");
    const int L = c->d <= 32 ? 8 : c->d <= 64 ? 16 : 32;
    /* Heads a group of lanes, where one a group fills the CUs twice. 1 and 4, us,
     * written and read: 4 heads of 128, 128 rows 5.0, 6.3; some 300 5.8, 7.0; 1200
     * 8.4, 8.1; 3000 13.8, 11.7; 8 heads of 32, 3000 9.4, 8.6. */
    const int R = c->nhk >= 4 && (long long)rows * c->nhk * L >= 512LL * o->ocl->cu_count ? 4 : 1;
    const long long items = (long long)rows * ((c->nhk + R - 1) / R);
    const unsigned n = grid_of((items * L + 255) / 256, 2 * 256, op);
    const device_scope on(o->ocl);
    const hipStream_t st = stream_of(o->ocl);

    prof_scope ps(o->ocl, write ? "cache_write" : "cache_read");
#define CACHE_KERNEL(L_, R_)                                                                  \
    do {                                                                                      \
        if (write)                                                                            \
            hipLaunchKernelGGL((cache_write_kernel<L_, R_>), dim3(n, 2), dim3(256), 0, st, a); \
        else                                                                                  \
            hipLaunchKernelGGL((cache_read_kernel<L_, R_>), dim3(n, 2), dim3(256), 0, st, a);  \
    } while (0)
#define CACHE_LAUNCH(L_)         \
    do {                         \
        if (R == 4)              \
            CACHE_KERNEL(L_, 4); \
        else                     \
            CACHE_KERNEL(L_, 1); \
    } while (0)
    if (L == 8)
        CACHE_LAUNCH(8);
    else if (L == 16)
        CACHE_LAUNCH(16);
    else
        CACHE_LAUNCH(32);
#undef CACHE_LAUNCH
#undef CACHE_KERNEL
    launch_check(op);
}

extern "C" void ops_cache_write(struct ops *o, const struct ops_cache *c, const struct ops_seqs *s,
                                int rows, struct opnd K, struct opnd V)
{
    ICOREG_API_BEGIN
    cache_move(o, c, s, rows, K, V, true, "ops_cache_write");
    ICOREG_API_END
}

extern "C" void ops_cache_read(struct ops *o, const struct ops_cache *c, const struct ops_seqs *s,
                               int rows, struct opnd K, struct opnd V)
{
    ICOREG_API_BEGIN
    cache_move(o, c, s, rows, K, V, false, "ops_cache_read");
    ICOREG_API_END
}
