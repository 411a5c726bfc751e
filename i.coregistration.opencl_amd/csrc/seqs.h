/* SPDX-License-Identifier: Unlicense */

/* Sequences kept in the pages of a cache (struct ops_cache, struct ops_seqs):
 * what kernels take of them, the lookups they share, and the host's checks.
 * The arrays live in device memory and may hold anything: every row and page
 * that is read from them is held to its range before it is used. */

#ifndef ICOREG_SEQS_H
#define ICOREG_SEQS_H

#include "common.h"
#include "q8.h"

#define SEQ_MAX_POS 0x7fffff00LL /* positions are counted in int, a tile past the last too */

struct cache_view {
    signed char *kc, *vc;
    float *ks, *vs;
    const int *start, *len, *table;
    int n, ldt, rows;                       /* sequences, pages of a row of the table, rows of the operands */
    int pages, page_log, nhk, d, pitch;
};

static inline __host__ __device__ int cache_pitch(int d) { return (d + 15) / 16 * 16; }

static __device__ __forceinline__ int seq_start(const cache_view &c, int b)
{
    return min(max(c.start[b], 0), c.rows);
}

/* The page of position p (0 <= p < ldt page) of sequence b, -1 for none. */
static __device__ __forceinline__ int seq_page(const cache_view &c, int b, int p)
{
    const int at = c.table[(long long)b * c.ldt + (p >> c.page_log)];

    return (unsigned)at < (unsigned)c.pages ? at : -1;
}

/* Row of codes and scales of place p of a page and key head. */
static __device__ __forceinline__ long long cache_row(const cache_view &c, int page, int h, int p)
{
    return (((long long)page * c.nhk + h) << c.page_log) + (p & ((1 << c.page_log) - 1));
}

namespace icoreg {

/* Fatal unless cache and sequences are sound; what kernels take of them. */
cache_view cache_check(const struct ops_cache *c, const struct ops_seqs *s, int rows, const char *op);

/* Fatal if [p, p + n) bytes overlap the cache's or the sequences' buffers
 * (inputs of a call: the cache's only where the call writes it). */
void cache_apart(const struct ops_cache *c, const struct ops_seqs *s, const void *p, long long n,
                 bool output, bool writes, const char *op, const char *name);

} // namespace icoreg

#endif /* ICOREG_SEQS_H */
