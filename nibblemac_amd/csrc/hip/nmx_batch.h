/* Shared by the kernels over a batch of sequences (nmx_attnbatch.hip, nmx_pages.hip): the layout of a
 * paged cache and the rows of a sequence. Not part of the ABI. */
#ifndef NMX_BATCH_H
#define NMX_BATCH_H

#include "nmx_attn.h"
#include "nmx_internal.h"

/* A paged cache as the kernels take it: position p of a sequence is row p & (page - 1) of the block that its
 * table names at p >> shift. */
struct PageDev {
    int seqs, npages, shift, max_pages;
    int32_t *table, *len;
    int nkv, hd;
    size_t block; /* bytes */
};

/* The rows [r0, r0 + count) of sequence s, within [0, n]; count is below 0 where row0 falls. */
struct SeqRows {
    int r0, count;
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t *row0, int s, int n) {
    const int a = row0[s], b = row0[s + 1];
    const int r0 = a < 0 ? 0 : a > n ? n : a, r1 = b < 0 ? 0 : b > n ? n : b;
    return {r0, r1 - r0};
}
/* The length of sequence s: its positions past max_pages << shift have no place in the table. */
__device__ __forceinline__ int seq_len(const int32_t *len, int s) { return len[s] < 0 ? 0 : len[s]; }
/* The sequence of row t: the last one that begins at or before it (every lane of the wave active). */
__device__ __forceinline__ int seq_of_row(const int32_t *row0, int seqs, int t) {
    const int lane = threadIdx.x & 63;
    int v[NMX_BATCH_MAX / 64], n = 0;
#pragma unroll
    for (int u = 0; u < NMX_BATCH_MAX / 64; u++) v[u] = row0[64 * u + lane < seqs ? 64 * u + lane : 0];
#pragma unroll
    for (int u = 0; u < NMX_BATCH_MAX / 64; u++) n += __popcll(__ballot(64 * u + lane < seqs && v[u] <= t));
    return n - 1;
}

/* Host: the layout from the arguments, refusing what the kernels do not take. */
static inline int nmx_pages_check(nmx_ctx *ctx, const nmx_pages &p, const char *what, PageDev *d) {
    int shift = 4;
    while (shift < 8 && (1 << shift) < p.page) shift++;
    if (p.seqs < 1 || p.seqs > NMX_BATCH_MAX || p.npages < 1 || p.npages > (1 << 20) || p.max_pages < 1 ||
        p.max_pages > (1 << 16) || (1 << shift) != p.page)
        return nmx_fail(ctx, "%s: seqs=%d npages=%d page=%d max_pages=%d", what, p.seqs, p.npages, p.page, p.max_pages);
    if (p.nkv < 1 || p.nkv > 1024 || p.hd < 64 || p.hd > 512 || p.hd % 64 || p.kv_dtype < KV_F32 || p.kv_dtype > KV_I8)
        return nmx_fail(ctx, "%s: nkv=%d hd=%d kv_dtype=%d", what, p.nkv, p.hd, p.kv_dtype);
    if (!p.table || !p.len) return nmx_fail(ctx, "%s: NULL table or len", what);
    *d = PageDev{p.seqs, p.npages, shift, p.max_pages, p.table, p.len, p.nkv, p.hd,
                 nmx_kv_bytes(p.kv_dtype, p.nkv, p.page, p.hd)};
    return 0;
}

struct NmxRange {
    const void *p;
    size_t bytes;
};
template <int N>
static inline bool nmx_hits(const NmxRange (&in)[N], const void *out, size_t bytes) {
    for (const NmxRange &x : in)
        if (x.p && nmx_overlap(out, bytes, x.p, x.bytes)) return true;
    return false;
}

#endif
