/* The pages of a step (include/nmx.h nmx_pages_update): sequences go on, are cut back, fork from each other or
 * end, and take pages for their new rows.
 *
 * pages_plan_k, one workgroup, does everything but move rows, so that no phase waits for another
 * workgroup: it counts the holders of every page as they will be (additions, exact in any order), decides which partly
 * filled pages have to be copied before their sequence writes into them, takes the lowest free pages by running
 * sums over the counts, and writes tables and lengths. Up to PP_LDS pages the counts stand in LDS meanwhile, and go back
 * only if the step fits; of more pages they are changed where they are and a step that does not fit is taken back by the
 * opposite additions. A fork's entries go through the workspace, so sequences may exchange places. pages_copy_k and, with
 * pack, pages_move_k then copy what the plan lists, in all caches at once.
 *
 * Times on MI355X: a token of 64 chats in 640 pages 11.4 us, of which the plan 7.8 and the copy of five pages in 14 caches 3.5 in
 * a trace, both chains of round trips (the bytes take 0.8); 16 of 64 chats end and the others are packed, 1200 pages, 12.8 + 4.6
 * + 21.3 in a trace, 26 as a copy. With the counts in memory, an atomic's round trip each, the first plan took 15.8. */
#include "nmx_internal.h"
#include "nmx_batch.h"
#include "nmx_lanes.h"

namespace {

constexpr int PP = 1024;          /* threads of the plan */
constexpr int PP_LDS = 16384;     /* pages whose counts, and as many page numbers, have room in LDS */
constexpr int PP_SEQS = 4;        /* sequences of a wave whose entries are requested together */
constexpr int PC = 256;           /* threads of a copy */
constexpr int PC_CHUNK = PC * 64; /* bytes of a workgroup's item: four 16-byte units a thread */

struct Lists { /* in the workspace, then the arrays below */
    int copies, moves;
    int4 copy[NMX_BATCH_MAX]; /* from, to, rows */
};
struct PagesDev {
    PageDev pg;
    int32_t *refs;
    const int32_t *from, *keep, *add;
    int pack;
    int32_t *out;
    Lists *lists;
    int32_t *fresh, *holes, *movers;      /* [npages] each */
    int32_t *rows;                        /* [seqs][max_pages]: the entries of sequences that fork */
};

/* The counts, in LDS or in memory. */
template <bool LDS>
struct Refs {
    int32_t *p;
    int npages;
    __device__ __forceinline__ int get(int page) const {
        return LDS ? p[page] : __hip_atomic_load(p + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ __forceinline__ void add(int page, int v) const {
        if ((uint32_t)page >= (uint32_t)npages) return;
        if (LDS) atomicAdd(p + page, v);
        else (void)__hip_atomic_fetch_add(p + page, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
};
/* What was written so far is seen by the whole workgroup. */
template <bool LDS>
__device__ __forceinline__ void settle() {
    if (!LDS) __threadfence();
    __syncthreads();
}

/* Running sum over the workgroup, the total in *all (sum_s: PP / 64 words; two barriers). */
__device__ __forceinline__ uint32_t scan_all(uint32_t v, uint32_t *sum_s, uint32_t *all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t inc = nmx_scan_wave(v);
    __syncthreads();
    if (lane == 63) sum_s[wave] = inc;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (int w = 0; w < PP / 64; w++) {
        if (w < wave) before += sum_s[w];
        total += sum_s[w];
    }
    *all = total;
    return before + inc - v;
}

/* Calls hit(page, rank) for the pages from `begin` on whose count want() wants, in order, while the rank is
 * below `most`; returns how many there are (all of them where it is less than most). */
template <bool LDS, typename Want, typename Hit>
__device__ uint32_t search(const Refs<LDS> &refs, int begin, int end, uint32_t most, uint32_t *sum_s, Want want, Hit hit) {
    constexpr int EACH = LDS ? 4 : 16; /* pages of a thread in a turn */
    uint32_t found = 0;
    for (int base = begin; base < end && found < most; base += PP * EACH) {
        int v[EACH];
        const int at = base + (int)threadIdx.x * EACH;
#pragma unroll
        for (int i = 0; i < EACH; i++) v[i] = refs.get(at + i < end ? at + i : end - 1);
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++)
            if (at + i < end && want(v[i])) mask |= 1u << i;
        uint32_t all, rank = found + scan_all(__popc(mask), sum_s, &all);
        for (; mask; mask &= mask - 1, rank++)
            if (rank < most) hit(at + __ffs(mask) - 1, rank);
        found += all;
    }
    return found;
}

template <bool LDS>
__global__ __launch_bounds__(PP) void pages_plan_k(const int32_t *from_, const int32_t *keep_, const int32_t *add_,
                                                   const int32_t *len_, int seqs, int npages, PagesDev a) {
    __shared__ int src_s[NMX_BATCH_MAX], kept_s[NMX_BATCH_MAX], old_s[NMX_BATCH_MAX], all_s[NMX_BATCH_MAX],
        last_s[NMX_BATCH_MAX], copy_s[NMX_BATCH_MAX], len_s[NMX_BATCH_MAX];
    __shared__ uint32_t base_s[NMX_BATCH_MAX], sum_s[PP / 64];
    __shared__ int wide_s, some_s;
    extern __shared__ int32_t pages_s[]; /* LDS: the counts, then page numbers */
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = seqs, mp = a.pg.max_pages;
    const int page = 1 << a.pg.shift, shift = a.pg.shift;
    const Refs<LDS> refs{LDS ? pages_s : a.refs, npages};
    int32_t *fresh = LDS ? pages_s + npages : a.fresh;
    auto pages_of = [&](long long r) { return (int)((r + page - 1) >> shift); };
    int f = -1, keep = 0, add = 0, old = 0;
    if (tid < S) {
        f = from_[tid], keep = keep_[tid], add = add_[tid], old = len_[tid];
        const long long room = (long long)mp << shift;
        old = old < 0 ? 0 : old > room ? (int)room : old;
        len_s[tid] = old;
    }
    if (LDS)
        for (int p = tid; p < npages; p += PP) pages_s[p] = a.refs[p];
    if (tid == 0) wide_s = S, some_s = 0;
    __syncthreads();
    int total = 0, part = 0, last = -1;
    if (tid < S) {
        const int src = f >= 0 && f < S ? f : -1, most = src < 0 ? 0 : len_s[src];
        keep = keep < 0 ? 0 : keep < most ? keep : most, add = add < 0 ? 0 : add;
        const long long len = (long long)keep + add;
        const bool wide = len > (long long)mp << shift;
        if (wide) atomicMin(&wide_s, tid);
        total = wide ? keep : (int)len, part = add > 0 ? keep & (page - 1) : 0;
        src_s[tid] = src, kept_s[tid] = pages_of(keep), old_s[tid] = pages_of(old), all_s[tid] = pages_of(total);
        if (part) last = a.pg.table[(size_t)src * mp + kept_s[tid] - 1];
        if ((uint32_t)last >= (uint32_t)npages) last = -1;
        if (src != tid || kept_s[tid] < old_s[tid]) some_s = 1; /* entries that change hands */
    }
    if (tid < NMX_BATCH_MAX) last_s[tid] = last;
    __syncthreads();
    const int wide = wide_s;
    if (wide < S) {
        if (tid < 4) a.out[tid] = tid ? 0 : -1 - wide;
        if (tid == 0) a.lists->copies = 0, a.lists->moves = 0;
        return;
    }
    /* who holds what after the step: entries given up, entries that a fork keeps. sign -1 takes it back */
    auto recount = [&](int sign) {
        for (int s0 = wave; s0 < S; s0 += PP_SEQS * (PP / 64)) {
            int begin[PP_SEQS], end[PP_SEQS], kept[PP_SEQS], src[PP_SEQS], longest = 0;
#pragma unroll
            for (int u = 0; u < PP_SEQS; u++) {
                const int s = s0 + u * (PP / 64);
                begin[u] = end[u] = kept[u] = src[u] = 0;
                if (s >= S) continue;
                const bool own = src_s[s] == s;
                begin[u] = own ? kept_s[s] : 0, end[u] = old_s[s], src[u] = src_s[s];
                kept[u] = own || src[u] < 0 ? 0 : kept_s[s];
                const int n = end[u] - begin[u] > kept[u] ? end[u] - begin[u] : kept[u];
                longest = n > longest ? n : longest;
            }
            for (int e0 = 0; e0 < longest; e0 += 64) {
                int mine[PP_SEQS], theirs[PP_SEQS];
#pragma unroll
                for (int u = 0; u < PP_SEQS; u++) {
                    const int s = s0 + u * (PP / 64), e = begin[u] + e0 + lane;
                    mine[u] = theirs[u] = -1;
                    if (e < end[u]) mine[u] = a.pg.table[(size_t)s * mp + e];
                    if (e0 + lane < kept[u]) theirs[u] = a.pg.table[(size_t)src[u] * mp + e0 + lane];
                }
#pragma unroll
                for (int u = 0; u < PP_SEQS; u++) {
                    refs.add(mine[u], -sign), refs.add(theirs[u], sign);
                    if (e0 + lane < kept[u]) a.rows[(size_t)(s0 + u * (PP / 64)) * mp + e0 + lane] = theirs[u];
                }
            }
        }
    };
    if (some_s) { /* uniform */
        recount(1);
        settle<LDS>();
    }
    /* a page that its sequence would add rows to is copied where another one holds it; where all who hold it
     * would, the first of them keeps it */
    bool copy = false;
    if (tid < S && last >= 0) {
        const int held = refs.get(last);
        if (held > 1) {
            int same = 0, before = 0;
            for (int s = 0; s < S; s++) same += last_s[s] == last, before += s < tid && last_s[s] == last;
            copy = !(held == same && before == 0);
        }
    }
    if (tid < S) copy_s[tid] = copy;
    const uint32_t need = tid < S ? (uint32_t)(all_s[tid] - kept_s[tid] + copy) : 0;
    uint32_t needed, copies;
    const uint32_t base = scan_all(need, sum_s, &needed), nth = scan_all(copy, sum_s, &copies);
    if (tid < S) base_s[tid] = base;
    if (needed) {
        const uint32_t found = search<LDS>(refs, 0, npages, needed, sum_s, [](int r) { return r == 0; },
                                           [&](int p, uint32_t i) { fresh[i] = p; });
        if (found < needed) {
            if (!LDS && some_s) recount(-1);
            if (tid < 4) a.out[tid] = tid ? 0 : (int)(needed - found);
            if (tid == 0) a.lists->copies = 0, a.lists->moves = 0;
            return;
        }
    }
    settle<LDS>();
    if (copy) {
        a.lists->copy[nth] = make_int4(last, fresh[base], part, 0);
        refs.add(last, -1);
    }
    if (tid < S) a.pg.len[tid] = total;
    /* tables: what a fork keeps, the fresh pages, -1 where there were more */
    for (int s = wave; s < S; s += PP / 64) {
        const int src = src_s[s], all = all_s[s], own = kept_s[s] - copy_s[s];
        int32_t *t = a.pg.table + (size_t)s * mp;
        if (src != s && src >= 0)
            for (int e = lane; e < own; e += 64) t[e] = a.rows[(size_t)s * mp + e];
        for (int e = own + lane; e < all; e += 64) {
            const int p = fresh[base_s[s] + e - own];
            t[e] = p, refs.p[p] = 1;
        }
        for (int e = all + lane; e < old_s[s]; e += 64) t[e] = -1;
    }
    if (tid < 4) a.out[tid] = tid == 1 ? (int)needed : 0;
    if (tid == 0) a.lists->copies = (int)copies, a.lists->moves = 0;
    if (a.pack) { /* the used pages from their number on move to the free ones below it */
        settle<false>(); /* the tables too */
        const uint32_t used = search<LDS>(refs, 0, npages, ~0u, sum_s, [](int r) { return r != 0; }, [](int, uint32_t) {});
        /* as many are free below it as used from it on, so holes' numbers never reach the pages that move: fresh[i] is the
         * i-th hole and fresh[p] where p goes */
        const uint32_t moves = search<LDS>(refs, 0, (int)used, ~0u, sum_s, [](int r) { return r == 0; },
                                           [&](int p, uint32_t i) { fresh[i] = p; });
        settle<LDS>();
        if (moves)
            (void)search<LDS>(refs, (int)used, npages, ~0u, sum_s, [](int r) { return r != 0; }, [&](int p, uint32_t i) {
                const int h = fresh[i];
                a.movers[i] = p, a.holes[i] = h, fresh[p] = h;
                refs.p[h] = refs.get(p), refs.p[p] = 0;
            });
        const int32_t *to = fresh;
        if (tid == 0) a.lists->moves = (int)moves;
        if (tid == 2 || tid == 3) a.out[tid] = (int)(tid == 2 ? used : moves);
        settle<LDS>();
        if (moves) {
            for (int s0 = wave; s0 < S; s0 += PP_SEQS * (PP / 64)) {
                int longest = 0;
#pragma unroll
                for (int u = 0; u < PP_SEQS; u++) {
                    const int s = s0 + u * (PP / 64);
                    if (s < S && all_s[s] > longest) longest = all_s[s];
                }
                for (int e = lane; e < longest; e += 64) {
                    int p[PP_SEQS];
#pragma unroll
                    for (int u = 0; u < PP_SEQS; u++) {
                        const int s = s0 + u * (PP / 64);
                        p[u] = s < S && e < all_s[s] ? a.pg.table[(size_t)s * mp + e] : -1;
                    }
#pragma unroll
                    for (int u = 0; u < PP_SEQS; u++)
                        if ((uint32_t)p[u] >= used && (uint32_t)p[u] < (uint32_t)npages)
                            a.pg.table[(size_t)(s0 + u * (PP / 64)) * mp + e] = to[p[u]];
                }
            }
        }
    }
    if (LDS) {
        __syncthreads();
        for (int p = tid; p < npages; p += PP) a.refs[p] = pages_s[p];
    }
}

struct CopyDev {
    const Lists *lists;
    const int32_t *movers, *holes;
    int caches, nkv, page, row_bytes; /* of one KV head */
    int scales;
    size_t block;
    int chunks; /* items of a head (a copy), of a block (a move) */
    void *kv[NMX_BATCH_KV_MAX];
};

/* n bytes (a multiple of 16), at most a chunk */
__device__ __forceinline__ void copy_chunk(char *dst, const char *src, size_t n) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const size_t at = (size_t)(i * PC + (int)threadIdx.x) * 16;
        v[i] = *(const u32x4 *)(src + (at < n ? at : 0));
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const size_t at = (size_t)(i * PC + (int)threadIdx.x) * 16;
        if (at < n) *(u32x4 *)(dst + at) = v[i];
    }
}

/* The first rows of pages, head by head, in every cache. */
__global__ __launch_bounds__(PC) void pages_copy_k(CopyDev a) {
    const long long items = (long long)a.lists->copies * a.caches * a.nkv * a.chunks;
    for (long long i = blockIdx.x; i < items; i += gridDim.x) {
        const int chunk = (int)(i % a.chunks), g = (int)(i / a.chunks % a.nkv);
        const int cache = (int)(i / a.chunks / a.nkv % a.caches);
        const int4 c = a.lists->copy[i / a.chunks / a.nkv / a.caches];
        const char *src = (const char *)a.kv[cache] + c.x * a.block;
        char *dst = (char *)a.kv[cache] + c.y * a.block;
        const size_t head = (size_t)g * a.page * a.row_bytes, n = (size_t)c.z * a.row_bytes, at = (size_t)chunk * PC_CHUNK;
        if (at < n) copy_chunk(dst + head + at, src + head + at, n - at < PC_CHUNK ? n - at : PC_CHUNK);
        if (a.scales && chunk == 0 && (int)threadIdx.x < c.z) { /* a page has at most 256 rows */
            const size_t s = (size_t)a.nkv * a.page * a.row_bytes + ((size_t)g * a.page + threadIdx.x) * 4;
            *(float *)(dst + s) = *(const float *)(src + s);
        }
    }
}

/* Whole pages, in every cache. */
__global__ __launch_bounds__(PC) void pages_move_k(CopyDev a) {
    const long long items = (long long)a.lists->moves * a.caches * a.chunks;
    for (long long i = blockIdx.x; i < items; i += gridDim.x) {
        const int chunk = (int)(i % a.chunks), cache = (int)(i / a.chunks % a.caches), m = (int)(i / a.chunks / a.caches);
        const size_t at = (size_t)chunk * PC_CHUNK, n = a.block - at;
        copy_chunk((char *)a.kv[cache] + a.holes[m] * a.block + at, (const char *)a.kv[cache] + a.movers[m] * a.block + at,
                   n < PC_CHUNK ? n : PC_CHUNK);
    }
}

size_t up16(size_t x) { return (x + 15) / 16 * 16; }

} // namespace

extern "C" {

size_t nmx_pages_work_bytes(int npages, int seqs, int max_pages) {
    if (npages < 1 || npages > (1 << 20) || seqs < 1 || seqs > NMX_BATCH_MAX || max_pages < 1 || max_pages > (1 << 16)) return 0;
    return up16(sizeof(Lists)) + 3 * up16((size_t)npages * 4) + up16((size_t)seqs * max_pages * 4);
}

int nmx_pages_update(nmx_ctx *ctx, const nmx_pages_args *p, void *work) {
    if (!ctx) return -1;
    if (!p) return nmx_fail(ctx, "nmx_pages_update: NULL argument");
    PagesDev a{};
    if (nmx_pages_check(ctx, p->pages, "nmx_pages_update", &a.pg)) return -1;
    if (!p->refs || !p->from || !p->keep || !p->add || !p->out || !work) return nmx_fail(ctx, "nmx_pages_update: NULL argument");
    if ((uintptr_t)work % 16) return nmx_fail(ctx, "nmx_pages_update: work not 16-byte aligned");
    if (p->caches < 0 || p->caches > NMX_BATCH_KV_MAX || (p->caches && !p->kv))
        return nmx_fail(ctx, "nmx_pages_update: caches=%d", p->caches);
    const int S = a.pg.seqs, np = a.pg.npages, mp = a.pg.max_pages;
    const size_t cb = a.pg.block * np, sb = (size_t)S * 4, wb = nmx_pages_work_bytes(np, S, mp);
    const NmxRange in[] = {{p->from, sb}, {p->keep, sb}, {p->add, sb}};
    NmxRange out[5 + NMX_BATCH_KV_MAX] = {{work, wb}, {a.pg.table, (size_t)S * mp * 4}, {a.pg.len, sb}, {p->refs, (size_t)np * 4},
                                          {p->out, 16}};
    CopyDev c{};
    int no = 5;
    for (int i = 0; i < p->caches; i++) {
        if (!p->kv[i] || (uintptr_t)p->kv[i] % 16) return nmx_fail(ctx, "nmx_pages_update: cache %d", i);
        c.kv[i] = p->kv[i];
        out[no++] = {p->kv[i], cb};
    }
    for (int i = 0; i < no; i++) {
        if (nmx_hits(in, out[i].p, out[i].bytes)) return nmx_fail(ctx, "nmx_pages_update: what is written overlaps an input");
        for (int k = 0; k < i; k++)
            if (nmx_overlap(out[i].p, out[i].bytes, out[k].p, out[k].bytes))
                return nmx_fail(ctx, "nmx_pages_update: two of the tables, caches, out and work overlap");
    }
    char *w = (char *)work;
    const size_t nb = up16((size_t)np * 4);
    a.refs = p->refs, a.from = p->from, a.keep = p->keep, a.add = p->add, a.pack = p->pack != 0, a.out = p->out;
    a.lists = (Lists *)w, w += up16(sizeof(Lists));
    a.fresh = (int32_t *)w, a.holes = (int32_t *)(w + nb), a.movers = (int32_t *)(w + 2 * nb);
    a.rows = (int32_t *)(w + 3 * nb);
    const nmx_on_device on(ctx);
    if (np <= PP_LDS) {
        static std::atomic<uint64_t> set0;
        if (nmx_dyn_lds(ctx, (const void *)pages_plan_k<true>, (size_t)PP_LDS * 8, set0)) return -1;
        pages_plan_k<true><<<1, PP, (size_t)np * 8, ctx->stream>>>(a.from, a.keep, a.add, a.pg.len, S, np, a);
    } else {
        pages_plan_k<false><<<1, PP, 0, ctx->stream>>>(a.from, a.keep, a.add, a.pg.len, S, np, a);
    }
    NMX_LAUNCHED(ctx, "pages_plan");
    if (!p->caches) return 0;
    const int kv = p->pages.kv_dtype, page = p->pages.page;
    c.lists = a.lists, c.movers = a.movers, c.holes = a.holes, c.caches = p->caches, c.nkv = a.pg.nkv, c.page = page;
    c.row_bytes = a.pg.hd * (kv == KV_F32 ? 4 : kv == KV_F16 ? 2 : 1), c.scales = kv == KV_I8, c.block = a.pg.block;
    c.chunks = (page * c.row_bytes + PC_CHUNK - 1) / PC_CHUNK;
    pages_copy_k<<<1024, PC, 0, ctx->stream>>>(c);
    NMX_LAUNCHED(ctx, "pages_copy");
    if (!p->pack) return 0;
    c.chunks = (int)((c.block + PC_CHUNK - 1) / PC_CHUNK);
    pages_move_k<<<2048, PC, 0, ctx->stream>>>(c);
    NMX_LAUNCHED(ctx, "pages_move");
    return 0;
}

} /* extern "C" */
