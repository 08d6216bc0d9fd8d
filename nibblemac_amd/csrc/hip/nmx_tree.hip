/* The commit of a verified tree (include/nmx.h nmx_tree_commit): the walk from the root along the
 * drafts that were chosen, and the move of what it accepted to where a chain's pass would have left
 * it. One launch: every workgroup redoes the walk (64 nodes: six shuffles and a ballot), so no second
 * launch waits for it; the rest is a copy of a few rows, bound by round trips to memory that wait for each
 * other: the parents, tokens and choices, then the position, then rows, then their stores. A path of four nodes (three
 * drafts) over 18 layers and 14 caches 5.0 us (5.2 MB, 1.0 us as a copy), one of ten 6.7 us (8.8 MB,
 * 1.7 us). One row at a time, each behind the last one's store, took 6.4 and 11.4 us. */
#include "nmx_internal.h"
#include "nmx_lanes.h"
#include "nmx_tree.h"

namespace {

constexpr int TC_ROWS = 8; /* rows of a thread on their way at once */

struct Commit {
    int n;
    const int32_t *parent, *tok, *choice;
    int32_t *out, *ctl, *vt;
    int layers, C, S; /* S = conv_k - 1 rows of conv state */
    float *state;
    const float *xin, *log;
    float *pend;
    int cap, row;
    int caches, nkv, max_ctx, row_bytes, scales;
    const int32_t *pos;
    int pos_off;
    size_t scale_at; /* bytes from a cache's start to its row scales */
    int conv_wgs, log_wgs, kv_wgs; /* workgroups of one layer's conv state, of its log rows, of one
                                    * cache's head */
    void *kv[NMX_TREE_KV_MAX];
};

/* The accepted path: path[i] for i < the result (path[0] = 0), known to every thread. */
__device__ int walk(const Commit &a, int *path, int *bonus) {
    __shared__ int s_e, s_bonus;
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int p;
        const unsigned long long set = tree_ancestors(a.parent, a.n, &p);
        const int tok = lane < a.n ? a.tok[lane] : -1, ch = lane < a.n ? a.choice[lane] : -1;
        const int want = __shfl(ch, p < 0 ? 0 : p);
        bool hit = lane < a.n && p >= 0 && want >= 0 && tok == want;
        /* of several children with the chosen token the first counts */
        for (unsigned long long m = __ballot(hit); m; m &= m - 1) {
            const int k = __ffsll((long long)m) - 1;
            if (__shfl(p, k) == p && k < lane) hit = false;
        }
        const unsigned long long good = __ballot(hit || lane == 0);
        const bool on = lane < a.n && (set & 1) && !(set & ~good);
        const unsigned long long chain = __ballot(on);
        if (on) path[__popcll(chain & ((1ull << lane) - 1))] = lane;
        const int last = 63 - __clzll((long long)chain);
        const int b = __shfl(ch, last);
        if (lane == 0) s_e = __popcll(chain), s_bonus = b;
    }
    __syncthreads();
    *bonus = s_bonus;
    return s_e;
}

__global__ __launch_bounds__(256) void tree_commit_k(Commit a) {
    __shared__ int path[NMX_TREE_MAX];
    int bonus;
    const int e = walk(a, path, &bonus), tid = threadIdx.x;
    int b = blockIdx.x;
    if (b == 0) {
        if (tid < a.n) a.out[2 + tid] = tid < e ? path[tid] : -1;
        if (tid == 0) {
            a.out[0] = e - 1;
            a.out[1] = bonus;
            if (a.ctl) a.ctl[1] = e, a.ctl[2] = e;
            if (a.vt) a.vt[0] = bonus;
        }
        return;
    }
    b--;
    if (b < a.layers * a.conv_wgs) { /* conv state: the last S of [state; raw inputs of the path] */
        const int l = b / a.conv_wgs, c = b % a.conv_wgs * 256 + tid;
        if (c >= a.C) return;
        float *st = a.state + (size_t)l * a.S * a.C + c;
        const float *xi = a.xin + (size_t)l * a.cap * a.C + c;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (j >= a.S) continue;
            const int r = j + e;
            v[j] = r < a.S ? st[(size_t)r * a.C] : xi[(size_t)path[r - a.S] * a.C];
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < a.S) st[(size_t)j * a.C] = v[j];
        return;
    }
    b -= a.layers * a.conv_wgs;
    if (b < a.layers * a.log_wgs) { /* pending rows: the path's log rows */
        const int l = b / a.log_wgs, x = b % a.log_wgs * 256 + tid;
        if (x >= a.row) return;
        const float *lg = a.log + (size_t)l * a.cap * a.row + x;
        float *pd = a.pend + (size_t)l * a.cap * a.row + x;
        for (int i0 = 0; i0 < e; i0 += TC_ROWS) {
            float v[TC_ROWS];
#pragma unroll
            for (int k = 0; k < TC_ROWS; k++) v[k] = lg[(size_t)path[i0 + k < e ? i0 + k : e - 1] * a.row];
#pragma unroll
            for (int k = 0; k < TC_ROWS; k++)
                if (i0 + k < e) pd[(size_t)(i0 + k) * a.row] = v[k];
        }
        return;
    }
    b -= a.layers * a.log_wgs;
    /* cache rows to consecutive slots. path[i] >= i and grows: no row is written before it is read where
     * a thread takes its own bytes of the rows in order, or some rows' in order before any of theirs */
    const int cache = b / (a.nkv * a.kv_wgs), g = b / a.kv_wgs % a.nkv, w = b % a.kv_wgs;
    const long long p = (long long)*a.pos + a.pos_off;
    const int words = a.row_bytes / 4 + (a.scales ? 1 : 0), x = w * 256 + tid;
    if (x >= words) return;
    char *c = (char *)a.kv[cache];
    char *base;
    size_t step;
    if (x < a.row_bytes / 4) base = c + (size_t)g * a.max_ctx * a.row_bytes + 4 * x, step = a.row_bytes;
    else base = c + a.scale_at + (size_t)g * a.max_ctx * 4, step = 4;
    for (int i0 = 1; i0 < e; i0 += TC_ROWS) {
        uint32_t v[TC_ROWS];
#pragma unroll
        for (int k = 0; k < TC_ROWS; k++) { /* a row outside the cache is not moved: any row inside stands for it */
            const long long from = p + path[i0 + k < e ? i0 + k : e - 1];
            v[k] = *(const uint32_t *)(base + (size_t)(from >= 0 && from < a.max_ctx ? from : 0) * step);
        }
#pragma unroll
        for (int k = 0; k < TC_ROWS; k++) {
            if (i0 + k >= e) continue;
            const long long from = p + path[i0 + k], to = p + i0 + k;
            if (from == to || to < 0 || from >= a.max_ctx) continue;
            *(uint32_t *)(base + (size_t)to * step) = v[k];
        }
    }
}

/* Whether anything that the call writes overlaps anything else that it reads or writes (shapes checked). A
 * cache's rows and an array's may move within themselves; vt may be tok, whose first is never read. */
bool overlaps(const nmx_tree_commit_args &p) {
    struct Range {
        const void *p;
        size_t bytes;
    };
    const size_t nb = (size_t)p.n * 4, rows = (size_t)p.layers * p.cap, lb = rows * p.row * 4;
    const bool lin = p.layers > 0, conv = lin && p.conv_k > 1, kvs = p.caches > 0;
    Range w[5 + NMX_TREE_KV_MAX] = {{p.out, nb + 8}, {p.ctl ? p.ctl + 1 : nullptr, p.ctl ? 8u : 0u}, {p.vt, p.vt ? 4u : 0u},
                                    {p.state, conv ? (size_t)p.layers * (p.conv_k - 1) * p.C * 4 : 0}, {p.pend, lin ? lb : 0}};
    const Range in[] = {{p.parent, nb}, {p.tok, nb}, {p.choice, nb}, {p.pos, kvs ? 4u : 0u}, {p.log, lin ? lb : 0},
                        {p.xin, conv ? rows * p.C * 4 : 0}, {p.ctl, p.ctl ? 4u : 0u}};
    int nw = 5;
    const size_t kb = kvs ? nmx_kv_bytes(p.kv_dtype, p.nkv, p.max_ctx, p.hd) : 0;
    for (int i = 0; i < p.caches; i++) w[nw++] = {p.kv[i], kb};
    for (int i = 0; i < nw; i++) {
        for (const Range &x : in)
            if (nmx_overlap(w[i].p, w[i].bytes, x.p, x.bytes) && !(w[i].p == p.vt && x.p == p.tok && p.vt == p.tok)) return true;
        for (int k = 0; k < i; k++)
            if (nmx_overlap(w[i].p, w[i].bytes, w[k].p, w[k].bytes)) return true;
    }
    return false;
}

} // namespace

extern "C" {

int nmx_tree_commit(nmx_ctx *ctx, const nmx_tree_commit_args *p) {
    if (!ctx) return -1;
    if (!p) return nmx_fail(ctx, "nmx_tree_commit: NULL argument");
    if (p->n < 1 || p->n > NMX_TREE_MAX) return nmx_fail(ctx, "nmx_tree_commit: n=%d", p->n);
    if (!p->parent || !p->tok || !p->choice || !p->out) return nmx_fail(ctx, "nmx_tree_commit: NULL argument");
    Commit a{};
    a.n = p->n, a.parent = p->parent, a.tok = p->tok, a.choice = p->choice;
    a.out = p->out, a.ctl = p->ctl, a.vt = p->vt;
    if (p->layers) {
        if (p->layers < 0 || p->layers > 1024 || p->C < 1 || p->C > (1 << 20) || p->conv_k < 1 || p->conv_k > 8 ||
            p->cap < p->n || p->cap > 4096 || p->row < 1 || p->row > (1 << 24))
            return nmx_fail(ctx, "nmx_tree_commit: bad shape layers=%d C=%d conv_k=%d cap=%d row=%d", p->layers, p->C,
                            p->conv_k, p->cap, p->row);
        if (!p->log || !p->pend || (p->conv_k > 1 && (!p->state || !p->xin)))
            return nmx_fail(ctx, "nmx_tree_commit: NULL argument");
        a.layers = p->layers, a.C = p->C, a.S = p->conv_k - 1;
        a.state = p->state, a.xin = p->xin, a.log = p->log, a.pend = p->pend, a.cap = p->cap, a.row = p->row;
        a.conv_wgs = a.S ? (p->C + 255) / 256 : 0;
        a.log_wgs = (p->row + 255) / 256;
    }
    if (p->caches) {
        if (p->caches < 0 || p->caches > NMX_TREE_KV_MAX || p->nkv < 1 || p->nkv > 1024 || p->max_ctx < 1 ||
            p->max_ctx > (1 << 20) || p->hd < 64 || p->hd > 512 || p->hd % 64 || p->kv_dtype < 0 || p->kv_dtype > 2)
            return nmx_fail(ctx, "nmx_tree_commit: bad caches %d nkv=%d max_ctx=%d hd=%d kv_dtype=%d", p->caches, p->nkv,
                            p->max_ctx, p->hd, p->kv_dtype);
        if (!p->kv || !p->pos) return nmx_fail(ctx, "nmx_tree_commit: NULL argument");
        for (int i = 0; i < p->caches; i++) {
            if (!p->kv[i] || (uintptr_t)p->kv[i] % 4) return nmx_fail(ctx, "nmx_tree_commit: cache %d", i);
            a.kv[i] = p->kv[i];
        }
        a.caches = p->caches, a.nkv = p->nkv, a.max_ctx = p->max_ctx, a.pos = p->pos, a.pos_off = p->pos_off;
        a.row_bytes = p->hd * (p->kv_dtype == 0 ? 4 : p->kv_dtype == 1 ? 2 : 1);
        a.scales = p->kv_dtype == 2;
        a.scale_at = (size_t)p->nkv * p->max_ctx * p->hd;
        a.kv_wgs = (a.row_bytes / 4 + a.scales + 255) / 256;
    }
    if (overlaps(*p)) return nmx_fail(ctx, "nmx_tree_commit: what is written overlaps something else");
    const nmx_on_device on(ctx);
    const size_t wgs = 1 + (size_t)a.layers * (a.conv_wgs + a.log_wgs) + (size_t)a.caches * a.nkv * a.kv_wgs;
    tree_commit_k<<<(unsigned)wgs, 256, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "tree_commit");
    return 0;
}

} /* extern "C" */
