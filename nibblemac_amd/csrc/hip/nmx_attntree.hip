/* Gated attention of a tree of drafts over the KV cache (include/nmx.h nmx_attn_tree_prep,
 * nmx_attn_tree): o = softmax(q K^T scale) V sigmoid(gate) over the context's positions [0, pos) and
 * the node's own ancestors, whose rows are at pos + node.
 *
 * Every node sees the whole context, so that part has no mask: attn_tree_ctx_k takes it as dense
 * tiles on the matrix cores, split over the positions, with a running maximum and sum per row.
 * What differs by node are at most 64 rows of the tree itself; attn_tree_join_k, one workgroup per
 * (node, head), adds a node's ancestors in 32 bits (rows that it does not see are never read, so
 * whatever they hold cannot reach it) to the parts of the context, and gates and stores the row.
 *
 * 32-bit results from 16-bit matrix instructions: every operand is split into a binary16 high part
 * and the binary16 rest, which together hold 22 bits; a query row, an fp32 cache row and an int8
 * row's scale are first brought to a power of two of their own, so that neither part leaves
 * binary16's range, and the softmax weights are taken 2^12 high. A binary16 cache's rows and int8
 * codes are exact as they are: two products per pair (q or weight high, low); an fp32 row has
 * two parts itself: three products, the low-low one left out (2^-22 of the row).
 *
 * Times of both kernels on MI355X, 8 heads on 2 of 256 (and of each in a kernel trace, context + join): 64 nodes
 * over 100000 binary16 positions 122 us (the same ones again and again 113), 428 TFLOP/s of the definition's products and twice that of
 * the matrix cores', which a large binary16 product runs at 1106 (traced 111 at least and 120 at the median + 14);
 * 37 nodes over 4001 int8 25.3 us (17.3 + 8.9); 9 nodes over 600
 * fp32 15.1 us (10.3 + 5.6) and one node over 20000 binary16 16.8 us (11.2 + 6.1): the latter 41 MB, 8 us
 * as a copy; the others are chains of round trips to memory (position, rows, barrier, parts, position, parts,
 * rows). Long fp32 and int8 contexts (before the tiles' waves worked a phase apart): 5 nodes over 30000 fp32 40 us (123 MB, 24 as
 * a copy), 64 of them 87; 9 over 100000 int8 58 us (104 MB, 20), 64 of them 143.
 *
 * The largest case is bound by the matrix cores and the vector unit together (counted: either is active in 51 % of the CUs'
 * busy cycles, LDS in 32 % without a bank conflict): two waves of a SIMD leave the one idle while both need the other. */
#include "nmx_internal.h"
#include "nmx_a8.h"
#include "nmx_attn.h"
#include "nmx_attnmx.h"
#include "nmx_lanes.h"
#include "nmx_math.h"
#include "nmx_rms.h"
#include "nmx_tree.h"

namespace {

constexpr int AT_MAXS = 256;     /* parts that the context is split into, at most */
struct TreeAttn {
    int n, nh, nkv, hd, max_ctx;
    const float *q;
    const void *kc, *vc;
    const int32_t *pos, *parent;
    int pos_off;
    float scale;
    float *part;   /* [splits][n nh][hd] weighted values, 2^12 high */
    float4 *stat;  /* [splits][n nh]: maximum of the scores, the values' exponent (columns below 256),
                    * sum, the values' exponent (columns from 256) */
    int splits; /* a part is a whole number of tiles */
    int jcols;        /* columns of a join's workgroup: hd over a divisor of hd / 64 */
    float *o;
    int8_t *aq;
    float *ad, *afs;
};

/* The slot of node 0, kept within [-64, max_ctx]: past either end no node has a slot. */
__device__ __forceinline__ int tree_slot0(const int32_t *pos, int pos_off, int max_ctx) {
    const long long p = (long long)*pos + pos_off;
    return p < -NMX_TREE_MAX ? -NMX_TREE_MAX : p > max_ctx ? max_ctx : (int)p;
}
__device__ __forceinline__ int ctx_len(const TreeAttn &a) {
    const int p = tree_slot0(a.pos, a.pos_off, a.max_ctx);
    return p < 0 ? 0 : p;
}
__device__ __forceinline__ int part_len(const TreeAttn &a, int len) {
    const int per = (len + a.splits - 1) / a.splits;
    return (per + AT_P - 1) / AT_P * AT_P;
}

/* ---- the tree's keys, values and queries (attn_prep_k's operations, RoPE at the node's depth) */
template <int KVT>
__global__ __launch_bounds__(512) void attn_tree_prep_k(nmx_attn_dev a, const int32_t *parent) {
    extern __shared__ float sq[];
    __shared__ float buf[512];
    __shared__ float red[8];
    const int t = blockIdx.y, u = blockIdx.x, i = threadIdx.x, hd = a.hd, h2 = a.rot / 2;
    const unsigned long long set = __shfl(tree_ancestors(parent, a.n, nullptr), t);
    const int p0 = tree_slot0(a.pos, a.pos_off, a.max_ctx), slot = p0 + t;
    int p = p0 + __popcll(set) - 1;
    p = p < 0 ? 0 : p < a.max_ctx ? p : a.max_ctx - 1; /* the RoPE tables have max_ctx rows */
    const bool is_k = u < a.nkv;
    float v;
    if (is_k) v = a.k_in[(size_t)t * a.nkv * hd + u * hd + i];
    else v = a.q[((size_t)t * a.nh + (u - a.nkv)) * 2 * hd + i];
    sq[i] = v * v;
    __syncthreads();
    const float ss = ordered_sum4(sq, hd, red);
    const float r = 1.0f / sqrtf(ss / (float)hd + a.eps);
    v = (v * r) * (is_k ? a.k_norm[i] : a.q_norm[i]);
    buf[i] = v;
    __syncthreads();
    if (i < h2) {
        const float c = a.rcos[(size_t)p * h2 + i], s = a.rsin[(size_t)p * h2 + i];
        v = buf[i] * c - buf[i + h2] * s;
    } else if (i < 2 * h2) {
        const float c = a.rcos[(size_t)p * h2 + i - h2], s = a.rsin[(size_t)p * h2 + i - h2];
        v = buf[i] * c + buf[i - h2] * s;
    }
    if (!is_k) {
        a.q[((size_t)t * a.nh + (u - a.nkv)) * 2 * hd + i] = v;
    } else if (slot >= 0 && slot < a.max_ctx) { /* uniform per workgroup; no row outside the cache */
        const size_t R = (size_t)u * a.max_ctx + slot;
        kv_store<KVT>(a.kc, a, R, i, v, red);
        kv_store<KVT>(a.vc, a, R, i, a.v_in[(size_t)t * a.nkv * hd + u * hd + i], red);
    }
}

/* ---- the context (the tiles: nmx_attnmx.h) -------------------------------------------- */
/* One head of a cache: its rows and, int8, their scales. A head has at most 2^20 rows of 512 values, so
 * a byte offset in it has 32 bits and an address is a scalar base plus one register. */
template <int KVT>
struct Head {
    const char *rows;
    const float *scales;
    int hd;
    static constexpr int SIZE = KVT == KV_F32 ? 4 : KVT == KV_F16 ? 2 : 1;
    __device__ __forceinline__ Head(const TreeAttn &a, const void *cache, int g)
        : rows((const char *)cache + (size_t)g * a.max_ctx * a.hd * SIZE),
          scales((const float *)((const char *)cache + (size_t)a.nkv * a.max_ctx * a.hd) + (size_t)g * a.max_ctx), hd(a.hd) {}
    __device__ __forceinline__ const char *at(int p, int col) const { return rows + (uint32_t)(p * hd + col) * SIZE; }
    __device__ __forceinline__ int page_of(int) const { return 0; } /* one block */
    __device__ __forceinline__ uint32_t where(int, int p, int col) const { return (uint32_t)(p * hd + col) * SIZE; }
    __device__ __forceinline__ Raw8<KVT> load8(uint32_t where) const {
        Raw8<KVT> r;
        const char *s = rows + where;
        if constexpr (KVT == KV_F32) r.a = *(const uint4 *)s, r.b = *(const uint4 *)(s + 16);
        else if constexpr (KVT == KV_F16) r.a = *(const uint4 *)s;
        else r.a = *(const uint2 *)s;
        return r;
    }
    __device__ __forceinline__ float scale(int, int p) const {
        if constexpr (KVT == KV_I8) return scales[(uint32_t)p];
        return 1.0f;
    }
};
/* This part's result of a row: columns d0 .. of the weighted values, maximum, exponent and sum. */
template <int DT>
__device__ __forceinline__ void store_part(const TreeAttn &a, const Running<DT> &r, int s, int hrow, int d0, int gq) {
    const size_t at = (size_t)s * a.n * a.nh + hrow;
#pragma unroll
    for (int d = 0; d < DT; d++)
        if (d0 + 16 * d < a.hd) *(float4v *)(a.part + at * a.hd + d0 + 16 * d + 4 * gq) = r.o[d];
    if (gq == 0) { /* the halves of 512 columns have value exponents of their own */
        if (d0) a.stat[at].w = (float)r.ve;
        else a.stat[at].x = r.m, a.stat[at].y = (float)r.ve, a.stat[at].z = r.l;
    }
}

template <int HDP, int KVT>
__global__ __launch_bounds__(64 * ctx_waves<HDP>()) void attn_tree_ctx_k(TreeAttn a) {
    constexpr int OD = HDP > 256 ? 256 : HDP, KS = HDP / 32;
    extern __shared__ uint4 smem[];
    const int lane = lane_id(), wave = wave_id(), c = lane & 15, gq = lane >> 4;
    const int s = blockIdx.x % a.splits, g = blockIdx.x / a.splits % a.nkv, mt = blockIdx.x / a.splits / a.nkv;
    const int d0 = blockIdx.y * OD; /* the output columns: of 512, half */
    const int hd = a.hd, rep = a.nh / a.nkv, rows = a.n * rep;
    const int row0 = (mt * ctx_waves<HDP>() + wave) * 16, row = row0 + c;
    const int hrow = row < rows ? (row / rep) * a.nh + g * rep + row % rep : -1; /* (node, head) */
    const bool busy = row0 < rows;
    QueryRow<KS> qr(a.q + (size_t)(hrow < 0 ? 0 : hrow) * 2 * hd, hrow >= 0, hd, gq);
    const Head<KVT> kh(a, a.kc, g), vh(a, a.vc, g);
    const int len = ctx_len(a), per = part_len(a, len), p0 = s * per;
    if (per == 0 || p0 >= len) return;
    const int p1 = p0 + per < len ? p0 + per : len;
    Running<OD / 16> r;
    attend_tiles<HDP, KVT>(r, qr, a.scale, kh, vh, p0, p1, p1, d0, busy, smem);
    r.l -= r.lc;
    r.l = nmx_sum_quarters(r.l);
    if (hrow >= 0) store_part(a, r, s, hrow, d0, gq);
}

/* ---- the node's ancestors, and the join ---------------------------------------------------- */
constexpr int JT = 512; /* threads of a join: of 1024, two workgroups do not fit a CU's registers (64 nodes 21 against 14 us) */

/* Workgroup: a node and head, blockIdx.y a group of a.jcols columns of it. */
template <int KVT>
__global__ __launch_bounds__(JT) void attn_tree_join_k(TreeAttn a) {
    __shared__ float sc[64], red[2 * (JT / 64)], acc_s[JT * 4], w_s[2][AT_MAXS];
    __shared__ int anc_s[64];
    const int lane = lane_id(), wave = wave_id(), tid = 64 * wave + lane;
    const int hrow = blockIdx.x, t = hrow / a.nh, h = hrow % a.nh, hd = a.hd, nd = hd >> 6;
    const int g = h / (a.nh / a.nkv), rows = a.n * a.nh, c0 = blockIdx.y * a.jcols;
    const float *qp = a.q + (size_t)hrow * 2 * hd;
    /* requested at entry, whatever the context's length: a part's numbers past the last one are not used */
    const int above = lane < a.n ? tree_parent(a.parent, lane) : -1;
    float4 st = a.stat[(size_t)(tid < a.splits ? tid : 0) * rows + hrow]; /* thread = part */
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = qp[i < nd ? lane + 64 * i : lane];
    const float gate = qp[hd + c0 + (tid < a.jcols ? tid : 0)];
    const int len = ctx_len(a), per = part_len(a, len), parts = per ? (len + per - 1) / per : 0;
    /* slots of jcols / 4 threads: a thread takes 4 columns of every slots-th row of a sum */
    const int per_slot = a.jcols >> 2, slots = JT / per_slot, slot = tid / per_slot, col = c0 + tid % per_slot * 4;
    constexpr int PB = 8; /* rows of a slot requested at once */
    float4 pr[PB];
    auto ask = [&](int s0) {
#pragma unroll
        for (int u = 0; u < PB; u++) {
            const int s = s0 + u * slots;
            if (s < parts) pr[u] = *(const float4 *)(a.part + ((size_t)s * rows + hrow) * hd + col);
        }
    };
    if (slot < slots) ask(slot);
    /* the ancestors' rows inside the cache, from the node up: lane i keeps the i-th */
    const int p0 = tree_slot0(a.pos, a.pos_off, a.max_ctx);
    int na = 0, mine = 0;
    for (int x = t; x >= 0; x = __builtin_amdgcn_readlane(above, x)) {
        if (p0 + x < 0 || p0 + x >= a.max_ctx) continue;
        mine = lane == na ? x : mine;
        na++;
    }
    if (wave == 0) anc_s[lane] = mine;
    const Head<KVT> kh(a, a.kc, g);
    /* scores: a wave for each ancestor */
    float mt = -INFINITY;
    for (int i = wave; i < na; i += JT / 64) {
        const int p = p0 + __builtin_amdgcn_readlane(mine, i);
        const float rs = kh.scale(0, p);
        float d = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < nd) {
                const char *at = kh.at(p, lane + 64 * k);
                float x;
                if constexpr (KVT == KV_F32) x = *(const float *)at;
                else if constexpr (KVT == KV_F16) x = kv_half_value(*(const unsigned short *)at);
                else x = (float)*(const int8_t *)at * rs;
                d = __builtin_fmaf(q[k], x, d);
            }
        d = sum_lanes(d) * (a.scale * AT_LOG2E);
        if (lane == 0) sc[i] = d;
        mt = fmaxf(mt, d);
    }
    if (tid >= parts) st = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    mt = fmaxf(mt, nmx_max_f32_wave(st.x));
    if (lane == 0) red[wave] = mt;
    nmx_lds_sync();
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < JT / 64; w++) m = fmaxf(m, red[w]);
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    if (tid < parts) { /* a part's weight, for its sum and for its 2^12 high values */
        const float w = __builtin_amdgcn_exp2f(st.x - ref);
        l = st.z * w;
        w_s[0][tid] = ldexpf(w, (int)st.y - 12);
        w_s[1][tid] = hd > 256 ? ldexpf(w, (int)st.w - 12) : 0.0f;
    }
    if (tid < na) {
        const float w = __builtin_amdgcn_exp2f(sc[tid] - ref);
        sc[tid] = w; /* no other thread reads it before the next barrier */
        l += w;
    }
    l = sum_lanes(l);
    if (lane == 0) red[JT / 64 + wave] = l;
    nmx_lds_sync();
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float w, float4 x) {
        acc.x = __builtin_fmaf(w, x.x, acc.x), acc.y = __builtin_fmaf(w, x.y, acc.y);
        acc.z = __builtin_fmaf(w, x.z, acc.z), acc.w = __builtin_fmaf(w, x.w, acc.w);
    };
    if (slot < slots) {
        const float *ws = w_s[col >> 8];
        for (int s0 = slot; s0 < parts; s0 += PB * slots) {
            if (s0 != slot) ask(s0);
#pragma unroll
            for (int u = 0; u < PB; u++) {
                const int s = s0 + u * slots;
                if (s < parts) add(ws[s], pr[u]);
            }
        }
        for (int i = slot; i < na; i += slots)
            add(sc[i], kv_load4<KVT>(a.vc, (size_t)g * a.max_ctx + p0 + anc_s[i], hd, col,
                                     KVT == KV_I8 ? (const float *)((const int8_t *)a.vc + (size_t)a.nkv * a.max_ctx * hd) : nullptr));
        *(float4 *)(acc_s + slot * a.jcols + col - c0) = acc;
    }
    nmx_lds_sync();
    if (tid < a.jcols) {
        float sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < JT / 64; w++) sum += red[JT / 64 + w];
        for (int w = 0; w < slots; w++) v += acc_s[w * a.jcols + tid];
        v = sum > 0.0f || !(sum == sum) ? v / sum : 0.0f; /* no row at all in sight: 0 */
        v = v * nmx_sigmoid(gate);
        const int at = h * hd + c0 + tid;
        a.o[(size_t)t * a.nh * hd + at] = v;
        if (a.aq) a8_block(v, at >> 5, t, a.n, a.aq, a.ad, a.afs); /* jcols % 64 == 0: whole blocks */
    }
}

/* How the context is divided among workgroups. */
struct Plan {
    int hdp, mtiles, splits, halves, jcols;
    size_t part_bytes, bytes;
};

Plan make_plan(int n, int nh, int nkv, int hd) {
    Plan p;
    p.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512;
    const int tiles = (n * (nh / nkv) + 15) / 16, od = p.hdp > 256 ? 256 : p.hdp;
    const int waves = p.hdp > 256 ? 4 : 8;
    p.mtiles = (tiles + waves - 1) / waves;
    p.halves = p.hdp / od;
    /* a workgroup to a CU */
    const int s = 256 / (nkv * p.mtiles * p.halves);
    p.splits = s < 1 ? 1 : s > AT_MAXS ? AT_MAXS : s;
    /* with few rows their columns are shared out too, while the chip holds the workgroups in one round */
    int groups = 1;
    for (int k = 2; k <= hd / 64; k++)
        if (hd / 64 % k == 0 && n * nh * k <= 512) groups = k;
    p.jcols = hd / groups;
    p.part_bytes = (size_t)p.splits * n * nh * hd * 4;
    p.bytes = p.part_bytes + (size_t)p.splits * n * nh * sizeof(float4);
    return p;
}

template <int HDP, int KVT>
int launch_ctx(nmx_ctx *ctx, const TreeAttn &a, const Plan &p) {
    const dim3 grid((unsigned)(p.splits * a.nkv * p.mtiles), (unsigned)p.halves);
    static std::atomic<uint64_t> set0;
    constexpr int lds = ctx_lds<HDP, KVT>();
    if (nmx_dyn_lds(ctx, (const void *)attn_tree_ctx_k<HDP, KVT>, lds, set0)) return -1;
    attn_tree_ctx_k<HDP, KVT><<<grid, 64 * ctx_waves<HDP>(), lds, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "attn_tree_ctx");
    return 0;
}

template <int KVT>
int launch_tree(nmx_ctx *ctx, const TreeAttn &a, const Plan &p) {
    const int rc = p.hdp == 64 ? launch_ctx<64, KVT>(ctx, a, p) : p.hdp == 128 ? launch_ctx<128, KVT>(ctx, a, p) :
                   p.hdp == 256 ? launch_ctx<256, KVT>(ctx, a, p) : launch_ctx<512, KVT>(ctx, a, p);
    if (rc) return rc;
    attn_tree_join_k<KVT><<<dim3((unsigned)(a.n * a.nh), (unsigned)(a.hd / a.jcols)), JT, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "attn_tree_join");
    return 0;
}

struct Range {
    const void *p;
    size_t bytes;
};
template <int N>
bool hits(const Range (&in)[N], const void *out, size_t bytes) {
    for (const Range &x : in)
        if (x.p && nmx_overlap(out, bytes, x.p, x.bytes)) return true;
    return false;
}

/* the arguments that both calls use */
int tree_shape(nmx_ctx *ctx, const nmx_attn_args *p, const int32_t *parent, const char *what) {
    if (!p || !parent) return nmx_fail(ctx, "%s: NULL argument", what);
    if (p->n < 1 || p->n > NMX_TREE_MAX || p->nkv < 1 || p->nh < p->nkv || p->nh % p->nkv || p->nh > 1024 ||
        p->hd < 64 || p->hd > 512 || p->hd % 64 || p->max_ctx < 1 || p->max_ctx > (1 << 20))
        return nmx_fail(ctx, "%s: bad shape n=%d nh=%d nkv=%d hd=%d max_ctx=%d", what, p->n, p->nh, p->nkv, p->hd,
                        p->max_ctx);
    if (p->kv_dtype < KV_F32 || p->kv_dtype > KV_I8) return nmx_fail(ctx, "%s: kv_dtype %d", what, p->kv_dtype);
    if (!p->q || !p->kc || !p->vc || !p->pos) return nmx_fail(ctx, "%s: NULL argument", what);
    if ((uintptr_t)p->q % 16 || (uintptr_t)p->kc % 16 || (uintptr_t)p->vc % 16)
        return nmx_fail(ctx, "%s: q or a cache not 16-byte aligned", what);
    const size_t kb = nmx_kv_bytes(p->kv_dtype, p->nkv, p->max_ctx, p->hd), qb = (size_t)p->n * p->nh * 2 * p->hd * 4;
    if (nmx_overlap(p->q, qb, p->kc, kb) || nmx_overlap(p->q, qb, p->vc, kb) || nmx_overlap(p->kc, kb, p->vc, kb))
        return nmx_fail(ctx, "%s: q and the caches overlap", what);
    return 0;
}

} // namespace

extern "C" {

int nmx_attn_tree_prep(nmx_ctx *ctx, const nmx_attn_args *p, const int32_t *parent) {
    if (!ctx) return -1;
    if (tree_shape(ctx, p, parent, "nmx_attn_tree_prep")) return -1;
    if (p->rot < 0 || p->rot % 2 || p->rot > p->hd || !p->k_in || !p->v_in || !p->q_norm || !p->k_norm ||
        (p->rot && (!p->rope_cos || !p->rope_sin)))
        return nmx_fail(ctx, "nmx_attn_tree_prep: bad arguments");
    const size_t kb = nmx_kv_bytes(p->kv_dtype, p->nkv, p->max_ctx, p->hd), qb = (size_t)p->n * p->nh * 2 * p->hd * 4;
    const size_t ib = (size_t)p->n * p->nkv * p->hd * 4, hb = (size_t)p->hd * 4, rb = (size_t)p->max_ctx * (p->rot / 2) * 4;
    const Range in[] = {{p->k_in, ib}, {p->v_in, ib}, {p->q_norm, hb}, {p->k_norm, hb}, {p->rope_cos, rb},
                        {p->rope_sin, rb}, {p->pos, 4}, {parent, (size_t)p->n * 4}};
    if (hits(in, p->q, qb) || hits(in, p->kc, kb) || hits(in, p->vc, kb))
        return nmx_fail(ctx, "nmx_attn_tree_prep: q or a cache overlaps an input");
    const nmx_attn_dev a{p->n, p->nh, p->nkv, p->hd, p->rot, p->max_ctx, p->q, p->k_in, p->v_in, p->q_norm,
                         p->k_norm, p->eps, p->scale, p->rope_cos, p->rope_sin, p->kc, p->vc, p->pos,
                         p->pos_off, nullptr, nullptr, nullptr, nullptr, p->n};
    const nmx_on_device on(ctx);
    const dim3 grid((unsigned)(p->nkv + p->nh), (unsigned)p->n);
    const size_t lds = (size_t)p->hd * 4;
    if (p->kv_dtype == KV_F16) attn_tree_prep_k<KV_F16><<<grid, (unsigned)p->hd, lds, ctx->stream>>>(a, parent);
    else if (p->kv_dtype == KV_I8) attn_tree_prep_k<KV_I8><<<grid, (unsigned)p->hd, lds, ctx->stream>>>(a, parent);
    else attn_tree_prep_k<KV_F32><<<grid, (unsigned)p->hd, lds, ctx->stream>>>(a, parent);
    NMX_LAUNCHED(ctx, "attn_tree_prep");
    return 0;
}

size_t nmx_attn_tree_work_bytes(int n, int nh, int nkv, int hd) {
    if (n < 1 || n > NMX_TREE_MAX || nkv < 1 || nh < nkv || nh % nkv || nh > 1024 || hd < 64 || hd > 512 || hd % 64)
        return 0;
    return make_plan(n, nh, nkv, hd).bytes;
}

int nmx_attn_tree(nmx_ctx *ctx, const nmx_attn_args *p, const int32_t *parent, void *work) {
    if (!ctx) return -1;
    if (tree_shape(ctx, p, parent, "nmx_attn_tree")) return -1;
    if (!p->o || !work || (p->a8.q && (!p->a8.d || !p->a8.fs))) return nmx_fail(ctx, "nmx_attn_tree: NULL argument");
    if ((uintptr_t)work % 16) return nmx_fail(ctx, "nmx_attn_tree: work not 16-byte aligned");
    const Plan pl = make_plan(p->n, p->nh, p->nkv, p->hd);
    const size_t kb = nmx_kv_bytes(p->kv_dtype, p->nkv, p->max_ctx, p->hd), ob = (size_t)p->n * p->nh * p->hd * 4;
    const Range in[] = {{p->q, 2 * ob}, {p->kc, kb}, {p->vc, kb}, {p->pos, 4}, {parent, (size_t)p->n * 4}};
    const size_t ab = p->a8.q ? ob : 0; /* a byte a value, a float to 32 each in d and fs */
    const Range out[] = {{work, pl.bytes}, {p->o, ob}, {p->a8.q, ab / 4}, {p->a8.d, ab / 32}, {p->a8.fs, ab / 32}};
    for (int i = 0; i < 5; i++) {
        if (hits(in, out[i].p, out[i].bytes)) return nmx_fail(ctx, "nmx_attn_tree: an output or work overlaps an input");
        for (int k = 0; k < i; k++)
            if (nmx_overlap(out[i].p, out[i].bytes, out[k].p, out[k].bytes))
                return nmx_fail(ctx, "nmx_attn_tree: outputs and work overlap");
    }
    const TreeAttn a{p->n, p->nh, p->nkv, p->hd, p->max_ctx, p->q, p->kc, p->vc, p->pos, parent, p->pos_off,
                     p->scale, (float *)work, (float4 *)((char *)work + pl.part_bytes), pl.splits,
                     pl.jcols, p->o, p->a8.q, p->a8.d, p->a8.fs};
    const nmx_on_device on(ctx);
    if (p->kv_dtype == KV_F16) return launch_tree<KV_F16>(ctx, a, pl);
    if (p->kv_dtype == KV_I8) return launch_tree<KV_I8>(ctx, a, pl);
    return launch_tree<KV_F32>(ctx, a, pl);
}

} /* extern "C" */
