/* Gated attention of a batch of sequences over paged KV caches (include/nmx.h nmx_attn_batch_prep,
 * nmx_attn_batch): o = softmax(q K^T scale) V sigmoid(gate) of every row over its own sequence up to its
 * own position, prefixes that a group of sequences shares read once for the group.
 *
 * The work is a list of segments: for each group the rows of all its sequences against the shared prefix,
 * for each sequence its rows against what follows. A segment has units (KV head, tile of query rows), a
 * unit steps of 32 positions. Lengths are on the device, so every workgroup makes the list itself (one wave, a scan
 * over at most 512 segments) and takes its share of the steps, whatever the lengths: a share may end one unit and
 * begin others. What a share finds of a unit is a part (weighted values, maximum, sum); the join adds a row's parts in
 * order.
 *
 * Two kinds of segments. Up to 8 query rows (a token of a sequence: the heads of a KV group) are bound by the cache's bytes:
 * a wave streams rows from memory into its registers, the keys of the next positions requested while the values of the
 * current ones are added and the other way round, without a barrier on the way; shares are a wave's, so that
 * the round trips at which a short sequence begins and ends hide behind other waves' work (with a workgroup's, each piece
 * of one kept the CU for 12 us, and 48 sequences of 50 to 6000 positions took 40 instead of 32.5). More rows are bound by the
 * matrix cores: tiles in LDS that the workgroup shares (nmx_attnmx.h).
 *
 * Times of both kernels on MI355X, 8 heads on 2 of 256, and of the attention kernel in a trace: 4 sequences of 300 to 700 fp32
 * positions 13.7 us (9.6), 48 of 50 to 6000 binary16 31 (27; inputs out of the caches 37 in all; 118 MB, 23 as a copy), 64 of
 * 1500 binary16 42 (37) and fp32 78 (73; 393 MB, 76 as a copy), 64 with 30000 binary16 positions in common 60 (56; out of the caches
 * 69), 20 of up to 90 rows with 700 int8 ones in common 42 (32).
 *
 * Where the last two go, by clocks read in the kernel (medians of the workgroups of the matrix kind): 2.1 / 2.1 us until a workgroup
 * begins, 5.0 / 4.2 for the list, 5.6 / 6.4 until the first tile of a share lies in LDS, 18 / 4.7 tiles of 2.0 / 2.1, 1.9 / 1.8 to
 * store a part, 1.9 / 1.8 for the search of the next share; together 52.1 / 27.5. The last workgroup, whose share touches two units, ends
 * 4 us after them. Shares of few rows: 2.9 for the list; then 5.6 at least in fp32, 10.6 in binary16. */
#include <type_traits>

#include "nmx_internal.h"
#include "nmx_a8.h"
#include "nmx_attn.h"
#include "nmx_attnmx.h"
#include "nmx_batch.h"
#include "nmx_lanes.h"
#include "nmx_math.h"
#include "nmx_rms.h"
#include "nmx_rowpos.h"

namespace {

/* ---- norms, rotary positions, rows into pages ------------------------------------------------ */
struct PrepBatch {
    PageDev pg;
    int n, nh, rot;
    const int32_t *row0;
    float *q;
    const float *k_in, *v_in, *q_norm, *k_norm;
    float eps;
    const float *rcos, *rsin;
    int rope_rows, axes;
    const int32_t *rope_pos;
    void *kc, *vc;
    uint32_t axis[16]; /* two bits for each frequency */
};

/* A wave for each row and head (attn_prep_k's operations: its sum of squares runs in four chains, here of four lanes over the
 * wave's own LDS). Workgroups of a head and row, a thread a column, took 8.6 us for 460 rows of 8 + 2 heads, this 6.4; 8 rows 4.2
 * and 4.8. E: 64 columns each, at least hd / 64. */
constexpr int PREP_WAVES = 2;
template <int KVT, int E>
__device__ __forceinline__ void store_row(char *block, int nkv, int hd, int page, int R, int lane, const float (&x)[E]) {
    float inv = 0.0f, m = 0.0f;
    if constexpr (KVT == KV_I8) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (64 * e < hd) m = fmaxf(m, fabsf(x[e]));
        m = nmx_max_f32_wave(m);
        inv = m > 127.0f / 3.40282347e+38f ? 127.0f / m : 0.0f; /* stays finite */
        if (lane == 0) ((float *)(block + (size_t)nkv * page * hd))[R] = m / 127.0f;
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (64 * e >= hd) continue;
        const size_t at = (size_t)R * hd + 64 * e + lane;
        if constexpr (KVT == KV_F32) ((float *)block)[at] = x[e];
        else if constexpr (KVT == KV_F16) ((unsigned short *)block)[at] = (unsigned short)kv_half_bits(x[e]);
        else ((int8_t *)block)[at] = (int8_t)kv_i8_code(x[e], inv);
    }
}
template <int KVT, int E>
__global__ __launch_bounds__(64 * PREP_WAVES) void attn_batch_prep_k(const int32_t *row0, const int32_t *len, int seqs, int n,
                                                                     int heads, PrepBatch a) {
    __shared__ float row_s[PREP_WAVES][512], sum_s[PREP_WAVES][4];
    const int lane = lane_id(), wave = wave_id(), item = blockIdx.x * PREP_WAVES + wave, t = item / heads, u = item % heads;
    if (t >= n) return;
    const int hd = a.pg.hd, h2 = a.rot / 2, nkv = a.pg.nkv;
    const bool is_k = u < nkv;
    const float *in = is_k ? a.k_in + ((size_t)t * nkv + u) * hd : a.q + ((size_t)t * a.nh + (u - nkv)) * 2 * hd;
    const float *w = is_k ? a.k_norm : a.q_norm, *vi = a.v_in + ((size_t)t * nkv + (is_k ? u : 0)) * hd;
    float x[E], wt[E], val[E], cs[E], sn[E];
    int at[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (64 * e >= hd) continue; /* uniform */
        const int i = 64 * e + lane, f = i < h2 ? i : i - h2; /* the frequency of columns below rot */
        x[e] = in[i], wt[e] = w[i], val[e] = is_k ? vi[i] : 0.0f, at[e] = 0;
        if (i < 2 * h2 && a.rope_pos) at[e] = a.rope_pos[t * a.axes + (a.axis[f >> 4] >> 2 * (f & 15) & 3)];
    }
    const int s = seq_of_row(row0, seqs, t);
    if (s < 0) return; /* uniform over the wave */
    const SeqRows rows = seq_rows(row0, s, n);
    if (t >= rows.r0 + rows.count) return;
    const int p = row_position(seq_len(a.pg.len, s), rows.count, t - rows.r0); /* may be past the table */
    int id = -1;
    if (is_k && p >= 0 && p >> a.pg.shift < a.pg.max_pages) id = a.pg.table[(size_t)s * a.pg.max_pages + (p >> a.pg.shift)];
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (64 * e >= hd) continue;
        const int i = 64 * e + lane, f = i < h2 ? i : i - h2;
        cs[e] = sn[e] = 0.0f;
        if (i < 2 * h2) {
            int r = a.rope_pos ? at[e] : p;
            r = r < 0 ? 0 : r < a.rope_rows ? r : a.rope_rows - 1;
            cs[e] = a.rcos[(size_t)r * h2 + f], sn[e] = a.rsin[(size_t)r * h2 + f];
        }
    }
    float *buf = row_s[wave];
#pragma unroll
    for (int e = 0; e < E; e++)
        if (64 * e < hd) buf[64 * e + lane] = x[e] * x[e];
    nmx_lds_wave_sync();
    if (lane < 4) { /* ordered_sum4's chains */
        float c = 0.0f;
        for (int m0 = 0; m0 < hd / 4; m0 += 16) {
            float b[16];
#pragma unroll
            for (int k = 0; k < 16; k++) b[k] = buf[4 * (m0 + k) + lane];
#pragma unroll
            for (int k = 0; k < 16; k++) c = c + b[k];
        }
        sum_s[wave][lane] = c;
    }
    nmx_lds_wave_sync();
    const float *c4 = sum_s[wave];
    const float ss = ((c4[0] + c4[1]) + (c4[2] + c4[3])) + 0.0f;
    const float r = 1.0f / sqrtf(ss / (float)hd + a.eps);
#pragma unroll
    for (int e = 0; e < E; e++)
        if (64 * e < hd) buf[64 * e + lane] = x[e] = (x[e] * r) * wt[e];
    nmx_lds_wave_sync();
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (64 * e >= hd) continue;
        const int i = 64 * e + lane;
        if (i < h2) x[e] = buf[i] * cs[e] - buf[i + h2] * sn[e];
        else if (i < 2 * h2) x[e] = buf[i] * cs[e] + buf[i - h2] * sn[e];
    }
    if (!is_k) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (64 * e < hd) a.q[((size_t)t * a.nh + (u - nkv)) * 2 * hd + 64 * e + lane] = x[e];
    } else if ((uint32_t)id < (uint32_t)a.pg.npages) { /* uniform over the wave */
        const int page = 1 << a.pg.shift, R = (u << a.pg.shift) + (p & (page - 1));
        store_row<KVT, E>((char *)a.kc + id * a.pg.block, nkv, hd, page, R, lane, x);
        store_row<KVT, E>((char *)a.vc + id * a.pg.block, nkv, hd, page, R, lane, val);
    }
}

/* ---- the list of segments ---------------------------------------------------------------------- */
constexpr int AB_SEGS = 2 * NMX_BATCH_MAX; /* a prefix for each group, the rest of each sequence */
constexpr int AB_WGS = 256;                /* shares: a workgroup to a CU */
constexpr int AB_VR = 8;                   /* query rows that the vector kind takes: 4 a wave */
/* A step of 32 positions costs a workgroup this much: of the vector kind (4 query rows) what its bytes take at a CU's share of
 * the memory's rate, of the matrix kind 2.5 times as long (pieces of prompts among tokens 42.6 us, 64 questions about 30000
 * shared rows, binary16, 60.2; at 2 times 43.7 and 59.6, at 1.75 times 43.8 and 60.2; other heads and types take the same). A unit's beginning is round trips that its workgroup waits for, or
 * its wave beside others. Eight units of cost a step, so that a share of the smallest batches is one step.
 * A part's end (its store, and what the join reads of it) has no cost here. */
constexpr int AB_COST_V = 8, AB_COST_M = 20, AB_BEGIN_V = 8, AB_BEGIN_M = 80;

/* of a segment of m query rows */
__device__ __forceinline__ int step_cost(int m) { return m > AB_VR ? AB_COST_M : m > 4 ? 2 * AB_COST_V : AB_COST_V; }

struct Seg {
    unsigned long long c0; /* cost of all steps of its kind before this segment */
    uint32_t unit;         /* the cost of one unit: all its steps; 0: nothing to do */
    uint32_t u0;           /* units of its kind (vector, matrix) before it */
    int m;                 /* query rows: rows times heads of a KV group */
    int p0, p1;            /* positions */
    int r0, seq;           /* first row; the sequence whose table is read */
    int last;              /* what its rows see (positions_seen) */
    int group;             /* of a sequence: its group, -1 none */
};
/* Who takes what: of AB_WGS workgroups the first mx take the matrix kind's steps, the others the vector kind's.
 * A workgroup of those either lies within one unit, and its 8 waves take that part together, or its waves
 * take an eighth of its share each, by themselves. */
struct Shares {
    unsigned long long per_m, per_w; /* the cost of a workgroup's share, of a wave's */
    int mx;
};
/* What the join asks for: the shares, and for each row its sequence's segment and its group's prefix (r0 below 0: the row
 * belongs to nobody), at an address that the row's number gives. */
struct RowSeg {
    unsigned long long c0;
    uint32_t unit, u0;
    int m, r0;
};
struct Plan {
    Shares sh;
    RowSeg row[NMX_CHUNK_ROWS][2]; /* the prefix, the rest */
};
constexpr int AB_PARTS = 8; /* shares of a vector workgroup */

struct BatchAttn {
    PageDev pg;
    int n, nh, groups;
    const int32_t *row0, *group0, *shared;
    const float *q;
    const void *kc, *vc;
    float scale;
    Plan *plan;
    float *part_v, *part_m; /* parts of the vector kind [slot][vrows][hd], of the matrix kind [slot][tile][columns] */
    float4 *stat_v, *stat_m;
    int rep;          /* heads of a KV head */
    int jcols, vrows; /* vrows: AB_VR, or the query rows of a KV head if there are fewer */
    float *o;
    int8_t *aq;
    float *ad, *afs;
};

template <int HDP>
constexpr int tile_rows() { /* of the matrix kind */
    return 16 * ctx_waves<HDP>();
}
template <int HDP>
constexpr int halves() { /* of 512 columns, a unit makes 256 */
    return HDP > 256 ? 2 : 1;
}

/* What a kernel asks for first: arguments of their own, which are in registers when it begins. */
struct Head0 {
    const int32_t *row0, *len;
    int seqs, n, groups, room; /* room: positions of a table */
};

/* The list, by one wave: seg[0 .. groups + seqs) in LDS. Loops of 64 sequences, not
 * unrolled: most batches take one turn, and code that runs once is bound by its fetching. */
template <int HDP>
__device__ __forceinline__ Shares make_list(const Head0 &b, const BatchAttn &a, Seg *seg) {
    __shared__ int ctx_s[NMX_BATCH_MAX], first_s[NMX_BATCH_MAX], g0_s[NMX_BATCH_MAX + 1];
    const int lane = lane_id(), S = b.seqs, G = b.groups;
    bool falls = false;
#pragma unroll 1
    for (int s = lane; s < S; s += 64) {
        const SeqRows rows = seq_rows(b.row0, s, b.n);
        const int len = seq_len(b.len, s);
        Seg &x = seg[G + s];
        x.r0 = rows.r0, x.m = rows.count, x.p0 = 0, x.p1 = len < b.room ? len : b.room, x.seq = s, x.group = -1;
        x.last = rows.count < 0 ? 0 : row_position(len, rows.count, 0);
        falls |= rows.count < 0;
    }
#pragma unroll 1
    for (int g = lane; g < G; g += 64) {
        const int begin = a.group0[g], end = a.group0[g + 1];
        Seg &x = seg[g];
        x.m = 0, x.r0 = 0, x.p0 = 0, x.p1 = a.shared[g], x.seq = 0, x.last = ROWS_SEE_ALL, x.group = -1;
        ctx_s[g] = 0x7fffffff, first_s[g] = S, g0_s[g] = begin;
        if (g == G - 1) g0_s[G] = end;
        falls |= begin > end;
    }
    nmx_lds_wave_sync();
    if (__any(falls)) { /* a list that falls has no rows: the workspace holds the parts of lists that do not */
        for (int s = lane; s < S; s += 64) seg[G + s].m = 0;
        nmx_lds_wave_sync();
    }
    if (G) {
#pragma unroll 1
        for (int s = lane; s < S; s += 64) {
            int lo = -1, hi = G; /* the last group that begins at or before s: g0[lo] <= s < g0[hi] */
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (g0_s[mid] <= s) lo = mid;
                else hi = mid;
            }
            if (lo < 0 || s >= g0_s[lo + 1] || !seg[G + s].m) continue;
            seg[G + s].group = lo;
            atomicMin(&ctx_s[lo], seg[G + s].last), atomicMin(&first_s[lo], s);
        }
        nmx_lds_wave_sync();
#pragma unroll 1
        for (int g = lane; g < G; g += 64) {
            Seg &x = seg[g];
            const int first = first_s[g], ctx = ctx_s[g] < b.room ? ctx_s[g] : b.room, share = x.p1, end = g0_s[g + 1] < S ? g0_s[g + 1] : S;
            x.p1 = 0;
            if (first >= S) continue;
            x.seq = first, x.r0 = seg[G + first].r0, x.m = seg[G + end - 1].r0 + seg[G + end - 1].m - x.r0;
            x.p1 = share < 0 || ctx < 0 ? 0 : share < ctx ? share : ctx;
        }
        nmx_lds_wave_sync();
    }
    /* costs and units of its kind before each segment */
    unsigned long long cb[2] = {0, 0}, ub = 0; /* vector, matrix; units: vector in the lower half */
    const int rep = a.rep;
#pragma unroll 1
    for (int j0 = 0; j0 < G + S; j0 += 64) {
        const int j = j0 + lane;
        unsigned long long cost = 0, units = 0;
        bool mx = false;
        if (j < G + S) {
            Seg &x = seg[j];
            x.m *= rep;
            if (x.group >= 0) x.p0 = seg[x.group].p1;
            mx = x.m > AB_VR;
            const uint32_t steps = x.m > 0 && x.p1 > x.p0 ? (uint32_t)(x.p1 - x.p0 + AT_P - 1) / AT_P : 0;
            const uint32_t tiles = mx ? (uint32_t)(x.m + tile_rows<HDP>() - 1) / tile_rows<HDP>() * halves<HDP>() : 1;
            const uint32_t count = steps ? tiles * a.pg.nkv : 0;
            x.unit = count ? steps * step_cost(x.m) + (mx ? AB_BEGIN_M : AB_BEGIN_V) : 0;
            cost = (unsigned long long)count * x.unit, units = mx ? (unsigned long long)count << 32 : count;
        }
        const unsigned long long ui = nmx_scan_wave(units);
        unsigned long long mine = 0;
#pragma unroll 1
        for (int k = 0; k < 2; k++) {
            if (k && !__any(mx)) break;
            const unsigned long long own = mx == (k == 1) ? cost : 0, ci = nmx_scan_wave(own);
            if (mx == (k == 1)) mine = cb[k] + ci - own;
            cb[k] += __shfl(ci, 63);
        }
        if (j < G + S) seg[j].c0 = mine, seg[j].u0 = (uint32_t)(mx ? (ub + ui - units) >> 32 : ub + ui - units);
        ub += __shfl(ui, 63);
    }
    nmx_lds_wave_sync();
    /* workgroups in the proportion of the costs, one at least for each kind */
    Shares sh;
    const float part = (float)cb[1] / ((float)cb[0] + (float)cb[1] + 1.0f) * AB_WGS;
    sh.mx = !cb[1] ? 0 : !cb[0] ? AB_WGS : part < 1.0f ? 1 : part > AB_WGS - 1 ? AB_WGS - 1 : (int)part;
    const uint32_t waves = (uint32_t)(AB_WGS - sh.mx) * AB_PARTS;
    auto over = [](unsigned long long c, uint32_t n) { return n ? c >> 32 ? (c + n - 1) / n : ((uint32_t)c + (unsigned long long)n - 1) >> 32 ? (c + n - 1) / n : ((uint32_t)c + n - 1) / n : 0; };
    sh.per_m = over(cb[1], sh.mx), sh.per_w = over(cb[0], waves);
    return sh;
}

/* What a share does next: the part of a unit that begins at cost c, by one wave (x.unit 0: nothing more). */
struct Piece {
    Seg x;
    int tile, g, p0, p1;
    uint32_t unit; /* units of its kind before this one */
    unsigned long long next;
};
template <int HDP>
__device__ __forceinline__ void find_piece(const BatchAttn &a, int segs, const Seg *seg, bool matrix, unsigned long long c,
                                           unsigned long long end, Piece *piece) {
    const int lane = lane_id(), nkv = a.pg.nkv;
    if (lane == 0) piece->x.unit = 0;
    nmx_lds_wave_sync();
    if (c < end)
#pragma unroll 1
        for (int j = lane; j < segs; j += 64) {
            const unsigned long long c0 = seg[j].c0;
            const uint32_t unit = seg[j].unit;
            const bool mx = seg[j].m > AB_VR;
            if (!unit || mx != matrix || c < c0) continue;
            const int tiles = mx ? (seg[j].m + tile_rows<HDP>() - 1) / tile_rows<HDP>() * halves<HDP>() : 1;
            if (c - c0 >= (unsigned long long)unit * (uint32_t)(tiles * nkv)) continue;
            const unsigned long long off = c - c0; /* one lane comes here */
            const uint32_t u = off >> 32 ? (uint32_t)(off / unit) : (uint32_t)off / unit;
            const unsigned long long cu = c0 + (unsigned long long)u * unit, cn = cu + unit < end ? cu + unit : end;
            const int each = step_cost(seg[j].m), begin = mx ? AB_BEGIN_M : AB_BEGIN_V;
            auto steps = [&](unsigned long long cost) { /* of a unit, begun by the first part of its cost */
                return cost <= (uint32_t)begin ? 0 : ((int)(uint32_t)cost - begin + each - 1) / each;
            };
            const Seg x = seg[j];
            piece->x = x;
            piece->tile = u / nkv, piece->g = u % nkv;
            piece->p0 = x.p0 + steps(c - cu) * AT_P;
            const int p1 = x.p0 + steps(cn - cu) * AT_P;
            piece->p1 = p1 < x.p1 ? p1 : x.p1;
            piece->unit = x.u0 + u, piece->next = cn;
        }
    nmx_lds_wave_sync();
}

/* ---- the shares ---------------------------------------------------------------------------------- */
/* One KV head of a paged cache as a sequence sees it. */
template <int KVT>
struct PagedHead {
    const char *cache;
    const int32_t *table;
    uint32_t block; /* bytes, at most 2^29 and some scales */
    int npages, shift, mask, hd;
    uint32_t row, scales; /* the head's first row and first scale in a block, bytes */
    static constexpr int SIZE = KVT == KV_F32 ? 4 : KVT == KV_F16 ? 2 : 1;
    __device__ __forceinline__ PagedHead(const PageDev &pg, const void *cache, int seq, int g)
        : cache((const char *)cache), table(pg.table + (size_t)seq * pg.max_pages), block((uint32_t)pg.block), npages(pg.npages),
          shift(pg.shift), mask((1 << pg.shift) - 1), hd(pg.hd), row(((uint32_t)g << pg.shift) * pg.hd * SIZE),
          scales((((uint32_t)pg.nkv << pg.shift) * pg.hd) + ((uint32_t)g << pg.shift) * 4) {}
    /* An entry as it stands in the table. It is looked at when its rows are requested, a turn later: here that would wait for the
     * entry, and for everything that was requested before it (a tile of many rows 2.4 instead of 2.1 us). */
    __device__ __forceinline__ int page_of(int p) const { return table[p >> shift]; }
    __device__ __forceinline__ unsigned long long page(int id) const { /* no page of the cache: any page stands for it */
        return (unsigned long long)((uint32_t)id < (uint32_t)npages ? (uint32_t)id : 0) * block;
    }
    __device__ __forceinline__ unsigned long long where(int id, int p, int col) const {
        return page(id) + (row + (uint32_t)((p & mask) * hd + col) * SIZE);
    }
    __device__ __forceinline__ const char *at(int id, int p, int col) const { return cache + where(id, p, col); }
    __device__ __forceinline__ Raw8<KVT> load8(unsigned long long where) const {
        Raw8<KVT> r;
        const char *s = cache + where;
        if constexpr (KVT == KV_F32) r.a = *(const uint4 *)s, r.b = *(const uint4 *)(s + 16);
        else if constexpr (KVT == KV_F16) r.a = *(const uint4 *)s;
        else r.a = *(const uint2 *)s;
        return r;
    }
    __device__ __forceinline__ float scale(int id, int p) const {
        if constexpr (KVT == KV_I8) return *(const float *)(cache + page(id) + (scales + (uint32_t)(p & mask) * 4));
        return 1.0f;
    }
};

/* acc + sum over i of 8 values times x[i] */
__device__ __forceinline__ float widen(const Raw8<KV_F32> &r, int i) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    return __uint_as_float(w[i]);
}
__device__ __forceinline__ float widen(const Raw8<KV_F16> &r, int i) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
    return kv_half_value(w[i >> 1] >> 16 * (i & 1));
}
__device__ __forceinline__ float widen(const Raw8<KV_I8> &r, int i) {
    return (float)(int8_t)((i < 4 ? r.a.x : r.a.y) >> 8 * (i & 3));
}

/* the sum over W neighbouring lanes, in each of them */
template <int W>
__device__ __forceinline__ float sum_group(float v) {
    auto with = [&](int o) { v += __int_as_float(o); };
    if (W >= 2) with(nmx_dpp<NMX_DPP_XOR1>(__float_as_int(v)));
    if (W >= 4) with(nmx_dpp<NMX_DPP_XOR2>(__float_as_int(v)));
    if (W >= 8) with(nmx_dpp<NMX_DPP_HALF_MIRROR>(__float_as_int(v)));
    if (W >= 16) with(nmx_dpp<NMX_DPP_MIRROR>(__float_as_int(v)));
    if (W >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return v;
}
/* v of lane r of each four neighbours, in all four */
template <int R>
__device__ __forceinline__ float of_quad(float v) {
    return __int_as_float(nmx_dpp<0x55 * R>(__float_as_int(v)));
}
__device__ __forceinline__ float quad_row(float v, int r) { /* r constant where it is unrolled */
    return r == 0 ? of_quad<0>(v) : r == 1 ? of_quad<1>(v) : r == 2 ? of_quad<2>(v) : of_quad<3>(v);
}

/* What a wave finds of a unit of few rows: 4 query rows, the rq-th, of segment x's KV head g over the ws-th of NS
 * shares of the positions [p0, p1), which change hands every 4 positions; to part and stat, where `together` is set with the
 * workgroup's other waves.
 *
 * Values: a lane adds 16 columns (two chunks of 8) of its positions' rows by vector instructions, a row's weight comes
 * from a lane of its quad: lane (quarter gq, column c) has the weights of row c mod 4.
 * Scores of 16-bit keys on the matrix cores, 16 positions at a time and straight from memory: as first operand keys lie in
 * a lane as they lie in a row. The second operand has 16 columns for 4 query rows, so their high and low parts
 * stand in columns 4 apart and one product makes both. (By vector instructions a turn took 3.4 us of issue for 128
 * positions and CU, this 1.3.) fp32 keys are loaded as values are and take vector instructions too: they come at half
 * the positions a second, and the matrix cores' fp32 products, 16 columns for 4 rows, took 20.5 against 14.9 us over
 * 4 x 500 positions. */
template <int HDP, int KVT>
__device__ __forceinline__ void vector_piece(const BatchAttn &a, const Seg &x, int g, int p0, int p1, int rq, int ws, int NS,
                                             bool together, float *part, float4 *stat, uint4 *smem) {
    constexpr int WV = ctx_waves<HDP>(), LPP = HDP / 16;   /* lanes of a position's values */
    constexpr int NT = HDP < 256 ? 256 / HDP : 1;          /* tiles of 16 positions a turn */
    constexpr bool F32 = KVT == KV_F32;
    constexpr int VT = !F32 ? 4 : HDP > 256 ? 1 : 2;       /* positions of a quarter in a tile (fp32: no room for four) */
    constexpr int VP = HDP > 256 ? 2 * VT : VT;            /* positions whose values a lane adds in a turn */
    constexpr int KN = F32 ? 1 : HDP / 32;                 /* a key's chunks of 32 columns over the quarters */
    constexpr int NW = F32 ? VP : NT * VT;                 /* scores of a lane in a turn */
    const int lane = lane_id(), wave = wave_id(), l = lane % LPP, c = lane & 15, gq = lane >> 4, hd = a.pg.hd, rep = a.rep;
    const PagedHead<KVT> kh(a.pg, a.kc, x.seq, g), vh(a.pg, a.vc, x.seq, g);
    int col[2];
#pragma unroll
    for (int j = 0; j < 2; j++) col[j] = (l + LPP * j) * 8, col[j] = col[j] < hd ? col[j] : 0;
    /* the positions of a turn: position v of quarter q in tile n is 4 NS (VT n + v) + 4 ws + q, so that few positions
     * spread over all waves; behind the end the last one stands in and has no weight */
    const int turn = 4 * VT * NT * NS;
    auto at = [&](int base, int n, int q, int v) { return base + 4 * NS * (VT * n + v) + 4 * ws + q; };
    auto in = [&](int p) { return p < p1 ? p : p1 - 1; };
    /* a lane's values: those of its quarter in the tile that its LPP lanes have (HDP 512: of two quarters) */
    const int vt = lane / LPP % (LPP < 16 ? 16 / LPP : 1);
    auto at_v = [&](int base, int v) { return HDP > 256 ? at(base, 0, (gq & 2) + v / VT, v % VT) : at(base, vt, gq, v); };
    int pk[NT], pv[VP];
    auto ask = [&](int base) {
#pragma unroll
        for (int n = 0; n < NT && !F32; n++) pk[n] = kh.page_of(in(at(base, n, c >> 2, c & 3)));
#pragma unroll
        for (int v = 0; v < VP; v++) pv[v] = vh.page_of(in(at_v(base, v)));
    };
    typedef typename std::conditional<KVT == KV_I8, uint2, uint4>::type KeyChunk;
    KeyChunk rk[NT][KN];
    Raw8<KVT> rf[F32 ? VP : 1][2], rv[VP][2]; /* rf: fp32 keys */
    float sk[NT], sv[NT]; /* int8: scales of position c of a tile (four of them are those of the lane's scores) */
    auto fetch_k = [&](int base) {
        if constexpr (F32) {
#pragma unroll
            for (int v = 0; v < VP; v++)
#pragma unroll
                for (int j = 0; j < 2; j++) rf[v][j] = kh.load8(kh.where(pv[v], in(at_v(base, v)), col[j]));
        } else {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int p = in(at(base, n, c >> 2, c & 3));
                const char *row = kh.at(pk[n], p, 8 * gq);
#pragma unroll
                for (int k = 0; k < KN; k++)
                    if (32 * k < HDP / 2 + 64 || 32 * k < hd) rk[n][k] = *(const KeyChunk *)(row + 32 * k * PagedHead<KVT>::SIZE);
                    else rk[n][k] = KeyChunk{}; /* columns behind hd */
                if (KVT == KV_I8) sk[n] = kh.scale(pk[n], p), sv[n] = vh.scale(pk[n], p);
            }
        }
    };
    auto fetch_v = [&](int base) {
#pragma unroll
        for (int v = 0; v < VP; v++)
#pragma unroll
            for (int j = 0; j < 2; j++) rv[v][j] = vh.load8(vh.where(pv[v], in(at_v(base, v)), col[j]));
    };
    ask(p0);
    /* the query rows: row c mod 4 of this wave's; rows past the last one are of no use to anyone */
    const int rr = rq * 4 + (c & 3), ri = rr < x.m ? rr : 0;
    const float *qp = a.q + ((size_t)(x.r0 + ri / rep) * a.nh + g * rep + ri % rep) * 2 * hd;
    half8 qx[KN];
    float qf = a.scale * AT_LOG2E;
    float *qs = (float *)smem + wave * 4 * HDP; /* fp32: this wave's rows in LDS, they have no registers to stay in */
    if constexpr (F32) {
        constexpr int QU = HDP / 64;
        float4 qv[QU];
#pragma unroll
        for (int u = 0; u < QU; u++) { /* lane: row c mod 4, 16-byte pieces lane / 4 + 16 u of it */
            const int q4 = (lane / 4 + 16 * u) * 4;
            qv[u] = *(const float4 *)(qp + (q4 < hd ? q4 : 0));
            if (q4 >= hd) qv[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        fetch_k(p0);
        fetch_v(p0);
        nmx_lds_wave_sync();
#pragma unroll
        for (int u = 0; u < QU; u++) { /* [row][chunk][half][lane][4], as the lanes of a position read them */
            const int piece = lane / 4 + 16 * u, chunk = piece / 2 / LPP;
            *(float4 *)(qs + (c & 3) * HDP + ((chunk * 2 + piece % 2) * LPP + piece / 2 % LPP) * 4) = qv[u];
        }
        nmx_lds_wave_sync();
    } else {
        QueryRow<KN> qr(qp, true, hd, gq);
        fetch_k(p0);
        fetch_v(p0);
        half8 ql[KN];
        qf = qr.split(a.scale, qx, ql);
#pragma unroll
        for (int k = 0; k < KN; k++) qx[k] = c & 4 ? ql[k] : qx[k];
    }
    const int lim = rr >= x.m ? 0 : positions_seen(x.last, ri / rep, p1);
    ask(p0 + turn);
    float acc[4][16], m = -INFINITY, sum = 0.0f, lost = 0.0f; /* m is the wave's, sum this lane's */
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[r][i] = 0.0f;
    int q_at = 4 * l;
    for (int base = p0; base < p1; base += turn) {
        /* scores of row c mod 4 at this lane's positions: its quarter's in each tile, or (fp32) those of its values */
        float w[NW], fv[NW];
        if constexpr (F32) {
            asm volatile("" : "+v"(q_at)); /* the query rows are read anew each turn: they have no registers to stay in */
            float s[VP][4];
#pragma unroll
            for (int v = 0; v < VP; v++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[v][r] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float4 q[4];
#pragma unroll
                for (int r = 0; r < 4; r++) q[r] = *(const float4 *)(qs + q_at + r * HDP + e * 4 * LPP);
#pragma unroll
                for (int v = 0; v < VP; v++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float k = widen(rf[v][e >> 1], 4 * (e & 1) + i);
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            s[v][r] = __builtin_fmaf(k, i == 0 ? q[r].x : i == 1 ? q[r].y : i == 2 ? q[r].z : q[r].w, s[v][r]);
                    }
            }
#pragma unroll
            for (int v = 0; v < VP; v++) {
                const float r0 = sum_group<LPP>(s[v][0]), r1 = sum_group<LPP>(s[v][1]);
                const float r2 = sum_group<LPP>(s[v][2]), r3 = sum_group<LPP>(s[v][3]);
                const float low = c & 1 ? r1 : r0, high = c & 1 ? r3 : r2;
                w[v] = c & 2 ? high : low;
            }
        } else {
            float4v s4[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) s4[n] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KN; k++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    half8 y;
                    if constexpr (KVT == KV_F16) y = __builtin_bit_cast(half8, rk[n][k]);
                    else y = codes8(rk[n][k]);
                    s4[n] = mfma16(y, qx[k], s4[n]);
                }
#pragma unroll
            for (int i = 0; i < NW; i++) {
                float s = s4[i / VT][i % VT];
                s += __int_as_float(nmx_dpp<0x124>(__float_as_int(s))); /* high and low: 4 columns on */
                if (KVT == KV_I8) { /* the scales are with lane c = 4 quarter + v of a quarter */
                    const int from = (lane & 48) + 4 * gq + i % VT;
                    s *= __shfl(sk[i / VT], from), fv[i] = __shfl(sv[i / VT], from);
                }
                w[i] = s;
            }
        }
        fetch_k(base + turn); /* behind the last turn the last position again */
        float top = m;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const int p = F32 ? at_v(base, i) : at(base, i / VT, gq, i % VT);
            w[i] = p < lim ? w[i] * qf : -INFINITY;
            top = fmaxf(top, w[i]);
        }
        if (F32 && LPP <= 4) top = fmaxf(top, __int_as_float(nmx_dpp<0x124>(__float_as_int(top))));
        if (F32 && LPP <= 8) top = fmaxf(top, __int_as_float(nmx_dpp<0x128>(__float_as_int(top))));
        top = max_quarters(top);
        if (__any(top > m)) {
            const float down = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
            m = top, sum *= down, lost *= down;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float d = quad_row(down, r);
#pragma unroll
                for (int i = 0; i < 16; i++) acc[r][i] *= d;
            }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float all = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            w[i] = __builtin_amdgcn_exp2f(w[i] - ref);
            all += w[i];
            if (KVT == KV_I8) w[i] *= fv[i];
        }
        const float gain = all - lost, now = sum + gain; /* the roundings of a long share's sum are kept */
        lost = (now - sum) - gain, sum = now;
        /* the weights of the positions whose values this lane adds */
        float u[VP];
#pragma unroll
        for (int v = 0; v < VT; v++) {
            if constexpr (F32) {
                u[v] = w[v];
                if (HDP > 256) u[v + VT] = w[(v + VT) % NW];
            } else if constexpr (HDP > 256) { /* of both quarters of its half */
                const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(w[v]), __float_as_uint(w[v]), false, false);
                u[v] = __uint_as_float(y[0]), u[v + VT] = __uint_as_float(y[1]);
            } else {
                u[v] = w[v];
#pragma unroll
                for (int n = 1; n < NT; n++) u[v] = vt == n ? w[VT * n + v] : u[v];
            }
        }
#pragma unroll
        for (int v = 0; v < VP; v++) {
            float wr[4];
#pragma unroll
            for (int r = 0; r < 4; r++) wr[r] = quad_row(u[v], r);
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = widen(rv[v][j], i);
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[r][8 * j + i] = __builtin_fmaf(y, wr[r], acc[r][8 * j + i]);
                }
        }
        fetch_v(base + turn);
        ask(base + 2 * turn);
    }
    /* a lane's sums over the wave's quarters */
    float total = sum - lost;
    if (F32 && LPP <= 4) total += __int_as_float(nmx_dpp<0x124>(__float_as_int(total)));
    if (F32 && LPP <= 8) total += __int_as_float(nmx_dpp<0x128>(__float_as_int(total)));
    if (F32 && LPP > 16) { /* the quarters of a half have the same positions */
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(total), __float_as_uint(total), false, false);
        total = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    } else {
        total = nmx_sum_quarters(total);
    }
    if (LPP < 16) { /* within a quarter first: rows of 16 lanes turned by 4 and by 8 */
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (LPP <= 4) acc[r][i] += __int_as_float(nmx_dpp<0x124>(__float_as_int(acc[r][i])));
                acc[r][i] += __int_as_float(nmx_dpp<0x128>(__float_as_int(acc[r][i])));
            }
    }
    /* halves of the wave, then (rows of HDP / 16 <= 16 lanes) its quarters exchange two rows and add: a lane
     * keeps its columns of row 2 (its half), or of that and of its quarter */
    float keep[2][16];
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[r][i]), __float_as_uint(acc[r + 2][i]), false, false);
            keep[r][i] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
        }
    if constexpr (LPP <= 16) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(keep[0][i]), __float_as_uint(keep[1][i]), false, false);
            keep[0][i] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
        }
    }
    float *vals = (float *)smem;                  /* together: [WV][4][HDP] */
    float2 *ml = (float2 *)(vals + WV * 4 * HDP); /* [WV][4]: maximum, sum */
    if (together && lane < 4) ml[wave * 4 + lane] = make_float2(m, total);
    if (!together && lane < 4 && rq * 4 + lane < x.m) stat[rq * 4 + lane] = make_float4(m, 12.0f, total, 0.0f); /* as 2^12 high values */
    if (LPP >= 16 || lane % 16 < LPP) {
#pragma unroll
        for (int k = 0; k < (LPP <= 16 ? 1 : 2); k++) {
            const int r = LPP <= 16 ? 2 * (lane >> 5) + (lane >> 4 & 1) : 2 * (lane >> 5) + k;
            if (!together && rq * 4 + r >= x.m) continue;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int c8 = (l + LPP * j) * 8;
                if (!together && c8 >= hd) continue;
                float *y = together ? vals + (wave * 4 + r) * HDP + c8 : part + (size_t)(rq * 4 + r) * hd + c8;
                *(float4 *)y = make_float4(keep[k][8 * j], keep[k][8 * j + 1], keep[k][8 * j + 2], keep[k][8 * j + 3]);
                *(float4 *)(y + 4) = make_float4(keep[k][8 * j + 4], keep[k][8 * j + 5], keep[k][8 * j + 6], keep[k][8 * j + 7]);
            }
        }
    }
    if (!together) return;
    __syncthreads();
    const int c4 = hd / 4, quads = WV / NS;
    for (int e = 64 * wave + lane; e < x.m * c4; e += 64 * WV) {
        const int rr = e / c4, cc = e % c4 * 4, r = rr & 3, first = rr >> 2;
        float top = -INFINITY;
        for (int w = first; w < WV; w += quads) top = fmaxf(top, ml[w * 4 + r].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float all = 0.0f;
        for (int w = first; w < WV; w += quads) {
            const float2 y = ml[w * 4 + r];
            const float f = __builtin_amdgcn_exp2f(y.x - ref);
            const float4 z = *(const float4 *)(vals + (w * 4 + r) * HDP + cc);
            all = __builtin_fmaf(y.y, f, all);
            v.x = __builtin_fmaf(z.x, f, v.x), v.y = __builtin_fmaf(z.y, f, v.y);
            v.z = __builtin_fmaf(z.z, f, v.z), v.w = __builtin_fmaf(z.w, f, v.w);
        }
        *(float4 *)(part + (size_t)rr * hd + cc) = v;
        if (cc == 0) stat[rr] = make_float4(top, 12.0f, all, 0.0f);
    }
}

/* What a share finds of a unit of many rows, one tile of them. */
template <int HDP, int KVT>
__device__ __forceinline__ void matrix_piece(const BatchAttn &a, const Seg &x, int g, int tile, int half, int p0, int p1,
                                             float *part, float4 *stat, uint4 *smem) {
    constexpr int OD = HDP > 256 ? 256 : HDP, KS = HDP / 32;
    const int lane = lane_id(), wave = wave_id(), c = lane & 15, gq = lane >> 4, hd = a.pg.hd, rep = a.rep;
    const int row0 = tile * tile_rows<HDP>() + wave * 16, rr = row0 + c, d0 = half * OD;
    const bool live = rr < x.m;
    const int i = (live ? rr : 0) / rep, h = g * rep + (live ? rr : 0) % rep;
    QueryRow<KS> qr(a.q + ((size_t)(x.r0 + i) * a.nh + h) * 2 * hd, live, hd, gq);
    const PagedHead<KVT> kh(a.pg, a.kc, x.seq, g), vh(a.pg, a.vc, x.seq, g);
    const int lim = positions_seen(x.last, i, p1);
    Running<OD / 16> r;
    attend_tiles<HDP, KVT>(r, qr, a.scale, kh, vh, p0, p1, lim, d0, row0 < x.m, smem);
    r.l -= r.lc;
    r.l = nmx_sum_quarters(r.l);
    if (!live) return;
    const int at = wave * 16 + c;
#pragma unroll
    for (int d = 0; d < OD / 16; d++)
        if (d0 + 16 * d < hd) *(float4v *)(part + (size_t)at * OD + 16 * d + 4 * gq) = r.o[d];
    if (gq == 0) stat[at] = make_float4(r.m, (float)r.ve, r.l, 0.0f);
}

template <int HDP, int KVT>
__global__ __launch_bounds__(64 * ctx_waves<HDP>()) void attn_batch_k(const int32_t *row0, const int32_t *len, int seqs, int n,
                                                                     int groups, int room, BatchAttn a) {
    constexpr int OD = HDP > 256 ? 256 : HDP;
    extern __shared__ uint4 smem[];
    constexpr int WV = ctx_waves<HDP>();
    __shared__ Seg seg[AB_SEGS];
    __shared__ Piece piece_s[WV];
    __shared__ Shares sh_s;
    const int tid = threadIdx.x, segs = groups + seqs, w = blockIdx.x, wave = wave_id();
    if (wave == 0) {
        const Shares sh = make_list<HDP>({row0, len, seqs, n, groups, room}, a, seg);
        const bool mx = w < sh.mx;
        const unsigned long long per = mx ? sh.per_m : sh.per_w * AB_PARTS, c = (unsigned long long)(mx ? w : w - sh.mx) * per;
        find_piece<HDP>(a, segs, seg, mx, c, c + per, piece_s);
        if (tid == 0) sh_s = sh;
        if (w == 0 && tid == 0) a.plan->sh = sh;
    }
    __syncthreads();
    if (wave == WV - 1) /* the join's rows, each by one workgroup */
#pragma unroll 1
        for (int t = w; t < n; t += AB_WGS) {
            auto put = [&](int k, const Seg &x, uint32_t unit) { a.plan->row[t][k] = RowSeg{x.c0, unit, x.u0, x.m, x.r0}; };
            bool found = false;
#pragma unroll 1
            for (int s = tid % 64; s < seqs; s += 64) {
                const Seg &x = seg[groups + s];
                if (t < x.r0 || (t - x.r0) * a.rep >= x.m) continue; /* a row has one sequence */
                found = true;
                put(1, x, x.unit);
                const Seg &y = seg[x.group < 0 ? groups + s : x.group];
                put(0, y, x.group < 0 ? 0 : y.unit);
            }
            if (!__any(found) && tid % 64 == 0) a.plan->row[t][1].r0 = -1;
        }
    /* between pieces everything is in LDS: a piece has no registers to spare */
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    int p0, p1, g, tile;
    size_t unit;
    Seg x{};
    auto take = [&](const Piece &p) {
        x.m = same(p.x.m), x.r0 = same(p.x.r0), x.seq = same(p.x.seq), x.last = same(p.x.last);
        p0 = same(p.p0), p1 = same(p.p1), g = same(p.g), tile = same(p.tile), unit = (uint32_t)same(p.unit);
        return same(p.x.unit) != 0;
    };
    const int mxs = same(sh_s.mx);
    if (w < mxs) {
        while (take(piece_s[0])) {
            const size_t slot = w + unit;
            float4 *stat = a.stat_m + slot * tile_rows<HDP>();
            if (p0 < p1) matrix_piece<HDP, KVT>(a, x, g, tile / halves<HDP>(), tile % halves<HDP>(), p0, p1,
                                                a.part_m + slot * tile_rows<HDP>() * OD, stat, smem);
            else if (tid < tile_rows<HDP>()) stat[tid] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
            __syncthreads();
            if (wave == 0) find_piece<HDP>(a, segs, seg, true, piece_s[0].next, (w + 1) * sh_s.per_m, piece_s);
            __syncthreads();
        }
        return;
    }
    if (!take(piece_s[0])) return;
    /* together in one unit (4 waves: as if they were 8), or each share by a wave alone */
    const bool together = same(piece_s[0].next == (unsigned long long)(w - mxs + 1) * AB_PARTS * sh_s.per_w);
    const int quads = x.m > 4 ? 2 : 1;
    if (together) {
        const size_t slot = (size_t)(w - mxs) * AB_PARTS + unit;
        float4 *stat = a.stat_v + slot * a.vrows;
        if (p0 < p1) vector_piece<HDP, KVT>(a, x, g, p0, p1, wave % quads, wave / quads, WV / quads, true,
                                            a.part_v + slot * a.vrows * a.pg.hd, stat, smem);
        else if (tid < a.vrows) stat[tid] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        return;
    }
    __syncthreads(); /* everyone has read the first piece */
    /* the waves that a row's heads take (4 each) go over the same positions at the same time */
    const int heads = a.rep, team = heads > 4 ? 2 : 1;
#pragma unroll 1
    for (int share = (w - mxs) * AB_PARTS + wave / team; share < (w - mxs + 1) * AB_PARTS; share += WV / team) {
        if (tid % 64 == 0) piece_s[wave].next = share * sh_s.per_w;
        nmx_lds_wave_sync();
#pragma unroll 1
        for (;;) {
            find_piece<HDP>(a, segs, seg, false, piece_s[wave].next, (share + 1) * sh_s.per_w, piece_s + wave);
            if (!take(piece_s[wave])) break;
            const size_t slot = share + unit;
            float4 *stat = a.stat_v + slot * a.vrows;
            if (p0 >= p1 && tid % 64 < a.vrows) stat[tid % 64] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (int k = wave % team; 4 * k < x.m && p0 < p1; k += team) {
                /* nothing of a pass is kept for the next one */
                asm volatile("" : "+s"(p0), "+s"(p1), "+s"(g), "+s"(x.seq), "+s"(x.r0), "+s"(x.m), "+s"(x.last));
                vector_piece<HDP, KVT>(a, x, g, p0, p1, k, 0, 1, false, a.part_v + slot * a.vrows * a.pg.hd, stat, smem);
            }
        }
    }
}

/* ---- the join -------------------------------------------------------------------------------------- */
constexpr int JB = 256;              /* threads */
/* rows, heads and halves from which a wave takes one alone (423 rows of 8 heads: 47.1 us against 52.6, 64 rows: 74.0 against
 * 71.5; nothing between 512 and 3384 items is measured) */
constexpr int JB_WAVES = 1024;
constexpr int JB_PARTS = 2 * (AB_WGS + 2 * AB_PARTS);

/* The parts of a row's head and half: those of the prefix, then the sequence's own. Of a unit of few rows: those of single
 * waves, of workgroups whose share lies in it, of single waves. */
template <int HDP>
struct Parts {
    int count[2], solo[2], whole[2];
    const float *val[2]; /* of the half's first column */
    const float4 *st[2];
    uint32_t vstep[2], sstep[2];
    bool any; /* the row belongs to a sequence */
    __device__ __forceinline__ Parts(const BatchAttn &a, int t, int h, int half) {
        constexpr int OD = HDP > 256 ? 256 : HDP;
        const int hd = a.pg.hd, nkv = a.pg.nkv, rep = a.rep, g = h / rep;
        const Shares sh = a.plan->sh;
        const RowSeg pre = a.plan->row[t][0], own = a.plan->row[t][1];
        any = own.r0 >= 0;
        if (!any) return; /* uniform over the wave */
        auto over = [](unsigned long long c, unsigned long long n) {
            return c >> 32 || n >> 32 ? (uint32_t)(c / n) : (uint32_t)c / (uint32_t)n;
        };
#pragma unroll 1
        for (int k = 0; k < 2; k++) {
            const RowSeg &x = k ? own : pre;
            const int rr = (t - x.r0) * rep + h % rep;
            int n = 0, so = 0, wh = 0;
            const float *v = nullptr;
            const float4 *f = nullptr;
            uint32_t vs = 0, ss = 0;
            if (x.unit && rr >= 0 && rr < x.m) {
                const bool mx = x.m > AB_VR;
                constexpr int TR = tile_rows<HDP>(); /* few rows: one tile */
                const int tr = mx ? TR : a.vrows, tile = mx ? rr / TR : 0, in = mx ? rr % TR : rr, width = mx ? OD : hd;
                const uint32_t u = (mx ? tile * halves<HDP>() + half : 0) * nkv + g;
                const unsigned long long cu = x.c0 + (unsigned long long)u * x.unit, per = mx ? sh.per_m : sh.per_w;
                const uint32_t w0 = over(cu, per), w1 = over(cu + x.unit - 1, per);
                n = so = (int)(w1 - w0) + 1;
                if (!mx) {
                    const uint32_t f0 = (w0 * per == cu ? w0 + AB_PARTS - 1 : w0 + AB_PARTS) / AB_PARTS, f1 = (w1 + (cu + x.unit == (w1 + 1) * per)) / AB_PARTS;
                    if (f1 > f0) so = (int)(f0 * AB_PARTS - w0), wh = (int)(f1 - f0), n -= wh * (AB_PARTS - 1);
                }
                const size_t slot = (size_t)w0 + x.u0 + u;
                v = (mx ? a.part_m : a.part_v) + (slot * tr + in) * width + (mx ? 0 : half * OD);
                f = (mx ? a.stat_m : a.stat_v) + slot * tr + in;
                vs = tr * width, ss = tr;
            }
            if (k) count[1] = n, solo[1] = so, whole[1] = wh, val[1] = v, st[1] = f, vstep[1] = vs, sstep[1] = ss;
            else count[0] = n, solo[0] = so, whole[0] = wh, val[0] = v, st[0] = f, vstep[0] = vs, sstep[0] = ss;
        }
    }
    __device__ __forceinline__ int all() const { return count[0] + count[1]; }
    /* slots from the first one to part i */
    __device__ __forceinline__ int step(int i) const {
        const bool b = i >= count[0];
        const int nth = b ? i - count[0] : i, inner = nth - (b ? solo[1] : solo[0]), w = b ? whole[1] : whole[0];
        return inner <= 0 ? nth : nth + (inner < w ? inner : w) * (AB_PARTS - 1);
    }
    __device__ __forceinline__ const float *values(int i) const {
        return i >= count[0] ? val[1] + (size_t)step(i) * vstep[1] : val[0] + (size_t)step(i) * vstep[0];
    }
    __device__ __forceinline__ float4 stat(int i) const { return i >= count[0] ? st[1][step(i) * sstep[1]] : st[0][step(i) * sstep[0]]; }
};

/* A wave for each row, head and half, where there are many of them: its parts' numbers stay in its lanes. */
template <int HDP>
__global__ __launch_bounds__(JB) void attn_batch_join_waves_k(BatchAttn a) {
    constexpr int OD = HDP > 256 ? 256 : HDP, HV = halves<HDP>(), PT = (JB_PARTS + 63) / 64;
    const int lane = lane_id(), item = __builtin_amdgcn_readfirstlane((int)blockIdx.x * (JB / 64) + wave_id());
    if (item >= a.n * a.nh * HV) return;
    const int hd = a.pg.hd, half = item % HV, h = item / HV % a.nh, t = item / HV / a.nh;
    const int col = half * OD + 4 * lane, cols = hd - half * OD < OD ? hd - half * OD : OD;
    const bool in = 4 * lane < cols;
    const float *qp = a.q + ((size_t)t * a.nh + h) * 2 * hd + hd;
    const float4 gate = *(const float4 *)(qp + (in ? col : 0));
    const Parts<HDP> p(a, t, h, half);
    if (!p.any) return; /* a row of no sequence is left as it is */
    const int parts = p.all();
    float top = -INFINITY, w[PT], sum[PT];
    int ex[PT];
#pragma unroll
    for (int k = 0; k < PT; k++) {
        w[k] = -INFINITY, sum[k] = 0.0f, ex[k] = 0;
        if (64 * k >= parts) continue;
        const int i = 64 * k + lane;
        if (i < parts) {
            const float4 y = p.stat(i);
            w[k] = y.x, sum[k] = y.z, ex[k] = (int)y.y;
        }
        top = fmaxf(top, w[k]);
    }
    top = nmx_max_f32_wave(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float all = 0.0f;
#pragma unroll
    for (int k = 0; k < PT; k++) {
        if (64 * k >= parts) continue;
        const float f = __builtin_amdgcn_exp2f(w[k] - ref);
        all += sum[k] * f;
        w[k] = w[k] == -INFINITY ? 0.0f : ldexpf(f, ex[k] - 12);
    }
    all = sum_lanes(all);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int PB = 8;
#pragma unroll
    for (int k = 0; k < PT; k++) {
        for (int i0 = 64 * k; i0 < parts && i0 < 64 * k + 64; i0 += PB) {
            float4 v[PB];
            float f[PB];
#pragma unroll
            for (int b = 0; b < PB; b++) {
                const int i = i0 + b < parts ? i0 + b : i0;
                f[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w[k]), i - 64 * k));
                if (i0 + b >= parts) f[b] = 0.0f;
                v[b] = *(const float4 *)(p.values(i) + (in ? 4 * lane : 0));
            }
#pragma unroll
            for (int b = 0; b < PB; b++)
                if (f[b] != 0.0f) { /* a part without a visible position was never written */
                    acc.x = __builtin_fmaf(f[b], v[b].x, acc.x), acc.y = __builtin_fmaf(f[b], v[b].y, acc.y);
                    acc.z = __builtin_fmaf(f[b], v[b].z, acc.z), acc.w = __builtin_fmaf(f[b], v[b].w, acc.w);
                }
        }
    }
    const bool some = all > 0.0f || !(all == all); /* nothing in sight: 0 */
    const float x[4] = {some ? acc.x / all : 0.0f, some ? acc.y / all : 0.0f, some ? acc.z / all : 0.0f, some ? acc.w / all : 0.0f};
    const float gx[4] = {gate.x, gate.y, gate.z, gate.w};
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = x[i] * nmx_sigmoid(gx[i]);
    const int at = h * hd + col;
    if (in) *(float4 *)(a.o + (size_t)t * a.nh * hd + at) = make_float4(o[0], o[1], o[2], o[3]);
    if (a.aq) { /* blocks of 32 columns: 8 lanes of 4 */
        float m = fmaxf(fmaxf(fabsf(o[0]), fabsf(o[1])), fmaxf(fabsf(o[2]), fabsf(o[3])));
        m = max_lanes<8>(m);
        const float id = m > 0.0f ? 127.0f / m : 0.0f;
        int c[4], n = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[i] = (int)rintf(o[i] * id), n += c[i];
            c[i] = c[i] > 127 ? 127 : c[i] < -128 ? -128 : c[i];
        }
        n += nmx_dpp<NMX_DPP_XOR1>(n);
        n += nmx_dpp<NMX_DPP_XOR2>(n);
        n += nmx_dpp<NMX_DPP_HALF_MIRROR>(n);
        if (in) {
            const size_t u = (size_t)(at >> 5) * a.n + t;
            *(uint32_t *)(a.aq + u * 32 + (at & 31)) = (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 | (uint32_t)c[3] << 24;
            if (lane % 8 == 0) {
                const float d = m / 127.0f;
                a.ad[u] = d, a.afs[u] = d * (float)n;
            }
        }
    }
}

/* Workgroup: a row and head, blockIdx.y a group of a.jcols columns of it (of one half). */
template <int HDP>
__global__ __launch_bounds__(JB) void attn_batch_join_k(BatchAttn a) {
    constexpr int OD = HDP > 256 ? 256 : HDP;
    __shared__ float red[2][JB / 64], acc_s[JB * 4], w_s[JB_PARTS];
    __shared__ const float *at_s[JB_PARTS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t = blockIdx.x / a.nh, h = blockIdx.x % a.nh;
    const int hd = a.pg.hd, c0 = blockIdx.y * a.jcols, half = c0 / OD;
    const float gate = a.q[((size_t)t * a.nh + h) * 2 * hd + hd + c0 + (tid < a.jcols ? tid : 0)];
    const Parts<HDP> p(a, t, h, half);
    if (!p.any) return; /* a row of no sequence is left as it is; uniform over the workgroup */
    const int parts = p.all();
    constexpr int PT = (JB_PARTS + JB - 1) / JB;
    float4 y[PT];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < PT; k++) {
        const int i = tid + JB * k;
        y[k] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        if (i < parts) y[k] = p.stat(i), at_s[i] = p.values(i) + c0 - half * OD;
        top = fmaxf(top, y[k].x);
    }
    top = nmx_max_f32_wave(top);
    if (lane == 0) red[0][wave] = top;
    nmx_lds_sync();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float ref = top == -INFINITY ? 0.0f : top;
    float all = 0.0f;
#pragma unroll
    for (int k = 0; k < PT; k++) {
        const int i = tid + JB * k;
        if (i >= parts) continue;
        const float f = __builtin_amdgcn_exp2f(y[k].x - ref);
        all += y[k].z * f;
        w_s[i] = y[k].x == -INFINITY ? 0.0f : ldexpf(f, (int)y[k].y - 12);
    }
    all = sum_lanes(all);
    if (lane == 0) red[1][wave] = all;
    nmx_lds_sync();
    all = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    /* slots of jcols / 4 threads: a thread takes 4 columns of every slots-th part */
    const int per_slot = a.jcols >> 2, slots = JB / per_slot, slot = tid / per_slot, col = tid % per_slot * 4;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (slot < slots) {
        constexpr int PB = 8;
        for (int i0 = slot; i0 < parts; i0 += PB * slots) {
            float4 v[PB];
            float f[PB];
#pragma unroll
            for (int k = 0; k < PB; k++) {
                const int i = i0 + k * slots, j = i < parts ? i : i0;
                f[k] = i < parts ? w_s[j] : 0.0f;
                v[k] = *(const float4 *)(at_s[j] + col);
            }
#pragma unroll
            for (int k = 0; k < PB; k++)
                if (f[k] != 0.0f) { /* a part without a visible position was never written */
                    acc.x = __builtin_fmaf(f[k], v[k].x, acc.x), acc.y = __builtin_fmaf(f[k], v[k].y, acc.y);
                    acc.z = __builtin_fmaf(f[k], v[k].z, acc.z), acc.w = __builtin_fmaf(f[k], v[k].w, acc.w);
                }
        }
        *(float4 *)(acc_s + slot * a.jcols + col) = acc;
    }
    nmx_lds_sync();
    if (tid < a.jcols) {
        float v = 0.0f;
        for (int k = 0; k < slots; k++) v += acc_s[k * a.jcols + tid];
        v = all > 0.0f || !(all == all) ? v / all : 0.0f; /* nothing in sight: 0 */
        v = v * nmx_sigmoid(gate);
        const int at = h * hd + c0 + tid;
        a.o[(size_t)t * a.nh * hd + at] = v;
        if (a.aq) a8_block(v, at >> 5, t, a.n, a.aq, a.ad, a.afs); /* jcols % 64 == 0: whole blocks */
    }
}

/* ---- the workspace ----------------------------------------------------------------------------------- */
struct Room {
    int hdp, jcols, vrows;
    size_t stat_v, part_m, stat_m, plan, bytes; /* part_v at 0 */
};

Room make_room(int n, int seqs, int groups, int nh, int nkv, int hd) {
    Room r;
    r.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512;
    const size_t tr = r.hdp > 256 ? 64 : 128, od = r.hdp > 256 ? 256 : r.hdp, hv = r.hdp > 256 ? 2 : 1;
    const size_t qr = (size_t)n * (nh / nkv); /* query rows of a KV head */
    const size_t sv = AB_WGS * AB_PARTS + (size_t)(seqs + groups) * nkv;
    /* segments of the matrix kind, each a tile more than its whole ones; every row in two of them */
    const size_t some = qr / (AB_VR + 1);
    const size_t big = (some < (size_t)seqs ? some : seqs) + (some < (size_t)groups ? some : groups);
    const size_t sm = big ? AB_WGS + (2 * (qr / tr) + big) * hv * nkv : 0;
    r.vrows = qr < AB_VR ? (int)qr : AB_VR; /* the clamped rows of all sequences are n at most */
    size_t at = sv * r.vrows * hd * 4;
    r.stat_v = at, at += sv * r.vrows * sizeof(float4);
    r.part_m = at, at += sm * tr * od * 4;
    r.stat_m = at, at += sm * tr * sizeof(float4);
    r.plan = at, at += (sizeof(Plan) + 15) / 16 * 16;
    r.bytes = at;
    /* columns of a join's workgroup: of one half; few rows share their columns out too */
    int cols = hd;
    if (hd > 256)
        for (cols = 256; hd % cols; cols /= 2) {}
    while ((size_t)n * nh * (hd / cols) < 256 && cols % 128 == 0) cols /= 2;
    r.jcols = cols;
    return r;
}

bool shape_ok(int n, int seqs, int groups, int nh, int nkv, int hd) {
    return n >= 1 && n <= NMX_CHUNK_ROWS && seqs >= 1 && seqs <= NMX_BATCH_MAX && groups >= 0 && groups <= seqs && nkv >= 1 &&
           nh >= nkv && nh % nkv == 0 && nh <= 1024 && hd >= 64 && hd <= 512 && hd % 64 == 0;
}

template <int HDP, int KVT>
int launch(nmx_ctx *ctx, const BatchAttn &a) {
    static std::atomic<uint64_t> set0;
    constexpr int vec = ctx_waves<HDP>() * 4 * (HDP * 4 + 8), mat = ctx_lds<HDP, KVT>();
    constexpr int lds = vec > mat ? vec : mat;
    if (nmx_dyn_lds(ctx, (const void *)attn_batch_k<HDP, KVT>, lds, set0)) return -1;
    attn_batch_k<HDP, KVT><<<AB_WGS, 64 * ctx_waves<HDP>(), lds, ctx->stream>>>(a.row0, a.pg.len, a.pg.seqs, a.n, a.groups,
                                                                              a.pg.max_pages << a.pg.shift, a);
    NMX_LAUNCHED(ctx, "attn_batch");
    const int items = a.n * a.nh * halves<HDP>();
    if (items >= JB_WAVES && (uintptr_t)a.aq % 4 == 0) attn_batch_join_waves_k<HDP><<<(items + JB / 64 - 1) / (JB / 64), JB, 0, ctx->stream>>>(a);
    else attn_batch_join_k<HDP><<<dim3((unsigned)(a.n * a.nh), (unsigned)(a.pg.hd / a.jcols)), JB, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "attn_batch_join");
    return 0;
}
template <int KVT>
int launch_hd(nmx_ctx *ctx, const BatchAttn &a, int hdp) {
    return hdp == 64 ? launch<64, KVT>(ctx, a) : hdp == 128 ? launch<128, KVT>(ctx, a) :
           hdp == 256 ? launch<256, KVT>(ctx, a) : launch<512, KVT>(ctx, a);
}

/* the arguments that both calls use, and their byte ranges */
struct Sizes {
    size_t q, cache, table, len, row0;
};
int batch_shape(nmx_ctx *ctx, const nmx_attn_batch_args *p, const char *what, PageDev *pg, Sizes *z) {
    if (!p) return nmx_fail(ctx, "%s: NULL argument", what);
    if (nmx_pages_check(ctx, p->pages, what, pg)) return -1;
    if (!shape_ok(p->n, pg->seqs, 0, p->nh, pg->nkv, pg->hd))
        return nmx_fail(ctx, "%s: bad shape n=%d nh=%d nkv=%d", what, p->n, p->nh, pg->nkv);
    if (!p->row0 || !p->q || !p->kc || !p->vc) return nmx_fail(ctx, "%s: NULL argument", what);
    if ((uintptr_t)p->q % 16 || (uintptr_t)p->kc % 16 || (uintptr_t)p->vc % 16)
        return nmx_fail(ctx, "%s: q or a cache not 16-byte aligned", what);
    *z = Sizes{(size_t)p->n * p->nh * 2 * pg->hd * 4, pg->block * pg->npages, (size_t)pg->seqs * pg->max_pages * 4,
               (size_t)pg->seqs * 4, (size_t)(pg->seqs + 1) * 4};
    if (nmx_overlap(p->q, z->q, p->kc, z->cache) || nmx_overlap(p->q, z->q, p->vc, z->cache) ||
        nmx_overlap(p->kc, z->cache, p->vc, z->cache))
        return nmx_fail(ctx, "%s: q and the caches overlap", what);
    return 0;
}

} // namespace

extern "C" {

int nmx_attn_batch_prep(nmx_ctx *ctx, const nmx_attn_batch_args *p) {
    if (!ctx) return -1;
    PrepBatch a{};
    Sizes z;
    if (batch_shape(ctx, p, "nmx_attn_batch_prep", &a.pg, &z)) return -1;
    const int hd = a.pg.hd, h2 = p->rot / 2;
    if (!p->k_in || !p->v_in || !p->q_norm || !p->k_norm) return nmx_fail(ctx, "nmx_attn_batch_prep: NULL argument");
    if (p->rot < 0 || p->rot % 2 || p->rot > hd || (p->rot && (!p->rope_cos || !p->rope_sin || p->rope_rows < 1)))
        return nmx_fail(ctx, "nmx_attn_batch_prep: rot=%d rope_rows=%d", p->rot, p->rope_rows);
    if (p->axes < 1 || p->axes > 4) return nmx_fail(ctx, "nmx_attn_batch_prep: axes=%d", p->axes);
    for (int i = 0; i < h2 && p->axis; i++) {
        if (p->axis[i] >= p->axes) return nmx_fail(ctx, "nmx_attn_batch_prep: frequency %d on axis %d of %d", i, p->axis[i], p->axes);
        a.axis[i >> 4] |= (uint32_t)p->axis[i] << 2 * (i & 15);
    }
    const size_t ib = (size_t)p->n * a.pg.nkv * hd * 4, hb = (size_t)hd * 4, rb = (size_t)p->rope_rows * h2 * 4;
    const NmxRange in[] = {{p->k_in, ib}, {p->v_in, ib}, {p->q_norm, hb}, {p->k_norm, hb}, {p->rope_cos, p->rot ? rb : 0},
                           {p->rope_sin, p->rot ? rb : 0}, {p->rope_pos, p->rope_pos ? (size_t)p->n * p->axes * 4 : 0},
                           {p->row0, z.row0}, {a.pg.len, z.len}, {a.pg.table, z.table}};
    if (nmx_hits(in, p->q, z.q) || nmx_hits(in, p->kc, z.cache) || nmx_hits(in, p->vc, z.cache))
        return nmx_fail(ctx, "nmx_attn_batch_prep: q or a cache overlaps an input");
    a.n = p->n, a.nh = p->nh, a.rot = p->rot, a.row0 = p->row0, a.q = p->q, a.k_in = p->k_in, a.v_in = p->v_in;
    a.q_norm = p->q_norm, a.k_norm = p->k_norm, a.eps = p->eps, a.rcos = p->rope_cos, a.rsin = p->rope_sin;
    a.rope_rows = p->rope_rows, a.axes = p->axes, a.rope_pos = p->rope_pos, a.kc = p->kc, a.vc = p->vc;
    const nmx_on_device on(ctx);
    const int heads = a.pg.nkv + p->nh, kv = p->pages.kv_dtype;
    const unsigned wgs = (unsigned)(((size_t)p->n * heads + PREP_WAVES - 1) / PREP_WAVES);
    auto go = [&](auto kernel) { kernel<<<wgs, 64 * PREP_WAVES, 0, ctx->stream>>>(a.row0, a.pg.len, a.pg.seqs, a.n, heads, a); };
    auto go_kv = [&](auto e) {
        if (kv == KV_F16) go(attn_batch_prep_k<KV_F16, e.value>);
        else if (kv == KV_I8) go(attn_batch_prep_k<KV_I8, e.value>);
        else go(attn_batch_prep_k<KV_F32, e.value>);
    };
    if (hd <= 64) go_kv(std::integral_constant<int, 1>{});
    else if (hd <= 128) go_kv(std::integral_constant<int, 2>{});
    else if (hd <= 256) go_kv(std::integral_constant<int, 4>{});
    else go_kv(std::integral_constant<int, 8>{});
    NMX_LAUNCHED(ctx, "attn_batch_prep");
    return 0;
}

size_t nmx_attn_batch_work_bytes(int n, int seqs, int groups, int nh, int nkv, int hd) {
    return shape_ok(n, seqs, groups, nh, nkv, hd) ? make_room(n, seqs, groups, nh, nkv, hd).bytes : 0;
}

int nmx_attn_batch(nmx_ctx *ctx, const nmx_attn_batch_args *p, void *work) {
    if (!ctx) return -1;
    BatchAttn a{};
    Sizes z;
    if (batch_shape(ctx, p, "nmx_attn_batch", &a.pg, &z)) return -1;
    const int hd = a.pg.hd, seqs = a.pg.seqs, kv = p->pages.kv_dtype;
    if (p->groups < 0 || p->groups > seqs) return nmx_fail(ctx, "nmx_attn_batch: groups=%d of %d sequences", p->groups, seqs);
    if (!p->o || !work || (p->a8.q && (!p->a8.d || !p->a8.fs)) || (p->groups && (!p->group0 || !p->shared)))
        return nmx_fail(ctx, "nmx_attn_batch: NULL argument");
    if ((uintptr_t)work % 16 || (uintptr_t)p->o % 16) return nmx_fail(ctx, "nmx_attn_batch: work or o not 16-byte aligned");
    const Room r = make_room(p->n, seqs, p->groups, p->nh, a.pg.nkv, hd);
    const size_t ob = z.q / 2, ab = p->a8.q ? ob : 0; /* a byte a value, a float to 32 each in d and fs */
    const NmxRange in[] = {{p->q, z.q}, {p->kc, z.cache}, {p->vc, z.cache}, {p->row0, z.row0}, {a.pg.len, z.len},
                           {a.pg.table, z.table}, {p->group0, p->groups ? (size_t)(p->groups + 1) * 4 : 0},
                           {p->shared, (size_t)p->groups * 4}};
    const NmxRange out[] = {{work, r.bytes}, {p->o, ob}, {p->a8.q, ab / 4}, {p->a8.d, ab / 32}, {p->a8.fs, ab / 32}};
    for (int i = 0; i < 5; i++) {
        if (nmx_hits(in, out[i].p, out[i].bytes)) return nmx_fail(ctx, "nmx_attn_batch: an output or work overlaps an input");
        for (int k = 0; k < i; k++)
            if (nmx_overlap(out[i].p, out[i].bytes, out[k].p, out[k].bytes))
                return nmx_fail(ctx, "nmx_attn_batch: outputs and work overlap");
    }
    char *ws = (char *)work;
    a.n = p->n, a.nh = p->nh, a.rep = p->nh / a.pg.nkv, a.groups = p->groups, a.row0 = p->row0, a.group0 = p->group0, a.shared = p->shared;
    a.q = p->q, a.kc = p->kc, a.vc = p->vc, a.scale = p->scale, a.plan = (Plan *)(ws + r.plan);
    a.part_v = (float *)ws, a.stat_v = (float4 *)(ws + r.stat_v), a.part_m = (float *)(ws + r.part_m);
    a.stat_m = (float4 *)(ws + r.stat_m), a.jcols = r.jcols, a.vrows = r.vrows, a.o = p->o, a.aq = p->a8.q, a.ad = p->a8.d, a.afs = p->a8.fs;
    const nmx_on_device on(ctx);
    return kv == KV_F16 ? launch_hd<KV_F16>(ctx, a, r.hdp) : kv == KV_I8 ? launch_hd<KV_I8>(ctx, a, r.hdp) :
           launch_hd<KV_F32>(ctx, a, r.hdp);
}

} /* extern "C" */
