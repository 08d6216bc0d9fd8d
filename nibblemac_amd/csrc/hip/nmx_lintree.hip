/* The Gated DeltaNet mixer over a tree of drafts (include/nmx.h nmx_lin_mix_tree): causal conv, SiLU,
 * L2 norms and gates with each node's conv window taken along its ancestors, then the recurrence from
 * each node's parent's state, then the gated RMSNorm (nmx_lin_post).
 *
 * No node's state is ever formed. With S the state before the tree, g_t the product of the decays
 * from it to node t and D(t, a) the product of those after ancestor a, the recurrence
 *     S_t = S_parent decay_t + k_t delta_t^T,  delta_t = beta_t (v_t - decay_t S_parent^T k_t)
 * unrolls to sums over a node's ancestors:
 *     delta_t = beta_t (v_t - g_t S^T k_t - sum_{a above t} D(t, a) (k_t . k_a) delta_a)
 *     o_t     = g_t S^T q_t + sum_{a above t, t} D(t, a) (q_t . k_a) delta_a
 * so the state is read once, S^T k and S^T q are 32-bit matrix instructions, the products of nodes 16-bit
 * ones of two parts each, and only the deltas remain to be solved, one level of the tree after the other.
 *
 * A node's sums run over its own ancestors alone (no product with a masked zero), so whatever
 * another branch holds, NaN or infinity, does not reach it.
 *
 * On MI355X, 16 heads of 128 x 128: 9 nodes 15.7 us (3.0 MB, 0.6 us as a copy), 64 nodes 26.0 to 26.5 us (7.6 MB,
 * 1.5 us; traced: pre 5.8, rule 19.9, post 4.2). Both are chains of phases behind barriers, not bytes; of the rule's
 * at 64 nodes (before rows had powers of two of their own, about 0.2 us) the requests take 2.1 us, parts of the
 * rows 1.6, 5 pending rows 2.2, the state's products and the tree's tables 2.2, the products of nodes
 * 2.3, 15 levels 3.5. A level costs a barrier: a chain of 64 nodes takes 49 us. The whole mixer of a head
 * in one workgroup, for up to 16 nodes, took longer (9 nodes 18.0, 16 nodes 20.8 against 17.0 us). */
#include "nmx_internal.h"
#include "nmx_a8.h"
#include "nmx_lanes.h"
#include "nmx_math.h"
#include "nmx_tree.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

/* ---- conv, norms, gates: lin_pre_k's operations per node ----------------------------------- */
struct TreePre {
    int n, C, K, dk, kd;
    const float *raw;
    int raw_stride;
    float *out;
    const float *state, *conv_w;
    float *xin;
    float qscale, l2eps;
    const float *b_in, *a_in;
    int g_stride, heads;
    const float *A_log, *A, *dt_bias;
    float *beta, *decay;
    const int32_t *parent;
};

constexpr int TP_N = 4; /* nodes of a workgroup */

/* Partial sum l of 4 interleaved ones over the dk squares of a row (v: element l of it, dk / 4 elements 4
 * apart), in element order: the adds of lin_pre_k. */
__device__ __forceinline__ float square_chain(const float *v, int m4) {
    float c = 0.0f;
    int m = 0;
    for (; m + 8 <= m4; m += 8) {
        float b[8];
#pragma unroll
        for (int u = 0; u < 8; u++) b[u] = v[4 * (m + u)];
#pragma unroll
        for (int u = 0; u < 8; u++) c = c + b[u] * b[u];
    }
    for (; m < m4; m++) c = c + v[4 * m] * v[4 * m];
    return c;
}
/* (c0 + c1) + (c2 + c3) of a quad's lanes, in each of them */
__device__ __forceinline__ float quad_sum(float c) {
    const float o = __int_as_float(nmx_dpp<NMX_DPP_XOR1>(__float_as_int(c)));
    const float s = c + o;
    return s + __int_as_float(nmx_dpp<NMX_DPP_XOR2>(__float_as_int(s)));
}
__device__ __forceinline__ float tree_beta(const float b) { return 1.0f / (1.0f + nmx_gate_expf(-b)); }
__device__ __forceinline__ float tree_decay(const TreePre &a, float av, int h) {
    const float A = a.A ? a.A[h] : -nmx_gate_expf(a.A_log[h]);
    float sp = av + a.dt_bias[h];
    sp = sp > 20.0f ? sp : nmx_gate_log1pf(nmx_gate_expf(sp));
    return nmx_gate_expf(A * sp);
}

template <int KT>
__global__ __launch_bounds__(256) void lin_tree_pre_k(TreePre a) {
    extern __shared__ float sq[]; /* [TP_N][dk + 4] */
    __shared__ float red[TP_N];
    __shared__ int par[NMX_TREE_MAX];
    const int groups = (a.C + a.dk - 1) / a.dk, tid = threadIdx.x;
    const int t0 = blockIdx.y * TP_N, nb = a.n - t0 < TP_N ? a.n - t0 : TP_N;
    if ((int)blockIdx.x == groups) { /* gates */
        for (int u = tid; u < nb * a.heads; u += blockDim.x) {
            const int t = t0 + u / a.heads, h = u % a.heads;
            a.beta[t * a.heads + h] = tree_beta(a.b_in[(size_t)t * a.g_stride + h]);
            a.decay[t * a.heads + h] = tree_decay(a, a.a_in[(size_t)t * a.g_stride + h], h);
        }
        return;
    }
    for (int t = tid; t < a.n; t += blockDim.x) par[t] = tree_parent(a.parent, t);
    const int ch = blockIdx.x * a.dk + tid, K = KT ? KT : a.K, S = K - 1;
    const bool live = tid < a.dk && ch < a.C;
    const int cc = live ? ch : 0;
    constexpr int KM = KT ? KT : 8;
    float wc[KM], y[TP_N], win[TP_N][KM];
#pragma unroll
    for (int r = 0; r < KM; r++) wc[r] = r < K ? a.conv_w[(size_t)cc * K + r] : 0.0f;
    nmx_lds_sync();
    /* win[u][j]: tap j's input, the newest (the node itself) at K - 1, then its ancestors, then the state's
     * rows from the newest down; nodes past the end repeat the last one */
#pragma unroll
    for (int u = 0; u < TP_N; u++) {
        int at = t0 + (u < nb ? u : nb - 1), row = S; /* row: the state row above, once the path is over */
#pragma unroll
        for (int r = 0; r < KM; r++) {
            if (!KT && r >= K) break;
            const bool node = at >= 0;
            row -= !node;
            const float *src = node ? a.raw + (size_t)at * a.raw_stride : a.state + (size_t)row * a.C;
            win[u][r] = src[cc]; /* the r-th newest */
            at = node ? par[at] : at;
        }
    }
#pragma unroll
    for (int u = 0; u < TP_N; u++) {
        /* taps in order, the oldest first */
        float acc = 0.0f;
#pragma unroll
        for (int j = 0; j < KM; j++) {
            if (!KT && j >= K) break;
            float x = win[u][KT ? KT - 1 - j : 0];
            if constexpr (!KT) {
#pragma unroll
                for (int r = 0; r < KM; r++) x = r == K - 1 - j ? win[u][r] : x;
            }
            acc = j ? acc + wc[j] * x : wc[0] * x;
        }
        y[u] = nmx_silu(acc);
        if (a.xin && live && u < nb) a.xin[(size_t)(t0 + u) * a.C + ch] = win[u][0];
    }
    if ((int)(blockIdx.x * a.dk) < 2 * a.kd) { /* a q or k head: L2 norm, chains of 4 per node */
        const float scale = (int)(blockIdx.x * a.dk) < a.kd ? a.qscale : 1.0f;
        const int rs = a.dk + 4;
#pragma unroll
        for (int u = 0; u < TP_N; u++)
            if (tid < a.dk) sq[u * rs + tid] = live ? y[u] : 0.0f;
        nmx_lds_sync();
        if (tid < 4 * TP_N) {
            const float c = square_chain(sq + (tid >> 2) * rs + (tid & 3), a.dk >> 2);
            red[tid >> 2] = 1.0f / sqrtf((quad_sum(c) + 0.0f) + a.l2eps);
        }
        nmx_lds_sync();
#pragma unroll
        for (int u = 0; u < TP_N; u++) y[u] = (y[u] * red[u]) * scale;
    }
#pragma unroll
    for (int u = 0; u < TP_N; u++)
        if (u < nb && live) a.out[(size_t)(t0 + u) * a.C + ch] = y[u];
}

/* ---- the recurrence ------------------------------------------------------------------------- */
struct TreeRule {
    int n, heads, rep, dv, kd, C;
    const float *qkv;           /* [n][C]: conv outputs q | k | v */
    const float *beta, *decay;  /* [n][heads] */
    float *S, *o;
    int o_stride;
    float *log;
    const float *pend;
    int keep;
    const int32_t *keep_dev, *parent;
};

constexpr int TR_B = 8; /* pending rows staged at a time */

/* The tree in LDS: of node t, in order of depth, its ancestors (itself the last) and
 * the product of the decays after each of them up to t; the product of all of them from the state. */
struct TreeTables {
    static constexpr int N = NMX_TREE_MAX;
    unsigned long long sets[N];
    float dec[N], bet[N], gs[N], gap[N][N + 1];
    uint8_t depth[N];
    alignas(16) uint8_t anc[N][N]; /* past a node's depth: itself */
    int levels;
};
/* One wave; lane t < n: its parent p, decay d and beta bt. */
__device__ __forceinline__ void tree_tables(TreeTables &s, int n, unsigned long long set, int p, float d, float bt) {
    const int lane = threadIdx.x & 63;
    const bool in = lane < n;
    int at = in ? __popcll(set) - 1 : -1, cur = lane;
    int deep = at;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) deep = max(deep, __shfl_xor(deep, x));
    s.sets[lane] = set, s.dec[lane] = d, s.bet[lane] = bt, s.depth[lane] = (uint8_t)(at < 0 ? 0 : at);
    for (int k = at < 0 ? 0 : at; k <= deep; k++) s.anc[lane][k] = (uint8_t)lane;
    float g = 1.0f;
    for (int k = 0; k <= deep; k++) { /* up the path, every lane at once */
        if (at >= 0) s.gap[lane][at] = g, s.anc[lane][at] = (uint8_t)cur;
        const float dc = __shfl(d, cur);
        const int up = __shfl(p, cur);
        if (at >= 0) g *= dc;
        at--;
        cur = up < 0 ? cur : up;
    }
    s.gs[lane] = g;
    if (lane == 0) s.levels = deep + 1;
}

/* Rows of k and q for the products of nodes: a row is brought to a norm about 2^12 by a power of two of its
 * own (the norm's epsilon leaves small conv rows far below 1), an element then taken as its nearest
 * whole number and the rest, both binary16. Products of whole numbers add up to no more than about 2^24: exact in
 * the accumulator. The products of a whole number and a rest are 2^-12 of that and have an accumulator of
 * their own: beside a larger sum the matrix instruction drops what lies below 2^-26 of it from every
 * product, which was the largest error of o where q.k nearly cancels. The products of two rests go there
 * too: 2^-24 and random between different rows, but of rows alike (a token repeated) they add up to dk / 12
 * of that in every product. Four 16-bit instructions per 32 keys in place of 32 32-bit ones. */
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma16(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void split4(float4 x, float up, _Float16 *hi, _Float16 *lo) {
    const float v[4] = {x.x * up, x.y * up, x.z * up, x.w * up};
    half4 h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = (_Float16)rintf(v[i]), l[i] = (_Float16)(v[i] - (float)h[i]);
    *(half4 *)hi = h, *(half4 *)lo = l;
}
__device__ __forceinline__ float sum_squares(const float4 *x, int n) {
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < n; i++) {
        s.x = __builtin_fmaf(x[i].x, x[i].x, s.x), s.y = __builtin_fmaf(x[i].y, x[i].y, s.y);
        s.z = __builtin_fmaf(x[i].z, x[i].z, s.z), s.w = __builtin_fmaf(x[i].w, x[i].w, s.w);
    }
    return nmx_sum_quarters((s.x + s.y) + (s.z + s.w));
}
/* The power of two that a row scaled for its products is brought back by, from its sum of squares: 2^(e - 12)
 * for the least e with ss < 2^(2 e), e from -63 on (below, a product has no 32-bit value either) up to 65. */
__device__ __forceinline__ float row_down(float ss) {
    const int e = ((int)(__float_as_uint(ss) >> 23 & 255) - 125) >> 1;
    return __uint_as_float((uint32_t)(e - 12 + 127) << 23);
}
__device__ __forceinline__ float inverse_pow2(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

/* The pending rows of head h, TR_B at a time: keys and decays to LDS (pk, pdec), the deltas of column
 * col to registers. The first batch is requested at the kernel's entry, among its other requests. */
template <int DK4, int TMIN>
struct Replay {
    static constexpr int DK = 4 * DK4, NP = (TR_B * DK + TMIN - 1) / TMIN; /* TMIN: the least threads of a workgroup */
    float k[NP], w[TR_B], d;
    __device__ __forceinline__ void ask(const float *pend, int u0, int keep, int heads, int h, size_t logw, int col) {
        const int nb = keep - u0 < TR_B ? keep - u0 : TR_B;
        if (nb <= 0) return;
        auto row = [&](int u) { return pend + ((size_t)(u0 + (u < nb ? u : nb - 1)) * heads + h) * logw; };
#pragma unroll
        for (int e = 0; e < NP; e++) {
            const int x = e * (int)blockDim.x + (int)threadIdx.x;
            k[e] = row(x / DK)[x % DK];
        }
#pragma unroll
        for (int u = 0; u < TR_B; u++) w[u] = row(u)[DK + col];
        d = row(threadIdx.x < TR_B ? threadIdx.x : 0)[logw - 1];
    }
    /* into the state's columns held in s, as nmx_lin_apply makes them; a wave without columns only helps to
     * stage */
    __device__ __forceinline__ void run(float4 (&s)[DK4 / 4], const float *pend, int asked, int keep, int heads, int h, size_t logw,
                                        int col, float (*pk)[DK + 16], float *pdec, bool has) {
        const int tid = threadIdx.x, gq = (tid & 63) >> 4;
        for (int u0 = 0; u0 < keep; u0 += TR_B) {
            if (u0) ask(pend, u0, asked, heads, h, logw, col);
            const int nb = keep - u0 < TR_B ? keep - u0 : TR_B;
            nmx_lds_sync();
#pragma unroll
            for (int e = 0; e < NP; e++) {
                const int x = e * (int)blockDim.x + tid, i = x % DK;
                if (x < TR_B * DK) pk[x / DK][i + 4 * (i / DK4)] = k[e];
            }
            if (tid < TR_B) pdec[tid] = d;
            nmx_lds_sync();
#pragma unroll
            for (int u = 0; u < TR_B; u++) {
                if (u >= nb || !has) continue;
                const float dc = pdec[u];
                const float *kr = &pk[u][gq * (DK4 + 4)];
#pragma unroll
                for (int i = 0; i < DK4 / 4; i++) {
                    const float4 x = *(const float4 *)(kr + 4 * i);
                    s[i].x = s[i].x * dc, s[i].y = s[i].y * dc, s[i].z = s[i].z * dc, s[i].w = s[i].w * dc;
                    s[i].x = s[i].x + x.x * w[u], s[i].y = s[i].y + x.y * w[u], s[i].z = s[i].z + x.z * w[u], s[i].w = s[i].w + x.w * w[u];
                }
            }
        }
    }
};
__device__ __forceinline__ int keep_of(int keep, const int32_t *keep_dev) {
    if (!keep_dev) return keep;
    const int d = *keep_dev;
    return d < keep ? d : keep;
}

/* A wave of its own for the tree's tables; of 256 keys the four waves of 64 nodes need the registers. */
template <int DK4>
constexpr int tree_wave() {
    return DK4 < 64 ? 1 : 0;
}

/* One workgroup per head and 16 value columns (a group of the state's layout), a wave per 16 nodes. The
 * state's columns are a matrix operand as they lie: lane (column c, quarter gq) holds the float4 slots of
 * keys gq dk/4 .. of its column, and the wave's rows of k and q are read in the same order. */
template <int DK4>
__global__ __launch_bounds__(256 + 64 * tree_wave<DK4>()) void lin_tree_rule_k(TreeRule a) {
    constexpr int DK = 4 * DK4, NS = DK4 / 4, HS = DK + 8; /* halves of a row in LDS: 16 bytes on, no bank twice */
    extern __shared__ float4 smem4[];
    __shared__ TreeTables tt;
    __shared__ float del[2][NMX_TREE_MAX][16], pdec[TR_B];
    __shared__ float2 down[NMX_TREE_MAX]; /* of a node's k and q: what their scaled products are multiplied by */
    const int h = blockIdx.x, j0 = blockIdx.y * 16, tid = threadIdx.x, lane = tid & 63, T = tid >> 6, waves = (int)(blockDim.x >> 6) - tree_wave<DK4>();
    const int c = lane & 15, gq = lane >> 4, n = a.n, heads = a.heads, dv = a.dv, n16 = 16 * waves;
    _Float16 *kh2 = (_Float16 *)smem4, *qh2 = kh2 + 2 * n16 * HS;   /* [2][n16][HS]: high, low parts */
    constexpr bool QL = DK4 < 64; /* 256 keys: the parts of q are made when they are used, LDS has no room */
    float2 *co = (float2 *)(QL ? qh2 + 2 * n16 * HS : qh2);         /* [n16][n16 + 1]: D k.k, D q.k of a node's ancestors by depth */
    float(*pk)[DK + 16] = (float(*)[DK + 16])co;                    /* pending keys, before the products */
    const size_t logw = (size_t)DK + dv + 1;
    const int kh = h / a.rep;

    Replay<DK4, DK4 < 64 ? 128 : 64> rp;
    rp.ask(a.pend, 0, a.keep, heads, h, logw, j0 + c);
    float4 s[NS], kf[NS], qf[NS];
    float *Sp = a.S + ((size_t)h * dv + j0) * DK + (4 * c + gq) * 4;
#pragma unroll
    for (int k = 0; k < NS; k++) s[k] = *(const float4 *)(Sp + k * 256);
    /* rows past the end repeat the last one: their products are not used */
    const int tn = 16 * T + c;
    const float *row = a.qkv + (size_t)(tn < n ? tn : n - 1) * a.C + kh * DK + gq * DK4;
#pragma unroll
    for (int k = 0; k < NS; k++) kf[k] = *(const float4 *)(row + a.kd + 4 * k), qf[k] = *(const float4 *)(row + 4 * k);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int t = 16 * T + 4 * gq + j;
        v[j] = a.qkv[(size_t)(t < n ? t : n - 1) * a.C + 2 * a.kd + h * dv + j0 + c];
    }
    const bool nodes = T < waves; /* the last wave has the tree instead */
    const bool tree = T == (int)(blockDim.x >> 6) - 1;
    float dc = 1.0f, bt1 = 0.0f;
    int up = -1;
    unsigned long long set = 0;
    if (tree) {
        dc = lane < n ? a.decay[lane * heads + h] : 1.0f, bt1 = lane < n ? a.beta[lane * heads + h] : 0.0f;
        set = tree_ancestors(a.parent, n, &up);
    }
    if (nodes) {
        /* a little less than the squares: a norm of 1, give or take a rounding, stays 2^12; half of q's, whose
         * norm of dk^-1/2 then goes to 2^12 or 2^12.5 */
        const float kdown = row_down(sum_squares(kf, NS) * 0.998f), qdown = row_down(sum_squares(qf, NS) * 0.499f);
        const float k_up = inverse_pow2(kdown), q_up = inverse_pow2(qdown);
        if (gq == 0) down[tn] = make_float2(kdown, qdown);
#pragma unroll
        for (int k = 0; k < NS; k++) {
            const int at = tn * HS + gq * DK4 + 4 * k;
            split4(kf[k], k_up, kh2 + at, kh2 + n16 * HS + at);
            if (QL) split4(qf[k], q_up, qh2 + at, qh2 + n16 * HS + at);
        }
    }
    const int keep = keep_of(a.keep, a.keep_dev);
    rp.run(s, a.pend, a.keep, keep, heads, h, logw, j0 + c, pk, pdec, nodes);
    if (tree) tree_tables(tt, n, set, up, dc, bt1); /* while the others multiply */
    /* S^T k and S^T q of the wave's nodes: element j is node 16 T + 4 gq + j, column c */
    f32x4 sk = {0.0f, 0.0f, 0.0f, 0.0f}, sq = sk, sk2 = sk, sq2 = sk; /* two chains each: shorter ones round less */
#pragma unroll
    for (int k = 0; k < NS; k++) {
        sk = mfma4(kf[k].x, s[k].x, sk), sq = mfma4(qf[k].x, s[k].x, sq);
        sk2 = mfma4(kf[k].y, s[k].y, sk2), sq2 = mfma4(qf[k].y, s[k].y, sq2);
        sk = mfma4(kf[k].z, s[k].z, sk), sq = mfma4(qf[k].z, s[k].z, sq);
        sk2 = mfma4(kf[k].w, s[k].w, sk2), sq2 = mfma4(qf[k].w, s[k].w, sq2);
    }
    sk += sk2, sq += sq2;
    /* the rows, the tables; the pending keys have been read */
    if (keep > 0) {
        __syncthreads(); /* and every wave's request of the state's columns has come: one of them writes */
        if (T == 0)
#pragma unroll
            for (int k = 0; k < NS; k++) *(float4 *)(Sp + k * 256) = s[k];
    } else {
        nmx_lds_sync();
    }
    /* D(t, a) (k_t . k_a) and D(t, a) (q_t . k_a): the tiles (t, a) on and below the diagonal, in turn */
    const int all = (int)(blockDim.x >> 6);
    for (int job = T, X = 0; X < waves; job -= X + 1, X++) {
        for (; job <= X; job += all) {
            const int U = job, an = 16 * U + c;
            const _Float16 *ar = kh2 + an * HS + 8 * gq, *tr = kh2 + (16 * X + c) * HS + 8 * gq, *ur = qh2 + (16 * X + c) * HS + 8 * gq;
            const int lo = n16 * HS;
            const float q_up = QL ? 0.0f : inverse_pow2(down[16 * X + c].y);
            f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x, xr = x, yr = x, xs = x, ys = x;
#pragma unroll
            for (int k = 0; k < DK; k += 32) {
                const half8 ah = *(const half8 *)(ar + k), al = *(const half8 *)(ar + lo + k);
                const half8 th = *(const half8 *)(tr + k), tl = *(const half8 *)(tr + lo + k);
                half8 uh, ul;
                if constexpr (QL) {
                    uh = *(const half8 *)(ur + k), ul = *(const half8 *)(ur + lo + k);
                } else {
                    const int t = 16 * X + c < n ? 16 * X + c : n - 1;
                    const float *src = a.qkv + (size_t)t * a.C + kh * DK + k + 8 * gq;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float v = src[i] * q_up;
                        uh[i] = (_Float16)rintf(v), ul[i] = (_Float16)(v - (float)uh[i]);
                    }
                }
                x = mfma16(th, ah, x), y = mfma16(uh, ah, y);
                xr = mfma16(tl, ah, xr), yr = mfma16(ul, ah, yr);
                xs = mfma16(th, al, xs), ys = mfma16(uh, al, ys);
                xr = mfma16(tl, al, xr), yr = mfma16(ul, al, yr);
            }
            x += xr + xs, y += yr + ys;
            const int dp = tt.depth[an];
            const float down_a = down[an].x;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int t = 16 * X + 4 * gq + j;
                if (t >= n || !(tt.sets[t] >> an & 1)) continue;
                const float d = tt.gap[t][dp] * down_a;
                const float2 dt = down[t];
                co[t * (n16 + 1) + dp] = make_float2(x[j] * dt.x * d, y[j] * dt.y * d);
            }
        }
    }
    nmx_lds_sync();
    /* the deltas, level by level; four levels' ancestors and the next level's coefficients are at hand */
    float r[4], o[4], bt[4];
    float2 cf[4];
    int depth[4], tj[4];
    uint32_t an[4];
    const int levels = tt.levels;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int t = 16 * T + 4 * gq + j;
        const bool in = nodes && t < n;
        tj[j] = in ? t : n - 1;
        depth[j] = in ? tt.depth[t] : -1;
        const float g = tt.gs[tj[j]];
        bt[j] = tt.bet[tj[j]];
        r[j] = v[j] - g * sk[j], o[j] = g * sq[j];
        an[j] = *(const uint32_t *)tt.anc[tj[j]];
        cf[j] = co[tj[j] * (n16 + 1)];
    }
    /* the log rows' keys and decays: a share of the nodes for each workgroup of the head */
    constexpr int LB = 4; /* values of a thread on their way at once */
    const int mine = (n - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y * DK, TH = (int)blockDim.x; /* blockIdx.y >= n: none */
    float lk[LB];
    auto node_of = [&](int x) { return (int)blockIdx.y + x / DK * (int)gridDim.y; };
    auto ask_keys = [&](int x0) {
#pragma unroll
        for (int u = 0; u < LB; u++) {
            const int x = x0 + u * TH < mine ? x0 + u * TH : 0, t = node_of(x);
            lk[u] = a.qkv[(size_t)(t < n ? t : n - 1) * a.C + a.kd + kh * DK + x % DK];
        }
    };
    ask_keys(tid); /* there when the deltas are */
    for (int d = 0; d < levels; d++) {
        float(*dl)[16] = del[d & 1]; /* read in this level while the next one is written */
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool now = depth[j] == d;
            r[j] = now ? r[j] * bt[j] : r[j];
            if (now) dl[tj[j]][c] = r[j];
        }
        nmx_lds_sync();
        float x[4];
        float2 cn[4];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = dl[an[j] & 255][c];
#pragma unroll
        for (int j = 0; j < 4; j++) cn[j] = co[tj[j] * (n16 + 1) + d + 1];
#pragma unroll
        for (int j = 0; j < 4; j++) { /* chosen, not multiplied away: a node past its depth reads anything */
            o[j] = depth[j] >= d ? o[j] + cf[j].y * x[j] : o[j];
            r[j] = depth[j] > d ? r[j] - cf[j].x * x[j] : r[j];
            an[j] >>= 8, cf[j] = cn[j];
        }
        if ((d & 3) == 3)
#pragma unroll
            for (int j = 0; j < 4; j++) an[j] = *(const uint32_t *)(tt.anc[tj[j]] + ((d + 1) & 63));
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int t = 16 * T + 4 * gq + j;
        if (nodes && t < n) {
            a.o[(size_t)t * a.o_stride + h * dv + j0 + c] = o[j];
            a.log[((size_t)t * heads + h) * logw + DK + j0 + c] = r[j];
        }
    }
    for (int x0 = tid; x0 < mine; x0 += LB * TH) {
        if (x0 != tid) ask_keys(x0);
#pragma unroll
        for (int u = 0; u < LB; u++) {
            const int x = x0 + u * TH;
            if (x < mine) a.log[((size_t)node_of(x) * heads + h) * logw + x % DK] = lk[u];
        }
    }
    if (tid * DK < mine) a.log[((size_t)node_of(tid * DK) * heads + h) * logw + DK + dv] = tt.dec[node_of(tid * DK)];
}

template <int DK4>
int launch_rule(nmx_ctx *ctx, const TreeRule &a) {
    const int n16 = (a.n + 15) / 16 * 16;
    auto bytes = [](int m) {
        const size_t co = (size_t)m * (m + 1) * 8, pk = (size_t)TR_B * (4 * DK4 + 16) * 4;
        return (size_t)(DK4 < 64 ? 4 : 2) * m * (4 * DK4 + 8) * 2 + (co > pk ? co : pk);
    };
    static std::atomic<uint64_t> set;
    if (nmx_dyn_lds(ctx, (const void *)lin_tree_rule_k<DK4>, bytes(64), set)) return -1;
    lin_tree_rule_k<DK4><<<dim3((unsigned)a.heads, (unsigned)(a.dv / 16)), (unsigned)(4 * n16 + 64 * tree_wave<DK4>()),
                           bytes(n16), ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "lin_tree_rule");
    return 0;
}

} // namespace

extern "C" {

int nmx_lin_mix_tree(nmx_ctx *ctx, const nmx_lin_mix_args *m, const int32_t *parent) {
    if (!ctx) return -1;
    if (!m || !parent) return nmx_fail(ctx, "nmx_lin_mix_tree: NULL argument");
    const nmx_lin_pre_args &p = m->pre;
    const nmx_lin_args &r = m->rule;
    const int n = p.n, dk = p.dk, dv = r.dv, heads = r.heads;
    if (n < 1 || n > NMX_TREE_MAX || n != r.n || dk != r.dk || p.heads != heads || heads < 1 || heads > 256 ||
        r.rep < 1 || heads % r.rep || (dk != 32 && dk != 64 && dk != 128 && dk != 256) || dv < 32 || dv > 512 || dv % 32 ||
        p.conv_k < 1 || p.conv_k > 8 || p.kd != heads / r.rep * dk || p.C != 2 * p.kd + heads * dv ||
        p.raw_stride < p.C || p.g_stride < heads || r.o_stride < heads * dv || m->z_stride < heads * dv ||
        (m->y && m->y_stride < heads * dv) || r.keep < 0 || r.keep > 64)
        return nmx_fail(ctx, "nmx_lin_mix_tree: bad shape n=%d heads=%d rep=%d dk=%d dv=%d conv_k=%d keep=%d", n, heads,
                        r.rep, dk, dv, p.conv_k, r.keep);
    if (!p.raw || !p.out || (p.conv_k > 1 && !p.state) || !p.conv_w || !p.b_in || !p.a_in || !p.beta || !p.decay ||
        !p.dt_bias || (!p.A_log && !p.A) || !r.S || !r.o || !r.log || (r.keep > 0 && !r.pend) || !m->z || !m->norm_w ||
        (!m->y && !m->a8.q) || (m->a8.q && (!m->a8.d || !m->a8.fs)))
        return nmx_fail(ctx, "nmx_lin_mix_tree: NULL argument");
    if ((uintptr_t)p.out % 16 || (uintptr_t)r.S % 16)
        return nmx_fail(ctx, "nmx_lin_mix_tree: pre.out or the state not 16-byte aligned");
    /* what is written overlaps nothing else that is read or written */
    const size_t logw = (size_t)dk + dv + 1, vd = (size_t)heads * dv, gb = (size_t)heads * 4;
    struct Range {
        const void *p;
        size_t bytes;
    };
    const Range w[] = {{p.out, (size_t)n * p.C * 4}, {p.xin, p.xin ? (size_t)n * p.C * 4 : 0}, {p.beta, n * gb},
                       {p.decay, n * gb}, {r.S, vd * dk * 4}, {r.o, ((size_t)(n - 1) * r.o_stride + vd) * 4},
                       {r.log, n * gb * logw}, {m->y, m->y ? ((size_t)(n - 1) * m->y_stride + vd) * 4 : 0},
                       {m->a8.q, m->a8.q ? n * vd : 0}, {m->a8.d, m->a8.q ? n * vd / 8 : 0}, {m->a8.fs, m->a8.q ? n * vd / 8 : 0}};
    const Range in[] = {{p.raw, ((size_t)(n - 1) * p.raw_stride + p.C) * 4}, {p.state, (size_t)(p.conv_k - 1) * p.C * 4},
                        {p.conv_w, (size_t)p.C * p.conv_k * 4}, {r.pend, r.keep * gb * logw},
                        {m->z, ((size_t)(n - 1) * m->z_stride + vd) * 4}, {m->norm_w, (size_t)dv * 4},
                        {p.b_in, (size_t)(n - 1) * p.g_stride * 4 + gb}, {p.a_in, (size_t)(n - 1) * p.g_stride * 4 + gb},
                        {p.A_log, p.A_log ? gb : 0}, {p.A, p.A ? gb : 0}, {p.dt_bias, gb}, {parent, (size_t)n * 4},
                        {r.keep_dev, r.keep_dev ? sizeof(int32_t) : 0}};
    for (size_t i = 0; i < sizeof w / sizeof *w; i++) {
        for (const Range &x : in)
            if (nmx_overlap(w[i].p, w[i].bytes, x.p, x.bytes))
                return nmx_fail(ctx, "nmx_lin_mix_tree: an output overlaps an input");
        for (size_t k = 0; k < i; k++)
            if (nmx_overlap(w[i].p, w[i].bytes, w[k].p, w[k].bytes))
                return nmx_fail(ctx, "nmx_lin_mix_tree: outputs overlap");
    }
    const nmx_on_device on(ctx);
    const TreePre a{n, p.C, p.conv_k, dk, p.kd, p.raw, p.raw_stride, p.out, p.state, p.conv_w, p.xin, p.qscale, p.l2eps,
                    p.b_in, p.a_in, p.g_stride, heads, p.A_log, p.A, p.dt_bias, p.beta, p.decay, parent};
    const TreeRule t{n, heads, r.rep, dv, p.kd, p.C, p.out, p.beta, p.decay, r.S, r.o, r.o_stride, r.log, r.pend, r.keep,
                     r.keep_dev, parent};
    const dim3 grid((unsigned)((p.C + dk - 1) / dk + 1), (unsigned)((n + TP_N - 1) / TP_N));
    const unsigned threads = dk < 64 ? 64 : (unsigned)dk;
    const size_t lds = (size_t)TP_N * (dk + 4) * 4;
    if (p.conv_k == 4) lin_tree_pre_k<4><<<grid, threads, lds, ctx->stream>>>(a);
    else lin_tree_pre_k<0><<<grid, threads, lds, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "lin_tree_pre");
    const int rc = dk == 32 ? launch_rule<8>(ctx, t) : dk == 64 ? launch_rule<16>(ctx, t) :
                   dk == 128 ? launch_rule<32>(ctx, t) : launch_rule<64>(ctx, t);
    if (rc) return rc;
    return nmx_lin_post(ctx, r.o, r.o_stride, m->z, m->z_stride, m->norm_w, n, heads, dv, m->eps, m->y, m->y_stride,
                        m->a8);
}

} /* extern "C" */
