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
 * so the state is read once, S^T k, S^T q and the products of nodes are 32-bit matrix instructions,
 * and only the deltas remain to be solved, one level of the tree after the other.
 *
 * A node's sums run over its own ancestors alone (no product with a masked zero), so whatever
 * another branch holds, NaN or infinity, does not reach it. */
#include "nmx_internal.h"
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

constexpr int TP_N = 8; /* nodes of a workgroup */

__global__ __launch_bounds__(256) void lin_tree_pre_k(TreePre a) {
    extern __shared__ float sq[]; /* [TP_N][dk] squares */
    __shared__ float red[4 * TP_N];
    const int groups = (a.C + a.dk - 1) / a.dk, tid = threadIdx.x;
    const int t0 = blockIdx.y * TP_N, nb = a.n - t0 < TP_N ? a.n - t0 : TP_N;
    if ((int)blockIdx.x == groups) { /* gates */
        for (int u = tid; u < nb * a.heads; u += blockDim.x) {
            const int t = t0 + u / a.heads, h = u % a.heads;
            const float b = a.b_in[(size_t)t * a.g_stride + h], av = a.a_in[(size_t)t * a.g_stride + h];
            a.beta[t * a.heads + h] = 1.0f / (1.0f + nmx_gate_expf(-b));
            const float A = a.A ? a.A[h] : -nmx_gate_expf(a.A_log[h]);
            float sp = av + a.dt_bias[h];
            sp = sp > 20.0f ? sp : nmx_gate_log1pf(nmx_gate_expf(sp));
            a.decay[t * a.heads + h] = nmx_gate_expf(A * sp);
        }
        return;
    }
    const int ch = blockIdx.x * a.dk + tid, S = a.K - 1;
    const bool live = tid < a.dk && ch < a.C;
    const int cc = live ? ch : 0;
    float wc[8], y[TP_N];
#pragma unroll
    for (int r = 0; r < 8; r++) wc[r] = r < a.K ? a.conv_w[(size_t)cc * a.K + r] : 0.0f;
#pragma unroll
    for (int u = 0; u < TP_N; u++) {
        y[u] = 0.0f;
        if (u >= nb) continue;
        /* win[j]: tap j's input, the newest (the node itself) at K - 1, then its ancestors, then the
         * state's rows from the newest down */
        float win[8];
        int at = t0 + u, row = S; /* row: the state row above, once the path is over */
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const int j = a.K - 1 - r; /* the r-th newest */
            if (j < 0) continue;
            float x;
            if (at >= 0) {
                x = a.raw[(size_t)at * a.raw_stride + cc];
                at = tree_parent(a.parent, at);
            } else {
                row--;
                x = a.state[(size_t)row * a.C + cc];
            }
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k == j) win[k] = x;
            if (r == 0 && a.xin && live) a.xin[(size_t)(t0 + u) * a.C + ch] = x;
        }
        float acc = wc[0] * win[0];
#pragma unroll
        for (int j = 1; j < 8; j++)
            if (j < a.K) acc = acc + wc[j] * win[j];
        y[u] = nmx_silu(acc);
    }
    if ((int)(blockIdx.x * a.dk) < 2 * a.kd) { /* a q or k head: L2 norm, chains of 4 per node */
        const float scale = (int)(blockIdx.x * a.dk) < a.kd ? a.qscale : 1.0f;
#pragma unroll
        for (int u = 0; u < TP_N; u++)
            if (u < nb && tid < a.dk) sq[u * a.dk + tid] = live ? y[u] * y[u] : 0.0f;
        __syncthreads();
        if (tid < 4 * nb) {
            const float *v = sq + (tid >> 2) * a.dk + (tid & 3);
            float c = 0.0f;
            for (int m = 0; m < a.dk >> 2; m++) c = c + v[4 * m];
            red[tid] = c;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < TP_N; u++) {
            if (u >= nb) continue;
            const float ss = ((red[4 * u] + red[4 * u + 1]) + (red[4 * u + 2] + red[4 * u + 3])) + 0.0f;
            const float r = 1.0f / sqrtf(ss + a.l2eps);
            y[u] = (y[u] * r) * scale;
        }
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

/* One workgroup per head and 16 value columns (a group of the state's layout), a wave per 16 nodes.
 * The state's columns are a matrix operand as they lie: lane (column c, quarter gq) holds the float4
 * slots of keys gq dk/4 .. of its column, and the rows of k and q are read in the same order. */
template <int DK4>
__global__ __launch_bounds__(256) void lin_tree_rule_k(TreeRule a) {
    constexpr int DK = 4 * DK4, NS = DK4 / 4;
    __shared__ float kk[NMX_TREE_MAX][NMX_TREE_MAX + 1], qk[NMX_TREE_MAX][NMX_TREE_MAX + 1];
    __shared__ float del[NMX_TREE_MAX][16], pk[TR_B][DK], pdel[TR_B][16], pdec[TR_B];
    __shared__ float dec[NMX_TREE_MAX], bet[NMX_TREE_MAX], run[6][NMX_TREE_MAX], gs[NMX_TREE_MAX];
    __shared__ int up[6][NMX_TREE_MAX];
    __shared__ unsigned long long sets[NMX_TREE_MAX];
    const int h = blockIdx.x, j0 = blockIdx.y * 16, tid = threadIdx.x, lane = tid & 63, T = tid >> 6;
    const int c = lane & 15, gq = lane >> 4, n = a.n, heads = a.heads, dv = a.dv;
    const size_t logw = (size_t)DK + dv + 1;
    const int kh = h / a.rep;

    float4 s[NS];
    float *Sp = a.S + ((size_t)h * dv + j0) * DK + (4 * c + gq) * 4;
#pragma unroll
    for (int k = 0; k < NS; k++) s[k] = *(const float4 *)(Sp + k * 256);

    /* operands of this wave's nodes: row 16 T + c, keys gq DK4 + 4 k + e */
    const int tn = 16 * T + c;
    const float *row = a.qkv + (size_t)(tn < n ? tn : n - 1) * a.C + kh * DK + gq * DK4;
    float4 kf[NS], qf[NS];
#pragma unroll
    for (int k = 0; k < NS; k++) kf[k] = *(const float4 *)(row + a.kd + 4 * k), qf[k] = *(const float4 *)(row + 4 * k);

    if (T == 0) { /* the tree: sets, decays over 2^k steps, the decays from the state */
        int p;
        const unsigned long long set = tree_ancestors(a.parent, n, &p);
        sets[lane] = set;
        const float d = lane < n ? a.decay[lane * heads + h] : 1.0f;
        dec[lane] = d;
        bet[lane] = lane < n ? a.beta[lane * heads + h] : 0.0f;
        float r = d;
        int q = p;
#pragma unroll
        for (int k = 0; k < 6; k++) {
            run[k][lane] = r, up[k][lane] = q;
            const int from = q < 0 ? lane : q;
            const float ro = __shfl(r, from);
            const int qo = __shfl(q, from);
            if (q >= 0) r *= ro, q = qo;
        }
        gs[lane] = r; /* every node is at most 63 steps from the state */
    }

    /* the updates of the last commit, as nmx_lin_apply makes them */
    int keep = a.keep;
    if (a.keep_dev) {
        const int kd = *a.keep_dev;
        keep = kd < keep ? kd : keep;
    }
    for (int u0 = 0; u0 < keep; u0 += TR_B) {
        const int nb = keep - u0 < TR_B ? keep - u0 : TR_B;
        __syncthreads();
        for (int x = tid; x < nb * DK; x += blockDim.x) pk[x / DK][x % DK] = a.pend[((size_t)(u0 + x / DK) * heads + h) * logw + x % DK];
        for (int x = tid; x < nb * 16; x += blockDim.x) pdel[x >> 4][x & 15] = a.pend[((size_t)(u0 + (x >> 4)) * heads + h) * logw + DK + j0 + (x & 15)];
        if (tid < nb) pdec[tid] = a.pend[((size_t)(u0 + tid) * heads + h) * logw + DK + dv];
        __syncthreads();
        for (int u = 0; u < nb; u++) {
            const float d = pdec[u], w = pdel[u][c];
            const float *k = &pk[u][gq * DK4];
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const float4 x = *(const float4 *)(k + 4 * i);
                s[i].x = s[i].x * d, s[i].y = s[i].y * d, s[i].z = s[i].z * d, s[i].w = s[i].w * d;
                s[i].x = s[i].x + x.x * w, s[i].y = s[i].y + x.y * w, s[i].z = s[i].z + x.z * w, s[i].w = s[i].w + x.w * w;
            }
        }
    }
    if (keep > 0 && T == 0) {
#pragma unroll
        for (int k = 0; k < NS; k++) *(float4 *)(Sp + k * 256) = s[k];
    }

    /* S^T k and S^T q of the wave's nodes: element j is node 16 T + 4 gq + j, column c */
    f32x4 ks = {0.0f, 0.0f, 0.0f, 0.0f}, qs = ks;
#pragma unroll
    for (int k = 0; k < NS; k++) {
        ks = mfma4(kf[k].x, s[k].x, ks), qs = mfma4(qf[k].x, s[k].x, qs);
        ks = mfma4(kf[k].y, s[k].y, ks), qs = mfma4(qf[k].y, s[k].y, qs);
        ks = mfma4(kf[k].z, s[k].z, ks), qs = mfma4(qf[k].z, s[k].z, qs);
        ks = mfma4(kf[k].w, s[k].w, ks), qs = mfma4(qf[k].w, s[k].w, qs);
    }
    __syncthreads(); /* the tree's tables */
    /* D(t, a) (k_t . k_a) and D(t, a) (q_t . k_a), t of this wave, a of tile U */
    for (int U = 0; U <= T; U++) {
        const int an = 16 * U + c;
        const float *ar = a.qkv + (size_t)(an < n ? an : n - 1) * a.C + a.kd + kh * DK + gq * DK4;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
#pragma unroll
        for (int k = 0; k < NS; k++) {
            const float4 b = *(const float4 *)(ar + 4 * k);
            x = mfma4(kf[k].x, b.x, x), y = mfma4(qf[k].x, b.x, y);
            x = mfma4(kf[k].y, b.y, x), y = mfma4(qf[k].y, b.y, y);
            x = mfma4(kf[k].z, b.z, x), y = mfma4(qf[k].z, b.z, y);
            x = mfma4(kf[k].w, b.w, x), y = mfma4(qf[k].w, b.w, y);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int t = 16 * T + 4 * gq + j;
            if (t >= n || !(sets[t] >> an & 1)) continue;
            const int steps = __popcll(sets[t]) - __popcll(sets[an]);
            float d = 1.0f;
            int at = t;
#pragma unroll
            for (int k = 0; k < 6; k++)
                if (steps >> k & 1) d *= run[k][at], at = up[k][at];
            kk[t][an] = x[j] * d, qk[t][an] = y[j] * d;
        }
    }
    __syncthreads();
    /* the deltas, level by level */
    unsigned long long left[4];
    float r[4], o[4];
    int depth[4], levels = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int t = 16 * T + 4 * gq + j;
        left[j] = t < n ? sets[t] : 0;
        depth[j] = t < n ? __popcll(sets[t]) - 1 : -1;
        const float v = t < n ? a.qkv[(size_t)t * a.C + 2 * a.kd + h * dv + j0 + c] : 0.0f;
        const float g = t < n ? gs[t] : 0.0f;
        r[j] = v - g * ks[j], o[j] = g * qs[j];
    }
    for (int t = 0; t < n; t++) { /* uniform: the deepest node */
        const int d = __popcll(sets[t]);
        levels = d > levels ? d : levels;
    }
    for (int d = 0; d < levels; d++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int t = 16 * T + 4 * gq + j;
            if (depth[j] == d) {
                r[j] = r[j] * bet[t];
                del[t][c] = r[j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int t = 16 * T + 4 * gq + j;
            if (depth[j] >= d) {
                const int an = __ffsll((long long)left[j]) - 1; /* ancestors in order of depth */
                left[j] &= left[j] - 1;
                const float x = del[an][c];
                o[j] = o[j] + qk[t][an] * x;
                if (depth[j] > d) r[j] = r[j] - kk[t][an] * x;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int t = 16 * T + 4 * gq + j;
        if (t < n) {
            a.o[(size_t)t * a.o_stride + h * dv + j0 + c] = o[j];
            a.log[((size_t)t * heads + h) * logw + DK + j0 + c] = r[j];
        }
    }
    if (j0 == 0) { /* the log rows' keys and decays */
        for (int x = tid; x < n * DK; x += blockDim.x)
            a.log[((size_t)(x / DK) * heads + h) * logw + x % DK] = a.qkv[(size_t)(x / DK) * a.C + a.kd + kh * DK + x % DK];
        if (tid < n) a.log[((size_t)tid * heads + h) * logw + DK + dv] = dec[tid];
    }
}

template <int DK4>
int launch_rule(nmx_ctx *ctx, const TreeRule &a) {
    lin_tree_rule_k<DK4><<<dim3((unsigned)a.heads, (unsigned)(a.dv / 16)), (unsigned)((a.n + 15) / 16 * 64), 0,
                           ctx->stream>>>(a);
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
    const size_t logw = (size_t)dk + dv + 1, vd = (size_t)heads * dv;
    struct Range {
        const void *p;
        size_t bytes;
    };
    const Range w[] = {{p.out, (size_t)n * p.C * 4}, {p.xin, p.xin ? (size_t)n * p.C * 4 : 0}, {p.beta, (size_t)n * heads * 4},
                       {p.decay, (size_t)n * heads * 4}, {r.S, vd * dk * 4}, {r.o, ((size_t)(n - 1) * r.o_stride + vd) * 4},
                       {r.log, (size_t)n * heads * logw * 4}, {m->y, m->y ? ((size_t)(n - 1) * m->y_stride + vd) * 4 : 0}};
    const Range in[] = {{p.raw, ((size_t)(n - 1) * p.raw_stride + p.C) * 4}, {p.state, (size_t)(p.conv_k - 1) * p.C * 4},
                        {r.pend, (size_t)r.keep * heads * logw * 4}, {m->z, ((size_t)(n - 1) * m->z_stride + vd) * 4},
                        {p.b_in, ((size_t)(n - 1) * p.g_stride + heads) * 4}, {p.a_in, ((size_t)(n - 1) * p.g_stride + heads) * 4}};
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
    lin_tree_pre_k<<<dim3((unsigned)((p.C + dk - 1) / dk + 1), (unsigned)((n + TP_N - 1) / TP_N)),
                     (unsigned)(dk < 64 ? 64 : dk), (size_t)TP_N * dk * 4, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "lin_tree_pre");
    const TreeRule t{n, heads, r.rep, dv, p.kd, p.C, p.out, p.beta, p.decay, r.S, r.o, r.o_stride, r.log, r.pend, r.keep,
                     r.keep_dev, parent};
    const int rc = dk == 32 ? launch_rule<8>(ctx, t) : dk == 64 ? launch_rule<16>(ctx, t) :
                   dk == 128 ? launch_rule<32>(ctx, t) : launch_rule<64>(ctx, t);
    if (rc) return rc;
    return nmx_lin_post(ctx, r.o, r.o_stride, m->z, m->z_stride, m->norm_w, n, heads, dv, m->eps, m->y, m->y_stride,
                        m->a8);
}

} /* extern "C" */
