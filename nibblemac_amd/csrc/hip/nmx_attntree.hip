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
 * two parts itself: three products, the low-low one left out (2^-22 of the row). */
#include "nmx_internal.h"
#include "nmx_a8.h"
#include "nmx_attn.h"
#include "nmx_lanes.h"
#include "nmx_math.h"
#include "nmx_rms.h"
#include "nmx_tree.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int AT_P = 32;         /* positions of a wave's tile: the depth of one P.V instruction */
constexpr int AT_MAXS = 256;     /* parts that the context is split into, at most */
constexpr float AT_LOG2E = 1.44269504f;

struct TreeAttn {
    int n, nh, nkv, hd, max_ctx;
    const float *q;
    const void *kc, *vc;
    const int32_t *pos, *parent;
    int pos_off;
    float scale;
    float *part;   /* [splits][n nh][hd] weighted values, 2^12 high */
    float4 *stat;  /* [splits][n nh]: maximum of the scores, of scores + value exponent (columns
                    * below 256), sum, maximum of scores + value exponent (columns from 256) */
    int splits, unit; /* a part is a whole number of units of positions */
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
    return (per + a.unit - 1) / a.unit * a.unit;
}

/* Exponent e with |x| < 2^e for the largest |x| of a row (0 for a row of zeros), clamped so that
 * 2^(12 - e) and 2^(e - 12) are finite; bits of anything not finite give the upper end. */
__device__ __forceinline__ int row_exp(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23) - 126;
    return amax == 0.0f ? 0 : e < -100 ? -100 : e > 128 ? 128 : e;
}
__device__ __forceinline__ float pow2f(int e) { /* -149 < e < 128 */
    return e > -127 ? __uint_as_float((uint32_t)(e + 127) << 23) : ldexpf(1.0f, e);
}

__device__ __forceinline__ float4v mfma16(half8 a, half8 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half4 lds_tr(const _Float16 *p) {
    typedef __attribute__((address_space(3))) short4v *lp;
    return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)p));
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

/* ---- the context ------------------------------------------------------------------------ */

/* A tile of PT positions in LDS: HDP binary16 values per position (a second plane of low parts for
 * fp32 caches), 16-byte chunks moved by an XOR so that the matrix operands' reads (16 positions of
 * one chunk for the keys, 4 positions of two chunks for the values) meet no bank twice; columns past
 * hd and positions past the part hold zeros. */
template <int HDP>
__device__ __forceinline__ int k_at(int p, int chunk) {
    return p * HDP + ((chunk ^ (p & 7)) << 3);
}
template <int HDP>
__device__ __forceinline__ int v_at(int p, int chunk) {
    return p * HDP + ((chunk ^ ((p & 3) << 1)) << 3);
}

/* 8 values of row R, columns col .. col + 7, as floats (int8: the codes) */
template <int KVT>
__device__ __forceinline__ void load8(const void *cache, size_t R, int hd, int col, uint4 (&raw)[2]) {
    if constexpr (KVT == KV_F32) {
        const uint4 *s = (const uint4 *)((const float *)cache + R * hd + col);
        raw[0] = s[0], raw[1] = s[1];
    } else if constexpr (KVT == KV_F16) {
        raw[0] = *(const uint4 *)((const unsigned short *)cache + R * hd + col);
    } else {
        const uint2 w = *(const uint2 *)((const int8_t *)cache + R * hd + col);
        raw[0].x = w.x, raw[0].y = w.y;
    }
}

/* Rows pt .. pt + PT - 1 of a cache (zeros from row p1 on), columns c0 .. c0 + W - 1, into a tile.
 * Keys: aux0 the factor of a row's scores. Values: aux0, aux1 exponent and fraction of a row's factor.
 * W / 8 lanes stage a row, 8 columns each. */
template <int W, int KVT, int PT, bool VALUES>
__device__ __forceinline__ void stage(const TreeAttn &a, size_t R0, int pt, int p1, int c0, _Float16 *dst,
                                      float *aux0, float *aux1) {
    constexpr int CH = W / 8, TURNS = PT * CH / 256, BATCH = TURNS < 8 ? TURNS : 8;
    static_assert(PT * CH % 256 == 0, "whole turns");
    const void *cache = VALUES ? a.vc : a.kc;
    const int tid = threadIdx.x, hd = a.hd;
    for (int t0 = 0; t0 < TURNS; t0 += BATCH) {
        uint4 raw[BATCH][2];
        float sc[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            const int f = (t0 + u) * 256 + tid, p = f / CH, col = c0 + f % CH * 8;
            raw[u][0] = raw[u][1] = uint4{0, 0, 0, 0};
            sc[u] = 0.0f;
            if (pt + p < p1 && col < hd) load8<KVT>(cache, R0 + pt + p, hd, col, raw[u]);
            if constexpr (KVT == KV_I8)
                if (pt + p < p1)
                    sc[u] = ((const float *)((const int8_t *)cache + (size_t)a.nkv * a.max_ctx * hd))[R0 + pt + p];
        }
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            const int f = (t0 + u) * 256 + tid, p = f / CH, chunk = f % CH;
            const int at = VALUES ? v_at<W>(p, chunk) : k_at<W>(p, chunk);
            if constexpr (KVT == KV_F16) {
                *(uint4 *)(dst + at) = raw[u][0];
            } else if constexpr (KVT == KV_I8) {
                half8 h;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    h[i] = (_Float16)(float)(int8_t)((i < 4 ? raw[u][0].x : raw[u][0].y) >> (8 * (i & 3)));
                *(half8 *)(dst + at) = h;
                if (chunk == 0) {
                    if constexpr (VALUES) {
                        const int e = row_exp(sc[u]);
                        aux0[p] = (float)e;
                        aux1[p] = sc[u] * pow2f(-e);
                    } else {
                        aux0[p] = sc[u];
                    }
                }
            } else {
                const float *x = (const float *)&raw[u][0];
                float am = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) am = fmaxf(am, fabsf(x[i]));
#pragma unroll
                for (int w = 1; w < CH; w <<= 1) am = fmaxf(am, __shfl_xor(am, w));
                const int e = row_exp(am);
                const float up = pow2f(12 - e);
                half8 h, r;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float v = x[i] * up;
                    h[i] = (_Float16)v;
                    r[i] = (_Float16)(v - (float)h[i]);
                }
                *(half8 *)(dst + at) = h;
                *(half8 *)(dst + PT * W + at) = r;
                if (chunk == 0) {
                    if constexpr (VALUES) aux0[p] = (float)(e - 12), aux1[p] = 1.0f;
                    else aux0[p] = pow2f(e - 12);
                }
            }
        }
    }
}

template <int HDP, int KVT, int PW>
__global__ __launch_bounds__(256) void attn_tree_ctx_k(TreeAttn a) {
    constexpr int PT = AT_P * PW, RW = 4 / PW, OD = HDP > 256 ? 256 : HDP, KS = HDP / 32, DT = OD / 16;
    constexpr int PL = KVT == KV_F32 ? 2 : 1; /* planes */
    extern __shared__ uint4 smem[];
    _Float16 *sk = (_Float16 *)smem, *sv = sk + PL * PT * HDP;
    float *kscale = (float *)(sv + PL * PT * OD), *vexp = kscale + PT, *vfrac = vexp + PT;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, gq = lane >> 4;
    const int s = blockIdx.x % a.splits, g = blockIdx.x / a.splits % a.nkv, mt = blockIdx.x / a.splits / a.nkv;
    const int d0 = blockIdx.y * OD; /* the output columns: of 512, half */
    const int len = ctx_len(a), per = part_len(a, len), hd = a.hd, rep = a.nh / a.nkv, rows = a.n * rep;
    const int p0 = s * per;
    if (per == 0 || p0 >= len) return;
    const int p1 = p0 + per < len ? p0 + per : len;
    const int pw = wave % PW, row0 = (mt * RW + wave / PW) * 16, row = row0 + c;
    const int hrow = (row / rep) * a.nh + g * rep + row % rep; /* (node, head) */
    const bool live = row < rows;
    const size_t R0 = (size_t)g * a.max_ctx;

    /* the query row of this lane's column, split; its factor goes to the scores */
    half8 qh[KS], ql[KS];
    float qfac;
    {
        const float *qp = a.q + (size_t)(live ? hrow : 0) * 2 * hd;
        float am = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int col = k * 32 + gq * 8;
            if (!live || col >= hd) continue;
            const float4 x = *(const float4 *)(qp + col), y = *(const float4 *)(qp + col + 4);
            am = fmaxf(am, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
            am = fmaxf(am, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
        }
        am = fmaxf(am, __shfl_xor(am, 16));
        am = fmaxf(am, __shfl_xor(am, 32));
        const int e = row_exp(am);
        const float up = pow2f(12 - e);
        qfac = pow2f(e - 12) * (a.scale * AT_LOG2E);
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int col = k * 32 + gq * 8;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
            if (live && col < hd) x = *(const float4 *)(qp + col), y = *(const float4 *)(qp + col + 4);
            const float z[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = z[i] * up;
                qh[k][i] = (_Float16)v;
                ql[k][i] = (_Float16)(v - (float)qh[k][i]);
            }
        }
    }

    /* this lane's operand addresses in its wave's part of a tile: the XORs leave two bases for the
     * keys (chunk 4 k + gq by k's parity) and four for the values (by d mod 4), the rest is constant */
    const int kp = pw * AT_P + c, vp = pw * AT_P + 4 * gq + (c >> 2);
    const _Float16 *kb[2], *vb[4];
#pragma unroll
    for (int i = 0; i < 2; i++) kb[i] = sk + k_at<HDP>(kp, 4 * i + gq) - 32 * i;
#pragma unroll
    for (int i = 0; i < 4; i++) vb[i] = sv + v_at<OD>(vp, 2 * i + ((c & 3) >> 1)) + 4 * (c & 1) - 16 * i;

    float4v o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, mo = -INFINITY, l = 0.0f;

    for (int pt = p0; pt < p1; pt += PT) {
        __syncthreads(); /* the last tile has been read */
        stage<HDP, KVT, PT, false>(a, R0, pt, p1, 0, sk, kscale, nullptr);
        stage<OD, KVT, PT, true>(a, R0, pt, p1, d0, sv, vexp, vfrac);
        __syncthreads();
        const int b = pw * AT_P; /* this wave's positions of the tile */
        if (pt + b >= p1) continue;
        /* scores: positions 16 i + 4 gq + j of the wave's tile against row c */
        float4v sc[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            sc[i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const _Float16 *at = kb[k & 1] + 16 * i * HDP + 32 * k;
                const half8 x = *(const half8 *)at;
                sc[i] = mfma16(x, qh[k], sc[i]);
                sc[i] = mfma16(x, ql[k], sc[i]);
                if constexpr (KVT == KV_F32) sc[i] = mfma16(*(const half8 *)(at + PT * HDP), qh[k], sc[i]);
            }
        }
        float x[8], xv[8], vf[8], mx = -INFINITY, mxo = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int p = b + 16 * (i >> 2) + 4 * gq + (i & 3);
            float y = sc[i >> 2][i & 3] * qfac;
            if constexpr (KVT != KV_F16) y *= kscale[p];
            x[i] = pt + p < p1 ? y : -INFINITY;
            mx = fmaxf(mx, x[i]);
            if constexpr (KVT != KV_F16) {
                xv[i] = x[i] + vexp[p];
                vf[i] = vfrac[p];
                mxo = fmaxf(mxo, xv[i]);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)));
        if constexpr (KVT != KV_F16) {
            mxo = fmaxf(mxo, __shfl_xor(mxo, 16));
            mxo = fmaxf(mo, fmaxf(mxo, __shfl_xor(mxo, 32)));
        } else {
            mxo = mx;
        }
        const float ref = mx == -INFINITY ? 0.0f : mx, refo = mxo == -INFINITY ? 0.0f : mxo;
        l *= exp2f(m - ref);
        const float down = exp2f(mo - refo);
        m = mx, mo = mxo;
        half8 ph, pl;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float w = exp2f(x[i] - ref);
            l += w;
            const float v = KVT == KV_F16 ? w * 4096.0f : exp2f(xv[i] - refo) * (vf[i] * 4096.0f);
            ph[i] = (_Float16)v;
            pl[i] = (_Float16)(v - (float)ph[i]);
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            o[d] *= down;
            /* values of column c of the tile's 16, positions in the weights' order */
            const _Float16 *at = vb[d & 3] + 16 * d;
            half8 y, z;
            const half4 y0 = lds_tr(at), y1 = lds_tr(at + 16 * OD);
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = y0[i], y[4 + i] = y1[i];
            o[d] = mfma16(y, ph, o[d]);
            o[d] = mfma16(y, pl, o[d]);
            if constexpr (KVT == KV_F32) {
                const half4 z0 = lds_tr(at + PT * OD), z1 = lds_tr(at + PT * OD + 16 * OD);
#pragma unroll
                for (int i = 0; i < 4; i++) z[i] = z0[i], z[4 + i] = z1[i];
                o[d] = mfma16(z, ph, o[d]);
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    if constexpr (PW > 1) { /* the waves' positions joined: wave pw 0 of a row group adds the others' */
        __syncthreads();
        float *xo = (float *)smem; /* [RW][PW - 1][64][DT 4 + 4] would not fit: one wave at a time */
        for (int w = 1; w < PW; w++) {
            float *my = xo + (size_t)(wave / PW) * 64 * (4 * DT + 4) + lane;
            if (pw == w) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) my[(4 * d + j) * 64] = o[d][j];
                my[4 * DT * 64] = m, my[(4 * DT + 1) * 64] = mo, my[(4 * DT + 2) * 64] = l;
            }
            __syncthreads();
            if (pw == 0) {
                const float m2 = my[4 * DT * 64], mo2 = my[(4 * DT + 1) * 64], l2 = my[(4 * DT + 2) * 64];
                const float mn = fmaxf(m, m2), mon = fmaxf(mo, mo2);
                const float ref = mn == -INFINITY ? 0.0f : mn, refo = mon == -INFINITY ? 0.0f : mon;
                const float f1 = exp2f(mo - refo), f2 = exp2f(mo2 - refo);
                l = l * exp2f(m - ref) + l2 * exp2f(m2 - ref);
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[d][j] = o[d][j] * f1 + my[(4 * d + j) * 64] * f2;
                m = mn, mo = mon;
            }
            __syncthreads();
        }
        if (pw) return;
    }
    if (!live) return;
    const size_t at = (size_t)s * a.n * a.nh + hrow;
#pragma unroll
    for (int d = 0; d < DT; d++)
        if (d0 + 16 * d < hd) *(float4v *)(a.part + at * hd + d0 + 16 * d + 4 * gq) = o[d];
    if (gq == 0) { /* the halves of 512 columns have value exponents of their own */
        if (d0) a.stat[at].w = mo;
        else a.stat[at].x = m, a.stat[at].y = mo, a.stat[at].z = l;
    }
}

/* ---- the node's ancestors, and the join ---------------------------------------------------- */
template <int KVT>
__global__ __launch_bounds__(256) void attn_tree_join_k(TreeAttn a) {
    constexpr int ND = 8; /* columns lane + 64 i, hd <= 512 */
    __shared__ float sc[64], red[8], acc_s[4][512], w_s[2][AT_MAXS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int hrow = blockIdx.x, t = hrow / a.nh, h = hrow % a.nh, hd = a.hd, nd = hd >> 6;
    const int g = h / (a.nh / a.nkv), rows = a.n * a.nh;
    const int len = ctx_len(a), per = part_len(a, len), parts = per ? (len + per - 1) / per : 0;
    const size_t R0 = (size_t)g * a.max_ctx;
    const float *qp = a.q + (size_t)hrow * 2 * hd;
    const float *ksc = KVT == KV_I8 ? (const float *)((const int8_t *)a.kc + (size_t)a.nkv * a.max_ctx * hd) : nullptr;
    const float *vsc = KVT == KV_I8 ? (const float *)((const int8_t *)a.vc + (size_t)a.nkv * a.max_ctx * hd) : nullptr;
    float q[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) q[i] = i < nd ? qp[lane + 64 * i] : 0.0f;
    float4 st = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f); /* thread = part */
    if (tid < parts) st = a.stat[(size_t)tid * rows + hrow];
    /* the ancestors' rows inside the cache */
    const int p0 = tree_slot0(a.pos, a.pos_off, a.max_ctx);
    unsigned long long set = __shfl(tree_ancestors(a.parent, a.n, nullptr), t);
    const int lo = p0 < 0 ? -p0 : 0, hi = a.max_ctx - p0; /* nodes lo .. hi - 1 have a slot */
    if (lo > 63 || hi <= 0) set = 0;
    else {
        set &= ~0ull << lo;
        if (hi < 64) set &= (1ull << hi) - 1;
    }
    auto value = [&](const void *cache, const float *scales, size_t R, int col) -> float {
        if constexpr (KVT == KV_F32) return ((const float *)cache)[R * hd + col];
        else if constexpr (KVT == KV_F16) return kv_half_value(((const unsigned short *)cache)[R * hd + col]);
        else return (float)((const int8_t *)cache)[R * hd + col] * scales[R];
    };
    const int na = __popcll(set);
    auto nth = [&](int i) { /* the i-th node of the set */
        unsigned long long x = set;
        for (int k = 0; k < i; k++) x &= x - 1;
        return __ffsll((long long)x) - 1;
    };
    float mt = -INFINITY;
    for (int i = wave; i < na; i += 4) {
        const size_t R = R0 + p0 + nth(i);
        float d = 0.0f;
#pragma unroll
        for (int k = 0; k < ND; k++)
            if (k < nd) d = __builtin_fmaf(q[k], value(a.kc, ksc, R, lane + 64 * k), d);
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) d += __shfl_xor(d, x);
        d *= a.scale * AT_LOG2E;
        if (lane == 0) sc[i] = d;
        mt = fmaxf(mt, d);
    }
    mt = fmaxf(mt, nmx_max_f32_wave(st.x));
    if (lane == 0) red[wave] = mt;
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), ref = m == -INFINITY ? 0.0f : m;
    __syncthreads();
    float l = st.z * exp2f(st.x - ref); /* a part's sum */
    if (tid < parts) {
        w_s[0][tid] = exp2f(st.y - ref - 12.0f);
        if (hd > 256) w_s[1][tid] = exp2f(st.w - ref - 12.0f);
    }
    __syncthreads();
    float acc[ND];
#pragma unroll
    for (int i = 0; i < ND; i++) acc[i] = 0.0f;
    for (int s = wave; s < parts; s += 4) {
        const float w0 = w_s[0][s], w1 = hd > 256 ? w_s[1][s] : 0.0f;
        const float *pp = a.part + ((size_t)s * rows + hrow) * hd + lane;
#pragma unroll
        for (int i = 0; i < ND; i++)
            if (i < nd) acc[i] = __builtin_fmaf(i < 4 ? w0 : w1, pp[64 * i], acc[i]);
    }
    float lt = 0.0f;
    for (int i = wave; i < na; i += 4) {
        const float w = exp2f(sc[i] - ref);
        const size_t R = R0 + p0 + nth(i);
        lt += w;
#pragma unroll
        for (int k = 0; k < ND; k++)
            if (k < nd) acc[k] = __builtin_fmaf(w, value(a.vc, vsc, R, lane + 64 * k), acc[k]);
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) l += __shfl_xor(l, x);
    if (lane == 0) red[4 + wave] = l + lt;
#pragma unroll
    for (int i = 0; i < ND; i++)
        if (i < nd) acc_s[wave][lane + 64 * i] = acc[i];
    __syncthreads();
    const float sum = (red[4] + red[5]) + (red[6] + red[7]);
    for (int d = tid; d < hd; d += 256) {
        float v = (acc_s[0][d] + acc_s[1][d]) + (acc_s[2][d] + acc_s[3][d]);
        v = sum > 0.0f || !(sum == sum) ? v / sum : 0.0f; /* no row at all in sight: 0 */
        v = v * nmx_sigmoid(qp[hd + d]);
        const int col = h * hd + d;
        a.o[(size_t)t * a.nh * hd + col] = v;
        if (a.aq) a8_block(v, col >> 5, t, a.n, a.aq, a.ad, a.afs); /* hd % 64 == 0: whole blocks */
    }
}

/* How the context is divided among workgroups: PW of a workgroup's 4 waves side by side over the
 * positions, the others over rows; `splits` parts. */
struct Plan {
    int hdp, pw, mtiles, splits, unit, halves;
    size_t part_bytes, bytes, lds;
};

/* positions side by side that a tile of the format fits the LDS with */
int max_pw(int hdp, int kv_dtype) {
    const int planes = kv_dtype == KV_F32 ? 2 : 1;
    const int fit = hdp > 256 ? 1 : (128 << 10) / (2 * planes * AT_P * hdp * 2);
    return fit >= 4 ? 4 : fit >= 2 ? 2 : 1;
}

Plan make_plan(int n, int nh, int nkv, int hd, int kv_dtype) {
    Plan p;
    p.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512;
    const int tiles = (n * (nh / nkv) + 15) / 16;
    const int most = max_pw(p.hdp, kv_dtype);
    p.pw = tiles == 1 ? most : tiles == 2 ? (most < 2 ? most : 2) : 1;
    const int rw = 4 / p.pw;
    p.mtiles = (tiles + rw - 1) / rw;
    const int target = p.pw == 4 ? 256 : 512;
    int s = target / (nkv * p.mtiles);
    p.splits = s < 1 ? 1 : s > AT_MAXS ? AT_MAXS : s;
    p.unit = AT_P * p.pw;
    const int planes = kv_dtype == KV_F32 ? 2 : 1;
    const int od = p.hdp > 256 ? 256 : p.hdp;
    p.halves = p.hdp / od;
    p.lds = (size_t)p.unit * (p.hdp + od) * 2 * planes + (size_t)3 * p.unit * 4;
    const size_t join = p.pw > 1 ? (size_t)rw * 64 * (od / 4 + 4) * 4 : 0;
    if (join > p.lds) p.lds = join;
    p.part_bytes = (size_t)p.splits * n * nh * hd * 4;
    p.bytes = p.part_bytes + (size_t)p.splits * n * nh * sizeof(float4);
    return p;
}

template <int HDP, int KVT, int PW>
int launch_ctx(nmx_ctx *ctx, const TreeAttn &a, const Plan &p) {
    static std::atomic<uint64_t> set;
    if (nmx_dyn_lds(ctx, (const void *)attn_tree_ctx_k<HDP, KVT, PW>, p.lds, set)) return -1;
    attn_tree_ctx_k<HDP, KVT, PW><<<dim3((unsigned)(p.splits * a.nkv * p.mtiles), (unsigned)p.halves), 256, p.lds,
                                        ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "attn_tree_ctx");
    return 0;
}

template <int HDP, int KVT>
int launch_pw(nmx_ctx *ctx, const TreeAttn &a, const Plan &p) {
    constexpr int planes = KVT == KV_F32 ? 2 : 1, fit = HDP > 256 ? 1 : (128 << 10) / (2 * planes * AT_P * HDP * 2);
    if constexpr (fit >= 4)
        if (p.pw == 4) return launch_ctx<HDP, KVT, 4>(ctx, a, p);
    if constexpr (fit >= 2)
        if (p.pw == 2) return launch_ctx<HDP, KVT, 2>(ctx, a, p);
    return launch_ctx<HDP, KVT, 1>(ctx, a, p);
}

template <int KVT>
int launch_tree(nmx_ctx *ctx, const TreeAttn &a, const Plan &p) {
    int rc = p.hdp == 64 ? launch_pw<64, KVT>(ctx, a, p) : p.hdp == 128 ? launch_pw<128, KVT>(ctx, a, p) :
             p.hdp == 256 ? launch_pw<256, KVT>(ctx, a, p) : launch_pw<512, KVT>(ctx, a, p);
    if (rc) return rc;
    attn_tree_join_k<KVT><<<(unsigned)(a.n * a.nh), 256, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "attn_tree_join");
    return 0;
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
    size_t most = 0;
    for (int t = KV_F32; t <= KV_I8; t++) {
        const size_t b = make_plan(n, nh, nkv, hd, t).bytes;
        most = b > most ? b : most;
    }
    return most;
}

int nmx_attn_tree(nmx_ctx *ctx, const nmx_attn_args *p, const int32_t *parent, void *work) {
    if (!ctx) return -1;
    if (tree_shape(ctx, p, parent, "nmx_attn_tree")) return -1;
    if (!p->o || !work || (p->a8.q && (!p->a8.d || !p->a8.fs))) return nmx_fail(ctx, "nmx_attn_tree: NULL argument");
    if ((uintptr_t)work % 16) return nmx_fail(ctx, "nmx_attn_tree: work not 16-byte aligned");
    const Plan pl = make_plan(p->n, p->nh, p->nkv, p->hd, p->kv_dtype);
    const size_t kb = nmx_kv_bytes(p->kv_dtype, p->nkv, p->max_ctx, p->hd), ob = (size_t)p->n * p->nh * p->hd * 4;
    if (nmx_overlap(work, pl.bytes, p->q, 2 * ob) || nmx_overlap(work, pl.bytes, p->kc, kb) ||
        nmx_overlap(work, pl.bytes, p->vc, kb) || nmx_overlap(work, pl.bytes, p->o, ob) ||
        nmx_overlap(p->o, ob, p->q, 2 * ob) || nmx_overlap(p->o, ob, p->kc, kb) || nmx_overlap(p->o, ob, p->vc, kb))
        return nmx_fail(ctx, "nmx_attn_tree: o, work and the inputs overlap");
    const TreeAttn a{p->n, p->nh, p->nkv, p->hd, p->max_ctx, p->q, p->kc, p->vc, p->pos, parent, p->pos_off,
                     p->scale, (float *)work, (float4 *)((char *)work + pl.part_bytes), pl.splits, pl.unit,
                     p->o, p->a8.q, p->a8.d, p->a8.fs};
    const nmx_on_device on(ctx);
    if (p->kv_dtype == KV_F16) return launch_tree<KV_F16>(ctx, a, pl);
    if (p->kv_dtype == KV_I8) return launch_tree<KV_I8>(ctx, a, pl);
    return launch_tree<KV_F32>(ctx, a, pl);
}

} /* extern "C" */
