/* Attention's inner product on the matrix cores, shared by the kernels over a tree of drafts
 * (nmx_attntree.hip) and over a batch of sequences (nmx_attnbatch.hip). Not part of the ABI.
 *
 * Tiles of 32 positions against 16 query rows a wave, every operand a pair of binary16 parts: 22 bits.
 * Scores are made transposed (positions x rows: keys are the first matrix operand, the query rows the
 * second), so a lane holds its own row's weights of 8 positions in exactly the order in which the
 * second product (values transposed x weights) wants its second operand: nothing moves between
 * lanes, and a row's running maximum, sum and rescale are its lane's own. */
#ifndef NMX_ATTNMX_H
#define NMX_ATTNMX_H

#include "nmx_attn.h"
#include "nmx_lanes.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int AT_P = 32;         /* positions of a wave's tile: the depth of one P.V instruction */

constexpr float AT_LOG2E = 1.44269504f;


/* Exponent e with |x| < 2^e for the largest |x| of a row, clamped so that 2^(12 - e) and 2^(e - 12) are
 * finite; bits of anything not finite give the upper end. A row of zeros has the lower end: of the value
 * rows of a tile the weights follow the largest, which a row of zeros must not be. */
__device__ __forceinline__ int row_exp(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23) - 126;
    return e < -100 ? -100 : e > 128 ? 128 : e;
}
__device__ __forceinline__ float pow2f(int e) { /* -149 < e < 128 */
    return e > -127 ? __uint_as_float((uint32_t)(e + 127) << 23) : ldexpf(1.0f, e);
}

/* lane and wave as the hardware knows them: no register kept for them, the wave's in a scalar */
__device__ __forceinline__ int lane_id() {
    return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

__device__ __forceinline__ float max_quarters(float v) {
    return nmx_over_quarters(v, [](float a, float b) { return fmaxf(a, b); });
}
/* the largest of W neighbouring lanes, in each of them (W a power of two) */
template <int W>
__device__ __forceinline__ float max_lanes(float v) {
    auto with = [&](int o) { v = fmaxf(v, __int_as_float(o)); };
    if (W >= 2) with(nmx_dpp<NMX_DPP_XOR1>(__float_as_int(v)));
    if (W >= 4) with(nmx_dpp<NMX_DPP_XOR2>(__float_as_int(v)));
    if (W >= 8) with(nmx_dpp<NMX_DPP_HALF_MIRROR>(__float_as_int(v)));
    if (W >= 16) with(nmx_dpp<NMX_DPP_MIRROR>(__float_as_int(v)));
    if (W == 64) return max_quarters(v);
    if (W == 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    return v;
}
/* the sum over a wave, in each lane */
__device__ __forceinline__ float sum_lanes(float v) {
    v += __int_as_float(nmx_dpp<NMX_DPP_XOR1>(__float_as_int(v)));
    v += __int_as_float(nmx_dpp<NMX_DPP_XOR2>(__float_as_int(v)));
    v += __int_as_float(nmx_dpp<NMX_DPP_HALF_MIRROR>(__float_as_int(v)));
    v += __int_as_float(nmx_dpp<NMX_DPP_MIRROR>(__float_as_int(v)));
    return nmx_sum_quarters(v);
}

__device__ __forceinline__ float4v mfma16(half8 a, half8 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half4 lds_tr(const _Float16 *p) {
    typedef __attribute__((address_space(3))) short4v *lp;
    return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(uintptr_t)p));
}

/* A row's 16-byte chunks of binary16 in LDS, moved by an XOR so that the operands' reads (16 positions of one chunk
 * for the keys, 8 positions of two chunks for the values, 256 bytes a cycle) meet no bank twice. */
template <int W>
__device__ __forceinline__ int k_at(int p, int chunk) {
    return p * W + ((chunk ^ (W >= 128 ? p & 15 : p >> 1 & 7)) << 3);
}
template <int W>
__device__ __forceinline__ int v_at(int p, int chunk) {
    return p * W + ((chunk ^ (W >= 128 ? p & 7 : p >> 1 & 3) << 1) << 3);
}

/* 8 values of a cache row as they lie in it */
template <int KVT>
struct Raw8 {
    uint4 a, b;
};
template <>
struct Raw8<KV_F16> {
    uint4 a;
};
template <>
struct Raw8<KV_I8> {
    uint2 a;
};

__device__ __forceinline__ half8 codes8(uint2 w) {
    half8 h;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (_Float16)(float)(int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    return h;
}
__device__ __forceinline__ void floats8(const Raw8<KV_F32> &r, float (&x)[8]) {
    x[0] = __uint_as_float(r.a.x), x[1] = __uint_as_float(r.a.y), x[2] = __uint_as_float(r.a.z), x[3] = __uint_as_float(r.a.w);
    x[4] = __uint_as_float(r.b.x), x[5] = __uint_as_float(r.b.y), x[6] = __uint_as_float(r.b.z), x[7] = __uint_as_float(r.b.w);
}
__device__ __forceinline__ float amax8(const Raw8<KV_F32> &r) {
    float x[8];
    floats8(r, x);
    return fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))),
                 fmaxf(fmaxf(fabsf(x[4]), fabsf(x[5])), fmaxf(fabsf(x[6]), fabsf(x[7]))));
}
/* x up as a binary16 and the binary16 rest: 2^-22 of x is left */
__device__ __forceinline__ void split8(const float (&x)[8], float up, half8 &h, half8 &r) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = x[i] * up;
        h[i] = (_Float16)v;
        r[i] = (_Float16)__builtin_fmaf((float)h[i], -1.0f, v);
    }
}
/* two weights, the first part towards zero in one instruction: 2^-21 is left */
typedef __fp16 fp16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split2(float a, float b, half8 &h, half8 &r, int i) {
    const fp16x2 p = __builtin_amdgcn_cvt_pkrtz(a, b);
    h[i] = (_Float16)p.x, h[i + 1] = (_Float16)p.y;
    r[i] = (_Float16)__builtin_fmaf((float)h[i], -1.0f, a), r[i + 1] = (_Float16)__builtin_fmaf((float)h[i + 1], -1.0f, b);
}

/* Lane c of 16 (quarter gq) takes its query row's chunks 4 k + gq: requested first, split when the
 * cache's first rows have been requested too. Columns past hd are zeros. */
template <int KS>
struct QueryRow {
    const float *qp;
    bool live;
    int hd, gq;
    float4 x[KS][2];
    __device__ __forceinline__ void get(int k) {
        const int col = k * 32 + gq * 8, at = live && col < hd ? col : 0; /* qp is in bounds for every lane */
        x[k][0] = *(const float4 *)(qp + at), x[k][1] = *(const float4 *)(qp + at + 4);
    }
    __device__ __forceinline__ QueryRow(const float *qp, bool live, int hd, int gq) : qp(qp), live(live), hd(hd), gq(gq) {
#pragma unroll
        for (int k = 0; k < KS; k++) get(k);
    }
    /* the parts; the result is the factor that turns a product of parts into a score in powers of two */
    __device__ __forceinline__ float split(float scale, half8 (&qh)[KS], half8 (&ql)[KS]) {
        float am = 0.0f;
        auto in = [&](int k) { return live && k * 32 + gq * 8 < hd; };
#pragma unroll
        for (int k = 0; k < KS; k++) {
            float4(&y)[2] = x[k];
            float b = fmaxf(fmaxf(fmaxf(fabsf(y[0].x), fabsf(y[0].y)), fmaxf(fabsf(y[0].z), fabsf(y[0].w))),
                            fmaxf(fmaxf(fabsf(y[1].x), fabsf(y[1].y)), fmaxf(fabsf(y[1].z), fabsf(y[1].w))));
            am = fmaxf(am, in(k) ? b : 0.0f);
        }
        am = max_quarters(am);
        const int e = row_exp(am);
        const float up = pow2f(12 - e);
#pragma unroll
        for (int k = 0; k < KS; k++) {
            float4(&y)[2] = x[k];
            const float z[8] = {y[0].x, y[0].y, y[0].z, y[0].w, y[1].x, y[1].y, y[1].z, y[1].w};
            split8(z, up, qh[k], ql[k]);
            if (!in(k)) qh[k] = ql[k] = half8{0, 0, 0, 0, 0, 0, 0, 0};
        }
        return pow2f(e - 12) * (scale * AT_LOG2E);
    }
};

/* A row's running state: weights are 2^(score - m); a value's factor 2^(its exponent - ve), where ve
 * grows so that no weight times value leaves binary16; l is this lane's share of the sum, lc what its
 * roundings have added to it (a part may have a thousand tiles, and equal weights round alike). */
template <int DT>
struct Running {
    float4v o[DT];
    float m = -INFINITY, l = 0.0f, lc = 0.0f;
    int ve = -1000;
    __device__ __forceinline__ Running() {
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

/* One tile of 32 positions: x[8] the lane's scores (-inf: no position), e / f their values' exponents
 * and fractions (int8 and fp32 caches), vb the value operand's bases, OD columns, `plane` halves to
 * the low parts. */
template <int OD, int KVT>
__device__ __forceinline__ void add_tile(Running<OD / 16> &r, const float (&x)[8], const int (&e)[8], const float (&f)[8],
                                         const _Float16 *const (&vb)[8], int plane) {
    constexpr int DT = OD / 16;
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) mx = fmaxf(mx, x[i]);
    mx = fmaxf(r.m, max_quarters(mx));
    const float ref = mx == -INFINITY ? 0.0f : mx;
    int ve = 0;
    if constexpr (KVT != KV_F16) { /* the largest of score + exponent, above the largest score, rounded up */
        float t = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) t = fmaxf(t, (x[i] - ref) + (float)e[i]);
        t = max_quarters(t);
        /* the old values' bound moves with the maximum */
        t = fmaxf(t, (r.m - ref) + (float)r.ve);
        ve = (int)ceilf(fmaxf(t, -500.0f));
    }
    if (__any(mx > r.m || ve != (KVT == KV_F16 ? 0 : r.ve))) {
        const float down = __builtin_amdgcn_exp2f(r.m - ref);
        r.l *= down, r.lc *= down;
        const float dv = KVT == KV_F16 ? down : ldexpf(down, r.ve - ve < -300 ? -300 : r.ve - ve);
#pragma unroll
        for (int d = 0; d < DT; d++) r.o[d] *= dv;
        r.m = mx, r.ve = ve;
    }
    half8 ph, pl;
    float wv[8], sum;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float w = __builtin_amdgcn_exp2f(x[i] - ref);
        sum = i ? sum + w : w;
        if constexpr (KVT == KV_F16) wv[i] = w * 4096.0f;
        else wv[i] = ldexpf(w * f[i], e[i] - ve + 12);
    }
    const float more = sum - r.lc, all = r.l + more;
    r.lc = (all - r.l) - more, r.l = all;
#pragma unroll
    for (int i = 0; i < 8; i += 2) split2(wv[i], wv[i + 1], ph, pl, i);
    /* values of column c of the tile's 16, positions in the weights' order: those of the next G column tiles are on
     * their way while the products of these run */
    constexpr int G = KVT == KV_F32 ? 1 : 2; /* fp32: no registers for more */
    half8 y[2][G], z[2][G];
    auto read = [&](int d, half8 &to, int at_plane) {
        const _Float16 *at = vb[d & 7] + 16 * d + at_plane;
        const half4 y0 = lds_tr(at), y1 = lds_tr(at + 16 * OD);
#pragma unroll
        for (int i = 0; i < 4; i++) to[i] = y0[i], to[4 + i] = y1[i];
    };
    auto ask = [&](int d0, int b) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            read(d0 + g, y[b][g], 0);
            if constexpr (KVT == KV_F32) read(d0 + g, z[b][g], plane);
        }
    };
    ask(0, 0);
#pragma unroll
    for (int d = 0; d < DT; d += G) {
        const int b = d / G & 1;
        if (d + G < DT) ask(d + G, b ^ 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < G; g++) r.o[d + g] = mfma16(y[b][g], ph, r.o[d + g]);
#pragma unroll
        for (int g = 0; g < G; g++) r.o[d + g] = mfma16(y[b][g], pl, r.o[d + g]);
        if constexpr (KVT == KV_F32)
#pragma unroll
            for (int g = 0; g < G; g++) r.o[d + g] = mfma16(z[b][g], ph, r.o[d + g]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

/* 8 waves of 16 rows (4 where a row has 512 columns) share a tile of 32 positions. The tile after the next one is on its
 * way into registers while the matrix cores work on the current one, with two tiles in LDS (one for
 * 512 columns of fp32, which have neither the registers nor the room). Half of the waves, one on each SIMD, bring the next
 * tile to LDS before they work on the current one, the others afterwards, so that a SIMD's two waves need
 * its matrix core and its vector unit at different times. A tile of 128 rows, 256 columns, binary16 / int8 / fp32 takes
 * 1.8 / 2.2 / 4.2 us (0.85 / 0.85 / 1.3 on the matrix cores alone); with all waves in step 1.9 / 2.3 / 4.8, with each
 * operand waited for by itself 2.1 / 2.8 / 5.0. The same kernel serves few rows,
 * whose waves without rows only bring tiles: waves with tiles of their own, each staging for itself, took
 * as long over 20000 binary16 positions and much longer otherwise (5 nodes over 30000 fp32 positions 86
 * against 41 us, 2 over 16 int8 17 against 12). */
template <int HDP>
constexpr int ctx_waves() {
    return HDP > 256 ? 4 : 8;
}
template <int HDP, int KVT>
constexpr int ctx_bufs() {
    return HDP > 256 && KVT == KV_F32 ? 1 : 2;
}
/* LDS of the tiles in bytes */
template <int HDP, int KVT>
constexpr int ctx_lds() {
    constexpr int od = HDP > 256 ? 256 : HDP, planes = KVT == KV_F32 ? 2 : 1;
    return ctx_bufs<HDP, KVT>() * (planes * AT_P * (HDP + od) * 2 + 3 * AT_P * 4);
}

/* A wave's 16 query rows (qr; lane c its own) over the positions [p0, p1), added to r: a row sees those below
 * its lane's lim. All waves of the workgroup come here together (busy: this one has rows) and share the
 * tiles in smem: kh and vh bring the cache's rows (page_of: where a position's row is, asked for a tile
 * ahead of load8 and scale), d0 is the first of the OD output columns. */
template <int HDP, int KVT, typename Rows>
__device__ __forceinline__ void attend_tiles(Running<(HDP > 256 ? 256 : HDP) / 16> &r, QueryRow<HDP / 32> &qr, float scale,
                                             const Rows &kh, const Rows &vh, int p0, int p1, int lim, int d0, bool busy,
                                             uint4 *smem) {
    constexpr int TH = 64 * ctx_waves<HDP>();
    constexpr int OD = HDP > 256 ? 256 : HDP, KS = HDP / 32, NB = ctx_bufs<HDP, KVT>();
    constexpr int PL = KVT == KV_F32 ? 2 : 1; /* planes */
    constexpr int KC = HDP / 8, VC = OD / 8;  /* lanes that stage a row, 8 columns each */
    constexpr int KU = AT_P * KC / TH ? AT_P * KC / TH : 1, VU = AT_P * VC / TH ? AT_P * VC / TH : 1;
    constexpr int TILE = PL * AT_P * (HDP + OD);
    _Float16 *tiles = (_Float16 *)smem;
    float *aux = (float *)(tiles + NB * TILE); /* per tile: the keys' factors, the values' exponents and fractions */
    const int lane = lane_id(), tid = 64 * wave_id() + lane, c = lane & 15, gq = lane >> 4, hd = kh.hd;
    /* staging: columns and rows past the end repeat ones inside (finite, and their weight is 0) */
    Raw8<KVT> rk[KU], rv[VU];
    float sk[KU], sv[VU];
    int pk[KU], pv[VU]; /* the pages of the next tile's rows, asked for a tile ahead of the rows */
    auto ask = [&](int pt) {
#pragma unroll
        for (int u = 0; u < KU; u++) {
            const int p = (u * TH + tid) / KC & (AT_P - 1);
            pk[u] = kh.page_of(pt + p < p1 ? pt + p : p1 - 1);
        }
#pragma unroll
        for (int u = 0; u < VU && HDP > 256; u++) {
            const int p = (u * TH + tid) / VC & (AT_P - 1);
            pv[u] = vh.page_of(pt + p < p1 ? pt + p : p1 - 1);
        }
    };
    auto fetch_k = [&](int pt) {
#pragma unroll
        for (int u = 0; u < KU; u++) {
            const int f = u * TH + tid, p = f / KC & (AT_P - 1), col = f % KC * 8;
            const int at = pt + p < p1 ? pt + p : p1 - 1;
            const auto row = kh.where(pk[u], at, col < hd ? col : 0);
            rk[u] = kh.load8(row);
            if (HDP <= 256) rv[u] = vh.load8(row), sv[u] = vh.scale(pk[u], at);
            sk[u] = kh.scale(pk[u], at);
        }
    };
    auto fetch_v = [&](int pt) {
#pragma unroll
        for (int u = 0; u < VU && HDP > 256; u++) {
            const int f = u * TH + tid, p = f / VC & (AT_P - 1), col = d0 + f % VC * 8;
            const int at = pt + p < p1 ? pt + p : p1 - 1;
            rv[u] = vh.load8(vh.where(pv[u], at, col < hd ? col : 0));
            sv[u] = vh.scale(pv[u], at);
        }
    };
    auto put_k = [&](int buf) {
        _Float16 *tk = tiles + buf * TILE;
        float *kf = aux + buf * 3 * AT_P;
#pragma unroll
        for (int u = 0; u < KU; u++) {
            const int f = u * TH + tid, p = f / KC, ch = f % KC, at = k_at<HDP>(p, ch);
            if (AT_P * KC < TH && p >= AT_P) continue;
            if constexpr (KVT == KV_F16) {
                *(uint4 *)(tk + at) = rk[u].a;
            } else if constexpr (KVT == KV_I8) {
                *(half8 *)(tk + at) = codes8(rk[u].a);
                if (ch == 0) kf[p] = sk[u];
            } else {
                float x[8];
                const int e = row_exp(max_lanes<KC>(amax8(rk[u])));
                half8 h, r;
                floats8(rk[u], x);
                split8(x, pow2f(12 - e), h, r);
                *(half8 *)(tk + at) = h;
                *(half8 *)(tk + AT_P * HDP + at) = r;
                if (ch == 0) kf[p] = pow2f(e - 12);
            }
        }
    };
    auto put_v = [&](int buf) {
        _Float16 *tv = tiles + buf * TILE + PL * AT_P * HDP;
        float *vf = aux + buf * 3 * AT_P + AT_P;
        int *ve = (int *)(vf + AT_P);
#pragma unroll
        for (int u = 0; u < VU; u++) {
            const int f = u * TH + tid, p = f / VC, ch = f % VC, at = v_at<OD>(p, ch);
            if (AT_P * VC < TH && p >= AT_P) continue;
            if constexpr (KVT == KV_F16) {
                *(uint4 *)(tv + at) = rv[u].a;
            } else if constexpr (KVT == KV_I8) {
                *(half8 *)(tv + at) = codes8(rv[u].a);
                if (ch == 0) {
                    const int e = row_exp(sv[u]);
                    ve[p] = e, vf[p] = sv[u] * pow2f(-e);
                }
            } else {
                float x[8];
                const int e = row_exp(max_lanes<VC>(amax8(rv[u])));
                half8 h, r;
                floats8(rv[u], x);
                split8(x, pow2f(12 - e), h, r);
                *(half8 *)(tv + at) = h;
                *(half8 *)(tv + AT_P * OD + at) = r;
                if (ch == 0) ve[p] = e - 12, vf[p] = 1.0f;
            }
        }
    };
    ask(p0);
    if constexpr (NB == 2) fetch_k(p0), fetch_v(p0), ask(p0 + AT_P);
    half8 qh[KS], ql[KS];
    const float qfac = qr.split(scale, qh, ql);
    if (NB == 2) {
        put_k(0), put_v(0);
        fetch_k(p0 + AT_P), fetch_v(p0 + AT_P), ask(p0 + 2 * AT_P);
    }
    /* this lane's operand addresses in a tile: the XORs leave four bases for the keys (chunk 4 k + gq by
     * k mod 4) and eight for the values (by d mod 8), the rest is constant; the second half of them are the first with
     * the bit of 8 chunks, which the lane's position flips or not */
    const int vp = 4 * gq + (c >> 2), kflip = 128 * (c >> 3), vflip = 128 * (vp >> 2 & 1);
    int kb[2], vo[4];
#pragma unroll
    for (int i = 0; i < 2; i++) kb[i] = k_at<HDP>(c, 4 * i + gq) - 32 * i;
#pragma unroll
    for (int i = 0; i < 4; i++) vo[i] = PL * AT_P * HDP + v_at<OD>(vp, 2 * i + ((c & 3) >> 1)) + 4 * (c & 1) - 16 * i;
    auto stage = [&](int pt, int to) {
        if (NB == 2 && pt + AT_P < p1) {
            put_k(to), put_v(to);
            if (pt + 2 * AT_P < p1) fetch_k(pt + 2 * AT_P), fetch_v(pt + 2 * AT_P), ask(pt + 3 * AT_P);
        }
    };
    const bool late = wave_id() < ctx_waves<HDP>() / 2;
    int buf = 0;
    for (int pt = p0; pt < p1; pt += AT_P) {
        if (NB == 1) { /* one tile: no registers to hold the next one either */
            __syncthreads();
            fetch_k(pt), put_k(0);
            fetch_v(pt), put_v(0);
            ask(pt + AT_P);
        }
        __syncthreads();
        if (!late) stage(pt, buf ^ 1);
        if (busy) {
            const _Float16 *tk = tiles + buf * TILE;
            const float *kf = aux + buf * 3 * AT_P, *vf = kf + AT_P;
            const int *ve = (const int *)(vf + AT_P);
            float4v sc[2];
#pragma unroll
            for (int i = 0; i < 2; i++) sc[i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            /* the keys of the next 32 columns are on their way while the products of these run */
            half8 key[2][2], low[2]; /* fp32: no registers for the next low parts */
            auto ask_keys = [&](int k) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const _Float16 *at = (k & 2 ? tk - kflip : tk) + kb[k & 1] + 16 * i * HDP + 32 * k;
                    key[k & 1][i] = *(const half8 *)at;
                }
            };
            auto ask_low = [&](int k) {
#pragma unroll
                for (int i = 0; i < 2; i++)
                    low[i] = *(const half8 *)((k & 2 ? tk - kflip : tk) + kb[k & 1] + (16 * i + AT_P) * HDP + 32 * k);
            };
            ask_keys(0);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                if (KVT == KV_F32) ask_low(k);
                if (k + 1 < KS) ask_keys(k + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 2; i++) sc[i] = mfma16(key[k & 1][i], qh[k], sc[i]);
#pragma unroll
                for (int i = 0; i < 2; i++) sc[i] = mfma16(key[k & 1][i], ql[k], sc[i]);
                if constexpr (KVT == KV_F32)
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[i] = mfma16(low[i], qh[k], sc[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
            const int left = lim - pt - 4 * gq;
            float x[8], f[8];
            int e[8];
#pragma unroll
            for (int h = 0; h < 2; h++) { /* positions 16 h + 4 gq + j, seen below left */
                const int p = 16 * h + 4 * gq;
                float4v k4{1.0f, 1.0f, 1.0f, 1.0f}, f4 = k4;
                int4 e4 = make_int4(0, 0, 0, 0);
                if constexpr (KVT != KV_F16) k4 = *(const float4v *)(kf + p), f4 = *(const float4v *)(vf + p), e4 = *(const int4 *)(ve + p);
                const int ej[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float y = sc[h][j] * qfac;
                    if constexpr (KVT != KV_F16) y *= k4[j];
                    x[4 * h + j] = j < left - 16 * h ? y : -INFINITY, f[4 * h + j] = f4[j], e[4 * h + j] = ej[j];
                }
            }
            const _Float16 *const tf = tk - vflip, *const vb[8] = {tk + vo[0], tk + vo[1], tk + vo[2], tk + vo[3],
                                                                   tf + vo[0], tf + vo[1], tf + vo[2], tf + vo[3]};
            add_tile<OD, KVT>(r, x, e, f, vb, AT_P * OD);
        }
        if (late) stage(pt, buf ^ 1);
        if (NB == 2) buf ^= 1;
    }
}

} // namespace

#endif
