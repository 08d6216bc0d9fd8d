/* Low-rank adapters of many requests (include/nmx.h nmx_lora): y += scale B (A x), each row with its own
 * adapter, for the matrices that share x.
 *
 * Rows with one adapter are taken together, 16 at a time, so that A and B are read once for them: the first
 * of every 16 (counted over the rows by ballots) is the leader of its tile, and a workgroup whose row leads
 * none ends. lora_down_k: 16 ranks of A x, the columns shared out over the waves; lora_up_k: 16 rows of B at a
 * time, added to y. Products are fp32 matrix instructions (16 x 16 x 4): a lane takes 8 neighbouring
 * columns of a weight row and of a row of x, the sum over the 32 columns of a wave's step has no order to keep, so
 * weights go from 16-byte loads to the operand without passing through LDS. */
#include "nmx_internal.h"
#include "nmx_attn.h"
#include "nmx_batch.h"
#include "nmx_lanes.h"

namespace {

typedef float float4v __attribute__((ext_vector_type(4)));

enum { W_F32 = 0, W_F16 = 1, W_BF16 = 2 };
constexpr int LD_WAVES = 8; /* of lora_down_k */
constexpr int LU_WAVES = 4; /* of lora_up_k, 16 LU_EACH output rows each */
constexpr int LU_EACH = 4;

struct Lora {
    int n, cols, x_stride, count;
    const float *x;
    int adapters, rank;
    const int32_t *adapter, *ranks;
    const float *scale;
    float *low; /* [count][n][rank16]: A x */
    int rank16;
    const void *A[NMX_MAX_SEGS], *B[NMX_MAX_SEGS];
    int rows[NMX_MAX_SEGS], y_stride[NMX_MAX_SEGS];
    float *Y[NMX_MAX_SEGS];
    int first[NMX_MAX_SEGS + 1]; /* of lora_up_k's workgroups */
};

/* The tile that row t leads: its adapter (-1: t leads none) and this lane's row (lane & 15; rows past the last one
 * repeat t, live false). Every lane of the wave active. */
struct Tile {
    int adapter, row, rank;
    bool live;
};
__device__ __forceinline__ Tile lead(const Lora &a, int t) {
    const int lane = threadIdx.x & 63, c = lane & 15;
    int id[NMX_CHUNK_ROWS / 64];
    const int mine = a.adapter[t];
#pragma unroll
    for (int u = 0; u < NMX_CHUNK_ROWS / 64; u++) id[u] = 64 * u < a.n ? a.adapter[64 * u + lane < a.n ? 64 * u + lane : 0] : -1;
    Tile r{-1, t, 0, false};
    if (mine < 0 || mine >= a.adapters) return r;
    int before = 0, at = 0;
#pragma unroll
    for (int u = 0; u < NMX_CHUNK_ROWS / 64; u++) {
        unsigned long long m = __ballot(64 * u + lane < a.n && id[u] == mine);
        const int split = t - 64 * u; /* rows of this 64 before t */
        const unsigned long long early = split >= 64 ? ~0ull : split > 0 ? (1ull << split) - 1 : 0;
        before += __popcll(m & early);
        m &= ~early;
        /* the c-th of the rows from t on */
        const int have = __popcll(m);
        if (c >= at && c < at + have) {
            unsigned long long k = m;
            for (int i = at; i < c; i++) k &= k - 1;
            r.row = 64 * u + __ffsll((long long)k) - 1, r.live = true;
        }
        at += have;
    }
    if (before % 16) return r;
    r.adapter = mine;
    const int rk = a.ranks ? a.ranks[mine] : a.rank;
    r.rank = rk < 0 ? 0 : rk < a.rank ? rk : a.rank;
    return r;
}

/* 8 weights as they lie in memory, widened */
template <int WT>
struct W8 {
    uint4 v[WT == W_F32 ? 2 : 1];
    __device__ __forceinline__ float at(int i) const {
        if constexpr (WT == W_F32) {
            const uint4 &q = v[i >> 2];
            return __uint_as_float((i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w);
        } else {
            const uint32_t w = i < 2 ? v[0].x : i < 4 ? v[0].y : i < 6 ? v[0].z : v[0].w;
            if constexpr (WT == W_F16) return kv_half_value(i & 1 ? w >> 16 : w);
            return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
        }
    }
    __device__ __forceinline__ void load(const char *p) {
        v[0] = *(const uint4 *)p;
        if constexpr (WT == W_F32) v[1] = *(const uint4 *)(p + 16);
    }
};
template <int WT>
__device__ __forceinline__ float one_weight(const void *p, size_t i) {
    if constexpr (WT == W_F32) return ((const float *)p)[i];
    const uint32_t w = ((const unsigned short *)p)[i];
    if constexpr (WT == W_F16) return kv_half_value(w);
    return __uint_as_float(w << 16);
}
__device__ __forceinline__ float4v mfma4(float a, float b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

/* Workgroup: a row, blockIdx.y 16 ranks of a matrix. */
template <int WT>
__global__ __launch_bounds__(64 * LD_WAVES) void lora_down_k(Lora a) {
    __shared__ float4 sum_s[LD_WAVES][64];
    constexpr int SIZE = WT == W_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c = lane & 15, k = lane >> 4;
    const Tile t = lead(a, blockIdx.x);
    if (t.adapter < 0) return; /* uniform over the workgroup */
    const int blocks = a.rank16 / 16, s = blockIdx.y / blocks, r0 = blockIdx.y % blocks * 16;
    const int r = r0 + c < a.rank ? r0 + c : a.rank - 1;
    const char *wp = (const char *)a.A[s] + (((size_t)t.adapter * a.rank + r) * a.cols + 8 * k) * SIZE;
    const float *xp = a.x + (size_t)t.row * a.x_stride + 8 * k;
    float4v acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    constexpr int U = 4; /* steps of 32 columns requested at once */
    for (int c0 = wave * 32; c0 < a.cols; c0 += 32 * LD_WAVES * U) {
        W8<WT> w[U];
        float4 x[U][2];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = c0 + 32 * LD_WAVES * u, in = at < a.cols ? at : c0;
            w[u].load(wp + (size_t)in * SIZE);
            x[u][0] = *(const float4 *)(xp + in), x[u][1] = *(const float4 *)(xp + in + 4);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (c0 + 32 * LD_WAVES * u >= a.cols) break;
            const float y[8] = {x[u][0].x, x[u][0].y, x[u][0].z, x[u][0].w, x[u][1].x, x[u][1].y, x[u][1].z, x[u][1].w};
#pragma unroll
            for (int i = 0; i < 8; i++) acc[i & 1] = mfma4(w[u].at(i), y[i], acc[i & 1]);
        }
    }
    const float4v mine = acc[0] + acc[1];
    sum_s[wave][lane] = make_float4(mine[0], mine[1], mine[2], mine[3]);
    __syncthreads();
    if (wave) return;
    float4 v = sum_s[0][lane];
#pragma unroll
    for (int w = 1; w < LD_WAVES; w++) {
        const float4 y = sum_s[w][lane];
        v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
    }
    if (!t.live) return;
    /* ranks 4 k .. 4 k + 3 of row c; those that the adapter lacks are zeros, whatever A holds there */
    const int q = r0 + 4 * k;
    if (q >= t.rank) v.x = 0.0f;
    if (q + 1 >= t.rank) v.y = 0.0f;
    if (q + 2 >= t.rank) v.z = 0.0f;
    if (q + 3 >= t.rank) v.w = 0.0f;
    *(float4 *)(a.low + ((size_t)s * a.n + t.row) * a.rank16 + q) = v;
}

/* Workgroup: a row, blockIdx.y a run of output rows of a matrix. VEC: rows of B are 16-byte aligned. */
template <int WT, bool VEC>
__global__ __launch_bounds__(64 * LU_WAVES) void lora_up_k(Lora a) {
    constexpr int SIZE = WT == W_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c = lane & 15, k = lane >> 4;
    const Tile t = lead(a, blockIdx.x);
    if (t.adapter < 0) return;
    int s = 0;
    while (s + 1 < a.count && (int)blockIdx.y >= a.first[s + 1]) s++;
    const int rows = a.rows[s], o0 = (((int)blockIdx.y - a.first[s]) * LU_WAVES + wave) * 16 * LU_EACH;
    if (o0 >= rows) return;
    const float scale = a.scale[t.adapter];
    const float *lp = a.low + ((size_t)s * a.n + t.row) * a.rank16 + 8 * k;
    float4v acc[LU_EACH];
#pragma unroll
    for (int e = 0; e < LU_EACH; e++) acc[e] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    for (int q = 0; q < t.rank; q += 32) {
        const int at = q + 8 * k; /* this lane's ranks */
        float4 y0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y1 = y0;
        if (at < a.rank16) y0 = *(const float4 *)(lp + q), y1 = *(const float4 *)(lp + q + 4);
        const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
        float w[LU_EACH][8];
#pragma unroll
        for (int e = 0; e < LU_EACH; e++) {
            const int o = o0 + 16 * e + c < rows ? o0 + 16 * e + c : rows - 1;
            const size_t row = ((size_t)t.adapter * rows + o) * a.rank;
            if constexpr (VEC) {
                W8<WT> v;
                v.load((const char *)a.B[s] + (row + (at < a.rank ? at : 0)) * SIZE);
#pragma unroll
                for (int i = 0; i < 8; i++) w[e][i] = at + i < t.rank ? v.at(i) : 0.0f;
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float v = one_weight<WT>(a.B[s], row + (at + i < a.rank ? at + i : 0));
                    w[e][i] = at + i < t.rank ? v : 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < LU_EACH; e++) acc[e] = mfma4(w[e][i], y[i], acc[e]);
    }
    if (!t.live) return;
    float *yp = a.Y[s] + (size_t)t.row * a.y_stride[s];
#pragma unroll
    for (int e = 0; e < LU_EACH; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int o = o0 + 16 * e + 4 * k + i;
            if (o < rows) yp[o] = __builtin_fmaf(acc[e][i], scale, yp[o]);
        }
}

template <int WT>
int launch(nmx_ctx *ctx, const Lora &a) {
    lora_down_k<WT><<<dim3((unsigned)a.n, (unsigned)(a.count * a.rank16 / 16)), 64 * LD_WAVES, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "lora_down");
    const dim3 grid((unsigned)a.n, (unsigned)a.first[a.count]);
    if (a.rank % 8 == 0) lora_up_k<WT, true><<<grid, 64 * LU_WAVES, 0, ctx->stream>>>(a);
    else lora_up_k<WT, false><<<grid, 64 * LU_WAVES, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "lora_up");
    return 0;
}

} // namespace

extern "C" {

size_t nmx_lora_work_bytes(int n, int count, int rank) {
    if (n < 1 || n > NMX_CHUNK_ROWS || count < 1 || count > NMX_MAX_SEGS || rank < 1 || rank > 256) return 0;
    return (size_t)count * n * ((rank + 15) / 16 * 16) * 4;
}

int nmx_lora(nmx_ctx *ctx, const nmx_lora_args *p, void *work) {
    if (!ctx) return -1;
    if (!p) return nmx_fail(ctx, "nmx_lora: NULL argument");
    const size_t wb = nmx_lora_work_bytes(p->n, p->count, p->rank);
    if (!wb || p->cols < 32 || p->cols > 32768 || p->cols % 32 || p->adapters < 1 || p->adapters > (1 << 20) ||
        p->w_dtype < W_F32 || p->w_dtype > W_BF16)
        return nmx_fail(ctx, "nmx_lora: n=%d count=%d rank=%d cols=%d adapters=%d w_dtype=%d", p->n, p->count, p->rank, p->cols,
                        p->adapters, p->w_dtype);
    if (!p->x || !p->adapter || !p->scale || !work) return nmx_fail(ctx, "nmx_lora: NULL argument");
    if (p->x_stride < p->cols || p->x_stride % 4 || (uintptr_t)p->x % 16 || (uintptr_t)work % 16)
        return nmx_fail(ctx, "nmx_lora: x_stride=%d, or x or work not 16-byte aligned", p->x_stride);
    Lora a{};
    const size_t N = (size_t)p->n, ws = p->w_dtype == W_F32 ? 4 : 2, mb = (size_t)p->adapters * p->rank * ws;
    NmxRange in[5 + 2 * NMX_MAX_SEGS], out[1 + NMX_MAX_SEGS];
    int ni = 0, no = 0;
    in[ni++] = {p->x, ((N - 1) * p->x_stride + p->cols) * 4};
    in[ni++] = {p->adapter, N * 4};
    in[ni++] = {p->scale, (size_t)p->adapters * 4};
    in[ni++] = {p->ranks, p->ranks ? (size_t)p->adapters * 4 : 0};
    out[no++] = {work, wb};
    for (int s = 0; s < p->count; s++) {
        if (!p->A[s] || !p->B[s] || !p->Y[s] || p->rows[s] < 1 || p->rows[s] > (1 << 20) || p->y_stride[s] < p->rows[s])
            return nmx_fail(ctx, "nmx_lora: matrix %d: rows=%d y_stride=%d, or a NULL argument", s, p->rows[s], p->y_stride[s]);
        if ((uintptr_t)p->A[s] % 16 || (uintptr_t)p->B[s] % 16 || (uintptr_t)p->Y[s] % 4)
            return nmx_fail(ctx, "nmx_lora: matrix %d: A or B not 16-byte aligned", s);
        in[ni++] = {p->A[s], mb * p->cols};
        in[ni++] = {p->B[s], mb * p->rows[s]};
        out[no++] = {p->Y[s], ((N - 1) * p->y_stride[s] + p->rows[s]) * 4};
        a.A[s] = p->A[s], a.B[s] = p->B[s], a.Y[s] = p->Y[s], a.rows[s] = p->rows[s], a.y_stride[s] = p->y_stride[s];
        a.first[s + 1] = a.first[s] + (p->rows[s] + 16 * LU_EACH * LU_WAVES - 1) / (16 * LU_EACH * LU_WAVES);
    }
    for (int i = 0; i < no; i++) {
        for (int k = 0; k < ni; k++)
            if (nmx_overlap(out[i].p, out[i].bytes, in[k].p, in[k].bytes))
                return nmx_fail(ctx, "nmx_lora: an output or work overlaps an input");
        for (int k = 0; k < i; k++)
            if (nmx_overlap(out[i].p, out[i].bytes, out[k].p, out[k].bytes))
                return nmx_fail(ctx, "nmx_lora: outputs and work overlap");
    }
    if (a.first[p->count] > 65535) return nmx_fail(ctx, "nmx_lora: too many rows in all");
    a.n = p->n, a.cols = p->cols, a.x_stride = p->x_stride, a.count = p->count, a.x = p->x, a.adapters = p->adapters;
    a.rank = p->rank, a.adapter = p->adapter, a.ranks = p->ranks, a.scale = p->scale, a.low = (float *)work;
    a.rank16 = (p->rank + 15) / 16 * 16;
    const nmx_on_device on(ctx);
    return p->w_dtype == W_F32 ? launch<W_F32>(ctx, a) : p->w_dtype == W_F16 ? launch<W_F16>(ctx, a) : launch<W_BF16>(ctx, a);
}

} /* extern "C" */
