/* Low-rank adapters of many requests (include/nmx.h nmx_lora): y += scale B (A x), each row with its own
 * adapter, for the matrices that share x.
 *
 * Rows with one adapter are taken together, 16 at a time (a tile), so that A and B are read once for them. A row's rank
 * among those of its adapter is counted by ballots over the adapters that 64 rows have; the rows of rank 0, 16, ..
 * lead the tiles, which are numbered in the order of their leaders. lora_down_k makes the list in every workgroup, leaves it
 * in the workspace, and makes 16 ranks of A x, the columns shared out over its waves; lora_up_k adds 16 rows of B at a
 * time to y. Products are fp32 matrix instructions (16 x 16 x 4): a lane takes 8 neighbouring columns of a weight
 * row and of a row of x, the sum over the 32 columns of a wave's step has no order to keep, so weights go from
 * 16-byte loads to the operand without passing through LDS.
 *
 * Times on MI355X: 8 requests, 5 adapters of 16 ranks, 1024 columns to 4096 + 512 + 512 rows 7.7 us (one launch); 64 requests, 40
 * adapters of up to 64 ranks, 1024 to 3584 + 3584 21 (9.7 + 12.4 in a trace, 5.1 as a copy); 512 requests of one adapter of 64
 * ranks 25 (11.4 + 14.9, 5.7 as a copy). Two launches, each a chain of round trips: lora_up_k waits for each 32 ranks in turn
 * and asks for half of a 128-byte line of 64 16-bit ranks at a time; every tile of 16 rows asks for its adapter again. */
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
    float *low;         /* [count][n][rank16]: A x */
    struct Tile *tiles; /* [tiles] */
    int rank16;
    const void *A[NMX_MAX_SEGS], *B[NMX_MAX_SEGS];
    int rows[NMX_MAX_SEGS], y_stride[NMX_MAX_SEGS];
    float *Y[NMX_MAX_SEGS];
    int first[NMX_MAX_SEGS + 1]; /* of lora_up_k's workgroups */
};

/* Rows of one adapter (adapter -1: no such tile); row -1: fewer rows. */
struct Tile {
    int adapter, rank, row[16], pad[14];
};
/* Tile number `want`, by the whole workgroup (at least n threads). */
__device__ __forceinline__ void find_tile(const Lora &a, int want, Tile *tile) {
    constexpr int B = NMX_CHUNK_ROWS / 64;
    __shared__ int leads_s[B], first_s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int id[B];
#pragma unroll
    for (int u = 0; u < B; u++) {
        id[u] = -1;
        if (64 * u < a.n) { /* uniform */
            const int v = a.adapter[64 * u + lane < a.n ? 64 * u + lane : 0];
            id[u] = 64 * u + lane < a.n && v >= 0 && v < a.adapters ? v : -1;
        }
    }
    int mine = -1, rank = 0;
#pragma unroll
    for (int u = 0; u < B; u++) mine = u == wave ? id[u] : mine;
    for (unsigned long long left = __ballot(mine >= 0); left;) { /* an adapter of this wave's rows */
        const int m = __builtin_amdgcn_readlane(mine, __ffsll((long long)left) - 1);
        const unsigned long long same = __ballot(mine == m);
        int before = 0;
        for (int u = 0; u < wave; u++) {
            int v = id[0];
#pragma unroll
            for (int k = 1; k < B; k++) v = u == k ? id[k] : v;
            before += __popcll(__ballot(v == m));
        }
        if (mine == m) rank = before + __popcll(same & ((1ull << lane) - 1));
        left &= ~same;
    }
    const unsigned long long leads = __ballot(mine >= 0 && rank % 16 == 0);
    if (lane == 0 && wave < B) leads_s[wave] = __popcll(leads);
    if (tid < 16) tile->row[tid] = -1;
    if (tid == 0) tile->adapter = -1;
    __syncthreads();
    int number = __popcll(leads & ((1ull << lane) - 1));
    for (int w = 0; w < wave && w < B; w++) number += leads_s[w];
    if (mine >= 0 && rank % 16 == 0 && number == want) {
        const int rk = a.ranks ? a.ranks[mine] : a.rank;
        tile->adapter = mine, tile->rank = rk < 0 ? 0 : rk < a.rank ? rk : a.rank;
        first_s = rank;
    }
    __syncthreads();
    if (mine >= 0 && mine == tile->adapter && rank >= first_s && rank < first_s + 16) tile->row[rank - first_s] = tid;
    __syncthreads();
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

/* Ranks r0 + 4 k .. + 3 of A x for the tile's row c in lane (k, c) of the first wave, zeros where the adapter has no such
 * rank, whatever A holds there; by the whole workgroup. */
template <int WT>
__device__ __forceinline__ float4 down_block(const Lora &a, const Tile &tile, int s, int r0, float4 (*sum_s)[64]) {
    constexpr int SIZE = WT == W_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c = lane & 15, k = lane >> 4;
    const int row = tile.row[c], r = r0 + c < a.rank ? r0 + c : a.rank - 1;
    const char *wp = (const char *)a.A[s] + (((size_t)tile.adapter * a.rank + r) * a.cols + 8 * k) * SIZE;
    const float *xp = a.x + (size_t)(row < 0 ? tile.row[0] : row) * a.x_stride + 8 * k;
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
    float4 v = sum_s[0][lane];
    if (wave) return v;
#pragma unroll
    for (int w = 1; w < LD_WAVES; w++) {
        const float4 y = sum_s[w][lane];
        v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
    }
    const int q = r0 + 4 * k, own = tile.rank;
    if (q >= own) v.x = 0.0f;
    if (q + 1 >= own) v.y = 0.0f;
    if (q + 2 >= own) v.z = 0.0f;
    if (q + 3 >= own) v.w = 0.0f;
    return v;
}

/* Workgroup: a tile, blockIdx.y 16 ranks of a matrix. */
template <int WT>
__global__ __launch_bounds__(64 * LD_WAVES) void lora_down_k(Lora a) {
    __shared__ float4 sum_s[LD_WAVES][64];
    __shared__ Tile tile;
    find_tile(a, blockIdx.x, &tile);
    if (blockIdx.y == 0 && threadIdx.x < 18) ((int *)(a.tiles + blockIdx.x))[threadIdx.x] = ((int *)&tile)[threadIdx.x];
    if (tile.adapter < 0) return; /* uniform over the workgroup */
    const int blocks = a.rank16 / 16, s = blockIdx.y / blocks, r0 = blockIdx.y % blocks * 16, row = tile.row[threadIdx.x & 15];
    const float4 v = down_block<WT>(a, tile, s, r0, sum_s);
    if (threadIdx.x < 64 && row >= 0) *(float4 *)(a.low + ((size_t)s * a.n + row) * a.rank16 + r0 + 4 * (threadIdx.x >> 4)) = v;
}

/* 64 output rows of a wave: y, requested with the weights, and the products' accumulators. Four neighbouring rows of B are
 * four neighbours in y. */
template <int WT, bool VEC>
struct Up {
    static constexpr int SIZE = WT == W_F32 ? 4 : 2;
    const Lora &a;
    int s, o0, rows, adapter, own, c, k;
    bool live, quads;
    float *yp;
    float4 y[LU_EACH];
    float4v acc[LU_EACH];
    W8<WT> v[LU_EACH];
    float w[LU_EACH][8];
    __device__ __forceinline__ Up(const Lora &a, int s, int o0, int adapter, int own, int row, int lane)
        : a(a), s(s), o0(o0), rows(a.rows[s]), adapter(adapter), own(own), c(lane & 15), k(lane >> 4), live(row >= 0),
          quads(a.y_stride[s] % 4 == 0 && ((uintptr_t)a.Y[s] & 15) == 0), yp(a.Y[s] + (size_t)(row < 0 ? 0 : row) * a.y_stride[s]) {
#pragma unroll
        for (int e = 0; e < LU_EACH; e++) {
            const int o = o0 + 16 * e + 4 * k;
            y[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), acc[e] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            if (quads && o + 3 < rows && live) y[e] = *(const float4 *)(yp + o);
        }
    }
    __device__ __forceinline__ void request(int q) { /* ranks q + 8 k .. + 7 */
        const int at = q + 8 * k;
#pragma unroll
        for (int e = 0; e < LU_EACH; e++) {
            const int o = o0 + 16 * e + c < rows ? o0 + 16 * e + c : rows - 1;
            const size_t first = ((size_t)adapter * rows + o) * a.rank;
            if constexpr (VEC) {
                v[e].load((const char *)a.B[s] + (first + (at < a.rank ? at : 0)) * SIZE);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) w[e][i] = one_weight<WT>(a.B[s], first + (at + i < a.rank ? at + i : 0));
            }
        }
    }
    __device__ __forceinline__ void add(int q, const float4 (&x)[2]) {
        const int at = q + 8 * k;
        const float z[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int e = 0; e < LU_EACH; e++) {
                const float b = VEC ? v[e].at(i) : w[e][i]; /* behind the adapter's rank anything: not used */
                acc[e] = mfma4(at + i < own ? b : 0.0f, z[i], acc[e]);
            }
    }
    __device__ __forceinline__ void store(float scale) {
        if (!live) return;
#pragma unroll
        for (int e = 0; e < LU_EACH; e++) {
            const int o = o0 + 16 * e + 4 * k;
            if (quads && o + 3 < rows) {
                *(float4 *)(yp + o) = make_float4(__builtin_fmaf(acc[e][0], scale, y[e].x), __builtin_fmaf(acc[e][1], scale, y[e].y),
                                                  __builtin_fmaf(acc[e][2], scale, y[e].z), __builtin_fmaf(acc[e][3], scale, y[e].w));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (o + i < rows) yp[o + i] = __builtin_fmaf(acc[e][i], scale, yp[o + i]);
            }
        }
    }
};
__device__ __forceinline__ int seg_of(const Lora &a, int y) {
    int s = 0;
    while (s + 1 < a.count && y >= a.first[s + 1]) s++;
    return s;
}

/* Workgroup: a tile, blockIdx.y a run of output rows of a matrix. VEC: rows of B are 16-byte aligned. */
template <int WT, bool VEC>
__global__ __launch_bounds__(64 * LU_WAVES) void lora_up_k(Lora a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Tile *tile = a.tiles + blockIdx.x;
    const int adapter = __builtin_amdgcn_readfirstlane(tile->adapter), own = __builtin_amdgcn_readfirstlane(tile->rank);
    const int row = tile->row[lane & 15];
    if (adapter < 0 || own == 0) return; /* no ranks: the rows are left alone */
    const int s = seg_of(a, blockIdx.y), o0 = (((int)blockIdx.y - a.first[s]) * LU_WAVES + wave) * 16 * LU_EACH;
    if (o0 >= a.rows[s]) return;
    const float scale = a.scale[adapter];
    Up<WT, VEC> up(a, s, o0, adapter, own, row, lane);
    /* a column without a row takes the first one's: it is not stored */
    const int first = tile->row[0];
    const float *lp = a.low + ((size_t)s * a.n + (row < 0 ? first : row)) * a.rank16 + 8 * up.k;
    for (int q = 0; q < own; q += 32) {
        float4 x[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
        up.request(q);
        if (q + 8 * up.k < a.rank16) x[0] = *(const float4 *)(lp + q), x[1] = *(const float4 *)(lp + q + 4);
        up.add(q, x);
    }
    up.store(scale);
}

/* Both in one launch, where the A of a matrix is small: every workgroup makes A x of its tile again, while its rows of B and
 * y are on their way. */
template <int WT, bool VEC>
__global__ __launch_bounds__(64 * LD_WAVES) void lora_one_k(Lora a) {
    __shared__ float4 sum_s[LD_WAVES][64];
    __shared__ Tile tile;
    __shared__ __align__(16) float low_s[16 * 20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    find_tile(a, blockIdx.x, &tile);
    const int adapter = tile.adapter, own = tile.rank, row = tile.row[lane & 15];
    if (adapter < 0 || own == 0) return; /* uniform over the workgroup */
    const int s = seg_of(a, blockIdx.y), o0 = (((int)blockIdx.y - a.first[s]) * LD_WAVES + wave) * 16 * LU_EACH;
    const float scale = a.scale[adapter];
    Up<WT, VEC> up(a, s, o0 < a.rows[s] ? o0 : 0, adapter, own, o0 < a.rows[s] ? row : -1, lane); /* no rows left: nothing is stored */
    up.request(0);
    const float4 v = down_block<WT>(a, tile, s, 0, sum_s);
    if (wave == 0) *(float4 *)(low_s + up.c * 20 + 4 * up.k) = v;
    __syncthreads();
    float4 x[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    const float *lp = low_s + up.c * 20 + 8 * up.k;
    if (up.k < 2) x[0] = *(const float4 *)lp, x[1] = *(const float4 *)(lp + 4);
    up.add(0, x);
    up.store(scale);
}

/* an adapter has at most one tile that is not full */
int tiles_of(const Lora &a) {
    const int most = a.n / 16 + (a.adapters < a.n ? a.adapters : a.n);
    return most < a.n ? most : a.n;
}
/* workgroups of a tile's output rows, `run` rows each */
int runs_of(const nmx_lora_args &p, int run) {
    int n = 0;
    for (int s = 0; s < p.count; s++) n += (p.rows[s] + run - 1) / run;
    return n;
}
/* One launch where every workgroup may make A x again: 16 ranks (more are one block of them after the other) of up to
 * LO_BYTES, in up to two workgroups a CU, or one where the list of the tiles is longer than a wave. Ranks of 16, binary16: 8
 * requests to 4096 + 512 + 512 rows 7.7 us against 9.7 in two launches, from 3584 columns 11.6 against 13.7; 64 on 40 adapters
 * (440 workgroups) 12.4 against 13.5, to 3584 + 3584 (616) 16.1 against 13.5; 512 on 4 (360) 18.7 against 16.1, from 3584 columns
 * to 1024 rows (72) 17.8 against 18.9; 64 on 40 of 25 ranks, bfloat16, 22.6 against 18.9. */
constexpr size_t LO_BYTES = 128 * 1024;
constexpr int LO_RUN = 16 * LU_EACH * LD_WAVES;
bool in_one(const Lora &a, const nmx_lora_args &p, int size) {
    return a.rank16 == 16 && (size_t)a.rank16 * a.cols * size <= LO_BYTES &&
           (long long)tiles_of(a) * runs_of(p, LO_RUN) <= (a.n <= 64 ? 512 : 256);
}

template <int WT>
int launch(nmx_ctx *ctx, const Lora &a, bool one) {
    const int tiles = tiles_of(a);
    const dim3 grid((unsigned)tiles, (unsigned)a.first[a.count]);
    const bool vec = a.rank % 8 == 0;
    if (one) {
        if (vec) lora_one_k<WT, true><<<grid, 64 * LD_WAVES, 0, ctx->stream>>>(a);
        else lora_one_k<WT, false><<<grid, 64 * LD_WAVES, 0, ctx->stream>>>(a);
        NMX_LAUNCHED(ctx, "lora_one");
        return 0;
    }
    lora_down_k<WT><<<dim3((unsigned)tiles, (unsigned)(a.count * a.rank16 / 16)), 64 * LD_WAVES, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "lora_down");
    if (vec) lora_up_k<WT, true><<<grid, 64 * LU_WAVES, 0, ctx->stream>>>(a);
    else lora_up_k<WT, false><<<grid, 64 * LU_WAVES, 0, ctx->stream>>>(a);
    NMX_LAUNCHED(ctx, "lora_up");
    return 0;
}

/* Matrices i and k write columns of their own of the same rows. */
bool side_by_side(const nmx_lora_args &p, int i, int k) {
    const intptr_t by = (intptr_t)p.Y[k] - (intptr_t)p.Y[i], row = (intptr_t)p.y_stride[i] * 4;
    if (p.y_stride[i] != p.y_stride[k] || by % 4) return false;
    const intptr_t at = (by % row + row) % row; /* of k's first column from i's, within a row */
    return at >= (intptr_t)p.rows[i] * 4 && at + (intptr_t)p.rows[k] * 4 <= row;
}

} // namespace

extern "C" {

size_t nmx_lora_work_bytes(int n, int count, int rank) {
    if (n < 1 || n > NMX_CHUNK_ROWS || count < 1 || count > NMX_MAX_SEGS || rank < 1 || rank > 256) return 0;
    return (size_t)n * sizeof(Tile) + (size_t)count * n * ((rank + 15) / 16 * 16) * 4;
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
    }
    for (int i = 0; i < no; i++) {
        for (int k = 0; k < ni; k++)
            if (nmx_overlap(out[i].p, out[i].bytes, in[k].p, in[k].bytes))
                return nmx_fail(ctx, "nmx_lora: an output or work overlaps an input");
        for (int k = 0; k < i; k++)
            if (nmx_overlap(out[i].p, out[i].bytes, out[k].p, out[k].bytes) && !(k > 0 && side_by_side(*p, i - 1, k - 1)))
                return nmx_fail(ctx, "nmx_lora: outputs and work overlap");
    }
    a.rank16 = (p->rank + 15) / 16 * 16, a.cols = p->cols, a.n = p->n, a.adapters = p->adapters;
    const bool one = in_one(a, *p, (int)ws);
    const int run = one ? LO_RUN : 16 * LU_EACH * LU_WAVES; /* output rows of a workgroup */
    for (int s = 0; s < p->count; s++) a.first[s + 1] = a.first[s] + (p->rows[s] + run - 1) / run;
    if (a.first[p->count] > 65535) return nmx_fail(ctx, "nmx_lora: too many rows in all");
    a.x_stride = p->x_stride, a.count = p->count, a.x = p->x;
    a.rank = p->rank, a.adapter = p->adapter, a.ranks = p->ranks, a.scale = p->scale;
    a.tiles = (Tile *)work, a.low = (float *)((char *)work + N * sizeof(Tile));
    const nmx_on_device on(ctx);
    return p->w_dtype == W_F32 ? launch<W_F32>(ctx, a, one) : p->w_dtype == W_F16 ? launch<W_F16>(ctx, a, one) : launch<W_BF16>(ctx, a, one);
}

} /* extern "C" */
