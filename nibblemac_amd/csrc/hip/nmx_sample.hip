/* Sampling from rows of logits with temperature, top-k, top-p and min-p, from given uniform numbers
 * (include/nmx.h nmx_sample).
 *
 * A row's weights are w_i = exp((l_i - max l) / T), in 64 bits. The kept tokens are a prefix of the
 * row sorted by descending logit (ties: lower index first), the shortest of what the three filters
 * allow; the token is the first one, in index order, at which the running mass of the kept weights
 * passes u times their whole. So nothing is ever sorted: the filters need the logit at which the
 * prefix ends, the draw a running sum.
 *
 * sample_scan_k, one workgroup per 8192 logits of a row, reads the logits once. Rows without a
 * filter leave the chunk's maximum and its mass. Rows with one leave a histogram of the logits over
 * bins of 1/8 nat on a grid that every chunk shares (bin B covers 8 l / T in [B, B + 1)), 256 bins
 * down from the chunk's maximum: counts, masses, and the chunk's indices grouped by bin. What lies
 * 32 nats below a maximum weighs less than 2^-46 of it and is taken as zero.
 * sample_pick_k, one workgroup per row, adds the histograms, finds the bin where each filter ends,
 * selects within that bin among its own members (fetched through the grouped indices), and rescans
 * only the chunk that the draw falls into.
 *
 * Masses are whole numbers, the weight relative to its bin's lower edge (in [1, e^(1/8))) times
 * 2^40: their sums do not depend on the order in which lanes add them, so a call's result is the
 * same every time; between bins they are scaled and added in 64-bit floating point in a fixed
 * order. Each weight is thereby right to 2^-40 of itself (half a unit of rounding, and the polynomial's
 * next term).
 *
 * On MI355X (scan + pick): a row of 248320 with top-k and top-p 16.4 us (6.0 + 10.1), of 32768 with min-p
 * 13.6 (5.7 + 7.7), 5 rows at the temperature alone 12.2 (5.5 + 8.0), 64 rows of 248320 with top-p
 * 0.95 and no peaks 51 (27 + 27): 63.6 MB, 12.3 us as a copy; greedy, a row 7 to 8.6 and 64 rows 14.5. The scan
 * of 64 rows issues 40 vector
 * instructions a logit, the weight's polynomial and the bin among them (81 % of its cycles; neither more
 * copies of the bins nor two additions for one changed it). A pick is one workgroup's chain of phases. */
#include "nmx_internal.h"
#include "nmx_lanes.h"

namespace {

constexpr int SM_CHUNK = 8192; /* logits of a workgroup of sample_scan_k */
constexpr int SM_T1 = 512, SM_PER = SM_CHUNK / SM_T1, SM_SLICE = SM_CHUNK / (SM_T1 / 64);
constexpr int SM_T2 = 1024, SM_W2 = SM_T2 / 64, SM_RUN = SM_CHUNK / SM_T2; /* consecutive logits of a thread */
constexpr int SM_BINS = 256, SM_COPY = 4;
static_assert(2 * SM_BINS == SM_T1, "two threads of sample_scan_k to a bin");
constexpr int SM_MAXC = (1 << 20) / SM_CHUNK; /* chunks of the longest row */
constexpr int SM_LIST = 16384; /* members of a bin kept in LDS; a bin with more is read again */
constexpr int SM_RANK = 256;   /* members of a bin ranked by comparing all with all */
constexpr int SM_FEW = SM_T2;  /* tokens among which a row is decided one to a thread (500 of them 15 us against 22
                                * through the bins; up to 64 by one wave, 9.9 against 12.6) */
constexpr int SM_DIGIT = SM_T2; /* values of a selection's digit */
static_assert(SM_SLICE == SM_T2, "a wave's slice of a chunk is one logit a thread of sample_pick_k");

/* What sample_scan_k leaves of one chunk. */
struct Chunk {
    unsigned long long mass[SM_BINS]; /* by bin, relative to the bin's lower edge, in 2^-40 (without a
                                       * filter: the slices' masses, in 64-bit floating point) */
    double base;                      /* the top bin's number; without a filter the mass */
    unsigned long long key;           /* greedy rows: the first maximum's key */
    float max;                        /* -inf: nothing to choose in it */
    uint32_t pad;
    uint32_t seg[SM_BINS];            /* bin j's members: perm[seg & 0xffff ..], seg >> 16 of them */
    uint16_t perm[SM_CHUNK];          /* the chunk's indices, from its top bin down */
};

/* A row's parameters with every value outside its range read as "no filter". */
struct Par {
    double inv, min_p, top_p; /* inv = 8 / T */
    int top_k;
    bool greedy, filter;
};

__device__ __forceinline__ Par sample_par(const nmx_sample_params *p, int vocab) {
    Par r;
    const float T = p->temperature, tp = p->top_p, mp = p->min_p;
    r.greedy = !(T > 0.0f);
    r.inv = T < INFINITY ? 8.0 / (double)T : 0x1p-1000; /* infinite: every finite logit alike */
    r.top_k = p->top_k > 0 && p->top_k < vocab ? p->top_k : 0;
    r.top_p = tp < 1.0f ? fmaxf(tp, 0.0f) : 1.0;
    r.min_p = mp > 0.0f ? fminf(mp, 1.0f) : 0.0;
    r.filter = !r.greedy && (r.top_k || r.top_p < 1.0 || r.min_p > 0.0);
    return r;
}

/* NaN is never chosen, +inf is the largest finite value (ties among several). */
__device__ __forceinline__ float sample_value(float x) {
    return x == x ? fminf(x, 3.40282347e+38f) : -INFINITY;
}

/* order-preserving bits of a value that is not NaN (-0 and 0 alike) */
__device__ __forceinline__ uint32_t sample_key(float x) {
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sample_unkey(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ double grid_pos(float x, double inv) { return (double)x * inv; }
/* How far x lies above the lower edge fl of its bin (g = grid_pos, fl = floor(g)). g is off by 2^-52 of
 * itself, which from SM_FAR bins on would cost a weight more than 2^-43: there what the product and inv
 * left out is added (the result may leave [0, 1) by that much). Past 2^33 bins neighbouring floats are more
 * than 256 bins apart, and only equal logits are ever compared. */
constexpr double SM_FAR = 4096.0;
__device__ __forceinline__ bool grid_far(double top) { return !(top < SM_FAR && top - SM_BINS > -SM_FAR); }
/* what the rounding of inv = 8 / T left out */
__device__ __forceinline__ double grid_rest(float T, double inv) {
    return T < INFINITY ? __builtin_fma(-inv, (double)T, 8.0) / (double)T : 0.0;
}
__device__ __forceinline__ double grid_above(float x, double inv, double inv2, double g, double fl) {
    const double fr = g - fl, a = fabs(fl);
    return a >= SM_FAR && a < 0x1p33 ? fr + __builtin_fma((double)x, inv2, __builtin_fma((double)x, inv, -g)) : fr;
}

/* e^z for z <= 0, right to 2^-43 (2^(k + f), |f| <= 1/2, by the Taylor polynomial of degree 10 of
 * e^(f ln 2): the next term is below 2.1e-13 2^-1; the reduced argument's error is |z| 2^-52). What
 * lies below e^-700 is 0. */
__device__ __forceinline__ double exp_neg(double z) {
    const double t = z * 1.4426950408889634074, k = rint(t), x = (t - k) * 0.69314718055994530942;
    double p = 1.0 / 3628800;
    p = __builtin_fma(p, x, 1.0 / 362880);
    p = __builtin_fma(p, x, 1.0 / 40320);
    p = __builtin_fma(p, x, 1.0 / 5040);
    p = __builtin_fma(p, x, 1.0 / 720);
    p = __builtin_fma(p, x, 1.0 / 120);
    p = __builtin_fma(p, x, 1.0 / 24);
    p = __builtin_fma(p, x, 1.0 / 6);
    p = __builtin_fma(p, x, 0.5);
    p = __builtin_fma(p, x, 1.0);
    p = __builtin_fma(p, x, 1.0);
    return z > -700.0 ? ldexp(p, (int)k) : 0.0;
}
/* the weight of v where the largest logit is mx */
__device__ __forceinline__ double weight(float v, float mx, double inv) {
    return exp_neg(((double)v - (double)mx) * inv * 0.125);
}

/* The weight of grid position g relative to the lower edge of its bin, in 2^-40, for fr = g - floor(g):
 * 2^40 e^(fr / 8) about the bin's middle, degree 7 (the next term is below 6e-15), rounded to a whole
 * number by the addition of 2^52. */
struct BinPoly { /* the coefficients, in scalars: a lane's fma takes one from there without a move */
    double c[8];
    __device__ __forceinline__ BinPoly() {
        constexpr double M = 0x1p40 * 1.0644944589178594296; /* e^(1/16) */
        const double k[8] = {M, M / 8, M / (2 * 0x1p6), M / (6 * 0x1p9), M / (24 * 0x1p12), M / (120 * 0x1p15),
                             M / (720 * 0x1p18), M / (5040 * 0x1p21)};
#pragma unroll
        for (int i = 0; i < 8; i++) { /* the same polynomial, in powers of fr */
            double b = 0.0, w = 1.0; /* w: binomial(j, i) (-1/2)^(j - i) */
#pragma unroll
            for (int j = i; j < 8; j++) b += k[j] * w, w *= -0.5 * (j + 1) / (j + 1 - i);
            c[i] = b;
            asm("" : "+s"(c[i]));
        }
    }
    /* the bits of 2^52 + the mass: 0x433 << 52 | mass */
    __device__ __forceinline__ unsigned long long bits(double fr) const {
        double p = c[7];
#pragma unroll
        for (int i = 6; i >= 0; i--) p = __builtin_fma(p, fr, c[i]);
        return (unsigned long long)__double_as_longlong(p + 0x1p52);
    }
    __device__ __forceinline__ unsigned long long at(double fr) const { return bits(fr) & 0xfffffffffffffull; }
};
__device__ __forceinline__ unsigned long long bin_mass(float x, double inv, double inv2) {
    const double g = grid_pos(x, inv);
    return BinPoly().at(grid_above(x, inv, inv2, g, floor(g)));
}

__device__ __forceinline__ float block_max(float v, float *red, int waves) {
    v = nmx_max_f32_wave(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < waves; w++) v = fmaxf(v, red[w]);
    return v;
}

/* inclusive running sums over the SM_T2 threads, in thread order; *total is the last. red: SM_W2 words
 * that nothing else uses meanwhile. */
template <typename V>
__device__ __forceinline__ V block_scan(V v, unsigned long long *red8, V *total) {
    const int w = threadIdx.x >> 6;
    V *red = (V *)red8;
    v = nmx_scan_wave(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[w] = v;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < SM_W2; i++) {
        if (i == w) before = all;
        all += red[i];
    }
    *total = all;
    return before + v;
}

/* The first and the last thread for which a truth holds (SM_T2 and -1: none), known to all. */
__device__ __forceinline__ void block_find(bool first_of, bool last_of, unsigned long long *red1,
                                           unsigned long long *red2, int *first, int *last) {
    const unsigned long long a = __ballot(first_of), b = __ballot(last_of);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red1[threadIdx.x >> 6] = a, red2[threadIdx.x >> 6] = b;
    __syncthreads();
    /* lane w of every wave looks at wave w's word */
    const int lane = threadIdx.x & 63, at = lane & (SM_W2 - 1);
    const unsigned long long x = red1[at], y = red2[at], low = (1ull << SM_W2) - 1;
    const unsigned long long mx = __ballot(x != 0) & low, my = __ballot(y != 0) & low;
    const int f = __ffsll((long long)x) - 1, l = 63 - __clzll((long long)y);
    *first = mx ? 64 * (__ffsll((long long)mx) - 1) + __builtin_amdgcn_readlane(f, __ffsll((long long)mx) - 1) : SM_T2;
    *last = my ? 64 * (63 - __clzll((long long)my)) + __builtin_amdgcn_readlane(l, 63 - __clzll((long long)my)) : -1;
}

__global__ __launch_bounds__(SM_T1, 8) void sample_scan_k(const float *__restrict__ logits, int stride,
                                                       int vocab, Chunk *__restrict__ work,
                                                       const nmx_sample_params *par, int par_step) {
    __shared__ float redf[SM_T1 / 64];
    __shared__ double redd[SM_T1 / 64];
    __shared__ unsigned long long redk[SM_T1 / 64];
    __shared__ uint32_t wave_cnt[SM_T1 / 64], first_s[SM_BINS * SM_COPY];
    __shared__ unsigned long long bins[SM_BINS * SM_COPY]; /* members << 52 | mass */
    __shared__ uint32_t perm2[SM_CHUNK / 2];
    uint16_t *perm = (uint16_t *)perm2;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = blockIdx.x, row = blockIdx.y;
    const float *l = logits + (size_t)row * stride + (size_t)c * SM_CHUNK;
    const int len = vocab - c * SM_CHUNK < SM_CHUNK ? vocab - c * SM_CHUNK : SM_CHUNK;
    Chunk *out = work + (size_t)row * gridDim.x + c;
    /* a wave takes a slice of consecutive logits, 16 bytes a lane where the row allows it */
    const bool vec = len == SM_CHUNK && ((uintptr_t)l & 15) == 0;
    const int i0 = wave * SM_SLICE + (vec ? 4 * lane : lane);
    auto index = [&](int u) { return i0 + (vec ? (u >> 2) * 256 + (u & 3) : u * 64); };
    float v[SM_PER];
    if (vec) {
#pragma unroll
        for (int u = 0; u < SM_PER; u += 4) {
            const float4 x = *(const float4 *)(l + index(u));
            v[u] = x.x, v[u + 1] = x.y, v[u + 2] = x.z, v[u + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int u = 0; u < SM_PER; u++) v[u] = l[index(u) < len ? index(u) : len - 1]; /* no branch around a request */
#pragma unroll
        for (int u = 0; u < SM_PER; u++) v[u] = index(u) < len ? v[u] : -INFINITY;
    }
    const Par p = sample_par(par + (size_t)row * par_step, vocab);
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < SM_PER; u++) {
        v[u] = sample_value(v[u]);
        mx = fmaxf(mx, v[u]);
    }
    if (p.greedy) {
        unsigned long long best = 0;
#pragma unroll
        for (int u = 0; u < SM_PER; u++) {
            const unsigned long long k = (unsigned long long)sample_key(v[u]) << 32 |
                                         (0xffffffffu - (uint32_t)(c * SM_CHUNK + index(u)));
            if (v[u] > -INFINITY && k > best) best = k;
        }
        best = nmx_max_u64_wave(best);
        if (lane == 0) redk[wave] = best;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < SM_T1 / 64; w++) best = redk[w] > best ? redk[w] : best;
            out->key = best;
        }
        return;
    }
    mx = block_max(mx, redf, SM_T1 / 64);
    if (tid == 0) out->max = mx;
    if (!(mx > -INFINITY)) {
        if (tid == 0) out->base = 0.0;
        return;
    }
    if (!p.filter) {
        double s = 0.0;
#pragma unroll
        for (int u = 0; u < SM_PER; u++) s += weight(v[u], mx, p.inv);
        s = nmx_scan_wave(s);
        if (lane == 63) redd[wave] = s, ((double *)out->mass)[wave] = s;
        __syncthreads();
        if (tid == 0) {
            double total = 0.0;
            for (int w = 0; w < SM_T1 / 64; w++) total += redd[w];
            out->base = total;
        }
        return;
    }
    /* SM_COPY copies of each bin, by lane: neighbouring lanes of one bin do not wait for each other. A
     * copy has at most SM_CHUNK / SM_COPY members of less than 1.14 2^40 each: 12 bits for them and 52
     * for their mass, one addition for both */
    static_assert(SM_CHUNK / SM_COPY * 1.14 * 0x1p40 < 0x1p52 && SM_CHUNK / SM_COPY < 4096, "a copy's word");
#pragma unroll
    for (int i = 0; i < SM_BINS * SM_COPY; i += SM_T1) bins[i + tid] = 0;
    __syncthreads();
    const double base = floor(grid_pos(mx, p.inv));
    const uint32_t copy = (lane & (SM_COPY - 1)) * 8;
    const BinPoly poly;
    uint32_t at[SM_PER]; /* byte offset of a copy's word << 12 | rank in it; all ones: no weight */
    auto add = [&](int u, double fl, double above) {
        at[u] = 0xffffffffu;
        const double d = base - fl; /* inf for -inf */
        if (d < (double)SM_BINS) {
            const uint32_t j = (uint32_t)(int)d * (SM_COPY * 8) + copy;
            unsigned long long *w = (unsigned long long *)((char *)bins + j);
            const unsigned long long old = atomicAdd(w, poly.bits(above) - (0x432ull << 52));
            at[u] = __builtin_amdgcn_alignbit(j, (uint32_t)(old >> 32), 20);
        }
    };
    /* no bin of the chunk as far as SM_FAR: nothing to add, and three instructions a logit fewer */
    if (!__builtin_amdgcn_readfirstlane(grid_far(base))) {
#pragma unroll
        for (int u = 0; u < SM_PER; u++) {
            const double g = grid_pos(v[u], p.inv), fl = floor(g);
            add(u, fl, g - fl);
        }
    } else {
        const double inv2 = grid_rest(par[(size_t)row * par_step].temperature, p.inv);
#pragma unroll
        for (int u = 0; u < SM_PER; u++) {
            const double g = grid_pos(v[u], p.inv), fl = floor(g);
            add(u, fl, grid_above(v[u], p.inv, inv2, g, fl));
        }
    }
    __syncthreads();
    /* thread: SM_COPY / 2 copies of a bin */
    constexpr int PT = SM_BINS * SM_COPY / SM_T1;
    uint32_t mine[PT], n = 0;
    unsigned long long m = 0;
#pragma unroll
    for (int i = 0; i < PT; i++) {
        const unsigned long long x = bins[tid * PT + i];
        mine[i] = (uint32_t)(x >> 52), n += mine[i], m += x & 0xfffffffffffffull;
    }
    const uint32_t upto = nmx_scan_wave(n);
    if (lane == 63) wave_cnt[wave] = upto;
    __syncthreads();
    uint32_t first = upto - n, members = 0;
#pragma unroll
    for (int w = 0; w < SM_T1 / 64; w++) {
        if (w < wave) first += wave_cnt[w];
        members += wave_cnt[w];
    }
    {
        uint32_t f = first;
#pragma unroll
        for (int i = 0; i < PT; i++) first_s[tid * PT + i] = f, f += mine[i];
    }
    /* the two threads of a bin together */
    const uint32_t n2 = n + (uint32_t)nmx_dpp<NMX_DPP_XOR1>((int)n);
    m += (unsigned long long)(uint32_t)nmx_dpp<NMX_DPP_XOR1>((int)(m >> 32)) << 32 | (uint32_t)nmx_dpp<NMX_DPP_XOR1>((int)m);
    if (!(tid & 1)) out->seg[tid >> 1] = first | n2 << 16, out->mass[tid >> 1] = m;
    if (tid == 0) out->base = base;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < SM_PER; u++)
        if (at[u] != 0xffffffffu) perm[*(const uint32_t *)((const char *)first_s + (at[u] >> 13)) + (at[u] & 0xfffu)] = (uint16_t)index(u);
    __syncthreads();
    uint2 *po = (uint2 *)out->perm;
    for (uint32_t i = tid; 4 * i < members; i += SM_T1) po[i] = ((const uint2 *)perm2)[i];
}

/* The row's state in sample_pick_k. */
struct Pick {
    unsigned long long mass[SM_BINS];    /* the row's histogram, from its top bin down */
    unsigned long long cand[SM_MAXC];    /* masses of a bin's kept members by chunk */
    unsigned long long red1[SM_W2], red2[SM_W2], sel_m;
    double edge[SM_BINS];                /* e^(-b / 8): bin b's lower edge, the top bin's being 1 */
    double chunk_mass[SM_MAXC], sel_d;
    float redf[SM_W2];
    uint32_t cnt[SM_BINS];
    int off[SM_MAXC];                    /* the chunk's top bin below the row's */
    uint32_t seg[SM_MAXC + 1];           /* running sizes of the segments of the members in hand */
    uint32_t at[SM_MAXC];                /* where a chunk's segment begins in its order */
    uint32_t ties[SM_MAXC];
    uint32_t sel_n, sel_k;
    int hit;
    union {
        struct {
            unsigned long long tally[SM_DIGIT], part_m[3][SM_BINS]; /* masses of a selection's digit */
            unsigned long long small_mass[SM_RANK];
            uint32_t digit[SM_DIGIT], small[SM_RANK], part_n[3][SM_BINS];
            uint32_t list[SM_LIST];
        };
        unsigned long long few[SM_FEW];
    };
};

/* What a row keeps: the keys above key, and of those equal to it the first `ties` in index order. */
struct Cut {
    uint32_t key, ties;
};

/* A row as sample_pick_k sees it. */
struct Row {
    const Chunk *ch;
    const float *l;
    int C;
    double inv, inv2, top; /* top: the row's top bin */
};

/* Member i of those in hand (S.seg, S.at): its chunk, its index there, its logit. */
__device__ __forceinline__ float member(const Pick &S, const Row &r, uint32_t i, int *c_out, int *at_out) {
    int lo = 0, hi = r.C; /* the last chunk whose segment starts at or before i */
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (S.seg[m] <= i) lo = m;
        else hi = m;
    }
    const int at = r.ch[lo].perm[S.at[lo] + (i - S.seg[lo])];
    *c_out = lo, *at_out = at;
    return sample_value(r.l[(size_t)lo * SM_CHUNK + at]);
}

/* Takes in hand the members of the row's bins b0 .. b1; a chunk's lie together. The number of them. */
__device__ uint32_t take_bins(Pick &S, const Row &r, int b0, int b1) {
    const int tid = threadIdx.x;
    uint32_t x = 0, from = 0;
    if (tid < r.C) {
        int j0 = b0 - S.off[tid], j1 = b1 - S.off[tid];
        j0 = j0 < 0 ? 0 : j0, j1 = j1 < SM_BINS - 1 ? j1 : SM_BINS - 1;
        if (j0 <= j1) {
            const uint32_t s0 = r.ch[tid].seg[j0], s1 = r.ch[tid].seg[j1];
            from = s0 & 0xffff, x = (s1 & 0xffff) + (s1 >> 16) - from;
        }
    }
    uint32_t total;
    const uint32_t incl = block_scan(x, S.red1, &total);
    if (tid < r.C) S.seg[tid] = incl - x, S.at[tid] = from;
    if (tid == 0) S.seg[r.C] = total;
    __syncthreads();
    return total;
}

/* take_bins of bin b alone, and its keys into the list if they fit. */
__device__ void open_bin(Pick &S, const Row &r, int b) {
    __syncthreads();
    const uint32_t total = take_bins(S, r, b, b);
    if (total <= SM_LIST) {
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < total; i += SM_T2) {
            int c, at;
            S.list[i] = sample_key(member(S, r, i, &c, &at));
        }
    }
    __syncthreads();
}
__device__ __forceinline__ uint32_t key_of(const Pick &S, const Row &r, uint32_t i) {
    int c, at;
    return S.seg[r.C] <= SM_LIST ? S.list[i] : sample_key(member(S, r, i, &c, &at));
}

/* Among the members of the opened bin b with keys of at least floor_key: the key at which the run in
 * descending order reaches `want` members (by count) or the mass want_mass (in 2^-40 of the bin's
 * lower edge). above / above_mass: what lies strictly above that key. Digits of 10 bits of the keys
 * that the bin spans, until few enough are left to compare all with all. */
__device__ uint32_t select_key(Pick &S, const Row &r, int b, bool by_count, uint32_t want, double want_mass,
                               uint32_t floor_key, uint32_t *above, double *above_mass) {
    const int tid = threadIdx.x;
    const uint32_t total = S.seg[r.C];
    /* the bin's keys lie between those of its edges (one bin wider: the product's rounding) */
    const double lo_x = (r.top - b - 1.0) / r.inv, hi_x = (r.top - b + 2.0) / r.inv, most = 3.40282346638528859e+38;
    uint32_t klo = sample_key((float)fmin(fmax(lo_x, -most), most)), khi = sample_key((float)fmin(fmax(hi_x, -most), most));
    klo = klo < floor_key ? floor_key : klo;
    uint32_t n_above = 0, left = total;
    unsigned long long m_above = 0;
    while (left > SM_RANK && klo < khi) {
        const int bits = 32 - __clz((int)(khi - klo)), shift = bits > 10 ? bits - 10 : 0;
        __syncthreads();
        S.digit[tid] = 0, S.tally[tid] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < total; i += SM_T2) {
            const uint32_t k = key_of(S, r, i);
            if (k < klo || k > khi) continue;
            const uint32_t d = (khi - k) >> shift;
            atomicAdd(&S.digit[d], 1u);
            if (!by_count) atomicAdd(&S.tally[d], bin_mass(sample_unkey(k), r.inv, r.inv2));
        }
        __syncthreads();
        const uint32_t n = S.digit[tid];
        const unsigned long long m = S.tally[tid];
        uint32_t n_all;
        unsigned long long m_all = 0, m_to = 0;
        const uint32_t n_to = n_above + block_scan(n, S.red1, &n_all);
        if (!by_count) m_to = m_above + block_scan(m, S.red1, &m_all);
        /* the first digit that reaches the want; the last one where a rounding keeps it from any */
        int hit, last;
        block_find(n && (by_count ? n_to >= want : (double)m_to >= want_mass), n, S.red1, S.red2, &hit, &last);
        hit = hit < SM_DIGIT ? hit : last < 0 ? 0 : last;
        if (tid == hit) S.sel_n = n_to - n, S.sel_k = n, S.sel_m = m_to - m;
        __syncthreads();
        n_above = S.sel_n, left = S.sel_k, m_above = S.sel_m;
        khi -= (uint32_t)hit << shift;
        const uint32_t low = shift ? khi - ((1u << shift) - 1) : khi;
        klo = low > klo && low <= khi ? low : klo;
    }
    __syncthreads();
    if (klo == khi) { /* all that is left are ties */
        *above = n_above, *above_mass = (double)m_above;
        return khi;
    }
    if (tid == 0) S.sel_n = 0;
    __syncthreads();
    for (uint32_t i = tid; i < total; i += SM_T2) {
        const uint32_t k = key_of(S, r, i);
        if (k < klo || k > khi) continue;
        const uint32_t at = atomicAdd(&S.sel_n, 1u);
        S.small[at] = k; /* at < left <= SM_RANK */
        S.small_mass[at] = by_count ? 0 : bin_mass(sample_unkey(k), r.inv, r.inv2);
    }
    __syncthreads();
    const uint32_t N = S.sel_n;
    uint32_t k = 0, gt = 0, eq = 0;
    unsigned long long gm = 0, em = 0;
    if ((uint32_t)tid < N) {
        k = S.small[tid];
#pragma unroll 8
        for (uint32_t i = 0; i < N; i++) {
            const uint32_t o = S.small[i];
            const unsigned long long w = S.small_mass[i];
            if (o > k) gt++, gm += w;
            if (o == k) eq++, em += w;
        }
    }
    /* the greatest key whose run reaches the want; the least where none does */
    if (tid == 0) S.sel_k = 0;
    __syncthreads();
    if ((uint32_t)tid < N && (by_count ? n_above + gt + eq >= want : (double)(m_above + gm + em) >= want_mass)) atomicMax(&S.sel_k, k);
    __syncthreads();
    uint32_t key = S.sel_k;
    __syncthreads();
    if (key == 0) {
        if (tid == 0) S.sel_k = 0xffffffffu;
        __syncthreads();
        if ((uint32_t)tid < N) atomicMin(&S.sel_k, k);
        __syncthreads();
        key = S.sel_k;
    }
    if ((uint32_t)tid < N && k == key) S.sel_n = n_above + gt, S.sel_m = m_above + gm; /* the same of each tie */
    __syncthreads();
    *above = S.sel_n, *above_mass = (double)S.sel_m;
    return key;
}

/* The least logit whose weight is at least min_p of the largest: its key. Weights grow with the key, so a
 * wave looks at 64 keys about the logarithm's border first, where it nearly always is, and else cuts the span of
 * keys that it may lie in to a 64th at a time: 6 rounds for 32 bits, also where weights are alike over
 * millions of keys (logits next to 0, a high temperature, min_p of 1). The upper end is always in. */
__device__ uint32_t min_p_key(float mx, double inv, double min_p) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = sample_key(-3.40282347e+38f), hi = sample_key(mx);
    uint32_t step = 1, from = sample_key(sample_value((float)fmax((double)mx + 8.0 * log(min_p) / inv, -3.40282346638528859e+38)));
    from = from < lo + 32 ? lo : from - 32 < hi ? from - 32 : hi;
    for (int round = 0; lo < hi && round < 8; round++) {
        const uint32_t k = from + lane * step < hi ? from + lane * step : hi;
        const unsigned long long in = __ballot(k == hi || weight(sample_unkey(k), mx, inv) >= min_p);
        const int f = in ? __ffsll((long long)in) - 1 : 64; /* the first key that is in */
        if (f < 64) hi = from + f * step < hi ? from + f * step : hi;
        if (f > 0) lo = from + (f - 1) * step + 1;
        from = lo, step = (hi - lo + 63) >> 6;
    }
    return hi;
}

/* A step of a bitonic network: this lane and lane ^ J, the greater with the lower one where up holds. J < 16
 * goes without LDS. */
template <int CTRL>
__device__ __forceinline__ unsigned long long dpp64(unsigned long long v) {
    return (unsigned long long)(uint32_t)nmx_dpp<CTRL>((int)(v >> 32)) << 32 | (uint32_t)nmx_dpp<CTRL>((int)v);
}
template <int J>
__device__ __forceinline__ void sort_step(unsigned long long &v, bool up) {
    unsigned long long o;
    if constexpr (J == 1) o = dpp64<NMX_DPP_XOR1>(v);
    else if constexpr (J == 2) o = dpp64<NMX_DPP_XOR2>(v);
    else if constexpr (J == 4) o = dpp64<NMX_DPP_HALF_MIRROR>(dpp64<0x1B>(v)); /* lane ^ 3, then ^ 7 */
    else if constexpr (J == 8) o = dpp64<0x128>(v);                            /* row_ror:8 */
    else o = __shfl_xor(v, J);
    const bool low = (threadIdx.x & J) == 0;
    if ((o > v) == (low == up)) v = o;
}
__device__ __forceinline__ unsigned long long readlane64(unsigned long long v, int l) {
    return (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}

/* The threads' values below P (a power of two from 64 on) in descending order, thread 0's the largest: a bitonic
 * network, in a wave by shuffles, across waves through buf. Threads from P on keep what they have. */
__device__ unsigned long long sort_down(unsigned long long v, int P, unsigned long long *buf) {
    const int tid = threadIdx.x;
    const bool in = tid < P;
    for (int k = 2; k <= P; k <<= 1) {
        for (int j = k >> 1; j >= 64; j >>= 1) {
            __syncthreads();
            if (in) buf[tid] = v;
            __syncthreads();
            const unsigned long long o = buf[in ? tid ^ j : 0];
            if (in && (o > v) == (((tid & j) == 0) == ((tid & k) == 0))) v = o;
        }
        if ((tid & ~63) >= P) continue; /* a wave without values */
        const bool up = (tid & k) == 0;
        if (k >= 64) sort_step<32>(v, up);
        if (k >= 32) sort_step<16>(v, up);
        if (k >= 16) sort_step<8>(v, up);
        if (k >= 8) sort_step<4>(v, up);
        if (k >= 4) sort_step<2>(v, up);
        sort_step<1>(v, up);
    }
    return v;
}

/* pick_few for up to 64 tokens: the first wave's lanes, each compared with all through scalars. */
__device__ void pick_wave(const Pick &S, const Row &r, const Par &p, float mx, double whole, double ud, int32_t *tok, float *prob) {
    const int i = threadIdx.x, N = (int)S.seg[r.C];
    if (i >= 64) return;
    unsigned long long v = 0;
    double w = 0.0;
    uint32_t index = 0xffffffffu;
    if (i < N) {
        int c, at;
        const float x = member(S, r, i, &c, &at);
        index = (uint32_t)(c * SM_CHUNK + at);
        v = (unsigned long long)sample_key(x) << 32 | ~index;
        w = weight(x, mx, r.inv);
    }
    unsigned long long mine = (unsigned long long)(w * 0x1p52 + 0.5), before = 0;
    int rank = 0;
    for (int j = 0; j < N; j++) {
        const unsigned long long o = readlane64(v, j), m = readlane64(mine, j);
        if (o > v) rank++, before += m;
    }
    bool keep = i < N && w > 0.0;
    if (p.top_k) {
        const int k = p.top_k < N ? p.top_k : N;
        whole = (double)readlane64(before + mine, __ffsll((long long)__ballot(i < N && rank == k - 1)) - 1);
        keep = keep && rank < k;
    } else {
        whole *= 0x1p52;
    }
    if (p.top_p < 1.0) keep = keep && (rank == 0 || (double)before < p.top_p * whole);
    if (p.min_p > 0.0) keep = keep && w >= p.min_p;
    mine = keep ? mine : 0;
    unsigned long long upto = mine, all = 0;
    uint32_t last = 0;
    for (int j = 0; j < N; j++) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)index, j);
        const unsigned long long m = readlane64(mine, j);
        all += m;
        if (o < index) upto += m;
        last = m && o > last ? o : last;
    }
    const double goal = ud * (double)all;
    const bool hit = goal < (double)all ? (double)(upto - mine) <= goal && (double)upto > goal : index == last;
    if (keep && hit) {
        tok[blockIdx.x] = (int)index;
        if (prob) prob[blockIdx.x] = (float)(w / ((double)all * 0x1p-52));
    }
}

/* A row whose kept tokens are among the S.seg[C] <= SM_FEW in hand, one to a thread: sorted by order for
 * the filters, then what they keep by index for the draw. Masses are in 2^-52 of the largest weight.
 * whole: the mass that top-p counts against where there is no top-k. */
__device__ void pick_few(Pick &S, const Row &r, const Par &p, float mx, double whole, double ud, int32_t *tok, float *prob) {
    const int tid = threadIdx.x, N = (int)S.seg[r.C]; /* > 64 */
    const int P = 1 << (32 - __clz(N - 1));
    unsigned long long v = 0; /* greater: earlier in the sorted row */
    if (tid < N) {
        int c, at;
        const float x = member(S, r, tid, &c, &at);
        v = (unsigned long long)sample_key(x) << 32 | ~(uint32_t)(c * SM_CHUNK + at);
    }
    auto mass_of = [&](double w) { return (unsigned long long)(w * 0x1p52 + 0.5); };
    v = sort_down(v, P, S.few);
    const uint32_t key = (uint32_t)(v >> 32);
    double w = tid < N ? weight(sample_unkey(key), mx, r.inv) : 0.0;
    unsigned long long mine = mass_of(w), all;
    const unsigned long long before = block_scan(mine, S.red1, &all) - mine;
    bool keep = tid < N && w > 0.0;
    if (p.top_k) {
        const int k = p.top_k < N ? p.top_k : N;
        if (tid == k - 1) S.sel_m = before + mine;
        __syncthreads();
        whole = (double)S.sel_m;
        keep = keep && tid < k;
    } else {
        whole *= 0x1p52;
    }
    if (p.top_p < 1.0) keep = keep && (tid == 0 || (double)before < p.top_p * whole);
    if (p.min_p > 0.0) keep = keep && w >= p.min_p;
    v = sort_down(keep ? v << 32 | key : 0, P, S.few); /* the kept ones by index: ~index on top */
    const bool kept = v != 0;
    w = kept ? weight(sample_unkey((uint32_t)v), mx, r.inv) : 0.0, mine = mass_of(w);
    const unsigned long long upto = block_scan(mine, S.red2, &all);
    const double goal = ud * (double)all;
    /* the token whose share of the running mass holds the goal; past the whole the last one */
    int hit, last;
    block_find(kept && (double)upto > goal, kept, S.red1, S.red2, &hit, &last);
    if (tid == (hit < SM_T2 ? hit : last)) {
        tok[blockIdx.x] = (int)~(uint32_t)(v >> 32);
        if (prob) prob[blockIdx.x] = (float)(w / ((double)all * 0x1p-52));
    }
}

__global__ __launch_bounds__(SM_T2) void sample_pick_k(const float *__restrict__ logits, int stride,
                                                       int vocab, int C, const Chunk *__restrict__ work,
                                                       const nmx_sample_params *par, int par_step,
                                                       const float *__restrict__ uni,
                                                       int32_t *__restrict__ tok,
                                                       float *__restrict__ prob) {
    extern __shared__ uint4 smem[];
    Pick &S = *(Pick *)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    const float *l = logits + (size_t)row * stride;
    const Chunk *ch = work + (size_t)row * C;
    const float mc = tid < C ? ch[tid].max : -INFINITY; /* garbage in a greedy row, and not used there */
    const double bc = tid < C ? ch[tid].base : 0.0;
    const float u = uni[row];
    const Par p = sample_par(par + (size_t)row * par_step, vocab);
    auto answer = [&](int t, double pr) {
        tok[row] = t;
        if (prob) prob[row] = (float)pr;
    };
    if (p.greedy) {
        if (tid < 64) {
            unsigned long long k = 0;
            for (int c = tid; c < C; c += 64) k = ch[c].key > k ? ch[c].key : k;
            k = nmx_max_u64_wave(k);
            if (tid == 0) answer(k ? (int)(0xffffffffu - (uint32_t)k) : -1, k ? 1.0 : 0.0);
        }
        return;
    }
    const double ud = u > 0.0f ? (double)fminf(u, 1.0f) : 0.0;
    const float mx = block_max(mc, S.redf, SM_W2);
    if (!(mx > -INFINITY)) { /* nothing to choose from */
        if (tid == 0) answer(-1, 0.0);
        return;
    }
    Cut cut = {0, 0xffffffffu};
    double mass = 0.0; /* chunk tid's kept mass, the largest weight being 1 */
    if (!p.filter) {
        if (tid < C && mc > -INFINITY) mass = bc * weight(mc, mx, p.inv);
    } else {
        const double g_top = grid_pos(mx, p.inv), top = floor(g_top);
        const double inv2 = grid_far(top) ? grid_rest(par[(size_t)row * par_step].temperature, p.inv) : 0.0;
        const Row r = {ch, l, C, p.inv, inv2, top};
        if (tid < C) {
            const double d = mc > -INFINITY ? top - bc : (double)SM_BINS;
            S.off[tid] = d < (double)SM_BINS ? (int)d : SM_BINS;
            S.cand[tid] = 0, S.ties[tid] = 0;
        }
        __syncthreads();
        const int b = tid & (SM_BINS - 1), quarter = tid / SM_BINS;
        {
            uint32_t n = 0; /* a thread adds its bin over every 4th chunk, 8 requests at a time */
            unsigned long long m = 0;
            for (int c0 = quarter; c0 < C; c0 += 32) {
                uint32_t ns[8];
                unsigned long long ms[8];
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const int c = c0 + 4 * q < C ? c0 + 4 * q : C - 1, j = b - S.off[c]; /* no branch around a request */
                    ns[q] = ch[c].seg[j < 0 ? 0 : j] >> 16;
                    ms[q] = ch[c].mass[j < 0 ? 0 : j];
                }
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const int c = c0 + 4 * q;
                    if (c < C && b >= S.off[c]) n += ns[q], m += ms[q];
                }
            }
            if (quarter) S.part_n[quarter - 1][b] = n, S.part_m[quarter - 1][b] = m;
            __syncthreads();
            if (!quarter) {
                S.cnt[b] = n + S.part_n[0][b] + S.part_n[1][b] + S.part_n[2][b];
                S.mass[b] = m + S.part_m[0][b] + S.part_m[1][b] + S.part_m[2][b];
                S.edge[b] = exp_neg(-0.125 * b);
            }
            __syncthreads();
        }
        const double edge = S.edge[b];
        /* a mass of the top bin, as a weight */
        const double unit = exp_neg(grid_above(mx, p.inv, inv2, g_top, top) * -0.125) * 0x1p-40;
        /* a bin that the kept tokens do not reach below: of top-k's or top-p's end, of min-p's border (one
         * lower, for its rounding). Few tokens down to it: they decide among themselves */
        uint32_t n_all;
        const uint32_t n_mine = tid < SM_BINS ? S.cnt[tid] : 0, n_upto = block_scan(n_mine, S.red1, &n_all);
        const bool by_k = p.top_k && (uint32_t)p.top_k < n_all;
        double m_all = 0.0, m_mine = 0.0, m_upto = 0.0; /* the masses that top-p counts, top-k aside */
        int reach = SM_BINS, pb = SM_BINS, last;
        if (by_k) {
            block_find(tid < SM_BINS && n_upto >= (uint32_t)p.top_k, false, S.red1, S.red2, &reach, &last);
        } else if (p.top_p < 1.0) {
            if (tid < SM_BINS) m_mine = (double)S.mass[b] * edge;
            m_upto = block_scan(m_mine, S.red1, &m_all);
            block_find(m_mine > 0.0 && m_upto >= p.top_p * m_all, m_mine > 0.0, S.red1, S.red2, &pb, &last);
            pb = pb < SM_BINS ? pb : last; /* a whole missed by a rounding */
            reach = pb;
        }
        if (p.min_p > 0.0 && !(by_k && p.top_p < 1.0)) {
            const double d = top - floor(g_top + 8.0 * log(p.min_p)) + 1.0;
            if (d < (double)reach) reach = (int)d;
        }
        if (reach < SM_BINS) {
            if (tid == reach) S.sel_n = n_upto;
            __syncthreads();
            if (S.sel_n <= SM_FEW) {
                Par q = p;
                if (!by_k) q.top_k = 0;
                take_bins(S, r, 0, reach);
                if (S.seg[C] <= 64) pick_wave(S, r, q, mx, m_all * unit, ud, tok, prob);
                else pick_few(S, r, q, mx, m_all * unit, ud, tok, prob);
                return;
            }
        }
        int kb = SM_BINS;     /* the bin that top-k ends in */
        double k_mass = 0.0;  /* and the mass that it keeps of it, in 2^-40 of its lower edge */
        if (by_k) {
            const uint32_t k = (uint32_t)p.top_k;
            __syncthreads();
            if (n_mine && n_upto >= k && n_upto - n_mine < k) S.hit = tid, S.sel_n = k - (n_upto - n_mine);
            __syncthreads();
            kb = S.hit;
            const uint32_t want = S.sel_n;
            open_bin(S, r, kb);
            uint32_t above;
            double unused;
            cut.key = select_key(S, r, kb, true, want, 0.0, 0, &above, &unused);
            cut.ties = want - above;
            if (p.top_p < 1.0) {
                unsigned long long kept = 0, whole;
                for (uint32_t i = tid; i < S.seg[C]; i += SM_T2) {
                    const uint32_t key = key_of(S, r, i);
                    if (key > cut.key) kept += bin_mass(sample_unkey(key), p.inv, inv2);
                }
                block_scan(kept, S.red1, &whole);
                k_mass = (double)whole + (double)cut.ties * (double)bin_mass(sample_unkey(cut.key), p.inv, inv2);
            }
        }
        int opened = kb;
        if (p.top_p < 1.0) { /* over what top-k left */
            if (by_k) {
                m_mine = tid < SM_BINS ? (b < kb ? (double)S.mass[b] : b == kb ? k_mass : 0.0) * edge : 0.0;
                m_upto = block_scan(m_mine, S.red1, &m_all);
                block_find(m_mine > 0.0 && m_upto >= p.top_p * m_all, m_mine > 0.0, S.red1, S.red2, &pb, &last);
                pb = pb < SM_BINS ? pb : last;
            }
            if (tid == pb) S.sel_d = fmax(p.top_p * m_all - (m_upto - m_mine), 0.0) / edge;
            __syncthreads();
            const double rest = S.sel_d;
            if (pb != kb) open_bin(S, r, pb);
            opened = pb;
            uint32_t above;
            double m_above;
            const uint32_t key = select_key(S, r, pb, false, 0, rest, pb == kb ? cut.key : 0, &above, &m_above);
            const double need = ceil((rest - m_above) / (double)bin_mass(sample_unkey(key), p.inv, inv2));
            uint32_t ties = need < 1.0 ? 1u : need < 4e9 ? (uint32_t)need : 0xffffffffu;
            if (pb == kb && key == cut.key && cut.ties < ties) ties = cut.ties;
            cut.key = key, cut.ties = ties;
        }
        if (p.min_p > 0.0) {
            const uint32_t key = min_p_key(mx, p.inv, p.min_p); /* the same of every wave */
            if (key > cut.key) cut.key = key, cut.ties = 0xffffffffu;
        }
        /* the kept mass of each chunk: whole bins, then the members of the cut's own bin */
        const double d = cut.key ? top - floor(grid_pos(sample_unkey(cut.key), p.inv)) : (double)SM_BINS;
        const int cb = d < (double)SM_BINS ? (int)d : SM_BINS;
        if (cb < SM_BINS) {
            if (cb != opened) open_bin(S, r, cb);
            const uint32_t total = S.seg[C];
            for (int c = wave; c < C; c += SM_W2) { /* a wave adds a chunk's */
                uint32_t n = 0;
                unsigned long long m = 0;
                const uint32_t end = S.seg[c + 1];
                for (uint32_t i = S.seg[c] + lane; i < end; i += 64) {
                    uint32_t key;
                    if (total <= SM_LIST) key = S.list[i];
                    else key = sample_key(sample_value(l[(size_t)c * SM_CHUNK + ch[c].perm[S.at[c] + (i - S.seg[c])]]));
                    n += key == cut.key;
                    if (key > cut.key) m += bin_mass(sample_unkey(key), p.inv, inv2);
                }
                n = nmx_scan_wave(n), m = nmx_scan_wave(m);
                if (lane == 63) S.ties[c] = n, S.cand[c] = m;
            }
        }
        for (int c0 = wave; c0 < C; c0 += 2 * SM_W2) { /* a wave adds two chunks' whole bins, in a fixed order */
            unsigned long long m[2][4];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int q = 0; q < 4; q++) m[i][q] = ch[c0 + i * SM_W2 < C ? c0 + i * SM_W2 : C - 1].mass[lane + 64 * q];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int c = c0 + i * SM_W2;
                if (c >= C) break;
                double s = 0.0;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int k = lane + 64 * q + S.off[c];
                    if (k < cb) s += (double)m[i][q] * S.edge[k];
                }
                s = nmx_scan_wave(s);
                if (lane == 63) S.chunk_mass[c] = s;
            }
        }
        __syncthreads();
        uint32_t all;
        const uint32_t mine = tid < C ? S.ties[tid] : 0, to = block_scan(mine, S.red1, &all), before = to - mine;
        const uint32_t ties = before >= cut.ties ? 0 : cut.ties - before < mine ? cut.ties - before : mine;
        if (tid < C) {
            S.ties[tid] = ties;
            mass = S.chunk_mass[tid];
            if (cb < SM_BINS) {
                double m = (double)S.cand[tid];
                if (ties) m += (double)ties * (double)bin_mass(sample_unkey(cut.key), p.inv, inv2);
                mass += m * S.edge[cb];
            }
            mass *= unit;
        }
    }
    /* the chunk that the draw falls into */
    double whole;
    const double to = block_scan(mass, S.red1, &whole);
    const double goal = ud < 1.0 ? ud * whole : INFINITY; /* from 1 on: past every sum, however it was rounded */
    const bool some = mass > 1e-296; /* so that one of its slices has 1e-297, and one logit a weight of 1e-300 */
    int c, c_last;
    block_find(some && to > goal, some, S.red1, S.red2, &c, &c_last);
    c = c < SM_T2 ? c : c_last;
    if (tid == c) S.sel_d = to - mass;
    __syncthreads();
    double rest = goal - S.sel_d;
    const int len = vocab - c * SM_CHUNK < SM_CHUNK ? vocab - c * SM_CHUNK : SM_CHUNK;
    const float *lc = l + (size_t)c * SM_CHUNK;
    /* without a filter the scan left the masses of the chunk's slices: one logit to a thread; else 8
     * consecutive ones of the chunk */
    const int per = p.filter ? SM_RUN : 1;
    int i0 = tid * per;
    if (!p.filter) {
        const float mcc = ch[c].max;
        const double up = weight(mcc, mx, p.inv);
        double at = -1.0, run = 0.0;
        int slice = 0;
#pragma unroll
        for (int w = 0; w < SM_CHUNK / SM_SLICE; w++) { /* every thread the same few sums */
            const double m = ((const double *)ch[c].mass)[w] * up;
            if (m > 1e-297 && (run <= rest || at < 0.0)) slice = w, at = run; /* the last one that starts at or before */
            run += m;
        }
        rest -= at;
        i0 += slice * SM_SLICE;
    }
    float x[SM_RUN];
    uint32_t key[SM_RUN], same = 0;
    if (p.filter && len == SM_CHUNK && ((uintptr_t)lc & 15) == 0) {
#pragma unroll
        for (int e = 0; e < SM_RUN; e += 4) {
            const float4 y = *(const float4 *)(lc + i0 + e);
            x[e] = y.x, x[e + 1] = y.y, x[e + 2] = y.z, x[e + 3] = y.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < SM_RUN; e++) x[e] = lc[e < per && i0 + e < len ? i0 + e : len - 1];
#pragma unroll
        for (int e = 0; e < SM_RUN; e++) x[e] = e < per && i0 + e < len ? x[e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < SM_RUN; e++) {
        x[e] = sample_value(x[e]);
        key[e] = sample_key(x[e]);
        same += x[e] > -INFINITY && key[e] == cut.key;
    }
    uint32_t rank = 0xffffffffu, allowed = 0xffffffffu;
    if (p.filter) {
        uint32_t all;
        rank = block_scan(same, S.red1, &all) - same;
        allowed = S.ties[c];
    }
    double w[SM_RUN], s = 0.0;
#pragma unroll
    for (int e = 0; e < SM_RUN; e++) {
        w[e] = 0.0;
        if (e >= per) continue;
        bool keep = x[e] > -INFINITY && key[e] >= cut.key;
        if (p.filter && keep && key[e] == cut.key) keep = rank++ < allowed;
        if (keep) w[e] = weight(x[e], mx, p.inv);
        s += w[e];
    }
    double in_chunk;
    double run = block_scan(s, S.red1, &in_chunk) - s;
    double wf = 0.0, wl = 0.0; /* the thread's first token past the goal, and its last one */
    int first = -1, final = -1;
#pragma unroll
    for (int e = 0; e < SM_RUN; e++) {
        run += w[e];
        if (w[e] > 0.0) {
            final = i0 + e, wl = w[e];
            if (run > rest && first < 0) first = i0 + e, wf = w[e];
        }
    }
    int who, who_last;
    block_find(first >= 0, final >= 0, S.red1, S.red2, &who, &who_last);
    if (who < SM_T2) {
        if (tid == who) answer(c * SM_CHUNK + first, wf / whole);
    } else if (tid == who_last) { /* a whole missed by a rounding: the last one */
        answer(c * SM_CHUNK + final, wl / whole);
    }
}

} // namespace

extern "C" {

size_t nmx_sample_work_bytes(int n, int vocab) {
    if (n < 1 || n > 4096 || vocab < 1 || vocab > (1 << 20)) return 0;
    return (size_t)n * ((vocab + SM_CHUNK - 1) / SM_CHUNK) * sizeof(Chunk);
}

int nmx_sample(nmx_ctx *ctx, const float *logits, int stride, int vocab, int n,
               const nmx_sample_params *params, int per_row, const float *u, void *work, int32_t *tok,
               float *prob) {
    if (!ctx) return -1;
    if (n < 1 || n > 4096 || vocab < 1 || vocab > (1 << 20) || stride < vocab)
        return nmx_fail(ctx, "nmx_sample: bad shape n=%d vocab=%d stride=%d", n, vocab, stride);
    if (!logits || !params || !u || !work || !tok) return nmx_fail(ctx, "nmx_sample: NULL argument");
    if ((uintptr_t)work % 16) return nmx_fail(ctx, "nmx_sample: work not 16-byte aligned");
    const int C = (vocab + SM_CHUNK - 1) / SM_CHUNK;
    const size_t lb = ((size_t)(n - 1) * stride + vocab) * 4, wb = nmx_sample_work_bytes(n, vocab);
    const size_t pb = sizeof(nmx_sample_params) * (per_row ? (size_t)n : 1), ob = (size_t)n * 4;
    const void *in[] = {logits, params, u};
    const size_t ib[] = {lb, pb, ob};
    for (int i = 0; i < 3; i++)
        if (nmx_overlap(tok, ob, in[i], ib[i]) || nmx_overlap(work, wb, in[i], ib[i]) ||
            (prob && nmx_overlap(prob, ob, in[i], ib[i])))
            return nmx_fail(ctx, "nmx_sample: an output or the workspace overlaps an input");
    if (nmx_overlap(tok, ob, work, wb) || (prob && (nmx_overlap(prob, ob, work, wb) || nmx_overlap(prob, ob, tok, ob))))
        return nmx_fail(ctx, "nmx_sample: outputs overlap");
    const nmx_on_device on(ctx);
    sample_scan_k<<<dim3((unsigned)C, (unsigned)n), SM_T1, 0, ctx->stream>>>(
        logits, stride, vocab, (Chunk *)work, params, per_row ? 1 : 0);
    NMX_LAUNCHED(ctx, "sample_scan");
    static std::atomic<uint64_t> lds_set;
    if (nmx_dyn_lds(ctx, (const void *)sample_pick_k, sizeof(Pick), lds_set)) return -1;
    sample_pick_k<<<(unsigned)n, SM_T2, sizeof(Pick), ctx->stream>>>(logits, stride, vocab, C, (const Chunk *)work,
                                                          params, per_row ? 1 : 0, u, tok, prob);
    NMX_LAUNCHED(ctx, "sample_pick");
    return 0;
}

} /* extern "C" */
