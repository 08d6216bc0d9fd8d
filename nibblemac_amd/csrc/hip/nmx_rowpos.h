/* Positions of a batch's rows (nmx_attnbatch.hip), whatever the lengths on the device hold: no step of these leaves 32 bits.
 * Needs no header of HIP, so tests compile it for the host with checks of overflow. */
#ifndef NMX_ROWPOS_H
#define NMX_ROWPOS_H

/* Position of row i of the count rows that end at length len (0 <= len, i < count). */
__host__ __device__ __forceinline__ int row_position(int len, int count, int i) { return len - (count - i); }

/* A segment's rows see the positions below last + 1, the next ones one more each; ROWS_SEE_ALL: all of them. */
constexpr int ROWS_SEE_ALL = 1 << 28;
/* How many of the positions [0, p1) (at most 2^24) row i of a segment sees; below 1: none. */
__host__ __device__ __forceinline__ int positions_seen(int last, int i, int p1) {
    if (last >= p1) return p1; /* last + 1 + i is not formed: it may leave 32 bits */
    return last + 1 + i < p1 ? last + 1 + i : p1;
}

#endif
