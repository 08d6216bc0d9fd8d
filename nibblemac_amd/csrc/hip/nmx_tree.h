/* Shared by the kernels over a tree of drafts (nmx_attntree.hip, nmx_lintree.hip, nmx_tree.hip): the
 * ancestors of a node. Not part of the ABI. */
#ifndef NMX_TREE_H
#define NMX_TREE_H

#include "nmx_internal.h"

/* The parent of node t as the kernels take it: -1 (the context) for any value outside [-1, t). */
__device__ __forceinline__ int tree_parent(const int32_t *parent, int t) {
    const int p = parent[t];
    return p >= 0 && p < t ? p : -1;
}

/* Lane t < n of a wave (every lane active) gets the set of node t and its ancestors; lanes past n
 * their own bit. Pointer doubling: after round k a lane's set holds the 2^k nearest. *above (may be
 * NULL): the lane's parent. The depth of a node is the size of its set - 1. */
__device__ __forceinline__ unsigned long long tree_ancestors(const int32_t *parent, int n, int *above) {
    const int lane = threadIdx.x & 63;
    int p = lane < n ? tree_parent(parent, lane) : -1;
    if (above) *above = p;
    unsigned long long set = 1ull << lane;
#pragma unroll
    for (int k = 0; k < 6; k++) {
        const int from = p < 0 ? lane : p;
        const unsigned long long s = __shfl(set, from);
        const int q = __shfl(p, from);
        if (p >= 0) set |= s, p = q;
    }
    return set;
}

#endif
