// What the kernels over drafted trees share: a tree's shape in shared memory and what its nodes see of one another.
//
// A tree is a run of nodes of which each names its parent by its place in the run: -1 hangs on the request's last committed
// token, anything below -1 marks padding. A parent stands before its child, so a walk from parent to parent ends. Padding, and
// what hangs on it, sees nothing and is seen by nobody.
#pragma once
#include "common.cuh"

namespace {

constexpr int TREE_MAX = 256;                  // nodes of a tree
constexpr int TREE_WORDS = TREE_MAX / 32;

struct __align__(16) TreeShape {
    int parents[TREE_MAX];
    int depth[TREE_MAX];                       // ancestors of a node; -1: padding
    uint32_t line[TREE_MAX][TREE_WORDS];       // bit j: node j is the node itself or an ancestor no more than window - 1 steps up
};

// By `threads` threads of which this is number `me`; `sync` is their barrier, and the caller needs none behind it. A parent that does
// not stand before its child is reported, and the child taken as padding.
template <typename Sync>
__device__ __forceinline__ void read_tree(TreeShape& t, const int* __restrict__ parents, int n, int window, int* __restrict__ err, int me, int threads, const Sync& sync) {
    for (int i = me; i < n; i += threads) {
        int p = parents[i];
        if (p >= i) { atomicOr(err, CELLM_DEV_BAD_TREE); p = -2; }
        t.parents[i] = p;
    }
    sync();
    for (int i = me; i < n; i += threads) {
        // the walk up is a chain of loads; the bits gather in registers beside it
        uint32_t line[TREE_WORDS] = {};
        int at = i, d = 0;
        while (at >= 0) {
            const uint32_t bit = window <= 0 || d < window ? 1u << (at & 31) : 0u;
#pragma unroll
            for (int w = 0; w < TREE_WORDS; ++w) line[w] |= at >> 5 == w ? bit : 0u;
            ++d;
            at = t.parents[at];
        }
        uint4* to = reinterpret_cast<uint4*>(t.line[i]);
        to[0] = make_uint4(line[0], line[1], line[2], line[3]);
        to[1] = make_uint4(line[4], line[5], line[6], line[7]);
        t.depth[i] = at == -1 ? d - 1 : -1;
    }
    sync();
}
__device__ __forceinline__ void read_tree(TreeShape& t, const int* parents, int n, int window, int* err) {
    read_tree(t, parents, n, window, err, (int)threadIdx.x, (int)blockDim.x, [] { __syncthreads(); });
}

}  // namespace
