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

struct TreeShape {
    int parents[TREE_MAX];
    int depth[TREE_MAX];                       // ancestors of a node; -1: padding
    uint32_t line[TREE_MAX][TREE_WORDS];       // bit j: node j is the node itself or an ancestor no more than window - 1 steps up
};

// All threads of the block; the caller synchronises behind it. A parent that does not stand before its child is reported, and
// the child taken as padding.
__device__ __forceinline__ void read_tree(TreeShape& t, const int* __restrict__ parents, int n, int window, int* __restrict__ err) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        int p = parents[i];
        if (p >= i) { atomicOr(err, CELLM_DEV_BAD_TREE); p = -2; }
        t.parents[i] = p;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
#pragma unroll
        for (int w = 0; w < TREE_WORDS; ++w) t.line[i][w] = 0u;
        int at = i, d = 0;
        while (at >= 0) {
            if (window <= 0 || d < window) t.line[i][at >> 5] |= 1u << (at & 31);
            ++d;
            at = t.parents[at];
        }
        t.depth[i] = at == -1 ? d - 1 : -1;
    }
    __syncthreads();
}

}  // namespace
