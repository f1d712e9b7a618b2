// What the kernels of drafted trees' attention share: their arguments, a block's share of the work, and which keys a node sees.
#pragma once
#include "draft_tree.cuh"

struct TreeArgs {
    void* out;                    // [T, nh * hd]
    float* part_o;                // [pieces, T * nh, hd], where pieces meet in the workspace
    float* part_ml;               // [pieces, T * nh, 2]
    const void *q, *k_new, *v_new;   // rows of node t at q + t * q_ld, k_new + t * k_ld, ...
    long long q_ld, k_ld, v_ld;   // in elements
    const int* parents;           // [T]
    const void *k_pool, *v_pool;  // [pages][nkv][page_size][hd]
    const int *cu_seqlens, *ctx_lens, *block_table;
    int bt_stride, B, T, most, num_pages, page_size, nh, nkv, hd, tiles, nsplit, window;
    float scale_log2e;
    int* err;
};

// The tcgen05 kernel (attention_tree_tc.cu): whether it takes a call, and its launch; pieces as for the others.
bool attention_tree_tc_takes(const TreeArgs& a);
int attention_tree_tc_launch(const TreeArgs& a, cudaStream_t stream);

namespace {

// A block's share of the work: request, key/value head, piece of the keys, tile of rows.
struct TreeTile {
    int b, kvh, split, tile, t_base, n, ctx;
    bool live;
};
__device__ __forceinline__ TreeTile tree_tile(const TreeArgs& a) {
    TreeTile t;
    int i = blockIdx.x;
    t.split = i % a.nsplit, i /= a.nsplit;
    t.tile = i % a.tiles, i /= a.tiles;
    t.kvh = i % a.nkv;
    t.b = i / a.nkv;
    t.t_base = a.cu_seqlens[t.b];
    t.n = a.cu_seqlens[t.b + 1] - t.t_base;
    t.ctx = a.ctx_lens[t.b];
    t.live = t.n > 0 && t.t_base >= 0 && t.t_base + t.n <= a.T;
    if (t.n > a.most || t.n < 0 || t.t_base < 0 || t.t_base + t.n > a.T) {
        if (threadIdx.x == 0) atomicOr(a.err, CELLM_DEV_BAD_TREE);
        t.live = false;
    }
    // keys beyond what a row of the block table can name are reported and left out
    if (t.ctx < 0 || t.ctx > (long long)a.bt_stride * a.page_size) {
        if (threadIdx.x == 0) atomicOr(a.err, CELLM_DEV_BAD_PAGE);
        t.ctx = t.ctx < 0 ? 0 : (int)((long long)a.bt_stride * a.page_size);
    }
    return t;
}

// Which of a block's KT keys a node sees, a bit a key: committed ones from position key0 on, or (node0 >= 0) the nodes from node0 on.
template <int KT>
__device__ __forceinline__ uint64_t seen_bits(const TreeShape& tree, int node, int window, int ctx, int key0, int node0) {
    static_assert(KT == 16 || KT == 32 || KT == 64, "a power of two of keys");
    if (node0 >= 0) {
        uint64_t m = tree.line[node][node0 >> 5];
        if (KT == 16) m >>= node0 & 31;
        if (KT == 64 && (node0 >> 5) + 1 < TREE_WORDS) m |= (uint64_t)tree.line[node][(node0 >> 5) + 1] << 32;
        return m;
    }
    const int lo = window > 0 ? max(0, ctx + tree.depth[node] - window + 1) : 0;
    const int below = min(max(lo - key0, 0), KT), upto = min(max(ctx - key0, 0), KT);
    const uint64_t in = upto >= 64 ? ~0ull : (1ull << upto) - 1ull, out = below >= 64 ? ~0ull : (1ull << below) - 1ull;
    return in & ~out;
}

}  // namespace
