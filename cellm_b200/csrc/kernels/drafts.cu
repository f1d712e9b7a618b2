// Which tokens of drafted trees stand, and their keys and values into the cache.
//
// Node 0 of a tree is the token the last step chose; it stands. From a node that stands the walk goes to its child whose token
// is the model's choice after the node (the first among equals), until there is none or `longest` nodes stand; the choice after
// the last node is the request's next token. Every child's test is made at once: a child that fits leaves its place with its
// parent (the smallest stays), and the walk then follows one word a step.
//
// The kept rows of all layers are written to places ctx, ctx + 1, ... of the request's pages. Every block repeats the walk
// (a microsecond at most) and takes its share of the copies, so that one launch does it all. Bound by latency: one tree of 8 nodes takes
// 2.8 us in a CUDA graph, 64 trees of 63 nodes with 16 layers' rows 7.4 us (17 MB, 2.6 us at a copy's rate).
#include <algorithm>

#include "draft_tree.cuh"

namespace {

struct DraftRows {             // keys or values: [items][T] rows beside the cache, the pool [items][pages][nkv][page_size][units]
    const void* rows;
    void* pool;
    long long item_ld, row_ld; // bytes between items and between nodes of `rows`
    int row_bytes;             // of one head
};

template <typename W>
__global__ void __launch_bounds__(TREE_MAX)
accept_drafts_kernel(int* __restrict__ out_count, int* __restrict__ out_path, int* __restrict__ out_next, const int* __restrict__ tokens,
                     const int* __restrict__ parents, const int* __restrict__ choices, const int* __restrict__ cu_seqlens, int T, int longest,
                     const DraftRows k, const DraftRows v, const int* __restrict__ ctx_lens, const int* __restrict__ block_table, int bt_stride,
                     int items, int nkv, int pages, int page_size, int* __restrict__ err) {
    __shared__ int child[TREE_MAX], choice[TREE_MAX], path[TREE_MAX], place_page[TREE_MAX];
    __shared__ int count_s;
    pdl_wait();
    // what does not depend on the walk is asked for before it
    const int b = blockIdx.y, t_base = cu_seqlens[b], ctx = items > 0 ? ctx_lens[b] : 0;
    int n = cu_seqlens[b + 1] - t_base;
    if (n > TREE_MAX || n < 0 || t_base < 0 || t_base + n > T) {
        if (threadIdx.x == 0) atomicOr(err, CELLM_DEV_BAD_TREE);
        n = 0;
    }
    const int me = threadIdx.x, node_parent = me < n ? parents[t_base + me] : -1, node_token = me < n ? tokens[t_base + me] : 0;
    if (me < n) child[me] = TREE_MAX, choice[me] = choices[t_base + me];
    if (items > 0 && me < min(longest, n)) {
        const long long at = ((long long)ctx + me) / page_size;
        const int page = ctx >= 0 && at < bt_stride ? block_table[(long long)b * bt_stride + at] : -1;
        place_page[me] = page < 0 || page >= pages ? -1 : page;
    }
    __syncthreads();
    if (me < n) {
        if (node_parent >= me) atomicOr(err, CELLM_DEV_BAD_TREE);
        else if (node_parent >= 0 && node_token == choice[node_parent]) atomicMin(&child[node_parent], me);
    }
    __syncthreads();
    if (me == 0) {
        int c = 0;
        // (a tree whose first node is padding keeps nothing)
        for (int at = n > 0 && node_parent == -1 ? 0 : n; at < n && c < longest; at = child[at]) path[c++] = at;
        count_s = c;
    }
    __syncthreads();
    const int count = count_s;
    if (blockIdx.x == 0) {
        for (int j = me; j < longest; j += TREE_MAX) out_path[(long long)b * longest + j] = j < count ? path[j] : -1;
        if (me == 0) out_count[b] = count, out_next[b] = count > 0 ? choice[path[count - 1]] : -1;
        if (items > 0 && me < count && place_page[me] < 0) atomicOr(err, CELLM_DEV_BAD_PAGE);
    }
    // the kept rows: neighbouring threads take a head's pieces, then the kept nodes, whose rows lie one behind the other on a page
    const unsigned k_units = (unsigned)k.row_bytes / sizeof(W), v_units = (unsigned)v.row_bytes / sizeof(W);
    const unsigned k_item = (unsigned)(count * nkv) * k_units, per_item = k_item + (unsigned)(count * nkv) * v_units;
    for (unsigned long long u = (unsigned long long)blockIdx.x * TREE_MAX + me; u < (unsigned long long)items * per_item; u += (unsigned long long)gridDim.x * TREE_MAX) {
        const unsigned item = (unsigned)(u / per_item), in_item = (unsigned)(u - (unsigned long long)item * per_item);
        const bool value = in_item >= k_item;
        const DraftRows& d = value ? v : k;
        const unsigned units = value ? v_units : k_units, rest = value ? in_item - k_item : in_item;
        const unsigned x = rest % units, j = rest / units % count, h = rest / units / count;
        const int page = place_page[j];
        if (page < 0) continue;
        const W* src = reinterpret_cast<const W*>(static_cast<const char*>(d.rows) + item * d.item_ld + (long long)(t_base + path[j]) * d.row_ld) + h * units + x;
        static_cast<W*>(d.pool)[((((size_t)item * pages + page) * nkv + h) * page_size + (ctx + j) % page_size) * units + x] = *src;
    }
}

}  // namespace

// tokens, parents, choices [T]; out_path [B][longest], out_count and out_next [B]. items > 0: the rows k_new [items][T][nkv][k_bytes]
// (k_item and k_row bytes between items and nodes; heads dense) go into k_pool [items][pages][nkv][page_size][k_bytes], and likewise
// the values where v_new is not null.
CELLM_API int cellm_accept_drafts(int* out_count, int* out_path, int* out_next, const int* tokens, const int* parents, const int* choices, const int* cu_seqlens,
                                  int B, int T, int longest, const void* k_new, long long k_item, long long k_row, int k_bytes, void* k_pool, const void* v_new,
                                  long long v_item, long long v_row, int v_bytes, void* v_pool, const int* ctx_lens, const int* block_table, int bt_stride,
                                  int items, int nkv, int pages, int page_size, int* err, cudaStream_t stream) {
    if (B <= 0) return CELLM_OK;
    if (B > 65535 || T < 0 || longest <= 0 || items < 0 || (items > 0 && (nkv <= 0 || pages <= 0 || page_size <= 0 || k_bytes <= 0 || bt_stride < 0))) return CELLM_ERR_SIZE;
    if (!out_count || !out_path || !out_next || !cu_seqlens || !err || (T > 0 && (!tokens || !parents || !choices))) return CELLM_ERR_ARG;
    if (T == 0) items = 0;                // (trees without nodes: nothing stands)
    if (items > 0 && (!k_new || !k_pool || !ctx_lens || !block_table || (v_new && (!v_pool || v_bytes <= 0)))) return CELLM_ERR_ARG;
    const DraftRows k = {items > 0 ? k_new : nullptr, k_pool, k_item, k_row, items > 0 ? k_bytes : 0},
                    v = {items > 0 ? v_new : nullptr, v_pool, v_item, v_row, items > 0 && v_new ? v_bytes : 0};
    uintptr_t at = 0;
    if (k.rows) at |= (uintptr_t)k.rows | (uintptr_t)k.pool | (uintptr_t)k_item | (uintptr_t)k_row | (uintptr_t)k_bytes;
    if (v.rows) at |= (uintptr_t)v.rows | (uintptr_t)v.pool | (uintptr_t)v_item | (uintptr_t)v_row | (uintptr_t)v_bytes;
    const int width = at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 2;
    if (at % 2) return CELLM_ERR_ALIGN;
    // blocks for three kept nodes of every request; more nodes take a block's threads round again
    const long long units = items > 0 ? (long long)items * nkv * ((k.row_bytes + v.row_bytes) / width) * std::min(longest, 3) : 1;
    const dim3 grid((unsigned)std::max<long long>(1, std::min<long long>((units + TREE_MAX - 1) / TREE_MAX, 256)), (unsigned)B);
#define GO(W_) CELLM_RUN(accept_drafts_kernel<W_>, grid, TREE_MAX, 0, stream, out_count, out_path, out_next, tokens, parents, choices, cu_seqlens, T, longest, k, v, \
                         ctx_lens, block_table, bt_stride, items, nkv, pages, page_size, err)
    if (width == 16) GO(uint4);
    else if (width == 4) GO(uint32_t);
    else GO(uint16_t);
#undef GO
    return CELLM_OK;
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_accept_drafts_packed(const long long* a, cudaStream_t stream) {
    return cellm_accept_drafts((int*)a[0], (int*)a[1], (int*)a[2], (const int*)a[3], (const int*)a[4], (const int*)a[5], (const int*)a[6], (int)a[7],
        (int)a[8], (int)a[9], (const void*)a[10], (long long)a[11], (long long)a[12], (int)a[13], (void*)a[14], (const void*)a[15], (long long)a[16],
        (long long)a[17], (int)a[18], (void*)a[19], (const int*)a[20], (const int*)a[21], (int)a[22], (int)a[23], (int)a[24], (int)a[25], (int)a[26],
        (int*)a[27], stream);
}
