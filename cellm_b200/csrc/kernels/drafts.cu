// Which tokens of drafted trees stand, and their keys and values into the cache.
//
// Node 0 of a tree is the token the last step chose; it stands. From a node that stands the walk goes to its child whose token
// is the model's choice after the node (the first among equals), until there is none or `longest` nodes stand; the choice after
// the last node is the request's next token. Every child's test is made at once: a child that fits leaves its place with its
// parent (the smallest stays), and the walk then follows one word a step.
//
// The kept rows of all layers are written to places ctx, ctx + 1, ... of the request's pages. Every block repeats the walk
// (a microsecond at most) and takes its share of the copies, so that one launch does it all.
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
__device__ __forceinline__ void copy_rows(const DraftRows& d, int items, int nkv, int pages, int page_size, const int* path, const int* place_page,
                                          int count, int t_base, int ctx) {
    const int units = d.row_bytes / (int)sizeof(W), per_node = nkv * units;
    const long long total = (long long)items * count * per_node;
    const char* rows = static_cast<const char*>(d.rows);
    W* pool = static_cast<W*>(d.pool);
    for (long long u = (long long)blockIdx.x * blockDim.x + threadIdx.x; u < total; u += (long long)gridDim.x * blockDim.x) {
        const int item = (int)(u / ((long long)count * per_node)), rest = (int)(u % ((long long)count * per_node));
        const int j = rest / per_node, hx = rest % per_node, h = hx / units, x = hx % units;
        const int page = place_page[j];
        if (page < 0) continue;
        const W v = *reinterpret_cast<const W*>(rows + item * d.item_ld + (long long)(t_base + path[j]) * d.row_ld + (long long)hx * sizeof(W));
        pool[((((size_t)item * pages + page) * nkv + h) * page_size + (ctx + j) % page_size) * units + x] = v;
    }
}

template <typename W>
__global__ void __launch_bounds__(256)
accept_drafts_kernel(int* __restrict__ out_count, int* __restrict__ out_path, int* __restrict__ out_next, const int* __restrict__ tokens,
                     const int* __restrict__ parents, const int* __restrict__ choices, const int* __restrict__ cu_seqlens, int T, int longest,
                     const DraftRows k, const DraftRows v, const int* __restrict__ ctx_lens, const int* __restrict__ block_table, int bt_stride,
                     int items, int nkv, int pages, int page_size, int* __restrict__ err) {
    __shared__ int child[TREE_MAX], path[TREE_MAX], place_page[TREE_MAX];
    __shared__ int count_s;
    pdl_wait();
    const int b = blockIdx.y, t_base = cu_seqlens[b];
    int n = cu_seqlens[b + 1] - t_base;
    if (n > TREE_MAX || n < 0 || t_base < 0 || t_base + n > T) {
        if (threadIdx.x == 0) atomicOr(err, CELLM_DEV_BAD_TREE);
        n = 0;
    }
    for (int i = threadIdx.x; i < n; i += blockDim.x) child[i] = TREE_MAX;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int p = parents[t_base + i];
        if (p >= i) atomicOr(err, CELLM_DEV_BAD_TREE);
        else if (p >= 0 && tokens[t_base + i] == choices[t_base + p]) atomicMin(&child[p], i);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int c = 0;
        // (a tree whose first node is padding keeps nothing)
        for (int at = n > 0 && parents[t_base] == -1 ? 0 : n; at < n && c < longest && c < TREE_MAX; at = child[at]) path[c++] = at;
        count_s = c;
    }
    __syncthreads();
    const int count = count_s;
    if (blockIdx.x == 0) {
        for (int j = threadIdx.x; j < longest; j += blockDim.x) out_path[(long long)b * longest + j] = j < count ? path[j] : -1;
        if (threadIdx.x == 0) out_count[b] = count, out_next[b] = count > 0 ? choices[t_base + path[count - 1]] : -1;
    }
    if (items == 0) return;
    const int ctx = ctx_lens[b];
    for (int j = threadIdx.x; j < count; j += blockDim.x) {
        const long long at = ((long long)ctx + j) / page_size;
        int page = ctx >= 0 && at < bt_stride ? block_table[(long long)b * bt_stride + at] : -1;
        if (page < 0 || page >= pages) {
            atomicOr(err, CELLM_DEV_BAD_PAGE);
            page = -1;
        }
        place_page[j] = page;
    }
    __syncthreads();
    copy_rows<W>(k, items, nkv, pages, page_size, path, place_page, count, t_base, ctx);
    if (v.rows != nullptr) copy_rows<W>(v, items, nkv, pages, page_size, path, place_page, count, t_base, ctx);
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
    if (!out_count || !out_path || !out_next || !tokens || !parents || !choices || !cu_seqlens || !err) return CELLM_ERR_ARG;
    if (items > 0 && (!k_new || !k_pool || !ctx_lens || !block_table || (v_new && (!v_pool || v_bytes <= 0)))) return CELLM_ERR_ARG;
    const DraftRows k = {items > 0 ? k_new : nullptr, k_pool, k_item, k_row, k_bytes}, v = {items > 0 ? v_new : nullptr, v_pool, v_item, v_row, v_bytes};
    uintptr_t at = 0;
    if (k.rows) at |= (uintptr_t)k.rows | (uintptr_t)k.pool | (uintptr_t)k_item | (uintptr_t)k_row | (uintptr_t)k_bytes;
    if (v.rows) at |= (uintptr_t)v.rows | (uintptr_t)v.pool | (uintptr_t)v_item | (uintptr_t)v_row | (uintptr_t)v_bytes;
    const int width = at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 2;
    if (at % 2) return CELLM_ERR_ALIGN;
    // blocks for three kept nodes of every request; more nodes take a block's threads round again
    const long long units = items > 0 ? (long long)items * nkv * (k_bytes / width) * std::min(longest, 3) : 1;
    const dim3 grid((unsigned)std::max<long long>(1, std::min<long long>((units + 255) / 256, 256)), (unsigned)B);
#define GO(W_) CELLM_RUN(accept_drafts_kernel<W_>, grid, 256, 0, stream, out_count, out_path, out_next, tokens, parents, choices, cu_seqlens, T, longest, k, v, \
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
