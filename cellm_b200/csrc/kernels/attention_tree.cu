// Attention of drafted trees over the paged cache: every node of a request's tree sees the request's committed keys (all of
// them, or those of its window) and, among the nodes, its ancestors and itself,
//     o_i = sum_j w_ij v_j,   w_i = softmax over the keys j that i sees of  scale q_i . k_j,
// node i standing at position ctx + depth(i). The committed keys and values lie in pages, the nodes' own in rows beside the
// cache (only what is accepted later moves into pages), so the keys are walked in blocks of two kinds: committed ones by
// position, then the nodes by their place in the tree, each with a mask of one bit a key.
//
// Sums, maxima and the output's accumulators are 32-bit; a row is rounded once, when it is written (the tensor-core kernel
// rounds the weights too). Where the keys are cut into pieces (few rows, long contexts), a piece leaves its maximum, sum and
// unnormalised output in a workspace, and a second kernel merges them in their order.
#include <algorithm>
#include <climits>

#include "attention_tree.cuh"
#include "mma_tiles.cuh"

namespace {

// ---------------------------------------------------------------- any type, any head size up to 256
// 128 threads take 32 rows ((node, query head) pairs of one key/value head) through blocks of KT keys in 32-bit arithmetic: a
// thread forms 4 x KT/16 scores out of shared memory, a row's maximum and sum go over half a warp, and the thread then owns 4 x
// HDP/16 entries of the output.
template <int HDP> struct PlainTile { static constexpr int KEYS = HDP <= 128 ? 64 : 32; };

template <typename T>
__device__ __forceinline__ void row_to_floats(float* dst, const T* src, int hd, int padded, int lane, int lanes, bool quads) {
    if (quads) {
        for (int d = lane * 4; d < padded; d += lanes * 4) {
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (src != nullptr && d < hd) {
                if constexpr (sizeof(T) == 4) {
                    f = *reinterpret_cast<const float4*>(src + d);
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(src + d);
                    f = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
                }
            }
            *reinterpret_cast<float4*>(dst + d) = f;
        }
    } else {
        for (int d = lane; d < padded; d += lanes) dst[d] = src != nullptr && d < hd ? to_float(src[d]) : 0.f;
    }
}

template <typename T, int HDP>
__global__ void __launch_bounds__(128)
attention_tree_plain_kernel(const TreeArgs a, int quads) {
    constexpr int RT = 32, KT = PlainTile<HDP>::KEYS, LD = HDP + 4, KC = KT / 16;
    constexpr int VEC = HDP % 64 == 0 ? 4 : 2, NV = HDP / (16 * VEC);
    extern __shared__ __align__(16) uint8_t plain_smem[];
    TreeShape& tree = *reinterpret_cast<TreeShape*>(plain_smem);
    float* qs = reinterpret_cast<float*>(plain_smem + sizeof(TreeShape));     // [RT][LD]
    float* ks = qs + RT * LD;                                          // [KT][LD]
    float* vs = ks + KT * LD;                                          // [KT][LD]
    float* ps = vs + KT * LD;                                          // [KT][RT + 4]
    pdl_wait();
    pdl_trigger();
    const TreeTile t = tree_tile(a);
    const int G = a.nh / a.nkv, rows = t.n * G;
    if (!t.live || t.tile * RT >= rows) return;
    read_tree(tree, a.parents + t.t_base, t.n, a.window, a.err);

    const int hd = a.hd, rg = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp; r < RT; r += 4) {
        const int row = t.tile * RT + r;
        const T* src = row < rows ? static_cast<const T*>(a.q) + (long long)(t.t_base + row / G) * a.q_ld + (long long)(t.kvh * G + row % G) * hd : nullptr;
        row_to_floats(qs + r * LD, src, hd, HDP, lane, 32, quads);
    }
    // a thread's rows are rg, rg + 8, rg + 16, rg + 24 of the tile
    int node[4];
    float m[4], l[4], o[4][NV * VEC];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = t.tile * RT + rg + i * 8;
        node[i] = row < rows && tree.depth[row / G] >= 0 ? row / G : -1;
        m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < NV * VEC; ++d) o[i][d] = 0.f;
    }
    const int lo = a.window > 0 ? max(0, t.ctx - a.window + 1) : 0;
    const int first = lo / KT, committed = lo < t.ctx ? (t.ctx + KT - 1) / KT - first : 0, blocks = committed + (t.n + KT - 1) / KT;
    const int per = (blocks + a.nsplit - 1) / a.nsplit, begin = min(blocks, t.split * per), end = min(blocks, begin + per);
    const int* bt = a.block_table + (size_t)t.b * a.bt_stride;
    for (int blk = begin; blk < end; ++blk) {
        const bool paged = blk < committed;
        const int key0 = (first + blk) * KT, node0 = paged ? -1 : (blk - committed) * KT;
        __syncthreads();
        for (int r = warp; r < KT; r += 4) {
            const T *k = nullptr, *v = nullptr;
            if (paged) {
                const int j = key0 + r;
                if (j >= lo && j < t.ctx) {
                    const int page = bt[j / a.page_size];
                    if (page < 0 || page >= a.num_pages) {
                        if (lane == 0) atomicOr(a.err, CELLM_DEV_BAD_PAGE);
                    } else {
                        const size_t off = (((size_t)page * a.nkv + t.kvh) * a.page_size + j % a.page_size) * hd;
                        k = static_cast<const T*>(a.k_pool) + off, v = static_cast<const T*>(a.v_pool) + off;
                    }
                }
            } else if (node0 + r < t.n && tree.depth[node0 + r] >= 0) {
                k = static_cast<const T*>(a.k_new) + (long long)(t.t_base + node0 + r) * a.k_ld + (long long)t.kvh * hd;
                v = static_cast<const T*>(a.v_new) + (long long)(t.t_base + node0 + r) * a.v_ld + (long long)t.kvh * hd;
            }
            row_to_floats(ks + r * LD, k, hd, HDP, lane, 32, quads);
            row_to_floats(vs + r * LD, v, hd, HDP, lane, 32, quads);
        }
        __syncthreads();
        float s[4][KC];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < KC; ++k) s[i][k] = 0.f;
#pragma unroll 2
        for (int d = 0; d < HDP; d += 4) {
            float4 q4[4], k4[KC];
#pragma unroll
            for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const float4*>(qs + (rg + i * 8) * LD + d);
#pragma unroll
            for (int k = 0; k < KC; ++k) k4[k] = *reinterpret_cast<const float4*>(ks + (c + k * 16) * LD + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < KC; ++k)
                    s[i][k] = fmaf(q4[i].w, k4[k].w, fmaf(q4[i].z, k4[k].z, fmaf(q4[i].y, k4[k].y, fmaf(q4[i].x, k4[k].x, s[i][k]))));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t seen = node[i] >= 0 ? seen_bits<KT>(tree, node[i], a.window, t.ctx, key0, node0) : 0ull;
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                s[i][k] = (seen >> (c + k * 16) & 1ull) ? s[i][k] * a.scale_log2e : -INFINITY;
                top = fmaxf(top, s[i][k]);
            }
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float now = fmaxf(m[i], top), use = now == -INFINITY ? 0.f : now, corr = exp2f(m[i] - use);
            m[i] = now;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                const float p = exp2f(s[i][k] - use);
                sum += p;
                ps[(c + k * 16) * (RT + 4) + rg * 4 + i] = p;
            }
            l[i] = l[i] * corr + sum;
#pragma unroll
            for (int d = 0; d < NV * VEC; ++d) o[i][d] *= corr;
        }
        __syncwarp();                          // a half-warp writes and reads the columns of its own rows alone
#pragma unroll 4
        for (int k = 0; k < KT; ++k) {
            const float4 p = *reinterpret_cast<const float4*>(ps + k * (RT + 4) + rg * 4);
#pragma unroll
            for (int g = 0; g < NV; ++g) {
                float v[VEC];
                const float* src = vs + k * LD + (g * 16 + c) * VEC;
                if constexpr (VEC == 4) {
                    const float4 w = *reinterpret_cast<const float4*>(src);
                    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
                } else {
                    const float2 w = *reinterpret_cast<const float2*>(src);
                    v[0] = w.x, v[1] = w.y;
                }
#pragma unroll
                for (int x = 0; x < VEC; ++x) {
                    o[0][g * VEC + x] = fmaf(p.x, v[x], o[0][g * VEC + x]);
                    o[1][g * VEC + x] = fmaf(p.y, v[x], o[1][g * VEC + x]);
                    o[2][g * VEC + x] = fmaf(p.z, v[x], o[2][g * VEC + x]);
                    o[3][g * VEC + x] = fmaf(p.w, v[x], o[3][g * VEC + x]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
        const int row = t.tile * RT + rg + i * 8;
        if (row >= rows) continue;
        const long long gr = (long long)(t.t_base + row / G) * a.nh + t.kvh * G + row % G;
        if (a.nsplit > 1) {
            float* dst = a.part_o + ((long long)t.split * a.T * a.nh + gr) * hd;
#pragma unroll
            for (int g = 0; g < NV; ++g)
#pragma unroll
                for (int x = 0; x < VEC; ++x)
                    if ((g * 16 + c) * VEC + x < hd) dst[(g * 16 + c) * VEC + x] = o[i][g * VEC + x];
            if (c == 0) {
                float* ml = a.part_ml + ((long long)t.split * a.T * a.nh + gr) * 2;
                ml[0] = m[i], ml[1] = l[i];
            }
        } else {
            const float inv = l[i] > 0.f ? 1.f / l[i] : l[i];          // 0 where nothing is seen; NaN stays
            T* dst = static_cast<T*>(a.out) + gr * hd;
#pragma unroll
            for (int g = 0; g < NV; ++g)
#pragma unroll
                for (int x = 0; x < VEC; ++x)
                    if ((g * 16 + c) * VEC + x < hd) dst[(g * 16 + c) * VEC + x] = from_float<T>(o[i][g * VEC + x] * inv);
        }
    }
}

// ---------------------------------------------------------------- bfloat16, head sizes 32, 64, 96, 128: mma.sync
// Four warps take 16 * RG rows through blocks of 64 keys that all threads bring in with cp.async (a ring of ST stages, one barrier
// a block). RG groups of 16 rows share a block; the 4 / RG warps of a group take its keys in equal parts, each with a softmax
// state of its own, and meet in shared memory at the end. Few rows (small trees) so still use every warp.
template <int HD, int RG>
struct MmaTile {
    static constexpr int KG = 4 / RG, RT = 16 * RG;
    static constexpr int ST = HD <= 32 ? 4 : HD <= 96 ? 3 : 2;
    static constexpr int KV = FA_BN * HD * 2;
    static constexpr int q_off = 0, kv_off = RT * HD * 2, tree_off = kv_off + ST * 2 * KV, bytes = tree_off + (int)sizeof(TreeShape);
    static_assert(4 * 16 * (HD + 2) * 4 <= ST * 2 * KV, "the warps' outputs must fit the ring");
};

template <int HD, int RG>
__global__ void __launch_bounds__(128)
attention_tree_mma_kernel(const TreeArgs a) {
    using L = MmaTile<HD, RG>;
    constexpr int BN = FA_BN, CH = HD / 8, NT = HD / 8, ST = L::ST, KG = L::KG, WK = BN / KG, ITERS = BN * CH / 128;
    extern __shared__ __align__(128) uint8_t mma_smem[];
    uint8_t *q_s = mma_smem + L::q_off, *kv_s = mma_smem + L::kv_off;
    TreeShape& tree = *reinterpret_cast<TreeShape*>(mma_smem + L::tree_off);
    pdl_wait();
    pdl_trigger();
    const TreeTile t = tree_tile(a);
    const int G = a.nh / a.nkv, rows = t.n * G, row0 = t.tile * L::RT;
    if (!t.live || row0 >= rows) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rg = warp % RG, kg = warp / RG;

    const int lo = a.window > 0 ? max(0, t.ctx - a.window + 1) : 0;
    const int first = lo / BN, committed = lo < t.ctx ? (t.ctx + BN - 1) / BN - first : 0, blocks = committed + (t.n + BN - 1) / BN;
    const int per = (blocks + a.nsplit - 1) / a.nsplit, begin = min(blocks, t.split * per), n_blk = min(blocks, begin + per) - begin;
    const int* bt = a.block_table + (size_t)t.b * a.bt_stride;
    const int shift = (a.page_size & (a.page_size - 1)) == 0 ? __ffs(a.page_size) - 1 : -1;
    const size_t page_elems = (size_t)a.nkv * a.page_size * HD;
    // this thread's rows of a block lie 128 / CH apart; the table's entries of the block after the next are under way while
    // a block is computed
    const int row_t = threadIdx.x / CH, chunk_t = threadIdx.x % CH;
    constexpr bool EVEN = 128 % CH == 0;
    auto row_of = [&](int it) { return EVEN ? row_t + it * (128 / CH) : (threadIdx.x + it * 128) / CH; };
    auto chunk_of = [&](int it) { return EVEN ? chunk_t : (threadIdx.x + it * 128) % CH; };
    int entry[ITERS];
    auto look_up = [&](int i) {
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            const int blk = begin + i, j = (first + blk) * BN + row_of(it);
            entry[it] = i < n_blk && blk < committed && j >= lo && j < t.ctx ? bt[shift >= 0 ? j >> shift : j / a.page_size] : -2;
        }
    };
    auto load_kv = [&](int i) {
        if (i < n_blk) {
            uint8_t* ks = kv_s + (size_t)(i % ST) * 2 * L::KV;
            const int blk = begin + i;
#pragma unroll
            for (int it = 0; it < ITERS; ++it) {
                const int row = row_of(it), chunk = chunk_of(it);
                const __nv_bfloat16 *k = static_cast<const __nv_bfloat16*>(a.k_pool), *v = static_cast<const __nv_bfloat16*>(a.v_pool);
                bool have = false;
                if (blk < committed) {
                    const int j = (first + blk) * BN + row, page = entry[it];
                    if (page >= 0 && page < a.num_pages) {
                        const size_t off = (size_t)page * page_elems + ((size_t)t.kvh * a.page_size + (shift >= 0 ? j & (a.page_size - 1) : j % a.page_size)) * HD + chunk * 8;
                        k += off, v += off, have = true;
                    } else if (page != -2) {
                        atomicOr(a.err, CELLM_DEV_BAD_PAGE);
                    }
                } else {
                    const int node = (blk - committed) * BN + row;
                    if (node < t.n && tree.depth[node] >= 0) {
                        k = static_cast<const __nv_bfloat16*>(a.k_new) + (t.t_base + node) * a.k_ld + t.kvh * HD + chunk * 8;
                        v = static_cast<const __nv_bfloat16*>(a.v_new) + (t.t_base + node) * a.v_ld + t.kvh * HD + chunk * 8;
                        have = true;
                    }
                }
                cp_async16(ks + tile_offset<HD>(row, chunk), k, have ? 16 : 0);
                cp_async16(ks + L::KV + tile_offset<HD>(row, chunk), v, have ? 16 : 0);
            }
        }
        cp_async_commit();
    };
    // Committed blocks leave before the tree's shape is known; the nodes' own wait for it.
    look_up(0);
    for (int i = threadIdx.x; i < L::RT * CH; i += 128) {
        const int r = i / CH, chunk = i % CH, row = min(row0 + r, rows - 1);
        cp_async16(q_s + tile_offset<HD>(r, chunk), static_cast<const __nv_bfloat16*>(a.q) + (t.t_base + row / G) * a.q_ld + (t.kvh * G + row % G) * HD + chunk * 8, 16);
    }
    const int old = max(0, min(min(n_blk, ST - 1), committed - begin));
    for (int i = 0; i < old; ++i) {
        load_kv(i);
        look_up(i + 1);
    }
    read_tree(tree, a.parents + t.t_base, t.n, a.window, a.err);
    for (int i = old; i < ST - 1; ++i) {
        load_kv(i);
        look_up(i + 1);
    }
    const int ra = row0 + rg * 16 + (lane >> 2), rb = ra + 8;
    const int node_a = ra < rows && tree.depth[ra / G] >= 0 ? ra / G : -1, node_b = rb < rows && tree.depth[rb / G] >= 0 ? rb / G : -1;
    const int open_from = a.window > 0 ? t.ctx + t.n - a.window : 0;        // no row's window starts behind it
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    uint32_t qf[HD / 16][4];

    for (int i = 0; i < n_blk; ++i) {
        cp_async_wait<ST - 2>();
        __syncthreads();
        if (i == 0) {
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) ldmatrix_x4(qf[ks], q_s + tile_offset<HD>(rg * 16 + (lane & 15), ks * 2 + (lane >> 4)));
        }
        load_kv(i + ST - 1);               // into the stage that everybody left before the barrier
        look_up(i + ST);
        const uint8_t *k_s = kv_s + (size_t)(i % ST) * 2 * L::KV, *v_s = k_s + L::KV;
        const int k0 = kg * WK;
        float s[WK / 8][4];
#pragma unroll
        for (int n = 0; n < WK / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
#pragma unroll
            for (int n2 = 0; n2 < WK / 16; ++n2) {
                uint32_t kf[4];
                ldmatrix_x4(kf, k_s + tile_offset<HD>(k0 + n2 * 16 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
                mma_bf16(s[2 * n2], qf[ks], kf[0], kf[1]);
                mma_bf16(s[2 * n2 + 1], qf[ks], kf[2], kf[3]);
            }
        }
        const int blk = begin + i, key0 = (first + blk) * BN;
        const bool paged = blk < committed;
        if (!paged || key0 + BN > t.ctx || key0 < open_from) {
            const int node0 = paged ? -1 : (blk - committed) * BN;
            const uint64_t see_a = node_a >= 0 ? seen_bits<BN>(tree, node_a, a.window, t.ctx, key0, node0) >> (k0 + (lane & 3) * 2) : 0ull;
            const uint64_t see_b = node_b >= 0 ? seen_bits<BN>(tree, node_b, a.window, t.ctx, key0, node0) >> (k0 + (lane & 3) * 2) : 0ull;
#pragma unroll
            for (int n = 0; n < WK / 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[n][e] = (see_a >> (n * 8 + e) & 1ull) ? s[n][e] * a.scale_log2e : -INFINITY;
                    s[n][2 + e] = (see_b >> (n * 8 + e) & 1ull) ? s[n][2 + e] * a.scale_log2e : -INFINITY;
                }
        } else {
#pragma unroll
            for (int n = 0; n < WK / 8; ++n) s[n][0] *= a.scale_log2e, s[n][1] *= a.scale_log2e, s[n][2] *= a.scale_log2e, s[n][3] *= a.scale_log2e;
        }
        float mx_a = -INFINITY, mx_b = -INFINITY;
#pragma unroll
        for (int n = 0; n < WK / 8; ++n) mx_a = fmaxf(mx_a, fmaxf(s[n][0], s[n][1])), mx_b = fmaxf(mx_b, fmaxf(s[n][2], s[n][3]));
        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
        const float mn_a = fmaxf(m_a, mx_a), mn_b = fmaxf(m_b, mx_b);
        const float use_a = mn_a == -INFINITY ? 0.f : mn_a, use_b = mn_b == -INFINITY ? 0.f : mn_b;
        const float corr_a = fast_exp2(m_a - use_a), corr_b = fast_exp2(m_b - use_b);
        m_a = mn_a, m_b = mn_b;
        float sum_a = 0.f, sum_b = 0.f;
        uint32_t pf[WK / 16][4];
#pragma unroll
        for (int n = 0; n < WK / 8; ++n) {
            const float p0 = fast_exp2(s[n][0] - use_a), p1 = fast_exp2(s[n][1] - use_a);
            const float p2 = fast_exp2(s[n][2] - use_b), p3 = fast_exp2(s[n][3] - use_b);
            sum_a += p0 + p1, sum_b += p2 + p3;
            pf[n >> 1][(n & 1) * 2] = pack_bf16(p0, p1);               // the weights' rounding: what the tensor cores' operand holds
            pf[n >> 1][(n & 1) * 2 + 1] = pack_bf16(p2, p3);
        }
        l_a = l_a * corr_a + sum_a, l_b = l_b * corr_b + sum_b;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][0] *= corr_a, o[n][1] *= corr_a, o[n][2] *= corr_b, o[n][3] *= corr_b;
#pragma unroll
        for (int kk = 0; kk < WK / 16; ++kk) {
#pragma unroll
            for (int n2 = 0; n2 < NT / 2; ++n2) {
                uint32_t vf[4];
                ldmatrix_x4_trans(vf, v_s + tile_offset<HD>(k0 + kk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), n2 * 2 + (lane >> 4)));
                mma_bf16(o[2 * n2], pf[kk], vf[0], vf[1]);
                mma_bf16(o[2 * n2 + 1], pf[kk], vf[2], vf[3]);
            }
        }
    }
    cp_async_wait<0>();
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
    l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);

    // the warps' results meet in shared memory, where the ring was; 16 lanes of a warp then write a row together
    __syncthreads();
    float* o_s = reinterpret_cast<float*>(kv_s);                                       // [4][16][HD]
    float* ml_s = o_s + 4 * 16 * HD;                                                   // [4][16][2]
    {
        const int r = lane >> 2, col = (lane & 3) * 2;
        float* ow = o_s + warp * 16 * HD;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2*>(ow + r * HD + n * 8 + col) = make_float2(o[n][0], o[n][1]);
            *reinterpret_cast<float2*>(ow + (r + 8) * HD + n * 8 + col) = make_float2(o[n][2], o[n][3]);
        }
        if ((lane & 3) == 0) {
            ml_s[(warp * 16 + r) * 2] = m_a, ml_s[(warp * 16 + r) * 2 + 1] = l_a;
            ml_s[(warp * 16 + r + 8) * 2] = m_b, ml_s[(warp * 16 + r + 8) * 2 + 1] = l_b;
        }
    }
    __syncthreads();
    for (int r = threadIdx.x >> 4; r < L::RT; r += 8) {
        const int row = row0 + r, c = threadIdx.x & 15;
        if (row >= rows) break;
        const bool seen = tree.depth[row / G] >= 0;
        float M = -INFINITY;
#pragma unroll
        for (int g = 0; g < KG; ++g) M = fmaxf(M, ml_s[((g * RG + r / 16) * 16 + r % 16) * 2]);
        const float use = M == -INFINITY ? 0.f : M;
        float f[KG], l = 0.f;
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            const float* ml = ml_s + ((g * RG + r / 16) * 16 + r % 16) * 2;
            f[g] = exp2f(ml[0] - use);
            l += f[g] * ml[1];
        }
        const long long gr = (long long)(t.t_base + row / G) * a.nh + t.kvh * G + row % G;
        const float inv = !seen || l == 0.f ? 0.f : 1.f / l;
        if (a.nsplit > 1 && c == 0)
            *reinterpret_cast<float2*>(a.part_ml + ((long long)t.split * a.T * a.nh + gr) * 2) = seen ? make_float2(M, l) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int d = c * 2; d < HD; d += 32) {
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int g = 0; g < KG; ++g) {
                const float2 v = *reinterpret_cast<const float2*>(o_s + ((g * RG + r / 16) * 16 + r % 16) * HD + d);
                acc.x = fmaf(f[g], v.x, acc.x), acc.y = fmaf(f[g], v.y, acc.y);
            }
            if (a.nsplit > 1) *reinterpret_cast<float2*>(a.part_o + ((long long)t.split * a.T * a.nh + gr) * HD + d) = seen ? acc : make_float2(0.f, 0.f);
            else *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + gr * HD + d) = seen ? pack_bf16(acc.x * inv, acc.y * inv) : 0u;
        }
    }
}

// The pieces of a row merged in their order: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s. A warp takes a row.
template <typename T>
__global__ void __launch_bounds__(256)
attention_tree_merge_kernel(T* __restrict__ out, const float* __restrict__ part_o, const float* __restrict__ part_ml, long long rows, int hd, int nsplit) {
    pdl_wait();
    pdl_trigger();
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (r >= rows) return;
    float M = -INFINITY;
    for (int s = lane; s < nsplit; s += 32) M = fmaxf(M, part_ml[(s * rows + r) * 2]);
    M = warp_max(M);
    const float use = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    for (int s = 0; s < nsplit; ++s) L = fmaf(exp2f(part_ml[(s * rows + r) * 2] - use), part_ml[(s * rows + r) * 2 + 1], L);
    const float inv = L > 0.f ? 1.f / L : L;
    for (int d = lane; d < hd; d += 32) {
        float acc = 0.f;
        for (int s = 0; s < nsplit; ++s) {
            const float w = exp2f(part_ml[(s * rows + r) * 2] - use);
            if (w != 0.f) acc = fmaf(w, part_o[(s * rows + r) * hd + d], acc);       // (a piece that sees nothing holds zeros)
        }
        out[r * hd + d] = from_float<T>(acc * inv);
    }
}

template <typename T, int HDP>
int launch_plain(const TreeArgs& a, cudaStream_t stream) {
    constexpr int KT = PlainTile<HDP>::KEYS, LD = HDP + 4;
    const size_t smem = sizeof(TreeShape) + (size_t)((32 + 2 * KT) * LD + KT * 36) * 4;
    cudaError_t e = cudaFuncSetAttribute(attention_tree_plain_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool;
    const int quads = a.hd % 4 == 0 && a.q_ld % 4 == 0 && a.k_ld % 4 == 0 && a.v_ld % 4 == 0 && at % (4 * sizeof(T)) == 0;
    CELLM_RUN((attention_tree_plain_kernel<T, HDP>), (unsigned)((long long)a.B * a.nkv * a.nsplit * a.tiles), 128, smem, stream, a, quads);
    return CELLM_OK;
}

template <typename T>
int launch_plain_sized(const TreeArgs& a, cudaStream_t stream) {
    if (a.hd <= 32) return launch_plain<T, 32>(a, stream);
    if (a.hd <= 64) return launch_plain<T, 64>(a, stream);
    if (a.hd <= 96) return launch_plain<T, 96>(a, stream);
    if (a.hd <= 128) return launch_plain<T, 128>(a, stream);
    return launch_plain<T, 256>(a, stream);
}

template <int HD, int RG>
int launch_mma(TreeArgs a, cudaStream_t stream) {
    using L = MmaTile<HD, RG>;
    cudaError_t e = cudaFuncSetAttribute(attention_tree_mma_kernel<HD, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::bytes);
    if (e != cudaSuccess) return (int)e;
    a.tiles = (a.most * (a.nh / a.nkv) + L::RT - 1) / L::RT;
    CELLM_RUN((attention_tree_mma_kernel<HD, RG>), (unsigned)((long long)a.B * a.nkv * a.nsplit * a.tiles), 128, L::bytes, stream, a);
    return CELLM_OK;
}
template <int HD>
int launch_mma_rows(const TreeArgs& a, cudaStream_t stream) {
    const int rows = a.most * (a.nh / a.nkv);
    return rows <= 16 ? launch_mma<HD, 1>(a, stream) : rows <= 32 ? launch_mma<HD, 2>(a, stream) : launch_mma<HD, 4>(a, stream);
}
// Whether the tensor-core kernel takes a call: its copies are 16 bytes wide.
bool mma_takes(const TreeArgs& a) {
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool | (uintptr_t)a.out;
    return (a.hd == 32 || a.hd == 64 || a.hd == 96 || a.hd == 128) && at % 16 == 0 && a.q_ld % 8 == 0 && a.k_ld % 8 == 0 && a.v_ld % 8 == 0;
}
// Trees that fill tiles of 128 rows go to the tcgen05 kernel.
bool tc_rows(int rows) { return rows > 64; }
int launch_bf16(const TreeArgs& a, cudaStream_t stream) {
    const int G = a.nh / a.nkv;
    if (tc_rows(a.most * G) && attention_tree_tc_takes(a) && (a.most > 128 / G || a.nsplit % 2 == 0)) {
        TreeArgs b = a;
        if (a.most <= 128 / G) b.nsplit /= 2;               // its two tiles leave a piece each
        return attention_tree_tc_launch(b, stream);
    }
    if (!mma_takes(a)) return launch_plain_sized<__nv_bfloat16>(a, stream);
    if (a.hd == 32) return launch_mma_rows<32>(a, stream);
    if (a.hd == 64) return launch_mma_rows<64>(a, stream);
    if (a.hd == 96) return launch_mma_rows<96>(a, stream);
    return launch_mma_rows<128>(a, stream);
}

// How many pieces the keys of a tile of rows are cut into: of all counts the one whose rounds of blocks, each as long as its keys
// and a few blocks' worth of start and merge, take the least time.
int pieces(long long tiles, int key_blocks, long long at_once) {
    constexpr int START = 3;
    int best = 1;
    long long least = LLONG_MAX;
    for (int n = 1; n <= 64 && n <= std::max(1, key_blocks); ++n) {
        const long long cost = (tiles * n + at_once - 1) / at_once * ((key_blocks + n - 1) / n + START) + (n > 1 ? START : 0);
        if (cost < least) least = cost, best = n;
    }
    return best;
}

template <typename T>
int launch_merge(const TreeArgs& a, cudaStream_t stream) {
    const long long rows = (long long)a.T * a.nh;
    CELLM_RUN(attention_tree_merge_kernel<T>, (unsigned)((rows + 7) / 8), 256, 0, stream, (T*)a.out, a.part_o, a.part_ml, rows, a.hd, a.nsplit);
    return CELLM_OK;
}

}  // namespace

// The pieces the keys are best cut into: B trees of up to `most` nodes, `keys` the most that a node sees.
CELLM_API int cellm_attention_tree_pieces(int B, int most, int nh, int nkv, int hd, int keys, int dtype, int sms) {
    if (B <= 0 || most <= 0 || nkv <= 0 || nh < nkv) return 1;
    const int G = nh / nkv, rows = most * G;
    if (dtype == CELLM_BF16 && hd == 64 && tc_rows(rows) && G <= 128 && 128 / G * G >= 96) {
        const int tile = 128 / G, two = most > tile;
        const int n = pieces((long long)B * nkv * ((most + (1 + two) * tile - 1) / ((1 + two) * tile)), ((keys + 127) / 128 + 1 - two) / (2 - two), sms);
        return two ? n : 2 * n;
    }
    const bool mma = dtype == CELLM_BF16 && (hd == 32 || hd == 64 || hd == 96 || hd == 128);
    const int tile = !mma || (rows > 16 && rows <= 32) ? 32 : rows <= 16 ? 16 : 64;
    const int an_sm = !mma ? 2 : hd == 32 ? 4 : hd == 64 ? 3 : 2;             // blocks that an SM holds, by their shared memory
    return pieces((long long)B * nkv * ((rows + tile - 1) / tile), (keys + 63) / 64, (long long)an_sm * sms);
}

// out [T, nh * hd], q rows q_ld elements apart, the nodes' keys and values in rows k_ld and v_ld apart ([nkv * hd] each), parents
// [T]; request b owns the nodes cu_seqlens[b] .. cu_seqlens[b + 1] (at most 256, `most` of them in the largest tree) behind
// ctx_lens[b] committed tokens in the pages of its row of the block table. nsplit pieces of the keys need part_o [nsplit, T * nh,
// hd] and part_ml [nsplit, T * nh, 2] floats.
CELLM_API int cellm_attention_tree(void* out, float* part_o, float* part_ml, const void* q, long long q_ld, const void* k_new, long long k_ld,
                                   const void* v_new, long long v_ld, const int* parents, const void* k_pool, const void* v_pool,
                                   const int* cu_seqlens, const int* ctx_lens, const int* block_table, int bt_stride, int B, int T, int most,
                                   int num_pages, int page_size, int nh, int nkv, int hd, float scale, int window, int nsplit, int dtype, int* err,
                                   cudaStream_t stream) {
    if (T <= 0 || B <= 0 || most <= 0) return CELLM_OK;
    if (dtype != CELLM_F32 && dtype != CELLM_BF16) return CELLM_ERR_DTYPE;
    if (nkv <= 0 || nh <= 0 || nh % nkv || hd <= 0 || hd > 256 || page_size <= 0 || most > TREE_MAX || bt_stride < 0 || window < 0) return CELLM_ERR_SIZE;
    if (nsplit < 1 || nsplit > 128) return CELLM_ERR_SIZE;
    if (nsplit > 1 && (!part_o || !part_ml)) return CELLM_ERR_ARG;
    if (!out || !q || !k_new || !v_new || !parents || !cu_seqlens || !ctx_lens || !err) return CELLM_ERR_ARG;
    TreeArgs a = {out, part_o, part_ml, q, k_new, v_new, q_ld, k_ld, v_ld, parents, k_pool, v_pool, cu_seqlens, ctx_lens, block_table,
                  bt_stride, B, T, most, num_pages, page_size, nh, nkv, hd, 0, nsplit, window, scale * 1.4426950408889634f, err};
    a.tiles = (most * (nh / nkv) + 31) / 32;
    if ((long long)B * nkv * nsplit * a.tiles > 0x7fffffffLL) return CELLM_ERR_SIZE;
    int rc = dtype == CELLM_F32 ? launch_plain_sized<float>(a, stream) : launch_bf16(a, stream);
    if (rc != CELLM_OK || nsplit == 1) return rc;
    return dtype == CELLM_F32 ? launch_merge<float>(a, stream) : launch_merge<__nv_bfloat16>(a, stream);
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_attention_tree_packed(const long long* a, cudaStream_t stream) {
    return cellm_attention_tree((void*)a[0], (float*)a[1], (float*)a[2], (const void*)a[3], (long long)a[4], (const void*)a[5], (long long)a[6],
        (const void*)a[7], (long long)a[8], (const int*)a[9], (const void*)a[10], (const void*)a[11], (const int*)a[12], (const int*)a[13],
        (const int*)a[14], (int)a[15], (int)a[16], (int)a[17], (int)a[18], (int)a[19], (int)a[20], (int)a[21], (int)a[22], (int)a[23],
        (float)cellm_packed_double(a[24]), (int)a[25], (int)a[26], (int)a[27], (int*)a[28], stream);
}
