// Attention of drafted trees over the paged cache: every node of a request's tree sees the request's committed keys (all of
// them, or those of its window) and, among the nodes, its ancestors and itself,
//     o_i = sum_j w_ij v_j,   w_i = softmax over the keys j that i sees of  scale q_i . k_j,
// node i standing at position ctx + depth(i). The committed keys and values lie in pages, the nodes' own in rows beside the
// cache (only what is accepted later moves into pages), so the keys are walked in blocks of two kinds: committed ones by
// position, then the nodes by their place in the tree, each with a mask of one bit a key.
//
// Sums, maxima and the output's accumulators are 32-bit; a row is rounded once, when it is written (the tensor-core kernel
// rounds the weights too). Where the keys are cut into pieces (few rows, long contexts), up to eight pieces are one thread-block cluster:
// each keeps its maximum, sum and unnormalised output in its shared memory, and every CTA merges a share of the rows out of its
// peers' memory. More pieces leave them in a workspace, and a second kernel merges. Either way in the pieces' order.
#include <algorithm>
#include <climits>

#include "attention_tree.cuh"
#include "mma_tiles.cuh"
#include "pairs.cuh"

namespace {

// ---------------------------------------------------------------- a tile's results
// The barrier's forms here are executed by a warp as a whole; what comes before may have taken its lanes through loops of different
// lengths (two rows a warp, columns that are no multiple of 32), so they meet first.
__device__ __forceinline__ void cluster_meet() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What lies at `local` in the shared memory of CTA `rank` of this cluster.
__device__ __forceinline__ float2 peer_pair(const float* local, uint32_t rank) {
    uint32_t addr;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
template <typename T>
__device__ __forceinline__ void write_pair(T* out, float2 v, bool both) {
    if constexpr (sizeof(T) == 2) {
        if (both) *reinterpret_cast<uint32_t*>(out) = pack_bf16(v.x, v.y);
        else out[0] = from_float<T>(v.x);
    } else {
        if (both) *reinterpret_cast<float2*>(out) = v;
        else out[0] = v.x;
    }
}

// The block's rows, row0 .. row0 + RT - 1 of the tree's (node, head) pairs: o [RT][LD] and ml [RT][2] (maximum and sum) in shared
// memory, written before a barrier. 16 threads take a row. Rows of padding become zeros.
template <typename T, bool CL>
__device__ __forceinline__ void finish_rows(const TreeArgs& a, const TreeTile& t, const TreeShape& tree, const float* o, int LD, const float* ml, int RT, int row0) {
    const int G = a.nh / a.nkv, rows = t.n * G, hd = a.hd, c = threadIdx.x & 15;
    const bool even = hd % 2 == 0;
    if constexpr (CL) cluster_meet();                   // every piece of the rows is there
    const int first = CL ? t.split : 0, step = CL ? a.nsplit : 1;
    for (int r = first + (threadIdx.x >> 4) * step; r < RT && row0 + r < rows; r += (blockDim.x >> 4) * step) {
        const int node = (row0 + r) / G;
        const bool seen = tree.depth[node] >= 0;
        const long long gr = (long long)(t.t_base + node) * a.nh + t.kvh * G + (row0 + r) % G;
        if (!CL && a.nsplit > 1) {
            if (c == 0) *reinterpret_cast<float2*>(a.part_ml + ((long long)t.split * a.T * a.nh + gr) * 2) = seen ? make_float2(ml[r * 2], ml[r * 2 + 1]) : make_float2(-INFINITY, 0.f);
            float* dst = a.part_o + ((long long)t.split * a.T * a.nh + gr) * hd;
            for (int d = c; d < hd; d += 16) dst[d] = seen ? o[r * LD + d] : 0.f;
            continue;
        }
        float weight[CL ? 8 : 1], l = 0.f;
        if constexpr (CL) {
            float2 all[8];
            float M = -INFINITY;
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                all[s] = s < a.nsplit ? peer_pair(ml + r * 2, s) : make_float2(-INFINITY, 0.f);
                M = fmaxf(M, all[s].x);
            }
            const float use = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int s = 0; s < 8; ++s) weight[s] = exp2f(all[s].x - use), l = fmaf(weight[s], all[s].y, l);
        } else {
            weight[0] = 1.f, l = ml[r * 2 + 1];
        }
        const float inv = l != 0.f ? 1.f / l : 0.f;                            // 0 where nothing is seen; NaN stays
        for (int d = c * 2; d < hd; d += 32) {
            float2 v = make_float2(0.f, 0.f);
            if constexpr (CL) {
                float2 p[8];
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    if (s < a.nsplit) p[s] = peer_pair(o + r * LD + d, s);
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    if (s < a.nsplit && weight[s] != 0.f) v.x = fmaf(weight[s], p[s].x, v.x), v.y = fmaf(weight[s], p[s].y, v.y);
            } else {
                v = make_float2(o[r * LD + d], o[r * LD + d + 1]);
            }
            v = seen ? make_float2(v.x * inv, v.y * inv) : make_float2(0.f, 0.f);
            T* dst = static_cast<T*>(a.out) + gr * hd + d;
            if (even) {
                write_pair<T>(dst, v, true);
            } else {
                write_pair<T>(dst, v, false);
                if (d + 1 < hd) write_pair<T>(dst + 1, make_float2(v.y, 0.f), false);
            }
        }
    }
    if constexpr (CL) cluster_meet();                   // nobody leaves while its memory is read
}

// ---------------------------------------------------------------- any type, any head size up to 256
// A block takes 16 RG rows ((node, query head) pairs of one key/value head) through blocks of KT keys in 32-bit multiply-adds.
// RG groups of 16 rows times KG equal parts of the keys: a warp each, with a softmax state of its own; the KG warps of a
// group meet in shared memory at the end. In a warp four lanes stand for four rows each, eight for WK/8 keys each (then for an
// eighth of the output's columns), so 16 x WK scores are formed out of 16 + WK rows of shared memory (with 6 x 64 scores a
// warp its bandwidth was at 72 %). 32-bit rows on 16-byte borders (FAST) come in by cp.async, the next block while one is worked on;
// others element by element. A block of 64 keys for 48 rows of 64 takes 10,000 cycles alone on an SM: 3,400 for the scores and 3,000 for
// the output (their multiply-adds would be 3,072 of an SM's), 2,200 to issue the copies, 1,100 for the softmax. Five trees of 13 nodes
// behind windows of 1,024 keys, 24 heads over 8: 31 us. Tiles of 16 rows take 32 keys at a time, so that an SM holds four: 29 trees of one
// node behind 1,590 keys 92 us for 105 with 64, 16 behind 8,000 keys 178 for 249, one tree of 5 nodes behind 4,000 keys 29 for 26.
template <int HDP, int RG, bool FAST>
struct PlainTile {
    static constexpr int RT = 16 * RG, KT = HDP <= 64 ? (RG == 1 ? 32 : 64) : HDP <= 128 ? 32 : 16, LD = HDP + 4, ST = FAST ? 2 : 1;
    static constexpr int KG = RG == 3 || HDP > 128 ? 2 : 4, WK = KT / KG, THREADS = 32 * RG * KG, PLD = 20;
    static constexpr int KV = KT * LD;                                   // floats of a block's keys, and of its values
    static constexpr int O_FLOATS = KG * RT * (HDP + 2), RING = ST * 2 * KV > O_FLOATS ? ST * 2 * KV : O_FLOATS;     // the outputs meet where the ring was
    static constexpr size_t bytes = sizeof(TreeShape) + (size_t)(RT * LD + RING + RG * KG * WK * PLD) * 4;
    static_assert(WK >= 8, "a key a lane at least");
};

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

// What KG groups of warps found for the same RT rows, into the place of the first of them: o [KG][RT][HD], ml [KG][RT][2]. 16 threads a
// row; between barriers.
template <int KG>
__device__ __forceinline__ void join_groups(float* o, float* ml, int RT, int HD) {
    for (int r = threadIdx.x >> 4; r < RT; r += blockDim.x >> 4) {
        float2 w[KG];
        float M = -INFINITY, f[KG], l = 0.f;
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            w[g] = *reinterpret_cast<const float2*>(ml + (g * RT + r) * 2);
            M = fmaxf(M, w[g].x);
        }
        const float use = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int g = 0; g < KG; ++g) f[g] = exp2f(w[g].x - use), l += f[g] * w[g].y;
        __syncwarp();
        if ((threadIdx.x & 15) == 0) *reinterpret_cast<float2*>(ml + r * 2) = make_float2(M, l);
        for (int d = (threadIdx.x & 15) * 2; d < HD; d += 32) {
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int g = 0; g < KG; ++g) {
                const float2 v = *reinterpret_cast<const float2*>(o + (g * RT + r) * HD + d);
                acc.x = fmaf(f[g], v.x, acc.x), acc.y = fmaf(f[g], v.y, acc.y);
            }
            *reinterpret_cast<float2*>(o + r * HD + d) = acc;
        }
    }
}

template <typename T, int HDP, int RG, bool FAST, bool CL>
__global__ void __launch_bounds__(PlainTile<HDP, RG, FAST>::THREADS)
attention_tree_plain_kernel(const TreeArgs a, int quads) {
    using L = PlainTile<HDP, RG, FAST>;
    constexpr int RT = L::RT, KT = L::KT, LD = L::LD, KG = L::KG, WK = L::WK, KC = WK / 8, WARPS = RG * KG;
    constexpr int NV = HDP / 32, CHUNKS = HDP / 4, PIECES = KT * CHUNKS, ITERS = (PIECES + L::THREADS - 1) / L::THREADS;
    extern __shared__ __align__(16) uint8_t plain_smem[];
    TreeShape& tree = *reinterpret_cast<TreeShape*>(plain_smem);
    float* qs = reinterpret_cast<float*>(plain_smem + sizeof(TreeShape));     // [RT][LD]
    float* kv = qs + RT * LD;                                                 // [ST][keys | values][KT][LD]
    float* ps = kv + L::RING + (threadIdx.x >> 5) * WK * L::PLD;              // this warp's weights, [WK][16 rows]
    pdl_wait();
    pdl_trigger();
    const TreeTile t = tree_tile(a);
    const int G = a.nh / a.nkv, rows = t.n * G, row0 = t.tile * RT;
    if (!t.live || row0 >= rows) return;

    const int hd = a.hd, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rg = warp % RG, kg = warp / RG;
    const int rl = lane >> 3, c = lane & 7;            // the lane's rows: rl, rl + 4, ...; its keys and columns
    const int lo = a.window > 0 ? max(0, t.ctx - a.window + 1) : 0;
    const int first = lo / KT, committed = lo < t.ctx ? (t.ctx + KT - 1) / KT - first : 0, blocks = committed + (t.n + KT - 1) / KT;
    const int per = (blocks + a.nsplit - 1) / a.nsplit, begin = min(blocks, t.split * per), n_blk = min(blocks, begin + per) - begin;
    const int* bt = a.block_table + (size_t)t.b * a.bt_stride;
    const int shift = (a.page_size & (a.page_size - 1)) == 0 ? __ffs(a.page_size) - 1 : -1;
    const size_t page_elems = (size_t)a.nkv * a.page_size * hd;
    // FAST: as in the tensor-core kernel below; an entry of the table is asked for a block before its rows are
    int entry[FAST ? ITERS : 1];
    auto look_up = [&](int i) {
#pragma unroll
        for (int it = 0; it < (FAST ? ITERS : 0); ++it) {
            const int blk = begin + i, at = threadIdx.x + it * L::THREADS, j = (first + blk) * KT + at / CHUNKS;
            entry[it] = at < PIECES && i < n_blk && blk < committed && j >= lo && j < t.ctx ? bt[shift >= 0 ? j >> shift : j / a.page_size] : -1;
        }
    };
    auto load = [&](int i) {
        if (i < n_blk) {
            float* ks = kv + (i & 1) * 2 * L::KV;
            const int blk = begin + i;
#pragma unroll
            for (int it = 0; it < (FAST ? ITERS : 0); ++it) {
                const int row = (threadIdx.x + it * L::THREADS) / CHUNKS, chunk = (threadIdx.x + it * L::THREADS) % CHUNKS;
                if (PIECES % L::THREADS && row >= KT) break;
                const float *k = static_cast<const float*>(a.k_pool), *v = static_cast<const float*>(a.v_pool);
                bool have = chunk * 4 < hd;
                if (blk < committed) {
                    const int page = entry[it], j = (first + blk) * KT + row;
                    if (page >= 0 && page < a.num_pages) {
                        const size_t off = (size_t)page * page_elems + ((size_t)t.kvh * a.page_size + (shift >= 0 ? j & (a.page_size - 1) : j % a.page_size)) * hd + chunk * 4;
                        if (have) k += off, v += off;
                    } else {
                        if (j >= lo && j < t.ctx) atomicOr(a.err, CELLM_DEV_BAD_PAGE);
                        have = false;
                    }
                } else {
                    const int node = (blk - committed) * KT + row;
                    have = have && node < t.n && tree.depth[node] >= 0;
                    if (have) {
                        k = static_cast<const float*>(a.k_new) + (t.t_base + node) * a.k_ld + t.kvh * hd + chunk * 4;
                        v = static_cast<const float*>(a.v_new) + (t.t_base + node) * a.v_ld + t.kvh * hd + chunk * 4;
                    }
                }
                cp_async16(ks + row * LD + chunk * 4, k, have ? 16 : 0);
                cp_async16(ks + L::KV + row * LD + chunk * 4, v, have ? 16 : 0);
            }
        }
        cp_async_commit();
    };
    look_up(0);
    const bool early = FAST && begin < committed;          // the first block needs nothing of the tree's shape
    if (early) load(0);
    for (int r = warp; r < RT; r += WARPS) {
        const int row = row0 + r;
        const T* src = row < rows ? static_cast<const T*>(a.q) + (long long)(t.t_base + row / G) * a.q_ld + (long long)(t.kvh * G + row % G) * hd : nullptr;
        row_to_floats(qs + r * LD, src, hd, HDP, lane, 32, quads);
    }
    read_tree(tree, a.parents + t.t_base, t.n, a.window, a.err);
    if (FAST && !early) load(0);
    look_up(1);
    const int open_from = a.window > 0 ? t.ctx + t.n - a.window : 0;        // no row's window starts behind it
    int node[4];
    float m[4], l[4];
    uint64_t o[4][NV * 2];                     // in pairs of columns
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + rg * 16 + rl + i * 4;
        node[i] = row < rows && tree.depth[row / G] >= 0 ? row / G : -1;
        m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < NV * 2; ++d) o[i][d] = 0ull;
    }
    for (int i = 0; i < n_blk; ++i) {
        const int blk = begin + i;
        const bool paged = blk < committed;
        const int key0 = (first + blk) * KT, node0 = paged ? -1 : (blk - committed) * KT;
        float *ks = kv + (FAST ? (i & 1) * 2 * L::KV : 0), *vs = ks + L::KV;
        if constexpr (FAST) {
            cp_async_wait<0>();
            __syncthreads();
            load(i + 1);                       // into the stage that everybody left before the barrier
            look_up(i + 2);
        } else {
            __syncthreads();
            for (int r = warp; r < KT; r += WARPS) {
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
        }
        const float *q_row = qs + (rg * 16 + rl) * LD, *k_row = ks + (kg * WK + c) * LD;
        float s2[4][KC];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int k = 0; k < KC; ++k) s2[x][k] = 0.f;
#pragma unroll 2
        for (int d = 0; d < HDP; d += 4) {
            float4 q4[4], k4[KC];
#pragma unroll
            for (int x = 0; x < 4; ++x) q4[x] = *reinterpret_cast<const float4*>(q_row + x * 4 * LD + d);
#pragma unroll
            for (int k = 0; k < KC; ++k) k4[k] = *reinterpret_cast<const float4*>(k_row + k * 8 * LD + d);
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int k = 0; k < KC; ++k) s2[x][k] = fmaf(q4[x].w, k4[k].w, fmaf(q4[x].z, k4[k].z, fmaf(q4[x].y, k4[k].y, fmaf(q4[x].x, k4[k].x, s2[x][k]))));
        }
        float s[4][KC];
        const bool open = paged && key0 + KT <= t.ctx && key0 >= open_from;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < KC; ++k) s[x][k] = s2[x][k] * a.scale_log2e;
            if (!open) {
                const uint64_t seen = node[x] >= 0 ? seen_bits<KT>(tree, node[x], a.window, t.ctx, key0, node0) >> (kg * WK + c) : 0ull;
#pragma unroll
                for (int k = 0; k < KC; ++k)
                    if (!(seen >> (k * 8) & 1ull)) s[x][k] = -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < KC; ++k) top = fmaxf(top, s[x][k]);
#pragma unroll
            for (int y = 4; y > 0; y >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
            const float now = fmaxf(m[x], top), use = now == -INFINITY ? 0.f : now, corr = fast_exp2(m[x] - use);
            m[x] = now;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < KC; ++k) s[x][k] = fast_exp2(s[x][k] - use), sum += s[x][k];
            l[x] = l[x] * corr + sum;
#pragma unroll
            for (int d = 0; d < NV * 2; ++d) o[x][d] = fma2(o[x][d], pair_of(corr, corr), 0ull);
        }
#pragma unroll
        for (int k = 0; k < KC; ++k) *reinterpret_cast<float4*>(ps + (c + k * 8) * L::PLD + rl * 4) = make_float4(s[0][k], s[1][k], s[2][k], s[3][k]);
        __syncwarp();
        const float* v_row = vs + kg * WK * LD + c * 4;
#pragma unroll 4
        for (int k = 0; k < WK; ++k) {
            const float4 w = *reinterpret_cast<const float4*>(ps + k * L::PLD + rl * 4);
            const uint64_t p[4] = {pair_of(w.x, w.x), pair_of(w.y, w.y), pair_of(w.z, w.z), pair_of(w.w, w.w)};
#pragma unroll
            for (int g = 0; g < NV; ++g) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(v_row + k * LD + g * 32);
#pragma unroll
                for (int x = 0; x < 4; ++x) o[x][2 * g] = fma2(p[x], v.x, o[x][2 * g]), o[x][2 * g + 1] = fma2(p[x], v.y, o[x][2 * g + 1]);
            }
        }
        __syncwarp();                          // (the weights' place is written again by the next block)
    }
    if constexpr (FAST) cp_async_wait<0>();
    __syncthreads();                           // the ring's place is free
    float *o_s = kv, *ml_s = kv + KG * RT * HDP;             // [KG][RT][HDP], [KG][RT][2]
#pragma unroll
    for (int x = 0; x < 4; ++x) {
#pragma unroll
        for (int y = 4; y > 0; y >>= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], y);
        const int r = kg * RT + rg * 16 + rl + x * 4;
#pragma unroll
        for (int g = 0; g < NV; ++g) *reinterpret_cast<ulonglong2*>(o_s + r * HDP + g * 32 + c * 4) = make_ulonglong2(o[x][2 * g], o[x][2 * g + 1]);
        if (c == 0) ml_s[r * 2] = m[x], ml_s[r * 2 + 1] = l[x];
    }
    __syncthreads();
    join_groups<KG>(o_s, ml_s, RT, HDP);
    __syncthreads();
    finish_rows<T, CL>(a, t, tree, o_s, HDP, ml_s, RT, row0);
}

// ---------------------------------------------------------------- bfloat16, head sizes 32, 64, 96, 128: mma.sync
// Four warps take 16 * RG rows through blocks of 64 keys that all threads bring in with cp.async (a ring of ST stages, one barrier
// a block). RG groups of 16 rows share a block; the 4 / RG warps of a group take its keys in equal parts, each with a softmax
// state of its own, and meet in shared memory at the end. Few rows (small trees) so still use every warp. One tree of 8 nodes behind 500
// keys, 32 heads over 8: 9.2 us in a CUDA graph, bound by latency (the copies' first block, the merge); with many long trees by issue
// slots (42 %) and waits for shared memory, which is why those go to tcgen05.
template <int HD, int RG>
struct MmaTile {
    static constexpr int KG = 4 / RG, RT = 16 * RG;
    static constexpr int ST = HD <= 32 ? 4 : HD <= 96 ? 3 : 2;
    static constexpr int KV = FA_BN * HD * 2;
    static constexpr int q_off = 0, kv_off = RT * HD * 2, tree_off = kv_off + ST * 2 * KV, bytes = tree_off + (int)sizeof(TreeShape);
    static_assert(4 * 16 * (HD + 2) * 4 <= ST * 2 * KV, "the warps' outputs must fit the ring");
};

template <int HD, int RG, bool CL>
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
            entry[it] = i < n_blk && blk < committed && j >= lo && j < t.ctx ? bt[shift >= 0 ? j >> shift : j / a.page_size] : -1;
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
                    } else if (j >= lo && j < t.ctx) {
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

    // the warps' results meet in shared memory, where the ring was
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
    if constexpr (KG > 1) {
        join_groups<KG>(o_s, ml_s, L::RT, HD);
        __syncthreads();
    }
    finish_rows<__nv_bfloat16, CL>(a, t, tree, o_s, HD, ml_s, L::RT, row0);
}

// The pieces of a row merged in their order: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s. 16 threads a row, which work out the
// pieces' weights together and take four neighbouring entries (one where the rows do not allow it) of every piece, so that every load
// of a row's pieces is on its way at once: bound by their latency.
template <typename T>
__global__ void __launch_bounds__(256)
attention_tree_merge_kernel(T* __restrict__ out, const float* __restrict__ part_o, const float* __restrict__ part_ml, long long rows, int hd, int nsplit) {
    pdl_wait();
    pdl_trigger();
    const long long r = min((long long)blockIdx.x * 16 + (threadIdx.x >> 4), rows - 1);       // (a row twice is written twice alike)
    const int c = threadIdx.x & 15, group = threadIdx.x & 16;
    float2 ml[4];
    float M = -INFINITY, L = 0.f, w[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        ml[g] = make_float2(-INFINITY, 0.f);
        if (g * 16 + c < nsplit) ml[g] = *reinterpret_cast<const float2*>(part_ml + ((long long)(g * 16 + c) * rows + r) * 2);
        M = fmaxf(M, ml[g].x);
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    const float use = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int g = 0; g < 4; ++g) w[g] = exp2f(ml[g].x - use), L = fmaf(w[g], ml[g].y, L);
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
    const float inv = L != 0.f ? 1.f / L : 0.f;
    const int quad = hd % 4 == 0 ? 4 : 1;
    for (int d0 = 0; d0 < hd; d0 += 16 * quad) {
        const int d = d0 + c * quad;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (g * 16 >= nsplit) break;
#pragma unroll 8
            for (int s = 0; s < min(16, nsplit - g * 16); ++s) {
                const float f = __shfl_sync(0xffffffffu, w[g], group + s);
                if (d >= hd) continue;
                const float* src = part_o + ((long long)(g * 16 + s) * rows + r) * hd + d;
                const float4 v = quad == 4 ? *reinterpret_cast<const float4*>(src) : make_float4(*src, 0.f, 0.f, 0.f);
                if (f != 0.f) acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
            }
        }
        if (d >= hd) continue;
        T* dst = out + r * hd + d;
        dst[0] = from_float<T>(acc.x * inv);
        if (quad == 4) dst[1] = from_float<T>(acc.y * inv), dst[2] = from_float<T>(acc.z * inv), dst[3] = from_float<T>(acc.w * inv);
    }
}

// The grid; in_cluster: the pieces of a tile are one cluster (they are neighbours in the grid).
template <typename... KArgs, typename... Args>
int launch_tiles(std::atomic<unsigned long long>& allowed, void (*kernel)(KArgs...), const TreeArgs& a, bool in_cluster, int threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaError_t e = cellm_allow_smem(allowed, (const void*)kernel, smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)a.B * a.nkv * a.tiles * a.nsplit));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.nsplit;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = in_cluster ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, a, args...);
    return e == cudaSuccess ? CELLM_OK : (int)e;
}
// Up to this many pieces meet in a cluster.
constexpr int CLUSTER_MAX = 8;

template <typename T, int HDP, int RG, bool FAST>
int launch_plain_rows(TreeArgs a, int quads, cudaStream_t stream) {
    using L = PlainTile<HDP, RG, FAST>;
    static std::atomic<unsigned long long> allowed[2];
    a.tiles = (a.most * (a.nh / a.nkv) + L::RT - 1) / L::RT;
    return a.nsplit > 1 && a.nsplit <= CLUSTER_MAX ? launch_tiles(allowed[1], attention_tree_plain_kernel<T, HDP, RG, FAST, true>, a, true, L::THREADS, L::bytes, stream, quads)
                                                   : launch_tiles(allowed[0], attention_tree_plain_kernel<T, HDP, RG, FAST, false>, a, false, L::THREADS, L::bytes, stream, quads);
}
// Rows of 32-bit tiles: 48 where that leaves the last tile fuller than 32 would (not for the widest heads, whose tiles would not fit
// twice into an SM), 16 for the smallest trees.
int plain_rows(int rows, int hd) { return rows <= 16 ? 16 : hd > 128 || rows % 32 == 0 || rows <= 32 || (rows + 47) / 48 * 48 > (rows + 31) / 32 * 32 ? 32 : 48; }
template <typename T, int HDP>
int launch_plain(const TreeArgs& a, cudaStream_t stream) {
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool;
    const int quads = a.hd % 4 == 0 && a.q_ld % 4 == 0 && a.k_ld % 4 == 0 && a.v_ld % 4 == 0 && at % (4 * sizeof(T)) == 0;
    if constexpr (sizeof(T) == 4) {
        if (quads) {
            const int rows = plain_rows(a.most * (a.nh / a.nkv), a.hd);
            if (rows == 16) return launch_plain_rows<T, HDP, 1, true>(a, 1, stream);
            if constexpr (HDP <= 128) {
                if (rows == 48) return launch_plain_rows<T, HDP, 3, true>(a, 1, stream);
            }
            return launch_plain_rows<T, HDP, 2, true>(a, 1, stream);
        }
    }
    return launch_plain_rows<T, HDP, 2, false>(a, quads, stream);
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
    static std::atomic<unsigned long long> allowed[2];
    a.tiles = (a.most * (a.nh / a.nkv) + L::RT - 1) / L::RT;
    return a.nsplit > 1 && a.nsplit <= CLUSTER_MAX ? launch_tiles(allowed[1], attention_tree_mma_kernel<HD, RG, true>, a, true, 128, L::bytes, stream)
                                                   : launch_tiles(allowed[0], attention_tree_mma_kernel<HD, RG, false>, a, false, 128, L::bytes, stream);
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
int launch_mma_sized(const TreeArgs& a, cudaStream_t stream) {
    if (a.hd == 32) return launch_mma_rows<32>(a, stream);
    if (a.hd == 64) return launch_mma_rows<64>(a, stream);
    if (a.hd == 96) return launch_mma_rows<96>(a, stream);
    return launch_mma_rows<128>(a, stream);
}

// How many pieces the keys of a tile of rows are cut into: of all counts the one whose rounds of blocks, each as long as its keys
// and a few blocks' worth of start and merge, take the least time. Up to CLUSTER_MAX pieces merge at the cost of one block where they may be
// a cluster (clusters leave about an eighth of the blocks' places empty, since a cluster stays within a group of SMs: 280 blocks in clusters
// of 7 took two rounds on 296 places), more at that of a launch.
int pieces(long long tiles, int key_blocks, long long at_once, bool clusters) {
    constexpr int START = 3;
    int best = 1;
    long long least = LLONG_MAX;
    for (int n = 1; n <= 64 && n <= std::max(1, key_blocks); ++n) {
        const bool cluster = clusters && n > 1 && n <= CLUSTER_MAX;
        const long long room = cluster ? at_once - at_once / 8 : at_once;
        const long long cost = (tiles * n + room - 1) / room * ((key_blocks + n - 1) / n + START) + (n == 1 ? 0 : cluster ? 1 : START);
        if (cost < least) least = cost, best = n;
    }
    return best;
}

// Which trees of heads of 64 go to the tcgen05 kernel, whose tiles have 128 rows: those of more than 64 rows, and behind long contexts those
// of more than 16. Microseconds of mma.sync and of tcgen05, 32 heads over 8, for 1, 8 and 32 trees:
//   8 nodes (32 rows)    1,024 keys 10.0 12.0 | 12.7 15.3 | 33.9 30.5     4,096 keys 18.8 16.3 | 24.8 27.0 | 105 77
//   12 nodes (48 rows)   1,024 keys 10.7 12.5 | 14.2 15.4 | 39.7 30.8     4,096 keys 21.3 17.1 | 30.9 27.3 | 127 77
//   25 nodes (100 rows)  1,024 keys 12.3 12.9 | 21.8 15.6 | 76.2 31.2     4,096 keys 24.0 18.7 | 54.9 28.2 | 226 77
// The number of trees, on which the table depends too, does not enter: the rule gives away up to 9 us where many small trees stand behind
// fewer than 2,048 keys (32 of 12 nodes 39.7 for 30.8, 32 of 8 33.9 for 30.5), 2 us for 8 of 8 nodes behind 4,096 (27.0 for 24.8) and 0.6
// for one of 25 behind 1,024. Fewer than 1,024 keys were not measured.
bool tc_pays(int rows, int keys) { return rows > 64 || (rows > 16 && keys >= 2048); }

struct TreePlan {
    bool tc;            // for the tcgen05 kernel, if it takes the call
    int nsplit;         // pieces a tile's keys are cut into
    int parts;          // pieces that meet in the workspace; 0: none do
};
TreePlan tree_plan(int B, int most, int nh, int nkv, int hd, int keys, int dtype, int sms) {
    const int G = nh / nkv, rows = most * G;
    if (dtype == CELLM_BF16 && hd == 64 && tc_pays(rows, keys) && G <= 128 && 128 / G * G >= 96) {
        const int tile = 128 / G, two = most > tile;
        const int n = pieces((long long)B * nkv * ((most + (1 + two) * tile - 1) / ((1 + two) * tile)), ((keys + 127) / 128 + 1 - two) / (2 - two), sms, false);
        return {true, n, n > 1 ? n : 0};
    }
    const bool mma = dtype == CELLM_BF16 && (hd == 32 || hd == 64 || hd == 96 || hd == 128);
    const int tile = mma ? (rows <= 16 ? 16 : rows <= 32 ? 32 : 64) : dtype == CELLM_F32 ? plain_rows(rows, hd) : 32;
    const bool few = !mma && tile == 16 && hd <= 64;                          // (32-bit tiles of 16 rows)
    const int an_sm = few ? 4 : hd <= 32 ? (mma ? 4 : 3) : mma && hd == 64 ? 3 : 2;     // blocks that an SM holds, by their shared memory
    const int block = few ? 32 : mma || hd <= 64 ? 64 : hd <= 128 ? 32 : 16;
    const int n = pieces((long long)B * nkv * ((rows + tile - 1) / tile), (keys + block - 1) / block, (long long)an_sm * sms, true);
    return {false, n, n > CLUSTER_MAX ? n : 0};
}

template <typename T>
int launch_merge(const TreeArgs& a, int parts, cudaStream_t stream) {
    const long long rows = (long long)a.T * a.nh;
    CELLM_RUN(attention_tree_merge_kernel<T>, (unsigned)((rows + 15) / 16), 256, 0, stream, (T*)a.out, a.part_o, a.part_ml, rows, a.hd, parts);
    return CELLM_OK;
}

}  // namespace

// How a call of these sizes is best run (`keys`: the most that a node sees), in three bytes: the pieces that a tile's keys are cut into, the
// pieces that meet in the workspace, whether the tcgen05 kernel is to be taken.
CELLM_API int cellm_attention_tree_plan(int B, int most, int nh, int nkv, int hd, int keys, int dtype, int sms) {
    if (B <= 0 || most <= 0 || nkv <= 0 || nh < nkv) return 1;
    const TreePlan p = tree_plan(B, most, nh, nkv, hd, keys, dtype, sms);
    return p.nsplit | p.parts << 8 | (p.tc ? 1 : 0) << 16;
}

// out [T, nh * hd], q rows q_ld elements apart, the nodes' keys and values in rows k_ld and v_ld apart ([nkv * hd] each), parents
// [T]; request b owns the nodes cu_seqlens[b] .. cu_seqlens[b + 1] (at most 256, `most` of them in the largest tree) behind
// ctx_lens[b] committed tokens in the pages of its row of the block table. nsplit, parts and tc as planned: part_o [parts, T * nh, hd]
// and part_ml [parts, T * nh, 2] floats.
CELLM_API int cellm_attention_tree(void* out, float* part_o, float* part_ml, const void* q, long long q_ld, const void* k_new, long long k_ld,
                                   const void* v_new, long long v_ld, const int* parents, const void* k_pool, const void* v_pool,
                                   const int* cu_seqlens, const int* ctx_lens, const int* block_table, int bt_stride, int B, int T, int most,
                                   int num_pages, int page_size, int nh, int nkv, int hd, float scale, int window, int nsplit, int parts, int tc, int dtype, int* err,
                                   cudaStream_t stream) {
    if (T <= 0 || B <= 0 || most <= 0) return CELLM_OK;
    if (dtype != CELLM_F32 && dtype != CELLM_BF16) return CELLM_ERR_DTYPE;
    if (nkv <= 0 || nh <= 0 || nh % nkv || hd <= 0 || hd > 256 || page_size <= 0 || most > TREE_MAX || bt_stride < 0 || window < 0) return CELLM_ERR_SIZE;
    if (nsplit < 1 || nsplit > 64 || parts < 0) return CELLM_ERR_SIZE;
    if (parts > 0 && (!part_o || !part_ml)) return CELLM_ERR_ARG;
    if (!out || !q || !k_new || !v_new || !parents || !cu_seqlens || !ctx_lens || !err) return CELLM_ERR_ARG;
    if ((((uintptr_t)part_o) & 15) || (((uintptr_t)part_ml) & 7)) return CELLM_ERR_ALIGN;
    TreeArgs a = {out, part_o, part_ml, q, k_new, v_new, q_ld, k_ld, v_ld, parents, k_pool, v_pool, cu_seqlens, ctx_lens, block_table,
                  bt_stride, B, T, most, num_pages, page_size, nh, nkv, hd, 0, nsplit, window, scale * 1.4426950408889634f, err};
    const int G = nh / nkv;
    if ((long long)B * nkv * 64 * ((most * G + 15) / 16) > 0x7fffffffLL) return CELLM_ERR_SIZE;
    if (tc && dtype == CELLM_BF16 && attention_tree_tc_takes(a)) {
        const int need = nsplit > 1 ? nsplit : 0;
        if (parts >= need) {
            const int rc = attention_tree_tc_launch(a, stream);
            return rc != CELLM_OK || need == 0 ? rc : launch_merge<__nv_bfloat16>(a, need, stream);
        }
    }
    if (nsplit > CLUSTER_MAX && parts < nsplit) a.nsplit = CLUSTER_MAX;
    const int rc = dtype == CELLM_F32 ? launch_plain_sized<float>(a, stream) : mma_takes(a) ? launch_mma_sized(a, stream) : launch_plain_sized<__nv_bfloat16>(a, stream);
    if (rc != CELLM_OK || a.nsplit <= CLUSTER_MAX) return rc;
    return dtype == CELLM_F32 ? launch_merge<float>(a, a.nsplit, stream) : launch_merge<__nv_bfloat16>(a, a.nsplit, stream);
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_attention_tree_packed(const long long* a, cudaStream_t stream) {
    return cellm_attention_tree((void*)a[0], (float*)a[1], (float*)a[2], (const void*)a[3], (long long)a[4], (const void*)a[5], (long long)a[6],
        (const void*)a[7], (long long)a[8], (const int*)a[9], (const void*)a[10], (const void*)a[11], (const int*)a[12], (const int*)a[13],
        (const int*)a[14], (int)a[15], (int)a[16], (int)a[17], (int)a[18], (int)a[19], (int)a[20], (int)a[21], (int)a[22], (int)a[23],
        (float)cellm_packed_double(a[24]), (int)a[25], (int)a[26], (int)a[27], (int)a[28], (int)a[29], (int*)a[30], stream);
}
