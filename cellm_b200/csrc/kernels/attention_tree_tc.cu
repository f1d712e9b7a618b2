// Attention of drafted trees on the 5th-generation tensor cores (tcgen05): bfloat16, heads of 64, trees whose rows ((node, query
// head) pairs of one key/value head) fill tiles of 128.
//
// One CTA takes two tiles of 128 rows through blocks of 128 keys: committed ones, a TMA box a page, then the nodes' own, a box a
// block. Warps 0 and 2 bring queries, keys and values in, warp 1 issues the products (S = Q.K^T into tensor memory, O += P.V with P
// read from tensor memory and V as its rows lie), warps 4..7 and 8..11 do the softmax of a tile each, a row a thread, so that one
// tile's products run beside the other's softmax; they take the registers that the first warpgroup gives up. Trees of up to 128 rows
// have one tile: the same rows then stand in both, and the tiles take the blocks in turn; the second tile's result joins the first's
// through shared memory at the end.
//
// What it costs is exponentials: a block of 128 x 128 scores keeps the four special-function units of an SM 1,024 cycles, its
// two products the tensor cores 512. A quarter of the exponentials are formed by multiply-adds (none 240 us, an eighth 241, a quarter
// 237, three eighths 250 where it was measured).
//
// Eight trees of 63 nodes behind 32,768 keys, 32 heads over 8: 233 us, 581 TFLOP/s (the keys and values alone would take 82 us). Half of
// that is handing over: with the exponentials taken out it still took 134 us, a tile waiting for the other role about as long as it
// computes, and the two tiles of a CTA cover only part of one another's waits. Two CTAs an SM with blocks of 64 keys (258 us), a product
// warp a tile (240), the next half block's scores loaded under this half's exponentials (304, more code than the instruction cache
// holds) and fewer barriers a block (246) were slower.
//
// Every wait on an mbarrier is bounded: a role that gives up sets CELLM_DEV_WAIT_TIMEOUT and an abort flag; the CTA then waits (bounded
// again) for the copies and products it has under way, frees its tensor memory and returns. The lanes of a warp wait together, by one
// instruction on one barrier, so they give up together.
#include <climits>

#include "attention_tree.cuh"
#include "pairs.cuh"
#include "tcgen05_attn.cuh"

namespace {

constexpr int TM = 128, TN = 128, HD = 64;
constexpr int KV_STAGES = 5;
constexpr int TMEM_COLUMNS = 512;      // scores of tile 0 and 1 in columns 0 and 128, their outputs in 256 and 320, their weights
constexpr int O_COL = 256, P_COL = 384;    // (bfloat16, two keys a column) in 384 and 448
constexpr int THREADS = 384;
constexpr int POLY = 2;                // pairs of exponentials of every eight that the multiply-add units form

struct TreeTcSmem {                    // starts on a 1024-byte boundary (checked in the kernel)
    uint8_t q[2][TM * HD * 2];
    uint8_t k[KV_STAGES][TN * HD * 2];
    uint8_t v[KV_STAGES][TN * HD * 2];
    TreeShape tree;
    uint64_t q_full;
    uint64_t k_full[KV_STAGES], k_empty[KV_STAGES];
    uint64_t v_full[KV_STAGES], v_empty[KV_STAGES];
    uint64_t s_full[2], s_empty[2], p_full[2], pv_done[2];
    uint64_t drained;            // by the products that an abort has left under way
    uint32_t tmem_base;
    int abort_flag, never, issued[2];     // never: no abort; issued: blocks of keys and of values asked for before an abort
};

__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return d;
}
// 2^x of two numbers without the special-function units: x = n + f with |f| <= 1/2, n out of the rounding of an addition, 2^f = 1 + f
// P(f), P fitted (weighted least squares, reweighted towards the largest error) to 2.8e-6 relative, a thousandth of what rounding
// the weight to bfloat16 costs. What lies at -127 or below, -inf too, gives 0: a key that is not seen has no weight. (Between -127 and -126
// the exponent's field is 0 and the result a denormal below 2^-126.)
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x) {
    x = pair_of(fmaxf(low_of(x), -127.f), fmaxf(high_of(x), -127.f));
    const uint64_t r = add2(x, pair_of(12582912.f, 12582912.f)), n = add2(r, pair_of(-12582912.f, -12582912.f));
    const uint64_t f = fma2(n, pair_of(-1.f, -1.f), x);
    uint64_t p = pair_of(0.00958284828811884f, 0.00958284828811884f);
    p = fma2(p, f, pair_of(0.05590643361210823f, 0.05590643361210823f));
    p = fma2(p, f, pair_of(0.24024099111557007f, 0.24024099111557007f));
    p = fma2(p, f, pair_of(0.6931241750717163f, 0.6931241750717163f));
    p = fma2(p, f, pair_of(1.f, 1.f));
    return pair_of(__uint_as_float(__float_as_uint(low_of(p)) + (__float_as_uint(low_of(r)) << 23)),
                   __uint_as_float(__float_as_uint(high_of(p)) + (__float_as_uint(high_of(r)) << 23)));
}

__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}

// grid: (request, key/value head, pair of tiles, piece), the last fastest. alternate: one tile of rows, whose blocks the two tiles take
// in turn.
__global__ void __launch_bounds__(THREADS, 1)
attention_tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                         const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_vn, const TreeArgs a, const int alternate) {
    extern __shared__ __align__(1024) uint8_t tc_smem[];
    TreeTcSmem& sm = *reinterpret_cast<TreeTcSmem*>(tc_smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (smem_u32(tc_smem) & 1023u) {             // the swizzled tiles need 1024-byte alignment
        if (threadIdx.x == 0) atomicOr(a.err, CELLM_DEV_BAD_LAYOUT);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(&sm.q_full, 1);
        for (int i = 0; i < KV_STAGES; ++i) {
            mbar_init(&sm.k_full[i], 1), mbar_init(&sm.k_empty[i], 1);
            mbar_init(&sm.v_full[i], 1), mbar_init(&sm.v_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sm.s_full[t], 1), mbar_init(&sm.s_empty[t], 128);
            mbar_init(&sm.p_full[t], 128), mbar_init(&sm.pv_done[t], 1);
        }
        mbar_init(&sm.drained, 1);
        sm.abort_flag = sm.never = 0, sm.issued[0] = sm.issued[1] = INT_MAX;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (const CUtensorMap* map : {&map_q, &map_k, &map_v, &map_kn, &map_vn}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    if (warp == 1) tmem_alloc(&sm.tmem_base, TMEM_COLUMNS);
    tc_fence_before();
    pdl_wait();
    pdl_trigger();
    const TreeTile t = tree_tile(a);
    const int G = a.nh / a.nkv, tile_nodes = TM / G, node_first = t.tile * (alternate ? 1 : 2) * tile_nodes;
    const bool live = t.live && node_first < t.n;
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    volatile int* abort_flag = &sm.abort_flag;

    const int lo = a.window > 0 ? max(0, t.ctx - a.window + 1) : 0;
    const int first = lo / TN, committed = lo < t.ctx ? (t.ctx + TN - 1) / TN - first : 0, blocks = committed + (t.n + TN - 1) / TN;
    const int per = (blocks + a.nsplit - 1) / a.nsplit, begin = min(blocks, t.split * per), n_blk = live ? min(blocks, begin + per) - begin : 0;
    const bool two = alternate || node_first + tile_nodes < t.n;
    auto takes = [&](int tile, int j) { return alternate ? (j & 1) == tile : tile == 0 || two; };

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 || warp == 2) {
        // warp 0 brings the queries and the keys, warp 2 the values: a stage of keys is free a product earlier than one of values
        if (live) {
            const bool keys = warp == 0;
            if (keys && lane == 0) {
                mbar_expect_tx(&sm.q_full, (two ? 2 : 1) * tile_nodes * G * HD * 2);
                tma_load_3d(sm.q[0], &map_q, 0, t.kvh * G, t.t_base + node_first, &sm.q_full);
                if (two) tma_load_3d(sm.q[1], &map_q, 0, t.kvh * G, t.t_base + node_first + (alternate ? 0 : tile_nodes), &sm.q_full);
            }
            const int* bt = a.block_table + (size_t)t.b * a.bt_stride;
            const int pages_per_block = TN / a.page_size;
            const CUtensorMap *paged_map = keys ? &map_k : &map_v, *node_map = keys ? &map_kn : &map_vn;
            // lane i brings page i of a block, if something of it is seen; its entry of the table is asked for a block ahead. A page that
            // is none is reported and read from behind the pool's end, which is zeros.
            const int behind = a.num_pages * a.nkv * a.page_size;
            auto seen = [&](int j) {
                const int key0 = (first + begin + j) * TN + lane * a.page_size;
                return j < n_blk && begin + j < committed && lane < pages_per_block && key0 < t.ctx && key0 + a.page_size > lo;
            };
            auto entry = [&](int j) { return seen(j) ? bt[((first + begin + j) * TN + lane * a.page_size) / a.page_size] : 0; };
            int next = entry(0);
            for (int j = 0; j < n_blk; ++j) {
                const int st = j % KV_STAGES, blk = begin + j, page = next;
                uint64_t* full = keys ? &sm.k_full[st] : &sm.v_full[st];
                uint8_t* dst = keys ? sm.k[st] : sm.v[st];
                next = entry(j + 1);
                const bool paged = blk < committed, have = seen(j), none = page < 0 || page >= a.num_pages;
                if (keys && have && none) atomicOr(a.err, CELLM_DEV_BAD_PAGE);
                const uint32_t bytes = paged ? (uint32_t)__popc(__ballot_sync(0xffffffffu, have)) * (uint32_t)a.page_size * HD * 2 : TN * HD * 2;
                bool ok = true;
                if (lane == 0) ok = mbar_wait(keys ? &sm.k_empty[st] : &sm.v_empty[st], ((uint32_t)(j / KV_STAGES) & 1u) ^ 1u, abort_flag);
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                if (!ok) { if (lane == 0) { *abort_flag = 1; sm.issued[warp >> 1] = j; atomicOr(a.err, CELLM_DEV_WAIT_TIMEOUT); } break; }
                if (lane == 0) mbar_expect_tx(full, bytes);
                __syncwarp();
                if (have) tma_load_2d(dst + (size_t)lane * a.page_size * HD * 2, paged_map, 0, none ? behind : (page * a.nkv + t.kvh) * a.page_size, full);
                else if (!paged && lane == 0) tma_load_3d(dst, node_map, 0, t.kvh, t.t_base + (blk - committed) * TN, full);
            }
        }
    } else if (warp == 1) {
        // The whole warp walks the blocks and one lane of it issues: what the products' descriptors are made of then stays in uniform
        // registers (with the other lanes branched away, the moves into them took 3,200 cycles a pair of blocks, more than
        // everything else).
        if (live) {
            const uint32_t idesc_s = umma_idesc(TM, TN, false);      // S[128 x 128] = Q (K-major) . K^T (K-major)
            const uint32_t idesc_o = umma_idesc(TM, HD, true);       // O[128 x 64] += P (K-major) . V (MN-major)
            const bool leader = elect_one();
            bool ok = mbar_wait(&sm.q_full, 0, abort_flag);
            auto issue_s = [&](int j) -> bool {
                const int st = j % KV_STAGES, n = alternate ? j >> 1 : j;
                if (!mbar_wait(&sm.k_full[st], (uint32_t)(j / KV_STAGES) & 1u, abort_flag)) return false;
                const uint64_t dk = umma_desc(smem_u32(sm.k[st]));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!takes(i, j)) continue;
                    if (n > 0 && !mbar_wait(&sm.s_empty[i], (uint32_t)(n - 1) & 1u, abort_flag)) return false;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t dq = umma_desc(smem_u32(sm.q[i]));
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks)
                            umma_bf16(tmem + (uint32_t)(i * TN), dq + (uint64_t)(ks * 2), dk + (uint64_t)(ks * 2), idesc_s, ks != 0 ? 1u : 0u);
                        umma_commit(&sm.s_full[i]);
                    }
                    __syncwarp();
                }
                if (leader) umma_commit(&sm.k_empty[st]);
                __syncwarp();
                return true;
            };
            // a tile's next scores are under way while its softmax works: one block ahead, two where the tiles take turns
            const int ahead = alternate ? 2 : 1;
            for (int j = 0; ok && j < min(ahead, n_blk); ++j) ok = issue_s(j);
            for (int j = 0; ok && j < n_blk; ++j) {
                const int st = j % KV_STAGES, n = alternate ? j >> 1 : j;
                if (j + ahead < n_blk) { ok = issue_s(j + ahead); if (!ok) break; }
                ok = mbar_wait(&sm.v_full[st], (uint32_t)(j / KV_STAGES) & 1u, abort_flag);
                if (!ok) break;
                const uint64_t dv = umma_desc(smem_u32(sm.v[st]));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!takes(i, j)) continue;
                    ok = mbar_wait(&sm.p_full[i], (uint32_t)n & 1u, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int ks = 0; ks < TN / 16; ++ks) {
                            const uint32_t pa = tmem + (uint32_t)(P_COL + i * (TN / 2) + ks * 8);     // 16 keys = 8 columns of P
                            const uint64_t db = dv + (uint64_t)(ks * 16 * HD * 2 / 16);               // 16 keys = 16 rows of V
                            umma_bf16_ts(tmem + (uint32_t)(O_COL + i * HD), pa, db, idesc_o, (n | ks) != 0 ? 1u : 0u);
                        }
                        umma_commit(&sm.pv_done[i]);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (leader) umma_commit(&sm.v_empty[st]);
                __syncwarp();
            }
            if (!ok && lane == 0) { *abort_flag = 1; atomicOr(a.err, CELLM_DEV_WAIT_TIMEOUT); }
        }
    }
    } else {
        // 384 x 168 registers at launch: as many as 128 x 56 and 256 x 224
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int i = (warp >> 2) - 1;                                // which tile
        // the tree's shape: wanted only where the nodes' own keys are read, so the first committed blocks are on their way meanwhile
        if (live) read_tree(sm.tree, a.parents + t.t_base, t.n, a.window, a.err, (int)threadIdx.x - 128, 256, [] { asm volatile("bar.sync 1, 256;" ::: "memory"); });
        if (live && (i == 0 || two)) {
        const int r = (warp & 3) * 32 + lane;                         // row of the tile = lane of tensor memory
        const int node = node_first + (alternate ? 0 : i * tile_nodes) + r / G;
        const bool row_ok = r < tile_nodes * G && node < t.n, seeing = row_ok && sm.tree.depth[node] >= 0;
        const int open_from = a.window > 0 ? t.ctx + t.n - a.window : 0;      // no row's window starts behind it
        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_col = (uint32_t)(i * TN), o_col = (uint32_t)(O_COL + i * HD), p_col = (uint32_t)(P_COL + i * (TN / 2));
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        int it = 0;
        for (int j = alternate ? i : 0; j < n_blk; j += alternate ? 2 : 1, ++it) {
            ok = mbar_wait(&sm.s_full[i], (uint32_t)it & 1u, abort_flag);
            if (!ok) break;
            tc_fence_after();
            uint32_t s[TN];
#pragma unroll
            for (int c = 0; c < TN / 32; ++c) tmem_ld32_nowait(lane_base + s_col + (uint32_t)(c * 32), s + c * 32);
            tmem_ld_wait();
            tc_fence_before();
            mbar_arrive(&sm.s_empty[i]);                              // the scores are in registers now
            const int blk = begin + j, key0 = (first + blk) * TN, node0 = (blk - committed) * TN;
            const bool paged = blk < committed;
            if (!paged || key0 + TN > t.ctx || key0 < open_from) {
#pragma unroll
                for (int c = 0; c < TN; c += 64) {
                    const uint64_t seen = seeing && (paged || node0 + c < TREE_MAX) ? seen_bits<64>(sm.tree, node, a.window, t.ctx, key0 + c, paged ? -1 : node0 + c) : 0ull;
                    const uint32_t half[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
                    for (int k = 0; k < 64; ++k)
                        if (!(half[k / 32] >> (k % 32) & 1u)) s[c + k] = 0xff800000u;
                }
            }
            float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int k = 0; k < TN; k += 8) {
                mx0 = max3(mx0, s[k], s[k + 1]), mx1 = max3(mx1, s[k + 2], s[k + 3]);
                mx2 = max3(mx2, s[k + 4], s[k + 5]), mx3 = max3(mx3, s[k + 6], s[k + 7]);
            }
            mx0 = max3(mx0, __float_as_uint(mx1), __float_as_uint(mx2));
            const float m_new = max3(m, __float_as_uint(mx0 * a.scale_log2e), __float_as_uint(mx3 * a.scale_log2e));      // NaN stays
            // the output is rescaled only when the maximum has grown by more than 2^RESCALE_STEP; a stale one only scales P
            const bool want = !(m_new <= m + RESCALE_STEP);
            bool pv_seen = it == 0;
            if (__any_sync(0xffffffffu, want)) {
                if (it > 0) {
                    ok = mbar_wait(&sm.pv_done[i], (uint32_t)(it - 1) & 1u, abort_flag);
                    if (!ok) break;
                    pv_seen = true;
                    tc_fence_after();
                    const float corr = want ? (m == -INFINITY ? 0.f : fast_exp2(m - m_new)) : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(lane_base + o_col + (uint32_t)(c * 32), o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                        tmem_st32(lane_base + o_col + (uint32_t)(c * 32), o);
                    }
                    if (want) l *= corr;
                }
                if (want) m = m_new;
            }
            // P = 2^(s c - m), two at a time; of every eight, POLY pairs come out of the multiply-add units
            const uint64_t c2 = pair_of(a.scale_log2e, a.scale_log2e);
            const float neg_use = m == -INFINITY ? 0.f : -m;
            const uint64_t neg2 = pair_of(neg_use, neg_use);
            uint64_t sum0 = 0ull, sum1 = 0ull;
#pragma unroll
            for (int k = 0; k < TN; k += 2) {
                const uint64_t x = fma2(pair_of(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), c2, neg2);
                const uint64_t p = (k >> 1) % 8 < POLY ? exp2_poly(x) : pair_of(fast_exp2(low_of(x)), fast_exp2(high_of(x)));
                if (k & 2) sum1 = add2(sum1, p);
                else sum0 = add2(sum0, p);
                s[k >> 1] = pack_bf16(low_of(p), high_of(p));
            }
            sum0 = add2(sum0, sum1);
            l += low_of(sum0) + high_of(sum0);
            if (!pv_seen) {
                ok = mbar_wait(&sm.pv_done[i], (uint32_t)(it - 1) & 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
            }
#pragma unroll
            for (int c = 0; c < TN / 64; ++c) tmem_st32_nowait(lane_base + p_col + (uint32_t)(c * 32), s + c * 32);
            // Rows of V that nobody sees must not carry NaN bits into P.V (0 * NaN): those in front of the window and behind the context
            // (not loaded, or the rest of a page), of other trees and of padding become zeros before this block's P.V. Tile 0, whose
            // product is issued first, does it where both tiles take the block.
            if ((i == 0 || alternate) && (!paged || key0 + TN > t.ctx || key0 < lo)) {
                const int st = j % KV_STAGES;
                ok = mbar_wait(&sm.v_full[st], (uint32_t)(j / KV_STAGES) & 1u, abort_flag);
                if (!ok) break;
                if (paged ? key0 + r >= t.ctx || key0 + r < lo : node0 + r >= t.n || sm.tree.depth[node0 + r] < 0) {
#pragma unroll
                    for (int c = 0; c < HD * 2 / 16; ++c) reinterpret_cast<uint4*>(sm.v[st] + r * HD * 2)[c] = make_uint4(0, 0, 0, 0);
                }
                proxy_fence();
            }
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&sm.p_full[i]);
        }
        if (ok && it > 0) ok = mbar_wait(&sm.pv_done[i], (uint32_t)(it - 1) & 1u, abort_flag);
        if (!ok && lane == 0) { *abort_flag = 1; atomicOr(a.err, CELLM_DEV_WAIT_TIMEOUT); }
        tc_fence_after();
        // One tile of rows: the second tile's results go to the first through the place of the keys, a row of 65 floats each (64 and
        // the banks would be the same for all). Every warp meets at the barriers, whatever became of its waits.
        float* room = reinterpret_cast<float*>(sm.k[0]);              // [TM][HD + 1], then [TM][2]
        float w_own = 1.f, w_room = 0.f;
        if (alternate) {
            asm volatile("bar.sync 2, 256;" ::: "memory");            // all products are done
            if (i == 1) {
#pragma unroll 1
                for (int c = 0; c < (it > 0 ? HD / 32 : 0); ++c) {
                    uint32_t o[32];
                    tmem_ld32(lane_base + o_col + (uint32_t)(c * 32), o);
#pragma unroll
                    for (int k = 0; k < 32; ++k) room[r * (HD + 1) + c * 32 + k] = __uint_as_float(o[k]);
                }
                room[TM * (HD + 1) + r * 2] = it > 0 ? m : -INFINITY, room[TM * (HD + 1) + r * 2 + 1] = l;
            }
            asm volatile("bar.sync 2, 256;" ::: "memory");
            if (i == 0) {
                const float m_room = room[TM * (HD + 1) + r * 2], top = fmaxf(it > 0 ? m : -INFINITY, m_room), use = top == -INFINITY ? 0.f : top;
                w_own = it > 0 ? exp2f(m - use) : 0.f, w_room = exp2f(m_room - use);
                l = (it > 0 ? l * w_own : 0.f) + (w_room != 0.f ? room[TM * (HD + 1) + r * 2 + 1] * w_room : 0.f);
                m = top;
            }
        }
        if (ok && !(alternate && i == 1)) {
            const long long gr = (long long)(t.t_base + node) * a.nh + t.kvh * G + r % G;
            const bool parted = a.nsplit > 1, any = it > 0 || alternate;
            const long long piece = t.split;
            const float inv = seeing && l != 0.f ? 1.0f / l : 0.f;
            if (parted && row_ok)
                *reinterpret_cast<float2*>(a.part_ml + (piece * a.T * a.nh + gr) * 2) = any && seeing ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                if (it > 0) {
                    tmem_ld32(lane_base + o_col + (uint32_t)(c * 32), o);
                }
                if (alternate) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        float v = w_own != 0.f ? __uint_as_float(o[k]) * w_own : 0.f;
                        if (w_room != 0.f) v = fmaf(room[r * (HD + 1) + c * 32 + k], w_room, v);
                        o[k] = __float_as_uint(v);
                    }
                }
                if (!(any && seeing)) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = 0u;
                }
                if (parted && row_ok) {
                    float4* dst = reinterpret_cast<float4*>(a.part_o + (piece * a.T * a.nh + gr) * HD + c * 32);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        dst[k] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                } else if (row_ok) {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + gr * HD + c * 32);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t w[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            w[x] = pack_bf16(__uint_as_float(o[8 * k + 2 * x]) * inv, __uint_as_float(o[8 * k + 2 * x + 1]) * inv);
                        dst[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {            // what is under way must not outlive this CTA's memory
        if ((warp == 0 || warp == 2) && lane == 0 && live) {
            const int issued = min(sm.issued[warp >> 1], n_blk);
            if (warp == 0) mbar_wait(&sm.q_full, 0, &sm.never);
            for (int j = max(0, issued - KV_STAGES); j < issued; ++j)
                mbar_wait(warp == 0 ? &sm.k_full[j % KV_STAGES] : &sm.v_full[j % KV_STAGES], (uint32_t)(j / KV_STAGES) & 1u, &sm.never);
        }
        if (warp == 1 && elect_one()) {      // the lane that issued the products
            umma_commit(&sm.drained);
            mbar_wait(&sm.drained, 0, &sm.never);
        }
        __syncthreads();
    }
    if (warp == 1) tmem_dealloc(tmem, TMEM_COLUMNS);
}

bool encode(CUtensorMap* out, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint32_t estr[3] = {1, 1, 1};
    return enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// rows of T nodes, `heads` heads of 64 each, `ld` elements between nodes; boxes of box_heads x box_nodes
bool encode_rows(CUtensorMap* out, const void* base, int T, int heads, long long ld, int box_heads, int box_nodes) {
    const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)heads, (cuuint64_t)T};
    const cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)ld * 2};
    const cuuint32_t box[3] = {(cuuint32_t)HD, (cuuint32_t)box_heads, (cuuint32_t)box_nodes};
    return encode(out, base, 3, dims, strides, box);
}

}  // namespace

bool attention_tree_tc_takes(const TreeArgs& a) {
    const int G = a.nh / a.nkv;
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k_new | (uintptr_t)a.v_new | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool | (uintptr_t)a.out;
    return a.hd == HD && a.scale_log2e > 0.f && at % 16 == 0 && a.q_ld % 8 == 0 && a.k_ld % 8 == 0 && a.v_ld % 8 == 0 &&
           a.q_ld > 0 && a.k_ld > 0 && a.v_ld > 0 && G <= TM && TM / G * G >= 96 &&
           a.num_pages > 0 && a.page_size >= 8 && a.page_size <= TN && (a.page_size & (a.page_size - 1)) == 0 && (long long)a.num_pages * a.nkv * a.page_size <= 0x7fffffffLL;
}

// part_o and part_ml hold a.nsplit pieces where there are more than one.
int attention_tree_tc_launch(const TreeArgs& given, cudaStream_t stream) {
    TreeArgs a = given;
    const int G = a.nh / a.nkv, tile_nodes = TM / G, alternate = a.most <= tile_nodes;
    CUtensorMap mq, mk, mv, mkn, mvn;
    const cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)a.num_pages * a.nkv * a.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)HD * 2};
    const cuuint32_t box[2] = {(cuuint32_t)HD, (cuuint32_t)a.page_size};
    if (!encode(&mk, a.k_pool, 2, dims, strides, box) || !encode(&mv, a.v_pool, 2, dims, strides, box) || !encode_rows(&mq, a.q, a.T, a.nh, a.q_ld, G, tile_nodes) ||
        !encode_rows(&mkn, a.k_new, a.T, a.nkv, a.k_ld, 1, TN) || !encode_rows(&mvn, a.v_new, a.T, a.nkv, a.v_ld, 1, TN))
        return CELLM_ERR_ARG;
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = cellm_allow_smem(allowed, (const void*)attention_tree_tc_kernel, sizeof(TreeTcSmem));
    if (e != cudaSuccess) return (int)e;
    const int pair = alternate ? tile_nodes : 2 * tile_nodes;
    a.tiles = (a.most + pair - 1) / pair;
    CELLM_RUN(attention_tree_tc_kernel, (unsigned)((long long)a.B * a.nkv * a.nsplit * a.tiles), THREADS, sizeof(TreeTcSmem), stream, mq, mk, mv, mkn, mvn, a, alternate);
    return CELLM_OK;
}
