// Beam search: the best continuations of a request's beams, and the beams' states and cached rows in their new order.
//
// Selection. A continuation (beam k, token v) of a request scores  s_k + x_kv - log sum_u exp x_ku;  the `keep` best of all
// beams * V are wanted, best first, equal ones by (k, v). The logits are read once:
//   beam_rows_kernel   every lane takes 64 logits of a row into registers and leaves their maximum; every warp leaves the sum
//                      of its 2,048 exponentials.
//   beam_pick_kernel   a block a request: the rows' log-sums, a lower bound of the worst wanted score out of the lanes' maxima
//                      (the keep-th largest maximum of 128 disjoint sets of them), and the logits of the few lanes that reach it.
// Scores of different beams are compared, so the sums behind them must be good to more than a logit's own rounding: the
// exponentials carry an error of about 2^-25 each, their sums over lanes are 64-bit, and a score is the 64-bit sum
// s + ((x - max) - log sum exp(x - max)).
//
// Reordering is done in place: a thread reads its 16 bytes (or what the rows' alignment allows) of ALL beams of a request
// before it writes any, and no other thread touches those places, so no copy of the states is needed and no order of blocks
// matters.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int LANE_VALUES = 64;                       // logits of a row a lane holds
constexpr int WARP_VALUES = 32 * LANE_VALUES;
constexpr int ROW_WARPS = 4;
constexpr int MAX_BEAMS = 32, MAX_KEEP = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOG2E_REST = (float)(1.4426950408889634074 - (double)1.4426950408889634f);
constexpr float ROUND_MAGIC = 12582912.f;             // 1.5 * 2^23: adding it rounds to a whole number, held in the low bits
constexpr float FAST_LIMIT = 2.9e6f;                  // behind it x log2(e) leaves the range of that

// Of one warp's logits: the largest, and the sum of their exponentials over 2^power, or over exp(best) where power is LARGE.
struct RowPart {
    float best;
    int power;
    double sum;
};
constexpr int LARGE = 1 << 30;

// 2^(x log2 e - n0) with n0 a whole number near the largest x log2 e. x log2 e = n + f with |f| <= 1/2 comes out of one rounding
// (n) and two multiply-adds with log2 e as a float and its remainder; 2^f = 1 + f P(f), P fitted (weighted least squares,
// reweighted towards the largest error) to 2.0e-9.
__device__ __forceinline__ float exp_to(float x, int n0) {
    const float r = fmaf(x, LOG2E, ROUND_MAGIC), n = r - ROUND_MAGIC;
    const float f = fmaf(x, LOG2E_REST, fmaf(x, LOG2E, -n));
    float p = 0.00015353357593994588f;
    p = fmaf(p, f, 0.0013398876180872321f);
    p = fmaf(p, f, 0.009618437848985195f);
    p = fmaf(p, f, 0.055503323674201965f);
    p = fmaf(p, f, 0.24022647738456726f);
    p = fmaf(p, f, 0.6931471824645996f);
    p = fmaf(p, f, 1.0f);
    return __uint_as_float(__float_as_uint(p) + ((__float_as_uint(r) - (uint32_t)n0) << 23));
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The 16 bytes of a row from its logit `at` on, logits behind the last as -inf. Which logits a lane takes goes by their places in the
// row alone, so that equal rows have equal sums wherever they lie: a row that does not start on a 16-byte border (`off` bytes behind
// one) is read in aligned pieces of which each lane joins two (the second is its neighbour's first).
template <typename T>
__device__ __forceinline__ void load_logits(float* x, const T* row, int at, int V, int off) {
    constexpr int N = 16 / sizeof(T);
    if (at + N <= V) {
        uint32_t u[8];
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row + at) - off);
        const uint4 w = __ldcs(src);
        u[0] = w.x, u[1] = w.y, u[2] = w.z, u[3] = w.w;
        if (off != 0) {
            const uint4 z = __ldcs(src + 1);
            u[4] = z.x, u[5] = z.y, u[6] = z.z, u[7] = z.w;
            if (off & 8) {
#pragma unroll
                for (int i = 0; i < 6; ++i) u[i] = u[i + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int i = 0; i < 5; ++i) u[i] = u[i + 1];
            }
            if (sizeof(T) == 2 && (off & 2)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = __funnelshift_r(u[i], u[i + 1], 16);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                x[i] = __uint_as_float(u[i]);
            } else {
                x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = at + i < V ? to_float(row[at + i]) : -INFINITY;
    }
}

// The first logit of piece i of lane `lane` of warp part `part` of a row.
template <typename T>
__device__ __forceinline__ int piece_at(int part, int i, int lane) {
    return part * WARP_VALUES + (i * 32 + lane) * (16 / (int)sizeof(T));
}

// grid (ceil(parts / ROW_WARPS), rows): tops [rows][parts * 32], sums [rows][parts]
template <typename T>
__global__ void __launch_bounds__(ROW_WARPS * 32)
beam_rows_kernel(float* __restrict__ tops, RowPart* __restrict__ sums, const T* __restrict__ logits, long long ld, int V, int parts,
                 const uint8_t* __restrict__ done) {
    constexpr int N = 16 / sizeof(T), PIECES = LANE_VALUES / N;
    pdl_wait();
    pdl_trigger();
    const int row = blockIdx.y, part = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (part >= parts || (done != nullptr && done[row])) return;
    const T* src = logits + (long long)row * ld;
    const int off = (int)(reinterpret_cast<uintptr_t>(src) & 15);
    float x[LANE_VALUES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) load_logits<T>(x + i * N, src, piece_at<T>(part, i, lane), V, off);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < LANE_VALUES; ++i) top = fmaxf(top, x[i]);            // (a NaN is passed over)
    tops[((long long)row * parts + part) * 32 + lane] = top;
    const float best = warp_max(top);
    double sum = 0.0;
    int power = LARGE;
    if (fabsf(best) < FAST_LIMIT) {
        const int n0 = (int)rintf(best * LOG2E);
        const float least = (float)(n0 - 125) * 0.6931472f;                   // what is smaller adds 2^-125 instead: nothing
        float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
        for (int i = 0; i < LANE_VALUES; i += 4) {
            s0 += exp_to(fmaxf(x[i], least), n0), s1 += exp_to(fmaxf(x[i + 1], least), n0);
            s2 += exp_to(fmaxf(x[i + 2], least), n0), s3 += exp_to(fmaxf(x[i + 3], least), n0);
        }
        power = n0, sum = warp_sum_d((double)(s0 + s1) + (double)(s2 + s3));
    } else {
        if (best > -INFINITY && best < INFINITY) {
            for (int i = 0; i < PIECES; ++i) {            // (read again: an index known only here would move the 64 out of registers)
                const int at = piece_at<T>(part, i, lane);
                for (int c = at; c < min(at + N, V); ++c) {
                    const float v = to_float(src[c]);
                    if (v > -INFINITY) sum += exp((double)v - (double)best);
                }
            }
        }
        sum = warp_sum_d(sum);
    }
    if (lane == 0) sums[(long long)row * parts + part] = RowPart{best, power, sum};
}

constexpr int PICK_THREADS = 512, PICK_SETS = 128, PICK_ROOM = 1024;

struct Found {
    double score[PICK_ROOM];
    uint32_t at[PICK_ROOM];           // k * V + v
};
__device__ __forceinline__ bool better(double a, uint32_t ai, double b, uint32_t bi) { return a > b || (a == b && ai < bi); }

// The `keep` best of the n found, in order, to the front. All threads; ends with a barrier. A find's rank is the number of better ones.
__device__ void sort_found(Found& f, int n, int keep) {
    constexpr int PER = PICK_ROOM / PICK_THREADS;
    double s[PER];
    uint32_t at[PER];
    int rank[PER];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int me = threadIdx.x + i * PICK_THREADS;
        rank[i] = keep;
        if (me >= n) continue;
        s[i] = f.score[me], at[i] = f.at[me];
        int r = 0;
        for (int j = 0; j < n; ++j) r += better(f.score[j], f.at[j], s[i], at[i]) ? 1 : 0;
        rank[i] = r;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (rank[i] < keep) f.score[rank[i]] = s[i], f.at[rank[i]] = at[i];
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(PICK_THREADS)
beam_pick_kernel(float* __restrict__ out_scores, int* __restrict__ out_parents, int* __restrict__ out_tokens, const float* __restrict__ tops,
                 const RowPart* __restrict__ sums, const T* __restrict__ logits, long long ld, int V, int parts, const float* __restrict__ scores,
                 const uint8_t* __restrict__ done, int beams, int keep, int pad) {
    constexpr int N = 16 / sizeof(T);
    __shared__ Found found;
    __shared__ double base_s[MAX_BEAMS], best_s[MAX_BEAMS], log_s[MAX_BEAMS], set_top[PICK_SETS];
    __shared__ double least_s;
    __shared__ int n_found, n_hot;
    __shared__ uint32_t hot[PICK_THREADS];
    const int r = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) n_found = 0, n_hot = 0, least_s = -INFINITY;
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    // ---- the rows' log-sums; a finished beam offers itself alone
    for (int k = warp; k < beams; k += PICK_THREADS / 32) {
        const int row = r * beams + k;
        const double s = (double)scores[row];
        const bool over = done != nullptr && done[row];
        double best = -INFINITY, sum = 0.0;
        if (!over) {
            const RowPart* p = sums + (long long)row * parts;
            for (int i = lane; i < parts; i += 32) best = fmax(best, (double)p[i].best);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) best = fmax(best, __shfl_xor_sync(0xffffffffu, best, o));
            for (int i = lane; i < parts; i += 32) {
                const RowPart w = p[i];
                if (w.sum > 0.0) sum += w.sum * (w.power == LARGE ? exp((double)w.best - best) : exp2((double)w.power - best * 1.4426950408889634074));
            }
            sum = warp_sum_d(sum);
        }
        if (lane == 0) {
            // nothing of a beam with no score, or of a row without a finite logit, is offered
            base_s[k] = over || !(s > -INFINITY) || !(sum > 0.0) ? -INFINITY : s;
            best_s[k] = best, log_s[k] = log(sum);
            if (over && s > -INFINITY) {
                const int i = atomicAdd(&n_found, 1);
                found.score[i] = s, found.at[i] = (uint32_t)k * (uint32_t)V + (uint32_t)pad;
            }
        }
    }
    __syncthreads();
    // ---- a lower bound of the keep-th best score
    const int groups = parts * 32, all = beams * groups;
    const float* my_tops = tops + (long long)r * all;
    auto group_score = [&](int i) {
        const int k = i / groups;
        const double b = base_s[k];
        if (b == -INFINITY) return -(double)INFINITY;                         // (its maxima may never have been written)
        return b + (((double)my_tops[i] - best_s[k]) - log_s[k]);
    };
    {
        double top = -INFINITY;
        for (int i = threadIdx.x; i < all; i += PICK_THREADS) top = fmax(top, group_score(i));
        constexpr int PER_SET = PICK_THREADS / PICK_SETS;
#pragma unroll
        for (int o = PER_SET / 2; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (threadIdx.x % PER_SET == 0) set_top[threadIdx.x / PER_SET] = top;
        __syncthreads();
        if (threadIdx.x < PICK_SETS) {
            const double me = set_top[threadIdx.x];
            int above = 0;
            for (int j = 0; j < PICK_SETS; ++j) above += better(set_top[j], j, me, threadIdx.x) ? 1 : 0;
            if (above == keep - 1) least_s = me;
        }
        __syncthreads();
    }
    // ---- the logits of the groups that reach it, a run of groups after the other; when the room fills up the best so far stay, and
    // the worst of them is the new bound
    double least = least_s;
    uint32_t least_at = 0xffffffffu;          // a find must be better than (least, least_at), or equal least where that is the first bound
    for (int from = 0; from < all; from += PICK_THREADS) {
        const int g = from + threadIdx.x;
        const double gs = g < all ? group_score(g) : -INFINITY;
        if (gs >= least && gs > -INFINITY) hot[atomicAdd(&n_hot, 1)] = (uint32_t)g;
        __syncthreads();
        const int n = n_hot;
        for (int first = 0; first < n * LANE_VALUES; first += PICK_THREADS) {
            const int e = first + threadIdx.x;
            if (e < n * LANE_VALUES) {
                const int group = (int)hot[e / LANE_VALUES], k = group / groups, gi = group % groups, at = e % LANE_VALUES;
                const T* row = logits + (long long)(r * beams + k) * ld;
                const int v = piece_at<T>(gi >> 5, at / N, gi & 31) + at % N;
                if (v < V) {
                    const double s = base_s[k] + (((double)to_float(row[v]) - best_s[k]) - log_s[k]);
                    const uint32_t id = (uint32_t)k * (uint32_t)V + (uint32_t)v;
                    if (s > -INFINITY && (s > least || (s == least && id <= least_at))) {
                        const int i = atomicAdd(&n_found, 1);
                        found.score[i] = s, found.at[i] = id;
                    }
                }
            }
            __syncthreads();
            const int have = n_found;
            __syncthreads();                   // (nobody adds to it before all have read it)
            if (have > PICK_ROOM - PICK_THREADS) {
                sort_found(found, have, keep);
                if (threadIdx.x == 0) n_found = keep;
                least = found.score[keep - 1], least_at = found.at[keep - 1];
                __syncthreads();
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) n_hot = 0;
        __syncthreads();
    }
    const int have = n_found;
    sort_found(found, have, keep);
    for (int i = threadIdx.x; i < keep; i += PICK_THREADS) {
        const bool fine = i < have;
        out_scores[r * keep + i] = fine ? (float)found.score[i] : -INFINITY;
        out_parents[r * keep + i] = fine ? (int)(found.at[i] / (uint32_t)V) : -1;
        out_tokens[r * keep + i] = fine ? (int)(found.at[i] % (uint32_t)V) : -1;
    }
}

// ---------------------------------------------------------------- reordering
template <int KMAX, typename W, typename Place>
__device__ __forceinline__ void reorder_unit(int beams, const int* parents, const Place& place) {
    W held[KMAX];
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
        if (k < beams && parents[k] >= 0) held[k] = *place(parents[k]);
#pragma unroll
    for (int k = 0; k < KMAX; ++k)
        if (k < beams && parents[k] >= 0) *place(k) = held[k];
}

// The parents of request r into shared memory: -1 for a beam that stays as it is (its own parent, none, or one that is reported).
__device__ __forceinline__ void read_parents(int* to, const int* parents, int r, int beams, int* err) {
    if (threadIdx.x < beams) {
        int p = parents[r * beams + threadIdx.x];
        if (p >= beams) { atomicOr(err, CELLM_DEV_BAD_SLOT); p = -1; }
        to[threadIdx.x] = p < 0 || p == threadIdx.x ? -1 : p;
    }
}

// grid (blocks over a slot's units, items, requests); state [items][slots][units] of W
template <int KMAX, typename W>
__global__ void __launch_bounds__(256)
reorder_states_kernel(W* state, const int* __restrict__ slot_ids, const int* __restrict__ parents, int beams, int slots, long long units, int* __restrict__ err) {
    __shared__ int from[MAX_BEAMS];
    __shared__ long long slot_at[MAX_BEAMS];
    pdl_wait();
    const int r = blockIdx.z;
    read_parents(from, parents, r, beams, err);
    __syncthreads();
    if (threadIdx.x < beams) {
        const int s = slot_ids[r * beams + threadIdx.x];
        slot_at[threadIdx.x] = s < 0 || s >= slots ? -1 : s * units;
        if (s < 0 || s >= slots) atomicOr(err, CELLM_DEV_BAD_SLOT);
    }
    __syncthreads();
    // a beam without a slot, or whose parent has none, is left alone
    if (threadIdx.x < beams && from[threadIdx.x] >= 0 && (slot_at[threadIdx.x] < 0 || slot_at[from[threadIdx.x]] < 0)) from[threadIdx.x] = -1;
    __syncthreads();
    W* item = state + (long long)blockIdx.y * slots * units;
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256)
        reorder_unit<KMAX, W>(beams, from, [&](int k) { return item + slot_at[k] + u; });
}

// grid (blocks over rows, items, requests); pool [items][pages][nkv][page_size][units] of W; a beam's row of the block table names
// the pages of its rows. Rows starts[r] .. ends[r] - 1 of every beam of request r take those of its parent. An entry of -1 is a
// page that was given back: its rows are passed over.
template <int KMAX, typename W>
__global__ void __launch_bounds__(256)
reorder_pages_kernel(W* pool, const int* __restrict__ block_table, int bt_stride, const int* __restrict__ starts, const int* __restrict__ ends,
                     const int* __restrict__ parents, int beams, int pages, int nkv, int page_size, int units, int* __restrict__ err) {
    __shared__ int from[MAX_BEAMS];
    pdl_wait();
    const int r = blockIdx.z;
    read_parents(from, parents, r, beams, err);
    __syncthreads();
    const int begin = max(0, starts[r]), end = (int)min((long long)ends[r], (long long)bt_stride * page_size);
    if (end < ends[r] && threadIdx.x == 0) atomicOr(err, CELLM_DEV_BAD_PAGE);
    const int per_row = nkv * units;
    W* item = pool + (size_t)blockIdx.y * pages * per_row * page_size;
    const long long total = (long long)max(0, end - begin) * per_row;
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < total; u += (long long)gridDim.x * 256) {
        const int at = begin + (int)(u / per_row), rest = (int)(u % per_row), h = rest / units, x = rest % units;
        const int* entry = block_table + (long long)r * beams * bt_stride + at / page_size;
        const size_t in_page = ((size_t)h * page_size + at % page_size) * units + x;
        W held[KMAX];
        int to[KMAX];
#pragma unroll
        for (int k = 0; k < KMAX; ++k) {
            to[k] = -1;
            if (k >= beams || from[k] < 0) continue;
            const int p = entry[(long long)k * bt_stride], src = entry[(long long)from[k] * bt_stride];
            if (p >= pages || src >= pages) { atomicOr(err, CELLM_DEV_BAD_PAGE); continue; }
            if (p < 0 || src < 0) continue;
            to[k] = p;
            held[k] = item[(size_t)src * per_row * page_size + in_page];
        }
#pragma unroll
        for (int k = 0; k < KMAX; ++k)
            if (to[k] >= 0) item[(size_t)to[k] * per_row * page_size + in_page] = held[k];
    }
}

template <typename W>
int launch_states(void* state, const int* slot_ids, const int* parents, int requests, int beams, int items, int slots, long long bytes, int* err,
                  cudaStream_t stream) {
    const long long units = bytes / (long long)sizeof(W);
    const unsigned blocks = (unsigned)std::min<long long>((units + 255) / 256, 4096);
    const dim3 grid(blocks, (unsigned)items, (unsigned)requests);
#define GO(K_) CELLM_RUN((reorder_states_kernel<K_, W>), grid, 256, 0, stream, (W*)state, slot_ids, parents, beams, slots, units, err)
    if (beams <= 4) GO(4);
    else if (beams <= 8) GO(8);
    else if (beams <= 16) GO(16);
    else GO(32);
#undef GO
    return CELLM_OK;
}

template <typename W>
int launch_pages(void* pool, const int* block_table, int bt_stride, const int* starts, const int* ends, const int* parents, int requests, int beams,
                 int items, int pages, int nkv, int page_size, int row_bytes, int* err, cudaStream_t stream) {
    const int units = row_bytes / (int)sizeof(W);
    const long long most = (long long)bt_stride * page_size * nkv * units;
    const unsigned blocks = (unsigned)std::max<long long>(1, std::min<long long>((most + 255) / 256, 512));
    const dim3 grid(blocks, (unsigned)items, (unsigned)requests);
#define GO(K_) CELLM_RUN((reorder_pages_kernel<K_, W>), grid, 256, 0, stream, (W*)pool, block_table, bt_stride, starts, ends, parents, beams, pages, nkv, page_size, units, err)
    if (beams <= 4) GO(4);
    else if (beams <= 8) GO(8);
    else if (beams <= 16) GO(16);
    else GO(32);
#undef GO
    return CELLM_OK;
}

template <typename T>
int launch_select(float* out_scores, int* out_parents, int* out_tokens, float* tops, void* sums, const void* logits, long long ld, int V, int requests,
                  int beams, int keep, const float* scores, const uint8_t* done, int pad, int parts, cudaStream_t stream) {
    const dim3 grid((unsigned)((parts + ROW_WARPS - 1) / ROW_WARPS), (unsigned)(requests * beams));
    CELLM_RUN(beam_rows_kernel<T>, grid, ROW_WARPS * 32, 0, stream, tops, (RowPart*)sums, (const T*)logits, ld, V, parts, done);
    CELLM_RUN(beam_pick_kernel<T>, requests, PICK_THREADS, 0, stream, out_scores, out_parents, out_tokens, tops, (const RowPart*)sums, (const T*)logits, ld, V,
              parts, scores, done, beams, keep, pad);
    return CELLM_OK;
}

}  // namespace

// Warp parts of a row of V logits: the workspace holds 32 floats (tops) and 16 bytes (sums) for each part of every row.
CELLM_API int cellm_beam_parts(int V) { return (V + WARP_VALUES - 1) / WARP_VALUES; }

// The `keep` best continuations of each request's `beams` rows of logits [requests * beams][V] (rows ld apart) under the beams'
// scores: out_* [requests][keep], -1 and -inf where there are fewer. done: null, or a byte a row: such a beam offers (itself, pad) at
// its score and its logits are not read.
CELLM_API int cellm_beam_select(float* out_scores, int* out_parents, int* out_tokens, float* tops, void* sums, const void* logits, long long ld, int V,
                                int requests, int beams, int keep, const float* scores, const uint8_t* done, int pad, int dtype, cudaStream_t stream) {
    if (requests <= 0) return CELLM_OK;
    if (dtype != CELLM_F32 && dtype != CELLM_BF16) return CELLM_ERR_DTYPE;
    if (V <= 0 || beams <= 0 || beams > MAX_BEAMS || keep <= 0 || keep > MAX_KEEP || ld < V || pad < 0 || pad >= V) return CELLM_ERR_SIZE;
    if ((long long)beams * (V + WARP_VALUES) > 0x7fffffffLL || (long long)requests * beams > 65535) return CELLM_ERR_SIZE;
    if (!out_scores || !out_parents || !out_tokens || !tops || !sums || !logits || !scores) return CELLM_ERR_ARG;
    if ((((uintptr_t)sums) & 15) || (((uintptr_t)logits) & (dtype == CELLM_F32 ? 3 : 1))) return CELLM_ERR_ALIGN;
    const int parts = cellm_beam_parts(V);
    return dtype == CELLM_F32 ? launch_select<float>(out_scores, out_parents, out_tokens, tops, sums, logits, ld, V, requests, beams, keep, scores, done, pad, parts, stream)
                              : launch_select<__nv_bfloat16>(out_scores, out_parents, out_tokens, tops, sums, logits, ld, V, requests, beams, keep, scores, done, pad, parts, stream);
}

// state [items][slots][bytes], in place: the slot of beam k of request r takes what the slot of beam parents[r][k] held.
CELLM_API int cellm_reorder_states(void* state, const int* slot_ids, const int* parents, int requests, int beams, int items, int slots, long long bytes,
                                   int* err, cudaStream_t stream) {
    if (requests <= 0 || items <= 0 || bytes <= 0) return CELLM_OK;
    if (beams <= 0 || beams > MAX_BEAMS || slots <= 0 || items > 65535 || requests > 65535) return CELLM_ERR_SIZE;
    if (!state || !slot_ids || !parents || !err) return CELLM_ERR_ARG;
    const uintptr_t at = (uintptr_t)state | (uintptr_t)bytes;
#define GO(W_) return launch_states<W_>(state, slot_ids, parents, requests, beams, items, slots, bytes, err, stream)
    if (at % 16 == 0) GO(uint4);
    if (at % 4 == 0) GO(uint32_t);
    if (at % 2 == 0) GO(uint16_t);
#undef GO
    return CELLM_ERR_ALIGN;
}

// pool [items][pages][nkv][page_size][row_bytes], in place; block_table [requests * beams][bt_stride].
CELLM_API int cellm_reorder_pages(void* pool, const int* block_table, int bt_stride, const int* starts, const int* ends, const int* parents, int requests,
                                  int beams, int items, int pages, int nkv, int page_size, int row_bytes, int* err, cudaStream_t stream) {
    if (requests <= 0 || items <= 0 || row_bytes <= 0) return CELLM_OK;
    if (beams <= 0 || beams > MAX_BEAMS || pages <= 0 || nkv <= 0 || page_size <= 0 || bt_stride <= 0 || items > 65535 || requests > 65535) return CELLM_ERR_SIZE;
    if (!pool || !block_table || !starts || !ends || !parents || !err) return CELLM_ERR_ARG;
    const uintptr_t at = (uintptr_t)pool | (uintptr_t)row_bytes;
#define GO(W_) return launch_pages<W_>(pool, block_table, bt_stride, starts, ends, parents, requests, beams, items, pages, nkv, page_size, row_bytes, err, stream)
    if (at % 16 == 0) GO(uint4);
    if (at % 4 == 0) GO(uint32_t);
    if (at % 2 == 0) GO(uint16_t);
#undef GO
    return CELLM_ERR_ALIGN;
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_beam_select_packed(const long long* a, cudaStream_t stream) {
    return cellm_beam_select((float*)a[0], (int*)a[1], (int*)a[2], (float*)a[3], (void*)a[4], (const void*)a[5], (long long)a[6], (int)a[7],
        (int)a[8], (int)a[9], (int)a[10], (const float*)a[11], (const uint8_t*)a[12], (int)a[13], (int)a[14], stream);
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_reorder_states_packed(const long long* a, cudaStream_t stream) {
    return cellm_reorder_states((void*)a[0], (const int*)a[1], (const int*)a[2], (int)a[3], (int)a[4], (int)a[5], (int)a[6], (long long)a[7],
        (int*)a[8], stream);
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_reorder_pages_packed(const long long* a, cudaStream_t stream) {
    return cellm_reorder_pages((void*)a[0], (const int*)a[1], (int)a[2], (const int*)a[3], (const int*)a[4], (const int*)a[5], (int)a[6], (int)a[7],
        (int)a[8], (int)a[9], (int)a[10], (int)a[11], (int)a[12], (int*)a[13], stream);
}
