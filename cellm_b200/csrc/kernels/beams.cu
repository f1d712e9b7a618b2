// Beam search: the best continuations of a request's beams, and the beams' states and cached rows in their new order.
//
// Selection. A continuation (beam k, token v) of a request scores  s_k + x_kv - log sum_u exp x_ku;  the `keep` best of all
// beams * V are wanted, best first, equal ones by (k, v). The logits are read once:
//   beam_rows_kernel   every lane takes 64 logits of a row into registers and leaves their maximum; every warp leaves the sum
//                      of its 2,048 exponentials.
//   beam_pick_kernel   a block a request: the rows' log-sums, a lower bound of the worst wanted score out of the lanes' maxima
//                      (the keep-th largest maximum of 128 disjoint sets of them), and the logits of the few lanes that reach it.
// Scores of different beams are compared, so the sums behind them must be good to more than a logit's own rounding, and where a row's
// mass lies in many equal logits the errors of its exponentials add up: an exponential is off by 1.1e-7 of itself at most (mostly by
// 2^-25), eight are summed in 32 bits (another 1.8e-7 at most), the rest in 64, and a score is the 64-bit sum
// s + ((x - max) - log sum exp(x - max)), good to 3e-7.
//
// Reordering is done in place: a thread reads its 16 bytes (or what the rows' alignment allows) of ALL beams of a request
// before it writes any, and no other thread touches those places, so no copy of the states is needed and no order of blocks
// matters.
#include <algorithm>
#include <climits>

#include "mma_tiles.cuh"
#include "pairs.cuh"

namespace {

constexpr int LANE_VALUES = 64;                       // logits of a row a lane holds
constexpr int WARP_VALUES = 32 * LANE_VALUES;          // a warp's part of a row, worked on in halves
constexpr int HALF_VALUES = LANE_VALUES / 2;
constexpr int ROW_WARPS = 4;
constexpr int MAX_BEAMS = 32, MAX_KEEP = 64, MAX_VOCAB = 1 << 24;

// Of one half part's logits: the largest, and the sum of exp(x - unit). The unit is power * log 2, or the best where power is BY_BEST.
struct RowPart {
    float best;
    int power;
    double sum;
};
constexpr int BY_BEST = INT_MIN;
constexpr float BY_BEST_FROM = 32768.f;       // the best's magnitude from which on it is the unit: x - best is exact there for all that counts

// 2^-p exp(x) of two numbers. x log2 e = n + f with |f| <= 1/2: n comes out of the rounding of a multiply-add whose addend (1.5 * 2^23 - p) also
// takes p off, f out of two more that lose nothing of x (log2 e in two parts; x - best would be rounded where the two are far apart, and
// alike for equal logits). 2^f = 1 + f P(f), P fitted (weighted least squares, reweighted towards the largest error)
// with its first coefficient and then one after the other rounded to 32 bits: 3.0e-9 with the coefficients as they stand. What lies
// below `least`, best - 86, or is not a number, adds exp(-86) of the best: nothing.
__device__ __forceinline__ uint64_t exp_scaled(float a, float b, float least, uint64_t magic) {
    const uint64_t x = pair_of(fmaxf(a, least), fmaxf(b, least)), l2e = pair_of(1.4426950408889634f, 1.4426950408889634f);
    const uint64_t r = fma2(x, l2e, magic), rest = fma2(x, l2e, fma2(r, pair_of(-1.f, -1.f), magic));
    const uint64_t f = fma2(x, pair_of(1.925963033500011537e-8f, 1.925963033500011537e-8f), rest);
    uint64_t p = pair_of(0.00015326462744269520f, 0.00015326462744269520f);
    p = fma2(p, f, pair_of(0.0013390806270763278f, 0.0013390806270763278f));
    p = fma2(p, f, pair_of(0.0096185058355331421f, 0.0096185058355331421f));
    p = fma2(p, f, pair_of(0.055503599345684052f, 0.055503599345684052f));
    p = fma2(p, f, pair_of(0.24022647738456726f, 0.24022647738456726f));
    p = fma2(p, f, pair_of(0.6931471824645996f, 0.6931471824645996f));
    p = fma2(p, f, pair_of(1.0f, 1.0f));
    return pair_of(__uint_as_float(__float_as_uint(low_of(p)) + (__float_as_uint(low_of(r)) << 23)),
                   __uint_as_float(__float_as_uint(high_of(p)) + (__float_as_uint(high_of(r)) << 23)));
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The first logit of piece i of a lane from logit `from` of a row on.
template <typename T>
__device__ __forceinline__ int piece_at(int from, int i, int lane) {
    return from + (i * 32 + lane) * (16 / (int)sizeof(T));
}

// A warp's ring of half parts in shared memory: the aligned 16-byte pieces that they lie in.
template <typename T>
struct Ring {
    static constexpr int N = 16 / sizeof(T), PIECES = HALF_VALUES / N, STAGES = sizeof(T) == 4 ? 2 : 3;
    static constexpr int BLOCKS = 6;                                      // of ROW_WARPS warps that an SM holds
    uint4 piece[STAGES][PIECES * 32 + 1];
};

// Which logits a lane takes goes by their places in the row alone, so that equal rows have equal sums wherever they lie: of a row that
// starts `off` bytes behind a 16-byte border a lane joins its own piece and the next.
template <typename T>
__device__ __forceinline__ void ring_load(Ring<T>& ring, int stage, const T* row, int from, int V, int lane) {
    using R = Ring<T>;
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15);
    const char* src = reinterpret_cast<const char*>(row + from) - off + lane * 16;
    uint4* dst = &ring.piece[stage][lane];
    if (from + HALF_VALUES * 32 + R::N <= V) {
#pragma unroll
        for (int i = 0; i < R::PIECES; ++i) cp_async16(dst + i * 32, src + i * 512, 16);
        if (lane == 0) cp_async16(dst + R::PIECES * 32, src + R::PIECES * 512, 16);
    } else {
        const long long left = (long long)(V - from) * (int)sizeof(T) + off - lane * 16;       // bytes up to the row's end
#pragma unroll
        for (int i = 0; i <= R::PIECES; ++i)
            if (left > i * 512 && (i < R::PIECES || lane == 0)) cp_async16(dst + i * 32, src + i * 512, (int)min(16ll, left - i * 512));
    }
}
template <typename T>
__device__ __forceinline__ void ring_read(float (&x)[HALF_VALUES], const Ring<T>& ring, int stage, const T* row, int from, int V, int lane) {
    using R = Ring<T>;
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15);
#pragma unroll
    for (int i = 0; i < R::PIECES; ++i) {
        uint32_t u[8];
        const uint4 w = ring.piece[stage][i * 32 + lane];
        u[0] = w.x, u[1] = w.y, u[2] = w.z, u[3] = w.w;
        if (off != 0) {
            const uint4 z = ring.piece[stage][i * 32 + lane + 1];
            u[4] = z.x, u[5] = z.y, u[6] = z.z, u[7] = z.w;
            if (off & 8) {
#pragma unroll
                for (int c = 0; c < 6; ++c) u[c] = u[c + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int c = 0; c < 5; ++c) u[c] = u[c + 1];
            }
            if (sizeof(T) == 2 && (off & 2)) {
#pragma unroll
                for (int c = 0; c < 4; ++c) u[c] = __funnelshift_r(u[c], u[c + 1], 16);
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if constexpr (sizeof(T) == 4) {
                x[i * R::N + c] = __uint_as_float(u[c]);
            } else {
                x[i * R::N + 2 * c] = __uint_as_float(u[c] << 16), x[i * R::N + 2 * c + 1] = __uint_as_float(u[c] & 0xffff0000u);
            }
        }
    }
    if (from + WARP_VALUES / 2 > V) {             // a row's last logits: what lies behind them is none
#pragma unroll
        for (int k = 0; k < HALF_VALUES; ++k)
            if (piece_at<T>(from, k / R::N, lane) + k % R::N >= V) x[k] = -INFINITY;
    }
}

// tops [rows][parts * 32], sums [rows][parts * 2]. The warps of a grid that fills the SMs take parts in turn, the next halves on their
// way through a ring of the warp's own while it works on one. 512 rows of 65,536 32-bit logits (134 MB): 31 us,
// 4.3 TB/s, with 56 % of the issue slots taken: neither limit is reached, a warp's halves wait in turn for memory and for one another's
// instructions (pick included 40 us; 16-bit logits, 67 MB, 36 us; steps on the way, with an exponential of fewer bits: 83 us with the warps loading in step, 51 with the ring and exponentials of any sign, 42 with those below
// the best alone).
template <typename T>
__global__ void __launch_bounds__(ROW_WARPS * 32, Ring<T>::BLOCKS)
beam_rows_kernel(float* __restrict__ tops, RowPart* __restrict__ sums, const T* __restrict__ logits, long long ld, int V, int parts, int rows,
                 const uint8_t* __restrict__ done) {
    using R = Ring<T>;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    Ring<T>& ring = reinterpret_cast<Ring<T>*>(ring_smem)[threadIdx.x >> 5];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, stride = gridDim.x * ROW_WARPS, first = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    const int row_step = stride / parts, part_step = stride % parts;
    // a place among the warp's halves: one runs ahead to load, one works
    struct At {
        int row, part, half;
    };
    auto advance = [&](At& at) {
        if ((at.half ^= 1) != 0) return;
        at.row += row_step, at.part += part_step;
        if (at.part >= parts) at.part -= parts, ++at.row;
    };
    auto looked_at = [&](const At& at) { return at.row < rows && !(done != nullptr && done[at.row]); };
    At load = {first / parts, first % parts, 0}, at = load;
    auto fetch = [&](int stage) {
        if (looked_at(load)) ring_load<T>(ring, stage, logits + load.row * ld, load.part * WARP_VALUES + load.half * (WARP_VALUES / 2), V, lane);
        cp_async_commit();
        advance(load);
    };
#pragma unroll
    for (int s = 0; s < R::STAGES; ++s) fetch(s);
    float top = -INFINITY;
    for (int stage = 0; at.row < rows; advance(at), stage = stage + 1 == R::STAGES ? 0 : stage + 1) {
        const int from = at.part * WARP_VALUES + at.half * (WARP_VALUES / 2);
        const bool wanted = looked_at(at);
        cp_async_wait<R::STAGES - 1>();
        __syncwarp();
        float x[HALF_VALUES];
        if (wanted) ring_read<T>(x, ring, stage, logits + at.row * ld, from, V, lane);
        __syncwarp();
        fetch(stage);
        if (!wanted) continue;
        float mine = -INFINITY, other = -INFINITY;
#pragma unroll
        for (int k = 0; k < HALF_VALUES; k += 4)                              // (a NaN is passed over)
            mine = fmaxf(fmaxf(mine, x[k]), x[k + 1]), other = fmaxf(fmaxf(other, x[k + 2]), x[k + 3]);
        mine = fmaxf(mine, other);
        top = at.half ? fmaxf(top, mine) : mine;
        const float best = warp_max(mine);
        double sum = 0.0;
        int power = BY_BEST;
        if (fabsf(best) < INFINITY) {                                         // (no logit at all, or one that has no meaning: no sum)
            float unit = best;
            if (fabsf(best) < BY_BEST_FROM) {
                unit = 0.f, power = __float2int_rn(best * 1.4426950408889634f);
            } else {
#pragma unroll
                for (int k = 0; k < HALF_VALUES; ++k) x[k] -= best;
            }
            const float least = (best - unit) - 86.f, base = 12582912.f - (unit == 0.f ? (float)power : 0.f);
            const uint64_t magic = pair_of(base, base);
            auto quad = [&](int k) { return add2(exp_scaled(x[k], x[k + 1], least, magic), exp_scaled(x[k + 2], x[k + 3], least, magic)); };
            auto eight = [&](int k) { return add2(quad(k), quad(k + 4)); };
#pragma unroll
            for (int k = 0; k < HALF_VALUES; k += 16) {                       // (by halves: equal numbers add up without a rounding)
                const uint64_t s = add2(eight(k), eight(k + 8));
                sum += (double)low_of(s) + (double)high_of(s);
            }
            sum = warp_sum_d(sum);
        }
        const long long part = (long long)at.row * parts + at.part;
        if (lane == 0) sums[2 * part + at.half] = RowPart{best, power, sum};
        if (at.half) tops[part * 32 + lane] = top;
    }
}

// exp(d) for d <= 1/2 in 64 bits, to 2.0e-9: as exp_scaled, with the fit's own coefficients. The picking block runs its code once, so what
// it calls is short.
__device__ __forceinline__ double exp_short(double d) {
    d = fmax(d, -600.0) * 1.4426950408889634074;
    const double n = rint(d), f = d - n;
    double p = 0.00015353361911178411;
    p = fma(p, f, 0.0013398874414638218);
    p = fma(p, f, 0.0096184373576691552);
    p = fma(p, f, 0.055503324711243029);
    p = fma(p, f, 0.2402264791362882);
    p = fma(p, f, 0.69314720285506826);
    return fma(p, f, 1.0) * __hiloint2double((1023 + (int)n) << 20, 0);
}
// log(s) for s >= 1/2: the 32-bit logarithm and one step of Newton's method
__device__ __forceinline__ double log_short(double s) {
    const double y = (double)logf((float)s);
    return y + (s * exp_short(-y) - 1.0);
}

// exp(unit - best) of a part's unit and the best of its row
__device__ __forceinline__ double unit_over(const RowPart& w, float best) {
    return exp_short((w.power == BY_BEST ? (double)w.best : w.power * 0.69314718055994530942) - (double)best);
}

constexpr int PICK_THREADS = 512, PICK_SETS = 128, PICK_ROOM = 1024, SUMS_HELD = 4, HELD = 16, HOT_ROOM = HELD * PICK_THREADS;

struct Found {
    double score[PICK_ROOM];
    uint32_t at[PICK_ROOM];           // k * V + v
};
struct Best {
    double score[MAX_KEEP];
    uint32_t at[MAX_KEEP];
};
__device__ __forceinline__ bool better(double a, uint32_t ai, double b, uint32_t bi) { return a > b || (a == b && ai < bi); }

// The `keep` best of the n found, in order, to the front of `to`. All threads; ends with a barrier. A find's rank is the number of better
// ones, which eight threads count together.
__device__ void sort_found(const Found& f, Best& to, int n, int keep) {
    const int part = threadIdx.x & 7;
    __syncthreads();
    for (int base = 0; base < n; base += PICK_THREADS / 8) {
        const int me = min(base + (int)(threadIdx.x >> 3), n - 1);
        const double s = f.score[me];
        const uint32_t at = f.at[me];
        int rank = 0;
#pragma unroll 4
        for (int j = part; j < n; j += 8) rank += better(f.score[j], f.at[j], s, at) ? 1 : 0;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        if (part == 0 && rank < keep) to.score[rank] = s, to.at[rank] = at;       // (equal places hold equal values)
    }
    __syncthreads();
}

// A block a request, so that no launch comes behind it: 512 rows of 64 requests 10 us, bound by its barriers (a dozen phases of few
// instructions each) and not by its reads.
template <typename T>
__global__ void __launch_bounds__(PICK_THREADS)
beam_pick_kernel(float* __restrict__ out_scores, int* __restrict__ out_parents, int* __restrict__ out_tokens, const float* __restrict__ tops,
                 const RowPart* __restrict__ sums, const T* __restrict__ logits, long long ld, int V, int parts, const float* __restrict__ scores,
                 const uint8_t* __restrict__ done, int beams, int keep, int pad, unsigned long long per_part) {
    constexpr int N = 16 / sizeof(T), WARPS = PICK_THREADS / 32;
    __shared__ Found found;
    __shared__ Best kept;
    __shared__ double base_s[MAX_BEAMS], best_s[MAX_BEAMS], log_s[MAX_BEAMS];
    __shared__ __align__(16) float set_top[PICK_SETS + 16];
    __shared__ float least_s, base_f[MAX_BEAMS], best_f[MAX_BEAMS], size_f[MAX_BEAMS];
    __shared__ int n_found, n_hot;
    extern __shared__ uint32_t hot[];          // [HOT_ROOM]
    const int r = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) n_found = 0, n_hot = 0, least_s = -INFINITY;
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    // ---- the rows' log-sums; a finished beam offers itself alone
    for (int k = warp; k < beams; k += WARPS) {
        const int row = r * beams + k;
        // all that is read of a beam is asked for before any of it is used
        const RowPart* p = sums + 2ll * row * parts;
        RowPart w[SUMS_HELD];
#pragma unroll
        for (int c = 0; c < SUMS_HELD; ++c) {
            w[c] = RowPart{-INFINITY, 0, 0.0};
            if (lane + c * 32 < 2 * parts) w[c] = p[lane + c * 32];
        }
        const double s = (double)scores[row];
        const bool over = done != nullptr && done[row];           // (its sums were never written, and are not used)
        float best = -INFINITY;
#pragma unroll
        for (int c = 0; c < SUMS_HELD; ++c) best = fmaxf(best, w[c].best);
        for (int i = lane + SUMS_HELD * 32; i < 2 * parts; i += 32) best = fmaxf(best, p[i].best);
        best = warp_max(best);
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < SUMS_HELD; ++c)
            if (w[c].sum > 0.0) sum += w[c].sum * unit_over(w[c], best);
        for (int i = lane + SUMS_HELD * 32; i < 2 * parts; i += 32)
            if (p[i].sum > 0.0) sum += p[i].sum * unit_over(p[i], best);
        sum = warp_sum_d(sum);
        if (lane == 0) {
            // nothing of a beam with no score, or of a row without a finite logit, is offered
            const bool offers = !over && s > -INFINITY && sum > 0.0;
            const double log_sum = offers ? log_short(sum) : 0.0;
            base_s[k] = offers ? s : -INFINITY, best_s[k] = (double)best, log_s[k] = log_sum;
            base_f[k] = offers ? (float)(s - log_sum) : -INFINITY, best_f[k] = best;
            size_f[k] = offers ? fabsf((float)s) + fabsf((float)log_sum) : 0.f;
            if (over && s > -INFINITY) {
                const int i = atomicAdd(&n_found, 1);
                found.score[i] = s, found.at[i] = (uint32_t)k * (uint32_t)V + (uint32_t)pad;
            }
        }
    }
    __syncthreads();
    // ---- a lower bound of the keep-th best score, in 32 bits: a lane's best score is known to within 2^-21 of what it is made of, and
    // that margin is taken off here and added where lanes are held against the bound
    const int groups = parts * 32, all = beams * groups;
    auto beam_of = [&](int i) { return (int)((((uint32_t)i >> 5) * per_part) >> 32); };  // i / groups: per_part is 2^32 / parts, rounded up
    const float* my_tops = tops + (long long)r * all;
    float size = lane < beams ? size_f[lane] : 0.f;
    size = 2.f * warp_max(size);
    auto margin = [&](float s) { return (fabsf(s) + size) * 4.8e-7f; };
    // the best scores of the lanes from + threadIdx.x, from + threadIdx.x + PICK_THREADS, ... of the request
    float held[HELD];
    auto hold = [&](int from) {
#pragma unroll
        for (int c = 0; c < HELD; ++c) {
            const int i = from + threadIdx.x + c * PICK_THREADS;
            held[c] = i < all ? my_tops[i] : -INFINITY;                       // (a finished beam's were never written, and are not used)
        }
#pragma unroll
        for (int c = 0; c < HELD; ++c) {
            const int k = min(beam_of(from + (int)threadIdx.x + c * PICK_THREADS), beams - 1);         // (the same of a warp's lanes)
            held[c] = base_f[k] > -INFINITY && held[c] > -INFINITY ? base_f[k] + (held[c] - best_f[k]) : -INFINITY;
        }
    };
    {
        float top = -INFINITY;
        for (int from = 0; from < all; from += HOT_ROOM) {
            hold(from);
#pragma unroll
            for (int c = 0; c < HELD; ++c)
                if (held[c] > -INFINITY) top = fmaxf(top, held[c] - margin(held[c]));
        }
        constexpr int PER_SET = PICK_THREADS / PICK_SETS;
#pragma unroll
        for (int o = PER_SET / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // a set's rank: its four threads count the better ones among a quarter of the sets each (quarters lie four floats further than
        // the banks are wide, so that the four read side by side)
        constexpr int QUARTER = PICK_SETS / PER_SET;
        const int me = threadIdx.x / PER_SET, q = threadIdx.x % PER_SET;
        if (q == 0) set_top[me / QUARTER * (QUARTER + 4) + me % QUARTER] = top;
        __syncthreads();
        int above = 0;
#pragma unroll
        for (int j = 0; j < QUARTER; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(set_top + q * (QUARTER + 4) + j);
            const int at = q * QUARTER + j;
            above += (v.x > top || (v.x == top && at < me)) + (v.y > top || (v.y == top && at + 1 < me)) + (v.z > top || (v.z == top && at + 2 < me)) +
                     (v.w > top || (v.w == top && at + 3 < me));
        }
#pragma unroll
        for (int o = PER_SET / 2; o > 0; o >>= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
        if (above == keep - 1 && q == 0) least_s = top;
        __syncthreads();
    }
    // ---- the logits of the lanes that reach it, HOT_ROOM lanes' tops at a time. A find goes into the room, unless that is full: then the best
    // so far stay, the worst of them is the new bound, and the run of lanes is gone through again with barriers (rows of few
    // different values come to that)
    float least_f = least_s;
    double least = (double)least_f;
    uint32_t least_at = 0xffffffffu;          // a find must be better than (least, least_at), or equal least where that is the first bound
    struct Place {
        int k, v;
    };
    auto place = [&](int e) {                 // e counts the hot lanes' logits
        const int group = (int)hot[e / LANE_VALUES], k = beam_of(group), gi = group - k * groups, at = e % LANE_VALUES;
        return Place{k, piece_at<T>((gi >> 5) * WARP_VALUES, at / N, gi & 31) + at % N};
    };
    auto logit = [&](const Place& p) { return p.v < V ? to_float(logits[(long long)(r * beams + p.k) * ld + p.v]) : -INFINITY; };
    auto find = [&](const Place& p, float x) {
        const double s = base_s[p.k] + (((double)x - best_s[p.k]) - log_s[p.k]);
        const uint32_t id = (uint32_t)p.k * (uint32_t)V + (uint32_t)p.v;
        if (s > -INFINITY && (s > least || (s == least && id <= least_at))) {
            const int i = atomicAdd(&n_found, 1);
            if (i < PICK_ROOM) found.score[i] = s, found.at[i] = id;
        }
    };
    for (int from = 0; from < all; from += HOT_ROOM) {
        if (all > HOT_ROOM) hold(from);
#pragma unroll
        for (int c = 0; c < HELD; ++c)
            if (held[c] > -INFINITY && held[c] + margin(held[c]) >= least_f) hot[atomicAdd(&n_hot, 1)] = (uint32_t)(from + threadIdx.x + c * PICK_THREADS);
        __syncthreads();
        const int n = n_hot * LANE_VALUES, before = n_found;
        __syncthreads();
        for (int e = threadIdx.x; e < n; e += 4 * PICK_THREADS) {             // four logits under way at once
            Place p[4];
            float x[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) p[c] = place(min(e + c * PICK_THREADS, n - 1)), x[c] = e + c * PICK_THREADS < n ? logit(p[c]) : -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (x[c] > -INFINITY) find(p[c], x[c]);
        }
        __syncthreads();
        if (n_found > PICK_ROOM) {
            __syncthreads();
            if (threadIdx.x == 0) n_found = before;
            __syncthreads();
            for (int first = 0; first < n; first += PICK_THREADS) {
                const int have = n_found;
                __syncthreads();              // (nobody adds to it before all have read it)
                if (have > PICK_ROOM - PICK_THREADS) {
                    sort_found(found, kept, have, keep);
                    if (threadIdx.x == 0) n_found = keep;
                    if (threadIdx.x < keep) found.score[threadIdx.x] = kept.score[threadIdx.x], found.at[threadIdx.x] = kept.at[threadIdx.x];
                    least = kept.score[keep - 1], least_at = kept.at[keep - 1], least_f = __double2float_rd(least);
                    __syncthreads();
                }
                if (first + threadIdx.x < n) {
                    const Place p = place(first + threadIdx.x);
                    const float x = logit(p);
                    if (x > -INFINITY) find(p, x);
                }
                __syncthreads();
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) n_hot = 0;
        __syncthreads();
    }
    const int have = n_found;
    sort_found(found, kept, have, keep);
    for (int i = threadIdx.x; i < keep; i += PICK_THREADS) {
        const bool fine = i < have;
        out_scores[r * keep + i] = fine ? (float)kept.score[i] : -INFINITY;
        out_parents[r * keep + i] = fine ? (int)(kept.at[i] / (uint32_t)V) : -1;
        out_tokens[r * keep + i] = fine ? (int)(kept.at[i] % (uint32_t)V) : -1;
    }
}

// ---------------------------------------------------------------- reordering
// U units of all beams, `step` apart, of which the first `left` exist: out of source(k), into target(k), below zero: that beam's stay.
// The places lie in shared memory and are read again for the stores: kept in registers they would take more of those than the units do.
template <int KMAX, int U, typename W, typename Source, typename Target>
__device__ __forceinline__ void reorder_units(int beams, W* base, int step, int left, const Source& source, const Target& target) {
    W held[KMAX][U];
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
        if (k >= beams) continue;
        const long long at = source(k);
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (at >= 0 && i < left) held[k][i] = base[at + i * step];
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int k = 0; k < KMAX; ++k) {
        if (k >= beams || source(k) < 0) continue;
        const long long at = target(k);
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i < left) base[at + i * step] = held[k][i];
    }
}
// Units narrower than 16 bytes that a thread of reorder_states has under way at once: what 32 registers hold of all beams (2 beams in units
// of 4 bytes, 336 MB: 58 us; 185 with one, which leaves too few bytes under way).
template <int KMAX, typename W>
constexpr int UNITS_AT_ONCE = KMAX >= 32 || sizeof(W) == 16 ? 1 : 32 / KMAX;

// The parents of request r into shared memory: -1 for a beam that stays as it is (its own parent, none, or one that is reported).
__device__ __forceinline__ void read_parents(int* to, const int* parents, int r, int beams, int* err) {
    if (threadIdx.x < beams) {
        int p = parents[r * beams + threadIdx.x];
        if (p >= beams || p < -1) { atomicOr(err, CELLM_DEV_BAD_SLOT); p = -1; }
        to[threadIdx.x] = p < 0 || p == threadIdx.x ? -1 : p;
    }
}

// grid (blocks over a slot's units, items, requests); state [items][slots][units] of W. Bound by memory: 8 requests of 8 beams that all
// move, 10 layers of 1 MB a state, 1 GB in all: 147 us, 7.0 TB/s (a parent of several beams is read once; 176 us with every beam's two
// places in registers, three blocks an SM). 16 beams 7.2 TB/s, 32 beams (206 registers, a block an SM) 5.5.
template <int KMAX, typename W>
__global__ void __launch_bounds__(256, KMAX <= 8 ? 4 : 1)
reorder_states_kernel(W* state, const int* __restrict__ slot_ids, const int* __restrict__ parents, int beams, int slots, long long units, int* __restrict__ err) {
    __shared__ int from[MAX_BEAMS];
    __shared__ long long slot_at[MAX_BEAMS], source_at[MAX_BEAMS];
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
    if (threadIdx.x < beams) source_at[threadIdx.x] = from[threadIdx.x] >= 0 && slot_at[threadIdx.x] >= 0 ? slot_at[from[threadIdx.x]] : -1;
    __syncthreads();
    W* item = state + (long long)blockIdx.y * slots * units;
    constexpr int U = UNITS_AT_ONCE<KMAX, W>;
    for (long long u = (long long)blockIdx.x * (256 * U) + threadIdx.x; u < units; u += (long long)gridDim.x * (256 * U))
        reorder_units<KMAX, U, W>(beams, item + u, 256, U == 1 ? 1 : (int)min((long long)U, (units - u + 255) / 256), [&](int k) { return source_at[k]; }, [&](int k) { return slot_at[k]; });
}

// What reorder_pages works on: up to two pools [items][pages][nkv][page_size][units] of W that share their pages.
struct PagedPools {
    void* pool[2];
    int units[2], pools;
};

// grid (blocks over rows, items * pools, requests); a beam's row of the block table names the pages of its rows. Rows starts[r] ..
// ends[r] - 1 of every beam of request r take those of its parent. An entry of -1 is a page that was given back: its rows are passed
// over. The places of ROWS rows of all beams are looked up once, into shared memory. Bound by memory: 16 requests of 8 beams, 1 GB
// read and written: 160 us, 96 % of a plain copy's rate (275 us with neighbouring threads on a position's heads, which lie far apart;
// 219 us with a launch a pool).
template <int KMAX, int ROWS, typename W>
__global__ void __launch_bounds__(256)
reorder_pages_kernel(const PagedPools p, const int* __restrict__ block_table, int bt_stride, const int* __restrict__ starts, const int* __restrict__ ends,
                     const int* __restrict__ parents, int beams, int pages, int nkv, int page_size, int* __restrict__ err) {
    __shared__ int from[MAX_BEAMS];
    __shared__ long long row_at[KMAX][ROWS], source_at[KMAX][ROWS];        // a row's place in its item, in units; -1: it has none
    pdl_wait();
    const int r = blockIdx.z, which = blockIdx.y % p.pools;
    const unsigned units = (unsigned)(which ? p.units[1] : p.units[0]);
    read_parents(from, parents, r, beams, err);
    const int begin = max(0, starts[r]), end = (int)min((long long)ends[r], (long long)bt_stride * page_size);
    if ((end < ends[r] || starts[r] < 0) && threadIdx.x == 0) atomicOr(err, CELLM_DEV_BAD_PAGE);
    const unsigned per_row = (unsigned)nkv * units, head = (unsigned)page_size * units;
    W* item = static_cast<W*>(which ? p.pool[1] : p.pool[0]) + (size_t)(blockIdx.y / p.pools) * pages * per_row * page_size;
    for (int at = begin + blockIdx.x * ROWS; at < end; at += gridDim.x * ROWS) {
        const unsigned rows = min(ROWS, end - at);
        __syncthreads();
        for (int i = threadIdx.x; i < beams * ROWS; i += 256) {
            const int k = i / ROWS, j = i % ROWS;
            if (j >= (int)rows) continue;
            const int page = block_table[((long long)r * beams + k) * bt_stride + (at + j) / page_size];
            if (page >= pages || page < -1) atomicOr(err, CELLM_DEV_BAD_PAGE);
            row_at[k][j] = page < 0 || page >= pages ? -1 : ((long long)page * nkv * page_size + (at + j) % page_size) * units;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < beams * ROWS; i += 256) {
            const int k = i / ROWS, j = i % ROWS;
            if (j < (int)rows) source_at[k][j] = from[k] >= 0 && row_at[k][j] >= 0 ? row_at[from[k]][j] : -1;
        }
        __syncthreads();
        // neighbouring threads take a head's rows one behind the other, which lie so on their page
        for (unsigned u = threadIdx.x; u < ROWS * per_row; u += 256) {
            const unsigned x = u % units, j = u / units % ROWS, h = u / units / ROWS;
            if (j >= rows) continue;
            reorder_units<KMAX, 1, W>(beams, item + (size_t)h * head + x, 0, 1, [&](int k) { return source_at[k][j]; }, [&](int k) { return row_at[k][j]; });
        }
    }
}

template <typename W>
int launch_states(void* state, const int* slot_ids, const int* parents, int requests, int beams, int items, int slots, long long bytes, int* err,
                  cudaStream_t stream) {
    const long long units = bytes / (long long)sizeof(W);
    auto grid = [&](int at_once) {
        long long blocks = std::min<long long>((units + 256 * at_once - 1) / (256 * at_once), 4096);
        if (at_once == 1 && blocks * items * requests > 4096) blocks = (blocks + 1) / 2;        // (two units a thread, one behind the other)
        return dim3((unsigned)blocks, (unsigned)items, (unsigned)requests);
    };
#define GO(K_) CELLM_RUN((reorder_states_kernel<K_, W>), grid(UNITS_AT_ONCE<K_, W>), 256, 0, stream, (W*)state, slot_ids, parents, beams, slots, units, err)
    if (beams <= 4) GO(4);
    else if (beams <= 8) GO(8);
    else if (beams <= 16) GO(16);
    else GO(32);
#undef GO
    return CELLM_OK;
}

template <typename W>
int launch_pages(PagedPools p, const int* block_table, int bt_stride, const int* starts, const int* ends, const int* parents, int requests, int beams,
                 int items, int pages, int nkv, int page_size, int sms, int* err, cudaStream_t stream) {
    for (int i = 0; i < p.pools; ++i) p.units[i] /= (int)sizeof(W);
    const long long most = (long long)bt_stride * page_size, rest = (long long)items * p.pools * requests;
    // Few beams have little to move between two look-ups: 32 rows at a time where that leaves every SM two blocks (2 beams, 330 MB: 68 us
    // for 84 with 8; 4 beams 76 for 82; 8 beams 86 for 81).
    const int rows = beams <= 4 && most * rest > 64ll * sms ? 32 : 8;
    const unsigned blocks = (unsigned)std::max<long long>(1, std::min<long long>((most + rows - 1) / rows, 128ll * sms / rest));
    const dim3 grid(blocks, (unsigned)(items * p.pools), (unsigned)requests);
#define GO(K_, R_) CELLM_RUN((reorder_pages_kernel<K_, R_, W>), grid, 256, 0, stream, p, block_table, bt_stride, starts, ends, parents, beams, pages, nkv, page_size, err)
    if (beams <= 4 && rows == 32) GO(4, 32);
    else if (beams <= 4) GO(4, 8);
    else if (beams <= 8) GO(8, 8);
    else if (beams <= 16) GO(16, 8);
    else GO(32, 8);
#undef GO
    return CELLM_OK;
}

template <typename T>
int launch_select(float* out_scores, int* out_parents, int* out_tokens, float* tops, void* sums, const void* logits, long long ld, int V, int requests,
                  int beams, int keep, const float* scores, const uint8_t* done, int pad, int parts, int sms, cudaStream_t stream) {
    const long long all = (long long)requests * beams * parts;
    const unsigned blocks = (unsigned)std::min<long long>((all + ROW_WARPS - 1) / ROW_WARPS, (long long)Ring<T>::BLOCKS * sms);
    const size_t smem = ROW_WARPS * sizeof(Ring<T>);
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = cellm_allow_smem(allowed, (const void*)beam_rows_kernel<T>, smem);
    if (e != cudaSuccess) return (int)e;
    CELLM_RUN(beam_rows_kernel<T>, blocks, ROW_WARPS * 32, smem, stream, tops, (RowPart*)sums, (const T*)logits, ld, V, parts, requests * beams, done);
    CELLM_RUN(beam_pick_kernel<T>, requests, PICK_THREADS, HOT_ROOM * sizeof(uint32_t), stream, out_scores, out_parents, out_tokens, tops, (const RowPart*)sums, (const T*)logits, ld, V,
              parts, scores, done, beams, keep, pad, ((1ull << 32) + parts - 1) / parts);
    return CELLM_OK;
}

}  // namespace

// Warp parts of a row of V logits: the workspace holds 32 floats (tops) and 32 bytes (sums of its halves) for each part of every row.
CELLM_API int cellm_beam_parts(int V) { return (V + WARP_VALUES - 1) / WARP_VALUES; }

// The `keep` best continuations of each request's `beams` rows of logits [requests * beams][V] (rows ld apart) under the beams'
// scores: out_* [requests][keep], -1 and -inf where there are fewer. done: null, or a byte a row: such a beam offers (itself, pad) at
// its score and its logits are not read.
CELLM_API int cellm_beam_select(float* out_scores, int* out_parents, int* out_tokens, float* tops, void* sums, const void* logits, long long ld, int V,
                                int requests, int beams, int keep, const float* scores, const uint8_t* done, int pad, int dtype, int sms, cudaStream_t stream) {
    if (requests <= 0) return CELLM_OK;
    if (dtype != CELLM_F32 && dtype != CELLM_BF16) return CELLM_ERR_DTYPE;
    if (V <= 0 || V > MAX_VOCAB || beams <= 0 || beams > MAX_BEAMS || keep <= 0 || keep > MAX_KEEP || ld < V || pad < 0 || pad >= V || sms <= 0) return CELLM_ERR_SIZE;
    if ((long long)beams * (V + WARP_VALUES) > 0x7fffffffLL || (long long)requests * beams * cellm_beam_parts(V) > 0x3fffffffLL) return CELLM_ERR_SIZE;
    if (!out_scores || !out_parents || !out_tokens || !tops || !sums || !logits || !scores) return CELLM_ERR_ARG;
    if ((((uintptr_t)sums) & 15) || (((uintptr_t)logits) & (dtype == CELLM_F32 ? 3 : 1))) return CELLM_ERR_ALIGN;
    const int parts = cellm_beam_parts(V);
    return dtype == CELLM_F32 ? launch_select<float>(out_scores, out_parents, out_tokens, tops, sums, logits, ld, V, requests, beams, keep, scores, done, pad, parts, sms, stream)
                              : launch_select<__nv_bfloat16>(out_scores, out_parents, out_tokens, tops, sums, logits, ld, V, requests, beams, keep, scores, done, pad, parts, sms, stream);
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
    if (at % 4 == 0) GO(uint32_t);           // (8-byte borders too: in units of 4 bytes, several a thread, 2 beams move at 5.8 TB/s)
    if (at % 2 == 0) GO(uint16_t);
#undef GO
    return CELLM_ERR_ALIGN;
}

// k_pool [items][pages][nkv][page_size][k_bytes] and (or null) v_pool likewise, in place; block_table [requests * beams][bt_stride].
CELLM_API int cellm_reorder_pages(void* k_pool, int k_bytes, void* v_pool, int v_bytes, const int* block_table, int bt_stride, const int* starts, const int* ends,
                                  const int* parents, int requests, int beams, int items, int pages, int nkv, int page_size, int sms, int* err, cudaStream_t stream) {
    if (requests <= 0 || items <= 0) return CELLM_OK;
    if (beams <= 0 || beams > MAX_BEAMS || pages <= 0 || nkv <= 0 || page_size <= 0 || bt_stride <= 0 || items > 32767 || requests > 65535 || sms <= 0 || k_bytes <= 0 ||
        (v_pool && v_bytes <= 0) || (long long)nkv * page_size * std::max(k_bytes, v_bytes) > 0x7fffffffLL)
        return CELLM_ERR_SIZE;
    if (!k_pool || !block_table || !starts || !ends || !parents || !err) return CELLM_ERR_ARG;
    const PagedPools p = {{k_pool, v_pool}, {k_bytes, v_bytes}, v_pool ? 2 : 1};
    const uintptr_t at = (uintptr_t)k_pool | (uintptr_t)k_bytes | (v_pool ? (uintptr_t)v_pool | (uintptr_t)v_bytes : 0);
#define GO(W_) return launch_pages<W_>(p, block_table, bt_stride, starts, ends, parents, requests, beams, items, pages, nkv, page_size, sms, err, stream)
    if (at % 16 == 0 && beams <= 16) GO(uint4);
    if (at % 8 == 0) GO(uint2);              // (32 beams in units of 16 bytes leave no registers for a second block: 117 us for 103)
    if (at % 4 == 0) GO(uint32_t);
    if (at % 2 == 0) GO(uint16_t);
#undef GO
    return CELLM_ERR_ALIGN;
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_beam_select_packed(const long long* a, cudaStream_t stream) {
    return cellm_beam_select((float*)a[0], (int*)a[1], (int*)a[2], (float*)a[3], (void*)a[4], (const void*)a[5], (long long)a[6], (int)a[7],
        (int)a[8], (int)a[9], (int)a[10], (const float*)a[11], (const uint8_t*)a[12], (int)a[13], (int)a[14], (int)a[15], stream);
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_reorder_states_packed(const long long* a, cudaStream_t stream) {
    return cellm_reorder_states((void*)a[0], (const int*)a[1], (const int*)a[2], (int)a[3], (int)a[4], (int)a[5], (int)a[6], (long long)a[7],
        (int*)a[8], stream);
}

// The same with its arguments in order as 64-bit words (see common.cuh).
CELLM_API int cellm_reorder_pages_packed(const long long* a, cudaStream_t stream) {
    return cellm_reorder_pages((void*)a[0], (int)a[1], (void*)a[2], (int)a[3], (const int*)a[4], (int)a[5], (const int*)a[6], (const int*)a[7], (const int*)a[8], (int)a[9],
        (int)a[10], (int)a[11], (int)a[12], (int)a[13], (int)a[14], (int)a[15], (int*)a[16], stream);
}
