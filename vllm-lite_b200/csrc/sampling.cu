// Sampling of one token per row of float32 logits, on the device.
//
// Order of the steps, as in crates/core/src/sampling.rs:497-636 of the reference:
//   (1) repeat penalty   l >= 0 ? l / p : l * p    once per distinct seen id
//   (2) presence penalty l -= p                    once per distinct seen id
//   (3) logit bias       l[id] += b
//   (4) temperature      l /= T            (T > 0 and T != 1)
//   (5) top-k            the k-th largest value is the threshold, l < thr is dropped,
//                        ties at the threshold are kept
//   (6) T <= 0: argmax (ties: lowest index, NaN counts as -inf); else softmax with the
//       maximum subtracted; top_p < 1 keeps the most probable tokens, in descending
//       order, up to and including the one with which the cumulative probability
//       exceeds top_p; min_p > 0 then drops what is less than min_p times as probable as
//       the most probable token; the draw is the inverse CDF at u over the kept tokens.
// Two choices are this engine's own.  The draw walks the kept tokens in index order
// (the reference walks nucleus tokens in sorted order): same distribution, other
// token for the same u.  Tokens whose probability equals the nucleus' last one are
// all kept.  Probabilities are accumulated as 40-bit fixed-point integers, floor(exp(s - max) 2^40), so sums do
// not depend on the order in which threads add, or on how many blocks share a row, and a draw is reproducible; min_p's bound is one of
// these integers too, floor(min_p 2^40).
//
// vl_apply_penalties works on ragged per-row lists.
// vl_sample: a cluster of 1 to 8 blocks holds a row in shared memory, so that it is read from memory once, whatever the options.
//
// The first look: half-unit bins of the distance from the maximum (each lane counts in a column of its own, so no two meet) say how many tokens are near enough
// to be kept at all: those with which top-k's count is reached, or top-p's mass with room for what lies behind.  Few of them (SMP_FEW) go to one
// block with their places in the row, which sorts them (up to SMP_RANKED: each is compared with each) and finishes the row alone; the other blocks are done.
//
// Else a threshold (top-k's by counts, top-p's by masses) is found in three steps.  All values are sorted into SMP_BINS bins of their distance from the maximum, a
// partition that keeps their order (subtraction and the cut are monotone); the blocks add up a share of the bins each and a scan finds the bin with which the sum
// is reached.  The few values of that bin are brought together in every block, and there the threshold's key is found 8 bits at a time, until what is left
// is kept whole.  (Should they be more than SMP_LIST, as in a row of one value, the 8 bits at a time go over the cluster's whole row.)  Behind top-k, top-p's sum runs over
// what top-k left.  Values 32 and more below the maximum have mass 0 and are in no bin: no threshold need be found among them.  Any vocabulary
// size; what of a slice shared memory does not hold (in rows of more than 342,880) is read again in each pass.
//
// Bound by latencies: reading another block's shared memory takes 0.5 us, a barrier of the cluster 0.4, and there are some ten steps behind one another.  One row
// of 151,936 logits with top-k 20, top-p 0.95 and min-p 0.02: 15.5 us in a graph, 64 rows of mixed options 51 us (0.76 TB/s); through thresholds alone, a
// conversion a mass and 64-bit atomics a bin, 56 and 168.
#include "common.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

#define SMP_THREADS 512
#define SMP_WARPS (SMP_THREADS / 32)
#define SMP_FIX 1099511627776.0f /* 2^40 */
#define SMP_BINS 2048
#define SMP_PER_UNIT 64.0f       /* bins per unit of s: 32 units in all, and exp(-27.8) 2^40 is below one */
#define SMP_CLUSTER 8
#define SMP_LIST 2048            /* values of one bin that a block brings together */
#define SMP_OWN 512              /* ... of them its own */
#define SMP_COARSE 32            /* bins of the first look at a row, half a unit each: what lies 15.5 and more below the maximum is in none */
#define SMP_RANKED 256           /* most of those tokens that are compared each with each */
#define SMP_FEW 3000             /* most tokens that one block finishes a row with */

typedef unsigned long long u64;

__device__ __forceinline__ unsigned order_key(float v) {
    unsigned k = __float_as_uint(v);
    return (k & 0x80000000u) ? ~k : (k | 0x80000000u);
}
__device__ __forceinline__ float clean(float v, float inv_t) {
    v = v * inv_t;
    return (v != v) ? -INFINITY : v + 0.f;                  // (-0 becomes 0: the two are a tie, and their keys differ)
}

__global__ void apply_penalties_kernel(float* __restrict__ logits, long long row_stride, int V,
                                       const int* __restrict__ seen_off, const int* __restrict__ seen_ids,
                                       const float* __restrict__ repeat_p, const float* __restrict__ presence_p,
                                       const int* __restrict__ bias_off, const int* __restrict__ bias_ids,
                                       const float* __restrict__ bias_vals) {
    const int r = blockIdx.x;
    float* l = logits + (size_t)r * row_stride;
    if (seen_off) {
        const float rp = repeat_p ? repeat_p[r] : 1.f;
        const float pp = presence_p ? presence_p[r] : 0.f;
        for (int i = seen_off[r] + threadIdx.x; i < seen_off[r + 1]; i += blockDim.x) {
            const int id = seen_ids[i];          // the host passes each id once per row
            if (id < 0 || id >= V) continue;
            float v = l[id];
            if (rp != 1.f) v = v >= 0.f ? v / rp : v * rp;
            v -= pp;
            l[id] = v;
        }
    }
    __syncthreads();
    if (bias_off) {
        for (int i = bias_off[r] + threadIdx.x; i < bias_off[r + 1]; i += blockDim.x) {
            const int id = bias_ids[i];
            if (id >= 0 && id < V) l[id] += bias_vals[i];
        }
    }
}

struct ArgBest { float v; int i; };
__device__ __forceinline__ ArgBest better(ArgBest a, ArgBest b) {
    if (b.v > a.v || (b.v == a.v && b.i < a.i)) return b;
    return a;
}

// Adds to a 64-bit sum in shared memory, low word at p: 32-bit atomics are the hardware's own, and the high word is seldom touched.
__device__ __forceinline__ void add_mass(u64* p, u64 q) {
    unsigned* w = reinterpret_cast<unsigned*>(p);
    const unsigned lo = (unsigned)q, old = atomicAdd(w, lo), hi = (unsigned)(q >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(w + 1, hi);
}

__device__ __forceinline__ float from_key(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

struct SampleShared {
    union {                                 // (the bins are at rest when values are brought together)
        struct { u64 mass[SMP_BINS]; unsigned count[SMP_BINS]; };
        unsigned list[SMP_LIST];
        unsigned coarse[SMP_COARSE * 32];   // a column a lane, so that a warp's additions meet nowhere
        uint2 near[SMP_FEW];                // this block's tokens that may be kept: key, place in the row
    };
    unsigned coarse_count[SMP_COARSE], row_count[SMP_COARSE];
    unsigned own[SMP_OWN], own_count;       // this block's values of a bin, by their keys
    u64 fine_mass[2][256];                  // two levels of the search in a bin in turn: one is read by the cluster while the other is filled
    unsigned fine_count[2][256];
    u64 warp_sum[SMP_WARPS], all_mass, part_mass, near_mass;       // part: of this block, of its share of the bins; near: of its tokens that may be kept
    ArgBest warp_best[SMP_WARPS], best;
    int found_bin, found_digit;
    u64 found_value, found_before;
    unsigned found_count, found_key;
};

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// inclusive sums over the block in the order of the threads; all threads call it
__device__ __forceinline__ u64 block_scan_u64(u64 v, u64* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += warp_sums[w];
    return v;
}

// Sums of one number of each block of a cluster (x: this lane's block's, 0 beyond the last): all of them, and those of the blocks before each lane's.
__device__ __forceinline__ void cluster_sums(u64 x, u64* total, u64* before) {
    const int lane = threadIdx.x & 31;
    u64 upto = x;
#pragma unroll
    for (int o = 1; o < SMP_CLUSTER; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    *total = __shfl_sync(0xffffffffu, upto, SMP_CLUSTER - 1);
    *before = upto - x;
}

__global__ void __launch_bounds__(SMP_THREADS)
sample_kernel(const float* __restrict__ logits, long long row_stride, int V, int slice, int held, int room,
              const float* __restrict__ temperature, const int* __restrict__ top_k,
              const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniform,
              int* __restrict__ out_token, float* __restrict__ out_logprob) {
    extern __shared__ __align__(16) float s_val[];          // the block's slice of the row, scaled: `held` values
    __shared__ SampleShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int r = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* l = logits + (size_t)r * row_stride + (size_t)rank * slice;
    const int n = max(0, min(slice, V - rank * slice)), first = rank * slice;
    const float temp = temperature ? temperature[r] : 0.f;
    const bool greedy = !(temp > 0.f);
    const float inv_t = greedy ? 1.f : 1.f / temp;
    const int k = top_k ? top_k[r] : 0;
    const float tp = top_p ? top_p[r] : 1.f, mp = min_p ? min_p[r] : 0.f;

    // ---- the slice into shared memory, and the row's first largest value ----
    ArgBest best{-INFINITY, 0x7fffffff};
    auto take = [&](int i, float x) {
        const float v = clean(x, 1.f);
        best = better(best, ArgBest{v, first + i});
        if (i < held) s_val[i] = clean(x, inv_t);
    };
    const int n4 = ((uintptr_t)l & 15) == 0 ? (n & ~3) : 0;
    constexpr int LOADS = 8;                                            // 16 bytes each, on their way together
    for (int i0 = 4 * tid; i0 < n4; i0 += LOADS * 4 * SMP_THREADS) {
        float4 q[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
            if (i0 + u * 4 * SMP_THREADS < n4) q[u] = *reinterpret_cast<const float4*>(l + i0 + u * 4 * SMP_THREADS);
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int i = i0 + u * 4 * SMP_THREADS;
            if (i < n4) { take(i, q[u].x); take(i + 1, q[u].y); take(i + 2, q[u].z); take(i + 3, q[u].w); }
        }
    }
    for (int i = n4 + tid; i < n; i += SMP_THREADS) take(i, l[i]);
    for (int i = n + tid; i < held; i += SMP_THREADS) s_val[i] = -INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        ArgBest other{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)};
        best = better(best, other);
    }
    if (lane == 0) sh.warp_best[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < SMP_WARPS; ++w) best = better(best, sh.warp_best[w]);
        sh.best = best;
    }
    cluster.sync();
    const SampleShared* const peer = cluster.map_shared_rank(&sh, lane < C ? lane : rank);        // a lane a block
    best = peer->best;
#pragma unroll
    for (int o = SMP_CLUSTER / 2; o > 0; o >>= 1) {
        ArgBest other{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.i, o)};
        best = better(best, other);
    }
    best = ArgBest{__shfl_sync(0xffffffffu, best.v, 0), __shfl_sync(0xffffffffu, best.i, 0)};
    const int arg = best.i == 0x7fffffff ? 0 : best.i;
    const float row_max = best.v * inv_t;      // maximum of the scaled row (top-k keeps it)
    const bool degenerate = !(row_max > -INFINITY && row_max < INFINITY);
    auto value = [&](int i) { return i < held ? s_val[i] : clean(l[i], inv_t); };
    // floor(exp(s - max) 2^40), the number's own digits shifted (a conversion takes as long as the exponential)
    auto mass_of = [&](float s) -> u64 {
        const unsigned e = __float_as_uint(expf(s - row_max)), shift = e >> 23;                  // of 2^(shift - 127), at most 2^0
        const u64 digits = (e & 0x7fffffu) | 0x800000u;
        return shift >= 110 ? digits << (shift - 110) : (shift >= 87 ? digits >> (110 - shift) : 0);
    };
    // the bin of a value, by an addition that leaves the nearest whole number in a float's low bits; SMP_BINS for one without mass
    auto bin_of = [&](float s) {
        const float d = row_max - s;
        return d < (SMP_BINS - 1) / SMP_PER_UNIT ? (int)(__float_as_uint(fmaf(d, SMP_PER_UNIT, 8388608.f)) & (SMP_BINS - 1)) : SMP_BINS;
    };
    auto finish = [&](int token, float logprob) {
        out_token[r] = token;
        if (out_logprob) out_logprob[r] = logprob;
    };
    if ((greedy && !out_logprob) || degenerate) {
        if (rank == 0 && tid == 0) finish(arg, 0.f);
        cluster.sync();                        // nobody leaves while others read its shared memory
        return;
    }

    // every value of the slice and its place in it, in no order; shared memory holds a multiple of four, filled up with values without mass
    auto each = [&](auto f) {
        for (int i = 4 * tid; i < held; i += 4 * SMP_THREADS) {
            const float4 v = *reinterpret_cast<const float4*>(s_val + i);
            f(v.x, i); f(v.y, i + 1); f(v.z, i + 2); f(v.w, i + 3);
        }
        for (int i = held + tid; i < n; i += SMP_THREADS) f(clean(l[i], inv_t), i);
    };
    int level = 0;
    // Of `all` weighted keys: the key with which the sum of weights, from the largest key on, reaches `left`; this block alone.
    auto search = [&](unsigned all, auto key_of, auto weight_of, u64 left) -> unsigned {
        unsigned prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8, ++level) {
            u64* fm = sh.fine_mass[level & 1];
            unsigned* fc = sh.fine_count[level & 1];
            if (tid < 256) { fm[tid] = 0; fc[tid] = 0; }
            if (tid == 0) sh.found_key = 0xffffffffu;
            __syncthreads();
            const unsigned himask = shift == 24 ? 0u : (0xffffffffu << (shift + 8));
            for (unsigned i = tid; i < all; i += SMP_THREADS) {
                const unsigned key = key_of(i);
                if ((key & himask) != prefix) continue;
                const u64 q = weight_of(i);
                if (!q) continue;
                const unsigned d = 255u - ((key >> shift) & 255u);
                atomicAdd(&fc[d], 1u);
                add_mass(&fm[d], q);
            }
            __syncthreads();
            const u64 x = tid < 256 ? fm[tid] : 0, upto = block_scan_u64(x, sh.warp_sum);
            if (tid < 256 && upto >= left && upto - x < left) { sh.found_digit = 255 - tid; sh.found_before = upto - x; sh.found_count = fc[tid]; }
            __syncthreads();
            prefix |= (unsigned)sh.found_digit << shift;
            left -= sh.found_before;
            const bool one = sh.found_count == 1;
            __syncthreads();
            if (one && shift > 0) {            // the only one left
                for (unsigned i = tid; i < all; i += SMP_THREADS) {
                    const unsigned key = key_of(i);
                    if (key >> shift == prefix >> shift && weight_of(i)) sh.found_key = key;
                }
                __syncthreads();
                prefix = sh.found_key;
                ++level;
                break;
            }
        }
        return prefix;
    };
    float cut = -INFINITY;                     // a token is kept by top-k and top-p if its value is at least this
    const bool by_k = !greedy && k > 0 && k < V, by_p = !greedy && tp < 1.f, by_m = !greedy && mp > 0.f;
    const u64 floor_mass = by_m ? (u64)((double)fminf(mp, 1.f) * (double)SMP_FIX) : 0;
    const float u_draw = uniform ? uniform[r] : 0.f;

    // ---- a row of which few tokens can be kept: those are brought together, and one block finishes ----
    if (by_k || by_p || by_m) {
        const bool weigh = by_p && !by_k;      // top-p's sum runs over the whole row
        for (int i = tid; i < SMP_COARSE * 32; i += SMP_THREADS) sh.coarse[i] = 0;
        if (tid == 0) { sh.part_mass = 0; sh.near_mass = 0; sh.own_count = 0; }
        __syncthreads();
        auto coarse_of = [&](float s) {        // a bin of half a unit of the distance; SMP_COARSE for one that lies far off
            const float d = row_max - s;
            return d < (SMP_COARSE - 1) / 2.f ? (int)(__float_as_uint(fmaf(d, 2.f, 8388608.f)) & (SMP_COARSE - 1)) : SMP_COARSE;
        };
        u64 mine = 0;
        each([&](float s, int) {
            const int b = coarse_of(s);
            if (b < SMP_COARSE) atomicAdd(&sh.coarse[b * 32 + lane], 1u);
            if (weigh) mine += mass_of(s);
        });
        if (weigh) {
            mine = warp_sum_u64(mine);
            if (lane == 0) atomicAdd(&sh.part_mass, mine);
        }
        __syncthreads();
        for (int b = warp; b < SMP_COARSE; b += SMP_WARPS) {
            const unsigned c = __reduce_add_sync(0xffffffffu, sh.coarse[b * 32 + lane]);
            if (lane == 0) sh.coarse_count[b] = c;
        }
        cluster.sync();
        static_assert(SMP_COARSE * SMP_CLUSTER <= SMP_THREADS, "a thread a bin and block");
        if (tid < SMP_COARSE * SMP_CLUSTER) {
            const int b = tid / SMP_CLUSTER, other = tid % SMP_CLUSTER;
            unsigned c = other < C ? cluster.map_shared_rank(&sh, other)->coarse_count[b] : 0;
#pragma unroll
            for (int o = 1; o < SMP_CLUSTER; o <<= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
            if (other == 0) sh.row_count[b] = c;
        }
        u64 row_mass, unused;
        cluster_sums(weigh && lane < C ? peer->part_mass : 0, &row_mass, &unused);
        __syncthreads();
        // the last bin that can hold a kept token: exactly for top-k, by its bins' middles and two more for top-p (checked below), by the bound for min-p
        unsigned upto = sh.row_count[lane];
        float guess = upto * __expf(-0.5f * lane);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
            const float y = __shfl_up_sync(0xffffffffu, guess, o);
            if (lane >= o) { upto += x; guess += y; }
        }
        unsigned reach = 0;
        if (by_k) reach = __ballot_sync(0xffffffffu, upto >= (unsigned)k);
        else if (by_p) reach = __ballot_sync(0xffffffffu, guess >= tp * __shfl_sync(0xffffffffu, guess, 31)) << 2;
        else reach = 1u << (int)fminf(-2.f * logf(mp) + 2.f, 31.f);
        const int last = __ffs(reach) - 1;     // (-1: none)
        const unsigned count = last >= 0 && last < SMP_COARSE - 1 ? __shfl_sync(0xffffffffu, upto, max(last, 0)) : SMP_FEW + 1;
        if (count <= SMP_FEW && count <= (unsigned)room) {
            u64 near = 0;
            each([&](float s, int i) {
                if (coarse_of(s) <= last) {
                    sh.near[atomicAdd(&sh.own_count, 1u)] = make_uint2(order_key(s), (unsigned)(first + i));
                    if (weigh) near += mass_of(s);
                }
            });
            if (weigh) {
                near = warp_sum_u64(near);
                if (lane == 0) atomicAdd(&sh.near_mass, near);
            }
            cluster.sync();
            u64 near_mass, all, place;
            cluster_sums(weigh && lane < C ? peer->near_mass : 0, &near_mass, &unused);
            const u64 target = (u64)((double)tp * (double)row_mass);
            if (!weigh || near_mass > target) {
                const unsigned found = lane < C ? peer->own_count : 0;
                cluster_sums(found, &all, &place);
                unsigned* const keys = reinterpret_cast<unsigned*>(s_val);         // the slice is at rest: its room holds keys, places and masses
                unsigned* const places = keys + room;
                u64* const weights = reinterpret_cast<u64*>(places + room);
                if (rank == 0) {
                    unsigned begin[SMP_CLUSTER];
#pragma unroll
                    for (int b = 0; b < SMP_CLUSTER; ++b) begin[b] = (unsigned)__shfl_sync(0xffffffffu, place, b);
                    for (unsigned i = tid; i < (unsigned)all; i += SMP_THREADS) {
                        int b = 0;
                        unsigned at = 0;
#pragma unroll
                        for (int o = 1; o < SMP_CLUSTER; ++o)
                            if (i >= begin[o] && o < C) { b = o; at = begin[o]; }
                        const uint2 x = cluster.map_shared_rank(&sh, b)->near[i - at];
                        keys[i] = x.x;
                        places[i] = x.y;
                        weights[i] = mass_of(from_key(x.x));
                    }
                }
                cluster.sync();                // nobody leaves while others read its shared memory
                if (rank != 0) return;
                const unsigned L = (unsigned)all;
                auto sum_of = [&](auto weight_of) -> u64 {
                    u64 t = 0;
                    for (unsigned i = tid; i < L; i += SMP_THREADS) t += weight_of(i);
                    t = warp_sum_u64(t);
                    __syncthreads();
                    if (lane == 0) sh.warp_sum[warp] = t;
                    __syncthreads();
                    return warp_sum_u64(lane < SMP_WARPS ? sh.warp_sum[lane] : 0);
                };
                if (L <= SMP_RANKED) {         // few enough to be compared each with each: a thread a token
                    const unsigned key = tid < L ? keys[tid] : 0, mine_at = tid < L ? places[tid] : 0;
                    u64 w = tid < L ? weights[tid] : 0, above = 0;
                    unsigned greater = 0;
                    if (tid < (int)L)
                        for (unsigned i = 0; i < L; ++i)
                            if (keys[i] > key) { ++greater; above += weights[i]; }
                    if (by_k && greater >= (unsigned)k) w = 0;                     // (ties at the threshold stay)
                    auto sum = [&](u64 x) -> u64 {
                        x = warp_sum_u64(x);
                        __syncthreads();
                        if (lane == 0) sh.warp_sum[warp] = x;
                        __syncthreads();
                        return warp_sum_u64(lane < SMP_WARPS ? sh.warp_sum[lane] : 0);
                    };
                    if (by_p && above > (by_k ? (u64)((double)tp * (double)sum(w)) : target)) w = 0;
                    if (w < floor_mass) w = 0;
                    const u64 kept = sum(w);
                    if (tid < L) weights[tid] = w;
                    __syncthreads();
                    u64 goal = (u64)((double)u_draw * (double)kept), before = 0;
                    if (goal >= kept) goal = kept - 1;
                    if (tid < (int)L)
                        for (unsigned i = 0; i < L; ++i)
                            if (places[i] < mine_at) before += weights[i];
                    if (w && before <= goal && goal - before < w) finish((int)mine_at, logf((float)((double)w / (double)kept)));
                    return;
                }
                auto key_of = [&](unsigned i) { return keys[i]; };
                unsigned least = 0;            // the threshold's key
                if (by_k) least = search(L, key_of, [&](unsigned) -> u64 { return 1; }, (u64)k);
                if (by_p) {
                    auto weight_of = [&](unsigned i) { return keys[i] >= least ? weights[i] : 0; };
                    const u64 goal = (by_k ? (u64)((double)tp * (double)sum_of(weight_of)) : target) + 1;
                    least = max(least, search(L, key_of, weight_of, goal));
                }
                auto kept_of = [&](unsigned i) { return keys[i] >= least && weights[i] >= floor_mass ? weights[i] : 0; };
                const u64 kept = sum_of(kept_of);
                u64 goal = (u64)((double)u_draw * (double)kept);
                if (goal >= kept) goal = kept - 1;
                const unsigned token = ~search(L, [&](unsigned i) { return ~places[i]; }, kept_of, goal + 1);
                for (unsigned i = tid; i < L; i += SMP_THREADS)
                    if (places[i] == token) finish((int)token, logf((float)((double)weights[i] / (double)kept)));
                return;
            }
        }
        cluster.sync();                        // what was read of others has been read
    }

    // The value with which the sum, from the largest values on, of counts (masses) of all values from `cut` on reaches goal(their sum); -inf if all together do not.
    auto threshold = [&](bool masses, auto goal_of) -> float {
        for (int i = tid; i < SMP_BINS; i += SMP_THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
        if (tid == 0) { sh.part_mass = 0; sh.own_count = 0; }
        __syncthreads();
        each([&](float s, int) {
            const int b = bin_of(s);
            if (b >= SMP_BINS || s < cut) return;
            if (!masses) atomicAdd(&sh.count[b], 1u);
            else {
                const u64 q = mass_of(s);
                if (q) add_mass(&sh.mass[b], q);
            }
        });
        cluster.sync();
        // this block's share of the bins, summed over the cluster in its own array (nobody else reads that share there)
        const int share = SMP_BINS / C, lo = rank * share;
        u64 m = 0;
        for (int i = lo + tid; i < lo + share; i += SMP_THREADS) {
            u64 bm = 0;
#pragma unroll
            for (int b = 0; b < SMP_CLUSTER; ++b) {          // (all on their way together)
                const SampleShared* other = cluster.map_shared_rank(&sh, b < C ? b : rank);
                const u64 x = masses ? other->mass[i] : (u64)other->count[i];
                bm += b < C ? x : 0;
            }
            sh.mass[i] = bm;
            m += bm;
        }
        m = warp_sum_u64(m);
        if (lane == 0 && m) atomicAdd(&sh.part_mass, m);
        cluster.sync();
        u64 total, before;
        const u64 part = lane < C ? peer->part_mass : 0;
        cluster_sums(part, &total, &before);
        const u64 goal = goal_of(total);
        if (goal > total) return -INFINITY;    // (everything that has a mass is kept)
        const int owner = __ffs(__ballot_sync(0xffffffffu, lane < C && before + part >= goal)) - 1;
        before = __shfl_sync(0xffffffffu, before, owner);
        if (owner == rank) {
            const int per = (share + SMP_THREADS - 1) / SMP_THREADS, i0 = lo + tid * per, i1 = min(lo + share, i0 + per);
            u64 mine = 0;
            for (int i = i0; i < i1; ++i) mine += sh.mass[i];
            u64 cum = before + block_scan_u64(mine, sh.warp_sum) - mine;
            for (int i = i0; i < i1; ++i) {
                const u64 x = sh.mass[i];
                if (cum < goal && cum + x >= goal) { sh.found_bin = i; sh.found_value = cum; }
                cum += x;
            }
        }
        cluster.sync();
        const SampleShared* o = cluster.map_shared_rank(&sh, owner);
        const int bin = o->found_bin;
        u64 left = goal - o->found_value;

        // the bin's values, each block's own first
        each([&](float s, int) {
            if (bin_of(s) == bin && s >= cut) {
                const unsigned at = atomicAdd(&sh.own_count, 1u);
                if (at < SMP_OWN) sh.own[at] = order_key(s);
            }
        });
        cluster.sync();
        u64 all, place;
        const unsigned found = lane < C ? peer->own_count : 0;
        cluster_sums(found, &all, &place);
        const bool few = all <= SMP_LIST && __all_sync(0xffffffffu, found <= SMP_OWN);
        if (few) {
#pragma unroll
            for (int b = 0; b < SMP_CLUSTER; ++b) {
                const unsigned c = __shfl_sync(0xffffffffu, found, b), at = (unsigned)__shfl_sync(0xffffffffu, place, b);
                for (unsigned i = tid; i < c; i += SMP_THREADS) sh.list[at + i] = cluster.map_shared_rank(&sh, b < C ? b : rank)->own[i];
            }
        }
        if (few) {
            __syncthreads();
            return from_key(search((unsigned)all, [&](unsigned i) { return sh.list[i]; }, [&](unsigned i) -> u64 { return masses ? mass_of(from_key(sh.list[i])) : 1; },
                                   left));
        }
        unsigned prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8, ++level) {
            u64* fm = sh.fine_mass[level & 1];
            if (tid < 256) fm[tid] = 0;
            __syncthreads();
            const unsigned himask = shift == 24 ? 0u : (0xffffffffu << (shift + 8));
            each([&](float s, int) {
                const unsigned key = order_key(s);
                if (bin_of(s) == bin && s >= cut && (key & himask) == prefix) add_mass(&fm[255u - ((key >> shift) & 255u)], masses ? mass_of(s) : 1);
            });
            cluster.sync();
            u64 x = 0;                         // every block finds the same digit for itself
            if (tid < 256)
                for (int b = 0; b < C; ++b) x += cluster.map_shared_rank(&sh, b)->fine_mass[level & 1][tid];
            const u64 upto = block_scan_u64(x, sh.warp_sum);
            if (tid < 256 && upto >= left && upto - x < left) { sh.found_digit = 255 - tid; sh.found_before = upto - x; }
            __syncthreads();
            prefix |= (unsigned)sh.found_digit << shift;
            left -= sh.found_before;
            __syncthreads();
        }
        return from_key(prefix);
    };
    if (by_k) cut = threshold(false, [&](u64) { return (u64)k; });
    if (by_p) {
        if (by_k) cluster.sync();              // what the search before left has been read
        // (the target is less than the sum, so that there is such a value)
        cut = fmaxf(cut, threshold(true, [&](u64 total) { return (u64)((double)tp * (double)total) + 1; }));
    }
    // ---- the draw: masses of the kept tokens in index order; a warp owns a contiguous part of the slice ----
    auto kept_mass = [&](float s) -> u64 {
        if (!(s >= cut)) return 0;
        const u64 q = mass_of(s);
        return q >= floor_mass ? q : 0;
    };
    constexpr int GROUP = 128;                 // neighbouring values that a warp takes at once, four a lane
    const int span = (n + SMP_WARPS * GROUP - 1) / (SMP_WARPS * GROUP) * GROUP, from = min(n, warp * span), to = min(n, from + span);
    auto four = [&](int i, u64 (&q)[4]) {      // the masses of values i .. i + 3, and their sum
        float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (i + 4 <= held) v = *reinterpret_cast<const float4*>(s_val + i);
        else
            for (int j = 0; j < 4; ++j)
                if (i + j < n) (&v.x)[j] = value(i + j);
        q[0] = kept_mass(v.x); q[1] = kept_mass(v.y); q[2] = kept_mass(v.z); q[3] = kept_mass(v.w);
        return q[0] + q[1] + q[2] + q[3];
    };
    u64 sum = 0, q[4];
    for (int i = from + 4 * lane; i < to; i += GROUP) sum += four(i, q);
    sum = warp_sum_u64(sum);
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        const u64 t = warp_sum_u64(lane < SMP_WARPS ? sh.warp_sum[lane] : 0);
        if (lane == 0) sh.all_mass = t;
    }
    cluster.sync();
    u64 total, before;
    cluster_sums(lane < C ? peer->all_mass : 0, &total, &before);
    before = __shfl_sync(0xffffffffu, before, rank);
    if (greedy) {                              // log-softmax of the row at the argmax: exp(0) / sum
        if (rank == 0 && tid == 0) finish(arg, -logf((float)((double)total / (double)SMP_FIX)));
        cluster.sync();
        return;
    }
    u64 target = (u64)((double)u_draw * (double)total);
    if (target >= total) target = total - 1;
    before += warp_sum_u64(lane < warp ? sh.warp_sum[lane] : 0);
    if (target >= before && target - before < sum) {                    // (warp-uniform) the drawn token is this warp's
        u64 run = before;
        for (int base = from; base < to; base += GROUP) {
            const u64 mine = base + 4 * lane < to ? four(base + 4 * lane, q) : 0;
            u64 inc = mine;                    // inclusive scan over the warp
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            const unsigned hits = __ballot_sync(0xffffffffu, mine > 0 && run + inc > target);
            if (hits) {
                if (lane == __ffs(hits) - 1) {
                    u64 upto = run + inc - mine;
                    for (int j = 0; j < 4; ++j) {
                        upto += q[j];
                        if (q[j] > 0 && upto > target) {
                            finish(first + base + 4 * lane + j, logf((float)((double)q[j] / (double)total)));
                            break;
                        }
                    }
                }
                break;
            }
            run += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    cluster.sync();
}

extern "C" int vl_apply_penalties(float* logits, long long row_stride, int R, int V,
                                  const int* seen_off, const int* seen_ids,
                                  const float* repeat_p, const float* presence_p,
                                  const int* bias_off, const int* bias_ids, const float* bias_vals,
                                  void* stream) {
    if (R <= 0) return VL_OK;
    apply_penalties_kernel<<<R, 256, 0, (cudaStream_t)stream>>>(
        logits, row_stride, V, seen_off, seen_ids, repeat_p, presence_p, bias_off, bias_ids, bias_vals);
    return vl_launch_status();
}

// Values of a slice that a block's shared memory holds beside its tables, a multiple of the four that it is read by.
constexpr int SMP_HELD_MAX = (200 * 1024 - (int)sizeof(SampleShared)) / 16 * 4;
static_assert(SMP_HELD_MAX % 4 == 0, "shared memory is read in pieces of four values");

extern "C" int vl_sample(const float* logits, long long row_stride, int R, int V,
                         const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                         const float* uniform, int* out_token, float* out_logprob, void* stream) {
    if (R <= 0) return VL_OK;
    if (V <= 0) return VL_ERR_ARGUMENT;
    if ((long long)R * SMP_CLUSTER >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
    int C = SMP_CLUSTER;
    while (C > 1 && V <= 2048 * C / 2) C /= 2;
    const int slice = ((V + C - 1) / C + 3) & ~3, held = slice < SMP_HELD_MAX ? slice : SMP_HELD_MAX;
    cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMP_HELD_MAX * 4);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(R * C));
    cfg.blockDim = dim3(SMP_THREADS);
    // room for the tokens that a block finishes a row with: 16 bytes each, a multiple of 2 of them
    const int few = (V < SMP_FEW ? V : SMP_FEW) + 1 & ~1, bytes = held * 4 > few * 16 ? held * 4 : few * 16;
    cfg.dynamicSmemBytes = (size_t)bytes;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, sample_kernel, logits, row_stride, V, slice, held, few, temperature, top_k, top_p, min_p, uniform, out_token,
                                   out_logprob);
}
