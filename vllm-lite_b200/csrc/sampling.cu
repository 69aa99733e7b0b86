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
// vl_sample: a cluster of 1 to 8 blocks holds a row in shared memory, so that it is read from memory once, whatever the options.  A row that asks for top-k
// or top-p is sorted into SMP_BINS bins of its distance from the maximum (a partition that keeps the order of values: subtraction and the cut are
// monotone), with their counts and masses; each block adds up a share of the bins over the cluster and the bin in which a threshold lies is found by
// a scan of them.  Inside that bin the threshold's key is found 8 bits at a time, until what is left is kept whole; few values lie there, so these passes
// count little.  Values 32 and more below the maximum have mass 0 and are in no bin: no threshold need be found among them.  Any vocabulary size; what of
// a slice shared memory does not hold (rows of more than some 390,000) is read again in each pass.
#include "common.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

#define SMP_THREADS 512
#define SMP_WARPS (SMP_THREADS / 32)
#define SMP_FIX 1099511627776.0f /* 2^40 */
#define SMP_BINS 2048
#define SMP_PER_UNIT 64.0f       /* bins per unit of s: 32 units in all, and exp(-27.8) 2^40 is below one */
#define SMP_CLUSTER 8

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

struct SampleShared {
    u64 mass[SMP_BINS];
    unsigned count[SMP_BINS];
    u64 fine_mass[2][256];                  // two levels of the search in a bin in turn: one is read by the cluster while the other is filled
    unsigned fine_count[2][256];
    u64 warp_sum[SMP_WARPS], all_mass, part_mass;      // part: this block's share of the bins
    unsigned part_count;
    ArgBest warp_best[SMP_WARPS], best;
    int found_bin;
    u64 found_above_mass, found_mass, found_value;
    unsigned found_above, found_count;
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

__global__ void __launch_bounds__(SMP_THREADS)
sample_kernel(const float* __restrict__ logits, long long row_stride, int V, int slice, int held,
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
    for (int i0 = 4 * tid; i0 < n4; i0 += 16 * SMP_THREADS) {           // 16 bytes a load, four on their way
        float4 q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * 4 * SMP_THREADS < n4) q[u] = *reinterpret_cast<const float4*>(l + i0 + u * 4 * SMP_THREADS);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * 4 * SMP_THREADS;
            if (i < n4) { take(i, q[u].x); take(i + 1, q[u].y); take(i + 2, q[u].z); take(i + 3, q[u].w); }
        }
    }
    for (int i = n4 + tid; i < n; i += SMP_THREADS) take(i, l[i]);
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
    best = sh.best;
    for (int c = 0; c < C; ++c) best = better(best, cluster.map_shared_rank(&sh, c)->best);
    const int arg = best.i == 0x7fffffff ? 0 : best.i;
    const float row_max = best.v * inv_t;      // maximum of the scaled row (top-k keeps it)
    const bool degenerate = !(row_max > -INFINITY && row_max < INFINITY);
    auto value = [&](int i) { return i < held ? s_val[i] : clean(l[i], inv_t); };
    auto mass_of = [&](float s) { return (u64)(expf(s - row_max) * SMP_FIX); };
    // the bin of a value; SMP_BINS for one without mass
    auto bin_of = [&](float s) {
        const float d = (row_max - s) * SMP_PER_UNIT;
        return d < (float)SMP_BINS ? (int)d : SMP_BINS;
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

    // A token is kept if its bin lies before `cut_bin`, or in it with at least the key `cut_key`.
    int cut_bin = SMP_BINS;
    unsigned cut_key = 0;
    const bool by_k = !greedy && k > 0 && k < V, by_p = !greedy && tp < 1.f;
    if (by_k || by_p) {
        for (int i = tid; i < SMP_BINS; i += SMP_THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
        __syncthreads();
        for (int i = tid; i < n; i += SMP_THREADS) {
            const float s = value(i);
            const int b = bin_of(s);
            if (b < SMP_BINS) {
                atomicAdd(&sh.count[b], 1u);
                const u64 q = mass_of(s);
                if (q) atomicAdd(&sh.mass[b], q);
            }
        }
        cluster.sync();
        // this block's share of the bins, summed over the cluster in its own arrays (nobody else reads that share there)
        const int share = SMP_BINS / C, lo = rank * share;
        u64 m = 0;
        unsigned c = 0;
        for (int i = lo + tid; i < lo + share; i += SMP_THREADS) {
            unsigned bc = 0;
            u64 bm = 0;
            for (int b = 0; b < C; ++b) {
                const SampleShared* other = cluster.map_shared_rank(&sh, b);
                bc += other->count[i];
                bm += other->mass[i];
            }
            sh.count[i] = bc;
            sh.mass[i] = bm;
            c += bc;
            m += bm;
        }
        c = __reduce_add_sync(0xffffffffu, c);
        m = warp_sum_u64(m);
        if (tid == 0) { sh.part_count = 0; sh.part_mass = 0; }
        __syncthreads();
        if (lane == 0) { atomicAdd(&sh.part_count, c); atomicAdd(&sh.part_mass, m); }
        cluster.sync();

        // The bin with which the sum, from the largest values on, of counts (masses) reaches `goal`; false if all bins together do not.
        struct Found { int bin; unsigned above, count; u64 above_mass, mass; } f;
        auto cross = [&](bool masses, u64 goal) -> bool {
            int owner = -1;
            unsigned before_c = 0;
            u64 before_m = 0;
            for (int b = 0; b < C && owner < 0; ++b) {
                const SampleShared* other = cluster.map_shared_rank(&sh, b);
                const unsigned pc = other->part_count;
                const u64 pm = other->part_mass;
                if ((masses ? before_m + pm : (u64)(before_c + pc)) >= goal) owner = b;
                else { before_c += pc; before_m += pm; }
            }
            if (owner < 0) return false;
            if (owner == rank) {
                const int each = (share + SMP_THREADS - 1) / SMP_THREADS, i0 = lo + tid * each, i1 = min(lo + share, i0 + each);
                u64 mine_c = 0, mine_m = 0;
                for (int i = i0; i < i1; ++i) { mine_c += sh.count[i]; mine_m += sh.mass[i]; }
                u64 cum_c = before_c + block_scan_u64(mine_c, sh.warp_sum) - mine_c, cum_m = before_m + block_scan_u64(mine_m, sh.warp_sum) - mine_m;
                for (int i = i0; i < i1; ++i) {
                    const u64 x = masses ? sh.mass[i] : sh.count[i], cum = masses ? cum_m : cum_c;
                    if (cum < goal && cum + x >= goal) {
                        sh.found_bin = i;
                        sh.found_above = (unsigned)cum_c; sh.found_above_mass = cum_m;
                        sh.found_count = sh.count[i]; sh.found_mass = sh.mass[i];
                    }
                    cum_c += sh.count[i];
                    cum_m += sh.mass[i];
                }
            }
            cluster.sync();
            const SampleShared* o = cluster.map_shared_rank(&sh, owner);
            f.bin = o->found_bin; f.above = o->found_above; f.count = o->found_count; f.above_mass = o->found_above_mass; f.mass = o->found_mass;
            return true;
        };
        // Within bin f.bin, among keys of at least `least`: the key with which the sum of counts (masses) reaches `goal`, all of that key's values kept.
        // f.mass becomes the mass of the bin's kept values.
        int level = 0;
        auto refine = [&](bool masses, u64 goal, unsigned least) -> unsigned {
            unsigned prefix = 0;
            u64 kept = 0;                      // mass of the bin's values above the prefix
            for (int shift = 24; shift >= 0; shift -= 8, ++level) {
                u64* fm = sh.fine_mass[level & 1];
                unsigned* fc = sh.fine_count[level & 1];
                if (tid < 256) { fm[tid] = 0; fc[tid] = 0; }
                __syncthreads();
                const unsigned himask = shift == 24 ? 0u : (0xffffffffu << (shift + 8));
                for (int i = tid; i < n; i += SMP_THREADS) {
                    const float s = value(i);
                    const unsigned key = order_key(s);
                    if (bin_of(s) == f.bin && key >= least && (key & himask) == prefix) {
                        atomicAdd(&fc[255u - ((key >> shift) & 255u)], 1u);
                        atomicAdd(&fm[255u - ((key >> shift) & 255u)], mass_of(s));
                    }
                }
                cluster.sync();
                u64 x = 0, xm = 0;             // every block finds the same digit for itself
                unsigned xc = 0;
                if (tid < 256)
                    for (int b = 0; b < C; ++b) {
                        const SampleShared* other = cluster.map_shared_rank(&sh, b);
                        xc += other->fine_count[level & 1][tid];
                        xm += other->fine_mass[level & 1][tid];
                    }
                x = masses ? xm : xc;
                const u64 upto = block_scan_u64(x, sh.warp_sum), upto_m = block_scan_u64(xm, sh.warp_sum);
                __syncthreads();
                if (tid < 256 && upto >= goal && upto - x < goal) {
                    sh.found_bin = 255 - tid; sh.found_value = upto - x; sh.found_count = xc; sh.found_above_mass = upto_m - xm; sh.found_mass = xm;
                }
                __syncthreads();
                prefix |= (unsigned)sh.found_bin << shift;
                goal -= sh.found_value;
                kept += sh.found_above_mass;
                f.mass = kept + sh.found_mass;
                const bool whole = masses ? sh.found_count == 1 : goal == sh.found_count;
                __syncthreads();
                if (whole) { ++level; break; }
            }
            return max(prefix, least);
        };

        u64 total = 0;                         // mass after top-k
        for (int b = 0; b < C; ++b) total += cluster.map_shared_rank(&sh, b)->part_mass;
        if (by_k && cross(false, (u64)k)) {
            cut_bin = f.bin;
            if (f.above + f.count > (unsigned)k) cut_key = refine(false, (u64)(k - f.above), 0u);
            total = f.above_mass + f.mass;
        }
        if (by_p && total > 0) {
            if (by_k) cluster.sync();          // what the search before left has been read
            const u64 target = (u64)((double)tp * (double)total);
            if (cross(true, target + 1)) {     // (always: the target is less than the total)
                const unsigned least = f.bin == cut_bin ? cut_key : 0u;
                cut_bin = f.bin;
                cut_key = refine(true, target + 1 - f.above_mass, least);
            }
        }
    }
    // ---- the draw: masses of the kept tokens in index order; a warp owns a contiguous part of the slice ----
    const u64 floor_mass = greedy ? 0 : (u64)((double)fminf(fmaxf(mp, 0.f), 1.f) * (double)SMP_FIX);
    auto kept_mass = [&](float s) -> u64 {
        const int b = bin_of(s);
        if (b > cut_bin || (b == cut_bin && order_key(s) < cut_key)) return 0;
        const u64 q = mass_of(s);
        return q >= floor_mass ? q : 0;
    };
    const int span = (n + SMP_WARPS - 1) / SMP_WARPS, from = warp * span, to = min(n, from + span);
    u64 sum = 0;
    for (int i = from + lane; i < to; i += 32) sum += kept_mass(value(i));
    sum = warp_sum_u64(sum);
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        u64 t = 0;
        for (int w = 0; w < SMP_WARPS; ++w) t += sh.warp_sum[w];
        sh.all_mass = t;
    }
    cluster.sync();
    u64 total = 0, before = 0;
    for (int c = 0; c < C; ++c) {
        const u64 t = cluster.map_shared_rank(&sh, c)->all_mass;
        if (c < rank) before += t;
        total += t;
    }
    if (greedy) {                              // log-softmax of the row at the argmax: exp(0) / sum
        if (rank == 0 && tid == 0) finish(arg, -logf((float)((double)total / (double)SMP_FIX)));
        cluster.sync();
        return;
    }
    u64 target = (u64)((double)(uniform ? uniform[r] : 0.f) * (double)total);
    if (target >= total) target = total - 1;
    for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
    if (target >= before && target - before < sum) {                    // (warp-uniform) the drawn token is this warp's
        u64 run = before;
        for (int base = from; base < to; base += 32) {
            const u64 q = base + lane < to ? kept_mass(value(base + lane)) : 0;
            u64 inc = q;                       // inclusive scan over the warp
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            const unsigned hits = __ballot_sync(0xffffffffu, q > 0 && run + inc > target);
            if (hits) {
                if (lane == __ffs(hits) - 1) finish(first + base + lane, logf((float)((double)q / (double)total)));
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

// Values of a slice that a block's shared memory holds beside its tables.
#define SMP_HELD_MAX ((200 * 1024 - (int)sizeof(SampleShared)) / 4)

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
    cfg.dynamicSmemBytes = (size_t)held * 4;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, sample_kernel, logits, row_stride, V, slice, held, temperature, top_k, top_p, min_p, uniform, out_token,
                                   out_logprob);
}
