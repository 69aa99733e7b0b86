// Attention of prompt portions over a cache in 8 bits (csrc/cache_8bit.cuh) on the 5th-generation tensor cores (tcgen05.mma, accumulators in TMEM),
// compiled for one head size: -DFA_HD, a multiple of 16 up to 256.
//
// The function is that of csrc/flash_decode_8bit.cu for every token of a list of tiles: a query at position p reads the keys lo..p of its
// request (lo = 0 or p - window + 1).  Scores, maxima, sums and the output accumulate in float32.
//
// A block owns consecutive tokens of one request and ALL query heads of one KV head (up to 128): rows of its one or two query tiles of 128 are
// (token, head) pairs, so a short portion fills a tile as a long one does and a tile's mask is as sharp as its few tokens.  It walks that request's
// keys in tiles of 64, which both query tiles read.  Roles:
//   warps 0..3 (and 4..7), a thread per row   read the scores of a key tile from TMEM, write P as halves where the scores were, keep the sum of their row and,
//        beside that, its largest score: a row's base is an older maximum, and only when it has been passed by 2^8 it is moved, the row's output
//        in TMEM scaled and the scores weighed again.  While one query tile's rows are exponentiated the tensor cores work on the other's products;
//   one warp             looks up where the keys' rows are and their pages' scales, up to 8 tiles ahead;
//   four warps for keys, four for values   bring them: 16 bytes a load into registers, two tiles ahead, e4m3 to halves (exact), times a power of two, into two
//        stages of 128-byte swizzled rows.  The pages' scales are folded in here: page by page 2^(e - E + 7), E the largest
//        exponent of all pages that the block reads (found first; 448 * 2^7 is below the largest half), so that scores and outputs of all tiles are in one
//        unit, which a row's own factor and the end undo.  Exact down to pages 2^22 below the largest.  A block that reads pages further apart takes its rows
//        one by one, a warp a row, in float32 (some of its rows may read the small pages alone; pages of the least scale, 2^-100, are counted as zeros beside larger ones);
//        Rows that no query of the block reads, or that the table does not hold (flagged), are zeros.  A page whose scale is not a number gives
//        keys of NaN and values of zero: who may read it gets NaN, rows that may not replace the score;
//   one warp a query tile   issues S = Q K^T (both K-major) into one of two score buffers and O += P V (P from TMEM, V as stored: N contiguous).
// Where a launch has so few tokens that half of the SMs would be without a block, each item's keys are shared out among several, which leave base, sum and
// output as they are for a second launch to join.  So are the keys of the items that would be the few blocks of a last round.
//
// Measured in a graph (32 heads of 128, 8 KV heads), tiles and table settled: a prompt of 2,048 tokens 53 us, 0.65 PFLOP/s; three portions of 512 at position 2,500 90 us,
// 0.71 (every block whole: 112); 8 tokens behind 8,000 keys 27 us.  Where they are not, what follows from them begins behind the wait for the kernel ahead: 54, 92 and 32.  A step of 64 keys takes a block 1.0 us where exponentials alone (16 a cycle and SM) take 0.54, the products 0.55
// and shared memory's traffic 0.65.  No unit is full (issue slots and the exponential unit about half, ALUs and tensor cores a third): a step is a chain of waits, loads
// from TMEM, weights and votes.  What a block takes besides, some 8 us: queries and scales (3 us), the first keys (2), the last product and the output (2).
// Steps on the way: P through shared memory and keys and values by the same four warps 75 and 165 us.
// Taken back: two threads a row (three portions of 512 94 for 92), turns between the two query tiles' exponentials (103 and 119 for 117), scores in parts of
// 16 or 32 columns (119 and 116 for 114), two loading warps with more registers (115), one block walking several items (its state costs registers and a quarter of the speed).
// Roundings: queries times a power of two of their row (largest number in [2^14, 2^15)) and the probabilities, 2^7 p with p up to 2^8, are halves.
// Every wait on an mbarrier is bounded; when one expires the block records VL_DEV_WAIT_EXPIRED, stops, and still frees its TMEM.
#include "cache_8bit.cuh"
#include "tc5.cuh"

#ifndef FA_HD
#define FA_HD 128
#endif

using namespace tc5;
using namespace cache8;

namespace {
constexpr int HD = FA_HD;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head sizes in steps of 16 up to 256");
constexpr int GROUPS = HD <= 128 ? 2 : 1;              // query tiles of 128 rows
constexpr int BM = 128, BN = 64, CB = (HD + 63) / 64;  // CB: blocks of 64 columns (one swizzled row) a head
constexpr int SOFT = 4 * GROUPS, FIND_WARP = SOFT, MMA_WARP = SOFT + 1, LOAD0 = MMA_WARP + GROUPS, LOADERS = 4;   // (loaders of keys, and as many of values)
constexpr int NTHREADS = 32 * (LOAD0 + 2 * LOADERS), LOAD_THREADS = 32 * LOADERS, WORKERS = 32 * (SOFT + 2 * LOADERS);
constexpr unsigned ROW_BYTES = 128;
constexpr unsigned Q_BYTES = BM * CB * ROW_BYTES;      // CB blocks of [128 rows][128 bytes]
constexpr unsigned KV_STAGE = BN * CB * ROW_BYTES;     // CB blocks of [64 rows][128 bytes]
constexpr int STAGES = 2;                              // of keys, and of values (a prompt of 2,048: 2 52.9 us, 3 54.2, 4 56.3)
constexpr unsigned TILE_BYTES = GROUPS * Q_BYTES + 2 * STAGES * KV_STAGE;
constexpr int ROWS = GROUPS * BM;
constexpr int MIN_PART = 4, MOST_ITEMS = 160, MOST_ROUNDS = 8;        // splitting of keys: key tiles of a block at least, items a head and rounds at most
constexpr int FOUND = 8;                               // key tiles whose rows are looked up ahead
constexpr unsigned SMEM_BYTES = TILE_BYTES + 512 + GROUPS * BM * 4 + 2 * FOUND * BN * 8;
constexpr unsigned TMEM_COLS = 512;                    // scores 2 x 64 a query tile, behind them the outputs
constexpr unsigned O_COL = GROUPS * 2 * BN;
constexpr int PIECES = HD / 16, EACH = (BN * PIECES + LOAD_THREADS - 1) / LOAD_THREADS;   // 16-byte pieces of a row, of a tile a thread
constexpr int QL = HD <= 16 ? 2 : HD <= 32 ? 4 : HD <= 64 ? 8 : HD <= 128 ? 16 : 32;      // lanes a row of queries or of the output, 8 features each
constexpr float RESCALE_ABOVE = 8.0f, P_SHIFT = 7.0f;
constexpr int FOLD = 7;
constexpr int FAR = 24 - 9 + FOLD;                     // pages' exponents that e4m3 values, multiples of 2^-9, and halves, of 2^-24, leave room for

__host__ __device__ constexpr unsigned idesc_f16(int m, int n) {       // float32 sums of halves: bits 4-5 = 1, operand types 0
    return (1u << 4) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ unsigned long long pair(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(unsigned long long v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <bool ACC>
__device__ __forceinline__ void mma_lo(unsigned tmem_c, unsigned a_lo, unsigned b_lo, unsigned a_hi, unsigned b_hi, unsigned idesc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %5, 0;\n mov.b64 da, {%1, %2};\n mov.b64 db, {%3, %4};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %6, p;\n}"
        ::"r"(tmem_c), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(ACC ? 1u : 0u), "r"(idesc) : "memory");
}
// the same with A in TMEM: a row a lane, two halves a column
template <bool ACC>
__device__ __forceinline__ void mma_tmem(unsigned tmem_c, unsigned tmem_a, unsigned b_lo, unsigned b_hi, unsigned idesc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %3};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %5, p;\n}"
        ::"r"(tmem_c), "r"(tmem_a), "r"(b_lo), "r"(b_hi), "r"(ACC ? 1u : 0u), "r"(idesc) : "memory");
}
// byte offset of the 16-byte chunk `chunk` (0..7) of row `row` in a tile of 128-byte swizzled rows
__device__ __forceinline__ unsigned swizzled(int row, int chunk) { return (unsigned)row * ROW_BYTES + (unsigned)((chunk ^ (row & 7)) << 4); }
// (no tile of the cache is read twice by a block)
__device__ __forceinline__ uint4 load_once(const uint4* p) {
    uint4 r;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ unsigned times(unsigned h2, unsigned f2) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&h2), *reinterpret_cast<const __half2*>(&f2));
    return *reinterpret_cast<const unsigned*>(&r);
}
// Items of the list: cut i % cuts of tile i / cuts, the tokens that a block takes for one KV head (or a part of its query heads).
struct List { const int4* tiles; int num_tiles, cuts, tokens, window; };
struct Item {
    int req, tok0, pos0, count, lo, jt0, n;                              // tokens, the first key, the first key tile, key tiles (0: no tokens)
    __device__ __forceinline__ Item(const List& list, int i) {
        const int4 tile = list.tiles[i / list.cuts];
        const int skip = i % list.cuts * GROUPS * list.tokens;
        req = tile.x; tok0 = tile.y + skip; pos0 = tile.w + skip;
        count = min(GROUPS * list.tokens, tile.z - skip);
        lo = list.window > 0 && pos0 - list.window + 1 > 0 ? pos0 - list.window + 1 : 0;
        jt0 = lo / BN;
        n = count > 0 ? (pos0 + count - 1) / BN - jt0 + 1 : 0;
    }
};
// Splitting of keys: item i's key tiles go to parts[i] blocks in equal shares, of as few tiles as there are blocks for (MIN_PART at least).
// The blocks of a head are numbered from item 0's on; a lane holds items lane, lane + 32, ...
struct Split {
    static constexpr int U = MOST_ITEMS / 32;
    int n[U], parts[U], before[U], blocks;                               // `before`: blocks of the items ahead; `blocks`: of a head
    __device__ __forceinline__ Split(const List& list, int most) {       // (all lanes of a warp)
        const int lane = threadIdx.x & 31, in_list = list.num_tiles * list.cuts;
        int all = 0, longest = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            n[u] = u * 32 + lane < in_list ? Item(list, u * 32 + lane).n : 0;
            all += n[u];
            longest = max(longest, n[u]);
        }
        all = __reduce_add_sync(0xffffffffu, all);
        longest = max(1, __reduce_max_sync(0xffffffffu, longest));
        int share = min(longest, max(MIN_PART, (all + most - 1) / most)), enough = longest;
        while (share < enough) {                                         // the smallest share for which the blocks are enough
            const int mid = (share + enough) / 2;
            int sum = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) sum += (n[u] + mid - 1) / mid;
            if (__reduce_add_sync(0xffffffffu, sum) <= most) enough = mid;
            else share = mid + 1;
        }
        blocks = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            parts[u] = (n[u] + enough - 1) / enough;
            int x = parts[u];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
            before[u] = blocks + x - parts[u];
            blocks += __shfl_sync(0xffffffffu, x, 31);
        }
    }
};
// Where a launch has more blocks than SMs and its last round is short of blocks: that round's items, with the shortest rows of keys, in parts each.
struct Tail {
    int whole, parts;                                                    // items ahead of them; parts each, 0: none
    __device__ __forceinline__ int parts_of(const Item& item) const { return min(parts, (item.n + MIN_PART - 1) / MIN_PART); }
};
struct Partial { float4* out; float2* ml; };                             // out [blocks with parts][HD / 4][ROWS], ml (base, sum) [blocks with parts][ROWS]
// What a block reads and writes, for `rows_alone`.
struct Block {
    const bf16* q; int q_stride; bf16* out; const unsigned char *kcache, *vcache; const float *kscale, *vscale; const int* table; int max_blocks;
    int nq, nkv, page_size, num_pages; float scale_log2; int window; unsigned* err; int heads, tokens, kvh, h0, nheads, tok0, pos0, count, groups, lo, hi;
    int parts, place; Partial partial;
};
// The block's rows one by one, a warp a row, in float32: for pages too far apart for one unit, which are not met in earnest (a prompt of 2,048 tokens 7 ms).  It is
// called: within the kernel it cost the tensor cores' way 1 to 2 us of 53 and 92.
__device__ __noinline__ void rows_alone(const Block& b) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_head = 65536 / b.heads + 1;
    constexpr int W = (HD / 2 + 31) / 32, AT_ONCE = 4;               // pairs of features a lane, keys on their way together
#pragma unroll 1
    for (int r = warp; r < b.groups * BM; r += NTHREADS / 32) {
        const int rr = r & (BM - 1), t = (rr * per_head) >> 16, tk = (r / BM) * b.tokens + t, h = rr - t * b.heads;
        if (t >= b.tokens || tk >= b.count || h >= b.nheads) continue;
        const int qpos = b.pos0 + tk, last = min(b.hi, qpos);
        const bf16* row = b.q + (size_t)(b.tok0 + tk) * b.q_stride + (size_t)(b.h0 + h) * HD;
        float2 x[W], o[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int i = lane + 32 * w;
            x[w] = i < HD / 2 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(row + 2 * i)) : make_float2(0.f, 0.f);
            o[w] = make_float2(0.f, 0.f);
        }
        float m = -INFINITY, l = 0.f;
#pragma unroll 1
        for (int key = b.window > 0 ? max(b.lo, qpos - b.window + 1) : b.lo; key <= last;) {
            const int blk = key / b.page_size, end = min(last, blk * b.page_size + (b.page_size - 1)), page = blk < b.max_blocks ? b.table[blk] : -1;
            if (page < 0 || page >= b.num_pages) {
                if (lane == 0 && b.err) atomicOr(b.err, VL_DEV_BAD_PAGE);
                key = end + 1;
                continue;
            }
            const size_t head = (size_t)page * b.nkv + b.kvh, at = (head * b.page_size + (key - blk * b.page_size)) * HD;
            const unsigned char *kp = b.kcache + at, *vp = b.vcache + at;
            const float ks = b.kscale[head] * b.scale_log2, vs = b.vscale[head];
#pragma unroll 1
            for (; key <= end; key += AT_ONCE, kp += AT_ONCE * HD, vp += AT_ONCE * HD) {
                unsigned short k[AT_ONCE][W], v[AT_ONCE][W];
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const int i = lane + 32 * w;
                        const bool there = key + j <= end && i < HD / 2;
                        k[j][w] = there ? *reinterpret_cast<const unsigned short*>(kp + j * HD + 2 * i) : 0;
                        v[j][w] = there ? *reinterpret_cast<const unsigned short*>(vp + j * HD + 2 * i) : 0;
                    }
                auto two = [](unsigned short e) {
                    const unsigned half2 = to_half2(e);
                    return __half22float2(*reinterpret_cast<const __half2*>(&half2));
                };
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) {
                    if (key + j > end) continue;
                    float s = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const float2 y = two(k[j][w]);
                        s += x[w].x * y.x + x[w].y * y.y;
                    }
                    s = warp_sum(s) * ks;
                    if (s > m) {
                        const float corr = exp2f(m - s);
                        l *= corr;
#pragma unroll
                        for (int w = 0; w < W; ++w) { o[w].x *= corr; o[w].y *= corr; }
                        m = s;
                    }
                    const float p = exp2f(s - m), pv = p * vs;
                    l += p;
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const float2 y = two(v[j][w]);
                        o[w].x += pv * y.x; o[w].y += pv * y.y;
                    }
                }
            }
            key = end + 1;
        }
        if (b.parts > 1) {                                             // (in the units of the other shares)
            const float unit = power_of_two((int)P_SHIFT);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int i = lane + 32 * w;
                if (i < HD / 2)
                    reinterpret_cast<float2*>(b.partial.out + ((size_t)b.place * (HD / 4) + i / 2) * ROWS + r)[i & 1] = make_float2(o[w].x * unit, o[w].y * unit);
            }
            if (lane == 0) b.partial.ml[(size_t)b.place * ROWS + r] = make_float2(m, l * unit);
        } else {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            bf16* dst = b.out + ((size_t)(b.tok0 + tk) * b.nq + b.h0 + h) * HD;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int i = lane + 32 * w;
                if (i < HD / 2) *reinterpret_cast<__nv_bfloat162*>(dst + 2 * i) = __floats2bfloat162_rn(o[w].x * inv, o[w].y * inv);
            }
        }
    }
}
}  // namespace

// tiles[i] = {row of the block table, index of the tile's first token in the step, tokens (<= 128), position of the first}
__global__ void __launch_bounds__(NTHREADS, 1)
flash_tc5_8bit_kernel(const bf16* __restrict__ q, int q_stride, bf16* __restrict__ out, const unsigned char* __restrict__ kcache,
                      const unsigned char* __restrict__ vcache, const float* __restrict__ kscale, const float* __restrict__ vscale,
                      const int* __restrict__ block_table, int max_blocks, const int4* __restrict__ tiles, int num_tiles, int nq, int nkv, int page_size,
                      int num_pages, float scale_log2, int window, unsigned* err, int heads, int htiles, int tokens, int cuts, int split, Tail tail, Partial partial,
                      int settled) {
    extern __shared__ __align__(1024) unsigned char smem[];              // (the block's only shared memory, so it begins the window)
    unsigned char* Qs = smem;                                            // GROUPS
    unsigned char* Ks = Qs + GROUPS * Q_BYTES;                           // STAGES
    unsigned char* Vs = Ks + STAGES * KV_STAGE;                          // STAGES
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + TILE_BYTES);
    unsigned long long *k_full = bars, *k_empty = bars + STAGES, *v_full = bars + 2 * STAGES, *v_empty = bars + 3 * STAGES;
    unsigned long long *s_full = bars + 4 * STAGES, *p_full = s_full + 4, *pv_done = p_full + 4;           // [GROUPS][2 buffers]
    unsigned long long *found_full = pv_done + 4, *found_empty = found_full + FOUND;
    unsigned& tmem_slot = *reinterpret_cast<unsigned*>(found_empty + FOUND);
    int* words = reinterpret_cast<int*>(found_empty + FOUND + 1);
    int &failed = words[0], &top_k = words[1], &top_v = words[2], &low_k = words[3], &low_v = words[4];
    float* s_row_scale = reinterpret_cast<float*>(smem + TILE_BYTES + 512);                      // [GROUPS * BM]
    int2* s_found = reinterpret_cast<int2*>(s_row_scale + GROUPS * BM);                          // keys, values: [FOUND][BN] cache row (-1: zeros) and factor
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(smem) & 1023u) {                                        // (uniform) never expected; the tiles would be misread
        pdl_wait();
        if (tid == 0 && err) atomicOr(err, VL_DEV_WAIT_EXPIRED | VL_DEV_IN_FLASH_8BIT);
        return;
    }
    pdl_launch_dependents();
    if (!settled) pdl_wait();                                            // a kernel before this one may be writing the list or the table
    // This block's item and its key tiles from .. to; the items with the longest rows of keys first, or a share of an item's keys.
    const List list = {tiles, num_tiles, cuts, tokens, window};
    int head = (int)blockIdx.x, number = num_tiles * cuts - 1 - (int)blockIdx.y, part = 0, parts = 1, place = -1;
    if (tail.parts) {
        place = (int)blockIdx.x - tail.whole;
        const int id = place < 0 ? (int)blockIdx.x : tail.whole + place / tail.parts;
        head = id % (nkv * htiles);
        number = num_tiles * cuts - 1 - id / (nkv * htiles);
    }
    if (split) {
        const Split plan(list, split / (nkv * htiles));
        place = (int)blockIdx.x;
        head = plan.blocks ? (int)blockIdx.x / plan.blocks : nkv * htiles;
        if (head >= nkv * htiles) { pdl_wait(); return; }                // (a launch that does not wait would end before the ones ahead of it)
        const int x = (int)blockIdx.x - head * plan.blocks;
        number = -1;
#pragma unroll
        for (int u = 0; u < Split::U; ++u) {
            const unsigned here = __ballot_sync(0xffffffffu, x >= plan.before[u] && x < plan.before[u] + plan.parts[u]);
            if (here) {
                const int from = __ffs(here) - 1;
                number = u * 32 + from;
                part = x - __shfl_sync(0xffffffffu, plan.before[u], from);
                parts = __shfl_sync(0xffffffffu, plan.parts[u], from);
            }
        }
    }
    const Item item(list, number);
    if (tail.parts && place >= 0) { part = place % tail.parts; parts = tail.parts_of(item); }
    if (item.n == 0 || part >= parts) { pdl_wait(); return; }            // (the whole block)
    const int from = (int)((long long)item.n * part / parts), n_tiles = (int)((long long)item.n * (part + 1) / parts) - from;
    const int req = item.req, tok0 = item.tok0, pos0 = item.pos0, count = item.count, jt0 = item.jt0 + from;
    const int kvh = head / htiles, grp = nq / nkv, hbase = (head - kvh * htiles) * heads;
    const int nheads = min(heads, grp - hbase), h0 = kvh * grp + hbase;
    const int groups = GROUPS == 2 && count > tokens ? 2 : 1;
    // the keys that this block reads for any of its rows
    const int lo = max(item.lo, jt0 * BN), hi = min(pos0 + count - 1, (jt0 + n_tiles) * BN - 1);
    const int* table = block_table + (size_t)req * max_blocks;
    const int per_head = 65536 / heads + 1;                              // (r * per_head) >> 16 is r / heads for rows of a tile

    // (barrier i by thread i; the numbers of arrivals in the order of `bars`)
    if (tid < 4 * STAGES + 12 + 2 * FOUND) {
        const int i = tid;
        const int count = i < 4 * STAGES ? (i / STAGES % 2 ? groups : LOAD_THREADS) : i < 4 * STAGES + 4 ? 1 : i < 4 * STAGES + 8 ? BM : i < 4 * STAGES + 12 + FOUND ? 1 : 2 * LOADERS;
        mbar_init(&bars[i], count);
        mbar_fence_init();
    } else if (tid == NTHREADS - 1) {
        failed = 0;
        top_k = top_v = EXP_MIN;
        low_k = low_v = 128;
    }
    const int worker = warp < SOFT ? tid : tid - 32 * (LOAD0 - SOFT), first_page = lo / page_size, last_page = hi / page_size;
    auto page_at = [&](int blk) -> int {
        const int page = blk <= last_page && blk < max_blocks ? table[blk] : -1;
        return page < num_pages ? page : -1;
    };
    int page = page_at(first_page + worker);
    __syncthreads();

    // The finder: a lane looks up keys `lane` and lane + 32 of every tile, in three steps a tile apart, so that no load is waited for: the page, its
    // scales, and what they say.
    struct Found { int page, at; float ks, vs; };
    auto page_of = [&](int it, int u) -> Found {
        Found f = {-1, -1, 0.f, 0.f};
        const int key = (jt0 + it) * BN + u * 32 + lane;
        if (it >= n_tiles || key < lo || key > hi) return f;
        const int blk = key / page_size;
        f.at = key - blk * page_size;
        if (blk < max_blocks) f.page = table[blk];
        return f;
    };
    auto scales_of = [&](Found& f) {
        if (f.at < 0) return;
        if (f.page < 0 || f.page >= num_pages) {
            f.page = -1;
            if (err) atomicOr(err, VL_DEV_BAD_PAGE);
            return;
        }
        f.ks = kscale[(size_t)f.page * nkv + kvh];
        f.vs = vscale[(size_t)f.page * nkv + kvh];
    };
    Found a[BN / 32], b[BN / 32];
    // The largest exponents of the pages that the block reads, and the queries as halves; the first loads of both are on their way at once.
    // QL lanes a query row, 8 features each; rows of no token are zeros.
    if (warp < SOFT || warp >= LOAD0) {
        int ek = EXP_MIN, ev = EXP_MIN, lk = 128, lv = 128;
        pdl_wait();
        constexpr int AT_ONCE = WORKERS / QL;
        constexpr int AHEAD = (GROUPS * BM + AT_ONCE - 1) / AT_ONCE;
        const int r0 = worker / QL, c = worker - r0 * QL;
        uint4 raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int r = r0 + u * AT_ONCE, rr = r & (BM - 1), t = (rr * per_head) >> 16, tk = (r / BM) * tokens + t, h = rr - t * heads;
            const bool live = r < groups * BM && t < tokens && tk < count && h < nheads && c < HD / 8;
            raw[u] = make_uint4(0u, 0u, 0u, 0u);
            if (live) raw[u] = *reinterpret_cast<const uint4*>(q + (size_t)(tok0 + tk) * q_stride + (size_t)(h0 + h) * HD + c * 8);
        }
        auto exponents = [&](float ks, float vs) {
            const int k = (int)(__float_as_uint(ks) >> 23) - 127, v = (int)(__float_as_uint(vs) >> 23) - 127;
            if (ks == ks) ek = max(ek, k);
            if (vs == vs) ev = max(ev, v);
            if (k > EXP_MIN) lk = min(lk, k);                            // (NaN's is 128)
            if (v > EXP_MIN) lv = min(lv, v);
        };
        const float ks = page >= 0 ? kscale[(size_t)page * nkv + kvh] : 0.f, vs = page >= 0 ? vscale[(size_t)page * nkv + kvh] : 0.f;
        for (int blk = first_page + worker + WORKERS; blk <= last_page; blk += WORKERS) {
            page = page_at(blk);
            if (page >= 0) exponents(kscale[(size_t)page * nkv + kvh], vscale[(size_t)page * nkv + kvh]);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int r = r0 + u * AT_ONCE, rr = r & (BM - 1);
            unsigned* w = &raw[u].x;
            __nv_bfloat162 most = __habs2(*reinterpret_cast<__nv_bfloat162*>(&w[0]));
#pragma unroll
            for (int i = 1; i < 4; ++i) most = __hmax2(most, __habs2(*reinterpret_cast<__nv_bfloat162*>(&w[i])));
#pragma unroll
            for (int o = 1; o < QL; o <<= 1) most = __hmax2(most, __shfl_xor_sync(0xffffffffu, most, o));
            const unsigned both = *reinterpret_cast<unsigned*>(&most), top = max(both & 0x7fffu, both >> 16);
            const int e = top == 0 || top >= 0x7f80u ? 0 : max(-112, (int)(top >> 7) - 127 - 14);
            const float f = power_of_two(-e);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_half(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
            // a query with a NaN or an infinity is NaN all along: its scores might all be -inf as those of a row without keys are
            if (__builtin_expect(top >= 0x7f80u, 0)) raw[u] = make_uint4(0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u);
            if (r < groups * BM && c < HD / 8) {
                *reinterpret_cast<uint4*>(Qs + (r / BM) * Q_BYTES + (unsigned)(c >> 3) * (BM * ROW_BYTES) + swizzled(rr, c & 7)) = raw[u];
                if (c == 0) s_row_scale[r] = scale_log2 * power_of_two(e);
            }
        }
        exponents(ks, vs);
        ek = __reduce_max_sync(0xffffffffu, ek);
        ev = __reduce_max_sync(0xffffffffu, ev);
        lk = __reduce_min_sync(0xffffffffu, lk);
        lv = __reduce_min_sync(0xffffffffu, lv);
        if (lane == 0) { atomicMax(&top_k, ek); atomicMax(&top_v, ev); atomicMin(&low_k, lk); atomicMin(&low_v, lv); }
    } else {
        if (warp == FIND_WARP) {
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) { a[u] = page_of(0, u); b[u] = page_of(1, u); }
        }
        pdl_wait();                                                      // q, the cache and its scales are written by the kernel before
        if (warp == FIND_WARP) {
            __syncwarp();
            tc5_alloc(&tmem_slot, TMEM_COLS);                            // (not earlier: a block of that kernel may be about to take its own)
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) scales_of(a[u]);
        }
    }
    tc5_fence_before();
    fence_proxy_async_smem();
    __syncthreads();
    tc5_fence_after();
    const unsigned tmem_base = tmem_slot;

    const int role = warp_number();
    if (top_k - low_k > FAR || top_v - low_v > FAR) {                    // ---- pages too far apart for one unit ----
        rows_alone({q, q_stride, out, kcache, vcache, kscale, vscale, table, max_blocks, nq, nkv, page_size, num_pages, scale_log2, window, err, heads, tokens, kvh, h0,
                    nheads, tok0, pos0, count, groups, lo, hi, parts, place, partial});
    } else if (role >= LOAD0) {                                                 // ---- keys and values ----
        const bool values = role >= LOAD0 + LOADERS;
        const int ct = (tid - LOAD0 * 32) % LOAD_THREADS;
        const unsigned char* cache = values ? vcache : kcache;
        unsigned char* stages = values ? Vs : Ks;
        unsigned long long *full = values ? v_full : k_full, *empty = values ? v_empty : k_empty;
        const int2* found = s_found + (values ? FOUND * BN : 0);
        // Piece i of this thread: row r, 16-byte piece c.  Head sizes of a power of two have c and the row's place in the swizzle the same for all of
        // a thread's pieces, whose places are then a constant apart.
        constexpr int APART = LOAD_THREADS / PIECES;
        constexpr bool EVEN = LOAD_THREADS % PIECES == 0 && APART % 8 == 0 && BN % APART == 0;
        const int r0 = ct / PIECES, c0 = ct - r0 * PIECES;
        const unsigned char* my_cache = cache + c0 * 16;
        const int2* my_found = found + r0;
        auto place = [&](int r, int c, int half) { return (unsigned)(c >> 2) * (BN * ROW_BYTES) + swizzled(r, 2 * (c & 3) + half); };
        // (eight lanes store 16 bytes at a time, and pieces 4 on lie in another block of rows but in the banks of pieces 0 to 3: they store their second half first)
        const bool flip = PIECES >= 8 && (c0 & 4);
        unsigned char *my_a = stages + place(r0, c0, flip), *my_b = stages + place(r0, c0, !flip);
        auto load = [&](uint4 (&x)[EACH], int it) {
            const int2* f = my_found + (it % FOUND) * BN;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if constexpr (EVEN) {
                    const int row = f[i * APART].x;
                    if (row >= 0) x[i] = load_once(reinterpret_cast<const uint4*>(my_cache + (size_t)row * HD));
                } else {
                    const int idx = i * LOAD_THREADS + ct, r = idx / PIECES, c = idx - r * PIECES;
                    const int row = idx < BN * PIECES ? f[r - r0].x : -1;
                    if (row >= 0) x[i] = load_once(reinterpret_cast<const uint4*>(cache + (size_t)row * HD + c * 16));
                }
            }
        };
        auto store = [&](const uint4 (&x)[EACH], int it) {
            const int2* fold = my_found + (it % FOUND) * BN;
            const unsigned stage = (unsigned)(it % STAGES) * KV_STAGE;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int idx = i * LOAD_THREADS + ct, r = idx / PIECES, c = idx - r * PIECES;
                if (!EVEN && idx >= BN * PIECES) continue;
                const unsigned f = (unsigned)fold[EVEN ? i * APART : r - r0].y;
                const unsigned w[4] = {EVEN && flip ? x[i].z : x[i].x, EVEN && flip ? x[i].w : x[i].y, EVEN && flip ? x[i].x : x[i].z, EVEN && flip ? x[i].y : x[i].w};
                uint4 a, b;
                a.x = times(half2_low(w[0]), f); a.y = times(half2_high(w[0]), f); a.z = times(half2_low(w[1]), f); a.w = times(half2_high(w[1]), f);
                b.x = times(half2_low(w[2]), f); b.y = times(half2_high(w[2]), f); b.z = times(half2_low(w[3]), f); b.w = times(half2_high(w[3]), f);
                if constexpr (EVEN) {
                    *reinterpret_cast<uint4*>(my_a + stage + i * (APART * ROW_BYTES)) = a;
                    *reinterpret_cast<uint4*>(my_b + stage + i * (APART * ROW_BYTES)) = b;
                } else {
                    *reinterpret_cast<uint4*>(stages + stage + place(r, c, 0)) = a;
                    *reinterpret_cast<uint4*>(stages + stage + place(r, c, 1)) = b;
                }
            }
        };
        // two tiles on their way: the loads of tile it + 2 are issued when those of tile it have been used
        bool ok = true;
        auto ask = [&](uint4 (&x)[EACH], int it) {
            if (it >= n_tiles || !ok) return;
            ok = warp_wait(&found_full[it % FOUND], (unsigned)((it / FOUND) & 1));
            if (ok) load(x, it);
        };
        auto bring = [&](uint4 (&x)[EACH], int it) {
            if (it >= n_tiles || !ok) return;
            ok = it < STAGES || warp_wait(&empty[it % STAGES], (unsigned)((it / STAGES - 1) & 1));
            if (!ok) return;
            store(x, it);
            fence_proxy_async_smem();
            mbar_arrive(&full[it % STAGES]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&found_empty[it % FOUND]);
        };
        uint4 x[EACH], y[EACH];
        ask(x, 0);
        ask(y, 1);
        for (int it = 0; it < n_tiles && ok; it += 2) {
            bring(x, it);
            ask(x, it + 2);
            bring(y, it + 1);
            ask(y, it + 3);
        }
        if (!ok && lane == 0) atomicExch(&failed, 1);
    } else if (role == FIND_WARP) {                                      // ---- where the keys are ----
        const int EK = top_k, EV = top_v;
        auto note = [&](const Found& f, int it, int u) {
            const bool no_value = f.vs != f.vs, none = f.ks != f.ks || no_value;
            const __half fk = none ? __ushort_as_half(0x7e00) : __float2half_rn(f.ks * power_of_two(FOLD - EK));
            const __half fv = __float2half_rn(no_value ? 0.f : f.vs * power_of_two(FOLD - EV));
            const int at = (it % FOUND) * BN + u * 32 + lane, row = f.page < 0 ? -1 : (f.page * nkv + kvh) * page_size + f.at;
            s_found[at] = make_int2(row, (int)(0x10001u * __half_as_ushort(fk)));
            s_found[FOUND * BN + at] = make_int2(no_value ? -1 : row, (int)(0x10001u * __half_as_ushort(fv)));
        };
        bool ok = true;
        // `now`, whose scales are on their way, is said and takes up the tile two further on; `next`, whose pages are, asks for its scales.  (Two
        // names that change places every step: a copy of one into the other would wait for its loads.)
        auto step = [&](Found (&now)[BN / 32], Found (&next)[BN / 32], int it) {
            if (it >= n_tiles || !ok) return;
            ok = it < FOUND || warp_wait(&found_empty[it % FOUND], (unsigned)((it / FOUND - 1) & 1));
            if (!ok) return;
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) note(now[u], it, u);
            __syncwarp();
            if (lane == 0) mbar_arrive(&found_full[it % FOUND]);
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) { now[u] = page_of(it + 2, u); scales_of(next[u]); }
        };
        for (int it = 0; it < n_tiles && ok; it += 2) {
            step(a, b, it);
            step(b, a, it + 1);
        }
        if (!ok && lane == 0) atomicExch(&failed, 1);
    } else if (role >= MMA_WARP && role - MMA_WARP < groups) {           // ---- issuer of a query tile's products ----
        const int gr = role - MMA_WARP;
        const bool lead = elect_one();
        const unsigned tmem = __shfl_sync(0xffffffffu, tmem_base, 0);    // (the warp's own, like everything an instruction is issued with)
        constexpr unsigned s_idesc = idesc_f16(BM, BN), o_idesc = idesc_f16(BM, HD) | IDESC_B_MN_MAJOR;
        const unsigned long long dq = make_smem_desc(Qs + gr * Q_BYTES), dk = make_smem_desc(Ks);
        const unsigned long long dv = make_smem_desc_lbo_sbo(Vs, BN * ROW_BYTES, 8 * ROW_BYTES);
        const unsigned q_lo = (unsigned)dq, k_lo = (unsigned)dk, k_hi = (unsigned)(dq >> 32), v_lo = (unsigned)dv, v_hi = (unsigned)(dv >> 32);
        const unsigned to = tmem + O_COL + (unsigned)(gr * 128);
        bool ok = true;
        auto scores = [&](int it) {                                      // S = Q K^T
            const int s = gr * 2 + (it & 1), stage = it % STAGES;
            ok = warp_wait(&k_full[stage], (unsigned)((it / STAGES) & 1));
            if (!ok) return;
            tc5_fence_after();
            const unsigned kb = k_lo + (unsigned)stage * (KV_STAGE >> 4), tc = tmem + (unsigned)(s * BN);
            if (lead) {
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    // 16 columns further on: 32 bytes inside the swizzled row; 64 columns: the next block of rows
                    const unsigned qo = (unsigned)(ks >> 2) * (BM * ROW_BYTES >> 4) + (unsigned)(ks & 3) * 2;
                    const unsigned ko = (unsigned)(ks >> 2) * (BN * ROW_BYTES >> 4) + (unsigned)(ks & 3) * 2;
                    if (ks == 0) mma_lo<false>(tc, q_lo + qo, kb + ko, k_hi, k_hi, s_idesc);
                    else mma_lo<true>(tc, q_lo + qo, kb + ko, k_hi, k_hi, s_idesc);
                }
                tc5_commit(&k_empty[stage]);
                tc5_commit(&s_full[s]);
            }
        };
        scores(0);
        if (ok && n_tiles > 1) scores(1);
        for (int it = 0; it < n_tiles && ok; ++it) {
            const int s = gr * 2 + (it & 1), stage = it % STAGES;
            ok = warp_wait(&v_full[stage], (unsigned)((it / STAGES) & 1)) && warp_wait(&p_full[s], (unsigned)((it / 2) & 1));
            if (!ok) break;
            tc5_fence_after();
            const unsigned pb = tmem + (unsigned)(s * BN), vb = v_lo + (unsigned)stage * (KV_STAGE >> 4);
            if (lead) {                                                  // O += P V
#pragma unroll
                for (int k = 0; k < BN / 16; ++k) {
                    // 16 keys further on: 8 columns of P, 16 rows of 128 bytes of V
                    if (k == 0 && it == 0) mma_tmem<false>(to, pb, vb, v_hi, o_idesc);
                    else mma_tmem<true>(to, pb + (unsigned)k * 8, vb + (unsigned)k * (16 * ROW_BYTES >> 4), v_hi, o_idesc);
                }
                tc5_commit(&v_empty[stage]);
                tc5_commit(&pv_done[s]);
            }
            if (it + 2 < n_tiles) {                                      // (the scores take the place of P, once it has been read)
                ok = warp_wait(&pv_done[s], (unsigned)((it / 2) & 1));
                if (ok) scores(it + 2);
            }
        }
        if (!ok && lead) atomicExch(&failed, 1);
    } else if (role < SOFT && warp / 4 < groups) {                       // ---- softmax: a thread per row ----
        const int gr = warp / 4, row = (warp & 3) * 32 + lane, tk = gr * tokens + row / heads;
        const int qpos = pos0 + min(tk, count - 1);
        const int first_key = (window > 0 && qpos - window + 1 > 0) ? qpos - window + 1 : 0;
        // (warp-uniform) a tile that ends behind the first row's position or begins before the last row's window holds keys that some row must not read
        const int warp_last = __reduce_min_sync(0xffffffffu, qpos), warp_first = __reduce_max_sync(0xffffffffu, first_key);
        // (positive even where the product is too small for a float32, so that -inf stays -inf: no sum of products reaches 2^40)
        const float sl2 = fmaxf(s_row_scale[gr * BM + row] * power_of_two(top_k - FOLD), 1.1754944e-38f);
        const unsigned masked = 0xff800000u;                             // -inf
        const unsigned lane_base = (unsigned)((warp & 3) * 32) << 16;
        const unsigned o_col = tmem_base + lane_base + O_COL + (unsigned)(gr * 128);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int it = 0; it < n_tiles; ++it) {
            const int s = it & 1;
            if (!warp_wait(&s_full[gr * 2 + s], (unsigned)((it / 2) & 1))) { ok = false; break; }
            tc5_fence_after();
            const unsigned buffer = tmem_base + lane_base + (unsigned)((gr * 2 + s) * BN);
            const int j0 = (jt0 + it) * BN;
            const bool edge = j0 + BN - 1 > warp_last || j0 < warp_first;
            unsigned pk[BN / 2];
            float sum, most;
            auto scores = [&](unsigned (&sv)[BN]) {
                tc5_ld32_nowait(buffer, sv);
                tc5_ld32_nowait(buffer + 32, sv + 32);
                tc5_wait_ld();
                if (edge) {
#pragma unroll
                    for (int c = 0; c < BN; ++c)
                        if (j0 + c > qpos || j0 + c < first_key) sv[c] = masked;
                }
            };
            auto peek = [&]() -> float {                                 // the largest score
                unsigned sv[BN];
                scores(sv);
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < BN; c += 2) top[c / 2 % 4] = max3(top[c / 2 % 4], __uint_as_float(sv[c]), __uint_as_float(sv[c + 1]));
                return max3(fmaxf(top[0], top[1]), top[2], top[3]) * sl2;
            };
            auto weigh = [&] {                                           // P and its sum relative to the row's base, and the largest score
                unsigned sv[BN];
                scores(sv);
                const float base = m == -INFINITY ? 0.f : m;
                const unsigned long long scale2 = pair(sl2, sl2), nbase2 = pair(P_SHIFT - base, P_SHIFT - base);
                unsigned long long sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < BN; c += 2) {
                    float t0, t1;
                    top[c / 2 % 4] = max3(top[c / 2 % 4], __uint_as_float(sv[c]), __uint_as_float(sv[c + 1]));
                    unpair(fma2(pair(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])), scale2, nbase2), t0, t1);
                    const float p0 = exp2_fast(t0), p1 = exp2_fast(t1);
                    sums[c / 2 % 2] = add2(sums[c / 2 % 2], pair(p0, p1));
                    pk[c >> 1] = pack_half(p0, p1);
                }
                float sum_hi;
                unpair(add2(sums[0], sums[1]), sum, sum_hi);
                sum += sum_hi;
                most = max3(fmaxf(top[0], top[1]), top[2], top[3]) * sl2;
            };
            // The largest score is found beside the exponentials and not before them: a row's base is an older maximum, good until it has been passed by 2^8.
            // Then it is moved and the scores, still where they were, are weighed again.
            if (it == 0) m = peek();
            weigh();
            const float m_new = fmaxf(m, most);
            const bool bump = (m_new - m) > RESCALE_ABOVE;               // false when both are -inf (NaN compares false)
            const bool any_bump = __any_sync(0xffffffffu, bump);
            const float corr = bump ? exp2_fast(m - m_new) : 1.0f;
            if (any_bump) {
                if (bump) m = m_new;
                weigh();
            }
            l = l * corr + sum;
            tc5_st32(buffer, pk);                                        // where the scores were
            if (it > 0 && any_bump) {
                if (!warp_wait(&pv_done[gr * 2 + (s ^ 1)], (unsigned)(((it - 1) / 2) & 1))) { ok = false; break; }
                tc5_fence_after();                                       // O is at rest
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    unsigned ov[32];
                    tc5_ld32(o_col + (unsigned)c0, ov);
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * corr);
                    tc5_st32(o_col + (unsigned)c0, ov);
                }
            }
            tc5_wait_st();
            tc5_fence_before();
            mbar_arrive(&p_full[gr * 2 + s]);
        }
        if (!ok || !warp_wait(&pv_done[gr * 2 + ((n_tiles - 1) & 1)], (unsigned)(((n_tiles - 1) / 2) & 1))) {
            atomicExch(&failed, 1);
        } else if (parts > 1) {                                          // a share of the item's keys: sums and base as they are
            tc5_fence_after();
            const float unit = power_of_two(top_v - FOLD);
            const bool live = row < tokens * heads && tk < count;
            float4* dst = partial.out + (size_t)place * (HD / 4) * ROWS + gr * BM + row;
#pragma unroll
            for (int c0 = 0; c0 < HD; c0 += 32) {
                unsigned ov[32];
                tc5_ld32(o_col + (unsigned)c0, ov);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (live && c0 + 4 * i < HD)
                        dst[(size_t)(c0 / 4 + i) * ROWS] = make_float4(__uint_as_float(ov[4 * i]) * unit, __uint_as_float(ov[4 * i + 1]) * unit,
                                                                       __uint_as_float(ov[4 * i + 2]) * unit, __uint_as_float(ov[4 * i + 3]) * unit);
            }
            if (live) partial.ml[(size_t)place * ROWS + gr * BM + row] = make_float2(m, l);
        } else {
            tc5_fence_after();
            const float inv = l == 0.f ? 0.f : 1.0f / l, unit = power_of_two(top_v - FOLD);
            unsigned char* turn = Qs + gr * Q_BYTES;                     // (all products with the queries are done)
            constexpr int STEP = HD <= 32 ? 32 : 64;
#pragma unroll
            for (int c0 = 0; c0 < HD; c0 += STEP) {
                unsigned ov[STEP];
#pragma unroll
                for (int i = 0; i < STEP; i += 32) tc5_ld32_nowait(o_col + (unsigned)(c0 + i), ov + i);
                tc5_wait_ld();
#pragma unroll
                for (int i = 0; i < STEP / 8; ++i) {
                    if (c0 + 8 * i >= HD) continue;
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(ov[8 * i + j]) * inv * unit;
                    const int c = c0 / 8 + i;
                    store8(reinterpret_cast<bf16*>(turn + (unsigned)(c >> 3) * (BM * ROW_BYTES) + swizzled(row, c & 7)), v);
                }
            }
            __syncwarp();
            // this warp's 32 rows, QL lanes a row: neighbouring lanes write neighbouring bytes
            const int c = lane % QL;
#pragma unroll 4
            for (int r = (warp & 3) * 32 + lane / QL; r < (warp & 3) * 32 + 32; r += 32 / QL) {
                const int t = (r * per_head) >> 16, tk = gr * tokens + t, h = r - t * heads;
                if (t < tokens && tk < count && h < nheads && c < HD / 8)
                    *reinterpret_cast<uint4*>(out + ((size_t)(tok0 + tk) * nq + h0 + h) * HD + c * 8) =
                        *reinterpret_cast<const uint4*>(turn + (unsigned)(c >> 3) * (BM * ROW_BYTES) + swizzled(r, c & 7));
            }
        }
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    if (warp == FIND_WARP) tc5_dealloc(tmem_base, TMEM_COLS);
    if (tid == 0 && failed && err) atomicOr(err, VL_DEV_WAIT_EXPIRED | VL_DEV_IN_FLASH_8BIT);
}

// The shares of an item whose keys several blocks have walked: out = sum_r 2^(m_r - M) o_r / sum_r 2^(m_r - M) l_r, M the largest base.  A block an
// item and 16 columns, a thread a row.
__global__ void __launch_bounds__(ROWS)
flash_tc5_8bit_join_kernel(const int4* __restrict__ tiles, int num_tiles, int cuts, int tokens, int window, int nq, int nkv, int heads, int htiles, int split,
                           Tail tail, Partial partial, bf16* __restrict__ out, int settled) {
    pdl_launch_dependents();
    if (!settled) pdl_wait();
    const List list = {tiles, num_tiles, cuts, tokens, window};
    const int in_list = num_tiles * cuts, id = tail.whole + (int)blockIdx.x, head = id % (nkv * htiles), number = in_list - 1 - id / (nkv * htiles);
    const Item item(list, number);
    if (item.n <= MIN_PART) { pdl_wait(); return; }                      // (every block waits: the launch behind this one waits for no other)
    int first = (int)blockIdx.x * tail.parts, parts = tail.parts_of(item);
    if (split) {
        const Split plan(list, split / (nkv * htiles));
#pragma unroll
        for (int u = 0; u < Split::U; ++u)
            if (number / 32 == u) {
                first = head * plan.blocks + __shfl_sync(0xffffffffu, plan.before[u], number % 32);
                parts = __shfl_sync(0xffffffffu, plan.parts[u], number % 32);
            }
    }
    pdl_wait();
    if (parts <= 1) return;                                              // (one block had them all)
    const int grp = nq / nkv, kvh = head / htiles, hbase = (head - kvh * htiles) * heads, nheads = min(heads, grp - hbase);
    const int row = threadIdx.x, rr = row & (BM - 1), t = rr / heads, tk = row / BM * tokens + t, h = rr - t * heads;
    if (t >= tokens || tk >= item.count || h >= nheads) return;
    const float2* ml = partial.ml + (size_t)first * ROWS + row;
    float top = -INFINITY;
    for (int k = 0; k < parts; ++k) top = fmaxf(top, ml[(size_t)k * ROWS].x);
    float sum = 0.f, o[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) o[c] = 0.f;
#pragma unroll 2
    for (int k = 0; k < parts; ++k) {
        const float2 b = ml[(size_t)k * ROWS];
        const float w = b.x == -INFINITY ? 0.f : exp2f(b.x - top);
        const float4* src = partial.out + ((size_t)(first + k) * (HD / 4) + blockIdx.y * 4) * ROWS + row;
        sum += w * b.y;                                                  // (also where w is 0: NaN stays NaN)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4 v = src[c * ROWS];
            o[4 * c] += w * v.x; o[4 * c + 1] += w * v.y; o[4 * c + 2] += w * v.z; o[4 * c + 3] += w * v.w;
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    bf16* dst = out + ((size_t)(item.tok0 + tk) * nq + kvh * grp + hbase + h) * HD + blockIdx.y * 16;
#pragma unroll
    for (int c = 0; c < 16; c += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = o[c + j] * inv;
        store8(dst + c, v);
    }
}

extern "C" int vl_flash_prefill_8bit_head_dim() { return HD; }

namespace {
// scratch (may be null: no keys are shared out): SMs * ROWS * (hd + 2) floats from a 16-byte boundary.  q rows and `out` rows begin on 16 bytes; caches
// [pages, nkv, page_size, hd] e4m3, scales [pages, nkv]; pages of any number of positions.
int flash_prefill_8bit(const void* q, int q_stride, void* out, const void* kcache, const void* vcache, const float* kscale,
                       const float* vscale, const int* block_table, int max_blocks, const int* tiles, int num_tiles, int nq, int nkv,
                       int hd, int page_size, int num_pages, float scale, int window, float* scratch, long long floats, unsigned* err, void* stream, int settled) {
    if (num_tiles <= 0) return VL_OK;
    if (hd != HD) return VL_ERR_UNSUPPORTED;
    if (nq <= 0 || nkv <= 0 || nq % nkv || page_size <= 0 || max_blocks <= 0 || num_pages <= 0 || window < 0 || q_stride < nq * hd) return VL_ERR_ARGUMENT;
    if (q_stride % 8 || (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)tiles) & 15)) return VL_ERR_ARGUMENT;
    if (scratch && (((uintptr_t)scratch & 15) || floats < (long long)ROWS * (HD + 2))) return VL_ERR_ARGUMENT;
    if ((long long)num_pages * nkv * page_size >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
    const int grp = nq / nkv, heads = grp < BM ? grp : BM, htiles = (grp + heads - 1) / heads, tokens = BM / heads;
    const int cuts = (128 + GROUPS * tokens - 1) / (GROUPS * tokens);
    if ((long long)num_tiles * cuts > 65535 || (long long)num_tiles * cuts * nkv * htiles >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
    int device, sms;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(flash_tc5_8bit_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
    if (e != cudaSuccess) return (int)e;
    // Keys are shared out where their rows may be long, if at least every second SM would be without a block, or without one in the last of few rounds (three
    // portions of 512 at position 2,500, 184 blocks on 148 SMs: 112 us with every block whole).
    const int in_list = num_tiles * cuts;
    const long long blocks = (long long)in_list * nkv * htiles, reach = (long long)max_blocks * page_size;
    const long long near = (long long)window + GROUPS * tokens, keys = window > 0 && near < reach ? near : reach;
    const bool shared = scratch && keys >= 2 * MIN_PART * BN;
    const int split = shared && in_list <= MOST_ITEMS && 2 * blocks <= sms ? sms : 0, over = (int)(blocks % sms);
    const bool last = shared && blocks > sms && blocks <= MOST_ROUNDS * sms && over && 2 * over <= sms;
    const Tail tail = {(int)(last ? blocks - over : split ? 0 : blocks), last ? sms / over : 0};
    if ((split || last) && floats < (long long)sms * ROWS * (HD + 2)) return VL_ERR_ARGUMENT;
    const Partial partial = {(float4*)scratch, split || last ? (float2*)(scratch + (long long)sms * ROWS * HD) : nullptr};
    cudaStream_t s = (cudaStream_t)stream;
    const int rc = vl_launch_waiting(flash_tc5_8bit_kernel, split ? dim3(sms) : last ? dim3(tail.whole + over * tail.parts) : dim3(nkv * htiles, in_list),
                                     dim3(NTHREADS), SMEM_BYTES, s, (const bf16*)q, q_stride,
                                     (bf16*)out, (const unsigned char*)kcache, (const unsigned char*)vcache, kscale, vscale, block_table, max_blocks,
                                     (const int4*)tiles, num_tiles, nq, nkv, page_size, num_pages, scale * 1.4426950408889634f, window, err, heads, htiles, tokens,
                                     cuts, split, tail, partial, settled);
    if (rc != VL_OK || !(split || last)) return rc;
    return vl_launch_waiting(flash_tc5_8bit_join_kernel, dim3((unsigned)(split ? blocks : over), HD / 16), dim3(ROWS), 0, s, (const int4*)tiles, num_tiles, cuts,
                             tokens, window, nq, nkv, heads, htiles, split, tail, partial, (bf16*)out, settled);
}
}  // namespace

extern "C" int vl_flash_prefill_8bit(const void* q, int q_stride, void* out, const void* kcache, const void* vcache, const float* kscale,
                                     const float* vscale, const int* block_table, int max_blocks, const int* tiles, int num_tiles, int nq, int nkv,
                                     int hd, int page_size, int num_pages, float scale, int window, float* scratch, long long floats, unsigned* err, void* stream) {
    return flash_prefill_8bit(q, q_stride, out, kcache, vcache, kscale, vscale, block_table, max_blocks, tiles, num_tiles, nq, nkv, hd, page_size, num_pages, scale,
                              window, scratch, floats, err, stream, 0);
}
// ... whose tiles and block_table copies brought, not kernels: they are read before the kernels ahead in the stream have ended.
extern "C" int vl_flash_prefill_8bit_settled(const void* q, int q_stride, void* out, const void* kcache, const void* vcache, const float* kscale,
                                             const float* vscale, const int* block_table, int max_blocks, const int* tiles, int num_tiles, int nq, int nkv,
                                             int hd, int page_size, int num_pages, float scale, int window, float* scratch, long long floats, unsigned* err, void* stream) {
    return flash_prefill_8bit(q, q_stride, out, kcache, vcache, kscale, vscale, block_table, max_blocks, tiles, num_tiles, nq, nkv, hd, page_size, num_pages, scale,
                              window, scratch, floats, err, stream, 1);
}
