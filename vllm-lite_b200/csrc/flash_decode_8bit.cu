// Attention of single tokens over a cache in 8 bits (csrc/cache_8bit.cuh), compiled for one head size: -DFA_HD, a multiple of 16 up to 256.
//
//   a token at position p reads the keys lo..p of its request (lo = 0 or p - window + 1), head h those of KV head h / (nq / nkv):
//     s_j = (q . k_j) * sk_j * scale;   p = softmax_j(s);   o = sum_j p_j (v_j * sv_j),
// k_j, v_j e4m3 values, sk_j, sv_j the powers of two of their pages.
//
// Bound by one read of the keys and values, and next by what it takes to bring them from 8 bits to the tensor cores.  Products of 8-bit operands would
// save that, but mma.sync of them is not the tensor cores' own here (18 to 24 instructions each), and tcgen05's smallest tile has 64 rows or more where a token has
// 4 to 16 heads.  So e4m3 values become halves (exactly: cvt.rn.f16x2.e4m3x2, two cycles a warp) and mma.sync m16n8k16 multiplies them.
//
// A warp has a ring of two stages of its own in shared memory, into which it copies rows as they are (cp.async, 16 bytes a lane), a stage ahead: SUB
// tiles of 16 keys' and 16 values' rows, in strides with which no two of a quad's or an eighth's loads meet in a bank.  From there a lane takes 16 bytes
// in a row of each row it needs (features may be dealt out to the lanes in any order as long as queries and keys, or outputs and values, agree).  Two tiles
// side by side give the scheduler two independent chains: with one, rings were no faster than loads straight into registers (decode of 64 requests 74 us), with
// two 67.  Four blocks an SM would spill registers; two of four warps each do not.
//     S^T [16 keys, 8 heads] += K [16, 16] Q^T,      O^T [16 features, 8 heads] += V^T [16, 16 keys] P^T:
// keys and features are the tile's 16 rows, heads its 8 columns: groups of up to 8 query heads cost one such tile, up to 16 two (template NT).  V's rows
// come key by key; bytes of four keys are put side by side by byte permutations (4 for 16 values) before they become halves.  P leaves the
// first product with keys along the lanes and enters the second with heads along them: one movmatrix for 8 keys.
// Roundings to fewer bits: q times a power of two (its largest number lies in [2^14, 2^15), so bfloat16's bits stay down to 2^-28 of
// it) and p sv, as halves.  Sums, maxima and outputs are float32.  p sv is held in units of the largest sv so far, E, times 2^6: a running base
// lets p reach 2^8 before the row is rescaled, so numbers lie below 2^14 and are normal down to 2^-20 of the base's weight (and what lies 2^-31 below the
// largest value that the token reads may vanish).
// The maximum of a warp's keys is looked for only where some score has passed the base by 8 (one vote a tile instead of shuffles).
//
// The keys of all (token, KV head, tile of heads) items, one item behind the other, are cut into runs of equal length in steps of BN keys, one run a block, as many
// runs as blocks are resident at once (two or three rounds of shorter runs: 68 to 74 us where equal runs take 67).  Where items are few, none shares a run with another.  An
// item that lies in one run is finished there, the others leave partial results (numerator, maximum, sum) that the block which
// arrives last at the item's counter adds up in the order of the pieces; where an item's pieces are more than 64 KB a second launch adds them up.
// Where the cuts lie, and with them the last bits of a result, follows from the lengths of all requests and the room for pieces.
//
// Measured in a graph (heads of 128): 64 requests of 400 to 4,096 tokens, 8 KV heads: 67 us, 4.4 TB/s; 8 of 3,500 to 4,096: 19 us (runs that reach into a second item 21); two of 50,000 to
// 65,536 with 16 heads a KV head: 33 us (37); one of 2,800: 10.5 us.  A kernel that reads as many bytes and does nothing else takes 46, 11.5, 20 and 1.9 us.  The rest: some 5 us from the
// launch to the first product (position, table, data: three latencies behind one another), 4 for each further item that a block begins, 3 for the joining.
// Keys outside lo..p, or on pages that the table does not hold (flagged), weigh nothing whatever their bytes and scales are; a page whose scale is not a
// number makes the result NaN where one of its keys is read.
#include "cache_8bit.cuh"

#ifndef FA_HD
#define FA_HD 128
#endif

using namespace cache8;

namespace {
constexpr int HD = FA_HD;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head sizes in steps of 16 up to 256");
constexpr int SUB = HD <= 192 ? 2 : 1, WARPS = 4, BN = 16 * SUB * WARPS;   // a step: SUB tiles of 16 keys a warp
constexpr int NTHREADS = 32 * WARPS, OLD = HD + 4;
constexpr int KW = HD / 16;                            // words (4 features) of a key that a lane takes: lanes t of a quad, piece j -> words (4j + t) KL ..
constexpr int KL = KW % 4 == 0 ? 4 : (KW % 2 == 0 ? 2 : 1);      // words a load
constexpr int VW = HD / 32;                            // ... of a value: lanes g of eight, piece j -> words (8j + g) VL ..
constexpr int VL = VW % 4 == 0 ? 4 : (VW % 2 == 0 ? 2 : 1);
constexpr bool ODD = HD % 32 != 0;                     // and two features more: HD - 16 + 2g
constexpr int OT = HD / 16;                            // tiles of 16 features
constexpr float ROOM = 8.f;                            // log2 of what a weight may exceed the base's by
constexpr int SHIFT = 6;                               // p sv is held times 2^SHIFT
constexpr int MIN_RUN = 2;                             // fewest steps of a run

// A warp's ring: NS stages of 16 keys' rows and 16 values' rows, in strides with which the lanes' loads meet in no bank: a quad of lanes takes
// 16 KL bytes of a key's row side by side, four rows apart in the lanes' groups of eight, and values are taken two rows apart.
constexpr int stride_of(int at_least, int want, int mod) { return at_least % mod == want ? at_least : stride_of(at_least + 16, want, mod); }
constexpr int KS = stride_of(HD, 16 * KL, 128), VS = stride_of(HD, 16, 64), TILE = 16 * (KS + VS), STAGE = SUB * TILE;
constexpr int RESIDENT = 2;                            // blocks an SM
constexpr int NS = 2;
constexpr int PIECES = HD / 16;                        // 16-byte pieces of a row

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(unsigned dst, const void* src, int bytes) {       // bytes 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// N copies of 16 bytes, TO and FROM bytes apart (offsets within the instructions: an addition for each would cost more than the copies)
template <int TO, int FROM, int N, int I = 0> __device__ __forceinline__ void copies16(unsigned dst, const void* src) {
    if constexpr (I < N) {
        asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(I * TO), "n"(I * FROM) : "memory");
        copies16<TO, FROM, N, I + 1>(dst, src);
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void load_words(const unsigned char* p, unsigned* w) {
    if constexpr (N == 4) { const uint4 x = *reinterpret_cast<const uint4*>(p); w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; }
    else if constexpr (N == 2) { const uint2 x = *reinterpret_cast<const uint2*>(p); w[0] = x.x; w[1] = x.y; }
    else w[0] = *reinterpret_cast<const unsigned*>(p);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned turned(unsigned v) {          // an 8 x 8 matrix of halves, rows to columns
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
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
__device__ __forceinline__ int exponent_of(float s) { return (int)(__float_as_uint(s) >> 23) - 127; }

struct Piece { int tok, req, kvh, h0, heads, c0, c1, piece, pieces, item, slot, slot0, stop; };   // heads 0: the end of the run

// Adds up an item's pieces for one head: numerators at part + (slot of piece p) * stride, (maximum, sum) at ml + (slot of piece p) * heads.  The slots: `first`,
// then every second one from `next` on.  A thread takes 4 features at d; 8 pieces' numbers are on their way together.
__device__ __forceinline__ void add_pieces(const float* part, const float2* ml, size_t stride, int heads, int first, int next, int pieces, int d, bf16* dst) {
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = 0; p0 < pieces; p0 += 8) {
        float2 x[8];
        float4 a[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int i = min(p0 + p, pieces - 1);
            const size_t slot = i == 0 ? first : next + 2 * (i - 1);
            x[p] = __ldcg(ml + slot * heads);
            a[p] = __ldcg(reinterpret_cast<const float4*>(part + slot * stride + d));
        }
        float top = M;
#pragma unroll
        for (int p = 0; p < 8; ++p) top = fmaxf(top, x[p].x);
        const float base = top == -INFINITY ? 0.f : top, old = M == -INFINITY ? 1.f : exp2_fast(M - base);
        M = top;
        L *= old;
        acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            if (p0 + p >= pieces) continue;
            const float f = x[p].x == -INFINITY ? 1.f : exp2_fast(x[p].x - base);         // (a piece of NaN keeps its sums)
            L += x[p].y * f;
            acc.x += a[p].x * f; acc.y += a[p].y * f; acc.z += a[p].z * f; acc.w += a[p].w * f;
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    dst[d] = __float2bfloat16(acc.x * inv); dst[d + 1] = __float2bfloat16(acc.y * inv);
    dst[d + 2] = __float2bfloat16(acc.z * inv); dst[d + 3] = __float2bfloat16(acc.w * inv);
}
}  // namespace

// What of the scratch memory holds what: `runs` runs leave two pieces at most (of the item that a run begins in, of the one that it ends in), each of `heads` rows of
// HD numerators; behind them (maximum, sum) of each row; behind those four words for each item.
struct Scratch {
    float* part;
    float2* ml;
    int4* info;                                        // of an item in pieces: slot of the first, of the second, how many (0: none), token
    __host__ __device__ Scratch(float* p, long long runs, int heads)
        : part(p), ml(reinterpret_cast<float2*>(p + 2 * runs * heads * HD)), info(reinterpret_cast<int4*>(p + (2 * runs * heads * (HD + 2) + 3) / 4 * 4)) {}
};

// WIDE: pages of a multiple of 16 positions, so that 16 keys lie on one page.
template <int NT, bool WIDE>
__global__ void __launch_bounds__(NTHREADS, RESIDENT)
flash_decode_8bit_kernel(const bf16* __restrict__ q, int q_stride, const unsigned char* __restrict__ kcache, const unsigned char* __restrict__ vcache,
                         const float* __restrict__ kscale, const float* __restrict__ vscale, const int* __restrict__ block_table, int max_blocks,
                         const int* __restrict__ req_index, const int* __restrict__ positions, int T, int nq, int nkv, int page_size, int num_pages,
                         float scale_log2, int window, int bound, float* scratch, unsigned* err, const int* __restrict__ token_index,
                         bf16* __restrict__ out, int* arrivals, int settled) {      // arrivals null: another launch adds the pieces up
    constexpr int HEADS = 8 * NT;
    extern __shared__ __align__(16) unsigned char smem[];    // the warps' rings; where those are at rest, the warps' shares of a piece
    float (*s_o)[HEADS][OLD] = reinterpret_cast<float (*)[HEADS][OLD]>(smem);
    __shared__ float2 s_scale[WARPS][NS][SUB][WIDE ? 1 : 16];     // scales of a stage's keys and values
    __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS], s_e[WARPS];
    __shared__ int s_scan[WARPS], s_z, s_before, s_last[2];
    __shared__ int s_tok[NTHREADS], s_pos[NTHREADS], s_req[NTHREADS];            // of the launch's first tokens
    __shared__ Piece s_partial[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_launch_dependents();
    if (tid == 0) { s_z = T; s_before = 0; s_partial[0].heads = s_partial[1].heads = 0; }
    if (!settled) pdl_wait();                                // a kernel before this one may be writing the step's description
    const int grp = nq / nkv, htiles = (grp + HEADS - 1) / HEADS, ny = nkv * htiles;
    // the keys [lo, n) of token z (its number within the launch): none for a padded place or a position beyond the bound
    auto keys_of = [&](int z, int* tok, int* lo) -> int {
        const int k = token_index ? (z < NTHREADS ? s_tok[z] : token_index[z]) : z, pos = z < NTHREADS ? s_pos[z] : positions[k];
        if (tok) *tok = k;
        *lo = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
        return pos >= 0 && pos < bound ? pos + 1 : 0;
    };
    if (tid < T) {
        const int k = token_index ? token_index[tid] : tid;
        s_tok[tid] = k;
        s_pos[tid] = positions[k];
        s_req[tid] = req_index[k];
    }
    __syncthreads();
    auto steps_of = [&](int lo, int keys) { return keys > 0 ? (keys - 1) / BN - lo / BN + 1 : 0; };
    // Where this block's run lies: the number of steps, the longest item, and the token in which the run begins.  A round is a token a thread.
    int total = 0;
    auto round = [&](int z0, int& n) -> int {                // steps of token z0 + tid; steps of the tokens up to it
        int lo = 0;
        const int z = z0 + tid, keys = z < T ? keys_of(z, nullptr, &lo) : 0, most = steps_of(lo, keys);
        n = ny * most;
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
        if (lane == 31) s_scan[warp] = x;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < WARPS; ++w) { if (w == warp) x += all; all += s_scan[w]; }
        total += all;
        __syncthreads();
        return total - all + x;
    };
    const int grid = gridDim.x, run = blockIdx.x, held = min(HEADS, grp);                  // held: rows that a piece leaves
    const Scratch left(scratch, grid, held);
    // Few items: no run reaches into a second one (beginning that costs as much as four steps).  An item takes whole runs, the last one of which may be
    // shorter, and a run is as short as there are blocks for: a token a lane, each warp by itself.
    const bool apart = T <= 32 && 2 * T * ny <= grid;
    int per, first, last, z = T, before = 0;                 // the run, the token that it begins in, the steps ahead of that
    auto span_of = [&](int steps) { return apart ? (steps + per - 1) / per * per : steps; };
    if (apart) {
        int lo = 0;
        const int keys = lane < T ? keys_of(lane, nullptr, &lo) : 0, steps = steps_of(lo, keys);
        const int all = __reduce_add_sync(0xffffffffu, ny * steps);
        per = max((all + grid - 1) / grid, MIN_RUN);
        auto runs_of = [&](int length) { return __reduce_add_sync(0xffffffffu, ny * ((steps + length - 1) / length)); };
        if (runs_of(per) > grid)
            for (int enough = all / (grid - T * ny) + 1; per < enough;) {              // (as long, the runs' rounding up is made good)
                const int mid = (per + enough) / 2;
                if (runs_of(mid) <= grid) enough = mid;
                else per = mid + 1;
            }
        const int n = ny * span_of(steps);
        int u = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, u, o); if (lane >= o) u += y; }
        const int end = __shfl_sync(0xffffffffu, u, 31);
        first = min(run * per, end);
        last = min(first + per, end);
        const unsigned here = __ballot_sync(0xffffffffu, u > first && u - n <= first);
        if (here) { z = __ffs(here) - 1; before = __shfl_sync(0xffffffffu, u - n, z); }
    } else {
        int n0 = 0, u0 = 0;                                  // the first round is kept
        for (int z0 = 0; z0 < T; z0 += NTHREADS) {
            int n;
            const int u = round(z0, n);
            if (z0 == 0) { n0 = n; u0 = u; }
        }
        const int all_steps = total;
        per = max((all_steps + grid - 1) / grid, MIN_RUN);
        first = (int)min((long long)run * per, (long long)all_steps);
        last = min(first + per, all_steps);
        total = 0;
        for (int z0 = 0; z0 < T; z0 += NTHREADS) {
            int n = n0, u = u0;
            if (z0 > 0 || T > NTHREADS) u = round(z0, n);
            if (u > first && u - n <= first) { s_z = z0 + tid; s_before = u - n; }
        }
        __syncthreads();
        z = s_z;
        before = s_before;
    }
    pdl_wait();                                              // q and the cache are written by the kernel before
    // the places without keys: rows of zeros, and the ones beyond the bound are flagged
    for (int z = blockIdx.x; z < T; z += grid) {
        int tok, lo;
        if (keys_of(z, &tok, &lo) > 0) continue;
        if (tid == 0 && err && positions[tok] >= 0) atomicOr(err, VL_DEV_BEYOND_BOUND);
        for (int i = tid; i < nq * HD; i += NTHREADS) out[(size_t)tok * nq * HD + i] = __float2bfloat16(0.f);
        if (!arrivals)
            for (int y = tid; y < ny; y += NTHREADS) __stcg(left.info + z * ny + y, make_int4(0, 0, 0, 0));
    }

    auto piece_at = [&](int at) -> Piece {                   // the piece that begins with step `at`: its item's share of this run
        Piece p;
        int lo = 0, keys = 0, tz = 0;
        p.tok = 0;
        p.heads = 0;
        while (at < last && z < T) {
            keys = keys_of(z, &p.tok, &lo);
            tz = steps_of(lo, keys);
            if (at < before + ny * span_of(tz)) break;
            before += ny * span_of(tz);
            ++z;
        }
        if (at >= last || z >= T) return p;
        const int span = span_of(tz), y = (at - before) / span, start = before + y * span, htile = y % htiles;     // the item's first step
        p.req = z < NTHREADS ? s_req[z] : req_index[p.tok];
        p.kvh = y / htiles;
        p.stop = min(last, start + tz);
        p.h0 = p.kvh * grp + htile * HEADS;
        p.heads = min(HEADS, grp - htile * HEADS);
        const int step0 = lo / BN - start;                   // + a step's number in the launch = its number in the request
        p.c0 = max((at + step0) * BN, lo);
        p.c1 = min((p.stop + step0) * BN, keys);
        const int run0 = start / per;
        p.piece = run - run0;
        p.pieces = (start + tz - 1) / per - run0 + 1;
        p.item = z * ny + y;
        p.slot = 2 * run + (at > first ? 1 : 0);             // the item that the run begins in, or the one that it ends in
        p.slot0 = 2 * run0 + (start > run0 * per ? 1 : 0);                 // where its first piece is
        return p;
    };

    bool bad_page = false;
    int at = first;
    for (int number = 0;; ++number) {
        const Piece pc = piece_at(at);
        if (pc.heads == 0) break;
        at = apart ? last : pc.stop;
        const int* table = block_table + (size_t)pc.req * max_blocks;

        float o[NT][OT][4], less[NT][2], l[NT][2];           // less: SHIFT less the base, a maximum of the scores so far
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < OT; ++i) { o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f; }
            less[n][0] = less[n][1] = INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
        int E = EXP_MIN;
        float in_units = power_of_two(-EXP_MIN);             // 2^-E

        unsigned qf[NT][KW][2];
        float qs[NT][2];                                     // scale * log2(e) * what head 2t (+ 1) was divided by
        // the queries as the second operand of S^T: head 8 n + g, the features of this lane's words, as halves
        uint2 raw_q[NT][KW];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const bf16* row = q + (size_t)pc.tok * q_stride + (size_t)(pc.h0 + n * 8 + g) * HD;
                raw_q[n][w] = n * 8 + g < pc.heads ? *reinterpret_cast<const uint2*>(row + ((w / KL * 4 + t) * KL + w % KL) * 4) : make_uint2(0u, 0u);
            }
        auto queries = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint2 (&raw)[KW] = raw_q[n];
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < KW / KL; ++j)
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    const int w = j * KL + i;
                    top = max(top, max(max(raw[w].x & 0x7fffu, (raw[w].x >> 16) & 0x7fffu), max(raw[w].y & 0x7fffu, (raw[w].y >> 16) & 0x7fffu)));
                }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // to [2^14, 2^15); a row of zeros stays as it is, one with a NaN or an infinity has a factor that says so
            const int e = top == 0 ? 0 : max(-112, (int)(top >> 7) - 127 - 14);
            const float f = power_of_two(-e);
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                qf[n][w][0] = pack_half(__uint_as_float(raw[w].x << 16) * f, __uint_as_float(raw[w].x & 0xffff0000u) * f);
                qf[n][w][1] = pack_half(__uint_as_float(raw[w].y << 16) * f, __uint_as_float(raw[w].y & 0xffff0000u) * f);
            }
            const float back = top >= 0x7f80u ? __uint_as_float(0x7fc00000u) : scale_log2 * power_of_two(e);
            qs[n][0] = __shfl_sync(0xffffffffu, back, 8 * t);
            qs[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
        }
        };
        const int st0 = pc.c0 / BN, st1 = (pc.c1 - 1) / BN;
        // a cache row and its page's scales: of the key of this lane (of 16), or, WIDE, of the first key of a step's 16; row < 0: not read
        struct Where { int row; float ks, vs; };
        auto page_of = [&](int key) -> int {                 // -1 for one that is not read
            if (key >= pc.c1 || key + (WIDE ? 15 : 0) < pc.c0) return -1;
            const int blk = key / page_size;
            return blk < max_blocks ? table[blk] : -2;
        };
        auto where_of = [&](int page, int key) -> Where {
            Where w = {-1, 0.f, 0.f};
            if (page == -1 && (key >= pc.c1 || key + (WIDE ? 15 : 0) < pc.c0)) return w;
            if (page < 0 || page >= num_pages) { bad_page = true; return w; }
            const int head = page * nkv + pc.kvh;
            w.row = head * page_size + key % page_size;
            w.ks = kscale[head];
            w.vs = vscale[head];
            return w;
        };
        unsigned char* const ring = smem + warp * NS * STAGE;
        const unsigned ring_u32 = smem_u32(ring);
        // the keys of this warp's tile `tile`, of SUB a step, begin here
        auto first_key = [&](int tile) { return tile / SUB * BN + (warp * SUB + tile % SUB) * 16; };
        auto fetch = [&](const Where& w, int tile, int stage) {  // a tile's keys and values on their way; a row that is not read: zeros
            const int k0 = first_key(tile);
            const unsigned to = ring_u32 + stage * STAGE + tile % SUB * TILE;
            constexpr int COPIES = (16 * PIECES + 31) / 32;
            const bool whole = WIDE && w.row >= 0 && k0 >= pc.c0 && k0 + 16 <= pc.c1;             // (warp-uniform)
            if (whole) {                                     // 16 rows of a page lie side by side
                const unsigned char* const k = kcache + (size_t)w.row * HD + lane * 16;
                const unsigned char* const v = vcache + (size_t)w.row * HD + lane * 16;
                if constexpr (PIECES > 1 && 32 % PIECES == 0) {            // 32 / PIECES rows a round (one piece a row leaves half of the lanes without)
                    copies16<32 / PIECES * KS, 512, COPIES>(to + lane / PIECES * KS + lane % PIECES * 16, k);
                    copies16<32 / PIECES * VS, 512, COPIES>(to + 16 * KS + lane / PIECES * VS + lane % PIECES * 16, v);
                } else {
#pragma unroll
                    for (int j = 0; j < COPIES; ++j) {
                        const int i = j * 32 + lane, r = i / PIECES, c = i - r * PIECES;
                        if (16 * PIECES % 32 && i >= 16 * PIECES) continue;
                        copies16<0, 0, 1>(to + r * KS + c * 16, k + j * 512);
                        copies16<0, 0, 1>(to + 16 * KS + r * VS + c * 16, v + j * 512);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < COPIES; ++j) {
                    const int i = j * 32 + lane, r = i / PIECES, c = i - r * PIECES;
                    const int first_row = WIDE ? w.row : __shfl_sync(0xffffffffu, w.row, r & 15), row = WIDE ? first_row + r : first_row;
                    if (16 * PIECES % 32 && i >= 16 * PIECES) continue;
                    const int bytes = first_row >= 0 && k0 + r >= pc.c0 && k0 + r < pc.c1 ? 16 : 0;
                    const size_t at = (size_t)max(row, 0) * HD + c * 16;
                    copy16(to + r * KS + c * 16, kcache + at, bytes);
                    copy16(to + 16 * KS + r * VS + c * 16, vcache + at, bytes);
                }
            }
        };
        // values under a scale that is none: their keys' scores say so, so that only who reads them gets NaN
        auto note = [&](const Where& w, int u, int stage) {
            if (lane < (WIDE ? 1 : 16)) s_scale[warp][stage][u][lane] = w.vs != w.vs ? make_float2(w.vs, 0.f) : make_float2(w.ks, w.vs);
        };
        // The step's tiles side by side, so that one's chain of products, exponentials and conversions runs beside another's.  (One code for steps with and without
        // keys that are not read: with one for each, layers of a step took 0.3 us more, for what the comparisons save.)
        auto work = [&](int st, int stage) {
            const unsigned char* const keys = ring + stage * STAGE + g * KS + t * KL * 4;
            const unsigned char* const values = ring + stage * STAGE + 16 * KS + 2 * t * VS + g * VL * 4;
            float2 scale0[SUB], scale1[SUB];
            float s[SUB][NT][4], x[SUB][NT][4], top = -INFINITY;
            bool none0[SUB], none1[SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                scale0[u] = s_scale[warp][stage][u][WIDE ? 0 : g];
                scale1[u] = WIDE ? scale0[u] : s_scale[warp][stage][u][WIDE ? 0 : g + 8];
                unsigned k[2][KW];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < KW / KL; ++j) load_words<KL>(keys + u * TILE + i * 8 * KS + j * 16 * KL, &k[i][j * KL]);
                float odd[NT][4];                            // two chains a tile
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[u][n][c] = odd[n][c] = 0.f;
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    const unsigned a0 = half2_low(k[0][i]), a1 = half2_low(k[1][i]), a2 = half2_high(k[0][i]), a3 = half2_high(k[1][i]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(i & 1 ? odd[n] : s[u][n], a0, a1, a2, a3, qf[n][i][0], qf[n][i][1]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) s[u][n][c] += odd[n][c];
            }
            // a score less its base, in units of log2, and SHIFT more: what the halves of the weights are the powers of
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const int k0 = st * BN + (warp * SUB + u) * 16;
                // keys that are not read weigh nothing: those outside the piece, and those without a page, whose scale is left 0
                none0[u] = scale0[u].x == 0.f || k0 + g < pc.c0 || k0 + g >= pc.c1;
                none1[u] = scale1[u].x == 0.f || k0 + g + 8 < pc.c0 || k0 + g + 8 >= pc.c1;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        x[u][n][c] = fmaf(s[u][n][c], (c < 2 ? scale0[u].x : scale1[u].x) * qs[n][c & 1], less[n][c & 1]);
                        if (c < 2 ? none0[u] : none1[u]) x[u][n][c] = -INFINITY;
                        top = fmaxf(top, x[u][n][c]);        // (no base yet: +inf)
                    }
            }
            int tile_e = -128;
#pragma unroll
            for (int u = 0; u < SUB; ++u) tile_e = max(tile_e, max(exponent_of(scale0[u].y), exponent_of(scale1[u].y)));
            if (!WIDE) tile_e = __reduce_max_sync(0xffffffffu, tile_e);
            if (__any_sync(0xffffffffu, top > ROOM + SHIFT) || tile_e > E) {
                const int grown = max(E, tile_e);
                const float lower = power_of_two(E - grown);
                E = grown;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float was = SHIFT - less[n][c];
                        float mx = was, sc[SUB][2];
#pragma unroll
                        for (int u = 0; u < SUB; ++u) {
                            sc[u][0] = none0[u] ? -INFINITY : s[u][n][c] * (scale0[u].x * qs[n][c]);
                            sc[u][1] = none1[u] ? -INFINITY : s[u][n][c + 2] * (scale1[u].x * qs[n][c]);
                            mx = fmaxf(mx, fmaxf(sc[u][0], sc[u][1]));
                        }
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float corr = mx == -INFINITY ? 1.f : exp2_fast(was - mx), both = corr * lower, base = mx == -INFINITY ? 0.f : mx;
                        less[n][c] = SHIFT - mx;
                        l[n][c] *= corr;
#pragma unroll
                        for (int u = 0; u < SUB; ++u) {
                            x[u][n][c] = sc[u][0] - base + SHIFT;
                            x[u][n][c + 2] = sc[u][1] - base + SHIFT;
                        }
#pragma unroll
                        for (int i = 0; i < OT; ++i) { o[n][i][c] *= both; o[n][i][c + 2] *= both; }
                    }
                in_units = power_of_two(-E);
            }
            unsigned pf[SUB][NT][2];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const float f0 = scale0[u].y * in_units, f1 = scale1[u].y * in_units;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float p[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) p[c] = exp2_fast(x[u][n][c]);
                    l[n][0] += p[0] + p[2];
                    l[n][1] += p[1] + p[3];
                    pf[u][n][0] = turned(pack_half(p[0] * f0, p[1] * f0));
                    pf[u][n][1] = turned(pack_half(p[2] * f1, p[3] * f1));
                }
            }
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
#pragma unroll
                for (int j = 0; j < VW / VL; ++j) {
                    unsigned v[4][VL];
#pragma unroll
                    for (int i = 0; i < 4; ++i) load_words<VL>(values + u * TILE + ((i & 1) + 8 * (i >> 1)) * VS + j * 32 * VL, v[i]);
#pragma unroll
                    for (int c = 0; c < VL; ++c) {
                        const int i = j * VL + c;
                        const unsigned lo01 = __byte_perm(v[0][c], v[1][c], 0x5140), hi01 = __byte_perm(v[0][c], v[1][c], 0x7362);
                        const unsigned lo23 = __byte_perm(v[2][c], v[3][c], 0x5140), hi23 = __byte_perm(v[2][c], v[3][c], 0x7362);
                        const unsigned a0 = half2_low(lo01), a1 = half2_high(lo01), a2 = half2_low(lo23), a3 = half2_high(lo23);
                        const unsigned c0 = half2_low(hi01), c1 = half2_high(hi01), c2 = half2_low(hi23), c3 = half2_high(hi23);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_f16(o[n][2 * i], a0, a1, a2, a3, pf[u][n][0], pf[u][n][1]);
                            mma_f16(o[n][2 * i + 1], c0, c1, c2, c3, pf[u][n][0], pf[u][n][1]);
                        }
                    }
                }
                if constexpr (ODD) {
                    unsigned v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        v[i] = *reinterpret_cast<const unsigned short*>(values + u * TILE + ((i & 1) + 8 * (i >> 1)) * VS - g * VL * 4 + HD - 16 + 2 * g);
                    const unsigned lo01 = __byte_perm(v[0], v[1], 0x5140), lo23 = __byte_perm(v[2], v[3], 0x5140);
                    const unsigned a0 = half2_low(lo01), a1 = half2_high(lo01), a2 = half2_low(lo23), a3 = half2_high(lo23);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(o[n][OT - 1], a0, a1, a2, a3, pf[u][n][0], pf[u][n][1]);
                }
            }
        };
        if constexpr (WIDE) {
            // lane i knows the place of tile base + i; the next 32 tiles' are looked up on the way, a load at a time
            Where now = where_of(page_of(first_key(st0 * SUB + lane)), first_key(st0 * SUB + lane)), then = {-1, 0.f, 0.f};
            int from = 0, base = st0 * SUB, page = -1;
            auto ask = [&](int stage) {                      // the step that begins with tile base + from
#pragma unroll
                for (int u = 0; u < SUB; ++u) fetch(Where{__shfl_sync(0xffffffffu, now.row, from + u), 0.f, 0.f}, base + from + u, stage);
                copies_commit();
            };
            auto tell = [&](int stage) {                     // its scales
#pragma unroll
                for (int u = 0; u < SUB; ++u) note(Where{0, __shfl_sync(0xffffffffu, now.ks, from + u), __shfl_sync(0xffffffffu, now.vs, from + u)}, u, stage);
            };
            auto advance = [&]() {
                if (from == 8) page = page_of(first_key(base + 32 + lane));
                if (from == 20) then = where_of(page, first_key(base + 32 + lane));
                from += SUB;
                if (from == 32) { now = then; base += 32; from = 0; }
            };
            ask(0);
            queries();                                       // (while the first keys and their scales are on their way)
            tell(0);
            advance();
            int stage = 0;
            for (int st = st0; st <= st1; ++st, stage ^= 1) {
                ask(stage ^ 1);
                tell(stage ^ 1);
                advance();
                copies_wait<1>();
                __syncwarp();                                // every lane's copies have landed
                work(st, stage);
                __syncwarp();                                // the stage has been read
            }
        } else {
            auto find = [&](int tile) { return where_of(page_of(first_key(tile) + (lane & 15)), first_key(tile) + (lane & 15)); };
            Where w[SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) { w[u] = find(st0 * SUB + u); fetch(w[u], st0 * SUB + u, 0); note(w[u], u, 0); }
            copies_commit();
#pragma unroll
            for (int u = 0; u < SUB; ++u) w[u] = find((st0 + 1) * SUB + u);
            queries();
            int stage = 0;
            for (int st = st0; st <= st1; ++st, stage ^= 1) {
#pragma unroll
                for (int u = 0; u < SUB; ++u) { fetch(w[u], (st + 1) * SUB + u, stage ^ 1); note(w[u], u, stage ^ 1); }
                copies_commit();
#pragma unroll
                for (int u = 0; u < SUB; ++u) w[u] = find((st + 2) * SUB + u);             // (used a step later)
                copies_wait<1>();
                __syncwarp();
                work(st, stage);
                __syncwarp();
            }
        }
        copies_wait<0>();
        __syncthreads();                                     // all rings are at rest

        // the four warps' shares, put together in warp order
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[n][c];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) { s_m[warp][n * 8 + 2 * t + c] = SHIFT - less[n][c]; s_l[warp][n * 8 + 2 * t + c] = x; }
            }
        if (lane == 0) s_e[warp] = power_of_two(E);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float* row = &s_o[warp][n * 8 + 2 * t + c][0];
#pragma unroll
                for (int w = 0; w < VW; ++w)
                    *reinterpret_cast<float4*>(row + (((w / VL) * 8 + g) * VL + w % VL) * 4) =
                        make_float4(o[n][2 * w][c], o[n][2 * w][c + 2], o[n][2 * w + 1][c], o[n][2 * w + 1][c + 2]);
                if constexpr (ODD) *reinterpret_cast<float2*>(row + HD - 16 + 2 * g) = make_float2(o[n][OT - 1][c], o[n][OT - 1][c + 2]);
            }
        __syncthreads();
        for (int i = tid; i < pc.heads * (HD / 4); i += NTHREADS) {
            const int h = i / (HD / 4), d = (i - h * (HD / 4)) * 4;
            float M = -INFINITY, L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w][h]);
            const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {                // (a warp without a key has sums of zero; one of NaN keeps them)
                const float f = s_m[w][h] == -INFINITY ? 1.f : exp2_fast(s_m[w][h] - base), e = s_e[w];
                const float4 x = *reinterpret_cast<const float4*>(&s_o[w][h][d]);
                acc.x += x.x * f * e; acc.y += x.y * f * e; acc.z += x.z * f * e; acc.w += x.w * f * e;
                L += s_l[w][h] * f;
            }
            if (pc.pieces == 1) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                bf16* dst = out + ((size_t)pc.tok * nq + pc.h0 + h) * HD + d;
                dst[0] = __float2bfloat16(acc.x * inv); dst[1] = __float2bfloat16(acc.y * inv);
                dst[2] = __float2bfloat16(acc.z * inv); dst[3] = __float2bfloat16(acc.w * inv);
            } else {
                const size_t row = (size_t)pc.slot * held + h;
                __stcg(reinterpret_cast<float4*>(left.part + row * HD + d), acc);
                if (d == 0) __stcg(left.ml + row, make_float2(M, L));
            }
        }
        if (tid == 0) {
            if (pc.pieces > 1) s_partial[number > 0] = pc;
            if (!arrivals && pc.piece == 0)
                __stcg(left.info + pc.item, make_int4(pc.slot0, 2 * (run + 1), pc.pieces > 1 ? pc.pieces : 0, pc.tok));
        }
        __syncthreads();                                     // the shares may be written again
    }
    if (bad_page && err) atomicOr(err, VL_DEV_BAD_PAGE);
    // The items shared with other blocks (the run's first and last), at its end so that the stream does not wait for them: this block's pieces are
    // counted; whoever comes last adds up all of an item's, in their order.
    if (!arrivals || (s_partial[0].heads == 0 && s_partial[1].heads == 0)) return;
    __threadfence();                                         // this thread's parts, before the block's arrivals are counted
    __syncthreads();
    if (tid < 2) s_last[tid] = s_partial[tid].heads && atomicAdd(&arrivals[s_partial[tid].item], 1) == s_partial[tid].pieces - 1;
    __syncthreads();
    if (!s_last[0] && !s_last[1]) return;
    __threadfence();
    for (int k = 0; k < 2; ++k) {
        if (!s_last[k]) continue;
        const Piece pc = s_partial[k];
        const int run0 = run - pc.piece, slot0 = pc.slot0;
        for (int i = tid; i < pc.heads * (HD / 4); i += NTHREADS) {
            const int h = i / (HD / 4);
            add_pieces(left.part + (size_t)h * HD, left.ml + h, (size_t)held * HD, held, slot0, 2 * (run0 + 1), pc.pieces, (i - h * (HD / 4)) * 4,
                       out + ((size_t)pc.tok * nq + pc.h0 + h) * HD);
        }
        if (tid == 0) arrivals[pc.item] = 0;               // as the next launch finds it
    }
}

// The pieces of one head of one item, where a block of the launch above would take longer over all of an item's.
__global__ void __launch_bounds__(HD / 4 < 32 ? 32 : HD / 4)
flash_decode_8bit_merge_kernel(float* scratch, int runs, int held, int grp, int nq, int nkv, bf16* __restrict__ out) {
    pdl_launch_dependents();
    pdl_wait();
    const Scratch left(scratch, runs, held);
    const int htiles = (grp + held - 1) / held, item = blockIdx.x / held, h = blockIdx.x % held, y = item % (nkv * htiles);
    const int head = (y % htiles) * held + h;                // within the KV head's group
    if ((int)threadIdx.x >= HD / 4 || head >= grp) return;
    const int4 info = __ldcg(left.info + item);
    if (info.z == 0) return;
    add_pieces(left.part + (size_t)h * HD, left.ml + h, (size_t)held * HD, held, info.x, info.y, info.z, (int)threadIdx.x * 4,
               out + ((size_t)info.w * nq + (y / htiles) * grp + head) * HD);
}

extern "C" int vl_flash_decode_8bit_head_dim() { return HD; }

// q [T, q_stride] bfloat16, out [.., nq * hd]; caches [pages, nkv, page_size, hd] e4m3, scales [pages, nkv]; positions from `bound` on are
// flagged and get rows of zeros; it is 2^30 at most.  scratch: `floats` of them, the more the shorter the runs may be, 3 * T * nq * (hd + 2) at least; arrivals: T * nq counters, zero
// before and after.
extern "C" int vl_flash_decode_8bit(const void* q, int q_stride, const void* kcache, const void* vcache, const float* kscale, const float* vscale,
                                    const int* block_table, int max_blocks, const int* req_index, const int* positions, int T, int nq, int nkv, int hd,
                                    int page_size, int num_pages, float scale, int window, int bound, float* scratch, long long floats, unsigned* err,
                                    const int* token_index, void* out, int* arrivals, int settled, void* stream) {
    if (T <= 0) return VL_OK;
    if (hd != HD) return VL_ERR_UNSUPPORTED;
    if (nq <= 0 || nkv <= 0 || nq % nkv || page_size <= 0 || max_blocks <= 0 || num_pages <= 0 || q_stride < nq * hd || q_stride % 4) return VL_ERR_ARGUMENT;
    if (bound <= 0 || !out || !arrivals || !scratch) return VL_ERR_ARGUMENT;
    if (((uintptr_t)q & 7) || (((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)scratch) & 15)) return VL_ERR_ARGUMENT;
    const int grp = nq / nkv, wide_heads = grp > 8 && HD <= 128 ? 16 : 8, htiles = (grp + wide_heads - 1) / wide_heads;
    const long long most = (long long)T * nkv * htiles * ((bound - 1) / BN + 1);
    if (bound > (1 << 30)) return VL_ERR_UNSUPPORTED;        // (positions, rounded up to steps, are whole numbers of 32 bits)
    if ((long long)num_pages * nkv * page_size >= (1ll << 31) || most >= (1ll << 30)) return VL_ERR_UNSUPPORTED;
    if (floats < 3ll * T * nq * (hd + 2)) return VL_ERR_ARGUMENT;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return (int)e;
    const bool wide = page_size % 16 == 0;
    const int held = grp < wide_heads ? grp : wide_heads;
    const long long items = (long long)T * nkv * htiles, reach = window > 0 && window < bound ? window + BN : bound, steps = (reach + BN - 1) / BN;
    auto launch = [&](auto kernel) {
        const long long resident = (long long)sms * RESIDENT;
        long long runs = (floats - 8 - 4 * items) / (2ll * held * (HD + 2));
        if (runs > resident) runs = resident;
        if (runs > sms) runs -= runs % sms;                  // as many on every SM
        if (runs > most) runs = most;
        if (runs < 1) runs = 1;
        // pieces that an item may come in, were every place full, and what a block would read to add them up: above 64 KB another launch, a block a head, does
        const long long run = (most + resident - 1) / resident > MIN_RUN ? (most + resident - 1) / resident : MIN_RUN, pieces = (steps + run - 1) / run + 1;
        const bool apart = pieces * held * HD * 4 > 64 * 1024;
        const int rings = WARPS * NS * STAGE, shares = WARPS * wide_heads * OLD * 4, smem = rings > shares ? rings : shares;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
        // (unless it may read the step's description early it touches no memory before its wait)
        int rc = vl_launch_as(settled ? vl_pdl_enabled() : !vl_pdl_forbidden(), kernel, dim3((unsigned)runs), dim3(NTHREADS), (size_t)smem, (cudaStream_t)stream, (const bf16*)q, q_stride,
                           (const unsigned char*)kcache, (const unsigned char*)vcache, kscale, vscale, block_table, max_blocks, req_index, positions, T,
                           nq, nkv, page_size, num_pages, scale * 1.4426950408889634f, window, bound, scratch, err, token_index, (bf16*)out,
                           apart ? (int*)nullptr : arrivals, settled);
        if (rc == VL_OK && apart)
            rc = vl_launch_waiting(flash_decode_8bit_merge_kernel, dim3((unsigned)(items * held)), dim3(HD / 4 < 32 ? 32 : HD / 4), 0, (cudaStream_t)stream, scratch,
                           (int)runs, held, grp, nq, nkv, (bf16*)out);
        return rc;
    };
    if constexpr (HD <= 128) {
        if (wide_heads == 16) return wide ? launch(flash_decode_8bit_kernel<2, true>) : launch(flash_decode_8bit_kernel<2, false>);
    }
    return wide ? launch(flash_decode_8bit_kernel<1, true>) : launch(flash_decode_8bit_kernel<1, false>);
}
