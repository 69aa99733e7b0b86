// Attention of single tokens over a cache in 8 bits (csrc/cache_8bit.cuh), compiled for one head size: -DFA_HD, a multiple of 16 up to 256.
//
//   a token at position p reads the keys lo..p of its request (lo = 0 or p - window + 1), head h those of KV head h / (nq / nkv):
//     s_j = (q . k_j) * sk_j * scale;   p = softmax_j(s);   o = sum_j p_j (v_j * sv_j),
// k_j, v_j e4m3 values, sk_j, sv_j the powers of two of their pages.
//
// Bound by one read of the keys and values, and next by what it takes to bring them from 8 bits to the tensor cores.  No shared memory and no
// copies on the way: a warp loads 16 keys' rows and 16 values' rows straight into the registers that mma.sync m16n8k16 wants them in, the next 16
// while these are worked on, and a lane's share of a row is 16 bytes in a row (features may be dealt out to the lanes in any order as long as
// queries and keys, or outputs and values, agree).  e4m3 values are halves exactly (cvt.rn.f16x2.e4m3x2), so the products are of halves:
//     S^T [16 keys, 8 heads] += K [16, 16] Q^T,      O^T [16 features, 8 heads] += V^T [16, 16 keys] P^T:
// keys and features are the tile's 16 rows, heads its 8 columns: groups of up to 8 query heads cost one such tile, up to 16 two (template NT).  V's rows
// come key by key; bytes of four keys are put side by side by byte permutations (4 for 16 values) before they become halves.  P leaves the
// first product with keys along the lanes and enters the second with heads along them: one movmatrix for 8 keys.
// Roundings to fewer bits: q times a power of two (its largest number lies in [2^14, 2^15), so bfloat16's bits stay down to 2^-28 of
// it) and p sv, as halves.  Sums, maxima and outputs are float32.  p sv is held in units of the largest sv so far, E, times 2^6: a running base
// lets p reach 2^8 before the row is rescaled, so numbers lie below 2^14 and are normal down to 2^-20 of the base's weight.
// The maximum of a warp's keys is looked for only where some score has passed the base by 8 (one vote a tile instead of shuffles).
//
// The keys of all (token, KV head, tile of heads) items, one item behind the other, are cut into runs of equal length in steps of 64 keys, one run a block; an
// item that lies in one run is finished there, the others leave partial results (numerator, maximum, sum) that the block which
// arrives last at the item's counter adds up in the order of the pieces.  Where the cuts lie, and with them the last bits of a result, follows from the
// lengths of all requests and the room for pieces.
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
constexpr int BN = 64, WARPS = 4, NTHREADS = 32 * WARPS;
constexpr int KW = HD / 16;                            // words (4 features) of a key that a lane takes: lanes t of a quad, piece j -> words (4j + t) KL ..
constexpr int KL = KW % 4 == 0 ? 4 : (KW % 2 == 0 ? 2 : 1);      // words a load
constexpr int VW = HD / 32;                            // ... of a value: lanes g of eight, piece j -> words (8j + g) VL ..
constexpr int VL = VW % 4 == 0 ? 4 : (VW % 2 == 0 ? 2 : 1);
constexpr bool ODD = HD % 32 != 0;                     // and two features more: HD - 16 + 2g
constexpr int OT = HD / 16;                            // tiles of 16 features
constexpr float ROOM = 8.f;                            // log2 of what a weight may exceed the base's by
constexpr int SHIFT = 6;                               // p sv is held times 2^SHIFT
constexpr int AHEAD = 4;                               // steps whose keys and values are asked for into L2 ahead of their loads
constexpr int PIECES_MAX = 4 * (HD + 4) < 302 ? 4 * (HD + 4) : 302;     // most pieces of an item: a weight a head and piece in the room of s_o
constexpr int MIN_RUN = 2;                             // fewest steps of a run

struct Tile { unsigned k[2][KW], v[4][VW > 0 ? VW : 1]; unsigned short v2[4]; };

template <int N> __device__ __forceinline__ void load_words(const unsigned char* p, unsigned* w) {
    if constexpr (N == 4) { const uint4 x = __ldg(reinterpret_cast<const uint4*>(p)); w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; }
    else if constexpr (N == 2) { const uint2 x = __ldg(reinterpret_cast<const uint2*>(p)); w[0] = x.x; w[1] = x.y; }
    else w[0] = __ldg(reinterpret_cast<const unsigned*>(p));
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
__device__ __forceinline__ void prefetch_l2(const void* p, unsigned bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ int exponent_of(float s) { return (int)(__float_as_uint(s) >> 23) - 127; }

struct Piece { int tok, place, kvh, h0, heads, c0, c1, piece, pieces, counter, stop; };   // heads 0: the end of the run
}  // namespace

// WIDE: pages of a multiple of 16 positions, so that 16 keys lie on one page.
template <int NT, bool WIDE>
__global__ void __launch_bounds__(NTHREADS, NT == 1 && HD <= 128 ? 3 : 2)
flash_decode_8bit_kernel(const bf16* __restrict__ q, int q_stride, const unsigned char* __restrict__ kcache, const unsigned char* __restrict__ vcache,
                         const float* __restrict__ kscale, const float* __restrict__ vscale, const int* __restrict__ block_table, int max_blocks,
                         const int* __restrict__ req_index, const int* __restrict__ positions, int T, int nq, int nkv, int page_size, int num_pages,
                         float scale_log2, int window, int bound, int S, float* __restrict__ part, unsigned* err, const int* __restrict__ token_index,
                         bf16* __restrict__ out, int* arrivals, int settled) {
    constexpr int HEADS = 8 * NT;
    constexpr int OLD = HD + 4;
    __shared__ __align__(16) float s_o[WARPS][HEADS][OLD];
    __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS], s_e[WARPS];
    __shared__ int s_scan[WARPS], s_most, s_z, s_before, s_last[2];
    __shared__ Piece s_partial[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    float* const part_ml = part + (size_t)T * nq * S * HD;   // behind the numerators: (maximum, sum) of each
    pdl_launch_dependents();
    if (tid == 0) { s_most = 0; s_z = T; s_before = 0; s_partial[0].heads = s_partial[1].heads = 0; }
    if (!settled) pdl_wait();                                // a kernel before this one may be writing the step's description
    __syncthreads();
    const int grp = nq / nkv, htiles = (grp + HEADS - 1) / HEADS, ny = nkv * htiles;
    // the keys [lo, n) of token z (its number within the launch): none for a padded place or a position beyond the bound
    auto keys_of = [&](int z, int* tok, int* lo) -> int {
        const int k = token_index ? token_index[z] : z, pos = positions[k];
        if (tok) *tok = k;
        *lo = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
        return pos >= 0 && pos < bound ? pos + 1 : 0;
    };
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
        const int longest = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) atomicMax(&s_most, longest);
        if (lane == 31) s_scan[warp] = x;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < WARPS; ++w) { if (w == warp) x += all; all += s_scan[w]; }
        total += all;
        __syncthreads();
        return total - all + x;
    };
    int n0 = 0, u0 = 0;                                      // the first round is kept
    for (int z0 = 0; z0 < T; z0 += NTHREADS) {
        int n;
        const int u = round(z0, n);
        if (z0 == 0) { n0 = n; u0 = u; }
    }
    // (a run as long as S allows leaves no item in more than S runs)
    const int grid = gridDim.x, all_steps = total;
    const int per = max(max((all_steps + grid - 1) / grid, MIN_RUN), (s_most + S - 2) / (S - 1));
    const int first = (int)min((long long)blockIdx.x * per, (long long)all_steps), last = (int)min((long long)first + per, (long long)all_steps);
    total = 0;
    for (int z0 = 0; z0 < T; z0 += NTHREADS) {
        int n = n0, u = u0;
        if (z0 > 0 || T > NTHREADS) u = round(z0, n);
        if (u > first && u - n <= first) { s_z = z0 + tid; s_before = u - n; }
    }
    __syncthreads();
    pdl_wait();                                              // q and the cache are written by the kernel before
    // the places without keys: rows of zeros, and the ones beyond the bound are flagged
    for (int z = blockIdx.x; z < T; z += grid) {
        int tok, lo;
        if (keys_of(z, &tok, &lo) > 0) continue;
        if (tid == 0 && err && positions[tok] >= 0) atomicOr(err, VL_DEV_BEYOND_BOUND);
        for (int i = tid; i < nq * HD; i += NTHREADS) out[(size_t)tok * nq * HD + i] = __float2bfloat16(0.f);
    }

    int z = s_z, before = s_before;
    auto piece_at = [&](int at) -> Piece {                   // the piece that begins with step `at`: its item's share of this run
        Piece p;
        int lo = 0, keys = 0, tz = 0;
        p.tok = 0;
        p.heads = 0;
        while (at < last && z < T) {
            keys = keys_of(z, &p.tok, &lo);
            tz = steps_of(lo, keys);
            if (at < before + ny * tz) break;
            before += ny * tz;
            ++z;
        }
        if (at >= last || z >= T) return p;
        const int y = (at - before) / tz, start = before + y * tz, htile = y % htiles;       // the item's first step
        p.kvh = y / htiles;
        p.place = z;
        p.stop = min(last, start + tz);
        p.h0 = p.kvh * grp + htile * HEADS;
        p.heads = min(HEADS, grp - htile * HEADS);
        const int step0 = lo / BN - start;                   // + a step's number in the launch = its number in the request
        p.c0 = max((at + step0) * BN, lo);
        p.c1 = min((p.stop + step0) * BN, keys);
        p.piece = (int)blockIdx.x - start / per;
        p.pieces = (start + tz - 1) / per - start / per + 1;
        p.counter = z * ny + y;
        return p;
    };

    bool bad_page = false;
    int at = first;
    for (int number = 0;; ++number) {
        const Piece pc = piece_at(at);
        if (pc.heads == 0) break;
        at = pc.stop;
        const int* table = block_table + (size_t)req_index[pc.tok] * max_blocks;

        // the queries as the second operand of S^T: head n0 + g, the features of this lane's words
        unsigned qf[NT][KW][2];
        float qs[NT][2];                                     // scale * log2(e) * what head 2t (+ 1) was divided by
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int h = n * 8 + g;
            const bf16* row = q + (size_t)pc.tok * q_stride + (size_t)(pc.h0 + h) * HD;
            uint2 raw[KW];
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < KW / KL; ++j)
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    const int w = j * KL + i;
                    raw[w] = h < pc.heads ? *reinterpret_cast<const uint2*>(row + ((j * 4 + t) * KL + i) * 4) : make_uint2(0u, 0u);
                    top = max(top, max(max(raw[w].x & 0x7fffu, (raw[w].x >> 16) & 0x7fffu), max(raw[w].y & 0x7fffu, (raw[w].y >> 16) & 0x7fffu)));
                }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // to [2^14, 2^15); a row of zeros, a NaN or an infinity stays as it is
            const int e = top == 0 || top >= 0x7f80u ? 0 : max(-112, (int)(top >> 7) - 127 - 14);
            const float f = power_of_two(-e);
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                qf[n][w][0] = pack_half(__uint_as_float(raw[w].x << 16) * f, __uint_as_float(raw[w].x & 0xffff0000u) * f);
                qf[n][w][1] = pack_half(__uint_as_float(raw[w].y << 16) * f, __uint_as_float(raw[w].y & 0xffff0000u) * f);
            }
            const float back = scale_log2 * power_of_two(e);
            qs[n][0] = __shfl_sync(0xffffffffu, back, 8 * t);
            qs[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
        }

        float o[NT][OT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < OT; ++i) { o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f; }
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
        int E = EXP_MIN;

        // this warp's 16 keys of step st begin at st * 64 + warp * 16
        const int st0 = pc.c0 / BN, st1 = (pc.c1 - 1) / BN;
        // the cache row and the scales of key `lane` (of 16; WIDE: of the first one) of a step's keys: row < 0 for one that is not read
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
        // values under a scale that is none: their keys' scores say so, so that only who reads them gets NaN
        auto settle = [&](Where w) -> Where {
            if (w.vs != w.vs) { w.ks = w.vs; w.vs = 0.f; }
            return w;
        };
        auto ask = [&](int row) {                            // 16 keys' rows and their values' into L2
            if (row >= 0) { prefetch_l2(kcache + (size_t)row * HD, 16 * HD); prefetch_l2(vcache + (size_t)row * HD, 16 * HD); }
        };
        auto load = [&](Tile& x, const Where& w) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = WIDE ? (w.row < 0 ? -1 : w.row + g + 8 * i) : __shfl_sync(0xffffffffu, w.row, g + 8 * i);
                const unsigned char* p = kcache + (size_t)max(row, 0) * HD;
#pragma unroll
                for (int j = 0; j < KW / KL; ++j) {
                    if (row >= 0) load_words<KL>(p + (j * 4 + t) * KL * 4, &x.k[i][j * KL]);
                    else {
#pragma unroll
                        for (int c = 0; c < KL; ++c) x.k[i][j * KL + c] = 0u;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * t + (i & 1) + 8 * (i >> 1);
                const int row = WIDE ? (w.row < 0 ? -1 : w.row + key) : __shfl_sync(0xffffffffu, w.row, key);
                const unsigned char* p = vcache + (size_t)max(row, 0) * HD;
                if constexpr (VW > 0) {
#pragma unroll
                    for (int j = 0; j < VW / VL; ++j) {
                        if (row >= 0) load_words<VL>(p + (j * 8 + g) * VL * 4, &x.v[i][j * VL]);
                        else {
#pragma unroll
                            for (int c = 0; c < VL; ++c) x.v[i][j * VL + c] = 0u;
                        }
                    }
                }
                if constexpr (ODD) x.v2[i] = row >= 0 ? __ldg(reinterpret_cast<const unsigned short*>(p + HD - 16 + 2 * g)) : (unsigned short)0;
            }
        };
        auto work = [&](Tile& x, const Where& w, int st) {
            const int k0 = st * BN + warp * 16;              // the tile's first key
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f; }
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const unsigned a0 = half2_low(x.k[0][i]), a2 = half2_high(x.k[0][i]), a1 = half2_low(x.k[1][i]), a3 = half2_high(x.k[1][i]);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(s[n], a0, a1, a2, a3, qf[n][i][0], qf[n][i][1]);
            }
            const float ks0 = WIDE ? w.ks : __shfl_sync(0xffffffffu, w.ks, g), ks1 = WIDE ? w.ks : __shfl_sync(0xffffffffu, w.ks, g + 8);
            const float vs0 = WIDE ? w.vs : __shfl_sync(0xffffffffu, w.vs, g), vs1 = WIDE ? w.vs : __shfl_sync(0xffffffffu, w.vs, g + 8);
            const bool edge = k0 < pc.c0 || k0 + 16 > pc.c1;                     // (warp-uniform)
            const bool in0 = !edge || (k0 + g >= pc.c0 && k0 + g < pc.c1), in1 = !edge || (k0 + g + 8 >= pc.c0 && k0 + g + 8 < pc.c1);
            const int row0 = WIDE ? w.row : __shfl_sync(0xffffffffu, w.row, g), row1 = WIDE ? w.row : __shfl_sync(0xffffffffu, w.row, g + 8);
            const bool r0 = in0 && row0 >= 0, r1 = in1 && row1 >= 0;
            if (edge) {                                      // values that are not read may be anything, and 0 * NaN is NaN
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = k0 + 2 * t + (i & 1) + 8 * (i >> 1);
                    if (key < pc.c0 || key >= pc.c1) {
#pragma unroll
                        for (int c = 0; c < (VW > 0 ? VW : 1); ++c) x.v[i][c] = 0u;
                        x.v2[i] = 0;
                    }
                }
            }
            bool over = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s[n][c] = (c < 2 ? r0 : r1) ? s[n][c] * (c < 2 ? ks0 : ks1) * qs[n][c & 1] : -INFINITY;
                    over |= s[n][c] > m[n][c & 1] + ROOM;
                }
            const int ev = max(exponent_of(vs0), exponent_of(vs1)), tile_e = WIDE ? ev : __reduce_max_sync(0xffffffffu, ev);
            if (__any_sync(0xffffffffu, over) || tile_e > E) {
                const int grown = max(E, tile_e);
                const float lower = power_of_two(E - grown);
                E = grown;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = fmaxf(s[n][c], s[n][c + 2]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)), m[n][c]);
                        const float corr = mx == -INFINITY ? 1.f : exp2_fast(m[n][c] - mx), both = corr * lower;
                        m[n][c] = mx;
                        l[n][c] *= corr;
#pragma unroll
                        for (int i = 0; i < OT; ++i) { o[n][i][c] *= both; o[n][i][c + 2] *= both; }
                    }
            }
            const float in_units = power_of_two(SHIFT - E), f0 = vs0 * in_units, f1 = vs1 * in_units;
            unsigned pf[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float b0 = m[n][0] == -INFINITY ? 0.f : m[n][0], b1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
                const float p00 = exp2_fast(s[n][0] - b0), p01 = exp2_fast(s[n][1] - b1), p10 = exp2_fast(s[n][2] - b0), p11 = exp2_fast(s[n][3] - b1);
                l[n][0] += p00 + p10;
                l[n][1] += p01 + p11;
                pf[n][0] = turned(pack_half(p00 * f0, p01 * f0));
                pf[n][1] = turned(pack_half(p10 * f1, p11 * f1));
            }
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const unsigned lo01 = __byte_perm(x.v[0][i], x.v[1][i], 0x5140), hi01 = __byte_perm(x.v[0][i], x.v[1][i], 0x7362);
                const unsigned lo23 = __byte_perm(x.v[2][i], x.v[3][i], 0x5140), hi23 = __byte_perm(x.v[2][i], x.v[3][i], 0x7362);
                const unsigned a0 = half2_low(lo01), a1 = half2_high(lo01), a2 = half2_low(lo23), a3 = half2_high(lo23);
                const unsigned c0 = half2_low(hi01), c1 = half2_high(hi01), c2 = half2_low(hi23), c3 = half2_high(hi23);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_f16(o[n][2 * i], a0, a1, a2, a3, pf[n][0], pf[n][1]);
                    mma_f16(o[n][2 * i + 1], c0, c1, c2, c3, pf[n][0], pf[n][1]);
                }
            }
            if constexpr (ODD) {
                const unsigned lo01 = __byte_perm(x.v2[0], x.v2[1], 0x5140), lo23 = __byte_perm(x.v2[2], x.v2[3], 0x5140);
                const unsigned a0 = half2_low(lo01), a1 = half2_high(lo01), a2 = half2_low(lo23), a3 = half2_high(lo23);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(o[n][OT - 1], a0, a1, a2, a3, pf[n][0], pf[n][1]);
            }
        };
        {
            Tile x, y;
            if constexpr (WIDE) {
                // lane i knows the place of step base + i; the next 32 steps' are looked up on the way, a load at a time
                const int k_of = warp * 16;
                auto key_of = [&](int st) { return st * BN + k_of; };
                Where now = where_of(page_of(key_of(st0 + lane)), key_of(st0 + lane)), then = {-1, 0.f, 0.f};
                int base = st0, page = -1;
                auto at_step = [&](int st) -> Where {        // (of a step of the present 32)
                    Where w = {__shfl_sync(0xffffffffu, now.row, st - base), __shfl_sync(0xffffffffu, now.ks, st - base), __shfl_sync(0xffffffffu, now.vs, st - base)};
                    return settle(w);
                };
                if (lane <= AHEAD) ask(now.row);
                auto advance = [&](int st) {                 // before step st's work: what lies ahead of it
                    const int i = st - base;
                    if (i == 0) page = page_of(key_of(base + 32 + lane));
                    if (i == 16) then = where_of(page, key_of(base + 32 + lane));
                    const int j = i + 1 + AHEAD;             // step st + 1 + AHEAD
                    if (lane == (j & 31)) ask(j < 32 ? now.row : then.row);
                };
                auto next_of = [&](int st) -> Where {        // step st + 1
                    if (st + 1 - base == 32) { now = then; base += 32; }
                    return at_step(st + 1);
                };
                Where wx = at_step(st0), wy;
                load(x, wx);
                for (int st = st0; st <= st1; st += 2) {
                    advance(st);
                    wy = next_of(st);
                    load(y, wy);
                    work(x, wx, st);
                    if (st + 1 > st1) break;
                    advance(st + 1);
                    wx = next_of(st + 1);
                    load(x, wx);
                    work(y, wy, st + 1);
                }
            } else {
                auto find = [&](int st) -> Where { return settle(where_of(page_of(st * BN + warp * 16 + (lane & 15)), st * BN + warp * 16 + (lane & 15))); };
                Where wx = find(st0), wy = find(st0 + 1);
                load(x, wx);
                for (int st = st0; st <= st1; st += 2) {
                    load(y, wy);
                    Where next = find(st + 2);
                    work(x, wx, st);
                    wx = next;
                    if (st + 1 > st1) break;
                    load(x, wx);
                    next = find(st + 3);
                    work(y, wy, st + 1);
                    wy = next;
                }
            }
        }

        // the four warps' shares, put together in warp order
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[n][c];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) { s_m[warp][n * 8 + 2 * t + c] = m[n][c]; s_l[warp][n * 8 + 2 * t + c] = x; }
            }
        if (lane == 0) s_e[warp] = power_of_two(E - SHIFT);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < OT; ++i) {
                const int w = i / 2;
                const int d = (ODD && i == OT - 1) ? HD - 16 + 2 * g : (((w / VL) * 8 + g) * VL + w % VL) * 4 + 2 * (i & 1);
#pragma unroll
                for (int c = 0; c < 4; ++c) s_o[warp][n * 8 + 2 * t + (c & 1)][d + (c >> 1)] = o[n][i][c];
            }
        __syncthreads();
        for (int i = tid; i < pc.heads * HD; i += NTHREADS) {
            const int h = i / HD, d = i - h * HD;
            float M = -INFINITY, acc = 0.f, L = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w][h]);
            const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {                // (a warp without a key has sums of zero; one of NaN keeps them)
                const float f = s_m[w][h] == -INFINITY ? 1.f : exp2_fast(s_m[w][h] - base);
                acc += s_o[w][h][d] * f * s_e[w];
                L += s_l[w][h] * f;
            }
            if (pc.pieces == 1) {
                out[((size_t)pc.tok * nq + pc.h0 + h) * HD + d] = __float2bfloat16(L == 0.f ? 0.f : acc / L);
            } else {
                const size_t row = ((size_t)pc.place * nq + pc.h0 + h) * S + pc.piece;
                __stcg(part + row * HD + d, acc);
                if (d == 0) __stcg(reinterpret_cast<float2*>(part_ml) + row, make_float2(M, L));
            }
        }
        if (pc.pieces > 1 && tid == 0) s_partial[number > 0] = pc;
        __syncthreads();                                     // the shares may be written again
    }
    if (bad_page && err) atomicOr(err, VL_DEV_BAD_PAGE);
    // The items shared with other blocks (the run's first and last), at its end so that the stream does not wait for them: this block's pieces are
    // counted; whoever comes last adds up all of an item's, in their order.
    if (s_partial[0].heads == 0 && s_partial[1].heads == 0) return;
    __threadfence();                                         // this thread's parts, before the block's arrivals are counted
    __syncthreads();
    if (tid < 2) s_last[tid] = s_partial[tid].heads && atomicAdd(&arrivals[s_partial[tid].counter], 1) == s_partial[tid].pieces - 1;
    __syncthreads();
    if (!s_last[0] && !s_last[1]) return;
    __threadfence();
    for (int k = 0; k < 2; ++k) {
        if (!s_last[k]) continue;
        const Piece pc = s_partial[k];
        // the pieces' weights and the sums' quotient, in the memory of the warps' shares
        float* weight = &s_o[0][0][0];                       // [heads][pieces]
        const float2* ml = reinterpret_cast<const float2*>(part_ml) + ((size_t)pc.place * nq + pc.h0) * S;
        for (int h = warp; h < pc.heads; h += WARPS) {
            float M = -INFINITY, L = 0.f;
            for (int p = lane; p < pc.pieces; p += 32) M = fmaxf(M, __ldcg(ml + (size_t)h * S + p).x);
            M = warp_max(M);
            const float base = M == -INFINITY ? 0.f : M;
            for (int p = lane; p < pc.pieces; p += 32) {
                const float2 x = __ldcg(ml + (size_t)h * S + p);
                const float f = x.x == -INFINITY ? 1.f : exp2_fast(x.x - base);
                L += x.y * f;
                weight[h * pc.pieces + p] = f;
            }
            L = warp_sum(L);
            if (lane == 0) s_l[0][h] = L;
        }
        __syncthreads();
        for (int i = tid; i < pc.heads * (HD / 4); i += NTHREADS) {
            const int h = i / (HD / 4), d = (i - h * (HD / 4)) * 4;
            const float* row = part + ((size_t)pc.place * nq + pc.h0 + h) * S * HD + d;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int p = 0; p < pc.pieces; ++p) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(row + (size_t)p * HD));
                const float f = weight[h * pc.pieces + p];
                acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
            }
            const float L = s_l[0][h], inv = L == 0.f ? 0.f : 1.f / L;
            bf16* dst = out + ((size_t)pc.tok * nq + pc.h0 + h) * HD + d;
            dst[0] = __float2bfloat16(acc.x * inv); dst[1] = __float2bfloat16(acc.y * inv);
            dst[2] = __float2bfloat16(acc.z * inv); dst[3] = __float2bfloat16(acc.w * inv);
        }
        __syncthreads();                                     // the weights may be written again
        if (tid == 0) arrivals[pc.counter] = 0;              // as the next launch finds it
    }
}

extern "C" int vl_flash_decode_8bit_head_dim() { return HD; }

// q [T, q_stride] bfloat16, out [.., nq * hd]; caches [pages, nkv, page_size, hd] e4m3, scales [pages, nkv]; positions from `bound` on are
// flagged and get rows of zeros.  part: T * nq * S * (hd + 2) floats (T: tokens of the launch), S > 1 pieces an item; arrivals: T * nq counters,
// zero before and after.
extern "C" int vl_flash_decode_8bit(const void* q, int q_stride, const void* kcache, const void* vcache, const float* kscale, const float* vscale,
                                    const int* block_table, int max_blocks, const int* req_index, const int* positions, int T, int nq, int nkv, int hd,
                                    int page_size, int num_pages, float scale, int window, int bound, int S, float* part, unsigned* err,
                                    const int* token_index, void* out, int* arrivals, int settled, void* stream) {
    if (T <= 0) return VL_OK;
    if (hd != HD) return VL_ERR_UNSUPPORTED;
    if (nq <= 0 || nkv <= 0 || nq % nkv || page_size <= 0 || max_blocks <= 0 || num_pages <= 0 || q_stride < nq * hd || q_stride % 4) return VL_ERR_ARGUMENT;
    if (bound <= 0 || S < 2 || S > PIECES_MAX || !out || !arrivals || !part) return VL_ERR_ARGUMENT;
    if (((uintptr_t)q & 7) || (((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)part) & 15)) return VL_ERR_ARGUMENT;
    const int grp = nq / nkv, wide_heads = grp > 8 && HD <= 128 ? 16 : 8, htiles = (grp + wide_heads - 1) / wide_heads;
    const long long most = (long long)T * nkv * htiles * ((bound + BN - 1) / BN);
    if ((long long)num_pages * nkv * page_size >= (1ll << 31) || most >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return (int)e;
    const bool wide = page_size % 16 == 0;
    auto launch = [&](auto kernel, int blocks_an_sm) {
        const long long grid = (long long)sms * blocks_an_sm;
        return vl_launch(kernel, dim3((unsigned)(most < grid ? most : grid)), dim3(NTHREADS), 0, (cudaStream_t)stream, (const bf16*)q, q_stride,
                         (const unsigned char*)kcache, (const unsigned char*)vcache, kscale, vscale, block_table, max_blocks, req_index, positions, T,
                         nq, nkv, page_size, num_pages, scale * 1.4426950408889634f, window, bound, S, part, err, token_index, (bf16*)out, arrivals, settled);
    };
    if constexpr (HD <= 128) {
        if (wide_heads == 16) return wide ? launch(flash_decode_8bit_kernel<2, true>, 2) : launch(flash_decode_8bit_kernel<2, false>, 2);
    }
    return wide ? launch(flash_decode_8bit_kernel<1, true>, HD <= 128 ? 3 : 2) : launch(flash_decode_8bit_kernel<1, false>, HD <= 128 ? 3 : 2);
}
