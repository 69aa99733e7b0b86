// Products of 8-bit rows and 8-bit weights with everything that follows them in one pass:
//     y[m, n] = f(sa[m] sw[n] sum_k a[m, k] w[n, k] + bias[n]) + residual[m, n]
// a [M, width] e4m3 with a scale a row (rows_8bit.cu), w packed e4m3 with a scale an output row (vl_pack_8bit), sums,
// scales, bias, activation and residual in float32, one rounding to out's type.  A sum is multiplied by w's scale first and by its row's then, in
// every kernel: times the scale of a row of large numbers alone it may overflow, and the two scales' product alone may be no normal number.
// f: none, a function of one argument, or (gated) f(gate) * up with w's rows in blocks of 8 gates and their 8 ups: out then has N / 2 columns.
#include "tc5.cuh"
#include <cuda_fp8.h>
#include <math.h>

using namespace tc5;

namespace {
enum { ACT_NONE = -1, ACT_SILU = 0, ACT_RELU = 1, ACT_RELU2 = 16, ACT_TANH = 17, ACT_GELU = 18 };   // codes of csrc/ops.py

struct Epilogue {
    const float* a_scale;                    // [M]
    const float* w_scale;                    // [N]
    const float* bias;                       // [N] or null
    const void* residual;                    // as out, or null
    void* out;
    int M, N, act, gated;
};

// v / (1 + exp(-v)).  The quick quotient (2 units in the last place): the exact one leaves the straight path where exp(-v) overflows, and a tile's
// epilogue then takes longer than its products
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + __expf(-v)); }
__device__ __forceinline__ float relu(float v) { return v < 0.f ? 0.f : v; }
// v times the normal distribution function, max(v, 0) - |v| / 2 erfc(|v| / sqrt(2)).  erfc(x) = t exp(-x^2) P(t), t = 1 / (1 + 0.4 x), P the
// polynomial of degree 8 nearest to erfc(x) exp(x^2) / t in relative error for x up to 10 (least squares at Chebyshev nodes: 7e-8; in float32 4e-7),
// which holds far below zero, where 1 + erf cancels.  17 operations: with erfcf, 2,048 x 4,096 -> 8,192 took 66.5 us for 60.7 (52 without activation).
__device__ __forceinline__ float gelu(float v) {
    const float x = fabsf(v), t = __fdividef(1.0f, fmaf(0.282842712f, x, 1.0f));
    float p = 0.0419418029f;
    p = fmaf(p, t, -0.143589124f);
    p = fmaf(p, t, 0.0905594453f);
    p = fmaf(p, t, 0.0806835741f);
    p = fmaf(p, t, 0.0846026987f);
    p = fmaf(p, t, 0.191415131f);
    p = fmaf(p, t, 0.202369645f);
    p = fmaf(p, t, 0.226379126f);
    p = fmaf(p, t, 0.225637764f);
    return relu(v) - 0.5f * fminf(x, 20.0f) * (t * p * __expf(-0.5f * x * x));
}
// called, not repeated for each of a chunk's values
__device__ __noinline__ float tanh_of(float v) { return tanhf(v); }
template <int ACT> __device__ __forceinline__ float activate(float v) {
    if (ACT == ACT_SILU) return silu(v);
    if (ACT == ACT_RELU) return relu(v);
    if (ACT == ACT_RELU2) return v < 0.f ? 0.f : v * v;
    if (ACT == ACT_TANH) return tanh_of(v);
    if (ACT == ACT_GELU) return gelu(v);
    return v;
}
__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ACT_SILU: return silu(v);
        case ACT_RELU: return relu(v);
        case ACT_RELU2: return v < 0.f ? 0.f : v * v;
        case ACT_TANH: return tanh_of(v);
        case ACT_GELU: return gelu(v);
        default: return v;
    }
}

// ---- from an accumulator in TMEM to out ------------------------------------------------------------
// W's rows lie along the accumulator's lanes and the rows of a along its columns: a thread holds CHUNK values of its row n of W, for the
// rows t0 .. t0 + CHUNK - 1 of a, whose scales lie in shared memory; `end` is the row of a behind the tile's last.  A warp's 32 lanes are 32 neighbouring columns of out, 64 or 128 bytes of a row a store; gated, lanes 8 apart hold a gate and
// its up and take every second row each.  The instructions of a value are what a tile's epilogue costs: stores of two neighbouring columns, which
// lanes have to exchange values for, took three times as many as these (256 rows x 1,024 -> 1,024 on pairs of SMs: 11.5 us and 9.1).
constexpr int CHUNK = 16;

__device__ __forceinline__ void load_tmem(unsigned taddr, float (&v)[CHUNK]) {
    unsigned r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
    tc5_wait_ld();
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) v[i] = __uint_as_float(r[i]);
}

// What a thread adds to its values of such a chunk and where they go.
template <typename TO, bool GATED>
struct Place {
    static constexpr int STEP = GATED ? 2 : 1, COUNT = CHUNK / STEP;
    size_t at, step;
    int rows;
    __device__ __forceinline__ Place(const Epilogue& e, int n, int t0, int end) {
        const int up = GATED ? (threadIdx.x >> 3) & 1 : 0, ld = GATED ? e.N >> 1 : e.N;
        at = (size_t)(t0 + up) * ld + (GATED ? ((n >> 4) << 3) + (n & 7) : n);
        step = (size_t)STEP * ld;
        rows = n < e.N ? min(end, e.M) - t0 - up : 0;
    }
    __device__ __forceinline__ void load(const Epilogue& e, TO (&x)[COUNT]) const {
        const TO* r = reinterpret_cast<const TO*>(e.residual) + at;
#pragma unroll
        for (int c = 0; c < COUNT; ++c, r += step) x[c] = c * STEP < rows ? *r : from_f32<TO>(0.f);
    }
};

template <typename TO, int ACT, bool GATED>
__device__ __forceinline__ void finish(float (&v)[CHUNK], TO (&x)[CHUNK / (GATED ? 2 : 1)], int n, int t0, int end, int next, const Epilogue& e,
                                       const float* scales, float sw, float b) {
    const Place<TO, GATED> p(e, n, t0, end);
    const float4* s4 = reinterpret_cast<const float4*>(scales);
#pragma unroll
    for (int c = 0; c < CHUNK; c += 4) {
        const float4 s = s4[c / 4];
        v[c] = v[c] * sw * s.x + b;
        v[c + 1] = v[c + 1] * sw * s.y + b;
        v[c + 2] = v[c + 2] * sw * s.z + b;
        v[c + 3] = v[c + 3] * sw * s.w + b;
    }
    constexpr int STEP = Place<TO, GATED>::STEP, COUNT = Place<TO, GATED>::COUNT;
    if (GATED) {
        const int up = (threadIdx.x >> 3) & 1;
#pragma unroll
        for (int c = 0; c < CHUNK; c += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, up ? v[c] : v[c + 1], 8);
            v[c / 2] = activate<ACT>(up ? got : v[c]) * (up ? v[c + 1] : got);
        }
    } else {
#pragma unroll
        for (int c = 0; c < CHUNK; ++c) v[c] = activate<ACT>(v[c]);
    }
    if (e.residual) {
#pragma unroll
        for (int c = 0; c < COUNT; ++c) v[c] += to_f32(x[c]);
        if (next < end) Place<TO, GATED>(e, n, next, end).load(e, x);
    }
    TO* o = reinterpret_cast<TO*>(e.out) + p.at;
#pragma unroll
    for (int c = 0; c < COUNT; ++c, o += p.step)
        if (c * STEP < p.rows) *o = from_f32<TO>(v[c]);
}

// The chunks of a warp, one of PARTS of a tile's (rows t0 + c0 .. of a, c0 < cols): what they are added to is asked for ahead, the first
// before `ready` waits for the sums (-> whether they came), the others before the stores of the one in front; `sums(c0, v)` brings the sums.
// Residual and out may be the same memory: a thread reads what it writes, and before.
template <typename TO, int ACT, bool GATED, int PARTS, typename Ready, typename Sums>
__device__ __forceinline__ bool finish_chunks(const Epilogue& e, int n, const float* scales, float sw, float b, int t0, int end, int first, int cols, Ready ready,
                                              Sums sums) {
    TO x[Place<TO, GATED>::COUNT];
    end = min(end, t0 + cols);
    int c0 = first * CHUNK;
    if (c0 < cols && e.residual) Place<TO, GATED>(e, n, t0 + c0, end).load(e, x);
    if (!ready()) return false;
#pragma unroll 1
    for (; c0 < cols; c0 += PARTS * CHUNK) {
        float v[CHUNK];
        sums(c0, v);
        finish<TO, ACT, GATED>(v, x, n, t0 + c0, end, t0 + c0 + PARTS * CHUNK, e, scales + c0, sw, b);
    }
    return true;
}

// The last copies that a block issued, of `issued` through a ring of `stages`, have arrived (or each had its time): no block leaves with copies on
// their way into its shared memory, whatever happened to those who wait for them.  One thread; a fill nobody has waited for yet is no hurry.
__device__ __forceinline__ void see_copies_in(unsigned long long* full_bar, int issued, int stages) {
    for (int j = max(0, issued - stages); j < issued; ++j) mbar_wait_bounded(&full_bar[j % stages], (unsigned)((j / stages) & 1));
}

constexpr int STRIP = 16, KB = 128;          // a strip of W, a block of K: 128 bytes
constexpr int ROWS = 128;                    // W's rows of a block
constexpr unsigned W_BYTES = ROWS * KB;
}  // namespace

// ---- many rows: two SMs on a tile of 256 rows of W by 256 rows of a ---------------------------------
namespace pair8 {
constexpr int MOST = 256, STAGES = 6, PARTS = 4, EPILOGUE = PARTS * 128, NUM_THREADS = 64 + EPILOGUE;
constexpr unsigned STAGE_BYTES = W_BYTES + MOST / 2 * KB, TMEM_COLS = 512;

// Tile `place` of the pairs' order: its corner and its rows of a.  From `whole` on places are halves of tiles: where the last round of the pairs
// has at most half of them a tile, its tiles are cut in two (4,096 x 12,288 -> 4,096, 256 tiles for 74 pairs, in short
// runs: bfloat16 147 us in whole tiles, 140 so, the float32 stream 159 and 151).
__device__ __forceinline__ int tile_corner(int place, int whole, int tiles_t, int tiles_n, int bt, int& t0, int& n0) {
    const int beyond = place - whole, tile = beyond < 0 ? place : whole + (beyond >> 1);
    constexpr int BAND = 8;                                  // pairs that run together share W's tiles in L2
    const int band = tile / (BAND * tiles_n), in_band = tile - band * BAND * tiles_n;
    const int band_rows = min(BAND, tiles_t - band * BAND);
    t0 = (band * BAND + in_band % band_rows) * bt;
    n0 = (in_band / band_rows) * 2 * ROWS;
    if (beyond < 0) return bt;
    t0 += (beyond & 1) * (bt >> 1);
    return bt >> 1;
}

template <typename TO, int ACT, bool GATED>
__global__ void __launch_bounds__(NUM_THREADS, 1)
gemm_8bit_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_half, const __grid_constant__ CUtensorMap map_w,
                      Epilogue e, int k_blocks, int bt, int whole, int places, int tiles_t, int tiles_n, unsigned* err) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full_bar[2], acc_empty_bar[2];
    __shared__ __align__(16) float scales[2][MOST];          // of a tile's rows of a, by accumulator
    __shared__ unsigned tmem_base_slot;
    __shared__ int failed;
    const int warp = warp_number();
    const unsigned rank = cluster_rank();
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full_bar[i], 1); mbar_init(&empty_bar[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full_bar[i], 1); mbar_init(&acc_empty_bar[i], 2 * EPILOGUE); }
        mbar_fence_init();
        failed = 0;
    }
    // Never launched as a programmatic dependent (see launch_pair); the order is kept all the same: nothing of the SM pair, tensor memory or the
    // cluster's barrier, is taken while earlier kernels run.
    pdl_wait();
    __syncthreads();
    cluster_sync();                                          // the other block's mbarriers exist before anything arrives there
    unsigned tmem_base = 0;
    if (warp > 0) {                                          // tensor memory comes while the first copies are under way
        if (warp == 1) alloc_pair(&tmem_base_slot, TMEM_COLS);
        tc5_fence_before();
        asm volatile("bar.sync 2, %0;" ::"n"(NUM_THREADS - 32) : "memory");
        tc5_fence_after();
        tmem_base = tmem_base_slot;
    }

    if (warp == 0) {                                         // ---- copies ----
        const bool lead = elect_one();
        int s = 0, issued = 0;
        unsigned phase = 1;
        bool ok = true;
        for (int place = pair; place < places && ok; place += num_pairs) {
            int t0, n0;
            const int rows = tile_corner(place, whole, tiles_t, tiles_n, bt, t0, n0);
            const int strip = n0 / STRIP + (int)rank * (ROWS / STRIP), row = t0 + (int)rank * (rows / 2);
            const CUtensorMap* map = rows == bt ? &map_a : &map_half;
            for (int kb = 0; kb < k_blocks; ++kb) {
                if (!warp_wait(&empty_bar[s], phase)) {
                    if (lead) atomicOr(&failed, 1);
                    ok = false;
                    break;
                }
                if (lead) {
                    if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * W_BYTES + (unsigned)(rows * KB));     // the bytes of both blocks
                    const unsigned bar = map_to_rank(smem_u32(&full_bar[s]), 0);
                    unsigned char* st = smem + (size_t)s * STAGE_BYTES;
                    tma_load_3d_pair(st, &map_w, 0, kb * STRIP, strip, bar);
                    tma_load_2d_pair(st + W_BYTES, map, kb * KB, row, bar);
                }
                ++issued;
                if (++s == STAGES) { s = 0; phase ^= 1u; }
            }
        }
        if (lead && rank == 0) see_copies_in(full_bar, issued, STAGES);          // both blocks' (the other waits at the last barrier)
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {                                     // ---- the pair's products ----
            const bool lead = elect_one();
            int s = 0, local = 0;
            unsigned phase = 0;
            bool ok = true;
            for (int place = pair; place < places && ok; place += num_pairs, ++local) {
                const unsigned idesc = make_idesc_8bit(2 * ROWS, place < whole ? bt : bt >> 1);
                const int acc = local & 1;
                if (local >= 2 && !warp_wait(&acc_empty_bar[acc], (unsigned)((local / 2 - 1) & 1))) {
                    if (lead) atomicOr(&failed, 2);
                    break;
                }
                tc5_fence_after();
                const unsigned tmem_c = tmem_base + (unsigned)(acc * MOST);
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!warp_wait(&full_bar[s], phase)) {
                        if (lead) atomicOr(&failed, 4);
                        ok = false;
                        break;
                    }
                    tc5_fence_after();
                    const unsigned char* st = smem + (size_t)s * STAGE_BYTES;
                    const unsigned long long wdesc = make_smem_desc(st), adesc = make_smem_desc(st + W_BYTES);
                    if (lead) {
#pragma unroll
                        for (int k = 0; k < KB / 32; ++k)
                            mma_pair_8bit(tmem_c, wdesc + (unsigned long long)(k * 2), adesc + (unsigned long long)(k * 2), idesc, (kb > 0 || k > 0) ? 1u : 0u);
                        commit_pair(&empty_bar[s]);
                        if (kb + 1 == k_blocks) commit_pair(&acc_full_bar[acc]);
                    }
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                }
            }
        }
    } else {                                                 // ---- epilogue: warps 2..17 ----
        const int quarter = warp & 3, part = (warp - 2) >> 2, lane = threadIdx.x & 31;
        const unsigned freed = map_to_rank(smem_u32(&acc_empty_bar[0]), 0);
        int local = 0;
        for (int place = pair; place < places; place += num_pairs, ++local) {
            const int acc = local & 1;
            int t0, n0;
            const int rows = tile_corner(place, whole, tiles_t, tiles_n, bt, t0, n0);
            const int n = n0 + (int)rank * ROWS + quarter * 32 + lane;
            const float sw = n < e.N ? e.w_scale[n] : 0.f, b = e.bias && n < e.N ? e.bias[n] : 0.f;
            const int i = threadIdx.x - 64;                  // (who read this place last has passed the barrier of the tile between)
            if (i < MOST) scales[acc][i] = t0 + i < e.M ? e.a_scale[t0 + i] : 0.f;
            asm volatile("bar.sync 1, %0;" ::"n"(EPILOGUE) : "memory");
            const unsigned tmem = tmem_base + ((unsigned)(quarter * 32) << 16) + (unsigned)(acc * MOST);
            // no warp leaves the tiles before the others: they meet at the barrier above.  Where a wait ran out, nobody waits any more.
            if (!finish_chunks<TO, ACT, GATED, PARTS>(
                    e, n, scales[acc], sw, b, t0, t0 + rows, part, min(rows, e.M - t0),
                    [&] {
                        const bool there = __all_sync(0xffffffffu, *(volatile int*)&failed == 0) && warp_wait(&acc_full_bar[acc], (unsigned)((local / 2) & 1));
                        tc5_fence_after();
                        return there;
                    },
                    [&](int c0, float (&v)[CHUNK]) { load_tmem(tmem + (unsigned)c0, v); }))
                atomicOr(&failed, 8);
            tc5_fence_before();
            mbar_arrive_remote(freed + (unsigned)(acc * sizeof(unsigned long long)));
        }
    }
    tc5_fence_before();
    __syncthreads();
    cluster_sync();                                          // neither block frees or leaves while the other may still read it
    tc5_fence_after();
    if (warp == 1) dealloc_pair(tmem_base, TMEM_COLS);
    if (threadIdx.x == 0 && failed && err) atomicOr(err, VL_DEV_WAIT_EXPIRED | VL_DEV_IN_GEMM_8BIT | ((unsigned)failed << VL_DEV_ROLE_SHIFT));
}
}  // namespace pair8

// ---- in between: one SM on a tile of 128 rows of W by bt rows of a, several blocks sharing its K ------------------------
// A block multiplies a run of the blocks of K of `height` rows of W (the 128-row operand; 96 or 112 of them where that spreads the tiles better) and bt rows of a.  Where a tile's K is shared out, the blocks leave their sums in scratch memory,
// [blocks of a tile, rows of a, W's rows rounded up to whole tiles], and a second launch adds them in the order of K and finishes them; it starts behind the
// first without a gap.  (Joined through the shared memory of a cluster, x 12,288 -> 4,096 took 14.5 us in a graph at 64 rows and 16.4 in calls
// behind one another, 13.8 and 15.0 so; kernels of clusters are launched the plain way, and a step that holds one has the engine's switch off:
// only kernels that touch nothing before their wait keep the attribute in it.)
namespace split8 {
constexpr int PARTS = 2, NUM_THREADS = 64 + PARTS * 128;      // (sixteen warps of epilogue, as pairs have, start later: x 12,288 -> 4,096 at 64 rows 14.4 us and 15.1)

// bt: a multiple of 16 up to 256; ahead: W is a constant, its first copies begin before the kernel in front has ended.
template <typename TO, int ACT, bool GATED, int PER_SM>
__global__ void __launch_bounds__(NUM_THREADS, PER_SM)
gemm_8bit_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, Epilogue e, int k_blocks, int height, int bt,
                       int tiles_t, int splits, float* scratch, int stages, int ahead, unsigned* err) {
    const unsigned w_bytes = (unsigned)(height * KB), stage_bytes = w_bytes + (unsigned)(bt * KB);
    extern __shared__ __align__(1024) unsigned char smem[];   // (nothing else is shared: it begins on a kilobyte)
    unsigned long long* full_bar = reinterpret_cast<unsigned long long*>(smem + stages * stage_bytes);
    unsigned long long *empty_bar = full_bar + stages, *acc_bar = empty_bar + stages;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(acc_bar + 1);
    int* failed = reinterpret_cast<int*>(tmem_slot + 1);
    float* scales = reinterpret_cast<float*>(((uintptr_t)(failed + 1) + 15) & ~(uintptr_t)15);     // of the tile's rows of a
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x % splits), tile = (int)(blockIdx.x / splits);
    const int t0 = (tile % tiles_t) * bt, n0 = (tile / tiles_t) * height;
    const int kb0 = (int)((long long)k_blocks * rank / splits), kb1 = (int)((long long)k_blocks * (rank + 1) / splits);
    const unsigned tmem_cols = bt <= 32 ? 32 : bt <= 64 ? 64 : bt <= 128 ? 128 : 256;
    auto copy_w = [&](int s, int kb) {
        mbar_arrive_expect_tx(&full_bar[s], stage_bytes);
        tma_load_3d(smem + s * stage_bytes, &map_w, 0, kb * STRIP, n0 / STRIP, &full_bar[s]);
    };
    auto copy_a = [&](int s, int kb) { tma_load_2d(smem + s * stage_bytes + w_bytes, &map_a, kb * KB, t0, &full_bar[s]); };
    const int early = min(stages, kb1 - kb0);

    pdl_launch_dependents();
    if (!ahead) pdl_wait();                                  // W may be as young as a
    if (warp == 0) {
        if (elect_one()) {                                   // the first copies go out before anything else is set up
            for (int i = 0; i < stages; ++i) { mbar_init(&full_bar[i], 1); mbar_init(&empty_bar[i], 1); }
            mbar_init(acc_bar, 1);
            mbar_fence_init();
            *failed = 0;
            for (int i = 0; i < early; ++i) copy_w(i, kb0 + i);
        }
        __syncwarp();
    }
    if (ahead) pdl_wait();
    if (warp == 0) {
        if (elect_one())
            for (int i = 0; i < early; ++i) copy_a(i, kb0 + i);
        __syncwarp();
    }
    if (warp == 1) tc5_alloc(tmem_slot, tmem_cols);
    const int quarter = warp & 3, part = (warp - 2) >> 2;
    const int row = quarter * 32 + lane, n = row < height ? n0 + row : e.N;    // (lanes beyond the tile's height hold products with what lies behind it)
    float sw = 0.f, b = 0.f;
    if (warp >= 2) {
        const int i = threadIdx.x - 64;
        if (i < bt) scales[i] = t0 + i < e.M ? e.a_scale[t0 + i] : 0.f;
        if (n < e.N) {
            sw = e.w_scale[n];
            if (e.bias) b = e.bias[n];
        }
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    const unsigned tmem_base = *tmem_slot;

    if (warp == 0) {                                         // ---- copies ----
        const bool lead = elect_one();
        int s = 0, issued = early;
        unsigned phase = 0;
        for (int kb = kb0 + early; kb < kb1; ++kb) {
            if (!warp_wait(&empty_bar[s], phase)) {
                if (lead) atomicOr(failed, 1);
                break;
            }
            if (lead) {
                copy_w(s, kb);
                copy_a(s, kb);
            }
            ++issued;
            if (++s == stages) { s = 0; phase ^= 1u; }
        }
        if (lead) see_copies_in(full_bar, issued, stages);
        __syncwarp();
    } else if (warp == 1) {                                  // ---- products ----
        const bool lead = elect_one();
        const unsigned idesc = make_idesc_8bit(ROWS, bt);
        int s = 0;
        unsigned phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!warp_wait(&full_bar[s], phase)) {
                if (lead) atomicOr(failed, 4);
                break;
            }
            tc5_fence_after();
            const unsigned char* st = smem + s * stage_bytes;
            const unsigned long long wdesc = make_smem_desc(st), adesc = make_smem_desc(st + w_bytes);
            if (lead) {
#pragma unroll
                for (int k = 0; k < KB / 32; ++k)
                    tc5_mma_8bit(tmem_base, wdesc + (unsigned long long)(k * 2), adesc + (unsigned long long)(k * 2), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
                tc5_commit(&empty_bar[s]);
                if (kb + 1 == kb1) tc5_commit(acc_bar);
            }
            if (++s == stages) { s = 0; phase ^= 1u; }
        }
    }
    const unsigned tmem = tmem_base + ((unsigned)(quarter * 32) << 16);
    const int cols = min(bt, (e.M - t0 + CHUNK - 1) / CHUNK * CHUNK);          // columns that hold rows of a (bt is a multiple of 16)
    auto wait_sums = [&] {
        const bool there = warp_wait(acc_bar, 0);
        if (!there) atomicOr(failed, 8);
        tc5_fence_after();
        return there;
    };
    if (warp >= 2 && quarter * 32 < height) {
        if (splits == 1) {
            finish_chunks<TO, ACT, GATED, PARTS>(e, n, scales, sw, b, t0, t0 + bt, part, cols, wait_sums,
                                                 [&](int c0, float (&v)[CHUNK]) { load_tmem(tmem + (unsigned)c0, v); });
        } else if (wait_sums()) {
            const size_t ld = (size_t)((e.N + ROWS - 1) / ROWS) * ROWS;
#pragma unroll 1
            for (int c0 = part * CHUNK; c0 < cols; c0 += PARTS * CHUNK) {
                float v[CHUNK];
                load_tmem(tmem + (unsigned)c0, v);
                float* p = scratch + ((size_t)rank * e.M + t0 + c0) * ld + n;
                const int rows = min(t0 + bt, e.M) - t0 - c0;
#pragma unroll
                for (int c = 0; c < CHUNK; ++c, p += ld)
                    if (c < rows && n < e.N) *p = v[c];
            }
        }
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    if (warp == 1) tc5_dealloc(tmem_base, tmem_cols);
    if (threadIdx.x == 0 && *failed && err) atomicOr(err, VL_DEV_WAIT_EXPIRED | VL_DEV_IN_GEMM_8BIT | ((unsigned)*failed << VL_DEV_ROLE_SHIFT));
}

// Four neighbouring outputs a thread, a row of a by blockIdx.x (which has no limit of 65,535).  WIDE: rows of out hold a multiple of four and everything begins on 16 bytes.
template <bool WIDE, typename T>
__device__ __forceinline__ float4 load4(const T* p, int left) {
    if (WIDE) return Quad<T>::load(p);
    return make_float4(to_f32(p[0]), left > 1 ? to_f32(p[1]) : 0.f, left > 2 ? to_f32(p[2]) : 0.f, left > 3 ? to_f32(p[3]) : 0.f);
}
template <typename TO, int ACT, bool GATED, bool WIDE>
__global__ void __launch_bounds__(256)
gemm_8bit_join_kernel(const float* __restrict__ scratch, Epilogue e, int splits) {
    pdl_launch_dependents();
    pdl_wait();
    const int width = GATED ? e.N >> 1 : e.N, m = blockIdx.x, col = 4 * (blockIdx.y * 256 + threadIdx.x);
    if (col >= width) return;
    const int n = GATED ? 2 * col - (col & 7) : col, left = width - col;
    const size_t ld = (size_t)((e.N + ROWS - 1) / ROWS) * ROWS;
    const float* p = scratch + (size_t)m * ld + n;
    TO* out = reinterpret_cast<TO*>(e.out) + (size_t)m * width + col;
    const float s = e.a_scale[m];
    auto scaled = [&](int at) {                              // the sums of columns n + at .. with scales and bias
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r0 = 0; r0 < splits; r0 += 4) {             // four parts' loads at a time on their way
            float4 q[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                q[r] = r0 + r < splits ? *reinterpret_cast<const float4*>(p + at + (size_t)(r0 + r) * e.M * ld) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int r = 0; r < 4; ++r) v = make_float4(v.x + q[r].x, v.y + q[r].y, v.z + q[r].z, v.w + q[r].w);
        }
        const float4 w = load4<WIDE>(e.w_scale + n + at, left), b = e.bias ? load4<WIDE>(e.bias + n + at, left) : make_float4(0.f, 0.f, 0.f, 0.f);
        return make_float4(v.x * w.x * s + b.x, v.y * w.y * s + b.y, v.z * w.z * s + b.z, v.w * w.w * s + b.w);
    };
    float4 y = scaled(0), r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e.residual) r = load4<WIDE>(reinterpret_cast<const TO*>(e.residual) + (size_t)m * width + col, left);
    y = make_float4(activate<ACT>(y.x), activate<ACT>(y.y), activate<ACT>(y.z), activate<ACT>(y.w));
    if (GATED) {
        const float4 u = scaled(8);
        y = make_float4(y.x * u.x, y.y * u.y, y.z * u.z, y.w * u.w);
    }
    y = make_float4(y.x + r.x, y.y + r.y, y.z + r.z, y.w + r.w);
    if (WIDE) {
        Quad<TO>::store(out, y);
        return;
    }
    out[0] = from_f32<TO>(y.x);
    if (left > 1) out[1] = from_f32<TO>(y.y);
    if (left > 2) out[2] = from_f32<TO>(y.z);
    if (left > 3) out[3] = from_f32<TO>(y.w);
}
}  // namespace split8

// ---- few rows (a decode step): W's stream is all that counts ------------------------------------------
// A block walks tiles of NS strips of 16 rows of W.  A warp brings them in, with the rows of a they meet, through a ring of stages that
// goes on across tiles: 8 / NS blocks of K of every strip (they lie one behind the other: a bulk copy a strip; where W is known to be a constant, `ahead`,
// its first copies begin before the kernel in front has ended).  Eight warps multiply, each a block of K of a strip.  mma.sync m16n8k32 pairs operand
// elements by their index along K and mixes no rows, so the bytes a lane holds may stand for any columns as long as both operands
// agree: pieces t and t + 4 of W's row against pieces t and t + 4 of the row of a, 16 bytes at a time.  Row (column) g of the instruction
// is W's (a's) row (g >> 1) + 4 (g & 1): eight neighbouring lanes then read all 32 banks (rows 0 and 4 have their pieces exchanged by 4).
// The sums of a strip's warps are added in their order; a thread asks for its outputs' scales, bias and residual when the tile begins.
namespace few8 {
constexpr int WARPS = 8;
constexpr unsigned BLOCK_BYTES = STRIP * KB;

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_16832(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Who gives up notes that for the block and goes on as if the stage were there; from then on nobody waits long, and no lane leaves a loop by itself.
__device__ __forceinline__ void wait_or_note(unsigned long long* bar, unsigned parity, volatile int* gave_up) {
    if (mbar_try_wait(bar, parity)) return;
    const long long t0 = clock64();
    for (int i = 0; i < VL_WAIT_POLL_LIMIT; ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if ((i & 31) == 31 && (*gave_up || vl_wait_gave_up(i, t0))) break;
    }
    *gave_up = 1;
}

// MT: rows of a in eights, NS: strips of a tile
template <int MT, int NS> struct Shape {
    static constexpr int DEEP = WARPS / NS;                   // blocks of K of a stage
    static constexpr unsigned W_STRIP = DEEP * BLOCK_BYTES, A_OFF = NS * W_STRIP, A_BYTES = DEEP * MT * 8 * KB, STAGE_BYTES = A_OFF + A_BYTES;
    static constexpr int OUTS = MT * NS > 2 ? MT * NS / 2 : 1;       // outputs of a thread
    // the sums of a tile's warps: twice, so that a tile's are added while the next tile's arrive
    typedef float Sums[DEEP][MT * 8][NS * STRIP + 1];
    static constexpr unsigned smem(int stages) { return stages * STAGE_BYTES + 2 * (unsigned)sizeof(Sums) + 16 * stages + 16; }
};

template <typename TO, int MT, int NS, int STAGES, int PER_SM>
__global__ void __launch_bounds__(32 * WARPS + 32, PER_SM)
gemm_8bit_few_kernel(const __grid_constant__ CUtensorMap map_a, const unsigned char* __restrict__ W, Epilogue e, int k_blocks, int strips, int ahead, unsigned* err) {
    using S = Shape<MT, NS>;
    constexpr int DEEP = S::DEEP, OUTS = S::OUTS;
    extern __shared__ __align__(1024) unsigned char ring[];   // (nothing else is shared: it begins on a kilobyte)
    typename S::Sums* red = reinterpret_cast<typename S::Sums*>(ring + STAGES * S::STAGE_BYTES);
    unsigned long long* full_bar = reinterpret_cast<unsigned long long*>(red + 2);
    unsigned long long* empty_bar = full_bar + STAGES;
    volatile int& gave_up = *reinterpret_cast<volatile int*>(empty_bar + STAGES);
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const int per_tile = (k_blocks + DEEP - 1) / DEEP;
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full_bar[i], 1); mbar_init(&empty_bar[i], WARPS); }
        mbar_fence_init();
    }
    __syncthreads();
    if (warp == WARPS) {                                      // ---- copies ----
        if (elect_one()) {
            auto copy_w = [&](int s, int strip, int it) {
                const unsigned bytes = (unsigned)min(DEEP, k_blocks - it * DEEP) * BLOCK_BYTES;
                mbar_arrive_expect_tx(&full_bar[s], bytes * (unsigned)min(NS, strips - strip) + S::A_BYTES);
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (strip + i < strips)
                        bulk_copy(ring + (size_t)s * S::STAGE_BYTES + i * S::W_STRIP, W + ((size_t)(strip + i) * k_blocks + it * DEEP) * BLOCK_BYTES, bytes,
                                  &full_bar[s]);
            };
            auto copy_a = [&](int s, int it) { tma_load_3d(ring + (size_t)s * S::STAGE_BYTES + S::A_OFF, &map_a, 0, 0, it * DEEP, &full_bar[s]); };
            const int mine = (strips - (int)blockIdx.x * NS + (int)gridDim.x * NS - 1) / ((int)gridDim.x * NS), total = mine * per_tile;
            const int early = min(STAGES, total);
            int strip = blockIdx.x * NS, it = 0;
            auto step = [&]() { if (++it == per_tile) { it = 0; strip += gridDim.x * NS; } };
            if (!ahead) pdl_wait();                            // W may be as young as a
            for (int s = 0; s < early; ++s, step()) copy_w(s, strip, it);
            // What lies AHEAD stages behind the ring is asked for into L2: where half of a stage is a's, the ring alone does not keep memory busy (16
            // rows x 12,288 -> 4,096 11.9 us without, 10.1 two stages ahead, 10.6 four, overlapped; up to 8 rows 9.1 without, 9.6 four).
            constexpr int AHEAD = MT > 1 ? 2 : 0;
            int next_strip = strip, next_it = it, asked = early;
            auto ask = [&]() {
                if (asked >= total) return;
                const unsigned bytes = (unsigned)min(DEEP, k_blocks - next_it * DEEP) * BLOCK_BYTES;
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (next_strip + i < strips)
                        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                                     ::"l"(W + ((size_t)(next_strip + i) * k_blocks + next_it * DEEP) * BLOCK_BYTES), "r"(bytes) : "memory");
                ++asked;
                if (++next_it == per_tile) { next_it = 0; next_strip += gridDim.x * NS; }
            };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) ask();
            pdl_wait();                                       // a comes from the kernel before
            for (int s = 0; s < early; ++s) copy_a(s, s % per_tile);
            int s = 0;
            unsigned phase = 0;
            int i = early;
            for (; i < total; ++i, step()) {
                if (!mbar_wait_bounded(&empty_bar[s], phase)) {
                    gave_up = 1;
                    break;
                }
                copy_w(s, strip, it);
                copy_a(s, it);
                if (AHEAD) ask();
                if (++s == STAGES) { s = 0; phase ^= 1u; }
            }
            see_copies_in(full_bar, i, STAGES);
        }
        return;
    }
    pdl_wait();
    const int deep = warp % DEEP, mine = warp / DEEP;         // this warp's block of a stage's K, and its strip
    const int g = lane >> 2, t = lane & 3, row = (g >> 1) | ((g & 1) << 2);
    const int at = row * 128 + ((t ^ row) << 4);              // piece t of the row in a block of K; piece t + 4 is this xor 64
    const int each = NS * (e.gated ? STRIP / 2 : STRIP), ld = e.gated ? e.N >> 1 : e.N;
    TO* out = reinterpret_cast<TO*>(e.out);
    const TO* res = reinterpret_cast<const TO*>(e.residual);
    int s = 0, buf = 0;
    unsigned phase = 0;
    for (int strip = blockIdx.x * NS; strip < strips; strip += gridDim.x * NS, buf ^= 1) {
        // only asked for here: a use would wait for memory
        float am[OUTS], ws[OUTS], wb[OUTS], us[OUTS], ub[OUTS];
        TO yr[OUTS];
#pragma unroll
        for (int o = 0; o < OUTS; ++o) {
            const int i = threadIdx.x + o * 32 * WARPS, m = i / each, c = i % each, col = strip * (each / NS) + c;
            const int n = strip * STRIP + (e.gated ? 2 * c - (c & 7) : c);      // gated: eight gates, their eight ups, ...
            am[o] = ws[o] = wb[o] = us[o] = ub[o] = 0.f;
            yr[o] = from_f32<TO>(0.f);
            if (m < e.M && col < ld) {
                am[o] = e.a_scale[m];
                ws[o] = e.w_scale[n];
                if (e.bias) wb[o] = e.bias[n];
                if (e.gated) {
                    us[o] = e.w_scale[n + 8];
                    if (e.bias) ub[o] = e.bias[n + 8];
                }
                if (res) yr[o] = res[(size_t)m * ld + col];
            }
        }
        float acc[MT][4];
#pragma unroll
        for (int i = 0; i < MT * 4; ++i) (&acc[0][0])[i] = 0.f;
        for (int it = 0; it < per_tile; ++it) {
            wait_or_note(&full_bar[s], phase, &gave_up);
            if (it * DEEP + deep < k_blocks) {                // (a strip that is not there left the stage as it was: nothing of it is stored)
                const unsigned char* w = ring + (size_t)s * S::STAGE_BYTES + mine * S::W_STRIP + deep * BLOCK_BYTES;
                const unsigned char* a = ring + (size_t)s * S::STAGE_BYTES + S::A_OFF + deep * (MT * 8 * KB);
                const uint4 l0 = *reinterpret_cast<const uint4*>(w + at), h0 = *reinterpret_cast<const uint4*>(w + at + 1024);
                const uint4 l1 = *reinterpret_cast<const uint4*>(w + (at ^ 64)), h1 = *reinterpret_cast<const uint4*>(w + (at ^ 64) + 1024);
                uint4 x0[MT], x1[MT];
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    x0[j] = *reinterpret_cast<const uint4*>(a + j * 1024 + at);
                    x1[j] = *reinterpret_cast<const uint4*>(a + j * 1024 + (at ^ 64));
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) mma_16832(acc[j], l0.x, h0.x, l0.y, h0.y, x0[j].x, x0[j].y);
#pragma unroll
                for (int j = 0; j < MT; ++j) mma_16832(acc[j], l0.z, h0.z, l0.w, h0.w, x0[j].z, x0[j].w);
#pragma unroll
                for (int j = 0; j < MT; ++j) mma_16832(acc[j], l1.x, h1.x, l1.y, h1.y, x1[j].x, x1[j].y);
#pragma unroll
                for (int j = 0; j < MT; ++j) mma_16832(acc[j], l1.z, h1.z, l1.w, h1.w, x1[j].z, x1[j].w);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[s]);
            if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {                        // acc: (row g, columns 2t and 2t + 1), (row g + 8, the same): rows t and t + 4 of a
            red[buf][deep][8 * j + t][mine * STRIP + row] = acc[j][0];
            red[buf][deep][8 * j + t + 4][mine * STRIP + row] = acc[j][1];
            red[buf][deep][8 * j + t][mine * STRIP + row + 8] = acc[j][2];
            red[buf][deep][8 * j + t + 4][mine * STRIP + row + 8] = acc[j][3];
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
#pragma unroll
        for (int o = 0; o < OUTS; ++o) {
            const int i = threadIdx.x + o * 32 * WARPS, m = i / each, c = i % each, col = strip * (each / NS) + c;
            if (m >= e.M || col >= ld) continue;
            const int place = e.gated ? 2 * c - (c & 7) : c;
            float y = 0.f, u = 0.f;
#pragma unroll
            for (int v = 0; v < DEEP; ++v) y += red[buf][v][m][place];
            y = y * ws[o] * am[o] + wb[o];
            if (e.gated) {
#pragma unroll
                for (int v = 0; v < DEEP; ++v) u += red[buf][v][m][place + 8];
                y = activate(y, e.act) * (u * us[o] * am[o] + ub[o]);
            } else {
                y = activate(y, e.act);
            }
            out[(size_t)m * ld + col] = from_f32<TO>(y + to_f32(yr[o]));
        }
    }
    if (threadIdx.x == 0 && gave_up && err) atomicOr(err, VL_DEV_WAIT_EXPIRED | VL_DEV_IN_GEMM_8BIT);
}
}  // namespace few8

// ---- host side --------------------------------------------------------------------------------------
// rows [M, width] in boxes of `box` rows x 128 bytes with the 128-byte swizzle
static int map_rows(CUtensorMap* map, const void* a, int M, int width, int box_rows) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return VL_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)M};
    cuuint64_t strides[1] = {(cuuint64_t)width};
    cuuint32_t box[2] = {(cuuint32_t)KB, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(a), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : VL_ERR_ARGUMENT;
}
// the same rows as (128 columns, rows, blocks of 128 columns): a box brings `deep` blocks of `box_rows` rows, block after block
static int map_row_blocks(CUtensorMap* map, const void* a, int M, int width, int box_rows, int deep) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return VL_ERR_UNSUPPORTED;
    cuuint64_t dims[3] = {(cuuint64_t)KB, (cuuint64_t)M, (cuuint64_t)(width / KB)};
    cuuint64_t strides[2] = {(cuuint64_t)width, (cuuint64_t)KB};
    cuuint32_t box[3] = {(cuuint32_t)KB, (cuuint32_t)box_rows, (cuuint32_t)deep}, estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(a), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : VL_ERR_ARGUMENT;
}
// packed strips in boxes of whole strips x 16 rows x 128 bytes: 128 rows, or fewer, of one block of K, already in the swizzle's order
static int map_strips(CUtensorMap* map, const void* w, int N, int k_blocks, int rows = ROWS) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return VL_ERR_UNSUPPORTED;
    cuuint64_t dims[3] = {(cuuint64_t)KB, (cuuint64_t)STRIP * k_blocks, (cuuint64_t)((N + STRIP - 1) / STRIP)};
    cuuint64_t strides[2] = {(cuuint64_t)KB, (cuuint64_t)STRIP * k_blocks * KB};
    cuuint32_t box[3] = {(cuuint32_t)KB, (cuuint32_t)STRIP, (cuuint32_t)(rows / STRIP)}, estr[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(w), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : VL_ERR_ARGUMENT;
}

static int sm_count() {
    static int num_sms = 0;
    if (!num_sms) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || num_sms <= 0) num_sms = 148;
    }
    return num_sms;
}

// Whether the tiles of the pairs' last round are cut in two (halves of at least 64 rows, a multiple of 32).
static bool halves(int tiles, int bt) {
    const int pairs = sm_count() / 2, last = tiles % pairs;
    return tiles > pairs && last > 0 && 2 * last <= pairs && bt >= 128 && bt % 64 == 0;
}

template <typename TO, int ACT, bool GATED>
static int launch_pair(const void* a, const void* w, const Epilogue& e, int width, int bt, unsigned* err, cudaStream_t s) {
    const size_t smem = (size_t)pair8::STAGES * pair8::STAGE_BYTES + 1024;
    auto kern = pair8::gemm_8bit_pair_kernel<TO, ACT, GATED>;
    // first of all: a thread that has made no call yet has no context, and a tensor map wants one
    cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (ce != cudaSuccess) return (int)ce;
    const int tiles_t = (e.M + bt - 1) / bt, tiles_n = (e.N + 2 * ROWS - 1) / (2 * ROWS);
    const int total = tiles_t * tiles_n, pairs = sm_count() / 2, whole = halves(total, bt) ? total - total % pairs : total, places = 2 * total - whole;
    CUtensorMap map_a, map_half, map_w;
    int rc = map_rows(&map_a, a, e.M, width, bt / 2);
    if (!rc) rc = map_rows(&map_half, a, e.M, width, whole < total ? bt / 4 : bt / 2);
    if (!rc) rc = map_strips(&map_w, w, e.N, width / KB);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (total < pairs ? total : pairs));
    cfg.blockDim = dim3(pair8::NUM_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    // never as a programmatic dependent: see csrc/gemm_tc5_pair.cu
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kern, map_a, map_half, map_w, e, width / KB, bt, whole, places, tiles_t, tiles_n, err);
}

// Which kernel and tile for more than 16 rows: what it would take, in cycles of an SM at 1.85 GHz.  A block of K costs by the rows of a that meet it (an SM takes
// some 64 bytes a cycle in: that paces small tiles, the tensor cores large ones), 1,230 cycles of a copy's way where few stages are in flight; tiles
// run in rounds of the SMs, W comes at the memory's pace, and the two together take the root of the sum of their squares.  Beside it a start (longer for
// a block that leaves no room for the next launch's on its SM), what a further round costs, the epilogue's columns that no products hide, and where K is cut
// a second launch and its bytes.  The numbers were fitted to 311 sizes (17 to 4,096 rows, weights of 16 KB to 178 MB) in every way that this
// function weighs, calls behind one another and in graphs: the choice is on average 0.9 % slower than the fastest way measured, at worst 16 % (3,200 rows
// x 320 -> 768: 6.8 us for 5.8).  512 x 4,096 -> 6,144: one SM a tile of 176 rows 14.0 us, pairs with 192 rows 16.4 (14.9 in a graph).
// overlapped: among launches that start as programmatic dependents with W known as a constant (a decode step) a second launch costs its bytes and little
// else, and a block that has its SM to itself loses nothing; fitted to 113 sizes of 17 to 64 rows, 2.2 % slower than the fastest way measured, by the numbers
// above 6 % (24 x 4,096 -> 6,144 8.1 us for 9.6, 64 x 12,288 -> 4,096 12.8 for 13.7).
// Lower tiles of W, 96 or 112 rows: where two blocks an SM have room for all of them and 128 rows leave SMs with one block beside SMs with two (64 x 4,096
// -> 24,576, 256 tiles for 192: 20.0 us for 21.4 overlapped, 96 rows 21.9 for 23.5 in calls); not for a K of a few blocks (20 x 320 -> 20,032 4.8 for 4.6), and
// tiles of 64 to 16 rows in place of cutting K gain nothing at 20 to 512 rows of twelve weights (a comes in too often).
struct Plan {
    int pair, height, bt, splits, per_sm;
    long long scratch(int M, int N) const { return splits > 1 ? (long long)splits * M * ((N + ROWS - 1) / ROWS * ROWS) : 0; }
};
// A block's stages: what an SM's 228 KB leave it, less 1 KB that the system keeps of it; behind them barriers, a few words and the scales (SPLIT_BESIDE).  A
// product reads 128 rows of W whatever the tile's height: a stage (96 + 32 rows at least) and what lies behind the last one hold them.
constexpr unsigned SPLIT_BESIDE = 2048;
static int split_stages(int height, int bt, int per_sm) {
    return (int)(((per_sm == 2 ? 115712u : 232448u) - SPLIT_BESIDE) / (unsigned)((height + bt) * KB));
}
static Plan plan_of(int M, int N, int k_blocks, bool overlapped) {
    const int sms = sm_count();
    const double stream = (double)N * k_blocks * KB / 3370;
    const auto longer = [](double a, double b) { return a > b ? a : b; };
    const double join = overlapped ? 1180 : 3970, join_part = overlapped ? 263 : 0, alone = overlapped ? 0 : 466;
    Plan best{1, 2 * ROWS, 256, 1, 1};
    double least = -1;
    for (int tall : {256, 224, 192, 160, 128, 96, 64, 32}) {
        const int tiles_t = (M + tall - 1) / tall, each = (M + tiles_t - 1) / tiles_t;
        if (tall >= 128) {
            const int bt = each <= 128 ? 128 : (each + 31) / 32 * 32;
            const long long tiles = (long long)tiles_t * ((N + 2 * ROWS - 1) / (2 * ROWS)), rounds = (tiles + sms / 2 - 1) / (sms / 2);
            const int last = tiles < (1 << 30) && halves((int)tiles, bt) ? bt / 2 : bt;
            const auto step = [&](int rows) { return longer(85 + 2.41 * rows, 417); };
            const double paced = ((double)(rounds - 1) * step(bt) + step(last)) * k_blocks;
            const double cost = 6950 + 4860 * (double)(rounds - 1) + sqrt(paced * paced + stream * stream) + 12.4 * last;
            if (least < 0 || cost < least) { least = cost; best = {1, 2 * ROWS, bt, 1, 1}; }
        }
        const int bt = (each + 15) / 16 * 16;
        const long long tiles = (long long)tiles_t * ((N + ROWS - 1) / ROWS);
        for (int splits = 1; splits <= 8 && (splits == 1 || 2 * splits <= k_blocks + 1) && tiles * splits <= 3 * sms; ++splits) {
            const int rounds = (int)((tiles * splits + sms - 1) / sms);
            // two blocks an SM where there are more blocks than SMs, or little of a in a stage
            for (int per_sm = 1; per_sm <= (bt <= 160 && (rounds > 1 || bt <= 64) ? 2 : 1); ++per_sm) {
                const int turns = (rounds + per_sm - 1) / per_sm, in_flight = split_stages(ROWS, bt, per_sm) * (rounds > 1 ? per_sm : 1);
                const double paced = (double)rounds * ((k_blocks + splits - 1) / splits) * longer(longer(146 + 2.17 * bt, 266), 1230.0 / in_flight);
                const double cost = 6480 + (per_sm == 1 ? alone : 0) + sqrt(paced * paced + stream * stream) + 7.91 * bt * turns + 8430 * (turns - 1) +
                                    (splits > 1 ? join + join_part * splits + 3.5 * splits * M * N / 10000 : 0);
                if (cost < least) { least = cost; best = {0, ROWS, bt, splits, per_sm}; }
            }
        }
    }
    if (!best.pair && best.splits == 1 && best.per_sm == 2 && k_blocks >= 16) {
        const long long tiles_t = (M + best.bt - 1) / best.bt;
        const auto tiles = [&](int height) { return tiles_t * ((N + height - 1) / height); };
        if (tiles(ROWS) > sms)
            for (int height : {112, 96})
                if (tiles(height) <= 2 * sms) best.height = height;
    }
    return best;
}

template <typename TO, int ACT, bool GATED, int PER_SM>
static int launch_split(const void* a, const void* w, const Epilogue& e, int width, int height, int bt, int splits, float* scratch, unsigned* err, cudaStream_t s) {
    const int stages = split_stages(height, bt, PER_SM);
    const size_t smem = (size_t)stages * (unsigned)((height + bt) * KB) + SPLIT_BESIDE;
    auto kern = split8::gemm_8bit_split_kernel<TO, ACT, GATED, PER_SM>;
    cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (ce != cudaSuccess) return (int)ce;
    CUtensorMap map_a, map_w;
    int rc = map_rows(&map_a, a, e.M, width, bt);
    if (!rc) rc = map_strips(&map_w, w, e.N, width / KB, height);
    if (rc) return rc;
    const int tiles_t = (e.M + bt - 1) / bt, tiles_n = (e.N + height - 1) / height;
    rc = vl_launch_waiting(kern, dim3(tiles_t * tiles_n * splits), dim3(split8::NUM_THREADS), smem, s, map_a, map_w, e, width / KB, height, bt, tiles_t, splits,
                           scratch, stages, vl_pdl_enabled() ? 1 : 0, err);
    if (rc || splits == 1) return rc;
    const int cols = GATED ? e.N >> 1 : e.N;
    const bool wide = cols % 4 == 0 && (((uintptr_t)e.out | (uintptr_t)e.residual | (uintptr_t)e.w_scale | (uintptr_t)e.bias) & 15) == 0;
    const dim3 grid(e.M, (cols + 1023) / 1024);
    return wide ? vl_launch_waiting(split8::gemm_8bit_join_kernel<TO, ACT, GATED, true>, grid, dim3(256), 0, s, (const float*)scratch, e, splits)
                : vl_launch_waiting(split8::gemm_8bit_join_kernel<TO, ACT, GATED, false>, grid, dim3(256), 0, s, (const float*)scratch, e, splits);
}
template <typename TO, int MT, int NS, int STAGES, int PER_SM>
static int launch_few(const void* a, const void* w, const Epilogue& e, int width, unsigned* err, cudaStream_t s) {
    const size_t smem = few8::Shape<MT, NS>::smem(STAGES);
    auto kern = few8::gemm_8bit_few_kernel<TO, MT, NS, STAGES, PER_SM>;
    cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (ce != cudaSuccess) return (int)ce;
    CUtensorMap map_a;
    if (int rc = map_row_blocks(&map_a, a, e.M, width, MT * 8, few8::Shape<MT, NS>::DEEP)) return rc;
    const int strips = (e.N + STRIP - 1) / STRIP, tiles = (strips + NS - 1) / NS, places = PER_SM * sm_count();
    // W is a constant to the steps of the engine, which turns the switch on; to anybody else it may be what the kernel in front writes
    return vl_launch_waiting(kern, dim3(tiles < places ? tiles : places), dim3(32 * few8::WARPS + 32), smem, s, map_a, (const unsigned char*)w, e,
                             width / KB, strips, vl_pdl_enabled() ? 1 : 0, err);
}
template <typename TO, int ACT, bool GATED>
static int launch_many(const void* a, const void* w, const Epilogue& e, int width, float* scratch, long long floats, bool overlapped, unsigned* err,
                       cudaStream_t s) {
    const Plan p = plan_of(e.M, e.N, width / KB, overlapped);
    if (p.pair) return launch_pair<TO, ACT, GATED>(a, w, e, width, p.bt, err, s);
    if (p.scratch(e.M, e.N) > (scratch ? floats : 0)) return VL_ERR_ARGUMENT;
    if (p.splits > 1 && ((uintptr_t)scratch & 15)) return VL_ERR_UNSUPPORTED;      // the second launch reads four sums at a time
    return p.per_sm == 2 ? launch_split<TO, ACT, GATED, 2>(a, w, e, width, p.height, p.bt, p.splits, scratch, err, s)
                         : launch_split<TO, ACT, GATED, 1>(a, w, e, width, p.height, p.bt, p.splits, scratch, err, s);
}

template <typename TO>
static int launch(const void* a, const void* w, const Epilogue& e, int width, float* scratch, long long floats, bool overlapped, unsigned* err, cudaStream_t s) {
    // Two blocks an SM.  Up to 8 rows: strips one by one, four stages of 16 + 8 KB.  Up to 16: in twos where that leaves more tiles than SMs, each strip's copy of a
    // being half the bytes then, else one by one with two stages of 16 + 16 KB (a third passes half an SM).  16 rows of 4,096, in twos / one by one, us overlapped:
    // -> 4,096 6.5 / 4.9, -> 6,144 7.4 / 7.7, -> 8,192 7.6 / 8.1, -> 18,432 13.3 / 14.7; where the last round of the twos holds few tiles they lose: -> 10,240
    // 11.6 / 9.4, -> 24,576 18.4 / 17.9.
    if (e.M <= 8) return launch_few<TO, 1, 1, 4, 2>(a, w, e, width, err, s);
    if (e.M <= 16)
        return (e.N + 2 * STRIP - 1) / (2 * STRIP) > sm_count() ? launch_few<TO, 2, 2, 4, 2>(a, w, e, width, err, s) : launch_few<TO, 2, 1, 2, 2>(a, w, e, width, err, s);
    if (e.gated)
        return e.act == ACT_SILU ? launch_many<TO, ACT_SILU, true>(a, w, e, width, scratch, floats, overlapped, err, s)
                                 : launch_many<TO, ACT_RELU, true>(a, w, e, width, scratch, floats, overlapped, err, s);
    switch (e.act) {
        case ACT_NONE: return launch_many<TO, ACT_NONE, false>(a, w, e, width, scratch, floats, overlapped, err, s);
        case ACT_SILU: return launch_many<TO, ACT_SILU, false>(a, w, e, width, scratch, floats, overlapped, err, s);
        case ACT_RELU: return launch_many<TO, ACT_RELU, false>(a, w, e, width, scratch, floats, overlapped, err, s);
        case ACT_RELU2: return launch_many<TO, ACT_RELU2, false>(a, w, e, width, scratch, floats, overlapped, err, s);
        case ACT_TANH: return launch_many<TO, ACT_TANH, false>(a, w, e, width, scratch, floats, overlapped, err, s);
        case ACT_GELU: return launch_many<TO, ACT_GELU, false>(a, w, e, width, scratch, floats, overlapped, err, s);
        default: return VL_ERR_UNSUPPORTED;
    }
}

// What a product of these sizes wants: plan[0] floats of scratch memory; plan[1]: whether it runs as clusters of blocks; plan[2]: w's rows of a tile, 0 for
// few rows of a.  overlapped: whether it is among launches that start as programmatic dependents; the launch is told the same.
extern "C" int vl_gemm_8bit_plan(int M, int N, int width, int overlapped, long long* plan) {
    if (!plan || width <= 0 || width % KB) return VL_ERR_ARGUMENT;
    plan[0] = plan[1] = plan[2] = 0;
    if (M <= 16 || N <= 0) return VL_OK;
    const Plan p = plan_of(M, N, width / KB, overlapped != 0);
    plan[0] = p.scratch(M, N);
    plan[1] = p.pair;
    plan[2] = p.height;
    return VL_OK;
}

extern "C" int vl_gemm_8bit(const void* a, const float* a_scale, const void* w, const float* w_scale, void* out, int out_dtype, const float* bias,
                            const void* residual, int act, int gated, int M, int N, int width, float* scratch, long long floats, int overlapped,
                            unsigned* err, void* stream) {
    if (M <= 0 || N <= 0) return VL_OK;
    if (width <= 0 || width % KB || (gated && N % 16)) return VL_ERR_ARGUMENT;
    if (((uintptr_t)a | (uintptr_t)w) & 15) return VL_ERR_UNSUPPORTED;
    if (gated ? act != ACT_SILU && act != ACT_RELU : act != ACT_NONE && act != ACT_SILU && act != ACT_RELU && act != ACT_RELU2 && act != ACT_TANH && act != ACT_GELU)
        return VL_ERR_UNSUPPORTED;
    const Epilogue e{a_scale, w_scale, bias, residual, out, M, N, act, gated};
    if (out_dtype == VL_BF16) return launch<bf16>(a, w, e, width, scratch, floats, overlapped != 0, err, (cudaStream_t)stream);
    if (out_dtype == VL_F32) return launch<float>(a, w, e, width, scratch, floats, overlapped != 0, err, (cudaStream_t)stream);
    return VL_ERR_UNSUPPORTED;
}
