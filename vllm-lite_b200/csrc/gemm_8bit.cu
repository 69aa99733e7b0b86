// Products of 8-bit rows and 8-bit weights with everything that follows them in one pass:
//     y[m, n] = f(sa[m] sw[n] sum_k a[m, k] w[n, k] + bias[n]) + residual[m, n]
// a [M, width] e4m3 with a scale a row (rows_8bit.cu), w packed e4m3 with a scale an output row (vl_pack_8bit), sums,
// scales, bias, activation and residual in float32, one rounding to out's type.  f: none, a function of one argument, or
// (gated) f(gate) * up with w's rows in blocks of 8 gates and their 8 ups: out then has N / 2 columns.
#include "tc5.cuh"
#include <cuda_fp8.h>

using namespace tc5;

namespace {
enum { ACT_NONE = -1, ACT_SILU = 0, ACT_RELU = 1, ACT_RELU2 = 16, ACT_TANH = 17, ACT_GELU = 18 };

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
__device__ __forceinline__ float activate_gate(float v, int act) { return act == ACT_SILU ? silu(v) : v < 0.f ? 0.f : v; }
__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ACT_SILU: return silu(v);
        case ACT_RELU: return v < 0.f ? 0.f : v;
        case ACT_RELU2: return v < 0.f ? 0.f : v * v;
        case ACT_TANH: return tanhf(v);
        case ACT_GELU: return 0.5f * v * erfcf(v * -0.70710678118654752f);      // erfc: exact far below zero, where 1 + erf cancels
        default: return v;
    }
}

// ---- from an accumulator in TMEM to out ------------------------------------------------------------
// W's rows lie along the accumulator's lanes and the rows of a along its columns: a thread holds CH values of its row n of W, for the
// rows t0 .. t0 + CH - 1 of a.  MODE 0: no activation, 1: of one argument, 2: gated.
// A warp's 32 lanes are 32 neighbouring columns of out, 2 or 4 bytes each.  Two lanes that are neighbours exchange halves, so that each
// stores two neighbouring columns of every second row (`pairs`: out has an even number of columns and begins on 8 bytes); gated, lanes
// 8 apart hold a gate and its up and take turns likewise.
template <typename TO> struct Two;
template <> struct Two<float> {
    static __device__ __forceinline__ void load(const float* p, float& a, float& b) { const float2 v = *reinterpret_cast<const float2*>(p); a = v.x; b = v.y; }
    static __device__ __forceinline__ void store(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
};
template <> struct Two<bf16> {
    static __device__ __forceinline__ void load(const bf16* p, float& a, float& b) {
        const unsigned v = *reinterpret_cast<const unsigned*>(p);
        a = __uint_as_float(v << 16);
        b = __uint_as_float(v & 0xffff0000u);
    }
    static __device__ __forceinline__ void store(bf16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }
};

template <typename TO, int MODE, int CH>
__device__ __forceinline__ void finish(float (&v)[CH], const Epilogue& e, int n, float sw, float b, int t0, bool pairs) {
    const int lane = threadIdx.x & 31;
    const float mine = t0 + (lane & (CH - 1)) < e.M ? e.a_scale[t0 + (lane & (CH - 1))] : 0.f;
    TO* out = reinterpret_cast<TO*>(e.out);
    const TO* res = reinterpret_cast<const TO*>(e.residual);
#pragma unroll
    for (int c = 0; c < CH; ++c) v[c] = v[c] * (__shfl_sync(0xffffffffu, mine, c) * sw) + b;
    if (MODE == 2) {
        const int ld = e.N >> 1, up = (lane >> 3) & 1, col = ((n >> 4) << 3) + (n & 7);
        float r[CH / 2];
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            const int t = t0 + c + up;
            r[c / 2] = res && n < e.N && t < e.M ? to_f32(res[(size_t)t * ld + col]) : 0.f;
        }
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, up ? v[c] : v[c + 1], 8);
            const int t = t0 + c + up;
            const float y = activate_gate(up ? got : v[c], e.act) * (up ? v[c + 1] : got) + r[c / 2];
            if (n < e.N && t < e.M) out[(size_t)t * ld + col] = from_f32<TO>(y);
        }
        return;
    }
    if (MODE == 1) {
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = activate(v[c], e.act);
    }
    const int ld = e.N;
    if (pairs) {
        const int odd = lane & 1, col = n & ~1;
        float r[CH];
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            r[c] = r[c + 1] = 0.f;
            if (res && col < e.N && t0 + c + odd < e.M) Two<TO>::load(res + (size_t)(t0 + c + odd) * ld + col, r[c], r[c + 1]);
        }
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? v[c] : v[c + 1], 1);
            const float lo = odd ? got : v[c], hi = odd ? v[c + 1] : got;
            if (col < e.N && t0 + c + odd < e.M) Two<TO>::store(out + (size_t)(t0 + c + odd) * ld + col, lo + r[c], hi + r[c + 1]);
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if (n < e.N && t0 + c < e.M) {
            const size_t at = (size_t)(t0 + c) * ld + n;
            out[at] = from_f32<TO>(res ? v[c] + to_f32(res[at]) : v[c]);
        }
}

constexpr int STRIP = 16, KB = 128;          // a strip of W, a block of K: 128 bytes
constexpr int ROWS = 128;                    // W's rows of a block
constexpr unsigned W_BYTES = ROWS * KB;

__device__ __forceinline__ bool stores_pairs(const Epilogue& e) { return (e.N & 1) == 0 && (((uintptr_t)e.out | (uintptr_t)e.residual) & 7) == 0; }
}  // namespace

// ---- many rows: two SMs on a tile of 256 rows of W by 256 rows of a ---------------------------------
namespace pair8 {
constexpr int BT = 256, STAGES = 6, NUM_THREADS = 64 + 256;
constexpr unsigned A_BYTES = BT / 2 * KB, STAGE_BYTES = W_BYTES + A_BYTES, TMEM_COLS = 512;

__device__ __forceinline__ void tile_corner(int tile, int tiles_t, int tiles_n, int& t0, int& n0) {
    constexpr int BAND = 8;                                  // pairs that run together share W's tiles in L2
    const int band = tile / (BAND * tiles_n), in_band = tile - band * BAND * tiles_n;
    const int band_rows = min(BAND, tiles_t - band * BAND);
    t0 = (band * BAND + in_band % band_rows) * BT;
    n0 = (in_band / band_rows) * 2 * ROWS;
}

template <typename TO, int MODE>
__global__ void __launch_bounds__(NUM_THREADS, 1)
gemm_8bit_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, Epilogue e, int k_blocks, int tiles_t,
                      int tiles_n, unsigned* err) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full_bar[STAGES], empty_bar[STAGES], acc_full_bar[2], acc_empty_bar[2];
    __shared__ unsigned tmem_base_slot;
    __shared__ int failed;
    const int warp = warp_number();
    const unsigned rank = cluster_rank();
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1, total_tiles = tiles_t * tiles_n;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full_bar[i], 1); mbar_init(&empty_bar[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full_bar[i], 1); mbar_init(&acc_empty_bar[i], 2 * 256); }
        mbar_fence_init();
        failed = 0;
    }
    if (warp == 1) alloc_pair(&tmem_base_slot, TMEM_COLS);
    tc5_fence_before();
    __syncthreads();
    cluster_sync();                                          // the other block's mbarriers exist before anything arrives there
    tc5_fence_after();
    const unsigned tmem_base = tmem_base_slot;

    if (warp == 0) {                                         // ---- copies ----
        const bool lead = elect_one();
        int s = 0;
        unsigned phase = 1;
        bool ok = true;
        for (int tile = pair; tile < total_tiles && ok; tile += num_pairs) {
            int t0, n0;
            tile_corner(tile, tiles_t, tiles_n, t0, n0);
            const int strip = n0 / STRIP + (int)rank * (ROWS / STRIP), row = t0 + (int)rank * (BT / 2);
            for (int kb = 0; kb < k_blocks; ++kb) {
                if (!warp_wait(&empty_bar[s], phase)) {
                    if (lead) atomicOr(&failed, 1);
                    ok = false;
                    break;
                }
                if (lead) {
                    if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * STAGE_BYTES);       // the bytes of both blocks
                    const unsigned bar = map_to_rank(smem_u32(&full_bar[s]), 0);
                    unsigned char* st = smem + (size_t)s * STAGE_BYTES;
                    tma_load_3d_pair(st, &map_w, 0, kb * STRIP, strip, bar);
                    tma_load_2d_pair(st + W_BYTES, &map_a, kb * KB, row, bar);
                }
                if (++s == STAGES) { s = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {                                     // ---- the pair's products ----
            const bool lead = elect_one();
            constexpr unsigned idesc = make_idesc_8bit(2 * ROWS, BT);
            int s = 0, local = 0;
            unsigned phase = 0;
            bool ok = true;
            for (int tile = pair; tile < total_tiles && ok; tile += num_pairs, ++local) {
                const int acc = local & 1;
                if (local >= 2 && !warp_wait(&acc_empty_bar[acc], (unsigned)((local / 2 - 1) & 1))) {
                    if (lead) atomicOr(&failed, 2);
                    break;
                }
                tc5_fence_after();
                const unsigned tmem_c = tmem_base + (unsigned)(acc * BT);
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
    } else {                                                 // ---- epilogue: warps 2..9 ----
        const int quarter = warp & 3, half = (warp - 2) >> 2, lane = threadIdx.x & 31;
        const bool pairs = stores_pairs(e);
        const unsigned freed = map_to_rank(smem_u32(&acc_empty_bar[0]), 0);
        int local = 0;
        for (int tile = pair; tile < total_tiles; tile += num_pairs, ++local) {
            const int acc = local & 1;
            int t0, n0;
            tile_corner(tile, tiles_t, tiles_n, t0, n0);
            const int n = n0 + (int)rank * ROWS + quarter * 32 + lane;
            const float sw = n < e.N ? e.w_scale[n] : 0.f, b = e.bias && n < e.N ? e.bias[n] : 0.f;
            if (!warp_wait(&acc_full_bar[acc], (unsigned)((local / 2) & 1))) {
                atomicOr(&failed, 8);
                break;
            }
            tc5_fence_after();
            const unsigned tmem = tmem_base + ((unsigned)(quarter * 32) << 16) + (unsigned)(acc * BT);
            for (int c0 = half * 32; c0 < BT && t0 + c0 < e.M; c0 += 64) {
                unsigned raw[32];
                float v[32];
                tc5_ld32(tmem + (unsigned)c0, raw);
#pragma unroll
                for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(raw[c]);
                finish<TO, MODE, 32>(v, e, n, sw, b, t0 + c0, pairs);
            }
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
// packed strips in boxes of 8 strips x 16 rows x 128 bytes: 128 rows of one block of K, already in the swizzle's order
static int map_strips(CUtensorMap* map, const void* w, int N, int k_blocks) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return VL_ERR_UNSUPPORTED;
    cuuint64_t dims[3] = {(cuuint64_t)KB, (cuuint64_t)STRIP * k_blocks, (cuuint64_t)((N + STRIP - 1) / STRIP)};
    cuuint64_t strides[2] = {(cuuint64_t)KB, (cuuint64_t)STRIP * k_blocks * KB};
    cuuint32_t box[3] = {(cuuint32_t)KB, (cuuint32_t)STRIP, (cuuint32_t)(ROWS / STRIP)}, estr[3] = {1, 1, 1};
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

template <typename TO, int MODE>
static int launch_pair(const void* a, const void* w, const Epilogue& e, int width, unsigned* err, cudaStream_t s) {
    const size_t smem = (size_t)pair8::STAGES * pair8::STAGE_BYTES + 1024;
    auto kern = pair8::gemm_8bit_pair_kernel<TO, MODE>;
    // first of all: a thread that has made no call yet has no context, and a tensor map wants one
    cudaError_t ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (ce != cudaSuccess) return (int)ce;
    CUtensorMap map_a, map_w;
    int rc = map_rows(&map_a, a, e.M, width, pair8::BT / 2);
    if (!rc) rc = map_strips(&map_w, w, e.N, width / KB);
    if (rc) return rc;
    const int tiles_t = (e.M + pair8::BT - 1) / pair8::BT, tiles_n = (e.N + 2 * ROWS - 1) / (2 * ROWS);
    const int total = tiles_t * tiles_n, pairs = sm_count() / 2;
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
    return (int)cudaLaunchKernelEx(&cfg, kern, map_a, map_w, e, width / KB, tiles_t, tiles_n, err);
}

template <typename TO>
static int launch(const void* a, const void* w, const Epilogue& e, int width, unsigned* err, cudaStream_t s) {
    if (e.gated) return launch_pair<TO, 2>(a, w, e, width, err, s);
    if (e.act != ACT_NONE) return launch_pair<TO, 1>(a, w, e, width, err, s);
    return launch_pair<TO, 0>(a, w, e, width, err, s);
}

extern "C" int vl_gemm_8bit(const void* a, const float* a_scale, const void* w, const float* w_scale, void* out, int out_dtype, const float* bias,
                            const void* residual, int act, int gated, int M, int N, int width, unsigned* err, void* stream) {
    if (M <= 0 || N <= 0) return VL_OK;
    if (width <= 0 || width % KB || (gated && N % 16)) return VL_ERR_ARGUMENT;
    if (((uintptr_t)a | (uintptr_t)w) & 15) return VL_ERR_UNSUPPORTED;
    const Epilogue e{a_scale, w_scale, bias, residual, out, M, N, act, gated};
    if (out_dtype == VL_BF16) return launch<bf16>(a, w, e, width, err, (cudaStream_t)stream);
    if (out_dtype == VL_F32) return launch<float>(a, w, e, width, err, (cudaStream_t)stream);
    return VL_ERR_UNSUPPORTED;
}
