// Products of 8-bit rows and 8-bit weights with everything that follows them in one pass:
//     y[m, n] = f(sa[m] sw[n] sum_k a[m, k] w[n, k] + bias[n]) + residual[m, n]
// a [M, width] e4m3 with a scale a row (rows_8bit.cu), w packed e4m3 with a scale an output row (vl_pack_8bit), sums,
// scales, bias, activation and residual in float32, one rounding to out's type.  f: none, a function of one argument, or
// (gated) f(gate) * up with w's rows in blocks of 8 gates and their 8 ups: out then has N / 2 columns.
#include "common.cuh"
#include <cuda_fp8.h>

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

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ACT_SILU: return v / (1.0f + __expf(-v));
        case ACT_RELU: return v < 0.f ? 0.f : v;
        case ACT_RELU2: return v < 0.f ? 0.f : v * v;
        case ACT_TANH: return tanhf(v);
        case ACT_GELU: return 0.5f * v * erfcf(v * -0.70710678118654752f);      // erfc: exact far below zero, where 1 + erf cancels
        default: return v;
    }
}

__device__ __forceinline__ float of_packed(const unsigned char* w, int k_blocks, int n, int k) {
    const int row = n & 15, piece = (k & 127) >> 4;
    const size_t at = ((size_t)(n >> 4) * k_blocks + (k >> 7)) * 2048 + row * 128 + ((piece ^ (row & 7)) << 4) + (k & 15);
    __nv_fp8_e4m3 v;
    v.__x = w[at];
    return float(v);
}

constexpr int TILE = 64, DEPTH = 32;
}  // namespace

// A tile of 64 x 64 by 256 threads, 4 x 4 outputs a thread, float32 multiply-adds.
template <typename TO>
__global__ void __launch_bounds__(256)
gemm_8bit_plain_kernel(const unsigned char* __restrict__ A, const unsigned char* __restrict__ W, Epilogue e, int width) {
    __shared__ float sa[DEPTH][TILE + 1], sw[DEPTH][TILE + 1];
    pdl_launch_dependents();
    pdl_wait();
    const int m0 = blockIdx.y * TILE, n0 = blockIdx.x * TILE, k_blocks = width / 128;
    const int tm = threadIdx.x >> 4, tn = threadIdx.x & 15;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < width; k0 += DEPTH) {
        for (int i = threadIdx.x; i < TILE * DEPTH; i += 256) {
            const int r = i / DEPTH, k = i % DEPTH;
            __nv_fp8_e4m3 v;
            v.__x = m0 + r < e.M ? A[(size_t)(m0 + r) * width + k0 + k] : 0;
            sa[k][r] = float(v);
            sw[k][r] = n0 + r < e.N ? of_packed(W, k_blocks, n0 + r, k0 + k) : 0.f;
        }
        __syncthreads();
        for (int k = 0; k < DEPTH; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += sa[k][tm * 4 + i] * sw[k][tn + 16 * j];
        __syncthreads();
    }
    TO* out = (TO*)e.out;
    const TO* res = (const TO*)e.residual;
    const int out_n = e.gated ? e.N / 2 : e.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + tm * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tn + 16 * j;
            float y = 0.f;
            if (m < e.M && n < e.N) y = acc[i][j] * (e.a_scale[m] * e.w_scale[n]) + (e.bias ? e.bias[n] : 0.f);
            int col = n;
            if (e.gated) {                   // the gate's thread takes its up from eight lanes on
                const float up = __shfl_down_sync(0xffffffffu, y, 8);
                y = activate(y, e.act) * up;
                col = (n >> 4) * 8 + (n & 7);
                if (tn & 8) continue;
            } else {
                y = activate(y, e.act);
            }
            if (m >= e.M || n >= e.N) continue;
            const size_t at = (size_t)m * out_n + col;
            if (res) y += to_f32(res[at]);
            out[at] = from_f32<TO>(y);
        }
    }
}

extern "C" int vl_gemm_8bit(const void* a, const float* a_scale, const void* w, const float* w_scale, void* out, int out_dtype, const float* bias,
                            const void* residual, int act, int gated, int M, int N, int width, unsigned* err, void* stream) {
    if (M <= 0 || N <= 0) return VL_OK;
    if (width <= 0 || width % 128 || (gated && N % 16)) return VL_ERR_ARGUMENT;
    if (((uintptr_t)a | (uintptr_t)w) & 15) return VL_ERR_UNSUPPORTED;
    cudaStream_t s = (cudaStream_t)stream;
    const Epilogue e{a_scale, w_scale, bias, residual, out, M, N, act, gated};
    const dim3 grid((N + TILE - 1) / TILE, (M + TILE - 1) / TILE);
    if (grid.y > 65535) return VL_ERR_UNSUPPORTED;
    if (out_dtype == VL_BF16)
        return vl_launch(gemm_8bit_plain_kernel<bf16>, grid, dim3(256), 0, s, (const unsigned char*)a, (const unsigned char*)w, e, width);
    if (out_dtype == VL_F32)
        return vl_launch(gemm_8bit_plain_kernel<float>, grid, dim3(256), 0, s, (const unsigned char*)a, (const unsigned char*)w, e, width);
    return VL_ERR_UNSUPPORTED;
}
