// Rows in 8 bits (e4m3: 4 bits of exponent, 3 of mantissa, up to 448) with a float32 scale a row, the operand of the
// 8-bit products (gemm_8bit.cu):
//     scale = max |h| / 448,   q = e4m3(h * (448 / max |h|))      so that h ~ q * scale,
// h being a row as it is (vl_rows_8bit) or the RMS norm of a row of the residual stream, the pending delta added first
// (vl_add_rmsnorm_8bit):   x <- x + delta;   h = x / sqrt(mean(x^2) + eps) * w.
// Sums, the norm and the scale are float32; the one rounding to 8 bits is the conversion at the end (round to nearest even).
// A row holds zeros behind its `cols` values, up to `width` columns (a multiple of 128: the products read whole blocks of K).
// A row without a value of 2^-100 or more is a row of zeros (448 / max would overflow).  The largest magnitude is the
// largest bit pattern without its sign, which also carries a NaN through to the scale; an infinity becomes a NaN value.
#include "common.cuh"
#include <cuda_fp8.h>

namespace {
constexpr float TOP = 448.0f;                // e4m3's largest number
constexpr float SMALLEST = 0x1p-100f;

__device__ __forceinline__ float factor_of(float top) { return top >= SMALLEST ? TOP / top : 0.0f; }
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int NT>
__device__ __forceinline__ unsigned block_max(unsigned v, unsigned* scratch) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned t = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) t = max(t, scratch[w]);
    return t;
}
}  // namespace

// One block a row, element by element: any width, any alignment.
template <typename TX, typename TD>
__global__ void __launch_bounds__(256)
rows_8bit_kernel(const TX* x, const TD* __restrict__ delta, const int* __restrict__ rows, const float* __restrict__ w,
                 TX* into, unsigned char* __restrict__ out, float* __restrict__ scale, int cols, int width, float eps) {
    __shared__ float sums[32];
    __shared__ unsigned tops[32];
    pdl_launch_dependents();
    pdl_wait();
    const int r = blockIdx.x, src = rows ? rows[r] : r;
    const TX* xr = x + (size_t)src * cols;
    const TD* dr = delta ? delta + (size_t)src * cols : nullptr;
    float inv = 1.0f;
    if (w) {
        float ss = 0.f;
        for (int i = threadIdx.x; i < cols; i += 256) {
            float v = to_f32(xr[i]);
            if (dr) v += to_f32(dr[i]);
            ss += v * v;
        }
        inv = 1.0f / sqrtf(block_sum<256>(ss, sums) / (float)cols + eps);
    }
    unsigned top = 0;
    for (int i = threadIdx.x; i < cols; i += 256) {
        float v = to_f32(xr[i]);
        if (dr) v += to_f32(dr[i]);
        top = max(top, magnitude(w ? v * inv * w[i] : v));
    }
    top = block_max<256>(top, tops);
    const float f = factor_of(__uint_as_float(top));
    for (int i = threadIdx.x; i < width; i += 256) {
        float h = 0.f;
        if (i < cols) {
            float v = to_f32(xr[i]);
            if (dr) {
                v += to_f32(dr[i]);
                if (!rows) into[(size_t)r * cols + i] = from_f32<TX>(v);
            }
            h = (w ? v * inv * w[i] : v) * f;
        }
        out[(size_t)r * width + i] = __nv_cvt_float_to_fp8(h, __NV_SATFINITE, __NV_E4M3);
    }
    if (threadIdx.x == 0) scale[r] = __uint_as_float(top) / TOP;
}

// e4m3 weights [N, K] to the layout the products read: strips of 16 rows, a strip's blocks of 128 columns one behind the other,
// the eight 16-byte pieces of a block's row exchanged by xor with the row's last three bits.  Zeros fill N up to 16 and K up to 128.
__global__ void __launch_bounds__(128)
pack_8bit_kernel(const unsigned char* __restrict__ w, uint4* __restrict__ out, int N, int K, int k_blocks) {
    const int kb = blockIdx.x, strip = blockIdx.y, row = threadIdx.x >> 3, piece = threadIdx.x & 7;
    const int n = strip * 16 + row, k0 = kb * 128 + piece * 16;
    unsigned v[4] = {0, 0, 0, 0};
    if (n < N)
        for (int i = 0; i < 16 && k0 + i < K; ++i) v[i >> 2] |= (unsigned)w[(size_t)n * K + k0 + i] << (8 * (i & 3));
    out[((size_t)strip * k_blocks + kb) * 128 + row * 8 + (piece ^ (row & 7))] = make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename TX, typename TD>
static int launch_rows(const void* x, const void* delta, const int* rows, const float* w, void* into, void* out, float* scale, int R, int cols,
                       int width, float eps, cudaStream_t s) {
    return vl_launch(rows_8bit_kernel<TX, TD>, dim3(R), dim3(256), 0, s, (const TX*)x, (const TD*)delta, rows, w, (TX*)into,
                     (unsigned char*)out, scale, cols, width, eps);
}

// x float32 [T, cols]; delta float32 or bfloat16 [T, cols] or null; rows null or R row numbers; into: where x + delta goes (x itself
// or other memory; not written with `rows` or without delta)
extern "C" int vl_add_rmsnorm_8bit(const float* x, const void* delta, int delta_dtype, const int* rows, const float* w, float* into, void* out,
                                   float* scale, int R, int cols, int width, float eps, void* stream) {
    if (R <= 0) return VL_OK;
    if (cols <= 0 || width < cols || width % 128 || !w) return VL_ERR_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    if (delta_dtype == VL_BF16) return launch_rows<float, bf16>(x, delta, rows, w, into, out, scale, R, cols, width, eps, s);
    if (delta_dtype == VL_F32) return launch_rows<float, float>(x, delta, rows, w, into, out, scale, R, cols, width, eps, s);
    return VL_ERR_UNSUPPORTED;
}

extern "C" int vl_rows_8bit(const void* x, int dtype, void* out, float* scale, int R, int cols, int width, void* stream) {
    if (R <= 0) return VL_OK;
    if (cols <= 0 || width < cols || width % 128) return VL_ERR_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == VL_BF16) return launch_rows<bf16, bf16>(x, nullptr, nullptr, nullptr, nullptr, out, scale, R, cols, width, 0.f, s);
    if (dtype == VL_F32) return launch_rows<float, float>(x, nullptr, nullptr, nullptr, nullptr, out, scale, R, cols, width, 0.f, s);
    return VL_ERR_UNSUPPORTED;
}

extern "C" int vl_pack_8bit(const void* w, void* out, int N, int K, void* stream) {
    if (N <= 0) return VL_OK;
    if (K <= 0 || (N + 15) / 16 > 65535) return VL_ERR_UNSUPPORTED;
    const int k_blocks = (K + 127) / 128;
    return vl_launch(pack_8bit_kernel, dim3(k_blocks, (N + 15) / 16), dim3(128), 0, (cudaStream_t)stream, (const unsigned char*)w, (uint4*)out,
                     N, K, k_blocks);
}
