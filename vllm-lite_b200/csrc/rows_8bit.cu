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

// Sum and maximum over a block of up to 1,024 threads; `scratch` holds 32 words and is written once.
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return warp_sum(lane < (int)(blockDim.x >> 5) ? scratch[lane] : 0.f);
}
// The same of PIECES values a thread, each of which stands for a thread of a block PIECES times as large: the sum's order, and its bits, are those of that block.
template <int PIECES>
__device__ __forceinline__ float row_sum(const float (&v)[PIECES], float* scratch) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const float sum = warp_sum(v[i]);
        if (lane == 0) scratch[i * warps + (threadIdx.x >> 5)] = sum;
    }
    __syncthreads();
    float all = lane < PIECES * warps ? scratch[lane] : 0.f;
#pragma unroll
    for (int i = 32; i < 32 * PIECES; i += 32) all += i + lane < PIECES * warps ? scratch[i + lane] : 0.f;
    return warp_sum(all);
}
__device__ __forceinline__ unsigned row_max(unsigned v, unsigned* scratch) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < (int)(blockDim.x >> 5) ? scratch[lane] : 0u);
}

// A thread's pieces of a row, zeros behind the row's end.  ALIGNED: rows begin on 16 bytes and hold a multiple of eight values, a piece is eight
// neighbours.  Else they are read value by value, of float32 rows eight that are blockDim.x apart, so that neighbouring threads read neighbours (us,
// neighbours in a thread / apart: 4,096 norms of 1,001 20.2 / 14.3; 2,048 bfloat16 rows of 12,287 23.9 / 44.9).
template <bool ALIGNED, bool APART, int PIECES, typename T>
__device__ __forceinline__ void load_pieces(const T* row, int cols, float (&v)[PIECES][8]) {
    const int step = blockDim.x;
    int at = threadIdx.x;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int c = 8 * (threadIdx.x + i * step);
        if (ALIGNED) {
            if (c < cols) {
                load8(row + c, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
            }
        } else if (APART) {
#pragma unroll
            for (int j = 0; j < 8; ++j, at += step) v[i][j] = at < cols ? to_f32(row[at]) : 0.f;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = c + j < cols ? to_f32(row[c + j]) : 0.f;
        }
    }
}
template <bool ALIGNED, int PIECES>
__device__ __forceinline__ void store_stream(float* row, int cols, const float (&v)[PIECES][8]) {
    if (ALIGNED) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int c = 8 * (threadIdx.x + i * blockDim.x);
            if (c < cols) store8(row + c, v[i]);
        }
    } else {
        const int step = blockDim.x;
        int c = threadIdx.x;
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j, c += step)
                if (c < cols) row[c] = v[i][j];
    }
}
__device__ __forceinline__ void store_8bit(unsigned char* p, const float (&v)[8], float f) {
    unsigned w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * f, v[4 * i + 1] * f), __NV_SATFINITE, __NV_E4M3);
        const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * f, v[4 * i + 3] * f), __NV_SATFINITE, __NV_E4M3);
        w[i] = lo | hi << 16;
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
}  // namespace

// One block a row, the row in registers: a thread holds PIECES pieces of eight neighbouring columns, piece by piece over the block's threads.  Bound by
// the bytes: one read of x (and delta), one write of each result.  The order of the sums is a function of the row's length and of whether rows
// lie on 16-byte boundaries, whatever the block's shape and however many rows there are.
template <typename TX, typename TD, int PIECES, bool NORM, bool ALIGNED>
__global__ void __launch_bounds__(ALIGNED ? 1024 : 512)
rows_8bit_kernel(const TX* x, const TD* __restrict__ delta, const int* __restrict__ rows, const float* __restrict__ w, TX* into,
                 unsigned char* __restrict__ out, float* __restrict__ scale, int cols, int width, float eps) {
    constexpr bool APART = !ALIGNED && sizeof(TX) == 4;
    __shared__ float sums[32 * PIECES];
    __shared__ unsigned tops[32];
    pdl_launch_dependents();
    pdl_wait();
    const int r = blockIdx.x, src = NORM && rows ? rows[r] : r;
    const TX* xr = x + (size_t)src * cols;
    float v[PIECES][8];
    load_pieces<ALIGNED, APART>(xr, cols, v);
    if (NORM) {
        if (delta) {
            float d[PIECES][8];
            load_pieces<ALIGNED, APART>(delta + (size_t)src * cols, cols, d);
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] += d[i][j];
        }
        float g[PIECES][8];
        if (PIECES == 1) load_pieces<ALIGNED, APART>(w, cols, g);    // few rows: one wait for memory less
        if (delta && !rows) store_stream<ALIGNED>(reinterpret_cast<float*>(into) + (size_t)r * cols, cols, v);
        float ss[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            ss[i] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss[i] += v[i][j] * v[i][j];
        }
        const float inv = 1.0f / sqrtf(row_sum(ss, sums) / (float)cols + eps);
        if (PIECES > 1) load_pieces<ALIGNED, APART>(w, cols, g);
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * inv * g[i][j];
    }
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[i][j]));
    top = row_max(top, tops);
    const float f = factor_of(__uint_as_float(top));
    unsigned char* o = out + (size_t)r * width;
    if (!APART) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int c = 8 * (threadIdx.x + i * blockDim.x);
            if (c < width) store_8bit(o + c, v[i], f);
        }
    } else {
        // through shared memory: stores of single bytes cost more than all the rest
        __shared__ uint4 line[APART ? 512 * PIECES / 2 : 1];
        unsigned char* b = reinterpret_cast<unsigned char*>(line);
        const int step = blockDim.x;
        int c = threadIdx.x;
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j, c += step) b[c] = __nv_cvt_float_to_fp8(v[i][j] * f, __NV_SATFINITE, __NV_E4M3);
        __syncthreads();
        for (int p = threadIdx.x; p < width / 8; p += step) reinterpret_cast<uint2*>(o)[p] = reinterpret_cast<const uint2*>(b)[p];
    }
    if (threadIdx.x == 0) scale[r] = __uint_as_float(top) / TOP;
}

// Rows of bfloat16 as they are, kept in registers as they were read, two values a word: half the registers, so that an SM holds more of the long rows
// that feed a down projection (2,048 rows of 25,600: 36.7 us in float32, 28.2 so).
template <int PIECES>
__global__ void __launch_bounds__(1024)
bf16_rows_8bit_kernel(const bf16* __restrict__ x, unsigned char* __restrict__ out, float* __restrict__ scale, int cols, int width) {
    __shared__ unsigned tops[32];
    pdl_launch_dependents();
    pdl_wait();
    const int r = blockIdx.x;
    const uint4* xr = reinterpret_cast<const uint4*>(x + (size_t)r * cols);
    uint4 v[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        v[i] = 8 * c < cols ? xr[c] : make_uint4(0, 0, 0, 0);
    }
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const unsigned w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, max(w[j] << 16 & 0x7fff0000u, w[j] & 0x7fff0000u));
    }
    top = row_max(top, tops);
    const float f = factor_of(__uint_as_float(top));
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int c = 8 * (threadIdx.x + i * blockDim.x);
        const unsigned w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        float h[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[2 * j] = __uint_as_float(w[j] << 16);
            h[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
        if (c < width) store_8bit(out + (size_t)r * width + c, h, f);
    }
    if (threadIdx.x == 0) scale[r] = __uint_as_float(top) / TOP;
}

// The same for rows that no block's registers hold (more than 32,768 columns, 65,536 of bfloat16 rows as they are; off the 16-byte boundaries, or where
// the columns are no multiple of eight, 16,384): three passes, element by element.
template <typename TX, typename TD>
__global__ void __launch_bounds__(1024)
long_rows_8bit_kernel(const TX* x, const TD* __restrict__ delta, const int* __restrict__ rows, const float* __restrict__ w, TX* into,
                      unsigned char* __restrict__ out, float* __restrict__ scale, int cols, int width, float eps) {
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
        for (int i = threadIdx.x; i < cols; i += 1024) {
            const float v = to_f32(xr[i]) + (dr ? to_f32(dr[i]) : 0.f);
            ss += v * v;
        }
        inv = 1.0f / sqrtf(row_sum(ss, sums) / (float)cols + eps);
    }
    unsigned top = 0;
    for (int i = threadIdx.x; i < cols; i += 1024) {
        const float v = to_f32(xr[i]) + (dr ? to_f32(dr[i]) : 0.f);
        top = max(top, magnitude(w ? v * inv * w[i] : v));
    }
    top = row_max(top, tops);
    const float f = factor_of(__uint_as_float(top));
    for (int i = threadIdx.x; i < width; i += 1024) {
        float h = 0.f;
        if (i < cols) {
            const float v = to_f32(xr[i]) + (dr ? to_f32(dr[i]) : 0.f);
            if (dr && !rows) into[(size_t)r * cols + i] = from_f32<TX>(v);
            h = (w ? v * inv * w[i] : v) * f;
        }
        out[(size_t)r * width + i] = __nv_cvt_float_to_fp8(h, __NV_SATFINITE, __NV_E4M3);
    }
    if (threadIdx.x == 0) scale[r] = __uint_as_float(top) / TOP;
}

// e4m3 weights [N, width] to the layout the products read: strips of 16 rows, a strip's blocks of 128 columns one behind the other,
// the eight 16-byte pieces of a block's row exchanged by xor with the row's last three bits.  Rows of zeros fill N up to 16.
__global__ void __launch_bounds__(128)
pack_8bit_kernel(const uint4* __restrict__ w, uint4* __restrict__ out, int N, int k_blocks) {
    pdl_wait();
    const int kb = blockIdx.x, row = threadIdx.x >> 3, piece = threadIdx.x & 7;
    for (int strip = blockIdx.y; strip < (N + 15) / 16; strip += gridDim.y) {
        const int n = strip * 16 + row;
        out[((size_t)strip * k_blocks + kb) * 128 + row * 8 + (piece ^ (row & 7))] =
            n < N ? w[((size_t)n * k_blocks + kb) * 8 + piece] : make_uint4(0, 0, 0, 0);
    }
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

template <typename TX, typename TD, bool NORM>
static int launch_rows(const void* x, const void* delta, const int* rows, const float* w, void* into, void* out, float* scale, int R, int cols,
                       int width, float eps, cudaStream_t s) {
    // whole pieces on 16-byte boundaries: eight values of x are 16 or 32 bytes, of delta and the weight likewise (the results' rows always are)
    const bool aligned = cols % 8 == 0 && (((uintptr_t)x | (uintptr_t)delta | (uintptr_t)w | (uintptr_t)into) & 15) == 0;
    if ((uintptr_t)out & 7) return VL_ERR_UNSUPPORTED;
    // Pieces a thread: the longer the row, the fewer threads it is worth (us, one piece / two / four: rows of 4,096 bfloat16, 4,096 of them 13.4 / 10.7 / -, of 2,048 6.7 / 6.1 / 6.3,
    // of 12,288 - / 30.8 / 25.4, of 25,600 - / - / 35.2, eight 28.2).
    const int pieces = width / 8;
    if (!NORM && sizeof(TX) == 2 && aligned && pieces <= 8192) {
        const int each = pieces <= 128 ? 1 : pieces <= 1024 ? 2 : pieces <= 2048 ? 4 : 8;
        const dim3 threads(((pieces + each - 1) / each + 31) / 32 * 32);
#define ROWS(n) vl_launch_waiting(bf16_rows_8bit_kernel<n>, dim3(R), threads, 0, s, (const bf16*)x, (unsigned char*)out, scale, cols, width)
        switch (each) {
            case 1: return ROWS(1);
            case 2: return ROWS(2);
            case 4: return ROWS(4);
            default: return ROWS(8);
        }
#undef ROWS
    }
    // A norm: one piece while all rows run at once, two where they take turns (us, one piece / two: of 4,096 one row 2.15 / 2.30, 512 rows 6.7 / 6.8, 2,048
    // 20.0 / 18.0, 4,096 34.5 / 31.7; of 5,120 one row 2.40 / 2.52, 512 rows 8.6 / 7.6, 4,096 42.7 / 39.3; four pieces are slower everywhere).
    const bool at_once = pieces <= 1024 && (long long)R * ((pieces + 31) / 32 * 32) <= 2048LL * sm_count();
    const int each = aligned ? ((NORM ? at_once : pieces <= 256) ? 1 : pieces <= 2048 ? 2 : pieces <= 4096 ? 4 : 0)
                             : (pieces <= 256 ? 1 : pieces <= 1024 ? 2 : pieces <= 2048 ? 4 : 0);
    const dim3 threads(each ? ((pieces + each - 1) / each + 31) / 32 * 32 : 1024);
#define ROWS(kernel) vl_launch_waiting(kernel, dim3(R), threads, 0, s, (const TX*)x, (const TD*)delta, rows, w, (TX*)into, (unsigned char*)out, scale, cols, width, eps)
    switch (each) {
        case 1: return aligned ? ROWS((rows_8bit_kernel<TX, TD, 1, NORM, true>)) : ROWS((rows_8bit_kernel<TX, TD, 1, NORM, false>));
        case 2: return aligned ? ROWS((rows_8bit_kernel<TX, TD, 2, NORM, true>)) : ROWS((rows_8bit_kernel<TX, TD, 2, NORM, false>));
        case 4: return aligned ? ROWS((rows_8bit_kernel<TX, TD, 4, NORM, true>)) : ROWS((rows_8bit_kernel<TX, TD, 4, NORM, false>));
        default: return ROWS((long_rows_8bit_kernel<TX, TD>));
    }
#undef ROWS
}

// x float32 [T, cols]; delta float32 or bfloat16 [T, cols] or null; rows null or R row numbers; into: where x + delta goes (x itself
// or other memory; not written with `rows` or without delta)
extern "C" int vl_add_rmsnorm_8bit(const float* x, const void* delta, int delta_dtype, const int* rows, const float* w, float* into, void* out,
                                   float* scale, int R, int cols, int width, float eps, void* stream) {
    if (R <= 0) return VL_OK;
    if (cols <= 0 || width < cols || width % 128 || !w) return VL_ERR_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    if (delta_dtype == VL_BF16) return launch_rows<float, bf16, true>(x, delta, rows, w, into, out, scale, R, cols, width, eps, s);
    if (delta_dtype == VL_F32) return launch_rows<float, float, true>(x, delta, rows, w, into, out, scale, R, cols, width, eps, s);
    return VL_ERR_UNSUPPORTED;
}

extern "C" int vl_rows_8bit(const void* x, int dtype, void* out, float* scale, int R, int cols, int width, void* stream) {
    if (R <= 0) return VL_OK;
    if (cols <= 0 || width < cols || width % 128) return VL_ERR_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == VL_BF16) return launch_rows<bf16, bf16, false>(x, nullptr, nullptr, nullptr, nullptr, out, scale, R, cols, width, 0.f, s);
    if (dtype == VL_F32) return launch_rows<float, float, false>(x, nullptr, nullptr, nullptr, nullptr, out, scale, R, cols, width, 0.f, s);
    return VL_ERR_UNSUPPORTED;
}

extern "C" int vl_pack_8bit(const void* w, void* out, int N, int width, void* stream) {
    if (N <= 0) return VL_OK;
    if (width <= 0 || width % 128) return VL_ERR_ARGUMENT;
    if (((uintptr_t)w | (uintptr_t)out) & 15) return VL_ERR_UNSUPPORTED;
    const int strips = (N + 15) / 16;
    return vl_launch(pack_8bit_kernel, dim3(width / 128, strips < 65535 ? strips : 65535), dim3(128), 0, (cudaStream_t)stream, (const uint4*)w, (uint4*)out,
                     N, width / 128);
}
