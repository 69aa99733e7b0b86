// Head norm and rotation of a step's queries and keys, and the write of its keys and values into pages of 8 bits, in one launch.
//
//   q_head, k_head <- head / sqrt(mean(head^2) + eps) * w                                        (optional)
//   pairs (x[i], x[i + rot/2]) of the first `rot` features turned by the angle pos * inv_freq[i]      (optional)
//   q to q_out (or in place); k and v to the pages of csrc/cache_8bit.cuh: value = e4m3(x / s), s the page's and KV head's scale.
//
// A block of the first kind takes one page of one request, one KV head, and the keys or the values: the step's new rows of that page (up to
// 64 a pass in registers, a warp a row), their largest |x|, and with it and the scale of the rows that were there the new scale; then the
// rows are written, and where the scale has grown the page's earlier rows are read, multiplied by the quotient of the scales (a power of
// two) and written back.  A page's rows belong to one request and a request's tokens follow one another, so one block sees all that
// a page gets and nothing is exchanged between blocks.  Which page of which request a block takes follows from a sum over the requests
// that every block makes itself.  A block of the second kind gives each of its warps a token and some of its query heads.
//
// Angles: pos * inv_freq in float32 is off by up to 2^-24 of itself, at position 100,000 by 0.006; the product's error, which one fma
// gives, is added to first order, so that sines and cosines are those of the exact product.
// While dependent launches are on, positions and slots are read before the wait for the kernel ahead, as the other head work does (csrc/common.cuh).
#include "cache_8bit.cuh"

using namespace cache8;

namespace {
constexpr int NT = 256, WARPS = NT / 32;

// One head's row in a warp's registers: a lane holds pairs of neighbouring features of the rotated part's first half, their
// partners in the second half, and pairs of the features behind the rotated part.
template <int MAXHD>
struct Row {
    static constexpr int UR = MAXHD / 128, UT = MAXHD / 64;
    float2 a[UR], b[UR], t[UT];

    __device__ __forceinline__ void load(const bf16* src, int lane, int hd, int rot) {
        const int half = rot / 2;
#pragma unroll
        for (int k = 0; k < UR; ++k) {
            const int i = 2 * (lane + 32 * k);
            a[k] = b[k] = make_float2(0.f, 0.f);
            if (i < half) {
                a[k] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src + i));
                b[k] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src + i + half));
            }
        }
#pragma unroll
        for (int k = 0; k < UT; ++k) {
            const int i = rot + 2 * (lane + 32 * k);
            t[k] = i < hd ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src + i)) : make_float2(0.f, 0.f);
        }
    }
    __device__ __forceinline__ void norm(const float* w, float eps, int lane, int hd, int rot) {
        const int half = rot / 2;
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < UR; ++k) ss += a[k].x * a[k].x + a[k].y * a[k].y + b[k].x * b[k].x + b[k].y * b[k].y;
#pragma unroll
        for (int k = 0; k < UT; ++k) ss += t[k].x * t[k].x + t[k].y * t[k].y;
        ss = warp_sum(ss);
        const float inv = 1.0f / sqrtf(ss / (float)hd + eps);
#pragma unroll
        for (int k = 0; k < UR; ++k) {
            const int i = 2 * (lane + 32 * k);
            if (i < half) {
                a[k].x *= inv * w[i]; a[k].y *= inv * w[i + 1];
                b[k].x *= inv * w[i + half]; b[k].y *= inv * w[i + half + 1];
            }
        }
#pragma unroll
        for (int k = 0; k < UT; ++k) {
            const int i = rot + 2 * (lane + 32 * k);
            if (i < hd) { t[k].x *= inv * w[i]; t[k].y *= inv * w[i + 1]; }
        }
    }
    // the sine and cosine of this lane's pairs at a position: (cos, sin) of the pair's two angles
    static __device__ __forceinline__ void angles(float4 (&cs)[UR], int pos, const float* inv_freq, int lane, int rot) {
        const float p = (float)pos;
#pragma unroll
        for (int k = 0; k < UR; ++k) {
            const int i = 2 * (lane + 32 * k);
            cs[k] = make_float4(1.f, 0.f, 1.f, 0.f);
            if (i < rot / 2) {
                float* out = &cs[k].x;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float f = inv_freq[i + j], angle = p * f, left = fmaf(p, f, -angle);
                    float s, c;
                    sincosf(angle, &s, &c);
                    out[2 * j] = fmaf(-left, s, c);
                    out[2 * j + 1] = fmaf(left, c, s);
                }
            }
        }
    }
    __device__ __forceinline__ void turn(const float4 (&cs)[UR]) {
#pragma unroll
        for (int k = 0; k < UR; ++k) {
            const float2 x = a[k], y = b[k];
            a[k] = make_float2(x.x * cs[k].x - y.x * cs[k].y, x.y * cs[k].z - y.y * cs[k].w);
            b[k] = make_float2(y.x * cs[k].x + x.x * cs[k].y, y.y * cs[k].z + x.y * cs[k].w);
        }
    }
    // the largest |x| by its bits: NaN and infinities above all numbers
    __device__ __forceinline__ unsigned top() const {
        unsigned m = 0;
        auto take = [&](float2 v) { m = max(m, max(__float_as_uint(fabsf(v.x)), __float_as_uint(fabsf(v.y)))); };
#pragma unroll
        for (int k = 0; k < UR; ++k) { take(a[k]); take(b[k]); }
#pragma unroll
        for (int k = 0; k < UT; ++k) take(t[k]);
        return m;
    }
    template <typename Store>
    __device__ __forceinline__ void each(int lane, int hd, int rot, Store store) const {
        const int half = rot / 2;
#pragma unroll
        for (int k = 0; k < UR; ++k) {
            const int i = 2 * (lane + 32 * k);
            if (i < half) { store(i, a[k]); store(i + half, b[k]); }
        }
#pragma unroll
        for (int k = 0; k < UT; ++k) {
            const int i = rot + 2 * (lane + 32 * k);
            if (i < hd) store(i, t[k]);
        }
    }
};

// sixteen e4m3 values times a power of two
__device__ __forceinline__ uint4 times(uint4 v, float f) {
    unsigned* w = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned lo = half2_low(w[i]), hi = half2_high(w[i]);
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        w[i] = (unsigned)to_e4m3x2(x.x * f, x.y * f) | ((unsigned)to_e4m3x2(y.x * f, y.y * f) << 16);
    }
    return v;
}
}  // namespace

template <int MAXHD>
__global__ void __launch_bounds__(NT)
qk_norm_rope_write_8bit_kernel(const bf16* qkv, int row_stride, bf16* q_out, int q_stride, const int* __restrict__ positions,
                               const int* __restrict__ slots, const int* __restrict__ cu, int B, const float* __restrict__ qw,
                               const float* __restrict__ kw, float eps, const float* __restrict__ inv_freq, int rot, unsigned char* kcache,
                               unsigned char* vcache, float* kscale, float* vscale, int T, int nq, int nkv, int hd, int page_size, int num_pages,
                               unsigned* err, int page_blocks, int heads_a_warp, int early) {
    constexpr int ROWS = MAXHD <= 128 ? 8 : 4;               // rows a warp holds
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    if (!early) pdl_wait();
    if ((int)blockIdx.x >= page_blocks) {                    // ---- queries ----
        const int groups = (nq + heads_a_warp - 1) / heads_a_warp;
        const long long unit = (long long)((int)blockIdx.x - page_blocks) * WARPS + warp;
        const int tok = (int)(unit / groups), h0 = (int)(unit - (long long)tok * groups) * heads_a_warp;
        if (tok >= T) return;
        const int turned = inv_freq ? rot : 0;
        float4 cs[Row<MAXHD>::UR];
        if (inv_freq) Row<MAXHD>::angles(cs, positions[tok], inv_freq, lane, rot);
        pdl_wait();
        const bf16* src = qkv + (size_t)tok * row_stride;
        bf16* dst = q_out + (size_t)tok * q_stride;
        const int h1 = min(nq, h0 + heads_a_warp);
        for (int h = h0; h < h1; h += 2) {                   // two heads at a time: the loads of one beside the arithmetic of the other
            Row<MAXHD> r[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (h + u < h1) r[u].load(src + (size_t)(h + u) * hd, lane, hd, turned);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (h + u >= h1) continue;
                if (qw) r[u].norm(qw, eps, lane, hd, turned);
                if (inv_freq) r[u].turn(cs);
                bf16* o = dst + (size_t)(h + u) * hd;
                r[u].each(lane, hd, turned, [&](int i, float2 v) {
                    *reinterpret_cast<__nv_bfloat162*>(o + i) = __floats2bfloat162_rn(v.x, v.y);
                });
            }
        }
        return;
    }

    // ---- a page of keys or values ----
    __shared__ int s_sum[WARPS], s_req, s_visit;
    __shared__ unsigned s_top[WARPS];
    const bool values = blockIdx.x & 1;
    const int kvh = (int)(blockIdx.x >> 1) % nkv, visit = (int)(blockIdx.x >> 1) / nkv;
    if (threadIdx.x == 0) s_req = -1;
    __syncthreads();
    for (int b0 = 0, before = 0; b0 < B; b0 += NT) {         // the request whose pages the launch's page number `visit` falls into
        const int b = b0 + threadIdx.x;
        int n = 0;
        if (b < B) {
            const int lo = cu[b], hi = cu[b + 1];
            if (lo >= 0 && lo < hi && hi <= T) {
                const int p = positions[lo];
                n = p < 0 ? 0 : (p % page_size + hi - lo - 1) / page_size + 1;
            }
        }
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
        if (lane == 31) s_sum[warp] = x;
        __syncthreads();
        for (int w = 0; w < warp; ++w) x += s_sum[w];
        int all = 0;
        for (int w = 0; w < WARPS; ++w) all += s_sum[w];
        x += before;
        if (visit < x && visit >= x - n) { s_req = b; s_visit = visit - (x - n); }
        before += all;
        __syncthreads();
        if (before > visit) break;
    }
    const int req = s_req;
    if (req < 0) return;                                     // the launch has a block for every page that there could be
    const int lo = cu[req], off = positions[lo] % page_size, skip = s_visit ? s_visit * page_size - off : 0;
    const int row0 = s_visit ? 0 : off, tok0 = lo + skip, n = min(page_size - row0, cu[req + 1] - tok0);
    const int slot0 = slots[tok0];
    if (slot0 < 0) return;                                   // (a call that reads another call's cache, a padded token)
    const int page = slot0 / page_size;
    if (page >= num_pages || slot0 - page * page_size != row0) {
        if (threadIdx.x == 0 && err) atomicOr(err, VL_DEV_BAD_SLOT);
        return;
    }
    const size_t head = (size_t)page * nkv + kvh;
    unsigned char* cache = (values ? vcache : kcache) + head * page_size * hd;
    float* scale = (values ? vscale : kscale) + head;
    const int turned = values || !inv_freq ? 0 : rot;
    const float* w = values ? nullptr : kw;
    const bf16* src = qkv + (size_t)(nq + (values ? nkv : 0) + kvh) * hd;
    pdl_wait();                                              // qkv comes from the kernel before
    const float old = row0 ? *scale : 0.f;
    Row<MAXHD> r[ROWS];
    bool mine[ROWS];
    unsigned top = 0, strange = 0;
    auto take = [&](int base) {                              // this warp's rows of the pass that begins with row `base`
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const int i = base + u * WARPS + warp;
            mine[u] = i < n;
            if (mine[u] && slots[tok0 + i] != slot0 + i) { mine[u] = false; strange = 1; }
            if (mine[u]) r[u].load(src + (size_t)(tok0 + i) * row_stride, lane, hd, turned);
        }
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (!mine[u]) continue;
            if (w) r[u].norm(w, eps, lane, hd, turned);
            if (turned) {
                float4 cs[Row<MAXHD>::UR];
                Row<MAXHD>::angles(cs, positions[tok0 + base + u * WARPS + warp], inv_freq, lane, rot);
                r[u].turn(cs);
            }
        }
    };
    constexpr int PASS = ROWS * WARPS;
    const int last = (n - 1) / PASS * PASS;
    for (int base = 0; base <= last; base += PASS) {
        take(base);
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (mine[u]) top = max(top, r[u].top());
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[warp] = top;
    if (strange && lane == 0 && err) atomicOr(err, VL_DEV_BAD_SLOT);
    __syncthreads();
    for (int i = 0; i < WARPS; ++i) top = max(top, s_top[i]);
    float now = scale_of(top);
    if (row0) now = old == old && now == now ? fmaxf(old, now) : __uint_as_float(0x7fc00000u);
    const float inv = inverse_of(now);
    // Whole passes that registers no longer hold are made again, the last one first (pages of more than 64 rows, heads beyond 128).
    for (int base = last; base >= 0; base -= PASS) {
        if (base != last) take(base);
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (!mine[u]) continue;
            unsigned char* dst = cache + (size_t)(row0 + base + u * WARPS + warp) * hd;
            r[u].each(lane, hd, turned, [&](int i, float2 v) { *reinterpret_cast<unsigned short*>(dst + i) = to_e4m3x2(v.x * inv, v.y * inv); });
        }
    }
    if (row0 && now > old) {                                 // (false for NaN: rows under a scale that is none need no other)
        const float f = old * inv;
        uint4* rows = reinterpret_cast<uint4*>(cache);
        for (int i = threadIdx.x; i < row0 * hd / 16; i += NT) rows[i] = times(rows[i], f);
    }
    if (threadIdx.x == 0) *scale = now;
}

// qkv [T, row_stride] bfloat16 = q | k | v heads of hd features; q_out [T, q_stride] (may be qkv).  Tokens cu[b] .. cu[b + 1] are those of
// request b at consecutive positions; slots [T] = page * page_size + position % page_size, negative: not written; null: no cache at all.
// Caches [pages, nkv, page_size, hd] e4m3, scales [pages, nkv].
extern "C" int vl_qk_norm_rope_write_8bit(const void* qkv, int row_stride, void* q_out, int q_stride, const int* positions, const int* slots,
                                          const int* cu, int B, const float* qw, const float* kw, float eps, const float* inv_freq, int rot,
                                          void* kcache, void* vcache, float* kscale, float* vscale, int T, int nq, int nkv, int hd, int page_size,
                                          int num_pages, unsigned* err, void* stream) {
    if (T <= 0) return VL_OK;
    if (hd <= 0 || hd > 256 || hd % 16 || rot < 0 || rot > hd || rot % 4) return VL_ERR_UNSUPPORTED;
    if (nq <= 0 || nkv <= 0 || B < 0 || row_stride < (nq + 2 * nkv) * hd || row_stride % 2 || q_stride < nq * hd || q_stride % 2) return VL_ERR_ARGUMENT;
    if (slots && (page_size <= 0 || num_pages <= 0 || !cu || !kcache || !vcache || !kscale || !vscale)) return VL_ERR_ARGUMENT;
    if ((((uintptr_t)qkv | (uintptr_t)q_out) & 3) || (((uintptr_t)kcache | (uintptr_t)vcache) & 15)) return VL_ERR_ARGUMENT;
    if (slots && (long long)num_pages * page_size >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
    // pages that B requests of T tokens can reach: full ones and one broken at each end
    const long long pages = slots ? (T < (long long)T / page_size + 2ll * B ? T : (long long)T / page_size + 2ll * B) : 0;
    const int heads_a_warp = T >= 256 ? 8 : (T >= 32 ? 4 : 2);
    const long long units = (long long)T * ((nq + heads_a_warp - 1) / heads_a_warp), blocks = pages * nkv * 2 + (units + WARPS - 1) / WARPS;
    if (blocks >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
    auto kernel = hd <= 128 ? qk_norm_rope_write_8bit_kernel<128> : qk_norm_rope_write_8bit_kernel<256>;
    return vl_launch_waiting(kernel, dim3((unsigned)blocks), dim3(NT), 0, (cudaStream_t)stream, (const bf16*)qkv, row_stride, (bf16*)q_out, q_stride,
                     positions, slots, cu, B, qw, kw, eps, inv_freq, rot, (unsigned char*)kcache, (unsigned char*)vcache, kscale, vscale, T, nq, nkv,
                     hd, page_size, num_pages, err, (int)(pages * nkv * 2), heads_a_warp, (int)vl_pdl_enabled());
}
