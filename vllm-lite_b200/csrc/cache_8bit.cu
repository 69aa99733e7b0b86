// Head norm and rotation of a step's queries and keys, and the write of its keys and values into pages of 8 bits, in one launch.
//
//   q_head, k_head <- head / sqrt(mean(head^2) + eps) * w                                        (optional)
//   pairs (x[i], x[i + rot/2]) of the first `rot` features turned by the angle pos * inv_freq[i]      (optional)
//   q to q_out (or in place); k and v to the pages of csrc/cache_8bit.cuh: value = e4m3(x / s), s the page's and KV head's scale.
//
// A page's rows belong to one request and a request's tokens follow one another, so one block sees all that a page gets of one KV head's keys or
// values, and nothing is exchanged between blocks: it takes the step's new rows of that page, their largest |x|, and with it and the scale of the rows
// that were there the new scale; then the rows are written, and where the scale has grown the page's earlier rows (and those between that are not written) are read, multiplied by
// the quotient of the scales (a power of two) and written back.  Which page of which request a block takes follows from a sum over the requests that every block makes itself.  Other blocks
// take the queries.  Three kernels:
//   singles: as many tokens as requests (a decode step), a warp a token and head, no sums over requests;
//   wide:    heads of 32, 64, 128 or 256 features that are rotated as a whole or not at all: 16-byte accesses, hd / 16 lanes a row, angles of a
//            page's rows once for several heads;
//   narrow:  any other head, a warp a row, 4-byte accesses.
//
// Measured in a graph: 64 single tokens of 32 + 2 x 8 heads of 128 4.4 us, 4.9 with q in place (a block a page took 16.4, most of it in blocks of one row); a portion of
// 4,096 tokens at position 700 27.8 us, 92 MB at 3.3 TB/s (through the narrow kernel, heads of 96 108 us, heads of 128 of which 64 features turn 112); five portions of 77 with
// heads of 80 and pages of 16 6.9 us.  Bound by latencies: single tokens by loads behind
// one another (position and slot, the scale, the row, the page's rows where a scale grows), a portion by the loads of a page's rows and the barrier before its scale is known.
//
// Angles are pos * inv_freq as a number of turns in double precision, of which the fraction alone is left (in float32 the product is off by up to 2^-24 of
// itself, at position 100,000 by 0.006): sines and cosines are those of the exact product to float32's own rounding.
// While dependent launches are on, positions and slots are read before the wait for the kernel ahead, as the other head work does (csrc/common.cuh).
#include "cache_8bit.cuh"

using namespace cache8;

namespace {
constexpr int NT = 256, WARPS = NT / 32;

__device__ __forceinline__ void sine_cosine(int pos, float freq, float* s, float* c) {
    double turns = (double)pos * ((double)freq * 0.15915494309189535);
    turns -= rint(turns);
    sincospif((float)(turns + turns), s, c);
}

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
#pragma unroll
        for (int k = 0; k < UR; ++k) {
            const int i = 2 * (lane + 32 * k);
            cs[k] = make_float4(1.f, 0.f, 1.f, 0.f);
            if (i < rot / 2) {
                sine_cosine(pos, inv_freq[i], &cs[k].y, &cs[k].x);
                sine_cosine(pos, inv_freq[i + 1], &cs[k].w, &cs[k].z);
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

struct Step {                                          // what every kernel is given
    const bf16* qkv; int row_stride; bf16* q_out; int q_stride;
    const int* positions; const int* slots; const int* cu; int B;
    const float* qw; const float* kw; float eps; const float* inv_freq; int rot;
    unsigned char* kcache; unsigned char* vcache; float* kscale; float* vscale;
    int T, nq, nkv, hd, page_size, num_pages; unsigned* err;
    int page_blocks, heads_a_warp, heads_a_block, early;
};

// The step's new rows of one page: tokens tok0 .. tok0 + n - 1 into rows row0 .., slots from slot0 on; n 0: none that the block may write.  Tokens of a negative
// slot are left out; `held`: the rows ahead of the first one that is written (0: the page begins anew).
struct Visit { int tok0, row0, n, slot0, page, held; };

// What the launch's page number `visit` is; all threads of the block call it.  Which request it falls into: a sum over the requests, a request a thread.
__device__ __forceinline__ Visit find_visit(const Step& st, int visit) {
    __shared__ int s_sum[WARPS], s_req, s_visit;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Visit v = {0, 0, 0, 0, 0, 0};
    if (threadIdx.x == 0) s_req = -1;
    __syncthreads();
    for (int b0 = 0, before = 0; b0 < st.B; b0 += NT) {
        const int b = b0 + threadIdx.x;
        int n = 0;
        if (b < st.B) {
            const int lo = st.cu[b], hi = st.cu[b + 1];
            if (lo >= 0 && lo < hi && hi <= st.T) {
                const int p = st.positions[lo];
                n = p < 0 ? 0 : (p % st.page_size + hi - lo - 1) / st.page_size + 1;
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
    if (req < 0) return v;                                   // the launch has a block for every page that there could be
    const int lo = st.cu[req], off = st.positions[lo] % st.page_size, skip = s_visit ? s_visit * st.page_size - off : 0;
    v.row0 = s_visit ? 0 : off;
    v.tok0 = lo + skip;
    const int n = min(st.page_size - v.row0, st.cu[req + 1] - v.tok0);
    int ahead = 0;
    v.slot0 = st.slots[v.tok0];
#pragma unroll 1
    while (v.slot0 < 0 && ++ahead < n) v.slot0 = st.slots[v.tok0 + ahead];
    if (v.slot0 < 0) return v;                               // (none of the page's tokens is written)
    v.slot0 -= ahead;
    v.held = v.row0 + ahead;
    v.page = v.slot0 / st.page_size;
    if (v.page >= st.num_pages || v.slot0 - v.page * st.page_size != v.row0) {
        if (threadIdx.x == 0 && st.err) atomicOr(st.err, VL_DEV_BAD_SLOT);
        return v;
    }
    v.n = n;
    return v;
}

// the scale of a page whose new rows' largest |x| has the bits `top`, and that held rows before (held > 0) under `old`
__device__ __forceinline__ float new_scale(unsigned top, int held, float old) {
    const float now = scale_of(top);
    if (!held) return now;
    return old == old && now == now ? fmaxf(old, now) : __uint_as_float(0x7fc00000u);
}
// `bytes` bytes of a page moved to a scale that has grown (f: old / new), by `count` threads
__device__ __forceinline__ void move_rows(unsigned char* cache, int bytes, float f, int thread, int count) {
    uint4* rows = reinterpret_cast<uint4*>(cache);
    for (int i = thread; i < bytes / 16; i += count) rows[i] = times(rows[i], f);
}

// Some query heads of one token, a warp.
template <int MAXHD>
__device__ __forceinline__ void query_heads(const Step& st, int tok, int h0, int h1) {
    const int lane = threadIdx.x & 31, turned = st.inv_freq ? st.rot : 0, hd = st.hd;
    float4 cs[Row<MAXHD>::UR];
    if (st.inv_freq) Row<MAXHD>::angles(cs, st.positions[tok], st.inv_freq, lane, st.rot);
    pdl_wait();
    const bf16* src = st.qkv + (size_t)tok * st.row_stride;
    bf16* dst = st.q_out + (size_t)tok * st.q_stride;
    for (int h = h0; h < h1; h += 2) {                       // two heads at a time: the loads of one beside the arithmetic of the other
        Row<MAXHD> r[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (h + u < h1) r[u].load(src + (size_t)(h + u) * hd, lane, hd, turned);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (h + u >= h1) continue;
            if (st.qw) r[u].norm(st.qw, st.eps, lane, hd, turned);
            if (st.inv_freq) r[u].turn(cs);
            bf16* o = dst + (size_t)(h + u) * hd;
            r[u].each(lane, hd, turned, [&](int i, float2 v) { *reinterpret_cast<__nv_bfloat162*>(o + i) = __floats2bfloat162_rn(v.x, v.y); });
        }
    }
}
}  // namespace

// As many tokens as requests, one each as a rule: a warp a token and key or value head, or a token and heads_a_warp query heads.
template <int MAXHD>
__global__ void __launch_bounds__(NT)
write_8bit_singles_kernel(const __grid_constant__ Step st) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = st.hd;
    pdl_launch_dependents();
    if (!st.early) pdl_wait();
    const int pages = st.slots ? 2 * st.nkv : 0, groups = (st.nq + st.heads_a_warp - 1) / st.heads_a_warp;
    const long long unit = (long long)blockIdx.x * WARPS + warp;
    const int tok = (int)(unit / (pages + groups)), u = (int)(unit - (long long)tok * (pages + groups));
    if (tok >= st.T) return;
    if (u >= pages) {
        query_heads<MAXHD>(st, tok, (u - pages) * st.heads_a_warp, min(st.nq, (u - pages + 1) * st.heads_a_warp));
        return;
    }
    const int pos = st.positions[tok], c0 = st.cu[tok], c1 = st.cu[tok + 1];
    int slot = st.slots[tok], n = 1, ahead = 0;
    if (pos < 0) return;
    const int row0 = pos % st.page_size;
    // as many tokens as requests, but not one each: the first token of a page takes the page's others, and looks for the first that is written
    if (__builtin_expect(c0 != tok || c1 != tok + 1, 0)) {
        int b = 0;
#pragma unroll 1
        for (int step = 1 << 30; step; step >>= 1)           // the last request that begins at this token or before
            if (b + step < st.B && st.cu[b + step] <= tok) b += step;
        const int lo = st.cu[b], hi = st.cu[b + 1];
        if (lo < 0 || lo > tok || hi <= tok || hi > st.T || (lo != tok && row0)) return;           // (padding, or not the first)
        n = min(st.page_size - row0, hi - tok);
#pragma unroll 1
        while (slot < 0 && ++ahead < n) slot = st.slots[tok + ahead];
    }
    if (slot < 0) return;
    slot -= ahead;
    const int page = slot / st.page_size;
    if (page >= st.num_pages || slot - page * st.page_size != row0) {
        if (lane == 0 && u == 0 && st.err) atomicOr(st.err, VL_DEV_BAD_SLOT);
        return;
    }
    const bool values = u & 1;
    const int kvh = u >> 1, turned = values || !st.inv_freq ? 0 : st.rot, held = row0 + ahead;
    const size_t head = (size_t)page * st.nkv + kvh;
    unsigned char* cache = (values ? st.vcache : st.kcache) + head * st.page_size * hd;
    float* scale = (values ? st.vscale : st.kscale) + head;
    // Two passes over the rows, one behind the other in the same code; a single row stays in registers in between.  (With the rare case in code of its own, unrolled
    // or called, each layer of a step took 4 us more: decode at batch 1 303 tokens/s, 318 so.)
    Row<MAXHD> r;
    unsigned top = 0;
    float old = 0.f, now = 0.f, inv = 0.f;
#pragma unroll 1
    for (int k = 0; k < 2 * n; ++k) {
        const int i = k < n ? k : k - n;
        if (k == n) {
            now = new_scale(__reduce_max_sync(0xffffffffu, top), held, old);
            inv = inverse_of(now);
        }
        if (__builtin_expect(n > 1, 0)) {
            const int mine = st.slots[tok + i];
            if (mine != slot + i) { if (lane == 0 && mine >= 0 && st.err) atomicOr(st.err, VL_DEV_BAD_SLOT); continue; }
        }
        if (k == 0 || n > 1) {
            float4 cs[Row<MAXHD>::UR];
            if (turned) Row<MAXHD>::angles(cs, pos + i, st.inv_freq, lane, turned);
            pdl_wait();
            if (k == ahead && held) old = *scale;
            r.load(st.qkv + (size_t)(tok + i) * st.row_stride + (size_t)(st.nq + (values ? st.nkv : 0) + kvh) * hd, lane, hd, turned);
            if (!values && st.kw) r.norm(st.kw, st.eps, lane, hd, turned);
            if (turned) r.turn(cs);
        }
        if (k < n) top = max(top, r.top());
        else {
            unsigned char* dst = cache + (size_t)(row0 + i) * hd;
            r.each(lane, hd, turned, [&](int c, float2 v) { *reinterpret_cast<unsigned short*>(dst + c) = to_e4m3x2(v.x * inv, v.y * inv); });
        }
    }
    if (held && now > old) {                                 // (false for NaN: rows under a scale that is none need no other)
        move_rows(cache, row0 * hd, old * inv, lane, 32);
        if (__builtin_expect(n > 1, 0))                      // rows between that are not written
#pragma unroll 1
            for (int i = 0; i < n; ++i)
                if (st.slots[tok + i] != slot + i && lane < hd / 16) {
                    uint4* row = reinterpret_cast<uint4*>(cache + (size_t)(row0 + i) * hd) + lane;
                    *row = times(*row, old * inv);
                }
    }
    if (lane == 0) *scale = now;
}

// Any head: a block a page's keys or values of one KV head, up to 64 rows a pass in registers, a warp a row.
template <int MAXHD>
__global__ void __launch_bounds__(NT)
write_8bit_narrow_kernel(const __grid_constant__ Step st) {
    constexpr int ROWS = MAXHD <= 128 ? 8 : 4;               // rows a warp holds
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = st.hd;
    pdl_launch_dependents();
    if (!st.early) pdl_wait();
    if ((int)blockIdx.x >= st.page_blocks) {                 // ---- queries ----
        const int groups = (st.nq + st.heads_a_warp - 1) / st.heads_a_warp;
        const long long unit = (long long)((int)blockIdx.x - st.page_blocks) * WARPS + warp;
        const int tok = (int)(unit / groups), h0 = (int)(unit - (long long)tok * groups) * st.heads_a_warp;
        if (tok < st.T) query_heads<MAXHD>(st, tok, h0, min(st.nq, h0 + st.heads_a_warp));
        return;
    }
    __shared__ unsigned s_top[WARPS];
    const bool values = blockIdx.x & 1;
    const int kvh = (int)(blockIdx.x >> 1) % st.nkv;
    const Visit v = find_visit(st, (int)(blockIdx.x >> 1) / st.nkv);
    if (v.n <= 0) return;
    const size_t head = (size_t)v.page * st.nkv + kvh;
    unsigned char* cache = (values ? st.vcache : st.kcache) + head * st.page_size * hd;
    float* scale = (values ? st.vscale : st.kscale) + head;
    const int turned = values || !st.inv_freq ? 0 : st.rot;
    const float* w = values ? nullptr : st.kw;
    const bf16* src = st.qkv + (size_t)(st.nq + (values ? st.nkv : 0) + kvh) * hd;
    pdl_wait();                                              // qkv comes from the kernel before
    const float old = v.held ? *scale : 0.f;
    Row<MAXHD> r[ROWS];
    bool mine[ROWS];
    unsigned top = 0, left_out = 0, strange = 0;
    auto take = [&](int base) {                              // this warp's rows of the pass that begins with row `base`
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const int i = base + u * WARPS + warp;
            mine[u] = i < v.n;
            const int slot = mine[u] ? st.slots[v.tok0 + i] : 0;
            if (mine[u] && slot != v.slot0 + i) { mine[u] = false; left_out = 1; strange |= slot >= 0; }
            if (mine[u]) r[u].load(src + (size_t)(v.tok0 + i) * st.row_stride, lane, hd, turned);
        }
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (!mine[u]) continue;
            if (w) r[u].norm(w, st.eps, lane, hd, turned);
            if (turned) {
                float4 cs[Row<MAXHD>::UR];
                Row<MAXHD>::angles(cs, st.positions[v.tok0 + base + u * WARPS + warp], st.inv_freq, lane, turned);
                r[u].turn(cs);
            }
        }
    };
    constexpr int PASS = ROWS * WARPS;
    const int last = (v.n - 1) / PASS * PASS;
    for (int base = 0; base <= last; base += PASS) {
        take(base);
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (mine[u]) top = max(top, r[u].top());
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[warp] = top;
    if (strange && lane == 0 && st.err) atomicOr(st.err, VL_DEV_BAD_SLOT);
    left_out = __syncthreads_or(left_out);
    for (int i = 0; i < WARPS; ++i) top = max(top, s_top[i]);
    const float now = new_scale(top, v.held, old), inv = inverse_of(now);
    // Whole passes that registers no longer hold are made again, the last one first (pages of more than 64 rows, heads beyond 128).
    for (int base = last; base >= 0; base -= PASS) {
        if (base != last) take(base);
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            if (!mine[u]) continue;
            unsigned char* dst = cache + (size_t)(v.row0 + base + u * WARPS + warp) * hd;
            r[u].each(lane, hd, turned, [&](int i, float2 x) { *reinterpret_cast<unsigned short*>(dst + i) = to_e4m3x2(x.x * inv, x.y * inv); });
        }
    }
    if (v.held && now > old) {
        move_rows(cache, v.row0 * hd, old * inv, threadIdx.x, NT);
        if (left_out)
            for (int i = warp; i < v.n; i += WARPS)
                if (st.slots[v.tok0 + i] != v.slot0 + i) move_rows(cache + (size_t)(v.row0 + i) * hd, hd, old * inv, lane, 32);
    }
    if (threadIdx.x == 0) *scale = now;
}

// Heads of HD features, all of them rotated or none: a lane holds 8 neighbouring features of a row's first half and their 8 partners in the second,
// so HD / 16 lanes share a row and a warp works on 512 / HD rows at once.
template <int HD>
struct WideRow {
    static constexpr int LANES = HD / 16, AT_ONCE = 32 / LANES, HALF = HD / 2;
    float a[8], b[8];

    __device__ __forceinline__ void load(const bf16* row, int i0) { load8(row + i0, a); load8(row + i0 + HALF, b); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
    }
    __device__ __forceinline__ void norm(const float (&wa)[8], const float (&wb)[8], float eps) {        // (all lanes of the warp)
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = 1.0f / sqrtf(ss / (float)HD + eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) { a[j] *= inv * wa[j]; b[j] *= inv * wb[j]; }
    }
    __device__ __forceinline__ void turn(const float2* table) {          // (cosine, sine) of this lane's 8 features
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float4 cs = *reinterpret_cast<const float4*>(table + j);
            const float x0 = a[j], y0 = b[j], x1 = a[j + 1], y1 = b[j + 1];
            a[j] = x0 * cs.x - y0 * cs.y; b[j] = y0 * cs.x + x0 * cs.y;
            a[j + 1] = x1 * cs.z - y1 * cs.w; b[j + 1] = y1 * cs.z + x1 * cs.w;
        }
    }
    __device__ __forceinline__ unsigned top() const {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, max(__float_as_uint(fabsf(a[j])), __float_as_uint(fabsf(b[j]))));
        return m;
    }
    static __device__ __forceinline__ uint2 eight(const float (&x)[8], float f) {
        return make_uint2((unsigned)to_e4m3x2(x[0] * f, x[1] * f) | ((unsigned)to_e4m3x2(x[2] * f, x[3] * f) << 16),
                          (unsigned)to_e4m3x2(x[4] * f, x[5] * f) | ((unsigned)to_e4m3x2(x[6] * f, x[7] * f) << 16));
    }
    __device__ __forceinline__ void store(unsigned char* row, int i0, float f) const {
        *reinterpret_cast<uint2*>(row + i0) = eight(a, f);
        *reinterpret_cast<uint2*>(row + i0 + HALF) = eight(b, f);
    }
};

// AT: warps on a head, whose rows of a page they hold in one pass where that is possible; other heads of the block are beside them.
template <int HD, int AT>
__global__ void __launch_bounds__(NT, HD <= 128 ? 4 : 2)           // (a portion of 2,048 tokens: 64 registers 17.6 us, 80 20.6, 121 20.9)
write_8bit_wide_kernel(const __grid_constant__ Step st) {
    using R = WideRow<HD>;
    constexpr int TURNS = HD <= 128 ? 2 : 4;                 // groups of rows a warp holds
    extern __shared__ __align__(16) float2 s_table[];        // keys: [the pass's rows][HD / 2]; queries: [WARPS][HD / 2]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / R::LANES, i0 = 8 * (lane % R::LANES);
    pdl_launch_dependents();
    if (!st.early) pdl_wait();
    float wa[8], wb[8];
    auto weights = [&](const float* w) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { wa[j] = w ? w[i0 + j] : 1.f; wb[j] = w ? w[i0 + R::HALF + j] : 1.f; }
    };
    if ((int)blockIdx.x >= st.page_blocks) {                 // ---- queries: a warp a token and heads_a_warp of its heads ----
        const int groups = (st.nq + st.heads_a_warp - 1) / st.heads_a_warp;
        const long long unit = (long long)((int)blockIdx.x - st.page_blocks) * WARPS + warp;
        const int tok = (int)(unit / groups), h0 = (int)(unit - (long long)tok * groups) * st.heads_a_warp, h1 = min(st.nq, h0 + st.heads_a_warp);
        if (tok >= st.T) return;
        float2* table = s_table + warp * R::HALF;
        if (st.inv_freq) {
            const int pos = st.positions[tok];
            for (int i = lane; i < R::HALF; i += 32) sine_cosine(pos, st.inv_freq[i], &table[i].y, &table[i].x);
            __syncwarp();
        }
        weights(st.qw);
        pdl_wait();
        const bf16* src = st.qkv + (size_t)tok * st.row_stride;
        bf16* dst = st.q_out + (size_t)tok * st.q_stride;
        for (int h = h0; h < h1; h += 2 * R::AT_ONCE) {      // (the loads of one group beside the arithmetic of the other)
            R r[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int mine = h + u * R::AT_ONCE + sub;
                if (mine < h1) r[u].load(src + (size_t)mine * HD, i0);
                else r[u].clear();
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int mine = h + u * R::AT_ONCE + sub;
                if (st.qw) r[u].norm(wa, wb, st.eps);
                if (st.inv_freq) r[u].turn(table + i0);
                if (mine < h1) { store8(dst + (size_t)mine * HD + i0, r[u].a); store8(dst + (size_t)mine * HD + i0 + R::HALF, r[u].b); }
            }
        }
        return;
    }
    // ---- a page of keys or values of heads_a_block KV heads, of which as many at a time as there are warps for ----
    constexpr int GROUP = AT * R::AT_ONCE, PASS = TURNS * GROUP;
    const int my_warp = warp % AT;
    __shared__ unsigned s_top[2][WARPS];
    const bool values = blockIdx.x & 1;
    const int parts = (st.nkv + st.heads_a_block - 1) / st.heads_a_block, part = (int)(blockIdx.x >> 1) % parts;
    const Visit v = find_visit(st, (int)(blockIdx.x >> 1) / parts);
    if (v.n <= 0) return;
    const bool turned = !values && st.inv_freq;
    const float* w = values ? nullptr : st.kw;
    weights(w);
    auto angles = [&](int base) {                            // of the pass's rows
        const int p0 = st.positions[v.tok0] + base, rows = min(PASS, v.n - base);
        for (int i = threadIdx.x; i < rows * R::HALF; i += NT) sine_cosine(p0 + i / R::HALF, st.inv_freq[i % R::HALF], &s_table[i].y, &s_table[i].x);
    };
    const int last = (v.n - 1) / PASS * PASS;
    if (turned && last == 0) angles(0);
    unsigned left_out = 0;
    for (int i = threadIdx.x; i < v.n; i += NT) {
        const int slot = st.slots[v.tok0 + i];
        if (slot == v.slot0 + i) continue;
        left_out = 1;
        if (slot >= 0 && st.err) atomicOr(st.err, VL_DEV_BAD_SLOT);
    }
    left_out = __syncthreads_or(left_out);
    pdl_wait();                                              // qkv comes from the kernel before
    const int end = min(st.nkv, (part + 1) * st.heads_a_block);
    for (int first = part * st.heads_a_block, turn = 0; first < end; first += WARPS / AT, turn ^= 1) {
        const bool none = first + warp / AT >= end;       // (no head is left for this warp: it goes along)
        const int kvh = none ? first : first + warp / AT;
        const size_t head = (size_t)v.page * st.nkv + kvh;
        unsigned char* cache = (values ? st.vcache : st.kcache) + head * st.page_size * HD;
        float* scale = (values ? st.vscale : st.kscale) + head;
        const bf16* src = st.qkv + (size_t)(st.nq + (values ? st.nkv : 0) + kvh) * HD;
        const float old = v.held ? *scale : 0.f;
        R r[TURNS];
        bool mine[TURNS];
        unsigned top = 0;
        auto take = [&](int base) {
            if (turned && last) {                            // (pages of more rows than a pass: their angles anew)
                __syncthreads();
                angles(base);
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                const int i = base + u * GROUP + my_warp * R::AT_ONCE + sub;
                mine[u] = !none && i < v.n && !(left_out && st.slots[v.tok0 + i] != v.slot0 + i);
                if (mine[u]) r[u].load(src + (size_t)(v.tok0 + i) * st.row_stride, i0);
                else r[u].clear();
            }
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                if (w) r[u].norm(wa, wb, st.eps);
                if (turned && mine[u]) r[u].turn(s_table + (u * GROUP + my_warp * R::AT_ONCE + sub) * R::HALF + i0);
            }
        };
        for (int base = 0; base <= last; base += PASS) {
            take(base);
#pragma unroll
            for (int u = 0; u < TURNS; ++u)
                if (mine[u]) top = max(top, r[u].top());
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) s_top[turn][warp] = top;
        __syncthreads();
        for (int i = 0; i < AT; ++i) top = max(top, s_top[turn][warp - my_warp + i]);
        const float now = new_scale(top, v.held, old), inv = inverse_of(now);
        for (int base = last; base >= 0; base -= PASS) {     // (the last pass is still held)
            if (base != last) take(base);
#pragma unroll
            for (int u = 0; u < TURNS; ++u)
                if (mine[u]) r[u].store(cache + (size_t)(v.row0 + base + u * GROUP + my_warp * R::AT_ONCE + sub) * HD, i0, inv);
        }
        if (none) continue;
        if (v.held && now > old) {
            move_rows(cache, v.row0 * HD, old * inv, my_warp * 32 + lane, AT * 32);
            if (left_out)
                for (int i = my_warp; i < v.n; i += AT)
                    if (st.slots[v.tok0 + i] != v.slot0 + i) move_rows(cache + (size_t)(v.row0 + i) * HD, HD, old * inv, lane, 32);
        }
        if (my_warp == 0 && lane == 0) *scale = now;         // (everybody has read it: a barrier ago)
    }
}

// qkv [T, row_stride] bfloat16 = q | k | v heads of hd features; q_out [T, q_stride] (may be qkv).  Tokens cu[b] .. cu[b + 1] are those of
// request b at consecutive positions; slots [T] = page * page_size + position % page_size, negative: not written (the row keeps what it stands for, unless the
// page begins anew with its first row); null: no cache at all.
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
    Step st = {(const bf16*)qkv, row_stride, (bf16*)q_out, q_stride, positions, slots, cu, B, qw, kw, eps, inv_freq, rot, (unsigned char*)kcache,
               (unsigned char*)vcache, kscale, vscale, T, nq, nkv, hd, page_size, num_pages, err, 0, 0, 0, (int)vl_pdl_enabled()};
    cudaStream_t s = (cudaStream_t)stream;
    if (T == B || (!slots && T < 256)) {
        st.heads_a_warp = T >= 32 ? 4 : 2;
        const long long units = (long long)T * ((slots ? 2 * nkv : 0) + (nq + st.heads_a_warp - 1) / st.heads_a_warp), blocks = (units + WARPS - 1) / WARPS;
        if (blocks >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
        return vl_launch_waiting(hd <= 128 ? write_8bit_singles_kernel<128> : write_8bit_singles_kernel<256>, dim3((unsigned)blocks), dim3(NT), 0, s, st);
    }
    // pages that B requests of T tokens can reach: full ones and one broken at each end
    const long long pages = slots ? (T < (long long)T / page_size + 2ll * B ? T : (long long)T / page_size + 2ll * B) : 0;
    const bool wide = (hd == 32 || hd == 64 || hd == 128 || hd == 256) && (!inv_freq || rot == hd) && row_stride % 8 == 0 && q_stride % 8 == 0 &&
                      (((uintptr_t)qkv | (uintptr_t)q_out) & 15) == 0;
    // Several heads share a page's angles where blocks are enough without and a page has rows for its threads (4,096 tokens, 8 KV heads: 4 heads 27.8 us, 2 29.7,
    // 1 34.5; 8 portions of 300, 4 KV heads: 4 heads 21, 1 12).
    st.heads_a_warp = wide ? (T >= 256 ? 16 : 8) : (T >= 256 ? 8 : (T >= 32 ? 4 : 2));
    st.heads_a_block = !wide || T < 32 * pages || pages * nkv < 256 ? 1 : (pages * nkv < 512 ? 2 : 4);
    // Two warps a head where they hold the rows that a page can get: small pages and short portions leave none idle (32 + 2 x 8 heads of 128: 2,048 tokens on pages
    // of 16 17.6 us, 29 with eight; 300 portions of 8 tokens 28 and 71).
    const int rows = page_size < (T + B - 1) / (B > 0 ? B : 1) ? page_size : (T + B - 1) / (B > 0 ? B : 1), a_warp = (hd <= 128 ? 2 : 4) * (512 / hd);
    const bool few = wide && rows <= 2 * a_warp;
    if (few && st.heads_a_block < WARPS / 2) st.heads_a_block = WARPS / 2 < nkv ? WARPS / 2 : nkv;
    st.page_blocks = (int)(pages * ((nkv + st.heads_a_block - 1) / st.heads_a_block) * 2);
    const long long units = (long long)T * ((nq + st.heads_a_warp - 1) / st.heads_a_warp), blocks = st.page_blocks + (units + WARPS - 1) / WARPS;
    if (blocks >= (1ll << 31) || pages * nkv * 2 >= (1ll << 31)) return VL_ERR_UNSUPPORTED;
    if (!wide)
        return vl_launch_waiting(hd <= 128 ? write_8bit_narrow_kernel<128> : write_8bit_narrow_kernel<256>, dim3((unsigned)blocks), dim3(NT), 0, s, st);
    const int angles = a_warp * (few ? 2 : WARPS) > WARPS ? a_warp * (few ? 2 : WARPS) : WARPS, smem = inv_freq ? angles * hd / 2 * 8 : 0;
    auto launch = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
        return vl_launch_waiting(kernel, dim3((unsigned)blocks), dim3(NT), (size_t)smem, s, st);
    };
    if (hd == 32) return few ? launch(write_8bit_wide_kernel<32, 2>) : launch(write_8bit_wide_kernel<32, WARPS>);
    if (hd == 64) return few ? launch(write_8bit_wide_kernel<64, 2>) : launch(write_8bit_wide_kernel<64, WARPS>);
    if (hd == 128) return few ? launch(write_8bit_wide_kernel<128, 2>) : launch(write_8bit_wide_kernel<128, WARPS>);
    return few ? launch(write_8bit_wide_kernel<256, 2>) : launch(write_8bit_wide_kernel<256, WARPS>);
}
