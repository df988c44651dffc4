// A cache of keys and values in one byte an element with a fp32 scale for each block of tokens
// and head: written as tokens arrive, and read back.
//
//   scale = max |x| / 127 over the block, byte = 128 + nearest_even(x / scale)
//
// A block that keeps tokens from before takes the larger of its scale and the new elements'; its
// kept bytes are then rounded anew from the values that they stood for.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace mi355 {

namespace {
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef v4f v4f_a4 __attribute__((aligned(4)));
}  // namespace

// eight consecutive elements at any alignment of their type
template <bool F16>
struct Eight {
    u32x4 raw[F16 ? 1 : 2];
    __device__ __forceinline__ void load(const char* p) {
        raw[0] = *reinterpret_cast<const u32x4_a2*>(p);
        if constexpr (!F16) raw[1] = *reinterpret_cast<const u32x4_a2*>(p + 16);
    }
    __device__ __forceinline__ void clear() {
        raw[0] = u32x4{0, 0, 0, 0};
        if constexpr (!F16) raw[1] = raw[0];
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (F16) return h2f((uint16_t)(raw[0][i >> 1] >> (16 * (i & 1))));
        else return __uint_as_float(raw[i >> 2][i & 3]);
    }
};

__device__ __forceinline__ int kv_len(const KvView& c, int s) {
    return (int)min((int64_t)max(c.n_kv[s], 0), (int64_t)c.max_blocks * c.bt);
}

// What division by a block's scale needs: d and its reciprocal, both times up, a power of two
// that keeps scales near the bottom of fp32 out of the subnormal range.
struct KvStep {
    float d, id, up;
};
__device__ __forceinline__ KvStep kv_step(float d) {
    KvStep k;
    k.up = d < 5.4210109e-20f ? 1.8446744e19f : 1.0f;  // 2^-64, 2^64
    k.d = d * k.up;
    k.id = d > 0.0f && d < __builtin_inff() ? 1.0f / k.d : 0.0f;
    return k;
}
// 128 + x / d rounded to nearest even, as a float: the product with the reciprocal is at most one off, and the
// remainder x - q d is exact in one fma, since x lies within a step of q d
__device__ __forceinline__ float kv_byte(float x, const KvStep& k) {
    const float xs = x * k.up;
    float q = rintf(xs * k.id);
    const float r = __builtin_fmaf(-q, k.d, xs), half = 0.5f * k.d;
    if (fabsf(r) > half || (fabsf(r) == half && ((int)q & 1))) q += __builtin_copysignf(1.0f, r);
    return k.id == 0.0f ? 128.0f : fminf(fmaxf(q, -127.0f), 127.0f) + 128.0f;
}
__device__ __forceinline__ uint32_t kv_pack(float a, float b, float c, float d) {
    uint32_t v = __builtin_amdgcn_cvt_pk_u8_f32(a, 0, 0);
    v = __builtin_amdgcn_cvt_pk_u8_f32(b, 1, v);
    v = __builtin_amdgcn_cvt_pk_u8_f32(c, 2, v);
    return __builtin_amdgcn_cvt_pk_u8_f32(d, 3, v);
}

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    v = max(v, (uint32_t)lane_swap<1>((int)v));
    v = max(v, (uint32_t)lane_swap<2>((int)v));
    v = max(v, (uint32_t)lane_swap<4>((int)v));
    v = max(v, (uint32_t)lane_swap<8>((int)v));
    v = max(v, (uint32_t)lane_swap<16>((int)v));
    return max(v, (uint32_t)lane_swap<32>((int)v));
}

// T threads (64: a wavefront) for a touched block of one head, keys or values: its new elements wait in registers,
// V times eight to a thread, for the block's largest magnitude; kept bytes are touched only where the scale grew.
// Bound by memory (each new element read once: 4 sequences of 5101 tokens, 8 heads of 128 halves, written and read back,
// 189 MB in 50.6 us), for single tokens by the chain length - block - scale (64 sequences, written and read back: 11.8 us
// in two launches).
template <bool F16, int T, int V>
__global__ __launch_bounds__(256) void kv_write_kernel(const KvView c, const KvRows r, const int D8, const int nb, const int units) {
    __shared__ uint32_t red[4];
    const int w = T == 256 ? (int)blockIdx.x : (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), t = threadIdx.x & (T - 1);
    if (w >= units) return;  // (T = 64: no barrier follows)
    const bool val = w & 1;
    const int j = (w >> 1) % nb, h = (w >> 1) / nb % c.heads, s = (w >> 1) / nb / c.heads;
    const int end = kv_len(c, s), n_new = r.idx ? min(max(r.idx[s], 0), r.n_tok) : r.n_tok;
    const int first = end - n_new, start = max(first, 0);
    const int b = start / c.bt + j, lo = max(start, b * c.bt), hi = min(end, (b + 1) * c.bt);
    if (lo >= hi) return;
    const int id = c.table[(int64_t)s * c.max_blocks + b];
    if (id < 0 || id >= c.n_blocks) return;
    const int64_t row = val ? r.v_nb[0] : r.k_nb[0], at = (int64_t)id * c.heads + h;
    const char* src = (val ? r.v + h * r.v_nb[1] + s * r.v_nb[2] : r.k + h * r.k_nb[1] + s * r.k_nb[2]) + (lo - first) * row;
    uint8_t* dst = (val ? c.v : c.k) + at * c.bt * (8 * D8);
    float* scale = (val ? c.v_scale : c.k_scale) + at;
    const int kept = (lo - b * c.bt) * D8, fresh = (hi - lo) * D8;  // pieces of eight
    Eight<F16> x[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = v * T + t, tok = i / D8;
        x[v].clear();
        if (i < fresh) x[v].load(src + tok * row + (i - tok * D8) * (F16 ? 16 : 32));
    }
    const float was = *scale;
    uint32_t top = 0;  // magnitudes order as their bits do, NaN above infinity
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[v][e]) & 0x7fffffffu);
    top = wave_max_u(top);
    if constexpr (T == 256) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(red[0], red[1]), max(red[2], red[3]));
    }
    float d = __uint_as_float(top) / 127.0f;
    if (kept > 0) d = __uint_as_float(max(__float_as_uint(d) & 0x7fffffffu, __float_as_uint(was) & 0x7fffffffu));
    const KvStep k = kv_step(d);
    if (kept > 0 && __float_as_uint(d) != __float_as_uint(was)) {
        uint32_t* old = reinterpret_cast<uint32_t*>(dst);
        for (int i = t; i < 2 * kept; i += T) {
            const uint32_t u = old[i];
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = kv_byte(((float)(u >> (8 * e) & 255) - 128.0f) * was, k);
            old[i] = kv_pack(y[0], y[1], y[2], y[3]);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = v * T + t;
        if (i >= fresh) break;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = kv_byte(x[v][e], k);
        reinterpret_cast<u32x2*>(dst)[kept + i] = u32x2{kv_pack(y[0], y[1], y[2], y[3]), kv_pack(y[4], y[5], y[6], y[7])};
    }
    if (t == 0) *scale = d;
}

// Thread per eight elements of a row; blockIdx.y: keys or values.  Bound by memory (15552 tokens of 8 heads of 64 to halves,
// 48 MB, in 11.2 us).
template <bool F16>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvView c, const KvRows r, const int D8, const int64_t total) {
    const bool val = r.k ? blockIdx.y == 1 : true;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const uint32_t row = (uint32_t)(i / D8);
    const int e = (int)(i - (int64_t)row * D8);
    const uint32_t hs = row / (uint32_t)r.n_tok;
    const int t = (int)(row - hs * r.n_tok), s = (int)(hs / (uint32_t)c.heads), h = (int)(hs - (uint32_t)s * c.heads);
    const int p = r.idx ? r.idx[(int64_t)s * r.n_tok + t] : t;
    const int id = c.table[(int64_t)s * c.max_blocks + min(max(p, 0) >> c.bt_log2, c.max_blocks - 1)];  // (on its way beside the length)
    if (p < 0 || p >= kv_len(c, s) || id < 0 || id >= c.n_blocks) return;
    const int64_t at = (int64_t)id * c.heads + h;
    const u32x2 u = reinterpret_cast<const u32x2*>(val ? c.v : c.k)[(at * c.bt + (p & (c.bt - 1))) * D8 + e];
    const float scale = (val ? c.v_scale : c.k_scale)[at];
    char* o = (val ? r.v + t * r.v_nb[0] + h * r.v_nb[1] + s * r.v_nb[2] : r.k + t * r.k_nb[0] + h * r.k_nb[1] + s * r.k_nb[2]) + e * (F16 ? 16 : 32);
    float y[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) y[x] = ((float)(u[x >> 2] >> (8 * (x & 3)) & 255) - 128.0f) * scale;
    if constexpr (F16) {
        u32x4 z;
#pragma unroll
        for (int x = 0; x < 4; ++x) z[x] = (uint32_t)f2h(y[2 * x]) | (uint32_t)f2h(y[2 * x + 1]) << 16;
        *reinterpret_cast<u32x4_a2*>(o) = z;
    } else {
        *reinterpret_cast<v4f_a4*>(o) = v4f{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<v4f_a4*>(o + 16) = v4f{y[4], y[5], y[6], y[7]};
    }
}

template <bool F16>
static void kv_write_go(const KvView& c, const KvRows& r, int D8, int nb, int units, hipStream_t st) {
    const int pieces = std::min(r.n_tok, c.bt) * D8;  // new ones of a block, at most
    auto go = [&](auto t, auto v) {
        constexpr int T = decltype(t)::value, V = decltype(v)::value;
        const int per = 256 / T;
        kv_write_kernel<F16, T, V><<<(unsigned)((units + per - 1) / per), 256, 0, st>>>(c, r, D8, nb, units);
    };
    using T64 = std::integral_constant<int, 64>;
    using T256 = std::integral_constant<int, 256>;
    if (pieces <= 64) go(T64(), std::integral_constant<int, 1>());
    else if (pieces <= 256) go(T64(), std::integral_constant<int, 4>());
    else if (pieces <= 512) go(T256(), std::integral_constant<int, 2>());
    else if (pieces <= 1024) go(T256(), std::integral_constant<int, 4>());
    else go(T256(), std::integral_constant<int, 8>());
}

hipError_t launch_kv_write(const KvView& c, const KvRows& r, int D, hipStream_t st) {
    if (c.n_seq <= 0 || r.n_tok <= 0 || c.max_blocks <= 0 || c.n_blocks <= 0) return hipSuccess;
    // blocks that n_tok tokens from any offset may touch
    const int nb = (int)std::min<int64_t>(((int64_t)r.n_tok + c.bt - 2) / c.bt + 1, c.max_blocks);
    const int64_t units = (int64_t)nb * c.heads * c.n_seq * 2;
    if (units > INT32_MAX - 8) return hipErrorInvalidValue;
    if (r.f16) kv_write_go<true>(c, r, D / 8, nb, (int)units, st);
    else kv_write_go<false>(c, r, D / 8, nb, (int)units, st);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvView& c, const KvRows& r, int D, hipStream_t st) {
    const int64_t total = (int64_t)r.n_tok * c.heads * c.n_seq * (D / 8);
    if (total <= 0 || c.max_blocks <= 0 || c.n_blocks <= 0) return hipSuccess;
    if ((total + 255) / 256 > INT32_MAX) return hipErrorInvalidValue;
    const dim3 g((unsigned)((total + 255) / 256), r.k && r.v ? 2 : 1);
    if (r.f16) kv_read_kernel<true><<<g, 256, 0, st>>>(c, r, D / 8, total);
    else kv_read_kernel<false><<<g, 256, 0, st>>>(c, r, D / 8, total);
    return hipGetLastError();
}

}  // namespace mi355
