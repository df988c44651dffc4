// A cache of keys and values in one byte an element with a fp32 scale for each block of tokens
// and head: written as tokens arrive, and read back.
//
//   scale = max |x| / 127 over the block, byte = 128 + nearest_even(x / scale)
//
// A block that keeps tokens from before takes the larger of its scale and the new elements'; its
// kept bytes are then rounded anew from the values that they stood for.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace mi355 {

template <bool F16>
__device__ __forceinline__ float kv_ld(const char* p, int i) {
    return F16 ? h2f(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}

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
// 128 + x / d rounded to nearest even: the product with the reciprocal is at most one off, and the
// remainder x - q d is exact in one fma, since x lies within a step of q d
__device__ __forceinline__ uint32_t kv_byte(float x, const KvStep& k) {
    if (k.id == 0.0f) return 128;
    const float xs = x * k.up;
    float q = fminf(fmaxf(rintf(xs * k.id), -127.0f), 127.0f);
    const float r = __builtin_fmaf(-q, k.d, xs), half = 0.5f * k.d;
    if (fabsf(r) > half || (fabsf(r) == half && ((int)q & 1))) q += __builtin_copysignf(1.0f, r);
    return (uint32_t)((int)fminf(fmaxf(q, -127.0f), 127.0f) + 128);
}

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    v = max(v, (uint32_t)lane_swap<1>((int)v));
    v = max(v, (uint32_t)lane_swap<2>((int)v));
    v = max(v, (uint32_t)lane_swap<4>((int)v));
    v = max(v, (uint32_t)lane_swap<8>((int)v));
    v = max(v, (uint32_t)lane_swap<16>((int)v));
    return max(v, (uint32_t)lane_swap<32>((int)v));
}

// One workgroup for a touched block of one head, keys or values.
template <bool F16>
__global__ __launch_bounds__(256) void kv_write_kernel(const KvView c, const KvRows r, int D, int nb) {
    __shared__ uint32_t red[4];
    const int w = blockIdx.x;
    const bool val = w & 1;
    const int j = (w >> 1) % nb, h = (w >> 1) / nb % c.heads, s = (w >> 1) / nb / c.heads;
    const int end = kv_len(c, s), n_new = r.idx ? min(max(r.idx[s], 0), r.n_tok) : r.n_tok;
    const int first = end - n_new, start = max(first, 0);
    const int b = start / c.bt + j, lo = max(start, b * c.bt), hi = min(end, (b + 1) * c.bt);
    if (lo >= hi) return;
    const int id = c.table[(int64_t)s * c.max_blocks + b];
    if (id < 0 || id >= c.n_blocks) return;
    const char* src = val ? r.v + h * r.v_nb[1] + s * r.v_nb[2] : r.k + h * r.k_nb[1] + s * r.k_nb[2];
    const int64_t row = val ? r.v_nb[0] : r.k_nb[0], at = (int64_t)id * c.heads + h;
    uint8_t* dst = (val ? c.v : c.k) + at * c.bt * D;
    float* scale = (val ? c.v_scale : c.k_scale) + at;
    const int kept = (lo - b * c.bt) * D, all = (hi - b * c.bt) * D;
    auto value = [&](int i) {  // element i of the block, a new one
        const int t = i / D;
        return kv_ld<F16>(src + (int64_t)(b * c.bt + t - first) * row, i - t * D);
    };
    uint32_t top = 0;  // magnitudes order as their bits do, NaN above infinity
    for (int i = kept + (int)threadIdx.x; i < all; i += 256) top = max(top, __float_as_uint(value(i)) & 0x7fffffffu);
    top = wave_max_u(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    const float was = *scale;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
    float d = __uint_as_float(top) / 127.0f;
    if (kept > 0) d = __uint_as_float(max(__float_as_uint(d) & 0x7fffffffu, __float_as_uint(was) & 0x7fffffffu));
    const KvStep k = kv_step(d);
    if (kept > 0 && __float_as_uint(d) != __float_as_uint(was))
        for (int i = threadIdx.x; i < kept; i += 256) dst[i] = (uint8_t)kv_byte((float)((int)dst[i] - 128) * was, k);
    for (int i = kept + (int)threadIdx.x; i < all; i += 256) dst[i] = (uint8_t)kv_byte(value(i), k);
    if (threadIdx.x == 0) *scale = d;
}

// thread per element
template <bool F16>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvView c, const KvRows r, int D, int64_t total) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int e = (int)(i % D);
    const int64_t row = i / D;
    const int t = (int)(row % r.n_tok), h = (int)(row / r.n_tok % c.heads), s = (int)(row / r.n_tok / c.heads);
    const int p = r.idx ? r.idx[(int64_t)s * r.n_tok + t] : t;
    if (p < 0 || p >= kv_len(c, s)) return;
    const int b = p / c.bt, id = c.table[(int64_t)s * c.max_blocks + b];
    if (id < 0 || id >= c.n_blocks) return;
    const int64_t at = (int64_t)id * c.heads + h, src = (at * c.bt + p - b * c.bt) * D + e;
    auto put = [&](char* base, const int64_t* nb, const uint8_t* q, const float* scale) {
        char* o = base + t * nb[0] + h * nb[1] + s * nb[2];
        const float v = (float)((int)q[src] - 128) * scale[at];
        if (F16) reinterpret_cast<uint16_t*>(o)[e] = f2h(v);
        else reinterpret_cast<float*>(o)[e] = v;
    };
    if (r.k) put(r.k, r.k_nb, c.k, c.k_scale);
    if (r.v) put(r.v, r.v_nb, c.v, c.v_scale);
}

hipError_t launch_kv_write(const KvView& c, const KvRows& r, int D, hipStream_t st) {
    if (c.n_seq <= 0 || r.n_tok <= 0 || c.max_blocks <= 0) return hipSuccess;
    // blocks that n_tok tokens from any offset may touch
    const int nb = (int)std::min<int64_t>(((int64_t)r.n_tok + c.bt - 2) / c.bt + 1, c.max_blocks);
    const int64_t g = (int64_t)nb * c.heads * c.n_seq * 2;
    if (g > INT32_MAX) return hipErrorInvalidValue;
    if (r.f16) kv_write_kernel<true><<<(unsigned)g, 256, 0, st>>>(c, r, D, nb);
    else kv_write_kernel<false><<<(unsigned)g, 256, 0, st>>>(c, r, D, nb);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvView& c, const KvRows& r, int D, hipStream_t st) {
    const int64_t total = (int64_t)r.n_tok * c.heads * c.n_seq * D;
    if (total <= 0 || c.max_blocks <= 0) return hipSuccess;
    if ((total + 255) / 256 > INT32_MAX) return hipErrorInvalidValue;
    if (r.f16) kv_read_kernel<true><<<(unsigned)((total + 255) / 256), 256, 0, st>>>(c, r, D, total);
    else kv_read_kernel<false><<<(unsigned)((total + 255) / 256), 256, 0, st>>>(c, r, D, total);
    return hipGetLastError();
}

}  // namespace mi355
