// The residual's addition, RMS norm and the next product's 8-bit operand in one pass over the
// rows (ggml_add, ggml_rms_norm, ggml_mul, from_float), and ggml's to_float back.
//
//   h = x + add, y = h * (1 / sqrt(mean(h^2) + eps)) * w
//
// The squares are fp32 products summed in double, as ggml_rms_norm does, so the sum's order changes
// the fp32 mean about once in 10^7 rows and the 8-bit quants behind it do not depend on it.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace mi355 {

__device__ __forceinline__ int64_t span_at(const RowSpan& s, int64_t r, int64_t ne1, int64_t ne2) {
    const int64_t i1 = r % ne1, q = r / ne1;
    return i1 * s.nb[0] + (q % ne2) * s.nb[1] + (q / ne2) * s.nb[2];
}

template <bool F16>
__device__ __forceinline__ float ld_one(const char* row, int i) {
    return F16 ? h2f(reinterpret_cast<const uint16_t*>(row)[i]) : reinterpret_cast<const float*>(row)[i];
}
template <bool F16>
__device__ __forceinline__ void st_one(char* row, int i, float v) {
    if (F16) reinterpret_cast<uint16_t*>(row)[i] = f2h(v);
    else reinterpret_cast<float*>(row)[i] = v;
}

namespace {
typedef v4f v4f_a4 __attribute__((aligned(4)));
typedef v8h v8h_a2 __attribute__((aligned(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
}  // namespace

// The 16 bytes of elements i .. of a row at any alignment of their type, zeros for those from n on; and as E floats
template <bool F16>
__device__ __forceinline__ u32x4 ld_raw(const char* row, int i, int n) {
    constexpr int E = F16 ? 8 : 4;
    if (i + E <= n) return *reinterpret_cast<const u32x4_a2*>(row + i * (16 / E));
    u32x4 x = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (i + j < n) {
            if (F16) x[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[i + j] << (16 * (j & 1));
            else x[j] = reinterpret_cast<const uint32_t*>(row)[i + j];
        }
    return x;
}
template <bool F16, int E>
__device__ __forceinline__ void unpack_raw(u32x4 x, float (&v)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = F16 ? h2f((uint16_t)(x[j >> 1] >> (16 * (j & 1)))) : __uint_as_float(x[j & 3]);
}
template <bool F16, int E>
__device__ __forceinline__ void st_some(char* row, int i, int n, const float (&v)[E]) {
    if (i + E <= n) {
        if constexpr (F16) {
            uint32_t x[E / 2];
#pragma unroll
            for (int j = 0; j < E; j += 2) x[j / 2] = (uint32_t)f2h(v[j]) | (uint32_t)f2h(v[j + 1]) << 16;
            if constexpr (E == 8) *reinterpret_cast<u32x4_a2*>(row + 2 * i) = u32x4{x[0], x[1], x[2], x[3]};
            else *reinterpret_cast<u32x2_a2*>(row + 2 * i) = u32x2{x[0], x[1]};
        } else {
#pragma unroll
            for (int j = 0; j < E; j += 4) *reinterpret_cast<v4f_a4*>(row + 4 * (i + j)) = v4f{v[j], v[j + 1], v[j + 2], v[j + 3]};
        }
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (i + j < n) st_one<F16>(row, i + j, v[j]);
    }
}

// T threads a row (64: a wavefront each, four rows to a workgroup), thread t holding elements E (v T + t) .. + E - 1,
// v < V: 16 bytes a load.  A wavefront's rows follow one another at the grid's stride, so that the weights are
// read once; what bounds the pass is memory, each operand moving once (8191 rows of 4736 halves with residual: 310 MB in
// 62.7 us, which is past the copy rate since a part is still in the last-level cache; 5184 rows of 1024 floats to Q8_0:
// 19.6 us with the read-back's launch for 80 MB), and for single tokens the launch (4096 floats: 6.6 to 8.4 us with the
// read-back's).  Rows beyond 8192 floats or 16384 halves want more registers than 1024 threads have, and spill (140 to 656
// bytes a lane): 512 rows of 32768 floats with residual 133 us, of halves 72, where their bytes take 57 and 29; 2048 of
// 16384 floats 112 for 114.
template <int T, int V, bool XF16>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rms_norm_kernel(const RmsArgs a) {
#pragma clang fp contract(off)
    constexpr int E = XF16 ? 8 : 4, NW = T / 64, RPB = T < 256 ? 256 / T : 1;
    __shared__ double red[2][NW];
    const int t = threadIdx.x % T, n = a.n;
    float w[V][E];
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < E; ++j) w[v][j] = 1.0f;
        const int i = E * (v * T + t);
        if (a.w && i < n) {
#pragma unroll
            for (int j = 0; j < E; j += 4) {
                const u32x4 x = ld_raw<false>(reinterpret_cast<const char*>(a.w), i + j, n);
#pragma unroll
                for (int k = 0; k < 4; ++k) w[v][j + k] = __uint_as_float(x[k]);
            }
        }
    }
    u32x4 rx[V], ra[V];
    auto load = [&](int64_t r) {
        const char* x = a.x.base + span_at(a.x, r, a.ne1, a.ne2);
#pragma unroll
        for (int v = 0; v < V; ++v) rx[v] = ld_raw<XF16>(x, E * (v * T + t), n);
        if (!a.add.base) return;
        const char* add = a.add.base + span_at(a.add, r, a.ne1, a.ne2);
#pragma unroll
        for (int v = 0; v < V; ++v) ra[v] = ld_raw<XF16>(add, E * (v * T + t), n);
    };
    int turn = 0;
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / T;
    if (r < a.rows) load(r);
    for (; r < a.rows; r += step, turn ^= 1) {
        char* sum = a.sum.base ? a.sum.base + span_at(a.sum, r, a.ne1, a.ne2) : nullptr;
        char* dst = a.dst.base + span_at(a.dst, r, a.ne1, a.ne2);
        float h[V][E];
        double s = 0.0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            unpack_raw<XF16, E>(rx[v], h[v]);
            if (a.add.base) {
                float g[E];
                unpack_raw<XF16, E>(ra[v], g);
#pragma unroll
                for (int j = 0; j < E; ++j) h[v][j] = h[v][j] + g[j];
            }
#pragma unroll
            for (int j = 0; j < E; ++j) s += (double)(h[v][j] * h[v][j]);
        }
        if (r + step < a.rows) load(r + step);  // the next row's bytes, while this one is reduced and written
        s = group_sum_d(s, 64);
        if constexpr (NW > 1) {
            if ((t & 63) == 0) red[turn][t >> 6] = s;
            __syncthreads();
            s = 0.0;
#pragma unroll
            for (int k = 0; k < NW; ++k) s += red[turn][k];
        }
        const float mean = (float)(s / (double)n);
        const float scale = 1.0f / sqrtf(mean + a.eps);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int i = E * (v * T + t);
            if (i >= n) break;  // (Q8: n % 32 == 0, so the lanes of a block leave together)
            if (sum) st_some<XF16, E>(sum, i, n, h[v]);
            float y[E];
#pragma unroll
            for (int j = 0; j < E; ++j) {
                y[j] = h[v][j] * scale;
                y[j] = y[j] * w[v][j];  // (without weights by one: no change)
            }
            if (a.out == T_F32) st_some<false, E>(dst, i, n, y);
            else if (a.out == T_F16) st_some<true, E>(dst, i, n, y);
            else {
                float amax = fabsf(y[0]);  // (a block of nothing but NaN, as one in the row makes it, has a NaN scale)
#pragma unroll
                for (int j = 1; j < E; ++j) amax = fmaxf(amax, fabsf(y[j]));
                amax = group_max<32 / E>(amax);
                const float d = amax / 127.0f, id = amax != 0.0f ? 127.0f / amax : 0.0f;
                uint32_t q[E / 4] = {};
                int isum = 0;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const int k = (int)rintf(y[j] * id);
                    isum += k;
                    q[j >> 2] |= (uint32_t)(k & 0xff) << (8 * (j & 3));
                }
                char* blk = dst + (int64_t)(i >> 5) * (a.out == T_Q8_0 ? 34 : 36);
                if (a.out == T_Q8_1) isum = group_sum_i<32 / E>(isum);
                if ((i & 31) == 0) {
                    reinterpret_cast<uint16_t*>(blk)[0] = f2h(d);
                    if (a.out == T_Q8_1) reinterpret_cast<uint16_t*>(blk)[1] = f2h(d * (float)isum);
                }
                char* qs = blk + (a.out == T_Q8_0 ? 2 : 4) + (i & 31);
                if constexpr (E == 8) *reinterpret_cast<u32x2_a2*>(qs) = u32x2{q[0], q[1]};
                else *reinterpret_cast<u32_a2*>(qs) = q[0];
            }
        }
    }
}

template <int T, int V, bool XF16>
static void rms_go(const RmsArgs& a, hipStream_t st) {
    constexpr int RPB = T < 256 ? 256 / T : 1;
    // as many workgroups as are on the CUs at a time, each with rows one after another (8191 rows of 4736 halves:
    // 62.5 us with 768, 68 with 2048; 5184 of 1024 floats 19.1 with 1024, 19.6 with 2048, 20.2 with 768)
    const int64_t g = std::min<int64_t>((a.rows + RPB - 1) / RPB, T == 1024 ? 512 : T == 256 && V >= 3 ? 768 : 1024);
    rms_norm_kernel<T, V, XF16><<<(unsigned)g, T < 256 ? 256 : T, 0, st>>>(a);
}
// A wavefront a row up to 1024 elements (F16: 2048); beyond, and where there are too few rows to occupy the CUs with
// that, more threads.
template <bool XF16>
static void rms_launch(const RmsArgs& a, hipStream_t st) {
    constexpr int E = XF16 ? 8 : 4;
    const int c = (a.n + E - 1) / E;  // 16-byte pieces
    const bool few = a.rows <= 512;
    if (c <= 64) rms_go<64, 1, XF16>(a, st);
    else if (c <= 256 && few) rms_go<256, 1, XF16>(a, st);
    else if (c <= 1024 && few) rms_go<1024, 1, XF16>(a, st);
    else if (c <= 128) rms_go<64, 2, XF16>(a, st);
    else if (c <= 256) rms_go<64, 4, XF16>(a, st);
    else if (c <= 512) rms_go<256, 2, XF16>(a, st);
    else if (c <= 768) rms_go<256, 3, XF16>(a, st);
    else if (c <= 1024) rms_go<256, 4, XF16>(a, st);
    else if (c <= 1280 && !few) rms_go<256, 5, XF16>(a, st);
    else if (c <= 1536 && !few) rms_go<256, 6, XF16>(a, st);
    else if (c <= 2048 && !few) rms_go<256, 8, XF16>(a, st);
    else if (c <= 2048) rms_go<1024, 2, XF16>(a, st);
    else if (c <= 4096) rms_go<1024, 4, XF16>(a, st);
    else if constexpr (!XF16) rms_go<1024, 8, XF16>(a, st);  // (RMS_MAX halves are 4096 pieces)
}

hipError_t launch_rms_norm(const RmsArgs& a, hipStream_t st) {
    if (a.rows <= 0 || a.n <= 0) return hipSuccess;
    if (a.n > RMS_MAX || a.rows > INT32_MAX) return hipErrorInvalidValue;
    if (a.xf16) rms_launch<true>(a, st);
    else rms_launch<false>(a, st);
    return hipGetLastError();
}

// Thread per 16 elements, half a block: 16 (Q4: 8) bytes in, 32 or 64 out, all at the blocks' 2-byte alignment.  Bound
// by memory, nearly all of it the floats written.
// flat: the rows of dst lie back to back.
template <int TYPE, bool F16>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const uint8_t* __restrict__ src, RowSpan dst, int flat, int64_t n16,
                                                              int64_t total, int64_t ne1, int64_t ne2) {
#pragma clang fp contract(off)
    constexpr int SIZE = TYPE == T_Q8_0 ? 34 : TYPE == T_Q8_1 ? 36 : TYPE == T_Q4_0 ? 18 : 20;
    constexpr int HEAD = TYPE == T_Q8_0 || TYPE == T_Q4_0 ? 2 : 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const uint8_t* blk = src + (i >> 1) * SIZE;
    const int half = (int)(i & 1);
    const float d = h2f(*reinterpret_cast<const uint16_t*>(blk));
    float y[16];
    if constexpr (TYPE == T_Q8_0 || TYPE == T_Q8_1) {
        const u32x4 q = *reinterpret_cast<const u32x4_a2*>(blk + HEAD + 16 * half);
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = (float)(int8_t)(q[j >> 2] >> (8 * (j & 3))) * d;
    } else {  // the low nibbles are the first half, the high ones the second
        const float m = TYPE == T_Q4_1 ? h2f(reinterpret_cast<const uint16_t*>(blk)[1]) : 0.0f;
        const u32x4 q = *reinterpret_cast<const u32x4_a2*>(blk + HEAD);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int v = (int)(q[j >> 2] >> (8 * (j & 3) + 4 * half) & 15);
            y[j] = TYPE == T_Q4_0 ? (float)(v - 8) * d : (float)v * d + m;
        }
    }
    const int64_t r = flat ? 0 : i / n16, e = 16 * (i - r * n16);
    char* o = dst.base + (flat ? 0 : span_at(dst, r, ne1, ne2)) + e * (F16 ? 2 : 4);
#pragma unroll
    for (int j = 0; j < 16; j += 8) {
        const float z[8] = {y[j], y[j + 1], y[j + 2], y[j + 3], y[j + 4], y[j + 5], y[j + 6], y[j + 7]};
        st_some<F16, 8>(o, j, 16, z);
    }
}

hipError_t launch_dequantize_rows(const void* src, int type, const RowSpan& dst, bool f16, int64_t n, int64_t rows,
                                  int64_t ne1, int64_t ne2, hipStream_t st) {
    const int64_t total = rows * (n / 16);
    if (total <= 0) return hipSuccess;
    if ((total + 255) / 256 > INT32_MAX) return hipErrorInvalidValue;
    const int64_t pitch = n * (f16 ? 2 : 4);
    const int flat = (ne1 == 1 || dst.nb[0] == pitch) && (ne2 == 1 || dst.nb[1] == pitch * ne1) &&
                     (rows == ne1 * ne2 || dst.nb[2] == pitch * ne1 * ne2);
    const unsigned g = (unsigned)((total + 255) / 256);
    const uint8_t* s = static_cast<const uint8_t*>(src);
    auto go = [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        if (f16) dequantize_rows_kernel<TYPE, true><<<g, 256, 0, st>>>(s, dst, flat, n / 16, total, ne1, ne2);
        else dequantize_rows_kernel<TYPE, false><<<g, 256, 0, st>>>(s, dst, flat, n / 16, total, ne1, ne2);
    };
    switch (type) {
        case T_Q8_0: go(std::integral_constant<int, T_Q8_0>()); break;
        case T_Q8_1: go(std::integral_constant<int, T_Q8_1>()); break;
        case T_Q4_0: go(std::integral_constant<int, T_Q4_0>()); break;
        case T_Q4_1: go(std::integral_constant<int, T_Q4_1>()); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// thread per half block of 16 quants; the scale slots as act_store_scale's
__global__ __launch_bounds__(256) void unpack_q8_kernel(const uint8_t* __restrict__ src, int64_t nb1, int sums, int64_t nbpr,
                                                        int64_t total, int64_t K, int8_t* q, uint32_t* dl, uint32_t* dh,
                                                        uint16_t* s) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t r = (i >> 1) / nbpr, b = (i >> 1) - r * nbpr, nst = (nbpr + 1) / 2;
    const uint8_t* blk = src + r * nb1 + b * (sums ? 36 : 34);
    const uint8_t* p = blk + (sums ? 4 : 2) + 16 * (i & 1);
    const uint4 v = make_uint4(ld_u32_a2(p), ld_u32_a2(p + 4), ld_u32_a2(p + 8), ld_u32_a2(p + 12));
    *reinterpret_cast<uint4*>(q + r * K + 32 * b + 16 * (i & 1)) = v;
    if (i & 1) return;
    const uint32_t d = *reinterpret_cast<const uint16_t*>(blk);
    if ((b & 1) == 0) dl[r * nst + b / 2] = d;
    else dh[r * nst + b / 2] = d << 16;
    if (b == nbpr - 1 && (nbpr & 1)) dh[r * nst + b / 2] = 0;
    if (sums) {
        s[r * 2 * nst + b] = reinterpret_cast<const uint16_t*>(blk)[1];
        if (b == nbpr - 1 && (nbpr & 1)) s[r * 2 * nst + b + 1] = 0;
    }
}

hipError_t launch_unpack_q8(const void* src, int64_t nb1, int type, int64_t M, int64_t K, void* q, uint32_t* dl, uint32_t* dh,
                            void* s, hipStream_t st) {
    const int64_t total = M * (K / 32) * 2;
    if (total <= 0) return hipSuccess;
    unpack_q8_kernel<<<(unsigned)((total + 255) / 256), 256, 0, st>>>(static_cast<const uint8_t*>(src), nb1, type == T_Q8_1,
                                                                      K / 32, total, K, static_cast<int8_t*>(q), dl, dh,
                                                                      static_cast<uint16_t*>(s));
    return hipGetLastError();
}

}  // namespace mi355
