// The residual's addition, RMS norm and the next product's 8-bit operand in one pass over the
// rows (ggml_add, ggml_rms_norm, ggml_mul, from_float), and ggml's to_float back.
//
//   h = x + add, y = h * (1 / sqrt(mean(h^2) + eps)) * w
//
// The squares are fp32 products summed in double, as ggml_rms_norm does, so the sum's order changes
// the fp32 mean about once in 10^7 rows and the 8-bit quants behind it do not depend on it.
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

// One workgroup of T threads a row; thread t holds elements 8 (v T + t) .. + 7, v < V.
template <int T, int V, bool XF16>
__global__ __launch_bounds__(T) void rms_norm_kernel(const RmsArgs a) {
#pragma clang fp contract(off)
    __shared__ double red[T / 64];
    const int64_t r = blockIdx.x;
    const int t = threadIdx.x, n = a.n;
    const char* x = a.x.base + span_at(a.x, r, a.ne1, a.ne2);
    const char* add = a.add.base ? a.add.base + span_at(a.add, r, a.ne1, a.ne2) : nullptr;
    char* sum = a.sum.base ? a.sum.base + span_at(a.sum, r, a.ne1, a.ne2) : nullptr;
    char* dst = a.dst.base + span_at(a.dst, r, a.ne1, a.ne2);
    float h[V][8];
    double s = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = 8 * (v * T + t) + j;
            h[v][j] = 0.0f;
            if (i < n) {
                h[v][j] = ld_one<XF16>(x, i);
                if (add) h[v][j] += ld_one<XF16>(add, i);
                s += (double)(h[v][j] * h[v][j]);
            }
        }
    s = group_sum_d(s, 64);
    if ((t & 63) == 0) red[t >> 6] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) s += red[w];
    const float mean = (float)(s / (double)n);
    const float scale = 1.0f / sqrtf(mean + a.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i0 = 8 * (v * T + t);
        if (i0 >= n) break;  // (Q8: n % 32 == 0, so the four lanes of a block leave together)
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i0 + j < n && sum) st_one<XF16>(sum, i0 + j, h[v][j]);
            y[j] = h[v][j] * scale;
            if (a.w && i0 + j < n) y[j] = y[j] * a.w[i0 + j];
        }
        if (a.out == T_F32 || a.out == T_F16) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i0 + j < n) {
                    if (a.out == T_F16) st_one<true>(dst, i0 + j, y[j]);
                    else st_one<false>(dst, i0 + j, y[j]);
                }
            continue;
        }
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
        amax = group_max<4>(amax);
        const float d = amax / 127.0f, id = amax != 0.0f ? 127.0f / amax : 0.0f;
        int q[8], isum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q[j] = (int)rintf(y[j] * id);
            isum += q[j];
        }
        isum = group_sum_i<4>(isum);
        const int b = i0 >> 5, part = (i0 >> 3) & 3;
        uint16_t* blk = reinterpret_cast<uint16_t*>(dst + (int64_t)b * (a.out == T_Q8_0 ? 34 : 36));
        if (part == 0) {
            blk[0] = f2h(d);
            if (a.out == T_Q8_1) blk[1] = f2h(d * (float)isum);
        }
        uint16_t* qs = blk + (a.out == T_Q8_0 ? 1 : 2) + 4 * part;
#pragma unroll
        for (int j = 0; j < 4; ++j) qs[j] = (uint16_t)((q[2 * j] & 0xff) | ((q[2 * j + 1] & 0xff) << 8));
    }
}

template <bool XF16>
static void rms_launch(const RmsArgs& a, hipStream_t st) {
    const unsigned g = (unsigned)a.rows;
    if (a.n <= 512) rms_norm_kernel<64, 1, XF16><<<g, 64, 0, st>>>(a);
    else if (a.n <= 2048) rms_norm_kernel<256, 1, XF16><<<g, 256, 0, st>>>(a);
    else if (a.n <= 8192) rms_norm_kernel<256, 4, XF16><<<g, 256, 0, st>>>(a);
    else rms_norm_kernel<1024, 4, XF16><<<g, 1024, 0, st>>>(a);
}

hipError_t launch_rms_norm(const RmsArgs& a, hipStream_t st) {
    if (a.rows <= 0 || a.n <= 0) return hipSuccess;
    if (a.n > RMS_MAX || a.rows > INT32_MAX) return hipErrorInvalidValue;
    if (a.xf16) rms_launch<true>(a, st);
    else rms_launch<false>(a, st);
    return hipGetLastError();
}

// thread per four elements
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const uint8_t* __restrict__ src, int type, RowSpan dst, int f16,
                                                              int64_t n4, int64_t total, int64_t ne1, int64_t ne2) {
#pragma clang fp contract(off)
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t r = i / n4, c = i - r * n4, b = i / 8;
    const int e = (int)(i & 7) * 4;
    float y[4];
    if (type == T_Q8_0 || type == T_Q8_1) {
        const uint8_t* blk = src + b * (type == T_Q8_0 ? 34 : 36);
        const float d = h2f(*reinterpret_cast<const uint16_t*>(blk));
        const uint32_t q = ld_u32_a2(blk + (type == T_Q8_0 ? 2 : 4) + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = (float)(int8_t)(q >> (8 * j)) * d;
    } else {
        const uint8_t* blk = src + b * (type == T_Q4_0 ? 18 : 20);
        const float d = h2f(*reinterpret_cast<const uint16_t*>(blk));
        const float m = type == T_Q4_1 ? h2f(reinterpret_cast<const uint16_t*>(blk)[1]) : 0.0f;
        const uint32_t q = ld_u32_a2(blk + (type == T_Q4_0 ? 2 : 4) + (e & 15)) >> (e >= 16 ? 4 : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int v = (q >> (8 * j)) & 15;
            y[j] = type == T_Q4_0 ? (float)(v - 8) * d : (float)v * d + m;
        }
    }
    char* o = dst.base + span_at(dst, r, ne1, ne2);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (f16) st_one<true>(o, (int)(4 * c + j), y[j]);
        else st_one<false>(o, (int)(4 * c + j), y[j]);
    }
}

hipError_t launch_dequantize_rows(const void* src, int type, const RowSpan& dst, bool f16, int64_t n, int64_t rows,
                                  int64_t ne1, int64_t ne2, hipStream_t st) {
    const int64_t total = rows * (n / 4);
    if (total <= 0) return hipSuccess;
    if ((total + 255) / 256 > INT32_MAX) return hipErrorInvalidValue;
    dequantize_rows_kernel<<<(unsigned)((total + 255) / 256), 256, 0, st>>>(static_cast<const uint8_t*>(src), type, dst, f16,
                                                                            n / 4, total, ne1, ne2);
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
