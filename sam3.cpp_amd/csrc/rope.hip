// Rotary positions over several axes: pair i of a head turns by pos[axis(i)] * f(i).
//
// f is held as a fraction of a turn in 64-bit fixed point (turn = f / (2 pi) * 2^64), so
// pos * turn modulo 2^64 is the angle modulo a turn; turn itself is good to 2^-61 (rope_table), so
// the angle to 2^-30 of a turn at the ends of int32.  What is left within an eighth of a turn is a
// fp32 angle for two Taylor series.
#include "common.cuh"
#include "kernels.h"

namespace mi355 {

// cos and sin of 2 pi phase / 2^64
__device__ __forceinline__ void turn_sincos(uint64_t phase, float& c, float& s) {
    const uint32_t top = (uint32_t)(phase >> 32);
    const uint32_t quad = (top + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(top - (quad << 30)) * 1.46291807926715968e-9f;  // |x| <= pi / 4
    const float t = x * x;
    // sin to x^9 / 9!, cos to x^10 / 10!: the next terms are below 2e-9 and 1e-10 at pi / 4
    float ps = 2.75573192e-6f;
    ps = __builtin_fmaf(ps, t, -1.98412698e-4f);
    ps = __builtin_fmaf(ps, t, 8.33333333e-3f);
    ps = __builtin_fmaf(ps, t, -1.66666667e-1f);
    const float sn = __builtin_fmaf(x * t, ps, x);
    float pc = -2.75573192e-7f;
    pc = __builtin_fmaf(pc, t, 2.48015873e-5f);
    pc = __builtin_fmaf(pc, t, -1.38888889e-3f);
    pc = __builtin_fmaf(pc, t, 4.16666667e-2f);
    pc = __builtin_fmaf(pc, t, -0.5f);
    const float cs = __builtin_fmaf(pc, t, 1.0f);
    c = (quad & 1) ? sn : cs;
    s = (quad & 1) ? cs : sn;
    if (quad == 1 || quad == 2) c = -c;
    if (quad & 2) s = -s;
}

namespace {
typedef v4f v4f_a4 __attribute__((aligned(4)));
typedef v8h v8h_a2 __attribute__((aligned(2)));
typedef v4h v4h_a2 __attribute__((aligned(2)));
}  // namespace

// N consecutive elements (4 or 8) at any alignment of their type
template <bool F16, int N>
__device__ __forceinline__ void rope_ld(const char* p, float (&v)[N]) {
    if constexpr (!F16) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const v4f x = *reinterpret_cast<const v4f_a4*>(p + 4 * j);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j + k] = x[k];
        }
    } else if constexpr (N == 8) {
        const v8h x = *reinterpret_cast<const v8h_a2*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)x[j];
    } else {
        const v4h x = *reinterpret_cast<const v4h_a2*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)x[j];
    }
}
template <bool F16, int N>
__device__ __forceinline__ void rope_st(char* p, const float (&v)[N]) {
    if constexpr (!F16) {
#pragma unroll
        for (int j = 0; j < N; j += 4) *reinterpret_cast<v4f_a4*>(p + 4 * j) = v4f{v[j], v[j + 1], v[j + 2], v[j + 3]};
    } else if constexpr (N == 8) {
        v8h x;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (_Float16)v[j];
        *reinterpret_cast<v8h_a2*>(p) = x;
    } else {
        v4h x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (_Float16)v[j];
        *reinterpret_cast<v4h_a2*>(p) = x;
    }
}
template <bool F16>
__device__ __forceinline__ float rope_ld1(const char* p, int i) {
    return F16 ? h2f(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
template <bool F16>
__device__ __forceinline__ void rope_st1(char* p, int i, float v) {
    if (F16) reinterpret_cast<uint16_t*>(p)[i] = f2h(v);
    else reinterpret_cast<float*>(p)[i] = v;
}

// A thread turns four neighbouring pairs of a token in H heads, `across` heads apart, with one set of angles; its
// neighbours take the head's other pairs, then the next heads.  Pieces after the pairs copy eight elements each.  Bound
// by memory, every element moving once in 16-byte (halves of an F16 head: 8) accesses: 4 x 5184 tokens of 16 heads of 64
// floats, 170 MB, in 35.5 us (4.8 TB/s); 32 single tokens of 40 heads of 128 halves are a launch, 5.0 us.
template <bool F16, bool HALVES, int H>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a, const int pieces, const int across, const int items) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const int c = i % pieces, hb = i / pieces, h0 = hb % across, bt = hb / across;
    const int b = bt / a.tokens, t = bt - b * a.tokens;
    const char* src = a.src + t * a.s_nb[1] + b * a.s_nb[2];
    char* dst = a.dst + t * a.d_nb[1] + b * a.d_nb[2];
    const int turning = (a.pairs + 3) / 4;
    constexpr int ES = F16 ? 2 : 4;
    if (c >= turning) {
        const int e = 2 * a.pairs + 8 * (c - turning);
#pragma unroll
        for (int k = 0; k < H; ++k) {
            const int h = h0 + across * k;
            if (h >= a.heads) break;
            const char* s = src + h * a.s_nb[0];
            char* d = dst + h * a.d_nb[0];
            for (int j = e; j < e + 8 && j < a.ne0; ++j) rope_st1<F16>(d, j, rope_ld1<F16>(s, j));
        }
        return;
    }
    const int p0 = 4 * c;
    const bool whole = p0 + 4 <= a.pairs;
    const int e0 = HALVES ? p0 : 2 * p0, e1 = p0 + a.pairs;  // (HALVES) second elements
    float x[H][8];
    auto fetch = [&](const char* s, float (&v)[8]) {
        if (whole) {
            if constexpr (HALVES) {
                float lo[4], hi[4];
                rope_ld<F16, 4>(s + ES * e0, lo);
                rope_ld<F16, 4>(s + ES * e1, hi);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[2 * j] = lo[j], v[2 * j + 1] = hi[j];
            } else {
                rope_ld<F16, 8>(s + ES * e0, v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p0 + j < a.pairs) v[2 * j] = rope_ld1<F16>(s, HALVES ? e0 + j : e0 + 2 * j), v[2 * j + 1] = rope_ld1<F16>(s, HALVES ? e1 + j : e0 + 2 * j + 1);
        }
    };
#pragma unroll
    for (int k = 0; k < H; ++k)
        if (h0 + across * k < a.heads) fetch(src + (h0 + across * k) * a.s_nb[0], x[k]);
    float cs[4], sn[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int p = min(p0 + j, a.pairs - 1);
        const int pos = a.pos[(int64_t)a.axis[p] * a.batch * a.tokens + bt];
        turn_sincos((uint64_t)(int64_t)pos * a.turn[p], cs[j], sn[j]);
    }
#pragma unroll
    for (int k = 0; k < H; ++k) {
        const int h = h0 + across * k;
        if (h >= a.heads) break;
        char* d = dst + h * a.d_nb[0];
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            y[2 * j] = x[k][2 * j] * cs[j] - x[k][2 * j + 1] * sn[j];
            y[2 * j + 1] = x[k][2 * j] * sn[j] + x[k][2 * j + 1] * cs[j];
        }
        if (whole) {
            if constexpr (HALVES) {
                const float lo[4] = {y[0], y[2], y[4], y[6]}, hi[4] = {y[1], y[3], y[5], y[7]};
                rope_st<F16, 4>(d + ES * e0, lo);
                rope_st<F16, 4>(d + ES * e1, hi);
            } else {
                rope_st<F16, 8>(d + ES * e0, y);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (p0 + j < a.pairs) {
                    rope_st1<F16>(d, HALVES ? e0 + j : e0 + 2 * j, y[2 * j]);
                    rope_st1<F16>(d, HALVES ? e1 + j : e0 + 2 * j + 1, y[2 * j + 1]);
                }
        }
    }
}

template <bool F16, bool HALVES>
static void rope_go(const RopeArgs& a, int pieces, hipStream_t st) {
    const int64_t bt = (int64_t)a.tokens * a.batch;
    // four heads to a thread where that leaves enough threads to occupy the CUs
    if (bt * pieces * ((a.heads + 3) / 4) >= 1 << 17) {
        const int across = (a.heads + 3) / 4;
        const int64_t items = bt * pieces * across;
        rope_kernel<F16, HALVES, 4><<<(unsigned)((items + 255) / 256), 256, 0, st>>>(a, pieces, across, (int)items);
    } else {
        const int64_t items = bt * pieces * a.heads;
        rope_kernel<F16, HALVES, 1><<<(unsigned)((items + 255) / 256), 256, 0, st>>>(a, pieces, a.heads, (int)items);
    }
}

hipError_t launch_rope_multi(const RopeArgs& a, hipStream_t st) {
    const int rest = a.ne0 - 2 * a.pairs, pieces = (a.pairs + 3) / 4 + (rest + 7) / 8;
    const int64_t bt = (int64_t)a.tokens * a.batch;
    if (bt <= 0 || a.heads <= 0 || pieces <= 0) return hipSuccess;
    if (bt * pieces * ((a.heads + 3) / 4) > INT32_MAX - 256) return hipErrorInvalidValue;
    if (a.f16) a.halves ? rope_go<true, true>(a, pieces, st) : rope_go<true, false>(a, pieces, st);
    else a.halves ? rope_go<false, true>(a, pieces, st) : rope_go<false, false>(a, pieces, st);
    return hipGetLastError();
}

}  // namespace mi355
