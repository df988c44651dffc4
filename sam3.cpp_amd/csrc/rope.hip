// Rotary positions over several axes: pair i of a head turns by pos[axis(i)] * f(i).
//
// f is held as a fraction of a turn in 64-bit fixed point (turn = f / (2 pi) * 2^64), so
// pos * turn modulo 2^64 is the angle modulo a turn, exact to 2^-33 turns for every int32
// position; what is left within an eighth of a turn is a fp32 angle for two Taylor series.
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

template <bool F16>
__device__ __forceinline__ float rope_ld(const char* p, int i) {
    return F16 ? h2f(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
template <bool F16>
__device__ __forceinline__ void rope_st(char* p, int i, float v) {
    if (F16) reinterpret_cast<uint16_t*>(p)[i] = f2h(v);
    else reinterpret_cast<float*>(p)[i] = v;
}

// thread per pair (or copied element) of a token, over its heads
template <bool F16>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
    const int per = a.pairs + a.ne0 - 2 * a.pairs;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)per * a.tokens * a.batch) return;
    const int p = (int)(i % per);
    const int64_t bt = i / per, b = bt / a.tokens, t = bt - b * a.tokens;
    const char* src = a.src + t * a.s_nb[1] + b * a.s_nb[2];
    char* dst = a.dst + t * a.d_nb[1] + b * a.d_nb[2];
    if (p >= a.pairs) {  // past the turned elements
        for (int h = 0; h < a.heads; ++h)
            rope_st<F16>(dst + h * a.d_nb[0], a.pairs + p, rope_ld<F16>(src + h * a.s_nb[0], a.pairs + p));
        return;
    }
    const int pos = a.pos[(int64_t)a.axis[p] * a.batch * a.tokens + bt];
    float c, s;
    turn_sincos((uint64_t)(int64_t)pos * a.turn[p], c, s);
    const int e0 = a.halves ? p : 2 * p, e1 = a.halves ? p + a.pairs : 2 * p + 1;
    for (int h = 0; h < a.heads; ++h) {
        const float x0 = rope_ld<F16>(src + h * a.s_nb[0], e0), x1 = rope_ld<F16>(src + h * a.s_nb[0], e1);
        rope_st<F16>(dst + h * a.d_nb[0], e0, x0 * c - x1 * s);
        rope_st<F16>(dst + h * a.d_nb[0], e1, x0 * s + x1 * c);
    }
}

hipError_t launch_rope_multi(const RopeArgs& a, hipStream_t st) {
    const int64_t n = (int64_t)(a.ne0 - a.pairs) * a.tokens * a.batch;
    if (n <= 0 || a.heads <= 0) return hipSuccess;
    const int64_t g = (n + 255) / 256;
    if (g > INT32_MAX) return hipErrorInvalidValue;
    if (a.f16) rope_kernel<true><<<(unsigned)g, 256, 0, st>>>(a);
    else rope_kernel<false><<<(unsigned)g, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace mi355
