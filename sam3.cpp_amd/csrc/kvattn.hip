// Attention over the 8-bit cache of kvcache.hip:
//
//   dst[s][i][h] = sum_t softmax_t(scale q_i . k_t) v_t
//
// over the tokens t that query i sees (n_kv, causal, window), with fp32 online softmax.
#include "common.cuh"
#include "kernels.h"

namespace mi355 {

// One wavefront for each query and head, 64 tokens a step: a lane scores one token, then every lane
// adds the step's values for its elements lane, lane + 64 of the head.
template <int D>
__global__ __launch_bounds__(64) void kv_attn_simple_kernel(const KvAttnArgs a) {
    constexpr int NE = (D + 63) / 64;
    __shared__ float qs[D], ps[64];
    const KvView& c = a.c;
    const int lane = threadIdx.x;
    const int64_t w = blockIdx.x;
    const int h = (int)(w % a.heads), i = (int)(w / a.heads % a.n_q), s = (int)(w / a.heads / a.n_q);
    const int n_kv = (int)min((int64_t)max(c.n_kv[s], 0), (int64_t)c.max_blocks * c.bt);
    const int nq = a.nq ? min(max(a.nq[s], 0), a.n_q) : a.n_q;
    if (i >= nq) return;
    const int p = n_kv - nq + i;
    const int end = a.causal ? min(p + 1, n_kv) : n_kv, begin = a.window > 0 ? max(p - a.window + 1, 0) : 0;
    const char* q = a.q + i * a.q_nb[0] + h * a.q_nb[1] + s * a.q_nb[2];
    for (int e = lane; e < D; e += 64)
        qs[e] = a.q16 ? h2f(reinterpret_cast<const uint16_t*>(q)[e]) : reinterpret_cast<const float*>(q)[e];
    __syncthreads();
    float m = -__builtin_inff(), l = 0.0f, o[NE] = {};
    for (int t0 = begin; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        float sc = -__builtin_inff();
        if (t < end) {
            const int id = c.table[(int64_t)s * c.max_blocks + t / c.bt];
            if (id >= 0 && id < c.n_blocks) {
                const int64_t at = (int64_t)id * c.heads + h / a.group;
                const uint8_t* k = c.k + (at * c.bt + t % c.bt) * D;
                float dot = 0.0f;
                for (int e = 0; e < D; ++e) dot = __builtin_fmaf(qs[e], (float)((int)k[e] - 128), dot);
                sc = dot * (c.k_scale[at] * a.scale);
            }
        }
        const float mx = fmaxf(m, group_max<64>(sc));
        if (mx == -__builtin_inff()) continue;
        const float alpha = expf(m - mx), pr = expf(sc - mx);
        m = mx;
        l = l * alpha + group_sum<64>(pr);
        ps[lane] = pr;
        __syncthreads();
        for (int x = 0; x < NE; ++x) o[x] *= alpha;
        for (int j = 0; j < 64 && t0 + j < end; ++j) {
            if (ps[j] == 0.0f) continue;
            const int tt = t0 + j, id = c.table[(int64_t)s * c.max_blocks + tt / c.bt];
            const int64_t at = (int64_t)id * c.heads + h / a.group;
            const uint8_t* v = c.v + (at * c.bt + tt % c.bt) * D;
            const float f = ps[j] * c.v_scale[at];
            for (int x = 0; x < NE; ++x)
                if (lane + 64 * x < D) o[x] = __builtin_fmaf(f, (float)((int)v[lane + 64 * x] - 128), o[x]);
        }
        __syncthreads();
    }
    char* d = a.dst + h * a.d_nb[0] + i * a.d_nb[1] + s * a.d_nb[2];
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    for (int x = 0; x < NE; ++x)
        if (lane + 64 * x < D) {
            if (a.d16) reinterpret_cast<uint16_t*>(d)[lane + 64 * x] = f2h(o[x] * inv);
            else reinterpret_cast<float*>(d)[lane + 64 * x] = o[x] * inv;
        }
}

hipError_t launch_kv_attn(const KvAttnArgs& a, int D, hipStream_t st) {
    const int64_t g = (int64_t)a.n_q * a.heads * a.c.n_seq;
    if (g <= 0) return hipSuccess;
    if (g > INT32_MAX) return hipErrorInvalidValue;
    if (D == 64) kv_attn_simple_kernel<64><<<(unsigned)g, 64, 0, st>>>(a);
    else if (D == 96) kv_attn_simple_kernel<96><<<(unsigned)g, 64, 0, st>>>(a);
    else if (D == 128) kv_attn_simple_kernel<128><<<(unsigned)g, 64, 0, st>>>(a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace mi355
