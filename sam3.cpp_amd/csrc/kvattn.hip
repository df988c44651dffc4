// Attention over the 8-bit cache of kvcache.hip:
//
//   dst[s][i][h] = sum_t softmax_t(scale q_i . k_t) v_t
//
// over the tokens t that query i sees (n_kv, causal, window), with fp32 online softmax.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace mi355 {

namespace {
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef v4f v4f_a4 __attribute__((aligned(4)));
typedef v2f v2f_a4 __attribute__((aligned(4)));
typedef v8h v8h_a2 __attribute__((aligned(2)));
typedef v4h v4h_a2 __attribute__((aligned(2)));
typedef h2v h2v_a2 __attribute__((aligned(2)));
constexpr float KV_LOG2E = 1.44269504088896340736f;
constexpr float KV_NONE = -1e30f;    // a reference that nothing has been taken against yet
constexpr float KV_LIFT = 12.0f;     // probabilities are raised by 2^12 to keep small ones in fp16's normal range
constexpr float KV_ROOM = 15.0f;     // and their reference moves when one would pass 2^15
constexpr int KV_STEP = 32;          // tokens of one step of a wavefront
constexpr int KV_SPAN = 4 * KV_STEP; // tokens of one step of a workgroup
}  // namespace

// The tokens that a sequence's queries can see, and its queries.
struct KvRange {
    int n_kv, nq, pos0;  // length, queries, position of the first query
    int lo, hi;          // tokens lo .. hi - 1 (lo a multiple of a step) are seen by some query
};
__device__ __forceinline__ KvRange kv_range(const KvAttnArgs& a, int s) {
    KvRange r;
    r.n_kv = (int)min((int64_t)max(a.c.n_kv[s], 0), (int64_t)a.c.max_blocks * a.c.bt);
    r.nq = a.nq ? min(max(a.nq[s], 0), a.n_q) : a.n_q;
    r.pos0 = r.n_kv - r.nq;
    r.lo = a.window > 0 ? (int)(max((int64_t)r.pos0 - a.window + 1, (int64_t)0) & ~(int64_t)(KV_STEP - 1)) : 0;
    r.hi = r.n_kv;
    return r;
}
// Tokens of each of `splits` ranges: whole workgroup steps
__device__ __forceinline__ int kv_chunk(const KvRange& r, int splits) {
    const int n = max(r.hi - r.lo, 1), per = (n + splits - 1) / splits;
    return (per + KV_SPAN - 1) / KV_SPAN * KV_SPAN;
}

// four bytes of keys as the halves u - 128 (exact): 0x64uu is the half 1024 + u
__device__ __forceinline__ void key_halves(uint32_t v, uint32_t* o) {
    const h2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    o[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, v, 0x04010400u)) + off);
    o[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, v, 0x04030402u)) + off);
}
// byte b of two tokens' values as the halves (u - 128) / 512 (exact): 0x00uu is the half u 2^-24
__device__ __forceinline__ uint32_t value_halves(uint32_t t0, uint32_t t1, int b) {
    const h2v mul = {(_Float16)32768.0f, (_Float16)32768.0f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
    const h2v u = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(t1, t0, 0x0c040c00u | (uint32_t)b | (uint32_t)b << 16));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(u, mul, off));
}

// log2 of a block's scale, -inf for 0; the instruction takes no subnormals
__device__ __forceinline__ float scale_log2(float v) {
    const bool tiny = v < 7.8886091e-31f;  // 2^-100
    return __builtin_amdgcn_logf(tiny ? v * 1.1529215e18f : v) - (tiny ? 60.0f : 0.0f);
}

// max and sum over the four lanes of a column (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float col_max(float v) {
    v = fmaxf(v, lane_swap_f<16>(v));
    return fmaxf(v, lane_swap_f<32>(v));
}
__device__ __forceinline__ float col_sum(float v) {
    v += lane_swap_f<16>(v);
    return v + lane_swap_f<32>(v);
}

// Few query rows over many tokens.  A row is one query and head of the group that shares a key head: row
// r of a sequence and key head is query r / group, head r % group.  A workgroup takes 16 NT rows and
// one range of the tokens, its four wavefronts every fourth step of 32 tokens; nothing passes through
// LDS but the join of the four at the end, so that the cache's bytes go from memory to the registers
// that the matrix instructions read, each once.
//   scores  S^T[token][row] = K Q^T (v_mfma_f32_16x16x32_f16): a lane holds 16 bytes of each 64 of one
//           key row, and the rows' queries in the same order of elements;
//   output  O^T[d][row] += V^T P^T: a lane's eight scores (tokens 4g .. 4g + 3 of both 16-token halves, g =
//           lane / 16) are the eight places of its column in the B operand, and the A operand takes the
//           same tokens of D / 16 neighbouring elements, a pair of tokens to a register by one byte
//           permutation.
// A block's value scale is part of the exponent of its probabilities, P = 2^(s + log2(v_scale) - M), and
// comes out of the sum again with one factor for a block, l += 2^(M - m - log2(v_scale)) sum P; where
// that factor passes 2^90 (scales far below the others', and zero) the sum is taken of 2^(s - m) itself.
// QS: an F32 q enters as two halves of 11 bits, scaled by a power of two that brings the row's largest
// magnitude to about one.  PS: for an F32 output the probabilities enter as two halves too.
template <int D, int NT, bool QS, bool PS>
__global__ __launch_bounds__(256, 2) void kv_attn_rows_kernel(const KvAttnArgs a, const int splits, const int tiles) {
    constexpr int KC = D / 64, KM = D / 32, NB = D / 16;  // key chunks of 64, score products, output blocks
    constexpr bool TAIL = D % 64 != 0;                    // D = 96: 32 more elements
    const KvView& c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    // the row tiles of one item go to the same XCD, one after another, and find its bytes in that L2
    const int per = 8 * tiles, gb = blockIdx.x / per, rb = blockIdx.x % per;
    const int item = gb * 8 + (rb & 7), tile = rb >> 3;
    if (item >= splits * c.heads * c.n_seq) return;
    const int sp = item % splits, hk = item / splits % c.heads, s = item / splits / c.heads;
    const KvRange kr = kv_range(a, s);
    const int rows = kr.nq * a.group, row0 = tile * 16 * NT;
    if (row0 >= rows) return;
    const int chunk = kv_chunk(kr, splits), tb = kr.lo + sp * chunk;
    // tokens that some row of this tile can see
    const int last = min(row0 + 16 * NT, rows) - 1;
    const int hi_tile = a.causal ? min(kr.pos0 + last / a.group + 1, kr.hi) : kr.hi;
    const int te = min(min(tb + chunk, kr.hi), hi_tile);
    if (splits > 1 && sp > 0 && tb >= kr.hi) return;  // no such range (the first always answers)

    // queries
    v8h q[NT][KM], ql[QS ? NT : 1][KM];
    float qscale[NT];
    int see_lo[NT], see_hi[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + col, iq = r / a.group, h = hk * a.group + (r - iq * a.group);
        const bool on = r < rows;
        const char* p = a.q + (int64_t)iq * a.q_nb[0] + (int64_t)h * a.q_nb[1] + (int64_t)s * a.q_nb[2];
        const int pos = kr.pos0 + iq;
        see_hi[t] = on ? (a.causal ? min(pos + 1, kr.hi) : kr.hi) : 0;
        see_lo[t] = a.window > 0 ? pos - a.window + 1 : 0;
        qscale[t] = 1.0f;
        if constexpr (QS) {
            float x[KM][8], top = 0.0f;
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                const int e = TAIL && m == KM - 1 ? 64 + 8 * g : 64 * (m >> 1) + 16 * g + 8 * (m & 1);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[m][j] = 0.0f;
                if (on) {
                    const v4f lo = *reinterpret_cast<const v4f_a4*>(p + 4 * e), hi = *reinterpret_cast<const v4f_a4*>(p + 4 * e + 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[m][j] = lo[j];
                        x[m][4 + j] = hi[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[m][j]));
            }
            top = col_max(top);
            // 2^-e of top's exponent e, and 2^e for the scores
            const int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            const int ec = min(max(e, -126), 126);
            const float down = __uint_as_float((uint32_t)(127 - ec) << 23);
            qscale[t] = __uint_as_float((uint32_t)(127 + ec) << 23);
#pragma unroll
            for (int m = 0; m < KM; ++m)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = x[m][j] * down;
                    q[t][m][j] = (_Float16)y;
                    ql[t][m][j] = (_Float16)(y - (float)q[t][m][j]);
                }
        } else {
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                const int e = TAIL && m == KM - 1 ? 64 + 8 * g : 64 * (m >> 1) + 16 * g + 8 * (m & 1);
                v8h z = {0, 0, 0, 0, 0, 0, 0, 0};
                q[t][m] = on ? *reinterpret_cast<const v8h_a2*>(p + 2 * e) : z;
            }
        }
    }

    float m_ref[NT], p_ref[NT], l_sum[NT];
    v4f O[NT][NB];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m_ref[t] = p_ref[t] = KV_NONE;
        l_sum[t] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) O[t][b] = v4f{0, 0, 0, 0};
    }
    const int* table = c.table + (int64_t)s * c.max_blocks;
    const float sc = a.scale * KV_LOG2E;

    for (int t0 = tb + w * KV_STEP; t0 < te; t0 += KV_SPAN) {
        // the step's two halves of 16 tokens lie in one block each
        const uint8_t *kp[2], *vp[2];
        float ks[2], lv[2];
        bool there[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int tt = t0 + 16 * u, blk = min(tt >> c.bt_log2, c.max_blocks - 1);
            const int id = table[blk];
            there[u] = id >= 0 && id < c.n_blocks;
            const int64_t at = (int64_t)(there[u] ? id : 0) * c.heads + hk;
            const int64_t off = (at * c.bt + (tt & (c.bt - 1))) * D;
            kp[u] = c.k + off;
            vp[u] = c.v + off;
            ks[u] = there[u] ? c.k_scale[at] * sc : 0.0f;
            lv[u] = there[u] ? scale_log2(c.v_scale[at]) : 0.0f;
        }
        u32x4 kv[2][KC];
        u32x2 kt[2];
        uint32_t vv[2][4][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int x = 0; x < KC; ++x) kv[u][x] = *reinterpret_cast<const u32x4*>(kp[u] + col * D + 64 * x + 16 * g);
            if (TAIL) kt[u] = *reinterpret_cast<const u32x2*>(kp[u] + col * D + 64 + 8 * g);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* row = vp[u] + (4 * g + i) * D;
                if constexpr (D == 128) {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(row + 8 * col);
                    vv[u][i][0] = x[0];
                    vv[u][i][1] = x[1];
                } else {
                    vv[u][i][0] = *reinterpret_cast<const uint32_t*>(row + 4 * col);
                    if (TAIL) vv[u][i][1] = *reinterpret_cast<const uint16_t*>(row + 64 + 2 * col);
                }
            }

        // scores
        v4f S[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) S[t][0] = S[t][1] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                uint32_t f[4];
                const bool tail = TAIL && m == KM - 1;
                key_halves(tail ? kt[u][0] : kv[u][m >> 1][2 * (m & 1)], f);
                key_halves(tail ? kt[u][1] : kv[u][m >> 1][2 * (m & 1) + 1], f + 2);
                const v8h k8 = __builtin_bit_cast(v8h, u32x4{f[0], f[1], f[2], f[3]});
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    S[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, q[t][m], S[t][u], 0, 0, 0);
                    if (QS) S[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[t][m], S[t][u], 0, 0, 0);
                }
            }

        // probabilities
        uint32_t P[NT][4], PL[PS ? NT : 1][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float x[2][4], top[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float f = QS ? ks[u] * qscale[t] : ks[u];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tt = t0 + 16 * u + 4 * g + i;
                    x[u][i] = there[u] && tt >= see_lo[t] && tt < see_hi[t] && tt < te ? S[t][u][i] * f : -__builtin_inff();
                }
                top[u] = fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3]));
            }
            const float topp = fmaxf(top[0] + lv[0], top[1] + lv[1]), tops = fmaxf(top[0], top[1]);
            if (__builtin_amdgcn_ballot_w64(topp > p_ref[t] + KV_ROOM || tops > m_ref[t] + 60.0f)) {
                const float pn = fmaxf(p_ref[t], col_max(topp) - KV_LIFT), mn = fmaxf(m_ref[t], col_max(tops));
                const float ap = __builtin_amdgcn_exp2f(p_ref[t] - pn), am = __builtin_amdgcn_exp2f(m_ref[t] - mn);
                p_ref[t] = pn;
                m_ref[t] = mn;
                l_sum[t] *= am;
#pragma unroll
                for (int b = 0; b < NB; ++b) O[t][b] *= ap;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float p[4];
                const float shift = lv[u] - p_ref[t], back = p_ref[t] - m_ref[t] - lv[u];
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = x[u][i] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x[u][i] + shift);
                h2v h0 = __builtin_convertvector((v2f{p[0], p[1]}), h2v), h1 = __builtin_convertvector((v2f{p[2], p[3]}), h2v);
                P[t][2 * u] = __builtin_bit_cast(uint32_t, h0);
                P[t][2 * u + 1] = __builtin_bit_cast(uint32_t, h1);
                float sum;
                if constexpr (PS) {
                    sum = (p[0] + p[1]) + (p[2] + p[3]);
                    const h2v e0 = __builtin_convertvector((v2f{p[0] - (float)h0[0], p[1] - (float)h0[1]}), h2v);
                    const h2v e1 = __builtin_convertvector((v2f{p[2] - (float)h1[0], p[3] - (float)h1[1]}), h2v);
                    PL[t][2 * u] = __builtin_bit_cast(uint32_t, e0);
                    PL[t][2 * u + 1] = __builtin_bit_cast(uint32_t, e1);
                } else {  // the sum of what the product takes
                    const h2v ones = {(_Float16)1.0f, (_Float16)1.0f};
                    sum = __builtin_amdgcn_fdot2(h1, ones, __builtin_amdgcn_fdot2(h0, ones, 0.0f, false), false);
                }
                if (__builtin_amdgcn_ballot_w64(back > 90.0f)) {
                    float d = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) d += __builtin_amdgcn_exp2f(x[u][i] - m_ref[t]);
                    l_sum[t] += back > 90.0f ? d : sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_exp2f(back);
                } else {
                    l_sum[t] += sum == 0.0f ? 0.0f : sum * __builtin_amdgcn_exp2f(back);  // (0: no NaN of a block that the row does not see)
                }
            }
        }

        // output
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int wd = D == 128 ? b >> 2 : (b >= 4), by = D == 128 ? b & 3 : b & 3;
            const u32x4 f = {value_halves(vv[0][0][wd], vv[0][1][wd], by), value_halves(vv[0][2][wd], vv[0][3][wd], by),
                             value_halves(vv[1][0][wd], vv[1][1][wd], by), value_halves(vv[1][2][wd], vv[1][3][wd], by)};
            const v8h v8 = __builtin_bit_cast(v8h, f);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32x4 p = {P[t][0], P[t][1], P[t][2], P[t][3]};
                O[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, __builtin_bit_cast(v8h, p), O[t][b], 0, 0, 0);
                if constexpr (PS) {
                    const u32x4 e = {PL[t][0], PL[t][1], PL[t][2], PL[t][3]};
                    O[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, __builtin_bit_cast(v8h, e), O[t][b], 0, 0, 0);
                }
            }
        }
    }

    // join the wavefronts: 2 and 3 into 0 and 1, then 1 into 0
    __shared__ __attribute__((aligned(16))) v4f so[2][NT][NB][64];
    __shared__ float sm[2][NT][3][16];
#pragma unroll
    for (int t = 0; t < NT; ++t) l_sum[t] = col_sum(l_sum[t]);
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
        if (w >= half && w < 2 * half) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int b = 0; b < NB; ++b) so[w - half][t][b][lane] = O[t][b];
                if (g == 0) {
                    sm[w - half][t][0][col] = m_ref[t];
                    sm[w - half][t][1][col] = p_ref[t];
                    sm[w - half][t][2][col] = l_sum[t];
                }
            }
        }
        __syncthreads();
        if (w < half) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float m2 = sm[w][t][0][col], p2 = sm[w][t][1][col], l2 = sm[w][t][2][col];
                const float mn = fmaxf(m_ref[t], m2), pn = fmaxf(p_ref[t], p2);
                l_sum[t] = l_sum[t] * __builtin_amdgcn_exp2f(m_ref[t] - mn) + l2 * __builtin_amdgcn_exp2f(m2 - mn);
                const float a1 = __builtin_amdgcn_exp2f(p_ref[t] - pn), a2 = __builtin_amdgcn_exp2f(p2 - pn);
#pragma unroll
                for (int b = 0; b < NB; ++b) O[t][b] = O[t][b] * a1 + so[w][t][b][lane] * a2;
                m_ref[t] = mn;
                p_ref[t] = pn;
            }
        }
        __syncthreads();
    }
    if (w != 0) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + col, iq = r / a.group, h = hk * a.group + (r - iq * a.group);
        if (r >= rows) continue;
        float f = 1.0f;
        char* out;
        if (splits > 1) {
            const int64_t pr = (((int64_t)sp * c.n_seq + s) * a.n_q + iq) * a.heads + h;
            out = reinterpret_cast<char*>(a.part + pr * D);
            if (g == 0) {
                float* ml = a.part + (int64_t)splits * c.n_seq * a.n_q * a.heads * D + pr * 4;
                *reinterpret_cast<v4f*>(ml) = v4f{m_ref[t], p_ref[t], l_sum[t], 0.0f};
            }
        } else {
            f = l_sum[t] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(p_ref[t] - m_ref[t] + 9.0f) / l_sum[t];
            out = a.dst + (int64_t)h * a.d_nb[0] + (int64_t)iq * a.d_nb[1] + (int64_t)s * a.d_nb[2];
        }
        const bool h16 = splits == 1 && a.d16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ar = 4 * g + i;
            v4f y[2];
#pragma unroll
            for (int b = 0; b < 8; ++b) y[b >> 2][b & 3] = b < NB ? O[t][b < NB ? b : 0][i] * f : 0.0f;
            const int e = (D == 128 ? 8 : 4) * ar;
            if (h16) {
                *reinterpret_cast<v4h_a2*>(out + 2 * e) = __builtin_convertvector(y[0], v4h);
                if (D == 128) *reinterpret_cast<v4h_a2*>(out + 2 * e + 8) = __builtin_convertvector(y[1], v4h);
                if (TAIL) *reinterpret_cast<h2v_a2*>(out + 2 * (64 + 2 * ar)) = __builtin_convertvector((v2f{y[1][0], y[1][1]}), h2v);
            } else {
                *reinterpret_cast<v4f_a4*>(out + 4 * e) = y[0];
                if (D == 128) *reinterpret_cast<v4f_a4*>(out + 4 * e + 16) = y[1];
                if (TAIL) *reinterpret_cast<v2f_a4*>(out + 4 * (64 + 2 * ar)) = v2f{y[1][0], y[1][1]};
            }
        }
    }
}

// The ranges' joins: thread per four elements of a row
template <int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(const KvAttnArgs a, const int splits) {
    constexpr int C4 = D / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.c.n_seq * a.n_q * a.heads;
    const int64_t pr = i / C4;
    if (pr >= rows) return;
    const int e = (int)(i - pr * C4) * 4;
    const int h = (int)(pr % a.heads), iq = (int)(pr / a.heads % a.n_q), s = (int)(pr / a.heads / a.n_q);
    const KvRange kr = kv_range(a, s);
    if (iq >= kr.nq) return;
    const int chunk = kv_chunk(kr, splits), n = max((kr.hi - kr.lo + chunk - 1) / chunk, 1);
    const float* ml = a.part + (int64_t)splits * rows * D + pr * 4;
    const float* po = a.part + pr * D + e;
    float m = KV_NONE, p = KV_NONE, l = 0.0f;
    v4f o = {0, 0, 0, 0};
    for (int x = 0; x < n; ++x) {
        m = fmaxf(m, ml[x * rows * 4]);
        p = fmaxf(p, ml[x * rows * 4 + 1]);
    }
    for (int x = 0; x < n; ++x) {
        l += ml[x * rows * 4 + 2] * __builtin_amdgcn_exp2f(ml[x * rows * 4] - m);
        o = o + *reinterpret_cast<const v4f*>(po + x * rows * D) * __builtin_amdgcn_exp2f(ml[x * rows * 4 + 1] - p);
    }
    const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(p - m + 9.0f) / l;
    o = o * f;
    char* out = a.dst + (int64_t)h * a.d_nb[0] + (int64_t)iq * a.d_nb[1] + (int64_t)s * a.d_nb[2];
    if (a.d16) *reinterpret_cast<v4h_a2*>(out + 2 * e) = __builtin_convertvector(o, v4h);
    else *reinterpret_cast<v4f_a4*>(out + 4 * e) = o;
}

// Row tiles and ranges of the kernel above for n_q queries: enough workgroups to fill the CUs several times
// over, of at least one step each.
KvAttnPlan kv_attn_plan(int n_q, int heads, int heads_kv, int n_seq, int64_t max_tokens, int D, int cus) {
    KvAttnPlan p;
    const int64_t rows = (int64_t)n_q * (heads / heads_kv);
    p.nt = rows > 16 ? 2 : 1;
    p.tiles = (int)((rows + 16 * p.nt - 1) / (16 * p.nt));
    const int64_t wgs = std::max<int64_t>((int64_t)p.tiles * heads_kv * n_seq, 1);
    const int64_t most = std::max<int64_t>((max_tokens + KV_SPAN - 1) / KV_SPAN, 1);
    p.splits = (int)std::max<int64_t>(std::min<int64_t>({(16LL * std::max(cus, 1) + wgs - 1) / wgs, most, 128}), 1);
    p.bytes = p.splits > 1 ? (size_t)p.splits * n_seq * n_q * heads * (D + 4) * 4 : 0;
    return p;
}

template <int D, int NT, bool QS, bool PS>
static void rows_launch(const KvAttnArgs& a, const KvAttnPlan& p, hipStream_t st) {
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    kv_attn_rows_kernel<D, NT, QS, PS><<<(unsigned)((items + 7) / 8 * 8 * p.tiles), 256, 0, st>>>(a, p.splits, p.tiles);
}

template <int D>
static hipError_t kv_attn_d(const KvAttnArgs& a, const KvAttnPlan& p, hipStream_t st) {
    auto go = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        if (a.q16 && a.d16) rows_launch<D, NT, false, false>(a, p, st);
        else if (a.q16) rows_launch<D, NT, false, true>(a, p, st);
        else if (a.d16) rows_launch<D, NT, true, false>(a, p, st);
        else rows_launch<D, NT, true, true>(a, p, st);
    };
    if (p.nt == 1) go(std::integral_constant<int, 1>());
    else go(std::integral_constant<int, 2>());
    if (p.splits > 1) {
        const int64_t n = (int64_t)a.c.n_seq * a.n_q * a.heads * (D / 4);
        kv_attn_join_kernel<D><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a, p.splits);
    }
    return hipGetLastError();
}

hipError_t launch_kv_attn(const KvAttnArgs& a, const KvAttnPlan& p, int D, hipStream_t st) {
    const int64_t rows = (int64_t)a.n_q * a.heads * a.c.n_seq;
    if (rows <= 0) return hipSuccess;
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    if ((items + 7) / 8 * 8 * p.tiles > INT32_MAX || rows * (D / 4) > (int64_t)INT32_MAX * 256 || (p.splits > 1 && !a.part))
        return hipErrorInvalidValue;
    switch (D) {
        case 64: return kv_attn_d<64>(a, p, st);
        case 96: return kv_attn_d<96>(a, p, st);
        case 128: return kv_attn_d<128>(a, p, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mi355
