// Attention over the 8-bit cache of kvcache.hip:
//
//   dst[s][i][h] = sum_t softmax_t(scale q_i . k_t) v_t
//
// over the tokens t that query i sees (n_kv, causal, window), with fp32 online softmax.
#include <algorithm>
#include <type_traits>

#include "attn.cuh"
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
constexpr float KV_NO_P = -2e30f;    // the probabilities' own: below it, so that rows that see nothing are not taken for thin ones
constexpr float KV_LIFT = 12.0f;     // probabilities are raised by 2^12 to keep small ones in fp16's normal range
constexpr float KV_ROOM = 15.0f;     // and their reference moves when one would pass 2^15
constexpr float KV_LIFT_SUM = 8.0f;  // the same where a lane's sum of 32 of them, and not each, is held below 2^15
// A probability that a product takes as a half is 2^-b of its softmax weight (the largest weight one), b the negative lift
// where the blocks' value scales are alike, and more by the binades that a block's scale lies below the others'.  The sum
// of the rounded halves has the products' own roundings, which then cancel; but a half's step of 2^-24 is 2^(b - 24) of a
// weight, so that from these b on the unrounded probabilities are summed.  Steps of 2^-32 and 2^-29 of the largest weight are
// left, which a million tokens of such weights may lose once each.  Every second block's values 2^-10 of the others': 2 x
// 4096 queries over 5120 tokens 504 us, 459 where all are alike (those groups' exponentials a second time); single tokens
// of 32 sequences over 16384 186 us either way.
constexpr float KV_THIN = -8.0f, KV_THIN_SUM = -5.0f;
constexpr int KV_STEP = 32;          // tokens of one step of a wavefront
constexpr int KV_SPAN = 4 * KV_STEP; // tokens of one step of a workgroup
constexpr int KV_RANGES = 64;        // ranges of a row that one workgroup joins, at most
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

// log2 of a block's scale, -inf for 0; the instruction takes no subnormals
__device__ __forceinline__ float scale_log2(float v) {
    const bool tiny = v < 7.8886091e-31f;  // 2^-100
    return __builtin_amdgcn_logf(tiny ? v * 1.1529215e18f : v) - (tiny ? 60.0f : 0.0f);
}

// What the products need of 16 tokens, which lie in one block: lane i of a wavefront keeps it for the i-th
// group from a token on, and readlane gives it to the scalar unit when its step comes.  (A load for each
// step instead is a chain of two latencies in every step.)
struct KvGroups {
    int id;           // block, or -1
    float f, lv, rv;  // key scale times the score's scale; log2 of the value scale; 1 / value scale
};
__device__ __forceinline__ int group_block(const KvAttnArgs& a, const int* table, int t) {
    const int id = table[min(max(t, 0) >> a.c.bt_log2, a.c.max_blocks - 1)];
    return id >= 0 && id < a.c.n_blocks ? id : -1;
}
__device__ __forceinline__ void group_scales(const KvAttnArgs& a, int hk, float sc, KvGroups& x) {
    const int64_t at = (int64_t)max(x.id, 0) * a.c.heads + hk;
    const float ks = a.c.k_scale[at], vs = a.c.v_scale[at];
    const bool finite = fabsf(ks) < __builtin_inff() && fabsf(vs) < __builtin_inff();
    x.f = x.id < 0 ? 0.0f : finite ? ks * sc : __builtin_nanf("");  // (a score that is seen is then NaN)
    x.lv = x.id >= 0 ? scale_log2(vs) : 0.0f;
    x.rv = 1.0f / vs;
}
__device__ __forceinline__ float read_lane(float v, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i)); }

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

// 2^-e and 2^e of a magnitude's exponent e, both normal
struct Pow2 {
    float down, up;
};
__device__ __forceinline__ Pow2 pow2_of(float top) {
    const int e = min(max((int)((__float_as_uint(top) >> 23) & 255) - 127, -126), 126);
    return {__uint_as_float((uint32_t)(127 - e) << 23), __uint_as_float((uint32_t)(127 + e) << 23)};
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

// A store past the caches of the workgroup's XCD, for a workgroup on another one, and a load of such
__device__ __forceinline__ v2f get_through(const float* p) {
    return __builtin_bit_cast(v2f, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ void put_through(float* p, v2f v) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Four elements from e on of row pr (sequence, query, head in that order), joined from the row's n ranges in the ranges'
// order and written.  ONE: other workgroups of this launch wrote the partial sums.
template <int D, bool ONE>
__device__ __forceinline__ void join_ranges(const KvAttnArgs& a, int splits, int n, int64_t pr, int e) {
    const int64_t rows = (int64_t)a.c.n_seq * a.n_q * a.heads;
    const float* ml = a.part + (int64_t)splits * rows * D + pr * 4;
    const float* po = a.part + pr * D + e;
    auto get = [](const float* q) {
        if constexpr (!ONE) return *reinterpret_cast<const v4f*>(q);
        const v2f lo = get_through(q), hi = get_through(q + 2);
        return v4f{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int B = 8;  // ranges whose loads are on their way together
    float m = KV_NONE, p = KV_NONE, l = 0.0f;
    v4f o = {0, 0, 0, 0};
    for (int x0 = 0; x0 < n; x0 += B) {
        v4f z[B], y[B];
#pragma unroll
        for (int x = 0; x < B; ++x) {
            z[x] = v4f{KV_NONE, KV_NONE, 0, 0};
            y[x] = v4f{0, 0, 0, 0};
            if (x0 + x < n) {
                z[x] = get(ml + (x0 + x) * rows * 4);
                y[x] = get(po + (x0 + x) * rows * D);
            }
        }
        float mn = m, pn = p;
#pragma unroll
        for (int x = 0; x < B; ++x) mn = fmaxf(mn, z[x][0]), pn = fmaxf(pn, z[x][1]);
        l *= __builtin_amdgcn_exp2f(m - mn);
        o = o * __builtin_amdgcn_exp2f(p - pn);
        m = mn;
        p = pn;
#pragma unroll
        for (int x = 0; x < B; ++x) {
            l += z[x][2] * __builtin_amdgcn_exp2f(z[x][0] - m);
            o = o + y[x] * __builtin_amdgcn_exp2f(z[x][1] - p);
        }
    }
    o = o * (l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(p - m) / l);
    const int64_t h = pr % a.heads, iq = pr / a.heads % a.n_q, s = pr / a.heads / a.n_q;
    char* out = a.dst + h * a.d_nb[0] + iq * a.d_nb[1] + s * a.d_nb[2];
    if (a.d16) *reinterpret_cast<v4h_a2*>(out + 2 * e) = __builtin_convertvector(o, v4h);
    else *reinterpret_cast<v4f_a4*>(out + 4 * e) = o;
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
// that factor passes 2^90 (scales far below the others', and zero) the sum is taken of 2^(s - m) itself, and for an
// F16 output from 2^-8 on of P before its rounding (KV_THIN).
// QS: an F32 q enters as two halves of 11 bits, scaled by a power of two that brings the row's largest
// magnitude to about one.  PS: for an F32 output the probabilities enter as two halves too.
//
// With many conversations the cache's bytes bound it: 32 of 16384 tokens, 32 heads of 128 over 8 key heads, 815 MB in
// 153 us (5.3 TB/s).  With few tokens the chain of latencies does: table, block, scales, then the last workgroup's
// join (777 tokens, 16 heads of 64 over 2: 7.2 us).
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
    if (sp > 0 && tb >= kr.hi) return;  // no such range (the first always answers)
    const int ranges = max((kr.hi - kr.lo + chunk - 1) / chunk, 1);

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
            const Pow2 z = pow2_of(col_max(top));
            const float down = z.down;
            qscale[t] = z.up;
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
        m_ref[t] = KV_NONE;
        p_ref[t] = KV_NO_P;
        l_sum[t] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) O[t][b] = v4f{0, 0, 0, 0};
    }
    const int* table = c.table + (int64_t)s * c.max_blocks;
    const float sc = a.scale * KV_LOG2E;

    // A step's two halves of 16 tokens: where their bytes are, and their scales.  The keys of a step are asked for
    // when the step before has multiplied its own, its values when it begins, so that something is always on its way.
    struct Step {
        const uint8_t* vp[2];
        float ks[2], lv[2];
        bool there[2];
    };
    KvGroups gr = {-1, 0.0f, 0.0f, 0.0f};
    int at = 32;
    u32x4 kv[2][KC];
    u32x2 kt[2];
    auto ask = [&](int t0) {
        Step x;
        if (at == 32) {  // lane 2 i + u: half u of this wavefront's i-th step from here
            gr.id = group_block(a, table, t0 + (lane >> 1) * KV_SPAN + 16 * (lane & 1));
            group_scales(a, hk, sc, gr);
            at = 0;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int id = __builtin_amdgcn_readlane(gr.id, 2 * at + u);
            const int64_t off = (((int64_t)max(id, 0) * c.heads + hk) * c.bt + ((t0 + 16 * u) & (c.bt - 1))) * D;
            const uint8_t* kp = c.k + off;
            x.vp[u] = c.v + off;
            x.there[u] = id >= 0;
            x.ks[u] = read_lane(gr.f, 2 * at + u);
            x.lv[u] = read_lane(gr.lv, 2 * at + u);
#pragma unroll
            for (int y = 0; y < KC; ++y) kv[u][y] = *reinterpret_cast<const u32x4*>(kp + col * D + 64 * y + 16 * g);
            if (TAIL) kt[u] = *reinterpret_cast<const u32x2*>(kp + col * D + 64 + 8 * g);
        }
        ++at;
        return x;
    };
    Step next{};
    if (tb + w * KV_STEP < te) next = ask(tb + w * KV_STEP);
    for (int t0 = tb + w * KV_STEP; t0 < te; t0 += KV_SPAN) {
        const Step x0 = next;
        const float (&ks)[2] = x0.ks, (&lv)[2] = x0.lv;
        const bool (&there)[2] = x0.there;
        uint32_t vv[2][4][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* row = x0.vp[u] + (4 * g + i) * D;
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

        if (t0 + KV_SPAN < te) next = ask(t0 + KV_SPAN);

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
                } else {  // the sum of what the product takes (KV_THIN)
                    const h2v ones = {(_Float16)1.0f, (_Float16)1.0f};
                    sum = __builtin_amdgcn_fdot2(h1, ones, __builtin_amdgcn_fdot2(h0, ones, 0.0f, false), false);
                    if (__builtin_amdgcn_ballot_w64(back > KV_THIN)) sum = back > KV_THIN ? (p[0] + p[1]) + (p[2] + p[3]) : sum;
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
    if (ranges == 1) {
        if (w != 0) return;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = row0 + 16 * t + col, iq = r / a.group, h = hk * a.group + (r - iq * a.group);
            if (r >= rows) continue;
            // (2^9: the halves were the bytes' values over 512)
            const float f = l_sum[t] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(p_ref[t] - m_ref[t] + 9.0f) / l_sum[t];
            char* out = a.dst + (int64_t)h * a.d_nb[0] + (int64_t)iq * a.d_nb[1] + (int64_t)s * a.d_nb[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ar = 4 * g + i;
                v4f y[2];
#pragma unroll
                for (int b = 0; b < 8; ++b) y[b >> 2][b & 3] = b < NB ? O[t][b < NB ? b : 0][i] * f : 0.0f;
                const int e = (D == 128 ? 8 : 4) * ar;
                if (a.d16) {
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
        return;
    }
    // One of several ranges: its sums go to memory past the caches, rows whole.
    auto partial_row = [&](int r) {  // row r of the tile: its number among all
        const int iq = (row0 + r) / a.group;
        return row0 + r < rows ? ((int64_t)s * a.n_q + iq) * a.heads + hk * a.group + (row0 + r - iq * a.group) : (int64_t)-1;
    };
    if (w == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int b = 0; b < NB; ++b) so[0][t][b][lane] = O[t][b];
            const int64_t pr = partial_row(16 * t + col);
            if (g == 0 && pr >= 0) {
                const int64_t all = (int64_t)c.n_seq * a.n_q * a.heads;
                float* ml = a.part + (int64_t)splits * all * D + (sp * all + pr) * 4;
                put_through(ml, v2f{m_ref[t], p_ref[t] + 9.0f});
                put_through(ml + 2, v2f{l_sum[t], 0.0f});
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT * (D / 2); i += 256) {
        const int r = i / (D / 2), e = 2 * (i % (D / 2));
        const int64_t pr = partial_row(r);
        if (pr < 0) break;
        const int ar = D == 128 ? e >> 3 : e < 64 ? e >> 2 : (e - 64) >> 1, b = D == 128 ? e & 7 : e < 64 ? e & 3 : 4;
        const v4f* o = &so[0][r >> 4][b][(r & 15) + 16 * (ar >> 2)];
        put_through(a.part + ((int64_t)sp * c.n_seq * a.n_q * a.heads + pr) * D + e, v2f{o[0][ar & 3], o[64][ar & 3]});
    }
    // The workgroup that comes last joins the ranges.  What the others wrote is in memory before they count
    // themselves, and the counter goes back to zero for the next launch.
    __shared__ int join;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t* n = a.arrived + ((int64_t)s * c.heads + hk) * tiles + tile;
        join = __hip_atomic_fetch_add(n, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)ranges - 1;
        if (join) __hip_atomic_store(n, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!join) return;
    asm volatile("" ::: "memory");
    if constexpr (NT == 1) {  // (few elements: one round of loads more would cost more than the weights' reuse saves)
        for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
            const int64_t pr = partial_row(i / (D / 4));
            if (pr >= 0) join_ranges<D, true>(a, splits, ranges, pr, 4 * (i % (D / 4)));
        }
        return;
    }
    // First each row's weights of its ranges, lanes L to a row, then the rows' elements.
    constexpr int L = 256 / (16 * NT), MAXN = KV_RANGES;
    __shared__ float weight[16 * NT][MAXN];
    const int64_t all = (int64_t)c.n_seq * a.n_q * a.heads;
    {
        const int r = threadIdx.x / L, x0 = threadIdx.x % L;
        const int64_t pr = partial_row(r);
        const float* ml = a.part + (int64_t)splits * all * D + max(pr, (int64_t)0) * 4;
        v2f mp[MAXN / L];
        float l[MAXN / L], m = KV_NONE, p = KV_NONE, sum = 0.0f;
#pragma unroll
        for (int x = 0; x < MAXN / L; ++x) {
            mp[x] = v2f{KV_NONE, KV_NONE};
            l[x] = 0.0f;
            if (pr >= 0 && x0 + L * x < ranges) {
                mp[x] = get_through(ml + (x0 + L * x) * all * 4);
                l[x] = get_through(ml + (x0 + L * x) * all * 4 + 2)[0];
            }
        }
#pragma unroll
        for (int x = 0; x < MAXN / L; ++x) m = fmaxf(m, mp[x][0]), p = fmaxf(p, mp[x][1]);
        m = group_max<L>(m);
        p = group_max<L>(p);
        // (the lanes' sums meet in a fixed order)
#pragma unroll
        for (int x = 0; x < MAXN / L; ++x) sum += l[x] * __builtin_amdgcn_exp2f(mp[x][0] - m);
        sum = group_sum<L>(sum);
        const float f = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(p - m) / sum;
#pragma unroll
        for (int x = 0; x < MAXN / L; ++x)
            if (x0 + L * x < ranges) weight[r][x0 + L * x] = __builtin_amdgcn_exp2f(mp[x][1] - p) * f;
    }
    __syncthreads();
    constexpr int K = NT * D / 64, B = 4;  // pieces of a thread, ranges whose loads are on their way together
    int64_t place[K];
    int row[K];
    v4f o[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = threadIdx.x + 256 * k;
        row[k] = i / (D / 4);
        const int64_t pr = i < 16 * NT * (D / 4) ? partial_row(row[k]) : -1;
        place[k] = pr < 0 ? -1 : pr * D + 4 * (i % (D / 4));
        o[k] = v4f{0, 0, 0, 0};
    }
    for (int x0 = 0; x0 < ranges; x0 += B) {
        v2f y[K][B][2];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int x = 0; x < B; ++x) {
                y[k][x][0] = y[k][x][1] = v2f{0, 0};
                if (place[k] >= 0 && x0 + x < ranges) {
                    y[k][x][0] = get_through(a.part + (x0 + x) * all * D + place[k]);
                    y[k][x][1] = get_through(a.part + (x0 + x) * all * D + place[k] + 2);
                }
            }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int x = 0; x < B; ++x) {
                const float f = place[k] >= 0 && x0 + x < ranges ? weight[row[k]][x0 + x] : 0.0f;
                o[k] = o[k] + v4f{y[k][x][0][0], y[k][x][0][1], y[k][x][1][0], y[k][x][1][1]} * f;
            }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (place[k] < 0) continue;
        const int r = row0 + row[k], iq = r / a.group, h = hk * a.group + (r - iq * a.group), e = 4 * ((threadIdx.x + 256 * k) % (D / 4));
        char* out = a.dst + (int64_t)h * a.d_nb[0] + (int64_t)iq * a.d_nb[1] + (int64_t)s * a.d_nb[2];
        if (a.d16) *reinterpret_cast<v4h_a2*>(out + 2 * e) = __builtin_convertvector(o[k], v4h);
        else *reinterpret_cast<v4f_a4*>(out + 4 * e) = o[k];
    }
}

// Many query rows: a workgroup takes 128 rows (as above: queries times the heads of a key head's group) in four
// wavefronts of 32, and streams the tokens through LDS in tiles of 64, bytes becoming halves once for
// all four on the way: thread t loads 16 bytes (D = 96: 8) of a row ahead of time and writes 32 after
// the previous tile's products.  Scores and output as fattn.hip's (v_mfma_f32_32x32x16_f16, S^T = K Q^T, the
// probabilities' registers as the operand of O^T += V^T P^T, V^T by transposing reads); the tile's scores
// are computed one tile ahead of its softmax, so that the matrix pipe works beside the VALU.  A lane's
// eight scores (kh, hh) belong to 16 tokens of one block: scales and validity are uniform over them.
//
// Bounded by the VALU's work of a score (scale, exponential, sum, the bytes' conversion) and the matrix products, which
// two wavefronts of a SIMD overlap in part, at a clock that they pull down to 2.0 GHz: at 4096 causal F16 queries twice, 32 heads
// of 128 over 8 key heads, 355 us or 890 TFLOP/s (320 to 430 from one run to another), the matrix pipe is busy 40 % of the
// time, the VALU 50 %, the LDS 40 % (10 % bank conflicts).  F32 queries and probabilities as two halves cost twice the
// products: 5184 queries over 15552 tokens, 8 heads of 64, 346 us for 165 GFLOP as the formula counts them (matrix pipe 45 %,
// VALU 63 %).  Eight items at a time 388 us; beside it sixteen or thirty-two 466, one 482, the shortest row tiles first 497.
template <int D, bool QS, bool PS>
__global__ __launch_bounds__(256, 2) void kv_attn_tiles_kernel(const KvAttnArgs a, const int splits, const int tiles) {
    constexpr int NC = D / 16, NDB = D / 32;        // score products, output blocks
    constexpr bool AHEAD = !((QS && D > 64) || (PS && D > 96));  // scores a tile ahead; else the second halves have their registers
    constexpr int UB = D == 96 ? 8 : 16;            // bytes of a staging unit
    constexpr int UR = D / UB, NU = 16 * UR / 64;   // units of a row, units of a thread
    __shared__ __attribute__((aligned(16))) _Float16 sK[2][64 * D];
    __shared__ __attribute__((aligned(16))) _Float16 sV[2][64 * D];
    const KvView& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Eight items (one to an XCD, whose bytes stay in its L2) at a time, and of them the last row tiles
    // first: causal ones are the longest.
    const int items = splits * c.heads * c.n_seq, first = blockIdx.x / (8 * tiles) * 8, left = blockIdx.x - first * tiles;
    const int many = min(8, items - first), item = first + left % many, tile = tiles - 1 - left / many;
    const int sp = item % splits, hk = item / splits % c.heads, s = item / splits / c.heads;
    const KvRange kr = kv_range(a, s);
    const int rows = kr.nq * a.group, row0 = tile * 128;
    if (row0 >= rows) return;
    const int chunk = kv_chunk(kr, splits);
    if (sp > 0 && kr.lo + sp * chunk >= kr.hi) return;
    const int iq_first = row0 / a.group, iq_last = (min(row0 + 128, rows) - 1) / a.group;
    const int lo_tile = a.window > 0 ? max(kr.pos0 + iq_first - a.window + 1, 0) & ~63 : 0;
    const int tb = max(kr.lo + sp * chunk, lo_tile);  // (a multiple of 32: blocks are met at 16-token steps)
    const int te = min(min(kr.lo + sp * chunk + chunk, kr.hi), a.causal ? kr.pos0 + iq_last + 1 : kr.hi);

    // this lane's query row
    const int r = row0 + 32 * w + lr, iq = r / a.group, h = hk * a.group + (r - iq * a.group);
    const bool on = r < rows;
    const int pos = kr.pos0 + iq;
    const int see_hi = on ? (a.causal ? min(pos + 1, te) : te) : 0, see_lo = a.window > 0 ? pos - a.window + 1 : 0;
    // tokens that every row of the wavefront sees (rows past the last one see what they like)
    const int iq0 = __builtin_amdgcn_readfirstlane(iq), iq31 = min(__builtin_amdgcn_readlane(iq, 31), iq_last);
    const int all_hi = a.causal ? min(kr.pos0 + iq0 + 1, te) : te, all_lo = a.window > 0 ? kr.pos0 + iq31 - a.window + 1 : 0;
    v8h q[NC], ql[QS ? NC : 1];
    float qscale = a.scale < 0.0f ? -1.0f : 1.0f;
    {
        const char* p = a.q + (int64_t)iq * a.q_nb[0] + (int64_t)h * a.q_nb[1] + (int64_t)s * a.q_nb[2];
        if constexpr (QS) {
            float top = 0.0f;
#pragma unroll
            for (int m = 0; m < NC; ++m)
                if (on) {
                    const v4f x0 = *reinterpret_cast<const v4f_a4*>(p + 4 * (16 * m + 8 * g)), x1 = *reinterpret_cast<const v4f_a4*>(p + 4 * (16 * m + 8 * g) + 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(fabsf(x0[j]), fabsf(x1[j])));
                }
            const Pow2 z = pow2_of(xmax32(top));
            const float down = z.down * qscale;
            qscale = z.up;
#pragma unroll
            for (int m = 0; m < NC; ++m) {
                v4f x0 = {0, 0, 0, 0}, x1 = {0, 0, 0, 0};
                if (on) {
                    x0 = *reinterpret_cast<const v4f_a4*>(p + 4 * (16 * m + 8 * g)) * down;
                    x1 = *reinterpret_cast<const v4f_a4*>(p + 4 * (16 * m + 8 * g) + 16) * down;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = j < 4 ? x0[j & 3] : x1[j & 3];
                    q[m][j] = (_Float16)y;
                    ql[m][j] = (_Float16)(y - (float)q[m][j]);
                }
            }
        } else {
#pragma unroll
            for (int m = 0; m < NC; ++m) {
                const v8h z = {0, 0, 0, 0, 0, 0, 0, 0};
                q[m] = on ? *reinterpret_cast<const v8h_a2*>(p + 2 * (16 * m + 8 * g)) : z;
                if (a.scale < 0.0f) q[m] = -q[m];
            }
            qscale = 1.0f;
        }
    }
    const float sc = fabsf(a.scale) * KV_LOG2E;

    const int* table = c.table + (int64_t)s * c.max_blocks;
    int tile0 = 0;  // the step's tile
    // groups of the sixteen tiles that the step's tile is of, and of the sixteen after
    KvGroups cur, nxt;
    auto group_of = [&](int tile) { return tb + 64 * tile + 16 * lane; };
    auto staged = [&](int tile) {  // block of this wavefront's 16 rows of a tile of this or the next sixteen
        const int i = 4 * (tile & 15) + w;
        return max((tile >> 4) == (tile0 >> 4) ? __builtin_amdgcn_readlane(cur.id, i) : __builtin_amdgcn_readlane(nxt.id, i), 0);
    };
    // staging: wavefront w takes rows 16 w .. + 15 of a tile, unit j of a lane bytes UB (u % UR) of row u / UR, u = lane + 64 j
    typedef uint32_t unit_t __attribute__((ext_vector_type(UB / 4)));
    unit_t kreg[NU], vreg[NU];
    auto load_one = [&](const uint8_t* base, unit_t* reg, int tile) {
        const uint8_t* p = base + (((int64_t)staged(tile) * c.heads + hk) * c.bt + ((tb + 64 * tile + 16 * w) & (c.bt - 1))) * D;
#pragma unroll
        for (int j = 0; j < NU; ++j) reg[j] = *reinterpret_cast<const unit_t*>(p + UB * (lane + 64 * j));
    };
    constexpr int NW = NU * UB / 8;  // eight elements each
    // LDS addresses: 16-byte chunk c of row r lies in slot c ^ swizzle(r) of it.  A row's bytes are a power of two
    // (D = 96: are added afterwards), so that a chunk further on is one exclusive or away.
    int kst[NU], vst[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) {
        const int u = lane + 64 * j, row = 16 * w + u / UR, chunk8 = (UB / 8) * (u % UR);
        kst[j] = row * 2 * D + 16 * (chunk8 ^ kswz<D>(row));
        vst[j] = row * 2 * D + 16 * (chunk8 ^ vswz<D>(row));
    }
    auto store8 = [&](_Float16* lds, const unit_t* reg, const int* st, int i) {
        const int j = i / (UB / 8), e = i % (UB / 8);
        uint32_t f[4];
        key_halves(reg[j][2 * e], f);
        key_halves(reg[j][2 * e + 1], f + 2);
        *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(lds) + (st[j] ^ (16 * e))) = u32x4{f[0], f[1], f[2], f[3]};
    };
    auto store_one = [&](_Float16* lds, const unit_t* reg, const int* st) {
#pragma unroll
        for (int i = 0; i < NW; ++i) store8(lds, reg, st, i);
    };
    const int krow = lr * 2 * D, kchunk = 16 * (g ^ kswz<D>(lr));
    auto key_frag = [&](const _Float16* lds, int pre, int m, int kh) {
        const int at = D == 96 ? krow + (pre ^ (32 * m)) : pre ^ (32 * m);
        return *reinterpret_cast<const v8h*>(reinterpret_cast<const char*>(lds) + at + kh * 64 * D);
    };
    const int kpre = D == 96 ? kchunk : krow + kchunk;
    const int vrow = 4 * g + ((lane & 15) >> 2), vpre = vrow * 2 * D + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vswz<D>(vrow)) + 8 * (lane & 1);

    v16f O[NDB];
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[i][e] = 0.0f;
    float m_ref = KV_NONE, p_ref = KV_NONE, l_sum = 0.0f, back = 1.0f;  // back = 2^(p_ref - m_ref)
    auto score = [&](const _Float16* lds, v16f* S) {
        const v16f z = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        S[0] = S[1] = z;
#pragma unroll
        for (int m = 0; m < NC; ++m)
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) {
                const v8h k8 = key_frag(lds, kpre, m, kh);
                S[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, q[m], S[kh], 0, 0, 0);
                if constexpr (QS) S[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8, ql[m], S[kh], 0, 0, 0);
            }
    };
    uint64_t hide_groups = 0, nan_groups = 0, far_groups = 0;  // (sort_groups)
    // Whether a group with 1 / value scale rv is thin against some row's references (KV_THIN_SUM), and whether one of these
    // sixteen tiles' groups is, which have at most top_rv.
    auto is_thin = [&](float rv) { return __builtin_amdgcn_ballot_w64(m_ref > KV_NONE && rv * back > __builtin_exp2f(KV_THIN_SUM)) != 0; };
    float top_rv = 0.0f;
    bool thin = false;
    // The token of score i of group j from the lane's first one of the tile.
    auto token = [](int j, int i) { return 32 * (j >> 1) + 16 * (j & 1) + 8 * (i >> 2) + (i & 3); };
    // Probabilities of a tile from its scores, at the references as they stand; returns the lane's sum of
    // them, ls is what they add to l_sum (without the groups of far value scales, whose rv is 0).
    uint32_t P[2][8], PL[2][PS ? 8 : 1];
    struct Sums {
        float s[4];
    };
    // pair n of a tile's sixteen pairs of scores
    auto pair = [&](const v16f* S, int tile, int n, Sums& sums) {
        const int j = n >> 2, gi = 4 * (tile & 15) + j;
        const float f0 = read_lane(cur.f, gi), f = QS ? fmaxf(f0 * qscale, 1e-37f) : f0, shift = read_lane(cur.lv, gi) - p_ref;
        const v16f& x = S[n >> 3];
        const int i = 2 * (n & 7);
        const v2f p = {__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], f, shift)), __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], f, shift))};
        const h2v ph = __builtin_convertvector(p, h2v), ones = {(_Float16)1.0f, (_Float16)1.0f};
        P[n >> 3][n & 7] = __builtin_bit_cast(uint32_t, ph);
        if ((n & 3) == 0) sums.s[j] = 0.0f;
        if constexpr (PS) {
            const h2v pl = __builtin_convertvector((v2f{p[0] - (float)ph[0], p[1] - (float)ph[1]}), h2v);
            PL[n >> 3][n & 7] = __builtin_bit_cast(uint32_t, pl);
            sums.s[j] += p[0] + p[1];
        } else {  // the sum of what the product takes (KV_THIN)
            sums.s[j] = __builtin_amdgcn_fdot2(ph, ones, sums.s[j], false);
        }
    };
    auto add_up = [&](const Sums& sums, int tile) {
        float ls = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) ls = __builtin_fmaf(sums.s[j], read_lane(cur.rv, 4 * (tile & 15) + j), ls);
        return ls * back;
    };
    // What is left when a tile's pairs are done: the sums, and the references where they have to move.
    auto settle = [&](const v16f* S, int tile, Sums& sums) {
        const float all = (sums.s[0] + sums.s[1]) + (sums.s[2] + sums.s[3]);
        float ls = add_up(sums, tile);
        const uint32_t far = (uint32_t)(far_groups >> (4 * (tile & 15))) & 15;
        if (__builtin_amdgcn_ballot_w64((int)!(all <= 32768.0f) | (int)(far != 0))) {
            // some probability is too large, or may be: the references move to the tile's own largest
            float topp = -__builtin_inff(), tops = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int gi = 4 * (tile & 15) + j, o = 8 * (j & 1);
                const v16f& x = S[j >> 1];
                const float f0 = read_lane(cur.f, gi), f = QS ? fmaxf(f0 * qscale, 1e-37f) : f0;
                const float y = fmaxf(fmaxf(fmaxf(x[o], x[o + 1]), fmaxf(x[o + 2], x[o + 3])), fmaxf(fmaxf(x[o + 4], x[o + 5]), fmaxf(x[o + 6], x[o + 7]))) * f;
                tops = fmaxf(tops, y);
                topp = fmaxf(topp, y + read_lane(cur.lv, gi));
            }
            const float pn = fmaxf(p_ref, xmax32(topp) - KV_LIFT_SUM), mn = fmaxf(m_ref, xmax32(tops));
            const float ap = __builtin_amdgcn_exp2f(p_ref - pn), am = __builtin_amdgcn_exp2f(m_ref - mn);
            p_ref = pn;
            m_ref = mn;
            back = __builtin_amdgcn_exp2f(pn - mn);
            if constexpr (!PS) thin = is_thin(top_rv);
            l_sum *= am;
#pragma unroll
            for (int b = 0; b < NDB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) O[b][e] *= ap;
#pragma unroll
            for (int n = 0; n < 16; ++n) pair(S, tile, n, sums);
            ls = add_up(sums, tile);
            if (far)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int gi = 4 * (tile & 15) + j, o = 8 * (j & 1);
                    const float f0 = read_lane(cur.f, gi), f = QS ? fmaxf(f0 * qscale, 1e-37f) : f0, on = (float)(far >> j & 1);
#pragma unroll
                    for (int i = 0; i < 8; ++i) ls = __builtin_fmaf(on, __builtin_amdgcn_exp2f(__builtin_fmaf(S[j >> 1][o + i], f, -m_ref)), ls);
                }
        }
        if constexpr (!PS)
            if (thin)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int gi = 4 * (tile & 15) + j, o = 8 * (j & 1);
                    const float rv = read_lane(cur.rv, gi);
                    if (!is_thin(rv)) continue;
                    const float f0 = read_lane(cur.f, gi), f = QS ? fmaxf(f0 * qscale, 1e-37f) : f0, shift = read_lane(cur.lv, gi) - p_ref;
                    float sum = -sums.s[j];
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(S[j >> 1][o + i], f, shift));
                    ls = __builtin_fmaf(sum * rv, back, ls);
                }
        l_sum += ls;
    };
    // The scores Sn of the tile in lds beside the probabilities of the tile before it, whose scores S are there:
    // a product's fragments are read while the product before multiplies, and pairs go between the products.
    auto score_softmax = [&](const _Float16* lds, v16f* Sn, const v16f* S, int tile) {
        int pre = kpre;
        asm volatile("" : "+v"(pre));  // (the addresses are made here: kept over the loop, they would push the queries out)
        const v16f z = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        v8h k8[2], k8n[2];
        auto frag = [&](int m, v8h* o) {
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) o[kh] = key_frag(lds, pre, m, kh);
        };
        // With F32 queries' two products to a fragment a wavefront here goes before the other one of its SIMD, which
        // then has its output's reads and stores beside them (5184 queries over 15552 tokens 353 us, 371 without); with
        // one product it does not pay (4096 F16 queries twice 394 us, 388 without).
        if constexpr (QS) __builtin_amdgcn_s_setprio(1);
        frag(0, k8);
        Sn[0] = Sn[1] = z;
        Sums sums;
#pragma unroll
        for (int m = 0; m < NC; ++m) {
            if (m + 1 < NC) frag(m + 1, k8n);
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) {
                Sn[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[kh], q[m], Sn[kh], 0, 0, 0);
                if constexpr (QS) Sn[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[kh], ql[m], Sn[kh], 0, 0, 0);
            }
#pragma unroll
            for (int n = 16 * m / NC; n < 16 * (m + 1) / NC; ++n) pair(S, tile, n, sums);
            k8[0] = k8n[0];
            k8[1] = k8n[1];
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (QS) __builtin_amdgcn_s_setprio(0);
        settle(S, tile, sums);
    };
    // What the sixteen tiles of cur have that is out of the ordinary.  Scores of blocks that are not there
    // are hidden, and so are those that a row does not see, before anything is made of them; where a
    // block's scales are not finite the others become NaN, and the scales ones.  Value scales of zero or beyond
    // 2^40 either way add to l_sum on a way of their own.
    auto sort_groups = [&]() {
        const bool off = cur.id < 0, bad = !off && !(cur.f < __builtin_inff() && cur.lv < __builtin_inff() && cur.lv == cur.lv);
        const bool far = !off && !bad && !(fabsf(cur.lv) <= 40.0f);
        if (off || bad) cur.f = cur.rv = 1.0f, cur.lv = 0.0f;
        if (far) cur.rv = 0.0f;
        if constexpr (!PS) {
            top_rv = group_max<64>(off ? 0.0f : cur.rv);
            thin = is_thin(top_rv);
        }
        if constexpr (!QS) cur.f = fmaxf(cur.f, 1e-37f);  // (0 times a hidden score; an F32 q's own factor comes first)
        hide_groups = __builtin_amdgcn_ballot_w64(off);
        nan_groups = __builtin_amdgcn_ballot_w64(bad);
        far_groups = __builtin_amdgcn_ballot_w64(far);
    };
    auto hide = [&](v16f* S, int tile) {
        const int t = tb + 64 * tile + 4 * g, shift = 4 * (tile & 15);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t n = hide_groups >> (shift + j) & 1 ? 0u : (uint32_t)max(see_hi - see_lo, 0);
            const float add = nan_groups >> (shift + j) & 1 ? __builtin_nanf("") : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = S[j >> 1][8 * (j & 1) + i];
                S[j >> 1][8 * (j & 1) + i] = (uint32_t)(token(j, i) + t - see_lo) < n ? x + add : -__builtin_inff();
            }
        }
    };
    // V^T fragments by transposing reads (fattn.hip)
    // The output of the tile in lds, and the staged bytes of the next ones into their buffers between the products
    auto output_store = [&](const _Float16* lds, _Float16* vnext, _Float16* knext) {
        int pre = vpre;
        asm volatile("" : "+v"(pre));
        auto frag = [&](int i) {  // product i: 16 tokens i / NDB, output block i % NDB
            const int b = i % NDB;
            const char* vt = reinterpret_cast<const char*>(lds) + (D == 96 ? pre + 64 * b : pre ^ (64 * b)) + 16 * (i / NDB) * 2 * D;
            const uint2 lo = lds_read_tr16(vt), hi = lds_read_tr16(vt + 8 * 2 * D);
            return __builtin_bit_cast(v8h, (u32x4{lo.x, lo.y, hi.x, hi.y}));
        };
        v8h v8[2] = {frag(0), frag(1)}, v8n[2];
        static_assert(4 * NDB == 4 * NW, "a unit of both to two products");
#pragma unroll
        for (int x = 0; x < 2 * NDB; ++x) {
            if (x + 1 < 2 * NDB) {
                v8n[0] = frag(2 * x + 2);
                v8n[1] = frag(2 * x + 3);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int i = 2 * x + y, kh = i / NDB / 2, hh = i / NDB & 1, b = i % NDB;
                const u32x4 p = {P[kh][4 * hh], P[kh][4 * hh + 1], P[kh][4 * hh + 2], P[kh][4 * hh + 3]};
                O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[y], __builtin_bit_cast(v8h, p), O[b], 0, 0, 0);
                if constexpr (PS) {
                    const u32x4 e = {PL[kh][4 * hh], PL[kh][4 * hh + 1], PL[kh][4 * hh + 2], PL[kh][4 * hh + 3]};
                    O[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[y], __builtin_bit_cast(v8h, e), O[b], 0, 0, 0);
                }
            }
            if (x < NW) store8(vnext, vreg, vst, x);
            else store8(knext, kreg, kst, x - NW);
            v8[0] = v8n[0];
            v8[1] = v8n[1];
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    const int nt = te > tb ? (te - tb + 63) / 64 : 0;
    if (nt > 0) {
        // Step t: the scores of tile t + 1 beside the softmax of tile t (AHEAD; else its own before it), and its
        // output; then the bytes of K(t + 2) (t + 1) and V(t + 1), loaded a step before, become halves in the buffers
        // that step t - 1 read last.  One barrier a step.
        cur.id = group_block(a, table, group_of(0));
        nxt.id = group_block(a, table, group_of(16));
        group_scales(a, hk, sc, cur);
        sort_groups();
        v16f SA[2], SB[2];
        load_one(c.k, kreg, 0);
        store_one(sK[0], kreg, kst);
        load_one(c.v, vreg, 0);
        store_one(sV[0], vreg, vst);
        load_one(c.k, kreg, 1);
        if constexpr (AHEAD) {
            store_one(sK[1], kreg, kst);
            load_one(c.k, kreg, 2);
        }
        load_one(c.v, vreg, 1);
        __syncthreads();
        if constexpr (AHEAD) score(sK[0], SA);
        auto step = [&](int t, int cb, v16f* Sc, v16f* Sn) {
            const int t0 = tb + 64 * t;
            lds_barrier();
            tile0 = t;
            if ((t & 15) == 0 && t > 0) {
                cur = nxt;
                sort_groups();
                nxt.id = group_block(a, table, group_of(t + 16));
            }
            if ((t & 15) == 8) group_scales(a, hk, sc, nxt);
            if constexpr (!AHEAD) score(sK[cb], Sc);
            if (t0 < all_lo || t0 + 64 > all_hi || (((hide_groups | nan_groups) >> (4 * (t & 15))) & 15)) hide(Sc, t);
            if constexpr (AHEAD) {
                score_softmax(sK[cb ^ 1], Sn, Sc, t);
            } else {
                Sums sums;
#pragma unroll
                for (int n = 0; n < 16; ++n) pair(Sc, t, n, sums);
                settle(Sc, t, sums);
            }
            output_store(sV[cb], sV[cb ^ 1], sK[AHEAD ? cb : cb ^ 1]);
            load_one(c.v, vreg, t + 2);
            load_one(c.k, kreg, t + (AHEAD ? 3 : 2));
        };
        for (int t = 0; t < nt; t += 2) {
            step(t, 0, SA, AHEAD ? SB : SA);
            if (t + 1 < nt) step(t + 1, 1, AHEAD ? SB : SA, SA);
        }
    }

    if (!on) return;
    l_sum = xsum32(l_sum);
    float f = 1.0f;
    char* out;
    if (splits > 1) {
        const int64_t pr = (((int64_t)sp * c.n_seq + s) * a.n_q + iq) * a.heads + h;
        out = reinterpret_cast<char*>(a.part + pr * D);
        if (g == 0) *reinterpret_cast<v4f*>(a.part + (int64_t)splits * c.n_seq * a.n_q * a.heads * D + pr * 4) = v4f{m_ref, p_ref, l_sum, 0.0f};
    } else {
        f = l_sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(p_ref - m_ref) / l_sum;
        out = a.dst + (int64_t)h * a.d_nb[0] + (int64_t)iq * a.d_nb[1] + (int64_t)s * a.d_nb[2];
    }
    const bool h16 = splits == 1 && a.d16;
#pragma unroll
    for (int b = 0; b < NDB; ++b)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            const int e = 32 * b + 8 * i4 + 4 * g;
            const v4f y = v4f{O[b][4 * i4], O[b][4 * i4 + 1], O[b][4 * i4 + 2], O[b][4 * i4 + 3]} * f;
            if (h16) *reinterpret_cast<v4h_a2*>(out + 2 * e) = __builtin_convertvector(y, v4h);
            else *reinterpret_cast<v4f_a4*>(out + 4 * e) = y;
        }
}

// The joins of kv_attn_tiles_kernel's ranges: thread per four elements of a row
template <int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(const KvAttnArgs a, const int splits) {
    constexpr int C4 = D / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, pr = i / C4;
    if (pr >= (int64_t)a.c.n_seq * a.n_q * a.heads) return;
    const KvRange kr = kv_range(a, (int)(pr / a.heads / a.n_q));
    if (pr / a.heads % a.n_q >= kr.nq) return;
    const int chunk = kv_chunk(kr, splits);
    join_ranges<D, false>(a, splits, max((kr.hi - kr.lo + chunk - 1) / chunk, 1), pr, (int)(i - pr * C4) * 4);
}

// The kernel, its row tiles and the ranges of the tokens for n_q queries.
// Up to 16 rows (decoding) the number of ranges is the cheapest of: steps of 128 tokens of a range at 0.5 us, or 0.35 us
// for each workgroup of a CU where there are more than that; and, from two ranges on, the join's 1.3 us (more past the
// eight ranges of one round of its loads) and 1 us for each workgroup of a CU, which all write partial sums.  Four
// workgroups to a CU at most, and no more ranges than twice the root of the steps, since one workgroup joins them.
// 32 conversations of 16384 tokens, 8 key heads: two ranges 153 us, four 164, sixteen 189; one of 19328 tokens with 28
// heads: 16 us, and 26 with 128 ranges.
// Beyond, the kernels of 16, 32 and 128 rows are compared at their best number of ranges by the rounds of workgroups
// over the CUs times a step's time (tens of nanoseconds, heads of 128) with one and with two workgroups on a CU: the
// widest has the throughput of many rows, the narrowest the shortest steps and joins where the CUs are not full
// (63 F32 rows of two sequences of 2424 tokens: 13.9 us with 16 rows to a workgroup, 19.8 with 32, 20.4 with 128; 80
// rows of 32 sequences and heads of 3000 tokens: 24.5, 27.3 and 23.0).  An item's row tiles of 16 or 32 share an XCD, so
// that fewer than eight items leave XCDs idle (3160 rows of four key heads: 29.6 us with 32 rows, 15.5 with 128).
KvAttnPlan kv_attn_plan(int n_q, int heads, int heads_kv, int n_seq, int64_t max_tokens, int window, int D, bool q16, int cus) {
    if (window > 0) max_tokens = std::min<int64_t>(max_tokens, (int64_t)window + n_q + KV_STEP);  // (kv_range)
    const int64_t rows = (int64_t)n_q * (heads / heads_kv), items = std::max<int64_t>((int64_t)heads_kv * n_seq, 1);
    const int64_t steps = std::max<int64_t>((max_tokens + KV_SPAN - 1) / KV_SPAN, 1);  // of 128 tokens
    cus = std::max(cus, 1);
    int64_t root = 8;  // (as many as one round of a join's loads)
    while (root < KV_RANGES && root * root < 4 * steps) ++root;
    KvAttnPlan p;
    if (rows <= 16) {
        p.nt = 1;
        p.tiles = 1;
        p.splits = 1;
        double best = 0.0;
        const int64_t most = std::min<int64_t>({(4LL * cus + items - 1) / items, steps, root});
        for (int s = 1; s <= most; ++s) {
            const int64_t per = (steps + s - 1) / s;
            const double load = (double)(items * s) / cus;
            const double t = (per + 1) * 50.0 * std::max(1.0, 0.7 * load) + (s == 1 ? 0.0 : 130.0 + 10.0 * std::max(s - 8, 0) + 100.0 * load);
            if (s == 1 || t < best) best = t, p.splits = s;
        }
    } else {
        double best = 1e300;
        for (int nt : {1, 2, 0}) {
            if (nt == 0 && rows <= 64) break;
            const int64_t row = nt ? 16 * nt : 128, wgs = (rows + row - 1) / row;
            for (int s = 1; s <= std::min<int64_t>(steps, nt ? root : 32); ++s) {
                const int64_t n = wgs * (nt ? (items * s + 7) / 8 * 8 : items * s), rounds = (n + 2 * cus - 1) / (2 * cus), per = (steps + s - 1) / s;
                const bool alone = n <= cus;
                const double step = nt == 1   ? (alone ? (q16 ? 100.0 : 115.0) : (q16 ? 140.0 : 170.0))
                                    : nt == 2 ? (alone ? (q16 ? 155.0 : 185.0) : (q16 ? 165.0 : 200.0))
                                              : (alone ? (q16 ? 275.0 : 375.0) : (q16 ? 385.0 : 610.0));
                const double join = s == 1    ? 0.0
                                    : nt == 1 ? 340.0 + 30.0 * s
                                    : nt == 2 ? 480.0 + 50.0 * s
                                              : 650.0 + s * (double)(rows * items * D) / 10000.0;
                const double t = rounds * (per * step + (nt == 1 ? 180.0 : 250.0)) + join;
                if (t < best) {
                    best = t;
                    p.nt = nt;
                    p.splits = s;
                }
            }
        }
        const int rt = p.nt ? 16 * p.nt : 128;
        p.tiles = (int)((rows + rt - 1) / rt);
    }
    if (p.nt && items * p.tiles > KV_ARRIVALS) p.splits = 1;  // (workgroups enough without)
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
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    auto tile = [&](auto qs, auto ps) {
        kv_attn_tiles_kernel<D, decltype(qs)::value, decltype(ps)::value><<<(unsigned)(items * p.tiles), 256, 0, st>>>(a, p.splits, p.tiles);
    };
    if (p.nt == 0) {
        if (a.q16 && a.d16) tile(std::false_type(), std::false_type());
        else if (a.q16) tile(std::false_type(), std::true_type());
        else if (a.d16) tile(std::true_type(), std::false_type());
        else tile(std::true_type(), std::true_type());
    } else if (p.nt == 1) go(std::integral_constant<int, 1>());
    else go(std::integral_constant<int, 2>());
    if (p.nt == 0 && p.splits > 1) {
        const int64_t n = (int64_t)a.c.n_seq * a.n_q * a.heads * (D / 4);
        kv_attn_join_kernel<D><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a, p.splits);
    }
    return hipGetLastError();
}

hipError_t launch_kv_attn(const KvAttnArgs& a, const KvAttnPlan& p, int D, hipStream_t st) {
    const int64_t rows = (int64_t)a.n_q * a.heads * a.c.n_seq;
    if (rows <= 0) return hipSuccess;
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    if ((items + 7) / 8 * 8 * p.tiles > INT32_MAX || rows * (D / 4) > (int64_t)INT32_MAX * 256 || (p.splits > 1 && (!a.part || (p.nt && !a.arrived))))
        return hipErrorInvalidValue;
    switch (D) {
        case 64: return kv_attn_d<64>(a, p, st);
        case 96: return kv_attn_d<96>(a, p, st);
        case 128: return kv_attn_d<128>(a, p, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mi355
