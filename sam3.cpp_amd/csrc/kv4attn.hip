// Attention over the 4-bit cache (kv4.cuh), and the sums of its weights by token:
//
//   dst[s][i][h] = sum_t softmax_t(scale q_i . k_t) v_t,   lse[s][i][h] = log sum_t exp(scale q_i . k_t)
//   sums[s][hk][t] += sum over i and the heads h of hk's group of exp(scale q_i . k_t - lse[s][i][h])
//
// over the tokens t that query i sees (n_kv, causal, window), with fp32 online softmax.
#include <algorithm>
#include <type_traits>

#include "attn.cuh"
#include "kv4.cuh"

namespace mi355 {

namespace {
constexpr float KV4_LOG2E = 1.44269504088896340736f, KV4_LN2 = 0.69314718055994530942f;
constexpr float KV4_NONE = -1e30f;   // a reference that nothing has been taken against yet
constexpr float KV4_LIFT = 12.0f;    // probabilities are raised by 2^12 to keep small ones in fp16's normal range
constexpr float KV4_ROOM = 15.0f;    // and their reference moves when one would pass 2^15
constexpr int KV4_RANGES = 64;       // ranges of a row that one workgroup joins, at most
}  // namespace

// ---- operands of v_mfma_f32_16x16x32_f16 with 16 tokens on one side and 16 rows on the other.  A row is one query and
// head of the group that shares a key head: row r of a sequence and key head is query r / group, head r % group.
// Product m of a lane's quarter g takes eight elements from here on: a lane's bytes of a key row lie together.
template <int D>
__device__ __forceinline__ int piece_of(int m, int g) {
    return D == 128 ? 32 * g + 8 * m : m < 2 ? 16 * g + 8 * m : 64 + 8 * g;
}
// A lane's words of 16 keys, its scales, and the halves they make
template <int D>
struct Keys {
    uint32_t w[D / 32];
    uint16_t s[D == 96 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t* k, const uint16_t* scale, int col, int g) {
        if constexpr (D == 128) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(k + col * 64 + 16 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = x[i];
            s[0] = scale[col * 4 + g];
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(k + col * (D / 2) + 8 * g);
            w[0] = x[0];
            w[1] = x[1];
            s[0] = scale[col * (D / 32) + (g >> 1)];
            if constexpr (D == 96) {
                w[2] = *reinterpret_cast<const uint32_t*>(k + col * 48 + 32 + 4 * g);
                s[1] = scale[col * 3 + 2];
            }
        }
    }
    __device__ __forceinline__ v8h halves(int m) const {
        const _Float16 d = __builtin_bit_cast(_Float16, s[D == 96 && m == 2 ? 1 : 0]);
        uint32_t f[4];
        word_halves(w[m], h2v{d, d}, f);
        return __builtin_bit_cast(v8h, u32x4{f[0], f[1], f[2], f[3]});
    }
};
// A lane's part of a row of queries at p (none: zeros).  QS: an F32 row enters as two halves of 11 bits, scaled by a
// power of two that brings its largest magnitude to about one; up undoes it.
template <int D, bool QS>
struct Row {
    v8h q[D / 32], ql[QS ? D / 32 : 1];
    float up;
    __device__ __forceinline__ void load(const char* p, bool on, int g) {
        up = 1.0f;
        if constexpr (QS) {
            float x[D / 32][8], top = 0.0f;
#pragma unroll
            for (int m = 0; m < D / 32; ++m) {
                const int e = piece_of<D>(m, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[m][j] = 0.0f;
                if (on) {
                    const v4f lo = *reinterpret_cast<const v4f_a4*>(p + 4 * e), hi = *reinterpret_cast<const v4f_a4*>(p + 4 * e + 16);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[m][j] = j < 4 ? lo[j & 3] : hi[j & 3];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[m][j]));
            }
            const Pow2 z = pow2_of(col_max(top));
            up = z.up;
#pragma unroll
            for (int m = 0; m < D / 32; ++m)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = x[m][j] * z.down;
                    q[m][j] = (_Float16)y;
                    ql[m][j] = (_Float16)(y - (float)q[m][j]);
                }
        } else {
#pragma unroll
            for (int m = 0; m < D / 32; ++m) {
                const v8h z = {0, 0, 0, 0, 0, 0, 0, 0};
                q[m] = on ? *reinterpret_cast<const v8h_a2*>(p + 2 * piece_of<D>(m, g)) : z;
            }
        }
    }
};
__device__ __forceinline__ const char* row_at(const Kv4AttnArgs& a, int s, int iq, int h) {
    return a.q + (int64_t)iq * a.q_nb[0] + (int64_t)h * a.q_nb[1] + (int64_t)s * a.q_nb[2];
}

// A lane's words of the values of eight tokens, 4 g .. 4 g + 3 of both halves of 32, and their scales
template <int D>
struct Values {
    uint32_t w[2][4];
    u32x2 s[2];                       // of two tokens each
    uint32_t tw[D == 96 ? 2 : 1][4];  // the last 32 elements of 96
    u32x2 ts[D == 96 ? 2 : 1];
    __device__ __forceinline__ void load(int u, const uint8_t* v, const uint16_t* scale, int bt, int col, int g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint8_t* row = v + (4 * g + i) * (D / 2);
            if constexpr (D == 128) w[u][i] = *reinterpret_cast<const uint32_t*>(row + 4 * col);
            else w[u][i] = *reinterpret_cast<const uint16_t*>(row + 2 * col);
            if constexpr (D == 96) tw[u][i] = row[32 + col];
        }
        s[u] = *reinterpret_cast<const u32x2*>(scale + (D == 128 ? col >> 2 : col >> 3) * bt + 4 * g);
        if constexpr (D == 96) ts[u] = *reinterpret_cast<const u32x2*>(scale + 2 * bt + 4 * g);
    }
    // Scales of no value, of tokens that some row does not see: 0 times theirs must be 0
    __device__ __forceinline__ void clean() {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                s[u][x] = finite_scales(s[u][x]);
                if constexpr (D == 96) ts[u][x] = finite_scales(ts[u][x]);
            }
    }
    // Block b of 16 elements as an operand: a register holds two tokens
    __device__ __forceinline__ v8h halves(int b) const {
        u32x4 f;
        const bool tail = D == 96 && b >= 4;
#pragma unroll
        for (int x = 0; x < 4; ++x) {  // tokens 2 (x & 1), + 1 of half x >> 1
            const int u = x >> 1, i = 2 * (x & 1);
            const h2v d = __builtin_bit_cast(h2v, tail ? ts[D == 96 ? u : 0][x & 1] : s[u][x & 1]);
            const uint32_t t0 = tail ? tw[D == 96 ? u : 0][i] : w[u][i], t1 = tail ? tw[D == 96 ? u : 0][i + 1] : w[u][i + 1];
            const uint32_t two = __builtin_amdgcn_perm(t1, t0, D == 128 && b >= 4 ? 0x07060302u : 0x05040100u);
            const int n = tail ? b - 4 : b & 3;
            const uint32_t y = n >= 2 ? two >> 8 : two;
            f[x] = __builtin_bit_cast(uint32_t, (n & 1 ? nibble_pair<4>(y) : nibble_pair<0>(y)) * d);
        }
        return __builtin_bit_cast(v8h, f);
    }
};
// Where element e of an output row is: row 0 .. 15 of block b
template <int D>
__device__ __forceinline__ void block_of(int e, int& ar, int& b) {
    const int x = (e & 7) >> 1, odd = e & 1;  // nibble x of the word's half `odd`
    if (D == 128) {
        ar = e >> 3;
        b = x + 4 * odd;
    } else if (D == 64 || e < 64) {
        ar = 2 * (e >> 3) + odd;
        b = x;
    } else {  // a byte has nibbles x and x + 1, x even
        ar = 4 * ((e - 64) >> 3) + 2 * odd + (x >> 1);
        b = 4 + (x & 1);
    }
}

__device__ __forceinline__ void put_lse(const Kv4AttnArgs& a, int64_t pr, float m, float l) {
    if (a.lse) a.lse[pr] = l == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * KV4_LN2;
}
__device__ __forceinline__ char* out_at(const Kv4AttnArgs& a, int64_t pr) {
    const int64_t h = pr % a.heads, iq = pr / a.heads % a.n_q, s = pr / a.heads / a.n_q;
    return a.dst + h * a.d_nb[0] + iq * a.d_nb[1] + s * a.d_nb[2];
}
__device__ __forceinline__ void put_four(const Kv4AttnArgs& a, char* out, int e, v4f y) {
    if (a.d16) *reinterpret_cast<v4h_a2*>(out + 2 * e) = __builtin_convertvector(y, v4h);
    else *reinterpret_cast<v4f_a4*>(out + 4 * e) = y;
}

// A workgroup takes 16 rows and one range of the tokens, its four wavefronts every fourth step of 32 tokens; the cache's
// bytes go from memory to the registers that the matrix instructions read, each once.
//   scores  S^T[token][row] = K Q^T;
//   output  O^T[element][row] += V^T P^T: a lane's eight scores (tokens 4 g .. 4 g + 3 of both 16-token halves) are the
//           eight places of its column in the B operand.
// PS: for an F32 output the probabilities enter as two halves; for an F16 one the fp32 sum is of the halves that the
// product takes, whose roundings then cancel, and lse has a sum of its own of the probabilities before them.
template <int D, bool QS, bool PS>
__global__ __launch_bounds__(256) void kv4_rows_kernel(const Kv4AttnArgs a, const int splits, const int tiles) {
    constexpr int KM = D / 32, NB = D / 16;
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    // the row tiles of one item go to the same XCD, one after another, and find its bytes in that L2
    const int per = 8 * tiles, gb = blockIdx.x / per, rb = blockIdx.x % per;
    const int item = gb * 8 + (rb & 7), tile = rb >> 3;
    if (item >= splits * c.heads * c.n_seq) return;
    const int sp = item % splits, hk = item / splits % c.heads, s = item / splits / c.heads;
    const KvRange kr = kv_range(a, s);
    const int rows = kr.nq * a.group, row0 = tile * 16;
    if (row0 >= rows) return;
    const int chunk = kv_chunk(kr, splits), tb = kr.lo + sp * chunk;
    const int last = min(row0 + 16, rows) - 1, iq0 = row0 / a.group, iq1 = last / a.group;
    // tokens that some row of this tile can see, and those that all do (rows past the last one see what they like)
    const int te = min(min(tb + chunk, kr.hi), a.causal ? kr.pos0 + iq1 + 1 : kr.hi);
    const int all_hi = a.causal ? min(kr.pos0 + iq0 + 1, te) : te, all_lo = a.window > 0 ? kr.pos0 + iq1 - a.window + 1 : 0;
    if (sp > 0 && tb >= kr.hi) return;  // no such range (the first always answers)
    const int ranges = max((kr.hi - kr.lo + chunk - 1) / chunk, 1);

    const int r = row0 + col, iq = r / a.group;
    const bool on = r < rows;
    Row<D, QS> row;
    row.load(row_at(a, s, iq, hk * a.group + (r - iq * a.group)), on, g);
    const int pos = kr.pos0 + iq;
    const int see_hi = on ? (a.causal ? min(pos + 1, te) : te) : 0, see_lo = a.window > 0 ? pos - a.window + 1 : 0;
    const float f = a.scale * KV4_LOG2E * row.up;

    float m_ref = KV4_NONE, l_sum = 0.0f, l_all = 0.0f;  // (l_all: before the rounding)
    v4f O[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) O[b] = v4f{0, 0, 0, 0};

    // The blocks of 16 tokens each: lane 2 i + u keeps that of half u of this wavefront's i-th step from a token on.
    struct Step {
        int64_t tok[2];  // place of the first token among all of the cache
        bool there[2];
    };
    int ids = -1, at = 32;
    Keys<D> key[2];
    auto ask = [&](int t0) {
        Step x;
        if (at == 32) {
            ids = kv4_block(c, s, t0 + (lane >> 1) * KV_SPAN + 16 * (lane & 1));
            at = 0;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int id = __builtin_amdgcn_readlane(ids, 2 * at + u);
            x.there[u] = id >= 0;
            x.tok[u] = ((int64_t)max(id, 0) * c.heads + hk) * c.bt + ((t0 + 16 * u) & (c.bt - 1));
            key[u].load(c.k + x.tok[u] * (D / 2), c.k_scale + x.tok[u] * KM, col, g);
        }
        ++at;
        return x;
    };
    Step next{};
    if (tb + w * KV_STEP < te) next = ask(tb + w * KV_STEP);
    for (int t0 = tb + w * KV_STEP; t0 < te; t0 += KV_SPAN) {
        const Step x0 = next;
        Values<D> val;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int in = (t0 + 16 * u) & (c.bt - 1);
            val.load(u, c.v + x0.tok[u] * (D / 2), c.v_scale + (x0.tok[u] - in) * KM + in, c.bt, col, g);
        }
        v4f S[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            S[u] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                const v8h k8 = key[u].halves(m);
                S[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, row.q[m], S[u], 0, 0, 0);
                if constexpr (QS) S[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, row.ql[m], S[u], 0, 0, 0);
            }
        }
        if (t0 + KV_SPAN < te) next = ask(t0 + KV_SPAN);

        float x[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u][i] = S[u][i] * f;
        if (!(x0.there[0] && x0.there[1] && t0 >= all_lo && t0 + KV_STEP <= all_hi)) {
            val.clean();
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tt = t0 + 16 * u + 4 * g + i;
                    if (!(x0.there[u] && tt >= see_lo && tt < see_hi)) x[u][i] = -__builtin_inff();
                }
        }
        const float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
        if (__builtin_amdgcn_ballot_w64(top > m_ref + KV4_ROOM)) {
            const float mn = fmaxf(m_ref, col_max(top) - KV4_LIFT), am = __builtin_amdgcn_exp2f(m_ref - mn);
            m_ref = mn;
            l_sum *= am;
            l_all *= am;
#pragma unroll
            for (int b = 0; b < NB; ++b) O[b] *= am;
        }
        u32x4 P, PL;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(x[u][i] - m_ref);
            const h2v h0 = __builtin_convertvector((v2f{p[0], p[1]}), h2v), h1 = __builtin_convertvector((v2f{p[2], p[3]}), h2v);
            P[2 * u] = __builtin_bit_cast(uint32_t, h0);
            P[2 * u + 1] = __builtin_bit_cast(uint32_t, h1);
            if constexpr (PS) {
                l_sum += (p[0] + p[1]) + (p[2] + p[3]);
                const h2v e0 = __builtin_convertvector((v2f{p[0] - (float)h0[0], p[1] - (float)h0[1]}), h2v);
                const h2v e1 = __builtin_convertvector((v2f{p[2] - (float)h1[0], p[3] - (float)h1[1]}), h2v);
                PL[2 * u] = __builtin_bit_cast(uint32_t, e0);
                PL[2 * u + 1] = __builtin_bit_cast(uint32_t, e1);
            } else {
                const h2v ones = {(_Float16)1.0f, (_Float16)1.0f};
                l_sum = __builtin_amdgcn_fdot2(h1, ones, __builtin_amdgcn_fdot2(h0, ones, l_sum, false), false);
                if (a.lse) l_all += (p[0] + p[1]) + (p[2] + p[3]);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const v8h v8 = val.halves(b);
            O[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, __builtin_bit_cast(v8h, P), O[b], 0, 0, 0);
            if constexpr (PS) O[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, __builtin_bit_cast(v8h, PL), O[b], 0, 0, 0);
        }
    }

    // join the wavefronts: 2 and 3 into 0 and 1, then 1 into 0
    __shared__ __attribute__((aligned(16))) v4f so[2][NB][64];
    __shared__ float sm[2][3][16];
    l_sum = col_sum(l_sum);
    l_all = PS ? l_sum : col_sum(l_all);
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
        if (w >= half && w < 2 * half) {
#pragma unroll
            for (int b = 0; b < NB; ++b) so[w - half][b][lane] = O[b];
            if (g == 0) {
                sm[w - half][0][col] = m_ref;
                sm[w - half][1][col] = l_sum;
                sm[w - half][2][col] = l_all;
            }
        }
        __syncthreads();
        if (w < half) {
            const float m2 = sm[w][0][col], l2 = sm[w][1][col], mn = fmaxf(m_ref, m2);
            const float a1 = __builtin_amdgcn_exp2f(m_ref - mn), a2 = __builtin_amdgcn_exp2f(m2 - mn);
            l_sum = l_sum * a1 + l2 * a2;
            l_all = l_all * a1 + sm[w][2][col] * a2;
#pragma unroll
            for (int b = 0; b < NB; ++b) O[b] = O[b] * a1 + so[w][b][lane] * a2;
            m_ref = mn;
        }
        __syncthreads();
    }
    // row y of the tile: its number among all (sequence, query, head in that order)
    auto number = [&](int y) {
        const int q = (row0 + y) / a.group;
        return row0 + y < rows ? ((int64_t)s * a.n_q + q) * a.heads + hk * a.group + (row0 + y - q * a.group) : (int64_t)-1;
    };
    const int64_t all = (int64_t)c.n_seq * a.n_q * a.heads;
    float* ml = a.part + (int64_t)splits * all * D;
    if (w == 0) {
        const float z = ranges > 1 ? 1.0f : l_sum == 0.0f ? 0.0f : 1.0f / l_sum;
#pragma unroll
        for (int b = 0; b < NB; ++b) so[0][b][lane] = O[b] * z;
        const int64_t pr = number(col);
        if (g == 0 && pr >= 0) {
            if (ranges > 1) {
                put_through(ml + (sp * all + pr) * 4, v2f{m_ref, l_sum});
                put_through(ml + (sp * all + pr) * 4 + 2, v2f{l_all, 0.0f});
            } else {
                put_lse(a, pr, m_ref, l_all);
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
        const int y = i / (D / 4), e = 4 * (i % (D / 4));
        const int64_t pr = number(y);
        if (pr < 0) break;
        v4f o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            int ar, b;
            block_of<D>(e + j, ar, b);
            o[j] = so[0][b][y + 16 * (ar >> 2)][ar & 3];
        }
        if (ranges == 1) {
            put_four(a, out_at(a, pr), e, o);
        } else {  // one of several ranges: its sums go to memory past the caches
            float* to = a.part + ((int64_t)sp * all + pr) * D + e;
            put_through(to, v2f{o[0], o[1]});
            put_through(to + 2, v2f{o[2], o[3]});
        }
    }
    if (ranges == 1) return;
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
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
        const int y = i / (D / 4), e = 4 * (i % (D / 4));
        const int64_t pr = number(y);
        if (pr < 0) break;
        constexpr int B = 8;  // ranges whose loads are on their way together
        float m = KV4_NONE, l = 0.0f, la = 0.0f;
        v4f o = {0, 0, 0, 0};
        for (int x0 = 0; x0 < ranges; x0 += B) {
            v2f z[B], lo[B], hi[B];
            float za[B];
#pragma unroll
            for (int x = 0; x < B; ++x) {
                z[x] = v2f{KV4_NONE, 0.0f};
                za[x] = 0.0f;
                lo[x] = hi[x] = v2f{0, 0};
                if (x0 + x < ranges) {
                    z[x] = get_through(ml + ((x0 + x) * all + pr) * 4);
                    if (e == 0) za[x] = get_through(ml + ((x0 + x) * all + pr) * 4 + 2)[0];
                    lo[x] = get_through(a.part + ((x0 + x) * all + pr) * D + e);
                    hi[x] = get_through(a.part + ((x0 + x) * all + pr) * D + e + 2);
                }
            }
            float mn = m;
#pragma unroll
            for (int x = 0; x < B; ++x) mn = fmaxf(mn, z[x][0]);
            const float old = __builtin_amdgcn_exp2f(m - mn);
            l *= old;
            la *= old;
            o = o * old;
            m = mn;
#pragma unroll
            for (int x = 0; x < B; ++x) {
                const float y2 = __builtin_amdgcn_exp2f(z[x][0] - m);
                l += z[x][1] * y2;
                la += za[x] * y2;
                o = o + v4f{lo[x][0], lo[x][1], hi[x][0], hi[x][1]} * y2;
            }
        }
        put_four(a, out_at(a, pr), e, o * (l == 0.0f ? 0.0f : 1.0f / l));
        if (e == 0) put_lse(a, pr, m, la);
    }
}

// ---- the weights' sums by token
// A wavefront keeps 32 tokens' keys as halves and walks over the rows, 16 at a time: S[row][token] = Q K^T gives a lane four
// rows of one token.  exp(scale q . k - lse) is taken of the difference, so that the largest weights, which have the smallest
// ones, lose least.  The rows' sums are taken in two levels, 64 tiles and then those, for 32 bits to hold them.
template <int D, bool QS>
__global__ __launch_bounds__(256) void kv4_weights_kernel(const Kv4AttnArgs a, float* sums) {
    constexpr int KM = D / 32;
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int hk = blockIdx.y, s = blockIdx.z;
    const KvRange kr = kv_range(a, s);
    const int t0 = kr.lo + (blockIdx.x * 4 + w) * KV_STEP;
    if (t0 >= kr.hi) return;
    const int rows = kr.nq * a.group;
    // queries that see one of these tokens
    const int q_lo = a.causal ? max(t0 - kr.pos0, 0) : 0;
    const int q_hi = a.window > 0 ? (int)min((int64_t)kr.nq, (int64_t)t0 + KV_STEP - 1 + a.window - kr.pos0) : kr.nq;
    if (q_lo >= q_hi) return;
    Keys<D> key[2];
    bool there[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int id = kv4_block(c, s, t0 + 16 * u);
        there[u] = id >= 0;
        const int64_t tok = ((int64_t)max(id, 0) * c.heads + hk) * c.bt + ((t0 + 16 * u) & (c.bt - 1));
        key[u].load(c.k + tok * (D / 2), c.k_scale + tok * KM, col, g);
    }
    v8h k8[2][KM];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int m = 0; m < KM; ++m) k8[u][m] = key[u].halves(m);
    float total[2] = {0, 0}, some[2] = {0, 0};
    int n = 0;
    const int r_end = min(q_hi * a.group, rows);
    for (int row0 = q_lo * a.group; row0 < r_end; row0 += 16) {
        const int r = row0 + col, iq = r / a.group, h = hk * a.group + (r - iq * a.group);
        const bool on = r < r_end;
        Row<D, QS> row;
        row.load(row_at(a, s, iq, h), on, g);
        const float lse = on ? a.lse[((int64_t)s * a.n_q + iq) * a.heads + h] : 0.0f;
        v4f S[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            S[u] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                S[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(row.q[m], k8[u][m], S[u], 0, 0, 0);
                if constexpr (QS) S[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(row.ql[m], k8[u][m], S[u], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int y = 4 * g + i, q = (row0 + y) / a.group, pos = kr.pos0 + q;
            const float l = __shfl(lse, y, 64), f = QS ? a.scale * __shfl(row.up, y, 64) : a.scale;
            const int hi = row0 + y < r_end ? (a.causal ? min(pos + 1, kr.hi) : kr.hi) : 0, lo = a.window > 0 ? pos - a.window + 1 : 0;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int t = t0 + 16 * u + col;
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[u][i], f, -l) * KV4_LOG2E);
                some[u] += there[u] && t >= lo && t < hi ? p : 0.0f;
            }
        }
        if (++n == 64) {
            n = 0;
#pragma unroll
            for (int u = 0; u < 2; ++u) total[u] += some[u], some[u] = 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const float x = col_sum(total[u] + some[u]);
        const int t = t0 + 16 * u + col;
        if (g == 0 && there[u] && t < kr.hi) {
            float* p = sums + ((int64_t)s * c.heads + hk) * c.max_blocks * c.bt + t;
            *p += x;
        }
    }
}

// The ranges of the tokens for n_q queries.
Kv4AttnPlan kv4_attn_plan(int n_q, int heads, int heads_kv, int n_seq, int64_t max_tokens, int window, int D, bool q16, int cus) {
    if (window > 0) max_tokens = std::min<int64_t>(max_tokens, (int64_t)window + n_q + KV_STEP);  // (kv_range)
    const int64_t rows = (int64_t)n_q * (heads / heads_kv), items = std::max<int64_t>((int64_t)heads_kv * n_seq, 1);
    const int64_t steps = std::max<int64_t>((max_tokens + KV_SPAN - 1) / KV_SPAN, 1);  // of 128 tokens
    cus = std::max(cus, 1);
    Kv4AttnPlan p;
    p.tiles = (int)((rows + 15) / 16);
    const int64_t wgs = items * p.tiles;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(2 * cus + wgs - 1) / wgs, steps, KV4_RANGES}));
    if (wgs > KV_ARRIVALS) p.splits = 1;  // (workgroups enough without)
    p.bytes = p.splits > 1 ? (size_t)p.splits * n_seq * n_q * heads * (D + 4) * 4 : 0;
    return p;
}

template <int D>
static hipError_t kv4_attn_d(const Kv4AttnArgs& a, const Kv4AttnPlan& p, hipStream_t st) {
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    const unsigned n = (unsigned)((items + 7) / 8 * 8 * p.tiles);
    if (a.q16 && a.d16) kv4_rows_kernel<D, false, false><<<n, 256, 0, st>>>(a, p.splits, p.tiles);
    else if (a.q16) kv4_rows_kernel<D, false, true><<<n, 256, 0, st>>>(a, p.splits, p.tiles);
    else if (a.d16) kv4_rows_kernel<D, true, false><<<n, 256, 0, st>>>(a, p.splits, p.tiles);
    else kv4_rows_kernel<D, true, true><<<n, 256, 0, st>>>(a, p.splits, p.tiles);
    return hipGetLastError();
}

hipError_t launch_kv4_attn(const Kv4AttnArgs& a, const Kv4AttnPlan& p, int D, hipStream_t st) {
    if ((int64_t)a.n_q * a.heads * a.c.n_seq <= 0) return hipSuccess;
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    if ((items + 7) / 8 * 8 * p.tiles > INT32_MAX || (p.splits > 1 && (!a.part || !a.arrived))) return hipErrorInvalidValue;
    switch (D) {
        case 64: return kv4_attn_d<64>(a, p, st);
        case 96: return kv4_attn_d<96>(a, p, st);
        case 128: return kv4_attn_d<128>(a, p, st);
        default: return hipErrorInvalidValue;
    }
}

template <int D>
static hipError_t kv4_weights_d(const Kv4AttnArgs& a, float* sums, hipStream_t st) {
    int64_t tokens = (int64_t)a.c.max_blocks * a.c.bt;
    if (a.window > 0) tokens = std::min<int64_t>(tokens, (int64_t)a.window + a.n_q + KV_STEP);
    const dim3 n((unsigned)((tokens + KV_SPAN - 1) / KV_SPAN), (unsigned)a.c.heads, (unsigned)a.c.n_seq);
    if (a.q16) kv4_weights_kernel<D, false><<<n, 256, 0, st>>>(a, sums);
    else kv4_weights_kernel<D, true><<<n, 256, 0, st>>>(a, sums);
    return hipGetLastError();
}

hipError_t launch_kv4_weights(const Kv4AttnArgs& a, float* sums, int D, hipStream_t st) {
    if ((int64_t)a.n_q * a.heads * a.c.n_seq <= 0 || a.c.max_blocks <= 0 || a.c.n_blocks <= 0) return hipSuccess;
    switch (D) {
        case 64: return kv4_weights_d<64>(a, sums, st);
        case 96: return kv4_weights_d<96>(a, sums, st);
        case 128: return kv4_weights_d<128>(a, sums, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mi355
