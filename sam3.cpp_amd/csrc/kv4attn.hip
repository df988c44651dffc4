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
constexpr float KV4_LIFT = 12.0f;    // probabilities are raised by 2^12 to keep small ones in fp16's normal range, and their reference moves when one passes 2^15
constexpr float KV4_LIFT_SUM = 8.0f; // the same where a lane's sum of 32 of them, and not each, is held below 2^15
constexpr int KV4_TILE = 64;         // tokens of a tile of the many rows' kernel; where a sequence's seen tokens begin
constexpr int64_t KV4_GRID = UINT32_MAX / 256;  // workgroups of a launch, at most
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

// What turns a row's products into exponents of 2.  The row's power of two comes first, for the scale to be a normal number
// where the scores are of a size that counts.  Neither zero nor infinite: hidden scores are -inf, products may be zero.
__device__ __forceinline__ float score_factor(float scale, float up) {
    return fminf(fmaxf(fabsf(scale) * up * KV4_LOG2E, 1e-37f), 3e38f);
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

// Four elements from e on of row pr, joined from the row's n ranges in the ranges' order and written.  ONE: other workgroups
// of this launch wrote the partial sums.
template <int D, bool ONE>
__device__ __forceinline__ void join_ranges(const Kv4AttnArgs& a, int splits, int n, int64_t pr, int e) {
    const int64_t all = (int64_t)a.c.n_seq * a.n_q * a.heads;
    const float* ml = a.part + (int64_t)splits * all * D + pr * 4;
    const float* po = a.part + pr * D + e;
    auto get = [](const float* q) {
        if constexpr (!ONE) return *reinterpret_cast<const v4f*>(q);
        const v2f lo = get_through(q), hi = get_through(q + 2);
        return v4f{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int B = 8;  // ranges whose loads are on their way together
    float m = KV4_NONE, l = 0.0f, la = 0.0f;
    v4f o = {0, 0, 0, 0};
    for (int x0 = 0; x0 < n; x0 += B) {
        v4f z[B], y[B];
#pragma unroll
        for (int x = 0; x < B; ++x) {
            z[x] = v4f{KV4_NONE, 0, 0, 0};
            y[x] = v4f{0, 0, 0, 0};
            if (x0 + x < n) {
                z[x] = get(ml + (x0 + x) * all * 4);
                y[x] = get(po + (x0 + x) * all * D);
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
            const float up = __builtin_amdgcn_exp2f(z[x][0] - m);
            l += z[x][1] * up;
            la += z[x][2] * up;
            o = o + y[x] * up;
        }
    }
    put_four(a, out_at(a, pr), e, o * (l == 0.0f ? 0.0f : 1.0f / l));
    if (e == 0) put_lse(a, pr, m, la);
}

// A workgroup takes 16 rows and one range of the tokens, its four wavefronts every fourth step of 32 tokens; the cache's
// bytes go from memory to the registers that the matrix instructions read, each once.
//   scores  S^T[token][row] = K Q^T;
//   output  O^T[element][row] += V^T P^T: a lane's eight scores (tokens 4 g .. 4 g + 3 of both 16-token halves) are the
//           eight places of its column in the B operand.
// PS: for an F32 output the probabilities enter as two halves; for an F16 one the fp32 sum is of the halves that the
// product takes, whose roundings then cancel, and lse has a sum of its own of the probabilities before them.
// With many conversations the cache's bytes bound it, with four workgroups on a CU: 32 of 16384 tokens, 32 heads of 128 over 8,
// 459 MB in 104 us (4.4 TB/s; a step's 300 vector instructions are half of its time).  With few tokens the chain of
// latencies does: 777 tokens, 16 heads of 64 over 2 in 7.1 us.  Values asked for a step ahead as the keys are took the registers of
// the fourth workgroup and were no faster (110 us).
template <int D, bool QS, bool PS>
__global__ __launch_bounds__(256, QS && D > 64 ? 2 : 4) void kv4_rows_kernel(const Kv4AttnArgs a, const int splits, const int tiles) {
    constexpr int KM = D / 32, NB = D / 16;
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    // the row tiles of one item go to the same XCD, one after another, and find its bytes in that L2
    const int per = 8 * tiles, gb = blockIdx.x / per, rb = blockIdx.x % per;
    const int item = gb * 8 + (rb & 7), tile = rb >> 3;
    if (item >= splits * c.heads * c.n_seq) return;
    const int sp = item % splits, hk = item / splits % c.heads, s = item / splits / c.heads;
    const KvRange kr = kv_range<KV4_TILE>(a, s);
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
    const float f = score_factor(a.scale, row.up);
    if (a.scale < 0.0f)
#pragma unroll
        for (int m = 0; m < KM; ++m) {
            row.q[m] = -row.q[m];
            if constexpr (QS) row.ql[m] = -row.ql[m];
        }

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

        if (!(x0.there[0] && x0.there[1] && t0 >= all_lo && t0 + KV_STEP <= all_hi)) {
            val.clean();
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tt = t0 + 16 * u + 4 * g + i;
                    if (!(x0.there[u] && tt >= see_lo && tt < see_hi)) S[u][i] = -__builtin_inff();
                }
        }
        // at the reference as it stands, which moves to the step's largest where one would pass 2^15
        float p[2][4];
        auto raise = [&]() {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) p[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[u][i], f, -m_ref));
        };
        auto largest = [](const float (&x)[2][4]) {
            return fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
        };
        raise();
        if (__builtin_amdgcn_ballot_w64(largest(p) > 32768.0f)) {
            float top = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, S[u][i] * f);
            const float mn = fmaxf(m_ref, col_max(top) - KV4_LIFT), am = __builtin_amdgcn_exp2f(m_ref - mn);
            m_ref = mn;
            l_sum *= am;
            l_all *= am;
#pragma unroll
            for (int b = 0; b < NB; ++b) O[b] *= am;
            raise();
        }
        u32x4 P, PL;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const h2v h0 = __builtin_convertvector((v2f{p[u][0], p[u][1]}), h2v), h1 = __builtin_convertvector((v2f{p[u][2], p[u][3]}), h2v);
            P[2 * u] = __builtin_bit_cast(uint32_t, h0);
            P[2 * u + 1] = __builtin_bit_cast(uint32_t, h1);
            if constexpr (PS) {
                l_sum += (p[u][0] + p[u][1]) + (p[u][2] + p[u][3]);
                const h2v e0 = __builtin_convertvector((v2f{p[u][0] - (float)h0[0], p[u][1] - (float)h0[1]}), h2v);
                const h2v e1 = __builtin_convertvector((v2f{p[u][2] - (float)h1[0], p[u][3] - (float)h1[1]}), h2v);
                PL[2 * u] = __builtin_bit_cast(uint32_t, e0);
                PL[2 * u + 1] = __builtin_bit_cast(uint32_t, e1);
            } else {
                const h2v ones = {(_Float16)1.0f, (_Float16)1.0f};
                l_sum = __builtin_amdgcn_fdot2(h1, ones, __builtin_amdgcn_fdot2(h0, ones, l_sum, false), false);
                if (a.lse) l_all += (p[u][0] + p[u][1]) + (p[u][2] + p[u][3]);
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
        const int64_t pr = number(i / (D / 4));
        if (pr < 0) break;
        join_ranges<D, true>(a, splits, ranges, pr, 4 * (i % (D / 4)));
    }
}

// Many query rows: a workgroup takes 128 rows in four wavefronts of 32 and streams the tokens through LDS in tiles of 64,
// nibbles becoming halves once for all four on the way: a thread loads its words of a row ahead of time and
// writes them after the previous tile's products.  Scores and output as fattn.hip's (v_mfma_f32_32x32x16_f16, S^T = K Q^T,
// the probabilities' registers as the operand of O^T += V^T P^T, V^T by transposing reads); a tile's scores are
// computed one tile ahead of its softmax, so that the matrix pipe works beside the VALU: between a tile's score products go the
// first half's probabilities of the tile before, between that tile's first output products the second half's.
// 2 x 4096 causal F16 queries over 5120 tokens, 32 heads of 128 over 8: 336 to 390 us from one run to another (940 TFLOP/s), 20 of
// them for the halves, at a clock of 1.7 to 1.95 GHz.  No unit is full: matrix pipe busy 45 % of the time, VALU 42 %, LDS 23 %, 1.7
// wavefronts on a SIMD, which leave the first two one after another more often than side by side.
// 5184 F32 queries over 15552 tokens, 8 heads of 64, two halves of either operand: 330 us for 330 GFLOP (matrix pipe 54 %, VALU
// 58 %, LDS 13 %).  64 rows to a wavefront would halve the LDS reads, but leave one wavefront a SIMD: 673 and 407 us.
//
// V row slot of 16-byte chunk c in row r: c ^ this.  The transposing reads take four chunks from each of four rows, which lie
// in distinct quarters of the banks (as fattn.hip's vswz); with heads of 128 the chunks are turned within their
// quarter too, so that the sixteen lanes of a write, four rows of four quarters, take distinct banks.
template <int D>
__device__ __forceinline__ int v4swz(int r) { return D == 128 ? 5 * (r & 3) : vswz<D>(r); }

// A thread's words of a tile of 64 tokens: wavefront w has rows 16 w .. + 15, unit j of a lane words VW (u % UR) on of row
// u / UR, u = lane + 64 j.  As halves they lie in rows of D, a row's 16-byte chunks exchanged as kswz and v4swz say.
template <int D>
struct TileWords {
    static constexpr int NW = D / 32, VW = D == 96 ? 1 : NW, NV = NW / VW, G = D / 32, UR = D / 8 / VW;
    typedef uint32_t unit_t __attribute__((ext_vector_type(VW)));
    unit_t x[NV];
    uint16_t d[NV];
    // keys or values; at: place of the block's first token and head, in: the wavefront's first row in the block
    __device__ __forceinline__ void load(const Kv4View& c, bool val, int64_t at, int in, int lane) {
        const uint8_t* p = (val ? c.v : c.k) + (at + in) * (D / 2);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int u = lane + 64 * j, row = u / UR, grp = u % UR * VW / 4;
            x[j] = *reinterpret_cast<const unit_t*>(p + 4 * VW * u);
            d[j] = val ? c.v_scale[at * G + grp * c.bt + in + row] : c.k_scale[(at + in + row) * G + grp];
        }
    }
    static __device__ __forceinline__ int place(bool val, int j, int w, int lane) {
        const int u = lane + 64 * j, row = 16 * w + u / UR, chunk8 = VW * (u % UR);
        return row * 2 * D + 16 * (chunk8 ^ (val ? v4swz<D>(row) : kswz<D>(row)));
    }
    // eight elements of the thread's D / 4 as halves; chunks further on are one exclusive or away
    __device__ __forceinline__ void store(bool val, void* tile, const int* places, int i) const {
        const int j = i / VW, e = i % VW;
        // (values of no scale: their token's scores are NaN or hidden)
        const _Float16 s = __builtin_bit_cast(_Float16, val ? (uint16_t)finite_scales(d[j]) : d[j]);
        uint32_t o[4];
        word_halves(x[j][e], h2v{s, s}, o);
        *reinterpret_cast<u32x4*>(static_cast<char*>(tile) + (places[j] ^ (16 * e))) = u32x4{o[0], o[1], o[2], o[3]};
    }
};

// Tiles of 64 tokens as halves, keys then values, in memory as they will lie in LDS: where many row tiles read
// them, the conversion is done once.  A workgroup a tile.
template <int D>
__global__ __launch_bounds__(256) void kv4_halves_kernel(const Kv4AttnArgs a, char* tiles, const int max_tiles) {
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hk = blockIdx.y, s = blockIdx.z;
    const KvRange kr = kv_range<KV4_TILE>(a, s);
    const int t = kr.lo + KV4_TILE * blockIdx.x + 16 * w;
    if (kr.lo + KV4_TILE * (int)blockIdx.x >= kr.hi || kr.nq == 0) return;
    const int id = max(kv4_block(c, s, t), 0), in = t & (c.bt - 1);  // (what is not there or not yet is hidden later)
    const int64_t at = ((int64_t)id * c.heads + hk) * c.bt;
    char* out = tiles + (((int64_t)s * c.heads + hk) * max_tiles + blockIdx.x) * (KV4_TILE * D * 4);
    TileWords<D> z[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) z[v].load(c, v, at, in, lane);
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        int places[TileWords<D>::NV];
#pragma unroll
        for (int j = 0; j < TileWords<D>::NV; ++j) places[j] = TileWords<D>::place(v, j, w, lane);
#pragma unroll
        for (int i = 0; i < TileWords<D>::NW; ++i) z[v].store(v, out + v * (KV4_TILE * D * 2), places, i);
    }
}

// PRE: the tiles are kv4_halves_kernel's, and go to LDS past the registers.
template <int D, bool QS, bool PS, bool PRE>
__global__ __launch_bounds__(256, 2) void kv4_tiles_kernel(const Kv4AttnArgs a, const int splits, const int tiles, const char* halves, const int max_tiles) {
    constexpr int NC = D / 16, NDB = D / 32;        // score products, output blocks
    constexpr bool AHEAD = !((QS && D > 64) || (PS && D > 96));  // scores a tile ahead; else the second halves have their registers
    constexpr int NW = TileWords<D>::NW, NV = TileWords<D>::NV;
    __shared__ __attribute__((aligned(16))) _Float16 sK[2][64 * D];
    __shared__ __attribute__((aligned(16))) _Float16 sV[2][64 * D];
    const Kv4View& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Eight items (one to an XCD, whose bytes stay in its L2) at a time, and of them the last row tiles
    // first: causal ones are the longest.
    const int items = splits * c.heads * c.n_seq, first = blockIdx.x / (8 * tiles) * 8, left = blockIdx.x - first * tiles;
    const int many = min(8, items - first), item = first + left % many, tile = tiles - 1 - left / many;
    const int sp = item % splits, hk = item / splits % c.heads, s = item / splits / c.heads;
    const KvRange kr = kv_range<KV4_TILE>(a, s);
    const int rows = kr.nq * a.group, row0 = tile * 128;
    if (row0 >= rows) return;
    const int chunk = kv_chunk(kr, splits);
    if (sp > 0 && kr.lo + sp * chunk >= kr.hi) return;
    const int iq_first = row0 / a.group, iq_last = (min(row0 + 128, rows) - 1) / a.group;
    const int lo_tile = a.window > 0 ? max(kr.pos0 + iq_first - a.window + 1, 0) & ~63 : 0;
    const int tb = max(kr.lo + sp * chunk, lo_tile);  // (a multiple of 64)
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
        const char* p = row_at(a, s, iq, h);
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
    const float f = score_factor(a.scale, qscale);

    int tile0 = 0;  // the step's tile
    // blocks of 16 tokens each, of the sixteen tiles that the step's tile is of, and of the sixteen after
    int cur = -1, nxt = -1;
    auto group_of = [&](int t) { return kv4_block(c, s, tb + 64 * t + 16 * lane); };
    auto staged = [&](int t) {  // block of this wavefront's 16 rows of a tile of this or the next sixteen
        const int i = 4 * (t & 15) + w;
        return max((t >> 4) == (tile0 >> 4) ? __builtin_amdgcn_readlane(cur, i) : __builtin_amdgcn_readlane(nxt, i), 0);
    };
    TileWords<D> kreg, vreg;
    auto load_one = [&](bool val, TileWords<D>& z, int t) {
        z.load(c, val, ((int64_t)staged(t) * c.heads + hk) * c.bt, (tb + 64 * t + 16 * w) & (c.bt - 1), lane);
    };
    int kst[NV], vst[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        kst[j] = TileWords<D>::place(false, j, w, lane);
        vst[j] = TileWords<D>::place(true, j, w, lane);
    }
    auto store_one = [&](bool val, _Float16* lds, const TileWords<D>& z) {
#pragma unroll
        for (int i = 0; i < NW; ++i) z.store(val, lds, val ? vst : kst, i);
    };
    // PRE: a wavefront's quarter of a tile's keys or values, 1 KiB at a time
    v4i rsrc;
    if constexpr (PRE) rsrc = make_rsrc(halves + (((int64_t)s * c.heads + hk) * max_tiles + (tb - kr.lo) / 64) * (256 * D), (int64_t)((te - tb + 63) / 64) * (256 * D));
    auto dma = [&](bool val, _Float16* lds, int t) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int at = 1024 * (w * (D / 32) + i);
            dma_b128_so(rsrc, (uint32_t)__builtin_amdgcn_readfirstlane(lds_addr(lds) + at), 16 * lane, t * (256 * D) + (val ? 128 * D : 0) + at);
        }
    };
    const int krow = lr * 2 * D, kchunk = 16 * (g ^ kswz<D>(lr));
    auto key_frag = [&](const _Float16* lds, int pre, int m, int kh) {
        const int at = D == 96 ? krow + (pre ^ (32 * m)) : pre ^ (32 * m);
        return *reinterpret_cast<const v8h*>(reinterpret_cast<const char*>(lds) + at + kh * 64 * D);
    };
    const int kpre = D == 96 ? kchunk : krow + kchunk;
    const int vrow = 4 * g + ((lane & 15) >> 2), vpre = vrow * 2 * D + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v4swz<D>(vrow)) + 8 * (lane & 1);

    v16f O[NDB];
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[i][e] = 0.0f;
    float m_ref = KV4_NONE, l_sum = 0.0f, l_all = 0.0f;
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
    // The token of score i of group j from the lane's first one of the tile.
    auto token = [](int j, int i) { return 32 * (j >> 1) + 16 * (j & 1) + 8 * (i >> 2) + (i & 3); };
    // Probabilities of a tile from its scores, at the reference as it stands: pair n of its sixteen
    uint32_t P[2][8], PL[2][PS ? 8 : 1];
    struct Sums {
        float s, all;
    };
    auto pair = [&](const v16f* S, int n, Sums& sums) {
        const v16f& x = S[n >> 3];
        const int i = 2 * (n & 7);
        const v2f p = {__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], f, -m_ref)), __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], f, -m_ref))};
        const h2v ph = __builtin_convertvector(p, h2v), ones = {(_Float16)1.0f, (_Float16)1.0f};
        P[n >> 3][n & 7] = __builtin_bit_cast(uint32_t, ph);
        if constexpr (PS) {
            const h2v pl = __builtin_convertvector((v2f{p[0] - (float)ph[0], p[1] - (float)ph[1]}), h2v);
            PL[n >> 3][n & 7] = __builtin_bit_cast(uint32_t, pl);
            sums.s += p[0] + p[1];
        } else {
            sums.s = __builtin_amdgcn_fdot2(ph, ones, sums.s, false);
            if (a.lse) sums.all += p[0] + p[1];
        }
    };
    // What is left when the pairs of half a tile are done: the sums, and the reference where it has to move.
    auto settle = [&](const v16f* S, int kh, Sums& sums) {
        if (__builtin_amdgcn_ballot_w64(!(sums.s <= 32768.0f))) {
            // some probability is too large, or may be: the reference moves to the half's own largest
            float top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, S[kh][i] * f);
            const float mn = fmaxf(m_ref, xmax32(top) - KV4_LIFT_SUM), am = __builtin_amdgcn_exp2f(m_ref - mn);
            m_ref = mn;
            l_sum *= am;
            l_all *= am;
#pragma unroll
            for (int b = 0; b < NDB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) O[b][e] *= am;
            sums = Sums{0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < 8; ++n) pair(S, 8 * kh + n, sums);
        }
        l_sum += sums.s;
        l_all += sums.all;
    };
    // The scores Sn of the tile in lds beside the first half's probabilities of the tile before it, whose scores S are there:
    // a product's fragments are read while the product before multiplies, and pairs go between the products.
    auto score_softmax = [&](const _Float16* lds, v16f* Sn, const v16f* S) {
        int pre = kpre;
        asm volatile("" : "+v"(pre));  // (the addresses are made here: kept over the loop, they would push the queries out)
        const v16f z = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        v8h k8[2], k8n[2];
        auto frag = [&](int m, v8h* o) {
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) o[kh] = key_frag(lds, pre, m, kh);
        };
        if constexpr (QS) __builtin_amdgcn_s_setprio(1);
        frag(0, k8);
        Sn[0] = Sn[1] = z;
        Sums sums = {0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < NC; ++m) {
            if (m + 1 < NC) frag(m + 1, k8n);
#pragma unroll
            for (int kh = 0; kh < 2; ++kh) {
                Sn[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[kh], q[m], Sn[kh], 0, 0, 0);
                if constexpr (QS) Sn[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[kh], ql[m], Sn[kh], 0, 0, 0);
            }
#pragma unroll
            for (int n = 8 * m / NC; n < 8 * (m + 1) / NC; ++n) pair(S, n, sums);
            k8[0] = k8n[0];
            k8[1] = k8n[1];
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (QS) __builtin_amdgcn_s_setprio(0);
        settle(S, 0, sums);
    };
    // Scores of blocks that are not there are hidden, and so are those that a row does not see, before anything
    // is made of them.
    uint64_t off = 0;  // of the groups of cur
    auto hide = [&](v16f* S, int t) {
        const int t0 = tb + 64 * t + 4 * g, shift = 4 * (t & 15);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t n = off >> (shift + j) & 1 ? 0u : (uint32_t)max(see_hi - see_lo, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = S[j >> 1][8 * (j & 1) + i];
                S[j >> 1][8 * (j & 1) + i] = (uint32_t)(token(j, i) + t0 - see_lo) < n ? x : -__builtin_inff();
            }
        }
    };
    // The output of the tile in lds, and between the products of its first half the second one's probabilities, between
    // those of the second one the staged words of the next tiles into their buffers
    auto output_store = [&](const v16f* S, const _Float16* lds, _Float16* vnext, _Float16* knext) {
        int pre = vpre;
        asm volatile("" : "+v"(pre));
        auto frag = [&](int i) {  // product i: 16 tokens i / NDB, output block i % NDB
            const int b = i % NDB;
            const char* vt = reinterpret_cast<const char*>(lds) + (D == 96 ? pre + 64 * b : pre ^ (64 * b)) + 16 * (i / NDB) * 2 * D;
            const uint2 lo = lds_read_tr16(vt), hi = lds_read_tr16(vt + 8 * 2 * D);
            return __builtin_bit_cast(v8h, (u32x4{lo.x, lo.y, hi.x, hi.y}));
        };
        v8h v8[2] = {frag(0), frag(1)}, v8n[2];
        static_assert(NDB == NW, "a unit of both to two products");
        Sums sums = {0.0f, 0.0f};
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
            if (x < NDB) {
#pragma unroll
                for (int n = 8 * x / NDB; n < 8 * (x + 1) / NDB; ++n) pair(S, 8 + n, sums);
                if (x == NDB - 1) settle(S, 1, sums);
            } else if constexpr (!PRE) {
                vreg.store(true, vnext, vst, x - NDB);
                kreg.store(false, knext, kst, x - NDB);
            }
            v8[0] = v8n[0];
            v8[1] = v8n[1];
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    const int nt = te > tb ? (te - tb + 63) / 64 : 0;
    if (nt > 0) {
        // Step t: the scores of tile t + 1 beside the softmax of tile t (AHEAD; else its own before it), and its
        // output; then the words of K(t + 2) (t + 1) and V(t + 1), loaded a step before, become halves in the buffers
        // that step t - 1 read last.  One barrier a step.
        cur = group_of(0);
        nxt = group_of(16);
        off = __builtin_amdgcn_ballot_w64(cur < 0);
        v16f SA[2], SB[2];
        if constexpr (PRE) {
            dma(false, sK[0], 0);
            dma(true, sV[0], 0);
            if (AHEAD && nt > 1) dma(false, sK[1], 1);
            if (AHEAD) {  // (the others' are waited for at the first step)
                if (nt > 1) wait_vmcnt<D / 16>();
                else wait_vmcnt<D / 32>();
                lds_barrier();
            }
        } else {
            load_one(false, kreg, 0);
            store_one(false, sK[0], kreg);
            load_one(true, vreg, 0);
            store_one(true, sV[0], vreg);
            load_one(false, kreg, 1);
            if constexpr (AHEAD) {
                store_one(false, sK[1], kreg);
                load_one(false, kreg, 2);
            }
            load_one(true, vreg, 1);
            __syncthreads();
        }
        if constexpr (AHEAD) score(sK[0], SA);
        auto step = [&](int t, int cb, v16f* Sc, v16f* Sn) {
            const int t0 = tb + 64 * t;
            if constexpr (PRE) wait_vmcnt<0>();
            lds_barrier();
            if constexpr (PRE) {  // into the buffers that step t - 1 read last
                if (t + 1 < nt) dma(true, sV[cb ^ 1], t + 1);
                if (AHEAD ? t + 2 < nt : t + 1 < nt) dma(false, sK[AHEAD ? cb : cb ^ 1], t + (AHEAD ? 2 : 1));
            }
            tile0 = t;
            if ((t & 15) == 0 && t > 0) {
                cur = nxt;
                off = __builtin_amdgcn_ballot_w64(cur < 0);
                nxt = group_of(t + 16);
            }
            if constexpr (!AHEAD) score(sK[cb], Sc);
            if (t0 < all_lo || t0 + 64 > all_hi || ((off >> (4 * (t & 15))) & 15)) hide(Sc, t);
            if constexpr (AHEAD) {
                score_softmax(sK[cb ^ 1], Sn, Sc);
            } else {
                Sums sums = {0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < 8; ++n) pair(Sc, n, sums);
                settle(Sc, 0, sums);
            }
            output_store(Sc, sV[cb], sV[cb ^ 1], sK[AHEAD ? cb : cb ^ 1]);
            if constexpr (!PRE) {
                load_one(true, vreg, t + 2);
                load_one(false, kreg, t + (AHEAD ? 3 : 2));
            }
        };
        for (int t = 0; t < nt; t += 2) {
            step(t, 0, SA, AHEAD ? SB : SA);
            if (t + 1 < nt) step(t + 1, 1, AHEAD ? SB : SA, SA);
        }
    }

    if (!on) return;
    l_sum = xsum32(l_sum);
    l_all = PS ? l_sum : xsum32(l_all);
    const int64_t pr = ((int64_t)s * a.n_q + iq) * a.heads + h, all = (int64_t)c.n_seq * a.n_q * a.heads;
    const float z = splits > 1 ? 1.0f : l_sum == 0.0f ? 0.0f : 1.0f / l_sum;
    if (g == 0) {
        if (splits > 1) *reinterpret_cast<v4f*>(a.part + (int64_t)splits * all * D + (sp * all + pr) * 4) = v4f{m_ref, l_sum, l_all, 0.0f};
        else put_lse(a, pr, m_ref, l_all);
    }
    float* part = a.part + (sp * all + pr) * D;
    char* out = out_at(a, pr);
#pragma unroll
    for (int b = 0; b < NDB; ++b)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            const int e = 32 * b + 8 * i4 + 4 * g;
            const v4f y = v4f{O[b][4 * i4], O[b][4 * i4 + 1], O[b][4 * i4 + 2], O[b][4 * i4 + 3]} * z;
            if (splits > 1) *reinterpret_cast<v4f*>(part + e) = y;
            else put_four(a, out, e, y);
        }
}

// The joins of kv4_tiles_kernel's ranges: thread per four elements of a row
template <int D>
__global__ __launch_bounds__(256) void kv4_join_kernel(const Kv4AttnArgs a, const int splits) {
    constexpr int C4 = D / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, pr = i / C4, all = (int64_t)a.c.n_seq * a.n_q * a.heads;
    if (pr >= all) return;
    const KvRange kr = kv_range<KV4_TILE>(a, (int)(pr / a.heads / a.n_q));
    if (pr / a.heads % a.n_q >= kr.nq) return;
    const int chunk = kv_chunk(kr, splits);
    join_ranges<D, false>(a, splits, max((kr.hi - kr.lo + chunk - 1) / chunk, 1), pr, (int)(i - pr * C4) * 4);
}

// ---- the weights' sums by token
// S[row][token] = Q K^T gives a lane some rows of one token, whose sum it keeps.  exp(scale q . k - lse) is taken of the
// difference, so that the largest weights, which have the smallest ones, lose least: an error of log2(e) acts on it alone.

// Up to 16 rows: a wavefront keeps their queries and walks over the tokens, every fourth 32 of its workgroup's range, the
// next ones' keys and sums asked for a step ahead.  Bound by memory: 32 sequences of 16384 tokens, 8 key heads of 128, 254 MB in
// 57 us (4.5 TB/s).
template <int D, bool QS>
__global__ __launch_bounds__(256, 4) void kv4_weights_rows_kernel(const Kv4AttnArgs a, float* sums, const int splits) {
    constexpr int KM = D / 32;
    const Kv4View& c = a.c;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int item = blockIdx.x / splits, sp = blockIdx.x % splits, hk = item % c.heads, s = item / c.heads;
    const KvRange kr = kv_range<KV4_TILE>(a, s);
    const int rows = kr.nq * a.group, chunk = kv_chunk(kr, splits), tb = kr.lo + sp * chunk, te = min(tb + chunk, kr.hi);
    if (rows == 0 || tb >= te) return;
    Row<D, QS> row;
    const int iq = col / a.group, h = hk * a.group + (col - iq * a.group);
    const bool on = col < rows;
    row.load(row_at(a, s, iq, h), on, g);
    const float lse = on ? a.lse[((int64_t)s * a.n_q + iq) * a.heads + h] : 0.0f;
    float l[4], f[4];
    int lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int y = 4 * g + i, pos = kr.pos0 + y / a.group;
        l[i] = __shfl(lse, y, 64);
        f[i] = QS ? a.scale * __shfl(row.up, y, 64) : a.scale;
        hi[i] = y < rows ? (a.causal ? min(pos + 1, kr.hi) : kr.hi) : 0;
        lo[i] = a.window > 0 ? pos - a.window + 1 : 0;
    }
    float* out = sums + ((int64_t)s * c.heads + hk) * c.max_blocks * c.bt;
    int ids = -1, at = 32;
    struct Step {
        bool there[2];
        float old[2];
    };
    Keys<D> key[2];
    auto ask = [&](int t0) {
        Step x;
        if (at == 32) {  // lane 2 i + u: the block of half u of this wavefront's i-th step from here
            ids = kv4_block(c, s, t0 + (lane >> 1) * KV_SPAN + 16 * (lane & 1));
            at = 0;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int id = __builtin_amdgcn_readlane(ids, 2 * at + u), t = t0 + 16 * u;
            x.there[u] = id >= 0;
            const int64_t tok = ((int64_t)max(id, 0) * c.heads + hk) * c.bt + (t & (c.bt - 1));
            key[u].load(c.k + tok * (D / 2), c.k_scale + tok * KM, col, g);
            x.old[u] = t + col < te ? out[t + col] : 0.0f;
        }
        ++at;
        return x;
    };
    Step next{};
    if (tb + w * KV_STEP < te) next = ask(tb + w * KV_STEP);
    for (int t0 = tb + w * KV_STEP; t0 < te; t0 += KV_SPAN) {
        const Step x0 = next;
        v4f S[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            S[u] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < KM; ++m) {
                const v8h k8 = key[u].halves(m);
                S[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(row.q[m], k8, S[u], 0, 0, 0);
                if constexpr (QS) S[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(row.ql[m], k8, S[u], 0, 0, 0);
            }
        }
        if (t0 + KV_SPAN < te) next = ask(t0 + KV_SPAN);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int t = t0 + 16 * u + col;
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(S[u][i], f[i], -l[i]) * KV4_LOG2E);
                p[i] = t >= lo[i] && t < hi[i] ? e : 0.0f;
            }
            const float sum = col_sum((p[0] + p[1]) + (p[2] + p[3]));
            if (g == 0 && x0.there[u] && t < te) out[t] = x0.old[u] + sum;
        }
    }
}

// More rows: a workgroup takes 256 tokens, 64 to a wavefront as halves in registers, and a range of the rows, which pass
// through LDS 32 at a time (an F32 row as two halves, times a power of two).  A lane sums a tile's sixteen rows of a token in a
// tree, 32 tiles one after another and then those, for 32 bits to hold them.  A range's sums go to part, or are added at once
// where there is one range.  Bound by the VALU's work of a weight (difference, product, exponential, sum): 2 x 2048 causal F16
// queries over 4099, 32 heads of 128 over 8, 79 GFLOP in 124 us (139 with equal ranges, chunk by chunk, the product with log2(e) of
// each difference, and each row's place by a division); VALU busy 53 % of the time, matrix pipe 28 %, LDS 20 %, up to three wavefronts a SIMD.  The next
// tile's scores between this one's weights leave two of them and took 1.13 times as long, 32 tokens to a wavefront and four of
// them 1.12 times, rows loaded two tiles ahead the same.
template <int D, bool QS>
__global__ __launch_bounds__(256, 2) void kv4_weights_tiles_kernel(const Kv4AttnArgs a, float* sums, const int splits, const int chunks) {
    constexpr int NC = D / 16, NP = D / 32;  // products, pieces of four elements of a thread
    const Kv4View& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, g = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // a sequence and key head on one XCD: all chunks of its first rows, then of the next ones
    const int per = 8 * chunks * splits, gb = blockIdx.x / per, rb = blockIdx.x % per;
    const int item = gb * 8 + (rb & 7), sp = (rb >> 3) / chunks, x = (rb >> 3) % chunks;
    if (item >= c.heads * c.n_seq) return;
    const int hk = item % c.heads, s = item / c.heads;
    const KvRange kr = kv_range<KV4_TILE>(a, s);
    const int wg0 = kr.lo + 256 * x, t0 = wg0 + 64 * w;
    if (wg0 >= kr.hi) return;
    const int64_t room = (int64_t)c.max_blocks * c.bt;
    // rows of this range that see one of these tokens.  The first ranges are three times as long as the last ones, which end the
    // launch together.
    const int rows = kr.nq * a.group, all = (rows + 31) / 32;
    auto begin = [&](int i) { return (int)((int64_t)all * i * (3 * splits - i) / (2 * (int64_t)splits * splits)) * 32; };
    const int q_lo = a.causal ? max(wg0 - kr.pos0, 0) : 0;
    const int q_hi = a.window > 0 ? (int)max(min((int64_t)kr.nq, (int64_t)wg0 + 255 + a.window - kr.pos0), (int64_t)0) : kr.nq;
    const int r_lo = (int)max((int64_t)begin(sp), (int64_t)q_lo * a.group) & ~31, r_hi = (int)min(min((int64_t)begin(sp + 1), (int64_t)rows), (int64_t)q_hi * a.group);

    v8h k8[2][NC];
    bool there[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        // a lane's token, half g of its row's words one after another (the queries' chunks follow that order)
        const int t = t0 + 32 * b + lr, id = kv4_block(c, s, t);
#pragma unroll
        for (int u = 0; u < 2; ++u) there[b][u] = __builtin_amdgcn_readlane(id, 16 * u) >= 0;
        const int64_t tok = ((int64_t)max(id, 0) * c.heads + hk) * c.bt + (t & (c.bt - 1));
        const uint8_t* row = c.k + tok * (D / 2) + 4 * NC * g;
        const uint16_t* scale = c.k_scale + tok * (D / 32);
        uint32_t words[NC];
#pragma unroll
        for (int m = 0; m < NC; m += 2) {  // (a row starts on 16 bytes, its half on 8)
            const u32x2 x = *reinterpret_cast<const u32x2*>(row + 4 * m);
            words[m] = x[0];
            words[m + 1] = x[1];
        }
#pragma unroll
        for (int m = 0; m < NC; ++m) {
            const _Float16 d = __builtin_bit_cast(_Float16, scale[(NC * g + m) >> 2]);
            uint32_t o[4];
            word_halves(words[m], h2v{d, d}, o);
            k8[b][m] = __builtin_bit_cast(v8h, u32x4{o[0], o[1], o[2], o[3]});
        }
    }

    __shared__ __attribute__((aligned(16))) _Float16 sQ[2][QS ? 2 : 1][32 * D];
    __shared__ __attribute__((aligned(16))) float sL[2][32], sF[2][32];
    __shared__ __attribute__((aligned(16))) int sHi[2][32], sLo[2][32];
    // staging: eight threads to a row
    const int sr = tid >> 3, part = tid & 7;
    struct Staged {
        float q[QS ? 4 * NP : 1], lse;
        v4h h[QS ? 1 : NP];
        int pos;
    };
    // the thread's row of the next tile, 32 rows at a time: its query, head of the group, place in q and in lse
    const int step_q = 32 / a.group, step_h = 32 - step_q * a.group;
    int r = r_lo + sr, iq = r / a.group, hg = r - iq * a.group;
    const char* q_row = row_at(a, s, iq, hk * a.group + hg) + part * (D / 8) * (QS ? 4 : 2);
    const float* lse_row = a.lse + ((int64_t)s * a.n_q + iq) * a.heads + hk * a.group + hg;
    auto load = [&]() {
        Staged z;
        const bool on = r < r_hi;
        const char* p = q_row;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            if constexpr (QS) {
                const v4f y = on ? *reinterpret_cast<const v4f_a4*>(p + 16 * j) : v4f{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) z.q[4 * j + i] = y[i];
            } else {
                z.h[j] = on ? *reinterpret_cast<const v4h_a2*>(p + 8 * j) : v4h{0, 0, 0, 0};
            }
        }
        z.lse = on && part == 0 ? *lse_row : 0.0f;
        z.pos = on ? kr.pos0 + iq : INT32_MIN;
        r += 32;
        iq += step_q;
        hg += step_h;
        q_row += step_q * a.q_nb[0] + step_h * a.q_nb[1];
        lse_row += (int64_t)step_q * a.heads + step_h;
        if (hg >= a.group) {
            hg -= a.group;
            ++iq;
            q_row += a.q_nb[0] - a.group * a.q_nb[1];
            lse_row += a.heads - a.group;
        }
        return z;
    };
    // In base 2: scale log2(e) is off by its rounding, and lse takes the same error, so that it acts on their difference alone.
    // Both of the scale's mantissa, whatever its size; its exponent joins the row's power of two.
    int scale_e;
    const float scale_m = frexpf(a.scale, &scale_e), f1 = scale_m * KV4_LOG2E, ratio = scale_m != 0.0f ? f1 / scale_m : KV4_LOG2E;
    auto factor = [&](float up) { return fmaxf(fminf(f1 * ldexpf(up, scale_e), 3e38f), -3e38f); };  // (times a product of zero)
    const float f2 = factor(1.0f);
    auto store = [&](const Staged& z, int buf) {
        float up = 1.0f, down = 1.0f;
        if constexpr (QS) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 4 * NP; ++j) top = fmaxf(top, fabsf(z.q[j]));
            const Pow2 y = pow2_of(group_max<8>(top));
            up = y.up;
            down = y.down;
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int e = part * (D / 8) + 4 * j, at = sr * D + 8 * ((e >> 3) ^ kswz<D>(sr)) + (e & 4);
            if constexpr (QS) {
                v4h hi, lo;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = z.q[4 * j + i] * down;
                    hi[i] = (_Float16)y;
                    lo[i] = (_Float16)(y - (float)hi[i]);
                }
                *reinterpret_cast<v4h*>(&sQ[buf][0][at]) = hi;
                *reinterpret_cast<v4h*>(&sQ[buf][1][at]) = lo;
            } else {
                *reinterpret_cast<v4h*>(&sQ[buf][0][at]) = z.h[j];
            }
        }
        if (part == 0) {
            const bool on = z.pos != INT32_MIN;
            sL[buf][sr] = z.lse * ratio;
            sF[buf][sr] = factor(up);
            sHi[buf][sr] = on ? (a.causal ? min(z.pos + 1, kr.hi) : kr.hi) : 0;
            sLo[buf][sr] = on && a.window > 0 ? z.pos - a.window + 1 : 0;
        }
    };
    float total[2] = {0, 0}, some[2] = {0, 0};
    const bool all_there = there[0][0] && there[0][1] && there[1][0] && there[1][1];
    if (r_lo < r_hi) {
        store(load(), 0);
        __syncthreads();
        int n = 0, buf = 0;
        for (int row0 = r_lo; row0 < r_hi; row0 += 32, buf ^= 1) {
            Staged z;
            if (row0 + 32 < r_hi) z = load();
            v16f S[2];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) S[b][i] = 0.0f;
#pragma unroll
            for (int m = 0; m < NC; ++m) {
                const int at = lr * D + 8 * ((NC * g + m) ^ kswz<D>(lr));
                const v8h q = *reinterpret_cast<const v8h*>(&sQ[buf][0][at]);
#pragma unroll
                for (int b = 0; b < 2; ++b) S[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q, k8[b][m], S[b], 0, 0, 0);
                if constexpr (QS) {
                    const v8h ql = *reinterpret_cast<const v8h*>(&sQ[buf][1][at]);
#pragma unroll
                    for (int b = 0; b < 2; ++b) S[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql, k8[b][m], S[b], 0, 0, 0);
                }
            }
            // a lane's rows of the tile: 8 j + 4 g .. + 3
            float p[2][16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const v4f l = *reinterpret_cast<const v4f*>(&sL[buf][8 * j + 4 * g]);
                const v4f f = QS ? *reinterpret_cast<const v4f*>(&sF[buf][8 * j + 4 * g]) : v4f{f2, f2, f2, f2};
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[b][4 * j + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[b][4 * j + i], f[i], -l[i]));
            }
            // whether every row of the tile sees all of the wavefront's tokens
            const int first = kr.pos0 + row0 / a.group, last = kr.pos0 + (row0 + 31) / a.group;
            const bool full = all_there && row0 + 32 <= r_hi && t0 + 64 <= (a.causal ? min(first + 1, kr.hi) : kr.hi) && (a.window == 0 || t0 > last - a.window);
            if (!full) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    typedef int i4 __attribute__((ext_vector_type(4)));
                    const i4 hi = *reinterpret_cast<const i4*>(&sHi[buf][8 * j + 4 * g]), lo = *reinterpret_cast<const i4*>(&sLo[buf][8 * j + 4 * g]);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int t = t0 + 32 * b + lr;
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[b][4 * j + i] = t >= lo[i] && t < hi[i] ? p[b][4 * j + i] : 0.0f;
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < o; ++i) p[b][i] += p[b][i + o];
                some[b] += p[b][0];
            }
            if (++n == 32) {
                n = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) total[b] += some[b], some[b] = 0.0f;
            }
            if (row0 + 32 < r_hi) store(z, buf ^ 1);
            __syncthreads();
        }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float y = xsum32(total[b] + some[b]);
        const int t = t0 + 32 * b + lr;
        if (g == 0 && (lr < 16 ? there[b][0] : there[b][1]) && t < kr.hi) {
            if (splits > 1) a.part[((int64_t)sp * c.heads * c.n_seq + item) * chunks * 256 + (t - kr.lo)] = y;
            else sums[(int64_t)item * room + t] += y;
        }
    }
}

// sums += the ranges' parts, in their order
__global__ __launch_bounds__(256) void kv4_weights_join_kernel(const Kv4AttnArgs a, float* sums, const int splits) {
    const Kv4View& c = a.c;
    const int hk = blockIdx.y, s = blockIdx.z, item = s * c.heads + hk;
    const KvRange kr = kv_range<KV4_TILE>(a, s);
    const int t = kr.lo + blockIdx.x * 256 + threadIdx.x;
    if (kr.nq == 0 || t >= kr.hi || kv4_block(c, s, t) < 0) return;
    const int64_t span = (int64_t)gridDim.x * 256, at = (int64_t)item * span + (t - kr.lo);  // (of the tokens that are seen)
    float x = 0.0f;
    for (int i = 0; i < splits; ++i) x += a.part[(int64_t)i * c.heads * c.n_seq * span + at];
    sums[(int64_t)item * c.max_blocks * c.bt + t] += x;
}

// The kernel, its row tiles and the ranges of the tokens for n_q queries: of 16 rows, of 128, and of 128 with the tokens'
// halves made before, each at its best number of ranges, the cheapest by the rounds of workgroups over the CUs.  A step of
// 128 tokens takes a workgroup so long, in microseconds, with one, two .. workgroups on its CU (heads of 128 and 64, of 96
// between them; F32 queries); where one row tile reads a sequence's tokens alone, its share of the memory at least.  Then the
// partial sums, which a last workgroup joins past the caches or a second launch does, and the halves' launch.
// One token of 32 sequences over 16384, 32 heads of 128 over 8: four ranges 104 us, two 117, eight 106; of one sequence
// (26 by these steps): 24 ranges 16.1 us, 16 16.5, 8 22.9.  80 rows of 32 sequences and 4 heads of 3000 tokens: 16 rows 47, 128 41, with halves 90;
// 126 rows of 16 heads of 2424: 14.5, 18.2, 31; 1024 rows of 64 heads of 2048: 103, 77, 86; 5184 F16 rows of 8 heads of 64 over
// 15552: 443, 256, 215 (245 to 285 with inputs rotated).
Kv4AttnPlan kv4_attn_plan(int n_q, int heads, int heads_kv, int n_seq, int64_t max_tokens, int window, int D, bool q16, int cus) {
    if (window > 0) max_tokens = std::min<int64_t>(max_tokens, (int64_t)window + n_q + KV_STEP);  // (kv_range)
    const int64_t rows = (int64_t)n_q * (heads / heads_kv), items = std::max<int64_t>((int64_t)heads_kv * n_seq, 1);
    const int64_t steps = std::max<int64_t>((max_tokens + KV_SPAN - 1) / KV_SPAN, 1);  // of 128 tokens
    cus = std::max(cus, 1);
    Kv4AttnPlan p;
    p.max_tiles = (int)((max_tokens + KV4_TILE - 1) / KV4_TILE) + (window > 0);
    const double pre = (double)items * p.max_tiles * (KV4_TILE * D * 4), values = (double)rows * items * D;
    static const float us[3][2][2][4] = {
        // 16 rows                                             128 rows                                     with halves
        {{{1.35f, 1.75f, 2.1f, 2.4f}, {1.0f, 1.2f, 1.45f, 1.7f}}, {{1.5f, 1.95f, 2.35f, 2.35f}, {1.1f, 1.3f, 1.6f, 1.9f}}},
        {{{3.05f, 5.0f}, {2.45f, 3.9f}}, {{3.8f, 7.0f}, {2.6f, 4.6f}}},
        {{{2.45f, 4.2f}, {1.75f, 2.2f, 3.4f}}, {{3.4f, 6.0f}, {2.0f, 3.4f}}}};
    double best = 1e300;
    for (int kind = 0; kind < 3; ++kind) {
        if ((kind > 0 && rows <= 16) || (kind == 2 && (pre > (double)(1 << 30) || max_tokens <= 0))) break;  // (a table without blocks has no halves)
        const float *wide = us[kind][q16 ? 0 : 1][0], *narrow = us[kind][q16 ? 0 : 1][1];
        const int64_t row = kind ? 128 : 16, tiles = (rows + row - 1) / row;
        const int cap = kind == 0 ? (q16 || D == 64 ? 4 : 3) : kind == 2 && q16 && D == 64 ? 3 : 2;  // workgroups of a CU
        for (int s = 1; s <= std::min<int64_t>(steps, kind ? 32 : KV4_RANGES); ++s) {
            if (kind == 0 && s > 1 && items * tiles > KV_ARRIVALS) break;
            const double per = (double)((steps + s - 1) / s), mem = tiles == 1 ? D / 128.0 : 0.0;
            auto step = [&](int load) {
                const int i = load - 1;
                const double t = D == 128 ? wide[i] : D == 64 ? narrow[i] : 0.5 * (wide[std::min(i, 1)] + narrow[std::min(i, 1)]) * (i > 1 ? wide[i] / wide[1] : 1.0);
                return per * std::max(t, mem * (0.12 + 0.78 * load));
            };
            const int64_t n = tiles * (kind ? items * s : (items * s + 7) / 8 * 8), full = (int64_t)cap * cus, rest = n % full;
            double t = (double)(n / full) * step(cap) + (rest ? step((int)((rest + cus - 1) / cus)) : 0.0);
            if (s > 1) t += kind ? 4.0 + 1.2e-6 * s * values : 0.5 + 0.3 * s + 4e-6 * s * values;
            if (kind == 2) t += 4.0 + 1.3 * pre / 4.5e6;
            if (t < best) {
                best = t;
                p.rows = (int)row;
                p.splits = s;
                p.pre = kind == 2;
            }
        }
    }
    p.tiles = (int)((rows + p.rows - 1) / p.rows);
    p.halves = p.splits > 1 ? ((size_t)p.splits * n_seq * n_q * heads * (D + 4) * 4 + 255) / 256 * 256 : 0;
    p.bytes = p.halves + (p.pre ? (size_t)pre : 0);
    return p;
}

template <int D, bool QS, bool PS>
static void kv4_attn_go(const Kv4AttnArgs& a, const Kv4AttnPlan& p, hipStream_t st) {
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    if (p.rows == 16) kv4_rows_kernel<D, QS, PS><<<(unsigned)((items + 7) / 8 * 8 * p.tiles), 256, 0, st>>>(a, p.splits, p.tiles);
    else if (p.pre) kv4_tiles_kernel<D, QS, PS, true><<<(unsigned)(items * p.tiles), 256, 0, st>>>(a, p.splits, p.tiles, reinterpret_cast<char*>(a.part) + p.halves, p.max_tiles);
    else kv4_tiles_kernel<D, QS, PS, false><<<(unsigned)(items * p.tiles), 256, 0, st>>>(a, p.splits, p.tiles, nullptr, 0);
}

template <int D>
static hipError_t kv4_attn_d(const Kv4AttnArgs& a, const Kv4AttnPlan& p, hipStream_t st) {
    if (p.pre)
        kv4_halves_kernel<D><<<dim3((unsigned)p.max_tiles, (unsigned)a.c.heads, (unsigned)a.c.n_seq), 256, 0, st>>>(a, reinterpret_cast<char*>(a.part) + p.halves, p.max_tiles);
    if (a.q16 && a.d16) kv4_attn_go<D, false, false>(a, p, st);
    else if (a.q16) kv4_attn_go<D, false, true>(a, p, st);
    else if (a.d16) kv4_attn_go<D, true, false>(a, p, st);
    else kv4_attn_go<D, true, true>(a, p, st);
    if (p.rows != 16 && p.splits > 1) {
        const int64_t n = (int64_t)a.c.n_seq * a.n_q * a.heads * (D / 4);
        kv4_join_kernel<D><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a, p.splits);
    }
    return hipGetLastError();
}

hipError_t launch_kv4_attn(const Kv4AttnArgs& a, const Kv4AttnPlan& p, int D, hipStream_t st) {
    if ((int64_t)a.n_q * a.heads * a.c.n_seq <= 0) return hipSuccess;
    const int64_t items = (int64_t)p.splits * a.c.heads * a.c.n_seq;
    if ((items + 7) / 8 * 8 * p.tiles > KV4_GRID || (int64_t)a.n_q * a.heads * a.c.n_seq * (D / 4) > KV4_GRID * 256 ||
        (p.bytes && !a.part) || (p.splits > 1 && p.rows == 16 && !a.arrived))
        return hipErrorInvalidValue;
    switch (D) {
        case 64: return kv4_attn_d<64>(a, p, st);
        case 96: return kv4_attn_d<96>(a, p, st);
        case 128: return kv4_attn_d<128>(a, p, st);
        default: return hipErrorInvalidValue;
    }
}

// The sums' ranges.  Up to 16 rows of the tokens, to eight workgroups a CU: one token of 32 sequences over 16384, 8 key heads, 57 us
// with eight ranges, 73 with four, 60 with 32; of one sequence 6.0 us with 128, 11.4 with 16.  Beyond, of the rows, to twelve
// workgroups a CU and no fewer than 512 rows each: 2 x 2048 queries over 4099, 32 heads of 128 over 8, 124 us with
// twelve ranges, 1.2 times that with four, 2.4 with one; 64 rows of 64 heads over 2048 12.6 us with one, 20.2 with two.
Kv4WeightsPlan kv4_weights_plan(int n_q, int heads, int heads_kv, int n_seq, int64_t room, int window, int cus) {
    const int64_t tokens = window > 0 ? std::min<int64_t>(room, (int64_t)window + n_q + KV4_TILE) : room;
    const int64_t rows = (int64_t)n_q * (heads / heads_kv), items = std::max<int64_t>((int64_t)heads_kv * n_seq, 1);
    cus = std::max(cus, 1);
    Kv4WeightsPlan p;
    p.few = rows <= 16;
    p.chunks = (int)((tokens + 255) / 256);
    const int64_t have = p.few ? items : items * std::max(p.chunks, 1), most = p.few ? (tokens + KV_SPAN - 1) / KV_SPAN : rows / 512;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({((p.few ? 8 : 12) * (int64_t)cus + have - 1) / have, most, p.few ? 2048 : 32}));
    p.bytes = p.few || p.splits == 1 ? 0 : (size_t)p.splits * items * p.chunks * 1024;
    return p;
}

template <int D, bool QS>
static hipError_t kv4_weights_go(const Kv4AttnArgs& a, float* sums, const Kv4WeightsPlan& p, hipStream_t st) {
    const int64_t items = (int64_t)a.c.heads * a.c.n_seq, n = p.few ? items * p.splits : (items + 7) / 8 * 8 * p.chunks * p.splits;
    if (n > KV4_GRID) return hipErrorInvalidValue;
    if (p.few) kv4_weights_rows_kernel<D, QS><<<(unsigned)n, 256, 0, st>>>(a, sums, p.splits);
    else kv4_weights_tiles_kernel<D, QS><<<(unsigned)n, 256, 0, st>>>(a, sums, p.splits, p.chunks);
    if (!p.few && p.splits > 1)
        kv4_weights_join_kernel<<<dim3((unsigned)p.chunks, (unsigned)a.c.heads, (unsigned)a.c.n_seq), 256, 0, st>>>(a, sums, p.splits);
    return hipGetLastError();
}

hipError_t launch_kv4_weights(const Kv4AttnArgs& a, float* sums, const Kv4WeightsPlan& p, int D, hipStream_t st) {
    if ((int64_t)a.n_q * a.heads * a.c.n_seq <= 0 || a.c.max_blocks <= 0 || a.c.n_blocks <= 0) return hipSuccess;
    if (p.bytes && !a.part) return hipErrorInvalidValue;
    switch (D) {
        case 64: return a.q16 ? kv4_weights_go<64, false>(a, sums, p, st) : kv4_weights_go<64, true>(a, sums, p, st);
        case 96: return a.q16 ? kv4_weights_go<96, false>(a, sums, p, st) : kv4_weights_go<96, true>(a, sums, p, st);
        case 128: return a.q16 ? kv4_weights_go<128, false>(a, sums, p, st) : kv4_weights_go<128, true>(a, sums, p, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace mi355
