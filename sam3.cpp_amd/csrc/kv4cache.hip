// The 4-bit cache (kv4.cuh): written as tokens arrive, read back, and brought down to the tokens with the
// largest sums of softmax weights.
#include <algorithm>
#include <type_traits>

#include "attn.cuh"
#include "kv4.cuh"

namespace mi355 {

// -ext / 8 as the group's scale
__device__ __forceinline__ uint16_t kv4_scale(float hi, float lo) {
    const float ext = hi >= -lo ? hi : lo;
    uint32_t u = __float_as_uint(ext * -0.125f);
    u = (u + 0x7fffu + ((u >> 16) & 1)) & 0xffff0000u;  // eight significant bits, ties to even
    const float d = __uint_as_float(u);
    const uint16_t h = f2h(d);
    return !(fabsf(d) <= 8160.0f) ? KV4_NAN : h == 0x8000 ? (uint16_t)0 : h;  // (one zero, whatever the elements' signs)
}

// Eight elements, their largest and smallest, whether one is not a number, and their nibbles 8 + nearest_even(x / d) at
// a scale d and id = 1 / d (or both 0)
template <bool F16>
struct Eight4 {
    u32x4 raw[F16 ? 1 : 2];
    __device__ __forceinline__ void load(const char* p) {
        raw[0] = *reinterpret_cast<const u32x4_a2*>(p);
        if constexpr (!F16) raw[1] = *reinterpret_cast<const u32x4_a2*>(p + 16);
    }
    __device__ __forceinline__ void clear() {
        raw[0] = u32x4{0, 0, 0, 0};
        if constexpr (!F16) raw[1] = raw[0];
    }
    __device__ __forceinline__ h2v pair(int i) const {
        const uint32_t w = raw[0][i];
        return __builtin_bit_cast(h2v, w);
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (F16) {
            return (float)pair(i >> 1)[i & 1];
        } else {
            return __uint_as_float(raw[i >> 2][i & 3]);
        }
    }
    __device__ __forceinline__ void ends(float& hi, float& lo, bool& nan) const {
        if constexpr (F16) {
            h2v a = pair(0), b = a;
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const h2v x = pair(i);
                a = __builtin_elementwise_max(a, x);
                b = __builtin_elementwise_min(b, x);
                bad |= (raw[0][i] & 0x7fff7fffu) + 0x04000400u;  // (bit 15: infinite or no number)
            }
            hi = fmaxf((float)a[0], (float)a[1]);
            lo = fminf((float)b[0], (float)b[1]);
            nan = (bad & 0x80008000u) != 0;
        } else {
            hi = lo = (*this)[0];
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                hi = fmaxf(hi, (*this)[i]);
                lo = fminf(lo, (*this)[i]);
                z = __builtin_fmaf((*this)[i], 0.0f, z);
            }
            nan = z != z;
        }
    }
    __device__ __forceinline__ uint32_t word(float d, float id) const {
        float q[8];
        if constexpr (F16) {
            // An element has 11 bits and k + 1/2 steps have 12, so that a quotient is a tie or 2^-12 of it away from one: rounded to
            // 2^-14 by the sum with 768 ties are exact, whatever the reciprocal's rounding, and the others keep their side.
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = rintf(__builtin_fmaf((*this)[i], id, 768.0f) - 768.0f);
        } else {
            // The product with the reciprocal is within 2^-22 of the quotient: where one is near a tie, the remainder x - q d
            // decides, which is exact in one fma (q d has twelve bits, and x lies within a step of it).
            float near = 1.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = (*this)[i] * id;
                q[i] = rintf(y);
                near = fminf(near, 0.5f - fabsf(y - q[i]));
            }
            if (__builtin_amdgcn_ballot_w64(near < 1.52587890625e-5f)) {  // 2^-16
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float r = __builtin_fmaf(-q[i], d, (*this)[i]), half = 0.5f * fabsf(d);
                    if (fabsf(r) > half || (fabsf(r) == half && ((int)q[i] & 1))) q[i] += (r < 0.0f) == (d < 0.0f) ? 1.0f : -1.0f;
                }
            }
        }
        // four nibbles to a half of the word, as a number
        float h[2] = {34952.0f, 34952.0f};  // 8 (1 + 16 + 256 + 4096)
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i & 1] = __builtin_fmaf(__builtin_amdgcn_fmed3f(q[i], -8.0f, 7.0f), (float)(1 << (4 * (i >> 1))), h[i & 1]);
        return (uint32_t)h[0] | (uint32_t)h[1] << 16;
    }
};

// D / 4 lanes to a token and head, eight elements each, the keys' lanes before the values': four lanes share a
// group.  A token with an element that is not finite, or whose group's scale would pass 8160, has NaN scales in all its
// groups, of keys and values: a key's NaN score is then what stands for it wherever it is seen, and its values need not be
// told apart.
// Bound by memory: 4 sequences of 5101 tokens, 8 heads of 128 halves, 87 MB in 19.6 us (with a division's remainder for each
// element 27.8); several tokens to a lane were no faster.
template <int D, bool F16>
__global__ __launch_bounds__(256) void kv4_write_kernel(const Kv4View c, const KvRows r) {
    constexpr int L = D / 4, TW = 64 / L;  // lanes of a token, tokens of a wavefront
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int h = blockIdx.y, s = blockIdx.z;
    const int i = (blockIdx.x * 4 + w) * TW + lane / L, p = lane % L;
    const int end = kv4_len(c, s), n_new = r.idx ? min(max(r.idx[s], 0), r.n_tok) : r.n_tok;
    const int t = end - n_new + i;
    const bool on = lane < TW * L && i < n_new && t >= 0;
    const bool val = p >= L / 2;
    const int piece = val ? p - L / 2 : p;
    Eight4<F16> x;
    x.clear();
    if (on) x.load((val ? r.v + i * r.v_nb[0] + h * r.v_nb[1] + s * r.v_nb[2] : r.k + i * r.k_nb[0] + h * r.k_nb[1] + s * r.k_nb[2]) + piece * (F16 ? 16 : 32));
    const int id = on ? kv4_block(c, s, t) : -1;
    if (__builtin_amdgcn_ballot_w64(id >= 0) == 0) return;
    float hi, lo;
    bool nan;
    x.ends(hi, lo, nan);
    hi = fmaxf(hi, lane_swap_f<1>(hi));
    hi = fmaxf(hi, lane_swap_f<2>(hi));
    lo = fminf(lo, lane_swap_f<1>(lo));
    lo = fminf(lo, lane_swap_f<2>(lo));
    uint16_t s16 = kv4_scale(hi, lo);
    const uint64_t bad = __builtin_amdgcn_ballot_w64(nan || s16 == KV4_NAN);
    if (bad >> (lane / L * L) & ((1ull << L) - 1)) s16 = KV4_NAN;
    const float d = s16 == KV4_NAN ? 0.0f : h2f(s16);
    // (a scale of 0 or none: 8 for all, whatever the elements are)
    const uint32_t word = d == 0.0f ? 0x88888888u : x.word(d, 1.0f / d);
    if (id < 0) return;
    const int64_t at = ((int64_t)id * c.heads + h) * c.bt;
    const int tok = t & (c.bt - 1);
    *reinterpret_cast<uint32_t*>((val ? c.v : c.k) + (at + tok) * (D / 2) + 4 * piece) = word;
    if ((piece & 3) == 0) {
        if (val) c.v_scale[at * (D / 32) + (piece >> 2) * c.bt + tok] = s16;
        else c.k_scale[(at + tok) * (D / 32) + (piece >> 2)] = s16;
    }
}

// Four lanes to a group of a row: eight elements each; a workgroup takes 256 / (D / 8) rows of a sequence and head at a time,
// keys and values, so that a lane's places follow from its row's alone.  Bound by memory: the same tokens read back, 87 MB in
// 14.0 us (24.3 with a place worked out for every eight elements of either).
template <int D, bool F16>
__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4View c, const KvRows r) {
    constexpr int D8 = D / 8, G = D / 32, R = 256 / D8;
    const int e = threadIdx.x % D8, t = blockIdx.x * R + threadIdx.x / D8, h = blockIdx.y, s = blockIdx.z;
    if ((D == 96 && threadIdx.x >= R * D8) || t >= r.n_tok) return;
    const int p = r.idx ? r.idx[(int64_t)s * r.n_tok + t] : t;
    const int id = kv4_block(c, s, p);  // (on its way beside the length)
    if (p < 0 || p >= kv4_len(c, s) || id < 0) return;
    const int64_t at = ((int64_t)id * c.heads + h) * c.bt;
    const int tok = p & (c.bt - 1);
    uint32_t w[2] = {0, 0};
    uint16_t d[2] = {0, 0};
    if (r.k) {
        w[0] = reinterpret_cast<const uint32_t*>(c.k)[(at + tok) * D8 + e];
        d[0] = c.k_scale[(at + tok) * G + (e >> 2)];
    }
    if (r.v) {
        w[1] = reinterpret_cast<const uint32_t*>(c.v)[(at + tok) * D8 + e];
        d[1] = c.v_scale[at * G + (e >> 2) * c.bt + tok];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        char* o = x ? r.v : r.k;
        if (!o) continue;
        o += x ? t * r.v_nb[0] + h * r.v_nb[1] + s * r.v_nb[2] : t * r.k_nb[0] + h * r.k_nb[1] + s * r.k_nb[2];
        const _Float16 f = __builtin_bit_cast(_Float16, d[x]);
        uint32_t y[4];
        word_halves(w[x], h2v{f, f}, y);
        if constexpr (F16) {
            *reinterpret_cast<u32x4_a2*>(o + 16 * e) = u32x4{y[0], y[1], y[2], y[3]};
        } else {
            v4f z[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const h2v q = __builtin_bit_cast(h2v, y[i]);
                z[i >> 1][2 * (i & 1)] = (float)q[0];
                z[i >> 1][2 * (i & 1) + 1] = (float)q[1];
            }
            *reinterpret_cast<v4f_a4*>(o + 32 * e) = z[0];
            *reinterpret_cast<v4f_a4*>(o + 32 * e + 16) = z[1];
        }
    }
}

// ---- eviction
namespace {
constexpr int EV_T = 1024;
struct EvictSpan {
    int n, keep, first, body;  // length; kept; tokens 0 .. first - 1 and body .. n - 1 are kept anyway
};
}  // namespace
__device__ __forceinline__ EvictSpan evict_span(const Kv4EvictArgs& a, int s) {
    EvictSpan e;
    e.n = kv4_len(a.c, s);
    e.keep = min(e.n, a.n_keep ? min(max(a.n_keep[s], 0), a.max_keep) : a.max_keep);
    const int recent = min(a.recent, e.keep);
    e.first = min(a.first, e.keep - recent);
    e.body = e.n - recent;
    return e;
}
// floats in the order of unsigned keys: tokens that are not there 0, NaN 1, then the numbers (both zeros alike)
__device__ __forceinline__ uint32_t evict_key(float x, bool there) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return !there ? 0u : x != x ? 1u : u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint32_t lanes_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// The sum of v over this lane and those before it: shifts within rows of 16 lanes, then the rows' last lanes to those after
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
}

// Counts of a workgroup's wavefronts, 64 PER of them in the order of tokens, to the sums of those before each; the sum of
// all goes behind them.  The first wavefront does it.
template <int PER>
__device__ __forceinline__ void scan_counts(uint32_t* count) {
    typedef uint32_t some __attribute__((ext_vector_type(PER)));
    __syncthreads();
    if (threadIdx.x < 64) {
        some v = reinterpret_cast<some*>(count)[threadIdx.x];
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t x = v[i];
            v[i] = mine;
            mine += x;
        }
        uint32_t before = wave_scan(mine);
        if (threadIdx.x == 63) count[64 * PER] = before;
        before -= mine;
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] += before;
        reinterpret_cast<some*>(count)[threadIdx.x] = v;
    }
    __syncthreads();
}

// The tokens that one sequence and head keeps, in their order, and their sums: a workgroup each.  The m-th largest key
// among the tokens that are not kept anyway is found digit by digit (11, 11 and 10 bits, a histogram each, until a bin's are all needed); what lies above
// it is kept, and of its equals the first ones, as many as are missing.  Eight copies of the histogram, by lane, keep a
// wavefront's lanes off one another's counter: many sums may be alike.
// A thread has PER tokens in registers, 1024 apart.  Longer sequences (LONG) are walked PER at a time, once for each digit and
// twice at the end.  Bound by what one CU does for a sequence and head (the loads, two or three histograms, two scans, the
// lists): 8 sequences of 16384 tokens and 8 heads in 24 us, 1280 tokens in 7.5.
template <int PER, bool LONG>
__global__ __launch_bounds__(EV_T) void kv4_select_kernel(const Kv4EvictArgs a) {
    constexpr int W = EV_T / 64, SPAN = PER * EV_T;
    __shared__ __attribute__((aligned(16))) uint32_t hist[8][2048 + 8];  // (a digit's copies in different banks)
    __shared__ __attribute__((aligned(16))) uint32_t count[PER * W + 1];
    __shared__ uint32_t found[3];  // the bin, how many of it are needed, how many it has
    const Kv4View& c = a.c;
    const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x, w = t >> 6;
    const EvictSpan e = evict_span(a, s);
    const int64_t room = (int64_t)c.max_blocks * c.bt, row = (int64_t)s * c.heads + h;
    const float* sums = a.sums + row * room;
    float* out = a.sums_out + row * room;
    int32_t* kept = a.kept + row * a.max_keep;
    if (h == 0 && t == 0) a.n_out[s] = e.keep;
    if (e.keep == e.n) {
        for (int i = t; i < e.n; i += EV_T) {
            kept[i] = i;
            out[i] = sums[i];
        }
        return;
    }
    const int32_t* table = c.table + (int64_t)s * c.max_blocks;
    float x[PER];
    uint32_t key[PER], in = 0, middle = 0;  // bit j: token j is one of the sequence's, is one to choose among
    auto load = [&](int i0) {
        int id[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = i0 + j * EV_T + t;
            x[j] = i < e.n ? sums[i] : 0.0f;
            id[j] = i < e.n ? table[i >> c.bt_log2] : -1;
        }
        in = middle = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = i0 + j * EV_T + t;
            key[j] = evict_key(x[j], (uint32_t)id[j] < (uint32_t)c.n_blocks);
            in |= (uint32_t)(i < e.n) << j;
            middle |= (uint32_t)(i >= e.first && i < e.body) << j;
        }
    };
    uint32_t need = e.keep - e.first - (e.n - e.body);  // of the middle ones; fewer than there are
    uint32_t cut = 0, mask = 0;                         // the key's digits so far
    if (!LONG) load(0);
    const int steps = LONG ? (e.n + SPAN - 1) / SPAN : 1;
    if (need > 0) {
        for (int i = t; i < 2056 * 2; i += EV_T) reinterpret_cast<u32x4*>(&hist[0][0])[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    for (int pass = 0; need > 0 && pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        for (int step = 0; step < steps; ++step) {
            if (LONG) load(step * SPAN);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if ((middle >> j & 1) && ((key[j] ^ cut) & mask) == 0) atomicAdd(&hist[t & 7][key[j] >> shift & (bins - 1)], 1u);
            }
        }
        __syncthreads();
        // from the top: the bin in which the need-th lies.  A thread has the bins 2 (1023 - t) + 1 and 2 (1023 - t), and clears them.
        uint32_t v[2] = {0, 0};  // (the higher bin first)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            u32x2* b = reinterpret_cast<u32x2*>(&hist[i][2 * (EV_T - 1 - t)]);
            const u32x2 n = *b;
            *b = u32x2{0, 0};
            v[0] += n[1];
            v[1] += n[0];
        }
        uint32_t above = wave_scan(v[0] + v[1]);
        if ((t & 63) == 63) count[w] = above;
        __syncthreads();
        above -= v[0] + v[1];
#pragma unroll
        for (int i = 0; i < W; ++i) above += i < w ? count[i] : 0;
        if (above < need && need <= above + v[0] + v[1]) {
            const bool low = above + v[0] < need;
            found[0] = 2 * (EV_T - 1 - t) + (low ? 0 : 1);
            found[1] = need - above - (low ? v[0] : 0);
            found[2] = v[low];
        }
        __syncthreads();
        cut |= found[0] << shift;
        mask |= (uint32_t)(bins - 1) << shift;
        need = found[1];
        if (need == found[2]) break;  // all that have these digits
    }
    __syncthreads();
    // kept: the first and the last ones, keys above cut, and the first `need` that equal it
    int at = 0;
    uint32_t equals = 0;
    for (int step = 0; step < steps; ++step) {
        if (LONG) load(step * SPAN);
        uint64_t eq[PER], keep[PER];
        bool equal[PER], kept_here[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            equal[j] = need > 0 && (middle >> j & 1) && ((key[j] ^ cut) & mask) == 0;
            eq[j] = __builtin_amdgcn_ballot_w64(equal[j]);
            if ((t & 63) == 0) count[j * W + w] = (uint32_t)__popcll(eq[j]);
        }
        scan_counts<PER * W / 64>(count);
        uint32_t before[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) before[j] = equals + count[j * W + w];
        equals += count[PER * W];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            kept_here[j] = (in >> j & 1) && (!(middle >> j & 1) || (need > 0 && (equal[j] ? before[j] + lanes_below(eq[j]) < need : (key[j] & mask) > cut)));
            keep[j] = __builtin_amdgcn_ballot_w64(kept_here[j]);
            if ((t & 63) == 0) count[j * W + w] = (uint32_t)__popcll(keep[j]);
        }
        scan_counts<PER * W / 64>(count);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (!kept_here[j]) continue;
            const int to = at + (int)(count[j * W + w] + lanes_below(keep[j]));
            kept[to] = step * SPAN + j * EV_T + t;
            out[to] = x[j];
        }
        at += (int)count[PER * W];
        __syncthreads();
    }
    for (int i = e.keep + t; i < e.n; i += EV_T) out[i] = 0.0f;
}

// Kept rows go to their places, in order and in place: place j's row comes from kept[j] >= j.  A workgroup moves the
// keys or values of a sequence and head (heads of 128: half of each row) or either's scales, U rows to a thread at a time: all of
// these rows are read before any place is written, and no later place's source is among the places before it.
// Each such round is a chain of loads (index, block, row) behind the last round's stores, about 8 us, so that rounds are few and
// long: half of 16384 tokens of 8 sequences and 8 heads of 128, 120 MB read and written, in 42 us, 49 with rounds of 1536
// whole rows, 53 with 16 bytes of 4096.
template <int D>
__global__ __launch_bounds__(EV_T) void kv4_move_kernel(const Kv4EvictArgs a, const int items) {
    constexpr int G = D / 32, L = D == 96 ? 3 : 2, NS = D / 32 / L, U = 8;  // groups, 16-byte lanes of a slice, slices
    const Kv4View& c = a.c;
    const int item = blockIdx.x % items, what = blockIdx.x / items;  // (what: the slices of keys, of values, and the scales, which are short)
    const bool wide = what < 2 * NS, val = wide ? what >= NS : what > 2 * NS;
    const int h = item % c.heads, s = item / c.heads;
    const EvictSpan e = evict_span(a, s);
    if (e.keep == e.n) return;
    const int32_t* kept = a.kept + (int64_t)item * a.max_keep;
    const int lanes = wide ? L : 1, tokens = EV_T / lanes, tok0 = (int)threadIdx.x / lanes, part = (int)threadIdx.x - tok0 * lanes;
    const bool on = tok0 < tokens;
    char* rows = reinterpret_cast<char*>(val ? c.v : c.k) + 16 * (part + L * (what % NS));
    auto wide_at = [&](int id, int tok) { return reinterpret_cast<u32x4*>(rows + (((int64_t)id * c.heads + h) * c.bt + tok) * (D / 2)); };
    auto scale_at = [&](int id, int tok, int g) {
        const int64_t at = ((int64_t)id * c.heads + h) * c.bt;
        return val ? c.v_scale + at * G + g * c.bt + tok : c.k_scale + (at + tok) * G + g;
    };
    int src[U], to[U], next[U], next_to[U];
    auto look_up = [&](int j0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * tokens + tok0;
            const bool in = on && j < e.keep;
            next[u] = in ? kept[j] : -1;
            next_to[u] = in ? kv4_block(c, s, j) : -1;
            if (next[u] <= j) next_to[u] = -1;  // (where it is already)
        }
    };
    look_up(0);
    for (int j0 = 0; j0 < e.keep; j0 += U * tokens) {
        int from[U];
        u32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            src[u] = next[u];
            to[u] = next_to[u];
            from[u] = to[u] >= 0 ? kv4_block(c, s, src[u]) : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x[u] = u32x4{0, 0, 0, 0};
            const int tok = src[u] & (c.bt - 1);
            if (from[u] < 0) {  // a row whose block is not there leaves NaN scales: its place never shows what stood there
                if (!wide) x[u] = u32x4{KV4_NAN, KV4_NAN, KV4_NAN, KV4_NAN};
            } else if (wide) {
                x[u] = *wide_at(from[u], tok);
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g) x[u][g] = *scale_at(from[u], tok, g);
            }
        }
        if (j0 + U * tokens < e.keep) look_up(j0 + U * tokens);
#pragma unroll
        for (int u = 0; u < U; ++u) asm volatile("" ::"v"(x[u]) : "memory");  // (these rows have arrived)
        lds_barrier();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int tok = (j0 + u * tokens + tok0) & (c.bt - 1);
            if (to[u] < 0) continue;
            if (wide) {
                if (from[u] >= 0) *wide_at(to[u], tok) = x[u];
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g) *scale_at(to[u], tok, g) = (uint16_t)x[u][g];
            }
        }
    }
}

template <int D>
static void kv4_write_go(const Kv4View& c, const KvRows& r, hipStream_t st) {
    constexpr int per = kv4_write_tokens(D);
    const dim3 g((unsigned)(((int64_t)r.n_tok + per - 1) / per), (unsigned)c.heads, (unsigned)c.n_seq);
    if (r.f16) kv4_write_kernel<D, true><<<g, 256, 0, st>>>(c, r);
    else kv4_write_kernel<D, false><<<g, 256, 0, st>>>(c, r);
}

hipError_t launch_kv4_write(const Kv4View& c, const KvRows& r, int D, hipStream_t st) {
    if (c.n_seq <= 0 || r.n_tok <= 0 || c.max_blocks <= 0 || c.n_blocks <= 0) return hipSuccess;
    switch (D) {
        case 64: kv4_write_go<64>(c, r, st); break;
        case 96: kv4_write_go<96>(c, r, st); break;
        case 128: kv4_write_go<128>(c, r, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4View& c, const KvRows& r, int D, hipStream_t st) {
    if (r.n_tok <= 0 || c.n_seq <= 0 || c.max_blocks <= 0 || c.n_blocks <= 0) return hipSuccess;
    auto go = [&](auto d) {
        constexpr int DD = decltype(d)::value, R = 256 / (DD / 8);
        const dim3 g((unsigned)(((int64_t)r.n_tok + R - 1) / R), (unsigned)c.heads, (unsigned)c.n_seq);
        if (r.f16) kv4_read_kernel<DD, true><<<g, 256, 0, st>>>(c, r);
        else kv4_read_kernel<DD, false><<<g, 256, 0, st>>>(c, r);
        return hipGetLastError();
    };
    switch (D) {
        case 64: return go(std::integral_constant<int, 64>());
        case 96: return go(std::integral_constant<int, 96>());
        case 128: return go(std::integral_constant<int, 128>());
        default: return hipErrorInvalidValue;
    }
}

template <int D>
static void kv4_move_go(const Kv4EvictArgs& a, hipStream_t st) {
    const int items = a.c.heads * a.c.n_seq;
    kv4_move_kernel<D><<<(unsigned)((D == 128 ? 6 : 4) * items), EV_T, 0, st>>>(a, items);
}

hipError_t launch_kv4_evict(const Kv4EvictArgs& a, int D, hipStream_t st) {
    if (a.c.n_seq <= 0) return hipSuccess;
    if (6 * EV_T * (int64_t)a.c.heads * a.c.n_seq > UINT32_MAX) return hipErrorInvalidValue;
    const int64_t room = (int64_t)a.c.max_blocks * a.c.bt;
    const dim3 g((unsigned)a.c.heads, (unsigned)a.c.n_seq);
    if (room <= 4 * EV_T) kv4_select_kernel<4, false><<<g, EV_T, 0, st>>>(a);
    else if (room <= 16 * EV_T) kv4_select_kernel<16, false><<<g, EV_T, 0, st>>>(a);
    else kv4_select_kernel<16, true><<<g, EV_T, 0, st>>>(a);
    if (a.c.n_blocks <= 0 || a.c.max_blocks <= 0 || a.max_keep <= 0) return hipGetLastError();
    switch (D) {
        case 64: kv4_move_go<64>(a, st); break;
        case 96: kv4_move_go<96>(a, st); break;
        case 128: kv4_move_go<128>(a, st); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace mi355
