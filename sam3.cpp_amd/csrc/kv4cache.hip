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
// keys and values, so that a lane's places follow from its row's alone.
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
// The tokens that one sequence and head keeps, in their order, and their sums: a workgroup each.  The m-th largest key
// among the tokens that are not kept anyway is found digit by digit (11, 11 and 10 bits, a histogram each), then one
// walk over the tokens keeps what lies above it and as many of its equals, the first ones, as are missing.
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
__device__ __forceinline__ uint64_t lanes_below() { return (1ull << (threadIdx.x & 63)) - 1; }

__global__ __launch_bounds__(EV_T) void kv4_select_kernel(const Kv4EvictArgs a) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t wave[2][EV_T / 64];
    __shared__ uint32_t found[2];
    const Kv4View& c = a.c;
    const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
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
    auto key_at = [&](int i) { return evict_key(sums[i], kv4_block(c, s, i) >= 0); };
    const int body = e.body - e.first;                 // tokens to choose among
    uint32_t need = e.keep - e.first - (e.n - e.body); // and how many
    uint32_t cut = 0, mask = 0;                        // the key's digits so far
    const bool choose = need > 0 && (int)need < body;
    if (choose) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
            for (int i = t; i < bins; i += EV_T) hist[i] = 0;
            __syncthreads();
            for (int i0 = 0; i0 < body; i0 += EV_T) {
                const int i = i0 + t;
                const uint32_t k = i < body ? key_at(e.first + i) : 0;
                const bool on = i < body && (k & mask) == cut;
                const uint32_t digit = k >> shift & (bins - 1);
                // the digit of the wavefront's first lane is counted at once: most weights may be alike
                const uint64_t act = __builtin_amdgcn_ballot_w64(on);
                if (act == 0) continue;
                const uint32_t lead = __builtin_amdgcn_readlane(digit, __builtin_ctzll(act));
                const uint64_t same = __builtin_amdgcn_ballot_w64(on && digit == lead);
                if ((t & 63) == 0) atomicAdd(&hist[lead], (uint32_t)__popcll(same));
                if (on && digit != lead) atomicAdd(&hist[digit], 1u);
            }
            __syncthreads();
            // from the top: the bin in which the need-th lies.  The first wavefront's lanes take bins / 64 each.
            if (t < 64) {
                const int per = bins / 64, b1 = bins - t * per;  // bins b1 - per .. b1 - 1
                uint32_t mine = 0;
                for (int b = 0; b < per; ++b) mine += hist[b1 - 1 - b];
                uint32_t above = mine;
                for (int o = 1; o < 64; o <<= 1) {
                    const uint32_t v = __shfl_up(above, o, 64);
                    if (t >= o) above += v;
                }
                above -= mine;
                if (above < need && need <= above + mine) {
                    int b = b1 - 1;
                    while (above + hist[b] < need) above += hist[b--];
                    found[0] = (uint32_t)b;
                    found[1] = need - above;
                }
            }
            __syncthreads();
            cut |= found[0] << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            need = found[1];
            __syncthreads();
        }
    }
    // kept: the first and the last ones, keys above cut, and the first `need` that equal it
    int at = 0;
    uint32_t equals = 0;
    for (int i0 = 0; i0 < e.n; i0 += EV_T) {
        const int i = i0 + t;
        const bool in = i < e.n, mid = in && i >= e.first && i < e.body;
        const float x = in ? sums[i] : 0.0f;
        const uint32_t k = mid && choose ? evict_key(x, kv4_block(c, s, i) >= 0) : 0;
        const bool eq = mid && choose && k == cut;
        const uint64_t be = __builtin_amdgcn_ballot_w64(eq);
        if ((t & 63) == 0) wave[0][t >> 6] = (uint32_t)__popcll(be);
        __syncthreads();
        uint32_t before = equals;
        for (int w = 0; w < EV_T / 64; ++w) {
            if (w == t >> 6) before = equals;
            equals += wave[0][w];
        }
        const bool keep = in && (!mid || (choose ? k > cut || (eq && before + __popcll(be & lanes_below()) < need) : need > 0));
        const uint64_t bk = __builtin_amdgcn_ballot_w64(keep);
        if ((t & 63) == 0) wave[1][t >> 6] = (uint32_t)__popcll(bk);
        __syncthreads();
        int mine = at;
        for (int w = 0; w < EV_T / 64; ++w) {
            if (w == t >> 6) mine = at;
            at += wave[1][w];
        }
        if (keep) {
            mine += __popcll(bk & lanes_below());
            kept[mine] = i;
            out[mine] = x;
        }
    }
    for (int i = e.keep + t; i < e.n; i += EV_T) out[i] = 0.0f;
}

// Kept rows go to their places, in order and in place: place j's row comes from kept[j] >= j.  A workgroup moves one
// slice of a sequence and head's rows (16 bytes of the keys' or values' nibbles, or a scale of a group),
// 1024 places at a time; the next places' rows are asked for before these are written, which no later row's
// source is among, and written once all of the workgroup has what it asked for.
template <int D>
__global__ __launch_bounds__(EV_T) void kv4_move_kernel(const Kv4EvictArgs a, const int items) {
    constexpr int NS = D / 32, G = D / 32, SL = 2 * NS + 2 * G;  // 16-byte slices of a row, groups, slices in all
    const Kv4View& c = a.c;
    // the slices of an item run on one XCD, whose L2 has their common lines
    const int gb = blockIdx.x / (8 * SL), rb = blockIdx.x % (8 * SL), item = gb * 8 + (rb & 7), sl = rb >> 3;
    if (item >= items) return;
    const int h = item % c.heads, s = item / c.heads;
    const EvictSpan e = evict_span(a, s);
    if (e.keep == e.n) return;
    const int32_t* kept = a.kept + (int64_t)item * a.max_keep;
    const bool wide = sl < 2 * NS, val = wide ? sl >= NS : sl >= 2 * NS + G;
    const int part = wide ? sl % NS : (sl - 2 * NS) % G;
    struct Piece {
        u32x4 x;
        int j;
        bool nan;
    };
    auto place = [&](int id, int tok) -> char* {
        const int64_t at = ((int64_t)id * c.heads + h) * c.bt;
        if (wide) return reinterpret_cast<char*>(val ? c.v : c.k) + (at + tok) * (D / 2) + 16 * part;
        return reinterpret_cast<char*>(val ? c.v_scale + at * G + part * c.bt + tok : c.k_scale + (at + tok) * G + part);
    };
    auto fetch = [&](int j0) {
        Piece p;
        p.j = j0 + (int)threadIdx.x;
        p.x = u32x4{0, 0, 0, 0};
        p.nan = false;
        const int src = p.j < e.keep ? kept[p.j] : -1;
        if (src <= p.j) {  // (none, or where it is already)
            p.j = -1;
            return p;
        }
        const int id = kv4_block(c, s, src);
        if (id < 0) p.nan = true;
        else if (wide) p.x = *reinterpret_cast<const u32x4*>(place(id, src & (c.bt - 1)));
        else p.x[0] = *reinterpret_cast<const uint16_t*>(place(id, src & (c.bt - 1)));
        return p;
    };
    Piece next = fetch(0);
    for (int j0 = 0; j0 < e.keep; j0 += EV_T) {
        const Piece p = next;
        if (j0 + EV_T < e.keep) next = fetch(j0 + EV_T);
        asm volatile("" ::"v"(p.x) : "memory");  // (this step's row has arrived)
        lds_barrier();
        if (p.j < 0) continue;
        const int id = kv4_block(c, s, p.j);
        if (id < 0) continue;
        char* d = place(id, p.j & (c.bt - 1));
        // a row whose block is not there leaves a NaN key: its place never shows what stood there
        if (p.nan) {
            if (!wide) *reinterpret_cast<uint16_t*>(d) = KV4_NAN;
        } else if (wide) *reinterpret_cast<u32x4*>(d) = p.x;
        else *reinterpret_cast<uint16_t*>(d) = (uint16_t)p.x[0];
    }
}

template <int D>
static void kv4_write_go(const Kv4View& c, const KvRows& r, hipStream_t st) {
    constexpr int per = 4 * (64 / (D / 4));
    const dim3 g((unsigned)((r.n_tok + per - 1) / per), (unsigned)c.heads, (unsigned)c.n_seq);
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
    kv4_move_kernel<D><<<(unsigned)((int64_t)(items + 7) / 8 * 8 * (D / 8)), EV_T, 0, st>>>(a, items);
}

hipError_t launch_kv4_evict(const Kv4EvictArgs& a, int D, hipStream_t st) {
    if (a.c.n_seq <= 0) return hipSuccess;
    if ((int64_t)(a.c.heads * (int64_t)a.c.n_seq + 7) / 8 * 8 * (D / 8) > INT32_MAX) return hipErrorInvalidValue;
    kv4_select_kernel<<<dim3((unsigned)a.c.heads, (unsigned)a.c.n_seq), EV_T, 0, st>>>(a);
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
