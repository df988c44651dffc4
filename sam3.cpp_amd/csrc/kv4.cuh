// The 4-bit cache's format, and what its kernels share.
//
// Elements of a token and head in groups of 32: d = -ext / 8 rounded to eight significant bits and
// fp16, ext being the group's element farthest from zero; nibble u = 8 + nearest_even(x / d) within
// 0 .. 15, which stands for (u - 8) d.  Four bits times eight are a half's eleven and one to spare, so
// that every value is exact in fp16 and a matrix instruction reads the cache as it is.
// A 32-bit word holds eight elements: element 2 i in nibble i, element 2 i + 1 in nibble i + 4, the
// two halves of a register once the word is shifted and masked.
// Keys' scales lie [block][head][token][group], beside the row that a lane reads; values'
// [block][head][group][token], the pairs of tokens that a product's registers hold.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace mi355 {

namespace {
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef v4f v4f_a4 __attribute__((aligned(4)));
typedef v8h v8h_a2 __attribute__((aligned(2)));
typedef v4h v4h_a2 __attribute__((aligned(2)));
constexpr uint16_t KV4_NAN = 0x7E00;
}  // namespace

__device__ __forceinline__ int kv4_len(const Kv4View& c, int s) {
    return (int)min((int64_t)max(c.n_kv[s], 0), (int64_t)c.max_blocks * c.bt);
}
// block of token t, or -1 (the table has blocks)
__device__ __forceinline__ int kv4_block(const Kv4View& c, int s, int t) {
    const int id = c.table[(int64_t)s * c.max_blocks + min(max(t, 0) >> c.bt_log2, c.max_blocks - 1)];
    return id >= 0 && id < c.n_blocks ? id : -1;
}

// nibbles 0 and 4 (SHIFT 0) or 1 and 5 (SHIFT 4) of w as the halves u - 8: 0x640u is the half 1024 + u, 0x64u0 1024 + 16 u.
// (Of an instruction's operands one may be a scalar: with the exponents in a vector register the mask is one, and both
// take one instruction.)
template <int SHIFT>
__device__ __forceinline__ h2v nibble_pair(uint32_t w) {
    uint32_t exps = 0x64006400u;
    asm("" : "+v"(exps));
    if constexpr (SHIFT == 0) {
        const h2v off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
        return __builtin_bit_cast(h2v, (w & 0x000f000fu) | exps) + off;
    } else {
        const h2v mul = {(_Float16)0.0625f, (_Float16)0.0625f}, off = {(_Float16)-72.0f, (_Float16)-72.0f};
        return __builtin_elementwise_fma(__builtin_bit_cast(h2v, (w & 0x00f000f0u) | exps), mul, off);
    }
}
// the four pairs of a word, times d
__device__ __forceinline__ void word_halves(uint32_t w, h2v d, uint32_t* o) {
    o[0] = __builtin_bit_cast(uint32_t, nibble_pair<0>(w) * d);
    o[1] = __builtin_bit_cast(uint32_t, nibble_pair<4>(w) * d);
    o[2] = __builtin_bit_cast(uint32_t, nibble_pair<0>(w >> 8) * d);
    o[3] = __builtin_bit_cast(uint32_t, nibble_pair<4>(w >> 8) * d);
}
// two scales, 0 in the place of those beyond 8160 (0x6ff8), infinities and NaN: their values would not be finite
__device__ __forceinline__ uint32_t finite_scales(uint32_t w) {
    const uint32_t bad = ((w & 0x7fff7fffu) + 0x10071007u) & 0x80008000u;
    return w & ~((bad >> 15) * 0xffffu);
}

}  // namespace mi355
