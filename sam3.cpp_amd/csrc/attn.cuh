// Device code that the attention kernels share: reductions over the two halves of a wavefront, LDS
// layouts of key and value tiles, transposing LDS reads; and those over a cache: the tokens that queries see,
// sums over a column's lanes, accesses past the caches.
#pragma once
#include "common.cuh"

namespace mi355 {

// max / sum over lanes l and l ^ 32 (the two halves of the wavefront hold the same
// queries): v_permlane32_swap of x with itself leaves x_l and x_(l^32) in its two
// results, in an order that depends on the half, and both operations are commutative
__device__ __forceinline__ float xmax32(float x) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return fmaxf(__int_as_float((int)p[0]), __int_as_float((int)p[1]));
}
// Workgroup barrier for LDS hazards only: waits for this wavefront's LDS accesses,
// not for its global loads still in flight (__syncthreads() also waits for those).
// The "memory" clobber keeps the compiler from moving LDS accesses across it.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ float xsum32(float x) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return __int_as_float((int)p[0]) + __int_as_float((int)p[1]);
}

// K row slot of 16-byte chunk c in row r of an unpadded fp16 K tile (DMA staging):
// the 32-row fragment reads of one chunk then fall in distinct bank quads
// (D = 96: 192-byte rows, four to three bank lines; (r >> 2) & 3 keeps a chunk inside its
// aligned group of four, so the twelve slots stay twelve)
template <int D>
__device__ __forceinline__ int kswz(int r) { return D == 64 ? ((r & 7) ^ ((r >> 3) & 1)) : D == 96 ? ((r >> 2) & 3) : (r & 15); }
// V row slot of 16-byte chunk c in row r of an unpadded fp16 V tile (DMA staging): slot
// c ^ vswz(r).  A transposing read of the PV operand takes 64 bytes (4 chunks 4 db .. +3)
// from each of 4 consecutive rows per half-wavefront; the 64 banks of 4 bytes then hold each
// byte once when the 4 rows' chunks land in distinct 64-byte quarters of a 256-byte bank
// line: D = 64 (128-byte rows: odd rows are the upper bank half) moves rows 2, 3 (mod 4) to
// the other half of their row's slots and rows 4..7 (mod 8) by one chunk; D = 128 (256-byte
// rows) moves row r by 4 (r % 4) chunks; D = 96 (192-byte rows) needs none: the 4 rows start
// at 0, 192, 384 and 576 bytes, so their 64-byte pieces fall in distinct quarters already.
// (The transposing reads add whole 8-row blocks to a swizzled row offset, so vswz may
// depend on r % 8 only.)
template <int D>
__device__ __forceinline__ int vswz(int r) { return D == 64 ? (((r & 2) << 1) | ((r >> 2) & 1)) : D == 96 ? 0 : ((r & 3) << 2); }

// 4 fp16 of LDS by the transposing read of gfx950 (ds_read_b64_tr_b16): within each group
// of 16 lanes, lane i receives element i % 4 of the 8 bytes addressed by lanes i / 4,
// 4 + i / 4, 8 + i / 4 and 12 + i / 4 of its group, in that order
__device__ __forceinline__ uint2 lds_read_tr16(const void* a) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    const v4s r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(a));
    return __builtin_bit_cast(uint2, r);
}

namespace {
constexpr int KV_STEP = 32;          // tokens of one step of a wavefront
constexpr int KV_SPAN = 4 * KV_STEP; // tokens of one step of a workgroup
}  // namespace

// The tokens that a sequence's queries can see, and its queries.
struct KvRange {
    int n_kv, nq, pos0;  // length, queries, position of the first query
    int lo, hi;          // tokens lo .. hi - 1 (lo a multiple of STEP) are seen by some query
};
template <int STEP = KV_STEP, class Args>
__device__ __forceinline__ KvRange kv_range(const Args& a, int s) {
    KvRange r;
    r.n_kv = (int)min((int64_t)max(a.c.n_kv[s], 0), (int64_t)a.c.max_blocks * a.c.bt);
    r.nq = a.nq ? min(max(a.nq[s], 0), a.n_q) : a.n_q;
    r.pos0 = r.n_kv - r.nq;
    r.lo = a.window > 0 ? (int)(max((int64_t)r.pos0 - a.window + 1, (int64_t)0) & ~(int64_t)(STEP - 1)) : 0;
    r.hi = r.n_kv;
    return r;
}
// Tokens of each of `splits` ranges: whole workgroup steps
__device__ __forceinline__ int kv_chunk(const KvRange& r, int splits) {
    const int n = max(r.hi - r.lo, 1), per = (n + splits - 1) / splits;
    return (per + KV_SPAN - 1) / KV_SPAN * KV_SPAN;
}

__device__ __forceinline__ float read_lane(float v, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i)); }


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

}  // namespace mi355
