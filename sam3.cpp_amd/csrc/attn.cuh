// Device code that the attention kernels share: reductions over the two halves of a wavefront, LDS
// layouts of key and value tiles, transposing LDS reads.
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

}  // namespace mi355
