// Tile conventions shared by the attention kernels: operand types, the key
// permutation and chunk swizzles of the LDS tiles, lane-half reductions and the
// copy to LDS.
#pragma once

#include "fd_common.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) void lds_void_t;
typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16_t lds_v4i16_t;

namespace {

// Key (within a 32-key block) supplied by MFMA row m, chosen so that the
// accumulator registers 8j..8j+7 of lane half g hold keys 16j + 8g + 0..7.
__device__ __forceinline__ int sigma(int m) {
  return ((m >> 4) << 4) + (((m >> 2) & 1) << 3) + (((m >> 3) & 1) << 2) + (m & 3);
}

// Chunk swizzles (physical chunk = logical chunk ^ f(row)).  K: the MFMA A
// operand reads rows sigma(0..7) = {0,1,2,3,8,9,10,11} (then +4) at one chunk;
// a bit permutation of row & 15 sends any 8 of them to 8 distinct chunks.
// V: 16 lanes of a transposing read touch 4 consecutive rows x 2 adjacent
// chunks, 32 lanes 4 rows x 4 chunks; the xor keeps chunk pairs adjacent.
template <int CR>
__device__ __forceinline__ int swz_k(int row) {
  const int r = row & 15;
  return ((r & 3) | ((r & 8) >> 1) | ((r & 4) << 1)) & (CR - 1);
}
template <int CR>
__device__ __forceinline__ int swz_v(int row) {
  // 16+ chunks per row: xor with 4*(row & 3) puts the 4 rows x 4 chunks that
  // 32 lanes of a transposing read touch on 16 distinct chunks (all banks).
  return CR >= 16 ? 4 * (row & 3) : (2 * (row & 3)) & (CR - 1);
}

// Max / sum of a value over lanes l and l^32 (the two lane halves hold the two
// 16-key halves of one query's scores).  v_permlane32_swap with the value in
// both operands leaves this lane's value in one result and its partner's in
// the other, so max and sum of the pair need no lane-index select.
__device__ __forceinline__ float half_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Copies 16 bytes per lane from `base` (uniform) + `off` to 1 KiB of LDS at
// `lds`, in flight until a vmcnt wait: an asm that the compiler does not count.
// The hardware needs one wait state between a write of M0 and the copy that
// reads it; the compiler keeps it for its own copies, not inside an asm.
__device__ __forceinline__ void copy_to_lds(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

}  // namespace
