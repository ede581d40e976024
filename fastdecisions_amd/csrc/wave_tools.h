// Arithmetic of one wavefront that finds its work: sums over lanes, scalar loads, uniform values.
#pragma once

#include "fd_common.h"

namespace {

// Inclusive sums over the lanes, on DPP: within rows of 16 lanes, then a row's last lane into the next row(s).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// p[i] for a uniform i, by a scalar load: a vector load here would make the compiler wait for
// the copies in flight.  Nothing writes the page table while the kernel runs.
// i is not negative and 4 i fits 32 bits.
__device__ __forceinline__ int scalar_load(const int32_t* p, int i) {
  typedef const __attribute__((address_space(4))) char const_char;
  typedef const __attribute__((address_space(4))) int32_t const_i32;
  const uint32_t at = static_cast<uint32_t>(i) * 4u;
  return *reinterpret_cast<const_i32*>(reinterpret_cast<const_char*>(reinterpret_cast<uintptr_t>(p)) + at);
}

// An index that is the same in all lanes, in a scalar register.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ceil(x / c) for x and c up to 2^22: a reciprocal whose error is put right by one step.
__device__ __forceinline__ int tiles_over(int x, int c) {
  const int y = x + c - 1;
  int q = static_cast<int>(static_cast<float>(y) * __builtin_amdgcn_rcpf(static_cast<float>(c)));
  const int r = y - q * c;
  return q + (r >= c ? 1 : 0) - (r < 0 ? 1 : 0);
}

}  // namespace
