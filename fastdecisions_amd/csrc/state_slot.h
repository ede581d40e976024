// Which row of a state pool a request owns.
#pragma once

#include "fd_common.h"

namespace {

// indices[r], or r itself without indices; -1 where that is no row of the pool or an earlier
// request of the call names it already: of requests with one index the first owns the state, so no
// two workgroups ever write it.  All 64 lanes take part; r is uniform.
__device__ __forceinline__ int owned_slot(const int32_t* indices, int r, int n_pool, int lane) {
  if (indices == nullptr) return r;
  const int mine = indices[r];
  bool taken = static_cast<unsigned>(mine) >= static_cast<unsigned>(n_pool);
  for (int r0 = 0; r0 < r; r0 += 64) {
    const int other = r0 + lane < r ? indices[r0 + lane] : -1;
    taken |= __builtin_amdgcn_ballot_w64(other == mine) != 0;
  }
  return taken ? -1 : mine;
}

}  // namespace
