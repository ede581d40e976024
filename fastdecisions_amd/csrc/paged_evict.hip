// Eviction from a paged cache, gfx950: of every request the `recent` last keys and, per key head, those of largest
// weight stay, `keep` in all, and move in their order to pages of their own.
//
//   select  one workgroup per (request, head): the weight of the last key that stays by up to three counting passes
//           over 11, 11 and 10 bits of the weights in an order-preserving integer form (fewer where all keys of a count
//           stay), then one pass that numbers the keys that stay in their order (a key above the weight, and as many at
//           it as there is room for, lowest first) and moves their weights
//   move    rows and scales of the kept keys, a lane per 16 bytes, two rows each; streaming
//
// Select is bound by the latency of one workgroup (12 requests x 4 heads: 48 of 256 CUs): weights of up to 16384 keys are
// loaded once and stay in registers (from memory in every pass: 21 us for 1500 to 10411 keys, now 14 to 15; 700 keys
// 7.0, with three passes always 7.8), then passes of LDS atomics over 2048 bins, and a barrier per 4096 keys when they are
// numbered.  Atomics that meet in a bin are not what it waits for: LDS conflicts are 4 % of its cycles, and weights spread over
// many bins take 13.4 us where those that fall into a few dozen take 15.2.  Longer requests load their weights in every pass:
// one request cut to 2048 keys (4 heads x 128, E4M3, a call) 21 us for 16384 keys, 29 for one key more, 46 for 32768, 153 for
// 131072.  A cut of a head over several workgroups would need a launch per pass, 3 to 4 us each.  Move: 50 MB in 10.4 us,
// 4.8 TB/s.
#include <algorithm>
#include <type_traits>

#include "paged_common.h"
#include "state_slot.h"
#include "wave_tools.h"

namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kBins = 2048;
constexpr int kPer = 4;                            // consecutive keys of a thread and chunk
constexpr int kChunk = kSelectThreads * kPer;
constexpr int kHeld = 4;                           // chunks whose weights stay in registers: all of up to 16384 keys
constexpr int kMoveThreads = 256;

struct EvictArgs {
  PagedView c;
  const float* w;
  float* w_out;
  int64_t w_row, w_head;
  const int32_t* index;       // or null
  const int32_t* new_table;
  int64_t new_stride;
  int32_t* kept;              // [requests, heads, keep]
  int32_t* new_lens;
  int w_rows, n_req, heads, keep, recent;
};

// Larger weight, larger integer; +0 and -0 alike, NaN below everything.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return w != w ? 0u : (u >> 31) != 0 ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ int bins[kBins];
  __shared__ int wave_sums[2][kSelectWaves];
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int req = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const int len = request_keys(a.c, req), left = min(len, a.keep), recent = min(a.recent, left);
  const int fixed = len - recent, need = left - recent;  // `need` of the keys [0, fixed) stay, and all behind them
  const int slot = owned_slot(a.index, req, a.w_rows, lane);
  const float* const w = slot < 0 ? nullptr : a.w + slot * a.w_row + head * a.w_head;
  float* const w_out = slot < 0 ? nullptr : a.w_out + slot * a.w_row + head * a.w_head;
  int32_t* const kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.keep;
  auto weight = [&](int j) { return w == nullptr ? 0.0f : w[j]; };  // a request without weights: the first keys stay
  if (tid == 0 && head == 0) a.new_lens[req] = left;

  // The row's weights are loaded once where they fit, else in every pass.  (four keys of a thread lie in a row)
  const bool held = len <= kHeld * kChunk;
  float x[kHeld][kPer];
  auto load = [&](int j0, float (&y)[kPer]) {
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int j = j0 + tid * kPer + u;
      y[u] = j < len ? weight(j) : 0.0f;
    }
  };
  if (held) {
#pragma unroll
    for (int c = 0; c < kHeld; ++c) load(c * kChunk, x[c]);
  }
  auto each = [&](int end, auto use) {  // use(first key, weights) of the chunks of [0, end)
    if (held) {
#pragma unroll
      for (int c = 0; c < kHeld; ++c)
        if (c * kChunk < end) use(c * kChunk, x[c]);
    } else {
      for (int j0 = 0; j0 < end; j0 += kChunk) {
        float y[kPer];
        load(j0, y);
        use(j0, y);
      }
    }
  };

  // ---- the weight at the border: its leading bits, and how many keys of those bits stay
  uint32_t border = 0;
  int room = need, bits = 0;  // of a weight below the leading ones
  if (need > 0 && need < fixed) {
    const int shifts[3] = {21, 10, 0};
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = shifts[pass], width = pass < 2 ? 11 : 10;
      for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
      each(fixed, [&](int j0, const float (&y)[kPer]) {
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          const uint32_t key = order_of(y[u]);
          if (j0 + tid * kPer + u < fixed && (pass == 0 || key >> (shift + width) == border >> (shift + width)))
            atomicAdd(&bins[(key >> shift) & ((1 << width) - 1)], 1);
        }
      });
      __syncthreads();
      // two bins per thread, largest first: the bin where the running count reaches `room`
      const int b0 = kBins - 1 - 2 * tid, c0 = bins[b0], c1 = bins[b0 - 1];
      const int incl_wave = wave_scan(c0 + c1);
      if (lane == 63) wave_sums[pass & 1][wave] = incl_wave;
      __syncthreads();
      // (16 wavefronts: lane v of each holds the sum of wavefront v)
      const int sums = wave_scan(lane < kSelectWaves ? wave_sums[pass & 1][lane] : 0);
      const int incl = incl_wave + (wave == 0 ? 0 : __builtin_amdgcn_readlane(sums, max(wave - 1, 0)));
      const int before = incl - c0 - c1;
      if (before < room && room <= incl) {
        const bool first = room <= before + c0;
        found[0] = first ? b0 : b0 - 1;
        found[1] = room - before - (first ? 0 : c0);
        found[2] = first ? c0 : c1;
      }
      __syncthreads();
      border |= static_cast<uint32_t>(found[0]) << shift;
      room = found[1];
      bits = shift;
      if (room == found[2]) break;  // all of these bits stay: what follows them does not matter
    }
  }
  const bool all = need >= fixed;

  // ---- the keys that stay, in their order
  int above = 0, equal = 0;  // of the keys before this chunk
  __syncthreads();           // the sums are read
  each(len, [&](int j0, const float (&y)[kPer]) {
    bool is_above[kPer], is_equal[kPer];
    int mine = 0;  // keys above in the low half, at the border in the high one
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int j = j0 + tid * kPer + u;
      const uint32_t key = order_of(y[u]) >> bits, last = border >> bits;
      is_above[u] = j < len && (j >= fixed || all || (need > 0 && key > last));
      is_equal[u] = !is_above[u] && j < fixed && need > 0 && key == last;
      mine += (is_above[u] ? 1 : 0) + (is_equal[u] ? 1 << 16 : 0);
    }
    const int incl = wave_scan(mine), parity = (j0 / kChunk) & 1;
    if (lane == 63) wave_sums[parity][wave] = incl;
    __syncthreads();  // every weight of the chunk is read, too
    const int sums = wave_scan(lane < kSelectWaves ? wave_sums[parity][lane] : 0), total = __builtin_amdgcn_readlane(sums, 63);
    const int before = incl - mine + (wave == 0 ? 0 : __builtin_amdgcn_readlane(sums, max(wave - 1, 0)));
    int n_above = above + (before & 0xffff), n_equal = equal + (before >> 16);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if (is_above[u] || (is_equal[u] && n_equal < room)) {
        const int place = n_above + min(n_equal, room);
        kept[place] = j0 + tid * kPer + u;
        if (w_out != nullptr) w_out[place] = y[u];
      }
      n_above += is_above[u] ? 1 : 0;
      n_equal += is_equal[u] ? 1 : 0;
    }
    above += total & 0xffff;
    equal += total >> 16;
  });
  __syncthreads();  // weights that move into [0, left) are read
  for (int i = left + tid; i < a.keep; i += kSelectThreads) kept[i] = -1;
  if (w_out != nullptr)
    for (int j = left + tid; j < len; j += kSelectThreads) w_out[j] = 0.0f;
}

// U rows per thread side by side.
template <int D, Format F, int U>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  constexpr int kRowBytes = F == kBf16 ? 2 * D : F == kE4m3 ? D : D / 2;
  constexpr int kLanes = kRowBytes / 16, kSide = kMoveThreads / kLanes;
  constexpr int kScales = F == kE2m1 ? D / kScaleBlock : 1;
  using Scales = std::conditional_t<kScales == 8, uint64_t, std::conditional_t<kScales == 4, uint32_t, std::conditional_t<kScales == 2, uint16_t, uint8_t>>>;
  const int side = blockIdx.y, li = threadIdx.x % kLanes;
  unsigned char* const pool = side == 0 ? a.c.k : a.c.v;
  uint8_t* const scales = side == 0 ? a.c.k_scale : a.c.v_scale;
  const int64_t rows = static_cast<int64_t>(a.n_req) * a.heads * a.keep;
  const int mask = (1 << a.c.shift) - 1;
  int head[U], from[U], to[U], src[U], dst[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * U + u) * kSide + threadIdx.x / kLanes;
    from[u] = row < rows ? a.kept[row] : -1;
    const int64_t rh = row / a.keep;
    to[u] = static_cast<int>(row - rh * a.keep);
    head[u] = static_cast<int>(rh % a.heads);
    const int req = static_cast<int>(rh / a.heads);
    src[u] = from[u] >= 0 ? a.c.table[req * a.c.table_stride + (from[u] >> a.c.shift)] : -1;
    dst[u] = from[u] >= 0 ? a.new_table[req * a.new_stride + (to[u] >> a.c.shift)] : -1;
  }
  uint4 w[U];
  Scales s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    w[u] = {0, 0, 0, 0};  // what a key on no page reads as
    s[u] = static_cast<Scales>(0x7f7f7f7f7f7f7f7full);
    if (static_cast<unsigned>(src[u]) < static_cast<unsigned>(a.c.n_pages)) {
      w[u] = *reinterpret_cast<const uint4*>(pool + src[u] * a.c.page + head[u] * a.c.head + (from[u] & mask) * a.c.row + li * 16);
      if (F != kBf16 && li == 0)
        s[u] = *reinterpret_cast<const Scales*>(scales + src[u] * a.c.s_page + head[u] * a.c.s_head + (from[u] & mask) * kScales);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (static_cast<unsigned>(dst[u]) >= static_cast<unsigned>(a.c.n_pages)) continue;
    *reinterpret_cast<uint4*>(pool + dst[u] * a.c.page + head[u] * a.c.head + (to[u] & mask) * a.c.row + li * 16) = w[u];
    if (F != kBf16 && li == 0)
      *reinterpret_cast<Scales*>(scales + dst[u] * a.c.s_page + head[u] * a.c.s_head + (to[u] & mask) * kScales) = s[u];
  }
}

}  // namespace

extern "C" int fd_paged_kv_evict(const fd_paged_cache* cache, const float* weights, float* weights_out,
                                 const int64_t weight_strides[2], int weight_rows, const int32_t* row_indices,
                                 const int32_t* new_table, int64_t new_table_stride, int new_max_pages, int requests,
                                 int keep, int recent, int32_t* kept, int32_t* new_lens, void* stream) {
  static const char* what = "fd_paged_kv_evict";
  FD_REQUIRE(weights && weights_out && weight_strides && new_table && kept && new_lens, FD_ERR_INVALID_ARGUMENT,
             "%s: weights, the new table, kept and new_lens must be non-null", what);
  EvictArgs a;
  if (int rc = fill_view(what, cache, true, &a.c)) return rc;
  FD_REQUIRE(requests >= 0 && keep >= 1 && recent >= 0 && recent <= keep, FD_ERR_INVALID_ARGUMENT,
             "%s: requests >= 0, keep >= 1 and recent in [0, keep]", what);
  FD_REQUIRE(new_max_pages >= 1 && static_cast<int64_t>(new_max_pages) * cache->page_size >= keep, FD_ERR_INVALID_ARGUMENT,
             "%s: the new table must hold %d keys", what, keep);
  FD_REQUIRE(weight_rows >= 0 && (row_indices || weight_rows >= requests), FD_ERR_INVALID_ARGUMENT,
             "%s: the weights need a row for every request", what);
  FD_REQUIRE(weight_strides[0] >= 0 && weight_strides[1] >= 0, FD_ERR_INVALID_ARGUMENT, "%s: weight strides must be >= 0", what);
  const int64_t select = static_cast<int64_t>(requests) * cache->kv_heads, rows = select * keep;
  FD_REQUIRE(select < (1LL << 32) / kSelectThreads && rows < (1LL << 27), FD_ERR_UNSUPPORTED, "%s: problem too large", what);
  if (requests == 0) return FD_OK;
  a.w = weights;
  a.w_out = weights_out;
  a.w_row = weight_strides[0];
  a.w_head = weight_strides[1];
  a.index = row_indices;
  a.new_table = new_table;
  a.new_stride = new_table_stride;
  a.kept = kept;
  a.new_lens = new_lens;
  a.w_rows = weight_rows;
  a.n_req = requests;
  a.heads = cache->kv_heads;
  a.keep = keep;
  a.recent = recent;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(evict_select_kernel, dim3(static_cast<unsigned>(select)), dim3(kSelectThreads), 0, s, a);
  if (int rc = fd_check_launch(what)) return rc;
  by_kind(cache, [&](auto d, auto f) {
    constexpr int D = decltype(d)::value;
    constexpr Format F = decltype(f)::value;
    constexpr int U = 2, per = kMoveThreads / ((F == kBf16 ? 2 * D : F == kE4m3 ? D : D / 2) / 16) * U;
    hipLaunchKernelGGL((evict_move_kernel<D, F, U>), dim3(static_cast<unsigned>((rows + per - 1) / per), 2), dim3(kMoveThreads), 0, s, a);
  });
  return fd_check_launch(what);
}
