// The attention weight that cached keys draw from new tokens, gfx950 (bf16 MFMA, fp32 sums).
//
//   w[r, h, j] += sum over rows p of head h of exp(s_pj - m_p) / l_p,   s = scale q_p . k_j
//
// with m_p, l_p a row's maximum and denominator over the keys that it sees.  A sum over rows needs every row's
// denominator first, so there are two kernels, each one product Q K^T with one exponential per score:
//
//   row stats   m and l of every row over ranges of keys (S^T = K Q^T: a lane's scores are of one row)
//   key sums    the rows' probabilities summed key by key (S = Q K^T: a lane's scores are of one key)
//
// In both the operand that stays is in registers and the other one streams through LDS.  Everything is added in an
// order that the sizes fix: no atomics.
#include <algorithm>
#include <type_traits>

#include "mfma_types.h"
#include "paged_common.h"
#include "state_slot.h"
#include "wave_tools.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

struct WeightArgs {
  PagedView c;                  // K alone
  const uint16_t* q;
  int64_t qs[3];                // b, h, t
  const int32_t* cu;
  const int32_t* index;         // or null
  float* w;
  int64_t w_row, w_head;
  int n_req, seq_len, group, kv_heads, last, w_rows;
  int target;                   // items that the row stats are cut into, about
  int part_items;
  float scale_log2;
  float* part;                  // per item of the row stats: its rows' (m, l)
};

// Row stats: RW row wavefronts of NB blocks of 32 rows, times 4 / RW key parts of a tile.
template <int RW_, int NB_>
struct Stats {
  static constexpr int RW = RW_, NB = NB_, KW = kWaves / RW;
  static constexpr int kRows = 32 * RW * NB;
  static constexpr int kKeys = KW == 1 ? 64 : 32 * KW;
};
using Few = Stats<1, 1>;
using Many = Stats<4, 2>;

// One request's part of the call: the rows that count, and the keys.
struct Req {
  int start, n_new, len;  // first counted token on the T axis, counted tokens, keys
};
__device__ __forceinline__ Req request(const WeightArgs& a, int r) {
  Req x{0, 0, 0};
  if (r < a.n_req) {
    int end;
    request_rows(a.cu, r, a.seq_len, &x.start, &end);
    x.n_new = min(end - x.start, a.last);
    x.start = end - x.n_new;
    x.len = request_keys(a.c, r);
  }
  return x;
}

// ceil(x / n) for x >= 0, and of products past 31 bits.
__device__ __forceinline__ int over(int64_t x, int n) { return static_cast<int>((x + n - 1) / n); }

template <typename T>
__device__ __forceinline__ T wave_total(T v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// Key tiles of a range of the row stats: all (row tile, key tile) pairs in about `target` items.
template <class S>
__device__ __forceinline__ int range_tiles(const WeightArgs& a, int lane) {
  int64_t work = 0;
  for (int r0 = 0; r0 < a.n_req; r0 += 64) {
    const Req x = request(a, r0 + lane);
    work += static_cast<int64_t>(over(static_cast<int64_t>(x.n_new) * a.group, S::kRows)) * over(x.len, S::kKeys);
  }
  work = wave_total(work) * a.kv_heads;
  const int64_t share = (work + a.target - 1) / a.target;
  return static_cast<int>(min(max(share, static_cast<int64_t>(256 / S::kKeys)), static_cast<int64_t>(1 << 22)));
}

// Request that holds item `at` when request r has count(r) items: false if none does; *base: items before it.
template <typename Count>
__device__ __forceinline__ bool find_request(const WeightArgs& a, int lane, int64_t at, Count count, int* req, int64_t* base) {
  int64_t before = 0;
  for (int r0 = 0; r0 < a.n_req; r0 += 64) {
    const int mine = r0 + lane < a.n_req ? count(request(a, r0 + lane)) : 0;
    const int incl = wave_scan(mine);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + incl > at);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      *req = uniform(r0 + l);
      *base = before + __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(mine, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// Eight cached values (chunk `chunk` of key `key` of a request) as bf16.
template <int D, Format F>
struct Chunk {
  std::conditional_t<F == kBf16, uint4, std::conditional_t<F == kE4m3, uint2, uint32_t>> w;
  uint8_t scale;
};
template <int D, Format F>
__device__ __forceinline__ Chunk<D, F> load_chunk(const WeightArgs& a, const int32_t* table, int head, int key, int chunk) {
  Chunk<D, F> x;
  const int slot = table[key >> a.c.shift];
  const int page = static_cast<unsigned>(slot) < static_cast<unsigned>(a.c.n_pages) ? slot : 0;
  const int at = key & ((1 << a.c.shift) - 1);
  const unsigned char* p = a.c.k + page * a.c.page + head * a.c.head + at * a.c.row;
  x.w = reinterpret_cast<const decltype(x.w)*>(p)[chunk];
  x.scale = 0;
  if constexpr (F != kBf16) {
    constexpr int per = F == kE2m1 ? D / kScaleBlock : 1;
    x.scale = a.c.k_scale[page * a.c.s_page + head * a.c.s_head + at * per + (F == kE2m1 ? chunk / 4 : 0)];
  }
  return x;
}
template <int D, Format F>
__device__ __forceinline__ bf16x8_t decoded(const Chunk<D, F>& x) {
  if constexpr (F == kBf16) {
    return __builtin_bit_cast(bf16x8_t, x.w);
  } else if constexpr (F == kE2m1) {
    return e2m1_to_bf16(x.w, scale_of(x.scale));
  } else {
    const float s = scale_of(x.scale);
    const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w.x, s, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w.x, s, true);
    const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w.y, s, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.w.y, s, true);
    return bf16x8_t{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
  }
}

// Place of chunk c of row `row` in a staged tile: 8 rows in a row at one chunk lie on 8 chunks.
template <int D>
__device__ __forceinline__ int place(int row, int c) { return (row * (D / 8) + (c ^ (row & 7))) * 16; }

// Row `row` of a request's head: its token, its query head's address, and the last key that it sees.
struct Row {
  const uint16_t* q;
  int pos;
};
__device__ __forceinline__ Row row_of(const WeightArgs& a, const Req& x, int req, int head, int row) {
  const int token = row / a.group;
  const int b = a.cu == nullptr ? req : 0;
  return {a.q + b * a.qs[0] + static_cast<int64_t>(head * a.group + row - token * a.group) * a.qs[1] +
              static_cast<int64_t>(x.start + token) * a.qs[2],
          x.len - x.n_new + token};
}

// Keys that any of a request's rows [row0, row1] sees.
__device__ __forceinline__ int seen_by(const WeightArgs& a, const Req& x, int row1) {
  return max(0, min(x.len, x.len - x.n_new + row1 / a.group + 1));
}

__device__ __forceinline__ bool on_a_page(const WeightArgs& a, const int32_t* table, int key) {
  return static_cast<unsigned>(table[key >> a.c.shift]) < static_cast<unsigned>(a.c.n_pages);
}

template <int D, Format F, class S>
__global__ __launch_bounds__(kThreads) void row_stats_kernel(WeightArgs a) {
  constexpr int CR = D / 8, kSteps = D / 16, NB = S::NB, kMoves = S::kKeys * CR / kThreads;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * S::kKeys * CR * 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int rw = wave % S::RW, kw = wave / S::RW, col = lane & 31, half = lane >> 5;
  const int c = uniform(range_tiles<S>(a, lane));
  auto tiles = [&](const Req& x) { return over(static_cast<int64_t>(x.n_new) * a.group, S::kRows); };
  auto ranges = [&](const Req& x) { return max(over(over(x.len, S::kKeys), c), 1); };
  for (int64_t item = blockIdx.x;; item += gridDim.x) {
    int req;
    int64_t base;
    if (!find_request(a, lane, item, [&](const Req& x) { return tiles(x) * ranges(x) * a.kv_heads; }, &req, &base)) return;
    const Req x = request(a, req);
    const int n_rt = uniform(tiles(x)), n_ranges = uniform(ranges(x)), k = uniform(static_cast<int>(item - base));
    const int rtile = k % n_rt, hr = k / n_rt, range = hr % n_ranges, head = hr / n_ranges;
    const int row0 = rtile * S::kRows, rows = x.n_new * a.group;
    const int kend = uniform(seen_by(a, x, min(row0 + S::kRows, rows) - 1));
    const int key0 = range * c * S::kKeys;
    const int nt = uniform(min(c, over(max(kend - key0, 0), S::kKeys)));
    if (item >= a.part_items || (range > 0 && nt == 0)) continue;
    const int32_t* const table = a.c.table + req * a.c.table_stride;
    bool bad = false;
    for (int i = (key0 >> a.c.shift) + lane; i <= ((min(key0 + nt * S::kKeys, kend) - 1) >> a.c.shift); i += 64)
      bad |= static_cast<unsigned>(table[i]) >= static_cast<unsigned>(a.c.n_pages);
    const bool absent = __builtin_amdgcn_ballot_w64(bad) != 0;

    int pos[NB];
    bf16x8_t qf[NB][kSteps];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const Row r = row_of(a, x, req, head, min(row0 + (rw * NB + n) * 32 + col, rows - 1));
      pos[n] = r.pos;
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk) qf[n][kk] = *reinterpret_cast<const bf16x8_t*>(r.q + kk * 16 + half * 8);
    }
    const int pos_min = x.len - x.n_new + min(row0 + rw * NB * 32, rows - 1) / a.group;
    float m_run[NB], l_run[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) m_run[n] = -__builtin_inff(), l_run[n] = 0.0f;

    Chunk<D, F> in[kMoves];
    auto load = [&](int t) {
#pragma unroll
      for (int i = 0; i < kMoves; ++i) {
        const int at = i * kThreads + tid;
        in[i] = load_chunk<D, F>(a, table, head, min(key0 + t * S::kKeys + at / CR, kend - 1), at % CR);
      }
    };
    auto store = [&](int t) {
#pragma unroll
      for (int i = 0; i < kMoves; ++i) {
        const int at = i * kThreads + tid;
        *reinterpret_cast<bf16x8_t*>(smem + (t & 1) * S::kKeys * CR * 16 + place<D>(at / CR, at % CR)) = decoded<D, F>(in[i]);
      }
    };
    __syncthreads();  // the item before has read its tiles
    if (nt > 0) {
      load(0);
      store(0);
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
      if (t + 1 < nt) load(t + 1);
      const unsigned char* const tile = smem + (t & 1) * S::kKeys * CR * 16;
#pragma unroll
      for (int sub = 0; sub < S::kKeys / 32 / S::KW; ++sub) {
        const int first = (S::KW == 1 ? sub : kw) * 32, kb0 = key0 + t * S::kKeys + first;
        f32x16_t s[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n] = f32x16_t{};
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
          const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(tile + place<D>(first + col, 2 * kk + half));
#pragma unroll
          for (int n = 0; n < NB; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[n][kk], s[n], 0, 0, 0);
        }
        if (kb0 + 31 > pos_min || absent) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = kb0 + 8 * (r >> 2) + 4 * half + (r & 3);
            const bool there = !absent || on_a_page(a, table, max(min(key, kend - 1), 0));
#pragma unroll
            for (int n = 0; n < NB; ++n)
              if (key > pos[n] || !there) s[n][r] = -__builtin_inff();
          }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float mx = s[n][0];
#pragma unroll
          for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
          mx = half_max(mx) * a.scale_log2;
          if (__builtin_amdgcn_ballot_w64(mx > m_run[n] + 8.0f) != 0) {
            const float m_new = fmaxf(m_run[n], mx);
            l_run[n] *= m_new == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m_run[n] - m_new);
            m_run[n] = m_new;
          }
          const float m_sub = m_run[n] == -__builtin_inff() ? 0.0f : m_run[n];
          float sum = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], a.scale_log2, -m_sub));
          l_run[n] += sum;
        }
      }
      if (t + 1 < nt) store(t + 1);
      __syncthreads();
    }

    float* const part = a.part + item * (2 * S::kRows);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float m = m_run[n], l = half_sum(l_run[n]);
      if constexpr (S::KW > 1) {  // the key parts of these rows
        float* const ml = reinterpret_cast<float*>(smem);
        if (half == 0) ml[(wave * 32 + col) * 2] = m, ml[(wave * 32 + col) * 2 + 1] = l;
        __syncthreads();
        if (wave == 0) {
#pragma unroll
          for (int v = 1; v < S::KW; ++v) {
            const float m2 = ml[(v * 32 + col) * 2], l2 = ml[(v * 32 + col) * 2 + 1];
            const float top = fmaxf(m, m2), sub = top == -__builtin_inff() ? 0.0f : top;
            l = l * __builtin_amdgcn_exp2f(m - sub) + l2 * __builtin_amdgcn_exp2f(m2 - sub);
            m = top;
          }
        }
      }
      if (half == 0 && (S::KW == 1 || wave == 0)) {
        const int row = (rw * NB + n) * 32 + col;
        part[row * 2] = m;
        part[row * 2 + 1] = l;
      }
    }
  }
}

// Key sums: every wavefront holds 32 keys in registers; rows stream by in tiles of 32.
template <int D, Format F, class S>
__global__ __launch_bounds__(kThreads) void key_sums_kernel(WeightArgs a) {
  constexpr int CR = D / 8, kSteps = D / 16, kKeys = 32 * kWaves, kRows = 32;
  constexpr int kTile = kRows * CR * 16, kMoves = kRows * CR / kThreads;
  static_assert(kMoves >= 1 && kKeys * CR * 16 >= 2 * kTile, "LDS holds the keys first, then two tiles of rows");
  __shared__ __attribute__((aligned(16))) unsigned char smem[kKeys * CR * 16];
  __shared__ __attribute__((aligned(16))) float row_m[2][kRows], row_inv[2][kRows];
  __shared__ __attribute__((aligned(16))) int row_pos[2][kRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int c = uniform(range_tiles<S>(a, lane));
  auto tiles = [&](const Req& x) { return over(static_cast<int64_t>(x.n_new) * a.group, S::kRows); };
  auto ranges = [&](const Req& x) { return max(over(over(x.len, S::kKeys), c), 1); };
  for (int64_t item = blockIdx.x;; item += gridDim.x) {
    int req;
    int64_t base;
    auto count = [&](const Req& x) { return x.n_new > 0 ? over(x.len, kKeys) * a.kv_heads : 0; };
    if (!find_request(a, lane, item, count, &req, &base)) return;
    const Req x = request(a, req);
    const int k = uniform(static_cast<int>(item - base)), n_kt = uniform(over(x.len, kKeys));
    const int head = k / n_kt, key0 = (k % n_kt) * kKeys;
    const int slot = uniform(owned_slot(a.index, req, a.w_rows, lane));
    if (slot < 0) continue;
    const int32_t* const table = a.c.table + req * a.c.table_stride;
    // first item of the request in the row stats
    int64_t stats = 0;
    for (int r0 = 0; r0 < req; r0 += 64) {
      const Req y = request(a, r0 + lane);
      stats += r0 + lane < req ? static_cast<int64_t>(tiles(y)) * ranges(y) * a.kv_heads : 0;
    }
    stats = wave_total(stats);
    const int n_rt = tiles(x), n_ranges = ranges(x), rows = x.n_new * a.group;

    // ---- the keys, through LDS into registers
    __syncthreads();  // the item before has read its tiles
#pragma unroll
    for (int i = 0; i < kKeys * CR / kThreads; ++i) {
      const int at = i * kThreads + tid;
      const auto in = load_chunk<D, F>(a, table, head, min(key0 + at / CR, x.len - 1), at % CR);
      *reinterpret_cast<bf16x8_t*>(smem + place<D>(at / CR, at % CR)) = decoded<D, F>(in);
    }
    __syncthreads();
    bf16x8_t kf[kSteps];
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) kf[kk] = *reinterpret_cast<const bf16x8_t*>(smem + place<D>(wave * 32 + col, 2 * kk + half));
    __syncthreads();
    const int key = key0 + wave * 32 + col;

    // ---- the rows that see the first key, tile by tile
    const int first = max(0, min(key0 - (x.len - x.n_new), x.n_new)) * a.group / kRows, nt = over(rows, kRows);
    bf16x8_t in[kMoves];
    float in_m = 0.0f, in_inv = 0.0f;
    int in_pos = -1;
    auto load = [&](int t) {
#pragma unroll
      for (int i = 0; i < kMoves; ++i) {
        const int at = i * kThreads + tid;
        in[i] = *reinterpret_cast<const bf16x8_t*>(row_of(a, x, req, head, min(t * kRows + at / CR, rows - 1)).q + at % CR * 8);
      }
      if (tid < kRows) {  // the row's maximum and denominator over all ranges
        const int row = t * kRows + tid, rtile = min(row, rows - 1) / S::kRows;
        const int kend = seen_by(a, x, min((rtile + 1) * S::kRows, rows) - 1);
        const int n = max(1, over(over(kend, S::kKeys), c));
        const int64_t slot0 = stats + static_cast<int64_t>(head) * n_ranges * n_rt + rtile;
        const float* const p = a.part + slot0 * (2 * S::kRows) + (min(row, rows - 1) - rtile * S::kRows) * 2;
        // (every part has its place but those of an offset table that is not ascending)
        const bool held = slot0 >= 0 && slot0 + static_cast<int64_t>(n - 1) * n_rt < a.part_items;
        float m = -__builtin_inff(), l = 0.0f;
        for (int i = 0; i < (held ? n : 0); ++i) {
          const float m2 = p[static_cast<int64_t>(i) * n_rt * (2 * S::kRows)], l2 = p[static_cast<int64_t>(i) * n_rt * (2 * S::kRows) + 1];
          const float top = fmaxf(m, m2), sub = top == -__builtin_inff() ? 0.0f : top;
          l = l * __builtin_amdgcn_exp2f(m - sub) + l2 * __builtin_amdgcn_exp2f(m2 - sub);
          m = top;
        }
        in_m = m == -__builtin_inff() ? 0.0f : m;
        in_inv = l == 0.0f ? 0.0f : 1.0f / l;
        in_pos = row < rows ? x.len - x.n_new + row / a.group : -1;
      }
    };
    auto store = [&](int t) {
#pragma unroll
      for (int i = 0; i < kMoves; ++i) {
        const int at = i * kThreads + tid;
        *reinterpret_cast<bf16x8_t*>(smem + (t & 1) * kTile + place<D>(at / CR, at % CR)) = in[i];
      }
      if (tid < kRows) row_m[t & 1][tid] = in_m, row_inv[t & 1][tid] = in_inv, row_pos[t & 1][tid] = in_pos;
    };
    float sum = 0.0f;
    if (first < nt) {
      load(first);
      store(first);
    }
    __syncthreads();
    for (int t = first; t < nt; ++t) {
      if (t + 1 < nt) load(t + 1);
      f32x16_t s = f32x16_t{};
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk) {
        const bf16x8_t qf = *reinterpret_cast<const bf16x8_t*>(smem + (t & 1) * kTile + place<D>(col, 2 * kk + half));
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf, kf[kk], s, 0, 0, 0);
      }
      float tile_sum = 0.0f;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int row = 8 * r4 + 4 * half;
        const f32x4_t m = *reinterpret_cast<const f32x4_t*>(&row_m[t & 1][row]), inv = *reinterpret_cast<const f32x4_t*>(&row_inv[t & 1][row]);
        const int4 pos = *reinterpret_cast<const int4*>(&row_pos[t & 1][row]);
        const int ps[4] = {pos.x, pos.y, pos.z, pos.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * r4 + e], a.scale_log2, -m[e])) * inv[e];
          tile_sum += key <= ps[e] ? p : 0.0f;
        }
      }
      sum += tile_sum;
      if (t + 1 < nt) store(t + 1);
      __syncthreads();
    }
    sum = half_sum(sum);
    if (half == 0 && key < x.len && on_a_page(a, table, key)) a.w[slot * a.w_row + head * a.w_head + key] += sum;
  }
}

// The kernels of a call, and its items and workspace, whatever the lengths turn out to be.
struct Plan {
  bool few;
  int target;
  int64_t items, bytes;
};
Plan plan_of(int64_t requests, int64_t tokens, int group, int kv_heads, int max_rows) {
  Plan p;
  p.few = max_rows <= 64;
  const int rows = p.few ? Few::kRows : Many::kRows;
  p.target = 1024;
  // a share alone may add a range per row tile
  p.items = p.target + kv_heads * (tokens * group / rows + requests);
  p.bytes = p.items * rows * 8;
  return p;
}

int check_sizes(const char* what, int batch, int q_heads, int kv_heads, int seq_len, int n_seqs, int max_seqlen, int last) {
  FD_REQUIRE(batch >= 0 && seq_len >= 0 && q_heads >= 1 && kv_heads >= 1 && q_heads % kv_heads == 0 && n_seqs >= 0,
             FD_ERR_INVALID_ARGUMENT, "%s: sizes must be >= 0 and q_heads a multiple of kv_heads >= 1", what);
  FD_REQUIRE(n_seqs == 0 || batch == 1, FD_ERR_INVALID_ARGUMENT, "%s: cu_seqlens requires batch == 1", what);
  FD_REQUIRE(q_heads / kv_heads <= 2048, FD_ERR_UNSUPPORTED, "%s: at most 2048 query heads per key head", what);
  FD_REQUIRE(max_seqlen >= 0 && max_seqlen <= seq_len && last >= 0, FD_ERR_INVALID_ARGUMENT,
             "%s: max_seqlen must be in [0, seq_len] and last >= 0", what);
  FD_REQUIRE(static_cast<int64_t>(batch) * seq_len * q_heads < (1LL << 30), FD_ERR_UNSUPPORTED,
             "%s: batch * seq_len * q_heads must be below 2^30", what);
  return FD_OK;
}

}  // namespace

extern "C" int64_t fd_paged_key_weights_workspace_bytes(int batch, int q_heads, int kv_heads, int seq_len, int n_seqs,
                                                        int max_seqlen, int last) {
  static const char* what = "fd_paged_key_weights_workspace_bytes";
  if (int rc = check_sizes(what, batch, q_heads, kv_heads, seq_len, n_seqs, max_seqlen, last)) return rc;
  const int group = q_heads / kv_heads, top = last > 0 ? std::min(last, max_seqlen) : max_seqlen;
  return plan_of(n_seqs > 0 ? n_seqs : batch, static_cast<int64_t>(batch) * seq_len, group, kv_heads,
                 static_cast<int>(std::min<int64_t>(static_cast<int64_t>(top) * group, 1 << 30))).bytes;
}

extern "C" int fd_paged_key_weights(const void* q, const fd_paged_cache* cache, float* weights, const int64_t q_strides[4],
                                    const int64_t weight_strides[2], int weight_rows, const int32_t* row_indices, int batch,
                                    int q_heads, int seq_len, float scale, int last, const int32_t* cu_seqlens, int n_seqs,
                                    int max_seqlen, void* workspace, int64_t workspace_bytes, void* stream) {
  static const char* what = "fd_paged_key_weights";
  FD_REQUIRE(q && weights && q_strides && weight_strides, FD_ERR_INVALID_ARGUMENT, "%s: tensors and strides must be non-null", what);
  WeightArgs a;
  if (int rc = fill_view(what, cache, true, &a.c)) return rc;
  FD_REQUIRE((cu_seqlens != nullptr) == (n_seqs > 0), FD_ERR_INVALID_ARGUMENT, "%s: cu_seqlens and n_seqs >= 1 come together", what);
  if (int rc = check_sizes(what, batch, q_heads, cache->kv_heads, seq_len, n_seqs, max_seqlen, last)) return rc;
  FD_REQUIRE(scale > 0.0f && scale < 1e30f, FD_ERR_INVALID_ARGUMENT, "%s: scale must be positive", what);
  FD_REQUIRE(fd_aligned16(q) && q_strides[3] == 1 && q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0 && q_strides[2] % 8 == 0,
             FD_ERR_ALIGNMENT, "%s: rows must be contiguous and 16-byte aligned", what);
  const int requests = n_seqs > 0 ? n_seqs : batch;
  FD_REQUIRE(weight_rows >= 0 && (row_indices || weight_rows >= requests), FD_ERR_INVALID_ARGUMENT,
             "%s: the weights need a row for every request", what);
  FD_REQUIRE(weight_strides[0] >= 0 && weight_strides[1] >= 0, FD_ERR_INVALID_ARGUMENT, "%s: weight strides must be >= 0", what);
  if (requests == 0 || seq_len == 0) return FD_OK;
  const int group = q_heads / cache->kv_heads, top = last > 0 ? std::min(last, max_seqlen) : max_seqlen;
  const Plan p = plan_of(requests, static_cast<int64_t>(batch) * seq_len, group, cache->kv_heads,
                         static_cast<int>(std::min<int64_t>(static_cast<int64_t>(top) * group, 1 << 30)));
  FD_REQUIRE(workspace && fd_aligned16(workspace) && workspace_bytes >= p.bytes, FD_ERR_INVALID_ARGUMENT,
             "%s: the workspace must be 16-byte aligned and hold %lld bytes", what, static_cast<long long>(p.bytes));
  a.q = static_cast<const uint16_t*>(q);
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i];
  a.cu = cu_seqlens;
  a.index = row_indices;
  a.w = weights;
  a.w_row = weight_strides[0];
  a.w_head = weight_strides[1];
  a.n_req = requests;
  a.seq_len = seq_len;
  a.group = group;
  a.kv_heads = cache->kv_heads;
  a.last = last > 0 ? last : seq_len;
  a.w_rows = weight_rows;
  a.target = p.target;
  a.part_items = static_cast<int>(std::min<int64_t>(p.items, 0x7fffffff));
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part = static_cast<float*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_kind(cache, [&](auto d, auto f) {
    constexpr int D = decltype(d)::value;
    constexpr Format F = decltype(f)::value;
    auto go = [&](auto kind) {
      using S = decltype(kind);
      const dim3 grid(static_cast<unsigned>(std::min<int64_t>(p.items, 2048)));
      hipLaunchKernelGGL((row_stats_kernel<D, F, S>), grid, dim3(kThreads), 0, s, a);
      hipLaunchKernelGGL((key_sums_kernel<D, F, S>), dim3(2048), dim3(kThreads), 0, s, a);
    };
    if (p.few) go(Few{});
    else go(Many{});
  });
  return fd_check_launch(what);
}
