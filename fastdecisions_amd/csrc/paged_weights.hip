// The attention weight that cached keys draw from new tokens, gfx950 (bf16 MFMA, fp32 sums).
//
//   w[r, h, j] += sum over rows p of head h of exp(s_pj - m_p) / l_p,   s = scale q_p . k_j
//
// with m_p, l_p a row's maximum and denominator over the keys that it sees.  A sum over rows needs every row's
// denominator first.
//
// Many rows: two kernels, each one product Q K^T with one exponential per score, the operand that stays in registers and
// the other one through a ring of tiles in LDS:
//
//   row stats   m and l of every row over ranges of keys (S^T = K Q^T: a lane's scores are of one row); 256 rows of a
//               workgroup, ranges joined by a launch of their own
//   key sums    the rows' probabilities summed key by key (S = Q K^T: a lane's scores are of one key); 256 keys of a
//               workgroup, cut into ranges of rows, joined likewise
//
// The wavefronts of a SIMD fall into step, so a loop of products and then exponentials leaves one unit idle at a time:
// the products of a block are written between the exponentials of the one before, slot by slot, held there by
// scheduling barriers.  A slot (one 32x32x16 product, 2 scores of exponential and sums) takes about 41 cycles of a SIMD,
// the product alone 32; a row's maximum is looked for only where a block's sum shows that it is needed.  2900 tokens on
// 2048 keys, 16/4 heads x 128 (41.6 GFLOP a product): 67.5 + 4.7 + 74.5 + 6.4 us of kernels, 135 a call; without the ring
// and the ranges of rows 870, with maxima of every block 195, with products first and exponentials after them 177.  Beyond
// the loops: 7 to 9 us until the first product (finding the item, Q or K into registers, three tiles), and ranges that
// end before the longest one.
//
// Few rows (up to 16 of a key head in a request, kMostScores): K is read once.
//
//   scores      S^T in fp32 into the workspace and the rows' (m, l) over the item's keys; streaming, no LDS
//   scores add  the ranges joined, exp(s - m) / l summed over the rows; w read and written
//
// The scores' rows are as wide as the page table, which is all that the host knows of the lengths.  A table so wide that they
// would pass kMostScores takes the two kernels above: a token each of 64 requests of 256 to 8192 keys behind up to 1024 pages
// of 64 takes 40, 27 and 22 us a call (bf16, e4m3, 4 bits), behind 1025 pages 108, 105 and 98.
//
// bound by K's bytes and, for short calls, by the chain from lengths to items to pages (3.5 us).  A token each of 64
// requests of 256 to 8192 keys (4 bits, 16/4 x 128, 37 MB): 15.7 + 6.4 us; by the two kernels above 94.  64 x 8192 keys:
// bf16 144 us (3.7 TB/s of K alone, the scores are 67 MB more), 4 bits 48.
//
// Items: workgroups do not start alike when their times differ, and a few more than the card holds at once cost a whole
// round, so every workgroup sums up the requests (a lane each), picks the range that makes the items fill whole rounds
// (tiles_of_item, fit) and finds its own; only items that exist are counted.  Everything is added in an order that the
// sizes fix: no atomics.
#include <algorithm>
#include <type_traits>

#include "mfma_types.h"
#include "paged_common.h"
#include "state_slot.h"
#include "wave_tools.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kCus = 256;
constexpr int kMostKeys = 1 << 27, kMostRows = 1 << 30;  // of a request
constexpr int64_t kMostScores = 1LL << 28;  // bytes of kept scores at the page table's width: what the last-level cache may hold

struct WeightArgs {
  PagedView c;                  // K alone
  const uint16_t* q;
  int64_t qs[3];                // b, h, t
  const int32_t* cu;
  const int32_t* index;         // or null
  float* w;
  int64_t w_row, w_head;
  int n_req, seq_len, group, kv_heads, last, w_rows;
  float scale_log2;
  int stats_items, sums_items;  // items that each kernel cuts its work into at most, but for one per tile that stays
  int slots;                    // workgroups that run at once
  int part_items;               // items of the row stats whose places the workspace holds
  int32_t* cuts;                // what the kernels before have cut by: row stats (or scores), key sums
  float* part;                  // per item of the row stats: its rows' (m, l)
  float* scores;                // [heads, tokens of the call x group, score_stride], few rows
  int64_t score_stride;
  float* stats;                 // [heads, tokens of the call x group]: (m, 1 / l) of every row over all its keys
  float* sums;                  // per item of the key sums of a request cut into row ranges: its keys' sums
};

// Row stats: a wavefront holds two blocks of 32 rows; keys stream by through a ring of tiles.
template <int D_>
struct Stats {
  static constexpr int D = D_, NB = 2;
  static constexpr int kRows = 32 * NB * kWaves;
  static constexpr int kSubs = D == 256 ? 1 : D == 128 ? 2 : 4;  // blocks of 32 keys of a tile
  static constexpr int kKeys = 32 * kSubs;
  static constexpr int kTileBytes = kKeys * D * 2;
  static constexpr int kRing = 4;
  // how far ahead of its products a tile is there: its first operands are read a block of keys before
  static constexpr int kEarly = kSubs == 1 ? 1 : 0;
};

// Key sums: every wavefront holds 64 keys; rows stream by in tiles of 32 through a ring of eight.
constexpr int kSumKeys = 64 * kWaves, kSumRows = 32, kSumRing = 8;
constexpr int kInfoRows = 1024;  // rows whose maxima and denominators are in LDS at a time

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

// All requests: the first 64 are loaded once, a lane each.
struct Requests {
  Req first;
  __device__ __forceinline__ Requests(const WeightArgs& a, int lane) : first(request(a, lane)) {}
  __device__ __forceinline__ Req lanes(const WeightArgs& a, int r0, int lane) const { return r0 == 0 ? first : request(a, r0 + lane); }
  __device__ __forceinline__ Req one(const WeightArgs& a, int r) const {  // r is uniform
    Req x = first;
    if (r >= 64) x = request(a, r);
    const int l = r < 64 ? r : 0;
    return {__builtin_amdgcn_readlane(x.start, l), __builtin_amdgcn_readlane(x.n_new, l), __builtin_amdgcn_readlane(x.len, l)};
  }
};

__device__ __forceinline__ int over(int x, int n) { return static_cast<int>((static_cast<uint32_t>(x) + n - 1) / static_cast<uint32_t>(n)); }

__device__ __forceinline__ int64_t wave_total(int64_t v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// What a kernel's cut needs of a request: pairs of tiles of a key head, those of them that are seen (about), and the tiles
// of the operand that stays, each of which wastes half a range or so.
struct Size {
  int64_t pairs;
  float seen, stays;
};
// Streamed tiles of an item.  Items that just fill m rounds of the workgroups that run at once take m (c + overhead) tiles of
// time, and the best of a few m is taken; a few items more than workgroups would cost a whole round.  `items` bounds them
// whatever the estimate: no more than that many places (and one per tile that stays) are needed.  `most`: what holds any
// request whole.
template <typename SizeOf>
__device__ __forceinline__ int tiles_of_item(const WeightArgs& a, const Requests& all_req, int lane, int items, int least, int most, int overhead, SizeOf size_of) {
  constexpr int kRounds = 4;
  Size all{0, 0.0f, 0.0f};
  for (int r0 = 0; r0 < a.n_req; r0 += 64) {
    const Req x = all_req.lanes(a, r0, lane);
    if (x.n_new == 0) continue;
    const Size y = size_of(x);
    all.pairs += y.pairs, all.seen += y.seen, all.stays += y.stays;
  }
  const int64_t pairs = wave_total(all.pairs) * a.kv_heads;
  const float seen = fd_xor_sum_up<64>(all.seen) * static_cast<float>(a.kv_heads);
  const float stays = fd_xor_sum_up<64>(all.stays) * static_cast<float>(a.kv_heads);
  float best = 1e9f, cost = 1e30f;  // without room for any cut: whole
#pragma unroll
  for (int m = 1; m <= kRounds; ++m) {
    const float room = static_cast<float>(m * a.slots) - 0.6f * stays;
    if (room < 1.0f) continue;
    const float c = ceilf(seen / room), now = static_cast<float>(m) * (c + static_cast<float>(overhead));
    if (now < cost) best = c, cost = now;
  }
  const int64_t floor = max((pairs + items - 1) / items, static_cast<int64_t>(least));
  return uniform(static_cast<int>(max(min(static_cast<int64_t>(best), static_cast<int64_t>(most)), min(floor, static_cast<int64_t>(most)))));
}

// Request that holds item `at` when request r has count(r) items: false if none does; *base: items before it.
template <typename Count>
__device__ __forceinline__ bool find_request(const WeightArgs& a, const Requests& all, int lane, int at, Count count, int* req, int* base) {
  int before = 0;
  for (int r0 = 0; r0 < a.n_req; r0 += 64) {
    const int mine = r0 + lane < a.n_req ? count(all.lanes(a, r0, lane)) : 0;
    const int incl = wave_scan(mine);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + incl > at);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      *req = uniform(r0 + l);
      *base = before + __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(mine, l);
      return at >= *base;  // sums past 31 bits: only of an offset table that is not ascending
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// Items of the requests before `req`.
template <typename Count>
__device__ __forceinline__ int items_before(const WeightArgs& a, const Requests& all, int lane, int req, Count count) {
  int n = 0;
  for (int r0 = 0; r0 < req; r0 += 64) n += __builtin_amdgcn_readlane(wave_scan(r0 + lane < req ? count(all.lanes(a, r0, lane)) : 0), 63);
  return n;
}

// The estimate put right: a few items more than whole rounds of workgroups are made fewer.
template <class C>
__device__ __forceinline__ void fit(C& cut, const WeightArgs& a, const Requests& all, int lane) {
  for (int i = 0; i < 4; ++i) {
    const int n = items_before(a, all, lane, a.n_req, [&](const Req& x) { return cut.items(a, x); });
    const int more = n & (a.slots - 1);  // of the last round
    if (n <= a.slots || n > 4 * a.slots || more == 0 || 8 * more > a.slots) break;
    cut.c += max(cut.c >> 4, 1);
  }
}

// How the row stats cut a request.
template <class S>
struct Cut {
  int c;  // key tiles of a range
  __device__ __forceinline__ Cut(const WeightArgs& a, const Requests& all, int lane)
      : c(tiles_of_item(a, all, lane, a.stats_items, 256 / S::kKeys, kMostKeys / S::kKeys, 5, [&](const Req& x) {
          const int rt = over(x.n_new * a.group, S::kRows), kt = over(x.len, S::kKeys);
          const float mean = 0.5f * static_cast<float>(min(x.len, x.len - x.n_new + S::kRows / a.group) + x.len);
          return Size{static_cast<int64_t>(rt) * kt, static_cast<float>(rt) * (mean / S::kKeys + 0.5f), static_cast<float>(rt)};
        })) {
    fit(*this, a, all, lane);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.cuts[0] = c;
  }
  __device__ __forceinline__ explicit Cut(const WeightArgs& a) : c(scalar_load(a.cuts, 0)) {}
  __device__ __forceinline__ int rtiles(const WeightArgs& a, const Req& x) const { return over(x.n_new * a.group, S::kRows); }
  __device__ __forceinline__ int ranges(const Req& x) const { return max(over(over(x.len, S::kKeys), c), 1); }
  // first row tile with keys in range v: later tokens see more keys
  __device__ __forceinline__ int rtile0(const WeightArgs& a, const Req& x, int v) const {
    const int rows = max(v * c * S::kKeys - (x.len - x.n_new), 0) * a.group;  // of the tokens that see none of the range
    return v == 0 ? 0 : min(rows / S::kRows, rtiles(a, x));
  }
  __device__ __forceinline__ int per_head(const WeightArgs& a, const Req& x) const {
    int n = 0;
    for (int v = 0; v < ranges(x); ++v) n += rtiles(a, x) - rtile0(a, x, v);
    return n;
  }
  __device__ __forceinline__ int items(const WeightArgs& a, const Req& x) const { return x.n_new > 0 ? per_head(a, x) * a.kv_heads : 0; }
};

// 16 bytes of codes (or bf16) of a cached row, as bf16 in pieces of eight.
template <Format F>
constexpr int kWordChunks = F == kBf16 ? 1 : F == kE4m3 ? 2 : 4;
template <Format F>
__device__ __forceinline__ void decode(const uint4& w, float s, bf16x8_t (&out)[kWordChunks<F>]) {
  if constexpr (F == kBf16) {
    out[0] = __builtin_bit_cast(bf16x8_t, w);
  } else if constexpr (F == kE2m1) {
    out[0] = e2m1_to_bf16(w.x, s), out[1] = e2m1_to_bf16(w.y, s), out[2] = e2m1_to_bf16(w.z, s), out[3] = e2m1_to_bf16(w.w, s);
  } else {
    auto eight = [&](uint32_t lo, uint32_t hi) {
      const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
      const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
      return bf16x8_t{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    };
    out[0] = eight(w.x, w.y), out[1] = eight(w.z, w.w);
  }
}

__device__ __forceinline__ int valid_page(const WeightArgs& a, int page) {  // page 0 for none: such keys are masked
  return static_cast<unsigned>(page) < static_cast<unsigned>(a.c.n_pages) ? page : 0;
}
__device__ __forceinline__ bool on_a_page(const WeightArgs& a, const int32_t* table, int key) {
  return static_cast<unsigned>(table[key >> a.c.shift]) < static_cast<unsigned>(a.c.n_pages);
}
template <Format F, int D>
__device__ __forceinline__ const uint8_t* scales_of(const WeightArgs& a, int page, int head, int at) {
  return a.c.k_scale + page * a.c.s_page + head * a.c.s_head + at * (F == kE2m1 ? D / kScaleBlock : 1);
}

// A product's step kk takes any 16 features, the same ones of both operands: lane half h those of chunk h D/16 + kk, so
// that a lane's share of a row lies in a row.  Staged rows: 8 rows in a row at one chunk lie on 8 chunks.
template <int D>
__device__ __forceinline__ int chunk_of(int kk, int half) { return half * (D / 16) + kk; }
template <int D>
__device__ __forceinline__ int place(int row, int chunk) { return (row * (D / 8) + (chunk ^ (row & 7))) * 16; }

// Address of a request's row (token, query head of the key head), tokens counted from its first counted one.
__device__ __forceinline__ const uint16_t* q_row(const WeightArgs& a, const Req& x, int req, int head, int token, int g) {
  return a.q + (a.cu == nullptr ? req : 0) * a.qs[0] + static_cast<int64_t>(head * a.group + g) * a.qs[1] +
         static_cast<int64_t>(x.start + token) * a.qs[2];
}

// Place of a request's row among the call's rows (m, 1 / l); inside them whatever the offset table holds.
__device__ __forceinline__ int64_t stat_row(const WeightArgs& a, const Req& x, int req, int head) {
  const int64_t tokens = a.cu == nullptr ? static_cast<int64_t>(a.n_req) * a.seq_len : a.seq_len;
  return (head * tokens + (a.cu == nullptr ? static_cast<int64_t>(req) * a.seq_len : 0) + x.start) * a.group;
}
__device__ __forceinline__ float2 stat_of(float m, float l) {
  return {m == -__builtin_inff() ? 0.0f : m, l == 0.0f ? 0.0f : 1.0f / l};
}

// Keys that a request's rows up to row1 see.
__device__ __forceinline__ int seen_by(const WeightArgs& a, const Req& x, int row1) {
  return max(0, min(x.len, x.len - x.n_new + row1 / a.group + 1));
}

__device__ __forceinline__ void lane_to_lds(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// The compiler's own loads of these end here: a wait of its own for them inside the loops would be one for the copies.
template <int N, int M>
__device__ __forceinline__ void loaded(bf16x8_t (&x)[N][M]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int m = 0; m < M; ++m) asm volatile("" : "+v"(x[n][m]));
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)p));
}

template <int D, Format F>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void row_stats_kernel(WeightArgs a) {
  using S = Stats<D>;
  constexpr int kSteps = D / 16, NB = S::NB, R = S::kRing;
  constexpr int kRowBytes = F == kBf16 ? 2 * D : F == kE4m3 ? D : D / 2;
  constexpr int kMoves = S::kKeys * kRowBytes / 16 / kThreads;      // 16-byte moves of a thread and tile
  constexpr int kLanes = kRowBytes / 16, kMoveRows = 64 / kLanes;  // lanes of a row, rows of a wavefront's move
  static_assert(kMoves >= 1, "a tile gives every thread a move");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[R * S::kTileBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const uint32_t lds0 = lds_address(smem);
  const Requests all(a, lane);
  const Cut<S> cut(a, all, lane);
  for (int item = blockIdx.x; item < a.part_items; item += gridDim.x) {
    int req, base;
    if (!find_request(a, all, lane, item, [&](const Req& x) { return cut.items(a, x); }, &req, &base)) return;
    const Req x = all.one(a, req);
    const int n_rt = uniform(cut.rtiles(a, x)), n_ranges = uniform(cut.ranges(x)), per_head = uniform(cut.per_head(a, x));
    const int head = uniform((item - base) / per_head);
    int rtile = item - base - head * per_head, range = 0;  // place within the head, range by range
    for (;; ++range) {
      const int first = uniform(cut.rtile0(a, x, range));
      if (rtile < n_rt - first || range + 1 == n_ranges) {
        rtile += first;
        break;
      }
      rtile -= n_rt - first;
    }
    const int row0 = rtile * S::kRows, rows = x.n_new * a.group;
    const int kend = uniform(seen_by(a, x, min(row0 + S::kRows, rows) - 1));
    const int key0 = range * cut.c * S::kKeys;
    const int nt = uniform(min(cut.c, over(max(kend - key0, 0), S::kKeys)));
    if (range > 0 && nt == 0) continue;
    const int32_t* const table = a.c.table + req * a.c.table_stride;
    bool bad = false;
    for (int i = (key0 >> a.c.shift) + lane; i <= ((min(key0 + nt * S::kKeys, kend) - 1) >> a.c.shift); i += 64)
      bad |= static_cast<unsigned>(table[i]) >= static_cast<unsigned>(a.c.n_pages);
    const bool absent = __builtin_amdgcn_ballot_w64(bad) != 0;

    // ---- tiles: bf16 rows are copied to LDS as they are, codes pass through registers.  Keys past kend repeat the last
    // one (the mask discards them).  A move's rows lie on one page, 32 of them on two.
    const unsigned char* const base_k = a.c.k + head * a.c.head;
    const int mask = (1 << a.c.shift) - 1, lrow = lane / kLanes, word = lane % kLanes;
    uint4 in[F == kBf16 ? 1 : kMoves];
    uint8_t in_scale[F == kBf16 ? 1 : kMoves];
    const uint32_t lane_at = static_cast<uint32_t>(lrow) * static_cast<uint32_t>(a.c.row);
    auto move = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kMoves; ++i) {
        const int row = (i * kWaves + wave) * kMoveRows, first = key0 + t * S::kKeys + row;
        const int first_key = uniform(min(first, kend - 1));
        int page = valid_page(a, scalar_load(table, first_key >> a.c.shift)), at;
        const unsigned char* p;
        if constexpr (kMoveRows > 16) {
          const int second = valid_page(a, scalar_load(table, uniform(min(first + 16, kend - 1)) >> a.c.shift));
          const int key = min(first + lrow, kend - 1);
          page = (key >> a.c.shift) == (first_key >> a.c.shift) ? page : second;
          at = key & mask;
          p = base_k + page * a.c.page + at * a.c.row;
        } else {
          uint32_t lane_row = lane_at;
          at = (first_key & mask) + lrow;
          if (first + kMoveRows > kend) {
            const int live = max(0, min(lrow, kend - 1 - first));
            lane_row = static_cast<uint32_t>(live) * static_cast<uint32_t>(a.c.row);
            at += live - lrow;
          }
          p = base_k + (page * a.c.page + (first_key & mask) * a.c.row) + lane_row;
        }
        if constexpr (F == kBf16) {
          lane_to_lds(p + (word ^ ((row + lrow) & 7)) * 16, lds0 + static_cast<uint32_t>((t & (R - 1)) * S::kTileBytes + (i * kWaves + wave) * 1024));
        } else {
          in[i] = reinterpret_cast<const uint4*>(p)[word];
          in_scale[i] = scales_of<F, D>(a, page, head, at)[F == kE2m1 ? word : 0];
        }
      }
    };
    auto store = [&](int t) __attribute__((always_inline)) {
      if constexpr (F != kBf16) {
#pragma unroll
        for (int i = 0; i < kMoves; ++i) {
          bf16x8_t y[kWordChunks<F>];
          decode<F>(in[i], scale_of(in_scale[i]), y);
#pragma unroll
          for (int u = 0; u < kWordChunks<F>; ++u)
            *reinterpret_cast<bf16x8_t*>(smem + (t & (R - 1)) * S::kTileBytes + place<D>((i * kWaves + wave) * kMoveRows + lrow, word * kWordChunks<F> + u)) = y[u];
        }
      }
    };
    // Tile t + 1 (+ kEarly) is there for every wavefront, and tile t - 1 is read, whose stage is the next move's.
    constexpr int E = S::kEarly;
    auto advance = [&](int t) __attribute__((always_inline)) {
      if constexpr (F == kBf16) {
        if (E == 0 && t + 2 < nt) wait_copies<kMoves>();
        else wait_copies<0>();
        __syncthreads();
        if (t + 3 < nt) move(t + 3);
      } else {
        __syncthreads();
        if (t + 2 + E < nt) store(t + 2 + E);
        if (t + 3 + E < nt) move(t + 3 + E);
      }
    };
    __syncthreads();  // the item before has read its tiles
    if constexpr (F == kBf16) {
#pragma unroll
      for (int u = 0; u < 3; ++u)
        if (u < nt) move(u);
    } else {
#pragma unroll
      for (int u = 0; u < 2 + E; ++u) {
        if (u >= nt) continue;
        move(u);
        store(u);
      }
      if (nt > 2 + E) move(2 + E);
    }

    int pos[NB];
    bf16x8_t qf[NB][kSteps];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int row = min(row0 + (wave * NB + n) * 32 + col, rows - 1), token = row / a.group;
      const uint16_t* const q = q_row(a, x, req, head, token, row - token * a.group);
      pos[n] = x.len - x.n_new + token;
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk) qf[n][kk] = *reinterpret_cast<const bf16x8_t*>(q + chunk_of<D>(kk, half) * 8);
    }
    loaded(qf);
    float m_run[NB], l_run[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) m_run[n] = -__builtin_inff(), l_run[n] = 0.0f;

    // ---- blocks of 32 keys, S::kSubs per tile
    constexpr int kAhead = 4, kSlots = NB * kSteps, kScores = 16 * NB, kPer = kScores >= kSlots ? kScores / kSlots : 1;
    static_assert(kScores % kSlots == 0 || kSlots % kScores == 0, "scores per product");
    auto operand = [&](int block, int kk) __attribute__((always_inline)) {
      const unsigned char* const tile = smem + ((block / S::kSubs) & (R - 1)) * S::kTileBytes;
      return *reinterpret_cast<const bf16x8_t*>(tile + place<D>((block % S::kSubs) * 32 + col, chunk_of<D>(kk, half)));
    };
    f32x4_t sums[NB];  // four side by side: a chain of 16 additions would take as long as the block's products
    float m_sub[NB];
    auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < NB; ++n) sums[n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, m_sub[n] = m_run[n];
    };
    auto score = [&](int i, const f32x16_t (&s)[NB]) __attribute__((always_inline)) {
      const int n = i % NB, r = i / NB;
      float y = sums[n][r & 3] + __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], a.scale_log2, -m_sub[n]));
      asm volatile("" : "+v"(y));  // computed here, not sunk towards the block's end
      sums[n][r & 3] = y;
    };
    // A row's maximum may lag: its exponentials are summed as they are while they stay far from fp32's end, which their sum
    // shows.  Only a row's first keys, and keys 2^64 above its maximum, take the maximum first.
    auto finish = [&](const f32x16_t (&s)[NB]) __attribute__((always_inline)) {
      float sum[NB];
      bool far = false;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        sum[n] = (sums[n][0] + sums[n][1]) + (sums[n][2] + sums[n][3]);
        far |= !(sum[n] < 0x1p64f);
      }
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(far) != 0, 0)) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float mx = s[n][0];
#pragma unroll
          for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
          mx = half_max(mx) * a.scale_log2;
          const float m_new = fmaxf(m_run[n], mx), sub = m_new == -__builtin_inff() ? 0.0f : m_new;
          l_run[n] *= m_new == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m_run[n] - m_new);
          m_run[n] = m_new;
          sum[n] = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) sum[n] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], a.scale_log2, -sub));
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) l_run[n] += sum[n];
    };
    auto softmax = [&](const f32x16_t (&s)[NB]) __attribute__((always_inline)) {
      begin();
#pragma unroll
      for (int i = 0; i < kScores; ++i) score(i, s);
      finish(s);
    };
    auto products = [&](int block, f32x16_t (&s)[NB]) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n] = f32x16_t{};
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk) {
        const bf16x8_t kf = operand(block, kk);
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[n][kk], s[n], 0, 0, 0);
      }
    };
    if (F == kBf16) wait_copies<0>();
    __syncthreads();
    // tiles [0, n_full) are seen whole by every row
    const int pos_first = x.len - x.n_new + row0 / a.group;
    const int n_full = uniform(absent ? 0 : max(0, min(nt, (pos_first + 1 - key0) / S::kKeys)));
    if (n_full > 0) {
      // Products of a block between the exponentials of the one before: wavefronts of a SIMD would run the same phase side by
      // side, one unit idle at a time.
      f32x16_t sA[NB], sB[NB];
      bf16x8_t kf[kAhead];
      products(0, sA);
#pragma unroll
      for (int kk = 0; kk < kAhead; ++kk) kf[kk] = operand(1, kk);  // (of a last block: unused)
      auto step = [&](int block, f32x16_t (&sc)[NB], f32x16_t (&sn)[NB]) __attribute__((always_inline)) {  // softmax of `block`, products of the next one
        begin();
#pragma unroll
        for (int n = 0; n < NB; ++n) sn[n] = f32x16_t{};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int slot = 0; slot < kSlots; ++slot) {
          const int kk = slot / NB, n = slot % NB;
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            if (kScores >= kSlots || slot % (kSlots / kScores) == 0) score(kScores >= kSlots ? slot * kPer + i : slot / (kSlots / kScores), sc);
          sn[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk % kAhead], qf[n][kk], sn[n], 0, 0, 0);
          if (n == NB - 1) kf[kk % kAhead] = kk + kAhead < kSteps ? operand(block + 1, kk + kAhead) : operand(block + 2, kk + kAhead - kSteps);
          __builtin_amdgcn_sched_barrier(0);
        }
        finish(sc);
      };
      if constexpr (S::kSubs > 1) {
#pragma unroll 1
        for (int t = 0; t + 1 < n_full; ++t) {
          advance(t);
#pragma unroll
          for (int sub = 0; sub < S::kSubs; sub += 2) {
            step(t * S::kSubs + sub, sA, sB);
            step(t * S::kSubs + sub + 1, sB, sA);
          }
        }
        advance(n_full - 1);
#pragma unroll
        for (int sub = 0; sub < S::kSubs; sub += 2) {
          step((n_full - 1) * S::kSubs + sub, sA, sB);
          if (sub + 2 < S::kSubs) step((n_full - 1) * S::kSubs + sub + 1, sB, sA);
        }
        softmax(sB);
      } else {
        int t = 0;
#pragma unroll 1
        for (; t + 2 < n_full; t += 2) {
          advance(t);
          step(t, sA, sB);
          advance(t + 1);
          step(t + 1, sB, sA);
        }
        if (t + 1 < n_full) {
          advance(t);
          step(t, sA, sB);
#pragma unroll
          for (int n = 0; n < NB; ++n) sA[n] = sB[n];
        }
        advance(n_full - 1);
        softmax(sA);
      }
    }
#pragma unroll 1
    for (int t = n_full; t < nt; ++t) {
      advance(t);
#pragma unroll 1
      for (int sub = 0; sub < S::kSubs; ++sub) {
        const int kb0 = key0 + t * S::kKeys + sub * 32;
        f32x16_t s[NB];
        products(t * S::kSubs + sub, s);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kb0 + 8 * (r >> 2) + 4 * half + (r & 3);
          const bool there = !absent || on_a_page(a, table, max(min(key, kend - 1), 0));
#pragma unroll
          for (int n = 0; n < NB; ++n)
            if (key > pos[n] || !there) s[n][r] = -__builtin_inff();
        }
        softmax(s);
      }
    }

    float* const part = a.part + static_cast<int64_t>(item) * (2 * S::kRows);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float m = m_run[n], l = half_sum(l_run[n]);
      const int row = (wave * NB + n) * 32 + col;
      if (half != 0 || row0 + row >= rows) continue;
      if (n_ranges == 1) {
        reinterpret_cast<float2*>(a.stats)[stat_row(a, x, req, head) + row0 + row] = stat_of(m, l);
      } else {
        part[row * 2] = m;
        part[row * 2 + 1] = l;
      }
    }
  }
}

// (m, 1 / l) of the rows whose keys were cut into ranges, one row tile per workgroup.
template <class S>
__global__ __launch_bounds__(S::kRows) void row_stats_join_kernel(WeightArgs a) {
  const int lane = threadIdx.x & 63;
  const Requests all(a, lane);
  const Cut<S> cut(a);
  for (int item = blockIdx.x;; item += gridDim.x) {
    int req, base;
    if (!find_request(a, all, lane, item, [&](const Req& x) { return cut.ranges(x) > 1 ? cut.rtiles(a, x) * a.kv_heads : 0; }, &req, &base)) return;
    const Req x = all.one(a, req);
    const int n_rt = uniform(cut.rtiles(a, x)), n_ranges = uniform(cut.ranges(x)), k = uniform(item - base);
    const int rtile = k % n_rt, head = k / n_rt, row0 = rtile * S::kRows, rows = x.n_new * a.group;
    const int place = uniform(items_before(a, all, lane, req, [&](const Req& y) { return cut.items(a, y); })) + head * uniform(cut.per_head(a, x)) + rtile;
    const int row = threadIdx.x;
    const float2* const p = reinterpret_cast<const float2*>(a.part) + row;
    float m = -__builtin_inff(), l = 0.0f;
    int at = place;  // of range v's first row tile, were this one that
    for (int v0 = 0; v0 < n_ranges; v0 += 4) {  // four loads in flight
      float2 y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int v = min(v0 + u, n_ranges - 1), first = cut.rtile0(a, x, v), here = at - first;
        // (every part has its place but those of an offset table that is not ascending)
        const bool seen = v0 + u < n_ranges && rtile >= first && here >= 0 && here < a.part_items;
        y[u] = float2{-__builtin_inff(), 0.0f};
        if (seen) y[u] = p[static_cast<int64_t>(here) * S::kRows];
        at += n_rt - first;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float top = fmaxf(m, y[u].x), sub = top == -__builtin_inff() ? 0.0f : top;
        l = l * __builtin_amdgcn_exp2f(m - sub) + y[u].y * __builtin_amdgcn_exp2f(y[u].x - sub);
        m = top;
      }
    }
    if (row0 + row < rows) reinterpret_cast<float2*>(a.stats)[stat_row(a, x, req, head) + row0 + row] = stat_of(m, l);
  }
}

// How the key sums cut a request: tiles of kSumKeys keys times ranges of c row tiles.
struct SumCut {
  int c;
  __device__ __forceinline__ SumCut(const WeightArgs& a, const Requests& all, int lane)
      : c(tiles_of_item(a, all, lane, a.sums_items, 4, kMostRows / kSumRows, 10, [&](const Req& x) {
          const int rt = over(x.n_new * a.group, kSumRows), kt = over(x.len, kSumKeys);
          const float fresh = 0.5f * static_cast<float>(x.n_new) / kSumKeys;  // half of the new tokens' keys are seen
          return Size{static_cast<int64_t>(rt) * kt, static_cast<float>(rt) * (static_cast<float>(kt) - fresh), static_cast<float>(kt)};
        })) {
    fit(*this, a, all, lane);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.cuts[1] = c;
  }
  __device__ __forceinline__ explicit SumCut(const WeightArgs& a) : c(scalar_load(a.cuts, 1)) {}
  __device__ __forceinline__ int ktiles(const WeightArgs& a, const Req& x) const { return x.n_new > 0 ? over(x.len, kSumKeys) * a.kv_heads : 0; }
  __device__ __forceinline__ int ranges(const WeightArgs& a, const Req& x) const { return max(over(over(x.n_new * a.group, kSumRows), c), 1); }
  // Ranges are counted from the last one on, which all key tiles have: the first `seen` key tiles have range j.
  __device__ __forceinline__ int seen(const WeightArgs& a, const Req& x, int n_ranges, int j) const {
    const int keys = x.len - x.n_new + over((n_ranges - j) * c * kSumRows, a.group);  // that the range's rows and those before see
    return min(max(over(max(keys, 0), kSumKeys), 0), over(x.len, kSumKeys));
  }
  __device__ __forceinline__ int per_head(const WeightArgs& a, const Req& x) const {
    const int n_ranges = ranges(a, x);
    int n = 0;
    for (int j = 0; j < n_ranges; ++j) n += seen(a, x, n_ranges, j);
    return n;
  }
  __device__ __forceinline__ int items(const WeightArgs& a, const Req& x) const { return x.n_new > 0 ? per_head(a, x) * a.kv_heads : 0; }
  // of requests that are cut into row ranges: their items' sums have places in the workspace, below 2 sums_items
  __device__ __forceinline__ int places(const WeightArgs& a, const Req& x) const { return ranges(a, x) > 1 ? items(a, x) : 0; }
  __device__ __forceinline__ int joins(const WeightArgs& a, const Req& x) const { return ranges(a, x) > 1 ? ktiles(a, x) : 0; }
};
// First row of a request that sees key `key` (of its counted rows).
__device__ __forceinline__ int first_row(const WeightArgs& a, const Req& x, int key) {
  return max(0, min(key - (x.len - x.n_new), x.n_new)) * a.group;
}

template <int D, Format F>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void key_sums_kernel(WeightArgs a) {
  constexpr int CR = D / 8, kSteps = D / 16, kTile = kSumRows * CR * 16, kCopies = kTile / 1024 / kWaves;
  constexpr int kRowBytes = F == kBf16 ? 2 * D : F == kE4m3 ? D : D / 2, kWords = kRowBytes / 32;  // of a lane's half row
  static_assert(kCopies >= 1, "a tile gives every wavefront a copy");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kSumRing * kTile];
  __shared__ __attribute__((aligned(16))) float row_m[kInfoRows], row_inv[kInfoRows];
  __shared__ __attribute__((aligned(16))) int row_last[kInfoRows];  // key that the row sees last
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const uint32_t lds0 = lds_address(smem);
  const Requests all(a, lane);
  const SumCut cut(a, all, lane);
  for (int item = blockIdx.x;; item += gridDim.x) {
    int req, base;
    if (!find_request(a, all, lane, item, [&](const Req& x) { return cut.items(a, x); }, &req, &base)) return;
    const Req x = all.one(a, req);
    const int n_ranges = uniform(cut.ranges(a, x)), k = uniform(item - base), per_head = uniform(cut.per_head(a, x));
    const int head = uniform(k / per_head);
    int kt = k - head * per_head, j = 0;  // place within the head, range by range
    for (;; ++j) {
      const int n = uniform(cut.seen(a, x, n_ranges, j));
      if (kt < n || j + 1 == n_ranges) break;
      kt -= n;
    }
    const int range = n_ranges - 1 - j;
    const int key0 = kt * kSumKeys, rows = x.n_new * a.group;
    const int t0 = uniform(max(first_row(a, x, key0) / kSumRows, range * cut.c));
    const int t1 = uniform(min(over(rows, kSumRows), (range + 1) * cut.c));
    if (t0 >= t1) continue;  // none of these rows sees the keys
    const int slot = uniform(owned_slot(a.index, req, a.w_rows, lane));
    if (slot < 0) continue;
    const int32_t* const table = a.c.table + req * a.c.table_stride;
    const float2* const stats = reinterpret_cast<const float2*>(a.stats) + stat_row(a, x, req, head);

    // ---- rows: tile t's are copied to stage t % kSumRing, in order; every lane's pointers move on by 32 rows (rows behind the
    // last one read the first: the mask discards them)
    const int step_tokens = uniform(kSumRows / a.group), step_rem = kSumRows - step_tokens * a.group;
    const uint16_t* const q_first = q_row(a, x, req, head, 0, 0);
    const int64_t step_bytes = 2 * (step_tokens * a.qs[2] + step_rem * a.qs[1]), wrap_bytes = 2 * (a.qs[2] - a.group * a.qs[1]);
    int copy_g[kCopies];
    const char* copy_at[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = (i * kWaves + wave) * 64 + lane, r = at / CR, row = t0 * kSumRows + r, token = row / a.group;
      copy_g[i] = row - token * a.group;
      copy_at[i] = reinterpret_cast<const char*>(q_first + token * a.qs[2] + copy_g[i] * a.qs[1] + ((at % CR) ^ (r & 7)) * 8);
    }
    auto copy = [&](int t) __attribute__((always_inline)) {
      const int left = rows - t * kSumRows;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int at = (i * kWaves + wave) * 64 + lane;
        const char* p = copy_at[i];
        if (left < kSumRows) p = at / CR < left ? p : reinterpret_cast<const char*>(q_first);
        lane_to_lds(p, lds0 + static_cast<uint32_t>((t & (kSumRing - 1)) * kTile + (i * kWaves + wave) * 1024));
        copy_at[i] += step_bytes;
        if (step_rem != 0) {
          copy_g[i] += step_rem;
          const bool wrap = copy_g[i] >= a.group;
          copy_g[i] -= wrap ? a.group : 0;
          copy_at[i] += wrap ? wrap_bytes : 0;
        }
      }
    };
    __syncthreads();  // the item before has read its tiles
#pragma unroll
    for (int u = 0; u < kSumRing - 1; ++u)
      if (t0 + u < t1) copy(t0 + u);

    // ---- this lane's keys
    bf16x8_t kf[2][kSteps];
    int key[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      key[n] = key0 + wave * 64 + n * 32 + col;
      const int held = min(key[n], x.len - 1), page = valid_page(a, table[held >> a.c.shift]), at = held & ((1 << a.c.shift) - 1);
      const uint4* const p = reinterpret_cast<const uint4*>(a.c.k + page * a.c.page + head * a.c.head + at * a.c.row) + half * kWords;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        float scale = 1.0f;
        if constexpr (F != kBf16) scale = scale_of(scales_of<F, D>(a, page, head, at)[F == kE2m1 ? half * kWords + i : 0]);
        bf16x8_t y[kWordChunks<F>];
        decode<F>(p[i], scale, y);
#pragma unroll
        for (int u = 0; u < kWordChunks<F>; ++u) kf[n][i * kWordChunks<F> + u] = y[u];
      }
    }

    loaded(kf);
    float sum[2] = {0.0f, 0.0f};
    int info0 = -1;  // first row of those in row_m
    auto info = [&](int row0) __attribute__((always_inline)) {
      if (info0 >= 0 && row0 < info0 + kInfoRows) return;
      __syncthreads();  // the rows before are done with theirs
      info0 = row0;
#pragma unroll
      for (int u = 0; u < kInfoRows / kThreads; ++u) {
        const int i = u * kThreads + tid;
        const int row = info0 + i;
        const float2 y = stats[min(row, rows - 1)];
        row_m[i] = y.x;
        row_inv[i] = y.y;
        row_last[i] = row < rows ? x.len - x.n_new + row / a.group : -1;
      }
      __syncthreads();
    };
    auto operand = [&](int t, int kk) __attribute__((always_inline)) {
      return *reinterpret_cast<const bf16x8_t*>(smem + (t & (kSumRing - 1)) * kTile + place<D>(col, chunk_of<D>(kk, half)));
    };
    // Tile t + 2 has landed for every wavefront (tile t + 1 at its first operands' reads), and tile t - 1 is read, whose
    // stage is the next copy's.
    auto advance = [&](int t) __attribute__((always_inline)) {
      if (t + 6 < t1) wait_copies<4 * kCopies>();
      else if (t + 4 < t1) wait_copies<2 * kCopies>();
      else wait_copies<0>();
      __syncthreads();
      if (t + kSumRing - 1 < t1) copy(t + kSumRing - 1);
    };
    // Scores one by one: exp(score - m) / l of row 8 r4 + 4 half + e and key block n, into four sums per block side by
    // side (a chain of 16 additions would take as long as the tile's products).
    f32x4_t tile_sum[2], mv[2], iv[2];
    int4 lv[2];
    int info_at = 0;
    auto values = [&](auto masked_c, int r4) __attribute__((always_inline)) {
      const int at = info_at + 8 * r4;
      mv[r4 & 1] = *static_cast<const f32x4_t*>(__builtin_assume_aligned(row_m + at, 16));
      iv[r4 & 1] = *static_cast<const f32x4_t*>(__builtin_assume_aligned(row_inv + at, 16));
      if constexpr (decltype(masked_c)::value) lv[r4 & 1] = *static_cast<const int4*>(__builtin_assume_aligned(row_last + at, 16));
    };
    auto score = [&](auto masked_c, int i, const f32x16_t (&s)[2]) __attribute__((always_inline)) {
      const int r4 = i / 8, e = (i / 2) % 4, n = i % 2;
      if (i % 8 == 0 && r4 < 3) values(masked_c, r4 + 1);
      float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][4 * r4 + e], a.scale_log2, -mv[r4 & 1][e]));
      y = __builtin_fmaf(y, iv[r4 & 1][e], tile_sum[n][e]);
      if constexpr (decltype(masked_c)::value) {  // (a row of NaN is none of a key that it does not see)
        const int4 l = lv[r4 & 1];
        y = key[n] <= (e == 0 ? l.x : e == 1 ? l.y : e == 2 ? l.z : l.w) ? y : tile_sum[n][e];
      }
      asm volatile("" : "+v"(y));  // computed here, not sunk towards the tile's end
      tile_sum[n][e] = y;
    };
    // Products of tile t + 1 between the exponentials of tile t: two wavefronts of a SIMD would run the same phase side by
    // side, one unit idle at a time.  (Behind the last tile they are of whatever lies in LDS, and unused.)
    constexpr int kAhead = 4, kSlots = 2 * kSteps, kPer = 32 / kSlots;
    static_assert(32 % kSlots == 0, "scores per product");
    f32x16_t sA[2], sB[2];
    bf16x8_t qf[kAhead];
    auto step = [&](auto masked_c, int t, f32x16_t (&sc)[2], f32x16_t (&sn)[2]) __attribute__((always_inline)) {
      advance(t);
      info(t * kSumRows);
      info_at = t * kSumRows - info0 + 4 * half;
      values(masked_c, 0);
      tile_sum[0] = tile_sum[1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      sn[0] = sn[1] = f32x16_t{};
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int slot = 0; slot < kSlots; ++slot) {
        const int kk = slot / 2, n = slot % 2;
#pragma unroll
        for (int i = 0; i < kPer; ++i) score(masked_c, slot * kPer + i, sc);
        sn[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qf[kk % kAhead], kf[n][kk], sn[n], 0, 0, 0);
        if (n == 1) qf[kk % kAhead] = kk + kAhead < kSteps ? operand(t + 1, kk + kAhead) : operand(t + 2, kk + kAhead - kSteps);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) sum[n] += (tile_sum[n][0] + tile_sum[n][1]) + (tile_sum[n][2] + tile_sum[n][3]);
    };
    auto run = [&](auto masked_c, int from, int to) __attribute__((always_inline)) {  // products of tile `from` are in sA, and of tile `to` afterwards
      int t = from;
#pragma unroll 1
      for (; t + 1 < to; t += 2) {
        step(masked_c, t, sA, sB);
        step(masked_c, t + 1, sB, sA);
      }
      if (t < to) {
        step(masked_c, t, sA, sB);
        sA[0] = sB[0], sA[1] = sB[1];
      }
    };
    wait_copies<0>();
    __syncthreads();
    sA[0] = sA[1] = f32x16_t{};
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
      const bf16x8_t y = operand(t0, kk);
#pragma unroll
      for (int n = 0; n < 2; ++n) sA[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, kf[n][kk], sA[n], 0, 0, 0);
    }
#pragma unroll
    for (int kk = 0; kk < kAhead; ++kk) qf[kk] = operand(t0 + 1, kk);
    // tiles [t0, whole) have rows that do not see every key, the last one may have rows behind the request's
    const int whole = uniform(min(max(over(first_row(a, x, min(key0 + kSumKeys, x.len) - 1), kSumRows), t0), t1));
    const int whole_end = uniform(max(whole, min(t1, rows / kSumRows)));
    run(std::true_type{}, t0, whole);
    run(std::false_type{}, whole, whole_end);
    run(std::true_type{}, whole_end, t1);
    int at = 0;
    if (n_ranges > 1) at = uniform(items_before(a, all, lane, req, [&](const Req& y) { return cut.places(a, y); })) + k;
    if (at < 0 || at >= 2 * a.sums_items) continue;  // only of an offset table that is not ascending
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const float y = half_sum(sum[n]);
      if (half != 0) continue;
      if (n_ranges > 1) a.sums[static_cast<int64_t>(at) * kSumKeys + wave * 64 + n * 32 + col] = y;
      else if (key[n] < x.len && on_a_page(a, table, key[n])) a.w[slot * a.w_row + head * a.w_head + key[n]] += y;
    }
  }
}

// The row ranges' sums of every key tile of the requests that are cut into such, added range by range.
__global__ __launch_bounds__(kSumKeys) void key_sums_join_kernel(WeightArgs a) {
  const int lane = threadIdx.x & 63;
  const Requests all(a, lane);
  const SumCut cut(a);
  for (int item = blockIdx.x;; item += gridDim.x) {
    int req, base;
    if (!find_request(a, all, lane, item, [&](const Req& x) { return cut.joins(a, x); }, &req, &base)) return;
    const Req x = all.one(a, req);
    const int n_ranges = uniform(cut.ranges(a, x)), k = uniform(item - base), n_kt = uniform(over(x.len, kSumKeys));
    const int kt = k % n_kt, head = k / n_kt, key = kt * kSumKeys + static_cast<int>(threadIdx.x);
    const int slot = uniform(owned_slot(a.index, req, a.w_rows, lane));
    if (slot < 0) continue;
    int at = uniform(items_before(a, all, lane, req, [&](const Req& y) { return cut.places(a, y); })) + head * uniform(cut.per_head(a, x)) + kt;
    float sum = 0.0f;
    for (int j = 0; j < n_ranges; ++j) {
      const int n = uniform(cut.seen(a, x, n_ranges, j));
      if (kt < n && at >= 0 && at < 2 * a.sums_items) sum += a.sums[static_cast<int64_t>(at) * kSumKeys + threadIdx.x];
      at += n;
    }
    if (key < x.len && on_a_page(a, a.c.table + req * a.c.table_stride, key)) a.w[slot * a.w_row + head * a.w_head + key] += sum;
  }
}

// ---------------------------------------------------------------- few rows

// How the scores cut a request: tiles of 16 rows times ranges of c tiles of kScoreKeys keys.
constexpr int kScoreRows = 16, kScoreKeys = 64 * kWaves;
struct ScoreCut {
  int c;
  __device__ __forceinline__ ScoreCut(const WeightArgs& a, const Requests& all, int lane)
      : c(tiles_of_item(a, all, lane, a.stats_items, 1, kMostKeys / kScoreKeys, 3, [&](const Req& x) {
          const int rt = rtiles(a, x), kt = over(x.len, kScoreKeys);
          return Size{static_cast<int64_t>(rt) * kt, static_cast<float>(rt * kt), static_cast<float>(rt)};
        })) {
    fit(*this, a, all, lane);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.cuts[0] = c;
  }
  __device__ __forceinline__ explicit ScoreCut(const WeightArgs& a) : c(scalar_load(a.cuts, 0)) {}
  static __device__ __forceinline__ int rtiles(const WeightArgs& a, const Req& x) { return over(x.n_new * a.group, kScoreRows); }
  __device__ __forceinline__ int ranges(const Req& x) const { return max(over(over(x.len, kScoreKeys), c), 1); }
  __device__ __forceinline__ int items(const WeightArgs& a, const Req& x) const { return rtiles(a, x) * ranges(x) * a.kv_heads; }
};

// Scores of up to 16 rows, kept in the workspace in fp32, and their rows' (m, l) over the item's keys.  Every wavefront
// takes blocks of 64 keys of its own, loaded straight into the operands' registers a block ahead: a lane's share of a
// key is every fourth word of 16 bytes (the steps of the product take any 32 features, the same ones of Q), so that
// four lanes read 64 bytes in a row.
template <int D, Format F>
constexpr int kScoreGroups = D == 256 && F == kBf16 ? 1 : D == 256 || (D == 128 && F == kBf16) ? 2 : 4;  // of a CU
template <int D, Format F>
__global__ __launch_bounds__(kThreads, (kScoreGroups<D, F>)) void key_scores_kernel(WeightArgs a) {
  constexpr int kSteps = D / 32, kRowBytes = F == kBf16 ? 2 * D : F == kE4m3 ? D : D / 2;
  constexpr int kBytes = kRowBytes / 4, kWords = kBytes < 16 ? 1 : kBytes / 16;  // of a lane and key
  constexpr int kChunks = kBytes < 16 ? 2 : kWordChunks<F>;                      // eights of features in a word
  constexpr int kScales = F == kE2m1 && D == 256 ? 2 : 1;
  using Word = std::conditional_t<kBytes < 16, uint2, uint4>;
  __shared__ float join[kWaves][kScoreRows][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int li = lane & 15, grp = lane >> 4;
  const Requests all(a, lane);
  const ScoreCut cut(a, all, lane);
  for (int item = blockIdx.x; item < a.part_items; item += gridDim.x) {
    int req, base;
    if (!find_request(a, all, lane, item, [&](const Req& x) { return cut.items(a, x); }, &req, &base)) return;
    const Req x = all.one(a, req);
    const int n_rt = uniform(cut.rtiles(a, x)), n_ranges = uniform(cut.ranges(x)), k = uniform(item - base);
    const int rtile = uniform(k % n_rt), hr = uniform(k / n_rt), range = uniform(hr % n_ranges), head = uniform(hr / n_ranges);
    const int row0 = rtile * kScoreRows, rows = x.n_new * a.group, row = min(row0 + li, rows - 1), token = row / a.group;
    const int pos = x.len - x.n_new + token, pos_min = uniform(x.len - x.n_new + row0 / a.group);
    const int32_t* const table = a.c.table + req * a.c.table_stride;
    const int first = range * cut.c * kScoreKeys + wave * 64, end = min(x.len, (range + 1) * cut.c * kScoreKeys);
    const int mask = (1 << a.c.shift) - 1;
    const unsigned char* const base_k = a.c.k + head * a.c.head + grp * sizeof(Word);

    struct Block {
      Word w[4][kWords];
      uint32_t s[4];   // E2M1: the bytes of the lane's features, E4M3: of the key
    };
    auto page_at = [&](int key) __attribute__((always_inline)) { return scalar_load(table, uniform(max(min(key, x.len - 1), 0)) >> a.c.shift); };
    auto load = [&](int kb0, Block& b) __attribute__((always_inline)) {  // keys behind the last repeat it (the mask discards them)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int page = valid_page(a, page_at(kb0 + 16 * u)), at = max(min(kb0 + 16 * u + li, x.len - 1), 0) & mask;
        const Word* const p = reinterpret_cast<const Word*>(base_k + page * a.c.page + at * a.c.row);
#pragma unroll
        for (int i = 0; i < kWords; ++i) b.w[u][i] = p[4 * i];
        if constexpr (F == kE4m3) b.s[u] = *scales_of<F, D>(a, page, head, at);
        if constexpr (F == kE2m1) {
          const uint8_t* const sp = scales_of<F, D>(a, page, head, at);
          b.s[u] = kScales == 2 ? sp[grp] | sp[4 + grp] << 8 : sp[kBytes < 16 ? grp / 2 : grp];
        }
      }
    };
    Block cur, next;
    if (first < end) load(first, cur);
    bf16x8_t qf[kSteps];
    const uint16_t* const q = q_row(a, x, req, head, token, row - token * a.group) + grp * (8 * kChunks);
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) qf[kk] = *reinterpret_cast<const bf16x8_t*>(q + (kk / kChunks * 4 * kChunks + kk % kChunks) * 8);
    float* const out = a.scores + (stat_row(a, x, req, head) + row) * a.score_stride + 4 * grp;
    float m = -__builtin_inff(), l = 0.0f;  // of this lane's keys
    for (int kb0 = first; kb0 < end; kb0 += kScoreKeys) {
      if (kb0 + kScoreKeys < end) load(kb0 + kScoreKeys, next);
      f32x4_t s[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        bf16x8_t kf[kSteps];
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          if constexpr (kBytes < 16) {
            kf[0] = e2m1_to_bf16(cur.w[u][i].x, scale_of(cur.s[u]));
            kf[1] = e2m1_to_bf16(cur.w[u][i].y, scale_of(cur.s[u]));
          } else {
            bf16x8_t y[kWordChunks<F>];
            decode<F>(cur.w[u][i], F == kBf16 ? 1.0f : scale_of(kScales == 2 ? cur.s[u] >> (8 * i) & 255u : cur.s[u]), y);
#pragma unroll
            for (int e = 0; e < kChunks; ++e) kf[i * kChunks + e] = y[e];
          }
        }
        s[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kk], qf[kk], s[u], 0, 0, 0);
      }
      bool there = true;
#pragma unroll
      for (int u = 0; u < 4; ++u) there &= static_cast<unsigned>(page_at(kb0 + 16 * u)) < static_cast<unsigned>(a.c.n_pages);
      if (kb0 + 63 > pos_min || !there) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool here = static_cast<unsigned>(page_at(kb0 + 16 * u)) < static_cast<unsigned>(a.c.n_pages);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (kb0 + 16 * u + 4 * grp + e > pos || !here) s[u][e] = -__builtin_inff();
        }
      }
      // as in the row stats: the maximum is looked for where the sum shows that it is needed
      auto exp_sum = [&](float sub) __attribute__((always_inline)) {
        f32x4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e], a.scale_log2, -sub));
        return (y[0] + y[1]) + (y[2] + y[3]);
      };
      float sum = exp_sum(m);
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum < 0x1p64f)) != 0, 0)) {
        float mx = s[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i / 4][i % 4]);
        const float m_new = fmaxf(m, mx * a.scale_log2), sub = m_new == -__builtin_inff() ? 0.0f : m_new;
        l *= m_new == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        sum = exp_sum(sub);
      }
      l += sum;
      if (row0 + li < rows) {
#pragma unroll
        for (int u = 0; u < 4; ++u) *reinterpret_cast<f32x4_t*>(out + kb0 + 16 * u) = s[u];
      }
      cur = next;
    }
    // ---- the lane groups' and the wavefronts' keys joined
    auto join2 = [](float m, float l, float m2, float l2, float* mo, float* lo) __attribute__((always_inline)) {
      const float top = fmaxf(m, m2), sub = top == -__builtin_inff() ? 0.0f : top;
      *lo = l * __builtin_amdgcn_exp2f(m - sub) + l2 * __builtin_amdgcn_exp2f(m2 - sub);
      *mo = top;
    };
#pragma unroll
    for (int d = 16; d < 64; d *= 2) {
      const float m2 = __shfl_xor(m, d), l2 = __shfl_xor(l, d);
      join2(m, l, m2, l2, &m, &l);
    }
    __syncthreads();  // the item before has read its join
    if (grp == 0) join[wave][li][0] = m, join[wave][li][1] = l;
    __syncthreads();
    if (wave == 0 && grp == 0) {
#pragma unroll
      for (int v = 1; v < kWaves; ++v) join2(m, l, join[v][li][0], join[v][li][1], &m, &l);
      reinterpret_cast<float2*>(a.part)[static_cast<int64_t>(item) * kScoreRows + li] = float2{m, l};
    }
  }
}

// The kept scores' probabilities summed key by key, kAddKeys of a request's head per workgroup.
constexpr int kAddKeys = 4 * kThreads;
__global__ __launch_bounds__(kThreads) void key_scores_add_kernel(WeightArgs a) {
  constexpr int kHold = 256;  // rows whose (m, 1 / l) are in LDS at a time
  constexpr int kAhead = 4;   // rows whose scores are asked for before those are joined
  __shared__ float2 stats[kHold];
  const int lane = threadIdx.x & 63;
  const Requests all(a, lane);
  const ScoreCut cut(a);
  for (int item = blockIdx.x;; item += gridDim.x) {
    int req, base;
    if (!find_request(a, all, lane, item, [&](const Req& x) { return x.n_new > 0 ? over(x.len, kAddKeys) * a.kv_heads : 0; }, &req, &base)) return;
    const Req x = all.one(a, req);
    const int n_kt = uniform(over(x.len, kAddKeys)), head = uniform((item - base) / n_kt), kt = item - base - head * n_kt;
    const int slot = uniform(owned_slot(a.index, req, a.w_rows, lane));
    if (slot < 0) continue;
    const int first = uniform(items_before(a, all, lane, req, [&](const Req& y) { return cut.items(a, y); }));
    const int n_rt = uniform(cut.rtiles(a, x)), n_ranges = uniform(cut.ranges(x)), rows = x.n_new * a.group;
    const int key0 = kt * kAddKeys + static_cast<int>(threadIdx.x);
    const float* const scores = a.scores + stat_row(a, x, req, head) * a.score_stride;
    float* const w = a.w + slot * a.w_row + head * a.w_head;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ahead[kAhead][4], old[4];
    int keys[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      keys[u] = min(key0 + u * kThreads, x.len - 1);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ahead[i][u] = scores[min(i, rows - 1) * a.score_stride + keys[u]];
      old[u] = w[keys[u]];
    }
    auto add = [&](const float2& y, const float (&s)[4]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // -inf: not seen (also where the row is NaN)
        const float p = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[u], a.scale_log2, -y.x)), y.y, sum[u]);
        sum[u] = s[u] == -__builtin_inff() ? sum[u] : p;
      }
    };
    for (int r0 = 0; r0 < rows; r0 += kHold) {
      __syncthreads();  // the rows before are done with theirs
      // 16 lanes share a row's ranges
      for (int i = static_cast<int>(threadIdx.x) / 16; i < min(kHold, rows - r0); i += kThreads / 16) {
        const int row = r0 + i, at = first + head * n_ranges * n_rt + row / kScoreRows, mine = threadIdx.x % 16;
        const float2* const p = reinterpret_cast<const float2*>(a.part) + static_cast<int64_t>(at) * kScoreRows + row % kScoreRows;
        // (every part has its place but those of an offset table that is not ascending)
        const int n = at >= 0 && at + static_cast<int64_t>(n_ranges - 1) * n_rt < a.part_items ? n_ranges : 0;
        float m = -__builtin_inff(), l = 0.0f;
        auto join = [&](float m2, float l2) __attribute__((always_inline)) {
          const float top = fmaxf(m, m2), sub = top == -__builtin_inff() ? 0.0f : top;
          l = l * __builtin_amdgcn_exp2f(m - sub) + l2 * __builtin_amdgcn_exp2f(m2 - sub);
          m = top;
        };
        for (int v = mine; v < n; v += 16) {
          const float2 y = p[static_cast<int64_t>(v) * n_rt * kScoreRows];
          join(y.x, y.y);
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) join(__shfl_xor(m, d), __shfl_xor(l, d));
        if (mine == 0) stats[i] = stat_of(m, l);
      }
      __syncthreads();
      if (r0 == 0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (i < rows) add(stats[i], ahead[i]);
      }
      for (int i = r0 == 0 ? kAhead : 0; i < min(kHold, rows - r0); ++i) {
        float s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = scores[(r0 + i) * a.score_stride + keys[u]];
        add(stats[i], s);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (key0 + u * kThreads < x.len && sum[u] != 0.0f) w[keys[u]] = old[u] + sum[u];
  }
}

// The kernels of a call, and its items and workspace, whatever the lengths turn out to be.
struct Plan {
  bool few, may_cut;
  int stats_items, sums_items, slots;
  int64_t score_stride, part_items, part_bytes, stats_bytes, bytes;
};
constexpr int kHeaderBytes = 256;  // of the workspace: the cuts
Plan plan_of(int64_t requests, int64_t tokens, int group, int kv_heads, int head_dim, int64_t max_keys, int64_t max_rows) {
  Plan p;
  const int64_t rows_all = kv_heads * tokens * group;
  p.score_stride = (max_keys + 63) / 64 * 64;
  const int64_t score_bytes = rows_all * p.score_stride * 4;
  p.few = max_rows <= kScoreRows && score_bytes <= kMostScores;
  const int rows = p.few ? kScoreRows : Stats<64>::kRows;
  p.slots = kCus * (head_dim == 256 && !p.few ? 1 : 2);
  p.stats_items = 2048;
  p.sums_items = 2048;
  // a share alone may add a range per row tile
  p.part_items = p.stats_items + kv_heads * (tokens * group / rows + requests);
  p.part_bytes = (p.part_items * rows * 8 + 15) / 16 * 16;
  p.stats_bytes = p.few ? score_bytes : (rows_all * 8 + 15) / 16 * 16;
  // a range of row tiles is four at least, and a request without more is never cut
  p.may_cut = !p.few && tokens * group > 4 * kSumRows;
  p.bytes = kHeaderBytes + p.part_bytes + p.stats_bytes + (p.may_cut ? 2LL * p.sums_items * kSumKeys * 4 : 0);
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

extern "C" int64_t fd_paged_key_weights_workspace_bytes(int batch, int q_heads, int kv_heads, int seq_len, int head_dim,
                                                        int page_size, int max_pages, int n_seqs, int max_seqlen, int last) {
  static const char* what = "fd_paged_key_weights_workspace_bytes";
  if (int rc = check_sizes(what, batch, q_heads, kv_heads, seq_len, n_seqs, max_seqlen, last)) return rc;
  FD_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, FD_ERR_UNSUPPORTED,
             "%s: head_dim must be 64, 128 or 256 (got %d)", what, head_dim);
  FD_REQUIRE(page_size >= 1 && max_pages >= 1, FD_ERR_INVALID_ARGUMENT, "%s: page_size and max_pages must be >= 1", what);
  return plan_of(n_seqs > 0 ? n_seqs : batch, static_cast<int64_t>(batch) * seq_len, q_heads / kv_heads, kv_heads, head_dim,
                 static_cast<int64_t>(max_pages) * page_size,
                 static_cast<int64_t>(last > 0 ? std::min(last, max_seqlen) : max_seqlen) * (q_heads / kv_heads)).bytes;
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
  const int group = q_heads / cache->kv_heads;
  const int64_t max_keys = static_cast<int64_t>(cache->max_pages) * cache->page_size;
  const Plan p = plan_of(requests, static_cast<int64_t>(batch) * seq_len, group, cache->kv_heads, cache->head_dim, max_keys,
                         static_cast<int64_t>(last > 0 ? std::min(last, max_seqlen) : max_seqlen) * group);
  FD_REQUIRE(p.part_items < (1LL << 31), FD_ERR_UNSUPPORTED, "%s: problem too large", what);
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
  a.stats_items = p.stats_items;
  a.sums_items = p.sums_items;
  a.slots = p.slots;
  a.part_items = static_cast<int>(p.part_items);
  a.scale_log2 = scale * 1.4426950408889634f;
  char* const work = static_cast<char*>(workspace);
  a.cuts = reinterpret_cast<int32_t*>(work);
  a.part = reinterpret_cast<float*>(work + kHeaderBytes);
  a.scores = a.stats = reinterpret_cast<float*>(work + kHeaderBytes + p.part_bytes);
  a.score_stride = p.score_stride;
  a.sums = reinterpret_cast<float*>(work + kHeaderBytes + p.part_bytes + p.stats_bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // workgroups: no more than the sizes can make items
  const int64_t heads = static_cast<int64_t>(requests) * cache->kv_heads, key_tiles = heads * ((max_keys + kSumKeys - 1) / kSumKeys);
  const int64_t row_tiles = (static_cast<int64_t>(batch) * seq_len * group + kSumRows - 1) / kSumRows;
  const unsigned stats_grid = static_cast<unsigned>(std::min<int64_t>(p.part_items, 2 * p.slots));
  const unsigned sums_grid = static_cast<unsigned>(std::min<int64_t>(key_tiles * std::max<int64_t>(row_tiles / 4, 1), 2 * p.slots));
  const unsigned join_grid = static_cast<unsigned>(std::min<int64_t>(key_tiles, p.sums_items));
  by_kind(cache, [&](auto d, auto f) {
    constexpr int D = decltype(d)::value;
    constexpr Format F = decltype(f)::value;
    if (p.few) {
      a.slots = kCus * kScoreGroups<D, F>;
      hipLaunchKernelGGL((key_scores_kernel<D, F>), dim3(static_cast<unsigned>(std::min<int64_t>(p.part_items, 2 * a.slots))), dim3(kThreads), 0, s, a);
      return;
    }
    hipLaunchKernelGGL((row_stats_kernel<D, F>), dim3(stats_grid), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL((row_stats_join_kernel<Stats<D>>), dim3(static_cast<unsigned>(std::min<int64_t>(p.part_items - p.stats_items, 1024))),
                       dim3(Stats<D>::kRows), 0, s, a);
    hipLaunchKernelGGL((key_sums_kernel<D, F>), dim3(sums_grid), dim3(kThreads), 0, s, a);
  });
  if (p.few) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(heads * ((max_keys + kAddKeys - 1) / kAddKeys), 4096));
    hipLaunchKernelGGL(key_scores_add_kernel, dim3(grid), dim3(kThreads), 0, s, a);
  }
  if (p.may_cut) hipLaunchKernelGGL(key_sums_join_kernel, dim3(join_grid), dim3(kSumKeys), 0, s, a);
  return fd_check_launch(what);
}
