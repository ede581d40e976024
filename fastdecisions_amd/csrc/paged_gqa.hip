// Grouped-query attention of new tokens over a paged key/value cache, gfx950
// (bf16 MFMA, fp32 softmax; bf16, e4m3 or e2m1 pages).
//
// The rows of one KV head are the (token, query head of its group) pairs of a
// request, token by token: row p is token p / G, head p % G.  A row sees the
// keys up to its token's position.  An item of work is one tile of rows of one
// (request, KV head) against one range of its keys:
//
//   few rows   16 or 32 rows, 4 wavefronts that each take every fourth block of
//              32 keys into LDS of their own: no barrier in the loop, the cache
//              streams through at the rate of the memory.  Up to 64 rows, small
//              calls up to 128 (plan_of).
//   pieces     128 rows, wavefronts share the staged key tiles.  Suffixes.
//
// Key ranges are sized on the device: the lengths are there, and a grid sized by
// the longest possible request would be mostly empty.  Every workgroup sums the
// row tiles times key tiles of all requests and cuts every request into ranges
// of c tiles (best_range), so items are alike whatever the mix of lengths; the
// host only bounds their number.  Items of a split row tile leave (o, max,
// denominator) in the workspace and paged_gqa_join_kernel joins them.
//
// In both, scores are computed transposed (S^T = K Q^T on MFMA), with the K rows
// permuted so that a lane's scores are those of the 8 consecutive keys whose
// probabilities it must supply to P V: P never leaves registers, and V^T comes
// from transposing LDS reads.
//
// The matrix product takes P in bf16.  Few rows, bound by the cache's bytes, take
// it in two parts (two_bf16), so that nothing but the output is rounded: errors
// against 64 bits as with P in fp32 (0.00164 of the output, the output's own
// rounding; one part 0.0020), for 0 to 4 % of the time with single tokens, up to 9 %
// with 17 to 64 rows.  Pieces, bound by the MFMAs' and the softmax's issue, take one
// part, as the uncached attention does: with two, 2048 tokens on 6144 keys take 139
// us (64 features, 103 with one), 192 (128, 143) and 191 (256, 148).  Their
// denominator sums the rounded p.
//
// e2m1 pages: v_cvt_scalef32_pk_bf16_fp4 takes codes times a block's scale to bf16,
// exactly.  Few rows copy codes to LDS as they are, and a block's leave it for
// registers at once, so that the next copies may follow.  K is widened there; V is
// widened into LDS of the wavefront as bf16, 32 keys of up to 128 features at a time
// (8 KiB), and read by the 16-bit transposing reads that bf16 pages take: 256 to 8192
// keys of 64 requests (97 MB) 33 us and 4.8 for the join, 64 x 8192 keys 65 us (4.4
// TB/s; e4m3 106, bf16 187).  The decoding, 4.4 cycles per 2 values and SIMD, and V's
// way through LDS then cost as much as the bytes.
// Pieces decode into their bf16 stages: 2048 tokens on 6144 keys 157 us (128
// features; e4m3 159, bf16 139) and 174 (256; 175, 147).
#include <algorithm>
#include <type_traits>

#include "gqa_tile.h"
#include "paged_common.h"
#include "wave_tools.h"

namespace {

constexpr int kNumXcd = 8;
constexpr int kCus = 256;  // a power of two (slots_log2)

// Few rows: NR blocks of 16 rows; every wavefront stages blocks of 32 keys of its own.
template <int D_, Format F_, int NR_>
struct Few {
  static constexpr int D = D_, NR = NR_;
  static constexpr Format F = F_;
  static constexpr bool FP8 = F == kE4m3, FP4 = F == kE2m1;
  static constexpr int kWaves = 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kRows = 16 * NR;
  static constexpr int kKeys = 32 * kWaves;             // keys of a tile: a block of each wavefront
  static constexpr int kRowBytes = FP4 ? D / 2 : FP8 ? D : 2 * D;  // of a cached row, staged as it is
  static constexpr int kBlockBytes = 32 * kRowBytes;    // K or V of a block
  // 32 K scales and 32 V scales, a word each; of E2M1 the D / 32 bytes of 32 rows of each, at least a word a row
  static constexpr int kScaleCopies = FP8 ? 1 : FP4 ? (D == 256 ? 2 : 1) : 0;
  static constexpr int kScaleBytes = 256 * kScaleCopies;
  static constexpr int kStageBytes = 2 * kBlockBytes + kScaleBytes;
  // E2M1 blocks leave their stage for registers at once, so half as many do
  static constexpr int kStages = FP4 ? 4096 / kBlockBytes : kBlockBytes >= 8192 ? 1 : 8192 / kBlockBytes;
  static constexpr int kWide = D < 128 ? D : 128;       // features of an E2M1 V block that are bf16 in LDS at a time
  static constexpr int kDecoded = FP4 ? 32 * 2 * kWide : 0;
  static constexpr int kCopies = kBlockBytes / 1024;    // copy instructions of a block's K (or V)
  static constexpr int kCopyRows = 1024 / kRowBytes;
  static constexpr int kKGroup = kCopies + kScaleCopies;
  static constexpr int kRowFloats = D + 4;
  static constexpr int kEpilogueBytes = kWaves * kRows * (kRowFloats + 2) * 4;
  static constexpr int kLoopBytes = kWaves * (kStages * kStageBytes + kDecoded);
  static constexpr int kSmemBytes = kLoopBytes > kEpilogueBytes ? kLoopBytes : kEpilogueBytes;
  static constexpr int kPerCu = kSmemBytes > 80 * 1024 ? 1 : 2;  // workgroups that a CU's LDS holds
};

// Pieces: RW row wavefronts of NB blocks of 32 rows, times KS key parts of a tile.
template <int D_, Format F_, int RW_, int NB_, int KS_>
struct Piece {
  static constexpr int D = D_, RW = RW_, NB = NB_, KS = KS_;
  static constexpr Format F = F_;
  static constexpr bool CODES = F != kBf16;
  static constexpr int kWaves = RW * KS;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kRows = 32 * RW * NB;
  static constexpr int kKeys = 32 * KS;                 // keys of a tile
  static constexpr int CR = D / 8;                      // 16-byte chunks of a staged (bf16) row
  static constexpr int kTileBytes = kKeys * CR * 16;    // K or V
  static constexpr int kStages = 4;
  static constexpr int kEpilogueBytes = KS == 1 ? 0 : kWaves * 64 * (NB * D / 4 + 2) * 4;  // what the key parts give each other
  static constexpr int kLoopBytes = 2 * kStages * kTileBytes;
  static constexpr int kSmemBytes = kLoopBytes > kEpilogueBytes ? kLoopBytes : kEpilogueBytes;
  // 1 KiB copies of a bf16 K (or V) tile per wavefront, and the rows of each
  static constexpr int kCopies = kTileBytes / 1024 / kWaves;
  static constexpr int kCopyRows = 1024 / (2 * D);
  // loads of 16 codes per lane of a tile per wavefront, and their rows
  static constexpr int kLoads = kKeys * D / 1024 / kWaves;
  static constexpr int kLoadRows = 1024 / D;
  static_assert(kCopies >= 1 && kLoads >= 1, "a tile gives every wavefront a whole copy");
  static_assert(kSmemBytes <= 160 * 1024, "LDS");
};

struct PagedArgs {
  PagedView c;
  const uint16_t* q;
  const uint16_t* gate;
  uint16_t* o;
  int64_t qs[3], gs[3], os[3];  // b, h, t
  const int32_t* cu;
  int n_req, seq_len, group, kv_heads;
  uint32_t group_magic;         // ceil(2^24 / group)
  int slots_log2, min_tiles, overhead;  // workgroups that run at once; tiles of a range at least, and that one costs besides
  int part_items;               // items whose parts the workspace holds
  float scale_log2;
  int32_t* range_tiles;         // the key tiles of a range, for the joining kernel; null where nothing can be split
  float* part;                  // per item: rows x D of o, then rows x 2 of (max, denominator)
};

// The work of one (request, row tile, KV head, key range).
struct Item {
  int req, head, rtile, range;
  int row0, rows;               // first row of the tile, rows of the request
  int token0, rem0;             // row0 / group and row0 % group
  int start, n_new, len;        // new tokens on the T axis, keys
  int tiles;                    // key tiles of a range
  int base, n_rtiles, n_ranges; // first item of the request; its row tiles and key ranges
};

// The key tiles of a range, for up to 64 requests of rt row tiles and kt key tiles (a lane each) and
// `work` tile pairs in all heads.  A range of c tiles gives sum rt ceil(kt / c) heads items; the smallest
// c whose items fit m times the workgroups that run at once takes about m (c + overhead) tiles of time,
// and the better of m = 1 .. kMaxRounds is taken: a few items more than workgroups would cost a whole
// round (six suffixes of 30 to 400 tokens: 344 items of 35 tiles on 256 CUs 107 us, 232 of 42 tiles 76).
constexpr int kMaxRounds = 2;
static_assert(kMaxRounds == 2, "m << slots_log2 and >> (slots_log2 + m - 1) are the same for m = 1 and 2");
__device__ __forceinline__ int best_range(const PagedArgs& a, int rt, int kt, int64_t work) {
  auto items = [&](int c) { return __builtin_amdgcn_readlane(wave_scan(rt * max(tiles_over(kt, c), 1)), 63) * a.kv_heads; };
  const float longest = fd_xor_max<32>(fd_xor_max<16>(fd_xor_max<8>(fd_xor_max<4>(fd_xor_max<2>(fd_xor_max<1>(static_cast<float>(kt)))))));
  const int top = max(uniform(static_cast<int>(longest)) + 1, a.min_tiles);
  int best = top, cost = 0x7fffffff;
  for (int m = 1; m <= kMaxRounds; ++m) {
    const int fit = m << a.slots_log2;
    const int64_t share = max(static_cast<int64_t>(a.min_tiles), (work + fit - 1) >> (a.slots_log2 + m - 1));
    if (share >= top || items(top) > fit) continue;
    int lo = static_cast<int>(share);
    if (items(lo) > fit) {  // items(hi) <= fit < items(lo)
      int hi = top;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (items(mid) > fit) lo = mid;
        else hi = mid;
      }
      lo = hi;
    }
    const int now = m * (lo + a.overhead);
    if (now < cost) {
      cost = now;
      best = lo;
    }
    if (lo == a.min_tiles || 8 * lo <= 9 * share) break;  // one round within an eighth of an even share: no better two
  }
  return best;
}

// Row tile at place j of n of a key range, of which XCDs take runs of `per` items: the later tiles see more keys, so
// they go first, and where a range's tiles fill q runs, run s takes every q-th of them (one half of the tiles in a row
// would be three quarters of the work).  Prompts without a prefix, 16/4 heads x 128: 6000 tokens 240 -> 197 us, 16384
// 1440 -> 1103 (1000 TFLOP/s); at most one tile per CU the same.
__device__ __forceinline__ int spread(int j, int n, int per) {
  const int q = min(max((n + per / 2) / per, 1), n), whole = n / q, more = n - whole * q;  // the first `more` runs have one more
  const int late = j - more * (whole + 1);
  const int s = late < 0 ? j / (whole + 1) : more + late / whole;
  const int i = late < 0 ? j - s * (whole + 1) : late - (s - more) * whole;
  return n - 1 - (i * q + s);
}

// Finds work item `want(total items)` (JOIN: row tile, whatever its ranges).  One wavefront
// looks at 64 requests at a time; false if there is no such item.  Beyond 64 requests ranges are a round's share.
template <int ROWS, int KEYS, bool JOIN, typename Want>
__device__ __forceinline__ bool find_item(const PagedArgs& a, int lane, Want want, Item* it) {
  auto sizes = [&](int r, int* start, int* n_new, int* len, int* rt, int* kt) {
    *start = *n_new = *len = *rt = *kt = 0;
    if (r < a.n_req) {
      int end;
      request_rows(a.cu, r, a.seq_len, start, &end);
      *n_new = end - *start;
      *len = request_keys(a.c, r);
      *rt = static_cast<int>((static_cast<int64_t>(*n_new) * a.group + ROWS - 1) / ROWS);
      *kt = (*len + KEYS - 1) / KEYS;
    }
  };
  auto at_lane = [](int v, int l) { return __builtin_amdgcn_readlane(v, l); };
  int start, n_new, len, rt, kt;
  int tiles;
  if constexpr (JOIN) {
    tiles = scalar_load(a.range_tiles, 0);  // what the items' kernel worked with, 0: it split nothing
    if (tiles == 0) return false;
    if (a.n_req <= 64) sizes(lane, &start, &n_new, &len, &rt, &kt);
  } else {
    int64_t work = 0;
    for (int r0 = 0; r0 < a.n_req; r0 += 64) {
      sizes(r0 + lane, &start, &n_new, &len, &rt, &kt);
      const int64_t w = static_cast<int64_t>(rt) * kt;  // below 2^49: summed in two parts
      work += at_lane(wave_scan(static_cast<int>(w & 0xffffff)), 63);
      work += static_cast<int64_t>(at_lane(wave_scan(static_cast<int>(w >> 24)), 63)) << 24;
    }
    if (a.n_req <= 64) {
      tiles = best_range(a, rt, kt, work * a.kv_heads);
    } else {
      const int log2 = a.slots_log2 + 1;  // of kMaxRounds rounds
      const int64_t share = (work * a.kv_heads + (1LL << log2) - 1) >> log2;
      tiles = static_cast<int>(min(max(static_cast<int64_t>(a.min_tiles), share), static_cast<int64_t>(1 << 22)));
    }
    if (a.range_tiles != nullptr && blockIdx.x == 0) {
      bool split = false;
      for (int r0 = 0; r0 < a.n_req; r0 += 64) {
        if (a.n_req > 64) sizes(r0 + lane, &start, &n_new, &len, &rt, &kt);
        split |= __builtin_amdgcn_ballot_w64(kt > tiles) != 0;
      }
      if (threadIdx.x == 0) *a.range_tiles = split ? tiles : 0;
    }
  }
  auto ranges_of = [&](int k) { return max(tiles_over(k, tiles), 1); };
  int total = 0, at = 0;
  if (a.n_req > 64) {
    for (int r0 = 0; r0 < a.n_req; r0 += 64) {
      sizes(r0 + lane, &start, &n_new, &len, &rt, &kt);
      total += at_lane(wave_scan(rt * (JOIN ? 1 : ranges_of(kt)) * a.kv_heads), 63);
    }
    at = want(total);
    if (at < 0 || at >= total) return false;
  }
  int base = 0, before = 0;  // items of the requests before r0 (all ranges), and in terms of `at`
  for (int r0 = 0; r0 < a.n_req; r0 += 64) {
    if (a.n_req > 64) sizes(r0 + lane, &start, &n_new, &len, &rt, &kt);
    const int ranges = ranges_of(kt);
    const int all = rt * ranges * a.kv_heads;
    const int mine = JOIN ? rt * a.kv_heads : all;
    const int incl = wave_scan(mine);
    const int incl_all = JOIN ? wave_scan(all) : incl;
    if (a.n_req <= 64) {
      total = at_lane(incl, 63);
      at = want(total);
      if (at < 0 || at >= total) return false;
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + incl > at);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      it->req = r0 + l;
      const int k = at - (before + at_lane(incl, l) - at_lane(mine, l));  // within the request
      if (k < 0) return false;  // sums past 31 bits: only of an offset table that is not ascending
      it->base = base + at_lane(incl_all, l) - at_lane(all, l);
      it->n_rtiles = at_lane(rt, l);
      it->n_ranges = at_lane(ranges, l);
      it->start = at_lane(start, l);
      it->n_new = at_lane(n_new, l);
      it->len = at_lane(len, l);
      it->tiles = max(tiles_over(at_lane(kt, l), it->n_ranges), 1);  // a request's ranges are alike
      it->rtile = k % it->n_rtiles;  // row tiles of a key range one after the other: they share its keys
      if constexpr (!JOIN && ROWS >= 128) it->rtile = spread(it->rtile, it->n_rtiles, (total + kNumXcd - 1) / kNumXcd);
      const int hr = k / it->n_rtiles;
      it->range = JOIN ? 0 : hr % it->n_ranges;
      it->head = JOIN ? hr : hr / it->n_ranges;
      it->row0 = it->rtile * ROWS;
      it->rows = it->n_new * a.group;
      it->token0 = it->row0 / a.group;
      it->rem0 = it->row0 - it->token0 * a.group;
      return true;
    }
    before += at_lane(incl, 63);
    base += at_lane(incl_all, 63);
  }
  return false;
}

// Token (from the tile's first one on) of row `row` of a tile: (rem0 + row) / group, below 2^24 / group.
__device__ __forceinline__ int token_of(const PagedArgs& a, const Item& it, int row) {
  return static_cast<int>((static_cast<uint32_t>(it.rem0 + row) * a.group_magic) >> 24);
}

// Keys that the last row of the tile sees (the tile's keys).
template <int ROWS>
__device__ __forceinline__ int keys_of_tile(const PagedArgs& a, const Item& it) {
  const int last = min(ROWS, it.rows - it.row0) - 1;
  return max(0, min(it.len, it.len - it.n_new + it.token0 + token_of(a, it, last) + 1));
}

template <int ROWS>
__device__ __forceinline__ int64_t part_floats(int D) {
  return static_cast<int64_t>(ROWS) * (D + 2);
}

// out = acc * inv (* sigmoid(gate)), four features of a row.
__device__ __forceinline__ void store4(const PagedArgs& a, const Item& it, int row, int d, f32x4_t acc, float inv) {
  const int local = token_of(a, it, row);
  const int head = it.head * a.group + (it.rem0 + row - local * a.group);
  const int b = a.cu == nullptr ? it.req : 0;
  const int64_t t = it.start + it.token0 + local;
  f32x4_t v = acc * inv;
  if (a.gate != nullptr) {
    const bf16x4_t g4 = *reinterpret_cast<const bf16x4_t*>(a.gate + b * a.gs[0] + head * a.gs[1] + t * a.gs[2] + d);
    const f32x4_t g = __builtin_convertvector(g4, f32x4_t);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] / (1.0f + __expf(-g[e]));
  }
  *reinterpret_cast<bf16x4_t*>(a.o + b * a.os[0] + head * a.os[1] + t * a.os[2] + d) = __builtin_convertvector(v, bf16x4_t);
}

__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Block b's item and the keys its rows see; false if there is none or none of its range's keys is seen.
struct Job {
  Item it;
  int kend, t0, nt, slot;  // keys seen; first tile, tiles, and place of the item
  bool split;
};
template <class S>
__device__ __forceinline__ bool open_job(const PagedArgs& a, int lane, Job* j) {
  Item it;
  // XCD x takes one contiguous run of the items: row tiles that share keys meet in one L2
  const int b = blockIdx.x;
  auto want = [&](int total) {
    const int per = (total + kNumXcd - 1) / kNumXcd;
    const int i = b / kNumXcd;
    return i < per ? (b % kNumXcd) * per + i : -1;
  };
  if (!find_item<S::kRows, S::kKeys, false>(a, lane, want, &it)) return false;
  it.req = uniform(it.req), it.head = uniform(it.head), it.rtile = uniform(it.rtile), it.range = uniform(it.range);
  it.row0 = uniform(it.row0), it.rows = uniform(it.rows), it.start = uniform(it.start), it.n_new = uniform(it.n_new);
  it.len = uniform(it.len), it.tiles = uniform(it.tiles), it.base = uniform(it.base);
  it.n_rtiles = uniform(it.n_rtiles), it.n_ranges = uniform(it.n_ranges);
  it.token0 = uniform(it.token0), it.rem0 = uniform(it.rem0);
  j->it = it;
  j->kend = uniform(keys_of_tile<S::kRows>(a, it));
  const int nt_all = (j->kend + S::kKeys - 1) / S::kKeys;
  j->t0 = it.range * it.tiles;
  if (it.range > 0 && j->t0 >= nt_all) return false;
  j->nt = min(it.tiles, nt_all - j->t0);  // 0 where no key is visible at all
  j->split = nt_all > it.tiles;
  // where a part goes; the workspace has a place for every part of a well-formed offset table
  j->slot = it.base + (it.head * it.n_ranges + it.range) * it.n_rtiles + it.rtile;
  return !j->split || (j->slot >= 0 && j->slot < a.part_items);
}

// Is any key of the job's tiles on no page?
template <class S>
__device__ __forceinline__ bool any_absent(const PagedArgs& a, const Job& j, const int32_t* table, int lane) {
  if (j.nt <= 0) return false;
  const int first = (j.t0 * S::kKeys) >> a.c.shift;
  const int last = (min((j.t0 + j.nt) * S::kKeys, j.kend) - 1) >> a.c.shift;
  bool bad = false;
  for (int i = first + lane; i <= last; i += 64)
    bad |= static_cast<unsigned>(table[i]) >= static_cast<unsigned>(a.c.n_pages);
  return __builtin_amdgcn_ballot_w64(bad) != 0;
}

// The key parts' rows in LDS (S::kRowFloats apart) and their (max, denominator), joined row by row: stored, or
// left as the item's part.
template <class S, int PARTS>
__device__ __forceinline__ void close_job(const PagedArgs& a, const Job& j, const float* rowsf, const float* ml) {
  constexpr int D = S::D;
  const int rows = min(S::kRows, j.it.rows - j.it.row0);
  float* const part = a.part + j.slot * part_floats<S::kRows>(D);
  for (int i = threadIdx.x; i < rows * (D / 4); i += S::kThreads) {
    const int row = i / (D / 4), d = (i % (D / 4)) * 4;
    float m = ml[row * 2];
#pragma unroll
    for (int s = 1; s < PARTS; ++s) m = fmaxf(m, ml[(s * S::kRows + row) * 2]);
    const float m_sub = m == -__builtin_inff() ? 0.0f : m;
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
      const int at = s * S::kRows + row;
      const float w = __builtin_amdgcn_exp2f(ml[at * 2] - m_sub);
      l += ml[at * 2 + 1] * w;
      acc += *reinterpret_cast<const f32x4_t*>(rowsf + at * S::kRowFloats + d) * w;
    }
    if (!j.split) {
      store4(a, j.it, row, d, acc, l == 0.0f ? 0.0f : 1.0f / l);
    } else {
      *reinterpret_cast<f32x4_t*>(part + row * D + d) = acc;
      if (d == 0) {
        part[S::kRows * D + row * 2] = m;
        part[S::kRows * D + row * 2 + 1] = l;
      }
    }
  }
}

// ---------------------------------------------------------------- few rows

// Key (within a 32-key block) that row m of the block's score MFMA a supplies: lane group g then
// holds the scores of keys 8 g .. 8 g + 7, those whose P it supplies as the B operand of P V.
__device__ __forceinline__ int sigma16(int a, int m) { return 8 * (m >> 2) + 4 * a + (m & 3); }

// Chunk swizzles of the staged rows (physical chunk = logical chunk ^ f(row)), such that rows read
// together lie in different banks: 16 permuted rows at one chunk for K; for V the 4 (bf16, chunk
// pairs) or 8 (codes) rows of a transposing read and the next lane group's.
template <int ROW_BYTES>
constexpr int kRowShift = ROW_BYTES >= 256 ? 0 : ROW_BYTES == 128 ? 1 : ROW_BYTES == 64 ? 2 : 3;
template <int ROW_BYTES>
__device__ __forceinline__ int few_swz_k(int row) {
  return ((row & 3) | ((row >> 3) & 3) << 2) >> kRowShift<ROW_BYTES>;
}
template <int ROW_BYTES, Format F>
__device__ __forceinline__ int few_swz_v(int row) {
  if constexpr (F == kE2m1) return (row >> 2) & (ROW_BYTES / 16 < 4 ? 1 : 3);
  else if constexpr (F == kE4m3) return ((row & 7) | ((row >> 3) & 1) << 3) >> kRowShift<ROW_BYTES>;
  else return 2 * (((row & 3) | ((row >> 3) & 1) << 2) >> kRowShift<ROW_BYTES>);
}

// Eight codes times a power of two as bf16 (exact).
__device__ __forceinline__ bf16x8_t codes_to_bf16(uint32_t lo, uint32_t hi, float scale = 1.0f) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x plus the eight bf16 of p.
__device__ __forceinline__ float sum8(bf16x8_t p, float x) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const bf16x2_t one = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{p[2 * i], p[2 * i + 1]}, one, x, false);
  return x;
}

// p >= 0 as the sum of two bf16 up to 2^-16 of it.  The first is below p wherever p is not 0, so that the second is
// not 0 there either: a seen infinity times the two parts is one infinity, never NaN.
__device__ __forceinline__ void two_bf16(f32x8_t p, bf16x8_t* hi, bf16x8_t* lo) {
  f32x8_t first;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    first[e] = __uint_as_float(__builtin_elementwise_sub_sat(__float_as_uint(p[e]), 1u) & 0xffff0000u);
  *hi = __builtin_convertvector(first, bf16x8_t);
  *lo = __builtin_convertvector(p - first, bf16x8_t);
}

// Infinities and NaN ("odd" values) among V's operands: are there any, the operand without them, element i
// (uniform) of one, and o + p x for the odd ones of four values x that a row sees (p is not 0).
__device__ __forceinline__ bool any_odd(bf16x8_t v) {
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return odd;
}
__device__ __forceinline__ bf16x8_t without_odd(bf16x8_t v) {
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  u32x4_t w = __builtin_bit_cast(u32x4_t, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((w[i] & 0x7f80u) == 0x7f80u) w[i] &= 0xffff0000u;
    if ((w[i] & 0x7f800000u) == 0x7f800000u) w[i] &= 0xffffu;
  }
  return __builtin_bit_cast(bf16x8_t, w);
}
__device__ __forceinline__ float element(bf16x8_t v, int i) {
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
  const uint32_t pair = i < 2 ? w[0] : i < 4 ? w[1] : i < 6 ? w[2] : w[3];
  return fd_bf16_to_f32((i & 1) ? pair >> 16 : pair & 0xffffu);
}
__device__ __forceinline__ f32x4_t add_odd(f32x4_t o, f32x4_t x, float p) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (!(fabsf(x[e]) < __builtin_inff()) && p != 0.0f) o[e] += p * x[e];
  return o;
}

// One byte per lane, zero-extended, to a word of LDS at lds + 4 * lane.
__device__ __forceinline__ void byte_to_lds(const uint8_t* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}

// Two bytes (zero-extended), four or sixteen per lane, likewise, each lane's from an address of its own.
__device__ __forceinline__ void short_to_lds(const uint8_t* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ushort %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void word_to_lds(const uint8_t* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void lane_to_lds(const unsigned char* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory", "m0");
}

// A block of 32 keys costs a wavefront 24 (NR) MFMAs of 16x16x32 and, at the memory's rate, several
// times as long to arrive, so what counts is that copies are always in flight: rows go to LDS as they
// are (codes are converted where they are read, scales multiply scores and probabilities), K and V
// of kStages blocks each, the next K leaving as soon as a block's scores have read theirs, the next
// V as soon as P V has.
// Measured (16 / 4 heads x 128, pages of 64, kernel and join): 64 requests of 8192 keys 195 us, 5.5 TB/s of
// keys and values (a large copy here: 5.1), E4M3 108 us, 5.0 TB/s; of 256 to 8192 keys 80 and 48 us; one
// request of 8192 keys 14 us, of 200 keys 8 us, latency: arguments, lengths, page, keys, scores, store.
template <class S>
__global__ __launch_bounds__(S::kThreads, S::kPerCu) void paged_gqa_few_kernel(PagedArgs a) {
  constexpr int D = S::D, NR = S::NR, RBY = S::kRowBytes, kKk = D / 32, kNdb = D / 16, NS = S::kStages;
  constexpr bool FP8 = S::FP8, FP4 = S::FP4;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[S::kSmemBytes];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int grp = lane >> 4, li = lane & 15;

  Job job;
  if (!open_job<S>(a, lane, &job)) return;
  const Item& it = job.it;
  const int kend = job.kend;
  const int32_t* const table = a.c.table + it.req * a.c.table_stride;

  // ---- copies.  Block j of this wavefront: keys first + 128 j .. + 31; rows past kend repeat row kend - 1 (the
  // mask discards them).  Its two halves of 16 keys lie on a page each.
  const int first = job.t0 * S::kKeys + wave * 32;
  const int mine = max(0, min(job.nt, (kend - first + S::kKeys - 1) / S::kKeys));
  struct Pages {
    int p[2];
  };
  auto pages_of = [&](int j) {
    Pages x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = uniform(max(min(first + j * S::kKeys + 16 * h, kend - 1), 0));
      const int page = scalar_load(table, key >> a.c.shift);
      x.p[h] = static_cast<unsigned>(page) < static_cast<unsigned>(a.c.n_pages) ? page : 0;
    }
    return x;
  };
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_t*)smem)) +
                        static_cast<uint32_t>(wave * NS * S::kStageBytes);
  const unsigned char* const stage0 = smem + wave * NS * S::kStageBytes;
  const int page_mask = (1 << a.c.shift) - 1;
  constexpr int kChunks = RBY / 16;
  const unsigned char* const head_base[2] = {a.c.k + it.head * a.c.head, a.c.v + it.head * a.c.head};
  auto copy_side = [&](const Pages& pg, int j, int v) {
    const int kb0 = first + j * S::kKeys;
    const uint32_t lds = lds0 + static_cast<uint32_t>((j & (NS - 1)) * S::kStageBytes + v * S::kBlockBytes);
#pragma unroll
    for (int i = 0; i < S::kCopies; ++i) {
      const int row = i * S::kCopyRows + lane / kChunks;
      const int chunk = (lane % kChunks) ^ (v ? few_swz_v<RBY, S::F>(row) : few_swz_k<RBY>(row));
      const int key = min(kb0 + row, kend - 1) & page_mask;
      const uint32_t at = static_cast<uint32_t>(key * static_cast<int>(a.c.row) + chunk * 16);
      if constexpr (S::kCopyRows > 16)  // rows of both pages
        lane_to_lds(head_base[v] + (row < 16 ? pg.p[0] : pg.p[1]) * a.c.page + at, lds + static_cast<uint32_t>(i * 1024));
      else
        copy_to_lds(head_base[v] + pg.p[i * S::kCopyRows / 16] * a.c.page, at, lds + static_cast<uint32_t>(i * 1024));
    }
  };
  auto copy_k = [&](const Pages& pg, int j) {
    copy_side(pg, j, 0);
    if constexpr (FP8) {
      const int row = lane & 31;
      const int key = min(first + j * S::kKeys + row, kend - 1) & page_mask;
      const int page = row < 16 ? pg.p[0] : pg.p[1];
      byte_to_lds((lane < 32 ? a.c.k_scale : a.c.v_scale) + page * a.c.s_page + it.head * a.c.s_head + key,
                  lds0 + static_cast<uint32_t>((j & (NS - 1)) * S::kStageBytes + 2 * S::kBlockBytes));
    }
    if constexpr (FP4) {  // a row's scales in one word per lane, of 256 features in two
#pragma unroll
      for (int i = 0; i < S::kScaleCopies; ++i) {
        const int row = D == 256 ? lane >> 1 : lane & 31;
        const bool of_k = D == 256 ? i == 0 : lane < 32;
        const int key = min(first + j * S::kKeys + row, kend - 1) & page_mask;
        const int page = row < 16 ? pg.p[0] : pg.p[1];
        const uint8_t* const p = (of_k ? a.c.k_scale : a.c.v_scale) + page * a.c.s_page + it.head * a.c.s_head +
                                 key * (D / kScaleBlock) + (D == 256 ? 4 * (lane & 1) : 0);
        const uint32_t lds = lds0 + static_cast<uint32_t>((j & (NS - 1)) * S::kStageBytes + 2 * S::kBlockBytes + i * 256);
        if constexpr (D == 64) short_to_lds(p, lds);
        else word_to_lds(p, lds);
      }
    }
  };
  auto copy_v = [&](const Pages& pg, int j) { copy_side(pg, j, 1); };
  // the first blocks leave at once; Q and the table are loaded behind them
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    if (j < mine) {
      const Pages pg = pages_of(j);
      copy_k(pg, j);
      copy_v(pg, j);
    }
  }

  // ---- this lane's rows (li of each block of 16)
  int pos[NR];
  bf16x8_t qf[NR][kKk];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int row = min(n * 16 + li, it.rows - it.row0 - 1);  // rows behind the last one repeat it and are not stored
    const int local = token_of(a, it, row), token = it.token0 + local;
    pos[n] = it.len - it.n_new + token;
    const int b = a.cu == nullptr ? it.req : 0;
    const int head = it.head * a.group + (it.rem0 + row - local * a.group);
    const uint16_t* qp = a.q + b * a.qs[0] + head * a.qs[1] + static_cast<int64_t>(it.start + token) * a.qs[2];
    // the features of a product's step are any 32, the same ones of Q and K: of E2M1 a lane takes D / 4 in a row, so that
    // its codes of a key are one read with few scales
#pragma unroll
    for (int kk = 0; kk < kKk; ++kk)
      qf[n][kk] = *reinterpret_cast<const bf16x8_t*>(qp + (FP4 ? grp * (D / 4) + kk * 8 : kk * 32 + grp * 8));
  }
  const int pos_min = it.len - it.n_new + it.token0;
  const bool absent = any_absent<S>(a, job, table, lane);

  f32x4_t o[NR][kNdb];
  float m_run[NR], l_run[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m_run[n] = -__builtin_inff();  // running maximum (log2 units), may lag the true one by 8
    l_run[n] = 0.0f;               // this lane's part of the denominator
#pragma unroll
    for (int db = 0; db < kNdb; ++db) o[n][db] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  bf16x8_t pb[NR], pl[NR];  // probabilities, in two parts
  // E2M1: a block's codes and scales on their way from LDS: K of this lane's two keys, V of half a row
  uint32_t k_codes[2][FP4 ? kKk : 1], v_codes[FP4 ? D / 16 : 1], v_scales[D == 256 ? 2 : 1];
  float k_scales[2][D == 256 ? 2 : 1];
  auto take = [&](int j) {
    const unsigned char* const st = stage0 + (j & (NS - 1)) * S::kStageBytes;
    const unsigned char* const sc = st + 2 * S::kBlockBytes;
    auto words = [](const unsigned char* p, uint32_t* to) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      to[0] = w.x, to[1] = w.y, to[2] = w.z, to[3] = w.w;
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = sigma16(h, li), swz = few_swz_k<RBY>(row);
      if constexpr (D == 64) {
        const uint2 w = *reinterpret_cast<const uint2*>(st + row * RBY + ((grp >> 1) ^ swz) * 16 + 8 * (grp & 1));
        k_codes[h][0] = w.x, k_codes[h][1] = w.y;
        k_scales[h][0] = scale_of(sc[row * 4 + (grp >> 1)]);
      } else {
#pragma unroll
        for (int c = 0; c < D / 128; ++c) {
          words(st + row * RBY + ((grp * (D / 128) + c) ^ swz) * 16, &k_codes[h][4 * c]);
          k_scales[h][c] = scale_of(sc[row * (D / kScaleBlock) + grp * (D / 128) + c]);
        }
      }
    }
    // V: of every S::kWide features of row lane / 2 the lane takes half, in 16-byte chunks
    const int row = lane >> 1, half = lane & 1, swz = few_swz_v<RBY, kE2m1>(row);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      constexpr int kHalf = S::kWide / 64;  // chunks of a lane in S::kWide features
      words(st + S::kBlockBytes + row * RBY + (((c / kHalf) * 2 * kHalf + half * kHalf + c % kHalf) ^ swz) * 16, &v_codes[4 * c]);
    }
#pragma unroll
    for (int c = 0; c < (D == 256 ? 2 : 1); ++c)
      v_scales[c] = reinterpret_cast<const uint32_t*>(sc + (D == 256 ? 256 : 128))[row * (D == 256 ? 2 : 1) + c];
  };

  auto scores = [&](int j) {
    const unsigned char* const st = stage0 + (j & (NS - 1)) * S::kStageBytes;
    const int kb0 = first + j * S::kKeys;
    f32x4_t s[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) s[n][0] = s[n][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = sigma16(h, li);
      const int swz = few_swz_k<RBY>(row);
#pragma unroll
      for (int kk = 0; kk < kKk; ++kk) {
        bf16x8_t kf;
        if constexpr (FP4) {
          kf = e2m1_to_bf16(k_codes[h][kk], k_scales[h][kk / 4]);
        } else if constexpr (FP8) {
          const uint2 w = *reinterpret_cast<const uint2*>(st + row * RBY + ((2 * kk + (grp >> 1)) ^ swz) * 16 + 8 * (grp & 1));
          kf = codes_to_bf16(w.x, w.y);
        } else {
          kf = *reinterpret_cast<const bf16x8_t*>(st + row * RBY + ((4 * kk + grp) ^ swz) * 16);
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][kk], s[n][h], 0, 0, 0);
      }
    }
    float ks[8], vs[8];
    if constexpr (FP8) {
      const uint4* const sc = reinterpret_cast<const uint4*>(st + 2 * S::kBlockBytes);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 kw = sc[2 * grp + h], vw = sc[8 + 2 * grp + h];
        const uint32_t ku[4] = {kw.x, kw.y, kw.z, kw.w}, vu[4] = {vw.x, vw.y, vw.z, vw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ks[4 * h + e] = scale_of(ku[e]);
          vs[4 * h + e] = scale_of(vu[e]);
        }
      }
    }
    const bool masked = kb0 + 31 > pos_min || absent;
    bool there = true;
    if (absent) {
      bool t[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = uniform(min(kb0 + 16 * h, kend - 1));
        t[h] = static_cast<unsigned>(scalar_load(table, key >> a.c.shift)) < static_cast<unsigned>(a.c.n_pages);
      }
      there = grp < 2 ? t[0] : t[1];
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[n][e >> 2][e & 3];
        if constexpr (FP8) x[e] *= ks[e];
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (kb0 + 8 * grp + e > pos[n] || !there) x[e] = -__builtin_inff();
      }
      float mx = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
      mx = fd_xor_max<32>(fd_xor_max<16>(mx)) * a.scale_log2;
      const bool grow = mx > m_run[n] + 8.0f;
      const float m_new = grow ? mx : m_run[n];
      const float alpha = grow ? __builtin_amdgcn_exp2f(m_run[n] - m_new) : 1.0f;
      const float m_sub = m_new == -__builtin_inff() ? 0.0f : m_new;  // nothing seen so far: p = 0
      m_run[n] = m_new;
      if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
        for (int db = 0; db < kNdb; ++db) o[n][db] *= alpha;
      }
      f32x8_t pv;
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale_log2, -m_sub));
      float psum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) psum += pv[e];
      l_run[n] = l_run[n] * alpha + psum;
      if constexpr (FP8) {  // V's scales go to P
#pragma unroll
        for (int e = 0; e < 8; ++e) pv[e] = masked && pv[e] == 0.0f ? 0.0f : pv[e] * vs[e];
      }
      two_bf16(pv, &pb[n], &pl[n]);
    }
  };

  auto p_v = [&](int j) {
    const unsigned char* const st = stage0 + (j & (NS - 1)) * S::kStageBytes + S::kBlockBytes;
    bf16x8_t vf[kNdb];  // V[key 8 grp + i][16 db + li]
#pragma unroll
    for (int db = 0; db < kNdb; ++db) {
      if constexpr (FP8) {
        typedef int v2i_t __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) v2i_t lds_v2i_t;
        const int row = 8 * grp + (li >> 1);
        const v2i_t w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_v2i_t*)(st + row * RBY + (db ^ few_swz_v<RBY, kE4m3>(row)) * 16 + 8 * (li & 1)));
        vf[db] = codes_to_bf16(static_cast<uint32_t>(w[0]), static_cast<uint32_t>(w[1]));
      } else {
        const int row = 8 * grp + (li >> 2);
        const unsigned char* vp = st + row * RBY + ((2 * db + ((li & 3) >> 1)) ^ few_swz_v<RBY, kBf16>(row)) * 16 + 8 * (li & 1);
        const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)vp);
        const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(vp + 4 * RBY));
        const short __attribute__((ext_vector_type(8))) vv = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        vf[db] = __builtin_bit_cast(bf16x8_t, vv);
      }
    }
    // a block with masked keys: their values must not reach a row as 0 * NaN or 0 * inf
    if (first + j * S::kKeys + 31 > pos_min || absent) {
      bool odd = false;
#pragma unroll
      for (int db = 0; db < kNdb; ++db) odd |= any_odd(vf[db]);
      if (__builtin_amdgcn_ballot_w64(odd) != 0) {
        // Infinities and NaN leave the product and are added by hand to the rows that see them: o[n][db][r]
        // is feature 16 db + 4 grp + r of this lane's row.
#pragma unroll
        for (int db = 0; db < kNdb; ++db) vf[db] = without_odd(vf[db]);
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {
          float ph[NR];
#pragma unroll
          for (int n = 0; n < NR; ++n) ph[n] = __shfl(element(pb[n], key & 7) + element(pl[n], key & 7), 16 * (key >> 3) + li);
#pragma unroll
          for (int db = 0; db < kNdb; ++db) {
            f32x4_t x;
            if constexpr (FP8) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(st + key * RBY + (db ^ few_swz_v<RBY, kE4m3>(key)) * 16 + 4 * grp);
              x = __builtin_convertvector(__builtin_shufflevector(codes_to_bf16(w, w), bf16x8_t{}, 0, 1, 2, 3), f32x4_t);
            } else {
              x = __builtin_convertvector(*reinterpret_cast<const bf16x4_t*>(
                  st + key * RBY + ((2 * db + (grp >> 1)) ^ few_swz_v<RBY, kBf16>(key)) * 16 + 8 * (grp & 1)), f32x4_t);
            }
#pragma unroll
            for (int n = 0; n < NR; ++n) o[n][db] = add_odd(o[n][db], x, ph[n]);
          }
        }
      }
    }
#pragma unroll
    for (int db = 0; db < kNdb; ++db)
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        o[n][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[db], pb[n], o[n][db], 0, 0, 0);
        o[n][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[db], pl[n], o[n][db], 0, 0, 0);
      }
  };

  // E2M1: V becomes bf16 in LDS of the wavefront, S::kWide features at a time, from where the transposing reads take it.
  constexpr int VBY = 2 * S::kWide;  // bytes of a row there
  unsigned char* const wide = smem + S::kWaves * NS * S::kStageBytes + wave * S::kDecoded;
  auto widen_v = [&](int part) {
    const int row = lane >> 1, half = lane & 1, swz = few_swz_v<VBY, kBf16>(row);
    constexpr int kEights = S::kWide / 16;  // of a lane
#pragma unroll
    for (int c = 0; c < kEights; ++c) {
      const int block = part * (S::kWide / kScaleBlock) + c / 4;  // scale of half 0; half 1's lies S::kWide / 64 further
      const uint32_t word = v_scales[block / 4] >> (half * (S::kWide / 64) * 8);
      const float scale = scale_of(word >> (8 * (block % 4)) & 255u);
      *reinterpret_cast<bf16x8_t*>(wide + row * VBY + ((half * kEights + c) ^ swz) * 16) = e2m1_to_bf16(v_codes[part * kEights + c], scale);
    }
  };
  auto p_v_wide = [&](int j, int part) {
    constexpr int kDb = S::kWide / 16;
    bf16x8_t vf[kDb];  // V[key 8 grp + i][S::kWide part + 16 db + li]
#pragma unroll
    for (int db = 0; db < kDb; ++db) {
      const int row = 8 * grp + (li >> 2);
      const unsigned char* vp = wide + row * VBY + ((2 * db + ((li & 3) >> 1)) ^ few_swz_v<VBY, kBf16>(row)) * 16 + 8 * (li & 1);
      const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)vp);
      const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(vp + 4 * VBY));
      const short __attribute__((ext_vector_type(8))) vv = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      vf[db] = __builtin_bit_cast(bf16x8_t, vv);
    }
    if (first + j * S::kKeys + 31 > pos_min || absent) {
      bool odd = false;
#pragma unroll
      for (int db = 0; db < kDb; ++db) odd |= any_odd(vf[db]);
      if (__builtin_amdgcn_ballot_w64(odd) != 0) {  // blocks of NaN: as in p_v
#pragma unroll
        for (int db = 0; db < kDb; ++db) vf[db] = without_odd(vf[db]);
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {
          float ph[NR];
#pragma unroll
          for (int n = 0; n < NR; ++n) ph[n] = __shfl(element(pb[n], key & 7) + element(pl[n], key & 7), 16 * (key >> 3) + li);
#pragma unroll
          for (int db = 0; db < kDb; ++db) {
            const f32x4_t x = __builtin_convertvector(*reinterpret_cast<const bf16x4_t*>(
                wide + key * VBY + ((2 * db + (grp >> 1)) ^ few_swz_v<VBY, kBf16>(key)) * 16 + 8 * (grp & 1)), f32x4_t);
#pragma unroll
            for (int n = 0; n < NR; ++n) o[n][part * kDb + db] = add_odd(o[n][part * kDb + db], x, ph[n]);
          }
        }
      }
    }
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        f32x4_t& y = o[n][part * kDb + db];
        y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[db], pb[n], y, 0, 0, 0);
        y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[db], pl[n], y, 0, 0, 0);
      }
  };

  // ---- the loop: copies in the queue, oldest first, at block j's scores: K(j) V(j) .. K(j + NS - 1) V(j + NS - 1)
  constexpr int kBoth = S::kKGroup + S::kCopies;
  Pages next = pages_of(NS);
  for (int j = 0; j < mine; ++j) {
    const bool more = j + NS < mine;
    if constexpr (FP4) {
      // the block leaves its stage for registers, and the stage's next copies leave before any of its work
      if (more || j + NS == mine) wait_copies<(NS - 1) * kBoth>();
      else wait_copies<0>();
      take(j);
      wait_lds_reads();
      if (more) {
        copy_k(next, j + NS);
        copy_v(next, j + NS);
      }
      next = pages_of(j + NS + 1);
      widen_v(0);
      scores(j);
      p_v_wide(j, 0);
#pragma unroll
      for (int part = 1; part < D / S::kWide; ++part) {
        widen_v(part);
        p_v_wide(j, part);
      }
      continue;
    }
    if (more || j + NS == mine) wait_copies<S::kCopies + (NS - 1) * kBoth>();  // K(j) has landed
    else wait_copies<0>();
    scores(j);
    wait_lds_reads();
    if (more) {
      copy_k(next, j + NS);
      wait_copies<(NS - 1) * kBoth + S::kKGroup>();  // V(j) has landed
    } else {
      wait_copies<0>();
    }
    p_v(j);
    wait_lds_reads();
    if (more) copy_v(next, j + NS);
    next = pages_of(j + NS + 1);
  }

  // ---- join the wavefronts' keys
  __syncthreads();  // the stages are free
  float* const rowsf = reinterpret_cast<float*>(smem);
  float* const ml = rowsf + S::kWaves * S::kRows * S::kRowFloats;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int at = wave * S::kRows + n * 16 + li;
#pragma unroll
    for (int db = 0; db < kNdb; ++db)
      *reinterpret_cast<f32x4_t*>(rowsf + at * S::kRowFloats + db * 16 + 4 * grp) = o[n][db];
    const float l = fd_xor_sum<32>(fd_xor_sum<16>(l_run[n]));
    if (grp == 0) {
      ml[at * 2] = m_run[n];
      ml[at * 2 + 1] = l;
    }
  }
  __syncthreads();
  close_job<S, S::kWaves>(a, job, rowsf, ml);
}

// ---------------------------------------------------------------- pieces

// Runs f(u) for the softmax pieces u (8 per row block) that go behind MFMA m of a phase of NB * STEPS MFMAs.
template <int NB, int STEPS, typename F>
__device__ __forceinline__ void pieces(int m, F f) {
  constexpr int kAll = 8 * NB, kMfma = NB * STEPS;
  if constexpr (kAll >= kMfma) {
#pragma unroll
    for (int u = 0; u < kAll / kMfma; ++u) f(m * (kAll / kMfma) + u);
  } else {
    if (m % (kMfma / kAll) == 0) f(m / (kMfma / kAll));
  }
}

// A wavefront owns NB blocks of 32 rows and every KS-th block of 32 keys.  A block of 128 features is 64 registers of
// O^T and 32 of Q.  Two blocks per wavefront, four wavefronts: an operand read from LDS feeds two MFMAs, one wavefront
// per SIMD.  One block, eight wavefronts: two per SIMD fill each other's waits, each operand read feeds one MFMA (1 KiB
// per 32-cycle MFMA on 4 SIMDs is all of LDS's 128 bytes per cycle, at a half-busy matrix core half of it).  Measured at
// 128 features, four and eight wavefronts: 2048 tokens on 6144 keys 149 and 141 us, E4M3 189 and 163, on 14336 267 and
// 263, 2048 alone 46.1 and 42.3.  256 features (128 + 64 registers of a block) leave room for one wavefront per SIMD; at
// 64 the four of a workgroup leave room for a second workgroup.
//
// Tiles that all rows see whole run in a pipelined loop without masks; the rest (the new tokens' own
// tiles, and everything of a request with absent pages) in a plain one.  A pipelined step t has two
// phases with one barrier between them:
//   A: the score MFMAs of tile t + 1; between them the second half of tile t's softmax and the reads
//      of tile t's V operands
//   B: the P V MFMAs of tile t; between them the first half of tile t + 1's softmax and the reads of
//      tile t + 2's K operands
// so that the softmax's VALU and exp work runs under both halves of the MFMAs and every operand is
// read a phase before it is used.  Four LDS stages: bf16 tiles are copied three steps ahead (asm copies,
// counted by hand), codes are loaded into registers three steps ahead and stored as bf16 two ahead.
//
// Measured, 2048 new tokens on 6144 cached ones: 16 / 4 heads x 128 features 142 us, 845 TFLOP/s (14336 cached
// 263 us, 978; a large library product here: 1370), x 64 104 us, 8 / 2 x 256 148 us, 810; E4M3 164, 127 and
// 175.  2048 tokens alone: 42 to 46 us.  A workgroup (128 features) spends 1.8 us on finding its item, 3.4 to 3.9 until
// its first tiles and Q are there, 1.05 per whole tile of 64 keys, 0.7 on the last one, 1.9 to 3 on the masked ones, 1.9
// on its rows.  In the loop MFMA, VALU, and LDS reads are each busy for a third to a half of the time, with a
// barrier per tile.  LDS conflicts are not the bound: E4M3's 8% of cycles could be removed without any gain.
template <class S>
__global__ __launch_bounds__(S::kThreads) void paged_gqa_piece_kernel(PagedArgs a) {
  constexpr int D = S::D, NB = S::NB, CR = S::CR, kNdb = D / 32, kSteps = D / 16, kAhead = 4;
  constexpr bool CODES = S::CODES;
  constexpr int kScales = S::F == kE2m1 ? D / kScaleBlock : 1;  // scale bytes of a row
  __shared__ __attribute__((aligned(1024))) unsigned char smem[S::kSmemBytes];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int rw = wave % S::RW;   // row wavefront
  const int kp = wave / S::RW;   // key part
  const int col = lane & 31, half = lane >> 5;

  Job job;
  if (!open_job<S>(a, lane, &job)) return;
  const Item& it = job.it;
  const int kend = job.kend, t0 = uniform(job.t0), nt = uniform(job.nt);

  // ---- this lane's rows: col of each of the wavefront's row blocks
  int pos[NB];
  bf16x8_t qf[NB][kSteps];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int row = min((rw * NB + n) * 32 + col, it.rows - it.row0 - 1);  // rows behind the last repeat it, not stored
    const int local = token_of(a, it, row), token = it.token0 + local;
    pos[n] = it.len - it.n_new + token;
    const int b = a.cu == nullptr ? it.req : 0;
    const int head = it.head * a.group + (it.rem0 + row - local * a.group);
    const uint16_t* qp = a.q + b * a.qs[0] + head * a.qs[1] + static_cast<int64_t>(it.start + token) * a.qs[2] + half * 8;
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) qf[n][kk] = *reinterpret_cast<const bf16x8_t*>(qp + kk * 16);
  }
  const int32_t* const table = a.c.table + it.req * a.c.table_stride;
  const int page_mask = (1 << a.c.shift) - 1;
  const bool absent = any_absent<S>(a, job, table, lane);
  // tiles [0, n_full) of the job are seen whole by every row of the workgroup
  const int pos_first = it.len - it.n_new + it.token0;
  const int n_full = uniform(absent ? 0 : max(0, min(nt, (pos_first + 1) / S::kKeys - t0)));

  // ---- staging.  The kMoveRows rows of a copy (or load) lie on one page: its address is a scalar base plus
  // a lane offset that depends on no tile.  Tiles that reach past kend repeat row kend - 1 there (the mask
  // discards it).
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_t*)smem));
  unsigned char* const k_lds = smem;
  unsigned char* const v_lds = smem + S::kStages * S::kTileBytes;
  constexpr int kMoves = CODES ? S::kLoads : S::kCopies;  // per wavefront and side
  constexpr int kMoveRows = CODES ? S::kLoadRows : S::kCopyRows;
  constexpr int kLanesRow = 64 / kMoveRows;             // lanes of a row, 16 bytes each (of E2M1: 8)
  using Word = std::conditional_t<S::F == kE2m1, uint2, uint4>;  // 16 codes
  const int lrow = lane / kLanesRow, lcol = lane % kLanesRow;
  struct Pages {
    int p[kMoves];
  };
  auto move_row = [&](int i) { return (i * S::kWaves + wave) * kMoveRows; };  // first row of move i within a tile
  // whole: tiles of [0, n_full), all of whose pages are there
  auto pages_of = [&](auto whole_c, int t) {
    Pages x;
    const int first = (t0 + (decltype(whole_c)::value ? min(t, n_full - 1) : t)) * S::kKeys;
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int key = first + move_row(i);
      const int page = scalar_load(table, uniform(decltype(whole_c)::value ? key : max(min(key, kend - 1), 0)) >> a.c.shift);
      x.p[i] = decltype(whole_c)::value || static_cast<unsigned>(page) < static_cast<unsigned>(a.c.n_pages) ? page : 0;
    }
    return x;
  };
  // first row of move i of tile t on its page, and this lane's row from there
  auto first_row = [&](auto whole_c, int t, int i) {
    const int key = (t0 + t) * S::kKeys + move_row(i);
    return uniform(decltype(whole_c)::value ? key : min(key, kend - 1)) & page_mask;
  };
  auto lane_row = [&](auto whole_c, int t, int i) {
    if constexpr (decltype(whole_c)::value) return lrow;
    else return max(0, min(lrow, kend - 1 - ((t0 + t) * S::kKeys + move_row(i))));
  };
  // K (v = 0) and V of this head, at one offset; pages lie a multiple of 16 bytes apart, 32 bits of it
  const unsigned char* const head_base[2] = {a.c.k + it.head * a.c.head, a.c.v + it.head * a.c.head};
  const uint32_t page16 = static_cast<uint32_t>(a.c.page >> 4), row_bytes = static_cast<uint32_t>(a.c.row);
  const uint8_t* const scale_base[2] = {a.c.k_scale + it.head * a.c.s_head, a.c.v_scale + it.head * a.c.s_head};
  auto move_offset = [&](int page, int row) {
    return ((static_cast<uint64_t>(page16) * static_cast<uint32_t>(page)) << 4) + static_cast<uint32_t>(row) * row_bytes;
  };
  auto copy_piece = [&](auto whole_c, const Pages& pg, int t, int buf, int i, int v) {
    const int row = move_row(i) + lrow;
    const int chunk = (lane % CR) ^ (v ? swz_v<CR>(row) : swz_k<CR>(row));
    copy_to_lds(head_base[v] + move_offset(pg.p[i], first_row(whole_c, t, i)),
                static_cast<uint32_t>(lane_row(whole_c, t, i)) * row_bytes + static_cast<uint32_t>(chunk * 16),
                lds0 + static_cast<uint32_t>((v * S::kStages + buf) * S::kTileBytes + (i * S::kWaves + wave) * 1024));
  };
  auto copy_tile = [&](auto whole_c, const Pages& pg, int t, int buf) {
#pragma unroll
    for (int i = 0; i < S::kCopies; ++i)
#pragma unroll
      for (int v = 0; v < 2; ++v) copy_piece(whole_c, pg, t, buf, i, v);
  };
  struct Codes {
    Word w[CODES ? 2 * S::kLoads : 1];
    uint32_t s[CODES ? 2 * S::kLoads : 1];
  };
  auto load_piece = [&](auto whole_c, const Pages& pg, int t, Codes& x, int i, int v) {
    const uint32_t row = static_cast<uint32_t>(lane_row(whole_c, t, i));
    const int first = first_row(whole_c, t, i);
    x.w[2 * i + v] = *reinterpret_cast<const Word*>(head_base[v] + move_offset(pg.p[i], first) + (row * row_bytes + lcol * static_cast<int>(sizeof(Word))));
    x.s[2 * i + v] = (scale_base[v] + static_cast<uint64_t>(static_cast<uint32_t>(a.c.s_page)) * static_cast<uint32_t>(pg.p[i]) + first * kScales)
        [row * kScales + (kScales > 1 ? lcol / 2 : 0)];
  };
  auto store_piece = [&](const Codes& x, int buf, int i, int v) {
    const int row = move_row(i) + lrow;
    const float s = scale_of(x.s[2 * i + v]);
    unsigned char* const dst = (v ? v_lds : k_lds) + buf * S::kTileBytes + row * CR * 16;
    const int swz = v ? swz_v<CR>(row) : swz_k<CR>(row);
    const Word w = x.w[2 * i + v];
    bf16x8_t lo, hi;
    if constexpr (S::F == kE2m1) lo = e2m1_to_bf16(w.x, s), hi = e2m1_to_bf16(w.y, s);
    else lo = codes_to_bf16(w.x, w.y, s), hi = codes_to_bf16(w.z, w.w, s);
    *reinterpret_cast<bf16x8_t*>(dst + ((lcol * 2) ^ swz) * 16) = lo;
    *reinterpret_cast<bf16x8_t*>(dst + ((lcol * 2 + 1) ^ swz) * 16) = hi;
  };
  auto load_tile = [&](auto whole_c, const Pages& pg, int t, Codes& x) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i)
#pragma unroll
      for (int v = 0; v < 2; ++v) load_piece(whole_c, pg, t, x, i, v);
  };
  auto store_tile = [&](const Codes& x, int buf) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i)
#pragma unroll
      for (int v = 0; v < 2; ++v) store_piece(x, buf, i, v);
  };

  f32x16_t o[NB][kNdb];
  float m_run[NB], l_run[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m_run[n] = -__builtin_inff();  // running maximum (log2 units), may lag the true one by 8
    l_run[n] = 0.0f;               // this lane's part of the denominator
#pragma unroll
    for (int db = 0; db < kNdb; ++db) o[n][db] = f32x16_t{};
  }

  // ---- operand addresses within a tile.  K: row kp * 32 + sigma(col), chunk 2 kk + half.  V^T of O
  // block db: two transposing reads (keys + 0..3, + 4..7) per 16-key slice.
  const int grp = lane >> 4, li = lane & 15;
  int k_rd[kSteps], v_rd[kNdb];
#pragma unroll
  for (int kk = 0; kk < kSteps; ++kk) {
    const int row = kp * 32 + sigma(col);
    k_rd[kk] = row * CR * 16 + (((2 * kk + half) ^ swz_k<CR>(row)) * 16);
  }
#pragma unroll
  for (int db = 0; db < kNdb; ++db) {
    const int dim = db * 32 + 16 * (grp & 1) + 4 * (li & 3);
    const int row = kp * 32 + 8 * (grp >> 1) + (li >> 2);
    v_rd[db] = S::kStages * S::kTileBytes + row * CR * 16 + (((dim >> 3) ^ swz_v<CR>(row)) * 16) + (dim & 7) * 2;
  }
  bf16x8_t kf[kAhead];               // K operands a few MFMAs ahead
  v4i16_t vlo[kSteps], vhi[kSteps];  // V operands of a tile; MFMA i: slice i / kNdb, O block i % kNdb
  auto read_k = [&](int buf, int kk) {
    kf[kk % kAhead] = *reinterpret_cast<const bf16x8_t*>(k_lds + buf * S::kTileBytes + k_rd[kk]);
  };
  auto read_v = [&](int buf, int i) {
    const unsigned char* vt = smem + buf * S::kTileBytes + v_rd[i % kNdb] + (i / kNdb) * 16 * CR * 16;
    vlo[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)vt);
    vhi[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(vt + 4 * CR * 16));
  };
  auto v_operand = [&](int i) {
    const short __attribute__((ext_vector_type(8))) vv = {vlo[i][0], vlo[i][1], vlo[i][2], vlo[i][3],
                                                          vhi[i][0], vhi[i][1], vhi[i][2], vhi[i][3]};
    return __builtin_bit_cast(bf16x8_t, vv);
  };

  // ---- softmax of a row block's scores, in pieces that fit behind one MFMA each: maximum and first half
  // of the probabilities (head), second half, rounding and denominator (tail)
  float p[NB][16], alpha[NB], m_sub[NB], mx[NB];
  bf16x8_t pb[NB][2];
  bool grow[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) alpha[n] = 1.0f, m_sub[n] = 0.0f, mx[n] = 0.0f, grow[n] = false;
  auto exps = [&](int n, const f32x16_t& s, int r0) {
#pragma unroll
    for (int r = r0; r < r0 + 2; ++r) {
      p[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.scale_log2, -m_sub[n]));
      asm volatile("" : "+v"(p[n][r]));  // computed here, not sunk towards its use in P V
    }
  };
  auto head = [&](int n, int k, const f32x16_t& s) {
    if (k < 2) {
      if (k == 0) mx[n] = s[0];
#pragma unroll
      for (int r = k == 0 ? 1 : 9; r < (k == 0 ? 9 : 16); ++r) mx[n] = fmaxf(mx[n], s[r]);
    } else if (k == 2) {
      mx[n] = half_max(mx[n]) * a.scale_log2;
      grow[n] = mx[n] > m_run[n] + 8.0f;
      const float m_new = grow[n] ? mx[n] : m_run[n];
      alpha[n] = grow[n] ? __builtin_amdgcn_exp2f(m_run[n] - m_new) : 1.0f;
      m_sub[n] = m_new == -__builtin_inff() ? 0.0f : m_new;  // nothing seen so far: p = 0
      m_run[n] = m_new;
    } else if (k < 7) {
      exps(n, s, 2 * (k - 3));
    }
  };
  auto round8 = [&](int n, int j) {
    pb[n][j] = __builtin_convertvector(f32x8_t{p[n][8 * j], p[n][8 * j + 1], p[n][8 * j + 2], p[n][8 * j + 3], p[n][8 * j + 4],
                                               p[n][8 * j + 5], p[n][8 * j + 6], p[n][8 * j + 7]}, bf16x8_t);
    asm volatile("" : "+v"(pb[n][j]));
  };
  auto tail = [&](int n, int k, const f32x16_t& s) {
    if (k < 4) {
      exps(n, s, 8 + 2 * k);
    } else if (k == 4) {
      round8(n, 0);
    } else if (k == 5) {
      round8(n, 1);
    } else if (k == 6) {
      // the denominator takes the rounded p: its error then cancels where a few keys carry the row
      l_run[n] = sum8(pb[n][1], sum8(pb[n][0], l_run[n] * alpha[n]));
      asm volatile("" : "+v"(l_run[n]));
    }
  };
  auto rescale = [&]() {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if (__builtin_amdgcn_ballot_w64(grow[n]) != 0) {
#pragma unroll
        for (int db = 0; db < kNdb; ++db) o[n][db] *= alpha[n];
      }
    }
  };

  const std::true_type whole{};
  const std::false_type part{};
  Codes codes;
  // The tiles behind the whole ones go to stage t % 4 too; the first of them (three, or one of codes) leave
  // before the pipelined loop's last step.
  constexpr int kAheadTiles = 3;
  auto ahead = [&]() {
    if constexpr (CODES) {
      if (n_full < nt) load_tile(part, pages_of(part, n_full), n_full, codes);
    } else {
#pragma unroll
      for (int u = 0; u < kAheadTiles; ++u)
        if (n_full + u < nt) copy_tile(part, pages_of(part, n_full + u), n_full + u, (n_full + u) & 3);
    }
  };
  if (n_full > 0) {
    f32x16_t sA[NB], sB[NB];
    Pages next;
    // Prologue: tiles 0 and 1 landed (Q too), tile 2 on its way; scores of tile 0 and the head of its softmax.
    if constexpr (!CODES) {
      copy_tile(whole, pages_of(whole, 0), 0, 0);
      if (n_full > 1) copy_tile(whole, pages_of(whole, 1), 1, 1);
      next = pages_of(whole, 2);
      wait_copies<0>();
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) asm volatile("" : "+v"(qf[n][kk]));  // the compiler's own loads end here
      if (n_full > 2) copy_tile(whole, next, 2, 2);
    } else {
      load_tile(part, pages_of(whole, 0), 0, codes);
      next = pages_of(whole, 1);
      store_tile(codes, 0);
      load_tile(part, next, 1, codes);  // (tiles behind the last whole one may reach past kend)
      next = pages_of(whole, 2);
      store_tile(codes, 1);
      load_tile(part, next, 2, codes);
    }
    next = pages_of(whole, 3);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; ++n) sA[n] = f32x16_t{};
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
      read_k(0, kk);
#pragma unroll
      for (int n = 0; n < NB; ++n) sA[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk % kAhead], qf[n][kk], sA[n], 0, 0, 0);
    }
    if (n_full > 1) {
#pragma unroll
      for (int kk = 0; kk < kAhead; ++kk) read_k(1, kk);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int k = 0; k < 8; ++k) head(n, k, sA[n]);

    // BUF = t % 4; LAST: no tile t + 1
    auto step = [&](auto last_c, int t, int BUF, f32x16_t (&sc)[NB], f32x16_t (&sn)[NB]) {
      constexpr bool LAST = decltype(last_c)::value;
      const bool issued = !LAST && t + 3 < n_full;
      // the moves of a step, one behind every kMoveEvery-th score MFMA: their scalar arithmetic is issued while
      // the matrix core works
      constexpr int kMoveEvery = NB * kSteps / (2 * kMoves);
      auto move_piece = [&](int u) {
        if constexpr (CODES) {
          if (t + 2 < n_full) store_piece(codes, (BUF + 2) & 3, u / 2, u % 2);
          if (issued) load_piece(whole, next, t + 3, codes, u / 2, u % 2);
        } else {
          if (issued) copy_piece(whole, next, t + 3, (BUF + 3) & 3, u / 2, u % 2);
        }
      };
      // ---- phase A
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!LAST) {
        // the pages are waited for here, not where they were asked for; Q stays in the accumulation half
#pragma unroll
        for (int i = 0; i < kMoves; ++i) asm volatile("" : "+s"(next.p[i]));
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) asm volatile("" : "+a"(qf[n][kk]));
#pragma unroll
        for (int n = 0; n < NB; ++n) sn[n] = f32x16_t{};
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            sn[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk % kAhead], qf[n][kk], sn[n], 0, 0, 0);
            if (n == NB - 1) {
              if (kk + kAhead < kSteps) read_k((BUF + 1) & 3, kk + kAhead);
              read_v(BUF, kk);
            }
            pieces<NB, kSteps>(kk * NB + n, [&](int u) { tail(u % NB, u / NB, sc[u % NB]); });
            if ((kk * NB + n) % kMoveEvery == 0) move_piece((kk * NB + n) / kMoveEvery);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) read_v(BUF, i);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int k = 0; k < 8; ++k) tail(n, k, sc[n]);
      }
      rescale();  // by tile t's alpha: phase B moves it on to tile t + 1
      if constexpr (!LAST) {
        if constexpr (!CODES) {
          if (issued) wait_copies<2 * S::kCopies>();  // all but this step's: tile t + 2 has landed
          else wait_copies<0>();
        }
        wait_lds_reads();  // the V operands have arrived, their stage is free after the barrier
        __syncthreads();
        next = pages_of(whole, t + 4);
      }
      // ---- phase B
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          o[n][i % kNdb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v_operand(i), pb[n][i / kNdb], o[n][i % kNdb], 0, 0, 0);
          if constexpr (!LAST) {
            if (n == 0 && i >= kSteps - kAhead) read_k((BUF + 2) & 3, i - (kSteps - kAhead));
            pieces<NB, kSteps>(i * NB + n, [&](int u) { head(u % NB, u / NB, sn[u % NB]); });
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    const std::false_type mid{};
    const std::true_type last{};
    const int n1 = n_full - 1;
    int t = 0;
    for (; t + 4 <= n1; t += 4) {
      step(mid, t, 0, sA, sB);
      step(mid, t + 1, 1, sB, sA);
      step(mid, t + 2, 2, sA, sB);
      step(mid, t + 3, 3, sB, sA);
    }
    if (t < n1) step(mid, t, 0, sA, sB);
    if (t + 1 < n1) step(mid, t + 1, 1, sB, sA);
    if (t + 2 < n1) step(mid, t + 2, 2, sA, sB);
    if (n1 & 1) {
#pragma unroll
      for (int n = 0; n < NB; ++n) sA[n] = sB[n];
    }
    ahead();  // every stage but tile n1's is free since the last barrier
    step(last, n1, n1 & 3, sA, sB);
  } else {
    ahead();
  }

  // ---- the other tiles: masked, and with values of masked keys kept out
#pragma unroll 1
  for (int t = n_full; t < nt; ++t) {
    const bool early = t < n_full + kAheadTiles;  // copied ahead
    const int buf = CODES || early ? t & 3 : 0;
    if constexpr (CODES) {
      store_tile(codes, buf);  // (the stages being read are those of tiles t - 1 and earlier)
      if (t + 1 < nt) load_tile(part, pages_of(part, t + 1), t + 1, codes);
      __syncthreads();
    } else if (!early || t == n_full) {
      if (!early) {
        __syncthreads();  // every wavefront has read the tile before
        copy_tile(part, pages_of(part, t), t, 0);
      }
      wait_copies<0>();
      __syncthreads();
    }
    const int kb0 = (t0 + t) * S::kKeys + kp * 32;
    bool there[2] = {true, true};
    if (absent) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = uniform(min(kb0 + 16 * j, kend - 1));
        there[j] = static_cast<unsigned>(scalar_load(table, key >> a.c.shift)) < static_cast<unsigned>(a.c.n_pages);
      }
    }
    f32x16_t s[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) s[n] = f32x16_t{};
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
      read_k(buf, kk);
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk % kAhead], qf[n][kk], s[n], 0, 0, 0);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kb0 + (r >> 3) * 16 + half * 8 + (r & 7);
        if (key > pos[n] || !there[r >> 3]) s[n][r] = -__builtin_inff();
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) head(n, k, s[n]);
#pragma unroll
      for (int k = 0; k < 8; ++k) tail(n, k, s[n]);
    }
    rescale();
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int j = i / kNdb, db = i % kNdb;
      read_v(buf, i);
      bf16x8_t vf = v_operand(i);  // V[key 16 j + 8 half + e][32 db + col]
      if (__builtin_amdgcn_ballot_w64(any_odd(vf)) != 0) {
        // infinities and NaN leave the product (0 times one is NaN) and are added by hand to the rows that see them
#pragma unroll 1
        for (int u = 0; u < 8; ++u) {
          const float v = element(vf, u);
          const float x = fabsf(v) < __builtin_inff() ? 0.0f : v;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const float pu = element(pb[n][j], u);
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              const float ph = __shfl(pu, h * 32 + col);  // this lane's row, key 16 j + 8 h + u
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const float xd = __shfl(x, h * 32 + (r & 3) + 8 * (r >> 2) + 4 * half);  // feature of o[n][db][r]
                if (xd != 0.0f && ph != 0.0f) o[n][db][r] += ph * xd;
              }
            }
          }
        }
        vf = without_odd(vf);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) o[n][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pb[n][j], o[n][db], 0, 0, 0);
    }
  }

  // ---- the key parts joined: with two of them each keeps half (of two row blocks one, of one block half its features)
  // and gives the other one away through LDS, in registers' order.  Then the rows leave from registers, 8 features (of
  // 16) of a row per lane.  (Through LDS row by row, 16 rounds of a few dependent reads each, it took 5 us of every item.)
  constexpr int kOwn = S::KS == 2 && NB == 1 ? kNdb / 2 : kNdb;  // blocks of 32 features that this wavefront stores
  f32x16_t acc[kOwn];
  float m = m_run[0], l = half_sum(l_run[0]);
  int n_own = 0, d_own = 0;
  if constexpr (S::KS == 2) {
    n_own = NB == 2 ? kp : 0;
    d_own = NB == 2 ? 0 : kp * (D / 2);
    __syncthreads();  // the stages are free
    constexpr int kGave = kOwn * 4;
    float* const gave = reinterpret_cast<float*>(smem) + lane * 4;
    float* const gave_ml = reinterpret_cast<float*>(smem) + S::kWaves * 256 * kGave + lane * 2;
    float m_give = m, l_give = l;
    if constexpr (NB == 2) {
      const float l1 = half_sum(l_run[1]);
      m_give = kp ? m : m_run[1], l_give = kp ? l : l1;
      m = kp ? m_run[1] : m;
      l = kp ? l1 : l;
    }
#pragma unroll
    for (int db = 0; db < kOwn; ++db) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        f32x4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = o[0][db][4 * r4 + e];
          const float p1 = NB == 2 ? o[NB - 1][db][4 * r4 + e] : o[0][(db + kOwn) % kNdb][4 * r4 + e];
          x[e] = kp ? p0 : p1;
          acc[db][4 * r4 + e] = kp ? p1 : p0;
        }
        *reinterpret_cast<f32x4_t*>(gave + (wave * kGave + db * 4 + r4) * 256) = x;
      }
    }
    gave_ml[wave * 128] = m_give;
    gave_ml[wave * 128 + 1] = l_give;
    __syncthreads();
    const int other = kp ? wave - S::RW : wave + S::RW;  // the other key part of these rows
    const float m2 = gave_ml[other * 128], l2 = gave_ml[other * 128 + 1];
    const float top = fmaxf(m, m2), sub = top == -__builtin_inff() ? 0.0f : top;
    const float w = __builtin_amdgcn_exp2f(m - sub), w2 = __builtin_amdgcn_exp2f(m2 - sub);
    m = top;
    l = l * w + l2 * w2;
#pragma unroll
    for (int db = 0; db < kOwn; ++db) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(gave + (other * kGave + db * 4 + r4) * 256);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[db][4 * r4 + e] = acc[db][4 * r4 + e] * w + x[e] * w2;
      }
    }
  } else {
    static_assert(S::KS == 1 && NB == 1, "nothing to join");
#pragma unroll
    for (int db = 0; db < kNdb; ++db) acc[db] = o[0][db];
  }
  // features 32 db + 16 j + 4 half + 0..3 and the same + 8: the halves exchange theirs for 8 in a row, from 8 half on
#pragma unroll
  for (int db = 0; db < kOwn; ++db) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[db][8 * j + e]), __float_as_uint(acc[db][8 * j + 4 + e]), false, false);
        acc[db][8 * j + e] = __uint_as_float(r[0]);
        acc[db][8 * j + 4 + e] = __uint_as_float(r[1]);
      }
    }
  }
  const int row = (rw * NB + n_own) * 32 + col;
  if (row >= it.rows - it.row0) return;
  if (job.split) {
    float* const at = a.part + job.slot * part_floats<S::kRows>(D);
    if (half == 0 && d_own == 0) {
      at[S::kRows * D + row * 2] = m;
      at[S::kRows * D + row * 2 + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < 2 * kOwn; ++i) {
      f32x4_t* const dst = reinterpret_cast<f32x4_t*>(at + row * D + d_own + 16 * i + 8 * half);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x16_t& x = acc[i / 2];
        const int e = 8 * (i % 2) + 4 * u;
        dst[u] = f32x4_t{x[e], x[e + 1], x[e + 2], x[e + 3]};
      }
    }
    return;
  }
  const int local = token_of(a, it, row);
  const int head_q = it.head * a.group + (it.rem0 + row - local * a.group);
  const int b = a.cu == nullptr ? it.req : 0;
  const int64_t tok = it.start + it.token0 + local;
  uint16_t* const dst = a.o + b * a.os[0] + head_q * a.os[1] + tok * a.os[2] + d_own + 8 * half;
  const uint16_t* const gate = a.gate == nullptr ? nullptr : a.gate + b * a.gs[0] + head_q * a.gs[1] + tok * a.gs[2] + d_own + 8 * half;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 2 * kOwn; ++i) {
    f32x8_t v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = acc[i / 2][8 * (i % 2) + e] * inv;
    if (gate != nullptr) {
      const f32x8_t g = __builtin_convertvector(*reinterpret_cast<const bf16x8_t*>(gate + 16 * i), f32x8_t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] / (1.0f + __expf(-g[e]));
    }
    *reinterpret_cast<bf16x8_t*>(dst + 16 * i) = __builtin_convertvector(v, bf16x8_t);
  }
}

// Joins the key ranges of every split row tile and stores its rows, ROWS of them per workgroup.  16, many row tiles:
// bound by the fp32 parts it reads: 2048 tokens x 8 heads x 256 features in two ranges, 34 MB in 11 us.  2 or 4, few
// row tiles: there are many ranges then, read in turn they would cost a memory latency per four of them; the threads
// that the rows leave over take ranges of their own, joined through LDS.
template <class S, int ROWS>
__global__ __launch_bounds__(256) void paged_gqa_join_kernel(PagedArgs a) {
  constexpr int D = S::D;
  constexpr int kLanes = D / 4;  // of a row
  constexpr int kRowsAtOnce = ROWS < 256 / kLanes ? ROWS : 256 / kLanes;
  constexpr int kGroups = 256 / kLanes / kRowsAtOnce;  // of ranges
  Item it;
  const int b = blockIdx.x;
  if (!find_item<S::kRows, S::kKeys, true>(a, threadIdx.x & 63, [&](int) { return b; }, &it)) return;
  const int nt_all = (keys_of_tile<S::kRows>(a, it) + S::kKeys - 1) / S::kKeys;
  const int ranges = (nt_all + it.tiles - 1) / it.tiles;
  if (ranges <= 1) return;  // its one item has stored the rows
  const int slot = it.base + it.head * it.n_ranges * it.n_rtiles + it.rtile;
  if (slot < 0 || slot + (ranges - 1) * static_cast<int64_t>(it.n_rtiles) >= a.part_items) return;
  const int row_end = min(min(S::kRows, it.rows - it.row0), static_cast<int>(blockIdx.y + 1) * ROWS);
  const int64_t step = it.n_rtiles * part_floats<S::kRows>(D);  // from one range's part to the next one's
  const float* const part = a.part + slot * part_floats<S::kRows>(D);
  const int d = (threadIdx.x % kLanes) * 4;
  const int own = threadIdx.x / kLanes % kRowsAtOnce, group = threadIdx.x / kLanes / kRowsAtOnce;
  for (int row0 = blockIdx.y * ROWS; row0 < row_end; row0 += kRowsAtOnce) {
    const int row = min(row0 + own, row_end - 1);
    // four ranges at a time: their loads are in flight together
    float m = -__builtin_inff(), l = 0.0f;
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 4 * group; s0 < ranges; s0 += 4 * kGroups) {
      float ms[4], ls[4];
      f32x4_t os[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* ps = part + min(s0 + u, ranges - 1) * step;
        ms[u] = ps[S::kRows * D + row * 2];
        ls[u] = ps[S::kRows * D + row * 2 + 1];
        os[u] = *reinterpret_cast<const f32x4_t*>(ps + row * D + d);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (s0 + u >= ranges) ms[u] = -__builtin_inff(), ls[u] = 0.0f, os[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        top = fmaxf(top, ms[u]);
      }
      const float sub = top == -__builtin_inff() ? 0.0f : top;
      const float keep = __builtin_amdgcn_exp2f(m - sub);
      l *= keep;
      acc *= keep;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = __builtin_amdgcn_exp2f(ms[u] - sub);
        l += ls[u] * w;
        acc += os[u] * w;
      }
      m = top;
    }
    if constexpr (kGroups > 1) {
      static_assert(ROWS == kRowsAtOnce, "one round of rows: LDS is used once");
      __shared__ float ml[kGroups][kRowsAtOnce][2];
      __shared__ f32x4_t os[kGroups][kRowsAtOnce][kLanes];
      os[group][own][d / 4] = acc;
      if (d == 0) ml[group][own][0] = m, ml[group][own][1] = l;
      __syncthreads();
      if (group != 0) return;
#pragma unroll
      for (int g = 1; g < kGroups; ++g) {
        const float mg = ml[g][own][0], top = fmaxf(m, mg), sub = top == -__builtin_inff() ? 0.0f : top;
        const float w = __builtin_amdgcn_exp2f(m - sub), wg = __builtin_amdgcn_exp2f(mg - sub);
        l = l * w + ml[g][own][1] * wg;
        acc = acc * w + os[g][own][d / 4] * wg;
        m = top;
      }
    }
    if (row0 + own < row_end) store4(a, it, row, d, acc, l == 0.0f ? 0.0f : 1.0f / l);
  }
}

// 128 rows (see the kernel): 4 wavefronts, at 128 features 8
template <int D, Format F>
using PieceOf = std::conditional_t<D == 256, Piece<D, F, 4, 1, 1>,
                                   std::conditional_t<D == 128, Piece<D, F, 4, 1, 2>, Piece<D, F, 2, 2, 2>>>;

template <Format F>
constexpr bool kCodesPerCu = Few<64, F, 1>::kPerCu == 2 && Few<128, F, 1>::kPerCu == 2 && Few<256, F, 1>::kPerCu == 2 &&
                             Few<64, F, 2>::kPerCu == 2 && Few<128, F, 2>::kPerCu == 2 && Few<256, F, 2>::kPerCu == 1;
static_assert(Few<64, kBf16, 1>::kPerCu == 2 && Few<64, kBf16, 2>::kPerCu == 2 && kCodesPerCu<kE4m3> && kCodesPerCu<kE2m1>,
              "plan_of's workgroups per CU");
constexpr int kHeaderBytes = 256;  // of the workspace: range_tiles

// The kernel of a call, and its items, row tiles and workspace, whatever the lengths turn out to be.
struct Plan {
  int few;  // blocks of 16 rows of the few-rows kernel, 0: pieces
  int rows, keys, slots, min_tiles;
  int64_t items, part_items, rtiles, bytes;
  bool may_split;
};

Plan plan_of(int64_t requests, int64_t tokens, int group, int kv_heads, int head_dim, int64_t max_keys, int max_seqlen,
             Format format) {
  const bool codes = format != kBf16;
  Plan p;
  const int64_t rows = static_cast<int64_t>(max_seqlen) * group;
  // Measured with 16 rows, 32 rows and pieces (us; 16/4 heads x 128 unless noted, 64 requests on 2048 keys):
  //   rows 32: 47, 52, 51; 8/2 x 256 49, 60, 59; E4M3 39, 40, 54: two tiles of 16 rows
  //   rows 64: 73, 51, 52; 8/2 x 256 84, 60, 61; E4M3 66, 51, 52: two of 32; 8/2 x 256 with E4M3, whose kernel for 32
  //            rows fills a CU alone: four of 16 (50; pieces 60)
  //   rows 96: 103, 78, 54; 8/2 x 256 123, 112, 70; E4M3 88, 75, 53: pieces, unless the call is so small that latency
  //            counts, up to 128 rows in all (one request of 4096 keys 19, 19, 24)
  const int64_t all_rows = tokens * group;
  p.few = rows <= 32 ? 1 : rows > 64 && (all_rows > 128 || max_keys > 16384) ? 0 : head_dim == 256 && codes ? 1 : 2;
  p.rows = p.few ? 16 * p.few : PieceOf<64, kBf16>::kRows;
  p.keys = p.few ? Few<64, kBf16, 1>::kKeys
                 : head_dim == 64 ? PieceOf<64, kBf16>::kKeys : head_dim == 128 ? PieceOf<128, kBf16>::kKeys : PieceOf<256, kBf16>::kKeys;
  // Workgroups per CU.  Few rows: by LDS (Few::kPerCu).  Pieces with 64 features: 245 registers and 64 KiB of LDS, two
  // (2048 tokens on 6144 keys, 16/4 heads: 103 us with ranges for two, 114 for one); with E4M3 265 registers and one
  // (137 us; 150 with ranges for two).
  const int per_cu = p.few == 1   ? (head_dim == 256 && !codes ? Few<256, kBf16, 1>::kPerCu : Few<128, kBf16, 1>::kPerCu)
                     : p.few == 2 ? (head_dim == 256 ? Few<256, kBf16, 2>::kPerCu : Few<128, kBf16, 2>::kPerCu)
                                  : (head_dim == 64 && !codes ? 2 : 1);
  p.slots = kCus * per_cu;
  p.min_tiles = 256 / p.keys;
  // a request's last row tile may be partly empty, its last key range too
  p.rtiles = kv_heads * (tokens * group / p.rows + requests);
  // best_range gives at most kMaxRounds * slots items, or splits nothing; a share alone may add a range per row tile
  p.items = requests <= 64 ? std::max<int64_t>(kMaxRounds * p.slots, p.rtiles) : kMaxRounds * p.slots + p.rtiles;
  p.may_split = max_keys > static_cast<int64_t>(p.min_tiles) * p.keys;
  // best_range splits only where all items fit its rounds: the row tiles of long pieces need no place for parts
  // (131072 tokens, 16/4 heads x 128: 34 MB, 1.09 GB with one for every row tile)
  p.part_items = requests <= 64 ? kMaxRounds * p.slots : p.items;
  p.bytes = p.may_split ? kHeaderBytes + p.part_items * p.rows * (head_dim + 2) * 4 : 0;
  return p;
}

template <class S, typename K>
void launch(K kernel, const PagedArgs& a, const Plan& p, hipStream_t s) {
  const int64_t blocks = (p.items + kNumXcd - 1) / kNumXcd * kNumXcd;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(S::kThreads), 0, s, a);
  if (!p.may_split) return;
  auto join = [&](auto kernel, int rows) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.rtiles), S::kRows / rows), dim3(256), 0, s, a);
  };
  // Two rows per workgroup while a CU gets at most 4 of them, four while it gets 4 (128 features) or 8 (256).  Whole
  // calls with 16, 4 and 2 rows (us): one request of 4 tokens on 4096 keys, 16/4 x 128, 16.9, -, 12.4, 8/2 x 256 25.0, -,
  // 16.4; two of 64 tokens on 8192 keys 34.7, 31.8, -; four on 4096, 8/2 x 256, 40.6, 34.3, -.  More row tiles: 64
  // requests of 4 tokens, 16/4 x 128, 50.7, -, 54.7; four of 100 tokens 38.4, 39.9, -.
  if (p.rtiles * (S::kRows / 2) <= 4 * kCus) return join(paged_gqa_join_kernel<S, 2>, 2);
  if constexpr (S::D > 64) {
    if (p.rtiles * (S::kRows / 4) <= S::D / 32 * kCus) return join(paged_gqa_join_kernel<S, 4>, 4);
  }
  join(paged_gqa_join_kernel<S, 16>, 16);
}

template <int D, Format F>
void launch_as(const PagedArgs& a, const Plan& p, hipStream_t s) {
  if (p.few == 1) launch<Few<D, kBf16, 1>>(paged_gqa_few_kernel<Few<D, F, 1>>, a, p, s);
  else if (p.few == 2) launch<Few<D, kBf16, 2>>(paged_gqa_few_kernel<Few<D, F, 2>>, a, p, s);
  else launch<PieceOf<D, kBf16>>(paged_gqa_piece_kernel<PieceOf<D, F>>, a, p, s);
}

int check_sizes(const char* what, int batch, int q_heads, int kv_heads, int seq_len, int n_seqs, int max_seqlen) {
  FD_REQUIRE(batch >= 0 && seq_len >= 0 && q_heads >= 1 && kv_heads >= 1 && q_heads % kv_heads == 0 && n_seqs >= 0,
             FD_ERR_INVALID_ARGUMENT, "%s: sizes must be >= 0 and q_heads a multiple of kv_heads >= 1", what);
  FD_REQUIRE(n_seqs == 0 || batch == 1, FD_ERR_INVALID_ARGUMENT, "%s: cu_seqlens requires batch == 1", what);
  FD_REQUIRE(q_heads / kv_heads <= 2048, FD_ERR_UNSUPPORTED, "%s: at most 2048 query heads per key head", what);
  FD_REQUIRE(max_seqlen >= 0 && max_seqlen <= seq_len, FD_ERR_INVALID_ARGUMENT,
             "%s: max_seqlen must be in [0, seq_len]", what);
  FD_REQUIRE(static_cast<int64_t>(batch) * seq_len * q_heads < (1LL << 30), FD_ERR_UNSUPPORTED,
             "%s: batch * seq_len * q_heads must be below 2^30", what);
  return FD_OK;
}

}  // namespace

extern "C" int64_t fd_paged_gqa_workspace_bytes(int batch, int q_heads, int kv_heads, int seq_len, int head_dim,
                                                int page_size, int max_pages, int n_seqs, int max_seqlen) {
  static const char* what = "fd_paged_gqa_workspace_bytes";
  if (int rc = check_sizes(what, batch, q_heads, kv_heads, seq_len, n_seqs, max_seqlen)) return rc;
  FD_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, FD_ERR_UNSUPPORTED,
             "%s: head_dim must be 64, 128 or 256 (got %d)", what, head_dim);
  FD_REQUIRE(page_size >= 1 && max_pages >= 1, FD_ERR_INVALID_ARGUMENT, "%s: page_size and max_pages must be >= 1", what);
  auto bytes = [&](Format format) {
    return plan_of(n_seqs > 0 ? n_seqs : batch, static_cast<int64_t>(batch) * seq_len, q_heads / kv_heads, kv_heads,
                   head_dim, static_cast<int64_t>(max_pages) * page_size, max_seqlen, format).bytes;
  };
  return std::max({bytes(kBf16), bytes(kE4m3), bytes(kE2m1)});
}

extern "C" int fd_paged_gqa_fwd(const void* q, const fd_paged_cache* cache, const void* gate, void* out,
                                const int64_t q_strides[4], const int64_t gate_strides[4], const int64_t out_strides[4],
                                int batch, int q_heads, int seq_len, float scale, const int32_t* cu_seqlens, int n_seqs,
                                int max_seqlen, void* workspace, int64_t workspace_bytes, void* stream) {
  static const char* what = "fd_paged_gqa_fwd";
  FD_REQUIRE(q && out && q_strides && out_strides && (!gate || gate_strides), FD_ERR_INVALID_ARGUMENT,
             "%s: tensors and strides must be non-null", what);
  PagedArgs a;
  if (int rc = fill_view(what, cache, true, &a.c)) return rc;
  FD_REQUIRE((cu_seqlens != nullptr) == (n_seqs > 0), FD_ERR_INVALID_ARGUMENT,
             "%s: cu_seqlens and n_seqs >= 1 come together", what);
  if (int rc = check_sizes(what, batch, q_heads, cache->kv_heads, seq_len, n_seqs, max_seqlen)) return rc;
  FD_REQUIRE(scale > 0.0f && scale < 1e30f, FD_ERR_INVALID_ARGUMENT, "%s: scale must be positive", what);
  auto rows_ok = [](const void* p, const int64_t* s) {
    return fd_aligned16(p) && s[3] == 1 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
  };
  FD_REQUIRE(rows_ok(q, q_strides) && rows_ok(out, out_strides) && (!gate || rows_ok(gate, gate_strides)),
             FD_ERR_ALIGNMENT, "%s: rows must be contiguous and 16-byte aligned", what);
  const int requests = n_seqs > 0 ? n_seqs : batch;
  if (requests == 0 || seq_len == 0) return FD_OK;
  const Plan p = plan_of(requests, static_cast<int64_t>(batch) * seq_len, q_heads / cache->kv_heads, cache->kv_heads,
                         cache->head_dim, static_cast<int64_t>(cache->max_pages) * cache->page_size, max_seqlen, format_of(cache));
  FD_REQUIRE(p.items < (1LL << 32) / 512 - kNumXcd, FD_ERR_UNSUPPORTED, "%s: problem too large", what);
  FD_REQUIRE(p.bytes == 0 || (workspace && fd_aligned16(workspace) && workspace_bytes >= p.bytes),
             FD_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned and hold %lld bytes", what,
             static_cast<long long>(p.bytes));
  a.q = static_cast<const uint16_t*>(q);
  a.gate = static_cast<const uint16_t*>(gate);
  a.o = static_cast<uint16_t*>(out);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i];
    a.gs[i] = gate ? gate_strides[i] : 0;
    a.os[i] = out_strides[i];
  }
  a.cu = cu_seqlens;
  a.n_req = requests;
  a.seq_len = seq_len;
  a.group = q_heads / cache->kv_heads;
  a.kv_heads = cache->kv_heads;
  a.group_magic = ((1u << 24) + a.group - 1) / a.group;
  a.slots_log2 = __builtin_ctz(static_cast<unsigned>(p.slots));
  a.min_tiles = p.min_tiles;
  a.overhead = p.few ? 2 : 4;
  a.part_items = static_cast<int>(p.part_items);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.range_tiles = p.may_split ? static_cast<int32_t*>(workspace) : nullptr;
  a.part = p.may_split ? static_cast<float*>(workspace) + kHeaderBytes / 4 : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_kind(cache, [&](auto d, auto f) { launch_as<decltype(d)::value, decltype(f)::value>(a, p, s); });
  return fd_check_launch(what);
}
