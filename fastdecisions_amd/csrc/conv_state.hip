// The packed causal depthwise conv1d + activation continued from a state, gfx950.
//
// y[t] = act(sum_j w[j] x[t - W + 1 + j] + bias) with x before a request's first
// new token taken from its state, the last W - 1 inputs of its earlier tokens;
// afterwards the state holds the last W - 1 inputs.  Values as in the uncached
// conv (packed_conv.hip): products summed in fp64, one rounding to fp32, bias,
// SiLU, one rounding to bf16; a request fed in pieces gets the bits of the
// request in one piece.
//
// HBM-bound, 2 channels per thread as there (4-byte accesses, 256 bytes per
// wavefront and row).  Two kinds of workgroups in one launch: a head block owns a
// request's first W - 1 new tokens and its state for 512 channels, so that one
// thread alone reads the old state and writes the new one (in place is then
// safe); body blocks take runs of the remaining tokens, which need no state.
// Steps of at most W - 1 tokens have no body.
//
// Measured (6144 channels): 64 requests of one token 3.9 us; 12 suffixes, 85 MB in 21 us, 4.0 TB/s (the
// uncached conv's rate: the fp64 taps take about as long as the bytes).
#include "../../include/fd_cache.h"
#include "state_slot.h"

namespace {

constexpr int kThreads = 256;
constexpr int kNumXcd = 8;
constexpr int kRun = 8;  // rows of a body block

struct ConvStateArgs {
  const uint16_t* x;
  const uint16_t* w;
  const uint16_t* bias;
  uint16_t* q;
  uint16_t* k;
  uint16_t* v;
  const uint16_t* state;
  uint16_t* state_out;
  const int32_t* indices;
  const int32_t* cu;
  int64_t x_row;
  int rows, seq_len, key_dim, value_dim;  // rows: batch * seq_len
  int n_req, n_pool, n_runs, n_col, head_blocks;
};

__device__ __forceinline__ uint32_t load4(const uint16_t* p) { return *reinterpret_cast<const uint32_t*>(p); }

// A thread's 2 channels: taps, bias and where its outputs go.
template <int WIDTH, bool SILU>
struct Channels {
  double w[WIDTH][2];
  float bias[2];
  bool has_bias;
  uint16_t* dst;
  int dst_row;

  __device__ __forceinline__ Channels(const ConvStateArgs& a, int c0) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int j = 0; j < WIDTH; ++j) w[j][e] = fd_bf16_to_f32(a.w[static_cast<int64_t>(c0 + e) * WIDTH + j]);
    }
    has_bias = a.bias != nullptr;
    const uint32_t b = has_bias ? load4(a.bias + c0) : 0u;
    bias[0] = fd_lo(b);
    bias[1] = fd_hi(b);
    if (c0 < a.key_dim) {
      dst = a.q + c0;
      dst_row = a.key_dim;
    } else if (c0 < 2 * a.key_dim) {
      dst = a.k + (c0 - a.key_dim);
      dst_row = a.key_dim;
    } else {
      dst = a.v + (c0 - 2 * a.key_dim);
      dst_row = a.value_dim;
    }
  }

  // Row r from the window win[0 .. WIDTH - 1], oldest first.
  __device__ __forceinline__ void store(const uint32_t (&win)[WIDTH], int64_t r) const {
    float y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      double acc = 0.0;
#pragma unroll
      for (int j = 0; j < WIDTH; ++j)
        acc = __builtin_fma(w[j][e], static_cast<double>(e == 0 ? fd_lo(win[j]) : fd_hi(win[j])), acc);
      float t = static_cast<float>(acc);
      if (has_bias) t = t + bias[e];
      y[e] = SILU ? fd_silu_bf16(t) : t;
    }
    *reinterpret_cast<uint32_t*>(dst + r * dst_row) = fd_pack2(y[0], y[1]);
  }
};

// New tokens [start, end) of request r on the flattened rows, inside [0, rows].
__device__ __forceinline__ void bounds(const ConvStateArgs& a, int r, int* start, int* end) {
  if (a.cu == nullptr) {
    *start = r * a.seq_len;
    *end = *start + a.seq_len;
  } else {
    *start = min(max(a.cu[r], 0), a.rows);
    *end = min(max(a.cu[r + 1], *start), a.rows);
  }
}

template <int WIDTH, bool SILU>
__device__ __forceinline__ void head_block(const ConvStateArgs& a, int b) {
  constexpr int H = WIDTH - 1;
  const int r = b / a.n_col;
  const int c0 = ((b - r * a.n_col) * kThreads + static_cast<int>(threadIdx.x)) * 2;
  const int C = 2 * a.key_dim + a.value_dim;
  const int slot = owned_slot(a.indices, r, a.n_pool, threadIdx.x & 63);
  if (c0 >= C) return;
  int start, end;
  bounds(a, r, &start, &end);
  const int n = end - start;
  const Channels<WIDTH, SILU> ch(a, c0);
  // the state, then the first new rows; the last H rows of a long request
  uint32_t in[2 * H], last[H];
  const int64_t at = static_cast<int64_t>(max(slot, 0)) * H * C + c0;
#pragma unroll
  for (int j = 0; j < H; ++j) in[j] = slot >= 0 ? load4(a.state + at + static_cast<int64_t>(j) * C) : 0u;
#pragma unroll
  for (int i = 0; i < H; ++i) in[H + i] = i < n ? load4(a.x + (start + i) * a.x_row + c0) : 0u;
#pragma unroll
  for (int j = 0; j < H; ++j) {
    last[j] = in[j];
    if (n >= H) {
      last[j] = load4(a.x + static_cast<int64_t>(end - H + j) * a.x_row + c0);
    } else {
#pragma unroll
      for (int i = 1; i < H; ++i)
        if (n == i) last[j] = in[i + j];  // shifted by the n new rows
    }
  }
#pragma unroll
  for (int i = 0; i < H; ++i) {
    if (i < n) {
      uint32_t win[WIDTH];
#pragma unroll
      for (int j = 0; j < WIDTH; ++j) win[j] = in[i + j];
      ch.store(win, start + i);
    }
  }
  if (slot >= 0) {
#pragma unroll
    for (int j = 0; j < H; ++j) *reinterpret_cast<uint32_t*>(a.state_out + at + static_cast<int64_t>(j) * C) = last[j];
  }
}

template <int WIDTH, bool SILU>
__device__ __forceinline__ void body_block(const ConvStateArgs& a, int b, int n_blocks) {
  constexpr int H = WIDTH - 1;
  // XCD x takes one contiguous range of the runs: a run's halo rows are in the L2 of the run before
  const int logical = (b % kNumXcd) * (n_blocks / kNumXcd) + b / kNumXcd;
  const int run = logical / a.n_col;
  const int c0 = ((logical - run * a.n_col) * kThreads + static_cast<int>(threadIdx.x)) * 2;
  const int C = 2 * a.key_dim + a.value_dim;
  if (run >= a.n_runs || c0 >= C) return;
  const int r0 = run * kRun, r1 = min(r0 + kRun, a.rows);
  int req, start, end;
  if (a.cu == nullptr) {
    req = r0 / a.seq_len;
  } else {
    int lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= r0) lo = mid;
      else hi = mid;
    }
    req = lo;
  }
  bounds(a, req, &start, &end);
  const Channels<WIDTH, SILU> ch(a, c0);
  const uint16_t* const x = a.x + c0;
  if (r0 - start >= H && r0 + kRun <= end) {  // all of the run lies behind the head of one request
    uint32_t in[H + kRun];
#pragma unroll
    for (int m = 0; m < H + kRun; ++m) in[m] = load4(x + static_cast<int64_t>(r0 - H + m) * a.x_row);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      uint32_t win[WIDTH];
#pragma unroll
      for (int j = 0; j < WIDTH; ++j) win[j] = in[i + j];
      ch.store(win, r0 + i);
    }
    return;
  }
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    while (r >= end && req + 1 < a.n_req) bounds(a, ++req, &start, &end);
    if (r < start + H || r >= end) continue;  // a head block's row, or behind the last request
    uint32_t win[WIDTH];
#pragma unroll
    for (int j = 0; j < WIDTH; ++j) win[j] = load4(x + static_cast<int64_t>(r - H + j) * a.x_row);
    ch.store(win, r);
  }
}

template <int WIDTH, bool SILU>
__global__ __launch_bounds__(kThreads) void conv_state_kernel(ConvStateArgs a) {
  const int b = blockIdx.x;
  if (b < a.head_blocks) {
    if (b < a.n_req * a.n_col) head_block<WIDTH, SILU>(a, b);
  } else {
    body_block<WIDTH, SILU>(a, b - a.head_blocks, gridDim.x - a.head_blocks);
  }
}

template <int WIDTH>
void launch(const ConvStateArgs& a, bool silu, int64_t blocks, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(blocks));
  if (silu) hipLaunchKernelGGL((conv_state_kernel<WIDTH, true>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((conv_state_kernel<WIDTH, false>), grid, dim3(kThreads), 0, s, a);
}

}  // namespace

extern "C" int fd_packed_conv_state(const void* x, int64_t x_row_stride, const void* weight, const void* bias,
                                    const void* state, void* state_out, int n_pool, const int32_t* state_indices,
                                    void* q, void* k, void* v, int batch, int seq_len, int key_dim, int value_dim,
                                    int width, const int32_t* cu_seqlens, int n_seqs, int activation, void* stream) {
  static const char* what = "fd_packed_conv_state";
  FD_REQUIRE(x && weight && state && state_out && q && k && v, FD_ERR_INVALID_ARGUMENT,
             "%s: tensor pointers must be non-null", what);
  FD_REQUIRE(batch >= 0 && seq_len >= 0 && key_dim >= 8 && value_dim >= 8 && key_dim % 8 == 0 && value_dim % 8 == 0,
             FD_ERR_INVALID_ARGUMENT, "%s: key_dim and value_dim must be positive multiples of 8", what);
  FD_REQUIRE(width >= 2 && width <= 4, FD_ERR_UNSUPPORTED, "%s: width must be in [2, 4] (got %d)", what, width);
  FD_REQUIRE(activation == FD_ACT_NONE || activation == FD_ACT_SILU, FD_ERR_INVALID_ARGUMENT,
             "%s: unknown activation %d", what, activation);
  FD_REQUIRE((cu_seqlens != nullptr) == (n_seqs > 0) && (n_seqs == 0 || batch == 1), FD_ERR_INVALID_ARGUMENT,
             "%s: cu_seqlens and n_seqs >= 1 come together, with batch == 1", what);
  const int64_t c = 2LL * key_dim + value_dim;
  FD_REQUIRE(c < (1 << 24), FD_ERR_UNSUPPORTED, "%s: too many channels", what);
  FD_REQUIRE(x_row_stride >= c && x_row_stride % 8 == 0, FD_ERR_ALIGNMENT,
             "%s: x_row_stride must be a multiple of 8, at least the channels", what);
  FD_REQUIRE(fd_aligned16(x) && fd_aligned16(weight) && fd_aligned16(bias) && fd_aligned16(state) &&
                 fd_aligned16(state_out) && fd_aligned16(q) && fd_aligned16(k) && fd_aligned16(v),
             FD_ERR_ALIGNMENT, "%s: pointers must be 16-byte aligned", what);
  const int requests = n_seqs > 0 ? n_seqs : batch;
  FD_REQUIRE(n_pool >= (state_indices ? 1 : requests), FD_ERR_INVALID_ARGUMENT,
             "%s: the state needs a row for every request", what);
  const int64_t rows = static_cast<int64_t>(batch) * seq_len;
  FD_REQUIRE(rows < (1LL << 31) - kRun, FD_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (requests == 0) return FD_OK;
  ConvStateArgs a;
  a.x = static_cast<const uint16_t*>(x);
  a.w = static_cast<const uint16_t*>(weight);
  a.bias = static_cast<const uint16_t*>(bias);
  a.q = static_cast<uint16_t*>(q);
  a.k = static_cast<uint16_t*>(k);
  a.v = static_cast<uint16_t*>(v);
  a.state = static_cast<const uint16_t*>(state);
  a.state_out = static_cast<uint16_t*>(state_out);
  a.indices = state_indices;
  a.cu = cu_seqlens;
  a.x_row = x_row_stride;
  a.rows = static_cast<int>(rows);
  a.seq_len = seq_len;
  a.key_dim = key_dim;
  a.value_dim = value_dim;
  a.n_req = requests;
  a.n_pool = n_pool;
  a.n_col = static_cast<int>((c / 2 + kThreads - 1) / kThreads);
  const bool body = seq_len > width - 1;  // of a packed batch: some request may be longer than a head
  a.n_runs = body ? static_cast<int>((rows + kRun - 1) / kRun) : 0;
  const int64_t heads = (static_cast<int64_t>(requests) * a.n_col + kNumXcd - 1) / kNumXcd * kNumXcd;
  const int64_t bodies = (static_cast<int64_t>(a.n_runs) * a.n_col + kNumXcd - 1) / kNumXcd * kNumXcd;
  FD_REQUIRE(heads + bodies < (1LL << 32) / kThreads, FD_ERR_UNSUPPORTED, "%s: grid too large", what);
  a.head_blocks = static_cast<int>(heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (width == 2) launch<2>(a, activation == FD_ACT_SILU, heads + bodies, s);
  else if (width == 3) launch<3>(a, activation == FD_ACT_SILU, heads + bodies, s);
  else launch<4>(a, activation == FD_ACT_SILU, heads + bodies, s);
  return fd_check_launch(what);
}
