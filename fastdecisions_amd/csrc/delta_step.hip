// The gated delta rule token by token, from and into its state, gfx950.
//
// Per value head, with S [128, 128] in fp32 and q, k l2-normalised in fp32:
//   S <- e^g S;  d = beta (v - S^T k);  S <- S + k d^T;  o = S^T (scale q)
// A column of S depends on no other column, so a wavefront owns 32 columns of one
// (request, head) and needs no other one: no LDS, no barrier.  Lane l holds rows
// 16 (l / 8) .. + 15 of columns 4 (l % 8) .. + 3 in 64 registers (loads and stores
// of whole 128-byte lines), and both products come from one pass over them,
//   a = S^T k, b = S^T q, c = k . q  =>  d = beta (v - e^g a),  o = scale (e^g b + c d),
// reduced together over the 8 lane groups, so a token costs one chain of
// cross-lane adds.
//
// Bound: the state, read once and written once however many tokens the call has
// (64 KiB each way per request and head); for few requests the latency of its
// loads.  The chunked rule moves it too and adds work that only pays from tens
// of tokens on.
//
// Measured (16 heads): one token of one request 4.4 us, of 64 requests 22.7 us, 5.9 TB/s of state (134 MB,
// in part from the last-level cache; a large copy here: 5.1).  A further token of a request costs 1.25 us:
// its chain of products and cross-lane adds.
#include "../../include/fd_cache.h"
#include "state_slot.h"

namespace {

constexpr int kD = 128;
constexpr int kCols = 32;   // columns of a wavefront
constexpr int kRowsLane = 16;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct StepArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const float* g;
  const void* beta;
  uint16_t* out;
  const float* state;   // or null: zeros
  float* state_out;     // or null
  const int32_t* indices;
  const int32_t* cu;
  int rows, seq_len, k_heads, v_heads, n_req, n_pool;
  float scale;
  int beta_f32, l2norm;
};

// 16 consecutive bf16 as fp32.
__device__ __forceinline__ void widen(const uint4 (&w)[2], float (&x)[kRowsLane]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[8 * i + 2 * j] = fd_lo(u[j]);
      x[8 * i + 2 * j + 1] = fd_hi(u[j]);
    }
  }
}

// Sum over the 8 lane groups (lanes of equal l % 8).
__device__ __forceinline__ float over_rows(float s) {
  s = fd_xor_sum<8>(s);
  s = fd_xor_sum<16>(s);
  return fd_xor_sum<32>(s);
}

struct Token {
  uint4 q[2], k[2];
  uint2 v;
  float g, beta;
};

__global__ __launch_bounds__(64) void delta_step_kernel(StepArgs a) {
  const int lane = threadIdx.x;
  const int rg = lane >> 3, cg = lane & 7;
  const int part = blockIdx.x % (kD / kCols);
  const int head = (blockIdx.x / (kD / kCols)) % a.v_heads;
  const int r = blockIdx.x / (kD / kCols) / a.v_heads;
  int start, end;
  if (a.cu == nullptr) {
    start = r * a.seq_len;
    end = start + a.seq_len;
  } else {
    start = min(max(a.cu[r], 0), a.rows);
    end = min(max(a.cu[r + 1], start), a.rows);
  }
  const int khead = head / (a.v_heads / a.k_heads);
  const int col = part * kCols + cg * 4;
  const int slot = owned_slot(a.indices, r, a.n_pool, lane);
  const int64_t at = ((static_cast<int64_t>(max(slot, 0)) * a.v_heads + head) * kD + rg * kRowsLane) * kD + col;
  f32x4_t s[kRowsLane];
  if (a.state != nullptr && slot >= 0) {
#pragma unroll
    for (int i = 0; i < kRowsLane; ++i) s[i] = *reinterpret_cast<const f32x4_t*>(a.state + at + i * kD);
  } else {
#pragma unroll
    for (int i = 0; i < kRowsLane; ++i) s[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  auto fetch = [&](int t, Token& x) {
    const int64_t kr = (static_cast<int64_t>(t) * a.k_heads + khead) * kD + rg * kRowsLane;
    const int64_t vr = static_cast<int64_t>(t) * a.v_heads + head;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x.q[i] = *reinterpret_cast<const uint4*>(a.q + kr + 8 * i);
      x.k[i] = *reinterpret_cast<const uint4*>(a.k + kr + 8 * i);
    }
    x.v = *reinterpret_cast<const uint2*>(a.v + vr * kD + col);
    x.g = a.g[vr];
    x.beta = a.beta_f32 ? static_cast<const float*>(a.beta)[vr]
                        : fd_bf16_to_f32(static_cast<const uint16_t*>(a.beta)[vr]);
  };
  Token next;
  if (start < end) fetch(start, next);
  for (int t = start; t < end; ++t) {
    const Token x = next;
    if (t + 1 < end) fetch(t + 1, next);
    float q[kRowsLane], k[kRowsLane];
    widen(x.q, q);
    widen(x.k, k);
    float c = 0.0f, qq = 0.0f, kk = 0.0f;
#pragma unroll
    for (int i = 0; i < kRowsLane; ++i) {
      c = __builtin_fmaf(q[i], k[i], c);
      qq = __builtin_fmaf(q[i], q[i], qq);
      kk = __builtin_fmaf(k[i], k[i], kk);
    }
    f32x4_t sk = {0.0f, 0.0f, 0.0f, 0.0f}, sq = sk;
#pragma unroll
    for (int i = 0; i < kRowsLane; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sk[e] = __builtin_fmaf(s[i][e], k[i], sk[e]);
        sq[e] = __builtin_fmaf(s[i][e], q[i], sq[e]);
      }
    }
    c = over_rows(c);
    qq = over_rows(qq);
    kk = over_rows(kk);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sk[e] = over_rows(sk[e]);
      sq[e] = over_rows(sq[e]);
    }
    // the products are linear in q and k: their norms scale the sums
    const float kn = a.l2norm ? 1.0f / __builtin_sqrtf(kk + 1e-6f) : 1.0f;
    const float qn = (a.l2norm ? 1.0f / __builtin_sqrtf(qq + 1e-6f) : 1.0f) * a.scale;
    const float decay = expf(x.g);
    const float v[4] = {fd_lo(x.v.x), fd_hi(x.v.x), fd_lo(x.v.y), fd_hi(x.v.y)};
    f32x4_t d, o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      d[e] = x.beta * (v[e] - decay * (sk[e] * kn));
      o[e] = __builtin_fmaf(c * kn, d[e], decay * sq[e]) * qn;
      d[e] *= kn;
    }
#pragma unroll
    for (int i = 0; i < kRowsLane; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = __builtin_fmaf(k[i], d[e], s[i][e] * decay);
    }
    if (rg == 0)
      *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(t) * a.v_heads + head) * kD + col) =
          uint2{fd_pack2(o[0], o[1]), fd_pack2(o[2], o[3])};
  }
  if (a.state_out != nullptr && slot >= 0) {
#pragma unroll
    for (int i = 0; i < kRowsLane; ++i) *reinterpret_cast<f32x4_t*>(a.state_out + at + i * kD) = s[i];
  }
}

}  // namespace

extern "C" int fd_gated_delta_step(const void* q, const void* k, const void* v, const float* g, const void* beta,
                                   void* out, const float* state, float* state_out, int n_pool,
                                   const int32_t* state_indices, int batch, int seq_len, int k_heads, int v_heads,
                                   int head_k_dim, int head_v_dim, float scale, int beta_dtype, int l2norm_qk,
                                   const int32_t* cu_seqlens, int n_seqs, void* stream) {
  static const char* what = "fd_gated_delta_step";
  FD_REQUIRE(q && k && v && g && beta && out, FD_ERR_INVALID_ARGUMENT, "%s: tensor pointers must be non-null", what);
  FD_REQUIRE(batch >= 0 && seq_len >= 0 && k_heads >= 1 && v_heads >= 1 && v_heads % k_heads == 0,
             FD_ERR_INVALID_ARGUMENT, "%s: sizes must be >= 0 and v_heads a multiple of k_heads >= 1", what);
  FD_REQUIRE(head_k_dim == kD && head_v_dim == kD, FD_ERR_UNSUPPORTED, "%s: head dims must be 128 (got %d, %d)", what,
             head_k_dim, head_v_dim);
  FD_REQUIRE(beta_dtype == FD_DTYPE_BF16 || beta_dtype == FD_DTYPE_F32, FD_ERR_INVALID_ARGUMENT,
             "%s: beta must be bf16 or fp32", what);
  FD_REQUIRE((cu_seqlens != nullptr) == (n_seqs > 0) && (n_seqs == 0 || batch == 1), FD_ERR_INVALID_ARGUMENT,
             "%s: cu_seqlens and n_seqs >= 1 come together, with batch == 1", what);
  FD_REQUIRE(fd_aligned16(q) && fd_aligned16(k) && fd_aligned16(v) && fd_aligned16(out) && fd_aligned16(state) &&
                 fd_aligned16(state_out),
             FD_ERR_ALIGNMENT, "%s: pointers must be 16-byte aligned", what);
  const int requests = n_seqs > 0 ? n_seqs : batch;
  FD_REQUIRE((!state && !state_out) || n_pool >= (state_indices ? 1 : requests), FD_ERR_INVALID_ARGUMENT,
             "%s: the state needs a row for every request", what);
  const int64_t rows = static_cast<int64_t>(batch) * seq_len;
  const int64_t blocks = static_cast<int64_t>(requests) * v_heads * (kD / kCols);
  FD_REQUIRE(rows < (1LL << 31) && blocks < (1LL << 32) / 64, FD_ERR_UNSUPPORTED, "%s: problem too large", what);
  if (blocks == 0) return FD_OK;
  const StepArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), g,
                   beta, static_cast<uint16_t*>(out), state, state_out, state_indices, cu_seqlens,
                   static_cast<int>(rows), seq_len, k_heads, v_heads, requests, n_pool, scale,
                   beta_dtype == FD_DTYPE_F32, l2norm_qk != 0};
  hipLaunchKernelGGL(delta_step_kernel, dim3(static_cast<unsigned>(blocks)), dim3(64), 0,
                     static_cast<hipStream_t>(stream), a);
  return fd_check_launch(what);
}
