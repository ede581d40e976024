// Writing and reading a paged key/value cache, gfx950.
//
// Streaming kernels, bound by HBM (and by the launch for a few tokens).  head_dim
// / 8 lanes own one (token, head) row of K or V, 16 bytes of bf16 each, so a
// wavefront moves 1 KiB in one instruction; blockIdx.y picks K or V.
//
// Quantising (E4M3): a row's scale is the smallest power of two 2^E with
// max|x| <= 448 2^E.  With A = max|x| = m 2^k, m in [1, 2), and 448 = 1.75 2^8 that
// is E = k - 8 for m <= 1.75, else k - 7: read off the exponent and mantissa bits,
// no logarithm and no division.  x 2^-E is exact in fp32 (or below a code's
// smallest step), so the one rounding is the conversion's; floating codes lose
// nothing to a scale that is not the tightest, except a binade of subnormals.
//
// Measured (4 heads x 128): 64 tokens 3.5 us, the launch; prompts of 24 MB (bf16 in, E4M3 out)
// 10.4 us, 2.3 TB/s, and 37 MB read back (E4M3 in, bf16 out) 13.1 us, 2.8 TB/s: a few microseconds of
// launch and of the page table's, then the pages' latencies besides the bytes' 4.6 and 7.2.
#include <initializer_list>
#include <type_traits>

#include "paged_common.h"

namespace {

constexpr int kThreads = 256;
constexpr float kE4m3Max = 448.0f;

struct WriteArgs {
  const uint16_t* x[2];       // k, v
  int64_t xs[2][3];           // b, h, t (elements)
  PagedView c;
  const int32_t* cu;
  int n_seqs, batch, seq_len, kv_heads;
};

template <int N>
__device__ __forceinline__ float group_max(float v) {
  v = fd_xor_max<1>(v);
  v = fd_xor_max<2>(v);
  v = fd_xor_max<4>(v);
  if constexpr (N >= 16) v = fd_xor_max<8>(v);
  if constexpr (N >= 32) v = fd_xor_max<16>(v);
  return v;
}

// Exponent byte E + 127 of the smallest 2^E with a <= 448 * 2^E (127 for a == 0).
__device__ __forceinline__ int scale_byte(float a) {
  const uint32_t u = __float_as_uint(a);
  if (u == 0) return 127;
  const int e = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, 1);
}

// x / 2^E for a code: infinities become the largest code, NaN stays.
__device__ __forceinline__ float to_code_range(float x, float inv) {
  const float y = x * inv;
  return y != y ? y : fminf(fmaxf(y, -kE4m3Max), kE4m3Max);
}

template <int D, bool FP8>
__global__ __launch_bounds__(kThreads) void paged_kv_write_kernel(WriteArgs a) {
  constexpr int kLanes = D / 8;  // lanes of a row
  const int side = blockIdx.y;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  const int li = threadIdx.x % kLanes;
  const int64_t token = row / a.kv_heads;
  const int head = static_cast<int>(row - token * a.kv_heads);
  const int64_t tokens = static_cast<int64_t>(a.batch) * a.seq_len;
  bool live = token < tokens;
  int b = 0, t = 0, r = 0, start = 0, end = 0;
  if (live) {
    if (a.cu == nullptr) {
      r = b = static_cast<int>(token / a.seq_len);
      t = static_cast<int>(token - static_cast<int64_t>(b) * a.seq_len);
    } else {
      t = static_cast<int>(token);
      r = request_of(a.cu, a.n_seqs, t);
      live = r >= 0;
    }
  }
  uint4 w = {0, 0, 0, 0};
  int pos = 0, page = -1;
  if (live) {
    const uint16_t* x = side == 0 ? a.x[0] : a.x[1];
    const int64_t xb = side == 0 ? a.xs[0][0] : a.xs[1][0], xh = side == 0 ? a.xs[0][1] : a.xs[1][1],
                  xt = side == 0 ? a.xs[0][2] : a.xs[1][2];
    w = *reinterpret_cast<const uint4*>(x + b * xb + head * xh + t * xt + li * 8);
    request_rows(a.cu, r, a.seq_len, &start, &end);
    const int len = request_keys(a.c, r);
    pos = len - (end - start) + (t - start);
    if (pos >= 0 && pos < len) page = a.c.table[r * a.c.table_stride + (pos >> a.c.shift)];
  }
  live = static_cast<unsigned>(page) < static_cast<unsigned>(a.c.n_pages);
  const int at = pos & ((1 << a.c.shift) - 1);
  unsigned char* dst = (side == 0 ? a.c.k : a.c.v) + page * a.c.page + head * a.c.head + at * a.c.row;
  if constexpr (!FP8) {
    if (live) *reinterpret_cast<uint4*>(dst + li * 16) = w;
  } else {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float x[8], top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = fd_lo(u[i]);
      x[2 * i + 1] = fd_hi(u[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float m = fabsf(x[i]);
      top = fmaxf(top, m < __builtin_inff() ? m : 0.0f);  // finite values only
    }
    top = group_max<kLanes>(top);  // every lane of the wavefront takes part
    const int byte = scale_byte(top);
    const float inv = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);  // 2^-E
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_code_range(x[i], inv);
    uint2 code;
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    code.x = static_cast<uint32_t>(lo);
    code.y = static_cast<uint32_t>(hi);
    if (live) {
      *reinterpret_cast<uint2*>(dst + li * 8) = code;
      if (li == 0) (side == 0 ? a.c.k_scale : a.c.v_scale)[page * a.c.s_page + head * a.c.s_head + at] = static_cast<uint8_t>(byte);
    }
  }
}

struct ReadArgs {
  uint16_t* out[2];
  int64_t os[2][2];           // h, t (elements)
  PagedView c;
  const int32_t* cu;
  int n_seqs, kv_heads;
  int total;
};

template <int D, bool FP8>
__global__ __launch_bounds__(kThreads) void paged_kv_read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8;
  const int side = blockIdx.y;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  const int li = threadIdx.x % kLanes;
  const int64_t t = row / a.kv_heads;
  const int head = static_cast<int>(row - t * a.kv_heads);
  if (t >= a.total) return;
  const int r = request_of(a.cu, a.n_seqs, static_cast<int>(t));
  if (r < 0) return;
  const int key = static_cast<int>(t) - max(a.cu[r], 0);
  const int slot = key >> a.c.shift, at = key & ((1 << a.c.shift) - 1);
  const int page = slot < a.c.max_pages ? a.c.table[r * a.c.table_stride + slot] : -1;
  uint4 w = {0, 0, 0, 0};
  if (static_cast<unsigned>(page) < static_cast<unsigned>(a.c.n_pages)) {
    const unsigned char* src = (side == 0 ? a.c.k : a.c.v) + page * a.c.page + head * a.c.head + at * a.c.row;
    if constexpr (!FP8) {
      w = *reinterpret_cast<const uint4*>(src + li * 16);
    } else {
      const uint2 code = *reinterpret_cast<const uint2*>(src + li * 8);
      const float s = scale_of((side == 0 ? a.c.k_scale : a.c.v_scale)[page * a.c.s_page + head * a.c.s_head + at]);
      typedef float f32x2_t __attribute__((ext_vector_type(2)));
      const f32x2_t f0 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code.x), false);
      const f32x2_t f1 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code.x), true);
      const f32x2_t f2 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code.y), false);
      const f32x2_t f3 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code.y), true);
      w.x = fd_pack2(f0[0] * s, f0[1] * s);
      w.y = fd_pack2(f1[0] * s, f1[1] * s);
      w.z = fd_pack2(f2[0] * s, f2[1] * s);
      w.w = fd_pack2(f3[0] * s, f3[1] * s);
    }
  }
  uint16_t* out = side == 0 ? a.out[0] + head * a.os[0][0] + t * a.os[0][1] : a.out[1] + head * a.os[1][0] + t * a.os[1][1];
  *reinterpret_cast<uint4*>(out + li * 8) = w;
}

template <typename F>
void by_head_dim(int head_dim, F&& launch) {
  if (head_dim == 64) launch(std::integral_constant<int, 64>{});
  else if (head_dim == 128) launch(std::integral_constant<int, 128>{});
  else launch(std::integral_constant<int, 256>{});
}

}  // namespace

extern "C" int fd_paged_kv_write(const void* k, const void* v, const int64_t k_strides[4], const int64_t v_strides[4],
                                 const fd_paged_cache* cache, int batch, int seq_len, const int32_t* cu_seqlens,
                                 int n_seqs, void* stream) {
  static const char* what = "fd_paged_kv_write";
  FD_REQUIRE(k && v && k_strides && v_strides, FD_ERR_INVALID_ARGUMENT, "%s: k, v and their strides must be non-null", what);
  WriteArgs a;
  if (int rc = fill_view(what, cache, true, &a.c)) return rc;
  FD_REQUIRE(batch >= 0 && seq_len >= 0, FD_ERR_INVALID_ARGUMENT, "%s: batch and seq_len must be >= 0", what);
  FD_REQUIRE(cu_seqlens == nullptr || (batch == 1 && n_seqs >= 1), FD_ERR_INVALID_ARGUMENT,
             "%s: cu_seqlens requires batch == 1 and n_seqs >= 1", what);
  for (const int64_t* s : {k_strides, v_strides})
    FD_REQUIRE(s[3] == 1 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0, FD_ERR_ALIGNMENT,
               "%s: k and v rows must be contiguous and 16-byte aligned", what);
  FD_REQUIRE(fd_aligned16(k) && fd_aligned16(v), FD_ERR_ALIGNMENT, "%s: k and v must be 16-byte aligned", what);
  a.x[0] = static_cast<const uint16_t*>(k);
  a.x[1] = static_cast<const uint16_t*>(v);
  for (int i = 0; i < 3; ++i) {
    a.xs[0][i] = k_strides[i];
    a.xs[1][i] = v_strides[i];
  }
  a.cu = cu_seqlens;
  a.n_seqs = n_seqs;
  a.batch = batch;
  a.seq_len = seq_len;
  a.kv_heads = cache->kv_heads;
  const int64_t rows = static_cast<int64_t>(batch) * seq_len * cache->kv_heads;
  const int per = kThreads / (cache->head_dim / 8);
  const int64_t blocks = (rows + per - 1) / per;
  FD_REQUIRE(blocks < (1LL << 31), FD_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (blocks == 0) return FD_OK;
  const bool fp8 = cache->dtype == FD_DTYPE_E4M3;
  by_head_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    if (fp8)
      hipLaunchKernelGGL((paged_kv_write_kernel<D, true>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    else
      hipLaunchKernelGGL((paged_kv_write_kernel<D, false>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
  });
  return fd_check_launch(what);
}

extern "C" int fd_paged_kv_read(const fd_paged_cache* cache, void* k_out, void* v_out, const int64_t k_strides[2],
                                const int64_t v_strides[2], int64_t total, const int32_t* cu_seqlens, int n_seqs,
                                void* stream) {
  static const char* what = "fd_paged_kv_read";
  FD_REQUIRE(k_out && v_out && k_strides && v_strides && cu_seqlens, FD_ERR_INVALID_ARGUMENT,
             "%s: outputs, strides and cu_seqlens must be non-null", what);
  ReadArgs a;
  if (int rc = fill_view(what, cache, false, &a.c)) return rc;
  FD_REQUIRE(total >= 0 && total < (1LL << 31) && n_seqs >= 1, FD_ERR_INVALID_ARGUMENT,
             "%s: total must be in [0, 2^31) and n_seqs >= 1", what);
  for (const int64_t* s : {k_strides, v_strides})
    FD_REQUIRE(s[0] % 8 == 0 && s[1] % 8 == 0, FD_ERR_ALIGNMENT, "%s: output rows must be 16-byte aligned", what);
  FD_REQUIRE(fd_aligned16(k_out) && fd_aligned16(v_out), FD_ERR_ALIGNMENT, "%s: outputs must be 16-byte aligned", what);
  a.out[0] = static_cast<uint16_t*>(k_out);
  a.out[1] = static_cast<uint16_t*>(v_out);
  for (int i = 0; i < 2; ++i) {
    a.os[0][i] = k_strides[i];
    a.os[1][i] = v_strides[i];
  }
  a.cu = cu_seqlens;
  a.n_seqs = n_seqs;
  a.kv_heads = cache->kv_heads;
  a.total = static_cast<int>(total);
  const int per = kThreads / (cache->head_dim / 8);
  const int64_t blocks = (total * cache->kv_heads + per - 1) / per;
  FD_REQUIRE(blocks < (1LL << 31), FD_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (blocks == 0) return FD_OK;
  const bool fp8 = cache->dtype == FD_DTYPE_E4M3;
  by_head_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    if (fp8)
      hipLaunchKernelGGL((paged_kv_read_kernel<D, true>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    else
      hipLaunchKernelGGL((paged_kv_read_kernel<D, false>), grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
  });
  return fd_check_launch(what);
}
