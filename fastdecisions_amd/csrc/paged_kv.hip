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
// Measured (4 heads x 128): 64 tokens 3.3 us, the launch; prompts of 24 MB (bf16 in, E4M3 out) 10.2 us,
// 2.3 TB/s, 37 MB read back (E4M3 in, bf16 out) 9.4 to 13 us (in or out of the last-level cache): a few microseconds of
// launch and of the page table's, then the pages' latencies besides the bytes' 4.6 and 7.2.  Long calls
// reach 4.9 TB/s (write) and 4.7 (read) with bf16 pages, 3.9 and 3.4 with E4M3: as long for fewer bytes.
#include <initializer_list>
#include <type_traits>

#include "paged_common.h"

namespace {

constexpr int kThreads = 256;
constexpr float kE4m3Max = 448.0f;
// The scale byte of rows whose largest value lies above 1.75 2^127.  From 248 2^120 on their values round to the code of
// 256, which is 2^128 and no bf16 number: it is read as 255 2^120, the largest one, no further from the value.
constexpr int kTopByte = 247;
// A thread takes several rows, their chains of loads side by side, once there is more than a round (write) or a few
// rounds (read) of workgroups: 1024 of a side (K, V) run at once.  Measured with 1, 2, 4 rows (us, 4 heads x 128 bf16):
// write 1.2, 5 and 48 thousand tokens 4.0, 4.1, 4.1; 9.6, 9.3, 10.0; 39, 40, 41, E4M3 40, 38, 41; read 12 and 96
// thousand 9.3, 9.4, 9.7; 120, 105, 81 (4.8 TB/s), E4M3 121, 108, 83.
constexpr int kAtOnce = 1024;
constexpr int kRows = 2, kManyRows = 4;  // beyond kAtOnce workgroups; of a read beyond four times as many

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

// The requests of U packed rows (the last one that starts at or before each; -1 for a row behind the last request),
// searched side by side: their loads are in flight together.
template <int U>
__device__ __forceinline__ void requests_of(const int32_t* cu, int n_seqs, const int (&t)[U], int (&r)[U]) {
  int hi[U];
#pragma unroll
  for (int u = 0; u < U; ++u) r[u] = 0, hi[u] = n_seqs;
  for (int width = n_seqs; width > 1; width = (width + 1) >> 1) {
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = cu[(r[u] + hi[u]) >> 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int mid = (r[u] + hi[u]) >> 1;
      if (hi[u] - r[u] > 1) (at[u] <= t[u] ? r[u] : hi[u]) = mid;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (!(cu[r[u]] <= t[u] && t[u] < cu[r[u] + 1])) r[u] = -1;
}

// U rows per thread, kThreads / kLanes apart, a stage of all of them at a time: rows, requests, pages, stores.
template <int D, bool FP8, int U>
__global__ __launch_bounds__(kThreads) void paged_kv_write_kernel(WriteArgs a) {
  constexpr int kLanes = D / 8, kSide = kThreads / kLanes;  // lanes of a row; rows of a workgroup side by side
  const int side = blockIdx.y;
  const int li = threadIdx.x % kLanes;
  const uint16_t* const x_side = side == 0 ? a.x[0] : a.x[1];
  const int64_t xb = side == 0 ? a.xs[0][0] : a.xs[1][0], xh = side == 0 ? a.xs[0][1] : a.xs[1][1],
                xt = side == 0 ? a.xs[0][2] : a.xs[1][2];
  const int64_t tokens = static_cast<int64_t>(a.batch) * a.seq_len;
  int head[U], t[U], r[U], pos[U], page[U];
  uint4 w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * U + u) * kSide + threadIdx.x / kLanes;
    const int64_t token = row / a.kv_heads;
    head[u] = static_cast<int>(row - token * a.kv_heads);
    const int b = a.cu == nullptr ? static_cast<int>(token / a.seq_len) : 0;
    t[u] = static_cast<int>(token - static_cast<int64_t>(b) * a.seq_len);
    r[u] = token < tokens ? b : -1;
    w[u] = {0, 0, 0, 0};
    if (token < tokens) w[u] = *reinterpret_cast<const uint4*>(x_side + b * xb + head[u] * xh + t[u] * xt + li * 8);
  }
  if (a.cu != nullptr) {
    int found[U];
    requests_of<U>(a.cu, a.n_seqs, t, found);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r[u] >= 0) r[u] = found[u];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int start, end;
    request_rows(a.cu, max(r[u], 0), a.seq_len, &start, &end);
    const int len = request_keys(a.c, max(r[u], 0));
    pos[u] = len - (end - start) + (t[u] - start);
    if (r[u] < 0 || pos[u] >= len) pos[u] = -1;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    page[u] = pos[u] >= 0 ? a.c.table[r[u] * a.c.table_stride + (pos[u] >> a.c.shift)] : -1;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool live = static_cast<unsigned>(page[u]) < static_cast<unsigned>(a.c.n_pages);
    const int at = pos[u] & ((1 << a.c.shift) - 1);
    unsigned char* dst = (side == 0 ? a.c.k : a.c.v) + page[u] * a.c.page + head[u] * a.c.head + at * a.c.row;
    if constexpr (!FP8) {
      if (live) *reinterpret_cast<uint4*>(dst + li * 16) = w[u];
    } else {
      const uint32_t h[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
      float x[8], top = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = fd_lo(h[i]);
        x[2 * i + 1] = fd_hi(h[i]);
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
        if (li == 0)
          (side == 0 ? a.c.k_scale : a.c.v_scale)[page[u] * a.c.s_page + head[u] * a.c.s_head + at] = static_cast<uint8_t>(byte);
      }
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

template <int D, bool FP8, int U>
__global__ __launch_bounds__(kThreads) void paged_kv_read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8, kSide = kThreads / kLanes;
  const int side = blockIdx.y;
  const int li = threadIdx.x % kLanes;
  int head[U], t[U], r[U], key[U], page[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * U + u) * kSide + threadIdx.x / kLanes;
    const int64_t token = row / a.kv_heads;
    head[u] = static_cast<int>(row - token * a.kv_heads);
    t[u] = token < a.total ? static_cast<int>(token) : -1;
  }
  requests_of<U>(a.cu, a.n_seqs, t, r);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (t[u] < 0) r[u] = -1;
    key[u] = t[u] - max(a.cu[max(r[u], 0)], 0);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int slot = key[u] >> a.c.shift;
    page[u] = r[u] >= 0 && slot < a.c.max_pages ? a.c.table[r[u] * a.c.table_stride + slot] : -1;
  }
  uint4 w[U];
  uint8_t byte[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = key[u] & ((1 << a.c.shift) - 1);
    w[u] = {0, 0, 0, 0};
    byte[u] = 0;
    if (static_cast<unsigned>(page[u]) < static_cast<unsigned>(a.c.n_pages)) {
      const unsigned char* src = (side == 0 ? a.c.k : a.c.v) + page[u] * a.c.page + head[u] * a.c.head + at * a.c.row;
      if constexpr (!FP8) {
        w[u] = *reinterpret_cast<const uint4*>(src + li * 16);
      } else {
        const uint2 code = *reinterpret_cast<const uint2*>(src + li * 8);
        w[u].x = code.x, w[u].y = code.y;
        byte[u] = (side == 0 ? a.c.k_scale : a.c.v_scale)[page[u] * a.c.s_page + head[u] * a.c.s_head + at];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (r[u] < 0) continue;
    if constexpr (FP8) {  // codes of no page are zeros, whatever their scale
      const float s = scale_of(byte[u]);
      typedef float f32x2_t __attribute__((ext_vector_type(2)));
      f32x2_t f0 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[u].x), false);
      f32x2_t f1 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[u].x), true);
      f32x2_t f2 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[u].y), false);
      f32x2_t f3 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[u].y), true);
      if (byte[u] == kTopByte) {
        for (f32x2_t* const f : {&f0, &f1, &f2, &f3})
#pragma unroll
          for (int e = 0; e < 2; ++e) (*f)[e] = fabsf((*f)[e]) == 256.0f ? copysignf(255.0f, (*f)[e]) : (*f)[e];
      }
      w[u].x = fd_pack2(f0[0] * s, f0[1] * s);
      w[u].y = fd_pack2(f1[0] * s, f1[1] * s);
      w[u].z = fd_pack2(f2[0] * s, f2[1] * s);
      w[u].w = fd_pack2(f3[0] * s, f3[1] * s);
    }
    uint16_t* out = side == 0 ? a.out[0] + head[u] * a.os[0][0] + t[u] * a.os[0][1] : a.out[1] + head[u] * a.os[1][0] + t[u] * a.os[1][1];
    *reinterpret_cast<uint4*>(out + li * 8) = w[u];
  }
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
  FD_REQUIRE(blocks < (1LL << 32) / kThreads, FD_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (blocks == 0) return FD_OK;
  const bool fp8 = cache->dtype == FD_DTYPE_E4M3;
  by_head_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    auto go = [&](auto kernel, int rows) {
      const dim3 grid(static_cast<unsigned>((blocks + rows - 1) / rows), 2);
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    };
    if (blocks <= kAtOnce) fp8 ? go(paged_kv_write_kernel<D, true, 1>, 1) : go(paged_kv_write_kernel<D, false, 1>, 1);
    else fp8 ? go(paged_kv_write_kernel<D, true, kRows>, kRows) : go(paged_kv_write_kernel<D, false, kRows>, kRows);
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
  FD_REQUIRE(blocks < (1LL << 32) / kThreads, FD_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (blocks == 0) return FD_OK;
  const bool fp8 = cache->dtype == FD_DTYPE_E4M3;
  by_head_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    auto go = [&](auto kernel, int rows) {
      const dim3 grid(static_cast<unsigned>((blocks + rows - 1) / rows), 2);
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    };
    if (blocks <= kAtOnce) fp8 ? go(paged_kv_read_kernel<D, true, 1>, 1) : go(paged_kv_read_kernel<D, false, 1>, 1);
    else if (blocks <= 4 * kAtOnce) fp8 ? go(paged_kv_read_kernel<D, true, kRows>, kRows) : go(paged_kv_read_kernel<D, false, kRows>, kRows);
    else fp8 ? go(paged_kv_read_kernel<D, true, kManyRows>, kManyRows) : go(paged_kv_read_kernel<D, false, kManyRows>, kManyRows);
  });
  return fd_check_launch(what);
}
