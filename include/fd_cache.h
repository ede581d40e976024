/*
 * fd_cache.h — C ABI of libfd_cache.so: the gfx950 kernels that continue a
 * request from its caches (paged keys/values, conv state, delta-rule state).
 *
 *   fd_paged_kv_write     keys and values of new tokens into a paged cache (bf16, or e4m3 quantised on the way)
 *   fd_paged_kv_read      the pages back as dense bf16 keys and values
 *   fd_paged_gqa_fwd      causal grouped-query attention of the new tokens over the paged cache
 *   fd_paged_key_weights  the attention weight that every cached key draws from the new tokens
 *   fd_paged_kv_evict     the keys of largest weight and the most recent ones, moved to pages of their own
 *   fd_gated_delta_step   the gated delta rule token by token, from and into its fp32 state
 *   fd_packed_conv_state  the packed causal conv + activation continued from its state
 *
 * They serve what the reference's prefix cache serves (ref: src/decider/shared_prefix.py:
 * keys/values, conv state and recurrent state of a prefix, continued by suffixes).
 *
 * Conventions as in fd_kernels.h: device pointers, bf16 as raw 16-bit storage, work
 * enqueued on `stream`, no allocation, no synchronisation, FD_OK or a negative FD_ERR_*
 * code, with the message in fd_cache_last_error() (of the calling thread).
 */
#ifndef FD_CACHE_H
#define FD_CACHE_H

#include "fd_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FD_CACHE_ABI_VERSION 1

/* Cache element types besides FD_DTYPE_BF16: OCP 8-bit floats with 4 exponent and 3 mantissa bits. */
#define FD_DTYPE_E4M3 2
/* OCP 4-bit floats with 2 exponent bits and 1 mantissa bit, two a byte (the even feature in the low bits). */
#define FD_DTYPE_E2M1 3

FD_API int fd_cache_abi_version(void);

/* Message describing the last failed call of this library on this thread ("" if none). */
FD_API const char* fd_cache_last_error(void);

/*
 * A paged key/value cache and the requests' view of it.
 *
 *   k, v      [n_pages, kv_heads, page_size, head_dim] of dtype (FD_DTYPE_BF16, FD_DTYPE_E4M3 or
 *             FD_DTYPE_E2M1); strides {page, head, row} in elements (E2M1: in bytes), head_dim contiguous;
 *             those of k and v the same
 *   k_scale, v_scale  with FD_DTYPE_E4M3: [n_pages, kv_heads, page_size] bytes, strides {page, head},
 *             rows contiguous; byte b stands for the scale 2^(b - 127), b in [1, 254], and a cached
 *             value is its code times that scale.  With FD_DTYPE_E2M1: [n_pages, kv_heads, page_size,
 *             head_dim / 32] bytes, one for 32 features, rows contiguous and aligned to their bytes; b in
 *             [0, 254], 255 makes its 32 values NaN (E8M0).  NULL with FD_DTYPE_BF16
 *   page_table  [requests, max_pages] int32 on the device, rows table_stride elements apart: key j of
 *             request r is row j % page_size of page page_table[r][j / page_size].  An entry outside
 *             [0, n_pages) is no page: its keys are not there (not written, read as zeros, not visible)
 *   cache_lens  [requests] int32 on the device: the keys of each request, the new tokens of the call
 *             included (clamped to [0, max_pages * page_size]); the last n new tokens of request r are
 *             its keys cache_lens[r] - n .. cache_lens[r] - 1.  Not used by fd_paged_kv_read
 *
 * Limits: head_dim 64, 128 or 256; page_size a power of two in [16, 256]; cache rows and
 * tensors 16-byte aligned; row strides below 2^20 and page strides below 2^35 elements;
 * max_pages * page_size < 2^27.
 */
typedef struct fd_paged_cache {
  void* k;
  void* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t k_strides[3];
  int64_t v_strides[3];
  int64_t k_scale_strides[2];
  int64_t v_scale_strides[2];
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* cache_lens;
  int32_t n_pages;
  int32_t page_size;
  int32_t max_pages;
  int32_t kv_heads;
  int32_t head_dim;
  int32_t dtype;
} fd_paged_cache;

/*
 * Writes the keys and values of new tokens into their pages.
 *
 *   k, v  [batch, kv_heads, seq_len, head_dim] bf16, strides {b, h, t, d} in elements (d contiguous)
 * Without cu_seqlens request r is batch row r with seq_len new tokens.  With cu_seqlens (device
 * int32[n_seqs + 1], non-decreasing from 0) batch is 1 and request r's new tokens are
 * [cu_seqlens[r], cu_seqlens[r + 1]) of the T axis; tokens behind the last request are ignored.
 *
 * FD_DTYPE_E4M3: per (token, head) the scale is the smallest 2^E with max|x| <= 448 * 2^E over the
 * row's finite values (E >= -126; 2^0 for a row of zeros), the code is x / 2^E rounded to nearest
 * even; an infinity becomes +-448 * 2^E, a NaN stays NaN.  Powers of two keep the division and the way
 * back exact, so a value is off by at most half a step of its code.
 * FD_DTYPE_E2M1: the same per 32 features with 6 in the place of 448; values from 3 * 2^126 on are held as
 * 3 * 2^126 (the next code's 2^128 is no bf16 number); an infinity becomes +-6 * 2^E (+-3 * 2^126 where E
 * is 126), and a NaN makes its 32 values NaN.
 * A page that two requests of a call write must not be shared between them at the same rows.
 */
FD_API int fd_paged_kv_write(const void* k, const void* v, const int64_t k_strides[4], const int64_t v_strides[4],
                             const fd_paged_cache* cache, int batch, int seq_len, const int32_t* cu_seqlens,
                             int n_seqs, void* stream);

/*
 * The first cu_seqlens[r + 1] - cu_seqlens[r] keys and values of every request r as dense bf16 rows
 * [cu_seqlens[r], cu_seqlens[r + 1]) of k_out and v_out [kv_heads, total, head_dim] (strides {h, t};
 * d contiguous).  Keys past the page table or on no page are zeros; rows behind the last request are
 * left as they were.  cache_lens is not used.  A cached value of 2^128 (values from 248 * 2^120 on are
 * held as one in E4M3) is read as bf16's largest, 255 * 2^120.
 */
FD_API int fd_paged_kv_read(const fd_paged_cache* cache, void* k_out, void* v_out, const int64_t k_strides[2],
                            const int64_t v_strides[2], int64_t total, const int32_t* cu_seqlens, int n_seqs,
                            void* stream);

/*
 * Causal grouped-query attention of the new tokens of every request over its paged cache, which
 * holds their own keys and values already (fd_paged_kv_write).  New token i of n of request r sees
 * the keys 0 .. cache_lens[r] - n + i; a row that sees no key is zeros.  fp32 softmax.  The P V product
 * takes each probability as the sum of two bf16 (good to 2^-16 of it) in the kernels for few rows, as one
 * bf16 in the one for pieces, whose denominator sums the rounded ones.  Pieces: more than 64 rows (tokens
 * times query heads of a key head) in the longest request, unless a key head has at most 128 rows in all
 * and the page table is at most 16384 keys wide.
 *
 *   q, out  [batch, q_heads, seq_len, head_dim] bf16, strides {b, h, t, d}; query head h reads key
 *           head h / (q_heads / kv_heads); at most 2048 query heads per key head
 *   gate    NULL, or logically like out: out = attention * sigmoid(gate), rounded to bf16 once
 *   cu_seqlens, n_seqs  as in fd_paged_kv_write; rows of out behind the last request are left as
 *           they were
 *   max_seqlen  (host) the longest request's new tokens (seq_len without cu_seqlens).  It chooses the
 *           kernel by the rows of a key head and bounds nothing: longer requests are computed too
 *   workspace  fd_paged_gqa_workspace_bytes(...) bytes, 16-byte aligned.  Long key ranges are split
 *           over workgroups, whose parts a second launch joins, both on `stream`: calls that may
 *           overlap need workspaces of their own
 * A row's last bits depend on how the call splits its keys, which follows from all requests' lengths.
 * Scores are fp32 sums, and p v is summed in fp32 before it is divided by the denominator, with a p of up to
 * 2^8: values from 2^120 / (keys seen) on may overflow where the quotient would not.
 * Masked or absent keys never reach a row, not even as NaN or infinities.  An E4M3 value of 2^128 (fd_paged_kv_read) is
 * infinite to the kernel for pieces.
 */
FD_API int fd_paged_gqa_fwd(const void* q, const fd_paged_cache* cache, const void* gate, void* out,
                            const int64_t q_strides[4], const int64_t gate_strides[4], const int64_t out_strides[4],
                            int batch, int q_heads, int seq_len, float scale, const int32_t* cu_seqlens, int n_seqs,
                            int max_seqlen, void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace of fd_paged_gqa_fwd for these sizes, or a negative FD_ERR_* code. */
FD_API int64_t fd_paged_gqa_workspace_bytes(int batch, int q_heads, int kv_heads, int seq_len, int head_dim,
                                            int page_size, int max_pages, int n_seqs, int max_seqlen);

/*
 * The attention weight that cached keys draw from new tokens, added to what they have drawn:
 *   weights[row(r)][h][j] += sum of softmax(scale q K^T)[.., j] over the new tokens of request r and the query heads of
 * key head h, for the keys j that the tokens see (as in fd_paged_gqa_fwd: causal, on a page; v of the cache is not read
 * and may be k).  fp32 throughout, in an order that the sizes fix.
 *
 *   q       as in fd_paged_gqa_fwd
 *   weights [weight_rows, kv_heads, >= max_pages * page_size] fp32, strides {row, head} in elements, keys contiguous;
 *           no two of its elements the same memory
 *   row_indices  device int32[requests]: request r's row of weights; NULL: row r.  An index outside [0, weight_rows), or
 *           one that an earlier request of the call names already, is no row: nothing is added for that request
 *   last    the last `last` new tokens of each request count; 0: all of them
 *   cu_seqlens, n_seqs, max_seqlen  as in fd_paged_gqa_fwd
 *   workspace  fd_paged_key_weights_workspace_bytes(...) bytes, 16-byte aligned; calls that may overlap need their own.
 *           With up to 16 rows (tokens times query heads of a key head) in the longest request it holds their scores, 4 bytes
 *           for each of max_pages * page_size keys, up to 2^28 bytes in all; beyond that a call takes the kernels for more
 *           rows, up to five times as long
 * Keys that no token sees keep their weight; a key that is NaN makes the weights of a row's keys NaN, as a softmax does.
 * Scores that overflow fp32 do so too, and E4M3 values of 2^128 (fd_paged_kv_read) are infinite here.
 */
FD_API int fd_paged_key_weights(const void* q, const fd_paged_cache* cache, float* weights, const int64_t q_strides[4],
                                const int64_t weight_strides[2], int weight_rows, const int32_t* row_indices, int batch,
                                int q_heads, int seq_len, float scale, int last, const int32_t* cu_seqlens, int n_seqs,
                                int max_seqlen, void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace of fd_paged_key_weights for these sizes, or a negative FD_ERR_* code. */
FD_API int64_t fd_paged_key_weights_workspace_bytes(int batch, int q_heads, int kv_heads, int seq_len, int head_dim,
                                                    int page_size, int max_pages, int n_seqs, int max_seqlen, int last);

/*
 * Cuts every request to at most `keep` keys: its `recent` last ones and, per key head, those of largest weight among the
 * others (of equal weights the lowest key; NaN below everything).  The kept keys' rows and scales move in their order to
 * the pages of new_table, their weights to the front of their row.
 *
 *   weights, weights_out  [weight_rows, kv_heads, >= max_pages * page_size] fp32 of the same strides {row, head}, keys
 *           contiguous; the same memory, or without overlap.  weights_out[..][0 .. n - 1] are the kept keys' weights,
 *           n = min(cache_lens, keep), and [n, cache_lens) are 0
 *   row_indices  as in fd_paged_key_weights; a request without a row counts as one of equal weights
 *   new_table  [requests, new_max_pages] int32, rows new_table_stride apart, new_max_pages * page_size >= keep.  Its
 *           pages must be distinct and not among those that the call's page table names for keys of any request.  Entries outside
 *           [0, n_pages) are no pages: their keys are not written.  Kept keys on no page become zeros
 *   kept    [requests, kv_heads, keep] int32, contiguous: the old place of every kept key, -1 behind the last one
 *   new_lens  [requests] int32: min(cache_lens, keep)
 * The old pages are left as they were.  Limit: requests * kv_heads * keep below 2^27.
 */
FD_API int fd_paged_kv_evict(const fd_paged_cache* cache, const float* weights, float* weights_out,
                             const int64_t weight_strides[2], int weight_rows, const int32_t* row_indices,
                             const int32_t* new_table, int64_t new_table_stride, int new_max_pages, int requests,
                             int keep, int recent, int32_t* kept, int32_t* new_lens, void* stream);

/*
 * The gated delta rule of the Gated-DeltaNet layers token by token (transformers'
 * torch_recurrent_gated_delta_rule), for the few new tokens of requests whose state is kept.
 * fd_gated_delta_fwd is the form for whole prompts and long pieces.
 *
 *   q, k  [batch, seq_len, k_heads, 128], v, out [batch, seq_len, v_heads, 128] bf16 contiguous
 *   g     [batch, seq_len, v_heads] fp32; beta likewise, of beta_dtype (FD_DTYPE_BF16 or FD_DTYPE_F32)
 *   state, state_out  [n_pool, v_heads, 128, 128] fp32 contiguous (key dimension first), or NULL (state:
 *         zeros, state_out: not kept).  They may be the same memory; otherwise they do not overlap
 *   state_indices  device int32[requests]: request r's state is row state_indices[r] of both; NULL:
 *         row r.  An index outside [0, n_pool), or one that an earlier request of the call names
 *         already, is no state: that request starts from zeros and keeps nothing
 * Requests: batch rows, or with cu_seqlens (batch 1) [cu_seqlens[r], cu_seqlens[r + 1]); a request
 * without new tokens hands its state on, rows of out behind the last request are left as they were.
 * With l2norm_qk q and k rows are divided by sqrt(sum of squares + 1e-6).  All arithmetic in fp32
 * without intermediate rounding (fd_gated_delta_fwd rounds the normalised q and k to bf16, as
 * transformers' l2norm does on bf16 tensors); out is rounded once.
 *
 * Limits: head dims 128; v_heads % k_heads == 0; 16-byte aligned pointers.
 */
FD_API int fd_gated_delta_step(const void* q, const void* k, const void* v, const float* g, const void* beta,
                               void* out, const float* state, float* state_out, int n_pool,
                               const int32_t* state_indices, int batch, int seq_len, int k_heads, int v_heads,
                               int head_k_dim, int head_v_dim, float scale, int beta_dtype, int l2norm_qk,
                               const int32_t* cu_seqlens, int n_seqs, void* stream);

/*
 * fd_packed_conv_strided_fwd continued from a state: the taps before a request's first new token
 * read its state, the last width - 1 inputs before it (oldest first), and state_out receives the
 * last width - 1 inputs after its new tokens.  Values as fd_packed_conv_fwd: a request fed in
 * pieces from a zero state gets the bits of the request in one piece.
 *
 *   state, state_out  [n_pool, width - 1, C] bf16 contiguous, C = 2 * key_dim + value_dim; the same
 *         memory, or without overlap
 *   state_indices, requests, rows behind the last request  as in fd_gated_delta_step
 *
 * Limits: width in [2, 4]; key_dim and value_dim multiples of 8; 16-byte aligned pointers;
 * x_row_stride a multiple of 8, at least C.
 */
FD_API int fd_packed_conv_state(const void* x, int64_t x_row_stride, const void* weight, const void* bias,
                                const void* state, void* state_out, int n_pool, const int32_t* state_indices,
                                void* q, void* k, void* v, int batch, int seq_len, int key_dim, int value_dim,
                                int width, const int32_t* cu_seqlens, int n_seqs, int activation, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FD_CACHE_H */
