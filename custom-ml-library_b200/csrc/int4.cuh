// The paged 4-bit KV cache: page layout, quantisation rule and the entry points of its kernels
// (kv_int4.cu, attn_int4*.cu, kv_pages.cu).
//
// One 4-bit value serves one channel of one token and KV head, one fp16 scale 32 channels of it:
//   scale = max|x| / 7, rounded up to 5 significant bits, held in [2^-20, 9216]
//   n     = round_half_even(x / scale) in [-7, 7], stored as the nibble n + 8
// n has 3 significant bits, so n * scale has at most 8 and is exact in bf16 and in fp16 (9216 * 7 <
// 65504, and a scale of at least 2^-20 with 5 bits is a multiple of 2^-24, fp16's smallest step).
// Every kernel therefore sees the same K and V whatever type it computes in; rounding the scale up
// costs at most 1/16 of the quantisation step.  Inputs beyond +-64512 (infinities too) saturate, a
// NaN becomes 0, so a cache never holds a non-finite value.
//
// The block of one page and KV head is contiguous, so one bulk copy fetches all of it:
//   K nibbles [page_size, D/2] | K scales fp16 [page_size, D/32] | V nibbles | V scales
// A row is D/8 32-bit words; word t * (D/32) + g holds the channels 32 g + 8 t + e in nibble e
// (bits 4e..4e+3).  Lane t of the four that share a key row in an mma fragment then reads D/32
// consecutive words, one of each scale group.
#pragma once
#include "common.cuh"

namespace tsa {

constexpr float kInt4ScaleMin = 9.5367431640625e-07f;  // 2^-20
constexpr float kInt4ScaleMax = 9216.f;

__host__ __device__ __forceinline__ int int4_row_bytes(int head_dim) { return head_dim / 2 + head_dim / 16; }
__host__ __device__ __forceinline__ int int4_block_bytes(int head_dim, int page_size) {
  return 2 * page_size * int4_row_bytes(head_dim);
}

__device__ __forceinline__ float int4_scale(float amax) {
  // amax / 7, correctly rounded: the quotient by 1/7's nearest float, corrected once with its remainder
  // (Markstein, IBM J. Res. Dev. 34, 1990)
  constexpr float seventh = 1.f / 7.f;
  float s = amax * seventh;
  s = fminf(fmaf(fmaf(-7.f, s, amax), seventh, s), kInt4ScaleMax);
  const float up = __uint_as_float((__float_as_uint(s) + 0x7FFFFu) & ~0x7FFFFu);
  return fminf(fmaxf(up, kInt4ScaleMin), kInt4ScaleMax);
}

// Page of row b's token, or -1 where the table has none (a bad entry is the caller's error: the
// kernels record it in the fault word and leave the page alone).
__device__ __forceinline__ int int4_page(const ts_kv4_cache& c, int b, int slot) {
  if ((unsigned)slot >= (unsigned)c.slots) return -1;
  const int page = c.table[(int64_t)b * c.table_stride + slot];
  return page >= 0 && page < c.pages ? page : -1;
}

cudaError_t kv_append_int4(const ts_view4& key, const ts_view4& value, int dtype, int steps, const ts_kv4_cache& c,
                           int64_t position, const int32_t* positions, int32_t* positions_out, uint32_t* fault,
                           cudaStream_t st);
// Dequantises tokens [starts[b] (or 0), + length) of every row; tokens at or past lens[b] (when
// given) are written as zeros, with `tile` > 0 (and no starts) only up to the end of the tile of that many tokens that
// the row ends in.
cudaError_t kv_gather_int4(const ts_kv4_cache& c, const int32_t* starts, const int32_t* lens, const ts_view4& key,
                           const ts_view4& value, int dtype, int length, int tile, uint32_t* fault, cudaStream_t st);

// The kernel that attends straight over the pages.  Its workspace; false where it takes not even one token of one
// row, whose line of work would pass what a launch counts (2^30 stages of 16 to 64 keys, over all KV heads).
bool attn_int4_workspace(const ts_attn_params& p, size_t* bytes);
cudaError_t attn_int4_forward(const ts_attn_params& p, const ts_kv4_cache& c, void* ws, uint32_t* fault,
                              cudaStream_t st);

cudaError_t kv_pages_copy(const ts_page_pool& src, const ts_page_pool& dst, const int32_t* from, const int32_t* to,
                          int count, cudaStream_t st);
cudaError_t kv_pages_fork(const int32_t* table, int64_t table_stride, const int32_t* lens, int rows,
                          const int32_t* index, int32_t* table_out, int64_t table_out_stride, int32_t* lens_out,
                          int rows_out, int slots, int page_size, int32_t* refs, int pages, int32_t* counters,
                          cudaStream_t st);
size_t kv_pages_reserve_workspace(int pages, int rows);
cudaError_t kv_pages_reserve(const ts_page_pool& pool, int32_t* table, int64_t table_stride, const int32_t* lens,
                             int rows, int slots, int page_size, int steps, const int32_t* row_steps, int32_t* refs,
                             int32_t* counters, void* ws, cudaStream_t st);
size_t kv_pages_compact_workspace(int pages);
cudaError_t kv_pages_compact(const ts_page_pool& pool, const int32_t* table, int32_t* table_out, int rows, int slots,
                             int64_t table_stride, int64_t table_out_stride, const int32_t* refs, int32_t* refs_out,
                             int32_t* counters, void* ws, cudaStream_t st);
}  // namespace tsa
