// Entry points of the CUDA-core attention under a window and over drafted tokens (attn_rows.cuh).
#pragma once
#include "common.cuh"
#include "tree.cuh"
#include "window.cuh"

namespace tsa {

struct RowsWindow {
  ts_attn_params p;
  WindowArgs win;
  __device__ __forceinline__ int kv_end(int b) const {
    return p.kv_lens ? min(p.kv_len, max(0, p.kv_lens[b])) : p.kv_len;
  }
  __device__ __forceinline__ int64_t offset(int b) const {
    return p.kv_lens ? (int64_t)kv_end(b) - p.q_len : p.causal_offset;
  }
};

// Row tiles of a forward block: four for up to 64 channels (2 x 2000 queries, 8 heads of 64: 425 us, with two 449), two
// for more (2 x 1500 of 128: 540 us, with four 600).
inline int rows_widest(int dim) { return dim <= 64 ? 4 : 2; }

// Row tiles of a block, at most `widest`.  A tile costs the reads of its columns, the same for any number of row tiles,
// and those of its rows (about 8 to 1), and the blocks of an SM share what it can read.
inline int rows_rt(int rows, int64_t slices, int widest) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int rt = 1; rt <= widest; rt *= 2) {
    const int64_t blocks = ceil_div(rows, 16 * rt) * slices, sms = device_sms();
    const int64_t cost = (blocks + sms - 1) / sms * (8 + rt);
    if (cost < least) least = cost, best = rt;
  }
  return best;
}

// Without arguments or a workspace (a null) rows_tree and rows_window_bwd only give the workspace's bytes.
#define TS_ROWS_DECLARE(suffix)                                                                                    \
  cudaError_t rows_window_fwd_##suffix(const RowsWindow& a, cudaStream_t st);                                      \
  cudaError_t rows_window_bwd_##suffix(const ts_attn_bwd_params& bp, const WindowArgs& win, size_t* bytes,         \
                                       void* ws, cudaStream_t st);                                                 \
  cudaError_t rows_tree_##suffix(const ts_attn_params& p, TreeArgs* a, size_t* bytes, void* ws, cudaStream_t st);
TS_ROWS_DECLARE(f32)
TS_ROWS_DECLARE(f64)
TS_ROWS_DECLARE(f16)
TS_ROWS_DECLARE(bf16)
#undef TS_ROWS_DECLARE

}  // namespace tsa
