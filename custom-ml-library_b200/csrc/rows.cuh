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
