// Entry points of the KV-cache maintenance kernels (kv_cache.cu).
#pragma once
#include "common.cuh"

namespace tsa {
cudaError_t kv_append(const ts_kv_append_params& p, cudaStream_t stream);
cudaError_t kv_reorder(const ts_view4& src, const ts_view4& dst, int dtype, int batch, int heads,
                       int length, int channels, const int32_t* index, cudaStream_t stream);

// kv_keep.cu: one launch over several layers' keys and values.
constexpr int kKeepTensors = 128;
struct KvKeep {
  void* data[kKeepTensors];  // keys and values of one layer after the other
  int64_t stride[2][3];      // bytes between rows, heads and slots of keys, of values
  int row_bytes[2];          // of a slot's channels
  int tensors, batch, heads, nodes;
  int64_t capacity;
  const int32_t *base, *path, *counts;
  int64_t path_stride;
};
cudaError_t kv_keep(const KvKeep& a, cudaStream_t stream);
// positions [batch, nodes] of drafted nodes behind lens[b] committed tokens.
cudaError_t tree_positions(const int32_t* parents, int64_t stride, const int32_t* lens, int batch, int nodes,
                           int32_t* positions, cudaStream_t stream);
}  // namespace tsa
