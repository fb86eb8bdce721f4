// Launch of the attention kernels over a 4-bit cache for one element type.
#pragma once
#include "attn_int4.cuh"

namespace tsa {

constexpr int kInt4Keys = 64;   // tokens of a stage
constexpr int kInt4Stages = 2;  // stages in flight for each warp
constexpr int kInt4Warps = 4;

template <typename T, int DG, int NT>
static cudaError_t int4_run(const Int4Attn& a, cudaStream_t st) {
  constexpr int D = DG * 32;
  constexpr size_t ring = (size_t)kInt4Warps * kInt4Stages * (2 * kInt4Keys * (D / 2 + D / 16) + sizeof(uint64_t));
  constexpr size_t red = (size_t)kInt4Warps * NT * 8 * (D + 4 + 2) * sizeof(float);
  constexpr size_t smem = ring > red ? ring : red;
  auto kernel = attn_int4_kernel<T, DG, NT, kInt4Keys, kInt4Stages, kInt4Warps>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int64_t blocks = (int64_t)a.p.batch * a.p.kv_heads * a.max_splits * a.col_blocks;
  const int64_t rows = (int64_t)a.p.batch * a.p.q_heads * a.p.q_len;
  if (blocks > 0x7FFFFFFF || rows > 0x7FFFFFFF) return cudaErrorInvalidValue;
  kernel<<<(unsigned)blocks, kInt4Warps * 32, smem, st>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess || a.max_splits == 1) return e;
  attn_int4_combine<T><<<(unsigned)rows, 128, 0, st>>>(a, NT * 8);
  return cudaGetLastError();
}

template <typename T>
cudaError_t attn_int4_launch(const Int4Attn& a, int nt, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {  // two column tiles: half types up to D = 128 (registers)
    if (nt == 2) {
      switch (a.p.head_dim) {
        case 32: return int4_run<T, 1, 2>(a, st);
        case 64: return int4_run<T, 2, 2>(a, st);
        case 96: return int4_run<T, 3, 2>(a, st);
        case 128: return int4_run<T, 4, 2>(a, st);
      }
      return cudaErrorInvalidValue;
    }
  }
  switch (a.p.head_dim) {
    case 32: return int4_run<T, 1, 1>(a, st);
    case 64: return int4_run<T, 2, 1>(a, st);
    case 96: return int4_run<T, 3, 1>(a, st);
    case 128: return int4_run<T, 4, 1>(a, st);
    case 160: return int4_run<T, 5, 1>(a, st);
    case 192: return int4_run<T, 6, 1>(a, st);
    case 224: return int4_run<T, 7, 1>(a, st);
    case 256: return int4_run<T, 8, 1>(a, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tsa
