// Launch of the attention kernels over a 4-bit cache for one element type.
#pragma once
#include "attn_int4.cuh"
#include "tc_util.cuh"

namespace tsa {

constexpr int kInt4Stages = 2;  // stages in a warp's ring

template <typename T, int DG, int NT, bool kTwin, int KT, int kWarps, int kMinBlocks>
static cudaError_t int4_run(const Int4Attn& a, int blocks, cudaStream_t st) {
  constexpr int D = DG * 32;
  constexpr size_t queries = NT > 1 ? (sizeof(T) == 4 ? 2 : 1) * NT * DG * 512 : 0;
  constexpr size_t barriers = int4_barrier_bytes(kWarps, kInt4Stages);
  constexpr size_t ring = barriers + (size_t)kWarps * (kInt4Stages * 2 * KT * (D / 2 + D / 16) + queries);
  constexpr size_t merge = barriers + (size_t)kWarps * NT * 8 * (D + 4 + 2) * sizeof(float);
  constexpr size_t most = ring + (size_t)2 * (kInt4MaxRows + 1) * sizeof(int);
  const size_t need = ring + (a.by_pair ? 0 : (size_t)2 * (a.p.batch + 1) * sizeof(int));
  const size_t smem = need > merge ? need : merge;
  auto kernel = attn_int4_kernel<T, DG, NT, kTwin, KT, kInt4Stages, kWarps, kMinBlocks>;
  cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(kernel), (int)(most > merge ? most : merge));
  if (e != cudaSuccess) return e;
  e = launch_dependent(kernel, dim3((unsigned)blocks), dim3(kWarps * 32), smem, st, a);
  if (e != cudaSuccess || a.by_pair) return e;
  const int64_t rows = (int64_t)a.p.batch * a.p.q_heads * a.p.q_len;
  // Warps that merge one row: about four parts each (of eight: 27.9 against 26.8 us for 16 rows x 8 heads), while
  // all of them fit on the GPU at once, two blocks a SM (2560 rows with up to ten parts: 51 against 59 us).
  int row_warps = a.parts > 16 ? 8 : a.parts > 8 ? 4 : a.parts > 4 ? 2 : 1;
  while (row_warps > 1 && rows * row_warps > 148 * 2 * 8) row_warps /= 2;
  return launch_dependent(attn_int4_combine<T, NT, kWarps>, dim3((unsigned)((rows * row_warps + 7) / 8)), dim3(256),
                          0, st, a, row_warps, KT);
}

template <typename T, int NT, bool kTwin, int KT, int kWarps, int kMinBlocks>
static cudaError_t int4_run_dims(const Int4Attn& a, int blocks, cudaStream_t st) {
  switch (a.p.head_dim / 32) {
    case 1: return int4_run<T, 1, NT, kTwin, KT, kWarps, kMinBlocks>(a, blocks, st);
    case 2: return int4_run<T, 2, NT, kTwin, KT, kWarps, kMinBlocks>(a, blocks, st);
    case 3: return int4_run<T, 3, NT, kTwin, KT, kWarps, kMinBlocks>(a, blocks, st);
    case 4: return int4_run<T, 4, NT, kTwin, KT, kWarps, kMinBlocks>(a, blocks, st);
  }
  return cudaErrorInvalidValue;
}

template <typename T, bool kTwin>
static cudaError_t int4_run_one(const Int4Attn& a, const Int4Shape& shape, int blocks, cudaStream_t st) {
  if (shape.keys == 16) return int4_run_dims<T, 1, kTwin, 16, 4, 3>(a, blocks, st);
  if (shape.warps == 12) return int4_run_dims<T, 1, kTwin, 64, 12, 1>(a, blocks, st);
  switch (a.p.head_dim / 32) {
    case 5: return int4_run<T, 5, 1, kTwin, 32, 4, 2>(a, blocks, st);
    case 6: return int4_run<T, 6, 1, kTwin, 32, 4, 2>(a, blocks, st);
    case 7: return int4_run<T, 7, 1, kTwin, 32, 4, 2>(a, blocks, st);
    case 8: return int4_run<T, 8, 1, kTwin, 32, 4, 2>(a, blocks, st);
  }
  return int4_run_dims<T, 1, kTwin, 64, 4, 3>(a, blocks, st);
}

// One column tile.
template <typename T>
cudaError_t attn_int4_launch(const Int4Attn& a, const Int4Shape& shape, int blocks, cudaStream_t st) {
  if (shape.nt > 1) return attn_int4_launch_wide<T>(a, shape, blocks, st);
  if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
    if (shape.twin) return int4_run_one<T, true>(a, shape, blocks, st);
  }
  return int4_run_one<T, false>(a, shape, blocks, st);
}

// Two or (half types) three column tiles, D up to 128.
template <typename T>
cudaError_t attn_int4_launch_wide(const Int4Attn& a, const Int4Shape& shape, int blocks, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (shape.nt == 3) return int4_run_dims<T, 3, false, 64, 4, 2>(a, blocks, st);
  }
  return int4_run_dims<T, 2, false, 64, 4, 2>(a, blocks, st);
}

// Instantiated once, in the sources of the wide kernels.
extern template cudaError_t attn_int4_launch_wide<__nv_bfloat16>(const Int4Attn&, const Int4Shape&, int, cudaStream_t);
extern template cudaError_t attn_int4_launch_wide<__half>(const Int4Attn&, const Int4Shape&, int, cudaStream_t);
extern template cudaError_t attn_int4_launch_wide<float>(const Int4Attn&, const Int4Shape&, int, cudaStream_t);

}  // namespace tsa
