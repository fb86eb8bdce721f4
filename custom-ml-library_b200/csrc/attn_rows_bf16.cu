// The CUDA-core attention under a window and over drafted tokens in __nv_bfloat16.
#include "attn_rows.cuh"

namespace tsa {
TS_ROWS_INSTANTIATE(bf16, __nv_bfloat16)
}  // namespace tsa
