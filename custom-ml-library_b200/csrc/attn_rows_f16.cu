// The CUDA-core attention under a window and over drafted tokens in __half.
#include "attn_rows.cuh"

namespace tsa {
TS_ROWS_INSTANTIATE(f16, __half)
}  // namespace tsa
