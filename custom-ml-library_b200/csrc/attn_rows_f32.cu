// The CUDA-core attention under a window and over drafted tokens in float.
#include "attn_rows.cuh"

namespace tsa {
TS_ROWS_INSTANTIATE(f32, float)
}  // namespace tsa
