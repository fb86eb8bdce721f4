// The CUDA-core attention under a window and over drafted tokens in double.
#include "attn_rows.cuh"

namespace tsa {
TS_ROWS_INSTANTIATE(f64, double)
}  // namespace tsa
