// f32 instances of the attention over a 4-bit cache (attn_int4.cuh): one column tile.
#include "attn_int4_launch.cuh"

namespace tsa {
template cudaError_t attn_int4_launch<float>(const Int4Attn& a, const Int4Shape& shape, int blocks, cudaStream_t st);
}  // namespace tsa
