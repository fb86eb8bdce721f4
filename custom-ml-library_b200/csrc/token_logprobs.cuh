// Entry points of the token log probabilities (token_logprobs.cu).
#pragma once
#include "common.cuh"

namespace tsa {
constexpr int kMaxTopTokens = 32;  // alternatives of a row
cudaError_t token_logprobs(const ts_token_logprobs& p, cudaStream_t st);
cudaError_t token_logprobs_bwd(const ts_token_logprobs& p, const float* grad_logprob, const float* grad_entropy,
                               const float* grad_top, void* grad_logits, int64_t grad_stride, cudaStream_t st);
}  // namespace tsa
