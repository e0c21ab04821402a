// Launchers of the logits operators.
#pragma once

#include "lkl_common.cuh"

namespace lkl {

// Rows of a [B, T, V] tensor with element strides (sb, st, 1).  low: what the rows'
// log-sum-exp in fp32 lacks, or nullptr.
struct LogitsView {
  const void* x;
  long long T, V, sb, st;
  int dtype;
  float* low;
};

cudaError_t launch_token_logprobs(const LogitsView& x, long long rows, const int64_t* targets,
                                  int64_t ignore, int top_k, float* logprob, float* entropy,
                                  float* lse, float* top_v, int64_t* top_i, cudaStream_t st);
cudaError_t launch_token_logprobs_backward(const LogitsView& x, long long rows,
                                           const int64_t* targets, int64_t ignore,
                                           const float* lse, const float* entropy,
                                           const float* g_lp, const float* g_en, void* dx,
                                           cudaStream_t st);
// row_kl: one float a row of scratch.
cudaError_t launch_logits_kl_forward(const LogitsView& s, const LogitsView& t, long long rows,
                                     const void* mask, int mdt, float inv_tau, float* lse_s,
                                     float* lse_t, float* row_kl, float* loss, cudaStream_t st);
cudaError_t launch_logits_kl_backward(const LogitsView& s, const LogitsView& t, long long rows,
                                      const void* mask, int mdt, float inv_tau,
                                      const float* lse_s, const float* lse_t, const float* dloss,
                                      void* ds, cudaStream_t st);

}  // namespace lkl
