// Host-side description of one attention call, shared by its launchers.
#pragma once

#include "lkl_common.cuh"

namespace lkl {

struct AttnProblem {
  int B, Hq, Hkv, T, D;
  int dtype, causal;
  float sc;
};

// Tensors of a call and their element strides; out, lse, ... as in lkl_attn_backward.
struct AttnTensors {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const void* dout;
  void *dq, *dk, *dv;
  TensorStrides sq, sk, sv, so, sdo, sdq, sdk, sdv;
};

// CUDA-core kernels: every head dim of the set, any strides and alignment.
cudaError_t launch_attn_generic_forward(const AttnProblem& p, const AttnTensors& t,
                                        const uint32_t* bits, cudaStream_t st);
// rows[b, h, i] = (-lse log2(e), delta_i); (-inf, 0) for a row the mask removes.
cudaError_t launch_attn_delta(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                              float2* rows, cudaStream_t st);
// delta_i = sum_j P_ij (dout_i . v_j) equals dout_i . out_i but for out's rounding and that
// of P behind it.  dS_ij = P_ij (dP_ij - delta_i) is a small difference where one key has
// most of a row, as in rows of few keys: with the rounded out, dk of two tokens was off by
// 17% (bf16), and 1% at eight.  Rows that see at most this many keys (in a causal sequence
// of any length, the first of its tokens that the mask keeps; else all rows of a sequence
// with no more tokens) therefore take the sum; beyond it rows of many keys carry the
// gradient and the roundings of dS and of the result outweigh that of out.  By how much goes
// by the head dim.  Error of dq in bf16, emulated, with these rows by the sum and with all
// (the result's rounding alone: 0.0017), causal and not:
//   D 128, T 4000: 0.00238 and 0.00235, 0.00239 and 0.00236
//   D 64, T 1000:  0.00247 and 0.00241, 0.00252 and 0.00242
//   D 32, T 3000:  0.00258 and 0.00246, 0.00269 and 0.00253
//   D 16, T 3000:  0.00275 and 0.00258, 0.00285 and 0.00258
//   D 8, T 6500:   0.0034 and 0.0027, 0.0033 and 0.0029
// A 16-bit remainder of out from the forward would bring the first of each pair near the
// second.  It has no place in the call: the backward takes what a forward returns, out and
// lse, and gives the same bits through autograd and by itself.
constexpr int kExactDeltaKeys = 256;
// The same into rows[] by that sum, for the rows that see at most kExactDeltaKeys keys.
cudaError_t launch_attn_exact_delta(const AttnProblem& p, const AttnTensors& t,
                                    const uint32_t* bits, float2* rows, cudaStream_t st);
// Those rows are the first tokens of a sequence.  Under a mask that leaves room for more
// (T > kExactDeltaKeys) they may stand anywhere, and a kernel finds them by their rank
// among the tokens that the mask keeps.
inline __host__ __device__ bool exact_delta_ranked(const AttnProblem& p, const uint32_t* bits) {
  return bits != nullptr && p.T > kExactDeltaKeys;
}

// A block of 256 threads finds the tokens of batch b whose rows see at most
// kExactDeltaKeys keys: their positions, ascending, in pos[] and their number in every
// thread.  sums: one int a warp.
__device__ __forceinline__ int few_key_tokens(const uint32_t* bits, const AttnProblem& p, int b,
                                              int* pos, int* sums) {
  const int words = (p.T + 31) >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n = 0;   // tokens of the words before
  for (int w0 = 0; w0 < words; w0 += 256) {
    const int w = w0 + threadIdx.x;
    uint32_t m = w < words ? bits[(size_t)b * words + w] : 0u;
    int upto = __popc(m);
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int at = n + upto - __popc(m);
    for (int k = 0; k < 8; ++k) {
      if (k < warp) at += sums[k];
      n += sums[k];
    }
    for (; m && at < kExactDeltaKeys; m &= m - 1) pos[at++] = w * 32 + __ffs(m) - 1;
    __syncthreads();
    if (n > kExactDeltaKeys) return p.causal ? kExactDeltaKeys : 0;
  }
  return n;
}
cudaError_t launch_attn_generic_backward(const AttnProblem& p, const AttnTensors& t,
                                         const uint32_t* bits, const float2* rows,
                                         cudaStream_t st);

// Tensor-core kernels: head dims up to 128, 16-byte aligned pointers, strides
// that are positive multiples of 8 elements, and more elements a head than this.  Up to it
// the CUDA-core kernels take a head in one or two 32-row tiles, and keep P and dS in fp32:
// dq and dk carry their own rounding alone (bf16 0.0017 of their size off instead of 0.0024;
// in a handful of tokens up to 0.0028).  Forward / backward of 2 and of 2048 heads,
// CUDA cores against tensor cores, us on the device: D 16, T 32: 4.9 / 16 against 5.5 / 13,
// 19 / 71 against 60 / 168; D 64, T 8: 6.0 / 21 against 5.4 / 13, 30 / 109 against 60 / 162.
// D 64, T 32 would take 10 / 39 against 5.6 / 13, 55 / 217 against 61 / 180.
constexpr int kAttnFewElements = 512;
bool attn_sm100_supports(const AttnProblem& p, const AttnTensors& t);
cudaError_t launch_attn_sm100_forward(const AttnProblem& p, const AttnTensors& t,
                                      const uint32_t* bits, cudaStream_t st);
bool attn_sm100_backward_supports(const AttnProblem& p, const AttnTensors& t);
// Scratch of the backward: row statistics (either path); dS tiles: what it asks
// for, the least it runs with, and what holds one kv group (below that, dq is
// summed over launches in attn_sm100_acc_bytes of fp32).
size_t attn_stats_bytes(const AttnProblem& p);
size_t attn_sm100_ds_bytes(const AttnProblem& p);
size_t attn_sm100_sums_bytes(const AttnProblem& p);   // behind the dS tiles, optional
size_t attn_sm100_ds_min_bytes(const AttnProblem& p);
size_t attn_sm100_group_bytes(const AttnProblem& p);
size_t attn_sm100_acc_bytes(const AttnProblem& p);
cudaError_t launch_attn_sm100_backward(const AttnProblem& p, const AttnTensors& t,
                                       const uint32_t* bits, float* stats, void* ds,
                                       size_t ds_bytes, float* acc, cudaStream_t st);

}  // namespace lkl
