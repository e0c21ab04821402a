// Operators over rows of logits: log probabilities of given tokens (with
// entropy and top alternatives) and the KL between two models' rows, each with
// its gradient.  One block a row.
#include <math_constants.h>

#include "lkl_logits.cuh"

namespace lkl {
namespace {

constexpr int kLThreads = 256;

__device__ __forceinline__ float logit(const LogitsView& x, size_t at) {
  if (x.dtype == LKL_F32) return reinterpret_cast<const float*>(x.x)[at];
  return load_elem(x.x, at, x.dtype);
}
__device__ __forceinline__ void put_logit(void* x, size_t at, int dtype, float v) {
  if (dtype == LKL_F32) reinterpret_cast<float*>(x)[at] = v;
  else if (dtype == LKL_BF16) reinterpret_cast<__nv_bfloat16*>(x)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(x)[at] = __float2half_rn(v);
}
__device__ __forceinline__ size_t row_at(const LogitsView& x, long long row) {
  return (size_t)((row / x.T) * x.sb + (row % x.T) * x.st);
}

template <typename Op>
__device__ __forceinline__ float block_reduce(float v, Op op) {
  __shared__ float red[kLThreads / 32];
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kLThreads / 32; ++w) v = op(v, red[w]);
  return v;
}
struct Add { __device__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };

__global__ void __launch_bounds__(kLThreads)
token_logprobs_kernel(const LogitsView x, const int64_t* __restrict__ targets, int64_t ignore,
                      int top_k, float* logprob, float* entropy, float* lse_out, float* top_v,
                      int64_t* top_i) {
  const long long row = blockIdx.x;
  const size_t at = row_at(x, row);
  float m = -CUDART_INF_F;
  for (long long c = threadIdx.x; c < x.V; c += kLThreads) m = fmaxf(m, logit(x, at + c));
  m = block_reduce(m, Max());
  float l = 0.f, a = 0.f;
  for (long long c = threadIdx.x; c < x.V; c += kLThreads) {
    const float d = logit(x, at + c) - m, e = expf(d);
    l += e;
    if (e != 0.f) a = fmaf(e, d, a);
  }
  l = block_reduce(l, Add());
  a = block_reduce(a, Add());
  const float lse = m + logf(l);
  if (threadIdx.x == 0) {
    const int64_t y = targets[row];
    float lp = CUDART_NAN_F;
    if (y == ignore) lp = 0.f;
    else if (y >= 0 && y < x.V) lp = (logit(x, at + y) - m) - logf(l);
    logprob[row] = lp;
    entropy[row] = logf(l) - a / l;
    lse_out[row] = lse;
  }
  // alternatives: the best that comes after the previous one in (value, -index)
  __shared__ float bv[kLThreads];
  __shared__ long long bi[kLThreads];
  float pv = CUDART_INF_F;
  long long pi = -1;
  for (int k = 0; k < top_k; ++k) {
    float v = -CUDART_INF_F;
    long long best = x.V;
    for (long long c = threadIdx.x; c < x.V; c += kLThreads) {
      const float w = logit(x, at + c);
      const bool after = w < pv || (w == pv && c > pi);
      if (after && (best == x.V || w > v)) {
        v = w;
        best = c;
      }
    }
    __syncthreads();
    bv[threadIdx.x] = v;
    bi[threadIdx.x] = best;
    __syncthreads();
    pv = bv[0];
    pi = bi[0];
    for (int i = 1; i < kLThreads; ++i)
      if (bi[i] < x.V && (pi == x.V || bv[i] > pv || (bv[i] == pv && bi[i] < pi))) {
        pv = bv[i];
        pi = bi[i];
      }
    if (threadIdx.x == 0) {
      top_v[row * top_k + k] = (pv - m) - logf(l);
      top_i[row * top_k + k] = pi < x.V ? pi : x.V - 1;  // a row of NaN
    }
  }
}

__global__ void __launch_bounds__(kLThreads)
token_logprobs_backward_kernel(const LogitsView x, const int64_t* __restrict__ targets,
                               int64_t ignore, const float* lse, const float* entropy,
                               const float* g_lp, const float* g_en, void* dx) {
  const long long row = blockIdx.x;
  const size_t at = row_at(x, row), out = (size_t)row * x.V;
  const int64_t y = targets[row];
  float g = g_lp && y != ignore ? g_lp[row] : 0.f;
  if (g_lp && y != ignore && (y < 0 || y >= x.V)) g = CUDART_NAN_F;
  const float h = g_en ? g_en[row] : 0.f, z = lse[row], H = entropy[row];
  for (long long c = threadIdx.x; c < x.V; c += kLThreads) {
    const float lp = logit(x, at + c) - z, p = expf(lp);
    float d = -p * g;
    if (p != 0.f) d -= h * p * (lp + H);
    if (c == y) d += g;
    put_logit(dx, out + c, x.dtype, d);
  }
}

__global__ void __launch_bounds__(kLThreads)
logits_kl_forward_kernel(const LogitsView s, const LogitsView t, const void* mask, int mdt,
                         float inv_tau, float* lse_s, float* lse_t, float* row_kl) {
  const long long row = blockIdx.x;
  if (mask && !mask_elem(mask, row, mdt)) {
    if (threadIdx.x == 0) lse_s[row] = lse_t[row] = row_kl[row] = 0.f;
    return;
  }
  const size_t as = row_at(s, row), at = row_at(t, row);
  float ms = -CUDART_INF_F, mt = -CUDART_INF_F;
  for (long long c = threadIdx.x; c < s.V; c += kLThreads) {
    ms = fmaxf(ms, logit(s, as + c));
    mt = fmaxf(mt, logit(t, at + c));
  }
  ms = block_reduce(ms, Max());
  mt = block_reduce(mt, Max());
  float ls = 0.f, lt = 0.f, a = 0.f;
  for (long long c = threadIdx.x; c < s.V; c += kLThreads) {
    const float xs = logit(s, as + c), xt = logit(t, at + c);
    const float e = expf((xt - mt) * inv_tau);
    ls += expf((xs - ms) * inv_tau);
    lt += e;
    if (e != 0.f) a = fmaf(e, xt - xs, a);
  }
  ls = block_reduce(ls, Add());
  lt = block_reduce(lt, Add());
  a = block_reduce(a, Add());
  if (threadIdx.x == 0) {
    // the difference of the two LSEs in 64 bits: the loss is what is left of it
    const double zs = (double)ms * inv_tau + log((double)ls);
    const double zt = (double)mt * inv_tau + log((double)lt);
    lse_s[row] = (float)zs;
    lse_t[row] = (float)zt;
    row_kl[row] = (float)((double)a * inv_tau / lt + (zs - zt));
  }
}

__global__ void __launch_bounds__(kLThreads)
logits_kl_backward_kernel(const LogitsView s, const LogitsView t, const void* mask, int mdt,
                          float inv_tau, const float* lse_s, const float* lse_t,
                          const float* dloss, void* ds) {
  const long long row = blockIdx.x;
  const bool on = !mask || mask_elem(mask, row, mdt);
  const size_t as = row_at(s, row), at = row_at(t, row), out = (size_t)row * s.V;
  const float g = (dloss ? *dloss : 1.f) * inv_tau, zs = lse_s[row], zt = lse_t[row];
  for (long long c = threadIdx.x; c < s.V; c += kLThreads) {
    float d = 0.f;
    if (on)
      d = g * (expf(fmaf(logit(s, as + c), inv_tau, -zs)) -
               expf(fmaf(logit(t, at + c), inv_tau, -zt)));
    put_logit(ds, out + c, s.dtype, d);
  }
}

}  // namespace

cudaError_t launch_token_logprobs(const LogitsView& x, long long rows, const int64_t* targets,
                                  int64_t ignore, int top_k, float* logprob, float* entropy,
                                  float* lse, float* top_v, int64_t* top_i, cudaStream_t st) {
  token_logprobs_kernel<<<(int)rows, kLThreads, 0, st>>>(x, targets, ignore, top_k, logprob,
                                                         entropy, lse, top_v, top_i);
  return cudaGetLastError();
}

cudaError_t launch_token_logprobs_backward(const LogitsView& x, long long rows,
                                           const int64_t* targets, int64_t ignore,
                                           const float* lse, const float* entropy,
                                           const float* g_lp, const float* g_en, void* dx,
                                           cudaStream_t st) {
  token_logprobs_backward_kernel<<<(int)rows, kLThreads, 0, st>>>(x, targets, ignore, lse, entropy,
                                                                  g_lp, g_en, dx);
  return cudaGetLastError();
}

cudaError_t launch_logits_kl_forward(const LogitsView& s, const LogitsView& t, long long rows,
                                     const void* mask, int mdt, float inv_tau, float* lse_s,
                                     float* lse_t, float* row_kl, float* loss, cudaStream_t st) {
  logits_kl_forward_kernel<<<(int)rows, kLThreads, 0, st>>>(s, t, mask, mdt, inv_tau, lse_s, lse_t,
                                                            row_kl);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess ? e : launch_reduce_partials(row_kl, (int)rows, loss, st);
}

cudaError_t launch_logits_kl_backward(const LogitsView& s, const LogitsView& t, long long rows,
                                      const void* mask, int mdt, float inv_tau,
                                      const float* lse_s, const float* lse_t, const float* dloss,
                                      void* ds, cudaStream_t st) {
  logits_kl_backward_kernel<<<(int)rows, kLThreads, 0, st>>>(s, t, mask, mdt, inv_tau, lse_s,
                                                             lse_t, dloss, ds);
  return cudaGetLastError();
}

}  // namespace lkl
