// CUDA-core attention, forward and recomputing backward: every head dim of the
// set and any layout.  The tensor-core kernels take the shapes that they cover;
// these take the rest (head dim 256, strides or pointers that TMA cannot read).
//
// Tiling: a 256-thread block owns 32 rows and walks 32-row tiles of the other
// side.  Eight neighbouring lanes share a row: thread t has row t / 8, the
// scores of columns t % 8 + 8 k and the features t % 8 + 8 m of that row's
// accumulators.  Rows that the mask removes are read as zeros, so that what
// they hold reaches no product.
#include <math_constants.h>

#include "lkl_attn.cuh"

namespace lkl {
namespace {

constexpr int kABM = 32;
constexpr int kAThreads = 256;

__device__ __forceinline__ void store_elem(void* base, size_t idx, int dtype, float v) {
  if (dtype == LKL_BF16) reinterpret_cast<__nv_bfloat16*>(base)[idx] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(base)[idx] = __float2half_rn(v);
}

// Rows [r0, r0 + 32) of head h of a [B, H, T, D] tensor into fp32 shared
// memory [32][D + 1]; zeros past T and where the mask removes the token.
template <int D>
__device__ __forceinline__ void attn_load_tile(float* dst, const void* src,
                                               const TensorStrides& s, int b, int h, int r0,
                                               int T, int dtype, const uint32_t* bits) {
  const int words = (T + 31) >> 5;
  const size_t base = (size_t)b * s.b + (size_t)h * s.h;
  for (int e = threadIdx.x; e < kABM * D; e += kAThreads) {
    const int r = e / D, d = e % D;
    float v = 0.f;
    if (r0 + r < T && token_valid(bits, words, b, r0 + r))
      v = load_elem(src, base + (size_t)(r0 + r) * s.t + d, dtype);
    dst[r * (D + 1) + d] = v;
  }
}

template <int D>
__device__ __forceinline__ float attn_dot(const float* a, const float* b) {
  float x = 0.f, y = 0.f;
#pragma unroll 8
  for (int d = 0; d < D; d += 2) {
    x = fmaf(a[d], b[d], x);
    y = fmaf(a[d + 1], b[d + 1], y);
  }
  return x + y;
}

__device__ __forceinline__ float max8(float v) {
  for (int o = 4; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float sum8(float v) {
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One pass over the key tiles with the running maximum and sum of the softmax.
template <int D>
__global__ void __launch_bounds__(kAThreads)
attn_generic_forward_kernel(const AttnProblem p, const AttnTensors a,
                            const uint32_t* __restrict__ bits) {
  extern __shared__ float smem[];
  float* sQ = smem;
  float* sK = sQ + kABM * (D + 1);
  float* sV = sK + kABM * (D + 1);
  float* sP = sV + kABM * (D + 1);  // [32][33]
  const int n_t = (p.T + kABM - 1) / kABM, words = (p.T + 31) >> 5;
  const int bh = blockIdx.x / n_t, mt = n_t - 1 - blockIdx.x % n_t;
  const int b = bh / p.Hq, h = bh % p.Hq, g = h / (p.Hq / p.Hkv);
  const int r = threadIdx.x >> 3, sub = threadIdx.x & 7, i = mt * kABM + r;
  const bool row = i < p.T && token_valid(bits, words, b, i);
  attn_load_tile<D>(sQ, a.q, a.sq, b, h, mt * kABM, p.T, p.dtype, bits);
  float m = -CUDART_INF_F, l = 0.f, o[D / 8] = {};
  const int n_j = p.causal ? mt + 1 : n_t;
  for (int j = 0; j < n_j; ++j) {
    __syncthreads();
    attn_load_tile<D>(sK, a.k, a.sk, b, g, j * kABM, p.T, p.dtype, bits);
    attn_load_tile<D>(sV, a.v, a.sv, b, g, j * kABM, p.T, p.dtype, bits);
    __syncthreads();
    float s[4], mx = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = j * kABM + sub + 8 * k;
      const bool ok = row && c < p.T && (!p.causal || c <= i) && token_valid(bits, words, b, c);
      s[k] = ok ? attn_dot<D>(sQ + r * (D + 1), sK + (sub + 8 * k) * (D + 1)) * p.sc * kLog2e
                : -CUDART_INF_F;
      mx = fmaxf(mx, s[k]);
    }
    const float m_new = fmaxf(m, max8(mx));
    const float ref = m_new == -CUDART_INF_F ? 0.f : m_new;  // nothing valid so far
    const float f = exp2f(m - ref);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float e = exp2f(s[k] - ref);
      sum += e;
      sP[r * 33 + sub + 8 * k] = e;
    }
    l = l * f + sum8(sum);
    m = m_new;
    __syncwarp();
#pragma unroll
    for (int x = 0; x < D / 8; ++x) o[x] *= f;
    for (int c = 0; c < kABM; ++c) {
      const float e = sP[r * 33 + c];
#pragma unroll
      for (int x = 0; x < D / 8; ++x) o[x] = fmaf(e, sV[c * (D + 1) + sub + 8 * x], o[x]);
    }
    __syncwarp();
  }
  if (i >= p.T) return;
  const size_t at = (size_t)b * a.so.b + (size_t)h * a.so.h + (size_t)i * a.so.t;
  const float inv = row ? 1.f / l : 0.f;
#pragma unroll
  for (int x = 0; x < D / 8; ++x)
    store_elem(a.out, at + sub + 8 * x, p.dtype, row ? o[x] * inv : 0.f);
  if (sub == 0) a.lse[(size_t)bh * p.T + i] = row ? (m + log2f(l)) * kLn2 : 0.f;
}

// rows[b, h, i] = (-lse_i log2(e), delta_i), delta_i = dout_i . out_i.  One
// warp a row.
__global__ void attn_delta_kernel(const AttnProblem p, const AttnTensors a,
                                  const uint32_t* __restrict__ bits, float2* __restrict__ rows) {
  const long long n = (long long)p.B * p.Hq * p.T;
  const int words = (p.T + 31) >> 5, lane = threadIdx.x & 31;
  for (long long x = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5; x < n;
       x += ((long long)gridDim.x * blockDim.x) >> 5) {
    const int i = (int)(x % p.T), bh = (int)(x / p.T), b = bh / p.Hq, h = bh % p.Hq;
    if (!token_valid(bits, words, b, i)) {
      if (lane == 0) rows[x] = make_float2(-CUDART_INF_F, 0.f);
      continue;
    }
    const size_t o = (size_t)b * a.so.b + (size_t)h * a.so.h + (size_t)i * a.so.t;
    const size_t d = (size_t)b * a.sdo.b + (size_t)h * a.sdo.h + (size_t)i * a.sdo.t;
    float s = 0.f;
    for (int c = lane; c < p.D; c += 32)
      s = fmaf(load_elem(a.out, o + c, p.dtype), load_elem(a.dout, d + c, p.dtype), s);
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    if (lane == 0) rows[x] = make_float2(-a.lse[x] * kLog2e, s);
  }
}

// Rows token(r0 .. r0 + 32) of head h, zeros where that is -1.
template <int D, typename Token>
__device__ __forceinline__ void attn_load_tokens(float* dst, const void* src,
                                                 const TensorStrides& s, int b, int h, int r0,
                                                 Token token, int dtype) {
  const size_t base = (size_t)b * s.b + (size_t)h * s.h;
  for (int e = threadIdx.x; e < kABM * D; e += kAThreads) {
    const int r = e / D, d = e % D, t = token(r0 + r);
    dst[r * (D + 1) + d] = t >= 0 ? load_elem(src, base + (size_t)t * s.t + d, dtype) : 0.f;
  }
}

// delta_i = sum_j P_ij (dout_i . v_j) for rows that see few keys; a block takes 32.  Rows
// and keys go by position or, where exact_delta_ranked() says so, by their rank.
template <int D>
__global__ void __launch_bounds__(kAThreads)
attn_exact_delta_kernel(const AttnProblem p, const AttnTensors a,
                        const uint32_t* __restrict__ bits, float2* __restrict__ rows,
                        int n_rt) {
  __shared__ int pos[kExactDeltaKeys], sums[8];
  extern __shared__ float smem[];
  float* sQ = smem;
  float* sG = sQ + kABM * (D + 1);
  float* sK = sG + kABM * (D + 1);
  float* sV = sK + kABM * (D + 1);
  const int bh = blockIdx.x / n_rt, mt = blockIdx.x % n_rt;   // n_rt: row tiles to take
  const int b = bh / p.Hq, h = bh % p.Hq, g = h / (p.Hq / p.Hkv), words = (p.T + 31) >> 5;
  const bool ranked = exact_delta_ranked(p, bits);
  const int n = ranked ? few_key_tokens(bits, p, b, pos, sums) : min(p.T, kExactDeltaKeys);
  if (mt * kABM >= n) return;
  auto token = [&](int r) {   // -1: none there, or one that the mask removes
    if (r >= n) return -1;
    return ranked ? pos[r] : token_valid(bits, words, b, r) ? r : -1;
  };
  const int r = threadIdx.x >> 3, sub = threadIdx.x & 7, rank = mt * kABM + r, i = token(rank);
  const float z = i >= 0 ? -a.lse[(size_t)bh * p.T + i] * kLog2e : -CUDART_INF_F;
  attn_load_tokens<D>(sQ, a.q, a.sq, b, h, mt * kABM, token, p.dtype);
  attn_load_tokens<D>(sG, a.dout, a.sdo, b, h, mt * kABM, token, p.dtype);
  float delta = 0.f;
  const int n_j = p.causal ? mt + 1 : (n + kABM - 1) / kABM;
  for (int j = 0; j < n_j; ++j) {
    __syncthreads();
    attn_load_tokens<D>(sK, a.k, a.sk, b, g, j * kABM, token, p.dtype);
    attn_load_tokens<D>(sV, a.v, a.sv, b, g, j * kABM, token, p.dtype);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int cl = sub + 8 * k, c = j * kABM + cl;
      if (i >= 0 && (!p.causal || c <= rank) && token(c) >= 0) {
        const float s = attn_dot<D>(sQ + r * (D + 1), sK + cl * (D + 1)) * p.sc * kLog2e;
        delta = fmaf(exp2f(s + z), attn_dot<D>(sG + r * (D + 1), sV + cl * (D + 1)), delta);
      }
    }
  }
  delta = sum8(delta);
  // by position, a removed token's row is written too
  const int at = ranked ? i : rank < n ? rank : -1;
  if (sub == 0 && at >= 0) rows[(size_t)bh * p.T + at] = make_float2(z, delta);
}

// dq_i = sc sum_j P_ij (dout_i . v_j - delta_i) k_j; query rows are stationary.
template <int D>
__global__ void __launch_bounds__(kAThreads)
attn_generic_dq_kernel(const AttnProblem p, const AttnTensors a,
                       const uint32_t* __restrict__ bits, const float2* __restrict__ rows) {
  extern __shared__ float smem[];
  float* sQ = smem;
  float* sG = sQ + kABM * (D + 1);
  float* sK = sG + kABM * (D + 1);
  float* sV = sK + kABM * (D + 1);
  float* sS = sV + kABM * (D + 1);  // dS [32][33]
  const int n_t = (p.T + kABM - 1) / kABM, words = (p.T + 31) >> 5;
  const int bh = blockIdx.x / n_t, mt = n_t - 1 - blockIdx.x % n_t;
  const int b = bh / p.Hq, h = bh % p.Hq, g = h / (p.Hq / p.Hkv);
  const int r = threadIdx.x >> 3, sub = threadIdx.x & 7, i = mt * kABM + r;
  const float2 st = i < p.T ? rows[(size_t)bh * p.T + i] : make_float2(-CUDART_INF_F, 0.f);
  const bool row = st.x != -CUDART_INF_F;
  attn_load_tile<D>(sQ, a.q, a.sq, b, h, mt * kABM, p.T, p.dtype, bits);
  attn_load_tile<D>(sG, a.dout, a.sdo, b, h, mt * kABM, p.T, p.dtype, bits);
  float acc[D / 8] = {};
  const int n_j = p.causal ? mt + 1 : n_t;
  for (int j = 0; j < n_j; ++j) {
    __syncthreads();
    attn_load_tile<D>(sK, a.k, a.sk, b, g, j * kABM, p.T, p.dtype, bits);
    attn_load_tile<D>(sV, a.v, a.sv, b, g, j * kABM, p.T, p.dtype, bits);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int cl = sub + 8 * k, c = j * kABM + cl;
      const bool ok = row && c < p.T && (!p.causal || c <= i) && token_valid(bits, words, b, c);
      float ds = 0.f;
      if (ok) {
        const float s = attn_dot<D>(sQ + r * (D + 1), sK + cl * (D + 1)) * p.sc * kLog2e;
        ds = exp2f(s + st.x) * (attn_dot<D>(sG + r * (D + 1), sV + cl * (D + 1)) - st.y);
      }
      sS[r * 33 + cl] = ds;
    }
    __syncwarp();
    for (int c = 0; c < kABM; ++c) {
      const float ds = sS[r * 33 + c];
#pragma unroll
      for (int x = 0; x < D / 8; ++x) acc[x] = fmaf(ds, sK[c * (D + 1) + sub + 8 * x], acc[x]);
    }
    __syncwarp();
  }
  if (i >= p.T) return;
  const size_t at = (size_t)b * a.sdq.b + (size_t)h * a.sdq.h + (size_t)i * a.sdq.t;
#pragma unroll
  for (int x = 0; x < D / 8; ++x)
    store_elem(a.dq, at + sub + 8 * x, p.dtype, row ? acc[x] * p.sc : 0.f);
}

// dk_j = sc sum_i dS_ij q_i and dv_j = sum_i P_ij dout_i over the query heads
// of the kv head; key rows are stationary, so each gradient row has one writer.
template <int D>
__global__ void __launch_bounds__(kAThreads)
attn_generic_dkv_kernel(const AttnProblem p, const AttnTensors a,
                        const uint32_t* __restrict__ bits, const float2* __restrict__ rows) {
  extern __shared__ float smem[];
  float* sQ = smem;
  float* sG = sQ + kABM * (D + 1);
  float* sK = sG + kABM * (D + 1);
  float* sV = sK + kABM * (D + 1);
  float* sP = sV + kABM * (D + 1);  // P^T [32 keys][33]
  float* sS = sP + kABM * 33;       // dS^T
  const int n_t = (p.T + kABM - 1) / kABM, words = (p.T + 31) >> 5, G = p.Hq / p.Hkv;
  const int bg = blockIdx.x / n_t, jt = blockIdx.x % n_t;
  const int b = bg / p.Hkv, g = bg % p.Hkv;
  const int r = threadIdx.x >> 3, sub = threadIdx.x & 7, j = jt * kABM + r;
  const bool key = j < p.T && token_valid(bits, words, b, j);
  attn_load_tile<D>(sK, a.k, a.sk, b, g, jt * kABM, p.T, p.dtype, bits);
  attn_load_tile<D>(sV, a.v, a.sv, b, g, jt * kABM, p.T, p.dtype, bits);
  float dk[D / 8] = {}, dv[D / 8] = {};
  for (int h = g * G; h < (g + 1) * G; ++h)
    for (int it = p.causal ? jt : 0; it < n_t; ++it) {
      __syncthreads();
      attn_load_tile<D>(sQ, a.q, a.sq, b, h, it * kABM, p.T, p.dtype, bits);
      attn_load_tile<D>(sG, a.dout, a.sdo, b, h, it * kABM, p.T, p.dtype, bits);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int cl = sub + 8 * k, i = it * kABM + cl;
        float pr = 0.f, ds = 0.f;
        if (key && i < p.T && (!p.causal || j <= i)) {
          const float2 st = rows[((size_t)b * p.Hq + h) * p.T + i];
          const float s = attn_dot<D>(sQ + cl * (D + 1), sK + r * (D + 1)) * p.sc * kLog2e;
          pr = exp2f(s + st.x);
          ds = pr * (attn_dot<D>(sG + cl * (D + 1), sV + r * (D + 1)) - st.y);
        }
        sP[r * 33 + cl] = pr;
        sS[r * 33 + cl] = ds;
      }
      __syncwarp();
      for (int c = 0; c < kABM; ++c) {
        const float pr = sP[r * 33 + c], ds = sS[r * 33 + c];
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          dv[x] = fmaf(pr, sG[c * (D + 1) + sub + 8 * x], dv[x]);
          dk[x] = fmaf(ds, sQ[c * (D + 1) + sub + 8 * x], dk[x]);
        }
      }
      __syncwarp();
    }
  if (j >= p.T) return;
  const size_t ak = (size_t)b * a.sdk.b + (size_t)g * a.sdk.h + (size_t)j * a.sdk.t;
  const size_t av = (size_t)b * a.sdv.b + (size_t)g * a.sdv.h + (size_t)j * a.sdv.t;
#pragma unroll
  for (int x = 0; x < D / 8; ++x) {
    store_elem(a.dk, ak + sub + 8 * x, p.dtype, key ? dk[x] * p.sc : 0.f);
    store_elem(a.dv, av + sub + 8 * x, p.dtype, key ? dv[x] : 0.f);
  }
}

template <typename K, typename... A>
cudaError_t attn_launch(K kernel, long long grid, int smem, cudaStream_t st, A... args) {
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  if (smem > (48 << 10)) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  kernel<<<(int)grid, kAThreads, smem, st>>>(args...);
  return cudaGetLastError();
}

template <int D>
cudaError_t attn_generic_fwd(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                             cudaStream_t st) {
  const int n_t = (p.T + kABM - 1) / kABM;
  return attn_launch(attn_generic_forward_kernel<D>, (long long)p.B * p.Hq * n_t,
                     (3 * kABM * (D + 1) + kABM * 33) * 4, st, p, t, bits);
}

template <int D>
cudaError_t attn_exact_delta(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                             float2* rows, cudaStream_t st) {
  const int n = p.T < kExactDeltaKeys ? p.T : kExactDeltaKeys, n_rt = (n + kABM - 1) / kABM;
  return attn_launch(attn_exact_delta_kernel<D>, (long long)p.B * p.Hq * n_rt,
                     4 * kABM * (D + 1) * 4, st, p, t, bits, rows, n_rt);
}

template <int D>
cudaError_t attn_generic_bwd(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                             const float2* rows, cudaStream_t st) {
  const int n_t = (p.T + kABM - 1) / kABM;
  const cudaError_t e = attn_launch(attn_generic_dq_kernel<D>, (long long)p.B * p.Hq * n_t,
                                    (4 * kABM * (D + 1) + kABM * 33) * 4, st, p, t, bits, rows);
  if (e != cudaSuccess) return e;
  return attn_launch(attn_generic_dkv_kernel<D>, (long long)p.B * p.Hkv * n_t,
                     (4 * kABM * (D + 1) + 2 * kABM * 33) * 4, st, p, t, bits, rows);
}

}  // namespace

cudaError_t launch_attn_generic_forward(const AttnProblem& p, const AttnTensors& t,
                                        const uint32_t* bits, cudaStream_t st) {
  switch (p.D) {
    case 8: return attn_generic_fwd<8>(p, t, bits, st);
    case 16: return attn_generic_fwd<16>(p, t, bits, st);
    case 32: return attn_generic_fwd<32>(p, t, bits, st);
    case 64: return attn_generic_fwd<64>(p, t, bits, st);
    case 128: return attn_generic_fwd<128>(p, t, bits, st);
    default: return attn_generic_fwd<256>(p, t, bits, st);
  }
}

cudaError_t launch_attn_exact_delta(const AttnProblem& p, const AttnTensors& t,
                                    const uint32_t* bits, float2* rows, cudaStream_t st) {
  switch (p.D) {
    case 8: return attn_exact_delta<8>(p, t, bits, rows, st);
    case 16: return attn_exact_delta<16>(p, t, bits, rows, st);
    case 32: return attn_exact_delta<32>(p, t, bits, rows, st);
    case 64: return attn_exact_delta<64>(p, t, bits, rows, st);
    case 128: return attn_exact_delta<128>(p, t, bits, rows, st);
    default: return attn_exact_delta<256>(p, t, bits, rows, st);
  }
}

cudaError_t launch_attn_delta(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                              float2* rows, cudaStream_t st) {
  const long long n = (long long)p.B * p.Hq * p.T;
  const int grid = (int)((n + 7) / 8 < 65536 ? (n + 7) / 8 : 65536);
  attn_delta_kernel<<<grid, 256, 0, st>>>(p, t, bits, rows);
  return cudaGetLastError();
}

cudaError_t launch_attn_generic_backward(const AttnProblem& p, const AttnTensors& t,
                                         const uint32_t* bits, const float2* rows,
                                         cudaStream_t st) {
  switch (p.D) {
    case 8: return attn_generic_bwd<8>(p, t, bits, rows, st);
    case 16: return attn_generic_bwd<16>(p, t, bits, rows, st);
    case 32: return attn_generic_bwd<32>(p, t, bits, rows, st);
    case 64: return attn_generic_bwd<64>(p, t, bits, rows, st);
    case 128: return attn_generic_bwd<128>(p, t, bits, rows, st);
    default: return attn_generic_bwd<256>(p, t, bits, rows, st);
  }
}

}  // namespace lkl
