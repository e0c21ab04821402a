// Operators over rows of logits: log probabilities of given tokens (with
// entropy and top alternatives) and the KL between two models' rows, each with
// its gradient.
//
// All four kernels are bound by HBM: a forward reads each logit once, a backward
// reads it once more and writes its gradient.  The forwards keep, per thread, a
// running maximum m and sums relative to it,
//   l = sum e^(x - m),  a = sum e^(x - m) (x - m)     (token: entropy = log l - a / l)
//   A = sum e^(t - m_t) (t - s)                       (KL = A / l_t - (lse_t - lse_s)),
// over batches of four 16-byte loads, and join threads, warps and blocks in a
// fixed order.  Differences from m are taken before they are scaled: the
// exponent of a likely token keeps all its bits, whatever the logits' offset.
//
// A row belongs to a cluster of 1, 2, 4 or 8 blocks that join their sums
// through distributed shared memory, so that few rows still fill the GPU and
// every call is one launch (and one more for the loss of the KL).
#include <cooperative_groups.h>
#include <math_constants.h>

#include "lkl_logits.cuh"

namespace lkl {
namespace {

namespace cg = cooperative_groups;

constexpr int kLThreads = 256;
constexpr int kLWarps = kLThreads / 32;
constexpr int kLBatch = 4;          // 16-byte loads in flight a thread and stream
constexpr int kMaxCluster = 8;
constexpr uint32_t kAll = 0xffffffffu;

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// ---------------------------------------------------------------- rows as vectors
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    return __uint_as_float(reinterpret_cast<const uint32_t*>(&v)[e]);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void put(uint4& v, int e, float x) {
    reinterpret_cast<uint32_t*>(&v)[e] = __float_as_uint(x);
  }
  static __device__ __forceinline__ void put1(float* p, float x) { *p = x; }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&v)[e >> 1];
    return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) {
    return __bfloat162float(*p);
  }
  static __device__ __forceinline__ void put(uint4& v, int e, float x) {
    reinterpret_cast<__nv_bfloat16*>(&v)[e] = __float2bfloat16_rn(x);
  }
  static __device__ __forceinline__ void put1(__nv_bfloat16* p, float x) {
    *p = __float2bfloat16_rn(x);
  }
};
template <>
struct Elem<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    return __half2float(reinterpret_cast<const __half*>(&v)[e]);
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void put(uint4& v, int e, float x) {
    reinterpret_cast<__half*>(&v)[e] = __float2half_rn(x);
  }
  static __device__ __forceinline__ void put1(__half* p, float x) { *p = __float2half_rn(x); }
};

template <typename T>
__device__ __forceinline__ const T* row_ptr(const LogitsView& x, long long row) {
  return static_cast<const T*>(x.x) + (row / x.T) * x.sb + (row % x.T) * x.st;
}

// A row of V elements: `lead` before the first 16-byte boundary, then nv
// vectors, then `tail`.  The ends are taken one element a thread.
template <typename T>
struct RowCut {
  int lead, nv, tail;
  __device__ __forceinline__ RowCut(const T* row, long long V) {
    constexpr int N = Elem<T>::N;
    const int off = (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    lead = (int)min((long long)(off ? N - off : 0), V);
    nv = (int)((V - lead) / N);
    tail = (int)(V - lead - (long long)nv * N);
  }
  // element of the row that thread k takes of its ends, or -1
  __device__ __forceinline__ long long end_elem(int k, long long V) const {
    if (k < lead) return k;
    return k - lead < tail ? V - tail + (k - lead) : -1;
  }
};

// The 16 bytes at p: one load, or element by element where p has another offset
// from 16 bytes than the row that was cut.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* p, bool vec) {
  if (vec) return __ldg(reinterpret_cast<const uint4*>(p));
  uint4 v;
#pragma unroll
  for (int e = 0; e < Elem<T>::N; ++e) reinterpret_cast<T*>(&v)[e] = p[e];
  return v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const uint4& v, bool vec) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < Elem<T>::N; ++e) p[e] = reinterpret_cast<const T*>(&v)[e];
}
template <typename T>
__device__ __forceinline__ bool same_offset(const T* a, const T* b) {
  return (reinterpret_cast<uintptr_t>(a) - reinterpret_cast<uintptr_t>(b)) % 16 == 0;
}

// ---------------------------------------------------------------- statistics
// Running sums relative to a maximum; c scales differences to exponents of two.
// Nothing above -inf so far: m = -inf, l = a = 0.
struct TokenStat {
  float m, l, a;
  __device__ __forceinline__ void move(float to, float c) {   // to >= m, to > -inf
    const float d = m - to, f = ex2(d * c);
    a = f == 0.f ? 0.f : f * fmaf(l, d, a);
    l *= f;
    m = to;
  }
  __device__ __forceinline__ void join(TokenStat o, float c) {
    const float to = max_nan(m, o.m);
    if (to == -CUDART_INF_F) return;
    if (m == -CUDART_INF_F) m = to;
    else move(to, c);
    if (o.m == -CUDART_INF_F) o.m = to;
    else o.move(to, c);
    l += o.l;
    a += o.a;
  }
};
struct KLStat {
  float ms, ls, mt, lt, a;
  __device__ __forceinline__ void move(float ns, float nt, float c) {
    if (ns != -CUDART_INF_F) {
      ls *= ms == -CUDART_INF_F ? 1.f : ex2((ms - ns) * c);
      ms = ns;
    }
    if (nt != -CUDART_INF_F) {
      const float f = mt == -CUDART_INF_F ? 1.f : ex2((mt - nt) * c);
      lt *= f;
      // a may be +inf, where the student excludes what the teacher gives
      a = f == 0.f && !isnan(a) ? 0.f : a * f;
      mt = nt;
    }
  }
  __device__ __forceinline__ void join(KLStat o, float c) {
    const float ns = max_nan(ms, o.ms), nt = max_nan(mt, o.mt);
    move(ns, nt, c);
    o.move(ns, nt, c);
    ls += o.ls;
    lt += o.lt;
    a += o.a;
  }
};

template <typename S>
__device__ __forceinline__ S shfl_stat(const S& s, int lane_xor) {
  S o;
  const float* a = reinterpret_cast<const float*>(&s);
  float* b = reinterpret_cast<float*>(&o);
#pragma unroll
  for (int k = 0; k < (int)(sizeof(S) / 4); ++k) b[k] = __shfl_xor_sync(kAll, a[k], lane_xor);
  return o;
}

// Joins the statistics of a cluster's threads; every thread gets the result.
// `shared`: kLWarps + 1 entries of this block.
template <typename S>
__device__ __forceinline__ S join_all(S s, S* shared, float c) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const S other = shfl_stat(s, o);
    // the same operand order in both lanes: the same bits
    if (lane & o) {
      S t = other;
      t.join(s, c);
      s = t;
    } else {
      s.join(other, c);
    }
  }
  if (lane == 0) shared[warp] = s;
  __syncthreads();
  s = shared[0];
#pragma unroll
  for (int w = 1; w < kLWarps; ++w) s.join(shared[w], c);
  cg::cluster_group cluster = cg::this_cluster();
  const int n = (int)cluster.num_blocks();
  if (n > 1) {
    if (threadIdx.x == 0) shared[kLWarps] = s;
    cluster.sync();
    s = *cluster.map_shared_rank(shared + kLWarps, 0);
    for (int r = 1; r < n; ++r) s.join(*cluster.map_shared_rank(shared + kLWarps, r), c);
    cluster.sync();   // the entries are free, and no block has left
  } else {
    __syncthreads();
  }
  return s;
}

// ---------------------------------------------------------------- top alternatives
// An element as one number: a larger logit first, then the lower index (0: none).
__device__ __forceinline__ uint64_t top_key(float v, uint32_t idx) {
  const uint32_t u = __float_as_uint(v + 0.f);   // -0 and 0 are equal
  const uint32_t ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)ord << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float top_value(uint64_t key) {
  const uint32_t ord = (uint32_t)(key >> 32);
  return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7fffffffu) : ~ord);
}

// The 32 best elements a warp has seen, lane k holding the k-th.
struct TopList {
  uint64_t key;
  __device__ __forceinline__ void insert(uint64_t x, int lane) {   // x: the same in every lane
    const uint64_t prev = __shfl_up_sync(kAll, key, 1);
    if (x > key) key = lane > 0 && x > prev ? prev : x;
  }
  // Value that an element has to reach to be among the best k (-inf: any does).
  __device__ __forceinline__ float threshold(int k) const {
    const uint64_t last = __shfl_sync(kAll, key, k - 1);
    return last ? top_value(last) : -CUDART_INF_F;
  }
};

// k-th largest of the lanes' values (NaN counts as -inf).
__device__ __forceinline__ float kth_of_lanes(float v, int k, int lane) {
  int rank = 0;
  if (isnan(v)) v = -CUDART_INF_F;
#pragma unroll
  for (int o = 0; o < 32; ++o) {
    const float w = __shfl_sync(kAll, v, o);
    rank += w > v || (w == v && o < lane);
  }
  return __shfl_sync(kAll, v, __ffs(__ballot_sync(kAll, rank == k - 1)) - 1);
}

// ---------------------------------------------------------------- token forward
// Sums over this block's share of the row.  GUARD: -inf logits add exactly 0 to
// a, where the plain form gives 0 x -inf = NaN; only rows that met one need it.
template <typename T, bool GUARD, bool TOP>
__device__ __forceinline__ TokenStat token_pass(const T* row, long long V, int top_k, TopList& top,
                                                volatile float* thr) {
  constexpr int N = Elem<T>::N;
  const RowCut<T> cut(row, V);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), n_blocks = (int)cluster.num_blocks();
  const int v0 = (int)((long long)cut.nv * rank / n_blocks);
  const int v1 = (int)((long long)cut.nv * (rank + 1) / n_blocks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TokenStat s{-CUDART_INF_F, 0.f, 0.f};
  bool fresh = true;
  auto add = [&](const float* x, int n) {   // n <= kLBatch * N values, unrolled by the caller
    float bm = x[0];
#pragma unroll
    for (int e = 1; e < n; ++e) bm = max_nan(bm, x[e]);
    const float to = max_nan(s.m, bm);
    if (to == -CUDART_INF_F) return bm;
    if (!(to == s.m)) {
      if (s.m == -CUDART_INF_F) s.m = to;
      else s.move(to, kLog2e);
    }
    float l0 = 0.f, l1 = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int e = 0; e < n; e += 2) {
      float d0 = x[e] - s.m, d1 = e + 1 < n ? x[e + 1] - s.m : -CUDART_INF_F;
      if (GUARD || n == 1) {
        d0 = max_nan(d0, -200.f);   // e^-200 is 0 in fp32
        d1 = max_nan(d1, -200.f);
      }
      const float e0 = ex2(d0 * kLog2e), e1 = ex2(d1 * kLog2e);
      l0 += e0;
      l1 += e1;
      a0 = fmaf(e0, d0, a0);
      a1 = fmaf(e1, d1, a1);
    }
    s.l += l0 + l1;
    s.a += a0 + a1;
    return bm;
  };
  for (int v = v0 + threadIdx.x - lane; v < v1; v += kLBatch * kLThreads) {
    uint4 raw[kLBatch];
    bool in[kLBatch];
#pragma unroll
    for (int u = 0; u < kLBatch; ++u) {
      const int at = v + lane + u * kLThreads;
      in[u] = at < v1;
      if (in[u]) raw[u] = __ldg(reinterpret_cast<const uint4*>(row + cut.lead) + at);
    }
    float x[kLBatch * N];
    float bm = -CUDART_INF_F;
    if (in[kLBatch - 1]) {
#pragma unroll
      for (int e = 0; e < kLBatch * N; ++e) x[e] = Elem<T>::get(raw[e / N], e % N);
      bm = add(x, kLBatch * N);
    } else {
#pragma unroll
      for (int u = 0; u < kLBatch; ++u)
        if (in[u]) {
#pragma unroll
          for (int e = 0; e < N; ++e) x[u * N + e] = Elem<T>::get(raw[u], e);
          bm = max_nan(bm, add(x + u * N, N));
        }
    }
    if (TOP) {
      __syncwarp();
      float need = top.threshold(top_k);
#pragma unroll
      for (int w = 0; w < kLWarps; ++w) need = fmaxf(need, thr[w]);
      if (fresh) need = fmaxf(need, kth_of_lanes(in[0] ? bm : -CUDART_INF_F, top_k, lane));
      fresh = false;
      if (__any_sync(kAll, in[0] && !(bm < need))) {
#pragma unroll
        for (int e = 0; e < kLBatch * N; ++e) {
          uint32_t hit = __ballot_sync(kAll, in[e / N] && x[e] >= need);
          if (!hit) continue;
          while (hit) {
            const int from = __ffs(hit) - 1;
            hit &= hit - 1;
            const float best = __shfl_sync(kAll, x[e], from);
            const uint32_t idx =
                (uint32_t)(cut.lead + (v + from + (e / N) * kLThreads) * N + e % N);
            top.insert(top_key(best, idx), lane);
          }
          need = fmaxf(need, top.threshold(top_k));
        }
        if (lane == 0) thr[warp] = need;
      }
    }
  }
  if (rank == 0 && warp == 0) {   // at most 14 elements
    const long long c = cut.end_elem(lane, V);
    const float x = c >= 0 ? Elem<T>::one(row + c) : -CUDART_INF_F;
    add(&x, 1);
    if (TOP) {
      uint32_t hit = __ballot_sync(kAll, c >= 0 && !isnan(x));
      while (hit) {
        const int from = __ffs(hit) - 1;
        hit &= hit - 1;
        top.insert(top_key(__shfl_sync(kAll, x, from),
                           (uint32_t)__shfl_sync(kAll, (int)c, from)), lane);
      }
    }
  }
  return s;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kLThreads)
token_logprobs_kernel(const LogitsView view, const int64_t* __restrict__ targets, int64_t ignore,
                      int top_k, float* __restrict__ logprob, float* __restrict__ entropy,
                      float* __restrict__ lse_out, float* __restrict__ top_v,
                      int64_t* __restrict__ top_i) {
  __shared__ TokenStat stat[kLWarps + 1];
  __shared__ float thr[kLWarps];
  __shared__ uint64_t lists[TOP ? kLWarps : 1][32];
  cg::cluster_group cluster = cg::this_cluster();
  const int n = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long row = blockIdx.x / n;
  const T* x = row_ptr<T>(view, row);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TopList top{0};
  if (TOP) {
    if (lane == 0) thr[warp] = -CUDART_INF_F;
    __syncthreads();
  }
  TokenStat s = join_all(token_pass<T, false, TOP>(x, view.V, top_k, top, thr), stat, kLog2e);
  if (isnan(s.a) && !isnan(s.l) && s.l > 0.f) {   // the same in every thread of the cluster
    TopList none{0};
    s = join_all(token_pass<T, true, false>(x, view.V, 0, none, thr), stat, kLog2e);
  }
  const bool empty = s.m == -CUDART_INF_F;
  const float log_l = empty ? CUDART_NAN_F : logf(s.l);
  if (rank == 0 && threadIdx.x == 0) {
    const int64_t y = targets[row];
    float lp = CUDART_NAN_F;
    if (y == ignore) lp = 0.f;
    else if (y >= 0 && y < view.V) lp = (Elem<T>::one(x + y) - s.m) - log_l;
    logprob[row] = lp;
    entropy[row] = log_l - s.a / s.l;
    lse_out[row] = s.m + log_l;
  }
  if (TOP) {
    lists[warp][lane] = top.key;
    if (n > 1) cluster.sync();
    else __syncthreads();
    if (rank == 0 && warp == 0) {
      for (int w = 1; w < n * kLWarps; ++w) {
        const uint64_t* from = n > 1 ? cluster.map_shared_rank(&lists[w % kLWarps][0], w / kLWarps)
                                     : &lists[w][0];
        const uint64_t mine = lane < top_k ? from[lane] : 0;
        for (int k = 0; k < top_k; ++k) {   // sorted: the first that does not fit ends the list
          const uint64_t key = __shfl_sync(kAll, mine, k);
          if (key <= __shfl_sync(kAll, top.key, top_k - 1)) break;
          top.insert(key, lane);
        }
      }
      if (lane < top_k) {
        const long long idx = (uint32_t)~(uint32_t)top.key;
        top_v[row * top_k + lane] = top.key ? (top_value(top.key) - s.m) - log_l : CUDART_NAN_F;
        top_i[row * top_k + lane] = top.key ? idx : view.V - 1;   // a row of NaN
      }
    }
    if (n > 1) cluster.sync();   // the lists stay until they are read
  }
}

// ---------------------------------------------------------------- KL forward
template <typename T, bool GUARD>
__device__ __forceinline__ KLStat kl_pass(const T* s, const T* t, long long V, float c) {
  constexpr int N = Elem<T>::N;
  constexpr int U = 2;   // loads in flight a thread and stream
  const RowCut<T> cut(s, V);
  const bool vec = same_offset(s, t);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), n_blocks = (int)cluster.num_blocks();
  const int v0 = (int)((long long)cut.nv * rank / n_blocks);
  const int v1 = (int)((long long)cut.nv * (rank + 1) / n_blocks);
  KLStat st{-CUDART_INF_F, 0.f, -CUDART_INF_F, 0.f, 0.f};
  auto add = [&](const float* x, const float* y, int n) {
    float bs = x[0], bt = y[0];
#pragma unroll
    for (int e = 1; e < n; ++e) {
      bs = max_nan(bs, x[e]);
      bt = max_nan(bt, y[e]);
    }
    const float ns = max_nan(st.ms, bs), nt = max_nan(st.mt, bt);
    if (!(ns == st.ms && nt == st.mt)) st.move(ns, nt, c);
    const float ms = ns == -CUDART_INF_F ? 0.f : ns, mt = nt == -CUDART_INF_F ? 0.f : nt;
    float ls = 0.f, lt = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const float es = ex2((x[e] - ms) * c), et = ex2((y[e] - mt) * c);
      ls += es;
      lt += et;
      float d = y[e] - x[e];
      if (GUARD && et == 0.f) d = 0.f;
      if (e & 1) a1 = fmaf(et, d, a1);
      else a0 = fmaf(et, d, a0);
    }
    st.ls += ls;
    st.lt += lt;
    st.a += a0 + a1;
  };
  const uint4* sv = reinterpret_cast<const uint4*>(s + cut.lead);
  const T* tv = t + cut.lead;
  int v = v0 + threadIdx.x;
  for (; v + (U - 1) * kLThreads < v1; v += U * kLThreads) {
    uint4 a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = __ldg(sv + v + u * kLThreads);
      b[u] = load_vec(tv + (size_t)(v + u * kLThreads) * N, vec);
    }
    float x[U * N], y[U * N];
#pragma unroll
    for (int e = 0; e < U * N; ++e) {
      x[e] = Elem<T>::get(a[e / N], e % N);
      y[e] = Elem<T>::get(b[e / N], e % N);
    }
    add(x, y, U * N);
  }
  for (; v < v1; v += kLThreads) {
    const uint4 a = __ldg(sv + v), b = load_vec(tv + (size_t)v * N, vec);
    float x[N], y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[e] = Elem<T>::get(a, e);
      y[e] = Elem<T>::get(b, e);
    }
    add(x, y, N);
  }
  if (rank == 0) {
    const long long k = cut.end_elem(threadIdx.x, V);
    if (k >= 0) {
      const float x = Elem<T>::one(s + k), y = Elem<T>::one(t + k);
      add(&x, &y, 1);
    }
  }
  return st;
}

template <typename T>
__global__ void __launch_bounds__(kLThreads)
logits_kl_forward_kernel(const LogitsView sv, const LogitsView tv, const void* __restrict__ mask,
                         int mdt, float inv_tau, float* __restrict__ lse_s,
                         float* __restrict__ lse_t, float* __restrict__ row_kl) {
  __shared__ KLStat stat[kLWarps + 1];
  cg::cluster_group cluster = cg::this_cluster();
  const long long row = blockIdx.x / cluster.num_blocks();
  const bool first = cluster.block_rank() == 0 && threadIdx.x == 0;
  if (mask && !mask_elem(mask, row, mdt)) {   // the whole cluster
    if (first) lse_s[row] = lse_t[row] = row_kl[row] = 0.f;
    return;
  }
  const T *s = row_ptr<T>(sv, row), *t = row_ptr<T>(tv, row);
  const float c = inv_tau * kLog2e;
  KLStat k = join_all(kl_pass<T, false>(s, t, sv.V, c), stat, c);
  if (isnan(k.a) && !isnan(k.ls) && !isnan(k.lt))
    k = join_all(kl_pass<T, true>(s, t, sv.V, c), stat, c);
  if (first) {
    // in 64 bits: the loss is what is left of the difference of the two LSEs
    const bool none = k.ms == -CUDART_INF_F || k.mt == -CUDART_INF_F;
    const double zs = none ? CUDART_NAN : (double)k.ms * inv_tau + log((double)k.ls);
    const double zt = none ? CUDART_NAN : (double)k.mt * inv_tau + log((double)k.lt);
    lse_s[row] = (float)zs;
    lse_t[row] = (float)zt;
    row_kl[row] = (float)((double)k.a * inv_tau / k.lt + (zs - zt));
  }
}

// ---------------------------------------------------------------- gradients
// Elements [begin, end) of a row of V: a block's share, cut at vectors.
constexpr int kLShare = 4 * kLThreads;   // vectors a block

// d = f(x, element) over a row: vectors in this block's share, the ends by the first block.
template <typename T, typename Load, typename F>
__device__ __forceinline__ void map_row(const T* cut_by, T* out, long long V, int share, Load load,
                                        F f) {
  constexpr int N = Elem<T>::N;
  const RowCut<T> cut(cut_by, V);
  const bool vec = same_offset(cut_by, out);
  const int end = min(cut.nv, (share + 1) * kLShare);
  for (int v = share * kLShare + threadIdx.x; v < end; v += 2 * kLThreads) {
    const bool two = v + kLThreads < end;
    auto a = load(cut.lead + (long long)v * N);
    auto b = a;
    if (two) b = load(cut.lead + (long long)(v + kLThreads) * N);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && !two) break;
      const long long at = cut.lead + (long long)(v + h * kLThreads) * N;
      uint4 d;
#pragma unroll
      for (int e = 0; e < N; ++e) Elem<T>::put(d, e, f(h ? b : a, e, at + e));
      store_vec(out + at, d, vec);
    }
  }
  if (share == 0) {
    const long long k = cut.end_elem(threadIdx.x, V);
    if (k >= 0) Elem<T>::put1(out + k, f(load.one(k), 0, k));
  }
}

template <typename T>
struct LoadOne {
  const T* x;
  __device__ __forceinline__ uint4 operator()(long long at) const {
    return __ldg(reinterpret_cast<const uint4*>(x + at));
  }
  __device__ __forceinline__ uint4 one(long long at) const {
    uint4 v = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<T*>(&v) = x[at];
    return v;
  }
};

template <typename T>
__global__ void __launch_bounds__(kLThreads)
token_logprobs_backward_kernel(const LogitsView view, const int64_t* __restrict__ targets,
                               int64_t ignore, const float* __restrict__ lse,
                               const float* __restrict__ entropy, const float* __restrict__ g_lp,
                               const float* __restrict__ g_en, T* __restrict__ dx, int shares) {
  const long long row = blockIdx.x / shares;
  const T* x = row_ptr<T>(view, row);
  const int64_t y = targets[row];
  float g = g_lp && y != ignore ? g_lp[row] : 0.f;
  if (g_lp && y != ignore && (y < 0 || y >= view.V)) g = CUDART_NAN_F;
  const float h = g_en ? g_en[row] : 0.f, z = lse[row], H = entropy[row];
  // -p (g + h (log p + H)) + g at the target
  const float gh = fmaf(h, H, g);
  map_row<T>(x, dx + row * view.V, view.V, (int)(blockIdx.x % shares), LoadOne<T>{x},
             [&](const uint4& v, int e, long long at) {
               // e^-200 is 0; 0 x -inf would not be
               const float lp = max_nan(Elem<T>::get(v, e) - z, -200.f);
               const float d = -ex2(lp * kLog2e) * fmaf(h, lp, gh);
               return at == y ? d + g : d;
             });
}

struct Pair {
  uint4 s, t;
};
template <typename T>
struct LoadPair {
  const T *s, *t;
  bool vec;
  __device__ __forceinline__ Pair operator()(long long at) const {
    return Pair{__ldg(reinterpret_cast<const uint4*>(s + at)), load_vec(t + at, vec)};
  }
  __device__ __forceinline__ Pair one(long long at) const {
    return Pair{LoadOne<T>{s}.one(at), LoadOne<T>{t}.one(at)};
  }
};

template <typename T>
__global__ void __launch_bounds__(kLThreads)
logits_kl_backward_kernel(const LogitsView sv, const LogitsView tv, const void* __restrict__ mask,
                          int mdt, float inv_tau, const float* __restrict__ lse_s,
                          const float* __restrict__ lse_t, const float* __restrict__ dloss,
                          T* __restrict__ ds, int shares) {
  const long long row = blockIdx.x / shares;
  const int share = (int)(blockIdx.x % shares);
  const T *s = row_ptr<T>(sv, row), *t = row_ptr<T>(tv, row);
  T* out = ds + row * sv.V;
  if (mask && !mask_elem(mask, row, mdt)) {
    struct Nothing {
      __device__ __forceinline__ int operator()(long long) const { return 0; }
      __device__ __forceinline__ int one(long long) const { return 0; }
    };
    map_row<T>(out, out, sv.V, share, Nothing{}, [](int, int, long long) { return 0.f; });
    return;
  }
  const float g = (dloss ? *dloss : 1.f) * inv_tau, c = inv_tau * kLog2e;
  const float zs = lse_s[row] * kLog2e, zt = lse_t[row] * kLog2e;
  map_row<T>(s, out, sv.V, share, LoadPair<T>{s, t, same_offset(s, t)},
             [&](const Pair& v, int e, long long) {
               return g * (ex2(fmaf(Elem<T>::get(v.s, e), c, -zs)) -
                           ex2(fmaf(Elem<T>::get(v.t, e), c, -zt)));
             });
}

// ---------------------------------------------------------------- launches
// Blocks a row: enough that all rows together fill the GPU twice, as long as a
// block keeps 2048 elements (below that, joining costs more than it saves).
int cluster_of(long long rows, long long V) {
  int n = 1;
  while (n < kMaxCluster && rows * n < 296 && V / (2 * n) >= 2048) n *= 2;
  return n;
}

template <typename K, typename... A>
cudaError_t launch_rows(K kernel, long long rows, int cluster, cudaStream_t st, A... args) {
  if (rows * cluster > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kLThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// f(T{}) for the element type of `dtype`
template <typename F>
cudaError_t with_type(int dtype, F f) {
  if (dtype == LKL_F32) return f(float{});
  if (dtype == LKL_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

template <typename T>
int shares_of(long long V) {
  return (int)(V / Elem<T>::N / kLShare + 1);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogitsView& x, long long rows, const int64_t* targets,
                                  int64_t ignore, int top_k, float* logprob, float* entropy,
                                  float* lse, float* top_v, int64_t* top_i, cudaStream_t st) {
  const int n = cluster_of(rows, x.V);
  return with_type(x.dtype, [&](auto t) {
    using T = decltype(t);
    return launch_rows(top_k ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>,
                       rows, n, st, x, targets, ignore, top_k, logprob, entropy, lse, top_v,
                       top_i);
  });
}

cudaError_t launch_token_logprobs_backward(const LogitsView& x, long long rows,
                                           const int64_t* targets, int64_t ignore,
                                           const float* lse, const float* entropy,
                                           const float* g_lp, const float* g_en, void* dx,
                                           cudaStream_t st) {
  return with_type(x.dtype, [&](auto t) {
    using T = decltype(t);
    const int shares = shares_of<T>(x.V);
    return launch_rows(token_logprobs_backward_kernel<T>, rows * shares, 1, st, x, targets, ignore,
                       lse, entropy, g_lp, g_en, static_cast<T*>(dx), shares);
  });
}

cudaError_t launch_logits_kl_forward(const LogitsView& s, const LogitsView& t, long long rows,
                                     const void* mask, int mdt, float inv_tau, float* lse_s,
                                     float* lse_t, float* row_kl, float* loss, cudaStream_t st) {
  const int n = cluster_of(rows, s.V);
  const cudaError_t e = with_type(s.dtype, [&](auto x) {
    return launch_rows(logits_kl_forward_kernel<decltype(x)>, rows, n, st, s, t, mask, mdt, inv_tau,
                       lse_s, lse_t, row_kl);
  });
  return e != cudaSuccess ? e : launch_reduce_partials(row_kl, (int)rows, loss, st);
}

cudaError_t launch_logits_kl_backward(const LogitsView& s, const LogitsView& t, long long rows,
                                      const void* mask, int mdt, float inv_tau,
                                      const float* lse_s, const float* lse_t, const float* dloss,
                                      void* ds, cudaStream_t st) {
  return with_type(s.dtype, [&](auto x) {
    using T = decltype(x);
    const int shares = shares_of<T>(s.V);
    return launch_rows(logits_kl_backward_kernel<T>, rows * shares, 1, st, s, t, mask, mdt, inv_tau,
                       lse_s, lse_t, dloss, static_cast<T*>(ds), shares);
  });
}

}  // namespace lkl
