// Operators over rows of logits: log probabilities of given tokens (with
// entropy and top alternatives) and the KL between two models' rows, each with
// its gradient.
//
// With many rows all four kernels are bound by HBM: a forward reads each logit once, a
// backward reads it once more and writes its gradient.  The forwards keep, per thread, a
// running maximum m and sums relative to it,
//   l = sum e^(x - m),  a = sum e^(x - m) (x - m)     (token: entropy = log l - a / l)
//   A = sum e^(t - m_t) ((t - m_t) - (s - m_s))       (KL = A / l_t + log l_s - log l_t),
// over batches of 16-byte loads, and join threads, warps and blocks in a fixed
// order: the maxima first, so that each thread rescales once.  Differences from m are
// taken before they are scaled: the exponent of a likely token keeps all its bits,
// whatever the logits' offset.  The backwards take p from the row's log-sum-exp.  An fp32
// number alone would leave 2^-24 of its size in p (0.6 10^-6 at 10, 6 10^-5 at 1000), so a
// forward hands over the rest of it as a second one, which costs a backward next to nothing
// (0 to 2%): the multiplication by log2(e) becomes a multiply-add.
//
// Measured at 16384 x 32000 bf16 (of 6561 GB/s, the copy rate): KL backward 6.4 TB/s, forward
// 6.0; token forward 5.9, backward 5.7 TB/s.  Blocks of 128 threads let ten rows of an SM
// overlap their ends, and 128 bytes in flight a thread fill HBM (64 bytes: 5.4 and 5.3;
// 256 threads and pairwise joins: 4.0 and 3.8; 64 threads: 3.8 and 3.7).  Fewer rows leave
// it idle at their ends: at 2004 x 50257 bf16 the KL takes 4.8 (forward) and 5.8 TB/s, the
// token operator 4.6 and 4.8; at 999 x 50257 fp16 4.0 and 5.4, 3.8 and 3.4.  There the
// rows of an SM are too few (7 of 999) for one's end to hide under another's loads, and the
// token backward, with two 16-byte loads in flight a thread, is short of issue slots as well
// (81% busy at 4096 x 32000).
//
// A row belongs to a cluster of 1, 2, 4 or 8 blocks that join their sums
// through distributed shared memory, so that few rows still fill the GPU and
// every call is one launch (and one more for the loss of the KL).
#include <cooperative_groups.h>
#include <math_constants.h>

#include "lkl_logits.cuh"
#include "sm100_ptx.cuh"

namespace lkl {
namespace {

namespace cg = cooperative_groups;

using namespace sm100;

constexpr int kLThreads = 128;      // a row's block: small, so that many rows overlap
constexpr int kLWarps = kLThreads / 32;
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
  static __device__ __forceinline__ float top(const uint4& v) {
    return max_nan(max_nan(get(v, 0), get(v, 1)), max_nan(get(v, 2), get(v, 3)));
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
  static __device__ __forceinline__ float top(const uint4& v) {   // the largest; NaN if one is
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
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
  static __device__ __forceinline__ float top(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
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
// Nothing above -inf so far: m = -inf and sums of 0.
struct TokenStat {
  static constexpr int kSums = 2;
  float m[1], sum[2];   // l, a
  __device__ __forceinline__ void move(const float* to, float c) {   // to >= m
    if (to[0] == -CUDART_INF_F || to[0] == m[0]) return;
    if (m[0] != -CUDART_INF_F) {
      const float d = m[0] - to[0], f = ex2(d * c);
      sum[1] = f == 0.f ? 0.f : f * fmaf(sum[0], d, sum[1]);
      sum[0] *= f;
    }
    m[0] = to[0];
  }
};
struct KLStat {
  static constexpr int kSums = 3;
  float m[2], sum[3];   // m_s, m_t; l_s, l_t, A
  __device__ __forceinline__ void move(const float* to, float c) {
    float shift = 0.f, f = 1.f;   // what every (t - m_t) - (s - m_s) grows by; e^(m_t - to)
    if (to[0] != -CUDART_INF_F && to[0] != m[0]) {
      if (m[0] != -CUDART_INF_F) {
        shift = to[0] - m[0];
        sum[0] *= ex2((m[0] - to[0]) * c);
      }
      m[0] = to[0];
    }
    if (to[1] != -CUDART_INF_F && to[1] != m[1]) {
      if (m[1] != -CUDART_INF_F) {
        shift += m[1] - to[1];
        f = ex2((m[1] - to[1]) * c);
      }
      m[1] = to[1];
    }
    // A may be +inf, where the student excludes what the teacher gives
    if (shift != 0.f && sum[1] > 0.f && f != 0.f) sum[2] = fmaf(sum[1], shift, sum[2]);
    sum[2] = f == 0.f && !isnan(sum[2]) ? 0.f : sum[2] * f;
    sum[1] *= f;
  }
};

// What a block shows the others of its cluster.
struct Joint {
  float warp[kLWarps][4];
  float block[2][4];   // maxima, sums
};

// Joins the statistics of a cluster's threads, in a fixed order: the maxima
// first, so that every thread rescales its sums once; every thread gets the result.
template <typename S>
__device__ __forceinline__ S join_all(S s, Joint& shared, float c) {
  constexpr int NM = S::kSums - 1, NS = S::kSums;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  cg::cluster_group cluster = cg::this_cluster();
  const int n = (int)cluster.num_blocks();
  float top[NM];
#pragma unroll
  for (int k = 0; k < NM; ++k) {
    top[k] = s.m[k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top[k] = max_nan(top[k], __shfl_xor_sync(kAll, top[k], o));
    if (lane == 0) shared.warp[warp][k] = top[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NM; ++k) {
    top[k] = shared.warp[0][k];
#pragma unroll
    for (int w = 1; w < kLWarps; ++w) top[k] = max_nan(top[k], shared.warp[w][k]);
  }
  if (n > 1) {
    if (threadIdx.x == 0)
      for (int k = 0; k < NM; ++k) shared.block[0][k] = top[k];
    cluster.sync();
    for (int r = 0; r < n; ++r) {
      const Joint* other = cluster.map_shared_rank(&shared, r);
#pragma unroll
      for (int k = 0; k < NM; ++k) top[k] = max_nan(top[k], other->block[0][k]);
    }
  }
  __syncthreads();
  s.move(top, c);
#pragma unroll
  for (int k = 0; k < NS; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.sum[k] += __shfl_xor_sync(kAll, s.sum[k], o);
    if (lane == 0) shared.warp[warp][k] = s.sum[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    s.sum[k] = shared.warp[0][k];
#pragma unroll
    for (int w = 1; w < kLWarps; ++w) s.sum[k] += shared.warp[w][k];
  }
  if (n > 1) {
    if (threadIdx.x == 0)
      for (int k = 0; k < NS; ++k) shared.block[1][k] = s.sum[k];
    cluster.sync();
#pragma unroll
    for (int k = 0; k < NS; ++k) s.sum[k] = 0.f;
    for (int r = 0; r < n; ++r) {
      const Joint* other = cluster.map_shared_rank(&shared, r);
#pragma unroll
      for (int k = 0; k < NS; ++k) s.sum[k] += other->block[1][k];
    }
    cluster.sync();   // the entries are free, and no block has left
  } else {
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < NM; ++k) s.m[k] = top[k];
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
  // Joins another such list: the better of each pair with the other reversed is a
  // bitonic sequence of the 32 best (Batcher), which five exchanges sort.
  __device__ __forceinline__ void merge(uint64_t other, int lane) {
    const uint64_t o = __shfl_sync(kAll, other, 31 - lane);
    key = o > key ? o : key;
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) exchange(j, (lane & j) == 0);
  }
  // Sorts 32 elements, one a lane.
  __device__ __forceinline__ void sort(int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1)
        exchange(j, ((lane & j) == 0) == ((lane & k) == 0 || k == 32));
  }
  __device__ __forceinline__ void exchange(int j, bool larger) {
    const uint64_t o = __shfl_xor_sync(kAll, key, j);
    key = (o > key) == larger ? o : key;
  }
  // Value that an element has to reach to be among the best k (-inf: any does).
  __device__ __forceinline__ float threshold(int k) const {
    const uint64_t last = __shfl_sync(kAll, key, k - 1);
    return last ? top_value(last) : -CUDART_INF_F;
  }
};

// ---------------------------------------------------------------- token forward
// Adds the pair x (two values as one register pair) to sums relative to m2.
template <bool GUARD>
__device__ __forceinline__ void token_pair(uint64_t x, uint64_t m2, uint64_t c2, uint64_t& l,
                                           uint64_t& a) {
  uint64_t d = fsub2(x, m2);
  if (GUARD) {
    float d0, d1;
    f2unpack(d, d0, d1);
    d = f2pack(max_nan(d0, -200.f), max_nan(d1, -200.f));   // e^-200 is 0 in fp32
  }
  float e0, e1;
  f2unpack(fmul2(d, c2), e0, e1);
  const uint64_t e = f2pack(ex2(e0), ex2(e1));
  l = fadd2(l, e);
  a = ffma2(e, d, a);
}

// The warps' bounds on the alternatives, and room for one lane's elements a warp.
struct TopShared {
  float kth[kLWarps], part[kLWarps];
  float lane[kLWarps][32];
  uint64_t lists[kLWarps][32];
};

// Sums over this block's share of the row.  GUARD: -inf logits add exactly 0 to
// a, where the plain form gives 0 x -inf = NaN; only rows that met one need it.
//
// TOP: an element can be among the best k only if it reaches the k-th best of any
// warp, and also the least of the warps' (k / warps)-th best.  Few elements do after
// the first batch; a batch's maximum, known for the sums, rules most batches out.
// U: 16-byte loads in flight a thread.
template <typename T, bool GUARD, bool TOP, int U>
__device__ __forceinline__ TokenStat token_pass(const T* row, long long V, int top_k, TopList& top,
                                                TopShared& ts) {
  constexpr int N = Elem<T>::N, E = U * N;
  static_assert(!TOP || E <= 32, "a lane's elements fit a warp");
  const RowCut<T> cut(row, V);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), n_blocks = (int)cluster.num_blocks();
  const int v0 = (int)((long long)cut.nv * rank / n_blocks);
  const int v1 = (int)((long long)cut.nv * (rank + 1) / n_blocks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint4* vec = reinterpret_cast<const uint4*>(row + cut.lead);
  volatile float* kth = ts.kth;
  volatile float* part = ts.part;
  const int share_k = (top_k + kLWarps - 1) / kLWarps;
  TokenStat s{{-CUDART_INF_F}, {0.f, 0.f}};
  const uint64_t c2 = f2pack(kLog2e, kLog2e);
  bool fresh = true;
  auto add = [&](const uint4* raw, int n) {   // n vectors; the sums, given their maximum
    float bm = Elem<T>::top(raw[0]);
#pragma unroll
    for (int u = 1; u < n; ++u) bm = max_nan(bm, Elem<T>::top(raw[u]));
    const float to = max_nan(s.m[0], bm);
    if (to == -CUDART_INF_F) return bm;
    if (!(to == s.m[0])) s.move(&to, kLog2e);
    const uint64_t m2 = f2pack(to, to);
    uint64_t l[2] = {0, 0}, a[2] = {0, 0};
#pragma unroll
    for (int u = 0; u < n; ++u)
#pragma unroll
      for (int e = 0; e < N; e += 2)
        token_pair<GUARD>(f2pack(Elem<T>::get(raw[u], e), Elem<T>::get(raw[u], e + 1)), m2, c2,
                          l[(e >> 1) & 1], a[(e >> 1) & 1]);
    float x, y;
    f2unpack(fadd2(l[0], l[1]), x, y);
    s.sum[0] += x + y;
    f2unpack(fadd2(a[0], a[1]), x, y);
    s.sum[1] += x + y;
    return bm;
  };
  for (int v = v0 + warp * 32; v < v1; v += U * kLThreads) {
    uint4 raw[U];
    const int mine = v + lane;
    const bool full = mine + (U - 1) * kLThreads < v1;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (full || mine + u * kLThreads < v1) raw[u] = __ldg(vec + mine + u * kLThreads);
    float bm = -CUDART_INF_F;
    if (full) {
      bm = add(raw, U);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (mine + u * kLThreads < v1) bm = max_nan(bm, add(raw + u, 1));
    }
    if (!TOP) continue;
    __syncwarp();
    float need = top.threshold(top_k), least = part[0];
#pragma unroll
    for (int w = 0; w < kLWarps; ++w) {
      need = fmaxf(need, kth[w]);
      least = fminf(least, part[w]);
    }
    need = fmaxf(need, least);
    const bool in = mine < v1;
    // what this lane still has to offer, and what it has offered already
    float offer = in ? bm : -CUDART_INF_F;
    bool any = in;
    uint64_t own = 0;
    if (fresh) {
      // the list starts with every lane's best element; the lane's next best decides
      // whether the rest is looked at
      fresh = false;
      float next = -CUDART_INF_F;
      int arg = -1;
      offer = -CUDART_INF_F;
      any = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x = Elem<T>::get(raw[e / N], e % N);
        if (!(full || mine + (e / N) * kLThreads < v1) || isnan(x)) continue;
        if (arg < 0 || x > offer) {
          any = arg >= 0;
          next = offer;
          offer = x;
          arg = e;
        } else {
          any = true;
          next = fmaxf(next, x);
        }
      }
      if (arg >= 0)
        own = top_key(offer, (uint32_t)(cut.lead + (mine + (arg / N) * kLThreads) * N + arg % N));
      top.key = own;
      top.sort(lane);
      offer = next;
      need = fmaxf(need, top.threshold(top_k));
    }
    uint32_t lanes = __ballot_sync(kAll, any && !(offer < need));
    // the elements of one lane after the other, one a lane
    while (lanes) {
      const int from = __ffs(lanes) - 1;
      lanes &= lanes - 1;
      if (lane == from) {
#pragma unroll
        for (int e = 0; e < E; ++e) ts.lane[warp][e] = Elem<T>::get(raw[e / N], e % N);
      }
      __syncwarp();
      const int at = v + from + (lane / N) * kLThreads;   // vector of this lane's element
      const float x = ts.lane[warp][lane];
      uint32_t hit = __ballot_sync(kAll, lane < E && at < v1 && x >= need);
      const uint64_t key = top_key(x, (uint32_t)(cut.lead + at * N + lane % N));
      hit &= __ballot_sync(kAll, key != __shfl_sync(kAll, own, from));
      while (hit) {
        const int h = __ffs(hit) - 1;
        hit &= hit - 1;
        top.insert(__shfl_sync(kAll, key, h), lane);
      }
      need = fmaxf(need, top.threshold(top_k));
      lanes &= __ballot_sync(kAll, !(offer < need));
      __syncwarp();
    }
    const float a_k = top.threshold(top_k), a_part = top.threshold(share_k);
    if (lane == 0) {
      kth[warp] = a_k;
      part[warp] = a_part;
    }
  }
  if (rank == 0 && warp == 0) {   // at most 14 elements
    const long long c = cut.end_elem(lane, V);
    const float x = c >= 0 ? Elem<T>::one(row + c) : -CUDART_INF_F;
    const float to = max_nan(s.m[0], x);
    if (to != -CUDART_INF_F) {
      if (!(to == s.m[0])) s.move(&to, kLog2e);
      const float d = max_nan(x - to, -200.f), e = ex2(d * kLog2e);
      s.sum[0] += e;
      s.sum[1] = fmaf(e, d, s.sum[1]);
    }
    if (TOP) {
      uint32_t hit = __ballot_sync(kAll, c >= 0 && !isnan(x));
      const uint64_t key = top_key(x, (uint32_t)c);
      while (hit) {
        const int h = __ffs(hit) - 1;
        hit &= hit - 1;
        top.insert(__shfl_sync(kAll, key, h), lane);
      }
    }
  }
  return s;
}

// Joins the warps' lists in warp 0.
__device__ __forceinline__ void join_lists(TopList& top, TopShared& ts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  ts.lists[warp][lane] = top.key;
  __syncthreads();
  if (warp == 0)
    for (int w = 1; w < kLWarps; ++w) top.merge(ts.lists[w][lane], lane);
}

// The best elements of this block's share, in warp 0 (one a lane, sorted).
//
// mine: the largest logit that this thread saw in the pass over the row.  The k-th
// largest of the threads' maxima is reached by k elements at least and, unless many
// logits are equal, by few more (22 expected for k = 20 of any row length).  So a
// second look at the share, which is in L2 by now, compares each 16 bytes' maximum with
// it and collects what reaches it.  Rows with more such elements than `cand` holds
// (equal logits) take the pass that keeps a sorted list a warp.
constexpr int kTopCand = 256;
struct TopLook {
  alignas(16) float mine[kLThreads];   // read four at a time
  float bound;
  int count;
  uint64_t cand[kTopCand];
};

template <typename T>
__device__ __forceinline__ TopList top_pass(const T* row, long long V, int top_k, float mine,
                                            TopShared& ts, TopLook& tc) {
  constexpr int N = Elem<T>::N, U = 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (isnan(mine)) mine = -CUDART_INF_F;
  tc.mine[threadIdx.x] = mine;
  if (threadIdx.x == 0) tc.count = 0;
  __syncthreads();
  int rank_of = 0;
  const float4* all = reinterpret_cast<const float4*>(tc.mine);
#pragma unroll 8
  for (int k = 0; k < kLThreads / 4; ++k) {
    const float4 o = all[k];
    const int at = 4 * k;
    rank_of += (o.x > mine || (o.x == mine && at < (int)threadIdx.x));
    rank_of += (o.y > mine || (o.y == mine && at + 1 < (int)threadIdx.x));
    rank_of += (o.z > mine || (o.z == mine && at + 2 < (int)threadIdx.x));
    rank_of += (o.w > mine || (o.w == mine && at + 3 < (int)threadIdx.x));
  }
  if (rank_of == top_k - 1) tc.bound = mine;
  __syncthreads();
  const float bound = tc.bound;
  const RowCut<T> cut(row, V);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), n_blocks = (int)cluster.num_blocks();
  const int v0 = (int)((long long)cut.nv * rank / n_blocks);
  const int v1 = (int)((long long)cut.nv * (rank + 1) / n_blocks);
  const uint4* vec = reinterpret_cast<const uint4*>(row + cut.lead);
  auto take = [&](float x, long long idx) {
    if (!(x >= bound)) return;
    const int at = atomicAdd(&tc.count, 1);
    if (at < kTopCand) tc.cand[at] = top_key(x, (uint32_t)idx);
  };
  auto look = [&](const uint4& raw, int at) {
    if (Elem<T>::top(raw) < bound) return;
#pragma unroll
    for (int e = 0; e < N; ++e) take(Elem<T>::get(raw, e), cut.lead + (long long)at * N + e);
  };
  int v = v0 + threadIdx.x;
  for (; v + (U - 1) * kLThreads < v1; v += U * kLThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = __ldg(vec + v + u * kLThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) look(raw[u], v + u * kLThreads);
  }
  for (; v < v1; v += kLThreads) look(__ldg(vec + v), v);
  if (rank == 0) {
    const long long c = cut.end_elem(threadIdx.x, V);
    if (c >= 0) take(Elem<T>::one(row + c), c);
  }
  __syncthreads();
  const int count = tc.count;
  TopList top{0};
  if (count <= kTopCand) {
    if (warp == 0)
      for (int at = 0; at < count; at += 32) {   // in any order: the keys are distinct
        TopList part{at + lane < count ? tc.cand[at + lane] : 0};
        part.sort(lane);
        if (at == 0) top = part;
        else top.merge(part.key, lane);
      }
    return top;
  }
  if (lane == 0) ts.kth[warp] = ts.part[warp] = -CUDART_INF_F;
  __syncthreads();
  token_pass<T, false, true, 4>(row, V, top_k, top, ts);
  join_lists(top, ts);
  return top;
}

// Alternatives are found in the one pass (kTopList) or by a second look (kTopLook).
enum TopMode { kTopNone, kTopList, kTopLook };

template <typename T, int MODE>
__global__ void __launch_bounds__(kLThreads)
token_logprobs_kernel(const LogitsView view, const int64_t* __restrict__ targets, int64_t ignore,
                      int top_k, float* __restrict__ logprob, float* __restrict__ entropy,
                      float* __restrict__ lse_out, float* __restrict__ top_v,
                      int64_t* __restrict__ top_i) {
  __shared__ Joint joint;
  __shared__ TopShared ts;
  __shared__ TopLook tc;
  cg::cluster_group cluster = cg::this_cluster();
  const int n = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long row = blockIdx.x / n;
  const T* x = row_ptr<T>(view, row);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TopList none{0}, top{0};
  if (MODE == kTopList) {
    if (lane == 0) ts.kth[warp] = ts.part[warp] = -CUDART_INF_F;
    __syncthreads();
  }
  // alone, 8 loads: 196 -> 177 us at 16384 x 32000 bf16; with alternatives, 4: 347, 8: 400
  constexpr int U = MODE == kTopNone ? 8 : 4;
  TokenStat s = token_pass<T, false, MODE == kTopList, U>(x, view.V, top_k, top, ts);
  const float mine = s.m[0];
  s = join_all(s, joint, kLog2e);
  if (isnan(s.sum[1]) && s.sum[0] > 0.f)   // the same in every thread of the cluster
    s = join_all(token_pass<T, true, false, U>(x, view.V, 0, none, ts), joint, kLog2e);
  const bool empty = s.m[0] == -CUDART_INF_F;
  const float log_l = empty ? CUDART_NAN_F : logf(s.sum[0]);
  if (rank == 0 && threadIdx.x == 0) {
    const int64_t y = targets[row];
    float lp = CUDART_NAN_F;
    if (y == ignore) lp = 0.f;
    else if (y >= 0 && y < view.V) lp = (Elem<T>::one(x + y) - s.m[0]) - log_l;
    logprob[row] = lp;
    entropy[row] = log_l - s.sum[1] / s.sum[0];
    lse_out[row] = s.m[0] + log_l;
    if (view.low) {
      const double z = empty ? CUDART_NAN : (double)s.m[0] + log((double)s.sum[0]);
      lse_out[row] = (float)z;
      view.low[row] = (float)(z - (double)(float)z);
    }
  }
  if (MODE != kTopNone) {
    if (MODE == kTopLook) top = top_pass<T>(x, view.V, top_k, mine, ts, tc);
    else join_lists(top, ts);
    if (n > 1) {
      if (warp == 0) ts.lists[0][lane] = top.key;
      cluster.sync();
    }
    if (rank == 0 && warp == 0) {
      for (int r = 1; r < n; ++r)
        top.merge(cluster.map_shared_rank(&ts.lists[0][0], r)[lane], lane);
      if (lane < top_k) {
        const long long idx = (uint32_t)~(uint32_t)top.key;
        top_v[row * top_k + lane] =
            top.key ? (top_value(top.key) - s.m[0]) - log_l : CUDART_NAN_F;
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
  constexpr int U = 4;   // loads in flight a thread and stream
  const RowCut<T> cut(s, V);
  const bool vec = same_offset(s, t);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), n_blocks = (int)cluster.num_blocks();
  const int v0 = (int)((long long)cut.nv * rank / n_blocks);
  const int v1 = (int)((long long)cut.nv * (rank + 1) / n_blocks);
  KLStat st{{-CUDART_INF_F, -CUDART_INF_F}, {0.f, 0.f, 0.f}};
  const uint64_t c2 = f2pack(c, c);
  auto add = [&](const uint4* x, const uint4* y, int n) {
    float to[2] = {st.m[0], st.m[1]};
#pragma unroll
    for (int u = 0; u < n; ++u) {
      to[0] = max_nan(to[0], Elem<T>::top(x[u]));
      to[1] = max_nan(to[1], Elem<T>::top(y[u]));
    }
    if (!(to[0] == st.m[0] && to[1] == st.m[1])) st.move(to, c);
    const float ms = to[0] == -CUDART_INF_F ? 0.f : to[0];
    const float mt = to[1] == -CUDART_INF_F ? 0.f : to[1];
    const uint64_t ms2 = f2pack(ms, ms), mt2 = f2pack(mt, mt);
    uint64_t ls = 0, lt = 0, a = 0;
#pragma unroll
    for (int u = 0; u < n; ++u)
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const uint64_t xs = f2pack(Elem<T>::get(x[u], e), Elem<T>::get(x[u], e + 1));
        const uint64_t xt = f2pack(Elem<T>::get(y[u], e), Elem<T>::get(y[u], e + 1));
        const uint64_t ds = fsub2(xs, ms2), dt = fsub2(xt, mt2);
        float s0, s1, t0, t1;
        f2unpack(fmul2(ds, c2), s0, s1);
        f2unpack(fmul2(dt, c2), t0, t1);
        const uint64_t es = f2pack(ex2(s0), ex2(s1)), et = f2pack(ex2(t0), ex2(t1));
        ls = fadd2(ls, es);
        lt = fadd2(lt, et);
        uint64_t d = fsub2(dt, ds);
        if (GUARD) {   // no teacher probability, nothing added
          float e0, e1, d0, d1;
          f2unpack(et, e0, e1);
          f2unpack(d, d0, d1);
          d = f2pack(e0 == 0.f ? 0.f : d0, e1 == 0.f ? 0.f : d1);
        }
        a = ffma2(et, d, a);
      }
    float u0, u1;
    f2unpack(ls, u0, u1);
    st.sum[0] += u0 + u1;
    f2unpack(lt, u0, u1);
    st.sum[1] += u0 + u1;
    f2unpack(a, u0, u1);
    st.sum[2] += u0 + u1;
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
    add(a, b, U);
  }
  for (; v < v1; v += kLThreads) {
    const uint4 a = __ldg(sv + v), b = load_vec(tv + (size_t)v * N, vec);
    add(&a, &b, 1);
  }
  if (rank == 0) {
    const long long k = cut.end_elem(threadIdx.x, V);
    if (k >= 0) {
      const float x = Elem<T>::one(s + k), y = Elem<T>::one(t + k);
      const float to[2] = {max_nan(st.m[0], x), max_nan(st.m[1], y)};
      st.move(to, c);
      const float dx = x - (to[0] == -CUDART_INF_F ? 0.f : to[0]);
      const float dy = y - (to[1] == -CUDART_INF_F ? 0.f : to[1]);
      const float et = ex2(dy * c);
      st.sum[0] += ex2(dx * c);
      st.sum[1] += et;
      st.sum[2] = fmaf(et, GUARD && et == 0.f ? 0.f : dy - dx, st.sum[2]);
    }
  }
  return st;
}

template <typename T>
__global__ void __launch_bounds__(kLThreads)
logits_kl_forward_kernel(const LogitsView sv, const LogitsView tv, const void* __restrict__ mask,
                         int mdt, float inv_tau, float* __restrict__ lse_s,
                         float* __restrict__ lse_t, float* __restrict__ row_kl) {
  __shared__ Joint joint;
  cg::cluster_group cluster = cg::this_cluster();
  const long long row = blockIdx.x / cluster.num_blocks();
  const bool first = cluster.block_rank() == 0 && threadIdx.x == 0;
  if (mask && !mask_elem(mask, row, mdt)) {   // the whole cluster
    if (first) {
      lse_s[row] = lse_t[row] = row_kl[row] = 0.f;
      if (sv.low) sv.low[row] = 0.f;
      if (tv.low) tv.low[row] = 0.f;
    }
    return;
  }
  const T *s = row_ptr<T>(sv, row), *t = row_ptr<T>(tv, row);
  const float c = inv_tau * kLog2e;
  KLStat k = join_all(kl_pass<T, false>(s, t, sv.V, c), joint, c);
  if (isnan(k.sum[2]) && !isnan(k.sum[0]) && !isnan(k.sum[1]))
    k = join_all(kl_pass<T, true>(s, t, sv.V, c), joint, c);
  if (first) {
    // in 64 bits: the loss is what is left of the difference of the two logarithms
    const bool none = k.m[0] == -CUDART_INF_F || k.m[1] == -CUDART_INF_F;
    const double zs = none ? CUDART_NAN : (double)k.m[0] * inv_tau + log((double)k.sum[0]);
    const double zt = none ? CUDART_NAN : (double)k.m[1] * inv_tau + log((double)k.sum[1]);
    lse_s[row] = (float)zs;
    lse_t[row] = (float)zt;
    if (sv.low) sv.low[row] = (float)(zs - (double)(float)zs);
    if (tv.low) tv.low[row] = (float)(zt - (double)(float)zt);
    row_kl[row] = none ? CUDART_NAN_F
                       : (float)((double)k.sum[2] * inv_tau / k.sum[1] +
                                 (log((double)k.sum[0]) - log((double)k.sum[1])));
  }
}

// ---------------------------------------------------------------- gradients
constexpr int kGThreadsL = 256;
constexpr int kLShare = 4 * kGThreadsL;   // vectors a block

// d = f(x, element) over a row: vectors in this block's share, the ends by the first block.
// zero: zeros instead, decided behind the loads so that they need not wait for it.
template <typename T, typename Load, typename F>
__device__ __forceinline__ void map_row(const T* cut_by, T* out, long long V, int share, Load load,
                                        F f, bool zero = false) {
  constexpr int N = Elem<T>::N;
  const RowCut<T> cut(cut_by, V);
  const bool vec = same_offset(cut_by, out);
  const int end = min(cut.nv, (share + 1) * kLShare);
  for (int v = share * kLShare + threadIdx.x; v < end; v += 2 * kGThreadsL) {
    const bool two = v + kGThreadsL < end;
    auto a = load(cut.lead + (long long)v * N);
    auto b = a;
    if (two) b = load(cut.lead + (long long)(v + kGThreadsL) * N);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && !two) break;
      const long long at = cut.lead + (long long)(v + h * kGThreadsL) * N;
      uint4 d = make_uint4(0, 0, 0, 0);
      if (!zero) {
#pragma unroll
        for (int e = 0; e < N; ++e) Elem<T>::put(d, e, f(h ? b : a, e, at + e));
      }
      store_vec(out + at, d, vec);
    }
  }
  if (share == 0) {
    const long long k = cut.end_elem(threadIdx.x, V);
    if (k >= 0) Elem<T>::put1(out + k, zero ? 0.f : f(load.one(k), 0, k));
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

// What a row's log-sum-exp in fp32 lacks, 0 where that was not kept.  Without a branch, which
// would keep the row's loads behind it (KL backward, 4096 x 32000 fp32: 258 instead of 242 us).
__device__ __forceinline__ float lse_rest(const float* low, const float* lse, long long row) {
  return (low ? 1.f : 0.f) * (low ? low : lse)[row];
}

template <typename T>
__global__ void __launch_bounds__(kGThreadsL)
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
  // Without gradient a row gives zeros whatever it holds: 0 x NaN is not 0.  Its logits are
  // read all the same: a branch here would have every row's loads wait for its target
  // (2004 x 50257 bf16, with the forward: 128 -> 144 us).
  const bool none = y == ignore && h == 0.f;
  // -p (g + h (log p + H)) + g at the target
  const float rest = lse_rest(view.low, lse, row);   // log p = (x - z) - rest
  const float gh = fmaf(h, H - rest, g), low = -rest * kLog2e;
  map_row<T>(x, dx + row * view.V, view.V, (int)(blockIdx.x % shares), LoadOne<T>{x},
             [&](const uint4& v, int e, long long at) {
               // e^-200 is 0; 0 x -inf would not be
               const float lp = max_nan(Elem<T>::get(v, e) - z, -200.f);
               const float d = -ex2(fmaf(lp, kLog2e, low)) * fmaf(h, lp, gh);
               return at == y ? d + g : d;
             }, none);
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

// a - b without rounding, as two numbers (Knuth's two-sum).
__device__ __forceinline__ float2 exact_difference(float a, float b) {
  const float d = a - b, bb = d - a;
  return make_float2(d, (a - (d - bb)) - (b + bb));
}

// ps - pt = pt (e^x - 1), x = (s - t) / tau - (lse_s - lse_t), where the two are near.  Their
// difference would carry the roundings of both: with logits of scale 2 and models 0.5 apart
// fp32 gradients were 4 10^-7 of their size off, 1.9 10^-6 at a temperature of 2; so they are
// 3 10^-7 and 5 10^-7 (models 0.05 apart: 4 10^-6 and 2 10^-5, now 1.3 and 2.5 10^-6, what the
// fp32 sums behind the log-sum-exps leave).  e^x - 1 by its Taylor series, off by less than
// 2 10^-7 up to 0.5.  For fp32 only: 16-bit gradients are rounded far coarser.  The 15
// instructions an element cost 6 to 12% there (4096 x 32000: 235 -> 250 us), 13 to 16% with
// the 48 registers that the compiler would take: six blocks an SM hide more.
struct NearDifference {
  float2 dz;   // lse_s - lse_t
  __device__ __forceinline__ float exponent(float s, float t, float inv_tau) const {
    const float2 e = exact_difference(s, t);
    return fmaf(e.x, inv_tau, -dz.x) + fmaf(e.y, inv_tau, -dz.y);
  }
  static __device__ __forceinline__ float expm1_small(float x) {
    float y = 1.f / 5040;
    y = fmaf(y, x, 1.f / 720);
    y = fmaf(y, x, 1.f / 120);
    y = fmaf(y, x, 1.f / 24);
    y = fmaf(y, x, 1.f / 6);
    y = fmaf(y, x, 0.5f);
    return x * fmaf(y, x, 1.f);
  }
};

template <typename T>
__global__ void __launch_bounds__(kGThreadsL, sizeof(T) == 4 ? 6 : 0)
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
  // the log probability first: a likely token's exponent is small and keeps its bits
  const float g = (dloss ? *dloss : 1.f) * inv_tau, zs = lse_s[row], zt = lse_t[row];
  const float rest_s = lse_rest(sv.low, lse_s, row), rest_t = lse_rest(tv.low, lse_t, row);
  const float low_s = -rest_s * kLog2e, low_t = -rest_t * kLog2e;
  NearDifference near{exact_difference(zs, zt)};
  near.dz.y += rest_s - rest_t;
  map_row<T>(s, out, sv.V, share, LoadPair<T>{s, t, same_offset(s, t)},
             [&](const Pair& v, int e, long long) {
               const float a = Elem<T>::get(v.s, e), b = Elem<T>::get(v.t, e);
               const float ps = ex2(fmaf(fmaf(a, inv_tau, -zs), kLog2e, low_s));
               const float pt = ex2(fmaf(fmaf(b, inv_tau, -zt), kLog2e, low_t));
               float d = ps - pt;
               if (sizeof(T) == 4) {   // not a number, or far apart: the difference itself
                 const float x = near.exponent(a, b, inv_tau);
                 const float y = pt * near.expm1_small(x);
                 d = fabsf(x) <= 0.5f ? y : d;
               }
               return g * d;
             });
}

// ---------------------------------------------------------------- launches
// Blocks a row: enough that all rows together give four blocks an SM, as long as a
// block keeps 1024 elements (below that, joining costs more than it saves).
int cluster_of(long long rows, long long V) {
  int n = 1;
  while (n < kMaxCluster && rows * n < 592 && V / (2 * n) >= 1024) n *= 2;
  return n;
}

// A second look needs the shares of all resident blocks (ten an SM) to stay in L2: up
// to 104 KB a block it is faster (2004 x 50257 bf16, top 20: 77 us, list 102), above
// it is not (4096 x 32000 fp32: 169 us, list 144; 2048 x 128256 bf16: 180, 177).
constexpr long long kTopLookBytes = 104 << 10;

template <typename K, typename... A>
cudaError_t launch_rows(K kernel, int threads, long long rows, int cluster, cudaStream_t st,
                        A... args) {
  if (rows * cluster > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(threads);
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
  return with_type(x.dtype, [&](auto t) {
    using T = decltype(t);
    const int n = cluster_of(rows, x.V);
    const bool look = x.V * (long long)sizeof(T) / n <= kTopLookBytes;
    return launch_rows(!top_k ? token_logprobs_kernel<T, kTopNone>
                       : look ? token_logprobs_kernel<T, kTopLook>
                              : token_logprobs_kernel<T, kTopList>,
                       kLThreads, rows, n, st, x, targets, ignore, top_k, logprob, entropy, lse,
                       top_v, top_i);
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
    return launch_rows(token_logprobs_backward_kernel<T>, kGThreadsL, rows * shares, 1, st, x,
                       targets, ignore, lse, entropy, g_lp, g_en, static_cast<T*>(dx), shares);
  });
}

cudaError_t launch_logits_kl_forward(const LogitsView& s, const LogitsView& t, long long rows,
                                     const void* mask, int mdt, float inv_tau, float* lse_s,
                                     float* lse_t, float* row_kl, float* loss, cudaStream_t st) {
  const int n = cluster_of(rows, s.V);
  const cudaError_t e = with_type(s.dtype, [&](auto x) {
    return launch_rows(logits_kl_forward_kernel<decltype(x)>, kLThreads, rows, n, st, s, t, mask,
                       mdt, inv_tau, lse_s, lse_t, row_kl);
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
    return launch_rows(logits_kl_backward_kernel<T>, kGThreadsL, rows * shares, 1, st, s, t, mask,
                       mdt, inv_tau, lse_s, lse_t, dloss, static_cast<T*>(ds), shares);
  });
}

}  // namespace lkl
