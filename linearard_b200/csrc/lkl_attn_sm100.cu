// sm_100a tensor-core attention: the forward.
//
// One CTA owns 256 query rows of one head as two tiles of 128 and walks the
// 128-key tiles from the diagonal down.  Per tile and key tile, two GEMMs
// (S = Q K^T, O += P V) and one exponential per score.  At head dim 128 the
// 16,384 exponentials of a tile take 1024 cycles of the SM's MUFU pipe and its
// two GEMMs about 1024 cycles of the tensor pipe, so neither may wait: while
// one tile's warpgroup computes P, the other tile's GEMMs run.
//
// Warps 0-3 / 4-7: softmax of tile 0 / 1, one row a thread, so a row's maximum
// and sum need no exchange.  Warp 8: TMA producer.  Warp 9: MMA issuer and TMEM
// owner.  Warp 10: with a padding mask, clears the rows of removed tokens in the
// loaded tiles (P is 0 there, but 0 x NaN is not).
//
// TMEM: S0, S1 (128 columns each; P, 16-bit, overwrites the first 64 of its S),
// then O0, O1.  tcgen05.mma of one thread run in order, so S_t(j+1), issued
// after O_t += P_t(j) V(j), may overwrite P_t(j), and its commit also says that
// O_t is complete up to j.
#include <math_constants.h>

#include "lkl_attn.cuh"
#include "sm100_ptx.cuh"

namespace lkl {
namespace {

constexpr int kFaThreads = 384;
// Registers a thread: three warpgroups are launched with 168 each; the softmax
// groups hold a row of 128 scores and take what the third does not need.
constexpr int kFaRegs = 168, kFaSoftmaxRegs = 208, kFaOtherRegs = 88;
static_assert(2 * kFaSoftmaxRegs + kFaOtherRegs <= 3 * kFaRegs, "register split");
static_assert(kFaThreads * kFaRegs <= 65536, "register file");
constexpr int kFaProducer = 8, kFaMma = 9, kFaCleaner = 10;
// A row's exponent offset is its running maximum as of the last rescale; it
// moves only when the maximum has grown by more than 2^8.  P then stays below
// 256, exact in neither type more or less than below 1 (the rounding is relative).
constexpr float kFaSlack = 8.f;
constexpr float kMaskedScore = -1.0e30f;

template <int D>
struct FaLayout {
  static constexpr int TILE = kBM * D * 2;      // one 128-row tile
  static constexpr int NS = D == 128 ? 5 : 8;   // ring of K and V tiles
  static constexpr int OFF_Q = 0, OFF_KV = 2 * TILE;
  static constexpr int OFF_MISC = OFF_KV + NS * TILE;
  static constexpr int BYTES = 1024 + OFF_MISC + kMisc;
  static_assert(BYTES <= kMaxDynSmem, "shared memory");
};

struct FaMisc {
  uint64_t q_full;
  uint64_t full[8], ready[8], empty[8];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(FaMisc) <= kMisc, "misc region too small");

// Validity bits of tokens [tile * 128, + 128): all of them without a mask
// (tokens past T then have to be cut by position).
struct TileBits {
  uint32_t w[4];
  __device__ __forceinline__ bool any() const { return (w[0] | w[1] | w[2] | w[3]) != 0; }
  __device__ __forceinline__ bool all() const { return (w[0] & w[1] & w[2] & w[3]) == ~0u; }
};

template <bool MASKED>
__device__ __forceinline__ TileBits tile_bits(const uint32_t* bits, int words, int b, int tile) {
  TileBits t;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    t.w[k] = ~0u;
    if (MASKED) {
      const int w = tile * 4 + k;
      t.w[k] = w < words ? __ldg(bits + (size_t)b * words + w) : 0u;
    }
  }
  return t;
}

// Next key tile at or below kt with a token in it, or -1.
template <bool MASKED>
__device__ __forceinline__ int live_tile(const uint32_t* bits, int words, int b, int kt) {
  if (MASKED)
    while (kt >= 0 && !tile_bits<true>(bits, words, b, kt).any()) --kt;
  return kt;
}

// Zeroes the rows of removed tokens in a loaded [128][D] tile.
template <int D>
__device__ __forceinline__ void clear_rows(uint8_t* tile, const TileBits& t, int lane) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if ((t.w[k] >> lane) & 1u) continue;
    uint8_t* row = tile + (k * 32 + lane) * 128;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int x = 0; x < 8; ++x)
        *reinterpret_cast<uint4*>(row + c * kChunk + (((x + lane) & 7) << 4)) =
            make_uint4(0, 0, 0, 0);
  }
}

// Query tiles in bands of heads whose keys and values stay in L2, the longest
// rows of a band first.
struct FaWork {
  int bh, m;
};
__device__ __forceinline__ FaWork fa_work(int blk, int heads, int band, int n_m) {
  const int k = blk / (band * n_m), r = blk % (band * n_m);
  const int size = min(band, heads - k * band);
  return FaWork{k * band + r % size, n_m - 1 - r / size};
}

template <int D, bool BF16, bool MASKED>
__global__ void __launch_bounds__(kFaThreads, 1)
attn_sm100_forward_kernel(const __grid_constant__ CUtensorMap tm_q,
                          const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v, const AttnProblem p,
                          const TensorStrides so, const uint32_t* __restrict__ bits,
                          uint16_t* __restrict__ out, float* __restrict__ lse, int band) {
  using L = FaLayout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  FaMisc* misc = reinterpret_cast<FaMisc*>(smem + L::OFF_MISC);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* err = &g_device_error;
  volatile int* abort = &misc->abort;

  const int n_kt = (p.T + kBN - 1) / kBN, words = (p.T + 31) >> 5;
  const FaWork wk = fa_work(blockIdx.x, p.B * p.Hq, band, (p.T + 2 * kBM - 1) / (2 * kBM));
  const int b = wk.bh / p.Hq, h = wk.bh % p.Hq, g = h / (p.Hq / p.Hkv);
  // key tiles of each query tile: 0 .. n_ct - 1 (none for a tile without a token)
  int n_ct[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int qt = wk.m * 2 + t;
    n_ct[t] = qt >= n_kt || !tile_bits<MASKED>(bits, words, b, qt).any() ? 0
              : p.causal ? qt + 1
                         : n_kt;
  }
  const int kt0 = live_tile<MASKED>(bits, words, b, max(n_ct[0], n_ct[1]) - 1);

  if (threadIdx.x == 0) {
    mbar_init(&misc->q_full, 1);
    for (int s = 0; s < L::NS; ++s) {
      mbar_init(&misc->full[s], 1);
      mbar_init(&misc->ready[s], 1);
      mbar_init(&misc->empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&misc->s_full[t], 1);
      mbar_init(&misc->p_full[t], 4);
      mbar_init(&misc->o_full[t], 1);
    }
    misc->abort = 0;
    fence_barrier_init();
  }
  if (warp == kFaMma) {
    tmem_alloc(&misc->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if (warp == kFaProducer && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc->tmem_base;
  constexpr uint32_t kColO = 256;

  if (warp >= 8) {
    reg_dec<kFaOtherRegs>();
    if (warp == kFaProducer) {
      if (lane == 0 && kt0 >= 0) {
        mbar_arrive_expect_tx(&misc->q_full, ((n_ct[0] > 0) + (n_ct[1] > 0)) * L::TILE);
  #pragma unroll
        for (int t = 0; t < 2; ++t)
          if (n_ct[t] > 0)
            issue_tile_loads(smem + L::OFF_Q + t * L::TILE, &tm_q, &misc->q_full, D,
                             (wk.m * 2 + t) * kBM, h, b);
        int n = 0;   // K(0), V(0), K(1), V(1), ...
        bool ok = true;
        for (int kt = kt0; ok && kt >= 0; kt = live_tile<MASKED>(bits, words, b, kt - 1))
          for (int v = 0; v < 2; ++v, ++n) {
            const int s = n % L::NS;
            if (n >= L::NS && !mbar_wait(&misc->empty[s], (n / L::NS - 1) & 1, abort, err)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&misc->full[s], L::TILE);
            issue_tile_loads(smem + L::OFF_KV + s * L::TILE, v ? &tm_v : &tm_k, &misc->full[s], D,
                             kt * kBN, g, b);
          }
      }
    } else if (warp == kFaMma) {
      if (lane == 0 && kt0 >= 0) {
        const uint32_t id_s = idesc_f16(kBM, kBN, BF16, BF16, 0, 0);
        const uint32_t id_o = idesc_f16(kBM, D, BF16, BF16, 0, 1);
        const uint32_t q_at = smem_u32(smem + L::OFF_Q), kv_at = smem_u32(smem + L::OFF_KV);
        uint64_t* loaded = MASKED ? misc->ready : misc->full;
        int done[2] = {0, 0};   // score tiles issued
        auto pv = [&](int t, int n_v) {   // O_t += P_t V with the V tile of load n_v
          const uint32_t v_at = kv_at + (n_v % L::NS) * L::TILE;
          if (!mbar_wait(&misc->p_full[t], (done[t] - 1) & 1, abort, err)) return false;
          tc_fence_after();
  #pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk)
            umma_f16_ts(tmem + kColO + t * D, tmem + t * 128 + kk * 8, mnmajor_desc(v_at, kk), id_o,
                        (done[t] > 1 || kk > 0) ? 1u : 0u);
          return true;
        };
        bool ok = mbar_wait(&misc->q_full, 0, abort, err);
        int n = 0;
        for (int kt = kt0; ok && kt >= 0; kt = live_tile<MASKED>(bits, words, b, kt - 1), n += 2) {
          ok = mbar_wait(&loaded[n % L::NS], (n / L::NS) & 1, abort, err);
          if (ok && n > 0)
            ok = mbar_wait(&loaded[(n - 1) % L::NS], ((n - 1) / L::NS) & 1, abort, err);
          if (!ok) break;
          tc_fence_after();
          const uint32_t k_at = kv_at + (n % L::NS) * L::TILE;
  #pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (kt >= n_ct[t]) continue;
            if (done[t] > 0 && !(ok = pv(t, n - 1))) break;
  #pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_f16_ss(tmem + t * 128, kmajor_desc(q_at + t * L::TILE, kk),
                          kmajor_desc(k_at, kk), id_s, kk > 0);
            umma_commit(&misc->s_full[t]);
            ++done[t];
          }
          if (!ok) break;
          umma_commit(&misc->empty[n % L::NS]);
          if (n > 0) umma_commit(&misc->empty[(n - 1) % L::NS]);
        }
        if (ok) ok = mbar_wait(&loaded[(n - 1) % L::NS], ((n - 1) / L::NS) & 1, abort, err);
        tc_fence_after();
  #pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && done[t] > 0 && (ok = pv(t, n - 1))) umma_commit(&misc->o_full[t]);
      }
    } else if (warp == kFaCleaner) {
      if (MASKED) {
        int n = 0;
        bool ok = true;
        for (int kt = kt0; ok && kt >= 0; kt = live_tile<MASKED>(bits, words, b, kt - 1)) {
          const TileBits tb = tile_bits<MASKED>(bits, words, b, kt);
          for (int v = 0; v < 2; ++v, ++n) {
            const int s = n % L::NS;
            if (!mbar_wait(&misc->full[s], (n / L::NS) & 1, abort, err)) {
              ok = false;
              break;
            }
            if (v && !tb.all()) {
              clear_rows<D>(smem + L::OFF_KV + s * L::TILE, tb, lane);
              fence_proxy_async_smem();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&misc->ready[s]);
          }
        }
      }
    }
  } else {
    // ---------------- softmax: thread = row r of tile t
    reg_inc<kFaSoftmaxRegs>();
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;
    const int qt = wk.m * 2 + t, i = qt * kBM + r;
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float cs = p.sc * kLog2e;
    const uint64_t cs2 = f2pack(cs, cs);
    float ref = -CUDART_INF_F, l = 0.f;   // exponent offset and sum of 2^(x cs - ref)
    const int my_ct = t ? n_ct[1] : n_ct[0];
    int n = 0;
    bool ok = true;
    for (int kt = live_tile<MASKED>(bits, words, b, my_ct - 1); kt >= 0;
         kt = live_tile<MASKED>(bits, words, b, kt - 1), ++n) {
      if (!mbar_wait(&misc->s_full[t], n & 1, abort, err)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(lane_addr + t * 128 + c * 32, x[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_wait_ld_dep(x[c]);
      const TileBits tb = tile_bits<MASKED>(bits, words, b, kt);
      if ((p.causal && kt == qt) || (kt + 1) * kBN > p.T || (MASKED && !tb.all())) {
        const int lim = (p.causal ? min(i, p.T - 1) : p.T - 1) - kt * kBN;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (!(c * 32 + k <= lim && ((tb.w[c] >> k) & 1u))) x[c][k] = kMaskedScore;
      }
      float mx = x[0][0];
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < 32; k += 2) mx = fmax3(mx, x[c][k], x[c][k + 1]);
      const float m_new = fmaxf(ref, mx * cs);
      if (__any_sync(0xffffffffu, m_new > ref + kFaSlack)) {
        if (n > 0) {
          const float f = ex2(ref - m_new);
          const uint64_t f2 = f2pack(f, f);
          l *= f;
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            float o[32];
            tmem_ld32(lane_addr + kColO + t * D + c, o);
            tmem_wait_ld_dep(o);
#pragma unroll
            for (int k = 0; k < 32; k += 2)
              f2unpack(fmul2(f2pack(o[k], o[k + 1]), f2), o[k], o[k + 1]);
            tmem_st32(lane_addr + kColO + t * D + c, reinterpret_cast<uint32_t(&)[32]>(o));
          }
        }
        ref = m_new;
      }
      const uint64_t nref2 = f2pack(-ref, -ref);
      uint64_t sum2[4] = {};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float a0, a1;
          f2unpack(ffma2(f2pack(x[c][k], x[c][k + 1]), cs2, nref2), a0, a1);
          a0 = ex2(a0);
          a1 = ex2(a1);
          sum2[c] = fadd2(sum2[c], f2pack(a0, a1));
          packed[k >> 1] = pack2t<BF16>(a0, a1);
        }
        tmem_st16(lane_addr + t * 128 + c * 16, packed);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&misc->p_full[t]);
      float s0, s1;
      f2unpack(fadd2(fadd2(sum2[0], sum2[1]), fadd2(sum2[2], sum2[3])), s0, s1);
      l += s0 + s1;
    }
    if (n > 0 && ok) ok = mbar_wait(&misc->o_full[t], 0, abort, err);
    tc_fence_after();
    if (ok) {
      const bool in = i < p.T;
      const bool live = in && my_ct > 0 && token_valid(MASKED ? bits : nullptr, words, b, i);
      const float inv = live ? 1.f / l : 0.f;
      uint16_t* row = out + (size_t)b * so.b + (size_t)h * so.h + (size_t)i * so.t;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (n > 0) {
          tmem_ld32(lane_addr + kColO + t * D + c, o);
          tmem_wait_ld_dep(o);
        }
        if (!in) continue;
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          if (c + k >= p.D) break;   // head dims below 64 run zero-padded
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = live ? pack2t<BF16>(o[k + 2 * e] * inv, o[k + 2 * e + 1] * inv) : 0u;
          *reinterpret_cast<uint4*>(row + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      if (in) lse[(size_t)wk.bh * p.T + i] = live ? (ref + lg2(l)) * kLn2 : 0.f;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kFaMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Heads per band: their keys and values stay within half of L2.
int fa_band(const AttnProblem& p) {
  const long long group = 2ll * p.T * p.D * 2, G = p.Hq / p.Hkv;
  const long long groups = std::max<long long>(1, (64ll << 20) / std::max<long long>(group, 1));
  return (int)std::min<long long>(groups * G, (long long)p.B * p.Hq);
}

bool attn_map(CUtensorMap* m, const void* x, const AttnProblem& p, int H, const TensorStrides& s) {
  return make_map(m, x, p.dtype, p.D, p.T, H, p.B, s);
}

template <int D, bool BF16, bool MASKED>
cudaError_t run_attn_forward(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                             cudaStream_t st) {
  using L = FaLayout<D>;
  CUtensorMap mq, mk, mv;
  if (!attn_map(&mq, t.q, p, p.Hq, t.sq) || !attn_map(&mk, t.k, p, p.Hkv, t.sk) ||
      !attn_map(&mv, t.v, p, p.Hkv, t.sv))
    return cudaErrorInvalidValue;
  auto k = attn_sm100_forward_kernel<D, BF16, MASKED>;
  const cudaError_t e = prep(k, L::BYTES);
  if (e != cudaSuccess) return e;
  const int grid = p.B * p.Hq * ((p.T + 2 * kBM - 1) / (2 * kBM));
  k<<<grid, kFaThreads, L::BYTES, st>>>(mq, mk, mv, p, t.so, bits, static_cast<uint16_t*>(t.out),
                                        t.lse, fa_band(p));
  return cudaGetLastError();
}

bool attn_readable(const void* x, const TensorStrides& s) {
  return reinterpret_cast<uintptr_t>(x) % 16 == 0 && s.b > 0 && s.h > 0 && s.t > 0 &&
         s.b % 8 == 0 && s.h % 8 == 0 && s.t % 8 == 0;
}

}  // namespace

bool attn_sm100_supports(const AttnProblem& p, const AttnTensors& t) {
  return p.D <= 128 && attn_readable(t.q, t.sq) && attn_readable(t.k, t.sk) &&
         attn_readable(t.v, t.sv) && attn_readable(t.out, t.so);
}

cudaError_t launch_attn_sm100_forward(const AttnProblem& p, const AttnTensors& t,
                                      const uint32_t* bits, cudaStream_t st) {
  const bool bf = p.dtype == LKL_BF16;
  if (tc_dim(p.D) == 64) {
    if (bits) return bf ? run_attn_forward<64, true, true>(p, t, bits, st)
                        : run_attn_forward<64, false, true>(p, t, bits, st);
    return bf ? run_attn_forward<64, true, false>(p, t, bits, st)
              : run_attn_forward<64, false, false>(p, t, bits, st);
  }
  if (bits) return bf ? run_attn_forward<128, true, true>(p, t, bits, st)
                      : run_attn_forward<128, false, true>(p, t, bits, st);
  return bf ? run_attn_forward<128, true, false>(p, t, bits, st)
            : run_attn_forward<128, false, false>(p, t, bits, st);
}

}  // namespace lkl
