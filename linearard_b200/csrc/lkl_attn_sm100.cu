// sm_100a tensor-core attention, forward and recomputing backward.
//
// Forward: one CTA owns 256 query rows of one head as two tiles of 128 and walks the
// 128-key tiles from the diagonal down.  Per tile and key tile, two GEMMs
// (S = Q K^T, O += P V) and one exponential per score.  At head dim 128 the
// 16,384 exponentials of a tile take 1024 cycles of the SM's MUFU pipe and its
// 16 MMA steps 1024 cycles of the tensor pipe at its peak, about 1370 as they run (S reads
// 8 KB of shared memory a step, all that an SM delivers in 64 cycles), so neither may
// wait: while one tile's warpgroup computes P, the other tile's GEMMs run.
//
// Measured at 32 / 8 heads x 8192 tokens, D 128, bf16, causal: 453 to 469 us in bursts
// (1213 TFLOP/s, 73% of the measured burst peak), 530 back to back at the power cap (1.67 GHz:
// 1037 TFLOP/s, 62%); two tiles x 128 keys take some 3300 cycles: softmax 1900,
// own GEMMs 1370 behind it.  Tried and slower there: P through shared memory, so
// that S is free early (384 KB of shared memory a period: 610 against 541 us then);
// 64-key units with two score buffers a tile (766); an MMA thread a tile (679);
// the maximum beside the exponentials (540 against 530).  Head dims up to 64 leave 128 TMEM
// columns free; P (and the backward's P and dS) in columns of their own, so that the next
// scores need not wait, gained nothing there (16 heads x 8192, D 64: forward 212
// either way, backward 585 against 630 us).
//
// Warps 0-3 / 4-7: softmax of tile 0 / 1, one row a thread, so a row's maximum
// and sum need no exchange.  Warp 8: TMA producer.  Warp 9: MMA issuer and TMEM
// owner.  Warp 10: with a padding mask, clears the rows of removed tokens in the
// loaded V tiles (P is 0 there, but 0 x NaN is not).
//
// TMEM: S0, S1 (128 columns each; P, 16-bit, overwrites the first 64 of its S),
// then O0, O1.  tcgen05.mma of one thread run in order, so S_t(j+1), issued
// after O_t += P_t(j) V(j), may overwrite P_t(j), and its commit also says that
// O_t is complete up to j.
//
// Roundings: scores, statistics and every sum are fp32 (products of 16-bit inputs are
// exact in it).  P is rounded to the inputs' type because the second GEMM takes 16-bit
// operands; the row sum adds the unrounded P.  That error and the output's own rounding
// are alike in size: 0.0022 of the output in bf16, 0.0016 with the latter alone (D 128).
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
// moves only when the maximum has grown by more than this power of two.  P then
// stays below 2^slack, where its rounding is as exact as below 1.  fp16 ends at 2^16.
template <bool BF16>
constexpr float kFaSlack = BF16 ? 40.f : 8.f;

template <int D>
struct FaLayout {
  static constexpr int TILE = kBM * D * 2;      // one 128-row tile
  static constexpr int NK = D == 128 ? 2 : 4, NV = D == 128 ? 3 : 4;   // rings of K, V tiles
  static constexpr int OFF_Q = 0, OFF_K = 2 * TILE, OFF_V = OFF_K + NK * TILE;
  static constexpr int OFF_MISC = OFF_V + NV * TILE;
  static constexpr int BYTES = 1024 + OFF_MISC + kMisc;
  static_assert(BYTES <= kMaxDynSmem, "shared memory");
};

struct FaMisc {
  uint64_t q_full;
  uint64_t k_full[4], k_empty[4], v_full[4], v_ready[4], v_empty[4];
  uint64_t s_full[2], p_full[2][2], o_full[2];   // p_full: keys 0-95, 96-127
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

// 32 16-bit columns from `col` on of row r into a [128][D] tile of 128-byte
// swizzled [128][64] chunks.
__device__ __forceinline__ void stage_row32(uint8_t* tile, int r, int col,
                                            const uint32_t (&w)[16]) {
  uint8_t* row = tile + (col >> 6) * kChunk + r * 128;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    *reinterpret_cast<uint4*>(row + (((((col & 63) >> 3) + e) ^ (r & 7)) << 4)) =
        make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
  fence_proxy_async_smem();
}

// Writes a warp's 32 rows of such a tile through a map with a {64, 32} box; rows
// past T and columns past the head dim are left as they are.
template <int D>
__device__ __forceinline__ void store_rows_tma(const CUtensorMap* map, const uint8_t* tile, int w,
                                               int lane, int row0, int T, int h, int b) {
  __syncwarp();
  if (lane == 0 && row0 + w * 32 < T) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      tma_store_4d(map, tile + c * kChunk + w * 32 * 128, c * 64, row0 + w * 32, h, b);
    bulk_commit_group();
    bulk_wait_read();
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
                          const __grid_constant__ CUtensorMap tm_v,
                          const __grid_constant__ CUtensorMap tm_o, const AttnProblem p,
                          const uint32_t* __restrict__ bits, float* __restrict__ lse, int band) {
  using L = FaLayout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  FaMisc* misc = reinterpret_cast<FaMisc*>(smem + L::OFF_MISC);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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

  // The producer sets the barriers up and starts the first loads before the block meets.
  if (warp == kFaProducer && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    mbar_init(&misc->q_full, 1);
    const int users = 4 * ((n_ct[0] > 0) + (n_ct[1] > 0));   // softmax warps
    for (int s = 0; s < 4; ++s) {
      mbar_init(&misc->k_full[s], 1);
      mbar_init(&misc->k_empty[s], users);
      mbar_init(&misc->v_full[s], 1);
      mbar_init(&misc->v_ready[s], 1);
      mbar_init(&misc->v_empty[s], users);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&misc->s_full[t], 1);
      mbar_init(&misc->p_full[t][0], 4);
      mbar_init(&misc->p_full[t][1], 4);
      mbar_init(&misc->o_full[t], 1);
    }
    misc->abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    if (kt0 >= 0) {
      mbar_arrive_expect_tx(&misc->q_full, ((n_ct[0] > 0) + (n_ct[1] > 0)) * L::TILE);
      mbar_arrive_expect_tx(&misc->k_full[0], L::TILE);
      mbar_arrive_expect_tx(&misc->v_full[0], L::TILE);
      issue_tile_loads(smem + L::OFF_K, &tm_k, &misc->k_full[0], D, kt0 * kBN, g, b);
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (n_ct[t] > 0)
          issue_tile_loads(smem + L::OFF_Q + t * L::TILE, &tm_q, &misc->q_full, D,
                           (wk.m * 2 + t) * kBM, h, b);
      issue_tile_loads(smem + L::OFF_V, &tm_v, &misc->v_full[0], D, kt0 * kBN, g, b);
    }
  }
  if (warp == kFaMma) {
    tmem_alloc(&misc->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, misc->tmem_base, 0);
  constexpr uint32_t kColO = 256;

  if (warp >= 8) {
    reg_dec<kFaOtherRegs>();
    if (warp == kFaProducer) {
      if (lane == 0 && kt0 >= 0) {
        int n = 1;   // the first tiles are on their way
        for (int kt = live_tile<MASKED>(bits, words, b, kt0 - 1); kt >= 0;
             kt = live_tile<MASKED>(bits, words, b, kt - 1), ++n) {
          const int sk = n % L::NK, sv = n % L::NV;
          if (n >= L::NK && !mbar_wait(&misc->k_empty[sk], (n / L::NK - 1) & 1, abort, err)) break;
          mbar_arrive_expect_tx(&misc->k_full[sk], L::TILE);
          issue_tile_loads(smem + L::OFF_K + sk * L::TILE, &tm_k, &misc->k_full[sk], D, kt * kBN,
                           g, b);
          if (n >= L::NV && !mbar_wait(&misc->v_empty[sv], (n / L::NV - 1) & 1, abort, err)) break;
          mbar_arrive_expect_tx(&misc->v_full[sv], L::TILE);
          issue_tile_loads(smem + L::OFF_V + sv * L::TILE, &tm_v, &misc->v_full[sv], D, kt * kBN,
                           g, b);
        }
      }
    } else if (warp == kFaMma) {
      // One warp issues both tiles' GEMMs, in turns: that keeps the tiles half a period
      // apart, so that one's softmax runs under the other's GEMMs.  The tensor pipe waits
      // for this warp, so it runs the loop as one: ring positions and descriptors are
      // then the same in every lane and stay in the uniform registers that the MMA
      // instructions read.  With the loop under `lane == 0` each MMA took 75 to 95 cycles to
      // issue instead of 25 (8192 tokens: 500 us instead of 453).
      if (kt0 >= 0) {
        const uint32_t leader = elect_one();
        const uint32_t id_s = idesc_f16(kBM, kBN, BF16, BF16, 0, 0);
        const uint32_t id_o = idesc_f16(kBM, D, BF16, BF16, 0, 1);
        const uint64_t q_desc = kmajor_desc(smem_u32(smem + L::OFF_Q), 0);
        const uint64_t k_desc = kmajor_desc(smem_u32(smem + L::OFF_K), 0);
        const uint64_t v_desc = mnmajor_desc(smem_u32(smem + L::OFF_V), 0);
        constexpr uint64_t kTile = L::TILE >> 4;   // descriptors count 16 bytes
        uint64_t* v_loaded = MASKED ? misc->v_ready : misc->v_full;
        int k_slot = 0, v_slot = 0;   // ring positions of the next K and V, and their phases
        uint32_t k_phase = 0, v_phase = 0;
        auto step = [](int& slot, uint32_t& phase, int n) {
          if (++slot == n) {
            slot = 0;
            phase ^= 1;
          }
        };
        auto score = [&](int t, uint64_t kd) {   // S_t = Q_t K^T
          const uint64_t qd = q_desc + t * kTile;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = (uint64_t)((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
            umma_f16_ss_by(leader, tmem + t * 128, qd + off, kd + off, id_s, kk > 0);
          }
          umma_commit_by(leader, &misc->s_full[t]);
        };
        // O_t += P_t V, in the order in which P arrives
        auto sum = [&](int t, uint64_t vd, uint32_t parity, bool first) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (!mbar_wait_warp(&misc->p_full[t][half], parity, abort, err)) return false;
            tc_fence_after();
#pragma unroll
            for (int kk = half * 6; kk < 6 + half * 2; ++kk)
              umma_f16_ts_by(leader, tmem + kColO + t * D, tmem + t * 128 + kk * 8,
                          vd + (uint64_t)(kk * 16 * 128 >> 4), id_o,
                          (!first || kk > 0) ? 1u : 0u);
          }
          return true;
        };
        bool ok = mbar_wait_warp(&misc->q_full, 0, abort, err) &&
                  mbar_wait_warp(&misc->k_full[0], 0, abort, err);
        uint32_t par[2] = {0, 0};
        bool on[2] = {false, false}, fresh[2] = {true, true};
        if (ok) {
          tc_fence_after();
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if ((on[t] = kt0 < n_ct[t])) score(t, k_desc);
          step(k_slot, k_phase, L::NK);
        }
        int kt = kt0;
        while (ok) {
          kt = live_tile<MASKED>(bits, words, b, kt - 1);
          const bool more = kt >= 0;
          if (!(ok = mbar_wait_warp(&v_loaded[v_slot], v_phase, abort, err) &&
                     (!more || mbar_wait_warp(&misc->k_full[k_slot], k_phase, abort, err))))
            break;
          tc_fence_after();
          const uint64_t vd = v_desc + v_slot * kTile, kd = k_desc + k_slot * kTile;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && on[t]) {
              ok = sum(t, vd, par[t], fresh[t]);
              par[t] ^= 1;
              fresh[t] = false;
              if (ok && !more) umma_commit_by(leader, &misc->o_full[t]);
            }
            if (ok && more && kt < n_ct[t]) {
              score(t, kd);
              on[t] = true;
            }
          }
          if (!ok || !more) break;
          step(k_slot, k_phase, L::NK);
          step(v_slot, v_phase, L::NV);
        }
      }
    } else if (warp == kFaCleaner) {
      if (MASKED) {
        int n = 0;
        for (int kt = kt0; kt >= 0; kt = live_tile<MASKED>(bits, words, b, kt - 1), ++n) {
          const TileBits tb = tile_bits<MASKED>(bits, words, b, kt);
          const int s = n % L::NV;
          if (!mbar_wait(&misc->v_full[s], (n / L::NV) & 1, abort, err)) break;
          if (!tb.all()) {
            clear_rows<D>(smem + L::OFF_V + s * L::TILE, tb, lane);
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&misc->v_ready[s]);
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
    // Exponent offset and sum of 2^(x cs - ref).  The offset starts finite: as long as a
    // row has nothing above -inf, its exponents are -inf and not inf - inf.
    float ref = -CUDART_MAX_NORMAL_F, l = 0.f;
    const int my_ct = t ? n_ct[1] : n_ct[0];
    // rows that are not written take no part in the warp's decisions
    const bool live = i < p.T && my_ct > 0 && token_valid(MASKED ? bits : nullptr, words, b, i);
    int n = 0, skip = 0;   // key tiles taken; those before them that are the other tile's alone
    bool ok = true;
    int kt = live_tile<MASKED>(bits, words, b, my_ct - 1);
    if (my_ct > 0 && kt != kt0) {
      skip = 1;
      if (lane == 0) {
        mbar_arrive(&misc->k_empty[0]);
        mbar_arrive(&misc->v_empty[0]);
      }
    }
    for (; kt >= 0; kt = live_tile<MASKED>(bits, words, b, kt - 1), ++n) {
      if (!mbar_wait(&misc->s_full[t], n & 1, abort, err)) {
        ok = false;
        break;
      }
      tc_fence_after();
      // S(n) is complete, and with it all that was issued before: K(n) and V(n - 1) are
      // free, without commits of their own.
      if (lane == 0) {
        mbar_arrive(&misc->k_empty[(n + skip) % L::NK]);
        if (n > 0) mbar_arrive(&misc->v_empty[(n + skip - 1) % L::NV]);
      }
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
            if (!(c * 32 + k <= lim && ((tb.w[c] >> k) & 1u))) x[c][k] = -CUDART_INF_F;
      }
      float mx[8];   // eight chains: a single one would wait 64 times for the last maximum
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float* y = x[c >> 1] + (c & 1) * 16;
        mx[c] = y[0];
#pragma unroll
        for (int k = 1; k < 15; k += 2) mx[c] = fmax3(mx[c], y[k], y[k + 1]);
        mx[c] = fmaxf(mx[c], y[15]);
      }
      const float m_new = fmaxf(ref, fmaxf(fmax3(fmax3(mx[0], mx[1], mx[2]), mx[3], mx[4]),
                                           fmax3(mx[5], mx[6], mx[7])) * cs);
      if (__any_sync(0xffffffffu, live && m_new > ref + kFaSlack<BF16>)) {
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
        if (c >= 2) {   // O += P V starts with the first 96 keys
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&misc->p_full[t][c - 2]);
        }
      }
      float s0, s1;
      f2unpack(fadd2(fadd2(sum2[0], sum2[1]), fadd2(sum2[2], sum2[3])), s0, s1);
      l += s0 + s1;
    }
    if (n > 0 && ok) ok = mbar_wait(&misc->o_full[t], 0, abort, err);
    tc_fence_after();
    if (ok) {
      const bool in = i < p.T;
      const float inv = live ? 1.f / l : 0.f;
      // through the query tile's shared memory, which no GEMM reads any more
      uint8_t* const tile = smem + L::OFF_Q + t * L::TILE;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (n > 0) {
          tmem_ld32(lane_addr + kColO + t * D + c, o);
          tmem_wait_ld_dep(o);
        }
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2)
          w[k >> 1] = live ? pack2t<BF16>(o[k] * inv, o[k + 1] * inv) : 0u;
        stage_row32(tile, r, c, w);
      }
      store_rows_tma<D>(&tm_o, tile, warp & 3, lane, qt * kBM, p.T, h, b);
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

bool attn_map(CUtensorMap* m, const void* x, const AttnProblem& p, int H, const TensorStrides& s,
              int box_rows = kBM) {
  return make_map(m, x, p.dtype, p.D, p.T, H, p.B, s, box_rows);
}

template <int D, bool BF16, bool MASKED>
cudaError_t run_attn_forward(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                             cudaStream_t st) {
  using L = FaLayout<D>;
  CUtensorMap mq, mk, mv, mo;
  if (!attn_map(&mq, t.q, p, p.Hq, t.sq) || !attn_map(&mk, t.k, p, p.Hkv, t.sk) ||
      !attn_map(&mv, t.v, p, p.Hkv, t.sv) || !attn_map(&mo, t.out, p, p.Hq, t.so, 32))
    return cudaErrorInvalidValue;
  auto k = attn_sm100_forward_kernel<D, BF16, MASKED>;
  const cudaError_t e = prep(k, L::BYTES);
  if (e != cudaSuccess) return e;
  const int grid = p.B * p.Hq * ((p.T + 2 * kBM - 1) / (2 * kBM));
  k<<<grid, kFaThreads, L::BYTES, st>>>(mq, mk, mv, mo, p, bits, t.lse, fa_band(p));
  return cudaGetLastError();
}

// ============================================================== backward
// Two launches per chunk of the dS buffer and no reductions.
//
// dkv launch (key-stationary): one CTA owns 128 keys of one kv head and walks
// the query tiles of the group's heads.  Scores are computed transposed (lanes
// = keys, columns = queries), so that P^T and dS^T, written to TMEM as 16-bit
// values, are the A operands of dV += P^T dO and dK += dS^T Q.  dS^T also goes to
// the dS buffer in HBM.
// dq launch (persistent GEMM): dq_i = sm_scale sum_j dS_ij K_j from that buffer.
//
// The hand-over costs 32 KB of HBM writes and reads a tile pair (10 ns of the
// whole GPU) and saves the second recomputation of S and dP: two GEMMs and
// 16,384 exponentials.  Reducing dq in L2 instead would move 64 KB of fp32 a
// pair, in an order that changes from run to run.
//
// Bound of the dkv launch: the tensor pipe, 32 MMA steps a tile pair (2048 cycles at the
// peak, some 3000 as they run) against 1024 cycles of exponentials.  Measured at
// 32 / 8 heads x 8192 tokens, D 128, causal: a pair every 3100 cycles, and as long without
// any exponential, TMEM access or TMA load; 4211 when one lane issued and eight row
// warps had 64 queries each.  The issue order dV(i), S(i+1), dK(i), dP(i+1) keeps the
// pipe busy: dS(i) is computed under dV(i) and S(i+1), P(i+1) under dK(i) and dP(i+1).
// All 512 TMEM columns are in use (S, dP, dV, dK at head dim 128; P and dS overwrite
// part of what they come from).  The dq launch reads dS at the copy rate (286 us for
// 1.84 GB at 8 heads x 15001).
//
// Roundings: P and dS are rounded to the inputs' type, the only one that the GEMMs take,
// and dS is handed over as rounded, which halves the dq launch's bytes.  The gradients
// carry that error beside their result's own: at D 64 and 128 0.0024 of their size in bf16
// instead of 0.0017, 0.0003 instead of 0.0002 in fp16.  dS as a sum of two 16-bit values would
// take that back for a third more MMA steps and twice the hand-over.
//
// Sixteen row warps, 32 queries of 128 each (eight warps with 64 queries left the
// exponentials of a tile at 1800 cycles for want of independent work).  P is handed
// over in two parts, so that half of dV's GEMM runs under its second part.
constexpr int kFbRowWarps = 16;
constexpr int kFbThreads = 640;
constexpr int kFbProducer = 16, kFbMma = 17, kFbCleaner = 18, kFbStats = 19;
// Registers a thread of the five warpgroups: 96 at launch
constexpr int kFbRegs = 96, kFbRowRegs = 104, kFbOtherRegs = 64;
static_assert(4 * kFbRowRegs + kFbOtherRegs <= 5 * kFbRegs, "register split");
static_assert(kFbThreads * kFbRegs <= 65536, "register file");

// One backward chunk: kv groups [g0, g1), key tiles [j0, j1).  `split`: not all
// key tiles, so that dq is summed over launches in fp32.
struct FbChunk {
  int g0, g1, j0, j1;
  int split;
  int band;            // kv groups per band of work items
  int parts;           // CTAs that share a key tile (its query tiles in turn)
  long long tph;       // dS tiles per query head
};

__host__ __device__ __forceinline__ long long fb_tile(const FbChunk& c, int causal, int n_t, int i,
                                                      int j) {
  if (c.split) return (long long)(i - (causal ? c.j0 : 0)) * (c.j1 - c.j0) + (j - c.j0);
  return causal ? (long long)i * (i + 1) / 2 + j : (long long)i * n_t + j;
}

// Query rows' statistics as the dkv launch reads them: per (head, query tile)
// 128 exponent offsets -lse log2(e) (-inf for a row without gradient), then
// 128 delta_i.
constexpr int kFbStatBytes = 2 * kBM * 4;

// c += A B for 16 rows x 16 x 8 columns, fp32 sums of 16-bit products.
template <bool BF16>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The 16-bit values 32 c + 8 (lane % 4) .. + 7 of a row of p.D, zeros past its end, for
// c < NC.  A contraction may take its terms in any order, as long as both operands take
// the same: words 0 and 1 are one step of 16, words 2 and 3 the next.
template <int NC>
__device__ __forceinline__ void load_fragment_row(uint4 (&x)[NC], const void* base, size_t at,
                                                  bool on, int D) {
  const int e = (threadIdx.x & 3) * 8;
#pragma unroll
  for (int c = 0; c < NC; ++c)
    x[c] = on && 32 * c + e < D
               ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at + 32 * c + e)
               : make_uint4(0u, 0u, 0u, 0u);
}

// delta_i = sum_j P_ij (dout_i . v_j) for 16 rows from `first` on, straight from global
// memory: a head's few keys come from L1 and L2, and 256 x 256 x D products a head are too
// few for staging tiles and TMEM to pay.  The eight warps take 8 keys each in turn, at
// most four times, and are joined in their order.  Bound by the latency of those
// steps: 11.8 us for the 256 rows of 32 heads, D 128.
//
// pos == nullptr: rows and keys by position.  Otherwise they are ranks among the n
// tokens at pos[], which the mask keeps.  stats: the head's.
template <int D, bool BF16>
__device__ __forceinline__ void exact_delta_rows(const AttnProblem& p, const AttnTensors& a,
                                                 const uint32_t* bits, int b, int h, int first,
                                                 const int* pos, int n, float* stats) {
  constexpr int NC = D / 32;
  __shared__ float part[8][16];
  const int words = (p.T + 31) >> 5, lane = threadIdx.x & 31, quad = lane >> 2;
  const int warp = threadIdx.x >> 5, r0 = first + quad, r1 = r0 + 8;
  auto token = [&](int r) { return pos && r < n ? pos[r] : r; };
  auto kept = [&](int r) { return r < n && (pos || token_valid(bits, words, b, r)); };
  const int i0 = token(r0), i1 = token(r1);
  const bool on0 = kept(r0), on1 = kept(r1);
  const float* lse = a.lse + ((size_t)b * p.Hq + h) * p.T;
  const float z0 = on0 ? -lse[i0] * kLog2e : -CUDART_INF_F;
  const float z1 = on1 ? -lse[i1] * kLog2e : -CUDART_INF_F;
  const size_t q = (size_t)b * a.sq.b + (size_t)h * a.sq.h;
  const size_t g = (size_t)b * a.sdo.b + (size_t)h * a.sdo.h;
  uint4 q0[NC], q1[NC], g0[NC], g1[NC];
  load_fragment_row(q0, a.q, q + (size_t)i0 * a.sq.t, on0, p.D);
  load_fragment_row(q1, a.q, q + (size_t)i1 * a.sq.t, on1, p.D);
  load_fragment_row(g0, a.dout, g + (size_t)i0 * a.sdo.t, on0, p.D);
  load_fragment_row(g1, a.dout, g + (size_t)i1 * a.sdo.t, on1, p.D);
  const int kv = h / (p.Hq / p.Hkv);
  const size_t kb = (size_t)b * a.sk.b + (size_t)kv * a.sk.h;
  const size_t vb = (size_t)b * a.sv.b + (size_t)kv * a.sv.h;
  const int keys = first >= n ? 0 : p.causal ? min(n, first + 16) : n;
  const float sl = p.sc * kLog2e;
  float d0 = 0.f, d1 = 0.f;
  for (int j = warp * 8; j < keys; j += 64) {
    const int row = token(j + quad);
    uint4 k[NC], v[NC];
    load_fragment_row(k, a.k, kb + (size_t)row * a.sk.t, j + quad < n, p.D);
    load_fragment_row(v, a.v, vb + (size_t)row * a.sv.t, j + quad < n, p.D);
    float s[4] = {}, x[4] = {};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      mma_16x8x16<BF16>(s, q0[c].x, q1[c].x, q0[c].y, q1[c].y, k[c].x, k[c].y);
      mma_16x8x16<BF16>(s, q0[c].z, q1[c].z, q0[c].w, q1[c].w, k[c].z, k[c].w);
      mma_16x8x16<BF16>(x, g0[c].x, g1[c].x, g0[c].y, g1[c].y, v[c].x, v[c].y);
      mma_16x8x16<BF16>(x, g0[c].z, g1[c].z, g0[c].w, g1[c].w, v[c].z, v[c].w);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = j + 2 * (lane & 3) + e;
      if (kept(col)) {
        if (on0 && (!p.causal || col <= r0)) d0 = fmaf(exp2f(fmaf(s[e], sl, z0)), x[e], d0);
        if (on1 && (!p.causal || col <= r1)) d1 = fmaf(exp2f(fmaf(s[e + 2], sl, z1)), x[e + 2], d1);
      }
    }
    __syncwarp();   // the next step's products take the whole warp
  }
  for (int o = 1; o < 4; o <<= 1) {
    d0 += __shfl_xor_sync(0xffffffffu, d0, o);
    d1 += __shfl_xor_sync(0xffffffffu, d1, o);
  }
  // by position, the tile's rows past T are set too: the dk/dv launch reads whole tiles
  auto at = [&](int i) { return stats + (size_t)(i / kBM) * 2 * kBM + i % kBM; };
  if ((lane & 3) == 0) {
    part[warp][quad] = d0;
    part[warp][quad + 8] = d1;
    if (warp == 0) {
      if (!pos || on0) *at(i0) = z0;
      if (!pos || on1) *at(i1) = z1;
    }
  }
  __syncthreads();
  if (threadIdx.x < 16 && (!pos || first + (int)threadIdx.x < n)) {
    float d = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) d += part[w][threadIdx.x];
    at(token(first + threadIdx.x))[kBM] = d;
  }
}

// Query tiles that are known by position to see at most kExactDeltaKeys keys, the first of
// a head.  None where they are found by rank: those rows replace what the launch below wrote.
__host__ __device__ __forceinline__ int exact_delta_tiles(const AttnProblem& p, bool ranked) {
  const int n_t = (p.T + kBM - 1) / kBM;
  return ranked ? 0 : p.T <= kExactDeltaKeys ? n_t : p.causal ? kExactDeltaKeys / kBM : 0;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(256, 2)
attn_sm100_exact_delta_kernel(const AttnProblem p, const AttnTensors a,
                              const uint32_t* __restrict__ bits, float* __restrict__ stats) {
  const int n_t = (p.T + kBM - 1) / kBM, units = exact_delta_tiles(p, false) * (kBM / 16);
  const int bh = blockIdx.x / units, first = blockIdx.x % units * 16;
  exact_delta_rows<D, BF16>(p, a, bits, bh / p.Hq, bh % p.Hq, first, nullptr, p.T,
                            stats + (size_t)bh * n_t * 2 * kBM);
}

// The rows found by rank; a block takes 16 of a head's up to kExactDeltaKeys.
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 2)
attn_sm100_exact_delta_ranked_kernel(const AttnProblem p, const AttnTensors a,
                                     const uint32_t* __restrict__ bits,
                                     float* __restrict__ stats) {
  constexpr int kUnits = kExactDeltaKeys / 16;
  __shared__ int pos[kExactDeltaKeys], sums[8];
  const int bh = blockIdx.x / kUnits, first = blockIdx.x % kUnits * 16, b = bh / p.Hq;
  const int n = few_key_tokens(bits, p, b, pos, sums);
  if (first >= n) return;
  exact_delta_rows<D, BF16>(p, a, bits, b, bh % p.Hq, first, pos, n,
                            stats + (size_t)bh * ((p.T + kBM - 1) / kBM) * 2 * kBM);
}

// The other tiles, one a block: delta_i = dout_i . out_i, D / 8 neighbouring lanes a row.
// Bound by HBM: 64 MB of 32 heads x 4096, D 128 in 14.1 us (4.7 TB/s; 17.5 with one row's
// loads at a time).  A launch of its own, since the 126 registers of the above leave too
// few warps to read with: both in one launch took 34 us there.
__global__ void __launch_bounds__(256)
attn_sm100_delta_kernel(const AttnProblem p, const AttnTensors a,
                        const uint32_t* __restrict__ bits, float* __restrict__ stats, int few) {
  const int n_t = (p.T + kBM - 1) / kBM, words = (p.T + 31) >> 5;
  const int bh = blockIdx.x / (n_t - few), qt = few + blockIdx.x % (n_t - few);
  const int b = bh / p.Hq, h = bh % p.Hq, lanes = p.D / 8, sub = threadIdx.x % lanes;
  float* dst = stats + ((size_t)bh * n_t + qt) * 2 * kBM;
  const uint16_t* out = static_cast<const uint16_t*>(a.out) + (size_t)b * a.so.b +
                        (size_t)h * a.so.h + sub * 8;
  const uint16_t* dout = static_cast<const uint16_t*>(a.dout) + (size_t)b * a.sdo.b +
                         (size_t)h * a.sdo.h + sub * 8;
  // four rows at a time, all loads before the first use
  for (int r0 = threadIdx.x / lanes; r0 < kBM; r0 += 4 * (256 / lanes)) {
    uint4 x[4], y[4];
    float z[4];
    bool on[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + k * (256 / lanes), i = qt * kBM + r;
      on[k] = r < kBM && i < p.T && token_valid(bits, words, b, i);
      x[k] = y[k] = make_uint4(0u, 0u, 0u, 0u);
      z[k] = CUDART_INF_F;
      if (on[k]) {
        x[k] = *reinterpret_cast<const uint4*>(out + (size_t)i * a.so.t);
        y[k] = *reinterpret_cast<const uint4*>(dout + (size_t)i * a.sdo.t);
        if (sub == 0) z[k] = a.lse[(size_t)bh * p.T + i];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + k * (256 / lanes);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s = fmaf(load_elem(&x[k], e, p.dtype), load_elem(&y[k], e, p.dtype), s);
      for (int o = lanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (sub == 0 && r < kBM) {
        dst[r] = -z[k] * kLog2e;
        dst[kBM + r] = s;
      }
    }
  }
}

template <int D>
struct FbLayout {
  static constexpr int TILE = kBM * D * 2;
  static constexpr int NS = D == 128 ? 5 : 8;   // ring of Q and dO tiles
  static constexpr int OFF_K = 0, OFF_V = TILE, OFF_RING = 2 * TILE;
  static constexpr int OFF_MISC = OFF_RING + NS * TILE;
  static constexpr int MISC = 512;
  // statistics: exponent offsets of two query tiles, delta of one
  static constexpr int OFF_LSE = OFF_MISC + MISC, OFF_DELTA = OFF_LSE + kFbStatBytes;
  static constexpr int BYTES = 1024 + OFF_DELTA + kFbStatBytes / 2;
  static_assert(BYTES <= kMaxDynSmem, "shared memory");
};

struct FbMisc {
  uint64_t kv_full;
  uint64_t full[8], ready[8], empty[8];
  uint64_t lse_full[2], lse_empty[2], delta_full, delta_empty;
  uint64_t s_full, p_full[2], dp_full, ds_full, acc_full;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(FbMisc) <= 512, "misc region too small");

// The (query head, query tile) pairs of a dkv CTA, in the order every role takes
// them: of each head the tiles first_, first_ + step, ... that have a token.
template <bool MASKED>
struct FbWalk {
  const uint32_t* bits;
  int words, b, n_t, step, first, h, h_end, i;
  __device__ __forceinline__ FbWalk(const uint32_t* bits_, int words_, int b_, int n_t_, int first_,
                                    int step_, int h0, int G)
      : bits(bits_), words(words_), b(b_), n_t(n_t_), step(step_), h(h0), h_end(h0 + G) {
    first = live(first_);
    i = first;
    if (first >= n_t) h = h_end;
  }
  __device__ __forceinline__ int live(int t) const {
    if (MASKED)
      while (t < n_t && !tile_bits<true>(bits, words, b, t).any()) t += step;
    return t;
  }
  __device__ __forceinline__ bool on() const { return h < h_end; }
  __device__ __forceinline__ void next() {
    i = live(i + step);
    if (i >= n_t) {
      i = first;
      ++h;
    }
  }
};

template <int D, bool BF16, bool MASKED>
__global__ void __launch_bounds__(kFbThreads, 1)
attn_sm100_dkv_kernel(const __grid_constant__ CUtensorMap tm_q,
                      const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_do,
                      const __grid_constant__ CUtensorMap tm_dk,
                      const __grid_constant__ CUtensorMap tm_dv, const AttnProblem p,
                      const FbChunk c, const uint32_t* __restrict__ bits,
                      const float* __restrict__ stats, uint16_t* __restrict__ dsbuf,
                      float* __restrict__ sums) {
  using L = FbLayout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  FbMisc* misc = reinterpret_cast<FbMisc*>(smem + L::OFF_MISC);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  int* err = &g_device_error;
  volatile int* abort = &misc->abort;
  constexpr uint32_t kColDp = 128, kColDv = 256, kColDk = 256 + D;

  const int n_t = (p.T + kBM - 1) / kBM, words = (p.T + 31) >> 5, G = p.Hq / p.Hkv;
  // bands of kv groups, key tiles ascending (the longest first when causal)
  const int part = (int)(blockIdx.x % c.parts);
  int lg, j;
  {
    const int n_j = c.j1 - c.j0, n_g = c.g1 - c.g0, blk = (int)(blockIdx.x / c.parts);
    const int k = blk / (c.band * n_j), r = blk % (c.band * n_j);
    const int size = min(c.band, n_g - k * c.band);
    lg = k * c.band + r % size;
    j = c.j0 + r / size;
  }
  const int grp = c.g0 + lg, b = grp / p.Hkv, g = grp % p.Hkv;
  const TileBits keys = tile_bits<MASKED>(bits, words, b, j);
  const FbWalk<MASKED> walk0(bits, words, b, n_t, (p.causal ? j : 0) + part, c.parts, g * G,
                             keys.any() ? G : 0);

  // The producer sets the barriers up and starts the first loads before the block meets.
  if (warp == kFbProducer && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_do);
    mbar_init(&misc->kv_full, 1);
    for (int s = 0; s < L::NS; ++s) {
      mbar_init(&misc->full[s], 1);
      mbar_init(&misc->ready[s], 1);
      mbar_init(&misc->empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&misc->lse_full[s], 1);
      mbar_init(&misc->lse_empty[s], kFbRowWarps);
      mbar_init(&misc->p_full[s], kFbRowWarps);
    }
    mbar_init(&misc->delta_full, 1);
    mbar_init(&misc->delta_empty, kFbRowWarps);
    mbar_init(&misc->s_full, 1);
    mbar_init(&misc->dp_full, 1);
    mbar_init(&misc->ds_full, kFbRowWarps);
    mbar_init(&misc->acc_full, 1);
    misc->abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    if (walk0.on()) {
      mbar_arrive_expect_tx(&misc->kv_full, 2 * L::TILE);
      issue_tile_loads(smem + L::OFF_K, &tm_k, &misc->kv_full, D, j * kBN, g, b);
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        mbar_arrive_expect_tx(&misc->full[o], L::TILE);
        issue_tile_loads(smem + L::OFF_RING + o * L::TILE, o ? &tm_do : &tm_q, &misc->full[o], D,
                         walk0.i * kBM, walk0.h, b);
        if (o == 0) issue_tile_loads(smem + L::OFF_V, &tm_v, &misc->kv_full, D, j * kBN, g, b);
      }
    }
  }
  if (warp == kFbMma) {
    tmem_alloc(&misc->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, misc->tmem_base, 0);

  if (warp >= kFbRowWarps) {
    reg_dec<kFbOtherRegs>();
    if (warp == kFbProducer) {
      if (lane == 0 && walk0.on()) {
        int n = 2;   // Q(0), dO(0), which are on their way, Q(1), dO(1), ...
        bool ok = true;
        FbWalk<MASKED> w = walk0;
        for (w.next(); ok && w.on(); w.next())
          for (int o = 0; o < 2; ++o, ++n) {
            const int s = n % L::NS;
            if (n >= L::NS && !mbar_wait(&misc->empty[s], (n / L::NS - 1) & 1, abort, err)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&misc->full[s], L::TILE);
            issue_tile_loads(smem + L::OFF_RING + s * L::TILE, o ? &tm_do : &tm_q,
                             &misc->full[s], D, w.i * kBM, w.h, b);
          }
      }
    } else if (warp == kFbStats) {
      if (lane == 0 && walk0.on()) {
        constexpr int kHalf = kFbStatBytes / 2;
        auto src = [&](const FbWalk<MASKED>& w) {
          return stats + ((size_t)(b * p.Hq + w.h) * n_t + w.i) * 2 * kBM;
        };
        auto load_lse = [&](const FbWalk<MASKED>& w, int it) {
          const int e = it & 1;
          if (it >= 2 && !mbar_wait(&misc->lse_empty[e], ((it >> 1) - 1) & 1, abort, err))
            return false;
          mbar_arrive_expect_tx(&misc->lse_full[e], kHalf);
          bulk_load(smem + L::OFF_LSE + e * kHalf, src(w), kHalf, &misc->lse_full[e]);
          return true;
        };
        FbWalk<MASKED> w = walk0;
        bool ok = load_lse(w, 0);
        for (int it = 0; ok && w.on(); ++it) {
          if (it >= 1 && !mbar_wait(&misc->delta_empty, (it - 1) & 1, abort, err)) break;
          mbar_arrive_expect_tx(&misc->delta_full, kHalf);
          bulk_load(smem + L::OFF_DELTA, src(w) + kBM, kHalf, &misc->delta_full);
          w.next();
          if (w.on()) ok = load_lse(w, it + 1);
        }
      }
    } else if (warp == kFbMma) {
      // the whole warp runs the loop, so that descriptors stay in uniform registers; one
      // lane issues
      if (walk0.on()) {
        const uint32_t leader = elect_one();
        const uint32_t id_s = idesc_f16(kBM, kBN, BF16, BF16, 0, 0);
        const uint32_t id_g = idesc_f16(kBM, D, BF16, BF16, 0, 1);
        const uint64_t k_desc = kmajor_desc(smem_u32(smem + L::OFF_K), 0);
        const uint64_t v_desc = kmajor_desc(smem_u32(smem + L::OFF_V), 0);
        const uint64_t km_desc = kmajor_desc(smem_u32(smem + L::OFF_RING), 0);
        const uint64_t mn_desc = mnmajor_desc(smem_u32(smem + L::OFF_RING), 0);
        constexpr uint64_t kTile = L::TILE >> 4;   // descriptors count 16 bytes
        uint64_t* loaded = MASKED ? misc->ready : misc->full;
        int slot = 0;            // ring position of the next load, and its phase
        uint32_t phase = 0;
        auto take = [&] {        // waits for the next load; its position, or -1
          const int at = slot;
          const bool got = mbar_wait_warp(&loaded[slot], phase, abort, err);
          if (++slot == L::NS) {
            slot = 0;
            phase ^= 1;
          }
          tc_fence_after();
          return got ? at : -1;
        };
        // S^T = K Q^T (ring tile: Q) and dP^T = V dO^T (ring tile: dO)
        auto scores = [&](uint64_t ad, int at, uint32_t col, uint64_t* bar) {
          const uint64_t bd = km_desc + at * kTile;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t off = (uint64_t)((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
            umma_f16_ss_by(leader, tmem + col, ad + off, bd + off, id_s, kk > 0);
          }
          umma_commit_by(leader, bar);
        };
        // One 16-query step of acc += A^T-from-TMEM x ring tile; the 32 queries of
        // warpgroup w have their 16-bit values from column 32 w on
        auto grad = [&](int at, uint32_t acc, uint32_t col, int kk, bool start) {
          umma_f16_ts_by(leader, tmem + acc, tmem + col + (kk >> 1) * 32 + (kk & 1) * 8,
                      mn_desc + at * kTile + (uint64_t)(kk * 16 * 128 >> 4), id_g, start ? 0u : 1u);
        };
        bool ok = mbar_wait_warp(&misc->kv_full, 0, abort, err);
        int q_at = ok ? take() : -1, do_at = -1;
        if ((ok = q_at >= 0)) {
          scores(k_desc, q_at, 0, &misc->s_full);
          do_at = take();
          if ((ok = do_at >= 0)) scores(v_desc, do_at, kColDp, &misc->dp_full);
        }
        uint32_t par = 0;
        bool first = true;
        FbWalk<MASKED> w = walk0;
        while (ok) {
          w.next();
          const bool more = w.on();
          for (int part = 0; part < 2; ++part) {
            if (!(ok = mbar_wait_warp(&misc->p_full[part], par, abort, err))) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k)
              grad(do_at, kColDv, 0, 2 * k + part, first && part == 0 && k == 0);
          }
          if (!ok) break;
          umma_commit_by(leader, &misc->empty[do_at]);
          int q_next = 0;
          if (more) {
            if (!(ok = (q_next = take()) >= 0)) break;
            scores(k_desc, q_next, 0, &misc->s_full);
          }
          if (!(ok = mbar_wait_warp(&misc->ds_full, par, abort, err))) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 8; ++k) grad(q_at, kColDk, kColDp, k, first && k == 0);
          umma_commit_by(leader, &misc->empty[q_at]);
          if (!more) break;
          q_at = q_next;
          if (!(ok = (do_at = take()) >= 0)) break;
          scores(v_desc, do_at, kColDp, &misc->dp_full);
          par ^= 1;
          first = false;
        }
        if (ok) umma_commit_by(leader, &misc->acc_full);
      }
    } else if (warp == kFbCleaner) {
      if (MASKED) {
        int n = 0;
        bool ok = true;
        for (FbWalk<MASKED> w = walk0; ok && w.on(); w.next()) {
          const TileBits tb = tile_bits<MASKED>(bits, words, b, w.i);
          for (int o = 0; o < 2; ++o, ++n) {
            const int s = n % L::NS;
            if (!mbar_wait(&misc->full[s], (n / L::NS) & 1, abort, err)) {
              ok = false;
              break;
            }
            if (!tb.all()) {
              clear_rows<D>(smem + L::OFF_RING + s * L::TILE, tb, lane);
              fence_proxy_async_smem();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&misc->ready[s]);
          }
        }
      }
    }
  } else {
    reg_inc<kFbRowRegs>();
    // ---------------- thread = key r; warpgroup wg owns 32 of the tile's 128 queries
    const int wg = warp >> 2, r = (warp & 3) * 32 + lane, key = j * kBN + r;
    const uint32_t row_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t lane_addr = row_addr + wg * 32;
    const float cs = p.sc * kLog2e;
    const uint64_t cs2 = f2pack(cs, cs);
    const bool key_ok = key < p.T && ((keys.w[warp & 3] >> lane) & 1u);
    uint4* const buf = reinterpret_cast<uint4*>(dsbuf) + (size_t)(wg * 4) * kBM + r;
    const float* const dl = reinterpret_cast<const float*>(smem + L::OFF_DELTA) + wg * 32;
    int it = 0;
    bool ok = true;
    for (FbWalk<MASKED> w = walk0; w.on(); w.next(), ++it) {
      const float* nl =
          reinterpret_cast<const float*>(smem + L::OFF_LSE + (it & 1) * (kFbStatBytes / 2)) +
          wg * 32;
      if (!mbar_wait(&misc->lse_full[it & 1], (it >> 1) & 1, abort, err) ||
          !mbar_wait(&misc->s_full, it & 1, abort, err)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float pr[32];
      tmem_ld32(lane_addr, pr);
      tmem_wait_ld_dep(pr);
      // causal: a query before this key takes no part (the diagonal tile only)
      const int from = p.causal && w.i == j ? r - wg * 32 : 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float* x = pr + half * 16;
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
          const float4 z = *reinterpret_cast<const float4*>(nl + half * 16 + k);
          f2unpack(ffma2(f2pack(x[k], x[k + 1]), cs2, f2pack(z.x, z.y)), x[k], x[k + 1]);
          f2unpack(ffma2(f2pack(x[k + 2], x[k + 3]), cs2, f2pack(z.z, z.w)), x[k + 2], x[k + 3]);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = ex2(x[k]);
        if (!key_ok || from > 0) {
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (!key_ok || half * 16 + k < from) x[k] = 0.f;
        }
        uint32_t packed[8];
#pragma unroll
        for (int k = 0; k < 16; k += 2) packed[k >> 1] = pack2t<BF16>(x[k], x[k + 1]);
        tmem_st8(lane_addr + half * 8, packed);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&misc->p_full[half]);
          if (half == 1) mbar_arrive(&misc->lse_empty[it & 1]);
        }
      }

      if (!mbar_wait(&misc->delta_full, it & 1, abort, err) ||
          !mbar_wait(&misc->dp_full, it & 1, abort, err)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t ds[16];
      {
        float x[32];
        tmem_ld32(lane_addr + kColDp, x);
        tmem_wait_ld_dep(x);
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 z = *reinterpret_cast<const float4*>(dl + k);
          f2unpack(fmul2(f2pack(pr[k], pr[k + 1]),
                         fsub2(f2pack(x[k], x[k + 1]), f2pack(z.x, z.y))), x[k], x[k + 1]);
          f2unpack(fmul2(f2pack(pr[k + 2], pr[k + 3]),
                         fsub2(f2pack(x[k + 2], x[k + 3]), f2pack(z.z, z.w))), x[k + 2], x[k + 3]);
        }
        if (MASKED && !key_ok) {   // 0 x what the removed key's v holds
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 32; k += 2) ds[k >> 1] = pack2t<BF16>(x[k], x[k + 1]);
      }
      tmem_st16(lane_addr + kColDp, ds);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&misc->ds_full);
        mbar_arrive(&misc->delta_empty);
      }
      // 16 groups of 8 queries, each [128 keys][16 bytes]: the no-swizzle core-matrix
      // layout that the dq GEMM reads; a warp's store covers 512 contiguous bytes
      const long long head = (long long)lg * G + (w.h - g * G);
      uint4* dst = buf + (size_t)(head * c.tph + fb_tile(c, p.causal, n_t, w.i, j)) *
                             (kDTileElems / 8);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        dst[k * kBM] = make_uint4(ds[4 * k], ds[4 * k + 1], ds[4 * k + 2], ds[4 * k + 3]);
    }
    if (ok && it > 0) ok = mbar_wait(&misc->acc_full, 0, abort, err);
    tc_fence_after();
    if (ok) {
      // warpgroups 0 and 1 write dv, 2 and 3 dk (half of the columns each), through the
      // tiles of V and K, which no GEMM reads any more
      const int which = wg >> 1, col0 = (wg & 1) * (D / 2);
      uint8_t* const tile = smem + (which ? L::OFF_K : L::OFF_V);
      const float scale = which ? p.sc : 1.f;
      const bool live = key_ok && it > 0;
      // several CTAs a key tile: this one's fp32 sums, [part][dv, dk][group][T][D]
      float* const sum_row =
          sums + ((((size_t)part * 2 + which) * (c.g1 - c.g0) + lg) * p.T + key) * p.D;
#pragma unroll
      for (int c2 = 0; c2 < D / 2; c2 += 32) {
        float v[32];
        tmem_ld32(row_addr + (which ? kColDk : kColDv) + col0 + c2, v);
        tmem_wait_ld_dep(v);
        if (c.parts > 1) {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            if (key < p.T && col0 + c2 + k < p.D)
              *reinterpret_cast<float4*>(sum_row + col0 + c2 + k) =
                  live ? make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]) : make_float4(0, 0, 0, 0);
          __syncwarp();   // the next step's TMEM load takes the whole warp
          continue;
        }
        uint32_t u[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2)
          u[k >> 1] = live ? pack2t<BF16>(v[k] * scale, v[k + 1] * scale) : 0u;
        stage_row32(tile, r, col0 + c2, u);
      }
      named_bar(1 + which, 256);
      if ((wg & 1) == 0 && c.parts == 1)
        store_rows_tma<D>(which ? &tm_dk : &tm_dv, tile, warp & 3, lane, j * kBN, p.T, g, b);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kFbMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// dk and dv of key rows [j0, j1) * 128 of a chunk: the parts' sums in their order, rounded.
template <bool BF16>
__global__ void __launch_bounds__(256)
attn_sm100_sum_parts_kernel(const AttnProblem p, const AttnTensors a, const FbChunk c,
                            const float* __restrict__ sums) {
  const int n8 = p.D / 8, r0 = c.j0 * kBN, rows = min(p.T, c.j1 * kBN) - r0, n_g = c.g1 - c.g0;
  const long long total = 2ll * n_g * rows * n8;
  for (long long x = blockIdx.x * 256ll + threadIdx.x; x < total; x += gridDim.x * 256ll) {
    const int col = (int)(x % n8) * 8;
    const long long y = x / n8;
    const int key = r0 + (int)(y % rows), lg = (int)(y / rows) % n_g, which = (int)(y / rows / n_g);
    float v[8] = {};
    for (int part = 0; part < c.parts; ++part) {
      const float4* from = reinterpret_cast<const float4*>(
          sums + ((((size_t)part * 2 + which) * n_g + lg) * p.T + key) * p.D + col);
      const float4 lo = from[0], hi = from[1];
      v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
      v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
    }
    const float sc = which ? p.sc : 1.f;
    const int grp = c.g0 + lg, b = grp / p.Hkv, g = grp % p.Hkv;
    const TensorStrides& st = which ? a.sdk : a.sdv;
    uint16_t* row = static_cast<uint16_t*>(which ? a.dk : a.dv) + (size_t)b * st.b +
                    (size_t)g * st.h + (size_t)key * st.t + col;
    *reinterpret_cast<uint4*>(row) =
        make_uint4(pack2t<BF16>(v[0] * sc, v[1] * sc), pack2t<BF16>(v[2] * sc, v[3] * sc),
                   pack2t<BF16>(v[4] * sc, v[5] * sc), pack2t<BF16>(v[6] * sc, v[7] * sc));
  }
}

// dq launch: a pipelined GEMM, one persistent CTA per SM.  Work item = (query
// head, query tile i): dq_i = sm_scale sum_j dS_ij K_j.  A = dS (one bulk copy of a
// stored tile, no swizzle, MN-major), B = K (TMA, 128-byte swizzle, MN-major).
// Bound by HBM: 32 KB of dS for 4.2 MFLOP.  Two accumulators, so that an item's
// epilogue runs under the next item's GEMM.
constexpr int kFqThreads = 224;   // producer, MMA, cleaner, four epilogue warps

template <int D>
struct FqLayout {
  static constexpr int DS_BYTES = kDTileElems * 2, K_BYTES = kBM * D * 2;
  static constexpr int STAGE = DS_BYTES + K_BYTES;
  static constexpr int NS = D == 128 ? 3 : 4;
  static constexpr int OFF_MISC = NS * STAGE;
  static constexpr int BYTES = 1024 + OFF_MISC + kMisc;
  static_assert(BYTES <= kMaxDynSmem, "shared memory");
};

struct FqMisc {
  uint64_t full[4], ready[4], empty[4];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort;
};

struct FqWork {
  int head, b, h, i, kt_last;   // head: within the chunk; kt_last: last key tile in it
};
__device__ __forceinline__ FqWork fq_work(const AttnProblem& p, const FbChunk& c, int n_t, int w) {
  FqWork k;
  const int G = p.Hq / p.Hkv, heads = (c.g1 - c.g0) * G;
  const int i0 = p.causal ? c.j0 : 0, band = c.band * G, n_i = n_t - i0;
  const int kb = w / (band * n_i), r = w % (band * n_i), size = min(band, heads - kb * band);
  k.head = kb * band + r % size;
  k.i = n_t - 1 - r / size;   // the longest first
  const int gh = c.g0 * G + k.head;   // kv groups and query heads are both head-major
  k.b = gh / p.Hq;
  k.h = gh % p.Hq;
  k.kt_last = (p.causal ? min(k.i, c.j1 - 1) : c.j1 - 1);
  return k;
}

template <int D, bool BF16, bool MASKED>
__global__ void __launch_bounds__(kFqThreads, 1)
attn_sm100_dq_kernel(const __grid_constant__ CUtensorMap tm_k, const AttnProblem p,
                     const AttnTensors a, const FbChunk c, const uint32_t* __restrict__ bits,
                     const uint16_t* __restrict__ dsbuf, float* __restrict__ acc32) {
  using L = FqLayout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  FqMisc* misc = reinterpret_cast<FqMisc*>(smem + L::OFF_MISC);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  int* err = &g_device_error;
  volatile int* abort = &misc->abort;
  const int n_t = (p.T + kBM - 1) / kBM, words = (p.T + 31) >> 5, G = p.Hq / p.Hkv;
  const int n_work = (c.g1 - c.g0) * G * (n_t - (p.causal ? c.j0 : 0));
  // "snake" order over the CTAs: evens out the causal lengths
  auto work_at = [&](int rd) {
    const int n = (int)gridDim.x, k = (int)blockIdx.x;
    return rd * n + ((rd & 1) ? n - 1 - k : k);
  };
  // key tiles of an item, from the last down (a query tile without a token has none)
  auto first_kt = [&](const FqWork& k) {
    if (MASKED && !tile_bits<MASKED>(bits, words, k.b, k.i).any()) return -1;
    const int kt = live_tile<MASKED>(bits, words, k.b, k.kt_last);
    return kt >= c.j0 ? kt : -1;
  };
  auto next_kt = [&](const FqWork& k, int kt) {
    kt = live_tile<MASKED>(bits, words, k.b, kt - 1);
    return kt >= c.j0 ? kt : -1;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 4; ++s) {
      mbar_init(&misc->full[s], 1);
      mbar_init(&misc->ready[s], 1);
      mbar_init(&misc->empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&misc->acc_full[s], 1);
      mbar_init(&misc->acc_empty[s], 4);
    }
    misc->abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&misc->tmem_base, 256);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) tma_prefetch_desc(&tm_k);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, misc->tmem_base, 0);

  if (warp == 0) {
    if (lane == 0) {
      int n = 0;
      bool ok = true;
      for (int rd = 0, w = work_at(0); ok && w < n_work; w = work_at(++rd)) {
        const FqWork k = fq_work(p, c, n_t, w);
        for (int kt = first_kt(k); kt >= 0; kt = next_kt(k, kt), ++n) {
          const int s = n % L::NS;
          if (n >= L::NS && !mbar_wait(&misc->empty[s], (n / L::NS - 1) & 1, abort, err)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * L::STAGE;
          mbar_arrive_expect_tx(&misc->full[s], L::STAGE);
          bulk_load(st,
                    dsbuf + ((long long)k.head * c.tph + fb_tile(c, p.causal, n_t, k.i, kt)) *
                                kDTileElems,
                    L::DS_BYTES, &misc->full[s]);
          issue_tile_loads(st + L::DS_BYTES, &tm_k, &misc->full[s], D, kt * kBN, k.h / G, k.b);
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_one();
    const uint32_t id = idesc_f16(kBM, D, BF16, BF16, 1, 1);
    const uint64_t a_desc = desc_interleave(smem_u32(smem), 128, kBM * 16);
    const uint64_t b_desc = mnmajor_desc(smem_u32(smem) + L::DS_BYTES, 0);
    uint64_t* loaded = MASKED ? misc->ready : misc->full;
    int slot = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int rd = 0, w = work_at(0); ok && w < n_work; w = work_at(++rd)) {
      const FqWork k = fq_work(p, c, n_t, w);
      int kt = first_kt(k);
      if (kt < 0) continue;
      const int ab = it & 1;
      if (it >= 2 && !mbar_wait_warp(&misc->acc_empty[ab], ((it >> 1) - 1) & 1, abort, err)) break;
      tc_fence_after();
      for (uint32_t more = 0; kt >= 0; kt = next_kt(k, kt), more = 1) {
        if (!(ok = mbar_wait_warp(&loaded[slot], phase, abort, err))) break;
        tc_fence_after();
        const uint64_t off = (uint64_t)slot * (L::STAGE >> 4);   // descriptors count 16 bytes
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk)
          umma_f16_ss_by(leader, tmem + ab * 128, a_desc + off + (uint64_t)(kk * 2 * 128 >> 4),
                         b_desc + off + (uint64_t)(kk * 16 * 128 >> 4), id,
                         (more || kk > 0) ? 1u : 0u);
        umma_commit_by(leader, &misc->empty[slot]);
        if (++slot == L::NS) {
          slot = 0;
          phase ^= 1;
        }
      }
      if (ok) umma_commit_by(leader, &misc->acc_full[ab]);
      ++it;
    }
  } else if (warp == 2) {
    if (MASKED) {
      int n = 0;
      bool ok = true;
      for (int rd = 0, w = work_at(0); ok && w < n_work; w = work_at(++rd)) {
        const FqWork k = fq_work(p, c, n_t, w);
        for (int kt = first_kt(k); kt >= 0; kt = next_kt(k, kt), ++n) {
          const int s = n % L::NS;
          if (!mbar_wait(&misc->full[s], (n / L::NS) & 1, abort, err)) {
            ok = false;
            break;
          }
          const TileBits tb = tile_bits<MASKED>(bits, words, k.b, kt);
          if (!tb.all()) {
            clear_rows<D>(smem + s * L::STAGE + L::DS_BYTES, tb, lane);
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&misc->ready[s]);
        }
      }
    }
  } else {
    const int r = (warp & 3) * 32 + lane;
    int it = 0;
    for (int rd = 0, w = work_at(0); w < n_work; w = work_at(++rd)) {
      const FqWork k = fq_work(p, c, n_t, w);
      const bool any = first_kt(k) >= 0;
      const int ab = it & 1, i = k.i * kBM + r;
      if (any && !mbar_wait(&misc->acc_full[ab], (it >> 1) & 1, abort, err)) break;
      tc_fence_after();
      const bool in = i < p.T;
      const bool live = any && in && token_valid(MASKED ? bits : nullptr, words, k.b, i);
      uint16_t* row = static_cast<uint16_t*>(a.dq) + (size_t)k.b * a.sdq.b + (size_t)k.h * a.sdq.h +
                      (size_t)i * a.sdq.t;
      const uint32_t taddr = tmem + ab * 128 + ((uint32_t)((warp & 3) * 32) << 16);
      // a split head: fp32 sums over its launches, rounded by the last of them
      const bool first = c.j0 == 0, last = p.causal ? k.i < c.j1 : c.j1 == n_t;
#pragma unroll
      for (int col = 0; col < D; col += 32) {
        float v[32];
        __syncwarp();   // lanes past the last row leave a step early; the load takes the warp
        if (any) {
          tmem_ld32(taddr + col, v);
          tmem_wait_ld_dep(v);
        }
        if (!in) continue;
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = live ? v[e] : 0.f;
        if (c.split) {
          float* sum = acc32 + ((size_t)k.head * p.T + i) * p.D + col;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            if (col + e >= p.D) break;
            float4* at = reinterpret_cast<float4*>(sum + e);
            if (!first) {
              const float4 o = *at;
              v[e] += o.x;
              v[e + 1] += o.y;
              v[e + 2] += o.z;
              v[e + 3] += o.w;
            }
            if (!last) *at = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
          if (!last) continue;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (col + e >= p.D) break;
          *reinterpret_cast<uint4*>(row + col + e) =
              make_uint4(pack2t<BF16>(v[e] * p.sc, v[e + 1] * p.sc),
                         pack2t<BF16>(v[e + 2] * p.sc, v[e + 3] * p.sc),
                         pack2t<BF16>(v[e + 4] * p.sc, v[e + 5] * p.sc),
                         pack2t<BF16>(v[e + 6] * p.sc, v[e + 7] * p.sc));
        }
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&misc->acc_empty[ab]);
        ++it;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

long long fb_tiles_per_head(const AttnProblem& p) {
  const long long n_t = (p.T + kBM - 1) / kBM;
  return p.causal ? n_t * (n_t + 1) / 2 : n_t * n_t;
}

// How the backward is cut: `per` whole kv groups a launch, or, where the buffer
// does not hold one group's dS tiles, `keys` key tiles of one group (split).
struct FbPlan {
  int per, keys;
  bool split;
};
FbPlan fb_plan(const AttnProblem& p, long long cap_tiles) {
  const int n_t = (p.T + kBM - 1) / kBM, G = p.Hq / p.Hkv, groups = p.B * p.Hkv;
  const long long group = (long long)G * fb_tiles_per_head(p);
  if (group <= cap_tiles) {
    // as few launches as fit, of near-equal size
    const long long most = std::min<long long>(groups, cap_tiles / group);
    const int n = (int)((groups + most - 1) / most);
    return FbPlan{(groups + n - 1) / n, n_t, false};
  }
  const long long keys = cap_tiles / ((long long)G * n_t);
  return FbPlan{1, (int)std::min<long long>(n_t, keys), true};
}

// CTAs a key tile.  Few and long work items leave the GPU waiting for the longest (2 kv
// heads of 4 query heads, 15001 tokens: 236 items, 472 query tiles in the longest, 379
// a SM on average): below three items a SM up to four CTAs share one, and their fp32
// sums of dk and dv are joined by a small launch (890 -> 815 + 17 us there; with 512
// items, 32 / 8 heads x 8192, it only costs 35 us).  Each keeps 16 query tiles on average.
constexpr int kFbSms = 148;
int fb_parts(const AttnProblem& p, const FbPlan& plan) {
  const long long n_t = (p.T + kBM - 1) / kBM, G = p.Hq / p.Hkv;
  const long long items = (long long)plan.per * plan.keys;
  const long long tiles = G * (p.causal ? (n_t + 1) / 2 : n_t);
  const long long want = (3 * kFbSms + items - 1) / items;
  return (int)std::max<long long>(1, std::min<long long>(std::min<long long>(want, 4), tiles / 16));
}
size_t fb_sums_bytes(const AttnProblem& p, const FbPlan& plan) {
  const int parts = fb_parts(p, plan);
  return parts > 1 ? (size_t)parts * 2 * plan.per * p.T * p.D * 4 : 0;
}

template <int D, bool BF16, bool MASKED>
cudaError_t run_attn_backward(const AttnProblem& p, const AttnTensors& t, const uint32_t* bits,
                              float* stats, uint16_t* dsbuf, size_t ds_bytes, float* acc32,
                              cudaStream_t st) {
  // [dS tiles][fp32 sums of dv and dk, where the scratch has room for them]
  const size_t tiles = std::min(ds_bytes, attn_sm100_ds_bytes(p));
  const FbPlan plan = fb_plan(p, (long long)(tiles / (kDTileElems * 2)));
  if (plan.keys <= 0) return cudaErrorInvalidValue;
  const size_t sums_at = (tiles + 255) & ~size_t(255), sums_bytes = fb_sums_bytes(p, plan);
  const int parts = sums_bytes && ds_bytes >= sums_at + sums_bytes ? fb_parts(p, plan) : 1;
  float* sums = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(dsbuf) + sums_at);
  CUtensorMap mq, mk, mv, mdo, mdk, mdv;
  if (!attn_map(&mq, t.q, p, p.Hq, t.sq) || !attn_map(&mk, t.k, p, p.Hkv, t.sk) ||
      !attn_map(&mv, t.v, p, p.Hkv, t.sv) || !attn_map(&mdo, t.dout, p, p.Hq, t.sdo) ||
      !attn_map(&mdk, t.dk, p, p.Hkv, t.sdk, 32) || !attn_map(&mdv, t.dv, p, p.Hkv, t.sdv, 32))
    return cudaErrorInvalidValue;
  auto kkv = attn_sm100_dkv_kernel<D, BF16, MASKED>;
  auto kq = attn_sm100_dq_kernel<D, BF16, MASKED>;
  cudaError_t e;
  int dev = 0, num_sms = 0;
  if ((e = prep(kkv, FbLayout<D>::BYTES)) != cudaSuccess ||
      (e = prep(kq, FqLayout<D>::BYTES)) != cudaSuccess ||
      (e = cudaGetDevice(&dev)) != cudaSuccess ||
      (e = cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
    return e;
  const int n_t = (p.T + kBM - 1) / kBM, G = p.Hq / p.Hkv, groups = p.B * p.Hkv;
  const bool ranked = exact_delta_ranked(p, bits);
  const int few = exact_delta_tiles(p, ranked), heads = p.B * p.Hq;
  if (few > 0)
    attn_sm100_exact_delta_kernel<D, BF16>
        <<<heads * few * (kBM / 16), 256, 0, st>>>(p, t, bits, stats);
  if (n_t > few)
    attn_sm100_delta_kernel<<<heads * (n_t - few), 256, 0, st>>>(p, t, bits, stats, few);
  if (ranked)
    attn_sm100_exact_delta_ranked_kernel<D, BF16>
        <<<heads * (kExactDeltaKeys / 16), 256, 0, st>>>(p, t, bits, stats);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const long long group_bytes = 4ll * G * p.T * p.D;   // queries and dO
  for (int g0 = 0; g0 < groups; g0 += plan.per)
    for (int j0 = 0; j0 < n_t; j0 += plan.keys) {
      FbChunk c{};
      c.g0 = g0;
      c.g1 = std::min(groups, g0 + plan.per);
      c.j0 = j0;
      c.j1 = std::min(n_t, j0 + plan.keys);
      c.split = plan.split;
      c.parts = parts;
      c.band = (int)std::max<long long>(
          1, std::min<long long>(c.g1 - g0, (64ll << 20) / std::max<long long>(group_bytes, 1)));
      const int i0 = p.causal ? j0 : 0;
      c.tph = plan.split ? (long long)(n_t - i0) * (c.j1 - j0) : fb_tiles_per_head(p);
      kkv<<<(c.g1 - c.g0) * (c.j1 - c.j0) * parts, kFbThreads, FbLayout<D>::BYTES, st>>>(
          mq, mk, mv, mdo, mdk, mdv, p, c, bits, stats, dsbuf, sums);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
      if (parts > 1) {
        const int rows = std::min(p.T, c.j1 * kBN) - j0 * kBN;
        const long long n = 2ll * (c.g1 - c.g0) * rows * (p.D / 8);
        attn_sm100_sum_parts_kernel<BF16><<<(int)std::min<long long>((n + 255) / 256, 4 * kFbSms),
                                            256, 0, st>>>(p, t, c, sums);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
      }
      const int work = (c.g1 - g0) * G * (n_t - i0);
      kq<<<std::min(work, num_sms), kFqThreads, FqLayout<D>::BYTES, st>>>(mk, p, t, c, bits, dsbuf,
                                                                          acc32);
      if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
  return cudaSuccess;
}

bool attn_readable(const void* x, const TensorStrides& s) {
  return reinterpret_cast<uintptr_t>(x) % 16 == 0 && s.b > 0 && s.h > 0 && s.t > 0 &&
         s.b % 8 == 0 && s.h % 8 == 0 && s.t % 8 == 0;
}

}  // namespace

bool attn_sm100_supports(const AttnProblem& p, const AttnTensors& t) {
  return p.D <= 128 && (long long)p.T * p.D > kAttnFewElements && attn_readable(t.q, t.sq) &&
         attn_readable(t.k, t.sk) && attn_readable(t.v, t.sv) && attn_readable(t.out, t.so);
}

bool attn_sm100_backward_supports(const AttnProblem& p, const AttnTensors& t) {
  return attn_sm100_supports(p, t) && attn_readable(t.dout, t.sdo) && attn_readable(t.dq, t.sdq) &&
         attn_readable(t.dk, t.sdk) && attn_readable(t.dv, t.sdv);
}

size_t attn_stats_bytes(const AttnProblem& p) {
  return (size_t)p.B * p.Hq * ((p.T + kBM - 1) / kBM) * kFbStatBytes;
}

size_t attn_sm100_group_bytes(const AttnProblem& p) {
  return (size_t)(p.Hq / p.Hkv) * fb_tiles_per_head(p) * kDTileElems * 2;
}

size_t attn_sm100_ds_bytes(const AttnProblem& p) {
  const long long all = fb_tiles_per_head(p) * p.B * p.Hq * kDTileElems * 2;
  const long long min = (long long)attn_sm100_ds_min_bytes(p);
  return (size_t)std::min(all, std::max(kDBufCapBytes, min));
}

size_t attn_sm100_sums_bytes(const AttnProblem& p) {
  return fb_sums_bytes(p, fb_plan(p, (long long)(attn_sm100_ds_bytes(p) / (kDTileElems * 2))));
}

size_t attn_sm100_ds_min_bytes(const AttnProblem& p) {
  return (size_t)(p.Hq / p.Hkv) * ((p.T + kBM - 1) / kBM) * kDTileElems * 2;
}

size_t attn_sm100_acc_bytes(const AttnProblem& p) {
  return (size_t)(p.Hq / p.Hkv) * p.T * p.D * 4;
}

cudaError_t launch_attn_sm100_backward(const AttnProblem& p, const AttnTensors& t,
                                       const uint32_t* bits, float* stats, void* ds,
                                       size_t ds_bytes, float* acc, cudaStream_t st) {
  uint16_t* d = static_cast<uint16_t*>(ds);
  const bool bf = p.dtype == LKL_BF16;
  auto run = [&](auto k) { return k(p, t, bits, stats, d, ds_bytes, acc, st); };
  if (tc_dim(p.D) == 64) {
    if (bits) return bf ? run(run_attn_backward<64, true, true>)
                        : run(run_attn_backward<64, false, true>);
    return bf ? run(run_attn_backward<64, true, false>) : run(run_attn_backward<64, false, false>);
  }
  if (bits) return bf ? run(run_attn_backward<128, true, true>)
                      : run(run_attn_backward<128, false, true>);
  return bf ? run(run_attn_backward<128, true, false>) : run(run_attn_backward<128, false, false>);
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
