// C ABI entry points of the attention and of the logits operators
// (include/linearard_b200.h): argument checks, scratch layout and dispatch.
#include "lkl_attn.cuh"
#include "lkl_logits.cuh"

namespace {

using lkl::AttnProblem;
using lkl::AttnTensors;
using lkl::LogitsView;
using lkl::TensorStrides;

int32_t check_attn(const lkl_attn_problem* p) {
  if (!p) return LKL_ERR_NULL_POINTER;
  if (p->B < 0 || p->T < 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv != 0)
    return LKL_ERR_BAD_SHAPE;
  if (!head_dim_ok(p->D)) return LKL_ERR_BAD_HEAD_DIM;
  if (p->dtype != LKL_F16 && p->dtype != LKL_BF16) return LKL_ERR_BAD_DTYPE;
  if (p->mask_dtype < LKL_MASK_BOOL || p->mask_dtype > LKL_MASK_I64) return LKL_ERR_BAD_DTYPE;
  // single precision holds the scale and its multiple by log2(e)
  if (!(p->sm_scale <= 0.f) && !(p->sm_scale >= 0x1p-126f && p->sm_scale < 0x1p127f))
    return LKL_ERR_BAD_SHAPE;
  // block counts and 32-bit token arithmetic
  if ((long long)p->B * p->Hq * (((long long)p->T + 31) / 32) > INT32_MAX ||
      p->T > INT32_MAX - 256)
    return LKL_ERR_TOO_LARGE;
  return LKL_OK;
}

AttnProblem to_attn(const lkl_attn_problem* p) {
  return AttnProblem{p->B, p->Hq, p->Hkv, p->T, p->D, p->dtype, p->causal ? 1 : 0,
                     p->sm_scale > 0.f ? p->sm_scale : 1.0f / sqrtf((float)p->D)};
}

inline size_t attn_bits_bytes(const lkl_attn_problem* p) {
  return round256((size_t)p->B * (size_t)((p->T + 31) / 32) * sizeof(uint32_t));
}
// Backward scratch: [mask bits][row statistics][fp32 dq sums][dS tiles ...]; the
// sums only where the tiles of one kv group do not fit at once.
size_t attn_stats_end(const lkl_attn_problem* p, bool has_mask) {
  return (has_mask ? attn_bits_bytes(p) : 0) + round256(lkl::attn_stats_bytes(to_attn(p)));
}
struct AttnScratch {
  size_t acc, ds, ds_bytes;   // offsets, and the bytes left from ds on
};
AttnScratch attn_scratch(const lkl_attn_problem* p, bool has_mask, size_t ws_bytes) {
  const AttnProblem a = to_attn(p);
  const size_t group = lkl::attn_sm100_group_bytes(a);
  AttnScratch s;
  s.acc = s.ds = attn_stats_end(p, has_mask);
  if (ws_bytes < s.ds + group || lkl::attn_sm100_ds_bytes(a) < group)
    s.ds += round256(lkl::attn_sm100_acc_bytes(a));
  s.ds_bytes = ws_bytes > s.ds ? ws_bytes - s.ds : 0;
  return s;
}

// Strides of tensor `which` (`strides` or the contiguous ones).
TensorStrides attn_strides(const lkl_strides* strides, int which, const lkl_attn_problem* p) {
  if (strides) return TensorStrides{strides[which].b, strides[which].h, strides[which].t};
  const bool kv = which == LKL_ATTN_K || which == LKL_ATTN_V || which == LKL_ATTN_DK ||
                  which == LKL_ATTN_DV;
  const long long n = (long long)p->T * p->D;
  return TensorStrides{n * (kv ? p->Hkv : p->Hq), n, p->D};
}

// Inputs may repeat elements (stride 0), outputs may not.
int32_t check_attn_strides(const lkl_strides* s, int n) {
  if (!s) return LKL_OK;
  for (int i = 0; i < n; ++i) {
    const bool output = i == LKL_ATTN_DQ || i == LKL_ATTN_DK || i == LKL_ATTN_DV ||
                        (i == LKL_ATTN_OUT && n == 4);
    if (s[i].b < 0 || s[i].h < 0 || s[i].t < 0) return LKL_ERR_BAD_SHAPE;
    if (output && (s[i].b == 0 || s[i].h == 0 || s[i].t == 0)) return LKL_ERR_BAD_SHAPE;
  }
  return LKL_OK;
}

int32_t attn_bits(const lkl_attn_problem* p, const void* mask, void* ws, uint32_t** bits,
                  cudaStream_t st) {
  *bits = nullptr;
  if (!mask) return LKL_OK;
  *bits = static_cast<uint32_t*>(ws);
  return launch_status(lkl::launch_pack_mask(mask, p->mask_dtype, p->B, p->T, *bits, st));
}

inline size_t logits_elem(int dtype) { return dtype == LKL_F32 ? 4 : 2; }

int32_t check_logits(const void* x, const lkl_logits* l) {
  if (!l) return LKL_ERR_NULL_POINTER;
  if (l->dtype != LKL_F16 && l->dtype != LKL_BF16 && l->dtype != LKL_F32) return LKL_ERR_BAD_DTYPE;
  if (l->B < 0 || l->T < 0 || l->V <= 0 || l->sb < 0 || l->st < 0) return LKL_ERR_BAD_SHAPE;
  if (l->V > INT32_MAX - 65536 || l->B > INT32_MAX || l->T > INT32_MAX ||
      l->B * l->T > INT32_MAX)
    return LKL_ERR_TOO_LARGE;
  if (l->B * l->T == 0) return LKL_OK;
  if (!x) return LKL_ERR_NULL_POINTER;
  return aligned(x, logits_elem(l->dtype)) && aligned(l->lse_low, 4) ? LKL_OK : LKL_ERR_MISALIGNED;
}

LogitsView to_view(const void* x, const lkl_logits* l) {
  return LogitsView{x, l->T, l->V, l->sb, l->st, l->dtype, l->lse_low};
}

// What a log-sum-exp lacks stands in an array of its own.
inline bool low_aliases(const lkl_logits* l, const void* other) {
  return l->lse_low && l->lse_low == other;
}

int32_t check_kl_lse(const lkl_logits* s, const lkl_logits* t, const float* lse_s,
                     const float* lse_t) {
  if (!lse_s || !lse_t) return LKL_ERR_NULL_POINTER;
  if (low_aliases(s, t->lse_low) || low_aliases(s, lse_s) || low_aliases(s, lse_t) ||
      low_aliases(t, lse_s) || low_aliases(t, lse_t))
    return LKL_ERR_BAD_ALIAS;
  return LKL_OK;
}

int32_t check_kl(const void* sx, const lkl_logits* s, const void* tx, const lkl_logits* t,
                 const void* mask, int32_t mdt, float temperature) {
  int32_t e;
  if ((e = check_logits(sx, s)) || (e = check_logits(tx, t))) return e;
  if (s->B != t->B || s->T != t->T || s->V != t->V) return LKL_ERR_BAD_SHAPE;
  if (s->dtype != t->dtype) return LKL_ERR_BAD_DTYPE;
  if (!(temperature > 0.f) || isinf(temperature) || isinf(1.f / temperature))
    return LKL_ERR_BAD_SHAPE;
  if (mask && (mdt < LKL_MASK_BOOL || mdt > LKL_MASK_I64)) return LKL_ERR_BAD_DTYPE;
  return check_mask(mask, mdt);
}

}  // namespace

extern "C" {

size_t lkl_attn_forward_workspace_size(const lkl_attn_problem* p, int32_t has_mask) {
  if (check_attn(p) != LKL_OK || p->B == 0 || p->T == 0) return 0;
  return has_mask ? attn_bits_bytes(p) : 0;
}

size_t lkl_attn_backward_workspace_size(const lkl_attn_problem* p, int32_t has_mask) {
  if (check_attn(p) != LKL_OK || p->B == 0 || p->T == 0) return 0;
  const AttnProblem a = to_attn(p);
  const size_t n = attn_stats_end(p, has_mask != 0);
  if (a.D > 128 || (long long)a.T * a.D <= lkl::kAttnFewElements) return n;
  return attn_scratch(p, has_mask != 0, SIZE_MAX).ds + round256(lkl::attn_sm100_ds_bytes(a)) +
         round256(lkl::attn_sm100_sums_bytes(a));
}

int32_t lkl_attn_forward(const void* q, const void* k, const void* v, const lkl_strides* strides,
                         const void* mask, const lkl_attn_problem* p, void* out, float* lse,
                         void* ws, size_t ws_bytes, void* stream) {
  int32_t s = check_attn(p);
  if (s) return s;
  if (p->B == 0 || p->T == 0) return LKL_OK;
  if (!q || !k || !v || !out || !lse) return LKL_ERR_NULL_POINTER;
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(out, 2) || !aligned(lse, 4))
    return LKL_ERR_MISALIGNED;
  if (out == q || out == k || out == v) return LKL_ERR_BAD_ALIAS;
  if ((s = check_mask(mask, p->mask_dtype)) || (s = check_attn_strides(strides, 4))) return s;
  if ((s = check_workspace(lkl_attn_forward_workspace_size(p, mask != nullptr), ws, ws_bytes)))
    return s;
  if (!bind_device_of(q) || !device_is_sm100()) return LKL_ERR_NO_DEVICE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t* bits;
  if ((s = attn_bits(p, mask, ws, &bits, st))) return s;
  AttnTensors t{};
  t.q = q, t.k = k, t.v = v, t.out = out, t.lse = lse;
  t.sq = attn_strides(strides, LKL_ATTN_Q, p);
  t.sk = attn_strides(strides, LKL_ATTN_K, p);
  t.sv = attn_strides(strides, LKL_ATTN_V, p);
  t.so = attn_strides(strides, LKL_ATTN_OUT, p);
  const AttnProblem a = to_attn(p);
  t_last_path = !g_force_generic.load() && lkl::attn_sm100_supports(a, t) ? 1 : 0;
  return launch_status(t_last_path ? lkl::launch_attn_sm100_forward(a, t, bits, st)
                                   : lkl::launch_attn_generic_forward(a, t, bits, st));
}

int32_t lkl_attn_backward(const void* q, const void* k, const void* v, const void* out,
                          const float* lse, const void* dout, const lkl_strides* strides,
                          const void* mask, const lkl_attn_problem* p, void* dq, void* dk,
                          void* dv, void* ws, size_t ws_bytes, void* stream) {
  int32_t s = check_attn(p);
  if (s) return s;
  if (p->B == 0 || p->T == 0) return LKL_OK;
  if (!q || !k || !v || !out || !lse || !dout || !dq || !dk || !dv) return LKL_ERR_NULL_POINTER;
  const void* const all[] = {q, k, v, out, dout, dq, dk, dv};
  for (const void* x : all)
    if (!aligned(x, 2)) return LKL_ERR_MISALIGNED;
  if (!aligned(lse, 4)) return LKL_ERR_MISALIGNED;
  for (int g = 5; g < 8; ++g)   // a gradient is neither an input nor another gradient
    for (int x = 0; x < g; ++x)
      if (all[g] == all[x]) return LKL_ERR_BAD_ALIAS;
  if ((s = check_mask(mask, p->mask_dtype)) || (s = check_attn_strides(strides, 8))) return s;
  if ((s = check_workspace(attn_stats_end(p, mask != nullptr), ws, ws_bytes))) return s;
  AttnTensors t{};
  t.q = q, t.k = k, t.v = v, t.out = const_cast<void*>(out), t.lse = const_cast<float*>(lse);
  t.dout = dout, t.dq = dq, t.dk = dk, t.dv = dv;
  t.sq = attn_strides(strides, LKL_ATTN_Q, p);
  t.sk = attn_strides(strides, LKL_ATTN_K, p);
  t.sv = attn_strides(strides, LKL_ATTN_V, p);
  t.so = attn_strides(strides, LKL_ATTN_OUT, p);
  t.sdo = attn_strides(strides, LKL_ATTN_DOUT, p);
  t.sdq = attn_strides(strides, LKL_ATTN_DQ, p);
  t.sdk = attn_strides(strides, LKL_ATTN_DK, p);
  t.sdv = attn_strides(strides, LKL_ATTN_DV, p);
  const AttnProblem a = to_attn(p);
  const bool tc = !g_force_generic.load() && lkl::attn_sm100_backward_supports(a, t);
  const AttnScratch at = attn_scratch(p, mask != nullptr, ws_bytes);
  if (tc && at.ds_bytes < lkl::attn_sm100_ds_min_bytes(a)) return LKL_ERR_WORKSPACE;
  if (!bind_device_of(q) || !device_is_sm100()) return LKL_ERR_NO_DEVICE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t* bits;
  if ((s = attn_bits(p, mask, ws, &bits, st))) return s;
  uint8_t* const base = static_cast<uint8_t*>(ws);
  float* const stats = reinterpret_cast<float*>(base + (mask ? attn_bits_bytes(p) : 0));
  t_last_path = tc ? 1 : 0;
  if (tc)
    return launch_status(lkl::launch_attn_sm100_backward(
        a, t, bits, stats, base + at.ds,
        at.ds_bytes,
        reinterpret_cast<float*>(base + at.acc), st));
  float2* rows = reinterpret_cast<float2*>(stats);
  // every row of a long sequence first, then those that see few keys
  const bool few = a.T <= lkl::kExactDeltaKeys;
  if (!few && (s = launch_status(lkl::launch_attn_delta(a, t, bits, rows, st)))) return s;
  if ((few || a.causal || bits) &&
      (s = launch_status(lkl::launch_attn_exact_delta(a, t, bits, rows, st))))
    return s;
  return launch_status(lkl::launch_attn_generic_backward(a, t, bits, rows, st));
}

int32_t lkl_token_logprobs(const void* logits, const lkl_logits* l, const int64_t* targets,
                           int64_t ignore_index, int32_t top_k, float* logprob, float* entropy,
                           float* lse, float* top_logprobs, int64_t* top_indices, void* stream) {
  int32_t s = check_logits(logits, l);
  if (s) return s;
  if (top_k < 0 || top_k > LKL_MAX_TOP_K || top_k > l->V) return LKL_ERR_BAD_SHAPE;
  if (l->B * l->T == 0) return LKL_OK;
  if (!targets || !logprob || !entropy || !lse || (top_k && (!top_logprobs || !top_indices)))
    return LKL_ERR_NULL_POINTER;
  if (!aligned(targets, 8) || !aligned(logprob, 4) || !aligned(entropy, 4) || !aligned(lse, 4) ||
      !aligned(top_logprobs, 4) || !aligned(top_indices, 8))
    return LKL_ERR_MISALIGNED;
  if (low_aliases(l, lse)) return LKL_ERR_BAD_ALIAS;
  if (!bind_device_of(logits) || !device_is_sm100()) return LKL_ERR_NO_DEVICE;
  return launch_status(lkl::launch_token_logprobs(
      to_view(logits, l), l->B * l->T, targets, ignore_index, top_k, logprob, entropy, lse,
      top_logprobs, top_indices, static_cast<cudaStream_t>(stream)));
}

int32_t lkl_token_logprobs_backward(const void* logits, const lkl_logits* l,
                                    const int64_t* targets, int64_t ignore_index,
                                    const float* lse, const float* entropy,
                                    const float* d_logprob, const float* d_entropy,
                                    void* d_logits, void* stream) {
  int32_t s = check_logits(logits, l);
  if (s) return s;
  if (l->B * l->T == 0) return LKL_OK;
  if (!targets || !lse || !entropy || !d_logits) return LKL_ERR_NULL_POINTER;
  if (d_logits == logits || low_aliases(l, lse)) return LKL_ERR_BAD_ALIAS;
  if (!aligned(targets, 8) || !aligned(lse, 4) || !aligned(entropy, 4) ||
      !aligned(d_logprob, 4) || !aligned(d_entropy, 4) ||
      !aligned(d_logits, logits_elem(l->dtype)))
    return LKL_ERR_MISALIGNED;
  if (!bind_device_of(logits) || !device_is_sm100()) return LKL_ERR_NO_DEVICE;
  return launch_status(lkl::launch_token_logprobs_backward(
      to_view(logits, l), l->B * l->T, targets, ignore_index, lse, entropy, d_logprob, d_entropy,
      d_logits, static_cast<cudaStream_t>(stream)));
}

size_t lkl_logits_kl_workspace_size(const lkl_logits* s) {
  if (!s || s->B <= 0 || s->T <= 0) return 0;
  return round256((size_t)s->B * s->T * sizeof(float));
}

int32_t lkl_logits_kl_forward(const void* s_logits, const lkl_logits* s, const void* t_logits,
                              const lkl_logits* t, const void* mask, int32_t mask_dtype,
                              float temperature, float* lse_s, float* lse_t, float* loss,
                              void* ws, size_t ws_bytes, void* stream) {
  int32_t e = check_kl(s_logits, s, t_logits, t, mask, mask_dtype, temperature);
  if (e) return e;
  if (!loss) return LKL_ERR_NULL_POINTER;
  if (!aligned(loss, 4) || !aligned(lse_s, 4) || !aligned(lse_t, 4)) return LKL_ERR_MISALIGNED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s->B * s->T == 0) {
    if (!bind_device_of(loss)) return LKL_ERR_NO_DEVICE;
    return launch_status(cudaMemsetAsync(loss, 0, sizeof(float), st));
  }
  if ((e = check_kl_lse(s, t, lse_s, lse_t))) return e;
  if ((e = check_workspace(lkl_logits_kl_workspace_size(s), ws, ws_bytes))) return e;
  if (!bind_device_of(s_logits) || !device_is_sm100()) return LKL_ERR_NO_DEVICE;
  return launch_status(lkl::launch_logits_kl_forward(
      to_view(s_logits, s), to_view(t_logits, t), s->B * s->T, mask, mask_dtype,
      1.f / temperature, lse_s, lse_t, static_cast<float*>(ws), loss, st));
}

int32_t lkl_logits_kl_backward(const void* s_logits, const lkl_logits* s, const void* t_logits,
                               const lkl_logits* t, const void* mask, int32_t mask_dtype,
                               float temperature, const float* lse_s, const float* lse_t,
                               const float* dloss, void* ds, void* stream) {
  int32_t e = check_kl(s_logits, s, t_logits, t, mask, mask_dtype, temperature);
  if (e) return e;
  if (s->B * s->T == 0) return LKL_OK;
  if (!ds) return LKL_ERR_NULL_POINTER;
  if ((e = check_kl_lse(s, t, lse_s, lse_t))) return e;
  if (ds == s_logits || ds == t_logits) return LKL_ERR_BAD_ALIAS;
  if (!aligned(lse_s, 4) || !aligned(lse_t, 4) || !aligned(dloss, 4) ||
      !aligned(ds, logits_elem(s->dtype)))
    return LKL_ERR_MISALIGNED;
  if (!bind_device_of(s_logits) || !device_is_sm100()) return LKL_ERR_NO_DEVICE;
  return launch_status(lkl::launch_logits_kl_backward(
      to_view(s_logits, s), to_view(t_logits, t), s->B * s->T, mask, mask_dtype,
      1.f / temperature, lse_s, lse_t, dloss, ds, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
