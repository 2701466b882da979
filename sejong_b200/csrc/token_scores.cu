// Scores of given tokens under rows of logits, and their gradient.
//
//   lse = m + log s,  m = max x,  s = sum e^(x - m);   logp = (x_t - m) - log s
//   H = -sum p log p = log s - sum e^(x - m) (x - m) / s     (both terms >= 0: nothing cancels)
//   dx_j = dlogp (1[j = t] - p_j) - dH p_j (log p_j + H)
//
// The alternatives are the `top` largest logits, the lowest index first among equal ones: a key of
// (value, ~index) orders them without ties.
#include <climits>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace sj {

namespace {
constexpr int kScoreMaxTop = 32;
}

SJ_DEVICE float score_load(const float* x) { return *x; }
SJ_DEVICE float score_load(const __nv_bfloat16* x) { return bf2f(*x); }

// Order-preserving key of a logit and its index: larger value first, then the lower index; NaN last.
SJ_DEVICE uint64_t score_key(float v, int index) {
  v += 0.f;  // -0 and +0 are equal
  const uint32_t bits = __float_as_uint(v);
  const uint32_t up = v != v ? 0u : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return static_cast<uint64_t>(up) << 32 | static_cast<uint32_t>(~index);
}
SJ_DEVICE float score_value(uint64_t key) {
  const uint32_t up = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(up == 0u ? 0x7fc00000u : up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

SJ_DEVICE uint64_t warp_max64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}

// One CTA per row: maximum, sums, then one pass for each alternative.
constexpr int kScoreThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kScoreThreads) token_scores_kernel(const T* logits, int ld, const int32_t* target,
                                                                     int vocab, int top, float* logp, float* entropy,
                                                                     float* lse, int32_t* top_id, float* top_logp) {
  pdl_wait();
  constexpr int W = kScoreThreads / 32;
  __shared__ float fa[W], fb[W];
  __shared__ uint64_t best[W];
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* x = logits + static_cast<size_t>(r) * ld;
  float m = -INFINITY;
  bool nan = false;
  for (int j = t; j < vocab; j += kScoreThreads) {
    const float v = score_load(x + j);
    nan |= v != v;
    m = fmaxf(m, v);
  }
  m = warp_max(m);
  if (lane == 0) fa[warp] = m;
  nan = __syncthreads_or(nan);
  for (int w = 0; w < W; ++w) m = fmaxf(m, fa[w]);
  __syncthreads();
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, u = 0.f;
  for (int j = t; j < vocab; j += kScoreThreads) {
    const float d = score_load(x + j) - base, e = expf(d);
    s += e;
    if (e > 0.f) u += e * d;
  }
  s = warp_sum(s);
  u = warp_sum(u);
  if (lane == 0) {
    fa[warp] = s;
    fb[warp] = u;
  }
  __syncthreads();
  s = u = 0.f;
  for (int w = 0; w < W; ++w) {
    s += fa[w];
    u += fb[w];
  }
  const float log_s = nan ? NAN : logf(s);
  if (t == 0) {
    const int at = target ? target[r] : -1;
    if (at >= vocab || at < -1) record_error(SJ_DEV_BAD_INDEX);
    if (logp) {
      const float v = at >= 0 && at < vocab ? score_load(x + at) : 0.f;
      logp[r] = at < 0 || at >= vocab ? 0.f : v == -INFINITY && !nan ? -INFINITY : (v - base) - log_s;
    }
    if (entropy) entropy[r] = s == 0.f && !nan ? 0.f : log_s - u / s;
    if (lse) lse[r] = base + log_s;
  }
  uint64_t bound = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t key = 0;
    for (int j = t; j < vocab; j += kScoreThreads) {
      const uint64_t v = score_key(score_load(x + j), j);
      if (v < bound && v > key) key = v;
    }
    key = warp_max64(key);
    if (lane == 0) best[warp] = key;
    __syncthreads();
    for (int w = 0; w < W; ++w) key = best[w] > key ? best[w] : key;
    __syncthreads();
    bound = key;
    if (t == 0) {
      const float v = score_value(key);
      top_id[static_cast<size_t>(r) * top + k] = static_cast<int32_t>(~static_cast<uint32_t>(key));
      top_logp[static_cast<size_t>(r) * top + k] = v == -INFINITY && !nan ? -INFINITY : (v - base) - log_s;
    }
  }
}

SJ_DEVICE void score_store(float* d, float g) { *d = g; }
SJ_DEVICE void score_store(__nv_bfloat16* d, float g) { *d = f2bf(g); }

template <typename T>
__global__ void __launch_bounds__(256) token_scores_bwd_kernel(const T* logits, int ld, const int32_t* target,
                                                               int vocab, const float* lse, const float* entropy,
                                                               const float* d_logp, const float* d_entropy, T* d_logits,
                                                               int ldd) {
  pdl_wait();
  const int r = blockIdx.x;
  const T* x = logits + static_cast<size_t>(r) * ld;
  T* d = d_logits + static_cast<size_t>(r) * ldd;
  int at = target ? target[r] : -1;
  if (at >= vocab || at < -1) {
    if (threadIdx.x == 0) record_error(SJ_DEV_BAD_INDEX);
    at = -1;
  }
  const float a = d_logp && at >= 0 ? d_logp[r] : 0.f, b = d_entropy ? d_entropy[r] : 0.f;
  const float z = lse[r], h = d_entropy ? entropy[r] : 0.f;
  for (int j = threadIdx.x; j < ldd; j += blockDim.x) {
    float g = 0.f;
    if (j < vocab && z != -INFINITY) {
      const float lp = score_load(x + j) - z, p = expf(lp);
      g = p == 0.f ? 0.f : -p * (a + b * (lp + h));
      if (j == at) g += a;
    }
    score_store(d + j, g);
  }
}

}  // namespace sj

using namespace sj;

extern "C" size_t sj_token_scores_workspace(int rows, int vocab, int top) {
  if (rows < 0 || vocab <= 0 || top < 0 || top > kScoreMaxTop) return 0;
  return 16;
}

extern "C" int sj_token_scores(const void* logits, int dtype, int ld, const int32_t* target, int rows, int vocab,
                               int top, float* logp, float* entropy, float* lse, int32_t* top_id, float* top_logp,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || vocab <= 0 || ld < vocab || top < 0 || top > kScoreMaxTop || top > vocab)
    return fail(SJ_ERR_SHAPE, "sj_token_scores: rows=%d vocab=%d ld=%d top=%d (up to %d)", rows, vocab, ld, top,
                kScoreMaxTop);
  if (dtype != SJ_F32 && dtype != SJ_BF16)
    return fail(SJ_ERR_UNSUPPORTED, "sj_token_scores: dtype %d (this build: f32 or bf16)", dtype);
  if (rows == 0) return SJ_OK;
  if (!logits || (logp && !target) || (top > 0 && (!top_id || !top_logp)) ||
      reinterpret_cast<uintptr_t>(logits) % (dtype == SJ_F32 ? 4 : 2))
    return fail(SJ_ERR_ARGUMENT, "sj_token_scores: null or unaligned operand");
  if (!workspace || !aligned16(workspace) || workspace_bytes < sj_token_scores_workspace(rows, vocab, top))
    return fail(SJ_ERR_CAPACITY, "sj_token_scores: workspace of %zu bytes", workspace_bytes);
  if (dtype == SJ_F32)
    launch(token_scores_kernel<float>, rows, kScoreThreads, 0, as_stream(stream), static_cast<const float*>(logits), ld,
           target, vocab, top, logp, entropy, lse, top_id, top_logp);
  else
    launch(token_scores_kernel<__nv_bfloat16>, rows, kScoreThreads, 0, as_stream(stream),
           static_cast<const __nv_bfloat16*>(logits), ld, target, vocab, top, logp, entropy, lse, top_id, top_logp);
  SJ_LAUNCH_CHECK("token_scores");
  return SJ_OK;
}

extern "C" int sj_token_scores_bwd(const void* logits, int dtype, int ld, const int32_t* target, int rows, int vocab,
                                   const float* lse, const float* entropy, const float* d_logp, const float* d_entropy,
                                   void* d_logits, int ldd, void* stream) {
  if (rows < 0 || vocab <= 0 || ld < vocab || ldd < vocab)
    return fail(SJ_ERR_SHAPE, "sj_token_scores_bwd: rows=%d vocab=%d ld=%d ldd=%d", rows, vocab, ld, ldd);
  if (dtype != SJ_F32 && dtype != SJ_BF16)
    return fail(SJ_ERR_UNSUPPORTED, "sj_token_scores_bwd: dtype %d (this build: f32 or bf16)", dtype);
  if (rows == 0) return SJ_OK;
  const uintptr_t mask = dtype == SJ_F32 ? 3 : 1;
  if (!logits || !lse || !d_logits || (!d_logp && !d_entropy) || (d_logp && !target) || (d_entropy && !entropy) ||
      ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(d_logits)) & mask))
    return fail(SJ_ERR_ARGUMENT, "sj_token_scores_bwd: null or unaligned operand");
  if (d_logits == logits && ld != ldd)
    return fail(SJ_ERR_ARGUMENT, "sj_token_scores_bwd: in place takes ld == ldd");
  if (dtype == SJ_F32)
    launch(token_scores_bwd_kernel<float>, rows, 256, 0, as_stream(stream), static_cast<const float*>(logits), ld,
           target, vocab, lse, entropy, d_logp, d_entropy, static_cast<float*>(d_logits), ldd);
  else
    launch(token_scores_bwd_kernel<__nv_bfloat16>, rows, 256, 0, as_stream(stream),
           static_cast<const __nv_bfloat16*>(logits), ld, target, vocab, lse, entropy, d_logp, d_entropy,
           static_cast<__nv_bfloat16*>(d_logits), ldd);
  SJ_LAUNCH_CHECK("token_scores_bwd");
  return SJ_OK;
}
