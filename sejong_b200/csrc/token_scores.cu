// Scores of given tokens under rows of logits, and their gradient.
//
//   lse = m + log s,  m = max x,  s = sum e^(x - m);   logp = (x_t - m) - log s
//   H = -sum p log p = log s - sum e^(x - m) (x - m) / s     (both terms >= 0: nothing cancels)
//   dx_j = dlogp (1[j = t] - p_j) - dH p_j (log p_j + H)
//
// The alternatives are the `top` largest logits, the lowest index first among equal ones: a key of
// (value, ~index) orders them without ties.
#include <algorithm>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace sj {

namespace {
constexpr int kScoreMaxTop = 32;
constexpr int kScoreNarrow = 1024;    // rows of at most this many logits are held by one warp
constexpr int kScoreThreads = 256;    // of the kernel for wider rows
constexpr int kScoreMaxSplits = 16;
constexpr int kScoreHeld = kScoreMaxTop * 32 + kScoreMaxTop;  // candidates: the best of 32 threads' 32, and the list
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
}  // namespace

SJ_DEVICE float score_load(const float* x) { return *x; }
SJ_DEVICE float score_load(const __nv_bfloat16* x) { return bf2f(*x); }

// 2^x to 2 ulp, results below 2^-126 flushed to 0.
SJ_DEVICE float exp2_flush(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order-preserving integer of a logit; NaN last.
SJ_DEVICE uint32_t score_order(float v) {
  v += 0.f;  // -0 and +0 are equal
  const uint32_t bits = __float_as_uint(v);
  return v != v ? 0u : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
SJ_DEVICE float score_value(uint32_t up) {
  return __uint_as_float(up == 0u ? 0x7fc00000u : up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
constexpr uint32_t kForbidden = 0x007fffffu;  // score_order(-inf)
// A key that orders logits and their indices without ties: the larger value first, then the lower index.
SJ_DEVICE uint64_t score_key(float v, int index) {
  return static_cast<uint64_t>(score_order(v)) << 32 | static_cast<uint32_t>(~index);
}

// A part of a row: its maximum m, s = sum e^(x - m) and u = sum e^(x - m) (x - m) log2(e); m = -inf: nothing yet.
struct ScoreSum {
  float m, s, u;
};
SJ_DEVICE ScoreSum score_join(ScoreSum a, ScoreSum b) {
  if (a.m < b.m) {
    const ScoreSum t = a;
    a = b;
    b = t;
  }
  if (b.m == -INFINITY) {
    a.s += b.s;  // 0, or the NaN of a part that is all NaN
    return a;
  }
  const float d = fmaxf((b.m - a.m) * kLog2e, -150.f), f = exp2_flush(d);
  a.u += f * fmaf(d, b.s, b.u);
  a.s += f * b.s;
  return a;
}
SJ_DEVICE ScoreSum score_warp_join(ScoreSum a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = score_join(a, ScoreSum{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                               __shfl_xor_sync(0xffffffffu, a.u, o)});
  return a;
}
// One logit into s and u.  The floor keeps 0 * -inf out of u (2^-150 is 0 as well) and lets a NaN pass.
SJ_DEVICE void score_add(float x, float base, float& s, float& u) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"((x - base) * kLog2e), "f"(-150.f));
  const float e = exp2_flush(d);
  s += e;
  u = fmaf(e, d, u);
}

// Floats of a part in the workspace: m, s, u, the number of keys, the keys.
__host__ __device__ constexpr int score_part(int top) { return (4 + 2 * top + 3) / 4 * 4; }

struct ScoreOut {
  const int32_t* target;
  float *logp, *entropy, *lse;
  int32_t* top_id;
  float* top_logp;
  int vocab, top;
};
// log softmax of x in a row of sums a (log_s = log a.s): -inf for a forbidden token.
SJ_DEVICE float score_logp(float x, const ScoreSum& a, float base, float log_s) {
  return x == -INFINITY && a.s == a.s ? -INFINITY : (x - base) - log_s;
}
template <typename T>
SJ_DEVICE void score_write_row(const ScoreOut& out, const T* x, int r, const ScoreSum& a) {
  const float base = a.m == -INFINITY ? 0.f : a.m, log_s = logf(a.s);
  const int at = out.target ? out.target[r] : -1;
  if (at >= out.vocab || at < -1) record_error(SJ_DEV_BAD_INDEX);
  if (out.logp) out.logp[r] = at < 0 || at >= out.vocab ? 0.f : score_logp(score_load(x + at), a, base, log_s);
  if (out.entropy) out.entropy[r] = a.s == 0.f ? 0.f : log_s - a.u / a.s * kLn2;
  if (out.lse) out.lse[r] = base + log_s;
}

// ---------------------------------------------------------------- narrow rows
// A warp holds a row in R registers a lane: one read, maximum, sums, then each alternative by two warp
// reductions (value, then lowest index) and the lane's own next best.
template <typename T, int R>
__global__ void __launch_bounds__(128) token_scores_narrow_kernel(const T* logits, int ld, int rows, ScoreOut out) {
  pdl_wait();
  const int lane = threadIdx.x & 31, r = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= rows) return;
  const T* x = logits + static_cast<size_t>(r) * ld;
  float v[R];
  ScoreSum a{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] = i * 32 + lane < out.vocab ? score_load(x + i * 32 + lane) : -INFINITY;
#pragma unroll
  for (int i = 0; i < R; ++i) a.m = fmaxf(a.m, v[i]);
  a.m = warp_max(a.m);
  const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int i = 0; i < R; ++i) score_add(v[i], base, a.s, a.u);
  a.s = warp_sum(a.s);
  a.u = warp_sum(a.u);
  if (lane == 0) score_write_row(out, x, r, a);
  if (out.top == 0) return;
  const float log_s = logf(a.s);
  uint32_t order[R];
#pragma unroll
  for (int i = 0; i < R; ++i) order[i] = score_order(v[i]);
  uint32_t bound = 0xffffffffu;  // the last alternative's order and index
  int bound_at = -1;
  for (int k = 0; k < out.top; ++k) {
    uint32_t best = 0;
    int best_at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int at = i * 32 + lane;
      const uint32_t up = order[i];
      const bool left = at < out.vocab && (up < bound || (up == bound && at > bound_at));
      if (left && (up > best || best_at == 0x7fffffff)) {
        best = up;
        best_at = at;
      }
    }
    bound = __reduce_max_sync(0xffffffffu, best_at == 0x7fffffff ? 0u : best);
    bound_at = static_cast<int>(
        __reduce_min_sync(0xffffffffu, best == bound ? static_cast<unsigned>(best_at) : 0x7fffffffu));
    if (lane == 0) {
      out.top_id[static_cast<size_t>(r) * out.top + k] = bound_at;
      out.top_logp[static_cast<size_t>(r) * out.top + k] = score_logp(score_value(bound), a, base, log_s);
    }
  }
}

// ---------------------------------------------------------------- wide rows
// Sixteen 4-byte (32 2-byte) logits of a thread's chunk as they are stored.
template <typename T>
struct ScoreChunk {
  static constexpr int PER = 16 / sizeof(T), N = 4 * PER, SIZE = kScoreThreads * N;
  uint4 raw[4];
  SJ_DEVICE static int index(int base, int i) {  // of element i: sixteen bytes of each thread side by side
    return base + (i / PER * kScoreThreads + static_cast<int>(threadIdx.x)) * PER + i % PER;
  }
  SJ_DEVICE float at(int i) const {
    const uint4& q = raw[i / PER];
    if (sizeof(T) == 4) return __uint_as_float(i % 4 == 0 ? q.x : i % 4 == 1 ? q.y : i % 4 == 2 ? q.z : q.w);
    const int w = i % PER / 2;
    const uint32_t pair = w == 0 ? q.x : w == 1 ? q.y : w == 2 ? q.z : q.w;
    return __uint_as_float(i % 2 ? pair & 0xffff0000u : pair << 16);
  }
  // Elements outside [0, vocab) are -inf.  base is a 16-byte boundary.
  SJ_DEVICE void load(const T* x, int base, int vocab) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int j = base + (v * kScoreThreads + static_cast<int>(threadIdx.x)) * PER;
      if (j >= 0 && j + PER <= vocab) {
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(raw[v].x), "=r"(raw[v].y), "=r"(raw[v].z), "=r"(raw[v].w)
                     : "l"(x + j)
                     : "memory");
      } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (sizeof(T) == 4) {
            w[e] = __float_as_uint(j + e >= 0 && j + e < vocab ? score_load(x + j + e) : -INFINITY);
          } else {
            const int a = j + 2 * e;
            const float lo = a >= 0 && a < vocab ? score_load(x + a) : -INFINITY;
            const float hi = a + 1 >= 0 && a + 1 < vocab ? score_load(x + a + 1) : -INFINITY;
            w[e] = __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xffff0000u);
          }
        }
        raw[v] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
};

// The best of the candidates so far.
struct ScoreBest {
  uint64_t held[kScoreHeld];
  uint64_t list[kScoreMaxTop];
  uint64_t thread_best[kScoreThreads];
  uint32_t group[64];
  uint32_t bar;  // order that a group of the first chunk reaches `top` times
  int count;     // of held
};

// held[0, n) cut down to the `top` largest keys, in order, among those whose index is below `before`.
SJ_DEVICE int score_compact(ScoreBest& b, int top, int before) {
  __syncthreads();
  const int n = min(b.count, kScoreHeld);
  for (int i = threadIdx.x; i < n; i += kScoreThreads) {
    const uint64_t key = b.held[i];
    int rank = static_cast<int>(~static_cast<uint32_t>(key)) < before ? 0 : top;
    for (int k = 0; k < n && rank < top; ++k) {
      const uint64_t other = b.held[k];
      rank += other > key && static_cast<int>(~static_cast<uint32_t>(other)) < before ? 1 : 0;
    }
    if (rank < top) b.list[rank] = key;
  }
  int kept = 0;
  for (int i = threadIdx.x; i < n; i += kScoreThreads)
    kept += static_cast<int>(~static_cast<uint32_t>(b.held[i])) < before ? 1 : 0;
  __syncthreads();
  if (threadIdx.x == 0) b.count = 0;
  __syncthreads();
  if (kept) atomicAdd(&b.count, kept);
  __syncthreads();
  kept = min(b.count, top);
  __syncthreads();
  if (threadIdx.x < kept) b.held[threadIdx.x] = b.list[threadIdx.x];
  if (threadIdx.x == 0) b.count = kept;
  __syncthreads();
  return kept;
}

// One CTA for a part of a row (splits > 1: as many parts of equal numbers of chunks), 16 KB at a time with the
// next chunk's loads in flight.  The sums are each thread's own until the part's end.  Alternatives: the
// `top`-th largest of 64 groups' maxima of the first chunk is a bar that at least `top` logits reach; what
// reaches it (of later chunks, exceeds it) goes to a list in shared memory that is ranked once at the end: about
// 24 candidates a chunk at top = 20.  A list that fills up is ranked at once, which raises the bar; a chunk with more
// candidates than the list holds (equal or rising logits) takes those of the `top` threads with the best maxima.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads, 4)
    token_scores_wide_kernel(const T* logits, int ld, int splits, int* counters, float* partial, ScoreOut out) {
  pdl_wait();
  using Chunk = ScoreChunk<T>;
  __shared__ ScoreBest best;
  __shared__ ScoreSum sums[kScoreThreads / 32];
  __shared__ int s_last;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int r = blockIdx.x / splits, split = blockIdx.x % splits, top = out.top, vocab = out.vocab;
  const T* x = logits + static_cast<size_t>(r) * ld;
  const int origin = -static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const int chunks = (vocab - origin + Chunk::SIZE - 1) / Chunk::SIZE;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * split / splits);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / splits);
  if (t == 0) best.count = 0;
  ScoreSum a{-INFINITY, 0.f, 0.f};
  uint32_t bar = 0;    // order to exceed, once `raised`
  bool raised = false;
  Chunk now, next;
  if (c0 < c1) next.load(x, origin + c0 * Chunk::SIZE, vocab);
  for (int c = c0; c < c1; ++c) {
    const int first = origin + c * Chunk::SIZE;
    now = next;
    if (c + 1 < c1) next.load(x, first + Chunk::SIZE, vocab);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < Chunk::N; ++i) m = fmaxf(m, now.at(i));
    if (m > a.m) a = score_join(ScoreSum{m, 0.f, 0.f}, a);
    const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int i = 0; i < Chunk::N; ++i) score_add(now.at(i), base, a.s, a.u);
    if (top == 0) continue;

    const bool any = Chunk::index(first, 0) < vocab;  // a thread's first element is its lowest
    const uint32_t order = any ? score_order(m) : 0u;
    uint32_t reach = raised ? bar + 1 : 0;
    if (!raised) {  // the first chunk: 64 groups of four threads
      uint32_t g = max(order, __shfl_xor_sync(0xffffffffu, order, 1));
      g = max(g, __shfl_xor_sync(0xffffffffu, g, 2));
      if ((lane & 3) == 0) best.group[t >> 2] = g;
      __syncthreads();
      int rank = 0;
      for (int i = 0; i < 16; ++i) {
        const int k = (t & 3) * 16 + i;
        const uint32_t o = best.group[k];
        rank += o > g || (o == g && k < t >> 2) ? 1 : 0;
      }
      rank += __shfl_xor_sync(0xffffffffu, rank, 1);
      rank += __shfl_xor_sync(0xffffffffu, rank, 2);
      if ((lane & 3) == 0 && rank == top - 1) best.bar = g;
      __syncthreads();
      bar = best.bar;
      raised = bar > kForbidden;  // fewer than `top` groups hold more than forbidden tokens: all are candidates
      reach = raised ? bar : 0;
    }
    int held = 0;
    if (any && order >= reach) {
#pragma unroll
      for (int i = 0; i < Chunk::N; ++i) {
        const float v = now.at(i);
        const int j = Chunk::index(first, i);
        if (j >= 0 && j < vocab && score_order(v) >= reach) {
          held = atomicAdd(&best.count, 1) + 1;
          if (held <= kScoreHeld) best.held[held - 1] = score_key(v, j);
        }
      }
    }
    if (__syncthreads_or(held > kScoreHeld)) {
      score_compact(best, top, first);
      uint64_t mine = 0;
      if (any && order >= reach) {
#pragma unroll
        for (int i = 0; i < Chunk::N; ++i) {
          const int j = Chunk::index(first, i);
          if (j >= 0 && j < vocab) mine = max(mine, score_key(now.at(i), j));
        }
      }
      best.thread_best[t] = mine;
      __syncthreads();
      int rank = 0;
      for (int k = 0; k < kScoreThreads; ++k) rank += best.thread_best[k] > mine ? 1 : 0;
      if (mine && rank < top) {
#pragma unroll
        for (int i = 0; i < Chunk::N; ++i) {
          const float v = now.at(i);
          const int j = Chunk::index(first, i);
          if (j >= 0 && j < vocab && score_order(v) >= reach)
            best.held[atomicAdd(&best.count, 1)] = score_key(v, j);
        }
      }
      held = kScoreHeld;
      __syncthreads();
    }
    if (__syncthreads_or(held > kScoreHeld / 2)) {
      if (score_compact(best, top, INT_MAX) == top) {
        bar = static_cast<uint32_t>(best.list[top - 1] >> 32);
        raised = true;
      }
    }
  }

  // ---- the part's sums and alternatives
  a = score_warp_join(a);
  if (lane == 0) sums[warp] = a;
  __syncthreads();
  a = sums[0];
  for (int w = 1; w < kScoreThreads / 32; ++w) a = score_join(a, sums[w]);
  int n = top > 0 ? score_compact(best, top, INT_MAX) : 0;
  if (splits > 1) {
    const int size = score_part(top);
    float* mine = partial + static_cast<size_t>(blockIdx.x) * size;
    if (t < n) reinterpret_cast<uint64_t*>(mine + 4)[t] = best.list[t];
    if (t == 0) *reinterpret_cast<float4*>(mine) = make_float4(a.m, a.s, a.u, __int_as_float(n));
    __syncthreads();
    if (t == 0) {
      __threadfence();
      s_last = atomicAdd(counters + r, 1) == splits - 1;
      if (s_last) counters[r] = 0;
      __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    // the parts in order
    const float* row = partial + static_cast<size_t>(r) * splits * size;
    a = ScoreSum{-INFINITY, 0.f, 0.f};
    for (int k = 0; k < splits; ++k) {
      const float4 p = __ldcg(reinterpret_cast<const float4*>(row + static_cast<size_t>(k) * size));
      a = score_join(a, ScoreSum{p.x, p.y, p.z});
    }
    if (top > 0) {
      if (t == 0) best.count = 0;
      __syncthreads();
      for (int i = t; i < splits * top; i += kScoreThreads) {
        const float* p = row + static_cast<size_t>(i / top) * size;
        if (i % top < __float_as_int(__ldcg(p + 3)))
          best.held[atomicAdd(&best.count, 1)] = __ldcg(reinterpret_cast<const unsigned long long*>(p + 4) + i % top);
      }
      n = score_compact(best, top, INT_MAX);
    }
  }
  if (t == 0) score_write_row(out, x, r, a);
  if (t < top) {  // top <= vocab: the list is full
    const float base = a.m == -INFINITY ? 0.f : a.m;
    const uint64_t key = best.list[t];
    out.top_id[static_cast<size_t>(r) * top + t] = static_cast<int32_t>(~static_cast<uint32_t>(key));
    out.top_logp[static_cast<size_t>(r) * top + t] =
        score_logp(score_value(static_cast<uint32_t>(key >> 32)), a, base, logf(a.s));
  }
}

// ---------------------------------------------------------------- gradient
struct ScoreGrad {
  const int32_t* target;
  const float *lse, *entropy, *d_logp, *d_entropy;
  int vocab;
};
// A row's part of the gradient: g = -p (a + b (log p + h)), + a at the target.
struct ScoreRow {
  float a, b, z, h;
  int at;
  SJ_DEVICE ScoreRow(const ScoreGrad& in, int r, bool reports) {
    at = in.target ? in.target[r] : -1;
    if (at >= in.vocab || at < -1) {
      if (reports) record_error(SJ_DEV_BAD_INDEX);
      at = -1;
    }
    a = in.d_logp && at >= 0 ? in.d_logp[r] : 0.f;
    b = in.d_entropy ? in.d_entropy[r] : 0.f;
    z = in.lse[r];
    h = in.d_entropy ? in.entropy[r] : 0.f;
  }
  SJ_DEVICE float grad(float x, int j) const {
    const float lp = x - z, p = exp2_flush(lp * kLog2e);
    float g = -p * fmaf(b, fmaxf(lp, -1e30f) + h, a);  // a forbidden token: p = 0, and no 0 * -inf
    if (z == -INFINITY) g = 0.f;                       // a row of nothing else
    if (j == at && z != -INFINITY) g += a;
    return g;
  }
};

SJ_DEVICE void score_store(float* d, float g) { *d = g; }
SJ_DEVICE void score_store(__nv_bfloat16* d, float g) { *d = f2bf(g); }

template <typename T>
SJ_DEVICE uint4 score_grad16(const ScoreRow& row, const uint4& q, int j) {
  uint4 y;
  if (sizeof(T) == 4) {
    y.x = __float_as_uint(row.grad(__uint_as_float(q.x), j));
    y.y = __float_as_uint(row.grad(__uint_as_float(q.y), j + 1));
    y.z = __float_as_uint(row.grad(__uint_as_float(q.z), j + 2));
    y.w = __float_as_uint(row.grad(__uint_as_float(q.w), j + 3));
  } else {
    auto pair = [&](uint32_t w, int at) {
      return pack_bf16x2(row.grad(__uint_as_float(w << 16), at), row.grad(__uint_as_float(w & 0xffff0000u), at + 1));
    };
    y.x = pair(q.x, j);
    y.y = pair(q.y, j + 2);
    y.z = pair(q.z, j + 4);
    y.w = pair(q.w, j + 6);
  }
  return y;
}

// Sixteen bytes of logits in, sixteen bytes of gradient out: rows on 16-byte boundaries.  The 16-byte pieces of
// all rows, one after the other, four to a thread (a CTA's side by side), so that narrow rows leave no
// thread idle; a piece that holds the row's end goes element by element.
template <typename T>
__global__ void __launch_bounds__(256) token_scores_bwd_kernel(const T* logits, int ld, T* d_logits, int ldd,
                                                               int64_t pieces, int per_row, ScoreGrad in) {
  pdl_wait();
  constexpr int PER = 16 / sizeof(T);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 1024;
  const int r0 = static_cast<int>(first / per_row), j0 = static_cast<int>(first - static_cast<int64_t>(r0) * per_row);
  uint4 raw[4];
  int r[4], j[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = i * 256 + static_cast<int>(threadIdx.x);
    raw[i] = make_uint4(0, 0, 0, 0);
    r[i] = -1;
    if (first + k < pieces) {
      const int down = (j0 + k) / per_row;
      r[i] = r0 + down;
      j[i] = (j0 + k - down * per_row) * PER;
      if (j[i] + PER <= in.vocab)
        raw[i] = *reinterpret_cast<const uint4*>(logits + static_cast<size_t>(r[i]) * ld + j[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r[i] < 0) continue;
    const ScoreRow row(in, r[i], j[i] == 0);
    T* d = d_logits + static_cast<size_t>(r[i]) * ldd + j[i];
    if (j[i] + PER <= in.vocab) {
      *reinterpret_cast<uint4*>(d) = score_grad16<T>(row, raw[i], j[i]);
    } else {
      for (int e = 0; e < PER; ++e) {
        const int at = j[i] + e;
        score_store(d + e, at < in.vocab ? row.grad(score_load(logits + static_cast<size_t>(r[i]) * ld + at), at) : 0.f);
      }
    }
  }
}

// Any strides and alignments: a CTA for 2048 elements of a row, side by side.
template <typename T>
__global__ void __launch_bounds__(256) token_scores_bwd_any_kernel(const T* logits, int ld, T* d_logits, int ldd,
                                                                   int parts, ScoreGrad in) {
  pdl_wait();
  const int r = blockIdx.x / parts, j0 = blockIdx.x % parts * 2048;
  const ScoreRow row(in, r, j0 == 0 && threadIdx.x == 0);
  const T* x = logits + static_cast<size_t>(r) * ld;
  T* d = d_logits + static_cast<size_t>(r) * ldd;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = j0 + i * 256 + threadIdx.x;
    if (j < ldd) score_store(d + j, j < in.vocab ? row.grad(score_load(x + j), j) : 0.f);
  }
}

}  // namespace sj

using namespace sj;

namespace {
// Parts of a row: enough CTAs for the GPU when the rows are few (4 fit an SM), of at least 4096 logits.
int score_splits(int rows, int vocab) {
  if (vocab <= kScoreNarrow || rows <= 0) return 1;
  const int fill = (4 * sm_count() + rows - 1) / rows, parts = (vocab + 4095) / 4096;
  return std::max(1, std::min({fill, parts, kScoreMaxSplits}));
}
size_t score_counter_bytes(int rows) { return (static_cast<size_t>(rows) * sizeof(int) + 255) / 256 * 256; }

template <typename T>
int scores(const T* logits, int ld, int rows, const ScoreOut& out, void* workspace, cudaStream_t stream) {
  if (out.vocab <= kScoreNarrow) {
    const int regs = (out.vocab + 31) / 32, grid = (rows + 3) / 4;
    launch(regs <= 4   ? token_scores_narrow_kernel<T, 4>
           : regs <= 9 ? token_scores_narrow_kernel<T, 9>
           : regs <= 16 ? token_scores_narrow_kernel<T, 16>
                        : token_scores_narrow_kernel<T, 32>,
           grid, 128, 0, stream, logits, ld, rows, out);
  } else {
    const int splits = score_splits(rows, out.vocab);
    launch(token_scores_wide_kernel<T>, rows * splits, kScoreThreads, 0, stream, logits, ld, splits,
           static_cast<int*>(workspace), reinterpret_cast<float*>(static_cast<char*>(workspace) + score_counter_bytes(rows)),
           out);
  }
  SJ_LAUNCH_CHECK("token_scores");
  return SJ_OK;
}

template <typename T>
int scores_bwd(const T* logits, int ld, T* d_logits, int ldd, int rows, const ScoreGrad& in, cudaStream_t stream) {
  constexpr int PER = 16 / sizeof(T);
  if (aligned16(logits) && aligned16(d_logits) && ld % PER == 0 && ldd % PER == 0) {
    const int per_row = ldd / PER;
    const int64_t pieces = static_cast<int64_t>(rows) * per_row;
    launch(token_scores_bwd_kernel<T>, static_cast<unsigned>((pieces + 1023) / 1024), 256, 0, stream, logits, ld,
           d_logits, ldd, pieces, per_row, in);
  } else {
    const int parts = (ldd + 2047) / 2048;
    if (static_cast<int64_t>(rows) * parts > INT_MAX)
      return fail(SJ_ERR_SHAPE, "sj_token_scores_bwd: rows=%d ldd=%d", rows, ldd);
    launch(token_scores_bwd_any_kernel<T>, static_cast<unsigned>(rows) * parts, 256, 0, stream, logits, ld, d_logits,
           ldd, parts, in);
  }
  SJ_LAUNCH_CHECK("token_scores_bwd");
  return SJ_OK;
}
}  // namespace

extern "C" size_t sj_token_scores_workspace(int rows, int vocab, int top) {
  if (rows < 0 || vocab <= 0 || top < 0 || top > kScoreMaxTop) return 0;
  const int splits = score_splits(rows, vocab);
  if (splits == 1) return 16;
  return score_counter_bytes(rows) + static_cast<size_t>(rows) * splits * score_part(top) * sizeof(float);
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
  const ScoreOut out{target, logp, entropy, lse, top_id, top_logp, vocab, top};
  return dtype == SJ_F32 ? scores(static_cast<const float*>(logits), ld, rows, out, workspace, as_stream(stream))
                         : scores(static_cast<const __nv_bfloat16*>(logits), ld, rows, out, workspace,
                                  as_stream(stream));
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
  const ScoreGrad in{target, lse, entropy, d_logp, d_entropy, vocab};
  if (dtype == SJ_F32)
    return scores_bwd(static_cast<const float*>(logits), ld, static_cast<float*>(d_logits), ldd, rows, in,
                      as_stream(stream));
  return scores_bwd(static_cast<const __nv_bfloat16*>(logits), ld, static_cast<__nv_bfloat16*>(d_logits), ldd, rows, in,
                    as_stream(stream));
}
