// Scores of given tokens under rows of logits, and their gradient.
//
//   lse = m + log s,  m = max x,  s = sum e^(x - m);   logp = (x_t - m) - log s
//   H = -sum p log p = log s - sum e^(x - m) (x - m) / s     (both terms >= 0: nothing cancels)
//   dx_j = dlogp (1[j = t] - p_j) - dH p_j (log p_j + H)
//
// The alternatives are the `top` largest logits, the lowest index first among equal ones: a key of
// (value, ~index) orders them without ties.
//
// Each logit is read once from memory.  Measured on B200 (graph replays): 2048 x 50001 bf16 with 20 alternatives 56 us
// (3.7 TB/s; without alternatives 43, 4.8 TB/s), where instructions bound it, not memory: of a warp's 400 for 1024
// logits, the exponentials' unit takes 32 (8 cycles each), floors and unpacking 64, the alternatives 80.
// 1024 x 50001 f32 40 us (5.1 TB/s).  The first simple kernel (a pass for the maximum, one for the sums, one for each
// alternative) took 1629.  Gradient: 2048 x 65537 bf16 85 us (6.3 TB/s), 1024 x 50001 f32 63 us (6.5).
#include <algorithm>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace sj {

namespace {
constexpr int kScoreMaxTop = 32;
constexpr int kScoreMaxColumns = INT_MAX - (1 << 14);  // 32 bits count to a chunk or a part past the last column
// Rows of at most this many logits are held by one warp: 8000 x 2000 f32 with 20 alternatives 22.2 us, 48.6 by the
// kernel for wide rows, bf16 25.8 and 52.2 (33.5 where the rows are not in L2); 4000 x 4096 f32 24.4 and 33.1, but
// bf16, loaded two bytes at a time, 33.0 and 27.8.
template <typename T>
constexpr int kScoreNarrow = sizeof(T) == 4 ? 4096 : 2048;
// CTAs of an SM, of the kernel that holds R logits a lane: 32768 x 257 f32 with 5 alternatives 20.6 us with nine, 20.2
// with ten, 19.9 with twelve; 32768 x 500 23.7 with ten, 24.2 with twelve, 28.1 without a limit on registers; 32768 x
// 1000 32.6 with seven, 31.8 with eight, 32.3 with nine, 42.5 without a limit; 16000 x 1100 36.9 with four, 34.5 with
// five; 4000 x 4096 28.8 with two, 24.3 with three.
template <int R>
constexpr int kScoreNarrowCtas = R <= 9 ? 12 : R <= 16 ? 10 : R <= 32 ? 8 : R <= 64 ? 5 : 3;
// Alternatives up to which their bar is found one by one, not by a sort: at 32768 x 257 one alternative takes 16.9 us,
// not 19.7, five 20.2, not 21.0, and ten the same either way.
constexpr int kScoreRounds = 8;
constexpr int kScoreThreads = 128, kScoreWarps = kScoreThreads / 32;  // of the kernel for wider rows
constexpr int kScorePieces = 5;       // 16-byte pieces of a chunk that a thread takes
constexpr int kScoreStage = kScoreThreads * kScorePieces * 16;
// CTAs of an SM, stages of a CTA's ring.  Small CTAs and small chunks waste less of a row's last chunk, many pieces a
// thread spread a chunk's fixed cost: with 128 threads, five pieces and seven CTAs, 2048 x 50001 bf16 with 20
// alternatives takes 55.7 us and 1024 x 50001 f32 40.0; with 256, four and four, 68.2 and 49.7; 128, four and eight,
// 62.2 and 43.0; 128, six and six, 59.9 and 51.2; 64, eight and nine, 61.7 and 45.8.  A third stage leaves room for
// five CTAs: 63.0 and 48.7.
constexpr int kScoreCtas = 7, kScoreStages = 2;
constexpr int kScoreMaxSplits = 16;
// The gradient of rows of at most 1024 pieces of 16 bytes: four rows a warp (32768 x 257 f32 13.0 us with eight CTAs of
// four warps an SM, 13.6 with nine; three rows and nine CTAs 15.3, two and eleven 17.1; 8192 x 2000 f32 25.4, 36.7 by
// the kernel for wide rows).
constexpr int kGradRows = 4, kGradNarrowCtas = 8, kGradNarrow = 1024;
// CTAs of an SM, of the gradient's kernel for wide rows: 2048 x 65537 bf16 85.6 us with four, 84.8 with five, 98.6 with
// six; 1024 x 50001 f32 65.6 with three, 62.9 with four, 68.7 with five.
template <typename T>
constexpr int kGradCtas = sizeof(T) == 2 ? 5 : 4;
constexpr int kScoreHeld = kScoreMaxTop * 16 + kScoreMaxTop;  // candidates: the best of 32 threads' 16, and the list
constexpr int kScoreNoted = 512, kScoreKept = 128;  // shares of chunks with candidates (of 2^20 logits, 128 noted)
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

// The largest x of a warp's lanes, none a NaN.
SJ_DEVICE float warp_largest(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 at a time: sm_100 adds, multiplies and fuses a register pair in one instruction.
SJ_DEVICE uint64_t pair2(float a, float b) {
  return static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a);
}
SJ_DEVICE float low2(uint64_t p) { return __uint_as_float(static_cast<uint32_t>(p)); }
SJ_DEVICE float high2(uint64_t p) { return __uint_as_float(static_cast<uint32_t>(p >> 32)); }
SJ_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
SJ_DEVICE uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
SJ_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
// The floor keeps 0 * -inf out of products with 2^x (2^-150 is 0 as well) and lets a NaN pass.
SJ_DEVICE float floor_exponent(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(-150.f));
  return y;
}

// Order-preserving integer of a logit that is no NaN.
SJ_DEVICE uint32_t score_up(float v) {
  const uint32_t bits = __float_as_uint(v);
  return bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
}
// The same where -0 and +0 are equal; NaN last.
SJ_DEVICE uint32_t score_order(float v) { return v != v ? 0u : score_up(v + 0.f); }
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
// The same part with a maximum of at least m.
SJ_DEVICE ScoreSum score_raise(ScoreSum a, float m) {
  const float top = fmaxf(a.m, m);
  const float d = a.m == top ? 0.f : fmaxf((a.m - top) * kLog2e, -150.f), f = exp2_flush(d);
  return ScoreSum{top, f * a.s, f * fmaf(d, a.s, a.u)};
}
// The parts of WIDTH lanes: the maximum first, then each part raised to it once.
template <int WIDTH>
SJ_DEVICE ScoreSum score_lanes_join(ScoreSum a) {
  float m = a.m;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  a = score_raise(a, m);
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  return a;
}

// Two logits into pairs of partial s and u: d = (x - base) log2(e), s += 2^d, u += 2^d d.
SJ_DEVICE void score_add2(uint64_t x, uint64_t minus_base, uint64_t& s, uint64_t& u) {
  uint64_t d = mul2(add2(x, minus_base), pair2(kLog2e, kLog2e));
  d = pair2(floor_exponent(low2(d)), floor_exponent(high2(d)));
  const uint64_t e = pair2(exp2_flush(low2(d)), exp2_flush(high2(d)));
  s = add2(s, e);
  u = fma2(e, d, u);
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
// A row's target and its logit.
struct ScoreTarget {
  int at;
  float x;
  SJ_DEVICE explicit ScoreTarget(int at_) : at(at_), x(0.f) {}
  template <typename T>
  SJ_DEVICE void load(const T* row, int vocab) {
    if (at >= 0 && at < vocab) x = score_load(row + at);
  }
};
SJ_DEVICE void score_write_row(const ScoreOut& out, const ScoreTarget& target, int r, const ScoreSum& a) {
  const float base = a.m == -INFINITY ? 0.f : a.m, log_s = logf(a.s);
  const int at = target.at;
  if (at >= out.vocab || at < -1) record_error(SJ_DEV_BAD_INDEX);
  if (out.logp) out.logp[r] = at < 0 || at >= out.vocab ? 0.f : score_logp(target.x, a, base, log_s);
  if (out.entropy) out.entropy[r] = a.s == 0.f ? 0.f : log_s - a.u / a.s * kLn2;
  if (out.lse) out.lse[r] = base + log_s;
}

// ---------------------------------------------------------------- narrow rows
// A warp holds a row in R registers a lane: one read, maximum, sums.  Alternatives: the `top`-th largest of the
// lanes' maxima is a bar that at least `top` logits reach; the few that do (31 are expected at top = 20) are
// listed and ranked by counting.  Where more than 64 do (ties), or too few are not forbidden, each alternative
// is found by two warp reductions instead (value, then lowest index).
template <typename T, int R>
__global__ void __launch_bounds__(128, kScoreNarrowCtas<R>)
    token_scores_narrow_kernel(const T* logits, int ld, int rows, ScoreOut out) {
  pdl_wait();
  __shared__ uint64_t listed[4][64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.x * 4 + warp;
  if (r >= rows) return;
  const T* x = logits + static_cast<size_t>(r) * ld;
  ScoreTarget target(lane == 0 && out.target ? out.target[r] : -1);
  float v[R + (R & 1)];
  ScoreSum a{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] = i * 32 + lane < out.vocab ? score_load(x + i * 32 + lane) : -INFINITY;
  if (R & 1) v[R] = -INFINITY;
  target.load(x, out.vocab);
#pragma unroll
  for (int i = 0; i < R; ++i) a.m = fmaxf(a.m, v[i]);
  const float lane_max = a.m;
  a.m = warp_largest(a.m);
  const float base = a.m == -INFINITY ? 0.f : a.m;
  uint64_t s = 0, u = 0;
#pragma unroll
  for (int i = 0; i < R; i += 2) score_add2(pair2(v[i], v[i + 1]), pair2(-base, -base), s, u);
  a.s = warp_sum(low2(s) + high2(s));
  a.u = warp_sum(low2(u) + high2(u));
  if (lane == 0) score_write_row(out, target, r, a);
  if (out.top == 0) return;
  const float log_s = logf(a.s);
  auto write = [&](int k, uint64_t key) {
    out.top_id[static_cast<size_t>(r) * out.top + k] = static_cast<int32_t>(~static_cast<uint32_t>(key));
    out.top_logp[static_cast<size_t>(r) * out.top + k] =
        score_logp(score_value(static_cast<uint32_t>(key >> 32)), a, base, log_s);
  };

  float bar = a.m;  // -inf: fewer than `top` lanes hold more than forbidden tokens
  if (out.top <= kScoreRounds) {
    float left = lane_max;
    for (int above = 0;;) {
      const bool is = left == bar;
      above += __popc(__ballot_sync(0xffffffffu, is));
      if (above >= out.top || bar == -INFINITY) break;
      if (is) left = -INFINITY;
      bar = warp_largest(left);
    }
  } else {
    bar = lane_max;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)  // a bitonic sort, the largest first
#pragma unroll
      for (int step = size / 2; step > 0; step /= 2) {
        const float o = __shfl_xor_sync(0xffffffffu, bar, step);
        bar = ((lane & step) == 0) == ((lane & size) == 0) ? fmaxf(bar, o) : fminf(bar, o);
      }
    bar = __shfl_sync(0xffffffffu, bar, out.top - 1);
  }
  int n = 0;
  if (bar > -INFINITY) {
#pragma unroll
    for (int i0 = 0; i0 < R; i0 += 32) {
      uint32_t left = 0;
#pragma unroll
      for (int i = i0; i < R && i < i0 + 32; ++i) left |= v[i] >= bar ? 1u << (i - i0) : 0u;
      for (uint32_t have; (have = __ballot_sync(0xffffffffu, left != 0)) != 0;) {
        const int at = n + __popc(have & ((1u << lane) - 1));
        if (left) {
          const int j = (i0 + __ffs(left) - 1) * 32 + lane;
          if (at < 64) listed[warp][at] = score_key(score_load(x + j), j);
          left &= left - 1;
        }
        n += __popc(have);
      }
    }
    __syncwarp();
  }
  if (n > 0 && n <= 64) {
    const uint64_t first = lane < n ? listed[warp][lane] : 0, second = lane + 32 < n ? listed[warp][lane + 32] : 0;
    int rank = 0, rank2 = 0;
    for (int k = 0; k < n; ++k) rank += listed[warp][k] > first ? 1 : 0;
    if (n > 32)
      for (int k = 0; k < n; ++k) rank2 += listed[warp][k] > second ? 1 : 0;
    if (lane < n && rank < out.top) write(rank, first);
    if (lane + 32 < n && rank2 < out.top) write(rank2, second);
    return;
  }
  uint32_t bound = 0xffffffffu;  // the last alternative's order and index
  int bound_at = -1;
  for (int k = 0; k < out.top; ++k) {
    uint32_t best = 0;
    int best_at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int at = i * 32 + lane;
      const uint32_t up = score_order(v[i]);
      const bool left = at < out.vocab && (up < bound || (up == bound && at > bound_at));
      if (left && (up > best || best_at == 0x7fffffff)) {
        best = up;
        best_at = at;
      }
    }
    bound = __reduce_max_sync(0xffffffffu, best_at == 0x7fffffff ? 0u : best);
    bound_at = static_cast<int>(
        __reduce_min_sync(0xffffffffu, best == bound ? static_cast<unsigned>(best_at) : 0x7fffffffu));
    if (lane == 0) write(k, static_cast<uint64_t>(bound) << 32 | static_cast<uint32_t>(~bound_at));
  }
}

// ---------------------------------------------------------------- wide rows
// A thread's pieces of a chunk of 10 KB of a row: each lies side by side with the other threads'.
template <typename T>
struct ScoreChunk {
  static constexpr int PER = 16 / sizeof(T), N = kScorePieces * PER, SIZE = kScoreThreads * N;
  static constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;  // -inf
  uint4 raw[kScorePieces];
  SJ_DEVICE static int index(int base, int i) {  // column of the thread's element i; base: of the chunk
    return base + (i / PER * kScoreThreads + static_cast<int>(threadIdx.x)) * PER + i % PER;
  }
  SJ_DEVICE static uint4 nothing() { return make_uint4(NONE, NONE, NONE, NONE); }
  SJ_DEVICE static uint32_t word(const uint4& q, int i) { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
  SJ_DEVICE float at(int i) const {
    const uint4& q = raw[i / PER];
    if (sizeof(T) == 4) return __uint_as_float(word(q, i % 4));
    const uint32_t w = word(q, i % PER / 2);
    return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
  }
  // The maximum: NaN left out, -inf where there is nothing else.
  SJ_DEVICE float largest() const {
    if (sizeof(T) == 4) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; ++i) m = fmaxf(m, at(i));
      return m;
    }
    uint32_t m = NONE;
#pragma unroll
    for (int v = 0; v < kScorePieces; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(word(raw[v], i)));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  // The chunk's pieces that lie in the row, on their way to `own`, the thread's place in a stage of shared memory.
  // A chunk inside the row needs no look at its pieces.
  SJ_DEVICE static void fetch(const T* x, int base, int vocab, uint32_t own) {
    const T* src = x + index(base, 0);
    const bool inside = base >= 0 && base + SIZE <= vocab;
#pragma unroll
    for (int v = 0; v < kScorePieces; ++v) {
      const int j = index(base, v * PER);
      if (inside || (j >= 0 && j + PER <= vocab))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(own + v * (16 * kScoreThreads)),
                     "l"(src + v * (PER * kScoreThreads))
                     : "memory");
    }
  }
  SJ_DEVICE static uint4 piece(uint32_t own, int v) {
    uint4 q;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                 : "r"(own + v * (16 * kScoreThreads))
                 : "memory");
    return q;
  }
  // The thread's pieces from its place in a stage, the row's ends from memory; -inf outside [0, vocab).
  SJ_DEVICE void read(const T* x, int base, int vocab, uint32_t own) {
    if (base >= 0 && base + SIZE <= vocab) {
#pragma unroll
      for (int v = 0; v < kScorePieces; ++v) raw[v] = piece(own, v);
      return;
    }
#pragma unroll
    for (int v = 0; v < kScorePieces; ++v) {
      const int j = index(base, v * PER);
      raw[v] = nothing();
      if (j >= 0 && j + PER <= vocab) {
        raw[v] = piece(own, v);
      } else if (j < vocab) {
        uint32_t w[4] = {NONE, NONE, NONE, NONE};
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          if (j + e < 0 || j + e >= vocab) continue;
          const uint32_t bits = __float_as_uint(score_load(x + j + e));
          if (sizeof(T) == 4)
            w[e % 4] = bits;
          else
            w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | (bits & 0xffff0000u) : (w[e / 2] & 0xffff0000u) | bits >> 16;
        }
        raw[v] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
};

// The chunks of the parts that a CTA takes: part blockIdx.x, + gridDim.x, ...; part p is the (p % splits)-th of
// equal numbers of chunks of row p / splits.  Columns are counted from the 16-byte boundary at or before the row.
template <typename T>
struct ScoreWalk {
  const T *logits, *x;
  int ld, vocab, splits, parts, part, origin, c, c1, start;
  SJ_DEVICE ScoreWalk(const T* all, int ld_, int vocab_, int splits_, int parts_)
      : logits(all), ld(ld_), vocab(vocab_), splits(splits_), parts(parts_), part(blockIdx.x) {
    enter();
  }
  SJ_DEVICE void enter() {
    if (part >= parts) return;
    const int r = splits == 1 ? part : part / splits, k = part - r * splits;
    x = logits + static_cast<size_t>(r) * ld;
    origin = -static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const int chunks = (vocab - origin + ScoreChunk<T>::SIZE - 1) / ScoreChunk<T>::SIZE;
    c = splits == 1 ? 0 : chunks * k / splits;  // at most 2^20 chunks, 16 splits; a chunk a part at least
    c1 = splits == 1 ? chunks : chunks * (k + 1) / splits;
    start = base();
  }
  SJ_DEVICE void leave() {
    part += gridDim.x;
    enter();
  }
  SJ_DEVICE int base() const { return origin + c * ScoreChunk<T>::SIZE; }
  SJ_DEVICE void fetch(uint32_t own) {  // the next chunk, whichever part it is of
    while (part < parts && c >= c1) leave();
    if (part < parts) {
      ScoreChunk<T>::fetch(x, base(), vocab, own);
      ++c;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
};

// The best of the candidates so far.
struct ScoreBest {
  uint64_t held[kScoreHeld];
  uint64_t list[kScoreMaxTop];
  uint64_t thread_best[kScoreThreads];
  __align__(4) uint16_t group[64];
  int noted[kScoreNoted];  // first columns of the threads' shares of chunks that reached the bar
  float met[kScoreNoted];  // their maxima
  int kept[kScoreKept];    // those that reach the last bar
  float bar;
  int count, notes, keeps;  // of held, noted, kept
  SJ_DEVICE void clear() {
    bar = -INFINITY;
    count = notes = keeps = 0;
  }
};

// The bar: a logit that at least `top` of the part's reach.  64 groups of threads keep the largest order that they
// have met, of which 16 bits make the bar no higher than it may be; the `top`-th largest of them is one.  One that is
// out of date still holds.  -inf when fewer than `top` groups hold more than forbidden tokens.
SJ_DEVICE void score_group(ScoreBest& b, uint32_t order) {
  constexpr int OF = kScoreThreads / 64;  // threads of a group
#pragma unroll
  for (int o = 1; o < OF; o <<= 1) order = max(order, __shfl_xor_sync(0xffffffffu, order, o));
  if (threadIdx.x % OF == 0) b.group[threadIdx.x / OF] = static_cast<uint16_t>(order >> 16);
}
// By one warp, whatever the others have come to: bitonic sorts of the low and of the high half of each lane, the
// largest first; of sorted a and b the k-th largest is the largest min(a_j, b_(k-j)).
SJ_DEVICE void score_raise_bar(ScoreBest& b, int top) {
  const int lane = threadIdx.x & 31;
  uint32_t v = reinterpret_cast<const volatile uint32_t*>(b.group)[lane];
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, v, step);
      const bool larger = ((lane & step) == 0) == ((lane & size) == 0);
      v = larger ? __vmaxu2(v, o) : __vminu2(v, o);
    }
  const uint32_t other = __shfl_sync(0xffffffffu, v, (top - 2 - lane) & 31) >> 16, low = v & 0xffffu;
  const uint32_t mine = lane < top - 1 ? min(low, other) : lane == top - 1 ? max(low, v >> 16) : 0u;
  const uint32_t bar = __reduce_max_sync(0xffffffffu, mine);
  if (lane == 0 && bar > kForbidden >> 16) *const_cast<volatile float*>(&b.bar) = score_value(bar << 16);
}

// The `top` largest keys of held, which all threads see, in order into list; returns how many there are.
SJ_DEVICE int score_rank(ScoreBest& b, int top) {
  const int n = b.count;
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kScoreThreads) {
    const uint64_t key = b.held[i];
    int rank = 0;
#pragma unroll 8
    for (int k = 0; k < n; ++k) rank += b.held[k] > key ? 1 : 0;
    if (rank < top) b.list[rank] = key;
  }
  __syncthreads();
  return min(n, top);
}

// The same where more logits reach the bar than the list holds (equal or rising logits): columns [base, end) once
// more, 2048 at a time, of which those of the `top` threads with the best maxima join the list; it is ranked each
// time.  Leaves best.list; returns its length.  2048 x 50001 bf16 with 20 alternatives take 550 us where all are equal,
// 1590 where they rise along the row, 333 where 100 tokens of a row are allowed and 605 where 11 are, since fewer than
// `top` groups of threads then hold one and there is no bar (57 us at random, 99 where they fall).
template <typename T>
SJ_DEVICE int score_rank_all(ScoreBest& best, const T* x, int base, int end, int top) {
  constexpr int N = 16;  // logits of a thread at a time
  __syncthreads();
  if (threadIdx.x == 0) best.count = 0;
  int n = 0;
  for (; base < end; base += kScoreThreads * N) {
    const uint32_t reach = n == top ? static_cast<uint32_t>(best.list[top - 1] >> 32) + 1 : 0u;
    uint64_t mine = 0;
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      const int j = base + i * kScoreThreads + static_cast<int>(threadIdx.x);
      if (j < 0 || j >= end) continue;
      const uint64_t key = score_key(score_load(x + j), j);
      if (static_cast<uint32_t>(key >> 32) >= reach) mine = max(mine, key);
    }
    __syncthreads();
    best.thread_best[threadIdx.x] = mine;
    __syncthreads();
    int rank = 0;
    for (int k = 0; k < kScoreThreads; ++k) rank += best.thread_best[k] > mine ? 1 : 0;
    if (mine && rank < top) {
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
        const int j = base + i * kScoreThreads + static_cast<int>(threadIdx.x);
        if (j < 0 || j >= end) continue;
        const uint64_t key = score_key(score_load(x + j), j);
        if (static_cast<uint32_t>(key >> 32) >= reach) best.held[atomicAdd(&best.count, 1)] = key;
      }
    }
    __syncthreads();
    n = score_rank(best, top);
    if (threadIdx.x < n) best.held[threadIdx.x] = best.list[threadIdx.x];
    if (threadIdx.x == 0) best.count = n;
    __syncthreads();
  }
  return n;
}

// Persistent CTAs over the parts of rows, 10 KB at a time; the next chunk, be it of the next part, is on its way
// to shared memory meanwhile (cp.async; a thread reads back only what it copied, so copies need no barrier).  The
// sums are each thread's own until the part's end.  Where a thread's share of a chunk reaches the bar of the
// alternatives is noted (of 50001 logits at top = 20 about 70 places); at the end, the pieces of those that reach the
// last bar (about 25) are looked at and the logits that do are ranked.  After the two barriers of a part's first bar
// the warps go on without any; in turn, they raise the bar at every other chunk (55.7 us; at every one 56.8).
template <typename T>
__global__ void __launch_bounds__(kScoreThreads, kScoreCtas)
    token_scores_wide_kernel(const T* logits, int ld, int splits, int parts, int* counters, float* partial,
                             ScoreOut out) {
  pdl_wait();
  using Chunk = ScoreChunk<T>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ ScoreBest best;
  __shared__ ScoreSum sums[2][kScoreWarps];
  __shared__ int s_last;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, top = out.top, vocab = out.vocab;
  const uint32_t stages = smem_u32(ring) + t * 16;
  int one;  // not a constant that the compiler sees: gathering a warp's additions costs more than they do
  asm volatile("mov.u32 %0, 1;" : "=r"(one));
  auto next = [&](int* count) {
    int at;
    asm volatile("atom.shared.add.u32 %0, [%1], %2;" : "=r"(at) : "r"(smem_u32(count)), "r"(one) : "memory");
    return at;
  };
  // Files the logits of the piece at column j0 that reach the bar.
  auto look = [&](const T* x, int j0) {
    const float bar = best.bar;
    auto push = [&](float y, int j) {
      const int at = next(&best.count);
      if (at < kScoreHeld) best.held[at] = score_key(y, j);
    };
    if (bar > -INFINITY && j0 >= 0 && j0 + Chunk::PER <= vocab) {
      const uint4 q = *reinterpret_cast<const uint4*>(x + j0);
      auto value = [&](int e) {
        const uint32_t w = Chunk::word(q, e * static_cast<int>(sizeof(T)) / 4);
        return __uint_as_float(sizeof(T) == 4 ? w : e % 2 ? w & 0xffff0000u : w << 16);
      };
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < Chunk::PER; ++e) hits |= value(e) >= bar ? 1u << e : 0u;
      for (; hits; hits &= hits - 1) push(value(__ffs(hits) - 1), j0 + __ffs(hits) - 1);
      return;
    }
#pragma unroll 1
    for (int j = max(j0, 0); j < min(j0 + Chunk::PER, vocab); ++j) {
      const float y = score_load(x + j);
      if (!(y < bar)) push(y, j);  // a NaN as well: it comes last
    }
  };
  ScoreWalk<T> ahead(logits, ld, vocab, splits, parts);
  for (int i = 0; i < kScoreStages - 1; ++i) ahead.fetch(stages + i * kScoreStage);
  int stage = 0, turn = 0;
  if (t == 0) best.clear();
  __syncthreads();
  for (ScoreWalk<T> here(logits, ld, vocab, splits, parts); here.part < parts; here.leave()) {
    const T* x = here.x;
    const int r = splits == 1 ? here.part : here.part / splits;
    ScoreTarget target(t == 0 && out.target ? out.target[r] : -1);
    float m = -INFINITY;  // the thread's maximum; s, u: its sums, in two halves
    uint64_t s = 0, u = 0;
    for (; here.c < here.c1; ++here.c) {
      const int first = here.base();
      asm volatile("cp.async.wait_group %0;" ::"n"(kScoreStages - 2) : "memory");
      const uint32_t own = stages + stage * kScoreStage;
      ahead.fetch(stages + (stage == 0 ? kScoreStages - 1 : stage - 1) * kScoreStage);
      stage = stage == kScoreStages - 1 ? 0 : stage + 1;
      if (t == 0 && here.c + 1 == here.c1) target.load(x, vocab);
      float here_m = -INFINITY;
      if (first + warp * 32 * Chunk::PER < vocab) {  // not past the row's end
        Chunk now;
        now.read(x, first, vocab, own);
        here_m = now.largest();
        if (__any_sync(0xffffffffu, here_m > m)) {  // as score_raise
          const float raised = fmaxf(m, here_m);
          const float d = m == raised ? 0.f : fmaxf((m - raised) * kLog2e, -150.f), f = exp2_flush(d);
          u = mul2(pair2(f, f), fma2(pair2(d, d), s, u));
          s = mul2(pair2(f, f), s);
          m = raised;
        }
        const float minus_base = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int i = 0; i < Chunk::N; i += 2)
          score_add2(pair2(now.at(i), now.at(i + 1)), pair2(minus_base, minus_base), s, u);
      }
      if (top == 0) continue;

      score_group(best, score_up(m));  // -inf from nothing: no more than kForbidden
      if (first == here.start) {
        __syncthreads();
        if (warp == 0) score_raise_bar(best, top);
        __syncthreads();
      } else if (here.c % 2 == 1 && warp == here.c / 2 % kScoreWarps) {
        score_raise_bar(best, top);
      }
      // the threads that meet the bar are few: they are noted, and looked at once the bar has risen
      const float bar = *const_cast<volatile float*>(&best.bar);
      const int column = Chunk::index(first, 0);  // a thread's first element is its lowest
      if (here_m >= bar && column < vocab) {
        const int at = next(&best.notes);
        if (at < kScoreNoted) {
          best.noted[at] = column;
          best.met[at] = here_m;
        }
      }
    }

    // ---- the part's sums and alternatives
    ScoreSum a = score_lanes_join<32>(ScoreSum{m, low2(s) + high2(s), low2(u) + high2(u)});
    if (lane == 0) sums[turn][warp] = a;
    int n = 0;
    __syncthreads();
    if (top > 0) {
      const int notes = best.notes;
      for (int i = t; i < min(notes, kScoreNoted); i += kScoreThreads)
        if (best.met[i] >= best.bar) {
          const int at = next(&best.keeps);
          if (at < kScoreKept) best.kept[at] = best.noted[i];
        }
      __syncthreads();
      const int keeps = best.keeps;
      for (int i = t; i < min(keeps, kScoreKept) * kScorePieces; i += kScoreThreads)
        look(x, best.kept[i / kScorePieces] + i % kScorePieces * (Chunk::PER * kScoreThreads));
      __syncthreads();
      n = notes > kScoreNoted || keeps > kScoreKept || best.count > kScoreHeld
              ? score_rank_all(best, x, here.start, min(vocab, here.origin + here.c1 * Chunk::SIZE), top)
              : score_rank(best, top);
      if (t == 0) best.clear();  // seen by all after the next part's first barrier
    }
    // What follows is warp 0's; the others go on.  Sums have two turns, since warp 0 may still read these.
    if (warp == 0) a = score_lanes_join<kScoreWarps>(sums[turn][lane % kScoreWarps]);
    turn ^= 1;
    bool writes = true;
    if (splits > 1) {
      const int size = score_part(top);
      float* mine = partial + static_cast<size_t>(here.part) * size;
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
      writes = s_last != 0;
      if (writes) {  // the row's parts, in order
        const float* row = partial + static_cast<size_t>(r) * splits * size;
        a = ScoreSum{-INFINITY, 0.f, 0.f};
        for (int k = 0; k < splits; ++k) {
          const float4 p = __ldcg(reinterpret_cast<const float4*>(row + static_cast<size_t>(k) * size));
          a = score_join(a, ScoreSum{p.x, p.y, p.z});
        }
        if (top > 0) {
          for (int i = t; i < splits * top; i += kScoreThreads) {
            const float* p = row + static_cast<size_t>(i / top) * size;
            if (i % top < __float_as_int(__ldcg(p + 3)))
              best.held[atomicAdd(&best.count, 1)] =
                  __ldcg(reinterpret_cast<const unsigned long long*>(p + 4) + i % top);
          }
          __syncthreads();
          n = score_rank(best, top);
          if (t == 0) best.clear();
        }
      }
    }
    if (writes && t == 0) score_write_row(out, target, r, a);
    if (writes && t < top) {  // top <= vocab: the list is full
      const float base = a.m == -INFINITY ? 0.f : a.m;
      const uint64_t key = best.list[t];
      out.top_id[static_cast<size_t>(r) * top + t] = static_cast<int32_t>(~static_cast<uint32_t>(key));
      out.top_logp[static_cast<size_t>(r) * top + t] =
          score_logp(score_value(static_cast<uint32_t>(key >> 32)), a, base, logf(a.s));
    }
  }
}

// ---------------------------------------------------------------- gradient
struct ScoreGrad {
  const int32_t* target;
  const float *lse, *entropy, *d_logp, *d_entropy;
  int vocab;
};
// A row's scalars, none of whose loads waits for another.
struct ScoreScalars {
  int at;
  float z, h, a, b;
  SJ_DEVICE ScoreScalars(const ScoreGrad& in, int r)
      : at(in.target ? in.target[r] : -1), z(in.lse[r]), h(in.d_entropy ? in.entropy[r] : 0.f),
        a(in.d_logp ? in.d_logp[r] : 0.f), b(in.d_entropy ? in.d_entropy[r] : 0.f) {}
};
// A row's part of the gradient: with d = (x - z) log2(e), g = 2^d (-(a + b h) - b ln(2) d), and + a at the target.
struct ScoreRow {
  float minus_z, c, b2, a;
  int at;
  SJ_DEVICE ScoreRow(const ScoreGrad& in, const ScoreScalars& row, bool reports) {
    at = row.at;
    if (at >= in.vocab || at < -1) {
      if (reports) record_error(SJ_DEV_BAD_INDEX);
      at = -1;
    }
    a = at >= 0 ? row.a : 0.f;
    if (row.z == -INFINITY) at = -1;  // a row of forbidden tokens only: no gradient
    minus_z = row.z == -INFINITY ? row.z : -row.z;
    c = row.z == -INFINITY ? 0.f : in.d_entropy ? -fmaf(row.b, row.h, a) : -a;
    b2 = row.z == -INFINITY ? 0.f : -row.b * kLn2;
  }
  SJ_DEVICE ScoreRow(const ScoreGrad& in, int r, bool reports) : ScoreRow(in, ScoreScalars(in, r), reports) {}
  SJ_DEVICE ScoreRow() {}
  SJ_DEVICE ScoreRow of_lane(int i) const {
    ScoreRow row;
    row.minus_z = __shfl_sync(0xffffffffu, minus_z, i);
    row.c = __shfl_sync(0xffffffffu, c, i);
    row.b2 = __shfl_sync(0xffffffffu, b2, i);
    row.a = __shfl_sync(0xffffffffu, a, i);
    row.at = __shfl_sync(0xffffffffu, at, i);
    return row;
  }
  SJ_DEVICE uint64_t grad2(uint64_t x) const {
    uint64_t d = mul2(add2(x, pair2(minus_z, minus_z)), pair2(kLog2e, kLog2e));
    d = pair2(floor_exponent(low2(d)), floor_exponent(high2(d)));
    const uint64_t p = pair2(exp2_flush(low2(d)), exp2_flush(high2(d)));
    return mul2(p, fma2(pair2(b2, b2), d, pair2(c, c)));
  }
  SJ_DEVICE float grad(float x, int j) const {
    const float g = low2(grad2(pair2(x, x)));
    return j == at ? g + a : g;
  }
};

SJ_DEVICE void score_store(float* d, float g) { *d = g; }
SJ_DEVICE void score_store(__nv_bfloat16* d, float g) { *d = f2bf(g); }

// Sixteen bytes of logits to sixteen bytes of gradient, but for the target's own.
template <typename T>
SJ_DEVICE uint4 score_grad16(const ScoreRow& row, const uint4& q) {
  if (sizeof(T) == 4) {
    const uint64_t a = row.grad2(pair2(__uint_as_float(q.x), __uint_as_float(q.y)));
    const uint64_t b = row.grad2(pair2(__uint_as_float(q.z), __uint_as_float(q.w)));
    return make_uint4(static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b),
                      static_cast<uint32_t>(b >> 32));
  }
  auto two = [&](uint32_t w) {
    const uint64_t g = row.grad2(pair2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
    return pack_bf16x2(low2(g), high2(g));
  };
  return make_uint4(two(q.x), two(q.y), two(q.z), two(q.w));
}

// The two kernels for rows on 16-byte boundaries take the pieces that lie whole in the row as such, and the columns
// after them one by one.  The target's gradient is computed before anything is written (d may be x) and written
// last.

// Narrow rows: a warp for four rows, their loads in flight together; lane i looks up row i's scalars.
template <typename T>
__global__ void __launch_bounds__(128, kGradNarrowCtas)
    token_scores_bwd_narrow_kernel(const T* logits, int ld, T* d_logits, int ldd, int rows, ScoreGrad in) {
  pdl_wait();
  constexpr int PER = 16 / sizeof(T), ROWS = kGradRows;
  const int lane = threadIdx.x & 31, r0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * ROWS, live = min(ROWS, rows - r0);
  if (live <= 0) return;
  const int whole = in.vocab / PER, tail = ldd - whole * PER;  // columns after the whole pieces, with the padding
  const T* x = logits + static_cast<size_t>(r0) * ld;
  T* d = d_logits + static_cast<size_t>(r0) * ldd;
  uint4 raw[ROWS][2];
  auto load = [&](int k) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        raw[i][e] = make_uint4(0, 0, 0, 0);
        if (i < live && k + e * 32 < whole)
          raw[i][e] = reinterpret_cast<const uint4*>(x + static_cast<size_t>(i) * ld)[k + e * 32];
      }
  };
  // Element e of the rows' tails.
  auto load_tail = [&](int e) {
    const int i = e / tail, j = whole * PER + e % tail;
    return i < live && j < in.vocab ? score_load(x + static_cast<size_t>(i) * ld + j) : 0.f;
  };
  load(lane);
  const float last = tail > 0 ? load_tail(lane) : 0.f;
  const int mine = min(lane, live - 1);
  const ScoreRow all(in, r0 + mine, lane < live);
  const float own =
      all.at >= 0 ? all.grad(score_load(x + static_cast<size_t>(mine) * ld + all.at), all.at) : 0.f;
  __syncwarp();
  for (int k0 = 0; k0 < whole; k0 += 64) {  // the same for every lane: they exchange the rows' scalars
    const int k = k0 + lane;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const ScoreRow row = all.of_lane(i);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (i < live && k + e * 32 < whole)
          reinterpret_cast<uint4*>(d + static_cast<size_t>(i) * ldd)[k + e * 32] = score_grad16<T>(row, raw[i][e]);
    }
    load(k + 64);
  }
  for (int e0 = 0; e0 < live * tail; e0 += 32) {
    const int e = e0 + lane, i = min(e / tail, live - 1), j = whole * PER + e % tail;
    const ScoreRow row = all.of_lane(i);
    if (e < live * tail)
      score_store(d + static_cast<size_t>(i) * ldd + j,
                  j < in.vocab ? row.grad(e0 == 0 ? last : load_tail(e), j) : 0.f);
  }
  __syncwarp();
  if (lane < live && all.at >= 0) score_store(d + static_cast<size_t>(lane) * ldd + all.at, own);
}

// Wide rows: persistent CTAs over parts of 1024 pieces, four pieces a thread; the next part's loads in flight.
template <typename T>
struct ScorePart {
  static constexpr int PER = 16 / sizeof(T);
  int r, k;  // row; this thread's first piece
  uint4 raw[4];
  SJ_DEVICE void load(const T* logits, int ld, int part, int per_row, int whole) {
    r = part / per_row;
    k = (part - r * per_row) * 1024 + static_cast<int>(threadIdx.x);
    const uint4* src = reinterpret_cast<const uint4*>(logits + static_cast<size_t>(r) * ld) + k;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i * 256 < whole) raw[i] = src[i * 256];
  }
};

template <typename T>
__global__ void __launch_bounds__(256, kGradCtas<T>)
    token_scores_bwd_wide_kernel(const T* logits, int ld, T* d_logits, int ldd, int parts, int per_row, ScoreGrad in) {
  pdl_wait();
  constexpr int PER = 16 / sizeof(T);
  const int whole = in.vocab / PER;
  ScorePart<T> next;
  next.load(logits, ld, blockIdx.x, per_row, whole);
  for (int part = blockIdx.x; part < parts;) {
    const ScorePart<T> now = next;
    part += gridDim.x;
    const ScoreRow row(in, now.r, now.k == 0);
    if (part < parts) next.load(logits, ld, part, per_row, whole);
    const T* x = logits + static_cast<size_t>(now.r) * ld;
    T* d = d_logits + static_cast<size_t>(now.r) * ldd;
    const int home = row.at / PER - now.k;  // the target's piece is this thread's
    const bool owner = row.at >= 0 && row.at < whole * PER && home >= 0 && home < 1024 && home % 256 == 0;
    const float own = owner ? row.grad(score_load(x + row.at), row.at) : 0.f;
    uint4* dst = reinterpret_cast<uint4*>(d) + now.k;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (now.k + i * 256 < whole) dst[i * 256] = score_grad16<T>(row, now.raw[i]);
    if (now.k - static_cast<int>(threadIdx.x) + 1024 > whole) {  // the row's end, which one part takes
      const int done = max(now.k - static_cast<int>(threadIdx.x), whole) * PER;
      for (int j = done + static_cast<int>(threadIdx.x); j < ldd && j < done + 1024 * PER; j += 256)
        score_store(d + j, j < in.vocab ? row.grad(score_load(x + j), j) : 0.f);
    }
    if (owner) score_store(d + row.at, own);
  }
}

// Any strides and alignments: a CTA for 2048 elements of a row, side by side.  1024 x 50001 f32 79 us (63 on 16-byte
// boundaries), 2048 x 65537 bf16 174 (83.5); narrow rows leave most of a CTA idle: 32768 x 257 f32 67 us (12.9), bf16
// 68 (10.3).
template <typename T>
__global__ void __launch_bounds__(256) token_scores_bwd_any_kernel(const T* logits, int ld, T* d_logits, int ldd,
                                                                   int parts, ScoreGrad in) {
  pdl_wait();
  const int r = blockIdx.x / parts, j0 = blockIdx.x % parts * 2048;
  const ScoreRow row(in, r, j0 == 0 && threadIdx.x == 0);
  const T* x = logits + static_cast<size_t>(r) * ld;
  T* d = d_logits + static_cast<size_t>(r) * ldd;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = j0 + i * 256 + static_cast<int>(threadIdx.x);
    v[i] = j < in.vocab ? score_load(x + j) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t g = row.grad2(pair2(v[i], v[i + 1]));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = j0 + (i + e) * 256 + static_cast<int>(threadIdx.x);
      const float y = e ? high2(g) : low2(g);
      if (j < ldd) score_store(d + j, j < in.vocab ? (j == row.at ? y + row.a : y) : 0.f);
    }
  }
}

}  // namespace sj

using namespace sj;

namespace {
int score_ctas() { return kScoreCtas * sm_count(); }
// Rows are cut into parts where there are fewer than this many of them.
int score_cut_rows() { return score_ctas() * 2 / 5; }
// Parts of a row, one for each 4096 logits at most: the fewest that give two CTAs of five one, since a CTA that has its
// SM to itself runs faster and a part costs its own ranking and a share of a join (128 x 130000 f32, which it cuts in
// four: 29.7 us in two, 23.4 in four, 25.8 in seven; 400 x 32000 f32, at its border: 18.4 us whole, 20.5 in two, 28.7
// in three).  For the same reason a partly filled last round of whole rows is left as it is.
int score_splits(int rows, int vocab) {
  if (rows <= 0 || rows >= score_cut_rows()) return 1;
  const int fill = (score_cut_rows() + rows - 1) / rows;
  return std::max(1, std::min({fill, (vocab + 4095) / 4096, kScoreMaxSplits}));
}
// Counters of a workspace, ahead of the parts: of a fixed size, so that no call's parts lie on another call's counters.
size_t score_counter_bytes() { return (static_cast<size_t>(score_cut_rows()) * sizeof(int) + 255) / 256 * 256; }

template <typename T>
int scores(const T* logits, int ld, int rows, const ScoreOut& out, void* workspace, cudaStream_t stream) {
  if (out.vocab <= kScoreNarrow<T>) {
    const int regs = (out.vocab + 31) / 32, grid = (rows - 1) / 4 + 1;
    launch(regs <= 4   ? token_scores_narrow_kernel<T, 4>
           : regs <= 9 ? token_scores_narrow_kernel<T, 9>
           : regs <= 16 ? token_scores_narrow_kernel<T, 16>
           : regs <= 32 ? token_scores_narrow_kernel<T, 32>
           : regs <= 64 ? token_scores_narrow_kernel<T, 64>
                        : token_scores_narrow_kernel<T, kScoreNarrow<T> / 32>,
           grid, 128, 0, stream, logits, ld, rows, out);
  } else {
    // No more parts than chunks: the CTA that ends a row writes with the target's logit that it read at its part's last
    // chunk.
    const int chunks = (out.vocab - 1) / ScoreChunk<T>::SIZE + 1, smem = kScoreStages * kScoreStage;
    const int splits = std::min(score_splits(rows, out.vocab), chunks);
    if (static_cast<int64_t>(rows) * splits > INT_MAX - score_ctas())
      return fail(SJ_ERR_SHAPE, "sj_token_scores: rows=%d vocab=%d", rows, out.vocab);
    static KernelAttrOnce once;
    const int rc = ensure_max_smem(once, reinterpret_cast<const void*>(token_scores_wide_kernel<T>), smem,
                                   "sj_token_scores: shared memory");
    if (rc != SJ_OK) return rc;
    launch(token_scores_wide_kernel<T>, std::min(rows * splits, score_ctas()), kScoreThreads, smem, stream, logits, ld,
           splits, rows * splits, static_cast<int*>(workspace),
           reinterpret_cast<float*>(static_cast<char*>(workspace) + score_counter_bytes()), out);
  }
  SJ_LAUNCH_CHECK("token_scores");
  return SJ_OK;
}

template <typename T>
int scores_bwd(const T* logits, int ld, T* d_logits, int ldd, int rows, const ScoreGrad& in, cudaStream_t stream) {
  constexpr int PER = 16 / sizeof(T);
  if (aligned16(logits) && aligned16(d_logits) && ld % PER == 0 && ldd % PER == 0) {
    if (ldd / PER <= kGradNarrow) {
      launch(token_scores_bwd_narrow_kernel<T>, (rows - 1) / (4 * kGradRows) + 1, 128, 0, stream, logits, ld, d_logits,
             ldd, rows, in);
    } else {
      const int per_row = (ldd / PER + 1023) / 1024;
      if (static_cast<int64_t>(rows) * per_row > INT_MAX / 2)
        return fail(SJ_ERR_SHAPE, "sj_token_scores_bwd: rows=%d ldd=%d", rows, ldd);
      const int parts = rows * per_row;
      launch(token_scores_bwd_wide_kernel<T>, std::min(parts, kGradCtas<T> * sm_count()), 256, 0, stream, logits, ld,
             d_logits, ldd, parts, per_row, in);
    }
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
  if (rows < 0 || vocab <= 0 || vocab > kScoreMaxColumns || top < 0 || top > kScoreMaxTop) return 0;
  const int splits = score_splits(rows, vocab);
  if (splits == 1) return 16;
  return score_counter_bytes() + static_cast<size_t>(rows) * splits * score_part(top) * sizeof(float);
}

extern "C" int sj_token_scores(const void* logits, int dtype, int ld, const int32_t* target, int rows, int vocab,
                               int top, float* logp, float* entropy, float* lse, int32_t* top_id, float* top_logp,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || vocab <= 0 || vocab > kScoreMaxColumns || ld < vocab || top < 0 || top > kScoreMaxTop || top > vocab)
    return fail(SJ_ERR_SHAPE, "sj_token_scores: rows=%d vocab=%d (up to %d) ld=%d top=%d (up to %d)", rows, vocab,
                kScoreMaxColumns, ld, top, kScoreMaxTop);
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
  if (rows < 0 || vocab <= 0 || ld < vocab || ldd < vocab || ldd > kScoreMaxColumns)
    return fail(SJ_ERR_SHAPE, "sj_token_scores_bwd: rows=%d vocab=%d ld=%d ldd=%d (up to %d)", rows, vocab, ld, ldd,
                kScoreMaxColumns);
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
