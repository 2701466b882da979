// Selection of a beam search (sj_beam_select).
//
//   total[b][t] = score[b] + (x[b][t] - lse[b]),  lse[b] = log sum_t e^x[b][t]
//
// and the `keep` largest of a request's beams * vocab totals, the lowest b * vocab + t first among equal ones.
// Within a beam the order is that of the logits, so a beam's candidates are found by their logits, next to its sum
// of exponentials; totals are compared in f64, since those of different beams lie next to one another.
//
//   beam_narrow_kernel  small vocabularies: a CTA for a request, a warp for a beam, the row in registers
//   beam_wide_kernel    parts of rows: sums and the `keep` best logits of each; the CTA that ends a request joins them
//
// Each logit is read once from memory; a bar that at least `keep` logits reach, found from the threads' maxima, picks
// the few threads whose logits are looked at again.
//
// Measured on B200 (graph replays): 128 requests of 8 beams, 50001 bf16 logits, 16 kept 43 us (2.4 TB/s; 27 without the
// candidates, which are chains of waits at a row's and a request's end), f32 70 (2.9 TB/s); one request of 5 beams,
// 131075 f32 logits 29; 16 requests of 4 beams, 257 f32 logits 6.4, where latency counts.  Candidates sought by each
// thread in its own logits took 53 us on the first, 25 waits one after the other.
#include <algorithm>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace sj {

namespace {
constexpr int kBeamMaxBeams = 64, kBeamMaxKeep = 64, kBeamMaxRequests = 4096;
constexpr int kBeamMaxColumns = INT_MAX - (1 << 16);  // 32 bits count to a chunk past the last column
// Logits of a row that a warp holds; at 1000 f32 logits the kernel for wide rows takes 10.2 us instead of 8.0 for 16 x 4 rows,
// 16.9 instead of 13.8 for 128 x 8.
constexpr int kBeamNarrow = 1024;
// Small CTAs, since a part's end is a chain of waits (its sums, bar, candidates, their ranks, the arrival: about 7 us) that
// only the others of its SM can cover: 1024 x 50001 bf16 43.0 us with eight CTAs of 128 threads an SM, 43.5 with ten (fewer
// registers), 44.6 with four of 256; rows cut in two 50.  As one wave its rows still end together, which is 16 of the 43.
constexpr int kBeamThreads = 128, kBeamWarps = kBeamThreads / 32, kBeamCtas = 8;
constexpr int kBeamPieces = 3;                          // 16-byte pieces of a thread at a time (four: as fast to 2%)
constexpr int kBeamLook = 4;                            // threads whose logits a warp looks at again at a time
constexpr int kBeamMaxSplits = 32;
constexpr int kBeamHeld = 512;                          // candidates of a part, or of a request
constexpr size_t kBeamCounterBytes = kBeamMaxRequests * sizeof(int);  // of any call, so that calls of all sizes share a workspace
constexpr float kLog2e = 1.4426950408889634f;
}  // namespace

SJ_DEVICE float beam_load(const float* x) { return *x; }
SJ_DEVICE float beam_load(const __nv_bfloat16* x) { return bf2f(*x); }

// 2^x to 2 ulp, results below 2^-126 flushed to 0.
SJ_DEVICE float beam_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SJ_DEVICE float beam_warp_largest(float x) {  // NaN left out
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// The n-th largest (n <= 8: one by one; else by a bitonic sort) of a warp's lanes.
SJ_DEVICE float beam_warp_nth(float x, int n) {
  if (n <= 8) {
    float left = x, bar = beam_warp_largest(x);
    for (int above = 0; bar > -INFINITY;) {
      const bool is = left == bar;
      above += __popc(__ballot_sync(0xffffffffu, is));
      if (above >= n) break;
      if (is) left = -INFINITY;
      bar = beam_warp_largest(left);
    }
    return bar;
  }
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2) {
      const float o = __shfl_xor_sync(0xffffffffu, x, step);
      x = ((lane & step) == 0) == ((lane & size) == 0) ? fmaxf(x, o) : fminf(x, o);
    }
  return __shfl_sync(0xffffffffu, x, n - 1);
}

// A key that orders logits and their columns without ties: the larger value first (-0 and 0 are equal), then the lower
// column.  0 stands for none: a forbidden token (-inf) or a NaN.
SJ_DEVICE uint64_t beam_key(float v, int column) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t bits = __float_as_uint(v + 0.f);
  const uint32_t up = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
  return static_cast<uint64_t>(up) << 32 | static_cast<uint32_t>(~column);
}
SJ_DEVICE float beam_value(uint64_t key) {
  const uint32_t up = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
SJ_DEVICE int beam_column(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

// A part of a row: its maximum m and s = sum e^(x - m); m = -inf: nothing yet.
struct BeamSum {
  float m, s;
};
SJ_DEVICE BeamSum beam_join(BeamSum a, BeamSum b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return BeamSum{m, a.s + b.s};  // 0, or the NaN of a part that is all NaN
  return BeamSum{m, a.s * beam_exp2((a.m - m) * kLog2e) + b.s * beam_exp2((b.m - m) * kLog2e)};
}

// Two f32 at a time: sm_100 adds and multiplies a register pair in one instruction.
SJ_DEVICE uint64_t beam_pair(float a, float b) {
  return static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a);
}
SJ_DEVICE float beam_low(uint64_t p) { return __uint_as_float(static_cast<uint32_t>(p)); }
SJ_DEVICE float beam_high(uint64_t p) { return __uint_as_float(static_cast<uint32_t>(p >> 32)); }
SJ_DEVICE uint64_t beam_add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
SJ_DEVICE uint64_t beam_mul2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
// s += 2^((x - base) log2(e)), of two logits.  The difference comes first: a product of the lowest f32 would overflow,
// and a rounded log2(e) base would move all of a row's terms the same way.
SJ_DEVICE uint64_t beam_sum2(uint64_t s, float a, float b, float base) {
  const uint64_t d = beam_mul2(beam_add2(beam_pair(a, b), beam_pair(-base, -base)), beam_pair(kLog2e, kLog2e));
  return beam_add2(s, beam_pair(beam_exp2(beam_low(d)), beam_exp2(beam_high(d))));
}

struct BeamOut {
  const float* score;
  int32_t *parent, *token;
  float* best;
  int beams, vocab, keep;
};
// A beam's totals: score - log s + (x - m), the difference first, since m + log s would lose log s where a mask has left
// nothing but the lowest f32.  NaN where it has no candidates.
struct BeamOffset {
  double add, m;
  SJ_DEVICE double total(float x) const { return add + (static_cast<double>(x) - m); }
};
SJ_DEVICE BeamOffset beam_offset(float score, float m, double s) {
  const bool is = score > -INFINITY && score < INFINITY && m > -INFINITY;
  return BeamOffset{is ? static_cast<double>(score) - log(s) : __longlong_as_double(0x7ff8000000000000ll), m};
}

// An order-preserving integer of a total; 0 where it is none.
SJ_DEVICE unsigned long long beam_up(double total) {
  if (!(total > -INFINITY)) return 0;
  const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(total + 0.0));
  return bits ^ (static_cast<unsigned long long>(static_cast<long long>(bits) >> 63) | 0x8000000000000000ull);
}
// The highest 32 bits that at least `keep` of the values reach of which each thread of the CTA counts its own, bit by
// bit (0 where there are fewer); it stops where exactly `keep` reach them.  counts: 32 in shared memory.
template <typename F>
SJ_DEVICE uint32_t beam_reach(int keep, int* counts, F count) {
  __syncthreads();
  if (threadIdx.x < 32) counts[threadIdx.x] = 0;
  __syncthreads();
  uint32_t reach = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t want = reach | 1u << bit;
    const int have = __reduce_add_sync(0xffffffffu, count(want));
    if ((threadIdx.x & 31) == 0 && have) atomicAdd(&counts[bit], have);
    __syncthreads();
    const int all = counts[bit];
    if (all >= keep) reach = want;
    if (all == keep) break;
  }
  return reach;
}

// A request's candidates: totals, and beams and columns as one order.
struct BeamList {
  double total[kBeamHeld];
  int beam[kBeamHeld], column[kBeamHeld];
  int count;
};
SJ_DEVICE void beam_write(const BeamOut& out, size_t at, int beam, int column, double total) {
  out.parent[at] = beam;
  out.token[at] = column;
  out.best[at] = static_cast<float>(total);
}
// The best of n <= kBeamHeld candidates, each ranked against all others, by the threads of a CTA.
SJ_DEVICE void beam_rank(const BeamOut& out, int request, const BeamList& c, int n, int threads) {
  const size_t row = static_cast<size_t>(request) * out.keep;
  for (int i = threadIdx.x; i < n; i += threads) {
    const double total = c.total[i];
    const int beam = c.beam[i], column = c.column[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) {
      const double other = c.total[k];
      rank += other > total || (other == total && (c.beam[k] < beam || (c.beam[k] == beam && c.column[k] < column)));
    }
    if (rank < out.keep) beam_write(out, row + rank, beam, column, total);
  }
  for (int i = n + threadIdx.x; i < out.keep; i += threads) beam_write(out, row + i, -1, -1, -INFINITY);
}

// ---------------------------------------------------------------- narrow rows
// R: logits of a lane.  Warps take the request's beams in turn.  Up to 16 kept: of a beam, `keep` logits reach a bar that the
// lanes' maxima give; with the beam's offset it is one for the whole request, and the highest of the beams' counts.  More of
// them come near the number of lanes, whose lowest maximum keeps little out, and many beams leave more than the list
// holds: then the bar is sought bit by bit (both ways, 257 logits: 16 x 4 with 8 kept 6.5 and 8.0 us, 128 x 8 with 16 11.6
// and 10.4, with 24 17.4 and 11.2, with 32 63 and 12.5; 128 x 1 with 64 100 and 19; 256 x 16 with 32 42 and 17.6).
template <typename T, int R>
__global__ void __launch_bounds__(1024) beam_narrow_kernel(const T* logits, int ld, BeamOut out) {
  pdl_wait();
  __shared__ BeamList list;
  __shared__ BeamOffset offset[kBeamMaxBeams];
  __shared__ double bars[kBeamMaxBeams];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, request = blockIdx.x;
  if (threadIdx.x == 0) list.count = 0;
  const T* rows = logits + static_cast<size_t>(request) * out.beams * ld;
  float v[R + (R & 1)];
  const bool few = out.keep <= 16 && out.beams * out.keep <= kBeamHeld / 2;
  auto load = [&](int b) {
    const T* x = rows + static_cast<size_t>(b) * ld;
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = i * 32 + lane < out.vocab ? beam_load(x + i * 32 + lane) : -INFINITY;
    if (R & 1) v[R] = -INFINITY;
  };
  for (int b = warp; b < out.beams; b += warps) {
    const float score = out.score[static_cast<size_t>(request) * out.beams + b];
    BeamOffset off = beam_offset(-INFINITY, 0.f, 1.0);
    double bar = -INFINITY;
    if (score > -INFINITY) {
      load(b);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < R; ++i) top = fmaxf(top, v[i]);  // NaN left out
      const float m = beam_warp_largest(top), base = m == -INFINITY ? 0.f : m;
      uint64_t s = 0;
#pragma unroll
      for (int i = 0; i < R; i += 2) s = beam_sum2(s, v[i], v[i + 1], base);
      off = beam_offset(score, m, warp_sum(static_cast<double>(beam_low(s) + beam_high(s))));
      if (few) bar = off.total(beam_warp_nth(top, out.keep));  // NaN where the row has none
    }
    if (lane == 0) {
      offset[b] = off;
      bars[b] = bar;
    }
  }
  __syncthreads();
  double bar = -INFINITY;
  for (int b = 0; b < out.beams; ++b) bar = fmax(bar, bars[b]);
  auto each = [&](auto use) {  // the totals of this thread
    for (int b = warp; b < out.beams; b += warps) {
      const BeamOffset off = offset[b];
      if (!(off.add == off.add)) continue;
      if (out.beams > warps) load(b);
#pragma unroll
      for (int i = 0; i < R; ++i) use(off.total(v[i]), b, i * 32 + lane);
    }
  };
  auto collect = [&](auto reaches) {
    each([&](double total, int b, int column) {
      if (!reaches(total) || !(total > -INFINITY)) return;
      const int at = atomicAdd(&list.count, 1);
      if (at < kBeamHeld) {
        list.total[at] = total;
        list.beam[at] = b;
        list.column[at] = column;
      }
    });
    __syncthreads();
    return list.count;
  };
  int n = few ? collect([&](double total) { return total >= bar; }) : kBeamHeld + 1;
  if (n > kBeamHeld) {
    __shared__ int counts[32];
    uint32_t high[R], reach;
    if (out.beams <= warps) {
      const BeamOffset off = warp < out.beams ? offset[warp] : beam_offset(-INFINITY, 0.f, 1.0);
#pragma unroll
      for (int i = 0; i < R; ++i) high[i] = static_cast<uint32_t>(beam_up(off.total(v[i])) >> 32);
      reach = beam_reach(out.keep, counts, [&](uint32_t want) {
        int have = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) have += high[i] >= want;
        return have;
      });
    } else {
      reach = beam_reach(out.keep, counts, [&](uint32_t want) {
        int have = 0;
        each([&](double total, int, int) { have += beam_up(total) >> 32 >= want; });
        return have;
      });
    }
    if (threadIdx.x == 0) list.count = 0;
    __syncthreads();
    n = collect([&](double total) { return beam_up(total) >> 32 >= reach; });
  }
  if (n <= kBeamHeld) {
    beam_rank(out, request, list, n, blockDim.x);
    return;
  }
  // more ties than the list holds: one after the other, each the best one after the last
  __shared__ double s_total[32];
  __shared__ int s_beam[32], s_column[32];
  double last = INFINITY;
  int last_beam = -1, last_column = -1;
  for (int k = 0; k < out.keep; ++k) {
    double best = -INFINITY;
    int beam = -1, column = -1;
    for (int b = warp; b < out.beams; b += warps) {
      const BeamOffset off = offset[b];
      if (!(off.add == off.add)) continue;
      const T* x = rows + static_cast<size_t>(b) * ld;
      for (int j = lane; j < out.vocab; j += 32) {
        const double total = off.total(beam_load(x + j));
        if (!(total > -INFINITY)) continue;
        const bool left = total < last || (total == last && (b > last_beam || (b == last_beam && j > last_column)));
        if (left && total > best) {
          best = total;
          beam = b;
          column = j;
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double t2 = __shfl_xor_sync(0xffffffffu, best, o);
      const int b2 = __shfl_xor_sync(0xffffffffu, beam, o), c2 = __shfl_xor_sync(0xffffffffu, column, o);
      if (b2 >= 0 && (beam < 0 || t2 > best || (t2 == best && (b2 < beam || (b2 == beam && c2 < column))))) {
        best = t2;
        beam = b2;
        column = c2;
      }
    }
    if (lane == 0) {
      s_total[warp] = best;
      s_beam[warp] = beam;
      s_column[warp] = column;
    }
    __syncthreads();
    best = -INFINITY;
    beam = column = -1;
    for (int w = 0; w < warps; ++w) {
      const int b2 = s_beam[w], c2 = s_column[w];
      const double t2 = s_total[w];
      if (b2 >= 0 && (beam < 0 || t2 > best || (t2 == best && (b2 < beam || (b2 == beam && c2 < column))))) {
        best = t2;
        beam = b2;
        column = c2;
      }
    }
    last = best;
    last_beam = beam;
    last_column = column;
    if (threadIdx.x == 0) beam_write(out, static_cast<size_t>(request) * out.keep + k, beam, column, best);
    __syncthreads();
  }
}

// ---------------------------------------------------------------- wide rows
// A row in pieces of 16 bytes from its first column on, so that equal rows have equal sums wherever they lie: beams that
// are alike tie.  A row that does not begin at a multiple of 16 bytes takes a piece from two aligned ones.
template <typename T, bool ALIGNED>
struct BeamRow {
  static constexpr int PER = 16 / sizeof(T);
  static constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;  // -inf
  const T* x;
  int vocab, shift;  // bytes from the boundary before the row
  SJ_DEVICE BeamRow(const T* row, int vocab_)
      : x(row), vocab(vocab_), shift(ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16)) {}
  SJ_DEVICE int pieces() const { return (vocab + PER - 1) / PER; }
  SJ_DEVICE uint4 load(int piece, int end) const {  // -inf outside the row, or from piece `end` on
    const int j = piece * PER;
    if (piece >= end) return make_uint4(NONE, NONE, NONE, NONE);
    if (shift == 0 && j + PER <= vocab) return *reinterpret_cast<const uint4*>(x + j);
    if (!ALIGNED && shift != 0 && piece > 0 && j + 2 * PER - shift / static_cast<int>(sizeof(T)) <= vocab) {
      const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x + j) - shift);
      const uint4 lo = from[0], hi = from[1];
      uint32_t w[6] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y};
      if (shift & 8) {
        w[0] = lo.z;
        w[1] = lo.w;
        w[2] = hi.x;
        w[3] = hi.y;
        w[4] = hi.z;
        w[5] = hi.w;
      }
      if (shift & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
      }
      if (shift & 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
    uint32_t w[4] = {NONE, NONE, NONE, NONE};
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (j + e >= vocab) continue;
      const uint32_t bits = __float_as_uint(beam_load(x + j + e));
      if (sizeof(T) == 4)
        w[e % 4] = bits;
      else
        w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | (bits & 0xffff0000u) : (w[e / 2] & 0xffff0000u) | bits >> 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  SJ_DEVICE static float at(const uint4& q, int e) {
    const uint32_t w = sizeof(T) == 4 ? (e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w)
                                      : (e / 2 == 0 ? q.x : e / 2 == 1 ? q.y : e / 2 == 2 ? q.z : q.w);
    return __uint_as_float(sizeof(T) == 4 ? w : e % 2 ? w & 0xffff0000u : w << 16);
  }
  SJ_DEVICE static float largest(const uint4& q) {  // NaN left out
    if (sizeof(T) == 4) return fmaxf(fmaxf(at(q, 0), at(q, 1)), fmaxf(at(q, 2), at(q, 3)));
    uint32_t m = q.x;
    asm volatile("max.bf16x2 %0, %0, %1;\n\tmax.bf16x2 %0, %0, %2;\n\tmax.bf16x2 %0, %0, %3;"
                 : "+r"(m)
                 : "r"(q.y), "r"(q.z), "r"(q.w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
};

// What a part leaves in the workspace: its sums and its best keys in order, 0 past the last.
__host__ __device__ constexpr size_t beam_part_bytes(int keep) { return 8 * (1 + static_cast<size_t>(keep)); }

// Keys of [first, last) pieces that the CTA's threads own: f(key).
template <typename Row, typename F>
SJ_DEVICE void beam_each_key(const Row& row, int first, int last, F f) {
  for (int p = first + static_cast<int>(threadIdx.x); p < last; p += kBeamThreads) {
    const uint4 q = row.load(p, last);
#pragma unroll
    for (int e = 0; e < Row::PER; ++e) f(beam_key(Row::at(q, e), p * Row::PER + e));
  }
}

// What the CTA that ends a request has in shared memory.
struct BeamJoin {
  BeamList list;
  BeamOffset offset[kBeamMaxBeams];
  int counts[32];
  unsigned long long bar, shares;
};
SJ_DEVICE unsigned long long beam_up(const BeamJoin& join, int splits, int list, uint64_t key) {
  return key == 0 ? 0ull : beam_up(join.offset[list / splits].total(beam_value(key)));
}
// What is rare in a join is not inlined: its registers and instructions would stand in the way of the rest.
//
// What `keep` of the lists' first totals reach, as many of each as the threads' registers hold.
__device__ __noinline__ unsigned long long beam_join_bar(BeamJoin& join, const uint64_t* all, size_t slot, int splits,
                                                         int members, int keep) {
  constexpr int MOST = (kBeamMaxBeams * kBeamMaxSplits + kBeamMaxKeep) / kBeamThreads + 1;  // of a thread
  const int firsts = min(keep, MOST * kBeamThreads / members);
  uint32_t high[MOST];
#pragma unroll
  for (int k = 0; k < MOST; ++k) {
    const int i = static_cast<int>(threadIdx.x) + k * kBeamThreads, list = i / firsts;
    high[k] = 0;
    if (list < members)
      high[k] = static_cast<uint32_t>(
          beam_up(join, splits, list, __ldcg(all + static_cast<size_t>(list) * slot + 1 + i % firsts)) >> 32);
  }
  const uint32_t reach = beam_reach(keep, join.counts, [&](uint32_t want) {
    int have = 0;
#pragma unroll
    for (int k = 0; k < MOST; ++k) have += high[k] >= want;
    return have;
  });
  return static_cast<unsigned long long>(reach) << 32;
}
// More ties than the list holds: one candidate after the other.
__device__ __noinline__ void beam_join_ties(const BeamOut& out, BeamJoin& join, const uint64_t* all, size_t slot,
                                            int splits, int request) {
  const int t = threadIdx.x, keep = out.keep, members = out.beams * splits;
  double done = INFINITY;
  int done_beam = -1, done_column = -1;
  double* s_total = join.list.total;
  for (int k = 0; k < keep; ++k) {
    double best = -INFINITY;
    int beam = -1, column = -1;
    for (int i = t; i < members * keep; i += kBeamThreads) {
      const int at = i / keep, b = at / splits;
      const uint64_t key = __ldcg(all + static_cast<size_t>(at) * slot + 1 + i % keep);
      if (key == 0) continue;
      const double total = join.offset[b].total(beam_value(key));
      const int c = beam_column(key);
      if (!(total > -INFINITY)) continue;
      const bool left = total < done || (total == done && (b > done_beam || (b == done_beam && c > done_column)));
      if (left && (beam < 0 || total > best || (total == best && (b < beam || (b == beam && c < column))))) {
        best = total;
        beam = b;
        column = c;
      }
    }
    __syncthreads();
    s_total[t] = best;
    join.list.beam[t] = beam;
    join.list.column[t] = column;
    __syncthreads();
    best = -INFINITY;
    beam = column = -1;
    for (int i = 0; i < kBeamThreads; ++i) {
      const int b2 = join.list.beam[i], c2 = join.list.column[i];
      const double t2 = s_total[i];
      if (b2 >= 0 && (beam < 0 || t2 > best || (t2 == best && (b2 < beam || (b2 == beam && c2 < column))))) {
        best = t2;
        beam = b2;
        column = c2;
      }
    }
    done = best;
    done_beam = beam;
    done_column = column;
    if (t == 0) beam_write(out, static_cast<size_t>(request) * keep + k, beam, column, best);
  }
}
// A request's parts joined by a CTA.
SJ_DEVICE void beam_join_parts(const BeamOut& out, const uint64_t* parts, int request, int splits,
                                             BeamJoin& join) {
  const int t = threadIdx.x, keep = out.keep, members = out.beams * splits;
  const size_t slot = beam_part_bytes(keep) / 8;
  if (t == 0) {
    join.list.count = 0;
    join.bar = 0;
    join.shares = ~0ull;
  }
  const uint64_t* all = parts + static_cast<size_t>(request) * members * slot;
  // where the list holds all candidates, they come over at once, next to the sums
  constexpr int HELD = kBeamHeld / kBeamThreads;
  const bool whole = members * keep <= kBeamHeld;
  uint64_t held[HELD];
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int i = t + k * kBeamThreads;
    held[k] = whole && i < members * keep ? __ldcg(all + static_cast<size_t>(i / keep) * slot + 1 + i % keep) : 0;
  }
  if (t < out.beams) {
    float top = -INFINITY;
    double sum = 0.0;
#pragma unroll 1
    for (int k = 0; k < splits; ++k) {
      const uint64_t word = __ldcg(all + static_cast<size_t>(t * splits + k) * slot);
      const float part_m = __uint_as_float(static_cast<uint32_t>(word >> 32));
      const float part_s = __uint_as_float(static_cast<uint32_t>(word));
      const float raised = fmaxf(top, part_m), base = raised == -INFINITY ? 0.f : raised;
      // (a part without a maximum has the sum 0, or the NaN of a row that has one, which stays)
      sum = sum * beam_exp2((top - base) * kLog2e) + static_cast<double>(part_s) * beam_exp2((part_m - base) * kLog2e);
      top = raised;
    }
    join.offset[t] = beam_offset(out.score[static_cast<size_t>(request) * out.beams + t], top, sum);
  }
  __syncthreads();
  // A bar again: what `keep` of the lists' first totals reach, as many of each as it takes; where the list holds all
  // candidates, the lowest of them or the last total of a list will do.
  auto up = [&](int list, uint64_t key) { return beam_up(join, splits, list, key); };
  auto file = [&](int list, uint64_t key) {
    const int at = atomicAdd(&join.list.count, 1);
    if (at < kBeamHeld) {
      join.list.total[at] = join.offset[list / splits].total(beam_value(key));
      join.list.beam[at] = list / splits;
      join.list.column[at] = beam_column(key);
    }
  };
  if (whole) {
    const int firsts = (keep + members - 1) / members;
    unsigned long long total[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int i = t + k * kBeamThreads, at = i % keep + 1;
      total[k] = i < members * keep ? up(i / keep, held[k]) : 0ull;
      if (i < members * keep && at == keep) atomicMax(&join.bar, total[k]);
      if (i < members * keep && at == firsts) atomicMin(&join.shares, total[k]);
    }
    __syncthreads();
    const unsigned long long bar = max(join.bar, join.shares);
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (total[k] != 0 && total[k] >= bar) file((t + k * kBeamThreads) / keep, held[k]);
  } else {
    const unsigned long long bar = beam_join_bar(join, all, slot, splits, members, keep);
    // a thread for a list, until one of its totals does not reach the bar (a thread for an entry reads them all: 10 x 20 x 5000
    // with 40 kept 38.5 us instead of 36.1, 1 x 32 x 131072 with 64 kept 229 instead of 62)
    for (int list = t; list < members; list += kBeamThreads)
      for (int k = 0; k < keep; ++k) {
        const uint64_t key = __ldcg(all + static_cast<size_t>(list) * slot + 1 + k);
        const unsigned long long total = up(list, key);
        if (total == 0 || total < bar) break;
        file(list, key);
      }
  }
  __syncthreads();
  const int n = join.list.count;
  if (n <= kBeamHeld) {
    beam_rank(out, request, join.list, n, kBeamThreads);
    return;
  }
  beam_join_ties(out, join, all, slot, splits, request);
}

// ALIGNED: every row begins at a multiple of 16 bytes (128 x 8 x 50001 bf16 43 us, otherwise 64).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kBeamThreads, kBeamCtas)
    beam_wide_kernel(const T* logits, int ld, int splits, int* counters, uint64_t* parts, BeamOut out) {
  pdl_wait();
  using Row = BeamRow<T, ALIGNED>;
  constexpr int PER = Row::PER, STEP = kBeamThreads * kBeamPieces;
  __shared__ union Shared {
    uint64_t held[kBeamHeld];
    BeamJoin join;
    __device__ Shared() {}
  } u;
  __shared__ float s_bar[32];
  __shared__ BeamSum s_sum[kBeamWarps];
  __shared__ int s_count, s_last;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, keep = out.keep;
  const int row_at = blockIdx.x / splits, split = blockIdx.x % splits;
  const int request = row_at / out.beams;
  const size_t slot = beam_part_bytes(keep) / 8;
  uint64_t* mine = parts + static_cast<size_t>(blockIdx.x) * slot;
  const float score = out.score[row_at];
  const Row row(logits + static_cast<size_t>(row_at) * ld, out.vocab);
  const int pieces = row.pieces();
  const int first = static_cast<int>(static_cast<int64_t>(pieces) * split / splits);
  const int last = static_cast<int>(static_cast<int64_t>(pieces) * (split + 1) / splits);
  float m = -INFINITY;
  uint64_t s = 0;
  if (t == 0) s_count = 0;
  uint4 ahead[kBeamPieces];  // on their way while the last ones are added up, the first ones while the score is
#pragma unroll
  for (int i = 0; i < kBeamPieces; ++i) ahead[i] = row.load(first + t + i * kBeamThreads, last);
  if (score > -INFINITY) {
    for (int p = first + t; p - t < last; p += STEP) {
      uint4 q[kBeamPieces];
#pragma unroll
      for (int i = 0; i < kBeamPieces; ++i) {
        q[i] = ahead[i];
        ahead[i] = row.load(p + STEP + i * kBeamThreads, last);
      }
      float here = -INFINITY;
#pragma unroll
      for (int i = 0; i < kBeamPieces; ++i) here = fmaxf(here, Row::largest(q[i]));
      if (here > m) {
        const float f = beam_exp2((m - here) * kLog2e);
        s = beam_mul2(s, beam_pair(f, f));
        m = here;
      }
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < kBeamPieces; ++i)
#pragma unroll
        for (int e = 0; e < PER; e += 2) s = beam_sum2(s, Row::at(q[i], e), Row::at(q[i], e + 1), base);
    }
  }
  // ---- the part's sums, and a bar that at least `keep` of its logits reach: each warp brings its share of them
  BeamSum w{m, beam_low(s) + beam_high(s)};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    w = beam_join(w, BeamSum{__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.s, o)});
  // `keep` <= 32: the keep-th largest of the four best maxima of each warp; more: the lowest of the warps' shares of them
  constexpr int BEST = 32 / kBeamWarps;
  const bool few = keep <= 32;
  if (few) {
    float left = m;
#pragma unroll
    for (int k = 0; k < BEST; ++k) {
      const float best = beam_warp_largest(left);
      const uint32_t is = __ballot_sync(0xffffffffu, left == best);
      if (lane == 0) s_bar[warp * BEST + k] = best;
      if (lane == __ffs(is) - 1) left = -INFINITY;
    }
  } else {
    const float nth = beam_warp_nth(m, (keep + kBeamWarps - 1) / kBeamWarps);
    if (lane < BEST) s_bar[warp * BEST + lane] = nth;
  }
  if (lane == 0) s_sum[warp] = w;
  __syncthreads();
  float bar = s_bar[lane];
  if (few) {
    int above = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) above += s_bar[k] > bar ? 1 : 0;
    if (above >= keep) bar = INFINITY;
  }
  bar = -beam_warp_largest(-bar);
  // the logits of the threads that hold candidates once more, a thread's by its whole warp, several threads' at a time
  for (uint32_t who = __ballot_sync(0xffffffffu, m >= bar && m > -INFINITY); who;) {
    int of[kBeamLook];
#pragma unroll
    for (int k = 0; k < kBeamLook; ++k) {
      of[k] = who ? first + warp * 32 + __ffs(who) - 1 : last;
      who &= who - 1;
    }
    for (int p = lane * kBeamThreads; first + p < last; p += 32 * kBeamThreads) {
      uint4 q[kBeamLook];
#pragma unroll
      for (int k = 0; k < kBeamLook; ++k) q[k] = row.load(of[k] + p, last);
#pragma unroll
      for (int k = 0; k < kBeamLook; ++k) {
        if (!(Row::largest(q[k]) >= bar)) continue;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const float v = Row::at(q[k], e);
          if (!(v >= bar) || v == -INFINITY) continue;
          const int at = atomicAdd(&s_count, 1);
          if (at < kBeamHeld) u.held[at] = beam_key(v, (of[k] + p) * PER + e);
        }
      }
    }
  }
  __syncthreads();
  int n = s_count;
  if (n > kBeamHeld) {
    // Ties, or too few threads with candidates: the keep-th largest key, bit by bit; then those that reach it.
    uint64_t reach = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t want = reach | 1ull << bit;
      int have = 0;
      beam_each_key(row, first, last, [&](uint64_t key) { have += key >= want; });
      have = __reduce_add_sync(0xffffffffu, have);
      __syncthreads();
      if (t == 0) s_count = 0;
      __syncthreads();
      if (lane == 0) atomicAdd(&s_count, have);
      __syncthreads();
      if (s_count >= keep) reach = want;
    }
    __syncthreads();
    if (t == 0) s_count = 0;
    __syncthreads();
    beam_each_key(row, first, last, [&](uint64_t key) {
      if (key != 0 && key >= reach) u.held[atomicAdd(&s_count, 1)] = key;
    });
    __syncthreads();
    n = s_count;
  }
  if (t >= n && t < keep) mine[1 + t] = 0;
  for (int i = t; i < n; i += kBeamThreads) {
    const uint64_t key = u.held[i];
    int rank = 0;
#pragma unroll 8
    for (int k = 0; k < n; ++k) rank += u.held[k] > key ? 1 : 0;
    if (rank < keep) mine[1 + rank] = key;
  }
  if (t == 0) {
    BeamSum sum = s_sum[0];
    for (int k = 1; k < kBeamWarps; ++k) sum = beam_join(sum, s_sum[k]);
    mine[0] = static_cast<uint64_t>(__float_as_uint(sum.m)) << 32 | __float_as_uint(sum.s);
  }
  // ---- the request's parts, by the CTA that ends the last of them
  __syncthreads();
  const int members = out.beams * splits;
  if (t == 0) {
    int before;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counters + request) : "memory");
    s_last = before == members - 1;
    if (s_last) counters[request] = 0;
  }
  __syncthreads();
  if (!s_last) return;
  beam_join_parts(out, parts, request, splits, u.join);
}

}  // namespace sj

using namespace sj;

namespace {
// Parts of a row: as many as fill the GPU, of at least a thread's pieces each.
int beam_splits(int64_t rows, int vocab) {
  const int64_t want = 8 * static_cast<int64_t>(sm_count()) / std::max<int64_t>(rows, 1);
  const int64_t most = vocab / (kBeamThreads * 16) + 1;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kBeamMaxSplits})));
}

template <typename T, int R>
int beam_narrow(const T* x, int ld, int requests, const BeamOut& out, cudaStream_t s) {
  launch(beam_narrow_kernel<T, R>, requests, 32 * std::min(out.beams, 32), 0, s, x, ld, out);
  SJ_LAUNCH_CHECK("beam_narrow");
  return SJ_OK;
}
template <typename T>
int beam_select(const T* x, int ld, int requests, const BeamOut& out, void* workspace, cudaStream_t s) {
  if (out.vocab <= kBeamNarrow) {
    // fewer registers for the vocabulary of bytes: 16 x 4 x 257 6.5 us instead of 7.8, 1000 x 4 x 257 8.6 instead of 11.8
    if (out.vocab <= 9 * 32) return beam_narrow<T, 9>(x, ld, requests, out, s);
    return beam_narrow<T, 32>(x, ld, requests, out, s);
  }
  const int64_t rows = static_cast<int64_t>(requests) * out.beams;
  const int splits = beam_splits(rows, out.vocab);
  const bool aligned = aligned16(x) && ld * sizeof(T) % 16 == 0;
  launch(aligned ? beam_wide_kernel<T, true> : beam_wide_kernel<T, false>, static_cast<unsigned>(rows * splits), kBeamThreads, 0, s, x, ld, splits,
         static_cast<int*>(workspace),
         reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + kBeamCounterBytes), out);
  SJ_LAUNCH_CHECK("beam_wide");
  return SJ_OK;
}
}  // namespace

extern "C" size_t sj_beam_select_workspace(int requests, int beams, int vocab, int keep) {
  if (requests <= 0 || requests > kBeamMaxRequests || beams <= 0 || beams > kBeamMaxBeams || vocab <= kBeamNarrow ||
      keep <= 0 || keep > kBeamMaxKeep)
    return 0;
  const int64_t rows = static_cast<int64_t>(requests) * beams;
  return kBeamCounterBytes + static_cast<size_t>(rows) * beam_splits(rows, vocab) * beam_part_bytes(keep);
}

extern "C" int sj_beam_select(const void* logits, int dtype, int ld, const float* score, int requests, int beams,
                              int vocab, int keep, int32_t* parent, int32_t* token, float* new_score, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (requests < 0 || requests > kBeamMaxRequests || beams <= 0 || beams > kBeamMaxBeams || vocab <= 0 ||
      vocab > kBeamMaxColumns || ld < vocab || keep <= 0 || keep > kBeamMaxKeep ||
      keep > static_cast<int64_t>(beams) * vocab)
    return fail(SJ_ERR_SHAPE, "sj_beam_select: requests=%d (up to %d) beams=%d (up to %d) vocab=%d ld=%d keep=%d (up to %d)",
                requests, kBeamMaxRequests, beams, kBeamMaxBeams, vocab, ld, keep, kBeamMaxKeep);
  if (dtype != SJ_F32 && dtype != SJ_BF16)
    return fail(SJ_ERR_ARGUMENT, "sj_beam_select: dtype %d (f32 or bf16)", dtype);
  if (requests == 0) return SJ_OK;
  if (!logits || !score || !parent || !token || !new_score ||
      reinterpret_cast<uintptr_t>(logits) % (dtype == SJ_F32 ? 4 : 2))
    return fail(SJ_ERR_ARGUMENT, "sj_beam_select: null or unaligned operand");
  const size_t need = sj_beam_select_workspace(requests, beams, vocab, keep);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(SJ_ERR_CAPACITY, "sj_beam_select: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const BeamOut out{score, parent, token, new_score, beams, vocab, keep};
  cudaStream_t s = as_stream(stream);
  return dtype == SJ_F32 ? beam_select(static_cast<const float*>(logits), ld, requests, out, workspace, s)
                         : beam_select(static_cast<const __nv_bfloat16*>(logits), ld, requests, out, workspace, s);
}
