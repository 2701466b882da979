// Attention of single rows over a paged key-value cache (sj_attn_paged).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = log2(e) / sqrt(dim)
//
// over the keys a row sees, with the running maximum m and f32 sums.  Each K and V element is used for the
// few query heads that share it (2 * hq / hk multiply-adds an element), far below the tensor cores'
// rate, so the kernel is bound by the cache bytes it reads and its design is about keeping enough
// of them in flight:
//   * a warp copies 4096 bytes of K and as many of V at a time (32 keys of 64 dims, 16 of 128) into a ring of two
//     stages of its own (cp.async, 16 bytes a lane, four whole 128-byte rows an instruction; keys out of sight
//     are zero-filled and never read), so no barrier joins the warps of a CTA while they read.  12 warps
//     an SM keep 96 to 192 KB in flight.  The page of each key is looked up one step ahead.
//   * K is the A operand of S^T = K Q^T (m16n8k16: 16 keys, 8 queries).  The order of the contracted dims is
//     free, so a lane's 16-byte pieces of a key row are its fragments as they are, and the same pieces of the query
//     rows its B fragments.  V^T is the A operand of O^T = V^T P^T: a lane reads 16 bytes of four keys and
//     interleaves pairs of keys by byte permutes; P^T comes from S^T by movmatrix.  8 query heads
//     fill the mma's 8 columns; with K as the B operand they would leave half of its 16 rows empty.
//   * the (row, KV head) units are cut into tiles of 128 keys, and the tiles of all units, one after the
//     other, are dealt to the CTAs in equal contiguous ranges: a step of ragged lengths, or one long
//     row, keeps every SM busy to the end.  A unit that spans CTAs is joined from the workspace by the CTA
//     that finishes it last; the parts are added in their order, so results do not depend on which.
//
// Measured on B200 (graph replays; the caches are larger than L2): 256 rows of 512 to 16384 keys, 12 / 4 heads of 64:
// 189 us, 6.35 TB/s of 1.2 GB (97% of the measured copy rate); two rows of 150 and 200 thousand keys, 16 / 4 heads:
// 64 us, 5.6 TB/s; 64 rows of 4 to 9 thousand keys, 16 / 2 heads of 128: 72 us, 5.6 TB/s.  The first simple kernel
// (a CTA for each row and query head) took 4730 us and 49200 us on the first two; K and V loaded straight into
// registers, 203 and 71 us (no copies in flight while a warp computes); 16- and 24-warp CTAs, one an SM, 10 to
// 20% more (all wait for the slowest warp at a unit's end); a last fifth of the tiles dealt to whoever is
// done first: the same.
#include <algorithm>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace sj {

namespace {
constexpr int kTile = 128;                   // keys of a tile
// Units of at most kWhole tiles are not split: a join through memory costs about 2.5 us, a second tile 0.5 (three
// short rows: 8.0 against 5.2 us).
constexpr int kWhole = 2;
// More parts than kGroup are joined in groups of about their square root: 444 parts of one unit by one CTA took 80 us,
// in two levels 9; 14 parts of 32 units took 2 us more in two levels than in one.  A group has at most kGroupMost
// parts: 1024 CTAs would be 32 groups of 32.
constexpr int kGroup = 20, kGroupMost = 32;
constexpr int kWarps = 4, kCtas = 3, kStages = 2;  // of a CTA, of an SM, of a warp's ring
constexpr int kLastPosition = INT_MAX - 4096;  // key indices step past the end by less than this
constexpr uint32_t kNoKey = 0xffffffffu;     // past any offset: buffers hold at most 2^32 16-byte chunks
}  // namespace

struct PagedAttention {
  const __nv_bfloat16 *q, *k, *v;
  const int32_t *table, *request, *position;
  __nv_bfloat16* o;
  float* lse;
  int* counters;   // parts written of each first group of a unit, of other groups, groups of a unit: a CTA one of each
  float* partial;  // two slots per CTA
  int64_t page_stride, head_stride, token_stride;
  int ldq, ldo, pages, page, ld_table, requests, rows, hq, hk, window;
};

// 16 bytes from global to shared memory without passing through registers; zeros when !seen.
SJ_DEVICE void copy16(uint32_t dst, const __nv_bfloat16* src, bool seen) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(seen ? 16 : 0) : "memory");
}
SJ_DEVICE void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
SJ_DEVICE void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
SJ_DEVICE uint4 read16(uint32_t src) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(src)
               : "memory");
  return r;
}
SJ_DEVICE void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
SJ_DEVICE uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// 2^x to 2 ulp, results below 2^-126 flushed to 0 (a weight that small adds nothing to an f32 sum that
// holds a weight of 1).
SJ_DEVICE float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SJ_DEVICE uint32_t swizzle(int row) { return ((row >> 1 & 3) << 1) ^ ((row & 1) << 2); }
SJ_DEVICE uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// Keys [lo, n) that a row sees.
SJ_DEVICE void row_span(const PagedAttention& a, int r, int& lo, int& n) {
  const int b = a.request ? a.request[r] : r, pos = a.position[r];
  n = b == -1 || pos > kLastPosition ? 0 : pos + 1;
  if (b < -1 || b >= a.requests || pos < -1 || pos > kLastPosition ||
      static_cast<int64_t>(n) > static_cast<int64_t>(a.ld_table) * a.page) {
    record_error(SJ_DEV_BAD_INDEX);
    n = 0;
  }
  lo = a.window > 0 ? max(0, n - a.window) : 0;
}
// The tiles of all units cut into consecutive ranges, one for a CTA.
struct Cut {
  unsigned long long total;
  int count;
  SJ_DEVICE Cut(unsigned long long tiles, int ctas)
      : total(tiles), count(static_cast<int>(min(static_cast<unsigned long long>(ctas), tiles))) {}
  SJ_DEVICE unsigned long long begin(int id) const { return total * id / count; }
  // the last range that begins at or before tile x, which holds it
  SJ_DEVICE int of(unsigned long long x) const {
    return static_cast<int>(((x + 1) * count + total - 1) / total) - 1;
  }
};
SJ_DEVICE int span_tiles(int lo, int n) { return max(1, (n - lo + kTile - 1) / kTile); }

// Parts first, first + stride, ... (count <= kGroupMost of them) of a unit added in that order by the whole CTA, left
// unnormalised in shared memory: sm[q] the maxima, sl[q] the sums, and the outputs as float4 [heads * DIM / 4] in
// `sums`.  Eight threads take a query's maxima and sums; a thread adds four dims of one query over every
// `shares`-th part, eight parts' loads in flight, the first ones before the weights are known.  Not inlined: its
// registers would push the main loop's into memory (193 instead of 187 us at 256 ragged rows, 135 instead of 81 at
// 16 heads of 128).
template <int DIM, int Q, int WARPS>
__device__ __noinline__ void join_parts(const float* partial, int from, int first, int count, int stride, int heads,
                                        float* sm, float* sl, float (*weight)[Q], float4* sums) {
  constexpr int SLOT = Q * (DIM + 2), THREADS = WARPS * 32;
  const int t = threadIdx.x;
  const int items = heads * (DIM / 4), shares = max(1, min(count, THREADS / items));
  auto slot_of = [&](int k) {
    const int at = first + k * stride;
    return partial + (at * 2 + (at == from ? 1 : 0)) * static_cast<size_t>(SLOT);
  };
  float4 x[8];
  auto fetch = [&](int i, int w) {
    const int item = i % items, at = 2 * Q + item / (DIM / 4) * DIM + item % (DIM / 4) * 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = min(w + e * shares, count - 1);
      x[e] = __ldcg(reinterpret_cast<const float4*>(slot_of(k) + at));
    }
  };
  int i = t;
  if (i < items * shares) fetch(i, i / items);
  static_assert(THREADS >= Q * 8 && kGroupMost == 32, "eight threads a query, four parts a thread");
  {
    const int qi = t >> 3;
    float m[4], l[4], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = (t & 7) + 8 * e;
      const bool is = qi < heads && k < count;
      m[e] = is ? __ldcg(slot_of(k) + qi) : -INFINITY;
      l[e] = is ? __ldcg(slot_of(k) + Q + qi) : 0.f;
      top = fmaxf(top, m[e]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = exp2_fast(m[e] - ref);
      sum += f * l[e];
      if (qi < heads) weight[(t & 7) + 8 * e][qi] = f;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (qi < heads && (t & 7) == 0) {
      sm[qi] = top;
      sl[qi] = sum;
    }
  }
  __syncthreads();
#pragma unroll 1
  while (i < items * shares) {
    const int qi = i % items / (DIM / 4);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int w = i / items; w < count; w += 8 * shares) {
      if (w >= shares) fetch(i, w);  // the first eight are here
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = w + e * shares < count ? weight[w + e * shares][qi] : 0.f;
        if (f != 0.f) {
          acc.x += f * x[e].x;
          acc.y += f * x[e].y;
          acc.z += f * x[e].z;
          acc.w += f * x[e].w;
        }
      }
    }
    sums[i] = acc;
    i += THREADS;
    if (i < items * shares) fetch(i, i / items);
  }
  __syncthreads();
  if (shares > 1) {
#pragma unroll 1
    for (int k = t; k < items; k += THREADS) {
      float4 out = sums[k];
#pragma unroll 1
      for (int w = 1; w < shares; ++w) {
        const float4 y = sums[w * items + k];
        out.x += y.x;
        out.y += y.y;
        out.z += y.z;
        out.w += y.w;
      }
      sums[k] = out;
    }
    __syncthreads();
  }
}

// One more on a counter, after what the CTA's threads have written (a barrier has passed it on to this one) and before
// what they read from others.
SJ_DEVICE int arrive(int* counter) {
  int before;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

// DIM: head_dim; NQ: query tiles of 8 that a unit holds (a query's columns of S^T; 2 above 8 heads a KV head).
template <int DIM, int NQ>
__global__ void __launch_bounds__(kWarps * 32, kCtas) attn_paged_kernel(const PagedAttention a) {
  pdl_wait();
  constexpr int WARPS = kWarps, STAGES = kStages, KT = 128 / DIM;  // KT: 16-key tiles of a warp's step
  constexpr int CC = DIM / 32, CH = DIM / 64, MT = DIM / 16, Q = NQ * 8, KEYS = KT * 16, STEP = WARPS * KEYS;
  constexpr int STAGE = KEYS * DIM * 4;    // bytes of K and V of a step
  constexpr int LD = DIM + 8;               // row of an output in shared memory
  constexpr int SLOT = Q * (DIM + 2);       // floats of a partial slot: m [Q], l [Q], o [Q][DIM]
  // 128-byte aligned: where a row of a stage straddles two lines of banks, its copy reads every sector twice
  // (231 instead of 190 us at 256 ragged rows)
  extern __shared__ uint8_t unaligned[];
  uint8_t* smem = unaligned + (-smem_u32(unaligned) & 127);
  float* so = reinterpret_cast<float*>(smem);  // [WARPS][Q][LD], once a unit's stages are read
  __shared__ float sm[WARPS][Q], sl[WARPS][Q], weight[kGroupMost][Q];
  __shared__ unsigned long long scan[WARPS], s_base;
  __shared__ int s_row, s_last;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
  const int group = a.hq / a.hk, sets = (group + Q - 1) / Q, units = a.hk * sets;
  const float scale = 1.4426950408889634f * rsqrtf(static_cast<float>(DIM));
  const uint32_t ring = smem_u32(smem) + warp * STAGES * STAGE;
  // shared-memory addresses inside a stage: 128-byte rows (of a half of DIM) whose 16-byte chunks are permuted
  // by swizzle(row), so that copies, K reads (rows 2 p and 2 p + 1) and V reads (rows 2 c) are free of conflicts
  const uint32_t put = (lane >> 3) * 128 + (((lane & 7) ^ swizzle(lane >> 3)) << 4);
  const uint32_t k_at = g * 128 + ((c ^ swizzle(g)) << 4);
  const uint32_t v_at = 2 * c * 128 + ((g ^ swizzle(2 * c)) << 4);

  // ---- this CTA's range of the tiles of all units
  const int per = (a.rows + WARPS * 32 - 1) / (WARPS * 32), r0 = min(t * per, a.rows), r1 = min(r0 + per, a.rows);
  unsigned long long mine = 0;
  for (int r = r0; r < r1; ++r) {
    int lo, n;
    row_span(a, r, lo, n);
    mine += static_cast<unsigned long long>(span_tiles(lo, n)) * units;
  }
  unsigned long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  unsigned long long total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w == warp) upto += total;
    total += scan[w];
  }
  const unsigned long long before = upto - mine;
  const Cut cut(total, gridDim.x);
  const int id = blockIdx.x;
  if (id >= cut.count) return;
  unsigned long long at = cut.begin(id);
  const unsigned long long end = cut.begin(id + 1);
  if (before <= at && at < before + mine) {
    unsigned long long base = before;
    for (int r = r0; r < r1; ++r) {
      int lo, n;
      row_span(a, r, lo, n);
      const unsigned long long next = base + static_cast<unsigned long long>(span_tiles(lo, n)) * units;
      if (at < next) {
        s_row = r;
        s_base = base;
        break;
      }
      base = next;
    }
  }
  __syncthreads();
  unsigned long long base = s_base;

  for (int r = s_row; at < end; ++r) {
    int lo, n;
    row_span(a, r, lo, n);
    const int tiles = span_tiles(lo, n);
    const int32_t* table = a.table + static_cast<size_t>(n > 0 ? (a.request ? a.request[r] : r) : 0) * a.ld_table;
    int unit = static_cast<int>((at - base) / tiles), first = static_cast<int>((at - base) % tiles);
    if (first > 0 && tiles <= kWhole) {  // a short unit stays with the CTA that its first tile falls to
      at += tiles - first;
      first = 0;
      ++unit;
    }
    for (; unit < units && at < end; ++unit, first = 0) {
      const int past = tiles <= kWhole
                           ? tiles
                           : static_cast<int>(min(static_cast<unsigned long long>(tiles), first + (end - at)));
      const int h = unit / sets, q0 = (unit % sets) * Q, heads = min(Q, group - q0);
      const int k0 = lo + first * kTile, k1 = min(n, lo + past * kTile);

      // ---- this warp's keys, KEYS at a time: lane i looks up the page of key i one step before it is needed, and
      // then resolves where the key lies (in 16-byte chunks)
      const int steps = k1 > k0 + warp * KEYS ? (k1 - k0 - warp * KEYS + STEP - 1) / STEP : 0;
      int key = k0 + warp * KEYS + lane, found = 0;
      int pg = key / a.page, off = key % a.page;
      const int step_page = STEP / a.page, step_off = STEP % a.page;
      auto look_up = [&]() {
        if (lane < KEYS && key < k1) found = table[pg];
      };
      auto resolve = [&]() {
        uint32_t where = kNoKey;
        if (lane < KEYS && key < k1) {
          if (found >= 0 && found < a.pages)
            where = static_cast<uint32_t>((found * a.page_stride + h * a.head_stride + off * a.token_stride) >> 3);
          else
            record_error(SJ_DEV_BAD_INDEX);
        }
        key += STEP;
        pg += step_page;
        off += step_off;
        if (off >= a.page) {
          off -= a.page;
          ++pg;
        }
        return where;
      };
      // four whole rows of 128 bytes an instruction
      auto fetch = [&](int stage, uint32_t where) {
#pragma unroll
        for (int i = 0; i < KEYS / 4; ++i) {
          const uint32_t w = __shfl_sync(0xffffffffu, where, i * 4 + (lane >> 3));
          const size_t at = w == kNoKey ? 0 : static_cast<size_t>(w) * 8 + (lane & 7) * 8;
          const uint32_t dst = ring + stage * STAGE + (i * 512 + put ^ (i & 1) * 64);  // rows 4 i + ..: swizzle(4) = 4
#pragma unroll
          for (int u = 0; u < CH; ++u) {
            const size_t part = w == kNoKey ? 0 : at + u * 64;
            copy16(dst + u * (KEYS * 128), a.k + part, w != kNoKey);
            copy16(dst + (CH + u) * (KEYS * 128), a.v + part, w != kNoKey);
          }
        }
      };
      uint32_t seen[STAGES - 1];  // keys of the stages in flight that are in sight
      look_up();

      // ---- queries: chunk c + 4 i of query row j * 8 + g, the B fragments of S^T
      uint4 qf[NQ][CC];
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int i = 0; i < CC; ++i) {
          qf[j][i] = make_uint4(0, 0, 0, 0);
          if (j * 8 + g < heads)
            qf[j][i] = *reinterpret_cast<const uint4*>(a.q + static_cast<size_t>(r) * a.ldq +
                                                       (h * group + q0 + j * 8 + g) * DIM + (c + 4 * i) * 8);
        }
      float o[NQ][MT][4], m[NQ][2], l[NQ][2];
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        m[j][0] = m[j][1] = -INFINITY;
        l[j][0] = l[j][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
      }

#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) {
        const uint32_t where = resolve();
        look_up();
        fetch(i, where);
        seen[i] = __ballot_sync(0xffffffffu, where != kNoKey);
        copy_commit();
      }
      for (int step = 0, stage = 0; step < steps; ++step) {
        copy_wait<STAGES - 2>();
        __syncwarp();  // the warp's copies are in, and its reads of the stage before are done
        const uint32_t where = resolve();
        look_up();
        fetch(stage == 0 ? STAGES - 1 : stage - 1, where);
        copy_commit();
        const uint32_t in_sight = seen[0];
#pragma unroll
        for (int i = 0; i < STAGES - 2; ++i) seen[i] = seen[i + 1];
        seen[STAGES - 2] = __ballot_sync(0xffffffffu, where != kNoKey);
        const uint32_t src = ring + stage * STAGE;
        float s[NQ][KT][4];
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          uint4 kf[2][CC];
#pragma unroll
          for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int u = 0; u < CC; ++u)
              kf[d][u] = read16(src + (u / 2) * (KEYS * 128) + (i * 16 + d * 8) * 128 + (k_at ^ (u & 1) * 64));
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            s[j][i][0] = s[j][i][1] = s[j][i][2] = s[j][i][3] = 0.f;
#pragma unroll
            for (int u = 0; u < CC; ++u) {
              mma_bf16(s[j][i], kf[0][u].x, kf[1][u].x, kf[0][u].y, kf[1][u].y, qf[j][u].x, qf[j][u].y);
              mma_bf16(s[j][i], kf[0][u].z, kf[1][u].z, kf[0][u].w, kf[1][u].w, qf[j][u].z, qf[j][u].w);
            }
          }
        }
        // s[j][i]: keys i * 16 + g (0, 1) and + 8 (2, 3) of queries 2 c and 2 c + 1
        uint32_t b[NQ][KT][2];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          if (in_sight != (KEYS == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(in_sight >> (i * 16 + g + (e >> 1) * 8) & 1)) s[j][i][e] = -INFINITY;
          }
          float top[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[e] = fmaxf(s[j][0][e], s[j][0][e + 2]);
            if (KT == 2) top[e] = fmaxf(top[e], fmaxf(s[j][KT - 1][e], s[j][KT - 1][e + 2]));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16)) * scale;
          }
          if (__any_sync(0xffffffffu, top[0] > m[j][0] || top[1] > m[j][1])) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              top[e] = fmaxf(top[e], m[j][e]);
              const float keep = exp2_fast(m[j][e] - (top[e] == -INFINITY ? 0.f : top[e]));
              m[j][e] = top[e];
              l[j][e] *= keep;
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                o[j][i][e] *= keep;
                o[j][i][e + 2] *= keep;
              }
            }
          }
          // P is rounded to bf16 (the mma's operand); the sums take it unrounded
          const float ref[2] = {m[j][0] == -INFINITY ? 0.f : m[j][0], m[j][1] == -INFINITY ? 0.f : m[j][1]};
#pragma unroll
          for (int i = 0; i < KT; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[j][i][e] = exp2_fast(fmaf(s[j][i][e], scale, -ref[e & 1]));
              l[j][e & 1] += s[j][i][e];
            }
            b[j][i][0] = transpose8x8(pack_bf16x2(s[j][i][0], s[j][i][1]));
            b[j][i][1] = transpose8x8(pack_bf16x2(s[j][i][2], s[j][i][3]));
          }
        }
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
          for (int u = 0; u < CH; ++u) {
            uint4 vf[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              vf[e] = read16(src + (CH + u) * (KEYS * 128) + (i * 16 + (e & 1) + (e >> 1) * 8) * 128 +
                             (v_at ^ (e & 1) * 64));
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t v0 = word(vf[0], x), v1 = word(vf[1], x), v2 = word(vf[2], x), v3 = word(vf[3], x);
              const uint32_t a0 = __byte_perm(v0, v1, 0x5410), a1 = __byte_perm(v0, v1, 0x7632);
              const uint32_t a2 = __byte_perm(v2, v3, 0x5410), a3 = __byte_perm(v2, v3, 0x7632);
#pragma unroll
              for (int j = 0; j < NQ; ++j) mma_bf16(o[j][u * 4 + x], a0, a1, a2, a3, b[j][i][0], b[j][i][1]);
            }
          }
        stage = stage == STAGES - 1 ? 0 : stage + 1;
      }
      copy_wait<0>();

      // ---- the warps' parts joined: o[j][x][e + 2 d] is dim (g + 8 (x / 4)) * 8 + 2 (x % 4) + d of query 2 c + e
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 4);
          l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 8);
          l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], 16);
          if (g == 0) {
            sm[warp][j * 8 + 2 * c + e] = m[j][e];
            sl[warp][j * 8 + 2 * c + e] = l[j][e];
          }
        }
      __syncthreads();  // and every warp is done with its ring, where the outputs go
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int qi = j * 8 + 2 * c + e;
          if (qi >= heads) continue;
          float top = sm[0][qi];
          for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm[w][qi]);
          const float f = exp2_fast(m[j][e] - (top == -INFINITY ? 0.f : top));
          float* dst = so + (warp * Q + qi) * LD;
#pragma unroll
          for (int u = 0; u < CH; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int x = u * 4 + 2 * i;
              *reinterpret_cast<float4*>(dst + (g + 8 * u) * 8 + 4 * i) =
                  make_float4(f * o[j][x][e], f * o[j][x][e + 2], f * o[j][x + 1][e], f * o[j][x + 1][e + 2]);
            }
        }
      __syncthreads();
      const bool whole = first == 0 && past == tiles;
      float* slot = a.partial + (static_cast<size_t>(id) * 2 + (first == 0 ? 1 : 0)) * SLOT;
      for (int i = t; i < heads * (DIM / 4); i += WARPS * 32) {
        const int qi = i / (DIM / 4), d = i % (DIM / 4) * 4;
        float top = sm[0][qi], sum = 0.f;
        for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm[w][qi]);
        const float ref = top == -INFINITY ? 0.f : top;
        float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < WARPS; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(so + (w * Q + qi) * LD + d);
          out.x += x.x;
          out.y += x.y;
          out.z += x.z;
          out.w += x.w;
          sum += exp2_fast(sm[w][qi] - ref) * sl[w][qi];
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          const int head = h * group + q0 + qi;
          *reinterpret_cast<uint2*>(a.o + static_cast<size_t>(r) * a.ldo + head * DIM + d) =
              make_uint2(pack_bf16x2(out.x * inv, out.y * inv), pack_bf16x2(out.z * inv, out.w * inv));
          if (d == 0 && a.lse)
            a.lse[static_cast<size_t>(r) * a.hq + head] =
                sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
        } else {
          *reinterpret_cast<float4*>(slot + 2 * Q + qi * DIM + d) = out;
          if (d == 0) {
            slot[qi] = top;
            slot[Q + qi] = sum;
          }
        }
      }
      if (!whole) {
        // ---- the unit's parts joined by the CTA that writes the last of them: tile x falls to the last chunk w
        // with w * total / count <= x.  Many parts are joined in groups, and the groups likewise.
        const unsigned long long begin = base + static_cast<unsigned long long>(unit) * tiles;
        const int from = cut.of(begin), to = cut.of(begin + tiles - 1);
        const int parts = to - from + 1;
        const int size = parts <= kGroup ? parts : static_cast<int>(ceilf(sqrtf(static_cast<float>(parts))));
        const int groups = (parts + size - 1) / size, mine_group = (static_cast<int>(id) - from) / size;
        const int lead = from + mine_group * size, members = min(size, parts - mine_group * size);
        auto last_of = [&](int* counter, int expected) {
          __syncthreads();
          if (t == 0) {
            s_last = arrive(counter) == expected - 1;
            if (s_last) *counter = 0;
          }
          __syncthreads();
          return s_last != 0;
        };
        float4* sums = reinterpret_cast<float4*>(so);
        bool joined = last_of(a.counters + (mine_group == 0 ? 0 : gridDim.x) + lead, members);
        if (joined) join_parts<DIM, Q, WARPS>(a.partial, from, lead, members, 1, heads, sm[0], sl[0], weight, sums);
        if (joined && groups > 1) {
          float* dst = a.partial + (static_cast<size_t>(lead) * 2 + (lead == from ? 1 : 0)) * SLOT;
          for (int i = t; i < heads * (DIM / 4); i += WARPS * 32) {
            const int qi = i / (DIM / 4), d = i % (DIM / 4) * 4;
            *reinterpret_cast<float4*>(dst + 2 * Q + qi * DIM + d) = sums[i];
            if (d == 0) {
              dst[qi] = sm[0][qi];
              dst[Q + qi] = sl[0][qi];
            }
          }
          joined = last_of(a.counters + 2 * gridDim.x + from, groups);
          if (joined) join_parts<DIM, Q, WARPS>(a.partial, from, from, groups, size, heads, sm[0], sl[0], weight, sums);
        }
        if (joined) {
          for (int i = t; i < heads * (DIM / 4); i += WARPS * 32) {
            const int qi = i / (DIM / 4), d = i % (DIM / 4) * 4, head = h * group + q0 + qi;
            const float sum = sl[0][qi], inv = sum == 0.f ? 0.f : 1.f / sum;
            const float4 out = sums[i];
            *reinterpret_cast<uint2*>(a.o + static_cast<size_t>(r) * a.ldo + head * DIM + d) =
                make_uint2(pack_bf16x2(out.x * inv, out.y * inv), pack_bf16x2(out.z * inv, out.w * inv));
            if (d == 0 && a.lse)
              a.lse[static_cast<size_t>(r) * a.hq + head] =
                  sum == 0.f ? -INFINITY : (sm[0][qi] + log2f(sum)) * 0.6931471805599453f;
          }
        }
      }
      __syncthreads();  // the next unit writes the shared arrays
      at += past - first;
    }
    base += static_cast<unsigned long long>(tiles) * units;
  }
}

}  // namespace sj

using namespace sj;

namespace {
int query_tiles(int hq, int hk) { return hq / hk > 8 ? 2 : 1; }
// CTAs of a launch; counters and partials are for as many.
int most_ctas() { return kCtas * sm_count(); }
size_t counter_bytes() { return (3 * static_cast<size_t>(most_ctas()) * sizeof(int) + 255) / 256 * 256; }

template <int DIM, int NQ>
int attend(const PagedAttention& a, cudaStream_t stream) {
  constexpr int outputs = kWarps * NQ * 8 * (DIM + 8) * 4, rings = kWarps * kStages * 8192;
  constexpr int smem = (outputs > rings ? outputs : rings) + 128;
  static KernelAttrOnce once;
  const int rc = ensure_max_smem(once, reinterpret_cast<const void*>(attn_paged_kernel<DIM, NQ>), smem,
                                 "sj_attn_paged: shared memory");
  if (rc != SJ_OK) return rc;
  launch(attn_paged_kernel<DIM, NQ>, most_ctas(), kWarps * 32, smem, stream, a);
  SJ_LAUNCH_CHECK("attn_paged");
  return SJ_OK;
}
}  // namespace

extern "C" size_t sj_attn_paged_workspace(int rows, int hq, int hk, int head_dim) {
  if (rows < 0 || hq <= 0 || hk <= 0 || hq % hk || (head_dim != 64 && head_dim != 128)) return 0;
  const int nq = query_tiles(hq, hk);
  return counter_bytes() + static_cast<size_t>(most_ctas()) * 2 * nq * 8 * (head_dim + 2) * sizeof(float);
}

extern "C" int sj_attn_paged(const void* q, int ldq, const void* k_cache, const void* v_cache, int pages, int page,
                             int64_t page_stride, int64_t head_stride, int64_t token_stride,
                             const int32_t* block_table, int ld_table, int requests, const int32_t* request,
                             const int32_t* position, int rows, int hq, int hk, int head_dim, int window, void* o,
                             int ldo, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || requests <= 0 || ld_table <= 0 || hq <= 0 || hk <= 0 || hq % hk || hq > 4096 || window < 0 ||
      (!request && rows > requests))
    return fail(SJ_ERR_SHAPE, "sj_attn_paged: rows=%d requests=%d ld_table=%d hq=%d hk=%d window=%d", rows, requests,
                ld_table, hq, hk, window);
  const int rc = check_paged_cache("sj_attn_paged", k_cache, v_cache, pages, page, page_stride, head_stride,
                                   token_stride, hk, head_dim);
  if (rc != SJ_OK) return rc;
  if (ldq < hq * head_dim || ldo < hq * head_dim)
    return fail(SJ_ERR_SHAPE, "sj_attn_paged: ldq=%d ldo=%d", ldq, ldo);
  if (rows == 0) return SJ_OK;
  if (!q || !o || !block_table || !position || !aligned16(q) || !aligned16(o) || ldq % 8 || ldo % 8)
    return fail(SJ_ERR_ARGUMENT, "sj_attn_paged: null or unaligned operand, or a row stride not a multiple of 8");
  if (!workspace || !aligned16(workspace) || workspace_bytes < sj_attn_paged_workspace(rows, hq, hk, head_dim))
    return fail(SJ_ERR_CAPACITY, "sj_attn_paged: workspace of %zu bytes", workspace_bytes);
  PagedAttention a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k_cache);
  a.v = static_cast<const __nv_bfloat16*>(v_cache);
  a.table = block_table;
  a.request = request;
  a.position = position;
  a.o = static_cast<__nv_bfloat16*>(o);
  a.lse = lse;
  a.counters = static_cast<int*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + counter_bytes());
  a.page_stride = page_stride;
  a.head_stride = head_stride;
  a.token_stride = token_stride;
  a.ldq = ldq;
  a.ldo = ldo;
  a.pages = pages;
  a.page = page;
  a.ld_table = ld_table;
  a.requests = requests;
  a.rows = rows;
  a.hq = hq;
  a.hk = hk;
  a.window = window;
  const int nq = query_tiles(hq, hk);
  cudaStream_t s = as_stream(stream);
  if (head_dim == 64) return nq == 1 ? attend<64, 1>(a, s) : attend<64, 2>(a, s);
  return nq == 1 ? attend<128, 1>(a, s) : attend<128, 2>(a, s);
}
