// The keys that the rows of a group have in common, read once for all of them (sj_attn_paged_shared).
//
//   shared_spans_kernel   each group's keys that all of its rows see, and the work that they are
//   attn_shared_kernel    the queries of a group against those keys, on the tensor cores
//   attn_paged_kernel     (attention_paged.cu) each row against its own keys
//   shared_join_kernel    the parts of each row and head joined
//
// With M queries a KV head, M multiply-adds are made of each cache element: memory bounds a few of them, the
// exponentials and the tensor cores many.  A row's keys outside [p0, p1), by its window or its length, are its own, so no
// tile needs a mask but for the last one's end, and a value that a row does not see reaches no sum of it.
//
// The weights P are rounded to bf16, the products' operand, as in attn_paged_kernel: each is off by 2^-8 of itself at most,
// and its sum takes it unrounded.  Against 64 bits outputs of random values are off by 0.0023 of their size (rms), where
// their own rounding to bf16 alone is 0.0017.
//
// Measured on B200 (graph replays, all four kernels): 509 rows that share 32768 keys, 16 / 4 heads of 128 198 us (693
// TFLOP/s; rows apart 2378); two pieces of 250 and 333 rows over 20 and 60 thousand keys, 16 / 2 heads of 128 223 (782
// TFLOP/s; 1548); 16 x 16 rows over 2048 to 16384 keys, 12 / 4 heads of 64 75 (164).  The tensor-core pass is about 153,
// 180 and 45 of these: 44% of the tensor pipe's cycles on the second, where softmax and products of a stream wait for
// one another and two streams do not fill the gaps.  Tiles that no box can fetch wait for their own copies, one at a time for
// each load warp: the first and third of these with pages of 4 271 and 131 us, and a window, whose first key is any number,
// 194 of 16000 keys where the first takes 137 without one.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <numeric>
#include <type_traits>

#include "attention_paged.cuh"
#include "common.cuh"
#include "internal.h"

namespace sj {

namespace {
constexpr int kSharedGroups = 1024;
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kLoadWarp = 9;  // two load warps: K and V
constexpr int kHalf = kSharedKeys / 2;     // keys whose P is handed over at a time
constexpr int kSharedThreads = 32 * (kLoadWarp + 2);
constexpr int kSeen = 8;                   // tiles whose masks of valid keys are kept
constexpr float kLazy = 8.f;               // a maximum may stand this far (of log2) below the true one (a published idea)
constexpr uint32_t kColO = 256;            // TMEM columns: S of two streams (their P over them), then O
constexpr uint32_t kTmemAll = 512;
constexpr uint32_t kNowhere = 0xffffffffu;
constexpr int kLastSeen = INT_MAX - 4096;
// When sharing pays: rows that each read the keys in common get them out of L2 at about 9 TB/s (134 MB in 16 us besides
// the kernel's own 5, 268 in 25), where the tensor-core pass costs 15 us to start and to join, and 1.6 (2.2 for wide
// heads) an item on each CTA.  Measured, rows apart against sharing: 8 rows of 16384 keys, 12 / 4 heads of 64 20.7 and
// 29.3 us; 32 rows of 2048 keys, 16 / 4 heads of 128 20.6 and 25.2, 64 rows 30.3 and 27.7; 16 x 16 rows of 2048 to 16384
// keys, 12 / 4 heads of 64 164 and 79.
constexpr double kSharedRate = 9e6, kSharedStart = 15.0;  // bytes a microsecond, microseconds
__host__ __device__ constexpr double shared_item_us(int head_dim) { return head_dim == 64 ? 1.6 : 2.2; }
}  // namespace

// ---------------------------------------------------------------- spans
struct SpansArgs {
  const int32_t *request, *position, *group;
  int rows, groups, requests, page, ld_table, window, hq, hk, head_dim, always;
  SharedSpans out;
};

// One CTA.  A group's p0 is the highest first key of its live rows, p1 the lowest end.
__global__ void __launch_bounds__(1024) shared_spans_kernel(const SpansArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ int first[kSharedGroups + 1], p0[kSharedGroups], p1[kSharedGroups], live[kSharedGroups];
  __shared__ unsigned long long s_scan[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int64_t most = static_cast<int64_t>(a.ld_table) * a.page;
  if (t < a.groups) {
    const bool fine = shared_group_fine(a.group, t, a.groups, a.rows, a.requests, most);
    if (!fine) record_error(SJ_DEV_BAD_INDEX);
    first[t] = a.group[3 * t];
    p0[t] = 0;
    p1[t] = fine ? a.group[3 * t + 2] : -1;
    live[t] = 0;
  }
  const bool ordered = __syncthreads_and(t >= a.groups || p1[t] >= 0);
  auto owner = [&](int r) {
    if (!ordered || a.groups == 0 || r < first[0]) return -1;
    int lo = 0, hi = a.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  };
  for (int r = t; r < a.rows; r += static_cast<int>(blockDim.x)) {
    const int b = a.request ? a.request[r] : r, pos = a.position[r];
    int n = b == -1 || pos > kLastSeen ? 0 : pos + 1;
    if (b < -1 || b >= a.requests || pos < -1 || pos > kLastSeen || n > most) {
      record_error(SJ_DEV_BAD_INDEX);
      n = 0;
    }
    const int lo = a.window > 0 ? max(0, n - a.window) : 0, g = owner(r);
    a.out.rows[r] = SharedRow{lo, n, 0, 0, g};
    if (g >= 0 && n > 0) {
      atomicMax(&p0[g], lo);
      atomicMin(&p1[g], n);
      atomicAdd(&live[g], 1);
    }
  }
  __syncthreads();
  unsigned long long items = 0;
  SharedGroup g{};
  if (t < a.groups) {
    g.first = first[t];
    g.rows = (t + 1 < a.groups ? first[t + 1] : a.rows) - first[t];
    g.request = a.group[3 * t + 1];
    g.p0 = p0[t];
    g.p1 = max(p1[t], p0[t]);
    if (!ordered || live[t] < 2) g.p1 = g.p0;
    const int per = kSharedQueries / (a.hq / a.hk);  // rows of a tile
    g.tiles = (g.rows + per - 1) / per;
    g.keys = (g.p1 - g.p0 + kSharedKeys - 1) / kSharedKeys;
    items = g.head_items() * a.hk;
  }
  unsigned long long total = 0;
  auto before = [&](unsigned long long mine) {  // the sum of the threads' before this one; total: of all
    unsigned long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = upto;
    __syncthreads();
    unsigned long long base = upto - mine;
    total = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) {
      if (w == warp) base += total;
      total += s_scan[w];
    }
    return base;
  };
  g.base = before(items);
  unsigned long long all = total;
  // bytes that the rows would read of the keys in common if each read them for itself
  before(static_cast<unsigned long long>(g.p1 - g.p0) * (t < a.groups ? live[t] : 0) * a.hk * a.head_dim * 4);
  if (!a.always && total < kSharedRate * (kSharedStart + all * shared_item_us(a.head_dim) / a.out.ctas)) {
    all = 0;
    g.p1 = g.p0;
    g.keys = 0;
    g.base = 0;
  }
  if (t < a.groups) p1[t] = g.p1;
  if (t == 0) *a.out.total = all;
  // about a CTA's items a chunk, so that a block is about a CTA's
  const unsigned long long ctas = min(static_cast<unsigned long long>(a.out.ctas), all);
  const unsigned long long chunks = all > 0 && g.tiles > 1 ? g.keys * ctas / all : 1;  // at most g.keys
  g.chunks = static_cast<int>(max(chunks, 1ull));
  const unsigned long long queries = static_cast<unsigned long long>(g.rows) * a.hq;
  g.main = before(t < a.groups ? queries * g.chunks : 0);
  if (total > a.out.main_queries) {  // not reached: a head's blocks are about as many as the CTAs
    g.chunks = 1;
    g.main = before(t < a.groups ? queries : 0);
  }
  g.blocks = static_cast<int>(before(t < a.groups ? static_cast<unsigned long long>(a.hk) * g.chunks * ((g.tiles + 1) / 2) : 0));
  if (t < a.groups) a.out.groups[t] = g;
  for (int r = t; r < a.rows; r += static_cast<int>(blockDim.x)) {
    SharedRow& row = a.out.rows[r];
    if (row.group >= 0 && row.n > 0 && p1[row.group] > p0[row.group]) {
      row.p0 = p0[row.group];
      row.p1 = p1[row.group];
    } else {
      row.group = -1;
    }
  }
}

// ---------------------------------------------------------------- tensor-core pass
struct SharedArgs {
  const __nv_bfloat16 *q, *k, *v;
  const int32_t* table;
  int64_t page_stride, head_stride, token_stride;
  int ldq, pages, page, ld_table, groups, hq, hk, fan;
  int box;      // rows of a page that a tensor copy takes: page's and the tile's common divisor; 0: copies of 16 bytes only
  float scale;  // log2(e) / sqrt(dim)
  SharedSpans s;
};

// A box of a cache: 64 dims from x, rows from y, of head z and page w.
SJ_DEVICE void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
SJ_DEVICE float shared_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SJ_DEVICE float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two f32 at a time: sm_100 adds and fuses a register pair in one instruction.
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
SJ_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
// 16 bytes from global to shared memory; zeros when !is.
SJ_DEVICE void shared_copy16(uint32_t dst, const __nv_bfloat16* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
SJ_DEVICE void shared_copy16(uint32_t dst, const __nv_bfloat16* src, bool is) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(is ? 16 : 0) : "memory");
}
// 32 lanes x 16 consecutive 32-bit columns, from thread i to lane (base + i).
SJ_DEVICE void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
SJ_DEVICE void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// One lane of a warp.
SJ_DEVICE uint32_t elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is;
}
// The instructions of the thread that issues products, as a whole warp executes them, by the lane that `is`: the
// operands are then uniform, where a branch of one lane would move each of them to uniform registers before every product
// (80 to 95 cycles a product).
//   D[tmem] (+)= A B: A from shared memory, or from TMEM with two bf16 of a row in each 32-bit column; B from shared memory
SJ_DEVICE void product_ss(uint32_t is, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(add), "r"(is)
      : "memory");
}
SJ_DEVICE void product_ts(uint32_t is, uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(add), "r"(is)
      : "memory");
}
SJ_DEVICE void commit_products(uint32_t is, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(is)
      : "memory");
}

template <int DIM>
struct SharedLay {
  static constexpr int SLOT = kSharedKeys * DIM * 2;  // a tile of K or of V
  static constexpr int HALF = kSharedKeys * 128;      // 64 dims of it: rows of 128 bytes
  static constexpr int QUERIES = kSharedQueries * DIM * 2, QUERIES_HALF = kSharedQueries * 128;
  static constexpr int STAGES = DIM == 64 ? 10 : 5;    // of the ring of K and V tiles
  static constexpr int Q = 0, RING = 2 * QUERIES, SEEN = RING + STAGES * SLOT, SUMS = SEEN + 2 * kSeen * 16,
                       BARS = SUMS + 2 * kSharedQueries * 4, SMEM = BARS + 512 + 1024;
};

// A CTA's share of a unit: items [i0, i1) of one KV head and one or two tiles of queries.
struct SharedPiece {
  SharedGroup g;
  int h, tile, chunk, i0, i1;
  bool begins, ends;  // a block
  bool two;  // two tiles of queries over the same keys; else one, over alternate tiles of keys
  int steps0, steps1;  // of the streams
  SJ_DEVICE int block() const { return g.blocks + (h * g.chunks + chunk) * ((g.tiles + 1) / 2) + tile / 2; }
  SJ_DEVICE int key(int stream, int step) const {
    return g.p0 + (two ? i0 + step : 2 * (i0 + step) + stream) * kSharedKeys;
  }
};
struct SharedWalk {
  const SharedArgs& a;
  unsigned long long at, end;
  SJ_DEVICE explicit SharedWalk(const SharedArgs& a_) : a(a_), at(0), end(0) {
    // the items in ranges of equal length, one for a CTA
    const unsigned long long total = *a.s.total, count = min(static_cast<unsigned long long>(gridDim.x), total);
    if (blockIdx.x >= count) return;
    at = total * blockIdx.x / count;
    end = total * (blockIdx.x + 1) / count;
  }
  SJ_DEVICE bool next(SharedPiece& p) {
    if (at >= end) return false;
    int lo = 0, hi = a.groups;
    while (hi - lo > 1) {  // the last group that begins at or before the item; those without items begin with the next
      const int mid = (lo + hi) >> 1;
      if (a.s.groups[mid].base <= at)
        lo = mid;
      else
        hi = mid;
    }
    p.g = a.s.groups[lo];
    const unsigned long long x = at - p.g.base, head = p.g.head_items();
    p.h = static_cast<int>(x / head);
    const unsigned long long y = x % head;
    const int pairs = p.g.tiles / 2;
    p.two = y < static_cast<unsigned long long>(pairs) * p.g.keys;
    int items;
    if (p.two) {
      const int column = static_cast<int>(y / pairs);  // the chunk that holds this tile of keys holds the item
      p.chunk = static_cast<int>((static_cast<long long>(column + 1) * p.g.chunks - 1) / p.g.keys);
      const int k0 = p.g.chunk(p.chunk), len = p.g.chunk(p.chunk + 1) - k0;
      const unsigned long long z = y - static_cast<unsigned long long>(pairs) * k0;
      p.tile = static_cast<int>(z / len) * 2;
      p.i0 = k0 + static_cast<int>(z % len);
      p.begins = p.i0 == k0;
      items = k0 + len;
    } else {
      p.chunk = 0;
      p.tile = p.g.tiles - 1;
      p.i0 = static_cast<int>(y - static_cast<unsigned long long>(pairs) * p.g.keys);
      p.begins = p.i0 == 0;
      items = p.g.halves();
    }
    p.i1 = static_cast<int>(min(static_cast<unsigned long long>(items), p.i0 + (end - at)));
    p.ends = p.i1 == items;
    at += p.i1 - p.i0;
    p.steps0 = p.i1 - p.i0;
    p.steps1 = p.two ? p.steps0 : min(p.g.keys - p.i1, p.i1) - p.i0;
    return true;
  }
};

// 11 warps, one CTA an SM.  Two streams of tiles, so that the products of one run under the softmax of the other:
//   warps 0-3, 4-7  softmax of streams 0 and 1: a thread for a query, which has the scores of half a tile in registers.  P
//                   goes over S in bf16, where the product with V reads it.  The output is
//                   rescaled only where a maximum has grown by more than 2^8: until then the sums are taken by the
//                   old one.
//   warp 8          issues S = Q K^T and O += P V of both streams.  S is 128 keys wide, since the tensor cores read Q
//                   from shared memory for every product: one of 64 keys takes 48 cycles, one of 128 64.
//   warps 9-10      pages of K and of V into a ring of tiles: tensor copies of the rows that a page and a tile have in
//                   common, a lane for each; where those are fewer than the 8 of a swizzled group, in the last tile of a
//                   group (rows past its end are zeros, whatever the cache holds there) and from a first key that is no
//                   multiple of them, copies of 16 bytes
template <int DIM>
__global__ void __launch_bounds__(kSharedThreads, 1)
    attn_shared_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const SharedArgs a) {
  using L = SharedLay<DIM>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* full = bars;                    // STAGES
  uint64_t* empty = full + L::STAGES;       // STAGES
  uint64_t* q_full = empty + L::STAGES;     // 2
  uint64_t* s_full = q_full + 2;            // 2
  uint64_t* p_full = s_full + 2;            // 2 halves of each stream
  uint64_t* o_half = p_full + 4;            // 2: the product of a tile's first half with V
  uint64_t* o_full = o_half + 2;            // 2: all products of a piece
  uint64_t* sums_full = o_full + 2;         // 1
  uint64_t* drain = sums_full + 1;          // 1
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* seen = reinterpret_cast<uint32_t*>(smem + L::SEEN);  // [2][kSeen][4]
  float* sums = reinterpret_cast<float*>(smem + L::SUMS);        // m and l of stream 1
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&o_half[i], 1);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&p_full[i], 4);
    mbar_init(sums_full, 4);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    if (a.box > 0) {
      tma_prefetch_map(&map_k);
      tma_prefetch_map(&map_v);
    }
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemAll);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  SharedWalk walk(a);
  SharedPiece p;
  uint32_t asked = 0;  // of a load warp's last tiles, the bits of those that it has asked for, and the slot after them
  int last_slot = 0, last_turn = 0;

  if (warp < kSoftmaxWarps) {
    const int stream = warp >> 2, row = (warp & 3) * 32 + lane, per = kSharedQueries / a.fan;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t col_s = tmem + lane_off + stream * kSharedKeys, col_o = tmem + lane_off + kColO + stream * DIM;
    int tile_at = 0, piece_at = 0, sums_at = 0;
    bool ok = true;
    // 16 bytes of a row of the stream's queries, which later serve to bring outputs into the order of memory
    auto cell = [&](int of_row, int c) {
      return reinterpret_cast<uint4*>(smem + L::Q + stream * L::QUERIES + (c >> 3) * L::QUERIES_HALF + of_row * 128 +
                                      (((c & 7) ^ (of_row & 7)) << 4));
    };
    const int row0 = (warp & 3) * 32;
    while (ok && walk.next(p)) {
      if (threadIdx.x == 0) {
        int2* block = a.s.blocks + p.block();
        if (p.begins) block->x = blockIdx.x;
        if (p.ends) block->y = blockIdx.x;
      }
      const int steps = stream == 0 ? p.steps0 : p.steps1;
      const int at = (p.tile + (p.two ? stream : 0)) * per + row / a.fan;  // the query's row in its group
      const int r = p.g.first + at, head = p.h * a.fan + row % a.fan;
      const bool is = row < per * a.fan && at < p.g.rows;
      if (stream == 0 || p.two) {  // this stream's queries, whole rows of a head at a time
        constexpr int LANES = DIM / 8, ROWS = 32 / LANES;
        const unsigned long long src = is ? static_cast<unsigned long long>(r) * a.ldq + head * DIM : ~0ull;
#pragma unroll
        for (int i0 = 0; i0 < 32 / ROWS; i0 += 8) {
          uint4 x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const unsigned long long from = __shfl_sync(0xffffffffu, src, (i0 + i) * ROWS + lane / LANES);
            x[i] = make_uint4(0, 0, 0, 0);
            if (from != ~0ull) x[i] = *reinterpret_cast<const uint4*>(a.q + from + lane % LANES * 8);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) *cell(row0 + (i0 + i) * ROWS + lane / LANES, lane % LANES) = x[i];
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[stream]);
      }
      const bool idle = !__any_sync(0xffffffffu, is);  // a warp without queries leaves S as it is
      float m = -INFINITY, l = 0.f;
      for (int step = 0; ok && step < steps; ++step, ++tile_at) {
        if (!mbar_wait_warp(&s_full[stream], tile_at & 1, abort_flag, SJ_DEV_ATTN_WAIT)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint2* masks = reinterpret_cast<const uint2*>(seen + (stream * kSeen + (tile_at & (kSeen - 1))) * 4);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const uint32_t col = col_s + half * kHalf;
          const uint2 valid = masks[half];
          // The exponentials are taken by the maximum so far while the new one is looked for; where that stands too far
          // above it, which is rare after the first tile, they are taken again.
          bool first = step == 0 && half == 0;
          while (!idle) {
            uint32_t x[kHalf], y[kHalf / 2];
#pragma unroll
            for (int c = 0; c < kHalf / 32; ++c)
              tmem_ld_32x32b_x32(col + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&x[c * 32]));
            const float base = m == -INFINITY ? 0.f : m;
            const uint64_t scale2 = pair2(a.scale, a.scale), base2 = pair2(-base, -base);
            uint64_t part[2] = {0, 0};
            float u[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            tmem_wait_ld();
            if ((valid.x & valid.y) != 0xffffffffu) {
#pragma unroll
              for (int i = 0; i < kHalf; ++i)
                if (!((i < 32 ? valid.x : valid.y) >> (i & 31) & 1)) x[i] = 0xff800000u;
            }
#pragma unroll
            for (int i = 0; i < kHalf / 2; ++i) {
              const float x0 = __uint_as_float(x[2 * i]), x1 = __uint_as_float(x[2 * i + 1]);
              const uint64_t d = fma2(pair2(x0, x1), scale2, base2);
              const float e0 = shared_exp2(low2(d)), e1 = shared_exp2(high2(d));
              u[i & 3] = max3(u[i & 3], x0, x1);
              part[i & 1] = add2(part[i & 1], pair2(e0, e1));
              y[i] = pack_bf16x2(e0, e1);  // the product's operand; the sums take it unrounded
            }
            const float top = fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])) * a.scale;
            const bool grown = first || !(top <= m + kLazy);
            if (!__any_sync(0xffffffffu, grown && top > m)) {
              l += (low2(part[0]) + high2(part[0])) + (low2(part[1]) + high2(part[1]));
#pragma unroll
              for (int c = 0; c < kHalf / 32; ++c)
                tmem_st_32x32b_x16(col + c * 16, *reinterpret_cast<uint32_t(*)[16]>(&y[c * 16]));
              tmem_wait_st();
              break;
            }
            const float next = fmaxf(m, top), f = m == next ? 1.f : shared_exp2(m - next);
            l *= f;
            m = next;
            if (step > 0 || half > 0) {
              // the output has the products of all tiles before, since S came after them, but maybe not this one's
              if (half == 1 && !mbar_wait_warp(&o_half[stream], tile_at & 1, abort_flag, SJ_DEV_ATTN_WAIT)) {
                ok = false;
                break;
              }
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < DIM / 16; ++c) {
                uint32_t z[16];
                tmem_ld_32x32b_x16(col_o + c * 16, z);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = __float_as_uint(f * __uint_as_float(z[i]));
                tmem_st_32x32b_x16(col_o + c * 16, z);
              }
              tmem_wait_st();
            }
            first = false;
          }
          if (!ok) break;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[stream * 2 + half]);
        }
        if (!ok) break;
      }
      if (!ok) break;
      if (steps > 0) {
        if (!mbar_wait_warp(&o_full[stream], piece_at & 1, abort_flag, SJ_DEV_ATTN_WAIT)) break;
        ++piece_at;
        tc_fence_after();
      }
      if (!p.two && stream == 1) {  // stream 0 has the same queries, and joins the two
        if (steps > 0) {
          sums[row] = m;
          sums[kSharedQueries + row] = l;
          __syncwarp();
          if (lane == 0) mbar_arrive(sums_full);
        }
        continue;
      }
      const bool joined = !p.two && p.steps1 > 0;
      float f = 1.f, g = 0.f;
      if (joined) {
        if (!mbar_wait_warp(sums_full, sums_at & 1, abort_flag, SJ_DEV_ATTN_WAIT)) break;
        ++sums_at;
        tc_fence_after();
        const float m2 = sums[row], top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
        f = shared_exp2(m - base);
        g = shared_exp2(m2 - base);
        l = f * l + g * sums[kSharedQueries + row];
        m = top;
      }
      if (idle) continue;
      const SharedParts& to = p.begins ? a.s.main : a.s.slots;
      const size_t query = p.begins ? p.g.main + (static_cast<size_t>(p.chunk) * p.g.rows + (is ? at : 0)) * a.hq + head
                                    : static_cast<size_t>(blockIdx.x) * (2 * kSharedQueries) +
                                          (p.two ? stream * kSharedQueries : 0) + row;
      const unsigned long long dst = is ? query * DIM : ~0ull;
      // half of the dims at a time through the cells of this warp's rows, so that stores are of whole lines
#pragma unroll
      for (int c0 = 0; c0 < DIM; c0 += DIM / 2) {
#pragma unroll
        for (int c = 0; c < DIM / 32; ++c) {
          uint32_t x[16], y[16];
          tmem_ld_32x32b_x16(col_o + c0 + c * 16, x);
          if (joined) tmem_ld_32x32b_x16(col_o + DIM + c0 + c * 16, y);
          tmem_wait_ld();
          if (joined) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float v = f == 0.f ? 0.f : f * __uint_as_float(x[i]), w = g == 0.f ? 0.f : g * __uint_as_float(y[i]);
              x[i] = __float_as_uint(v + w);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *cell(row, c * 4 + i) = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        }
        __syncwarp();
        constexpr int LANES = DIM / 8, ROWS = 32 / LANES;
#pragma unroll
        for (int i = 0; i < 32 / ROWS; ++i) {
          const int rr = i * ROWS + lane / LANES;
          const unsigned long long there = __shfl_sync(0xffffffffu, dst, rr);
          const uint4 x = *cell(row0 + rr, lane % LANES);
          if (there != ~0ull) *reinterpret_cast<uint4*>(to.o + there + c0 + lane % LANES * 4) = x;
        }
        __syncwarp();
      }
      if (is) {
        to.m[query] = m;
        to.l[query] = l;
      }
      tc_fence_before();
    }
  } else if (warp == kMmaWarp) {
    {
      const uint32_t is = elect_one();
      constexpr uint32_t kIdescS = umma_idesc_bf16(kSharedQueries, kSharedKeys, 0, 0);
      constexpr uint32_t kIdescO = umma_idesc_bf16(kSharedQueries, DIM, 0, 1);
      // descriptors differ in their addresses only, which are in the low words
      auto desc = [](uint32_t low, uint32_t off) {
        constexpr uint32_t high = (1024 >> 4) | 1u << 14 | 2u << 29;
        return static_cast<uint64_t>(high) << 32 | (low + (off >> 4));
      };
      auto low = [](const uint8_t* at, uint32_t lead) { return ((smem_u32(at) >> 4) & 0x3fffu) | (lead >> 4) << 16; };
      const uint32_t q_low = low(smem + L::Q, 16), k_low = low(smem + L::RING, 16), v_low = low(smem + L::RING, L::HALF);
      int slot = 0, turn = 0, q_at[2] = {0, 0}, tile_at[2] = {0, 0};
      // After a wait that gave up the piece's products are of no use, but harmless, and its other waits give up at once.
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        mbar_wait(bar, parity, abort_flag, SJ_DEV_ATTN_WAIT);
        tc_fence_after();
      };
      // A look at a barrier whose answer is needed after the next products only, so that its latency is hidden.
      auto peek = [&](uint64_t* bar, uint32_t parity) { return mbar_test_wait(bar, parity); };
      auto settle = [&](bool done, uint64_t* bar, uint32_t parity) {
        if (!done) mbar_wait(bar, parity, abort_flag, SJ_DEV_ATTN_WAIT);
        tc_fence_after();
      };
      auto wait_tile = [&]() { wait(&full[slot], turn); };
      auto release = [&]() {  // the tile at hand is done with when the products so far are
        commit_products(is, &empty[slot]);
        if (++slot == L::STAGES) {
          slot = 0;
          turn ^= 1;
        }
      };
      auto scores = [&](int stream, int queries, int of) {  // S = Q K^T
        const uint32_t q = q_low + queries * (L::QUERIES >> 4), k = k_low + of * (L::SLOT >> 4);
#pragma unroll
        for (int kk = 0; kk < DIM / 16; ++kk)
          product_ss(is, tmem + stream * kSharedKeys, desc(q, (kk >> 2) * L::QUERIES_HALF + (kk & 3) * 32),
                     desc(k, (kk >> 2) * L::HALF + (kk & 3) * 32), kIdescS, kk > 0 ? 1u : 0u);
        commit_products(is, &s_full[stream]);
      };
      auto outputs = [&](int stream, int half, int of, bool first) {  // O += P V
        const uint32_t v = v_low + of * (L::SLOT >> 4) + half * (kHalf * 128 >> 4);
#pragma unroll
        for (int kk = 0; kk < kHalf / 16; ++kk)
          product_ts(is, tmem + kColO + stream * DIM, tmem + stream * kSharedKeys + half * kHalf + kk * 8,
                     desc(v, kk * 2048), kIdescO, !first || kk > 0 ? 1u : 0u);
      };
      auto wait_q = [&](int stream) {
        wait(&q_full[stream], q_at[stream] & 1);
        ++q_at[stream];
      };
      // A tile of a stream, in two steps: the product of the first half of P with the V at hand; that of the second, and
      // S of the stream's next tile, whose K lies in the slot behind.
      auto first_half = [&](int stream, bool first) {
        const bool value = peek(&full[slot], turn);
        wait(&p_full[stream * 2], tile_at[stream] & 1);
        settle(value, &full[slot], turn);
        outputs(stream, 0, slot, first);
        commit_products(is, &o_half[stream]);
      };
      auto second_half = [&](int stream, int queries, bool more, bool last_user) {
        const int next = slot + 1 == L::STAGES ? 0 : slot + 1, next_turn = next == 0 ? turn ^ 1 : turn;
        const bool key = peek(&full[next], next_turn);
        wait(&p_full[stream * 2 + 1], tile_at[stream] & 1);
        outputs(stream, 1, slot, false);
        ++tile_at[stream];
        if (last_user) release();
        if (more) {
          settle(key, &full[next], next_turn);
          scores(stream, queries, next);
          if (last_user) release();
        } else {
          commit_products(is, &o_full[stream]);
        }
      };
      while (__shfl_sync(0xffffffffu, *abort_flag == 0 && walk.next(p) ? 1 : 0, 0)) {
        const int n0 = __shfl_sync(0xffffffffu, p.steps0, 0), n1 = __shfl_sync(0xffffffffu, p.steps1, 0);
        const bool two = __shfl_sync(0xffffffffu, p.two ? 1 : 0, 0) != 0;
        wait_q(0);
        wait_tile();
        scores(0, 0, slot);
        if (two) {
          wait_q(1);
          scores(1, 1, slot);
          release();
          for (int i = 0; i < n0; ++i) {
            first_half(0, i == 0);
            first_half(1, i == 0);
            second_half(0, 0, i + 1 < n0, false);
            second_half(1, 1, i + 1 < n0, true);
          }
        } else {
          release();
          if (n1 > 0) {
            wait_tile();
            scores(1, 0, slot);
            release();
          }
          for (int i = 0; i < n0; ++i) {
            first_half(0, i == 0);
            second_half(0, 0, i + 1 < n0, true);
            if (i >= n1) continue;
            first_half(1, i == 0);
            second_half(1, 0, i + 1 < n1, true);
          }
        }
      }
      commit_products(is, drain);
      mbar_wait(drain, 0, nullptr, SJ_DEV_ATTN_WAIT);
    }
  } else {
    // both warps follow the order of all tiles; one fetches those of K, the other those of V
    const bool of_k = warp == kLoadWarp;
    const __nv_bfloat16* from = of_k ? a.k : a.v;
    const CUtensorMap* map = of_k ? &map_k : &map_v;
    int slot = 0, turn = 0, seen_at[2] = {0, 0};
    bool ok = true;
    uint32_t fetched = 0;  // of the last tiles, those that this warp has asked for
    auto pass = [&](uint32_t mine) {
      fetched = fetched << 1 | mine;
      if (++slot == L::STAGES) {
        slot = 0;
        turn ^= 1;
      }
    };
    auto place = [&](int key) {  // where a key lies, in 16-byte pieces
      if (key >= p.g.p1) return kNowhere;
      const int index = key / a.page, page = a.table[static_cast<size_t>(p.g.request) * a.ld_table + index];
      if (page < 0 || page >= a.pages) {
        record_error(SJ_DEV_BAD_INDEX);
        return kNowhere;
      }
      return static_cast<uint32_t>(
          (page * a.page_stride + p.h * a.head_stride + (key - index * a.page) * a.token_stride) >> 3);
    };
    struct Box {  // this lane's of a tile: its page and the first row there
      int page, row;
    };
    const int boxes = a.box > 0 ? kSharedKeys / a.box : 0;
    auto look_up = [&](int key) {
      Box x{0, 0};
      key += lane * a.box;
      if (lane < boxes && key < p.g.p1) {
        const int index = key / a.page;
        x.page = a.table[static_cast<size_t>(p.g.request) * a.ld_table + index];
        x.row = key - index * a.page;
      }
      return x;
    };
    auto mark = [&](int stream, int word, uint32_t have) {
      if (lane == 0) seen[(stream * kSeen + (seen_at[stream] & (kSeen - 1))) * 4 + word] = have;
    };
    auto fetch = [&](int stream, int key, const Box& x) {
      ok = mbar_wait_warp(&empty[slot], turn ^ 1, abort_flag, SJ_DEV_ATTN_WAIT);
      if (!ok) return;
      const uint32_t dst = smem_u32(smem + L::RING + slot * L::SLOT);
      const bool boxed = boxes > 0 && key % a.box == 0 && key + kSharedKeys <= p.g.p1;
      if (boxed && __all_sync(0xffffffffu, lane >= boxes || (x.page >= 0 && x.page < a.pages))) {
        if (of_k) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mark(stream, i, 0xffffffffu);
            if (p.two) mark(1, i, 0xffffffffu);
          }
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[slot], L::SLOT);
        __syncwarp();
        if (lane < boxes) {
#pragma unroll
          for (int i = 0; i < DIM / 64; ++i)
            tma_load_4d(dst + i * L::HALF + lane * a.box * 128, map, &full[slot], i * 64, x.row, p.h, x.page);
        }
      } else {
        constexpr int LANES = DIM / 8, ROWS = 32 / LANES;  // of a row, in one instruction
#pragma unroll 1
        for (int i0 = 0; i0 < kSharedKeys; i0 += 32) {
          const uint32_t where = place(key + i0 + lane), have = __ballot_sync(0xffffffffu, where != kNowhere);
          if (of_k) {
            mark(stream, i0 >> 5, have);
            if (p.two) mark(1, i0 >> 5, have);
          }
#pragma unroll
          for (int i = 0; i < 32; i += ROWS) {
            const int row = i + lane / LANES;
            const uint32_t at = __shfl_sync(0xffffffffu, where, row);
            shared_copy16(dst + ((lane % LANES) >> 3) * L::HALF + (i0 + row) * 128 + (((lane & 7) ^ (row & 7)) << 4),
                          from + (at == kNowhere ? 0 : static_cast<size_t>(at) * 8 + lane % LANES * 8), at != kNowhere);
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[slot]);
      }
      ++seen_at[stream];
      if (p.two) ++seen_at[1];
      pass(1);
    };
    while (ok && walk.next(p)) {
      const int n0 = p.steps0, n1 = p.two ? 0 : p.steps1;
      Box next[2];  // of the next tile of each stream that this warp fetches
      next[0] = look_up(p.key(0, 0));
      if (n1 > 0) next[1] = look_up(p.key(1, 0));
      auto tile = [&](int stream, int step, bool mine) {
        if (!mine) {
          pass(0);
          return;
        }
        const Box x = next[stream];
        next[stream] = look_up(p.key(stream, step + 1));  // past the piece's end as well, where it is not used
        fetch(stream, p.key(stream, step), x);
      };
      tile(0, 0, of_k);
      if (ok && n1 > 0) tile(1, 0, of_k);
      for (int i = 0; i < n0 && ok; ++i) {
        tile(0, i, !of_k);
        if (ok && i + 1 < n0) tile(0, i + 1, of_k);
        if (ok && i < n1) tile(1, i, !of_k);
        if (ok && i + 1 < n1) tile(1, i + 1, of_k);
      }
    }
    asked = fetched;
    last_slot = slot;
    last_turn = turn;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemAll);
  }
  // Nothing lands after the CTA has gone: the products have waited for every tile that was asked for, unless a wait gave up,
  // which all warps know by now.
  for (int i = 0; warp >= kLoadWarp && *abort_flag != 0 && i < L::STAGES; ++i, asked >>= 1) {
    last_turn ^= last_slot == 0 ? 1 : 0;
    last_slot = last_slot == 0 ? L::STAGES - 1 : last_slot - 1;
    if (asked & 1) mbar_wait(&full[last_slot], last_turn, nullptr, SJ_DEV_ATTN_WAIT);
  }
}

// ---------------------------------------------------------------- join
// A warp for a row and head: its own part, then the parts of its keys in common, 32 at a time: of 16 chunks two CTAs
// each, or of one chunk 32 CTAs.  The lanes take the weights, then each its dims of all parts, in order.
template <int DIM>
__global__ void __launch_bounds__(256, 5) shared_join_kernel(const SharedSpans s, int rows, int hq, int fan, __nv_bfloat16* o,
                                                          int ldo, float* lse) {
  pdl_wait();
  constexpr int PER = DIM / 32, AT_ONCE = 4;
  using Dims = typename std::conditional<PER == 4, float4, float2>::type;
  const int lane = threadIdx.x & 31, at = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= rows * hq) return;
  const int r = at / hq, head = at - r * hq;
  const SharedRow row = s.rows[r];
  if (row.group < 0) return;  // written already
  float m = s.own.m[at], l = s.own.l[at], acc[PER];
  auto take = [&](float (&to)[PER], const float* from) {
    const Dims x = *reinterpret_cast<const Dims*>(from + lane * PER);
#pragma unroll
    for (int e = 0; e < PER; ++e) to[e] = reinterpret_cast<const float*>(&x)[e];
  };
  take(acc, s.own.o + static_cast<size_t>(at) * DIM);
  {
    const SharedGroup g = s.groups[row.group];
    const int per = kSharedQueries / fan, in = r - g.first, tile = in / per;
    const bool two = tile / 2 < g.tiles / 2;
    const int chunks = two ? g.chunks : 1;
    const int slot = (two ? (tile & 1) * kSharedQueries : 0) + in % per * fan + head % fan;
    const int2* blocks = s.blocks + g.blocks + (head / fan) * g.chunks * ((g.tiles + 1) / 2) + tile / 2;
    const int side = chunks > 1 ? 2 : 32;  // CTAs of a chunk at a time
    for (int c0 = 0; c0 < chunks; c0 += 32 / side) {
      const int c = c0 + lane / side;
      int2 span = c < chunks ? blocks[c * ((g.tiles + 1) / 2)] : make_int2(0, -1);
      if (!shared_span_fine(span, s.ctas)) span = make_int2(0, -1);
      for (int k = lane % side; __any_sync(0xffffffffu, span.x + k <= span.y); k += side) {
        const bool is = span.x + k <= span.y;
        const SharedParts& part = k == 0 ? s.main : s.slots;
        const size_t query = !is ? 0
                             : k == 0 ? g.main + (static_cast<size_t>(c) * g.rows + in) * hq + head
                                      : static_cast<size_t>(span.x + k) * (2 * kSharedQueries) + slot;
        const float pm = is ? part.m[query] : -INFINITY, pl = is ? part.l[query] : 0.f;
        const unsigned long long from = reinterpret_cast<unsigned long long>(part.o + query * DIM);
        const float top = fmaxf(m, warp_max(pm)), ref = top == -INFINITY ? 0.f : top;
        const float f = shared_exp2(m - ref), w = shared_exp2(pm - ref);
        l = f * l + warp_sum(w * pl);
        m = top;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] *= f;
        uint32_t left = __ballot_sync(0xffffffffu, is);
        while (left) {
          float x[AT_ONCE][PER], weight[AT_ONCE];
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j) {
            const int of = left ? __ffs(left) - 1 : -1;
            left &= left - 1;
            weight[j] = of < 0 ? 0.f : __shfl_sync(0xffffffffu, w, of);
            const unsigned long long src = __shfl_sync(0xffffffffu, from, max(of, 0));
#pragma unroll
            for (int e = 0; e < PER; ++e) x[j][e] = 0.f;
            if (of >= 0) take(x[j], reinterpret_cast<const float*>(src));
          }
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] += weight[j] * x[j][e];
        }
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t* dst = reinterpret_cast<uint32_t*>(o + static_cast<size_t>(r) * ldo + head * DIM + lane * PER);
#pragma unroll
  for (int e = 0; e < PER; e += 2) dst[e / 2] = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
  if (lane == 0 && lse) lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

namespace {
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Where the parts of the workspace lie, from its own start.
size_t shared_layout(SharedSpans* s, char* at, int rows, int groups, int hq, int hk, int head_dim) {
  size_t n = 0;
  auto take = [&](size_t bytes) {
    const size_t was = n;
    n += up256(bytes);
    return at + was;
  };
  char* total = take(sizeof(unsigned long long));
  char* group = take(sizeof(SharedGroup) * groups);
  char* row = take(sizeof(SharedRow) * rows);
  // of a group with pairs of tiles twice its chunks * pairs * hk at most, else a unit a KV head
  char* block = take(sizeof(int2) * (2 * static_cast<size_t>(sm_count()) + static_cast<size_t>(hk) * (2 * rows + groups)));
  auto parts = [&](size_t queries) {
    float* m = reinterpret_cast<float*>(take(queries * sizeof(float)));
    float* l = reinterpret_cast<float*>(take(queries * sizeof(float)));
    return SharedParts{m, l, reinterpret_cast<float*>(take(queries * head_dim * sizeof(float)))};
  };
  // chunks * pairs * hk of a group is at most its share of the CTAs, and a pair brings a third tile at most
  const size_t own = static_cast<size_t>(rows) * hq, ctas = static_cast<size_t>(sm_count());
  const size_t main_queries = own + ctas * 3 * kSharedQueries;
  const SharedSpans all{reinterpret_cast<unsigned long long*>(total), reinterpret_cast<SharedGroup*>(group),
                        reinterpret_cast<SharedRow*>(row), reinterpret_cast<int2*>(block), parts(own), parts(main_queries),
                        parts(ctas * 2 * kSharedQueries), main_queries, static_cast<int>(ctas)};
  if (s) *s = all;
  return n;
}

template <int DIM>
int shared_pass(SharedArgs a, cudaStream_t stream) {
  static KernelAttrOnce once;
  const int rc = ensure_max_smem(once, reinterpret_cast<const void*>(attn_shared_kernel<DIM>), SharedLay<DIM>::SMEM,
                                 "sj_attn_paged_shared: shared memory");
  if (rc != SJ_OK) return rc;
  CUtensorMap maps[2] = {};
  if (a.box > 0) {
    const uint64_t dims[4] = {DIM, static_cast<uint64_t>(a.page), static_cast<uint64_t>(a.hk),
                              static_cast<uint64_t>(a.pages)};
    const uint64_t strides[3] = {static_cast<uint64_t>(a.token_stride) * 2, static_cast<uint64_t>(a.head_stride) * 2,
                                 static_cast<uint64_t>(a.page_stride) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(a.box), 1, 1};
    for (int i = 0; i < 2; ++i) {
      const int map_rc = tensor_map(&maps[i], i == 0 ? a.k : a.v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, dims, strides, box,
                                    CU_TENSOR_MAP_SWIZZLE_128B);
      if (map_rc != SJ_OK) a.box = 0;  // copies of 16 bytes take any strides
    }
  }
  launch(attn_shared_kernel<DIM>, a.s.ctas, kSharedThreads, SharedLay<DIM>::SMEM, stream, maps[0], maps[1], a);
  SJ_LAUNCH_CHECK("attn_shared");
  return SJ_OK;
}
}  // namespace
}  // namespace sj

using namespace sj;

namespace {
// Groups that the tensor-core pass takes: tiles hold whole rows, and one CTA knows all groups.
bool shares(int groups, int hq, int hk) { return groups > 0 && groups <= kSharedGroups && hq / hk <= kSharedQueries; }
}  // namespace

extern "C" size_t sj_attn_paged_shared_workspace(int rows, int groups, int hq, int hk, int head_dim) {
  const size_t own = sj_attn_paged_workspace(rows, hq, hk, head_dim);
  if (own == 0 || groups < 0) return 0;
  if (!shares(groups, hq, hk)) return own;
  return up256(own) + shared_layout(nullptr, nullptr, rows, groups, hq, hk, head_dim);
}

extern "C" int sj_attn_paged_shared(const void* q, int ldq, const void* k_cache, const void* v_cache, int pages,
                                    int page, int64_t page_stride, int64_t head_stride, int64_t token_stride,
                                    const int32_t* block_table, int ld_table, int requests, const int32_t* request,
                                    const int32_t* position, int rows, const int32_t* group, int groups, int hq,
                                    int hk, int head_dim, int window, void* o, int ldo, float* lse, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  constexpr const char* who = "sj_attn_paged_shared";
  if (groups < 0 || (rows > 0 && groups > rows) || (hq > 0 && rows > INT_MAX / hq))
    return fail(SJ_ERR_SHAPE, "%s: groups=%d rows=%d", who, groups, rows);
  PagedAttention a;
  int rc = paged_attention_args(who, a, q, ldq, k_cache, v_cache, pages, page, page_stride, head_stride, token_stride,
                                block_table, ld_table, requests, request, position, rows, hq, hk, head_dim, window, o,
                                ldo, lse, workspace, workspace_bytes,
                                sj_attn_paged_shared_workspace(rows, groups, hq, hk, head_dim));
  if (rc != SJ_OK || rows == 0) return rc;
  if (groups > 0 && !group) return fail(SJ_ERR_ARGUMENT, "%s: null operand", who);
  cudaStream_t s = as_stream(stream);
  const double most = static_cast<double>(rows) * hk * head_dim * 4 * ld_table * page;  // bytes that rows apart read
  const char* wish = std::getenv("SJ_ATTN_SHARE");
  const bool always = wish && std::strcmp(wish, "always") == 0;
  if (!shares(groups, hq, hk) || (!always && most < kSharedRate * kSharedStart)) {
    a.group = group;
    a.groups = groups;
    return attn_paged_rows(a, nullptr, head_dim, s);
  }
  SharedSpans spans;
  shared_layout(&spans, static_cast<char*>(workspace) + up256(sj_attn_paged_workspace(rows, hq, hk, head_dim)), rows,
                groups, hq, hk, head_dim);
  const SpansArgs sa{request, position, group, rows, groups, requests, page, ld_table, window, hq, hk, head_dim, always ? 1 : 0, spans};
  // A thread takes a group, and the rows in turn.  The barriers and scans of 256 threads are shorter, which pays up to about 2048
  // rows (the whole call, 256 and 1024 threads: 256 rows 38.7 and 43.5 us, 2048 rows of 8 groups 80.3 and 82.1, 4096 rows 154.7
  // and 148.7, 16384 595 and 550).
  launch(shared_spans_kernel, 1, groups <= 256 && rows <= 2048 ? 256 : 1024, 0, s, sa);
  SJ_LAUNCH_CHECK("shared_spans");
  // Tensor copies of boxes that pages and tiles have in common, of whole swizzled groups of 8 rows; strides that a map
  // takes (not 0, below 2^40 bytes: a head or page that no index reaches may have any).
  const int divisor = std::gcd(page, kSharedKeys);
  auto fits = [](int64_t stride) { return stride > 0 && stride < int64_t{1} << 39; };
  const int box = divisor % 8 == 0 && fits(page_stride) && fits(head_stride) && fits(token_stride) ? divisor : 0;
  const SharedArgs ta{a.q, a.k, a.v, block_table, page_stride, head_stride, token_stride, ldq, pages, page, ld_table,
                      groups, hq, hk, hq / hk, box, 1.4426950408889634f / sqrtf(static_cast<float>(head_dim)), spans};
  rc = head_dim == 64 ? shared_pass<64>(ta, s) : shared_pass<128>(ta, s);
  if (rc == SJ_OK) rc = attn_paged_rows(a, &spans, head_dim, s);
  if (rc != SJ_OK) return rc;
  const int64_t queries = static_cast<int64_t>(rows) * hq;
  launch(head_dim == 64 ? shared_join_kernel<64> : shared_join_kernel<128>, static_cast<unsigned>((queries + 7) / 8), 256, 0,
         s, spans, rows, hq, hq / hk, a.o, ldo, lse);
  SJ_LAUNCH_CHECK("shared_join");
  return SJ_OK;
}
