// Pages of a cache that several requests share: a step's reordering of requests, copies of pages, and
// the pages in use moved to the front of the cache (paged.cu plans and ends the steps themselves).
//
//   paged_fork_kernel     block tables, owners and the free stack after each request took over another's pages
//   paged_copy_kernel     rows of pages to other pages, in every layer
//   paged_compact_kernel  the pages in use mapped to the lowest ids
//
// shares[p] is the number of requests that hold page p beyond the first, 0 for a free page, so that a page that
// sj_paged_plan takes from the stack needs no entry of its own.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "internal.h"

namespace cg = cooperative_groups;

namespace sj {

namespace {
constexpr int kShareMaxBatch = 4096, kShareMaxPages = 1 << 18;  // counters of an eighth of them fit shared memory, and masks of all
constexpr int kForkNoPages = 2, kForkTableNarrow = 3, kForkBad = 4;
constexpr int kCompactMovesOver = 1, kCompactBad = 4;
constexpr int kForkCluster = 8, kForkThreads = 1024;
constexpr int kForkChunk = 128;       // entries of a block table that a warp takes at a time
constexpr int kForkRun = 8;           // slots whose entries it counts together
constexpr int kForkUnits = 4;         // owners that a thread asks for at a time
constexpr int kNoEntry = INT_MIN;     // out of range as well, so that it need not be told from a table's
constexpr int kCopyThreads = 256, kCopyPieces = 8;  // 16-byte pieces of a thread
constexpr int kCompactThreads = 1024, kCompactIds = 8;  // of the stack, that a thread asks for at a time
}  // namespace

// ---------------------------------------------------------------- fork
struct Fork {
  const int32_t *parent, *cached, *table, *shares, *stack, *stack_count;
  int32_t *cached_out, *table_out, *shares_out, *stack_out, *count_out, *copies, *summary;
  int batch, page, ld_table, pages, per;  // per: pages whose owners a CTA counts
};

// A slot's pages pass to its children: full ones are shared, a half-filled last page goes to the lowest child and is
// copied to a fresh page for each of the others.  Every CTA scans the batch for itself.  The first cluster counts: an
// entry of a slot with c children changes its page's owners by c - 1 (the half-filled page of a slot without children
// by -1); the counters of a CTA's share of the pages lie in its shared memory, which the others add to (integers, so the
// order does not matter; in memory, with the fences that takes, 9.3 us instead of 8.8 for 32 requests).  Then each CTA
// knows which of its pages nobody holds, and after one exchange of numbers where on the stack they go.  The other
// clusters write tables.  Bound by latency, four phases of a few dependent loads: 32 requests 8.8 us (graph replays), 1024
// requests of 500 to 32768 tokens in pages of 64 22.2 (34 with an addition to another CTA's counter for each entry).
__global__ void __launch_bounds__(kForkThreads) paged_fork_kernel(const Fork a) {
  pdl_wait();
  extern __shared__ int dynamic[];
  int* children = dynamic;                       // [batch + 1]
  int* lowest = children + (a.batch + 1);        // [batch + 1]
  int* rank = lowest + (a.batch + 1);            // [batch + 1] copies of the slots before, -1: no copy
  int* parents = rank + (a.batch + 1);           // [batch + 1]
  int* lengths = parents + (a.batch + 1);        // [batch + 1]
  int* counter = lengths + (a.batch + 1);        // of the CTA's pages: the change of their owners
  __shared__ int s_bad, s_narrow, s_back, s_warp[kForkThreads / 32];
  cg::cluster_group cluster = cg::this_cluster();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, batch = a.batch, page = a.page;
  const int threads = blockDim.x, warps = threads >> 5;
  const int cta = cluster.block_rank(), ctas = cluster.num_blocks();
  const bool counts = blockIdx.x < static_cast<unsigned>(ctas);
  if (t == 0) s_bad = s_narrow = 0;
  for (int b = t; b < batch; b += threads) {
    children[b] = 0;
    lowest[b] = INT_MAX;
    parents[b] = a.parent[b];
    lengths[b] = a.cached[b];
  }
  // this CTA's share of the pages
  const int page0 = min(cta * a.per, a.pages), mine = counts ? min(a.per, a.pages - page0) : 0;
  for (int i = t; i < mine; i += threads) counter[i] = 0;
  __syncthreads();
  auto length = [&](int b) { return lengths[b]; };
  for (int b = t; b < batch; b += threads) {
    const int p = parents[b], n = length(b);
    if (p < -1 || p >= batch || n < 0 || n > INT_MAX - page) {
      s_bad = 1;
      continue;
    }
    if ((n + page - 1) / page > a.ld_table) s_narrow = 1;
    if (p >= 0) {
      atomicAdd(&children[p], 1);
      atomicMin(&lowest[p], b);
    }
  }
  const int count = *a.stack_count;
  if (count < 0 || count > a.pages) s_bad = 1;
  __syncthreads();
  int status = s_bad ? kForkBad : s_narrow ? kForkTableNarrow : 0;
  // copies of the slots before each, 32 slots a warp at a time
  {
    int taken = 0;
    for (int b0 = 0; b0 < batch; b0 += threads) {
      const int b = b0 + t, p = b < batch && !status ? parents[b] : -1;
      const bool copied = p >= 0 && lowest[p] != b && length(p) % page != 0;
      const unsigned have = __ballot_sync(0xffffffffu, copied);
      if (lane == 0) s_warp[warp] = __popc(have);
      __syncthreads();
      int before = taken, all = 0;
      for (int w = 0; w < warps; ++w) {
        if (w < warp) before += s_warp[w];
        all += s_warp[w];
      }
      if (b < batch) rank[b] = copied ? before + __popc(have & ((1u << lane) - 1)) : -1;
      taken += all;
      __syncthreads();
    }
    if (t == 0) s_back = taken;
    __syncthreads();
  }
  int taken = s_back;
  if (!status && taken > count) status = kForkNoPages;
  if (status) taken = 0;
  // with a status, every slot keeps what it holds
  auto source = [&](int b) { return status ? b : parents[b]; };
  auto held = [&](int p) {
    const int n = length(p);
    return n < 0 || n > INT_MAX - page ? 0 : min((n + page - 1) / page, a.ld_table);
  };
  auto fresh = [&](int b) { return a.stack[count - 1 - rank[b]]; };

  // ---- tables, lengths, copies, what stays of the stack
  const int writers = gridDim.x - ctas, writer = static_cast<int>(blockIdx.x) - ctas;
  if (writer >= 0) {
    const int chunks = (a.ld_table + kForkChunk - 1) / kForkChunk;
    for (int u = writer * warps + warp; u < batch * chunks; u += writers * warps) {
      const int b = u % batch, j0 = u / batch * kForkChunk, p = source(b);
      const bool copied = !status && rank[b] >= 0;
      const int n = p < 0 ? 0 : held(p), own = copied ? n - 1 : -1, end = min(n, j0 + kForkChunk);
      const int32_t* from = a.table + static_cast<size_t>(max(p, 0)) * a.ld_table;
      int32_t* to = a.table_out + static_cast<size_t>(b) * a.ld_table;
      int32_t id[kForkChunk / 32];
#pragma unroll
      for (int e = 0; e < kForkChunk / 32; ++e) id[e] = j0 + 32 * e + lane < end ? from[j0 + 32 * e + lane] : 0;
#pragma unroll
      for (int e = 0; e < kForkChunk / 32; ++e) {
        if (j0 + 32 * e + lane >= end) continue;
        if (!status && (id[e] < 0 || id[e] >= a.pages)) record_error(SJ_DEV_BAD_INDEX);
        if (j0 + 32 * e + lane != own) to[j0 + 32 * e + lane] = id[e];
      }
      if (!status && children[b] == 0) {  // whose entries nobody takes over: looked at here, where there is time, and counted below
        const int32_t* left = a.table + static_cast<size_t>(b) * a.ld_table;
        const int until = min(held(b), j0 + kForkChunk);
#pragma unroll
        for (int e = 0; e < kForkChunk / 32; ++e) id[e] = j0 + 32 * e + lane < until ? left[j0 + 32 * e + lane] : 0;
#pragma unroll
        for (int e = 0; e < kForkChunk / 32; ++e)
          if (id[e] < 0 || id[e] >= a.pages) record_error(SJ_DEV_BAD_INDEX);
      }
      if (lane == 0 && j0 == 0) {
        a.cached_out[b] = p < 0 ? 0 : length(p);
        if (copied) {
          const int dst = fresh(b), at = rank[b], src = from[own];
          to[own] = dst;
          const bool fine = dst >= 0 && dst < a.pages && src >= 0 && src < a.pages;
          if (!fine) record_error(SJ_DEV_BAD_INDEX);
          a.copies[3 * at] = fine ? src : -1;
          a.copies[3 * at + 1] = fine ? dst : -1;
          a.copies[3 * at + 2] = fine ? length(p) % page : 0;
        }
      }
    }
    const int first = writer * threads + t, step = writers * threads;
    for (int i = taken + first; i < batch; i += step) {
      a.copies[3 * i] = a.copies[3 * i + 1] = -1;
      a.copies[3 * i + 2] = 0;
    }
    const int stays = min(max(count, 0), a.pages) - taken;
    for (int i = first; i < stays; i += step) a.stack_out[i] = a.stack[i];
  }
  if (!counts) return;

  // ---- owners
  cluster.sync();  // every counter of the cluster is zero
  if (!status) {
    // A warp takes a chunk of the tables of kForkRun slots side by side.  Slots that came from one share their first pages,
    // and what their children take and leave there mostly adds up to nothing: it is added up here, as long as the page
    // is the same, before it goes to memory.
    const int chunks = (a.ld_table + kForkChunk - 1) / kForkChunk, runs = (batch + kForkRun - 1) / kForkRun;
    constexpr int PER = kForkChunk / 32;
    for (int u = cta * warps + warp; u < runs * chunks; u += ctas * warps) {
      const int p0 = u % runs * kForkRun, j0 = u / runs * kForkChunk + lane;
      int32_t id[kForkRun][PER];
#pragma unroll
      for (int k = 0; k < kForkRun; ++k) {
        const int p = min(p0 + k, batch - 1), change = p0 + k < batch ? children[p] - 1 : 0;
        const int end = change == 0 ? 0 : change < 0 ? held(p) : length(p) / page;
#pragma unroll
        for (int e = 0; e < PER; ++e)
          id[k][e] = j0 + 32 * e < end ? a.table[static_cast<size_t>(p) * a.ld_table + j0 + 32 * e] : kNoEntry;
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        int32_t now = kNoEntry;
        int sum = 0;
        auto add = [&]() {
          if (now == kNoEntry || sum == 0) return;
          if (now >= 0 && now < a.pages)  // others are reported above
            atomicAdd(cluster.map_shared_rank(counter, now / a.per) + now % a.per, sum);
        };
#pragma unroll
        for (int k = 0; k < kForkRun; ++k) {
          if (id[k][e] == kNoEntry) continue;
          if (id[k][e] != now) {
            add();
            now = id[k][e];
            sum = 0;
          }
          sum += children[min(p0 + k, batch - 1)] - 1;
        }
        add();
      }
    }
  }
  cluster.sync();
  // a warp's run of this CTA's pages, in order
  const int run = ((mine + warps - 1) / warps + 31) / 32 * 32;
  const int i0 = min(warp * run, mine), i1 = min(i0 + run, mine);
  int gone = 0;
  for (int i = i0 + lane; i - lane < i1; i += 32 * kForkUnits) {
    int more[kForkUnits];
#pragma unroll
    for (int e = 0; e < kForkUnits; ++e) more[e] = i + 32 * e < i1 ? a.shares[page0 + i + 32 * e] : 0;
#pragma unroll
    for (int e = 0; e < kForkUnits; ++e) {
      const int at = i + 32 * e;
      bool is = false;
      if (at < i1) {
        const int left = max(more[e], 0) + counter[at];
        is = left == -1;
        if (more[e] < 0 || left < -1) record_error(SJ_DEV_BAD_INDEX);  // given back more often than it was held
        a.shares_out[page0 + at] = max(left, 0);
        counter[at] = is;
      }
      gone += __popc(__ballot_sync(0xffffffffu, is));
    }
  }
  if (lane == 0) s_warp[warp] = gone;
  __syncthreads();
  if (t == 0) {
    int sum = 0;
    for (int w = 0; w < warps; ++w) sum += s_warp[w];
    s_back = sum;
  }
  cluster.sync();
  int back = count - taken, all = 0;
  for (int k = 0; k < ctas; ++k) {
    const int n = *cluster.map_shared_rank(&s_back, k);
    if (k < cta) back += n;
    all += n;
  }
  for (int w = 0; w < warp; ++w) back += s_warp[w];
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const bool is = i < i1 && counter[i] != 0;
    const unsigned have = __ballot_sync(0xffffffffu, is);
    const int at = back + __popc(have & ((1u << lane) - 1));
    if (is) {
      if (at >= 0 && at < a.pages)
        a.stack_out[at] = page0 + i;
      else
        record_error(SJ_DEV_BAD_INDEX);
    }
    back += __popc(have);
  }
  if (cta == 0 && t == 0) {
    const int left = min(count - taken + all, a.pages);
    *a.count_out = status ? count : left;
    a.summary[0] = taken;
    a.summary[1] = all;
    a.summary[2] = status;
    a.summary[3] = status ? count : left;
  }
  cluster.sync();  // nobody's shared memory goes while another reads it
}

// ---------------------------------------------------------------- copy
struct PagedCopy {
  const int32_t* copies;
  __nv_bfloat16 *k, *v;
  int64_t layer_stride, page_stride, head_stride, token_stride;
  int pages, page, hk, parts, tokens_outside;
};

// A CTA takes kCopyThreads * kCopyPieces pieces of 16 bytes of one copy, of K or of V of one layer; a page's rows and
// heads go in the order in which they lie in memory.  All loads of a thread are in flight before its first store.  2003
// pages of 64 rows of 8 heads of 128: 159 us, 6.6 TB/s in and out (the measured copy rate); 13 half-filled pages of six
// layers 2.1.
template <int DIM>
__global__ void __launch_bounds__(kCopyThreads) paged_copy_kernel(const PagedCopy a) {
  pdl_wait();
  const int entry = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int from = a.copies[3 * entry], to = a.copies[3 * entry + 1], rows = a.copies[3 * entry + 2];
  if (from == -1) return;
  if (from < 0 || from >= a.pages || to < 0 || to >= a.pages || rows < 0 || rows > a.page) {
    if (threadIdx.x == 0) record_error(SJ_DEV_BAD_INDEX);
    return;
  }
  constexpr int PER = DIM / 8;  // pieces of a row of a head
  const int inner = a.tokens_outside ? a.hk : rows, lines = rows * a.hk;
  __nv_bfloat16* base = (blockIdx.y & 1 ? a.v : a.k) + static_cast<int64_t>(blockIdx.y >> 1) * a.layer_stride;
  const __nv_bfloat16* src = base + from * a.page_stride;
  __nv_bfloat16* dst = base + to * a.page_stride;
  uint4 x[kCopyPieces];
  int64_t at[kCopyPieces];
#pragma unroll
  for (int i = 0; i < kCopyPieces; ++i) {
    const int piece = (part * kCopyPieces + i) * kCopyThreads + static_cast<int>(threadIdx.x), line = piece / PER;
    at[i] = -1;
    if (line < lines) {
      const int outer = line / inner, in = line - outer * inner;
      const int64_t head = a.tokens_outside ? in : outer, row = a.tokens_outside ? outer : in;
      at[i] = head * a.head_stride + row * a.token_stride + piece % PER * 8;
      x[i] = *reinterpret_cast<const uint4*>(src + at[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kCopyPieces; ++i)
    if (at[i] >= 0) *reinterpret_cast<uint4*>(dst + at[i]) = x[i];
}

// ---------------------------------------------------------------- compact
struct Compact {
  const int32_t *cached, *table, *shares, *stack, *stack_count;
  int32_t *table_out, *shares_out, *stack_out, *moves, *summary;
  int batch, page, ld_table, pages, most;
};

// Every CTA reads the whole stack into a bit mask of the free pages with the numbers of pages in use before each word,
// and writes its share of the results: the i-th page in use from `used` on goes to the i-th free page below it.  One launch
// without a wait for other CTAs; bound by the shared-memory atomics of the mask (1024 requests on 183 thousand pages, half of
// them free, 25 us; 32 requests on a thousand 6.5).
__global__ void __launch_bounds__(kCompactThreads) paged_compact_kernel(const Compact a) {
  pdl_wait();
  extern __shared__ uint32_t bits[];                          // a bit for each page: free
  const int words = (a.pages + 31) / 32, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int* before = reinterpret_cast<int*>(bits + words);         // [words + 1] pages in use before each word
  __shared__ int s_warp[32], s_bad;
  const int count = *a.stack_count;
  bool bad = count < 0 || count > a.pages;
  for (int w = t; w < words; w += kCompactThreads) bits[w] = 0;
  if (t == 0) s_bad = 0;
  __syncthreads();
  for (int i = t; i < (bad ? 0 : count); i += kCompactThreads * kCompactIds) {
    int id[kCompactIds];
#pragma unroll
    for (int e = 0; e < kCompactIds; ++e) id[e] = i + e * kCompactThreads < count ? a.stack[i + e * kCompactThreads] : 0;
#pragma unroll
    for (int e = 0; e < kCompactIds; ++e) {
      if (i + e * kCompactThreads >= count) break;
      if (id[e] < 0 || id[e] >= a.pages)
        s_bad = 1;
      else
        atomicOr(&bits[id[e] >> 5], 1u << (id[e] & 31));
    }
  }
  __syncthreads();
  const int per = (words + kCompactThreads - 1) / kCompactThreads, w0 = min(t * per, words), w1 = min(w0 + per, words);
  auto in_word = [&](int w) { return min(32, a.pages - w * 32) - __popc(bits[w]); };
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += in_word(w);
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) s_warp[warp] = upto;
  __syncthreads();
  int base = upto - mine;
  for (int w = 0; w < warp; ++w) base += s_warp[w];
  for (int w = w0; w < w1; ++w) {
    before[w] = base;
    base += in_word(w);
  }
  int in_use = 0;
  for (int w = 0; w < 32; ++w) in_use += s_warp[w];
  bad |= s_bad != 0 || in_use != a.pages - count;  // twice on the stack
  __syncthreads();
  const int used = bad ? 0 : a.pages - count;
  auto is_free = [&](int p) { return (bits[p >> 5] >> (p & 31) & 1) != 0; };
  auto in_use_before = [&](int p) {  // p < pages
    return before[p >> 5] + (p & 31) - __popc(bits[p >> 5] & ((1u << (p & 31)) - 1));
  };
  const int kept = bad || used == a.pages ? used : in_use_before(used), moved = used - kept;
  const int status = bad ? kCompactBad : moved > a.most ? kCompactMovesOver : 0;
  auto target = [&](int p) {
    if (status || p < used) return p;
    const int r = in_use_before(p) - kept;  // the r-th hole: the last word with at most r holes before it
    int lo = 0, hi = (used + 31) / 32;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (mid * 32 - before[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    uint32_t holes = bits[lo];
    int skip = r - (lo * 32 - before[lo]), at = 0;  // the skip-th set bit: by halves of what is left of the word
#pragma unroll
    for (int half = 16; half > 0; half >>= 1) {
      const int below = __popc(holes & ((1u << half) - 1));
      if (skip >= below) {
        skip -= below;
        at += half;
        holes >>= half;
      }
    }
    return lo * 32 + at;
  };
  const int first = blockIdx.x * kCompactThreads + t, step = gridDim.x * kCompactThreads;
  const int chunks = (a.ld_table + kForkChunk - 1) / kForkChunk;
  for (int u = first >> 5; u < a.batch * chunks; u += step >> 5) {
    const int b = u % a.batch, j0 = u / a.batch * kForkChunk, n = a.cached[b];
    if (n < 0 || n > INT_MAX - a.page || (n + a.page - 1) / a.page > a.ld_table) {
      if (lane == 0) record_error(SJ_DEV_BAD_INDEX);
      continue;
    }
    const size_t row = static_cast<size_t>(b) * a.ld_table;
    const int end = min((n + a.page - 1) / a.page, j0 + kForkChunk);
    int id[kForkChunk / 32];
#pragma unroll
    for (int e = 0; e < kForkChunk / 32; ++e) id[e] = j0 + 32 * e + lane < end ? a.table[row + j0 + 32 * e + lane] : 0;
#pragma unroll
    for (int e = 0; e < kForkChunk / 32; ++e) {
      if (j0 + 32 * e + lane >= end) continue;
      const bool fine = id[e] >= 0 && id[e] < a.pages && (bad || !is_free(id[e]));
      if (!fine) record_error(SJ_DEV_BAD_INDEX);
      a.table_out[row + j0 + 32 * e + lane] = fine ? target(id[e]) : id[e];
    }
  }
  for (int p = first; p < a.pages; p += step) {
    if (status) {
      a.shares_out[p] = a.shares[p];
      continue;
    }
    if (!is_free(p)) {
      const int to = target(p);
      a.shares_out[to] = a.shares[p];
      if (to != p) {
        const int i = in_use_before(p) - kept;
        a.moves[3 * i] = p;
        a.moves[3 * i + 1] = to;
        a.moves[3 * i + 2] = a.page;
      }
    }
    if (p >= used) a.shares_out[p] = 0;
  }
  for (int i = (status ? 0 : moved) + first; i < a.most; i += step) {
    a.moves[3 * i] = a.moves[3 * i + 1] = -1;
    a.moves[3 * i + 2] = 0;
  }
  for (int i = first; i < min(max(count, 0), a.pages); i += step) a.stack_out[i] = status ? a.stack[i] : a.pages - 1 - i;
  if (first == 0) {
    a.summary[0] = status ? 0 : moved;
    a.summary[1] = used;
    a.summary[2] = status;
    a.summary[3] = count;
  }
}

}  // namespace sj

using namespace sj;

extern "C" int sj_paged_fork(const int32_t* parent, int batch, int page, const int32_t* cached,
                             const int32_t* block_table, int ld_table, const int32_t* shares,
                             const int32_t* free_pages, const int32_t* free_count, int pages, int32_t* cached_out,
                             int32_t* table_out, int32_t* shares_out, int32_t* free_out, int32_t* count_out,
                             int32_t* copies, int32_t* summary, void* stream) {
  if (batch <= 0 || batch > kShareMaxBatch || page <= 0 || page > (1 << 20) || ld_table <= 0 ||
      ld_table > INT_MAX / kShareMaxBatch * kForkChunk - kForkChunk || pages <= 0 || pages > kShareMaxPages)
    return fail(SJ_ERR_SHAPE, "sj_paged_fork: batch=%d (up to %d) page=%d ld_table=%d pages=%d (up to %d)", batch,
                kShareMaxBatch, page, ld_table, pages, kShareMaxPages);
  if (!parent || !cached || !block_table || !shares || !free_pages || !free_count || !cached_out || !table_out ||
      !shares_out || !free_out || !count_out || !copies || !summary)
    return fail(SJ_ERR_ARGUMENT, "sj_paged_fork: null operand");
  if (cached == cached_out || block_table == table_out || shares == shares_out || free_pages == free_out ||
      free_count == count_out)
    return fail(SJ_ERR_ARGUMENT, "sj_paged_fork: the new state needs buffers of its own");
  Fork a{parent, cached, block_table, shares, free_pages, free_count, cached_out, table_out, shares_out,
         free_out, count_out, copies, summary, batch, page, ld_table, pages, 0};
  constexpr int ctas = kForkCluster;
  a.per = (pages + ctas - 1) / ctas;
  const int smem = (5 * (batch + 1) + a.per) * static_cast<int>(sizeof(int));
  static KernelAttrOnce once;
  constexpr int most = (5 * (kShareMaxBatch + 1) + kShareMaxPages / kForkCluster) * static_cast<int>(sizeof(int));
  const int rc = ensure_max_smem(once, reinterpret_cast<const void*>(paged_fork_kernel), most,
                                 "sj_paged_fork: shared memory");
  if (rc != SJ_OK) return rc;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  // A unit is a chunk of a request's table.  Few of them leave most warps of 1024 threads with the barriers only (256 and 1024
  // threads: 32 requests, 32 units 8.8 and 11.1 us; 512 units 11.2 and 14.3), many need the warps (1024 units 16.5 and 15.1;
  // 1024 requests, 5120 units 40.9 and 22.0).
  const int64_t units = static_cast<int64_t>(batch) * ((ld_table + kForkChunk - 1) / kForkChunk);
  const int threads = units <= 512 ? 256 : kForkThreads;
  const int64_t writers = std::min<int64_t>((units * 32 - 1) / threads + 1, sm_count() / 2);
  cfg.gridDim = dim3(static_cast<unsigned>(ctas * (1 + (writers + ctas - 1) / ctas)));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = as_stream(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  void* args[] = {&a};
  cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(paged_fork_kernel), args);
  SJ_LAUNCH_CHECK("paged_fork");
  return SJ_OK;
}

extern "C" int sj_paged_copy(const int32_t* copies, int most, void* k_cache, void* v_cache, int layers,
                             int64_t layer_stride, int pages, int page, int64_t page_stride, int64_t head_stride,
                             int64_t token_stride, int hk, int head_dim, void* stream) {
  if (most < 0 || hk <= 0 || hk > 4096 || layers <= 0 || layers > 4096)
    return fail(SJ_ERR_SHAPE, "sj_paged_copy: most=%d hk=%d layers=%d (up to 4096)", most, hk, layers);
  const int rc = check_paged_cache("sj_paged_copy", k_cache, v_cache, pages, page, page_stride, head_stride,
                                   token_stride, hk, head_dim);
  if (rc != SJ_OK) return rc;
  if (layer_stride < 0 || layer_stride % 8 || layer_stride > (int64_t{1} << 62) / layers)
    return fail(SJ_ERR_ARGUMENT, "sj_paged_copy: a layer stride that is a multiple of 8");
  if (most == 0) return SJ_OK;
  if (!copies) return fail(SJ_ERR_ARGUMENT, "sj_paged_copy: null operand");
  const int64_t pieces = static_cast<int64_t>(page) * hk * (head_dim / 8);
  constexpr int each = kCopyThreads * kCopyPieces;
  const int64_t parts = (pieces + each - 1) / each;
  if (pieces > INT_MAX - each || parts * most > INT_MAX)
    return fail(SJ_ERR_SHAPE, "sj_paged_copy: most=%d page=%d hk=%d", most, page, hk);
  PagedCopy a{copies, static_cast<__nv_bfloat16*>(k_cache), static_cast<__nv_bfloat16*>(v_cache), layer_stride,
              page_stride, head_stride, token_stride, pages, page, hk, static_cast<int>(parts),
              token_stride > head_stride ? 1 : 0};
  launch(head_dim == 64 ? paged_copy_kernel<64> : paged_copy_kernel<128>,
         dim3(static_cast<unsigned>(parts * most), 2 * layers), kCopyThreads, 0, as_stream(stream), a);
  SJ_LAUNCH_CHECK("paged_copy");
  return SJ_OK;
}

extern "C" int sj_paged_compact(const int32_t* cached, int batch, int page, const int32_t* block_table, int ld_table,
                                const int32_t* shares, const int32_t* free_pages, const int32_t* free_count,
                                int pages, int32_t* table_out, int32_t* shares_out, int32_t* free_out, int32_t* moves,
                                int most, int32_t* summary, void* stream) {
  if (batch <= 0 || batch > kShareMaxBatch || page <= 0 || page > (1 << 20) || ld_table <= 0 ||
      ld_table > INT_MAX / kShareMaxBatch * kForkChunk - kForkChunk || pages <= 0 || pages > kShareMaxPages || most < 0 || most > INT_MAX / 3)
    return fail(SJ_ERR_SHAPE, "sj_paged_compact: batch=%d (up to %d) page=%d ld_table=%d pages=%d (up to %d) most=%d",
                batch, kShareMaxBatch, page, ld_table, pages, kShareMaxPages, most);
  if (!cached || !block_table || !shares || !free_pages || !free_count || !table_out || !shares_out || !free_out ||
      !summary || (most > 0 && !moves))
    return fail(SJ_ERR_ARGUMENT, "sj_paged_compact: null operand");
  if (block_table == table_out || shares == shares_out || free_pages == free_out)
    return fail(SJ_ERR_ARGUMENT, "sj_paged_compact: the new state needs buffers of its own");
  const int words = (pages + 31) / 32;
  static KernelAttrOnce once;
  const int rc = ensure_max_smem(once, reinterpret_cast<const void*>(paged_compact_kernel),
                                 (kShareMaxPages / 32 * 2 + 1) * static_cast<int>(sizeof(int)),
                                 "sj_paged_compact: shared memory");
  if (rc != SJ_OK) return rc;
  const Compact a{cached, block_table, shares, free_pages, free_count, table_out, shares_out, free_out,
                  moves, summary, batch, page, ld_table, pages, most};
  const int64_t units = static_cast<int64_t>(batch) * ((ld_table + kForkChunk - 1) / kForkChunk);
  const int64_t work = std::max<int64_t>(units * 32, std::max(pages, most));
  const int grid = static_cast<int>(std::min<int64_t>((work + kCompactThreads - 1) / kCompactThreads, sm_count()));
  launch(paged_compact_kernel, grid, kCompactThreads, (2 * words + 1) * sizeof(int), as_stream(stream), a);
  SJ_LAUNCH_CHECK("paged_compact");
  return SJ_OK;
}
