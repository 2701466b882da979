// Batched decoding on a paged key-value cache: the step's block tables and slot maps, the rotated
// queries, and the keys and values written to their slots (attention_paged.cu reads them).
//
//   paged_plan_kernel     lengths -> new block-table entries, row maps, new lengths (idempotent)
//   paged_commit_kernel   makes a planned step final and takes back the pages of finished requests
//   rope_scaled_kernel    (cos, sin) tables of scaled rotary positions, angles in f64
//   paged_append_kernel   rotary positions of q and k, k and v into their cache slots
//
// A cache of one layer is `pages` pages of `page` slots; slot s is row s % page of page s / page.
// Element (page p, head h, row r, dim d) lies at p * page_stride + h * head_stride + r *
// token_stride + d of the K and of the V buffer, so both storage orders (heads outermost inside a
// page, or tokens outermost) and K and V halves of one buffer are covered.
#include <algorithm>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "internal.h"

namespace sj {

namespace {
constexpr int kPlanMaxBatch = 4096, kPlanMaxRows = (1 << 19) - 1;  // their product fits 31 bits, so sums do
constexpr int kCommitIds = 4;
constexpr int kPlanRowsOver = 1, kPlanNoPages = 2, kPlanTableNarrow = 3, kPlanBadCount = 4;
}  // namespace

// ---------------------------------------------------------------- plan
// Exclusive prefix sums of a[i] and b[i], i < n <= 4 * blockDim.x, into shared sa[0..n], sb[0..n].
template <typename F>
SJ_DEVICE void block_scan2(int n, int* sa, int* sb, F value) {
  __shared__ int wa[32], wb[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
  int a[4], b[4], ta = 0, tb = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = b[i] = 0;
    if (4 * t + i < n) value(4 * t + i, a[i], b[i]);
    ta += a[i];
    tb += b[i];
  }
  int ia = ta, ib = tb;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) {
      ia += ua;
      ib += ub;
    }
  }
  if (lane == 31) {
    wa[warp] = ia;
    wb[warp] = ib;
  }
  __syncthreads();
  int ba = ia - ta, bb = ib - tb;
  for (int w = 0; w < warps; ++w)
    if (w < warp) {
      ba += wa[w];
      bb += wb[w];
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (4 * t + i < n) {
      sa[4 * t + i] = ba;
      sb[4 * t + i] = bb;
      if (4 * t + i == n - 1) {
        sa[n] = ba + a[i];
        sb[n] = bb + b[i];
      }
    }
    ba += a[i];
    bb += b[i];
  }
  __syncthreads();
}

// The b with start[b] <= i < start[b + 1] (start[0] = 0 <= i < start[n]).
SJ_DEVICE int owner_of(const int* start, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Request b holds H_b = ceil(cached_b / page) pages and needs N_b = ceil((cached_b + added_b) / page);
// the i-th new page, requests in order, is the i-th from the top of the free stack.  Every CTA scans
// the batch for itself (a few KB out of L2) and writes its share of the rows and new table entries,
// so one launch does it all without a grid-wide wait.  Bound by latency: a launch, three dependent look-ups and the
// scan (64 requests 4.3 us, 1021 requests with 50000 rows 5.3; graph replays).
__global__ void __launch_bounds__(1024) paged_plan_kernel(const int32_t* cached, const int32_t* added, int batch,
                                                          int page, const int32_t* free_pages,
                                                          const int32_t* free_count, int32_t* table, int ld_table,
                                                          int32_t* lengths, int32_t* request, int32_t* position,
                                                          int32_t* slot, int rows_cap, int32_t* summary) {
  pdl_wait();
  __shared__ int row_start[kPlanMaxBatch + 1], page_start[kPlanMaxBatch + 1];
  __shared__ int bad, narrow, over;
  if (threadIdx.x == 0) bad = narrow = over = 0;
  __syncthreads();
  const int count = max(*free_count, 0);
  block_scan2(batch, row_start, page_start, [&](int b, int& rows, int& pages) {
    const int c = cached[b], n = added[b];
    if (c < 0 || n < 0 || c > INT_MAX - page - n) {
      bad = 1;
    } else if (n > rows_cap) {
      over = 1;
    } else {
      const int need = (c + n + page - 1) / page;
      rows = n;
      pages = need - (c + page - 1) / page;
      if (need > ld_table) narrow = 1;
    }
  });
  const int rows = row_start[batch], taken = page_start[batch];
  const int status = bad                        ? kPlanBadCount
                     : (over || rows > rows_cap) ? kPlanRowsOver
                     : narrow                   ? kPlanTableNarrow
                     : taken > count            ? kPlanNoPages
                                                : 0;
  const int first = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  for (int b = first; b < batch; b += step) lengths[b] = cached[b] + (status ? 0 : added[b]);
  if (first == 0) {
    summary[0] = status ? 0 : rows;
    summary[1] = status ? 0 : taken;
    summary[2] = status;
    summary[3] = status ? count : count - taken;
  }
  for (int r = first; r < rows_cap; r += step) {
    int b = -1, pos = -1, s = -1;
    if (!status && r < rows) {
      b = owner_of(row_start, batch, r);
      const int c = cached[b], held = (c + page - 1) / page;
      pos = c + (r - row_start[b]);
      const int at = pos / page;
      const int id = at < held ? table[static_cast<size_t>(b) * ld_table + at]
                               : free_pages[count - 1 - (page_start[b] + at - held)];
      if (id >= 0 && id <= (INT_MAX - page) / page)
        s = id * page + pos % page;
      else
        record_error(SJ_DEV_BAD_INDEX);
    }
    request[r] = b;
    position[r] = pos;
    slot[r] = s;
  }
  if (status) return;
  for (int i = first; i < taken; i += step) {
    const int b = owner_of(page_start, batch, i);
    const int held = (cached[b] + page - 1) / page;
    table[static_cast<size_t>(b) * ld_table + held + i - page_start[b]] = free_pages[count - 1 - i];
  }
}

// One CTA, so that what it refuses is known before anything is written: it looks at the returned pages twice.  Bound by
// latency: 64 requests of which none ends 2.5 us (graph replays), 652 pages back 4.9, 12349 pages of 1021 requests 25,
// 269844 pages 409; with a search of the requests for each page 5.4, 58 and 1277.
__global__ void __launch_bounds__(1024) paged_commit_kernel(int32_t* cached, int32_t* lengths, const int32_t* release,
                                                            int batch, int page, const int32_t* table, int ld_table,
                                                            int32_t* free_pages, int32_t* free_count, int pages,
                                                            int32_t* summary) {
  pdl_wait();
  __shared__ int page_start[kPlanMaxBatch + 1], unused[kPlanMaxBatch + 1];
  block_scan2(batch, page_start, unused, [&](int b, int& n, int&) {
    if (release && release[b]) n = min((max(lengths[b], 0) + page - 1) / page, ld_table);
  });
  const int top = *free_count - summary[1], back = page_start[batch];
  bool refused = top < 0 || back < 0 || back > pages - top;
  // The pages to return, a run of them for each warp, kCommitIds of a lane at a time: side by side in the table, so
  // that a request is looked for where a lane leaves the last one's pages only.
  const int run = (back / static_cast<int>(blockDim.x) + 1) * 32, i0 = (threadIdx.x >> 5) * run;
  const int i1 = refused ? 0 : min(i0 + run, back);
  auto each_page = [&](auto use) {
    int first = 0, past = 0;  // of the pages of the request at `own`
    const int32_t* own = table;
    for (int i = i0 + static_cast<int>(threadIdx.x & 31); i < i1; i += 32 * kCommitIds) {
      int id[kCommitIds];
#pragma unroll
      for (int e = 0; e < kCommitIds; ++e) {
        const int at = min(i + e * 32, i1 - 1);
        if (at >= past) {
          const int b = owner_of(page_start, batch, at);
          own = table + static_cast<size_t>(b) * ld_table;
          first = page_start[b];
          past = page_start[b + 1];
        }
        id[e] = own[at - first];
      }
#pragma unroll
      for (int e = 0; e < kCommitIds; ++e)
        if (i + e * 32 < i1) use(i + e * 32, id[e]);
    }
  };
  each_page([&](int, int id) { refused |= id < 0 || id >= pages; });
  if (__syncthreads_or(refused)) {  // nothing is written yet
    if (threadIdx.x == 0) record_error(SJ_DEV_BAD_INDEX);
    return;
  }
  each_page([&](int i, int id) { free_pages[top + i] = id; });
  for (int b = threadIdx.x; b < batch; b += blockDim.x) {
    const bool gone = release && release[b];
    if (gone) lengths[b] = 0;
    cached[b] = gone ? 0 : lengths[b];
  }
  if (threadIdx.x == 0) {
    *free_count = top + back;
    summary[0] = summary[1] = 0;
  }
}

// ---------------------------------------------------------------- scaled rotary tables
// Angles in f64: at position 131071 an f32 product p * freq is off by up to 2^-24 p = 0.008 rad, more
// than the bf16 it rotates can hide.
__global__ void rope_scaled_kernel(float* table, int t, int half, int offset, double theta, int scaling, double factor,
                                   double original, double fast, double slow) {
  pdl_wait();
  const size_t n = static_cast<size_t>(t) * half;
  const size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int p = static_cast<int>(i / half), k = static_cast<int>(i % half);
  double base = theta, amplitude = 1.0;
  if (scaling == SJ_ROPE_BASE && half > 1) base = theta * pow(factor, static_cast<double>(half) / (half - 1));
  double freq = pow(base, -static_cast<double>(k) / half);
  if (scaling == SJ_ROPE_LINEAR) freq /= factor;
  if (scaling == SJ_ROPE_RAMP) {
    const double turns = original * freq / 6.283185307179586476925286766559;
    const double keep = fmin(fmax((turns - slow) / (fast - slow), 0.0), 1.0);
    freq = freq * keep + freq / factor * (1.0 - keep);
    amplitude = 0.1 * log(factor) + 1.0;
  }
  double s, c;
  sincos(static_cast<double>(p + offset) * freq, &s, &c);
  table[2 * i] = static_cast<float>(c * amplitude);
  table[2 * i + 1] = static_cast<float>(s * amplitude);
}

// ---------------------------------------------------------------- append
constexpr int kAppendThreads = 128, kAppendHeads = 4, kAppendCtas = 8;

// Where keys and values go.
struct PagedWrite {
  __nv_bfloat16 *k, *v;
  int pages, page;
  int64_t page_stride, head_stride, token_stride;
};

SJ_DEVICE void rotate8(uint4& x, uint4& y, const float4* cs, bool half) {
  // interleaved: x and y are 16 consecutive elements, pairs (2i, 2i + 1); half: x holds the first
  // elements of eight pairs and y the second.  cs: the eight pairs' (cos, sin).
  uint32_t* a = &x.x;
  uint32_t* b = &y.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 w = cs[i];  // (cos, sin) of pairs 2i and 2i + 1
    if (half) {
      const float2 u = unpack_bf16x2(a[i]), v = unpack_bf16x2(b[i]);
      a[i] = pack_bf16x2(u.x * w.x - v.x * w.y, u.y * w.z - v.y * w.w);
      b[i] = pack_bf16x2(u.x * w.y + v.x * w.x, u.y * w.w + v.y * w.z);
    } else {
      uint32_t* p = i < 2 ? a + 2 * i : b + 2 * (i - 2);
      const float2 u = unpack_bf16x2(p[0]), v = unpack_bf16x2(p[1]);
      p[0] = pack_bf16x2(u.x * w.x - u.y * w.y, u.x * w.y + u.y * w.x);
      p[1] = pack_bf16x2(v.x * w.z - v.y * w.w, v.x * w.w + v.y * w.z);
    }
  }
}

// A warp for a row.  A lane takes 16 elements of a head (in the half layout the eight first and the eight second
// elements of eight pairs) of every 32 / (DIM / 16)-th head, so that it needs one piece of the row's angles
// for all of them, and has the loads of four heads in flight: two 16-byte loads, the f32 rotation, two 16-byte
// stores each.  Bound by the bytes of q, k and v, in and out: 32003 rows of 16 / 2 heads of 128 (64 rotated) 54.6 us,
// 6.2 TB/s (94% of the measured copy rate), a step of 64 rows 2.8.  A thread for 16 elements of one head, with its
// own look-ups, took 81; two heads in flight, 57; five CTAs an SM instead of eight, 64.
template <int DIM>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) paged_append_kernel(const __nv_bfloat16* qkv, int ld,
                                                                      const int32_t* position, const int32_t* slot,
                                                                      int rows, int hq, int hk, const float* table,
                                                                      int table_len, int rot, int half,
                                                                      __nv_bfloat16* q, int ldq, PagedWrite to) {
  pdl_wait();
  constexpr int LANES = DIM / 16, STEP = 32 / LANES;  // lanes of a head; heads side by side
  const int r = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= rows) return;
  const int c = lane % LANES, h0 = lane / LANES;
  const int s = slot[r], p = position[r];
  bool live = s != -1;
  if (live && (s < 0 || s >= to.pages * to.page || (rot > 0 && (p < 0 || p >= table_len)))) {
    if (lane == 0) record_error(SJ_DEV_BAD_INDEX);
    live = false;
  }
  const bool turns = live && c < rot / 16;
  float4 cs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    cs[i] = turns ? reinterpret_cast<const float4*>(table + static_cast<size_t>(p) * rot + c * 16)[i]
                  : make_float4(1.f, 0.f, 1.f, 0.f);
  const int page = live ? s / to.page : 0;
  const int64_t at = page * to.page_stride + (s - page * to.page) * to.token_stride;
  const __nv_bfloat16* src = qkv + static_cast<size_t>(r) * ld;
  const int heads = hq + 2 * hk, last = live ? heads : hq;
  // the half layout's pairs lie apart only where they are rotated: keys and queries
  const int first = c * 16, first_half = c * 8, second_half = first_half + rot / 2;
  for (int h = h0; h < last; h += kAppendHeads * STEP) {
    uint4 x[kAppendHeads], y[kAppendHeads];
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i) {
      const int head = h + i * STEP;
      const bool apart = half && turns && head < hq + hk;
      x[i] = y[i] = make_uint4(0, 0, 0, 0);
      if (live && head < last) {
        x[i] = *reinterpret_cast<const uint4*>(src + head * DIM + (apart ? first_half : first));
        y[i] = *reinterpret_cast<const uint4*>(src + head * DIM + (apart ? second_half : first + 8));
      }
    }
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i) {
      const int head = h + i * STEP;
      if (head >= last) continue;
      const bool turn = turns && head < hq + hk, apart = half && turn;
      if (turn) rotate8(x[i], y[i], cs, half != 0);
      __nv_bfloat16* dst = head < hq        ? q + static_cast<size_t>(r) * ldq + head * DIM
                           : head < hq + hk ? to.k + at + (head - hq) * to.head_stride
                                            : to.v + at + (head - hq - hk) * to.head_stride;
      *reinterpret_cast<uint4*>(dst + (apart ? first_half : first)) = x[i];
      *reinterpret_cast<uint4*>(dst + (apart ? second_half : first + 8)) = y[i];
    }
  }
}

// ---------------------------------------------------------------- host
int check_paged_cache(const char* who, const void* k, const void* v, int pages, int page, int64_t page_stride,
                int64_t head_stride, int64_t token_stride, int hk, int head_dim) {
  if (head_dim != 64 && head_dim != 128)
    return fail(SJ_ERR_UNSUPPORTED, "%s: head_dim %d (this build: 64 or 128)", who, head_dim);
  if (pages <= 0 || page <= 0 || static_cast<int64_t>(pages) * page > INT_MAX)
    return fail(SJ_ERR_SHAPE, "%s: pages=%d page=%d (below 2^31 slots)", who, pages, page);
  if (!k || !v || !aligned16(k) || !aligned16(v) || page_stride < 0 || head_stride < 0 || token_stride < 0 ||
      (page_stride | head_stride | token_stride) % 8)
    return fail(SJ_ERR_ARGUMENT, "%s: the cache takes 16-byte aligned buffers and strides that are multiples of 8",
                who);
  const int64_t limit = int64_t{1} << 35;
  if (page_stride > limit / pages || head_stride > limit / hk || token_stride > limit / page ||
      (pages - 1) * page_stride + (hk - 1) * head_stride + (page - 1) * token_stride + head_dim > limit)
    return fail(SJ_ERR_SHAPE, "%s: a cache buffer of more than 64 GiB", who);
  return SJ_OK;
}
}  // namespace sj

using namespace sj;

extern "C" int sj_paged_plan(const int32_t* cached, const int32_t* added, int batch, int page,
                             const int32_t* free_pages, const int32_t* free_count, int32_t* block_table, int ld_table,
                             int32_t* lengths, int32_t* request, int32_t* position, int32_t* slot, int rows,
                             int32_t* summary, void* stream) {
  if (batch <= 0 || batch > kPlanMaxBatch || page <= 0 || page > (1 << 20) || ld_table <= 0 || rows < 0 ||
      rows > kPlanMaxRows)
    return fail(SJ_ERR_SHAPE, "sj_paged_plan: batch=%d (up to %d) page=%d ld_table=%d rows=%d (up to %d)", batch,
                kPlanMaxBatch, page, ld_table, rows, kPlanMaxRows);
  if (!cached || !added || !free_pages || !free_count || !block_table || !lengths || !summary ||
      (rows > 0 && (!request || !position || !slot)))
    return fail(SJ_ERR_ARGUMENT, "sj_paged_plan: null operand");
  const int threads = batch <= 1024 ? 256 : 1024;
  const int grid = std::max(1, std::min((rows + threads - 1) / threads, 2 * sm_count()));
  launch(paged_plan_kernel, grid, threads, 0, as_stream(stream), cached, added, batch, page, free_pages, free_count,
         block_table, ld_table, lengths, request, position, slot, rows, summary);
  SJ_LAUNCH_CHECK("paged_plan");
  return SJ_OK;
}

extern "C" int sj_paged_commit(int32_t* cached, int32_t* lengths, const int32_t* release, int batch, int page,
                               const int32_t* block_table, int ld_table, int32_t* free_pages, int32_t* free_count,
                               int pages, int32_t* summary, void* stream) {
  if (batch <= 0 || batch > kPlanMaxBatch || page <= 0 || page > (1 << 20) || ld_table <= 0 || pages <= 0)
    return fail(SJ_ERR_SHAPE, "sj_paged_commit: batch=%d (up to %d) page=%d ld_table=%d pages=%d", batch,
                kPlanMaxBatch, page, ld_table, pages);
  if (!cached || !lengths || !block_table || !free_pages || !free_count || !summary)
    return fail(SJ_ERR_ARGUMENT, "sj_paged_commit: null operand");
  launch(paged_commit_kernel, 1, batch <= 1024 ? 256 : 1024, 0, as_stream(stream), cached, lengths, release, batch,
         page, block_table, ld_table, free_pages, free_count, pages, summary);
  SJ_LAUNCH_CHECK("paged_commit");
  return SJ_OK;
}

extern "C" int sj_rope_table_scaled(float* table, int t, int rope_dim, int offset, float theta, int scaling,
                                    float factor, int original, float fast, float slow, void* stream) {
  if (t <= 0 || rope_dim <= 0 || rope_dim % 2 || offset < 0 || offset > INT_MAX - t)
    return fail(SJ_ERR_SHAPE, "sj_rope_table_scaled: t=%d rope_dim=%d offset=%d", t, rope_dim, offset);
  if (!table || !(theta > 0.f) || scaling < SJ_ROPE_PLAIN || scaling > SJ_ROPE_RAMP)
    return fail(SJ_ERR_ARGUMENT, "sj_rope_table_scaled: null table, theta %g or scaling %d", theta, scaling);
  if (scaling != SJ_ROPE_PLAIN && !(factor >= 1.f))
    return fail(SJ_ERR_ARGUMENT, "sj_rope_table_scaled: factor %g (at least 1)", factor);
  if (scaling == SJ_ROPE_RAMP && (original <= 0 || !(fast > slow)))
    return fail(SJ_ERR_ARGUMENT, "sj_rope_table_scaled: original=%d fast=%g slow=%g", original, fast, slow);
  const size_t n = static_cast<size_t>(t) * (rope_dim / 2);
  if ((n + 255) / 256 > INT_MAX) return fail(SJ_ERR_SHAPE, "sj_rope_table_scaled: t=%d rope_dim=%d", t, rope_dim);
  launch(rope_scaled_kernel, static_cast<unsigned>((n + 255) / 256), 256, 0, as_stream(stream), table, t, rope_dim / 2,
         offset, theta, scaling, factor, original, fast, slow);
  SJ_LAUNCH_CHECK("rope_table_scaled");
  return SJ_OK;
}

extern "C" int sj_paged_append(const void* qkv, int ld, const int32_t* position, const int32_t* slot, int rows, int hq,
                               int hk, int head_dim, const float* rope_table, int rope_len, int rope_dim, int half,
                               void* q, int ldq, void* k_cache, void* v_cache, int pages, int page,
                               int64_t page_stride, int64_t head_stride, int64_t token_stride, void* stream) {
  if (rows < 0 || hq < 0 || hk <= 0 || hq > 4096 || hk > 4096)
    return fail(SJ_ERR_SHAPE, "sj_paged_append: rows=%d hq=%d hk=%d", rows, hq, hk);
  const int rc = check_paged_cache("sj_paged_append", k_cache, v_cache, pages, page, page_stride, head_stride,
                                   token_stride, hk, head_dim);
  if (rc != SJ_OK) return rc;
  if (rope_dim < 0 || rope_dim > head_dim || rope_dim % 16 || (rope_dim > 0 && rope_len <= 0) ||
      ld < (hq + 2 * hk) * head_dim || ldq < hq * head_dim)
    return fail(SJ_ERR_SHAPE, "sj_paged_append: rope_dim=%d (a multiple of 16) rope_len=%d ld=%d ldq=%d", rope_dim,
                rope_len, ld, ldq);
  if (rows == 0) return SJ_OK;
  if (!qkv || !position || !slot || (hq > 0 && !q) || (rope_dim > 0 && !rope_table) || !aligned16(qkv) ||
      !aligned16(q) || !aligned16(rope_table) || ld % 8 || ldq % 8)
    return fail(SJ_ERR_ARGUMENT, "sj_paged_append: null or unaligned operand, or a row stride not a multiple of 8");
  const PagedWrite to{static_cast<__nv_bfloat16*>(k_cache), static_cast<__nv_bfloat16*>(v_cache), pages, page,
                      page_stride, head_stride, token_stride};
  constexpr int per = kAppendThreads / 32;
  launch(head_dim == 64 ? paged_append_kernel<64> : paged_append_kernel<128>, (rows - 1) / per + 1, kAppendThreads, 0,
         as_stream(stream), static_cast<const __nv_bfloat16*>(qkv), ld, position, slot, rows, hq, hk, rope_table,
         rope_len, rope_dim, half, static_cast<__nv_bfloat16*>(q), ldq, to);
  SJ_LAUNCH_CHECK("paged_append");
  return SJ_OK;
}
