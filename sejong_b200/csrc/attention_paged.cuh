// The arguments of attn_paged_kernel, and what the kernels of sj_attn_paged_shared hand to one another through the
// workspace.
#pragma once
#include "common.cuh"

namespace sj {

// Lets the next kernel's CTAs come in beside this one; they wait for its end all the same (pdl_wait).  For a kernel of one
// CTA: 1 us less of 76 behind shared_spans_kernel, but 4 us more behind the kernels after it, whose room it takes.
SJ_DEVICE void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct PagedAttention {
  const __nv_bfloat16 *q, *k, *v;
  const int32_t *table, *request, *position;
  __nv_bfloat16* o;
  float* lse;
  int* counters;   // parts written of each first group of a unit, of other groups, groups of a unit: a CTA one of each
  float* partial;  // two slots per CTA
  int64_t page_stride, head_stride, token_stride;
  int ldq, ldo, pages, page, ld_table, requests, rows, hq, hk, window;
  // of rows that are left apart though a call names groups of them: looked at for the report only, else none
  const int32_t* group;
  int groups;
};

constexpr int kSharedKeys = 128;     // keys of a tile
constexpr int kSharedQueries = 128;  // queries of a tile: whole rows of hq / hk heads that share a KV head

// A group: its rows, the keys [p0, p1) that every live one of them sees, and its first item.  The queries of a KV head
// lie in `tiles` tiles.  An item is a tile of keys for two tiles of queries, or two tiles of keys for the one tile that
// may be left: the same work either way.  A head's items are those of its pairs of tiles, a chunk of the keys at a time,
// so that CTAs which run side by side read the same keys, then those of the tile that is left.
struct SharedGroup {
  unsigned long long base;
  size_t main;  // the first query of the group's parts that begin a block (chunk and pair): [chunks][rows][hq]
  int blocks;   // its first block: [kv head][chunk][unit], a unit being a pair of tiles or the tile that is left
  int first, rows, request, p0, p1, tiles, keys, chunks;  // keys: tiles of them
  SJ_DEVICE int halves() const { return (keys + 1) / 2; }
  SJ_DEVICE unsigned long long head_items() const {
    return static_cast<unsigned long long>(tiles / 2) * keys + (tiles & 1) * halves();
  }
  SJ_DEVICE int chunk(int c) const { return static_cast<int>(static_cast<long long>(keys) * c / chunks); }  // its first tile
};

// A row: keys [lo, p0) and [p1, n) are its own, group -1: all of [lo, n).
struct SharedRow {
  int lo, n, p0, p1, group;
};

// Whether group t of `groups` (first row, request, tokens) is in order and in range; `most`: the tokens that a table holds.
__host__ __device__ inline bool shared_group_fine(const int32_t* group, int t, int groups, int rows, int requests,
                                                  int64_t most) {
  const int at = group[3 * t], b = group[3 * t + 1], n = group[3 * t + 2], next = t + 1 < groups ? group[3 * t + 3] : rows;
  const bool ordered = at >= 0 && next <= rows && (at < next || (at == rows && next == rows));
  return ordered && b >= 0 && b < requests && n >= 0 && n <= most;
}

// Whether a block's first and last CTA can be those that attn_shared_kernel wrote.  Where a wait of it gave up it left blocks
// out, and a workspace may hold anything there.
__host__ __device__ inline bool shared_span_fine(int2 span, int ctas) {
  return span.x >= 0 && span.x <= span.y && span.y < ctas;
}

// A softmax's part: maximum (of log2), sum and outputs of each query.
struct SharedParts {
  float *m, *l, *o;  // o: [queries][dim]
};

struct SharedSpans {
  unsigned long long* total;  // items of all groups
  SharedGroup* groups;
  SharedRow* rows;
  int2* blocks;       // the first and the last CTA of each block
  SharedParts own;    // [rows, hq]: a row's own keys
  SharedParts main;   // the parts that begin a block
  SharedParts slots;  // [ctas][2 * kSharedQueries]: the part that goes on with a block, of each CTA
  size_t main_queries;
  int ctas;  // of attn_shared_kernel
};

// Checks the arguments of sj_attn_paged, or of a call (`who`) that has the same ones and a workspace of `need` bytes
// that begins with that of sj_attn_paged.
int paged_attention_args(const char* who, PagedAttention& a, const void* q, int ldq, const void* k_cache,
                         const void* v_cache, int pages, int page, int64_t page_stride, int64_t head_stride,
                         int64_t token_stride, const int32_t* block_table, int ld_table, int requests,
                         const int32_t* request, const int32_t* position, int rows, int hq, int hk, int head_dim,
                         int window, void* o, int ldo, float* lse, void* workspace, size_t workspace_bytes,
                         size_t need);
// Launches attn_paged_kernel: all of a row's keys, or (spans not null) its own ones, as a part.
int attn_paged_rows(const PagedAttention& a, const SharedSpans* spans, int head_dim, cudaStream_t stream);

}  // namespace sj
