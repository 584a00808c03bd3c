// What the kernels over a paged key-value cache share: addressing and argument checks.
#pragma once
#include "common.cuh"

namespace {

constexpr uint32_t kNoRow = 0xffffffffu;

// Pools [num_pages, kv_heads, page_size, head_dim] and the table that assigns pages to rows.
struct PagedLayout {
  const int* table;     // [batch, max_pages]
  const int* lengths;   // [batch]
  int kv_heads, head_dim, num_pages, page_size, max_pages;
  int page_shift;       // log2(page_size), or -1
  int capacity;         // max_pages * page_size
  int* flag;            // the context's error word
  uint64_t pool_bytes;  // of each pool
};

// Slots of row b, clamped to [0, capacity]; a length outside that is reported.
__device__ __forceinline__ int paged_length(const PagedLayout& g, int b) {
  const int n = __ldg(g.lengths + b);
  if (n < 0 || n > g.capacity) {
    atomicOr(g.flag, kBadLength);
    return n < 0 ? 0 : g.capacity;
  }
  return n;
}

// Index, in rows of head_dim values, of slot j of row b and head h in both pools; kNoRow (and
// a report, unless the caller makes it) when the table names no page of the pool for it.  The number of
// rows of a pool is below 2^31 (checked on the host), its byte offsets are not.
template <bool REPORT = true>
__device__ __forceinline__ uint32_t paged_row(const PagedLayout& g, int b, int h, int j) {
  const int pi = g.page_shift >= 0 ? j >> g.page_shift : j / g.page_size;
  const int page = __ldg(g.table + (size_t)b * g.max_pages + pi);
  if ((unsigned)page >= (unsigned)g.num_pages) {
    if (REPORT) atomicOr(g.flag, kBadPage);
    return kNoRow;
  }
  return (uint32_t)((page * g.kv_heads + h) * g.page_size + (j - pi * g.page_size));
}

// Checks the dimensions, the pools, the table and the lengths of a call.
int paged_layout(tfjs_cuda_ctx* ctx, const tfjs_cuda_paged_params* p, const char* who,
                 int32_t k_cache_id, int32_t v_cache_id, int32_t table_id, int32_t lengths_id,
                 PagedLayout* g, Buffer** kc, Buffer** vc) {
  if (!p) return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: null parameters", who);
  if (p->batch <= 0 || p->kv_heads <= 0 || p->head_dim <= 0 || p->num_pages <= 0 ||
      p->page_size <= 0 || p->max_pages <= 0)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: dimensions must be positive", who);
  const uint64_t page_heads = (uint64_t)p->num_pages * p->kv_heads;
  const uint64_t rows = page_heads < (1ull << 31) ? page_heads * p->page_size : ~0ull;
  const uint64_t cap = (uint64_t)p->max_pages * p->page_size;
  if (rows > 0x7fffffffull || cap > 0x3fffffffull || (uint64_t)p->batch * p->kv_heads > 0xffffffull || p->head_dim > 256)
    return ctx_fail(ctx, TFJS_CUDA_UNSUPPORTED,
                    "%s: heads of up to 256 values, pools below 2^31 rows, rows below 2^30 slots "
                    "and below 2^24 rows times heads", who);
  if (k_cache_id == v_cache_id)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: one pool cannot hold keys and values", who);
  Buffer *table, *lengths;
  int rc;
  const uint64_t pool = rows * (uint64_t)p->head_dim * 4;
  if ((rc = ctx_get(ctx, k_cache_id, pool, who, kc))) return rc;
  if ((rc = ctx_get(ctx, v_cache_id, pool, who, vc))) return rc;
  if ((rc = ctx_get(ctx, table_id, (uint64_t)p->batch * p->max_pages * 4, who, &table))) return rc;
  if ((rc = ctx_get(ctx, lengths_id, (uint64_t)p->batch * 4, who, &lengths))) return rc;
  g->pool_bytes = pool;
  g->table = (const int*)table->ptr;
  g->lengths = (const int*)lengths->ptr;
  g->kv_heads = p->kv_heads;
  g->head_dim = p->head_dim;
  g->num_pages = p->num_pages;
  g->page_size = p->page_size;
  g->max_pages = p->max_pages;
  g->capacity = (int)cap;
  g->page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (p->page_size == (1 << s)) g->page_shift = s;
  g->flag = ctx->d_flag;
  return TFJS_CUDA_OK;
}

}  // namespace
