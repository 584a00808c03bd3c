// Writing to a paged key-value cache and keeping it bounded: appending new tokens, and
// eviction by accumulated attention weight.  Both move rows of head_dim values and compute
// nothing, so bytes bound them: a row is read once and written once.  (8 prompts of up to 2048
// tokens, 8 heads of 64: 13 us for 71 MB.)
#include "paged.cuh"

namespace {

// One row of head_dim values of both pools, copied by a warp; V values a lane at a time.
template <int V>
__device__ __forceinline__ void copy_row(float* k_cache, float* v_cache, uint64_t src, uint64_t dst, int dim, int lane) {
  for (int d = lane * V; d < dim; d += 32 * V) {
    if (V == 4) {
      const float4 x = *reinterpret_cast<const float4*>(k_cache + src + d);
      const float4 y = *reinterpret_cast<const float4*>(v_cache + src + d);
      *reinterpret_cast<float4*>(k_cache + dst + d) = x;
      *reinterpret_cast<float4*>(v_cache + dst + d) = y;
    } else {
      const float x = k_cache[src + d], y = v_cache[src + d];
      k_cache[dst + d] = x;
      v_cache[dst + d] = y;
    }
  }
}

// ---- append ------------------------------------------------------------------------------
// k and v are [batch, kv_heads, tokens, head_dim]; the tokens of one row and head are
// contiguous at the source, and in runs of a page's places at the destination.  V values at a
// time: 4 where head_dim and the addresses allow 16-byte accesses, else 1.
template <int V>
__global__ void __launch_bounds__(256)
paged_append_kernel(const PagedLayout g, const float* __restrict__ k, const float* __restrict__ v,
                    const int* __restrict__ counts, float* __restrict__ k_cache,
                    float* __restrict__ v_cache, int* __restrict__ out_lengths, int batch,
                    int tokens, int blocks_per_head) {
  const int unit = blockIdx.x / blocks_per_head;           // row * kv_heads + head
  const int part = blockIdx.x - unit * blocks_per_head;
  const int b = unit / g.kv_heads, h = unit - b * g.kv_heads;
  const int n = paged_length(g, b);
  int c = counts ? __ldg(counts + b) : tokens;
  const bool bad = c < 0 || c > tokens || c > g.capacity - n;
  if (bad) c = c < 0 ? 0 : min(min(c, tokens), g.capacity - n);
  if (h == 0 && part == 0 && threadIdx.x == 0) {
    if (bad) atomicOr(g.flag, kBadLength);
    out_lengths[b] = n + c;
  }
  const int per_row = g.head_dim / V;
  const uint64_t total = (uint64_t)c * per_row;
  const uint64_t src0 = (uint64_t)unit * tokens * g.head_dim;
  for (uint64_t i = (uint64_t)part * 256 + threadIdx.x; i < total; i += (uint64_t)blocks_per_head * 256) {
    const int t = (int)(i / per_row);
    const int d = (int)(i - (uint64_t)t * per_row) * V;
    const uint32_t row = paged_row(g, b, h, n + t);
    if (row == kNoRow) continue;
    const uint64_t src = src0 + (uint64_t)t * g.head_dim + d;
    const uint64_t dst = (uint64_t)row * g.head_dim + d;
    if (V == 4) {
      *reinterpret_cast<float4*>(k_cache + dst) = __ldg(reinterpret_cast<const float4*>(k + src));
      *reinterpret_cast<float4*>(v_cache + dst) = __ldg(reinterpret_cast<const float4*>(v + src));
    } else {
      k_cache[dst] = __ldg(k + src);
      v_cache[dst] = __ldg(v + src);
    }
  }
}

// ---- evict -------------------------------------------------------------------------------
struct EvictArgs {
  const float* weights;     // [batch, kv_heads, capacity]
  const int* positions;     // or null
  const int* total;         // [batch], or null
  float* out_weights;
  int* out_positions;
  int* out_lengths;
  int* out_kept;            // [batch, kv_heads, budget]
  int* moves;               // [units]: how many slots move
  int* holes;               // [units][list]: where to, ascending
  int* tails;               // [units][list]: where from, ascending
  int list;                 // min(budget, capacity)
  int budget, recent;
  float *k_cache, *v_cache;
  int move;                 // the rows are moved by the block that chose them
};

// Weights as unsigned numbers of the same order: NaN above all, -0 equal to +0.
__device__ __forceinline__ uint32_t ordered(float w) {
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

struct SlotView {
  const float* w;
  const int* pos;     // null: by the slot
  long long total, n, first_recent;
  __device__ __forceinline__ long long position(int j) const {
    if (pos) {
      const int p = __ldg(pos + j);
      if (p >= 0) return p;
    }
    return total - (n - j);
  }
  // The recent ones first, whatever their weight.
  __device__ __forceinline__ uint32_t key(int j) const {
    return position(j) >= first_recent ? 0xffffffffu : ordered(__ldg(w + j));
  }
};

// Exclusive sum over the block of one value a thread, and the block's total.
template <int NT>
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* warp_sums,
                                                         unsigned long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    const unsigned long long mine = lane < NT / 32 ? warp_sums[lane] : 0;
    unsigned long long t = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    if (lane < NT / 32) warp_sums[lane] = t - mine;
    if (lane == 31) warp_sums[32] = t;
  }
  __syncthreads();
  const unsigned long long r = warp_sums[warp] + s - v;
  *total = warp_sums[32];
  __syncthreads();   // warp_sums is reused by the next call
  return r;
}

// One block decides for one row and head which slots stay: the m-th largest key by a radix
// select of 8 bits a pass (counting, no sorting), then one pass in slot order that ranks the
// slots equal to it, the free places below m and the kept slots from m on: every thread has a
// stretch of slots, so that each of these takes one sum over the block.  HELD: the keys are formed
// once and kept in shared memory, which a row of up to 48 k slots allows.  NT: threads.  V: values a
// lane moves at a time.
template <bool HELD, int V, int NT>
__global__ void __launch_bounds__(NT)
paged_evict_select_kernel(const PagedLayout g, const EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[256];
  __shared__ unsigned long long warp_sums[33];
  __shared__ uint32_t pick[2];
  const int unit = blockIdx.x;
  const int b = unit / g.kv_heads;
  const int tid = threadIdx.x;
  const int n = paged_length(g, b);
  const int m = min(n, a.budget);
  const uint64_t base = (uint64_t)unit * g.capacity;
  SlotView s;
  s.w = a.weights + base;
  s.pos = a.positions ? a.positions + base : nullptr;
  s.n = n;
  s.total = a.total ? __ldg(a.total + b) : n;
  s.first_recent = s.total - a.recent;
  float* ow = a.out_weights + base;
  int* op = a.out_positions + base;
  int* ok = a.out_kept + (uint64_t)unit * a.budget;
  if (unit == b * g.kv_heads && tid == 0) a.out_lengths[b] = m;
  for (int j = m + tid; j < g.capacity; j += NT) {
    ow[j] = 0.0f;
    op[j] = -1;
  }
  for (int j = m + tid; j < a.budget; j += NT) ok[j] = -1;
  if (n <= m) {   // nothing to lose
    for (int j = tid; j < m; j += NT) {
      ow[j] = __ldg(s.w + j);
      op[j] = (int)s.position(j);
      ok[j] = j;
    }
    if (tid == 0) a.moves[unit] = 0;
    return;
  }
  if (HELD) {
#pragma unroll 4
    for (int j = tid; j < n; j += NT) keys[j] = s.key(j);   // (read by the same thread or behind a barrier)
  }
  auto key_of = [&](int j) { return HELD ? keys[j] : s.key(j); };
  // the key that the m-th largest has, and how many of the slots that have it stay
  uint32_t prefix = 0, mask = 0;
  uint32_t want = (uint32_t)m;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += NT) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += NT) {
      const uint32_t key = key_of(j);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 32) {
      // lane l: the eight digits below 256 - 8 l, from the top
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = hist[255 - (tid * 8 + i)];
        sum += c[i];
      }
      uint32_t before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, before, o);
        if (tid >= o) before += u;
      }
      before -= sum;
      if (before < want && want <= before + sum) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < want && want <= before + c[i]) {
            pick[0] = 255u - (uint32_t)(tid * 8 + i);
            pick[1] = want - before;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    want = pick[1];
    mask |= 255u << shift;
  }
  // in slot order: slots equal to the threshold stay while `want` lasts.  (Stretches of an odd
  // number of slots, so that the threads of a warp read different banks.)
  const int stretch = ((n + NT - 1) / NT) | 1;
  const int j0 = min(tid * stretch, n), j1 = min(j0 + stretch, n);
  uint32_t equal = 0;
  for (int j = j0; j < j1; ++j) equal += key_of(j) == prefix;
  unsigned long long all;
  const uint32_t equal_before = (uint32_t)block_scan<NT>(equal, warp_sums, &all);
  auto each = [&](auto hole, auto tail) {
    uint32_t rank = equal_before;
    for (int j = j0; j < j1; ++j) {
      const uint32_t key = key_of(j);
      const bool keep = key > prefix || (key == prefix && rank++ < want);
      if (j < m && !keep) hole(j);
      if (j >= m && keep) tail(j);
    }
  };
  uint32_t my_holes = 0, my_tails = 0;
  each([&](int) { ++my_holes; }, [&](int) { ++my_tails; });
  const unsigned long long before = block_scan<NT>((unsigned long long)my_tails << 32 | my_holes, warp_sums, &all);
  const uint32_t holes = (uint32_t)all;
  int* hole_list = a.holes + (uint64_t)unit * a.list;
  int* tail_list = a.tails + (uint64_t)unit * a.list;
  uint32_t hole_at = (uint32_t)before, tail_at = (uint32_t)(before >> 32);
  each([&](int j) { hole_list[hole_at++] = j; }, [&](int j) { tail_list[tail_at++] = j; });
  for (int j = tid; j < m; j += NT) {
    ow[j] = __ldg(s.w + j);
    op[j] = (int)s.position(j);
    ok[j] = j;
  }
  __syncthreads();   // the lists of this block are read, and the free places written again, by other threads
  for (uint32_t r = tid; r < holes; r += NT) {
    const int to = hole_list[r], from = tail_list[r];
    ow[to] = __ldg(s.w + from);
    op[to] = (int)s.position(from);
    ok[to] = from;
  }
  if (tid == 0) a.moves[unit] = (int)holes;
  if (a.move) {
    const int h = unit - b * g.kv_heads;
    for (uint32_t r = tid >> 5; r < holes; r += NT / 32) {
      const uint32_t from = paged_row(g, b, h, tail_list[r]), to = paged_row(g, b, h, hole_list[r]);
      if (from != kNoRow && to != kNoRow)
        copy_row<V>(a.k_cache, a.v_cache, (uint64_t)from * g.head_dim, (uint64_t)to * g.head_dim, g.head_dim, tid & 31);
    }
  }
}

// The rows of the kept slots: sources are slots from m on, destinations slots below m, so no
// move touches another's source.  A warp takes kRowsAtOnce moves at a time: from list to page table to
// row each is a chain of three loads, and one chain a warp left memory waiting (128 rows and heads,
// 1.5 k moves of 128 values each: 61 us with one, 57 with four, 5.3 TB/s).
constexpr int kRowsAtOnce = 4;
template <int V>
__global__ void __launch_bounds__(256)
paged_evict_move_kernel(const PagedLayout g, const int* __restrict__ moves,
                        const int* __restrict__ holes, const int* __restrict__ tails, int list,
                        float* __restrict__ k_cache, float* __restrict__ v_cache,
                        int blocks_per_unit) {
  const int unit = blockIdx.x / blocks_per_unit;
  const int part = blockIdx.x - unit * blocks_per_unit;
  const int b = unit / g.kv_heads, h = unit - b * g.kv_heads;
  const int count = __ldg(moves + unit);
  const int lane = threadIdx.x & 31;
  const int step = blocks_per_unit * 8 * kRowsAtOnce;
  struct __align__(V * 4) Vec { float x[V]; };
  for (int r0 = (part * 8 + ((int)threadIdx.x >> 5)) * kRowsAtOnce; r0 < count; r0 += step) {
    // lane i < 2 kRowsAtOnce finds source (i even) or destination of move i / 2
    uint32_t mine = kNoRow;
    const int r = r0 + (lane >> 1);
    if (lane < 2 * kRowsAtOnce && r < count)
      mine = paged_row(g, b, h, __ldg((lane & 1 ? holes : tails) + (uint64_t)unit * list + r));
    uint64_t from[kRowsAtOnce], to[kRowsAtOnce];
    bool move[kRowsAtOnce];
#pragma unroll
    for (int u = 0; u < kRowsAtOnce; ++u) {
      const uint32_t f = __shfl_sync(0xffffffffu, mine, 2 * u), t = __shfl_sync(0xffffffffu, mine, 2 * u + 1);
      move[u] = f != kNoRow && t != kNoRow;
      from[u] = (uint64_t)f * g.head_dim;
      to[u] = (uint64_t)t * g.head_dim;
    }
    for (int d = lane * V; d < g.head_dim; d += 32 * V) {
      Vec x[kRowsAtOnce], y[kRowsAtOnce];
#pragma unroll
      for (int u = 0; u < kRowsAtOnce; ++u)
        if (move[u]) {
          x[u] = *reinterpret_cast<const Vec*>(k_cache + from[u] + d);
          y[u] = *reinterpret_cast<const Vec*>(v_cache + from[u] + d);
        }
#pragma unroll
      for (int u = 0; u < kRowsAtOnce; ++u)
        if (move[u]) {
          *reinterpret_cast<Vec*>(k_cache + to[u] + d) = x[u];
          *reinterpret_cast<Vec*>(v_cache + to[u] + d) = y[u];
        }
    }
  }
}

}  // namespace

extern "C" {

int tfjs_cuda_paged_cache_append(tfjs_cuda_ctx* ctx, const tfjs_cuda_paged_params* p,
                                 int32_t k_cache_id, int32_t v_cache_id, int32_t k_id,
                                 int32_t v_id, int32_t page_table_id, int32_t lengths_id,
                                 int32_t counts_id, int32_t out_lengths_id) {
  if (!ctx) return TFJS_CUDA_INVALID_ARG;
  const char* who = "paged cache append";
  PagedLayout g;
  Buffer *kc, *vc, *k, *v, *counts = nullptr, *ol;
  int rc = paged_layout(ctx, p, who, k_cache_id, v_cache_id, page_table_id, lengths_id, &g, &kc, &vc);
  if (rc) return rc;
  if (p->tokens <= 0)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: dimensions must be positive", who);
  const uint64_t units = (uint64_t)p->batch * p->kv_heads;
  const uint64_t n = units * p->tokens * (uint64_t)p->head_dim;
  if ((rc = ctx_get(ctx, k_id, n * 4, who, &k))) return rc;
  if ((rc = ctx_get(ctx, v_id, n * 4, who, &v))) return rc;
  if (counts_id && (rc = ctx_get(ctx, counts_id, (uint64_t)p->batch * 4, who, &counts))) return rc;
  if ((rc = ctx_get(ctx, out_lengths_id, (uint64_t)p->batch * 4, who, &ol))) return rc;
  if (out_lengths_id == lengths_id || k_id == k_cache_id || k_id == v_cache_id ||
      v_id == k_cache_id || v_id == v_cache_id)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: an output is also an input", who);
  const uint64_t rows = (uint64_t)p->batch * 4;
  const Span spans[] = {{kc->ptr, g.pool_bytes}, {vc->ptr, g.pool_bytes}, {ol->ptr, rows},
                        {k->ptr, n * 4}, {v->ptr, n * 4}, {g.table, rows * p->max_pages}, {g.lengths, rows},
                        {counts ? counts->ptr : nullptr, counts ? rows : 0}};
  if ((rc = ctx_apart(ctx, who, spans, 8, 3))) return rc;
  cudaSetDevice(ctx->device);
  const bool wide = p->head_dim % 4 == 0 &&
                    (((uintptr_t)kc->ptr | (uintptr_t)vc->ptr | (uintptr_t)k->ptr | (uintptr_t)v->ptr) & 15) == 0;
  const uint64_t items = (uint64_t)p->tokens * (p->head_dim / (wide ? 4 : 1));
  // a block handles up to four items a thread of one row and head
  uint64_t per = (items + 1023) / 1024;
  if (per > 0x7fffffffull / units) per = 0x7fffffffull / units;
  const unsigned grid = (unsigned)(units * per);
  const int* ct = counts ? (const int*)counts->ptr : nullptr;
  if (wide)
    paged_append_kernel<4><<<grid, 256, 0, ctx->stream>>>(
        g, (const float*)k->ptr, (const float*)v->ptr, ct, (float*)kc->ptr, (float*)vc->ptr,
        (int*)ol->ptr, p->batch, p->tokens, (int)per);
  else
    paged_append_kernel<1><<<grid, 256, 0, ctx->stream>>>(
        g, (const float*)k->ptr, (const float*)v->ptr, ct, (float*)kc->ptr, (float*)vc->ptr,
        (int*)ol->ptr, p->batch, p->tokens, (int)per);
  LAUNCH_CHECK(ctx, wide ? "paged_append_kernel<4>" : "paged_append_kernel<1>");
  ctx_mark_written(ctx, k_cache_id);
  ctx_mark_written(ctx, v_cache_id);
  ctx_mark_written(ctx, out_lengths_id);
  return TFJS_CUDA_OK;
}

int tfjs_cuda_paged_cache_evict(tfjs_cuda_ctx* ctx, const tfjs_cuda_paged_params* p,
                                int32_t k_cache_id, int32_t v_cache_id, int32_t weights_id,
                                int32_t page_table_id, int32_t lengths_id, int32_t positions_id,
                                int32_t total_id, int32_t out_weights_id,
                                int32_t out_positions_id, int32_t out_lengths_id,
                                int32_t out_kept_id) {
  if (!ctx) return TFJS_CUDA_INVALID_ARG;
  const char* who = "paged cache evict";
  PagedLayout g;
  Buffer *kc, *vc, *w, *pos = nullptr, *tot = nullptr, *ow, *op, *ol, *ok;
  int rc = paged_layout(ctx, p, who, k_cache_id, v_cache_id, page_table_id, lengths_id, &g, &kc, &vc);
  if (rc) return rc;
  if (p->budget <= 0 || p->recent < 0 || p->recent > p->budget)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG,
                    "%s: the budget must be positive and hold the recent slots", who);
  const uint64_t units = (uint64_t)p->batch * p->kv_heads;
  const uint64_t slots = units * (uint64_t)g.capacity * 4;
  if ((rc = ctx_get(ctx, weights_id, slots, who, &w))) return rc;
  if (positions_id && (rc = ctx_get(ctx, positions_id, slots, who, &pos))) return rc;
  if (total_id && (rc = ctx_get(ctx, total_id, (uint64_t)p->batch * 4, who, &tot))) return rc;
  if ((rc = ctx_get(ctx, out_weights_id, slots, who, &ow))) return rc;
  if ((rc = ctx_get(ctx, out_positions_id, slots, who, &op))) return rc;
  if ((rc = ctx_get(ctx, out_lengths_id, (uint64_t)p->batch * 4, who, &ol))) return rc;
  if ((rc = ctx_get(ctx, out_kept_id, units * (uint64_t)p->budget * 4, who, &ok))) return rc;
  const int32_t in[] = {k_cache_id, v_cache_id, weights_id, page_table_id, lengths_id, positions_id, total_id};
  const int32_t out[] = {out_weights_id, out_positions_id, out_lengths_id, out_kept_id};
  for (int i = 0; i < 4; ++i) {
    for (int32_t x : in)
      if (out[i] == x) return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: an output is also an input", who);
    for (int j = 0; j < i; ++j)
      if (out[i] == out[j]) return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: an output is given twice", who);
  }
  const uint64_t rows = (uint64_t)p->batch * 4;
  const Span spans[] = {{kc->ptr, g.pool_bytes}, {vc->ptr, g.pool_bytes}, {ow->ptr, slots}, {op->ptr, slots},
                        {ol->ptr, rows}, {ok->ptr, units * (uint64_t)p->budget * 4},
                        {w->ptr, slots}, {g.table, rows * p->max_pages}, {g.lengths, rows},
                        {pos ? pos->ptr : nullptr, pos ? slots : 0}, {tot ? tot->ptr : nullptr, tot ? rows : 0}};
  if ((rc = ctx_apart(ctx, who, spans, 11, 6))) return rc;
  float *kp = (float*)kc->ptr, *vp = (float*)vc->ptr;
  EvictArgs a;
  a.weights = (const float*)w->ptr;
  a.positions = pos ? (const int*)pos->ptr : nullptr;
  a.total = tot ? (const int*)tot->ptr : nullptr;
  a.out_weights = (float*)ow->ptr;
  a.out_positions = (int*)op->ptr;
  a.out_lengths = (int*)ol->ptr;
  a.out_kept = (int*)ok->ptr;
  a.budget = p->budget;
  a.recent = p->recent;
  a.list = p->budget < g.capacity ? p->budget : g.capacity;
  cudaSetDevice(ctx->device);
  TempBuffer ws(ctx);
  void* mem;
  if ((rc = ws.get(units * (1 + 2 * (uint64_t)a.list) * 4, &mem))) return rc;   // (Buffer pointers end here)
  a.moves = (int*)mem;
  a.holes = a.moves + units;
  a.tails = a.holes + units * a.list;
  const bool wide = p->head_dim % 4 == 0 && (((uintptr_t)kp | (uintptr_t)vp) & 15) == 0;
  // at most min(budget, capacity - budget) slots of a row move; a few the choosing block moves
  // itself, which saves a launch
  const int most = g.capacity - p->budget < a.list ? g.capacity - p->budget : a.list;
  a.k_cache = kp;
  a.v_cache = vp;
  a.move = most <= 64;
  const uint64_t held = (uint64_t)g.capacity * 4;
  // 256 threads where there are more rows and heads than SMs, which then hold several blocks, and rows
  // are short (256 of them with 1025 / 2049 / 4097 / 8193 slots: 10 / 14 / 23 / 41 us against 16 / 18 /
  // 22 / 32 with 1024 threads; 8 of them: 10 / 13 / 18 / 38 against 8 / 9 / 12 / 16)
  constexpr int kMostHeld = 192 * 1024;
  const bool small = g.capacity <= 4096 && units > (uint64_t)ctx->sm_count, keep_keys = held <= (uint64_t)kMostHeld;
  void (*kernel)(PagedLayout, EvictArgs) =
      small ? (wide ? paged_evict_select_kernel<true, 4, 256> : paged_evict_select_kernel<true, 1, 256>)
      : keep_keys ? (wide ? paged_evict_select_kernel<true, 4, 1024> : paged_evict_select_kernel<true, 1, 1024>)
                  : (wide ? paged_evict_select_kernel<false, 4, 1024> : paged_evict_select_kernel<false, 1, 1024>);
  // (Without asking for more, a launch has 48 KB for the keys and the kernel's own arrays together.  The
  // same amount whatever the row needs, so that two contexts of a process cannot lower it for each other.)
  if (held > 32 * 1024 && keep_keys)
    CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostHeld));
  kernel<<<(unsigned)units, small ? 256 : 1024, keep_keys ? held : 0, ctx->stream>>>(g, a);
  LAUNCH_CHECK(ctx, "paged_evict_select_kernel");
  if (!a.move) {
    uint64_t per = ((uint64_t)most + 31) / 32;
    if (per * units > (uint64_t)ctx->sm_count * 32) per = ((uint64_t)ctx->sm_count * 32 + units - 1) / units;
    const unsigned grid = (unsigned)(units * per);
    if (wide)
      paged_evict_move_kernel<4><<<grid, 256, 0, ctx->stream>>>(g, a.moves, a.holes, a.tails, a.list, kp, vp, (int)per);
    else
      paged_evict_move_kernel<1><<<grid, 256, 0, ctx->stream>>>(g, a.moves, a.holes, a.tails, a.list, kp, vp, (int)per);
    LAUNCH_CHECK(ctx, wide ? "paged_evict_move_kernel<4>" : "paged_evict_move_kernel<1>");
  }
  ctx_mark_written(ctx, k_cache_id);
  ctx_mark_written(ctx, v_cache_id);
  for (int32_t id : out) ctx_mark_written(ctx, id);
  return TFJS_CUDA_OK;
}

}  // extern "C"
