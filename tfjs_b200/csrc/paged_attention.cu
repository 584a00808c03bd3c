// Attention of one new token over a paged key-value cache:
//   s_j = q . k_j * scale + mask_j,  p = softmax(s),  out = sum_j p_j v_j
// Every key and value is read once and takes 4 G operations a byte pair of it (G query heads
// share a key-value head), so memory bounds it.  A row's slots are split over blocks
// (and a block's slots over its warps), each keeps a running maximum, sum and weighted
// sum of values, and a second kernel joins them.
#include "paged.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;
constexpr int kTile = 32;          // slots a warp takes at a time

struct PagedAttnArgs {
  const float* q;         // [batch, heads, head_dim]
  const float* k_cache;
  const float* v_cache;
  const float* mask;      // [batch, capacity], or null
  float* part_acc;        // [batch * heads][splits][head_dim]
  float2* part_ml;        // [batch * heads][splits]: maximum, sum
  float* scores;          // [batch * heads][capacity], or null: the scores are not kept
  int heads, group, group_chunks, split_len, splits;
  int has_scale;
  float scale;
};

// e^(x - m) for a maximum that may be -infinity (nothing seen yet: 0)
__device__ __forceinline__ float exp_from(float x, float m) {
  return exp2_approx(__fmul_rn(__fsub_rn(x, m == -INFINITY ? 0.0f : m), kLog2e));
}

template <bool WIDE>
__device__ __forceinline__ float4 load4(const float* p, int d, int dim) {
  if (WIDE) return d < dim ? __ldg(reinterpret_cast<const float4*>(p + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 r;
  r.x = d < dim ? __ldg(p + d) : 0.f;
  r.y = d + 1 < dim ? __ldg(p + d + 1) : 0.f;
  r.z = d + 2 < dim ? __ldg(p + d + 2) : 0.f;
  r.w = d + 3 < dim ? __ldg(p + d + 3) : 0.f;
  return r;
}

// DM: head_dim rounded up; GT: query heads of one key-value head that a block serves.
template <int DM, int GT, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32)
paged_attention_kernel(const PagedLayout g, const PagedAttnArgs a) {
  constexpr int NI = DM / 16;                    // steps of 16 values of a key, 4 a lane
  constexpr int LPR = DM / 4 < 32 ? DM / 4 : 32; // lanes that share a value row
  constexpr int VR = DM / 4 / LPR;               // 4-value pieces of it a lane holds
  constexpr int TPI = 32 / LPR;                  // value rows a warp reads at a time
  __shared__ __align__(16) float q_s[GT][DM];
  __shared__ float p_s[kWarps][kTile][GT];
  __shared__ float2 ml_s[kWarps][GT];
  __shared__ __align__(16) float acc_s[kWarps][GT][DM];
  int u = blockIdx.x;
  const int split = u % a.splits;
  u /= a.splits;
  const int gc = u % a.group_chunks;
  u /= a.group_chunks;
  const int h = u % g.kv_heads, b = u / g.kv_heads;
  const int n = paged_length(g, b);
  const int begin = split * a.split_len;
  const int end = min(n, begin + a.split_len);
  if (begin >= end && split != 0) return;        // (the join does not read this split)
  const int head0 = h * a.group + gc * GT;       // first query head
  const int live = min(GT, a.group - gc * GT);   // of them, real ones
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < GT * DM; i += kWarps * 32) {
    const int gi = i / DM, d = i - gi * DM;
    q_s[gi][d] = gi < live && d < g.head_dim ? __ldg(a.q + ((uint64_t)b * a.heads + head0 + gi) * g.head_dim + d) : 0.f;
  }
  __syncthreads();

  float m[GT], l[GT];
  float4 acc[GT][VR];
#pragma unroll
  for (int gi = 0; gi < GT; ++gi) {
    m[gi] = -INFINITY;
    l[gi] = 0.f;
#pragma unroll
    for (int r = 0; r < VR; ++r) acc[gi][r] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const int c = lane & 3, tok = lane >> 2;       // keys: four lanes a slot, eight slots at a time

  for (int t0 = begin + warp * kTile; t0 < end; t0 += kWarps * kTile) {
    const int mine = t0 + lane;
    const float my_mask = a.mask && mine < end ? __ldg(a.mask + (uint64_t)b * g.capacity + mine) : 0.f;
    // (a slot hidden by the mask is not read: what it holds, NaN included, does not count)
    const uint32_t my_row = mine < end && my_mask != -INFINITY ? paged_row(g, b, h, mine) : kNoRow;
    float s[GT][4];
#pragma unroll
    for (int gi = 0; gi < GT; ++gi)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[gi][x] = 0.f;
    uint32_t row[4];
    const float* kp[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      row[x] = __shfl_sync(0xffffffffu, my_row, x * 8 + tok);
      kp[x] = a.k_cache + (uint64_t)(row[x] == kNoRow ? 0u : row[x]) * g.head_dim;
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int d = (i * 4 + c) * 4;
      float4 kv[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        kv[x] = row[x] != kNoRow ? load4<WIDE>(kp[x], d, g.head_dim) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int gi = 0; gi < GT; ++gi) {
        const float4 qv = *reinterpret_cast<const float4*>(&q_s[gi][d]);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          s[gi][x] = fmaf(qv.w, kv[x].w, fmaf(qv.z, kv[x].z, fmaf(qv.y, kv[x].y, fmaf(qv.x, kv[x].x, s[gi][x]))));
      }
    }
    float mask4[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) mask4[x] = __shfl_sync(0xffffffffu, my_mask, x * 8 + tok);
#pragma unroll
    for (int gi = 0; gi < GT; ++gi) {
      float mx = m[gi];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float t = s[gi][x];
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        if (a.has_scale) t = __fmul_rn(t, a.scale);
        if (a.mask) t = __fadd_rn(t, mask4[x]);
        if (row[x] == kNoRow) t = -INFINITY;
        s[gi][x] = t;
        mx = fmaxf(mx, t);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      const float down = exp_from(m[gi], mx);
      m[gi] = mx;
      l[gi] *= down;
#pragma unroll
      for (int r = 0; r < VR; ++r) {
        acc[gi][r].x *= down;
        acc[gi][r].y *= down;
        acc[gi][r].z *= down;
        acc[gi][r].w *= down;
      }
      // lane c of a slot's four keeps the slot of sub-tile c
      const float mine_s = c == 0 ? s[gi][0] : c == 1 ? s[gi][1] : c == 2 ? s[gi][2] : s[gi][3];
      const float p = exp_from(mine_s, mx);
      l[gi] += p;
      p_s[warp][c * 8 + tok][gi] = p;
      const int slot = t0 + c * 8 + tok;
      if (a.scores && gi < live && slot < end)
        a.scores[((uint64_t)b * a.heads + head0 + gi) * g.capacity + slot] = mine_s;
    }
    __syncwarp();
#pragma unroll 4
    for (int it = 0; it < kTile / TPI; ++it) {
      const int t = it * TPI + lane / LPR;
      const uint32_t r0 = __shfl_sync(0xffffffffu, my_row, t);
      if (r0 == kNoRow) continue;                // (lanes of a value row agree)
      const float* vp = a.v_cache + (uint64_t)r0 * g.head_dim;
      float4 v[VR];
#pragma unroll
      for (int r = 0; r < VR; ++r) v[r] = load4<WIDE>(vp, (r * LPR + lane % LPR) * 4, g.head_dim);
#pragma unroll
      for (int gi = 0; gi < GT; ++gi) {
        const float p = p_s[warp][t][gi];
#pragma unroll
        for (int r = 0; r < VR; ++r) {
          acc[gi][r].x = fmaf(p, v[r].x, acc[gi][r].x);
          acc[gi][r].y = fmaf(p, v[r].y, acc[gi][r].y);
          acc[gi][r].z = fmaf(p, v[r].z, acc[gi][r].z);
          acc[gi][r].w = fmaf(p, v[r].w, acc[gi][r].w);
        }
      }
    }
    __syncwarp();
  }

  // across the lanes, then across the warps
#pragma unroll
  for (int gi = 0; gi < GT; ++gi) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) l[gi] += __shfl_xor_sync(0xffffffffu, l[gi], o);
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
      for (int r = 0; r < VR; ++r) {
        acc[gi][r].x += __shfl_xor_sync(0xffffffffu, acc[gi][r].x, o);
        acc[gi][r].y += __shfl_xor_sync(0xffffffffu, acc[gi][r].y, o);
        acc[gi][r].z += __shfl_xor_sync(0xffffffffu, acc[gi][r].z, o);
        acc[gi][r].w += __shfl_xor_sync(0xffffffffu, acc[gi][r].w, o);
      }
    if (lane == 0) ml_s[warp][gi] = make_float2(m[gi], l[gi]);
    if (lane < LPR)
#pragma unroll
      for (int r = 0; r < VR; ++r)
        *reinterpret_cast<float4*>(&acc_s[warp][gi][(r * LPR + lane) * 4]) = acc[gi][r];
  }
  __syncthreads();
  for (int i = tid; i < GT * DM; i += kWarps * 32) {
    const int gi = i / DM, d = i - gi * DM;
    if (gi >= live || d >= g.head_dim) continue;
    float mx = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml_s[w][gi].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp_from(ml_s[w][gi].x, mx);
      sum = fmaf(ml_s[w][gi].y, f, sum);
      o = fmaf(acc_s[w][gi][d], f, o);
    }
    const uint64_t part = ((uint64_t)b * a.heads + head0 + gi) * a.splits + split;
    a.part_acc[part * g.head_dim + d] = o;
    if (d == 0) a.part_ml[part] = make_float2(mx, sum);
  }
}

// Splits that row b's slots fill (at least one, which is empty for an empty row).
__device__ __forceinline__ int live_splits(const PagedLayout& g, const PagedAttnArgs& a, int b) {
  const int n = paged_length(g, b);
  return max(1, (n + a.split_len - 1) / a.split_len);
}

__global__ void __launch_bounds__(128)
paged_attention_join_kernel(const PagedLayout g, const PagedAttnArgs a, float* __restrict__ out) {
  const int unit = blockIdx.x;                   // row * heads + head
  const int ns = live_splits(g, a, unit / a.heads);
  const float2* ml = a.part_ml + (uint64_t)unit * a.splits;
  float mx = -INFINITY, sum = 0.f;
  for (int i = 0; i < ns; ++i) mx = fmaxf(mx, ml[i].x);
  for (int i = 0; i < ns; ++i) sum = fmaf(ml[i].y, exp_from(ml[i].x, mx), sum);
  for (int d = threadIdx.x; d < g.head_dim; d += 128) {
    float o = 0.f;
    for (int i = 0; i < ns; ++i)
      o = fmaf(a.part_acc[((uint64_t)unit * a.splits + i) * g.head_dim + d], exp_from(ml[i].x, mx), o);
    out[(uint64_t)unit * g.head_dim + d] = sum == 0.f ? 0.f : __fdiv_rn(o, sum);
  }
}

// Accumulated weights: a thread per slot, summing the query heads of the group in order.
__global__ void __launch_bounds__(256)
paged_attention_weights_kernel(const PagedLayout g, const PagedAttnArgs a,
                               const float* __restrict__ weights, float* __restrict__ out,
                               int blocks_per_unit) {
  extern __shared__ float2 stat[];               // [group]: maximum, 1 / sum (0 for an empty row)
  const int unit = blockIdx.x / blocks_per_unit; // row * kv_heads + head
  const int part = blockIdx.x - unit * blocks_per_unit;
  const int b = unit / g.kv_heads, h = unit - b * g.kv_heads;
  const int n = paged_length(g, b), ns = live_splits(g, a, b);
  const uint64_t head0 = (uint64_t)b * a.heads + h * a.group;
  for (int gi = threadIdx.x; gi < a.group; gi += 256) {
    const float2* ml = a.part_ml + (head0 + gi) * a.splits;
    float mx = -INFINITY, sum = 0.f;
    for (int i = 0; i < ns; ++i) mx = fmaxf(mx, ml[i].x);
    for (int i = 0; i < ns; ++i) sum = fmaf(ml[i].y, exp_from(ml[i].x, mx), sum);
    stat[gi] = make_float2(mx, sum == 0.f ? 0.f : __fdiv_rn(1.0f, sum));
  }
  __syncthreads();
  for (int j = part * 256 + threadIdx.x; j < g.capacity; j += blocks_per_unit * 256) {
    float w = 0.f;
    if (j < n) {
      for (int gi = 0; gi < a.group; ++gi) {
        const float2 st = stat[gi];
        const float s = a.scores[(head0 + gi) * g.capacity + j];
        // (an empty row has 1 / sum = 0 and scores of -infinity only)
        w = fmaf(exp_from(s, st.x), st.y, w);
      }
      w += weights[(uint64_t)unit * g.capacity + j];
    }
    out[(uint64_t)unit * g.capacity + j] = w;
  }
}

template <int DM, int GT, bool WIDE>
int launch_attention(tfjs_cuda_ctx* ctx, const PagedLayout& g, const PagedAttnArgs& a, unsigned grid) {
  paged_attention_kernel<DM, GT, WIDE><<<grid, kWarps * 32, 0, ctx->stream>>>(g, a);
  LAUNCH_CHECK(ctx, "paged_attention_kernel");
  return TFJS_CUDA_OK;
}
template <int GT, bool WIDE>
int launch_dim(tfjs_cuda_ctx* ctx, const PagedLayout& g, const PagedAttnArgs& a, unsigned grid) {
  if (g.head_dim <= 32) return launch_attention<32, GT, WIDE>(ctx, g, a, grid);
  if (g.head_dim <= 64) return launch_attention<64, GT, WIDE>(ctx, g, a, grid);
  if (g.head_dim <= 128) return launch_attention<128, GT, WIDE>(ctx, g, a, grid);
  return launch_attention<256, GT, WIDE>(ctx, g, a, grid);
}

}  // namespace

extern "C" int tfjs_cuda_paged_attention(tfjs_cuda_ctx* ctx, const tfjs_cuda_paged_params* p,
                                         int32_t q_id, int32_t k_cache_id, int32_t v_cache_id,
                                         int32_t page_table_id, int32_t lengths_id,
                                         int32_t mask_id, int32_t weights_id, int32_t out_id,
                                         int32_t out_weights_id) {
  if (!ctx) return TFJS_CUDA_INVALID_ARG;
  const char* who = "paged attention";
  PagedLayout g;
  Buffer *kc, *vc, *q, *mask = nullptr, *w = nullptr, *out, *ow = nullptr;
  int rc = paged_layout(ctx, p, who, k_cache_id, v_cache_id, page_table_id, lengths_id, &g, &kc, &vc);
  if (rc) return rc;
  if (p->heads <= 0 || p->heads % p->kv_heads != 0)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG,
                    "%s: %d query heads do not share %d key-value heads evenly", who, p->heads, p->kv_heads);
  if ((weights_id == 0) != (out_weights_id == 0))
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: weights need a place for the new ones", who);
  const uint64_t units = (uint64_t)p->batch * p->heads, kv_units = (uint64_t)p->batch * p->kv_heads;
  const uint64_t cap = (uint64_t)g.capacity;
  if (units > 0xffffffull || p->heads / p->kv_heads > 1024)
    return ctx_fail(ctx, TFJS_CUDA_UNSUPPORTED, "%s: too many heads", who);
  if ((rc = ctx_get(ctx, q_id, units * p->head_dim * 4, who, &q))) return rc;
  if (mask_id && (rc = ctx_get(ctx, mask_id, p->batch * cap * 4, who, &mask))) return rc;
  if (weights_id && (rc = ctx_get(ctx, weights_id, kv_units * cap * 4, who, &w))) return rc;
  if ((rc = ctx_get(ctx, out_id, units * p->head_dim * 4, who, &out))) return rc;
  if (weights_id && (rc = ctx_get(ctx, out_weights_id, kv_units * cap * 4, who, &ow))) return rc;
  const int32_t in[] = {q_id, k_cache_id, v_cache_id, page_table_id, lengths_id, mask_id, weights_id};
  for (int32_t x : in)
    if (x && (x == out_id || x == out_weights_id))
      return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: an output is also an input", who);
  if (out_id == out_weights_id)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: an output is given twice", who);

  PagedAttnArgs a;
  a.q = (const float*)q->ptr;
  a.k_cache = (const float*)kc->ptr;
  a.v_cache = (const float*)vc->ptr;
  a.mask = mask ? (const float*)mask->ptr : nullptr;
  a.heads = p->heads;
  a.group = p->heads / p->kv_heads;
  a.has_scale = p->has_scale;
  a.scale = p->scale;
  float* op = (float*)out->ptr;
  const float* wp = w ? (const float*)w->ptr : nullptr;
  float* owp = ow ? (float*)ow->ptr : nullptr;

  const bool wide = p->head_dim % 4 == 0 && (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) == 0;
  const int gt = a.group == 1 ? 1 : a.group == 2 ? 2 : a.group <= 4 ? 4 : 8;
  a.group_chunks = (a.group + gt - 1) / gt;
  // Splits: enough blocks to fill the GPU about eight times over (rows are ragged, and a
  // block that finds nothing to do leaves at once), each with at least one tile a warp.
  const uint64_t base = kv_units * a.group_chunks;
  const int step = kWarps * kTile;
  uint64_t splits = ((uint64_t)ctx->sm_count * 8 + base - 1) / base;
  const uint64_t most = (cap + step - 1) / step;
  if (splits > most) splits = most;
  uint64_t len = (cap + splits - 1) / splits;
  len = (len + step - 1) / step * step;
  splits = (cap + len - 1) / len;
  a.split_len = (int)len;
  a.splits = (int)splits;

  cudaSetDevice(ctx->device);
  TempBuffer ws(ctx), sc(ctx);
  void* mem;
  const uint64_t parts = units * splits;
  if ((rc = ws.get(parts * (8 + (uint64_t)p->head_dim * 4), &mem))) return rc;   // (Buffer pointers end here)
  a.part_ml = (float2*)mem;
  a.part_acc = (float*)(a.part_ml + parts);
  a.scores = nullptr;
  if (weights_id) {
    if ((rc = sc.get(units * cap * 4, &mem))) return rc;
    a.scores = (float*)mem;
  }
  const unsigned grid = (unsigned)(base * splits);
  if (wide)
    rc = gt == 1 ? launch_dim<1, true>(ctx, g, a, grid) : gt == 2 ? launch_dim<2, true>(ctx, g, a, grid)
         : gt == 4 ? launch_dim<4, true>(ctx, g, a, grid) : launch_dim<8, true>(ctx, g, a, grid);
  else
    rc = gt == 1 ? launch_dim<1, false>(ctx, g, a, grid) : gt == 2 ? launch_dim<2, false>(ctx, g, a, grid)
         : gt == 4 ? launch_dim<4, false>(ctx, g, a, grid) : launch_dim<8, false>(ctx, g, a, grid);
  if (rc) return rc;
  paged_attention_join_kernel<<<(unsigned)units, 128, 0, ctx->stream>>>(g, a, op);
  LAUNCH_CHECK(ctx, "paged_attention_join_kernel");
  if (weights_id) {
    uint64_t per = (cap + 1023) / 1024;
    paged_attention_weights_kernel<<<(unsigned)(kv_units * per), 256, a.group * sizeof(float2), ctx->stream>>>(
        g, a, wp, owp, (int)per);
    LAUNCH_CHECK(ctx, "paged_attention_weights_kernel");
    ctx_mark_written(ctx, out_weights_id);
  }
  ctx_mark_written(ctx, out_id);
  return TFJS_CUDA_OK;
}
