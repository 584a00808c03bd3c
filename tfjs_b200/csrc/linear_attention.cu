// Linear attention with a decay for each head:
//   S_t = g S_{t-1} + k_t v_t^T,  out_t = scale q_t S_t,  g = exp(log_decay)
// This file: the entry point and the recurrence over the tokens, the state in registers; prompts
// run in chunks (linear_attention_sm100.cu).
#include "linear_attention.h"

namespace {

// Up to here the recurrence, one dependent step a token: 8 / 16 / 32 tokens take 9 / 14 / 25 us for
// 12 states of 64 x 64 and 71 / 128 / 244 us for 1024 of 128 x 128 (ncu durations), where the three launches
// of the chunked form take 24 and 311 for 33 tokens.
constexpr int kFewTokens = 32;
constexpr int kTileV = 32;      // columns of the state that a block holds
constexpr int kRowGroups = 32;  // threads that share a column's rows

// A block holds dim_k x 32 of the state: thread (r, c) rows r, r + 32, ... of four columns.
// Steps are dependent and end in a sum over the block, so this is the form for single
// tokens, where reading and writing the state is all there is.
// WIDE: dim_v and the addresses allow 16-byte accesses.
template <int NR, bool WIDE>
__global__ void __launch_bounds__(256)
linear_recurrent_kernel(const LinearArgs a, int tiles) {
  __shared__ __align__(16) float part[8][kTileV];
  const int unit = blockIdx.x / tiles, tile = blockIdx.x - unit * tiles;
  const int b = unit / a.heads, h = unit - b * a.heads;
  const int n = linear_length(a, b);
  const int r = threadIdx.x >> 3, c0 = tile * kTileV + (threadIdx.x & 7) * 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t s0 = (uint64_t)unit * a.dk * a.dv;
  float s[NR][4];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int row = i * kRowGroups + r;
    const float* p = a.state + s0 + (uint64_t)row * a.dv + c0;
    const bool in = a.state && row < a.dk;
    if (WIDE) {
      const float4 v = in && c0 < a.dv ? __ldg(reinterpret_cast<const float4*>(p)) : make_float4(0.f, 0.f, 0.f, 0.f);
      s[i][0] = v.x;
      s[i][1] = v.y;
      s[i][2] = v.z;
      s[i][3] = v.w;
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) s[i][x] = in && c0 + x < a.dv ? __ldg(p + x) : 0.f;
    }
  }
  // (the next token's values are on their way while a step waits for the sum over the block)
  float v[4], kk[NR], qq[NR];
  auto fetch = [&](uint64_t tok) {
#pragma unroll
    for (int x = 0; x < 4; ++x) v[x] = c0 + x < a.dv ? __ldg(a.v + tok * a.dv + c0 + x) : 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int row = i * kRowGroups + r;
      kk[i] = row < a.dk ? __ldg(a.k + tok * a.dk + row) : 0.f;
      qq[i] = row < a.dk ? __ldg(a.q + tok * a.dk + row) : 0.f;
    }
  };
  if (n > 0) fetch((uint64_t)unit * a.seq);
  const Factor decay = factor_of(decay_power_exact(__ldg(a.log_decay + h), 1));
  for (int t = 0; t < n; ++t) {
    const uint64_t tok = (uint64_t)unit * a.seq + t;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[i][x] = times_plus(decay, s[i][x], kk[i] * v[x]);
        o[x] = fmaf(qq[i], s[i][x], o[x]);
      }
    if (t + 1 < n) fetch(tok + 1);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      o[x] += __shfl_xor_sync(0xffffffffu, o[x], 8);
      o[x] += __shfl_xor_sync(0xffffffffu, o[x], 16);
    }
    if (lane < 8)
#pragma unroll
      for (int x = 0; x < 4; ++x) part[warp][lane * 4 + x] = o[x];
    __syncthreads();
    if (threadIdx.x < kTileV && tile * kTileV + (int)threadIdx.x < a.dv) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) sum += part[w][threadIdx.x];
      if (a.has_scale) sum = __fmul_rn(sum, a.scale);
      a.out[(((uint64_t)b * a.seq + t) * a.heads + h) * a.dv + tile * kTileV + threadIdx.x] = sum;
    }
    __syncthreads();
  }
  for (int t = n + warp; t < a.seq; t += 8)
    if (tile * kTileV + lane < a.dv)
      a.out[(((uint64_t)b * a.seq + t) * a.heads + h) * a.dv + tile * kTileV + lane] = 0.f;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int row = i * kRowGroups + r;
    float* p = a.out_state + s0 + (uint64_t)row * a.dv + c0;
    if (row >= a.dk) continue;
    if (WIDE) {
      if (c0 < a.dv) *reinterpret_cast<float4*>(p) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (c0 + x < a.dv) p[x] = s[i][x];
    }
  }
}

}  // namespace

extern "C" int tfjs_cuda_linear_attention(tfjs_cuda_ctx* ctx, const tfjs_cuda_linear_attention_params* p,
                                          int32_t q_id, int32_t k_id, int32_t v_id,
                                          int32_t log_decay_id, int32_t state_id,
                                          int32_t lengths_id, int32_t out_id,
                                          int32_t out_state_id) {
  if (!ctx) return TFJS_CUDA_INVALID_ARG;
  const char* who = "linear attention";
  if (!p) return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: null parameters", who);
  if (p->batch <= 0 || p->heads <= 0 || p->seq <= 0 || p->dim_k <= 0 || p->dim_v <= 0)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: dimensions must be positive", who);
  const uint64_t units = (uint64_t)p->batch * p->heads;
  if (p->dim_k > 256 || p->dim_v > 256 || units > 0xffffffull || p->seq > 0x7fffff00)
    return ctx_fail(ctx, TFJS_CUDA_UNSUPPORTED,
                    "%s: heads of up to 256 values, fewer than 2^24 rows times heads, tokens below 2^31 - 255", who);
  const uint64_t tokens = units * p->seq, st = units * p->dim_k * p->dim_v * 4;
  Buffer *q, *k, *v, *d, *s = nullptr, *n = nullptr, *out, *os;
  int rc;
  if ((rc = ctx_get(ctx, q_id, tokens * p->dim_k * 4, who, &q))) return rc;
  if ((rc = ctx_get(ctx, k_id, tokens * p->dim_k * 4, who, &k))) return rc;
  if ((rc = ctx_get(ctx, v_id, tokens * p->dim_v * 4, who, &v))) return rc;
  if ((rc = ctx_get(ctx, log_decay_id, (uint64_t)p->heads * 4, who, &d))) return rc;
  if (state_id && (rc = ctx_get(ctx, state_id, st, who, &s))) return rc;
  if (lengths_id && (rc = ctx_get(ctx, lengths_id, (uint64_t)p->batch * 4, who, &n))) return rc;
  if ((rc = ctx_get(ctx, out_id, tokens * p->dim_v * 4, who, &out))) return rc;
  if ((rc = ctx_get(ctx, out_state_id, st, who, &os))) return rc;
  const int32_t in[] = {q_id, k_id, v_id, log_decay_id, state_id, lengths_id};
  for (int32_t x : in)
    if (x && (x == out_id || x == out_state_id))
      return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: an output is also an input", who);
  if (out_id == out_state_id)
    return ctx_fail(ctx, TFJS_CUDA_INVALID_ARG, "%s: an output is given twice", who);
  const Span spans[] = {{out->ptr, tokens * p->dim_v * 4}, {os->ptr, st}, {q->ptr, tokens * p->dim_k * 4},
                        {k->ptr, tokens * p->dim_k * 4}, {v->ptr, tokens * p->dim_v * 4}, {d->ptr, (uint64_t)p->heads * 4},
                        {s ? s->ptr : nullptr, s ? st : 0}, {n ? n->ptr : nullptr, n ? (uint64_t)p->batch * 4 : 0}};
  if ((rc = ctx_apart(ctx, who, spans, 8, 2))) return rc;
  LinearArgs a;
  a.q = (const float*)q->ptr;
  a.k = (const float*)k->ptr;
  a.v = (const float*)v->ptr;
  a.log_decay = (const float*)d->ptr;
  a.state = s ? (const float*)s->ptr : nullptr;
  a.lengths = n ? (const int*)n->ptr : nullptr;
  a.out = (float*)out->ptr;
  a.out_state = (float*)os->ptr;
  a.batch = p->batch;
  a.heads = p->heads;
  a.seq = p->seq;
  a.dk = p->dim_k;
  a.dv = p->dim_v;
  a.has_scale = p->has_scale;
  a.scale = p->scale;
  a.flag = ctx->d_flag;
  cudaSetDevice(ctx->device);
  if (p->seq > kFewTokens) {
    rc = launch_linear_chunked(ctx, a);
    if (rc) return rc;
    ctx_mark_written(ctx, out_id);
    ctx_mark_written(ctx, out_state_id);
    return TFJS_CUDA_OK;
  }
  const int tiles = (p->dim_v + kTileV - 1) / kTileV;
  const unsigned grid = (unsigned)(units * tiles);
  const bool wide = p->dim_v % 4 == 0 && (((uintptr_t)a.state | (uintptr_t)a.out_state) & 15) == 0;
  auto kernel = p->dim_k <= 64    ? (wide ? linear_recurrent_kernel<2, true> : linear_recurrent_kernel<2, false>)
                : p->dim_k <= 128 ? (wide ? linear_recurrent_kernel<4, true> : linear_recurrent_kernel<4, false>)
                                  : (wide ? linear_recurrent_kernel<8, true> : linear_recurrent_kernel<8, false>);
  kernel<<<grid, 256, 0, ctx->stream>>>(a, tiles);
  LAUNCH_CHECK(ctx, "linear_recurrent_kernel");
  ctx_mark_written(ctx, out_id);
  ctx_mark_written(ctx, out_state_id);
  return TFJS_CUDA_OK;
}
