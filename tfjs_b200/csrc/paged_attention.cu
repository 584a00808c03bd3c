// Attention of one new token over a paged key-value cache:
//   s_j = q . k_j * scale + mask_j,  p = softmax(s),  out = sum_j p_j v_j
// Every key and value is read once and takes 4 G operations a byte pair of it (G query heads
// share a key-value head), so memory bounds it.  A row's slots are split over blocks
// (and a block's slots over its warps), each keeps a running maximum, sum and weighted
// sum of values, and a second kernel joins them.
//
// The rows of one page and head are contiguous, so tiles of keys and values travel as bulk
// copies into a ring in shared memory, issued by a warp of their own and several tiles ahead of
// the four warps that compute: the bytes in flight do not depend on registers.  Head sizes that
// are no multiple of four values (rows not on 16 bytes) take a kernel with plain loads.
#include "paged.cuh"
#include "ptx.cuh"

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
  float* out;             // [batch * heads][head_dim], written here when there is one split
  int slots;              // bulk kernel: tiles of the ring
};

// e^(x - m) for a maximum that may be -infinity (nothing seen yet: 0)
__device__ __forceinline__ float exp_from(float x, float m) {
  return exp2_approx(__fmul_rn(__fsub_rn(x, m == -INFINITY ? 0.0f : m), kLog2e));
}

__device__ __forceinline__ float4 load4(const float* p, int d, int dim) {
  float4 r;
  r.x = d < dim ? __ldg(p + d) : 0.f;
  r.y = d + 1 < dim ? __ldg(p + d + 1) : 0.f;
  r.z = d + 2 < dim ? __ldg(p + d + 2) : 0.f;
  r.w = d + 3 < dim ? __ldg(p + d + 3) : 0.f;
  return r;
}

// The block's partial results: the warps' (maximum, sum) [kWarps][GT] and weighted sums
// [kWarps][GT][DM] joined, and written as a part, or as the result when there is only one.
template <int DM, int GT>
__device__ __forceinline__ void write_partial(const PagedLayout& g, const PagedAttnArgs& a, const float2* ml,
                                              const float* acc, int tid, int threads, int b, int head0,
                                              int live, int split) {
  for (int i = tid; i < GT * DM; i += threads) {
    const int gi = i / DM, d = i - gi * DM;
    if (gi >= live || d >= g.head_dim) continue;
    float mx = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml[w * GT + gi].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp_from(ml[w * GT + gi].x, mx);
      sum = fmaf(ml[w * GT + gi].y, f, sum);
      o = fmaf(acc[(w * GT + gi) * DM + d], f, o);
    }
    const uint64_t head = (uint64_t)b * a.heads + head0 + gi;
    const uint64_t part = head * a.splits + split;
    if (a.splits == 1)
      a.out[head * g.head_dim + d] = sum == 0.f ? 0.f : __fdiv_rn(o, sum);
    else
      a.part_acc[part * g.head_dim + d] = o;
    if (d == 0) a.part_ml[part] = make_float2(mx, sum);
  }
}

// What a block works on.
struct Piece {
  int b, h, split, head0, live, begin, end;
};
template <int GT>
__device__ __forceinline__ bool piece_of(const PagedLayout& g, const PagedAttnArgs& a, Piece& p) {
  int u = blockIdx.x;
  p.split = u % a.splits;
  u /= a.splits;
  const int gc = u % a.group_chunks;
  u /= a.group_chunks;
  p.h = u % g.kv_heads;
  p.b = u / g.kv_heads;
  const int n = paged_length(g, p.b);
  p.begin = p.split * a.split_len;
  p.end = min(n, p.begin + a.split_len);
  p.head0 = p.h * a.group + gc * GT;             // first query head
  p.live = min(GT, a.group - gc * GT);           // of GT, real ones
  return p.begin < p.end || p.split == 0;        // (the join does not read an empty later split)
}

// ---- bulk copies ---------------------------------------------------------------------------
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

constexpr int kBulkThreads = (kWarps + 1) * 32;
constexpr int kMaxSlots = 8;

// Shared memory: ring, queries [GT][DM], probabilities [warps][slots of a warp][GT], barriers.
template <int DM, int GT, int SUB>
constexpr int bulk_fixed_bytes() {
  return GT * DM * 4 + kWarps * SUB * 8 * GT * 4 + kWarps * GT * 8 + 2 * kMaxSlots * 8 + 128;
}

// A tile is 8 SUB slots for each of the four computing warps; the ring holds tiles of keys and
// of values in turn.  Scores: four lanes a slot, each 16-byte pieces of the key 64 bytes apart,
// eight slots at a time; odd slots take the pieces in another order, so that the two slots that
// a quarter of a warp reads lie in different banks (head sizes are mostly multiples of 32 values).
// Values: lanes along head_dim, a weighted sum in registers.
template <int DM, int GT, int SUB>
__global__ void __launch_bounds__(kBulkThreads)
paged_attention_bulk_kernel(const PagedLayout g, const PagedAttnArgs a) {
  constexpr int TW = 8 * SUB;                    // slots of a warp
  constexpr int T = kWarps * TW;
  constexpr int LPR = DM / 4 < 32 ? DM / 4 : 32; // lanes that share a value row
  constexpr int VR = DM / 4 / LPR;               // 4-value pieces of it a lane holds
  constexpr int TPI = 32 / LPR;                  // value rows a warp reads at a time
  extern __shared__ __align__(128) uint8_t smem[];
  Piece pc;
  if (!piece_of<GT>(g, a, pc)) return;
  const int D = g.head_dim;
  const uint32_t tile_bytes = (uint32_t)(T * D * 4);
  const uint32_t ring_bytes = (uint32_t)a.slots * tile_bytes;
  float* q_s = reinterpret_cast<float*>(smem + ring_bytes);
  float* p_all = q_s + GT * DM;
  float2* ml_s = reinterpret_cast<float2*>(p_all + kWarps * TW * GT);
  const uint32_t bars = smem_u32(ml_s + kWarps * GT);
  auto full = [&](int s) { return bars + 8u * (uint32_t)s; };
  auto empty = [&](int s) { return bars + 8u * (uint32_t)(kMaxSlots + s); };
  const uint32_t ring = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < a.slots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = tid; i < GT * DM; i += kBulkThreads) {
    const int gi = i / DM, d = i - gi * DM;
    q_s[i] = gi < pc.live && d < D ? __ldg(a.q + ((uint64_t)pc.b * a.heads + pc.head0 + gi) * D + d) : 0.f;
  }
  __syncthreads();
  const int tiles = pc.begin < pc.end ? (pc.end - pc.begin + T - 1) / T : 0;

  if (warp == kWarps) {
    // ------------------------------------------------------------------ producer --
    int used = 0;
    bool alive = true;
    for (int t = 0; alive && t < tiles; ++t) {
      const int first = pc.begin + t * T, last = min(first + T, pc.end);
      const int page0 = g.page_shift >= 0 ? first >> g.page_shift : first / g.page_size;
      const int page1 = g.page_shift >= 0 ? (last - 1) >> g.page_shift : (last - 1) / g.page_size;
      for (int kv = 0; kv < 2; ++kv, ++used) {
        const int s = used % a.slots;
        if (!warp_wait(empty(s), ((used / a.slots) & 1) ^ 1)) {
          if (lane == 0) atomicExch(g.flag, 1);
          alive = false;
          break;
        }
        const float* pool = kv ? a.v_cache : a.k_cache;
        // every lane one page after the other: how much of it is there, then the copies
        for (int pass = 0; pass < 2; ++pass) {
          uint32_t bytes = 0;
          for (int pi = page0 + lane; pi <= page1; pi += 32) {
            const int from = max(first, pi * g.page_size), to = min(last, (pi + 1) * g.page_size);
            const uint32_t row = paged_row(g, pc.b, pc.h, from);
            if (row == kNoRow) continue;
            const uint32_t n = (uint32_t)(to - from) * (uint32_t)(D * 4);
            if (pass)
              bulk_copy(ring + (uint32_t)s * tile_bytes + (uint32_t)(from - first) * (uint32_t)(D * 4),
                        pool + (uint64_t)row * D, n, full(s));
            bytes += n;
          }
          if (pass == 0) {
            for (int o = 16; o; o >>= 1) bytes += __shfl_xor_sync(0xffffffffu, bytes, o);
            if (lane == 0) mbar_expect_tx(full(s), bytes);
            __syncwarp();
          }
        }
      }
    }
    if (!alive)   // copies in flight must land before the block's memory goes away
      for (int u = used - a.slots > 0 ? used - a.slots : 0; u < used; ++u)
        warp_wait(full(u % a.slots), (u / a.slots) & 1);
  } else {
    // ------------------------------------------------------------------ computing --
    float m[GT], l[GT];
    float4 acc[GT][VR];
#pragma unroll
    for (int gi = 0; gi < GT; ++gi) {
      m[gi] = -INFINITY;
      l[gi] = 0.f;
#pragma unroll
      for (int r = 0; r < VR; ++r) acc[gi][r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float* p_s = p_all + warp * TW * GT;
    const int c = lane & 3, tok = lane >> 2;
    const int steps = ((D + 31) / 32) * 2;       // of 16 values; even
    for (int t = 0; t < tiles; ++t) {
      const int t0 = pc.begin + t * T + warp * TW;
      // lane j looks after slot t0 + j: is it there, and what does the mask add to it
      const int mine = t0 + lane;
      float add = 0.f;
      bool there = lane < TW && mine < pc.end;
      if (there) {
        const int pi = g.page_shift >= 0 ? mine >> g.page_shift : mine / g.page_size;
        there = (unsigned)__ldg(g.table + (size_t)pc.b * g.max_pages + pi) < (unsigned)g.num_pages;
        if (a.mask) {
          add = __ldg(a.mask + (uint64_t)pc.b * g.capacity + mine);
          there = there && add != -INFINITY;     // hidden: what it holds, NaN included, does not count
        }
      }
      const uint32_t seen = __ballot_sync(0xffffffffu, there);
      const int ks = (2 * t) % a.slots, vs = (2 * t + 1) % a.slots;
      if (!warp_wait(full(ks), ((2 * t) / a.slots) & 1)) {
        if (lane == 0) atomicExch(g.flag, 2);
        break;
      }
      float s[GT][SUB];
#pragma unroll
      for (int gi = 0; gi < GT; ++gi)
#pragma unroll
        for (int x = 0; x < SUB; ++x) s[gi][x] = 0.f;
      const float* kt = reinterpret_cast<const float*>(smem + (uint32_t)ks * tile_bytes) + (warp * TW + tok) * D;
#pragma unroll 4
      for (int i = 0; i < steps; ++i) {
        const int d = ((i ^ (tok & 1)) * 4 + c) * 4;
        float4 kv[SUB];
#pragma unroll
        for (int x = 0; x < SUB; ++x)
          kv[x] = d < D ? *reinterpret_cast<const float4*>(kt + x * 8 * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int gi = 0; gi < GT; ++gi) {
          const float4 qv = *reinterpret_cast<const float4*>(q_s + gi * DM + d);
#pragma unroll
          for (int x = 0; x < SUB; ++x)
            s[gi][x] = fmaf(qv.w, kv[x].w, fmaf(qv.z, kv[x].z, fmaf(qv.y, kv[x].y, fmaf(qv.x, kv[x].x, s[gi][x]))));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(ks));
      float add_x[SUB];
#pragma unroll
      for (int x = 0; x < SUB; ++x) add_x[x] = __shfl_sync(0xffffffffu, add, x * 8 + tok);
#pragma unroll
      for (int gi = 0; gi < GT; ++gi) {
        float mx = m[gi], own = -INFINITY;
#pragma unroll
        for (int x = 0; x < SUB; ++x) {
          float v = s[gi][x];
          v += __shfl_xor_sync(0xffffffffu, v, 1);
          v += __shfl_xor_sync(0xffffffffu, v, 2);
          if (a.has_scale) v = __fmul_rn(v, a.scale);
          if (a.mask) v = __fadd_rn(v, add_x[x]);
          if (!(seen >> (x * 8 + tok) & 1u)) v = -INFINITY;
          if (c == x) own = v;                   // lane c of a slot's four keeps slot c * 8 + tok
          mx = fmaxf(mx, v);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        if (mx != m[gi]) {                       // (the same for the whole warp)
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
        }
        if (c < SUB) {
          const float p = exp_from(own, mx);
          l[gi] += p;
          p_s[(c * 8 + tok) * GT + gi] = p;
          const int slot = t0 + c * 8 + tok;
          if (a.scores && gi < pc.live && slot < pc.end)
            a.scores[((uint64_t)pc.b * a.heads + pc.head0 + gi) * g.capacity + slot] = own;
        }
      }
      __syncwarp();
      if (!warp_wait(full(vs), ((2 * t + 1) / a.slots) & 1)) {
        if (lane == 0) atomicExch(g.flag, 3);
        break;
      }
      const float* vt = reinterpret_cast<const float*>(smem + (uint32_t)vs * tile_bytes) + (warp * TW) * D;
      const bool all = seen == (TW == 32 ? 0xffffffffu : (1u << TW) - 1u);
#pragma unroll 4
      for (int it = 0; it < TW / TPI; ++it) {
        const int row = it * TPI + lane / LPR;
        float4 v[VR];
#pragma unroll
        for (int r = 0; r < VR; ++r) {
          const int d = (r * LPR + lane % LPR) * 4;
          v[r] = d < D && (all || (seen >> row & 1u)) ? *reinterpret_cast<const float4*>(vt + row * D + d)
                                                      : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float p[GT];
        if constexpr (GT >= 4) {
#pragma unroll
          for (int gi = 0; gi < GT; gi += 4)
            *reinterpret_cast<float4*>(p + gi) = *reinterpret_cast<const float4*>(p_s + row * GT + gi);
        } else {
#pragma unroll
          for (int gi = 0; gi < GT; ++gi) p[gi] = p_s[row * GT + gi];
        }
#pragma unroll
        for (int gi = 0; gi < GT; ++gi)
#pragma unroll
          for (int r = 0; r < VR; ++r) {
            acc[gi][r].x = fmaf(p[gi], v[r].x, acc[gi][r].x);
            acc[gi][r].y = fmaf(p[gi], v[r].y, acc[gi][r].y);
            acc[gi][r].z = fmaf(p[gi], v[r].z, acc[gi][r].z);
            acc[gi][r].w = fmaf(p[gi], v[r].w, acc[gi][r].w);
          }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(vs));
    }
    // across the lanes, then (in the ring's memory) across the warps
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
      if (lane == 0) ml_s[warp * GT + gi] = make_float2(m[gi], l[gi]);
    }
    // all computing warps are done with the ring
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    float* acc_s = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int gi = 0; gi < GT; ++gi)
      if (lane < LPR)
#pragma unroll
        for (int r = 0; r < VR; ++r)
          *reinterpret_cast<float4*>(acc_s + (warp * GT + gi) * DM + (r * LPR + lane) * 4) = acc[gi][r];
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    write_partial<DM, GT>(g, a, ml_s, acc_s, tid, kWarps * 32, pc.b, pc.head0, pc.live, pc.split);
  }
}

// ---- plain loads -----------------------------------------------------------------------------
// Rows that are not on 16 bytes.  DM: head_dim rounded up; GT: query heads of one key-value head that a block serves.
template <int DM, int GT>
__global__ void __launch_bounds__(kWarps * 32)
paged_attention_loads_kernel(const PagedLayout g, const PagedAttnArgs a) {
  constexpr int NI = DM / 16;                    // steps of 16 values of a key, 4 a lane
  constexpr int LPR = DM / 4 < 32 ? DM / 4 : 32; // lanes that share a value row
  constexpr int VR = DM / 4 / LPR;               // 4-value pieces of it a lane holds
  constexpr int TPI = 32 / LPR;                  // value rows a warp reads at a time
  __shared__ __align__(16) float q_s[GT][DM];
  __shared__ float p_s[kWarps][kTile][GT];
  __shared__ float2 ml_s[kWarps][GT];
  __shared__ __align__(16) float acc_s[kWarps][GT][DM];
  Piece pc;
  if (!piece_of<GT>(g, a, pc)) return;
  const int b = pc.b, h = pc.h, split = pc.split, begin = pc.begin, end = pc.end, head0 = pc.head0, live = pc.live;
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
        kv[x] = row[x] != kNoRow ? load4(kp[x], d, g.head_dim) : make_float4(0.f, 0.f, 0.f, 0.f);
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
      for (int r = 0; r < VR; ++r) v[r] = load4(vp, (r * LPR + lane % LPR) * 4, g.head_dim);
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
  write_partial<DM, GT>(g, a, &ml_s[0][0], &acc_s[0][0][0], tid, kWarps * 32, b, head0, live, split);
}

// Splits that row b's slots fill (at least one, which is empty for an empty row).
__device__ __forceinline__ int live_splits(const PagedLayout& g, const PagedAttnArgs& a, int b) {
  const int n = paged_length(g, b);
  return max(1, (n + a.split_len - 1) / a.split_len);
}

__global__ void __launch_bounds__(128)
paged_attention_join_kernel(const PagedLayout g, const PagedAttnArgs a) {
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
    a.out[(uint64_t)unit * g.head_dim + d] = sum == 0.f ? 0.f : __fdiv_rn(o, sum);
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

// The ring: tiles of at most 32 KB, and as many as fit twice into an SM's shared memory (more
// than two blocks an SM where they are small).
template <int DM, int GT>
int launch_bulk(tfjs_cuda_ctx* ctx, const PagedLayout& g, PagedAttnArgs& a, unsigned grid) {
  constexpr int SUB = DM <= 128 ? 2 : 1;
  constexpr int fixed = bulk_fixed_bytes<DM, GT, SUB>();
  const int tile = kWarps * 8 * SUB * g.head_dim * 4;
  a.slots = (113 * 1024 - fixed) / tile;
  if (a.slots > 4) a.slots = 4;
  const int acc = kWarps * GT * DM * 4;
  const int bytes = (a.slots * tile > acc ? a.slots * tile : acc) + fixed;
  CUDA_TRY(ctx, cudaFuncSetAttribute(paged_attention_bulk_kernel<DM, GT, SUB>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  paged_attention_bulk_kernel<DM, GT, SUB><<<grid, kBulkThreads, bytes, ctx->stream>>>(g, a);
  LAUNCH_CHECK(ctx, "paged_attention_bulk_kernel");
  return TFJS_CUDA_OK;
}
template <int GT>
int launch_bulk(tfjs_cuda_ctx* ctx, const PagedLayout& g, PagedAttnArgs& a, unsigned grid) {
  if (g.head_dim <= 32) return launch_bulk<32, GT>(ctx, g, a, grid);
  if (g.head_dim <= 64) return launch_bulk<64, GT>(ctx, g, a, grid);
  if (g.head_dim <= 128) return launch_bulk<128, GT>(ctx, g, a, grid);
  return launch_bulk<256, GT>(ctx, g, a, grid);
}
template <int DM, int GT>
int launch_loads(tfjs_cuda_ctx* ctx, const PagedLayout& g, const PagedAttnArgs& a, unsigned grid) {
  paged_attention_loads_kernel<DM, GT><<<grid, kWarps * 32, 0, ctx->stream>>>(g, a);
  LAUNCH_CHECK(ctx, "paged_attention_loads_kernel");
  return TFJS_CUDA_OK;
}
template <int GT>
int launch_loads(tfjs_cuda_ctx* ctx, const PagedLayout& g, const PagedAttnArgs& a, unsigned grid) {
  if (g.head_dim <= 32) return launch_loads<32, GT>(ctx, g, a, grid);
  if (g.head_dim <= 64) return launch_loads<64, GT>(ctx, g, a, grid);
  if (g.head_dim <= 128) return launch_loads<128, GT>(ctx, g, a, grid);
  return launch_loads<256, GT>(ctx, g, a, grid);
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
  a.out = (float*)out->ptr;
  a.slots = 0;
  const float* wp = w ? (const float*)w->ptr : nullptr;
  float* owp = ow ? (float*)ow->ptr : nullptr;

  const bool wide = p->head_dim % 4 == 0 && (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) == 0;
  const int gt = a.group == 1 ? 1 : !wide ? 8 : a.group == 2 ? 2 : a.group <= 4 ? 4 : 8;
  a.group_chunks = (a.group + gt - 1) / gt;
  // Splits: about four blocks for each of the two an SM holds (rows are ragged, and a block that
  // finds nothing to do leaves at once), but one full wave where the rows and heads alone do
  // not fill it: each split then is as long as can be.  At least one tile a warp.
  const uint64_t base = kv_units * a.group_chunks, wave = (uint64_t)ctx->sm_count * 2;
  const int step = kWarps * kTile;
  uint64_t splits = base * 4 <= wave ? wave / base : (wave * 4 + base - 1) / base;
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
    rc = gt == 1   ? launch_bulk<1>(ctx, g, a, grid)
         : gt == 2 ? launch_bulk<2>(ctx, g, a, grid)
         : gt == 4 ? launch_bulk<4>(ctx, g, a, grid)
                   : launch_bulk<8>(ctx, g, a, grid);
  else
    rc = gt == 1 ? launch_loads<1>(ctx, g, a, grid) : launch_loads<8>(ctx, g, a, grid);
  if (rc) return rc;
  if (splits > 1) {
    paged_attention_join_kernel<<<(unsigned)units, 128, 0, ctx->stream>>>(g, a);
    LAUNCH_CHECK(ctx, "paged_attention_join_kernel");
  }
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
