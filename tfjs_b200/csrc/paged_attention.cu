// Attention of one new token over a paged key-value cache:
//   s_j = q . k_j * scale + mask_j,  p = softmax(s),  out = sum_j p_j v_j
// Every value of the cache is read once and takes 2 G operations (G query heads share a key-value
// head), so memory bounds it: 100003 slots of 8 heads of 128 (819 MB) take 133 us, 6.2 TB/s, 0.95 of a copy's.
// (Read once for each 16 query heads where more of them share a key-value head, for each 8 in the form with
// plain loads; those groups are not bound by memory.  Slots that the mask hides are read like the others.)
//
// Work: the slots of every row and head are cut into tiles, all tiles are numbered through, and
// each block takes an equal share of them, whatever the rows' lengths (a share may begin and end
// inside a row).  A row and head that several blocks work on is joined by a second kernel from
// their maxima, sums and weighted sums of values; otherwise the block writes the result.
//
// The rows of one page and head are contiguous, so tiles of keys and values travel as bulk
// copies into a ring in shared memory, issued by a warp of their own and several tiles ahead of
// the warps that compute: the bytes in flight do not depend on registers.  Head sizes that
// are no multiple of four values (rows not on 16 bytes) take a kernel with plain loads: 16 rows of 4096 slots
// of 8 heads of 127 take 187 us with one query head each and 385 with four, where 128 and four take 104.
//
// Arithmetic, for up to 4 query heads a key-value head: fp32 multiply-adds.  For more, the
// multiply-adds and the sums across lanes took four times as long as memory (8 heads of 64: 321 us
// where the bytes take 93; 138 with MMAs, whose 16 rows half a group of 4 would leave empty:
// 196 against 148 us with 4 heads of 128), so the products run as m16n8k8 TF32 MMAs with each operand split into
// two TF32 parts and three products (fp32 accuracy; the single query row of a decode step has no
// tile for the 128-row tcgen05 form); with up to 8 heads both parts of the queries, or of the
// probabilities, are the 16 rows of one.  Tensor cores cut sums off instead of rounding them, so
// sums over a tile start from zero and are added to fp32 registers.  What holds this form back is shared
// memory: rows of a tile lie a multiple of 128 bytes apart, so that the lanes of a load that have equal
// columns of different rows read one bank, four of them for values and two for keys.  Heads of 256 spill
// registers from 9 query heads on: 16 rows of 4096 slots, 4 key-value heads of 256, take 137 us with 8 query
// heads each and 361 with 16 (heads of 128 with 16: 96).
#include "paged.cuh"
#include "ptx.cuh"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4;            // that compute with plain loads

struct PagedAttnArgs {
  const float* q;         // [batch, heads, head_dim]
  const float* k_cache;
  const float* v_cache;
  const float* mask;      // [batch, capacity], or null
  float* out;             // [batch * heads][head_dim]
  float* part_acc;        // [parts][heads of a block][head_dim]
  float2* part_ml;        // [parts][heads of a block]: maximum, sum
  float* scores;          // [batch * heads][capacity], or null: the scores are not kept
  int batch, heads, group, group_chunks;
  int chunk;              // query heads of a block
  int tile;               // slots of a tile
  int shares;             // blocks
  int whole;              // a share is one row and head
  int has_scale;
  float scale;
  int slots;              // bulk kernel: tiles of the ring
};

// e^(x - m) for a maximum that may be -infinity (nothing seen yet: 0)
__device__ __forceinline__ float exp_from(float x, float m) {
  return exp2_approx(__fmul_rn(__fsub_rn(x, m == -INFINITY ? 0.0f : m), kLog2e));
}

// ---- shares --------------------------------------------------------------------------------
// Units are (row, key-value head, chunk of its query heads); a unit has a tile per `tile` slots,
// at least one.  Tiles are numbered unit by unit; share i is tiles [i size, (i + 1) size).
__device__ __forceinline__ int row_tiles(const PagedLayout& g, const PagedAttnArgs& a, int b) {
  const int n = paged_length(g, b);
  return n == 0 ? 1 : (n - 1) / a.tile + 1;
}
struct Shares {
  long long size;          // tiles of a share
  long long before;        // tiles of the rows in front of a row, per unit of a row
  int row;                 // that row
};
// A whole warp: the share size, and either the tiles in front of row `row` (find < 0) or the
// row in which tile `find * size` lies.
__device__ __forceinline__ Shares shares_of(const PagedLayout& g, const PagedAttnArgs& a, int row, int find) {
  const int lane = threadIdx.x & 31;
  const int per_row = g.kv_heads * a.group_chunks;
  Shares r;
  r.row = row;
  r.before = 0;
  if (a.whole) {
    r.size = 1;            // (in units; not used)
    return r;
  }
  long long total = 0, before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    long long t = b < a.batch ? row_tiles(g, a, b) : 0;
    long long lower = b < row ? t : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      t += __shfl_xor_sync(0xffffffffu, t, o);
      lower += __shfl_xor_sync(0xffffffffu, lower, o);
    }
    total += t;
    before += lower;
  }
  r.size = (total * per_row + a.shares - 1) / a.shares;
  if (find < 0) {
    r.before = before;
    return r;
  }
  const long long at = (long long)find * r.size;
  long long sum = 0;
  r.row = a.batch;         // behind the last tile
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    const long long t = b < a.batch ? row_tiles(g, a, b) : 0;
    long long incl = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, b < a.batch && at < (sum + incl) * per_row);
    if (hit) {
      const int src = __ffs(hit) - 1;
      r.row = b0 + src;
      r.before = sum + __shfl_sync(0xffffffffu, incl - t, src);
      break;
    }
    sum += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

// The pieces of a block's share, one unit after the other.
struct Piece {
  int b, h, head0, live;   // row, key-value head, first query head, query heads
  int begin, end;          // slots
  int tiles;
  int part;                // where its partial results go
  bool complete;           // all of the unit's slots
};
struct Walk {
  long long left;          // tiles
  long long off;           // tiles of the unit in front
  int b, hc;
  __device__ __forceinline__ void init(const PagedLayout& g, const PagedAttnArgs& a) {
    const int per_row = g.kv_heads * a.group_chunks;
    if (a.whole) {
      b = blockIdx.x / per_row;
      hc = blockIdx.x - b * per_row;
      off = 0;
      left = row_tiles(g, a, b);
      return;
    }
    const Shares s = shares_of(g, a, 0, (int)blockIdx.x);
    b = s.row;
    left = 0;
    if (b >= a.batch) return;
    const long long t = row_tiles(g, a, b), at = (long long)blockIdx.x * s.size - s.before * per_row;
    hc = (int)(at / t);
    off = at - hc * t;
    left = s.size;
  }
  __device__ __forceinline__ bool next(const PagedLayout& g, const PagedAttnArgs& a, Piece& p) {
    if (left <= 0 || b >= a.batch) return false;
    const int per_row = g.kv_heads * a.group_chunks;
    const long long t = row_tiles(g, a, b);
    const long long take = left < t - off ? left : t - off;
    const int n = paged_length(g, b);
    const int gc = hc % a.group_chunks;
    p.b = b;
    p.h = hc / a.group_chunks;
    p.head0 = p.h * a.group + gc * a.chunk;
    p.live = min(a.chunk, a.group - gc * a.chunk);
    p.begin = (int)(off * a.tile);
    p.end = (int)((off + take) * a.tile < n ? (off + take) * a.tile : n);
    p.tiles = p.begin < p.end ? (int)take : 0;
    p.part = (a.whole ? 0 : (int)blockIdx.x) + b * per_row + hc;   // (one more with every block and every unit)
    p.complete = off == 0 && take == t;
    left -= take;
    off = 0;
    if (++hc == per_row) {
      hc = 0;
      ++b;
    }
    return true;
  }
};

// The joined results of a piece: d of query head gi of its chunk.
template <int GT>
__device__ __forceinline__ void write_result(const PagedLayout& g, const PagedAttnArgs& a, const Piece& p, int gi,
                                             int d, float o, float m, float l) {
  if (gi >= p.live || d >= g.head_dim) return;
  if (p.complete)
    a.out[((uint64_t)p.b * a.heads + p.head0 + gi) * g.head_dim + d] = l == 0.f ? 0.f : __fdiv_rn(o, l);
  else
    a.part_acc[((uint64_t)p.part * GT + gi) * g.head_dim + d] = o;
  if (d == 0) a.part_ml[(uint64_t)p.part * GT + gi] = make_float2(m, l);
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
template <int NW>
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(NW * 32) : "memory"); }

constexpr int kMaxSlots = 8;
// Warps that compute and blocks of an SM.  The MMA form of small heads is bound by the latency of its
// instructions, so it has 16 warps on an SM.
constexpr int compute_warps(int dm, int gt, bool mma) { return mma && gt == 8 && dm <= 64 ? 8 : 4; }
constexpr int blocks_per_sm(int dm, int gt, bool mma) { return dm <= 64 && compute_warps(dm, gt, mma) == 4 ? 3 : 2; }

// x = hi + lo, hi rounded to TF32's 11 bits
__device__ __forceinline__ float tf32_hi(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
}
// d += a b for a 16 x 8 (rows lane / 4 and + 8, columns lane % 4 and + 4), b 8 x 8, d 16 x 8
__device__ __forceinline__ void mma_tf32(float (&d)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// Slots of a warp's share of a tile, and shared memory beside the ring: queries, probabilities
// (multiply-add form), places for the joining of the warps, their maxima and sums, barriers.
template <int DM>
constexpr int warp_slots() { return DM <= 128 ? 16 : 8; }
template <int DM, int GT, bool MMA>
constexpr int query_floats() { return MMA ? DM * 8 * (GT == 16 ? 4 : 2) : GT * DM; }
template <int DM, int GT, bool MMA>
constexpr int bulk_fixed_bytes() {
  constexpr int NW = compute_warps(DM, GT, MMA);
  return query_floats<DM, GT, MMA>() * 4 + (MMA ? 0 : NW * warp_slots<DM>() * GT * 4) + NW / 2 * GT * DM * 4 +
         NW * GT * 8 + 2 * kMaxSlots * 8 + 128;
}

// One warp's computing state, multiply-add form.  Scores: four lanes a slot, each 16-byte pieces
// of the key 64 bytes apart, eight slots at a time; odd slots take the pieces in another order, so
// that the two slots that a quarter of a warp reads lie in different banks.  Values: lanes along
// head_dim.
template <int DM, int GT>
struct FmaState {
  static constexpr int TW = warp_slots<DM>(), SUB = TW / 8;
  static constexpr int LPR = DM / 4 < 32 ? DM / 4 : 32;   // lanes that share a value row
  static constexpr int VR = DM / 4 / LPR;                 // 4-value pieces of it a lane holds
  static constexpr int TPI = 32 / LPR;                    // value rows a warp reads at a time
  float m[GT], l[GT];
  float4 acc[GT][VR];
  float* p_s;

  __device__ __forceinline__ static void load_queries(const PagedLayout& g, const PagedAttnArgs& a, const Piece& p,
                                                      float* q_s, int tid) {
    for (int i = tid; i < GT * DM; i += compute_warps(DM, GT, false) * 32) {
      const int gi = i / DM, d = i - gi * DM;
      q_s[i] = gi < p.live && d < g.head_dim
                   ? __ldg(a.q + ((uint64_t)p.b * a.heads + p.head0 + gi) * g.head_dim + d) : 0.f;
    }
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int gi = 0; gi < GT; ++gi) {
      m[gi] = -INFINITY;
      l[gi] = 0.f;
#pragma unroll
      for (int r = 0; r < VR; ++r) acc[gi][r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  // scores of the warp's slots from t0 on; `seen`: which are there; add: lane j's mask for slot j
  float s[GT][SUB];
  __device__ __forceinline__ void scores(const float* kt, const float* q_s, int D, int lane) {
    const int c = lane & 3, tok = lane >> 2;
    kt += tok * D;
#pragma unroll
    for (int gi = 0; gi < GT; ++gi)
#pragma unroll
      for (int x = 0; x < SUB; ++x) s[gi][x] = 0.f;
    const int steps = ((D + 31) / 32) * 2;                // of 16 values; even
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
  }
  __device__ __forceinline__ void softmax(const PagedLayout& g, const PagedAttnArgs& a, const Piece& pc, int t0,
                                          uint32_t seen, float add, int lane) {
    const int c = lane & 3, tok = lane >> 2;
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
        if (c == x) own = v;                              // lane c of a slot's four keeps slot c * 8 + tok
        mx = fmaxf(mx, v);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      if (mx != m[gi]) {                                  // (the same for the whole warp)
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
  }
  __device__ __forceinline__ void values(const float* vt, int D, uint32_t seen, int lane) {
    const bool all = seen == (1u << TW) - 1u;
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
      float p_row[GT];
      if constexpr (GT == 4)
        *reinterpret_cast<float4*>(p_row) = *reinterpret_cast<const float4*>(p_s + row * GT);
      else
#pragma unroll
        for (int gi = 0; gi < GT; ++gi) p_row[gi] = p_s[row * GT + gi];
#pragma unroll
      for (int gi = 0; gi < GT; ++gi) {
        const float p = p_row[gi];
#pragma unroll
        for (int r = 0; r < VR; ++r) {
          acc[gi][r].x = fmaf(p, v[r].x, acc[gi][r].x);
          acc[gi][r].y = fmaf(p, v[r].y, acc[gi][r].y);
          acc[gi][r].z = fmaf(p, v[r].z, acc[gi][r].z);
          acc[gi][r].w = fmaf(p, v[r].w, acc[gi][r].w);
        }
      }
    }
    __syncwarp();                                         // (p_s is rewritten by the next tile)
  }
  // sums across the lanes; afterwards lane 0 holds m and l, lanes < LPR the sums
  __device__ __forceinline__ void finish(float2* ml, int lane) {
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
      if (lane == 0) ml[gi] = make_float2(m[gi], l[gi]);
    }
  }
  // f(head of the chunk, first d of a pair, value, value)
  template <typename F>
  __device__ __forceinline__ void each(int lane, F f) {
#pragma unroll
    for (int gi = 0; gi < GT; ++gi)
#pragma unroll
      for (int r = 0; r < VR; ++r)
        if (lane < LPR) {
          const int d = (r * LPR + lane) * 4;
          f(gi, d, acc[gi][r].x, acc[gi][r].y);
          f(gi, d + 2, acc[gi][r].z, acc[gi][r].w);
        }
  }
};

// The same with MMAs: rows are query heads (lane / 4 and, for 16 of them, + 8), a lane's columns
// of the scores are slots 2 c and 2 c + 1 of each eight (c = lane % 4), which is also how the
// probabilities enter the second product: its K index c stands for slot 2 c and c + 4 for
// 2 c + 1.  In the first product K index c and c + 4 of steps 2 i and 2 i + 1 stand for values
// 16 i + 4 c + 0 .. 3, one 16-byte load.  In the second, column n of MMA e of a block of 32
// values stands for value 4 n + e, again one load.
template <int DM, int GT>
struct MmaState {
  static constexpr int TW = warp_slots<DM>(), NT = TW / 8;
  static constexpr int R = GT / 8;                        // heads of a lane
  static constexpr int JB = DM / 32;
  float m[R], l[R];
  float acc[JB][4][2 * R];                                // [block][MMA][head, column 2 c + x]
  float s[NT][2 * R];                                     // scores, then probabilities

  // [step of 8][lane][hi (row, K c), hi (row, K c + 4), then row + 8, then lo the same]
  __device__ __forceinline__ static void load_queries(const PagedLayout& g, const PagedAttnArgs& a, const Piece& p,
                                                      float* q_s, int tid) {
    for (int i = tid; i < GT * DM; i += compute_warps(DM, GT, true) * 32) {
      const int gi = i / DM, d = i - gi * DM;
      const float x = gi < p.live && d < g.head_dim
                          ? __ldg(a.q + ((uint64_t)p.b * a.heads + p.head0 + gi) * g.head_dim + d) : 0.f;
      const float hi = tf32_hi(x);
      const int j = d & 15, step = (d >> 4) * 2 + ((j >> 1) & 1);
      float* to = q_s + (step * 32 + (gi & 7) * 4 + (j >> 2)) * (4 * R) + (gi >> 3) * 2 + (j & 1);
      to[0] = hi;
      to[2 * R] = x - hi;
    }
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 2 * R; ++x) acc[j][e][x] = 0.f;
  }
  __device__ __forceinline__ void scores(const float* kt, const float* q_s, int D, int lane) {
    const int c = lane & 3, tok = lane >> 2;
    kt += tok * D + c * 4;
    q_s += lane * (4 * R);
    float hi[NT][4], lo[NT][4];                           // large and small products apart
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 4; ++x) hi[t][x] = lo[t][x] = 0.f;
    const int steps = (D + 15) / 16;
#pragma unroll 4
    for (int i = 0; i < steps; ++i) {
      const bool in = i * 16 + c * 4 < D;
      float kv[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float4 x = in ? *reinterpret_cast<const float4*>(kt + t * 8 * D + i * 16) : make_float4(0.f, 0.f, 0.f, 0.f);
        kv[t][0] = x.x;
        kv[t][1] = x.y;
        kv[t][2] = x.z;
        kv[t][3] = x.w;
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float qf[4 * R];
#pragma unroll
        for (int x = 0; x < R; ++x)
          *reinterpret_cast<float4*>(qf + 4 * x) = *reinterpret_cast<const float4*>(q_s + (2 * i + y) * 128 * R + 4 * x);
        const float *qh = qf, *ql = qf + 2 * R;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float b0 = tf32_hi(kv[t][2 * y]), b1 = tf32_hi(kv[t][2 * y + 1]);
          const float c0 = kv[t][2 * y] - b0, c1 = kv[t][2 * y + 1] - b1;
          if constexpr (R == 1) {                         // rows + 8: the queries' lo parts
            mma_tf32(lo[t], qh[0], ql[0], qh[1], ql[1], c0, c1);
            mma_tf32(hi[t], qh[0], ql[0], qh[1], ql[1], b0, b1);
          } else {
            mma_tf32(lo[t], qh[0], qh[2], qh[1], qh[3], c0, c1);
            mma_tf32(lo[t], ql[0], ql[2], ql[1], ql[3], b0, b1);
            mma_tf32(hi[t], qh[0], qh[2], qh[1], qh[3], b0, b1);
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2 * R; ++x)
        s[t][x] = R == 1 ? hi[t][x] + (hi[t][2 + x] + (lo[t][x] + lo[t][2 + x])) : hi[t][x] + lo[t][x];
  }
  float down[R];
  __device__ __forceinline__ void softmax(const PagedLayout& g, const PagedAttnArgs& a, const Piece& pc, int t0,
                                          uint32_t seen, float add, int lane) {
    const int c = lane & 3;
    float add_x[NT][2];
    if (a.mask) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) add_x[t][x] = __shfl_sync(0xffffffffu, add, t * 8 + 2 * c + x);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int gi = r * 8 + (lane >> 2);
      float mx = m[r];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float v = s[t][2 * r + x];
          if (a.has_scale) v = __fmul_rn(v, a.scale);
          if (a.mask) v = __fadd_rn(v, add_x[t][x]);
          if (!(seen >> (t * 8 + 2 * c + x) & 1u)) v = -INFINITY;
          s[t][2 * r + x] = v;
          mx = fmaxf(mx, v);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      down[r] = exp_from(m[r], mx);
      m[r] = mx;
      l[r] *= down[r];
      if (a.scores && gi < pc.live) {
        float* to = a.scores + ((uint64_t)pc.b * a.heads + pc.head0 + gi) * g.capacity + t0 + 2 * c;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (t0 + t * 8 + 2 * c + x < pc.end) to[t * 8 + x] = s[t][2 * r + x];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[t][2 * r + x] = exp_from(s[t][2 * r + x], mx);
          l[r] += s[t][2 * r + x];
        }
    }
  }
  __device__ __forceinline__ void values(const float* vt, int D, uint32_t seen, int lane) {
    const int c = lane & 3, n4 = (lane >> 2) * 4;
    const bool all = seen == (1u << TW) - 1u;
    float ph[NT][2 * R], pl[NT][2 * R];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < 2 * R; ++x) {
        ph[t][x] = tf32_hi(s[t][x]);
        pl[t][x] = s[t][x] - ph[t][x];
      }
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      if (j * 32 >= D) break;
      float o[4][4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[e][x] = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bool in = j * 32 + n4 < D;
        const float* p0 = vt + (t * 8 + 2 * c) * D + j * 32 + n4;
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 x0 = in && (all || (seen >> (t * 8 + 2 * c) & 1u)) ? *reinterpret_cast<const float4*>(p0) : zero;
        const float4 x1 = in && (all || (seen >> (t * 8 + 2 * c + 1) & 1u)) ? *reinterpret_cast<const float4*>(p0 + D) : zero;
        const float v0[4] = {x0.x, x0.y, x0.z, x0.w}, v1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float b0 = tf32_hi(v0[e]), b1 = tf32_hi(v1[e]);
          if constexpr (R == 1) {                         // rows + 8: the probabilities' lo parts
            mma_tf32(o[e], ph[t][0], pl[t][0], ph[t][1], pl[t][1], v0[e] - b0, v1[e] - b1);
            mma_tf32(o[e], ph[t][0], pl[t][0], ph[t][1], pl[t][1], b0, b1);
          } else {
            mma_tf32(o[e], ph[t][0], ph[t][2], ph[t][1], ph[t][3], v0[e] - b0, v1[e] - b1);
            mma_tf32(o[e], pl[t][0], pl[t][2], pl[t][1], pl[t][3], b0, b1);
            mma_tf32(o[e], ph[t][0], ph[t][2], ph[t][1], ph[t][3], b0, b1);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 2 * R; ++x)
          acc[j][e][x] = fmaf(acc[j][e][x], down[x >> 1], R == 1 ? o[e][x] + o[e][2 + x] : o[e][x]);
    }
  }
  __device__ __forceinline__ void finish(float2* ml, int lane) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if ((lane & 3) == 0) ml[r * 8 + (lane >> 2)] = make_float2(m[r], l[r]);
    }
  }
  // column 2 c + x of MMA e of block j is value 32 j + 4 (2 c + x) + e
  template <typename F>
  __device__ __forceinline__ void each(int lane, F f) {
    const int c = lane & 3;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
            f(r * 8 + (lane >> 2), j * 32 + (2 * c + x) * 4 + e, acc[j][e][2 * r + x], acc[j][e + 1][2 * r + x]);
  }
};

template <int DM, int GT, bool MMA> struct Chosen { typedef FmaState<DM, GT> State; };
template <int DM, int GT> struct Chosen<DM, GT, true> { typedef MmaState<DM, GT> State; };

template <int DM, int GT, bool MMA>
__global__ void __launch_bounds__((compute_warps(DM, GT, MMA) + 1) * 32, blocks_per_sm(DM, GT, MMA))
paged_attention_bulk_kernel(const PagedLayout g, const PagedAttnArgs a) {
  typedef typename Chosen<DM, GT, MMA>::State State;
  constexpr int TW = warp_slots<DM>(), NW = compute_warps(DM, GT, MMA), T = NW * TW;
  extern __shared__ __align__(128) uint8_t smem[];
  const int D = g.head_dim;
  const uint32_t tile_bytes = (uint32_t)(T * D * 4);
  float* q_s = reinterpret_cast<float*>(smem + (uint32_t)a.slots * tile_bytes);
  float* joined = q_s + query_floats<DM, GT, MMA>();      // [NW / 2][GT][DM]
  float* p_all = joined + NW / 2 * GT * DM;
  float2* ml_s = reinterpret_cast<float2*>(p_all + (MMA ? 0 : NW * TW * GT));
  const uint32_t bars = smem_u32(ml_s + NW * GT);
  auto full = [&](int s) { return bars + 8u * (uint32_t)s; };
  auto empty = [&](int s) { return bars + 8u * (uint32_t)(kMaxSlots + s); };
  const uint32_t ring = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < a.slots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), NW);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  Walk walk;
  walk.init(g, a);
  __syncthreads();
  Piece pc;
  int slot = 0;                                           // of the ring, and its phase
  uint32_t phase = 0;
  auto step = [&]() {
    if (++slot == a.slots) {
      slot = 0;
      phase ^= 1;
    }
  };

  if (warp == NW) {
    // ------------------------------------------------------------------ producer --
    int used = 0;
    bool alive = true;
    while (alive && walk.next(g, a, pc)) {
      for (int t = 0; alive && t < pc.tiles; ++t) {
        const int first = pc.begin + t * T, last = min(first + T, pc.end);
        const int page0 = g.page_shift >= 0 ? first >> g.page_shift : first / g.page_size;
        const int page1 = g.page_shift >= 0 ? (last - 1) >> g.page_shift : (last - 1) / g.page_size;
        for (int kv = 0; kv < 2; ++kv) {
          if (!warp_wait(empty(slot), phase ^ 1)) {
            if (lane == 0) atomicExch(g.flag, 1);
            alive = false;
            break;
          }
          const float* pool = kv ? a.v_cache : a.k_cache;
          // a lane for every page: how much of it is there, then the copies
          for (int pass = 0; pass < 2; ++pass) {
            uint32_t bytes = 0;
            for (int pi = page0 + lane; pi <= page1; pi += 32) {
              const int from = max(first, pi * g.page_size);
              const int to = (int)min((long long)last, (long long)(pi + 1) * g.page_size);
              const uint32_t row = paged_row<false>(g, pc.b, pc.h, from);
              if (row == kNoRow) continue;   // (reported below, if one of its slots counts)
              const uint32_t n = (uint32_t)(to - from) * (uint32_t)(D * 4);
              if (pass)
                bulk_copy(ring + (uint32_t)slot * tile_bytes + (uint32_t)(from - first) * (uint32_t)(D * 4),
                          pool + (uint64_t)row * D, n, full(slot));
              bytes += n;
            }
            if (pass == 0) {
              for (int o = 16; o; o >>= 1) bytes += __shfl_xor_sync(0xffffffffu, bytes, o);
              if (lane == 0) mbar_expect_tx(full(slot), bytes);
              __syncwarp();
            }
          }
          ++used;
          step();
        }
      }
    }
    if (!alive)   // copies in flight must land before the block's memory goes away
      for (int u = used > a.slots ? used - a.slots : 0; u < used; ++u)
        warp_wait(full(u % a.slots), (u / a.slots) & 1);
    return;
  }
  // -------------------------------------------------------------------- computing --
  State st;
  bool alive = true;
  if constexpr (!MMA) st.p_s = p_all + warp * TW * GT;
  while (walk.next(g, a, pc)) {
    State::load_queries(g, a, pc, q_s, tid);
    st.reset();
    compute_barrier<NW>();
    // lane j looks after slot t0 + j: its page, and what the mask adds to it (fetched a tile ahead)
    auto look = [&](int t, int& page, float& add) {
      const int mine = pc.begin + t * T + warp * TW + lane;
      page = -1;
      add = -INFINITY;
      if (lane < TW && mine < pc.end) {
        page = __ldg(g.table + (size_t)pc.b * g.max_pages + (g.page_shift >= 0 ? mine >> g.page_shift : mine / g.page_size));
        add = a.mask ? __ldg(a.mask + (uint64_t)pc.b * g.capacity + mine) : 0.f;
      }
    };
    int page, next_page;
    float add, next_add;
    look(0, next_page, next_add);
    for (int t = 0; t < pc.tiles; ++t) {
      const int t0 = pc.begin + t * T + warp * TW;
      page = next_page;
      add = next_add;
      look(t + 1, next_page, next_add);
      // (a slot hidden by the mask does not count, whatever it holds, NaN included)
      const bool counts = add != -INFINITY, there = (unsigned)page < (unsigned)g.num_pages;
      if (counts && !there) atomicOr(g.flag, kBadPage);
      const uint32_t seen = __ballot_sync(0xffffffffu, counts && there);
      // (a wait that gives up marks the launch as failed; the rest runs through without waiting)
      if (alive && !warp_wait(full(slot), phase)) {
        alive = false;
        if (lane == 0) atomicExch(g.flag, 2);
      }
      st.scores(reinterpret_cast<const float*>(smem + (uint32_t)slot * tile_bytes) + warp * TW * D, q_s, D, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(slot));
      step();
      st.softmax(g, a, pc, t0, seen, add, lane);
      if (alive && !warp_wait(full(slot), phase)) {
        alive = false;
        if (lane == 0) atomicExch(g.flag, 3);
      }
      st.values(reinterpret_cast<const float*>(smem + (uint32_t)slot * tile_bytes) + warp * TW * D, D, seen, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(slot));
      step();
    }
    // the warps' results: the upper half of them gives its to the lower half, until one has all
    st.finish(ml_s + warp * GT, lane);
    compute_barrier<NW>();
    auto top = [&](int gi) {
      float m = ml_s[gi].x;
#pragma unroll
      for (int w = 1; w < NW; ++w) m = fmaxf(m, ml_s[w * GT + gi].x);
      return m;
    };
    for (int round = NW / 2; round >= 1; round >>= 1) {
      const bool first = round == NW / 2;
      if (warp >= round && warp < 2 * round) {
        float* to = joined + (warp - round) * GT * DM;
        st.each(lane, [&](int gi, int d, float& x, float& y) {
          const float f = first ? exp_from(ml_s[warp * GT + gi].x, top(gi)) : 1.0f;
          to[gi * DM + d] = x * f;
          to[gi * DM + d + 1] = y * f;
        });
      }
      compute_barrier<NW>();
      if (warp < round) {
        const float* from = joined + warp * GT * DM;
        st.each(lane, [&](int gi, int d, float& x, float& y) {
          const float f = first ? exp_from(ml_s[warp * GT + gi].x, top(gi)) : 1.0f;
          x = fmaf(x, f, from[gi * DM + d]);
          y = fmaf(y, f, from[gi * DM + d + 1]);
        });
      }
      if (round > 1) compute_barrier<NW>();
    }
    if (warp == 0)
      st.each(lane, [&](int gi, int d, float& x, float& y) {
        const float mx = top(gi);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum = fmaf(ml_s[w * GT + gi].y, exp_from(ml_s[w * GT + gi].x, mx), sum);
        write_result<GT>(g, a, pc, gi, d, x, mx, sum);
        write_result<GT>(g, a, pc, gi, d + 1, y, mx, sum);
      });
    compute_barrier<NW>();                                    // queries, maxima and `joined` are free again
  }
}

// ---- plain loads -----------------------------------------------------------------------------
__device__ __forceinline__ float4 load4(const float* p, int d, int dim) {
  float4 r;
  r.x = d < dim ? __ldg(p + d) : 0.f;
  r.y = d + 1 < dim ? __ldg(p + d + 1) : 0.f;
  r.z = d + 2 < dim ? __ldg(p + d + 2) : 0.f;
  r.w = d + 3 < dim ? __ldg(p + d + 3) : 0.f;
  return r;
}

constexpr int kLoadTile = 32;      // slots a warp takes at a time

// Rows that are not on 16 bytes.  DM: head_dim rounded up; GT: query heads of one key-value head
// that a block serves.
template <int DM, int GT>
__global__ void __launch_bounds__(kWarps * 32)
paged_attention_loads_kernel(const PagedLayout g, const PagedAttnArgs a) {
  constexpr int NI = DM / 16;                    // steps of 16 values of a key, 4 a lane
  constexpr int LPR = DM / 4 < 32 ? DM / 4 : 32; // lanes that share a value row
  constexpr int VR = DM / 4 / LPR;               // 4-value pieces of it a lane holds
  constexpr int TPI = 32 / LPR;                  // value rows a warp reads at a time
  __shared__ __align__(16) float q_s[GT][DM];
  __shared__ float p_s[kWarps][kLoadTile][GT];
  __shared__ float2 ml_s[kWarps][GT];
  __shared__ __align__(16) float acc_s[kWarps][GT][DM];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c = lane & 3, tok = lane >> 2;       // keys: four lanes a slot, eight slots at a time
  Walk walk;
  walk.init(g, a);
  Piece pc;
  while (walk.next(g, a, pc)) {
    for (int i = tid; i < GT * DM; i += kWarps * 32) {
      const int gi = i / DM, d = i - gi * DM;
      q_s[gi][d] = gi < pc.live && d < g.head_dim
                       ? __ldg(a.q + ((uint64_t)pc.b * a.heads + pc.head0 + gi) * g.head_dim + d) : 0.f;
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
    for (int t0 = pc.begin + warp * kLoadTile; t0 < pc.end; t0 += kWarps * kLoadTile) {
      const int mine = t0 + lane;
      const float my_mask = a.mask && mine < pc.end ? __ldg(a.mask + (uint64_t)pc.b * g.capacity + mine) : 0.f;
      // (a slot hidden by the mask is not read: what it holds, NaN included, does not count)
      const uint32_t my_row = mine < pc.end && my_mask != -INFINITY ? paged_row(g, pc.b, pc.h, mine) : kNoRow;
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
        if (a.scores && gi < pc.live && slot < pc.end)
          a.scores[((uint64_t)pc.b * a.heads + pc.head0 + gi) * g.capacity + slot] = mine_s;
      }
      __syncwarp();
#pragma unroll 4
      for (int it = 0; it < kLoadTile / TPI; ++it) {
        const int t = it * TPI + lane / LPR;
        const uint32_t r0 = __shfl_sync(0xffffffffu, my_row, t);
        const float* vp = a.v_cache + (uint64_t)(r0 == kNoRow ? 0u : r0) * g.head_dim;
        float4 v[VR];
#pragma unroll
        for (int r = 0; r < VR; ++r)
          v[r] = r0 != kNoRow ? load4(vp, (r * LPR + lane % LPR) * 4, g.head_dim) : make_float4(0.f, 0.f, 0.f, 0.f);
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
      float mx = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml_s[w][gi].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp_from(ml_s[w][gi].x, mx);
        sum = fmaf(ml_s[w][gi].y, f, sum);
        o = fmaf(acc_s[w][gi][d], f, o);
      }
      write_result<GT>(g, a, pc, gi, d, o, mx, sum);
    }
    __syncthreads();
  }
}

// ---- join ------------------------------------------------------------------------------------
// A block takes query heads `part`, part + per, ... of a row and key-value head (results that
// several blocks worked on) and, with weights, every per-th stretch of its slots: the accumulated
// weights are the old ones plus the group's probabilities, summed in the order of the heads.
// V slots a thread: 4 where the rows of the weights are on 16 bytes, else 1.
constexpr int kJoinThreads = 256;

template <int V>
__global__ void __launch_bounds__(kJoinThreads)
paged_attention_join_kernel(const PagedLayout g, const PagedAttnArgs a, const float* __restrict__ weights,
                            float* __restrict__ out_weights, int per) {
  extern __shared__ float2 stat[];               // [group]: maximum, 1 / sum (0 for an empty row)
  __shared__ float sums[kJoinThreads];
  __shared__ int part0_s, parts_s;
  const int unit = blockIdx.x / per;             // row * kv_heads + head
  const int part = blockIdx.x - unit * per;
  const int b = unit / g.kv_heads, h = unit - b * g.kv_heads;
  const int n = paged_length(g, b);
  const uint64_t head0 = (uint64_t)b * a.heads + h * a.group;
  const int per_row = g.kv_heads * a.group_chunks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // threads side by side along head_dim, `lines` parts at a time
  const int width = g.head_dim <= 32 ? 32 : g.head_dim <= 64 ? 64 : g.head_dim <= 128 ? 128 : 256;
  const int lines = kJoinThreads / width, d = tid & (width - 1), line = tid / width;
  Shares sh;
  if (warp == 0) sh = shares_of(g, a, b, -1);
  for (int gc = 0; gc < a.group_chunks; ++gc) {
    if (tid == 0) {
      // the blocks among which this unit's tiles lie
      const int hc = h * a.group_chunks + gc;
      const long long t = row_tiles(g, a, b), first = sh.before * per_row + hc * t;
      const int c0 = a.whole ? 0 : (int)(first / sh.size), c1 = a.whole ? 0 : (int)((first + t - 1) / sh.size);
      part0_s = b * per_row + hc + c0;
      parts_s = c1 - c0 + 1;
    }
    __syncthreads();
    const int part0 = part0_s, parts = parts_s;
    const int heads = min(a.chunk, a.group - gc * a.chunk);
    if (parts == 1 && out_weights == nullptr) {  // one block has written the result
      __syncthreads();
      continue;
    }
    for (int gi = warp; gi < heads; gi += kJoinThreads / 32) {
      const float2* ml = a.part_ml + (uint64_t)part0 * a.chunk + gi;
      float mx = -INFINITY, sum = 0.f;
      for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, ml[(uint64_t)i * a.chunk].x);
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      for (int i = lane; i < parts; i += 32) {
        const float2 x = ml[(uint64_t)i * a.chunk];
        sum = fmaf(x.y, exp_from(x.x, mx), sum);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) stat[gc * a.chunk + gi] = make_float2(mx, sum == 0.f ? 0.f : __fdiv_rn(1.0f, sum));
    }
    __syncthreads();
    if (parts > 1)
      for (int gi = part; gi < heads; gi += per) {
        const float2* ml = a.part_ml + (uint64_t)part0 * a.chunk + gi;
        const float* acc = a.part_acc + ((uint64_t)part0 * a.chunk + gi) * g.head_dim + d;
        const float2 st = stat[gc * a.chunk + gi];
        float o = 0.f;
        if (d < g.head_dim) {
#pragma unroll 8
          for (int i = line; i < parts; i += lines)
            o = fmaf(acc[(uint64_t)i * a.chunk * g.head_dim], exp_from(ml[(uint64_t)i * a.chunk].x, st.x), o);
        }
        sums[tid] = o;
        __syncthreads();
        if (line == 0 && d < g.head_dim) {
          for (int x = 1; x < lines; ++x) o += sums[x * width + d];
          a.out[(head0 + gc * a.chunk + gi) * g.head_dim + d] = __fmul_rn(o, st.y);
        }
        __syncthreads();
      }
  }
  if (out_weights == nullptr) return;
  const float* sc = a.scores + head0 * g.capacity;
  const float* old = weights + (uint64_t)unit * g.capacity;
  for (int j = (part * kJoinThreads + tid) * V; j < g.capacity; j += per * kJoinThreads * V) {
    float w[V], o[V];
#pragma unroll
    for (int x = 0; x < V; ++x) w[x] = o[x] = 0.f;
    if (j < n) {
      if constexpr (V == 4)
        *reinterpret_cast<float4*>(o) = __ldg(reinterpret_cast<const float4*>(old + j));
      else
        o[0] = __ldg(old + j);
#pragma unroll 4
      for (int gi = 0; gi < a.group; ++gi) {
        const float2 st = stat[gi];
        float s[V];
        if constexpr (V == 4)
          *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sc + (uint64_t)gi * g.capacity + j);
        else
          s[0] = sc[(uint64_t)gi * g.capacity + j];
        // (an empty row has 1 / sum = 0 and scores of -infinity only)
#pragma unroll
        for (int x = 0; x < V; ++x) w[x] = fmaf(exp_from(s[x], st.x), st.y, w[x]);
      }
      // (what lies behind the row's end was never written and is dropped here)
#pragma unroll
      for (int x = 0; x < V; ++x) w[x] = j + x < n ? w[x] + o[x] : 0.f;
    }
    if constexpr (V == 4)
      *reinterpret_cast<float4*>(out_weights + (uint64_t)unit * g.capacity + j) = *reinterpret_cast<float4*>(w);
    else
      out_weights[(uint64_t)unit * g.capacity + j] = w[0];
  }
}

// ---- host ------------------------------------------------------------------------------------
constexpr int kBlockSmem = 226 * 1024;   // that a single block of an SM may ask for

// How a call is cut into shares, and what its blocks need.
struct Plan {
  int chunk, tile, blocks, slots, smem;
};

// The ring: as many tiles as fit beside another block (or two, for small heads), at least two
// (the keys and the values of one tile).
template <int DM, int GT, bool MMA>
Plan plan_bulk(const tfjs_cuda_ctx* ctx, int dim) {
  constexpr int fixed = bulk_fixed_bytes<DM, GT, MMA>(), T = compute_warps(DM, GT, MMA) * warp_slots<DM>();
  Plan p;
  p.chunk = GT;
  p.tile = T;
  int per_sm = blocks_per_sm(DM, GT, MMA);
  const int tile = T * dim * 4;
  do {
    const int room = (kBlockSmem + 1024) / per_sm - 1024 - fixed;   // (a block has 1 KB beside what it asks for)
    p.slots = room > 0 ? room / tile : 0;
  } while (p.slots < 2 && --per_sm > 0);
  if (p.slots > kMaxSlots) p.slots = kMaxSlots;
  p.smem = p.slots * tile + fixed;
  p.blocks = ctx->sm_count * per_sm;
  return p;
}
template <int DM, int GT, bool MMA>
int launch_bulk(tfjs_cuda_ctx* ctx, const PagedLayout& g, const PagedAttnArgs& a, const Plan& p) {
  // (the most that any call of it takes, so that two contexts of a process cannot lower it for each other)
  CUDA_TRY(ctx, cudaFuncSetAttribute(paged_attention_bulk_kernel<DM, GT, MMA>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, kBlockSmem));
  paged_attention_bulk_kernel<DM, GT, MMA><<<a.shares, (compute_warps(DM, GT, MMA) + 1) * 32, p.smem, ctx->stream>>>(g, a);
  LAUNCH_CHECK(ctx, MMA ? "paged_attention_bulk_kernel<mma>" : "paged_attention_bulk_kernel<fma>");
  return TFJS_CUDA_OK;
}
template <int DM, int GT>
Plan plan_loads(const tfjs_cuda_ctx* ctx, int) {
  Plan p;
  p.chunk = GT;
  p.tile = kWarps * kLoadTile;
  p.blocks = ctx->sm_count * 4;
  p.slots = p.smem = 0;
  return p;
}
template <int DM, int GT>
int launch_loads(tfjs_cuda_ctx* ctx, const PagedLayout& g, const PagedAttnArgs& a, const Plan&) {
  paged_attention_loads_kernel<DM, GT><<<a.shares, kWarps * 32, 0, ctx->stream>>>(g, a);
  LAUNCH_CHECK(ctx, "paged_attention_loads_kernel");
  return TFJS_CUDA_OK;
}

typedef Plan (*PlanFn)(const tfjs_cuda_ctx*, int);
typedef int (*LaunchFn)(tfjs_cuda_ctx*, const PagedLayout&, const PagedAttnArgs&, const Plan&);
struct Form {
  PlanFn plan;
  LaunchFn launch;
};
#define BULK_FORMS(GT, MMA)                                                                 \
  {                                                                                         \
    {plan_bulk<32, GT, MMA>, launch_bulk<32, GT, MMA>}, {plan_bulk<64, GT, MMA>, launch_bulk<64, GT, MMA>}, \
    {plan_bulk<128, GT, MMA>, launch_bulk<128, GT, MMA>}, {plan_bulk<256, GT, MMA>, launch_bulk<256, GT, MMA>} \
  }
#define LOAD_FORMS(GT)                                                                      \
  {                                                                                         \
    {plan_loads<32, GT>, launch_loads<32, GT>}, {plan_loads<64, GT>, launch_loads<64, GT>}, \
    {plan_loads<128, GT>, launch_loads<128, GT>}, {plan_loads<256, GT>, launch_loads<256, GT>} \
  }
// [query heads of a key-value head: 1, 2, to 4, to 8, more; plain loads: 1, more][head size]
const Form kForms[7][4] = {BULK_FORMS(1, false), BULK_FORMS(2, false), BULK_FORMS(4, false), BULK_FORMS(8, true),
                           BULK_FORMS(16, true), LOAD_FORMS(1), LOAD_FORMS(8)};

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
  const uint64_t values = units * p->head_dim * 4, sums = kv_units * cap * 4, rows = (uint64_t)p->batch * 4;
  const Span spans[] = {{out->ptr, values}, {ow ? ow->ptr : nullptr, ow ? sums : 0}, {q->ptr, values},
                        {kc->ptr, g.pool_bytes}, {vc->ptr, g.pool_bytes}, {g.table, rows * p->max_pages},
                        {g.lengths, rows}, {mask ? mask->ptr : nullptr, mask ? rows * cap : 0},
                        {w ? w->ptr : nullptr, w ? sums : 0}};
  if ((rc = ctx_apart(ctx, who, spans, 9, 2))) return rc;

  PagedAttnArgs a;
  a.q = (const float*)q->ptr;
  a.k_cache = (const float*)kc->ptr;
  a.v_cache = (const float*)vc->ptr;
  a.mask = mask ? (const float*)mask->ptr : nullptr;
  a.out = (float*)out->ptr;
  a.batch = p->batch;
  a.heads = p->heads;
  a.group = p->heads / p->kv_heads;
  a.has_scale = p->has_scale;
  a.scale = p->scale;
  const float* wp = w ? (const float*)w->ptr : nullptr;
  float* owp = ow ? (float*)ow->ptr : nullptr;

  const bool wide = p->head_dim % 4 == 0 && (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) == 0;
  const int by_group = !wide ? (a.group == 1 ? 5 : 6)
                             : a.group <= 2 ? a.group - 1 : a.group <= 4 ? 2 : a.group <= 8 ? 3 : 4;
  const int by_dim = p->head_dim <= 32 ? 0 : p->head_dim <= 64 ? 1 : p->head_dim <= 128 ? 2 : 3;
  const Form& form = kForms[by_group][by_dim];
  const Plan plan = form.plan(ctx, p->head_dim);
  a.chunk = plan.chunk;
  a.tile = plan.tile;
  a.slots = plan.slots;
  a.group_chunks = (a.group + a.chunk - 1) / a.chunk;
  // Short rows: a block each, whose result needs no joining.  (12 rows and heads of 128 / 256 / 512
  // slots: 6.5 / 9.9 / 16 us against 10 / 10 / 11 with equal shares and their joining; 128 of 256 / 512 /
  // 1024: 14 / 21 / 36 against 16 / 22 / 28; 256 of them: 15 / 24 / 43 against 32 / 37 / 54, but there a
  // single long row among short ones would be waited for.)
  const uint64_t blocks = kv_units * a.group_chunks;
  a.whole = cap <= (blocks * 4 >= (uint64_t)ctx->sm_count * 3 ? 8ull : 4ull) * a.tile;
  a.shares = a.whole ? (int)blocks : plan.blocks;

  cudaSetDevice(ctx->device);
  TempBuffer ws(ctx), sc(ctx);
  void* mem;
  const uint64_t parts = (blocks + (a.whole ? 0 : a.shares)) * a.chunk;
  if ((rc = ws.get(parts * (8 + (a.whole ? 0 : (uint64_t)p->head_dim * 4)), &mem))) return rc;   // (Buffer pointers end here)
  a.part_ml = (float2*)mem;
  a.part_acc = (float*)(a.part_ml + parts);
  a.scores = nullptr;
  if (weights_id) {
    if ((rc = sc.get(units * cap * 4, &mem))) return rc;
    a.scores = (float*)mem;
  }
  if ((rc = form.launch(ctx, g, a, plan))) return rc;
  if (weights_id || !a.whole) {
    // blocks for the heads to join (few, where the rows and heads are many), and one for every four
    // slots a thread
    uint64_t per = ((uint64_t)ctx->sm_count * 4 + kv_units - 1) / kv_units;
    if (per > (uint64_t)a.group) per = a.group;
    if (a.whole) per = 1;
    const bool four = weights_id && cap % 4 == 0 && (((uintptr_t)wp | (uintptr_t)owp) & 15) == 0;
    const uint64_t stretch = kJoinThreads * 4;
    if (weights_id) {
      // (all of them at once: finding the parts takes a block as long as a stretch of slots)
      uint64_t want = (cap + stretch - 1) / stretch;
      const uint64_t room = (uint64_t)ctx->sm_count * 8 / kv_units;
      if (want > room) want = room;
      if (per < want) per = want;
    }
    if (per * kv_units > 0x7fffffffull) per = 0x7fffffffull / kv_units;
    const unsigned grid = (unsigned)(kv_units * per);
    const unsigned stat = a.group * sizeof(float2);
    if (four)
      paged_attention_join_kernel<4><<<grid, kJoinThreads, stat, ctx->stream>>>(g, a, wp, owp, (int)per);
    else
      paged_attention_join_kernel<1><<<grid, kJoinThreads, stat, ctx->stream>>>(g, a, wp, owp, (int)per);
    LAUNCH_CHECK(ctx, "paged_attention_join_kernel");
    if (weights_id) ctx_mark_written(ctx, out_weights_id);
  }
  ctx_mark_written(ctx, out_id);
  return TFJS_CUDA_OK;
}
