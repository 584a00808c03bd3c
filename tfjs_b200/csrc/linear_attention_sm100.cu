// Linear attention with a decay for each head, in chunks of 128 tokens on the tensor cores.
// With g = exp(log_decay) and S the state in front of a chunk, its tokens t = 0 .. 127 give
//   out_t = scale * ( sum_{j <= t} g^(t-j) (q_t . k_j) v_j  +  g^(t+1) q_t S )
// and the chunk leaves  g^128 S + A,  A = sum_j g^(127-j) k_j v_j^T.  Three launches:
//   chunk_states   A^T of every chunk (tokens are the K dimension of the product)
//   chunk_scan     A^T of chunk c is replaced by the state in front of it, chunk after chunk,
//                  elementwise; what is left over is the new state
//   chunk_outputs  Q [K; S^T]^T, the decayed lower triangle of its left half, times V, on top of
//                  the decayed right half
// so that all chunks of all rows and heads run at once; the states between them are kept
// transposed, [dim_v][dim_k], which is what the last kernel's B operand wants.
//
// Products of fp32 values on TF32 tensor cores: every operand x is stored as hi = x rounded to
// 11 bits and lo = x - hi, and hi hi + hi lo + lo hi is accumulated in fp32, which leaves out
// about 2^-22 of each product.  The tensor core cuts its sums off instead of rounding them, a
// bias of about 0.4 * 2^-24 of the accumulator for each MMA, so the small products have an
// accumulator of their own (or come first) and only every third MMA meets the large sum.
// Operands come through registers (load, split, swizzled store)
// because the split has to happen on the way, so any size and alignment is a predicate there.
//
// 2 x 16 heads of 128 x 128 with 16384 tokens take 177 us for the states (805 MB), 90 for the scan (537 MB, 0.92
// of a copy's bandwidth) and 410 for the outputs (1342 MB).  No unit is full in the last: DRAM, tensor and
// shared-memory pipes are each near 0.4.  A chunk moves 1.5 MB through shared memory (the split doubles what is written,
// and each MMA reads its operands again), some 12 k of about 28 k clocks at 128 bytes each; the rest is most
// likely the chain of one chunk: tensor memory has no room for a second one's scores (for half of them it has).
#include "gemm_tf32_device.cuh"
#include "linear_attention.h"

namespace {

constexpr int kC = 128;            // tokens of a chunk = rows of an MMA
constexpr int kProducers = 8;      // warps 0-7: load, split, store operands; those from 8 on read tensor
                                   // memory, each in the quarter of its lanes that it may access
constexpr int kMaxStages = 4;
constexpr int kSmemCap = 232448;

struct ChunkArgs {
  LinearArgs a;
  float* states;                   // [units][chunks][dv][dk]
  int chunks, dv_tiles, items;
  int dvp, dkp;                    // columns of a dim_v tile and dim_k, in whole blocks of 32
  int stage_bytes, stages;
};

// a chunk's row, head, first token and tokens
struct Item {
  int unit, b, h, c, dv0;
  int n;                           // tokens of the chunk, 0 behind the row's end
};
__device__ __forceinline__ Item item_of(const ChunkArgs& g, int i) {
  Item t;
  const int dvt = i % g.dv_tiles;
  const int uc = i / g.dv_tiles;
  t.c = uc % g.chunks;
  t.unit = uc / g.chunks;
  t.b = t.unit / g.a.heads;
  t.h = t.unit - t.b * g.a.heads;
  t.dv0 = dvt * 128;
  const int left = linear_length(g.a, t.b) - t.c * kC;
  t.n = left < 0 ? 0 : (left > kC ? kC : left);
  return t;
}

// Four values, zeros where !in; load_cols4: of a row of `dim` that is not on 16 bytes, from column d
// on (p points there).  Volatile, so that a stage's loads are issued together and early: left to itself the compiler
// moves each one down to its use.  Predicated, since a branch a load costs as much as the rest.
__device__ __forceinline__ float4 load16(const float* p, bool in) {
  float4 r;
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.f32 %0, 0f00000000;\n\tmov.f32 %1, 0f00000000;\n\tmov.f32 %2, 0f00000000;\n\tmov.f32 %3, 0f00000000;\n\t"
      "@q ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w) : "l"(p), "r"((int)in));
  return r;
}
__device__ __forceinline__ float load1(const float* p, bool in) {
  float r;
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t@q ld.global.nc.f32 %0, [%1];\n\t}"
      : "=f"(r) : "l"(p), "r"((int)in));
  return r;
}
__device__ __forceinline__ float4 load_cols4(const float* p, int d, int dim, bool in) {
  return make_float4(load1(p, in && d < dim), load1(p + 1, in && d + 1 < dim), load1(p + 2, in && d + 2 < dim),
                     load1(p + 3, in && d + 3 < dim));
}
// Bits 0 .. of the places 0, 32, 64, ... (at most `most` of them) that lie below n.
__device__ __forceinline__ uint32_t places(int n, int most) {
  const int c = n <= 0 ? 0 : (n + 31) >> 5;
  return (1u << (c < most ? c : most)) - 1u;
}

// x rounded to TF32's 11 bits, to nearest
__device__ __forceinline__ float tf32_hi(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
}
__device__ __forceinline__ void store_split(uint32_t hi_addr, uint32_t lo_addr, const float4& x) {
  const float a = tf32_hi(x.x), b = tf32_hi(x.y), c = tf32_hi(x.z), d = tf32_hi(x.w);
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(hi_addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(lo_addr), "f"(x.x - a), "f"(x.y - b),
               "f"(x.z - c), "f"(x.w - d) : "memory");
}
// Byte offsets of 16-byte piece c4 (of 8) of a row in the two swizzled layouts: K-major rows of
// 32 values (16-byte pieces exchanged within eight rows), and MN-major blocks of 32 K rows x 32
// columns (32-byte pieces exchanged within four rows).
__device__ __forceinline__ uint32_t k_major(int row, int c4) {
  return (uint32_t)row * 128u + (uint32_t)((c4 ^ (row & 7)) << 4);
}
__device__ __forceinline__ uint32_t mn_major(int row, int c4) {
  return (uint32_t)row * 128u + (uint32_t)((((c4 >> 1) ^ (row & 3)) << 5) | ((c4 & 1) << 4));
}

// mbar_wait for a whole warp: true only if no lane gave up, so that its lanes stay together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

__device__ __forceinline__ void mma_tmem_a(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const float* f) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]),
      "f"(f[8]), "f"(f[9]), "f"(f[10]), "f"(f[11]), "f"(f[12]), "f"(f[13]), "f"(f[14]), "f"(f[15]),
      "f"(f[16]), "f"(f[17]), "f"(f[18]), "f"(f[19]), "f"(f[20]), "f"(f[21]), "f"(f[22]), "f"(f[23]),
      "f"(f[24]), "f"(f[25]), "f"(f[26]), "f"(f[27]), "f"(f[28]), "f"(f[29]), "f"(f[30]), "f"(f[31])
      : "memory");
}

// 32 columns of this thread's lane from two places at once: one wait for both.
__device__ __forceinline__ void tmem_load32_nowait(uint32_t taddr, float* f) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]),
        "=f"(f[8]), "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]),
        "=f"(f[16]), "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]), "=f"(f[21]), "=f"(f[22]), "=f"(f[23]),
        "=f"(f[24]), "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]), "=f"(f[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_load_sum32(uint32_t at, uint32_t at_lo, float* x) {
  float lo[32];
  tmem_load32_nowait(at, x);
  tmem_load32_nowait(at_lo, lo);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  // (the registers are there only now: nothing that reads them may come earlier)
#pragma unroll
  for (int j = 0; j < 32; ++j) asm volatile("" : "+f"(x[j]), "+f"(lo[j]));
#pragma unroll
  for (int j = 0; j < 32; ++j) x[j] += lo[j];
}

// 32 x 32 values, one row a lane, through a swizzled 4 KB tile of the warp so that global
// memory is written in rows of 128 bytes.  Row r goes to row_ptr(r) (null: not stored) at
// columns col .. col + 31 of `dim`.
template <bool WIDE, typename RowPtr>
__device__ __forceinline__ void store_rows32(uint32_t tile, int lane, const float* v, int col, int dim, RowPtr row_ptr) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(tile + k_major(lane, j)), "f"(v[4 * j]),
                 "f"(v[4 * j + 1]), "f"(v[4 * j + 2]), "f"(v[4 * j + 3]) : "memory");
  __syncwarp();
  const int c4 = lane & 7, d = col + c4 * 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3);
    float4 x;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                 : "r"(tile + k_major(r, c4)) : "memory");
    float* p = row_ptr(r);
    if (p == nullptr) continue;
    if (WIDE) {
      if (d < dim) *reinterpret_cast<float4*>(p + d) = x;
    } else {
      if (d < dim) p[d] = x.x;
      if (d + 1 < dim) p[d + 1] = x.y;
      if (d + 2 < dim) p[d + 2] = x.z;
      if (d + 3 < dim) p[d + 3] = x.w;
    }
  }
}

constexpr uint32_t kIdesc = (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(128 >> 4) << 24);  // f32 += tf32 x tf32, M = 128
constexpr uint32_t kAMN = 1u << 15, kBMN = 1u << 16;
__device__ __forceinline__ uint32_t n_field(int n) { return (uint32_t)(n >> 3) << 17; }

// ---- A^T of every chunk: M = dim_v tile, N = dim_k, K = tokens ------------------------------
constexpr int kStateThreads = (kProducers + 4 + 1) * 32;

// Warp 12's first thread issues the MMAs.  NK: at most that many blocks of 32 columns of K.
template <bool WIDE, int NK>
__global__ void __launch_bounds__(kStateThreads, 1)
linear_chunk_states_kernel(const ChunkArgs g) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t tiles = base + (uint32_t)(g.stages * g.stage_bytes);
  const uint32_t bars = tiles + 4 * 4096u;
  auto full = [&](int s) { return bars + 8u * (uint32_t)s; };
  auto empty = [&](int s) { return bars + 8u * (uint32_t)(kMaxStages + s); };
  auto acc_full = [&](int s) { return bars + 8u * (uint32_t)(2 * kMaxStages + s); };
  auto acc_empty = [&](int s) { return bars + 8u * (uint32_t)(2 * kMaxStages + 2 + s); };
  const uint32_t tmem_slot = bars + 8u * (2 * kMaxStages + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(full(s), kProducers);
      mbar_init(empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full(s), 1);
      mbar_init(acc_empty(s), 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

  // a stage: 32 tokens of V (four column blocks, hi then lo) and of decayed K
  const int nbv = g.dvp / 32, nbk = g.dkp / 32;
  const uint32_t k_off = 2 * 16384u, k_bytes = (uint32_t)nbk * 4096u;
  // accumulators of hi hi and of the small products: twice where 512 columns hold that
  const uint32_t bufs = g.dkp <= 128 ? 2u : 1u;
  if (warp < kProducers) {
    // A thread has a token of the stage and a 16-byte piece of each of its blocks.  Two stages are
    // in flight: the next one's loads are issued before this one's values are split and stored.
    const int r0 = (int)threadIdx.x >> 3, c4 = (int)threadIdx.x & 7;
    constexpr int S = 4 + NK;
    struct Stage {
      int i, ks;
      Item t;
      float ld;
    };
    auto settle = [&](Stage& s) {                  // the next item that has tokens, from s.i on
      for (; s.i < g.items; s.i += gridDim.x) {
        s.t = item_of(g, s.i);
        if (s.t.n > 0) break;
      }
      s.ks = 0;
      if (s.i < g.items) s.ld = __ldg(g.a.log_decay + s.t.h);
    };
    auto next = [&](Stage& s) {
      if ((++s.ks) * 32 >= s.t.n) {
        s.i += gridDim.x;
        settle(s);
      }
    };
    auto load = [&](const Stage& s, float4 (&x)[S]) {
      if (s.i >= g.items) return;
      const int j = s.ks * 32 + r0;
      const bool in = j < s.t.n;
      const uint64_t row = (uint64_t)s.t.unit * g.a.seq + (uint64_t)s.t.c * kC + (in ? j : 0);
      const float* pv = g.a.v + row * g.a.dv + s.t.dv0 + c4 * 4;
      const float* pk = g.a.k + row * g.a.dk + c4 * 4;
      if (WIDE) {
        const uint32_t mv = in ? places(g.a.dv - s.t.dv0 - c4 * 4, 4) : 0u, mk = in ? places(g.a.dk - c4 * 4, NK) : 0u;
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y] = load16(pv + y * 32, mv >> y & 1u);
#pragma unroll
        for (int y = 0; y < NK; ++y) x[4 + y] = load16(pk + y * 32, mk >> y & 1u);
      } else {
#pragma unroll
        for (int y = 0; y < 4; ++y)
          x[y] = load_cols4(pv + y * 32, s.t.dv0 + y * 32 + c4 * 4, g.a.dv, in && y < nbv);
#pragma unroll
        for (int y = 0; y < NK; ++y) x[4 + y] = load_cols4(pk + y * 32, y * 32 + c4 * 4, g.a.dk, in && y < nbk);
      }
    };
    uint32_t slot = 0, phase = 1;
    auto store = [&](const Stage& s, float4 (&x)[S]) -> bool {
      const uint32_t at = base + slot * (uint32_t)g.stage_bytes + mn_major(r0, c4);
      const int j = s.ks * 32 + r0;
      const float w = j < s.t.n ? decay_power(s.ld, s.t.n - 1 - j) : 0.f;
      if (!warp_wait(empty(slot), phase)) {
        if (lane == 0) atomicExch(g.a.flag, 1);
        return false;
      }
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (y < nbv) store_split(at + y * 4096u, at + 16384u + y * 4096u, x[y]);
      const uint32_t k_hi = at + k_off, k_lo = k_hi + k_bytes;
#pragma unroll
      for (int y = 0; y < NK; ++y)
        if (y < nbk)
          store_split(k_hi + y * 4096u, k_lo + y * 4096u,
                      make_float4(x[4 + y].x * w, x[4 + y].y * w, x[4 + y].z * w, x[4 + y].w * w));
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(full(slot));
      if (++slot == (uint32_t)g.stages) {
        slot = 0;
        phase ^= 1;
      }
      return true;
    };
    Stage a, b;
    float4 xa[S], xb[S];
    a.i = blockIdx.x;
    settle(a);
    load(a, xa);
    while (a.i < g.items) {
      b = a;
      next(b);
      load(b, xb);
      if (!store(a, xa) || b.i >= g.items) break;
      a = b;
      next(a);
      load(a, xa);
      if (!store(b, xb)) break;
    }
  } else if (warp == 12) {
    if (lane == 0) {
      const uint32_t idesc = kIdesc | kAMN | kBMN | n_field(g.dkp);
      uint32_t st = 0, done = 0;
      bool alive = true;
      for (int i = blockIdx.x; alive && i < g.items; i += gridDim.x) {
        const Item t = item_of(g, i);
        if (t.n == 0) continue;
        const uint32_t buf = done % bufs;
        if (!mbar_wait(acc_empty(buf), ((done / bufs) & 1) ^ 1)) {
          atomicExch(g.a.flag, 2);
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + buf * 256u, acc_lo = acc + (bufs == 2 ? 128u : 256u);
        const int steps = (t.n + 31) / 32;
        for (int ks = 0; ks < steps; ++ks, ++st) {
          const int s = st % g.stages;
          if (!mbar_wait(full(s), (st / g.stages) & 1)) {
            atomicExch(g.a.flag, 3);
            alive = false;
            break;
          }
          tc_fence_after();
          const uint32_t sb = base + (uint32_t)(s * g.stage_bytes);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t o = (uint32_t)kk * 1024u;
            const uint64_t vh = desc_mn_major(sb + o), vl = desc_mn_major(sb + 16384u + o);
            const uint64_t kh = desc_mn_major(sb + k_off + o), kl = desc_mn_major(sb + k_off + k_bytes + o);
            tc_mma_tf32(acc_lo, vl, kh, idesc, (ks | kk) != 0);
            tc_mma_tf32(acc_lo, vh, kl, idesc, 1);
            tc_mma_tf32(acc, vh, kh, idesc, (ks | kk) != 0);
          }
          tc_commit(empty(s));
        }
        if (!alive) break;
        tc_commit(acc_full(buf));
        ++done;
      }
    }
  } else {
    const int q = warp & 3;
    const uint32_t tile = tiles + (uint32_t)q * 4096u;
    uint32_t done = 0;
    for (int i = blockIdx.x; i < g.items; i += gridDim.x) {
      const Item t = item_of(g, i);
      if (t.n == 0) continue;
      const uint32_t buf = done % bufs;
      if (!warp_wait(acc_full(buf), (done / bufs) & 1)) {
        if (lane == 0) atomicExch(g.a.flag, 4);
        break;
      }
      tc_fence_after();
      float* out = g.states + ((uint64_t)t.unit * g.chunks + t.c) * g.a.dv * g.a.dk;
      if (q * 32 < g.dvp)
        for (int cb = 0; cb < nbk; ++cb) {
          float v[32];
          const uint32_t acc = tmem + buf * 256u + ((uint32_t)(q * 32) << 16) + (uint32_t)(cb * 32);
          tmem_load_sum32(acc, acc + (bufs == 2 ? 128u : 256u), v);
          store_rows32<WIDE>(tile, lane, v, cb * 32, g.a.dk, [&](int r) -> float* {
            const int row = t.dv0 + q * 32 + r;
            return row < g.a.dv ? out + (uint64_t)row * g.a.dk : nullptr;
          });
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(buf));
      ++done;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---- states between the chunks -----------------------------------------------------------
// A thread carries V neighbouring elements of the (transposed) state through all chunks of its
// row; eight chunks are in flight, since each is a dependent step of two multiply-adds (the decay of a
// chunk is in two parts: in one, its error grows by the same amount with every chunk, to 106 * 2^-24 over
// 128 chunks at decays of 1 - 10^-5 or so).
template <int V>
__global__ void __launch_bounds__(256)
linear_chunk_scan_kernel(const ChunkArgs g, int blocks_per_unit) {
  const int unit = blockIdx.x / blocks_per_unit;
  const int e = ((blockIdx.x - unit * blocks_per_unit) * 256 + (int)threadIdx.x) * V;
  const int size = g.a.dv * g.a.dk;
  if (e >= size) return;
  const int b = unit / g.a.heads, h = unit - b * g.a.heads;
  const int n = linear_length(g.a, b);
  const int nc = (n + kC - 1) / kC;
  const int row = e / g.a.dk, col = e - row * g.a.dk;      // dim_v, dim_k (V divides dim_k)
  const uint64_t at = (uint64_t)unit * size + (uint64_t)col * g.a.dv + row;
  const float ld = __ldg(g.a.log_decay + h);
  const Factor whole = factor_of(decay_power_exact(ld, kC)), last = factor_of(decay_power_exact(ld, n - (nc - 1) * kC));
  struct __align__(V * 4) Vec { float x[V]; };
  Vec s;
#pragma unroll
  for (int v = 0; v < V; ++v) s.x[v] = g.a.state ? __ldg(g.a.state + at + (uint64_t)v * g.a.dv) : 0.f;
  float* p = g.states + (uint64_t)unit * g.chunks * size + e;
  // (two batches: loads behind a batch's stores would otherwise wait for them; 2 x 16 heads of
  // 128 x 128, 128 chunks: 210 us with one batch of eight in flight)
  constexpr int U = 8;
  Vec x[2][U];
  auto load = [&](int c, Vec (&y)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + u < nc) y[u] = *reinterpret_cast<const Vec*>(p + (uint64_t)(c + u) * size);
  };
  auto step = [&](int c, const Vec (&y)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + u < nc) {
        *reinterpret_cast<Vec*>(p + (uint64_t)(c + u) * size) = s;
        const Factor w = c + u + 1 < nc ? whole : last;
#pragma unroll
        for (int v = 0; v < V; ++v) s.x[v] = times_plus(w, s.x[v], y[u].x[v]);
      }
  };
  load(0, x[0]);
  for (int c = 0; c < nc; c += 2 * U) {
    load(c + U, x[1]);
    step(c, x[0]);
    load(c + 2 * U, x[0]);
    step(c + U, x[1]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) g.a.out_state[at + (uint64_t)v * g.a.dv] = s.x[v];
}

// ---- outputs -------------------------------------------------------------------------------
// Tensor memory, in columns (hi hi sums left, sums of the small products right):
//   [0, 128) scores, later the probabilities' hi parts     [256, 384) scores, later their lo parts
//   [128, 256) Q S, later decayed                          [384, 512) Q S, later P V
// Eight producer warps, eight that read tensor memory.
constexpr int kOutThreads = 512;

// The second product multiplies values of v behind a token by zeros, which hides all but a NaN and an
// infinity (a value above 2^127 becomes one when it is split).  Where a chunk has such a value its outputs are
// computed once more, by the whole block, from the sums that the tokens have: slow, and nothing else needs it.
__device__ __noinline__ void outputs_again(const ChunkArgs& g, int item, float* scores) {
  const Item t = item_of(g, item);
  const int cols = g.a.dv - t.dv0 < 128 ? g.a.dv - t.dv0 : 128;
  const uint64_t row0 = (uint64_t)t.unit * g.a.seq + (uint64_t)t.c * kC;
  const float* v = g.a.v + row0 * g.a.dv + t.dv0;
  bool found = false;
  for (int i = threadIdx.x; i < t.n * cols; i += kOutThreads)
    found |= !(fabsf(__ldg(v + (uint64_t)(i / cols) * g.a.dv + i % cols)) <= 1.7014118e38f);
  if (!__syncthreads_or(found)) return;
  const float ld = __ldg(g.a.log_decay + t.h);
  for (int i = threadIdx.x; i < t.n * kC; i += kOutThreads) {
    const int row = i / kC, col = i % kC;
    if (col > row) continue;
    float sum = 0.f;
    for (int d = 0; d < g.a.dk; ++d)
      sum = fmaf(__ldg(g.a.q + (row0 + row) * g.a.dk + d), __ldg(g.a.k + (row0 + col) * g.a.dk + d), sum);
    scores[i] = sum * decay_power(ld, row - col);
  }
  __syncthreads();
  const float* state = g.states + (((uint64_t)t.unit * g.chunks + t.c) * g.a.dv + t.dv0) * g.a.dk;
  for (int i = threadIdx.x; i < t.n * cols; i += kOutThreads) {
    const int row = i / cols, col = i % cols;
    float sum = 0.f;
    for (int d = 0; d < g.a.dk; ++d)
      sum = fmaf(__ldg(g.a.q + (row0 + row) * g.a.dk + d), state[(uint64_t)col * g.a.dk + d], sum);
    sum *= decay_power(ld, row + 1);
    for (int j = 0; j <= row; ++j) sum = fmaf(scores[row * kC + j], __ldg(v + (uint64_t)j * g.a.dv + col), sum);
    g.a.out[(((uint64_t)t.b * g.a.seq + t.c * kC + row) * g.a.heads + t.h) * g.a.dv + t.dv0 + col] =
        g.a.has_scale ? __fmul_rn(sum, g.a.scale) : sum;
  }
  __syncthreads();
}

template <bool WIDE>
__global__ void __launch_bounds__(kOutThreads, 1)
linear_chunk_outputs_kernel(const __grid_constant__ ChunkArgs g) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t tiles = base + (uint32_t)(g.stages * g.stage_bytes);
  const uint32_t bars = tiles + 8 * 4096u;
  auto full = [&](int s) { return bars + 8u * (uint32_t)s; };
  auto empty = [&](int s) { return bars + 8u * (uint32_t)(kMaxStages + s); };
  const uint32_t s_full = bars + 8u * (2 * kMaxStages), o_full = s_full + 8u;
  const uint32_t tmem_slot = s_full + 16u;
  const uint32_t power_s = tmem_slot + 8u;                 // float[kC + 1]
  float* power = reinterpret_cast<float*>(smem_raw + (power_s - smem_u32(smem_raw)));
  int* again = reinterpret_cast<int*>(power + kC + 2);     // first and last item to compute again
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    again[0] = 0x7fffffff;
    again[1] = -1;
    for (int s = 0; s < g.stages; ++s) {
      mbar_init(full(s), kProducers);
      mbar_init(empty(s), 1);
    }
    mbar_init(s_full, 1);
    mbar_init(o_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kProducers) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  const uint32_t t_s = tmem, t_inter = tmem + 128u, t_lo = tmem + 256u, t_out = tmem + 384u;

  // a stage holds either 32 columns of Q (128 rows, hi then lo) and of [K; S^T] (128 + dvp rows,
  // hi then lo), or 64 tokens of V (two groups of 32, each dvp / 32 column blocks; hi then lo)
  const int nk = g.dkp / 32, nbv = g.dvp / 32;
  const uint32_t b_off = 32768u, b_bytes = (uint32_t)(128 + g.dvp) * 128u;
  const uint32_t v_bytes = 64u * (uint32_t)g.dvp * 4u;
  if (warp < kProducers) {
    // A thread has a 16-byte piece of every 32nd operand row: of 128 of Q, 128 of K, dvp of S^T; or of
    // each column block of two tokens of V.  Two stages are in flight, as above.
    const int r0 = (int)threadIdx.x >> 3, c4 = (int)threadIdx.x & 7;
    constexpr int S = 12;
    struct Stage {
      int i, ks;                                   // ks: nk stages of Q, K, S, then those of V
      Item t;
    };
    auto settle = [&](Stage& s) {
      for (; s.i < g.items; s.i += gridDim.x) {
        s.t = item_of(g, s.i);
        if (s.t.n > 0) break;
      }
      s.ks = 0;
    };
    auto next = [&](Stage& s) {
      if (++s.ks >= nk + (s.t.n + 63) / 64) {
        s.i += gridDim.x;
        settle(s);
      }
    };
    auto load = [&](const Stage& s, float4 (&x)[S]) {
      if (s.i >= g.items) return;
      // (One load a place whichever kind of stage it is: with two, the compiler copies what one of them
      // brings, which waits for it, and nothing is in flight any more.)
      const uint64_t row0 = (uint64_t)s.t.unit * g.a.seq + (uint64_t)s.t.c * kC;
      const bool is_v = s.ks >= nk;
      const int d = s.ks * 32 + c4 * 4;
      const int j0 = (s.ks - nk) * 64 + r0;                // V: this thread's tokens are j0 and j0 + 32
      const uint64_t at = (row0 + r0) * g.a.dk + d;
      const float* p0 = g.a.q + at;
      const float* p1 = g.a.k + at;
      const float* p2 = g.states + (((uint64_t)s.t.unit * g.chunks + s.t.c) * g.a.dv + s.t.dv0 + r0) * g.a.dk + d;
      uint32_t by = 32u * (uint32_t)g.a.dk;
      if (is_v) {
        p0 = g.a.v + (row0 + j0) * g.a.dv + s.t.dv0 + c4 * 4;
        p1 = p0 + 32u * (uint32_t)g.a.dv;
        by = 32u;
      }
      if (WIDE) {
        uint32_t m0 = 0u, m1 = 0u, m2 = 0u;
        if (is_v) {
          const uint32_t cols = places(g.a.dv - s.t.dv0 - c4 * 4, 4);
          m0 = j0 < s.t.n ? cols : 0u;
          m1 = j0 + 32 < s.t.n ? cols : 0u;
        } else if (d < g.a.dk) {
          m0 = m1 = places(s.t.n - r0, 4);
          m2 = places(g.a.dv - s.t.dv0 - r0, 4);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          x[y] = load16(p0 + y * by, m0 >> y & 1u);
          x[4 + y] = load16(p1 + y * by, m1 >> y & 1u);
          x[8 + y] = load16(p2 + y * by, m2 >> y & 1u);
        }
      } else {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int col = is_v ? s.t.dv0 + y * 32 + c4 * 4 : d, dim = is_v ? g.a.dv : g.a.dk;
          const bool row_in = y * 32 + r0 < s.t.n;
          x[y] = load_cols4(p0 + y * by, col, dim, is_v ? y < nbv && j0 < s.t.n : row_in);
          x[4 + y] = load_cols4(p1 + y * by, col, dim, is_v ? y < nbv && j0 + 32 < s.t.n : row_in);
          x[8 + y] = load_cols4(p2 + y * by, col, dim, !is_v && y < nbv && s.t.dv0 + y * 32 + r0 < g.a.dv);
        }
      }
    };
    uint32_t slot = 0, phase = 1;
    const uint32_t at_k = k_major(r0, c4), at_mn = mn_major(r0, c4);
    auto store = [&](const Stage& s, float4 (&x)[S]) -> bool {
      const uint32_t sb = base + slot * (uint32_t)g.stage_bytes;
      if (!warp_wait(empty(slot), phase)) {
        if (lane == 0) atomicExch(g.a.flag, 1);
        return false;
      }
      if (s.ks < nk) {
        const uint32_t q_at = sb + at_k, b_at = q_at + b_off, b_lo = b_at + b_bytes;
#pragma unroll
        for (int y = 0; y < 4; ++y) store_split(q_at + y * 4096u, q_at + 16384u + y * 4096u, x[y]);
#pragma unroll
        for (int y = 0; y < 8; ++y)                // rows 128 on of B are those of S^T
          if (y < 4 + nbv) store_split(b_at + y * 4096u, b_lo + y * 4096u, x[4 + y]);
      } else {
#pragma unroll
        for (int tg = 0; tg < 2; ++tg)
#pragma unroll
          for (int cb = 0; cb < 4; ++cb)
            if (cb < nbv) {
              const uint32_t at = sb + at_mn + (uint32_t)(tg * nbv + cb) * 4096u;
              store_split(at, at + v_bytes, x[tg * 4 + cb]);
            }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(full(slot));
      if (++slot == (uint32_t)g.stages) {
        slot = 0;
        phase ^= 1;
      }
      return true;
    };
    Stage a, b;
    float4 xa[S], xb[S];
    a.i = blockIdx.x;
    settle(a);
    load(a, xa);
    while (a.i < g.items) {
      b = a;
      next(b);
      load(b, xb);
      if (!store(a, xa) || b.i >= g.items) break;
      a = b;
      next(a);
      load(a, xa);
      if (!store(b, xb)) break;
    }
  } else {
    // The first of these warps also issues the MMAs, of which its first thread: they have nothing
    // else to do while the scores are formed.
    const bool issuer = warp == kProducers;
    const uint32_t idesc_s = kIdesc | n_field(128 + g.dvp);
    const uint32_t idesc_o = kIdesc | kBMN | n_field(g.dvp);
    uint32_t slot = 0, phase = 0;
    auto advance = [&](uint32_t& s, uint32_t& p) {
      if (++s == (uint32_t)g.stages) {
        s = 0;
        p ^= 1;
      }
    };
    // scores (and Q S) of an item, stage by stage
    auto issue_scores = [&]() -> bool {
      for (int ks = 0; ks < nk; ++ks) {
        if (!warp_wait(full(slot), phase)) {
          if (lane == 0) atomicExch(g.a.flag, 2);
          return false;
        }
        tc_fence_after();
        if (lane == 0) {
          const uint32_t sb = base + slot * (uint32_t)g.stage_bytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t o = (uint32_t)kk * 32u;
            const uint64_t qh = desc_k_major(sb + o), ql = desc_k_major(sb + 16384u + o);
            const uint64_t bh = desc_k_major(sb + b_off + o), bl = desc_k_major(sb + b_off + b_bytes + o);
            tc_mma_tf32(t_lo, ql, bh, idesc_s, (ks | kk) != 0);
            tc_mma_tf32(t_lo, qh, bl, idesc_s, 1);
            tc_mma_tf32(t_s, qh, bh, idesc_s, (ks | kk) != 0);
          }
          tc_commit(empty(slot));
          if (ks == nk - 1) tc_commit(s_full);
        }
        __syncwarp();
        advance(slot, phase);
      }
      return true;
    };
    // P V: all small products first, while the sum is small; both halves of V are there by then (at
    // least two stages).  (Straight code for each half: a branch an MMA makes one take 140 cycles to
    // issue, twice what it takes to run.)
    auto issue_values = [&](int n) -> bool {
      const bool two = n > 64;
      const uint32_t s0 = slot, sb0 = base + s0 * (uint32_t)g.stage_bytes;
      if (!warp_wait(full(slot), phase)) {
        if (lane == 0) atomicExch(g.a.flag, 4);
        return false;
      }
      advance(slot, phase);
      uint32_t s1 = s0;
      if (two) {
        s1 = slot;
        if (!warp_wait(full(slot), phase)) {
          if (lane == 0) atomicExch(g.a.flag, 4);
          return false;
        }
        advance(slot, phase);
      }
      const uint32_t sb1 = base + s1 * (uint32_t)g.stage_bytes;
      const uint32_t group = (uint32_t)nbv * 4096u;
      auto small = [&](uint32_t sb, uint32_t col0, uint32_t begun) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t o = sb + (kk >= 4 ? group : 0u) + (uint32_t)(kk & 3) * 1024u, col = col0 + (uint32_t)(kk * 8);
          mma_tmem_a(t_out, t_lo + col, desc_mn_major(o), idesc_o, kk ? 1u : begun);
          mma_tmem_a(t_out, t_s + col, desc_mn_major(o + v_bytes), idesc_o, 1u);
        }
      };
      auto large = [&](uint32_t sb, uint32_t col0) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          mma_tmem_a(t_out, t_s + col0 + (uint32_t)(kk * 8),
                     desc_mn_major(sb + (kk >= 4 ? group : 0u) + (uint32_t)(kk & 3) * 1024u), idesc_o, 1u);
      };
      tc_fence_after();
      if (lane == 0) {
        small(sb0, 0u, 0u);
        if (two) small(sb1, 64u, 1u);
        large(sb0, 0u);
        tc_commit(empty(s0));
        if (two) {
          large(sb1, 64u);
          tc_commit(empty(s1));
        }
        tc_commit(o_full);
      }
      __syncwarp();
      return true;
    };
    auto all_warps = []() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    const int q = warp & 3, half = (warp - kProducers) >> 2;   // two warps a quarter: every second block
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    const uint32_t tile = tiles + (uint32_t)(warp - kProducers) * 4096u;
    const int tok = q * 32 + lane;                         // this thread's row
    uint32_t done = 0;
    int powers_of = -1;
    bool alive = true;
    for (int i = blockIdx.x; i < g.items; i += gridDim.x) {
      const Item t = item_of(g, i);
      const uint64_t first = (uint64_t)t.b * g.a.seq + (uint64_t)t.c * kC;
      auto out_row = [&](int r) -> float* {
        const int token = q * 32 + r;
        return t.c * kC + token < g.a.seq ? g.a.out + ((first + token) * g.a.heads + t.h) * g.a.dv + t.dv0 : nullptr;
      };
      const int cols = g.a.dv - t.dv0 < 128 ? g.a.dv - t.dv0 : 128;
      if (t.n == 0) {
        float z[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) z[x] = 0.f;
        for (int cb = half; cb < nbv; cb += 2) store_rows32<WIDE>(tile, lane, z, cb * 32, cols, out_row);
        continue;
      }
      if (t.h != powers_of) {                              // (the same for all eight warps)
        all_warps();
        const float ld = __ldg(g.a.log_decay + t.h);
        const int e = (int)threadIdx.x - kProducers * 32;
        if (e <= kC) power[e] = decay_power(ld, e);
        all_warps();
        powers_of = t.h;
      }
      // (a warp that gave up takes part in the barriers alone)
      if (issuer && alive) alive = issue_scores();
      if (alive && !warp_wait(s_full, done & 1)) {
        if (lane == 0) atomicExch(g.a.flag, 5);
        alive = false;
      }
      tc_fence_after();
      if (alive) {
#pragma unroll 1
      for (int j0 = half * 32; j0 < kC; j0 += 64) {
        float x[32], lo[32];
        if (j0 <= q * 32) {
          tmem_load_sum32(t_s + lanes + (uint32_t)j0, t_lo + lanes + (uint32_t)j0, x);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int ago = tok - (j0 + j);
            const float p = ago >= 0 ? x[j] * power[ago < 0 ? 0 : ago] : 0.f;
            x[j] = tf32_hi(p);
            lo[j] = p - x[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = lo[j] = 0.f;
        }
        tmem_store32(t_s + lanes + (uint32_t)j0, x);
        tmem_store32(t_lo + lanes + (uint32_t)j0, lo);
      }
      const float w = power[tok + 1];
#pragma unroll 1
      for (int cb = half; cb < nbv; cb += 2) {
        float x[32];
        tmem_load_sum32(t_inter + lanes + (uint32_t)(cb * 32), t_out + lanes + (uint32_t)(cb * 32), x);
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] *= w;
        tmem_store32(t_inter + lanes + (uint32_t)(cb * 32), x);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      tc_fence_before();
      all_warps();                                        // the probabilities of all rows are there
      tc_fence_after();
      if (issuer && alive) alive = issue_values(t.n);
      if (alive && !warp_wait(o_full, done & 1)) {
        if (lane == 0) atomicExch(g.a.flag, 6);
        alive = false;
      }
      tc_fence_after();
      if (alive) {
      const bool real = tok < t.n;
      const float scale = g.a.has_scale ? g.a.scale : 1.0f;
#pragma unroll 1
      for (int cb = half; cb < nbv; cb += 2) {
        float x[32];
        tmem_load_sum32(t_out + lanes + (uint32_t)(cb * 32), t_inter + lanes + (uint32_t)(cb * 32), x);
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = real ? __fmul_rn(x[j], scale) : 0.0f;
        store_rows32<WIDE>(tile, lane, x, cb * 32, cols, out_row);
      }
      }
      tc_fence_before();
      all_warps();                                        // all sums are read: the next products may come
      tc_fence_after();
      ++done;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kProducers) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  // A value of v that is not finite has made its column NaN for all tokens of its chunk, so the first token
  // tells (read back here, since a look at the values on their way out took 3% of the time).
  int from = 0x7fffffff, to = -1;
#pragma unroll 8
  for (int i = blockIdx.x + (int)(threadIdx.x >> 7) * gridDim.x; i < g.items; i += kOutThreads / 128 * gridDim.x) {
    const int uc = i / g.dv_tiles, unit = uc / g.chunks, b = unit / g.a.heads;
    const int d = (i - uc * g.dv_tiles) * 128 + (int)(threadIdx.x & 127);
    // (behind a row's end are zeros)
    const uint64_t at = (((uint64_t)b * g.a.seq + (uint64_t)(uc - unit * g.chunks) * kC) * g.a.heads + (unit - b * g.a.heads)) * g.a.dv + d;
    const float x = d < g.a.dv ? __ldcg(g.a.out + at) : 0.f;
    if (!(fabsf(x) <= kMostFloat)) {
      from = min(from, i);
      to = i;
    }
  }
  if (to >= 0) {
    atomicMin(again, from);
    atomicMax(again + 1, to);
  }
  __syncthreads();
  const int last = again[1];
  for (int i = again[0]; i <= last; i += gridDim.x)
    outputs_again(g, i, reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw))));
}

template <bool WIDE>
int launch_chunks(tfjs_cuda_ctx* ctx, ChunkArgs& g) {
  // chunk_states: 32 tokens of V (four blocks whatever dim_v, the MMA reads 128 columns) and K
  ChunkArgs s = g;
  s.stage_bytes = 2 * 16384 + 2 * (g.dkp / 32) * 4096;
  const int s_fixed = 1024 + 4 * 4096 + 256;
  s.stages = (kSmemCap - s_fixed) / s.stage_bytes;
  if (s.stages > kMaxStages) s.stages = kMaxStages;
  const int s_smem = s_fixed + s.stages * s.stage_bytes;
  const unsigned grid = (unsigned)(g.items < ctx->sm_count ? g.items : ctx->sm_count);
  if (g.dkp <= 128) {
    CUDA_TRY(ctx, cudaFuncSetAttribute(linear_chunk_states_kernel<WIDE, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap));
    linear_chunk_states_kernel<WIDE, 4><<<grid, kStateThreads, s_smem, ctx->stream>>>(s);
  } else {
    CUDA_TRY(ctx, cudaFuncSetAttribute(linear_chunk_states_kernel<WIDE, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap));
    linear_chunk_states_kernel<WIDE, 8><<<grid, kStateThreads, s_smem, ctx->stream>>>(s);
  }
  LAUNCH_CHECK(ctx, "linear_chunk_states_kernel");
  const unsigned units = (unsigned)(g.a.batch * g.a.heads);
  const int V = g.a.dk % 4 == 0 ? 4 : 1, per = (g.a.dv * g.a.dk / V + 255) / 256;
  if (V == 4)
    linear_chunk_scan_kernel<4><<<units * per, 256, 0, ctx->stream>>>(g, per);
  else
    linear_chunk_scan_kernel<1><<<units * per, 256, 0, ctx->stream>>>(g, per);
  LAUNCH_CHECK(ctx, "linear_chunk_scan_kernel");
  const int qk = 32768 + 2 * (128 + g.dvp) * 128, v = 2 * 64 * g.dvp * 4;
  g.stage_bytes = qk > v ? qk : v;
  const int o_fixed = 1024 + 8 * 4096 + 256 + (kC + 4) * 4;
  g.stages = (kSmemCap - o_fixed) / g.stage_bytes;
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  const int o_smem = o_fixed + g.stages * g.stage_bytes;
  CUDA_TRY(ctx, cudaFuncSetAttribute(linear_chunk_outputs_kernel<WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap));
  linear_chunk_outputs_kernel<WIDE><<<grid, kOutThreads, o_smem, ctx->stream>>>(g);
  LAUNCH_CHECK(ctx, "linear_chunk_outputs_kernel");
  return TFJS_CUDA_OK;
}

}  // namespace

int launch_linear_chunked(tfjs_cuda_ctx* ctx, const LinearArgs& a) {
  ChunkArgs g;
  g.a = a;
  g.chunks = (a.seq + kC - 1) / kC;
  g.dv_tiles = (a.dv + 127) / 128;
  const uint64_t units = (uint64_t)a.batch * a.heads;
  if (units * g.chunks * g.dv_tiles > 0x7fffffffull || units * ((uint64_t)a.dv * a.dk / 256 + 1) > 0x7fffffffull)
    return ctx_fail(ctx, TFJS_CUDA_UNSUPPORTED, "linear attention: too many tokens for one call");
  g.items = (int)(units * g.chunks * g.dv_tiles);
  const int tile = a.dv < 128 ? a.dv : 128;
  g.dvp = (tile + 31) / 32 * 32;
  g.dkp = (a.dk + 31) / 32 * 32;
  TempBuffer ws(ctx);
  void* mem;
  int rc = ws.get(units * g.chunks * (uint64_t)a.dv * a.dk * 4, &mem);
  if (rc) return rc;
  g.states = (float*)mem;
  const bool wide = a.dk % 4 == 0 && a.dv % 4 == 0 &&
                    (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0;
  return wide ? launch_chunks<true>(ctx, g) : launch_chunks<false>(ctx, g);
}
