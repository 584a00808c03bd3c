// What the two forms of linear attention (linear_attention.cu: one token after the other;
// linear_attention_sm100.cu: chunks of 128 tokens on the tensor cores) share.
#pragma once
#include "common.cuh"

struct LinearArgs {
  const float *q, *k, *v, *log_decay, *state;   // state: or null
  const int* lengths;                           // or null
  float *out, *out_state;
  int batch, heads, seq, dk, dv;
  int has_scale;
  float scale;
  int* flag;
};

int launch_linear_chunked(tfjs_cuda_ctx* ctx, const LinearArgs& a);

namespace {

// Tokens of row b, clamped to [0, seq]; a length outside that is reported.
__device__ __forceinline__ int linear_length(const LinearArgs& a, int b) {
  if (!a.lengths) return a.seq;
  const int n = __ldg(a.lengths + b);
  if (n < 0 || n > a.seq) {
    atomicOr(a.flag, kBadLength);
    return n < 0 ? 0 : a.seq;
  }
  return n;
}

// A positive factor that is applied again and again, in two parts: rounded to one float, its error would
// have the same sign each time and grow with the steps.  The large part is rounded down and the small one
// is never 0 beside it (at least 2^-149), so that both keep the sign of an infinite value and it stays what
// it is; a test of every value for that took a quarter more time (1024 states of 128 x 128, 32 tokens:
// 299 us a call, here 236).
struct Factor {
  float hi, lo;
};
__device__ __forceinline__ Factor factor_of(double exact) {
  Factor f;
  f.hi = __double2float_rz(exact);
  f.lo = (float)(exact - (double)f.hi);
  if (f.hi > 0.0f && !(f.lo > 0.0f)) f.lo = __int_as_float(1);
  return f;
}
// f s + x
__device__ __forceinline__ float times_plus(Factor f, float s, float x) { return fmaf(f.hi, s, fmaf(f.lo, s, x)); }
constexpr float kMostFloat = 3.402823466e38f;
// decay^e, in double
__device__ __forceinline__ double decay_power_exact(float log_decay, int e) {
  return e == 0 ? 1.0 : exp((double)log_decay * e);
}

// decay^e for a whole number e >= 0 (decay 0 included: 0^0 = 1)
__device__ __forceinline__ float decay_power(float log_decay, int e) {
  return e == 0 ? 1.0f : expf(__fmul_rn(log_decay, (float)e));
}

}  // namespace
