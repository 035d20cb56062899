// tcb/nll_common.cuh -- what both forms of the cross entropy share: logits in units of log 2, maxima and sums of
// exponentials joined.
#pragma once

#ifndef TCB_BIAS
#define TCB_BIAS 1
#endif

namespace tcb {

constexpr float NLL_LOG2E = 1.44269504f, NLL_LN2 = 0.693147181f, NLL_MAX = 3.402823466e38f;
#define TCB_MINUS_INF bits(0xff800000u)

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// b log2(e); a mask of the lowest float stays finite
__device__ __forceinline__ float nll_bias2(float b) {
  return fabsf(b) <= NLL_MAX ? fmaxf(fminf(b * NLL_LOG2E, NLL_MAX), -NLL_MAX) : b;
}
// a row's class, or -1 when it takes no part
__device__ __forceinline__ int nll_class(float t, u64 V) { return t >= 0.0f && t < (float)V ? (int)t : -1; }
__device__ __forceinline__ void nll_join(float& m, float& s, const float2& x) {
  const float mx = fmaxf(m, x.x), safe = mx == TCB_MINUS_INF ? 0.0f : mx;
  s = s * ex2(m - safe) + x.y * ex2(x.x - safe);
  m = mx;
}
// A row's loss from its maximum, its sum of exponentials and the target's logit (units of log 2); bias: all of it,
// not read without one.  A bias below -2.36e38, a mask of the lowest float say, leaves the range in units of log 2
// and stands at its end, beyond what the others' logits can move: that target's loss takes the bias itself.
__device__ __forceinline__ float nll_loss(float m, float s, float z, int t, const float* bias) {
  if (t < 0) return 0.0f;
  if (TCB_BIAS && z <= -NLL_MAX && m > z) return fmaf(m, NLL_LN2, logf(s)) - __ldg(bias + t);
  return (m - z) * NLL_LN2 + logf(s);
}

}  // namespace tcb
