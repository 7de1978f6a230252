// What the kernels of log probabilities share (logprobs.cu, head_logprobs.cu): a row's running sums and their joining.
#pragma once
#include "common.cuh"

namespace mx {

constexpr float kLog2e = 1.4426950408889634f;

// What a part of a row adds up to: the largest logit m, s = sum e^(z - m), t = sum e^(z - m) (z - m).
struct LpSums {
  float m, s, t;
};
// z - m where both may be infinite: equal infinities are at distance 0.
__device__ __forceinline__ float lp_gap(float z, float m) { return z == m ? 0.f : z - m; }
__device__ __forceinline__ LpSums lp_rescale(LpSums a, float m) {
  const float d = lp_gap(a.m, m), e = exp2f(d * kLog2e);
  if (e == 0.f) return {m, 0.f, 0.f};                                 // (d can be -inf, or s * d overflow)
  return {m, a.s * e, (a.t + a.s * d) * e};
}
__device__ __forceinline__ LpSums lp_join(const LpSums& a, const LpSums& b) {
  if (a.s == 0.f) return b;
  if (b.s == 0.f) return a;
  const float m = fmaxf(a.m, b.m);
  const LpSums x = lp_rescale(a, m), y = lp_rescale(b, m);
  return {m, x.s + y.s, x.t + y.t};
}
__device__ __forceinline__ LpSums lp_warp_join(LpSums a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const LpSums b = {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)};
    // (both lanes of a pair join in the same order, so that all lanes end with the same bits)
    a = (threadIdx.x & o) ? lp_join(b, a) : lp_join(a, b);
  }
  return a;
}
// A logit as the row's distribution has it: softcap * tanh((x + bias[j]) * scale / softcap), NaN as -inf.
__device__ __forceinline__ float lp_transform(float x, int j, const void* bias, int bias_fp32, float scale, float softcap) {
  if (bias != nullptr) x += bias_fp32 ? static_cast<const float*>(bias)[j] : __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[j]);
  x *= scale;
  if (softcap > 0.f) x = softcap * tanhf(x / softcap);
  return x != x ? -INFINITY : x;
}
__device__ __forceinline__ float lp_log(float z, float m, float log_s) { return z == -INFINITY ? z : lp_gap(z, m) - log_s; }
__device__ __forceinline__ float lp_exp2(float x) {                    // 2 ulp; subnormal results are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace mx
