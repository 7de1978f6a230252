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
__device__ __forceinline__ LpSums lp_rescale(const LpSums& a, float m) {
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
// Log normaliser, entropy and log probability of a logit z of a row; nothing left: -inf, 0, -inf.
__device__ __forceinline__ float lp_lse(const LpSums& a) { return a.s == 0.f ? -INFINITY : a.m + logf(a.s); }
__device__ __forceinline__ float lp_entropy(const LpSums& a) { return a.s == 0.f ? 0.f : logf(a.s) - a.t / a.s; }
__device__ __forceinline__ float lp_log(float z, const LpSums& a) { return z == -INFINITY ? z : lp_gap(z, a.m) - logf(a.s); }
// A logit as the row's distribution has it: softcap * tanh((x + bias[j]) * scale / softcap), NaN as -inf.
__device__ __forceinline__ float lp_transform(float x, int j, const void* bias, int bias_fp32, float scale, float softcap) {
  if (bias != nullptr) x += bias_fp32 ? static_cast<const float*>(bias)[j] : __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[j]);
  x *= scale;
  if (softcap > 0.f) x = softcap * tanhf(x / softcap);
  return x != x ? -INFINITY : x;
}
__device__ __forceinline__ float lp_exp2(float x) {                    // 2 ulp; subnormal results are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Logits of ordinary size. Beyond, neighbouring numbers are so far apart that a logit weighs 1 where it equals m and nothing where not;
// that holds for infinities too.
__device__ __forceinline__ bool lp_plain(float m) { return fabsf(m) < 1e30f; }
// Logits below this weigh nothing beside m (e^-150 at most), and count as it: for masked values z - m would be no number that can be
// multiplied by a weight of 0. 256 below m or, where that is no step of m, |m| / 64. For m of ordinary size.
__device__ __forceinline__ float lp_floor(float m) { return m - fmaxf(256.f, fabsf(m) * 0.015625f); }

// Two fp32 operations in one instruction.
using lp_pair = unsigned long long;
__device__ __forceinline__ lp_pair lp_two(float a, float b) {
  lp_pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 lp_both(lp_pair a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ lp_pair lp_add2(lp_pair a, lp_pair b) {
  lp_pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ lp_pair lp_fma2(lp_pair a, lp_pair b, lp_pair c) {
  lp_pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ lp_pair lp_mul2(lp_pair a, lp_pair b) {
  lp_pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Adds the logits z[N], none below lp_floor(m), to (s, t) of the largest logit m.
template <int N>
__device__ __forceinline__ void lp_add(const float (&z)[N], lp_pair minus_m, lp_pair& s, lp_pair& t) {
  const lp_pair l2e = lp_two(kLog2e, kLog2e);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const lp_pair d = lp_add2(lp_two(z[j], z[j + 1]), minus_m);
    const float2 u = lp_both(lp_mul2(d, l2e));
    const lp_pair e = lp_two(lp_exp2(u.x), lp_exp2(u.y));
    s = lp_add2(s, e);
    t = lp_fma2(e, d, t);
  }
}

}  // namespace mx
