// Log probabilities of given tokens, entropy and the most likely tokens of every row of logits:
//
//   z = x (+ bias), times scale, soft-capped;  lse = log sum_j e^(z_j);  log p(id) = z_id - lse;  H = lse - sum_j p_j z_j
//
// NaN counts as -inf. A row with nothing left (all -inf) has lse = -inf, log probabilities -inf and entropy 0. Equal logits order by
// index. An id outside the vocabulary has log probability NaN.
#include "api.h"
#include "common.cuh"
#include "logprobs.cuh"
#include "typed.cuh"

namespace mx {

constexpr int kLpThreads = 512;
struct LpParams {
  const void* logits;
  const void* ids;
  const void* bias;
  float* logprob;
  float* entropy;
  float* lse;
  int* top_ids;
  float* top_logprobs;
  long long ld;
  int V, n_ids, ids64, bias_fp32, top;
  float scale, softcap;
};

// A logit as the row's distribution has it.
__device__ __forceinline__ float lp_value(const LpParams& p, float x, int j) { return lp_transform(x, j, p.bias, p.bias_fp32, p.scale, p.softcap); }

// Orders by value, then by lower index; 0 is below every pair.
__device__ __forceinline__ unsigned long long lp_key(float z, int j) {
  uint32_t u = __float_as_uint(z + 0.f);                              // (-0 equals 0)
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<unsigned long long>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(j));
}
__device__ __forceinline__ int lp_key_index(unsigned long long k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float lp_key_value(unsigned long long k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LpParams p) {
  __shared__ float part[3][kLpThreads / 32];
  __shared__ unsigned long long best[kLpThreads / 32];
  pdl_trigger();
  pdl_wait();
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  LpSums a{-INFINITY, 0.f, 0.f};
  for (int j = threadIdx.x; j < p.V; j += kLpThreads) {
    const float z = lp_value(p, to_f(x[j]), j);
    if (z == -INFINITY) continue;
    if (z > a.m) a = lp_rescale(a, z);
    const float d = lp_gap(z, a.m), e = exp2f(d * kLog2e);
    a.s += e;
    if (e > 0.f) a.t += e * d;
  }
  a = lp_warp_join(a);
  if (lane == 0) part[0][warp] = a.m, part[1][warp] = a.s, part[2][warp] = a.t;
  __syncthreads();
  a = {part[0][0], part[1][0], part[2][0]};
  for (int i = 1; i < kLpThreads / 32; ++i) a = lp_join(a, {part[0][i], part[1][i], part[2][i]});
  const float log_s = logf(a.s);
  if (threadIdx.x == 0) {
    p.lse[row] = a.s > 0.f ? a.m + log_s : -INFINITY;
    p.entropy[row] = a.s > 0.f ? log_s - a.t / a.s : 0.f;
  }
  for (int i = threadIdx.x; i < p.n_ids; i += kLpThreads) {
    const long long id = p.ids64 ? static_cast<const long long*>(p.ids)[row * p.n_ids + i] : static_cast<const int*>(p.ids)[row * p.n_ids + i];
    p.logprob[row * p.n_ids + i] =
        id < 0 || id >= p.V ? __int_as_float(0x7fc00000) : lp_log(lp_value(p, to_f(x[id]), static_cast<int>(id)), a.m, log_s);
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long top = 0;
    for (int j = threadIdx.x; j < p.V; j += kLpThreads) {
      const unsigned long long key = lp_key(lp_value(p, to_f(x[j]), j), j);
      if (key < last && key > top) top = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long b = __shfl_xor_sync(0xffffffffu, top, o);
      if (b > top) top = b;
    }
    __syncthreads();
    if (lane == 0) best[warp] = top;
    __syncthreads();
    last = best[0];
    for (int i = 1; i < kLpThreads / 32; ++i)
      if (best[i] > last) last = best[i];
    if (threadIdx.x == 0) {
      p.top_ids[row * p.top + k] = lp_key_index(last);
      p.top_logprobs[row * p.top + k] = lp_log(lp_key_value(last), a.m, log_s);
    }
  }
}

}  // namespace mx

extern "C" int mx_token_logprobs(const void* logits, int fp32, long long ld, const void* ids, int ids64, int n_ids, const void* bias,
                                 int bias_fp32, float scale, float softcap, float* logprob, float* entropy, float* lse, int* top_ids,
                                 float* top_logprobs, int top, int R, int V, void* stream_) {
  using namespace mx;
  if (R <= 0) return 0;
  if (V <= 0 || top < 0 || top > V || n_ids < 0 || scale <= 0.f || softcap < 0.f) return -1;
  const LpParams p{logits, ids, bias, logprob, entropy, lse, top_ids, top_logprobs, ld, V, n_ids, ids64, bias_fp32, top, scale, softcap};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const cudaError_t e = fp32 ? launch_kernel(token_logprobs_kernel<float>, dim3(R), dim3(kLpThreads), 0, stream, p)
                             : launch_kernel(token_logprobs_kernel<__nv_bfloat16>, dim3(R), dim3(kLpThreads), 0, stream, p);
  return static_cast<int>(e);
}
