// Log probabilities of given tokens, entropy and the most likely tokens of every row of logits:
//
//   z = x (+ bias), times scale, soft-capped;  lse = log sum_j e^(z_j);  log p(id) = z_id - lse;  H = lse - sum_j p_j z_j
//
// NaN counts as -inf. A row with nothing left (all -inf) has lse = -inf, log probabilities -inf and entropy 0. Equal logits order by
// index. An id outside the vocabulary has log probability NaN.
//
// A row is read once, by a cluster of 1 to 8 CTAs (its parts are joined through distributed shared memory), as 16-byte vectors with
// the next chunk in flight. Sums are per thread, rescaled at most once a chunk. The `top` best are found on the way: candidates
// above a threshold go to a list in shared memory. The threshold is below the `top` best of what has been read: at first the best
// but (top - 1) of 64 group maxima of a chunk (each group has an element at least that large), later the last of the list whenever
// that is cut down to `top`. Lists are ordered by counting, for each entry, the entries above it. Every key is unique (value, then
// index), so neither ties nor the order of arrival change a result.
#include <cooperative_groups.h>
#include <string.h>

#include <type_traits>

#include "api.h"
#include "common.cuh"
#include "logprobs.cuh"
#include "typed.cuh"

namespace mx {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 4;               // 16-byte vectors of a thread and chunk
constexpr int kLpTop = 64;
constexpr int kLpGroups = 64;            // of 4 neighbouring threads
constexpr int kLpList = 2048;
constexpr int kLpSlack = 32;             // entries of the list beyond twice those asked for before it is cut
constexpr int kLpCluster = 8;
using lp_key_t = unsigned long long;
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
__device__ __forceinline__ lp_key_t lp_key(float z, int j) {
  uint32_t u = __float_as_uint(z + 0.f);                              // (-0 equals 0)
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<lp_key_t>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(j));
}
__device__ __forceinline__ int lp_key_index(lp_key_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float lp_key_value(lp_key_t k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// A row's part: vectors [first, end) of 16 bytes, the first of them beginning `lead` elements before the row.
template <typename T>
struct LpPart {
  static constexpr int E = 16 / sizeof(T);
  const T* row;
  int V, lead, first, end;
  __device__ __forceinline__ int index(int v, int j) const { return v * E - lead + j; }
  __device__ __forceinline__ uint4 load(int v) const {
    const int j0 = index(v, 0);
    if (j0 >= 0 && j0 + E <= V) return __ldg(reinterpret_cast<const uint4*>(row + j0));
    T e[E];                                                            // the row's ends: what lies beyond is not read
#pragma unroll
    for (int j = 0; j < E; ++j) e[j] = j0 + j >= 0 && j0 + j < V ? row[j0 + j] : from_f<T>(-INFINITY);
    uint4 u;
    memcpy(&u, e, 16);
    return u;
  }
};
template <typename T>
__device__ __forceinline__ void lp_unpack(const uint4& u, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
    else f[i] = __uint_as_float(w[i]);
  }
}

struct LpNoLists {};
struct LpLists {
  lp_key_t list[kLpList];
  lp_key_t best[kLpTop];                   // this part's, in order (what the cluster reads)
  lp_key_t group[kLpGroups];
  lp_key_t threshold;
  int count[kLpWarps];
};

// Entries of a[n] above `key`.
__device__ __forceinline__ int lp_rank(const lp_key_t* a, int n, lp_key_t key) {
  int r = 0;
#pragma unroll 8
  for (int i = 0; i < n; ++i) r += a[i] > key ? 1 : 0;
  return r;
}
// The `top` best of list[n] in order to best[] (0 where there are fewer). Ends with a barrier.
__device__ __forceinline__ void lp_select(LpLists& sh, int n, int top) {
  for (int i = threadIdx.x; i < top; i += kLpThreads)
    if (i >= n) sh.best[i] = 0;
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const lp_key_t key = sh.list[i];
    const int r = lp_rank(sh.list, n, key);
    if (r < top) sh.best[r] = key;
  }
  __syncthreads();
}
// Places for `mine` entries of every thread behind each other: this thread's first, and the total. One barrier.
__device__ __forceinline__ int lp_places(LpLists& sh, int mine, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.count[warp] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kLpWarps; ++i) {
    if (i < warp) before += sh.count[i];
    total += sh.count[i];
  }
  return before + incl - mine;
}

template <typename T, bool TOP, bool SHAPED>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LpParams p) {
  constexpr int E = 16 / sizeof(T);
  __shared__ std::conditional_t<TOP, LpLists, LpNoLists> sh;
  __shared__ LpSums part_sums, warp_sums[kLpWarps];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  pdl_trigger();
  pdl_wait();
  const long long row = blockIdx.x / parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, top = p.top;
  LpPart<T> x;
  x.row = static_cast<const T*>(p.logits) + row * p.ld;
  x.V = p.V;
  x.lead = static_cast<int>(reinterpret_cast<uintptr_t>(x.row) % 16 / sizeof(T));
  const int vecs = (p.V + x.lead + E - 1) / E, per = (vecs + parts - 1) / parts;
  x.first = min(part * per, vecs);
  x.end = min(x.first + per, vecs);

  LpSums a{-INFINITY, 0.f, 0.f};
  lp_key_t threshold = 0;
  int listed = 0;
  uint4 now[kLpVecs], next[kLpVecs];
  auto fetch = [&](int v0, uint4 (&u)[kLpVecs]) {
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      const int v = v0 + i * kLpThreads + threadIdx.x;
      if (v < x.end) u[i] = x.load(v);
    }
  };
  auto values = [&](const uint4& u, int v, float (&f)[E]) {
    lp_unpack<T>(u, f);
    if constexpr (SHAPED) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int k = x.index(v, j);
        f[j] = k >= 0 && k < x.V ? lp_value(p, f[j], k) : -INFINITY;
      }
    }
  };
  fetch(x.first, now);
  for (int v0 = x.first; v0 < x.end; v0 += kLpVecs * kLpThreads) {
    fetch(v0 + kLpVecs * kLpThreads, next);
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      const int v = v0 + i * kLpThreads + threadIdx.x;
      if (v < x.end) {
        float f[E];
        values(now[i], v, f);
#pragma unroll
        for (int j = 0; j < E; ++j) most = fmaxf(most, f[j]);           // (passes over NaN)
      }
    }
    if (most > a.m) a = lp_rescale(a, most);
    // e^d is 0 from d = -104 on: -256 stands for all that is lower, for masked values and (fmaxf drops it) for NaN
    auto add = [&](auto&& gap) {
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) {
        const int v = v0 + i * kLpThreads + threadIdx.x;
        if (v < x.end) {
          float f[E];
          values(now[i], v, f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const float d = gap(f[j]), e = lp_exp2(d * kLog2e);
            a.s += e;
            a.t += e * d;
          }
        }
      }
    };
    if (a.m == INFINITY) add([](float z) { return z == INFINITY ? 0.f : -256.f; });
    else if (a.m != -INFINITY) add([&](float z) { return fmaxf(z - a.m, -256.f); });
    if constexpr (TOP) {
      // what the threshold's value lets pass is looked at again as keys; NaN passes too and becomes -inf there
      const float edge = threshold == 0 ? -INFINITY : lp_key_value(threshold);
      const bool some = v0 + static_cast<int>(threadIdx.x) < x.end && most >= edge;
      // the thread's elements above the threshold, in order of their index
      auto each = [&](auto&& take) {
        if (!some) return;
#pragma unroll
        for (int i = 0; i < kLpVecs; ++i) {
          const int v = v0 + i * kLpThreads + threadIdx.x;
          if (v < x.end) {
            float f[E];
            values(now[i], v, f);
#pragma unroll
            for (int j = 0; j < E; ++j) {
              if (!(f[j] < edge)) {
                const int k = x.index(v, j);
                const lp_key_t key = lp_key(f[j] != f[j] ? -INFINITY : f[j], k);
                if (k >= 0 && k < x.V && key > threshold) take(key);
              }
            }
          }
        }
      };
      // the list's best stay, and the last of them is the threshold
      auto cut = [&] {
        lp_select(sh, listed, top);
        listed = top;
        if (sh.best[top - 1] > threshold) threshold = sh.best[top - 1];
        for (int i = threadIdx.x; i < top; i += kLpThreads) sh.list[i] = sh.best[i];
      };
      const int threads = __syncthreads_count(some);
      if (threads > kLpGroups) {                                          // many: raise the threshold by this chunk's group maxima
        lp_key_t mine = 0;
        each([&](lp_key_t key) { mine = key > mine ? key : mine; });
#pragma unroll
        for (int o = 1; o < kLpThreads / kLpGroups; o <<= 1) {
          const lp_key_t other = __shfl_xor_sync(0xffffffffu, mine, o);
          mine = other > mine ? other : mine;
        }
        if (threadIdx.x % (kLpThreads / kLpGroups) == 0) sh.group[threadIdx.x / (kLpThreads / kLpGroups)] = mine;
        if (threadIdx.x == 0) sh.threshold = threshold;
        __syncthreads();
        if (threadIdx.x < kLpGroups) {
          const lp_key_t key = sh.group[threadIdx.x];
          // one below the key itself, which has to pass
          if (key > threshold && lp_rank(sh.group, kLpGroups, key) == top - 1) sh.threshold = key - 1;
        }
        __syncthreads();
        threshold = sh.threshold;
      }
      if (threads > 0) {
        int mine = 0, total;
        each([&](lp_key_t) { ++mine; });
        int at = lp_places(sh, mine, total);
        if (listed + total > kLpList && listed > top) {                   // make room: the list's best stay
          __syncthreads();
          cut();
          mine = 0;
          each([&](lp_key_t) { ++mine; });
          __syncthreads();
          at = lp_places(sh, mine, total);
        }
        if (listed + total <= kLpList) {
          at += listed;
          each([&](lp_key_t key) { sh.list[at++] = key; });
          listed += total;
          if (listed > 2 * top + kLpSlack) {                              // a current threshold lets 1 / n of the list pass in the nth chunk
            __syncthreads();
            cut();
          }
        } else {
          // still too many (large values side by side): one place of every thread's elements at a time
          for (int step = 0; step < kLpVecs * E; ++step) {
            lp_key_t held = 0;
#pragma unroll
            for (int i = 0; i < kLpVecs; ++i) {
              const int v = v0 + i * kLpThreads + threadIdx.x;
              if (v < x.end) {
                float f[E];
                values(now[i], v, f);
#pragma unroll
                for (int j = 0; j < E; ++j) {
                  const int k = x.index(v, j);
                  if (i * E + j == step && k >= 0 && k < x.V) held = lp_key(f[j] != f[j] ? -INFINITY : f[j], k);
                }
              }
            }
            if (listed + kLpThreads > kLpList) {
              __syncthreads();
              cut();
            }
            const bool take = held > threshold;
            __syncthreads();
            at = lp_places(sh, take ? 1 : 0, total);
            if (take) sh.list[listed + at] = held;
            listed += total;
            __syncthreads();
          }
        }
        __syncthreads();
      }
    }
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) now[i] = next[i];
  }
  a = lp_warp_join(a);
  if (lane == 0) warp_sums[warp] = a;
  __syncthreads();
  a = warp_sums[0];
#pragma unroll
  for (int i = 1; i < kLpWarps; ++i) a = lp_join(a, warp_sums[i]);
  if constexpr (TOP) lp_select(sh, listed, top);
  if (parts > 1) {
    if (threadIdx.x == 0) part_sums = a;
    cluster.sync();
    if (part == 0) {
      for (int i = 1; i < parts; ++i) a = lp_join(a, *cluster.map_shared_rank(&part_sums, i));
      if constexpr (TOP) {
        for (int i = threadIdx.x; i < parts * top; i += kLpThreads) sh.list[i] = cluster.map_shared_rank(sh.best, i / top)[i % top];
      }
    }
    cluster.sync();                                                       // the other parts' memory has been read
    if (part != 0) return;
    if constexpr (TOP) lp_select(sh, parts * top, top);
  }
  const float log_s = logf(a.s);
  if (threadIdx.x == 0) {
    p.lse[row] = a.s > 0.f ? a.m + log_s : -INFINITY;
    p.entropy[row] = a.s > 0.f ? log_s - a.t / a.s : 0.f;
  }
  for (int i = threadIdx.x; i < p.n_ids; i += kLpThreads) {
    const long long id = p.ids64 ? static_cast<const long long*>(p.ids)[row * p.n_ids + i] : static_cast<const int*>(p.ids)[row * p.n_ids + i];
    p.logprob[row * p.n_ids + i] =
        id < 0 || id >= p.V ? __int_as_float(0x7fc00000) : lp_log(lp_value(p, to_f(x.row[id]), static_cast<int>(id)), a.m, log_s);
  }
  if constexpr (TOP) {
    for (int i = threadIdx.x; i < top; i += kLpThreads) {
      p.top_ids[row * top + i] = lp_key_index(sh.best[i]);
      p.top_logprobs[row * top + i] = lp_log(lp_key_value(sh.best[i]), a.m, log_s);
    }
  }
}

template <typename T, bool TOP>
static cudaError_t launch_token_logprobs(const LpParams& p, int rows, cudaStream_t stream) {
  const bool shaped = p.bias != nullptr || p.scale != 1.f || p.softcap > 0.f;
  auto kern = shaped ? token_logprobs_kernel<T, TOP, true> : token_logprobs_kernel<T, TOP, false>;
  // Four CTAs are resident on an SM: rows are cut until they fill the SMs, into parts of at least one chunk.
  const long long slots = 4ll * device_sm_count(), chunk = static_cast<long long>(kLpVecs) * kLpThreads * 16 / sizeof(T);
  int parts = 1;
  while (parts < kLpCluster && 2ll * parts * rows <= slots && p.V > parts * chunk) parts *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * parts);
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace mx

extern "C" int mx_token_logprobs(const void* logits, int fp32, long long ld, const void* ids, int ids64, int n_ids, const void* bias,
                                 int bias_fp32, float scale, float softcap, float* logprob, float* entropy, float* lse, int* top_ids,
                                 float* top_logprobs, int top, int R, int V, void* stream_) {
  using namespace mx;
  if (R <= 0) return 0;
  if (V <= 0 || V > (1 << 30) || R > (1 << 27) || top < 0 || top > V || top > kLpTop || n_ids < 0 || scale <= 0.f || softcap < 0.f) return -1;
  const LpParams p{logits, ids, bias, logprob, entropy, lse, top_ids, top_logprobs, ld, V, n_ids, ids64, bias_fp32, top, scale, softcap};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  cudaError_t e;
  if (fp32) e = top ? launch_token_logprobs<float, true>(p, R, stream) : launch_token_logprobs<float, false>(p, R, stream);
  else e = top ? launch_token_logprobs<__nv_bfloat16, true>(p, R, stream) : launch_token_logprobs<__nv_bfloat16, false>(p, R, stream);
  return static_cast<int>(e);
}
