// Log probabilities of given tokens, entropy and the most likely tokens of every row of logits:
//
//   z = x (+ bias), times scale, soft-capped;  lse = log sum_j e^(z_j);  log p(id) = z_id - lse;  H = lse - sum_j p_j z_j
//
// NaN counts as -inf. A row with nothing left (all -inf) has lse = -inf, log probabilities -inf and entropy 0. Equal logits order by
// index. An id outside the vocabulary has log probability NaN.
//
// A row is read by a cluster of 1 to 8 CTAs whose parts are joined through distributed shared memory, as 16-byte vectors that each
// thread asks for two chunks ahead. Sums are per thread, rescaled at most once a chunk.
//
// The `top` best cost the pass over the row a maximum per thread and the chunk it came from. Behind it, each of 128 groups of threads
// has an element at least as large as its maximum, so all of the `top` best are at or above the (top)th of these maxima, and only
// groups whose own maximum is can hold one. Their vectors are read again (top 5 of 128 groups: 4 % of the row, top 20: 16 %), what
// reaches the bound goes to a list, and the list is ordered by counting, for each entry, the entries above it. Every key is unique
// (value, then index), so neither ties nor the order of arrival change a result. Should the list overflow (many of the largest logits a
// whole number of rows of vectors apart), each of the `top` best is searched for. Looking for candidates on the way instead (against a
// bound from the first chunk) cost more: every candidate sends its warp on a detour.
//
// Memory (19.9 us for 509 x 128256 bf16 logits), the exponentials (16 a cycle and SM: 14.5 us) and the other 5 instructions per element, for
// which additions and products are done in pairs, come close to one another; no unit is at its limit (top 5: exponentials 41 %, issue 61 %,
// memory 38 % busy), and 509 CTAs are four on some SMs and three on others. The way from the last logit to the result (joining, the search
// among groups) leaves a CTA without loads on their way: top 5 of 2000 x 32000, whose rows have no common end, takes 55 us in place of 32.
// Measured, back to back
// (us): 509 x 128256 bf16 31 without alternatives (24.6 without the exponentials), 45 with top 5, 53 with top 20; 512 x 151936 fp32 55
// (floor 47), 80, 107; one row of 151936 fp32 5.5, 10.2, 12.9.
#include <cooperative_groups.h>

#include <type_traits>

#include "api.h"
#include "common.cuh"
#include "logprobs.cuh"
#include "typed.cuh"

namespace mx {

constexpr int kLpVecs = 4;               // 16-byte vectors of a thread and chunk
constexpr int kLpStages = 2;             // chunks of a thread in flight
constexpr int kLpTop = 64;
constexpr int kLpGroups = 128;           // of neighbouring threads
constexpr int kLpList = 1088;            // at least kLpTop per CTA of a cluster, and the first vectors of kLpTop groups with the row's ends
constexpr int kLpCluster = 8;
using lp_key_t = unsigned long long;

// The sums of a warp's lanes, the same bits in all of them: each is rescaled once, to the largest logit of all.
__device__ __forceinline__ LpSums lp_warp_join(const LpSums& lane) {
  float m = lane.s > 0.f ? lane.m : -INFINITY;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  LpSums a = lane.s > 0.f ? lp_rescale(lane, m) : LpSums{m, 0.f, 0.f};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
  return a;
}

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

// Orders by value, then by lower index; NaN is -inf; 0 is below every key.
__device__ __forceinline__ lp_key_t lp_key(float z, int j) {
  uint32_t u = __float_as_uint((z != z ? -INFINITY : z) + 0.f);       // (-0 equals 0)
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (static_cast<lp_key_t>(u) << 32) | (0xffffffffu - static_cast<uint32_t>(j));
}
__device__ __forceinline__ int lp_key_index(lp_key_t k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float lp_key_value(lp_key_t k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

template <typename T>
__device__ __forceinline__ void lp_unpack(const uint4& u, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
    else f[i] = __uint_as_float(w[i]);
  }
}
__device__ __forceinline__ uint32_t lp_max2(uint32_t a, uint32_t b) {   // of two bf16 each; passes over NaN
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

struct LpNoLists {};
struct LpLists {
  lp_key_t list[kLpList];
  lp_key_t group[kLpGroups];
  lp_key_t best[kLpTop];
  lp_key_t bound;
  int chosen[kLpTop];                      // groups that reach the bound
  int n, groups;                           // entries that wanted into the list; chosen ones
};
// Calls take(i, how many of a[n] are above a[i]) for every entry but those that are 0, once. Up to 32 neighbouring threads count for
// one entry. n <= kLpList; all threads of the CTA call it.
template <int THREADS, typename F>
__device__ __forceinline__ void lp_ranks(const lp_key_t* a, int n, F&& take) {
  int share = 32;
  while (share > 1 && share * n > THREADS) share >>= 1;
  for (int i0 = 0; i0 < n; i0 += THREADS / share) {
    const int i = i0 + threadIdx.x / share;
    const lp_key_t key = i < n ? a[i] : ~0ull;
    int r = 0;
#pragma unroll 4
    for (int j = threadIdx.x % share; j < n; j += share) r += a[j] > key ? 1 : 0;
    for (int o = share >> 1; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    if (i < n && key != 0 && threadIdx.x % share == 0) take(i, r);
  }
}
__device__ __forceinline__ void lp_offer(LpLists& sh, lp_key_t key, lp_key_t bound) {
  if (key >= bound) {
    const int at = atomicAdd(&sh.n, 1);
    if (at < kLpList) sh.list[at] = key;
  }
}
// The `top` best of list[n], which is complete, in order to best[] (0 where there are fewer). Ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void lp_select(LpLists& sh, int n, int top) {
  for (int i = threadIdx.x; i < top; i += THREADS)
    if (i >= n) sh.best[i] = 0;
  lp_ranks<THREADS>(sh.list, n, [&](int i, int r) {
    if (r < top) sh.best[r] = sh.list[i];
  });
  __syncthreads();
}
template <typename T, bool TOP, bool SHAPED, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const LpParams p) {
  constexpr int E = 16 / sizeof(T), kWarps = THREADS / 32, kStep = kLpVecs * THREADS;
  constexpr bool kWhole = sizeof(T) == 2 && !SHAPED;                       // bf16 that needs no change: maxima without unpacking
  extern __shared__ __align__(16) unsigned char lp_smem[];
  uint4* ring = reinterpret_cast<uint4*>(lp_smem) + threadIdx.x;           // [stage][vector][thread]: a thread's own vectors on their way
  __shared__ std::conditional_t<TOP, LpLists, LpNoLists> sh;
  __shared__ float warp_m[kWarps], warp_s[kWarps], warp_t[kWarps];
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  pdl_trigger();
  pdl_wait();
  const long long row = blockIdx.x / parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = static_cast<int>(threadIdx.x), top = p.top;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  // `head` elements, then aligned vectors, then fewer than E elements
  const int past = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)), head = min(past ? E - past : 0, p.V);
  const int vecs = (p.V - head) / E, per = (vecs + parts - 1) / parts, first = min(part * per, vecs), end = min(first + per, vecs);
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);

  // A thread reads only what it asked for itself, so its own wait is all that is needed.
  auto ask = [&](int v0, int stage) {
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) {
      const int v = v0 + i * THREADS + tid;
      if (v < end)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(ring + (stage * kLpVecs + i) * THREADS)), "l"(xv + v) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kLpStages; ++i) ask(first + i * kStep, i);

  LpSums a{-INFINITY, 0.f, 0.f};
  lp_key_t loose = 0;                                                     // of the row's ends
  float peak = -INFINITY;                                                 // the thread's largest logit, and its chunk
  int peak_at = first;
  if (part == 0 && warp == 0) {                                           // the row's ends
    const int tail = p.V - head - vecs * E, j = lane < head ? lane : vecs * E + lane;
    if (lane < head + tail) {
      const float z = lp_value(p, to_f(x[j]), j);
      if (z != -INFINITY) a = {z, 1.f, 0.f};
      loose = lp_key(z, j);
    }
  }
  int stage = 0;
  for (int v0 = first; v0 < end; v0 += kStep) {
    uint4 now[kLpVecs];
    asm volatile("cp.async.wait_group %0;" ::"n"(kLpStages - 1) : "memory");
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i) now[i] = ring[(stage * kLpVecs + i) * THREADS];
    const bool full = v0 + kStep <= end;
    auto here = [&](int i) { return full || v0 + i * THREADS + tid < end; };
    auto index = [&](int i, int j) { return head + (v0 + i * THREADS + tid) * E + j; };
    auto values = [&](int i, float (&f)[E]) {
      lp_unpack<T>(now[i], f);
      if constexpr (SHAPED) {
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] = lp_value(p, f[j], index(i, j));
      }
    };
    auto largest = [&](int i) {                                           // of vector i; passes over NaN
      if constexpr (kWhole) {
        const uint32_t w = lp_max2(lp_max2(now[i].x, now[i].y), lp_max2(now[i].z, now[i].w));
        return fmaxf(fmaxf(bf16_lo(w), -INFINITY), bf16_hi(w));
      } else {
        float f[E], m = -INFINITY;
        values(i, f);
#pragma unroll
        for (int j = 0; j < E; ++j) m = fmaxf(m, f[j]);
        return m;
      }
    };
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLpVecs; ++i)
      if (here(i)) most = fmaxf(most, largest(i));
    // (every vector has been looked at: its place is free)
    ask(v0 + kLpStages * kStep, stage);
    stage = stage + 1 == kLpStages ? 0 : stage + 1;
    if (most > a.m) a = lp_rescale(a, most);
    if (lp_plain(a.m)) {
      const float low = lp_floor(a.m);
      const uint32_t low2 = pack_bf16(low, low);
      const lp_pair minus_m = lp_two(-a.m, -a.m);
      lp_pair s2 = lp_two(a.s, 0.f), t2 = lp_two(a.t, 0.f);
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) {
        if (here(i)) {
          float f[E];
          if constexpr (kWhole) {
            lp_unpack<T>(make_uint4(lp_max2(now[i].x, low2), lp_max2(now[i].y, low2), lp_max2(now[i].z, low2), lp_max2(now[i].w, low2)), f);
          } else {
            values(i, f);
#pragma unroll
            for (int j = 0; j < E; ++j) f[j] = fmaxf(f[j], low);
          }
          lp_add(f, minus_m, s2, t2);
        }
      }
      const float2 s = lp_both(s2), t = lp_both(t2);
      a.s = s.x + s.y;
      a.t = t.x + t.y;
    } else if (a.m != -INFINITY) {
#pragma unroll
      for (int i = 0; i < kLpVecs; ++i) {
        if (here(i)) {
          float f[E];
          values(i, f);
#pragma unroll
          for (int j = 0; j < E; ++j) a.s += f[j] == a.m ? 1.f : 0.f;
        }
      }
    }
    if (TOP && most > peak) peak = most, peak_at = v0;
  }
  a = lp_warp_join(a);
  if (lane == 0) warp_m[warp] = a.m, warp_s[warp] = a.s, warp_t[warp] = a.t;
  if constexpr (TOP) {
    auto key_at = [&](const uint4& u, int v, int j) {                   // of element j of vector v
      float f[E];
      lp_unpack<T>(u, f);
      const int k = head + v * E + j;
      return lp_key(SHAPED ? lp_value(p, f[j], k) : f[j], k);
    };
    // the thread's largest key: in the first chunk with its largest value
    constexpr int kGroup = THREADS / kLpGroups;
    lp_key_t own = 0;
    for (int i = 0; i < kLpVecs; ++i) {
      const int v = peak_at + i * THREADS + tid;
      if (v < end) {
        const uint4 u = __ldg(xv + v);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const lp_key_t k = key_at(u, v, j);
          own = k > own ? k : own;
        }
      }
    }
#pragma unroll
    for (int o = 1; o < kGroup; o <<= 1) {
      const lp_key_t other = __shfl_xor_sync(0xffffffffu, own, o);
      own = other > own ? other : own;
    }
    if (tid % kGroup == 0) sh.group[tid / kGroup] = own;
    if (tid == 0) {
      sh.bound = 0;
      sh.n = 0;
      sh.groups = 0;
    }
    __syncthreads();
    lp_ranks<THREADS>(sh.group, kLpGroups, [&](int i, int r) {            // (keys are unique: so are the ranks)
      if (r < top) {
        sh.chosen[r] = i;
        atomicMax(&sh.groups, r + 1);
        if (r == top - 1) sh.bound = sh.group[i];
      }
    });
    __syncthreads();
    const lp_key_t bound = sh.bound;
    const float edge = bound ? lp_key_value(bound) : -INFINITY;
    if (loose) lp_offer(sh, loose, bound);
    const int rows = (end - first + THREADS - 1) / THREADS, again = kGroup * sh.groups * rows;
    for (int q = tid; q < again; q += THREADS) {
      const int g = q / kGroup / rows, v = first + (q / kGroup - g * rows) * THREADS + sh.chosen[g] * kGroup + q % kGroup;
      if (v < end) {
        const uint4 u = __ldg(xv + v);
        float f[E];
        lp_unpack<T>(u, f);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (SHAPED || !(f[j] < edge)) lp_offer(sh, key_at(u, v, j), bound);       // (NaN passes and is -inf there)
      }
    }
    __syncthreads();
    if (sh.n <= kLpList) {
      lp_select<THREADS>(sh, sh.n, top);
    } else {
      lp_key_t last = ~0ull;
      for (int k = 0; k < top; ++k) {
        own = loose < last ? loose : 0;
        for (int v = first + tid; v < end; v += THREADS) {
          const uint4 u = __ldg(xv + v);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const lp_key_t c = key_at(u, v, j);
            if (c < last && c > own) own = c;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const lp_key_t c = __shfl_xor_sync(0xffffffffu, own, o);
          if (c > own) own = c;
        }
        if (lane == 0) sh.group[warp] = own;
        __syncthreads();
        last = sh.group[0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) last = sh.group[i] > last ? sh.group[i] : last;
        if (tid == 0) sh.best[k] = last;
        __syncthreads();
      }
    }
  } else {
    __syncthreads();
  }
  // every warp of part 0 joins the sums of all parts' warps (at most 64)
  if (parts > 1) cluster.sync();
  if (part == 0) {
    a = {-INFINITY, 0.f, 0.f};
    for (int i = lane; i < parts * kWarps; i += 32) {
      const int from = i / kWarps, w = i % kWarps;
      a = lp_join(a, {cluster.map_shared_rank(warp_m, from)[w], cluster.map_shared_rank(warp_s, from)[w], cluster.map_shared_rank(warp_t, from)[w]});
    }
    a = lp_warp_join(a);
    if constexpr (TOP) {
      if (parts > 1)
        for (int i = tid; i < parts * top; i += THREADS) sh.list[i] = cluster.map_shared_rank(sh.best, i / top)[i % top];
    }
  }
  if (parts > 1) {
    cluster.sync();                                                       // the other parts' memory has been read
    if (part != 0) return;
    if constexpr (TOP) lp_select<THREADS>(sh, parts * top, top);
  }
  if (tid == 0) {
    p.lse[row] = lp_lse(a);
    p.entropy[row] = lp_entropy(a);
  }
  for (int i = tid; i < p.n_ids; i += THREADS) {
    const long long id = p.ids64 ? static_cast<const long long*>(p.ids)[row * p.n_ids + i] : static_cast<const int*>(p.ids)[row * p.n_ids + i];
    p.logprob[row * p.n_ids + i] = id < 0 || id >= p.V ? __int_as_float(0x7fc00000) : lp_log(lp_value(p, to_f(x[id]), static_cast<int>(id)), a);
  }
  if constexpr (TOP) {
    for (int i = tid; i < top; i += THREADS) {
      p.top_ids[row * top + i] = lp_key_index(sh.best[i]);
      p.top_logprobs[row * top + i] = lp_log(lp_key_value(sh.best[i]), a);
    }
  }
}

// A row is cut while all CTAs still find an SM of their own, into parts of at least a chunk: with more CTAs the tails of the parts cost
// more than the cut gives (74 rows of 128256 fp32, top 5: 16.5 us in 2 parts, 21.2 in 4; one row: 10.2 us in 8 parts, 22.9 in one). In
// between it is not the best cut, as four CTAs fit on an SM and one alone does not fill it (us without alternatives / top 5 / top 20,
// 128256 bf16): 200 rows 22.2 / 29.6 / 32.8 in one part, which the rule takes, 18.3 / 27.6 / 30.2 in two; 32 rows 9.5 / 16.8 / 18.4 in four,
// which it takes, 8.7 / 14.6 / 16.5 in two.
template <typename T, bool TOP>
static cudaError_t launch_token_logprobs(const LpParams& p, int rows, cudaStream_t stream) {
  constexpr int THREADS = 256, chunk = THREADS * kLpVecs * 16 / sizeof(T);
  int parts = 1;
  while (parts < kLpCluster && 2ll * parts * rows <= device_sm_count() && p.V > static_cast<long long>(parts) * chunk) parts *= 2;
  const bool shaped = p.bias != nullptr || p.scale != 1.f || p.softcap > 0.f;
  auto kern = shaped ? token_logprobs_kernel<T, TOP, true, THREADS> : token_logprobs_kernel<T, TOP, false, THREADS>;
  constexpr int bytes = kLpStages * kLpVecs * THREADS * 16;
  static bool allowed[2][64] = {};
  const cudaError_t e = allow_shared(kern, bytes, allowed[shaped]);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * parts);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
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

extern "C" int mx_token_logprobs(const MxTokenLogprobs* a, void* stream_) {
  using namespace mx;
  if (a->R <= 0) return 0;
  if (a->V <= 0 || a->V > (1 << 30) || a->R > (1 << 27) || a->top < 0 || a->top > a->V || a->top > kLpTop || a->n_ids < 0 || !(a->scale > 0.f) ||
      !(a->softcap >= 0.f))
    return -1;
  const LpParams p{a->logits, a->ids, a->bias, a->logprob, a->entropy, a->lse, a->top_ids, a->top_logprobs, a->ld, a->V, a->n_ids, a->ids64, a->bias_fp32,
                   a->top, a->scale, a->softcap};
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  cudaError_t e;
  if (a->fp32) e = a->top ? launch_token_logprobs<float, true>(p, a->R, stream) : launch_token_logprobs<float, false>(p, a->R, stream);
  else e = a->top ? launch_token_logprobs<__nv_bfloat16, true>(p, a->R, stream) : launch_token_logprobs<__nv_bfloat16, false>(p, a->R, stream);
  return static_cast<int>(e);
}
