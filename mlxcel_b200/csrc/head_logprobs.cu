// Log probabilities of given tokens and entropy straight from hidden rows and the head's weights, without logits in memory:
// z = x[M, K] @ w[V, K]^T (+ bias), scaled and soft-capped, for each row lse = log sum e^z, log p(id) = z_id - lse, H = lse - sum p z.
//
// The products run as in gemm_pair.cu: 256 x 256 tiles on pairs of SMs, operands by TMA, accumulators in TMEM, double-buffered. The
// epilogue leaves a tile as the sums of its columns per row (m, s, t of logprobs.cuh, one set per half of the tile) in place of 256
// logits, and the row's own token's logit where the tile holds it. A second launch joins the column tiles of each row.
// Logits of 2047 rows over 128256 tokens would be 1 GB of fp32; what is written instead is 25 MB (three numbers per row and half tile).
// The logits are never rounded.
//
// Bound by the tensor cores under the power cap: a tile's products take 8 K cycles an SM, its epilogue about 3000 beside them, whose
// instructions cost power and with it clock. Measured, in a row (us): 2047 rows, K 4096, V 128256 1870 (1.15 PFLOP/s); the same product
// by gemm_pair.cu, which writes 525 MB of bf16 logits, 1750, by cuBLAS 1550. With the sums left in the tensor core over all of K 1790,
// and 3e-6 from the 64-bit result in place of 7e-7; with the changes of SHAPED made in any case 120 more. A tile is 256 rows whatever is
// left of them, which is what few rows and remainders cost: 256 rows 235 (floor 194), 300 rows 414 (227), 8 to 192 rows of K 1024, V 50257
// 40 to 42 (16). 168 registers a thread, 40 bytes of them spilled (44 where SHAPED).
#include <cooperative_groups.h>

#include "api.h"
#include "common.cuh"
#include "logprobs.cuh"
#include "pair_mma.cuh"

namespace mx {

// The tensor core truncates its fp32 sums, which draws every logit towards 0: by 4e-6 of it over K = 4096. Its sums are therefore taken
// out every 1024 of K and added up, rounded, in the epilogue's registers (128 columns of a row per thread, hence eight warps).
constexpr int kHlSegment = 1024 / kGpBK;             // K slices of a sum
constexpr int kHlWarps = 8;                          // of the epilogue
constexpr int kHlCols = 128;                         // columns of a thread: half a tile
constexpr int kHlThreads = 64 + 32 * kHlWarps;

bool make_tensor_map_bf16(CUtensorMap* out, const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, uint32_t box_cols);

struct HeadParams {
  const void* ids;
  const void* bias;
  float* partials;          // [2 tiles_n][3][M], then the rows' own logits [M]
  float* logprob;
  float* entropy;
  float* lse;
  int* status;
  int M, V, K, ids64, bias_fp32, tiles_m, tiles_n, raster;
  float scale, softcap;
};

__device__ __forceinline__ long long head_id(const HeadParams& p, int m) {
  return p.ids64 ? static_cast<const long long*>(p.ids)[m] : static_cast<const int*>(p.ids)[m];
}

// SHAPED: the products are not the logits yet (a bias, a scale or a soft cap).
template <bool SHAPED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kHlThreads, 1)
head_logprobs_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const HeadParams p) {
  extern __shared__ uint8_t hl_smem[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(hl_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(ring + kGpStages * kGpStageBytes);   // leader: both CTAs' slices landed
  uint64_t* empty_bar = full_bar + kGpStages;         // the products that read the stage are done
  uint64_t* tmem_full = empty_bar + kGpStages;
  uint64_t* tmem_empty = tmem_full + 2;               // leader: both CTAs' epilogues have read the accumulator
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmem_empty + 2);

  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int pair = static_cast<int>(blockIdx.x) >> 1, pairs = static_cast<int>(gridDim.x) >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = p.tiles_m * p.tiles_n, num_kb = (p.K + kGpBK - 1) / kGpBK;

  // tile t -> first token row and first vocabulary row: panels of `raster` row tiles, row tile fastest, so that the tokens of a
  // panel stay in L2 while the weights pass once per panel
  auto place = [&](int t, int& m0, int& f0) {
    const int per_panel = p.raster * p.tiles_n, g = t / per_panel, r = t - g * per_panel;
    const int rows = min(p.raster, p.tiles_m - g * p.raster);
    m0 = (g * p.raster + r % rows) * 256;
    f0 = (r / rows) * 256;
  };

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    for (int s = 0; s < kGpStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 2 * kHlWarps);        // the epilogue warps of both CTAs
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_ptr)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  cluster.sync();                                     // the other CTA's barriers are there
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_ptr;
  pdl_trigger();
  pdl_wait();                                         // (weights too may be the previous kernel's)

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t keep = l2_policy_evict_last(), stream = l2_policy_evict_first();
      const uint32_t bars = gp_leader(full_bar);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs) {
        int m0, f0;
        place(t, m0, f0);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!gp_wait(&empty_bar[stage], phase ^ 1u, p.status, kErrProducerWait)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * kGpStageBytes);
          gp_tma_load(ring + stage * kGpStageBytes + kGpHalf, &map_w, bars + 8 * stage, kb * kGpBK, f0 + rank * 128, stream);
          gp_tma_load(ring + stage * kGpStageBytes, &map_x, bars + 8 * stage, kb * kGpBK, m0 + rank * 128, keep);
          if (++stage == kGpStages) stage = 0, phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = umma_idesc_bf16(256, false, false, 256);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs) {
        for (int kb0 = 0; ok && kb0 < num_kb; kb0 += kHlSegment) {
          if (!gp_wait(&tmem_empty[acc], acc_phase ^ 1u, p.status, kErrMmaWaitTmem)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          for (int kb = kb0; kb < min(num_kb, kb0 + kHlSegment); ++kb) {
            if (!gp_wait(&full_bar[stage], phase, p.status, kErrMmaWaitFull)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint32_t sa = smem_u32(ring + stage * kGpStageBytes), sb = sa + kGpHalf;
#pragma unroll
            for (int kk = 0; kk < kGpBK / 16; ++kk)
              gp_mma(tmem + acc * 256, umma_desc_k_sw128(sa + kk * 32), umma_desc_k_sw128(sb + kk * 32), idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
            gp_commit(&empty_bar[stage]);
            if (++stage == kGpStages) stage = 0, phase ^= 1u;
          }
          if (!ok) break;
          gp_commit(&tmem_full[acc]);
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, row = q * 32 + lane, col0 = (warp - 2) / 4 * kHlCols;
    const uint32_t done = gp_leader(tmem_empty);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool all = true;
    for (int t = pair; all && t < tiles; t += pairs) {
      int m0, f0;
      place(t, m0, f0);
      f0 += col0;
      const int m = m0 + rank * 128 + row, valid = p.V - f0;            // (below 1 where the vocabulary ends in the first half)
      const bool live = m < p.M;
      const long long own_col = live ? head_id(p, m) - f0 : -1;
      float z[kHlCols];
      for (int kb0 = 0; kb0 < num_kb; kb0 += kHlSegment) {
        const bool ok = gp_wait(&tmem_full[acc], acc_phase, p.status, kErrEpilogueWait);
        all = __all_sync(0xffffffffu, ok);
        if (!all) break;
        tc_fence_after_sync();
        const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * 256 + col0;
#pragma unroll
        for (int c = 0; c < kHlCols; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32(taddr + c, r);
          tmem_ld_wait();
          if (kb0 == 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) z[c + i] = __uint_as_float(r[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) z[c + i] += __uint_as_float(r[i]);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) gp_arrive(done + 8 * acc);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!all) break;
      if constexpr (SHAPED) {
#pragma unroll
        for (int i = 0; i < kHlCols; ++i) z[i] = lp_transform(z[i], min(f0 + i, p.V - 1), p.bias, p.bias_fp32, p.scale, p.softcap);
      }
      if (valid < kHlCols) {
#pragma unroll
        for (int i = 0; i < kHlCols; ++i)
          if (i >= valid) z[i] = -INFINITY;
      }
      if (own_col >= 0 && own_col < min(valid, kHlCols)) {
        float own = 0.f;
#pragma unroll
        for (int i = 0; i < kHlCols; ++i)
          if (own_col == i) own = z[i] != z[i] ? -INFINITY : z[i];
        p.partials[static_cast<size_t>(p.tiles_n) * 6 * p.M + m] = own;
      }
      LpSums a{-INFINITY, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kHlCols; ++i) a.m = fmaxf(a.m, z[i]);          // (NaN is dropped here and by the floor below: it counts as -inf)
      if (lp_plain(a.m)) {
        const float low = lp_floor(a.m);
        lp_pair s2 = lp_two(0.f, 0.f), t2 = s2;
#pragma unroll
        for (int i = 0; i < kHlCols; ++i) z[i] = fmaxf(z[i], low);
        lp_add(z, lp_two(-a.m, -a.m), s2, t2);
        const float2 s = lp_both(s2), t = lp_both(t2);
        a.s = s.x + s.y;
        a.t = t.x + t.y;
      } else if (a.m != -INFINITY) {
#pragma unroll
        for (int i = 0; i < kHlCols; ++i) a.s += z[i] == a.m ? 1.f : 0.f;
      }
      if (live) {
        float* out = p.partials + static_cast<size_t>(f0 / kHlCols) * 3 * p.M + m;
        out[0] = a.m;
        out[p.M] = a.s;
        out[2 * static_cast<size_t>(p.M)] = a.t;
      }
    }
  }

  tc_fence_before_sync();
  cluster.sync();                                     // nothing more arrives from or is read in the other CTA
  if (warp == 1) {
    tc_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Joins the halves of the column tiles of 32 rows (a lane each), a warp every 32nd tile, in a fixed order.
__global__ void __launch_bounds__(1024) head_join_kernel(const HeadParams p) {
  __shared__ float part[3][32][33];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, m = blockIdx.x * 32 + lane;
  LpSums a{-INFINITY, 0.f, 0.f};
  if (m < p.M) {
#pragma unroll 4
    for (int t = warp; t < 2 * p.tiles_n; t += 32) {
      const float* src = p.partials + static_cast<size_t>(t) * 3 * p.M + m;
      a = lp_join(a, {src[0], src[p.M], src[2 * static_cast<size_t>(p.M)]});
    }
  }
  part[0][warp][lane] = a.m, part[1][warp][lane] = a.s, part[2][warp][lane] = a.t;
  __syncthreads();
  if (warp != 0 || m >= p.M) return;
  for (int i = 1; i < 32; ++i) a = lp_join(a, {part[0][i][lane], part[1][i][lane], part[2][i][lane]});
  const long long id = head_id(p, m);
  p.lse[m] = lp_lse(a);
  p.entropy[m] = lp_entropy(a);
  p.logprob[m] = id < 0 || id >= p.V ? __int_as_float(0x7fc00000) : lp_log(p.partials[static_cast<size_t>(p.tiles_n) * 6 * p.M + m], a);
}

}  // namespace mx

extern "C" int mx_head_logprobs(const void* x, const void* w, const void* ids, int ids64, const void* bias, int bias_fp32, float scale,
                                float softcap, float* partials, float* logprob, float* entropy, float* lse, int M, int V, int K, int ldx,
                                int ldw, void* status, void* stream_) {
  using namespace mx;
  if (M <= 0) return 0;
  if (V <= 0 || K <= 0 || scale <= 0.f || softcap < 0.f || status == nullptr || partials == nullptr) return -1;
  if (K % 8 || ldx % 8 || ldw % 8 || (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) % 16) return -10;
  HeadParams p{ids, bias, partials, logprob, entropy, lse, static_cast<int*>(status), M, V, K, ids64, bias_fp32, (M + 255) / 256, (V + 255) / 256, 8,
               scale, softcap};
  CUtensorMap map_x, map_w;
  if (!make_tensor_map_bf16(&map_x, x, M, K, ldx, 128, kGpBK) || !make_tensor_map_bf16(&map_w, w, V, K, ldw, 128, kGpBK)) return -4;
  const bool shaped = bias != nullptr || scale != 1.f || softcap > 0.f;
  auto kern = shaped ? head_logprobs_kernel<true> : head_logprobs_kernel<false>;
  static bool allowed[2][64] = {};
  cudaError_t e = allow_shared(kern, kGpSmem, allowed[shaped]);
  if (e != cudaSuccess) return static_cast<int>(e);
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n, most = device_sm_count() / 2;
  if (tiles > 0x7fffffffll) return -1;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  e = launch_kernel(kern, dim3(2 * static_cast<unsigned>(tiles < most ? tiles : most)), dim3(kHlThreads), kGpSmem, stream, map_x, map_w, p);
  if (e != cudaSuccess) return static_cast<int>(e);
  return static_cast<int>(launch_kernel(head_join_kernel, dim3((M + 31) / 32), dim3(1024), 0, stream, p));
}
