// Building blocks of the kernels that run 256 x 256 tiles on pairs of SMs (tcgen05 cta_group::2): gemm_pair.cu, head_logprobs.cu.
#pragma once
#include "common.cuh"

namespace mx {

constexpr int kGpBK = 64;
constexpr int kGpStages = 6;
constexpr int kGpHalf = 128 * kGpBK * 2;            // bytes of one operand slice of one CTA
constexpr int kGpStageBytes = 2 * kGpHalf;
constexpr int kGpThreads = 192;
constexpr int kGpSmem = kGpStages * kGpStageBytes + 1024 /* alignment */ + 256;

__device__ __forceinline__ uint32_t gp_leader(const void* p) {          // the leader's copy of a shared-memory location
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
__device__ __forceinline__ void gp_tma_load(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint"
               " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void gp_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred P;\n\tsetp.ne.b32 P, %4, 0;\n\t"
               "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, P;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void gp_commit(uint64_t* bar) {               // arrives on this barrier of BOTH CTAs
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
__device__ __forceinline__ void gp_arrive(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// mbar_wait with acquire at cluster scope: the arrivals come from the other SM too.
__device__ __forceinline__ bool gp_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  const unsigned long long t0 = globaltimer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 128; ++i) {
      uint32_t ok;
      asm volatile("{\n\t.reg .pred P;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\tselp.u32 %0, 1, 0, P;\n\t}"
                   : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
      if (ok) return true;
    }
    if (*reinterpret_cast<volatile int*>(status) != 0) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      atomicCAS(status, 0, code);
      return false;
    }
  }
}

}  // namespace mx
