// Rotary positions with several axes (time, row and column of an image or video patch). Frequency i of the rotated half turns with
// the position its axis has in this row: angle = positions[axis[i]][t] * inv_freq[i].
//
//   mx_mrope_append  q and k of the fused projection: optional per-head rms norm, rotation; q goes out, k and v into the paged pool
//                    (16-bit, or 8- / 4-bit codes with a bf16 scale and offset per 64 values)
//   mx_axial_rope    vision towers: q, k (rotated) and v of all heads as fp32 [H, R, D], what their attention reads
//
// An fp32 product of a position near 2^17 and its frequency is off by 2^-8 of a radian. The product and its reduction by whole turns
// are therefore done in fp64 (64 of them per token, shared by all heads), sine and cosine of the remainder in fp32.
#include "api.h"
#include "common.cuh"
#include "typed.cuh"

namespace mx {

constexpr int kMropeThreads = 256;
constexpr int kMropeMaxDim = 256;

struct MropeAngles {
  const int* positions;      // [axes][ldp]
  const int* axis;           // [half]
  const float* inv_freq;     // [half]
  long long ldp;
  int axes, half;
};

__device__ __forceinline__ void axis_angle(const MropeAngles& a, long long t, int i, float& sn, float& cs) {
  const int ax = min(max(a.axis[i], 0), a.axes - 1);
  const double ang = static_cast<double>(a.positions[ax * a.ldp + t]) * static_cast<double>(a.inv_freq[i]);
  const double turns = rint(ang * 0.15915494309189535);                               // 1 / (2 pi)
  const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, ang));     // 2 pi as a sum of two
  sincosf(static_cast<float>(r), &sn, &cs);
}

struct MropeParams {
  const __nv_bfloat16* qkv;
  __nv_bfloat16* q_out;
  const int* slots;
  void* k_pool;
  void* v_pool;
  __nv_bfloat16* k_meta;
  __nv_bfloat16* v_meta;
  const __nv_bfloat16* q_norm_w;
  const __nv_bfloat16* k_norm_w;
  MropeAngles ang;
  long long ldqkv, ldq, n_slots;
  int Hq, Hkv, D, block_size, pairs;       // pairs: neighbouring columns (2i, 2i + 1) turn together instead of (i, i + half)
  float eps, mscale;
};

// Codes of 64 values (two per lane): q = round((x - low) / scale), scale = (high - low) / levels, both kept in bf16.
template <int BITS>
__device__ __forceinline__ void store_codes(float a, float b, int lane, uint8_t* dst, __nv_bfloat16* meta) {
  constexpr float kLevels = BITS == 8 ? 255.f : 15.f;
  float mn = fminf(a, b), mx = fmaxf(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  // codes are taken against the rounded pair, which is what a reader expands them with
  float scale = __bfloat162float(__float2bfloat16((mx - mn) / kLevels));
  const float low = __bfloat162float(__float2bfloat16(mn));
  if (scale == 0.f) scale = 1.f;
  const int top = static_cast<int>(kLevels);
  const int qa = min(top, max(0, __float2int_rn((a - low) / scale)));
  const int qb = min(top, max(0, __float2int_rn((b - low) / scale)));
  if constexpr (BITS == 8) {
    dst[lane] = static_cast<uint8_t>(qa);
    dst[32 + lane] = static_cast<uint8_t>(qb);
  } else {                                                        // neighbouring lanes share a byte, the even one in the low half
    const int qa1 = __shfl_down_sync(0xffffffffu, qa, 1), qb1 = __shfl_down_sync(0xffffffffu, qb, 1);
    if ((lane & 1) == 0) {
      dst[lane >> 1] = static_cast<uint8_t>(qa | (qa1 << 4));
      dst[16 + (lane >> 1)] = static_cast<uint8_t>(qb | (qb1 << 4));
    }
  }
  if (lane == 0) {
    meta[0] = __float2bfloat16(scale);
    meta[1] = __float2bfloat16(low);
  }
}

// Any head size up to 256, any rotated width, every pool. A CTA is one token, a warp one head at a time, staged in shared memory.
template <int KV_BITS>
__global__ void __launch_bounds__(kMropeThreads) mrope_append_kernel(const MropeParams p) {
  __shared__ float sn[kMropeMaxDim / 2], cs[kMropeMaxDim / 2];
  __shared__ float stage[kMropeThreads / 32][kMropeMaxDim];
  pdl_trigger();
  pdl_wait();
  const long long t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.D, half = p.ang.half;
  for (int i = threadIdx.x; i < half; i += kMropeThreads) axis_angle(p.ang, t, i, sn[i], cs[i]);
  __syncthreads();
  const long long slot = p.slots[t];
  const bool kept = slot >= 0 && slot < p.n_slots;
  float* st = stage[warp];
  for (int s = warp; s < p.Hq + 2 * p.Hkv; s += kMropeThreads / 32) {
    const bool is_q = s < p.Hq, is_v = s >= p.Hq + p.Hkv;
    if (!is_q && !kept) break;                                   // a row without a slot leaves the pool alone
    const __nv_bfloat16* src = p.qkv + t * p.ldqkv + static_cast<long long>(s) * D;
    float ss = 0.f;
    for (int i = lane; i < D; i += 32) {
      const float v = __bfloat162float(src[i]);
      st[i] = v;
      ss += v * v;
    }
    __syncwarp();
    const __nv_bfloat16* nw = is_q ? p.q_norm_w : (is_v ? nullptr : p.k_norm_w);
    if (nw != nullptr) {                                         // (not rounded before the rotation)
      const float rstd = rsqrtf(warp_sum(ss) / D + p.eps);
      for (int i = lane; i < D; i += 32) st[i] *= rstd * __bfloat162float(nw[i]);
      __syncwarp();
    }
    if (!is_v) {
      for (int i = lane; i < half; i += 32) {
        const int i1 = p.pairs ? 2 * i : i, i2 = p.pairs ? 2 * i + 1 : i + half;
        const float a = st[i1], b = st[i2];
        st[i1] = (a * cs[i] - b * sn[i]) * p.mscale;
        st[i2] = (b * cs[i] + a * sn[i]) * p.mscale;
      }
      __syncwarp();
    }
    if (is_q) {
      __nv_bfloat16* dst = p.q_out + t * p.ldq + static_cast<long long>(s) * D;
      for (int i = lane; i < D; i += 32) dst[i] = __float2bfloat16(st[i]);
    } else {
      const int head = s - p.Hq - (is_v ? p.Hkv : 0);
      const long long blk = slot / p.block_size, off = slot - blk * p.block_size;
      const long long row = (blk * p.Hkv + head) * p.block_size + off;
      void* pool = is_v ? p.v_pool : p.k_pool;
      if constexpr (KV_BITS == 16) {
        for (int i = lane; i < D; i += 32) static_cast<__nv_bfloat16*>(pool)[row * D + i] = __float2bfloat16(st[i]);
      } else {
        __nv_bfloat16* meta = (is_v ? p.v_meta : p.k_meta) + row * (D / 64) * 2;
        uint8_t* dst = static_cast<uint8_t*>(pool) + row * (D * KV_BITS / 8);
        for (int g = 0; g < D / 64; ++g)
          store_codes<KV_BITS>(st[g * 64 + lane], st[g * 64 + 32 + lane], lane, dst + g * (64 * KV_BITS / 8), meta + g * 2);
      }
    }
    __syncwarp();
  }
}

struct AxialParams {
  const __nv_bfloat16* qkv;
  float* q;
  float* k;
  float* v;
  MropeAngles ang;
  long long ldqkv, rows;
  int H, D;
};

__global__ void __launch_bounds__(kMropeThreads) axial_rope_kernel(const AxialParams p) {
  __shared__ float sn[kMropeMaxDim / 2], cs[kMropeMaxDim / 2];
  pdl_trigger();
  pdl_wait();
  const long long t = blockIdx.x;
  const int half = p.ang.half, D = p.D, n = p.H * D;
  for (int i = threadIdx.x; i < half; i += kMropeThreads) axis_angle(p.ang, t, i, sn[i], cs[i]);
  __syncthreads();
  for (int j = threadIdx.x; j < p.H * half; j += kMropeThreads) {
    const int h = j / half, i = j - h * half;
    const __nv_bfloat16* src = p.qkv + t * p.ldqkv + h * D + i;
    const long long dst = (h * p.rows + t) * D + i;
    const float qa = __bfloat162float(src[0]), qb = __bfloat162float(src[half]);
    const float ka = __bfloat162float(src[n]), kb = __bfloat162float(src[n + half]);
    p.q[dst] = qa * cs[i] - qb * sn[i];
    p.q[dst + half] = qb * cs[i] + qa * sn[i];
    p.k[dst] = ka * cs[i] - kb * sn[i];
    p.k[dst + half] = kb * cs[i] + ka * sn[i];
    p.v[dst] = __bfloat162float(src[2 * n]);
    p.v[dst + half] = __bfloat162float(src[2 * n + half]);
  }
}

}  // namespace mx

extern "C" int mx_mrope_append(const void* qkv, long long ldqkv, void* q_out, long long ldq, const int* positions, long long ldp, int axes,
                               const int* axis, const int* slots, long long n_slots, const float* inv_freq, void* k_pool, void* v_pool,
                               void* k_meta, void* v_meta, const void* q_norm_w, const void* k_norm_w, float norm_eps, int T, int Hq,
                               int Hkv, int D, int rot_dim, int block_size, int pairs, float mscale, int kv_bits, void* stream_) {
  using namespace mx;
  if (T <= 0) return 0;
  if (D <= 0 || D > kMropeMaxDim || rot_dim < 0 || rot_dim > D || rot_dim % 2 || Hq < 0 || Hkv < 0 || axes < 1 || block_size < 1) return -1;
  if ((kv_bits != 16 && kv_bits != 8 && kv_bits != 4) || (kv_bits != 16 && (D % 64 || k_meta == nullptr || v_meta == nullptr))) return -1;
  MropeParams p{};
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.slots = slots;
  p.k_pool = k_pool, p.v_pool = v_pool;
  p.k_meta = static_cast<__nv_bfloat16*>(k_meta), p.v_meta = static_cast<__nv_bfloat16*>(v_meta);
  p.q_norm_w = static_cast<const __nv_bfloat16*>(q_norm_w), p.k_norm_w = static_cast<const __nv_bfloat16*>(k_norm_w);
  p.ang = {positions, axis, inv_freq, ldp, axes, rot_dim / 2};
  p.ldqkv = ldqkv, p.ldq = ldq, p.n_slots = n_slots;
  p.Hq = Hq, p.Hkv = Hkv, p.D = D, p.block_size = block_size, p.pairs = pairs;
  p.eps = norm_eps, p.mscale = mscale;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  cudaError_t e;
  if (kv_bits == 16) e = launch_kernel(mrope_append_kernel<16>, dim3(T), dim3(kMropeThreads), 0, stream, p);
  else if (kv_bits == 8) e = launch_kernel(mrope_append_kernel<8>, dim3(T), dim3(kMropeThreads), 0, stream, p);
  else e = launch_kernel(mrope_append_kernel<4>, dim3(T), dim3(kMropeThreads), 0, stream, p);
  return static_cast<int>(e);
}

extern "C" int mx_axial_rope(const void* qkv, long long ldqkv, float* q, float* k, float* v, const int* positions, long long ldp, int axes,
                             const int* axis, const float* inv_freq, int R, int H, int D, void* stream_) {
  using namespace mx;
  if (R <= 0 || H <= 0) return 0;
  if (D <= 0 || D > kMropeMaxDim || D % 2 || axes < 1) return -1;
  AxialParams p{static_cast<const __nv_bfloat16*>(qkv), q, k, v, {positions, axis, inv_freq, ldp, axes, D / 2}, ldqkv, R, H, D};
  return static_cast<int>(launch_kernel(axial_rope_kernel, dim3(R), dim3(kMropeThreads), 0, static_cast<cudaStream_t>(stream_), p));
}
