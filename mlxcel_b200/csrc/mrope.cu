// Rotary positions with several axes (time, row and column of an image or video patch). Frequency i of the rotated half turns with
// the position its axis has in this row: angle = positions[axis[i]][t] * inv_freq[i].
//
//   mx_mrope_append  q and k of the fused projection: optional per-head rms norm, rotation; q goes out, k and v into the paged pool
//                    (16-bit, or 8- / 4-bit codes with a bf16 scale and offset per 64 values)
//   mx_axial_rope    vision towers: q, k (rotated) and v of all heads as fp32 [H, R, D], what their attention reads
//
// An fp32 product of a position near 2^17 and its frequency is off by 2^-8 of a radian. The product and its reduction by whole turns
// are therefore done in fp64 (64 of them per token, shared by all heads), sine and cosine of what is left of a turn in fp32.
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
  const double turns = ang * 0.15915494309189535;                                     // 1 / (2 pi)
  sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn, &cs);
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

// The step and offset of 64 values between mn and mx as they are stored (bf16), and a value's code: round((x - low) / scale). Codes are
// taken against the rounded pair, which is what a reader expands them with.
template <int BITS>
struct KvCode {
  static constexpr int kTop = BITS == 8 ? 255 : 15;
  float scale, low;
  __device__ __forceinline__ KvCode(float mn, float mx)
      : scale(__bfloat162float(__float2bfloat16((mx - mn) / static_cast<float>(kTop)))), low(__bfloat162float(__float2bfloat16(mn))) {
    if (scale == 0.f) scale = 1.f;
  }
  __device__ __forceinline__ uint32_t operator()(float x) const { return static_cast<uint32_t>(min(kTop, max(0, __float2int_rn((x - low) / scale)))); }
  __device__ __forceinline__ uint32_t meta() const { return pack_bf16(scale, low); }
};

// Codes of 64 values, two per lane.
template <int BITS>
__device__ __forceinline__ void store_codes(float a, float b, int lane, uint8_t* dst, __nv_bfloat16* meta) {
  float mn = fminf(a, b), mx = fmaxf(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const KvCode<BITS> code(mn, mx);
  const uint32_t qa = code(a), qb = code(b);
  if constexpr (BITS == 8) {
    dst[lane] = static_cast<uint8_t>(qa);
    dst[32 + lane] = static_cast<uint8_t>(qb);
  } else {                                                        // neighbouring lanes share a byte, the even one in the low half
    const uint32_t qa1 = __shfl_down_sync(0xffffffffu, qa, 1), qb1 = __shfl_down_sync(0xffffffffu, qb, 1);
    if ((lane & 1) == 0) {
      dst[lane >> 1] = static_cast<uint8_t>(qa | (qa1 << 4));
      dst[16 + (lane >> 1)] = static_cast<uint8_t>(qb | (qb1 << 4));
    }
  }
  if (lane == 0) *reinterpret_cast<uint32_t*>(meta) = code.meta();
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

// ----------------------------------------------------------------------------- heads as vectors
// A lane holds 2 W columns of a head (W = 8 or 4, accesses of 16 or 8 bytes): the columns W u.. of the first half and their partners of
// the second, or (pairs) 2 W neighbours; the lanes behind the rotated width copy 2 W neighbours. LPH lanes work on a head, those beyond
// its D / (2 W) are idle. A CTA takes up to 4 tokens, so that its threads have an angle each; heads of all of them follow one another,
// two of a thread's in flight.
constexpr int kMropeTokens = 4;

template <int W>
struct MropeVec;
template <>
struct MropeVec<8> {
  using type = uint4;
  static __device__ __forceinline__ void widen(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
  }
  static __device__ __forceinline__ uint4 narrow(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
};
template <>
struct MropeVec<4> {
  using type = uint2;
  static __device__ __forceinline__ void widen(const uint2& v, float (&f)[4]) { f[0] = bf16_lo(v.x), f[1] = bf16_hi(v.x), f[2] = bf16_lo(v.y), f[3] = bf16_hi(v.y); }
  static __device__ __forceinline__ uint2 narrow(const float (&f)[4]) { return make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3])); }
};

// The first columns of a lane's two vectors, and whether they turn.
template <int W>
__device__ __forceinline__ bool unit_columns(int u, int half, int pairs, int& c0, int& c1) {
  const bool turns = u * W < half;
  if (pairs || !turns) {
    c0 = 2 * W * u;                        // (behind the rotated width, 2 half columns, too)
    c1 = c0 + W;
  } else {
    c0 = W * u;
    c1 = half + W * u;
  }
  return turns;
}
// Rows of n floats that lanes read W at a time are kept so that a warp's accesses of 16 bytes are neighbours: with W = 8 the first four
// of every eight, then the others.
template <int W>
__device__ __forceinline__ int kept_at(int i, int n) {
  return W == 8 ? (i >> 2 & 1) * (n >> 1) + (i >> 3) * 4 + (i & 3) : i;
}
template <int W>
__device__ __forceinline__ void read_kept(float (&d)[W], const float* row, int first, int n) {
#pragma unroll
  for (int i = 0; i < W; i += 4) *reinterpret_cast<float4*>(d + i) = *reinterpret_cast<const float4*>(row + kept_at<W>(first + i, n));
}

// Turns a lane's 2 W values by its W angles (from W u on, of `half`; they carry the scale).
template <int W>
__device__ __forceinline__ void turn_unit(float (&a)[W], float (&b)[W], const float* cs, const float* sn, int u, int half, int pairs) {
  alignas(16) float c[W], s[W];
  read_kept<W>(c, cs, W * u, half);
  read_kept<W>(s, sn, W * u, half);
  if (pairs) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const float x0 = a[2 * i], y0 = a[2 * i + 1], x1 = b[2 * i], y1 = b[2 * i + 1];
      a[2 * i] = x0 * c[i] - y0 * s[i];
      a[2 * i + 1] = y0 * c[i] + x0 * s[i];
      b[2 * i] = x1 * c[W / 2 + i] - y1 * s[W / 2 + i];
      b[2 * i + 1] = y1 * c[W / 2 + i] + x1 * s[W / 2 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  }
}

// (token, head) of an index that grows by a fixed step, without a division per step.
struct HeadWalk {
  int t, s;
  __device__ __forceinline__ HeadWalk(int item, int heads) : t(item / heads), s(item % heads) {}
  __device__ __forceinline__ void step(int by, int heads) {
    s += by;
    while (s >= heads) s -= heads, ++t;
  }
};

// Eight values' codes as they are stored: 8 bytes, or 4 with the first of two in the low half of a byte.
template <int BITS>
__device__ __forceinline__ void store_eight(const float (&x)[8], const KvCode<BITS>& code, uint8_t* dst) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[BITS == 8 ? i / 4 : 0] |= code(x[i]) << (BITS == 8 ? i % 4 * 8 : i * 4);
  if constexpr (BITS == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(dst) = w[0];
}

// BITS 8 and 4 (W = 8): 64 columns are those of four lanes, or (halves 64 or a multiple apart) one vector of eight lanes each.
template <int W, int LPH, bool NORM, int BITS>
__global__ void __launch_bounds__(kMropeThreads, W == 8 ? 3 : 4) mrope_append_vec_kernel(const MropeParams p, int tokens, int per_block) {
  using Vec = typename MropeVec<W>::type;
  __shared__ __align__(16) float cs[kMropeTokens * kMropeMaxDim / 2], sn[kMropeTokens * kMropeMaxDim / 2];
  __shared__ __align__(16) float norm_w[NORM ? 2 : 1][NORM ? kMropeMaxDim : 4];      // of q and k
  __shared__ long long kept[kMropeTokens];                      // the row of a token's first head in the pool; below 0: nowhere
  constexpr int HPI = kMropeThreads / LPH, HPW = 32 / LPH;      // heads at once: of the CTA, of a warp
  pdl_trigger();
  pdl_wait();
  const int t0 = blockIdx.x * per_block, rows = min(per_block, tokens - t0), heads = p.Hq + 2 * p.Hkv, half = p.ang.half, D = p.D;
  const int g = threadIdx.x / LPH, u = threadIdx.x % LPH;
  int c0, c1;
  const bool turns = unit_columns<W>(u, half, p.pairs, c0, c1), live = u * 2 * W < D;
  const __nv_bfloat16* src = p.qkv + t0 * p.ldqkv;
  Vec v[2][2];
  HeadWalk ahead(g, heads);
  auto load = [&](Vec (&x)[2]) {
    if (live && ahead.t < rows) {
      const __nv_bfloat16* from = src + ahead.t * p.ldqkv + ahead.s * D;
      x[0] = *reinterpret_cast<const Vec*>(from + c0);
      x[1] = *reinterpret_cast<const Vec*>(from + c1);
    }
    ahead.step(HPI, heads);
  };
  load(v[0]);
  load(v[1]);
  [[maybe_unused]] const float inv_dim = 1.f / static_cast<float>(D);
  if constexpr (NORM) {
    if (threadIdx.x < D) {
      const int to = kept_at<W>(threadIdx.x, D);
      norm_w[0][to] = p.q_norm_w ? __bfloat162float(p.q_norm_w[threadIdx.x]) : 1.f;
      norm_w[1][to] = p.k_norm_w ? __bfloat162float(p.k_norm_w[threadIdx.x]) : 1.f;
    }
  }
  if (threadIdx.x < rows) {
    const long long slot = p.slots[t0 + threadIdx.x], blk = slot / p.block_size;
    kept[threadIdx.x] = slot < 0 || slot >= p.n_slots ? -1 : blk * p.Hkv * p.block_size + (slot - blk * p.block_size);
  }
  for (int i = threadIdx.x; i < rows * half; i += kMropeThreads) {
    const int t = i / half;
    float sine, cosine;
    axis_angle(p.ang, t0 + t, i - t * half, sine, cosine);
    const int to = t * half + kept_at<W>(i - t * half, half);
    sn[to] = sine * p.mscale;
    cs[to] = cosine * p.mscale;
  }
  __syncthreads();
  HeadWalk at(g, heads);
  auto work = [&](Vec (&x)[2]) {
    alignas(16) float a[W], b[W];
    const bool here = live && at.t < rows;
    const bool is_q = at.s < p.Hq, is_v = at.s >= p.Hq + p.Hkv;
    if (here) {
      MropeVec<W>::widen(x[0], a);
      MropeVec<W>::widen(x[1], b);
    }
    load(x);
    if constexpr (NORM) {
      float2* a2 = reinterpret_cast<float2*>(a);
      float2* b2 = reinterpret_cast<float2*>(b);
      float2 sq = make_float2(0.f, 0.f);
      if (here) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) sq = __ffma2_rn(b2[i], b2[i], __ffma2_rn(a2[i], a2[i], sq));
      }
      float ss = sq.x + sq.y;
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (here && !is_v && (is_q ? p.q_norm_w : p.k_norm_w) != nullptr) {       // (not rounded before the rotation)
        const float rstd = rsqrtf(ss * inv_dim + p.eps);
        const float2 r2 = make_float2(rstd, rstd);
        alignas(16) float w[W];
        const float2* w2 = reinterpret_cast<const float2*>(w);
        read_kept<W>(w, norm_w[is_q ? 0 : 1], c0, D);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) a2[i] = __fmul2_rn(__fmul2_rn(a2[i], r2), w2[i]);
        read_kept<W>(w, norm_w[is_q ? 0 : 1], c1, D);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) b2[i] = __fmul2_rn(__fmul2_rn(b2[i], r2), w2[i]);
      }
    }
    if (here && turns && !is_v) turn_unit<W>(a, b, cs + at.t * half, sn + at.t * half, u, half, p.pairs);
    const int head = at.s - p.Hq - (is_v ? p.Hkv : 0);
    const long long row = here && !is_q ? kept[at.t] : -1;                 // (a row without a slot leaves the pool alone)
    const long long place = row + static_cast<long long>(head) * p.block_size;
    __nv_bfloat16* dst = nullptr;
    if (here && is_q) dst = p.q_out + (t0 + at.t) * p.ldq + at.s * D;
    else if (BITS == 16 && row >= 0) dst = static_cast<__nv_bfloat16*>(is_v ? p.v_pool : p.k_pool) + place * D;
    if (dst != nullptr) {
      *reinterpret_cast<Vec*>(dst + c0) = MropeVec<W>::narrow(a);
      *reinterpret_cast<Vec*>(dst + c1) = MropeVec<W>::narrow(b);
    }
    if constexpr (BITS != 16) {
      if (__any_sync(0xffffffffu, row >= 0)) {
        const bool apart = (c0 >> 6) != (c1 >> 6);
        float low[2], high[2];
        low[0] = high[0] = here ? a[0] : 0.f;
        low[1] = high[1] = here ? b[0] : 0.f;
        if (here) {
#pragma unroll
          for (int i = 1; i < W; ++i) {
            low[0] = fminf(low[0], a[i]), high[0] = fmaxf(high[0], a[i]);
            low[1] = fminf(low[1], b[i]), high[1] = fmaxf(high[1], b[i]);
          }
        }
        if (!apart) low[0] = low[1] = fminf(low[0], low[1]), high[0] = high[1] = fmaxf(high[0], high[1]);
#pragma unroll
        for (int o = 1; o <= 4; o <<= 1) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float l = __shfl_xor_sync(0xffffffffu, low[i], o), h = __shfl_xor_sync(0xffffffffu, high[i], o);
            if (o < 4 || apart) low[i] = fminf(low[i], l), high[i] = fmaxf(high[i], h);
          }
        }
        if (row >= 0) {
          const KvCode<BITS> code_a(low[0], high[0]), code_b(low[1], high[1]);
          uint8_t* codes = static_cast<uint8_t*>(is_v ? p.v_pool : p.k_pool) + place * (D * BITS / 8);
          store_eight<BITS>(a, code_a, codes + c0 * BITS / 8);
          store_eight<BITS>(b, code_b, codes + c1 * BITS / 8);
          uint32_t* meta = reinterpret_cast<uint32_t*>(is_v ? p.v_meta : p.k_meta) + place * (D / 64);
          if (u % (apart ? 8 : 4) == 0) meta[c0 >> 6] = code_a.meta();
          if (apart && u % 8 == 0) meta[c1 >> 6] = code_b.meta();
        }
      }
    }
    at.step(HPI, heads);
  };
  // whole warps stay in the loop (it goes by the warp's first head), as the norm's sums are exchanged between lanes
  for (int left = rows * heads - (g - g % HPW); left > 0; left -= 2 * HPI) {
    work(v[0]);
    if (left > HPI) work(v[1]);
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

// Units of 2 W columns of all heads (q, k, v) of up to 4 rows follow one another over the threads.
template <int W>
__global__ void __launch_bounds__(kMropeThreads, W == 8 ? 3 : 4) axial_rope_vec_kernel(const AxialParams p, int per_block) {
  using Vec = typename MropeVec<W>::type;
  __shared__ __align__(16) float cs[kMropeTokens * kMropeMaxDim / 2], sn[kMropeTokens * kMropeMaxDim / 2];
  pdl_trigger();
  pdl_wait();
  const long long t0 = static_cast<long long>(blockIdx.x) * per_block;
  const int rows = static_cast<int>(min(static_cast<long long>(per_block), p.rows - t0)), half = p.ang.half, D = p.D, heads = 3 * p.H;
  const int units = D / (2 * W), u_step = kMropeThreads % units, h_step = kMropeThreads / units;
  struct Place {
    int u;
    HeadWalk at;
  };
  auto step = [&](Place& x) {
    x.u += u_step;
    const int carry = x.u >= units;
    if (carry) x.u -= units;
    x.at.step(h_step + carry, heads);
  };
  const __nv_bfloat16* src = p.qkv + t0 * p.ldqkv;
  Place ahead{static_cast<int>(threadIdx.x) % units, HeadWalk(threadIdx.x / units, heads)}, now = ahead;
  // units of a thread on their way: 5476 patches of 16 heads of 80 26.5 us with 2, 25.3 with 4, 24.8 with 8 (4096 of 12 of 64 11.6, 9.7 with 4)
  constexpr int kAhead = 4;
  Vec v[kAhead][2];
  auto load = [&](Vec (&x)[2]) {
    if (ahead.at.t < rows) {
      const __nv_bfloat16* from = src + ahead.at.t * p.ldqkv + ahead.at.s * D + ahead.u * W;
      x[0] = *reinterpret_cast<const Vec*>(from);
      x[1] = *reinterpret_cast<const Vec*>(from + half);
    }
    step(ahead);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(v[i]);
  for (int i = threadIdx.x; i < rows * half; i += kMropeThreads) axis_angle(p.ang, t0 + i / half, i % half, sn[i], cs[i]);
  __syncthreads();
  auto work = [&](Vec (&x)[2]) {
    float a[W], b[W];
    MropeVec<W>::widen(x[0], a);
    MropeVec<W>::widen(x[1], b);
    load(x);
    const int part = (now.at.s >= p.H) + (now.at.s >= 2 * p.H), h = now.at.s - part * p.H, angles = now.at.t * half;
    if (part < 2) turn_unit<W>(a, b, cs + angles, sn + angles, now.u, half, 0);
    float* dst = (part == 0 ? p.q : part == 1 ? p.k : p.v) + (h * p.rows + t0 + now.at.t) * D + W * now.u;
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      *reinterpret_cast<float4*>(dst + i) = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
      *reinterpret_cast<float4*>(dst + half + i) = make_float4(b[i], b[i + 1], b[i + 2], b[i + 3]);
    }
    step(now);
  };
  while (now.at.t < rows) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (now.at.t < rows) work(v[i]);
  }
}

// Tokens of a CTA: as many as have an angle per thread, while every SM still gets four CTAs. Between 600 and 1200 tokens that is one a CTA
// and more CTAs than are resident (1031 on 592 places: 8.1 us, of which a copy of the bytes takes 2.9).
static int mrope_tokens(int T) {
  int n = kMropeTokens;
  while (n > 1 && T < 4 * n * device_sm_count()) n /= 2;
  return n;
}
// Columns per access (`most` or 4; 0: not in vectors) for heads of D whose first rot columns turn.
static int mrope_width(int most, int D, int rot, uintptr_t addresses, long long strides) {
  for (int w = most; w >= 4; w -= 4)
    if (rot > 0 && D % (2 * w) == 0 && rot % (2 * w) == 0 && strides % w == 0 && addresses % (2 * w) == 0) return w;
  return 0;
}

}  // namespace mx

extern "C" int mx_mrope_append(const MxMropeAppend* a, void* stream_) {
  using namespace mx;
  const int T = a->T, D = a->D, rot_dim = a->rot_dim, kv_bits = a->kv_bits;
  if (T <= 0) return 0;
  if (D <= 0 || D > kMropeMaxDim || rot_dim < 0 || rot_dim > D || rot_dim % 2 || a->Hq < 0 || a->Hkv < 0 || a->axes < 1 || a->block_size < 1) return -1;
  if (a->Hq + a->Hkv == 0) return -1;                        // (threads walk from head to head: without any they would not come to an end)
  if ((kv_bits != 16 && kv_bits != 8 && kv_bits != 4) || (kv_bits != 16 && (D % 64 || a->k_meta == nullptr || a->v_meta == nullptr))) return -1;
  MropeParams p{};
  p.qkv = static_cast<const __nv_bfloat16*>(a->qkv);
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.slots = a->slots;
  p.k_pool = a->k_pool, p.v_pool = a->v_pool;
  p.k_meta = static_cast<__nv_bfloat16*>(a->k_meta), p.v_meta = static_cast<__nv_bfloat16*>(a->v_meta);
  p.q_norm_w = static_cast<const __nv_bfloat16*>(a->q_norm_w), p.k_norm_w = static_cast<const __nv_bfloat16*>(a->k_norm_w);
  p.ang = {a->positions, a->axis, a->inv_freq, a->ldp, a->axes, rot_dim / 2};
  p.ldqkv = a->ldqkv, p.ldq = a->ldq, p.n_slots = a->n_slots;
  p.Hq = a->Hq, p.Hkv = a->Hkv, p.D = D, p.block_size = a->block_size, p.pairs = a->pairs;
  p.eps = a->norm_eps, p.mscale = a->mscale;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  cudaError_t e;
  auto bits_of = [](const void* a) { return reinterpret_cast<uintptr_t>(a); };
  // Accesses of 8 bytes leave room for more warps, those of 16 bytes take fewer instructions: 1031 tokens of 32 + 4 heads 8.1 us against 10.8,
  // 8191 of 64 + 16 heads with norms 81 against 73. Codes are made of 8 values of a lane at once; each takes a
  // division, and the 12 forms that make them spill 4 to 24 bytes (8191 tokens of 64 + 16 heads without norms 82 us with 8 bits, 80 with 4, 66
  // with 16; 4000 of 32 + 16 heads 34, 33, 23).
  const bool coded = kv_bits != 16;
  int w = mrope_width(coded || mrope_tokens(T) == kMropeTokens ? 8 : 4, D, rot_dim, bits_of(a->qkv) | bits_of(a->q_out) | bits_of(a->q_norm_w) | bits_of(a->k_norm_w) |
                      (coded ? 0 : bits_of(a->k_pool) | bits_of(a->v_pool)), a->ldqkv | a->ldq);
  if (coded && (w != 8 || !(a->pairs || rot_dim <= 64 || rot_dim % 128 == 0) || (bits_of(a->k_pool) | bits_of(a->v_pool)) % 8 ||
                (bits_of(a->k_meta) | bits_of(a->v_meta)) % 4))
    w = 0;
  if (w != 0) {
    const int lanes = D / (2 * w), per = mrope_tokens(T), blocks = (T + per - 1) / per;
    const bool norm = a->q_norm_w != nullptr || a->k_norm_w != nullptr;
    auto run = [&](auto kern) { return static_cast<int>(launch_kernel(kern, dim3(blocks), dim3(kMropeThreads), 0, stream, p, T, per)); };
#define MX_MROPE(W_, L_, B_) return norm ? run(mrope_append_vec_kernel<W_, L_, true, B_>) : run(mrope_append_vec_kernel<W_, L_, false, B_>)
#define MX_MROPE_LANES(B_)              \
  if (lanes <= 4) MX_MROPE(8, 4, B_);   \
  if (lanes <= 8) MX_MROPE(8, 8, B_);   \
  MX_MROPE(8, 16, B_)
    if (kv_bits == 8) { MX_MROPE_LANES(8); }
    if (kv_bits == 4) { MX_MROPE_LANES(4); }
    if (w == 8) { MX_MROPE_LANES(16); }
    if (lanes <= 8) MX_MROPE(4, 8, 16);
    if (lanes <= 16) MX_MROPE(4, 16, 16);
    MX_MROPE(4, 32, 16);
#undef MX_MROPE_LANES
#undef MX_MROPE
  }
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
  // (16-byte accesses: 33 us where 8-byte ones take 26 with as much in flight, 5476 patches of 16 heads of 80)
  const int w = mrope_width(4, D, D, reinterpret_cast<uintptr_t>(qkv), ldqkv);
  // (results are written 16 bytes at a time)
  if (w != 0 && aligned_to(q, 16) && aligned_to(k, 16) && aligned_to(v, 16)) {
    const int per = mrope_tokens(R), blocks = (R + per - 1) / per;
    return static_cast<int>(launch_kernel(axial_rope_vec_kernel<4>, dim3(blocks), dim3(kMropeThreads), 0, static_cast<cudaStream_t>(stream_), p, per));
  }
  return static_cast<int>(launch_kernel(axial_rope_kernel, dim3(R), dim3(kMropeThreads), 0, static_cast<cudaStream_t>(stream_), p));
}
