// The step between two sub-layers of a residual stream, in one pass over the row:
//
//   b = rms(x) * (post_w + w_bias)          (post_w == NULL: b = x)
//   h = round(residual + scale * gate * b)  (gate: a factor per channel)
//   y = rms(h) * (pre_w + w_bias), or layer norm of h times (pre_w + w_bias) + pre_b
//
// Statistics, the branch and the sum are fp32. h is the stored residual stream, so it is rounded to the row type, and y is the norm
// of the rounded row: what a later reader of the stream would compute. b and the scaled branch are not rounded in between.
//
// Bound by memory: x and residual in, h and y out, four rows. The row stays in registers between its reductions (two for rms, three
// with the mean of a layer norm). Measured (us, of what a copy of these bytes would take): 8192 x 5120 bf16 62 (82 %; 64 with one
// element per instruction, 83 with one access per thread and the weights asked for when they are needed, 70 with CTAs that stay and
// have their next row on its way to shared memory: fewer rows are then between their sums at a time), 8192 x 4096 45 (91 %), 2000 x 8192
// fp32 45 (89 %), one row of 2560 2.1; layer norm with gate, 1370 x 1024: 4.7 in bf16, 5.9 in fp32 (floors 1.7 and 3.4; launch and sums).
// Rows of an odd length: 8192 x 5119 136 (241 element by element), 8192 x 1003 26 (32); each row shifts its weights anew from two reads.
#include "api.h"
#include "common.cuh"
#include "typed.cuh"

namespace mx {

struct BranchNormParams {
  const void* x;
  const void* residual;
  const void* post_w;
  const void* gate;
  const void* pre_w;
  const void* pre_b;
  void* h;
  void* y;
  long long ldx, ldr, ldh, ldy;
  int dim;
  float scale, eps, w_bias;
};

// Sum over the CTA; `red` holds 32 floats that no other reduction in flight uses. One barrier: every thread adds the warps' sums.
__device__ __forceinline__ float row_sum(float v, float* red) {
  const int warps = blockDim.x >> 5;
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < warps; ++i) t += red[i];
  return t;
}

// V elements of type T in one access (16 bytes, or one element).
template <typename T, int V>
struct Pack {
  static_assert(V == 1 || V * sizeof(T) == 16, "one element or 16 bytes");
  uint4 w;
  T e;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) e = *p;
    else w = *reinterpret_cast<const uint4*>(p);
  }
  __device__ __forceinline__ void widen(float (&f)[V]) const {
    if constexpr (V == 1) {
      f[0] = to_f(e);
    } else {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (V == 8) f[2 * j] = bf16_lo(u[j]), f[2 * j + 1] = bf16_hi(u[j]);
        else f[j] = __uint_as_float(u[j]);
      }
    }
  }
  // Rounds f to the type and leaves what is stored in f.
  __device__ __forceinline__ void narrow(float (&f)[V]) {
    if constexpr (V == 1) {
      e = from_f<T>(f[0]);
    } else if constexpr (V == 8) {
      w = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    } else {
      w = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    widen(f);
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) *p = e;
    else *reinterpret_cast<uint4*>(p) = w;
  }
};

// a = a b + c (b and c as many or one number), a = a b, and a^2 added to s; rows of bf16, which take more instructions per byte, two
// elements at a time.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
template <int V>
__device__ __forceinline__ void mul_add(float (&a)[V], const float (&b)[V], const float (&c)[V]) {
#pragma unroll
  for (int j = 0; j < V; j += V == 8 ? 2 : 1) {
    if constexpr (V == 8) {
      const float2 r = __ffma2_rn(make_float2(a[j], a[j + 1]), make_float2(b[j], b[j + 1]), make_float2(c[j], c[j + 1]));
      a[j] = r.x, a[j + 1] = r.y;
    } else {
      a[j] = fmaf(a[j], b[j], c[j]);
    }
  }
}
template <int V>
__device__ __forceinline__ void mul_add(float (&a)[V], float b, float c) {
#pragma unroll
  for (int j = 0; j < V; j += V == 8 ? 2 : 1) {
    if constexpr (V == 8) {
      const float2 r = __ffma2_rn(make_float2(a[j], a[j + 1]), both(b), both(c));
      a[j] = r.x, a[j + 1] = r.y;
    } else {
      a[j] = fmaf(a[j], b, c);
    }
  }
}
template <int V>
__device__ __forceinline__ void mul(float (&a)[V], const float (&b)[V]) {
#pragma unroll
  for (int j = 0; j < V; j += V == 8 ? 2 : 1) {
    if constexpr (V == 8) {
      const float2 r = __fmul2_rn(make_float2(a[j], a[j + 1]), make_float2(b[j], b[j + 1]));
      a[j] = r.x, a[j + 1] = r.y;
    } else {
      a[j] *= b[j];
    }
  }
}
template <int V>
__device__ __forceinline__ void add_squares(float2& s, const float (&a)[V]) {
#pragma unroll
  for (int j = 0; j < V; j += V == 8 ? 2 : 1) {
    if constexpr (V == 8) s = __ffma2_rn(make_float2(a[j], a[j + 1]), make_float2(a[j], a[j + 1]), s);
    else s.x = fmaf(a[j], a[j], s.x);
  }
}

// Rows that do not start on 16 bytes but all at the same place within 16 bytes (rows of an odd length behind each other) are covered by
// the aligned vectors that hold them: vector v has the elements v V - o ... of a row that starts o elements behind a boundary. Ends are
// read and written element by element (what is beyond the row counts as 0 and is not touched).
template <typename T, int V>
__device__ __forceinline__ void load_part(Pack<T, V>& d, const T* row, int first, int dim) {
  if (first >= 0 && first + V <= dim) {
    d.load(row + first);
  } else {
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = first + j >= 0 && first + j < dim ? to_f(row[first + j]) : 0.f;
    d.narrow(f);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_part(const Pack<T, V>& s, T* row, int first, int dim) {
  if (first >= 0 && first + V <= dim) {
    s.store(row + first);
  } else {
    float f[V];
    s.widen(f);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (first + j >= 0 && first + j < dim) row[first + j] = from_f<T>(f[j]);
  }
}
// The last O elements of vector a and the first V - O of b.
template <typename T, int V, int O>
__device__ __forceinline__ uint4 joined(const uint4& a, const uint4& b) {
  constexpr int bytes = 16 - O * static_cast<int>(sizeof(T)), q = bytes / 4;
  const uint32_t w[9] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, 0u};
  if constexpr (bytes % 4 == 0) return make_uint4(w[q], w[q + 1], w[q + 2], w[q + 3]);
  else return make_uint4(__funnelshift_r(w[q], w[q + 1], 16), __funnelshift_r(w[q + 1], w[q + 2], 16), __funnelshift_r(w[q + 2], w[q + 3], 16),
                         __funnelshift_r(w[q + 3], w[q + 4], 16));
}
// Elements first .. first + V of a vector of weights that starts on 16 bytes, first = v V - o.
template <typename T, int V>
__device__ __forceinline__ void load_shifted(Pack<T, V>& d, const T* w, int v, int o, int dim) {
  Pack<T, V> a, b;
  load_part(b, w, v * V, dim);
  if (o == 0) {
    d = b;
    return;
  }
  load_part(a, w, (v - 1) * V, dim);
  switch (o) {
    case 1: d.w = joined<T, V, 1>(a.w, b.w); break;
    case 2: d.w = joined<T, V, 2>(a.w, b.w); break;
    case 3: d.w = joined<T, V, 3>(a.w, b.w); break;
    default:
      if constexpr (V == 8) {
        switch (o) {
          case 4: d.w = joined<T, V, 4>(a.w, b.w); break;
          case 5: d.w = joined<T, V, 5>(a.w, b.w); break;
          case 6: d.w = joined<T, V, 6>(a.w, b.w); break;
          default: d.w = joined<T, V, 7>(a.w, b.w); break;
        }
      }
  }
}

// (registers: 4 CTAs of 256 threads or 64 a thread cost more in spills than they hide: 8192 x 4096 48 us in place of 45)
template <typename T, int V, int VPT, int MOST, bool LAYER, bool SHIFT>
__global__ void __launch_bounds__(MOST, VPT > 4 ? 1 : MOST == 256 ? 3 : MOST == 512 ? 2 : 1) branch_norm_kernel(const BranchNormParams p) {
  __shared__ float red[3][32];
  pdl_trigger();
  pdl_wait();
  const size_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const int o = SHIFT ? static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)) : 0;
  const int nvec = SHIFT ? (p.dim + o + V - 1) / V : p.dim / V;
  auto get = [&](Pack<T, V>& d, const T* from, int v) {
    if constexpr (SHIFT) load_part(d, from, v * V - o, p.dim);
    else d.load(from + static_cast<size_t>(v) * V);
  };
  auto put = [&](const Pack<T, V>& d, T* to, int v) {
    if constexpr (SHIFT) store_part(d, to, v * V - o, p.dim);
    else d.store(to + static_cast<size_t>(v) * V);
  };
  auto weights = [&](Pack<T, V>& d, const T* from, int v) {
    if constexpr (SHIFT) load_shifted(d, from, v, o, p.dim);
    else d.load(from + static_cast<size_t>(v) * V);
  };
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
  const T* post = static_cast<const T*>(p.post_w);
  const T* gate = static_cast<const T*>(p.gate);
  const T* pre = static_cast<const T*>(p.pre_w);
  const T* bias = static_cast<const T*>(p.pre_b);
  // everything that does not wait for a sum is asked for before the first one
  Pack<T, V> xv[VPT], rv[VPT], wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      get(xv[i], x, v);
      if (res) get(rv[i], res, v);
      if (post) weights(wv[i], post, v);
    }
  }
  float rstd = 1.f;
  if (post) {
    float2 ss = both(0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (threadIdx.x + i * blockDim.x < nvec) {
        float f[V];
        xv[i].widen(f);
        add_squares(ss, f);
      }
    }
    rstd = rsqrtf(row_sum(ss.x + ss.y, red[0]) / static_cast<float>(p.dim) + p.eps);
  }
  float hv[VPT][V];
  float2 stat2 = both(0.f);
  const float factor = rstd * p.scale;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      Pack<T, V> t;
      float f[V], g[V];
      if (post) {                                            // what the branch is multiplied by
        wv[i].widen(f);
        mul_add(f, factor, factor * p.w_bias);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = factor;
      }
      if (gate) {
        weights(t, gate, v);
        t.widen(g);
        mul(f, g);
      }
      xv[i].widen(hv[i]);
      if (res) {
        rv[i].widen(g);
        mul_add(hv[i], f, g);
      } else {
        mul(hv[i], f);
      }
      t.narrow(hv[i]);
      put(t, static_cast<T*>(p.h) + row * p.ldh, v);
      if constexpr (LAYER) {
#pragma unroll
        for (int j = 0; j < V; ++j) stat2.x += hv[i][j];
      } else {
        add_squares(stat2, hv[i]);
      }
    }
  }
  if (pre == nullptr) return;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) weights(wv[i], pre, v);
  }
  float mean = 0.f;
  float stat = row_sum(stat2.x + stat2.y, red[1]) / static_cast<float>(p.dim);
  if constexpr (LAYER) {                    // the variance from the centred row: no cancellation where the mean is large
    mean = stat;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = hv[i][j] - mean;
          if (!SHIFT || static_cast<unsigned>(v * V - o + j) < static_cast<unsigned>(p.dim)) ss += d * d;
        }
      }
    }
    stat = row_sum(ss, red[2]) / static_cast<float>(p.dim);
  }
  rstd = rsqrtf(stat + p.eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      Pack<T, V> t;
      float f[V];
      wv[i].widen(f);
      mul_add(f, rstd, rstd * p.w_bias);
      if constexpr (LAYER) {
#pragma unroll
        for (int j = 0; j < V; ++j) hv[i][j] -= mean;
      }
      if (bias) {
        float g[V];
        weights(t, bias, v);
        t.widen(g);
        mul_add(hv[i], f, g);
      } else {
        mul(hv[i], f);
      }
      t.narrow(hv[i]);
      put(t, static_cast<T*>(p.y) + row * p.ldy, v);
    }
  }
}

template <typename T, int V, bool LAYER, bool SHIFT>
static int launch_branch_norm(const BranchNormParams& p, int rows, cudaStream_t stream) {
  const int nvec = SHIFT ? (p.dim + 2 * V - 2) / V : p.dim / V;
  // Few rows: one access per thread, the shortest way through a row. Many rows: several per thread, so that more rows are on an SM and
  // fewer warps meet at a row's barriers.
  int each = 1;
  const int most = V == 1 ? 8 : 4;
  while (each < most && nvec > 64 * each && rows > 2 * device_sm_count()) each *= 2;
  while (each < 32 / V && nvec > 1024 * each) each *= 2;
  const int threads = ((nvec + each - 1) / each + 31) / 32 * 32;
  if (threads > 1024) return -1;                            // (a shifted row of the greatest length: left to the form by elements)
  auto run = [&](auto kern) { return static_cast<int>(launch_kernel(kern, dim3(rows), dim3(threads), 0, stream, p)); };
  if (each == 1) return run(branch_norm_kernel<T, V, 1, 1024, LAYER, SHIFT>);
#define MX_BRANCH(VPT_)                                                                  \
  if (threads <= 256) return run(branch_norm_kernel<T, V, VPT_, 256, LAYER, SHIFT>);     \
  if (threads <= 512) return run(branch_norm_kernel<T, V, VPT_, 512, LAYER, SHIFT>);     \
  return run(branch_norm_kernel<T, V, VPT_, 1024, LAYER, SHIFT>)
  if (each == 2) { MX_BRANCH(2); }
  if (each == 4) { MX_BRANCH(4); }
  if constexpr (V < 8) {
    if (each == 8) { MX_BRANCH(8); }
  }
#undef MX_BRANCH
  if constexpr (V == 1) {
    if (each == 16) return run(branch_norm_kernel<T, V, 16, 1024, LAYER, SHIFT>);
    return run(branch_norm_kernel<T, V, 32, 1024, LAYER, SHIFT>);
  }
  return -1;
}

template <typename T, int V>
static int choose_branch_norm(const BranchNormParams& p, int rows, bool layer, bool wide, bool shifted, cudaStream_t stream) {
  if (wide) return layer ? launch_branch_norm<T, V, true, false>(p, rows, stream) : launch_branch_norm<T, V, false, false>(p, rows, stream);
  if (shifted) {
    const int rc = layer ? launch_branch_norm<T, V, true, true>(p, rows, stream) : launch_branch_norm<T, V, false, true>(p, rows, stream);
    if (rc != -1) return rc;
  }
  return layer ? launch_branch_norm<T, 1, true, false>(p, rows, stream) : launch_branch_norm<T, 1, false, false>(p, rows, stream);
}

}  // namespace mx

extern "C" int mx_branch_norm(const MxBranchNorm* a, void* stream_) {
  using namespace mx;
  if (a->rows <= 0) return 0;
  if (a->dim <= 0 || a->dim > 32768 || a->x == nullptr || a->h == nullptr || (a->pre_w != nullptr && a->y == nullptr)) return -1;
  const BranchNormParams p{a->x, a->residual, a->post_w, a->gate, a->pre_w, a->pre_b, a->h, a->y, a->ldx, a->ldr, a->ldh, a->ldy, a->dim, a->scale, a->eps, a->w_bias};
  const int rows = a->rows, dim = a->dim, fp32 = a->fp32, layer_norm = a->layer_norm;
  const int v = fp32 ? 4 : 8;
  bool wide = dim % v == 0 && a->ldx % v == 0 && a->ldr % v == 0 && a->ldh % v == 0 && a->ldy % v == 0, shifted = true;
  for (const void* t : {a->post_w, a->gate, a->pre_w, a->pre_b}) shifted = shifted && aligned_to(t, 16);
  wide = wide && shifted;
  const uintptr_t place = reinterpret_cast<uintptr_t>(a->x) % 16;
  auto row_at = [&](const void* t, long long ld) {           // wide: on a boundary; shifted: every row where x's is
    if (t == nullptr) return;
    wide = wide && aligned_to(t, 16);
    shifted = shifted && reinterpret_cast<uintptr_t>(t) % 16 == place && (rows == 1 || (ld - a->ldx) % v == 0);
  };
  row_at(a->x, a->ldx), row_at(a->residual, a->ldr), row_at(a->h, a->ldh), row_at(a->y, a->ldy);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return fp32 ? choose_branch_norm<float, 4>(p, rows, layer_norm != 0, wide, shifted, stream)
              : choose_branch_norm<__nv_bfloat16, 8>(p, rows, layer_norm != 0, wide, shifted, stream);
}
