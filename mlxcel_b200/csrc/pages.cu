// Pages of a cache on the move. A page id addresses the same slot of every slab (one slab per layer and for keys, values, ...), so a
// page's content is one run of bytes in each of them; all of it moves in one launch.
//
//   copy     page dst[i] <- page src[i], all sources as they were before the call. Pages that are read and written are put in order by
//            the caller (`starts` cuts the pairs into chains): a thread owns the same bytes of every page of a chain and moves them pair
//            after pair, so no other thread's store can come before its load. A chain may end in a cycle, whose first page is held in
//            registers until the last pair.
//   gather   buffer[slab][i] <- page ids[i];   scatter   page ids[i] <- buffer[slab][i]
//
// Bound by memory (two bytes moved per byte of a page); small calls by the launch, so ids of small calls travel in the parameters.
#include "api.h"
#include "common.cuh"
#include "typed.cuh"

namespace mx {

constexpr int kPageSlabs = 128;            // of one launch
constexpr int kPageInline = 320;           // ints of the table that fit into the parameters
constexpr int kPageThreads = 256;
constexpr int kPageUnits = 4;              // accesses of a thread in flight

enum { kPagesCopy = 0, kPagesGather = 1, kPagesScatter = 2 };

struct PagesParams {
  char* base[kPageSlabs];
  uint32_t bytes[kPageSlabs];              // of a page in this slab
  uint32_t first[kPageSlabs];              // bytes of one page in the slabs before it (buffer)
  char* buffer;
  const int* far;                          // the table in device memory, where it does not fit here
  int n;                                   // pages
  int table[kPageInline];                  // copy: n pairs (src, dst), then the chains' starts; else the ids
};

template <int JOB, typename U>
__global__ void __launch_bounds__(kPageThreads) pages_kernel(const __grid_constant__ PagesParams p) {
  pdl_trigger();
  pdl_wait();
  const int slab = blockIdx.y;
  const uint32_t units = p.bytes[slab] / sizeof(U);
  const int* table = p.far ? p.far : p.table;
  U* base = reinterpret_cast<U*>(p.base[slab]);
  auto page = [&](int id) { return base + static_cast<size_t>(id) * units; };
  for (uint32_t u0 = blockIdx.z * (kPageThreads * kPageUnits) + threadIdx.x; u0 < units; u0 += gridDim.z * (kPageThreads * kPageUnits)) {
    U r[kPageUnits];
    auto load = [&](const U* from) {
#pragma unroll
      for (int i = 0; i < kPageUnits; ++i)
        if (u0 + i * kPageThreads < units) r[i] = from[u0 + i * kPageThreads];
    };
    auto store = [&](U* to) {
#pragma unroll
      for (int i = 0; i < kPageUnits; ++i)
        if (u0 + i * kPageThreads < units) to[u0 + i * kPageThreads] = r[i];
    };
    if constexpr (JOB == kPagesCopy) {
      const int a = table[2 * p.n + blockIdx.x], b = table[2 * p.n + blockIdx.x + 1];
      int c = b;                                       // the cycle's first pair, if the chain ends in one
      if (b - a > 1) {
        for (c = a; c < b && table[2 * c + 1] != table[2 * (b - 1)]; ++c) {}
      }
      U held[kPageUnits];
      for (int i = a; i < b; ++i) {
        if (i == c) {
          load(page(table[2 * i + 1]));
#pragma unroll
          for (int j = 0; j < kPageUnits; ++j) held[j] = r[j];
        }
        if (i == b - 1 && c < b) {
#pragma unroll
          for (int j = 0; j < kPageUnits; ++j) r[j] = held[j];
        } else {
          load(page(table[2 * i]));
        }
        store(page(table[2 * i + 1]));
      }
    } else {
      U* flat = reinterpret_cast<U*>(p.buffer + static_cast<size_t>(p.first[slab]) * p.n) + static_cast<size_t>(blockIdx.x) * units;
      U* mine = page(table[blockIdx.x]);
      load(JOB == kPagesGather ? mine : flat);
      store(JOB == kPagesGather ? flat : mine);
    }
  }
}

template <int JOB>
static cudaError_t launch_pages(const PagesParams& p, int unit, dim3 grid, cudaStream_t stream) {
  switch (unit) {
    case 16: return launch_kernel(pages_kernel<JOB, uint4>, grid, dim3(kPageThreads), 0, stream, p);
    case 4: return launch_kernel(pages_kernel<JOB, uint32_t>, grid, dim3(kPageThreads), 0, stream, p);
    default: return launch_kernel(pages_kernel<JOB, uint8_t>, grid, dim3(kPageThreads), 0, stream, p);
  }
}

}  // namespace mx

extern "C" int mx_pages_inline_ints(void) { return mx::kPageInline; }

extern "C" int mx_pages(int job, const void* const* base, const long long* bytes, int n_slabs, void* buffer, const int* table,
                        const int* table_dev, int ints, int n, int chains, void* stream_) {
  using namespace mx;
  if (n <= 0 || n_slabs <= 0) return 0;
  if (job < 0 || job > 2 || (job != kPagesCopy && buffer == nullptr) || (job == kPagesCopy && chains <= 0)) return -1;
  if (ints > kPageInline ? table_dev == nullptr : table == nullptr) return -1;
  PagesParams p{};
  p.buffer = static_cast<char*>(buffer);
  p.n = n;
  if (ints > kPageInline) p.far = table_dev;
  else for (int i = 0; i < ints; ++i) p.table[i] = table[i];
  int unit = aligned_to(buffer, 16) ? 16 : (aligned_to(buffer, 4) ? 4 : 1);
  long long before = 0;
  for (int s = 0; s < n_slabs; ++s) {                       // the widest access that suits every slab
    if (bytes[s] < 0 || bytes[s] > 0x7fffffffll) return -1;
    while (bytes[s] % unit || !aligned_to(base[s], unit)) unit = unit == 16 ? 4 : 1;
    before += bytes[s];
  }
  if (before > 0xffffffffll) return -1;
  const long long per_block = static_cast<long long>(kPageThreads) * kPageUnits * unit;
  before = 0;
  for (int s0 = 0; s0 < n_slabs; s0 += kPageSlabs) {
    const int count = n_slabs - s0 < kPageSlabs ? n_slabs - s0 : kPageSlabs;
    long long most = 0;
    for (int s = 0; s < count; ++s) {
      p.base[s] = static_cast<char*>(const_cast<void*>(base[s0 + s]));
      p.bytes[s] = static_cast<uint32_t>(bytes[s0 + s]);
      p.first[s] = static_cast<uint32_t>(before);
      before += bytes[s0 + s];
      most = bytes[s0 + s] > most ? bytes[s0 + s] : most;
    }
    const long long z = (most + per_block - 1) / per_block;
    if (z == 0) continue;
    const dim3 grid(job == kPagesCopy ? chains : n, count, static_cast<unsigned>(z < 65535 ? z : 65535));
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const cudaError_t e = job == kPagesCopy ? launch_pages<kPagesCopy>(p, unit, grid, stream)
                          : job == kPagesGather ? launch_pages<kPagesGather>(p, unit, grid, stream)
                                                : launch_pages<kPagesScatter>(p, unit, grid, stream);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
}
