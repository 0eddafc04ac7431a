// Moves inside a cache of pages, [layers, 2, pages, page, kv_heads, dim]: rows of new tokens to their slots, pages to other pages.
// All layers and both of keys and values go in one launch. The indices travel as kernel parameters (host memory, read when the
// launch is issued), so that no copy to the device goes in front.
//
// Bound by memory: every byte that moves is read and written once, in pieces of 16 bytes, four in flight for a thread.
#include <algorithm>

#include "operators.cuh"

namespace b200 {
namespace {

// Parameters of a launch are at most 4 KB here: longer lists go in several launches.
constexpr int kIndices = 960;

struct Moves {
  int index[kIndices];
};

// A block moves `run` pieces of 16 bytes; the pieces of a plane and an index are `pieces`. blockIdx.y: index, blockIdx.z: plane.
template <typename F>
__device__ __forceinline__ void move_run(F&& ends, long long pieces) {
  const uint4* from;
  uint4* to;
  if (!ends(from, to)) return;
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < pieces; i += 4 * step) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) if (i + u * step < pieces) v[u] = from[i + u * step];
#pragma unroll
    for (int u = 0; u < 4; ++u) if (i + u * step < pieces) to[i + u * step] = v[u];
  }
}

__global__ void __launch_bounds__(128) write_pages_kernel(const __grid_constant__ Moves m, void* cache, const void* rows, long long first, long long n,
                                                          long long slots, long long pieces) {
  pdl_prologue();
  move_run([&](const uint4*& from, uint4*& to) {
    const int slot = m.index[blockIdx.y];
    if (slot < 0) return false;
    from = (const uint4*)rows + ((long long)blockIdx.z * n + first + blockIdx.y) * pieces;
    to = (uint4*)cache + ((long long)blockIdx.z * slots + slot) * pieces;
    return true;
  }, pieces);
}

// Pairs of a source and a destination; a source of -1 - i is page i of the stage.
__global__ void __launch_bounds__(128) copy_pages_kernel(const __grid_constant__ Moves m, void* cache, const void* stage, long long staged,
                                                         long long pages, long long pieces) {
  pdl_prologue();
  move_run([&](const uint4*& from, uint4*& to) {
    const int src = m.index[2 * blockIdx.y], dst = m.index[2 * blockIdx.y + 1];
    from = src >= 0 ? (const uint4*)cache + ((long long)blockIdx.z * pages + src) * pieces
                    : (const uint4*)stage + ((long long)blockIdx.z * staged - 1 - src) * pieces;
    to = (uint4*)cache + ((long long)blockIdx.z * pages + dst) * pieces;
    return true;
  }, pieces);
}

__global__ void __launch_bounds__(128) stage_pages_kernel(const __grid_constant__ Moves m, const void* cache, void* stage, long long first, long long n,
                                                          long long pages, long long pieces) {
  pdl_prologue();
  move_run([&](const uint4*& from, uint4*& to) {
    from = (const uint4*)cache + ((long long)blockIdx.z * pages + m.index[blockIdx.y]) * pieces;
    to = (uint4*)stage + ((long long)blockIdx.z * n + first + blockIdx.y) * pieces;
    return true;
  }, pieces);
}

unsigned blocks_for(long long pieces) { return (unsigned)std::max<long long>(1, std::min<long long>(1024, (pieces + 511) / 512)); }

}  // namespace

cudaError_t launch_write_pages(const CacheShape& c, void* cache, const void* rows, const int* slots, long long n, cudaStream_t stream, int* launches) {
  const long long pieces = c.token / 16;
  for (long long at = 0; at < n; at += kIndices) {
    const int count = (int)std::min<long long>(kIndices, n - at);
    Moves m;
    std::copy(slots + at, slots + at + count, m.index);
    if (cudaError_t e = launch_op(write_pages_kernel, dim3(blocks_for(pieces), (unsigned)count, (unsigned)c.planes), 128, 0, stream, launches, m, cache, rows, at, n,
                                  c.pages * c.page, pieces))
      return e;
  }
  return cudaSuccess;
}

cudaError_t launch_copy_pages(const CacheShape& c, void* cache, const int* pairs, const int* staged, const void* stage, long long n, cudaStream_t stream,
                              int* launches) {
  const long long pieces = c.page * c.token / 16;
  long long in_stage = 0;
  for (long long i = 0; staged && i < n; i++) in_stage = std::max<long long>(in_stage, staged[i] + 1);
  for (long long at = 0; at < n; at += kIndices / 2) {
    const int count = (int)std::min<long long>(kIndices / 2, n - at);
    Moves m;
    for (int i = 0; i < count; i++) {
      m.index[2 * i] = staged && staged[at + i] >= 0 ? -1 - staged[at + i] : pairs[2 * (at + i)];
      m.index[2 * i + 1] = pairs[2 * (at + i) + 1];
    }
    if (cudaError_t e = launch_op(copy_pages_kernel, dim3(blocks_for(pieces), (unsigned)count, (unsigned)c.planes), 128, 0, stream, launches, m, cache, stage,
                                  in_stage, c.pages, pieces))
      return e;
  }
  return cudaSuccess;
}

cudaError_t launch_stage_pages(const CacheShape& c, const void* cache, void* stage, const int* sources, long long n, cudaStream_t stream, int* launches) {
  const long long pieces = c.page * c.token / 16;
  for (long long at = 0; at < n; at += kIndices) {
    const int count = (int)std::min<long long>(kIndices, n - at);
    Moves m;
    std::copy(sources + at, sources + at + count, m.index);
    if (cudaError_t e = launch_op(stage_pages_kernel, dim3(blocks_for(pieces), (unsigned)count, (unsigned)c.planes), 128, 0, stream, launches, m, cache, stage, at, n,
                                  c.pages, pieces))
      return e;
  }
  return cudaSuccess;
}

}  // namespace b200
