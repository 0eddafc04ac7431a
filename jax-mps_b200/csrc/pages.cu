// Moves inside a cache of pages, [layers, 2, pages, page, kv_heads, dim]: rows of new tokens to their slots, pages to other pages.
// All layers and both of keys and values go in one launch. The indices travel as kernel parameters (host memory, read when the
// launch is issued), so that no copy to the device goes in front.
//
// Bound by memory: every byte that moves is read and written once, in pieces of 16 bytes, four in flight for a thread.
#include <algorithm>

#include "operators.cuh"

namespace b200 {
namespace {

// Indices of a launch: its parameters may be 32 KB, but the host copies them for every one.
constexpr int kFew = 240, kMany = 7680;

template <int N>
struct Moves {
  int index[N];
};

// `count` runs of `pieces` pieces of 16 bytes for each plane (blockIdx.y): a thread moves four of them, 256 apart. `ends` gives where a
// run's first piece comes from and goes to, or false.
template <typename F>
__device__ __forceinline__ void move_runs(int count, unsigned pieces, F&& ends) {
  const unsigned total = (unsigned)count * pieces, first = blockIdx.x * 1024u + threadIdx.x;
  uint4 v[4];
  uint4* to[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const unsigned at = first + 256u * u;
    to[u] = nullptr;
    if (at >= total) continue;
    const unsigned run = at / pieces, piece = at - run * pieces;
    const uint4* from;
    uint4* dst;
    if (!ends(run, from, dst)) continue;
    v[u] = from[piece];
    to[u] = dst + piece;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) if (to[u]) *to[u] = v[u];
}

template <int N>
__global__ void __launch_bounds__(256) write_pages_kernel(const __grid_constant__ Moves<N> m, int count, void* cache, const void* rows, long long first,
                                                          long long n, long long slots, unsigned pieces) {
  pdl_prologue();
  move_runs(count, pieces, [&](unsigned run, const uint4*& from, uint4*& to) {
    const int slot = m.index[run];
    if (slot < 0) return false;
    from = (const uint4*)rows + ((long long)blockIdx.y * n + first + run) * pieces;
    to = (uint4*)cache + ((long long)blockIdx.y * slots + slot) * pieces;
    return true;
  });
}

// Pairs of a source and a destination; a source of -1 - i is page i of the stage.
template <int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ Moves<N> m, int count, void* cache, const void* stage, long long staged,
                                                         long long pages, unsigned pieces) {
  pdl_prologue();
  move_runs(count, pieces, [&](unsigned run, const uint4*& from, uint4*& to) {
    const int src = m.index[2 * run], dst = m.index[2 * run + 1];
    from = src >= 0 ? (const uint4*)cache + ((long long)blockIdx.y * pages + src) * pieces
                    : (const uint4*)stage + ((long long)blockIdx.y * staged - 1 - src) * pieces;
    to = (uint4*)cache + ((long long)blockIdx.y * pages + dst) * pieces;
    return true;
  });
}

template <int N>
__global__ void __launch_bounds__(256) stage_pages_kernel(const __grid_constant__ Moves<N> m, int count, const void* cache, void* stage, long long first,
                                                          long long n, long long pages, unsigned pieces) {
  pdl_prologue();
  move_runs(count, pieces, [&](unsigned run, const uint4*& from, uint4*& to) {
    from = (const uint4*)cache + ((long long)blockIdx.y * pages + m.index[run]) * pieces;
    to = (uint4*)stage + ((long long)blockIdx.y * n + first + run) * pieces;
    return true;
  });
}

// Blocks for the runs of one launch: every thread moves four pieces. (Eight blocks an SM that go round: 472 MB of pages 87 us instead of 73.)
dim3 grid_for(const CacheShape& c, long long runs, long long pieces) { return dim3((unsigned)((runs * pieces + 1023) / 1024), (unsigned)c.planes); }

// Launches for `n` runs, whose indices (`each` a run) `fill` writes; as many of them at a time as have room and as 32 bits of pieces count.
template <typename Fill, typename Launch>
cudaError_t in_pieces(long long n, int each, long long pieces, Fill&& fill, Launch&& launch) {
  const long long most = std::max<long long>(1, (1LL << 30) / pieces);
  for (long long at = 0; at < n;) {
    const int count = (int)std::min(std::min<long long>(n - at, most), (long long)(n - at <= kFew / each ? kFew / each : kMany / each));
    if (count <= kFew / each) {
      Moves<kFew> m;
      fill(m.index, at, count);
      if (cudaError_t e = launch(m, at, count)) return e;
    } else {
      Moves<kMany> m;
      fill(m.index, at, count);
      if (cudaError_t e = launch(m, at, count)) return e;
    }
    at += count;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_write_pages(const CacheShape& c, void* cache, const void* rows, const int* slots, long long n, cudaStream_t stream, int* launches) {
  const long long pieces = c.token / 16;
  return in_pieces(n, 1, pieces, [&](int* to, long long at, int count) { std::copy(slots + at, slots + at + count, to); },
                   [&](auto& m, long long at, int count) {
                     constexpr int N = sizeof(m.index) / sizeof(int);
                     return launch_op(write_pages_kernel<N>, grid_for(c, count, pieces), 256, 0, stream, launches, m, count, cache, rows, at, n, c.pages * c.page,
                                      (unsigned)pieces);
                   });
}

cudaError_t launch_copy_pages(const CacheShape& c, void* cache, const int* pairs, const int* staged, const void* stage, long long n, cudaStream_t stream,
                              int* launches) {
  const long long pieces = c.page * c.token / 16;
  long long in_stage = 0;
  for (long long i = 0; i < n; i++) in_stage = std::max<long long>(in_stage, staged[i] + 1);
  return in_pieces(n, 2, pieces,
                   [&](int* to, long long at, int count) {
                     for (int i = 0; i < count; i++) {
                       to[2 * i] = staged[at + i] >= 0 ? -1 - staged[at + i] : pairs[2 * (at + i)];
                       to[2 * i + 1] = pairs[2 * (at + i) + 1];
                     }
                   },
                   [&](auto& m, long long, int count) {
                     constexpr int N = sizeof(m.index) / sizeof(int);
                     return launch_op(copy_pages_kernel<N>, grid_for(c, count, pieces), 256, 0, stream, launches, m, count, cache, stage, in_stage, c.pages,
                                      (unsigned)pieces);
                   });
}

cudaError_t launch_stage_pages(const CacheShape& c, const void* cache, void* stage, const int* sources, long long n, cudaStream_t stream, int* launches) {
  const long long pieces = c.page * c.token / 16;
  return in_pieces(n, 1, pieces, [&](int* to, long long at, int count) { std::copy(sources + at, sources + at + count, to); },
                   [&](auto& m, long long at, int count) {
                     constexpr int N = sizeof(m.index) / sizeof(int);
                     return launch_op(stage_pages_kernel<N>, grid_for(c, count, pieces), 256, 0, stream, launches, m, count, cache, stage, at, n, c.pages,
                                      (unsigned)pieces);
                   });
}

}  // namespace b200
