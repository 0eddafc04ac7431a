// Log probabilities of given tokens with the entropy and the best alternatives of each row (custom call b200.token_log_probs), and
// the gradient of the logits (b200.token_log_probs_grad).
//
//   n = log sum_j e^{x_j},  log_prob = x_t - n (0 for a token outside the vocabulary),  entropy = n - sum_j p_j x_j,  p_j = e^{x_j - n}
//   d x_j = d_log_prob (1[j = t] - p_j) + d_n p_j - d_entropy p_j (x_j - n + entropy)
//
// Bound by memory: the logits are read once (the gradient: once more, and written). Maxima and sums are held in 32 bits: the
// running maximum m, s = sum e^{x - m} and u = sum e^{x - m} (x - m), from which n = m + log s and entropy = log s - u / s, so that
// the entropy is no difference of large numbers. What n loses to its rounding is a result of its own, the remainder: log
// probabilities and the gradient's exponents are (x - n) - remainder, right where the logits are far larger than log s too.
#include <algorithm>

#include "operators.cuh"

namespace b200 {
namespace {

struct Sums {
  float m, s, u;                      // u in units of the logarithm to base 2
};
constexpr float kLowest = -3.4028235e38f;

// Maxima start at the type's lowest value, not at minus infinity, so that differences with them are numbers; a side that has no
// weight at the joint maximum adds nothing, however far below it is.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m), da = (a.m - m) * kLog2e, db = (b.m - m) * kLog2e, fa = power(da), fb = power(db);
  return {m, fa * a.s + fb * b.s, (fa == 0.f ? 0.f : fa * (a.u + a.s * da)) + (fb == 0.f ? 0.f : fb * (b.u + b.s * db))};
}
__device__ __forceinline__ Sums warp_join(Sums v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, {__shfl_xor_sync(0xFFFFFFFFu, v.m, o), __shfl_xor_sync(0xFFFFFFFFu, v.s, o), __shfl_xor_sync(0xFFFFFFFFu, v.u, o)});
  return v;
}

// Order of the alternatives: larger logits first, equal ones by their number; NaN behind every number, -0 like +0.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0u;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// The maximum and the sums of a block, in two steps: the maximum of all first, then everything in its units, so that joining is adding.
// (With a maximum for each thread and sums joined as above, the joins of 4096 x 30522 in 32 bits were a quarter of all instructions.)
template <int WARPS>
__device__ __forceinline__ float block_max(float v, float (&shared)[WARPS]) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[threadIdx.x % WARPS];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
template <int WARPS>
__device__ __forceinline__ void block_sums(float& s, float& u, float2 (&shared)[WARPS]) {
  s = warp_sum(s);
  u = warp_sum(u);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = make_float2(s, u);
  __syncthreads();
  s = shared[threadIdx.x % WARPS].x;
  u = shared[threadIdx.x % WARPS].y;
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
  }
}
// Two logits' share of the sums. The product of no weight and minus infinity is nothing, which the bound sees to; a NaN stays one.
__device__ __forceinline__ void add_weights(uint64_t x, uint64_t minus_max, uint64_t& s, uint64_t& u) {
  const uint64_t y = mul2(add2(x, minus_max), two(kLog2e, kLog2e)), e = two(power(first(y)), power(second(y)));
  s = add2(s, e);
  u = fma2(e, two(fmaxf(first(y), -200.f), fmaxf(second(y), -200.f)), u);
}
// p_j (c - d_entropy (x_j - n + entropy)) of two logits: d = x_j - n' with n = n' + rest, `scaled` -rest log2(e), `minus_dh` -d_entropy,
// `others` c - d_entropy (entropy - rest).
__device__ __forceinline__ uint64_t two_gradients(uint64_t d, uint64_t scaled, uint64_t minus_dh, uint64_t others) {
  const uint64_t y = fma2(d, two(kLog2e, kLog2e), scaled);
  return mul2(two(power(first(y)), power(second(y))), fma2(two(fmaxf(first(d), -200.f), fmaxf(second(d), -200.f)), minus_dh, others));
}

constexpr int kThreads = 256, kWarps = kThreads / 32, kHeld = 32;      // logits that a thread holds
constexpr int kSegment = kThreads * kHeld, kRoom = 1024, kMostTop = 128;
constexpr int kNobody = 0x7FFFFFFF;

struct Rows {
  const void* x;
  const int* tokens;
  float *log_prob, *entropy, *normalizer, *remainder, *top_values;
  int* top_ids;
  Sums* sums;                         // of a row's segments, when there are several
  uint2* best;                        // their `top` best as (order, number)
  int vocab, top, segments;
  long long rows;
};

// The first `top` keys of a block in order, of those that its threads hold: N a thread, `order` with `id` (kNobody: none). Fewer
// where there are fewer. `put(place, order, id)` gets each with its place. The top-th largest of the threads' own maxima is reached by
// `top` keys at least, and for keys in no particular order by hardly more: it is found by a search over the key's bits, two at a time,
// that ends when the number of maxima above is near enough. What reaches it is collected in shared memory and finds its place by
// counting the keys in front of it, so that the result does not depend on the order of collection. More than there is room for (rows
// of few distinct values): the search goes on over all keys, their numbers behind them, to the top-th itself.
struct TopShared {
  unsigned long long key[kRoom];
  int total[64], found;
};
template <int N, typename Order, typename Id, typename Put>
__device__ __forceinline__ void block_top(TopShared& sh, int top, Order&& order, Id&& id, Put&& put) {
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid < 64) sh.total[tid] = 0;
  if (tid == 0) sh.found = 0;
  uint32_t most = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) { const uint32_t v = id(i) == kNobody ? 0u : order(i); most = v > most ? v : most; }
  __syncthreads();
  uint32_t least = 0u;
  for (int b = 30, q = 0; b >= 0; b -= 2, q += 3) {
#pragma unroll
    for (int s = 1; s < 4; ++s) {
      const uint32_t vote = __ballot_sync(0xFFFFFFFFu, most >= (least | ((uint32_t)s << b)));
      if (lane == 0 && vote) atomicAdd(&sh.total[q + s - 1], __popc(vote));
    }
    __syncthreads();
    int reached = kThreads;
#pragma unroll
    for (int s = 3; s > 0; --s)
      if (sh.total[q + s - 1] >= top) { least |= (uint32_t)s << b; reached = sh.total[q + s - 1]; break; }
    if (reached <= top + top / 2 + 8) break;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = id(i);
    if (j != kNobody && order(i) >= least) {
      const int at = atomicAdd(&sh.found, 1);
      if (at < kRoom) sh.key[at] = (unsigned long long)order(i) << 32 | (0xFFFFFFFFu - (unsigned)j);
    }
  }
  __syncthreads();
  int count = sh.found;
  if (count > kRoom) {
    unsigned long long kth = 0;                               // the largest value that `top` keys reach
    for (int b = 63; b >= 0; --b) {
      const unsigned long long trial = kth | (1ull << b);
      __syncthreads();
      if (tid == 0) sh.found = 0;
      __syncthreads();
      int mine = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = id(i);
        mine += j != kNobody && ((unsigned long long)order(i) << 32 | (0xFFFFFFFFu - (unsigned)j)) >= trial ? 1 : 0;
      }
      mine = __reduce_add_sync(0xFFFFFFFFu, mine);
      if (lane == 0 && mine) atomicAdd(&sh.found, mine);
      __syncthreads();
      if (sh.found >= top) kth = trial;
    }
    __syncthreads();
    if (tid == 0) sh.found = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = id(i);
      const unsigned long long key = (unsigned long long)order(i) << 32 | (0xFFFFFFFFu - (unsigned)j);
      if (j != kNobody && key >= kth) sh.key[atomicAdd(&sh.found, 1)] = key;
    }
    __syncthreads();
    count = sh.found;                                         // `top`: no two keys are equal
  }
  for (int c = tid; c < count; c += kThreads) {
    const unsigned long long key = sh.key[c];
    int place = 0;
    for (int o = 0; o < count; ++o) place += sh.key[o] > key ? 1 : 0;
    if (place < top) put(place, (uint32_t)(key >> 32), (int)(0xFFFFFFFFu - (uint32_t)key));
  }
}

template <typename T>
__device__ __forceinline__ void finish_row(const Rows& a, long long row, const Sums& v) {
  // no weight at all: the logarithm of zero
  const float ls = logf(v.s), n = v.s == 0.f ? neg_inf() : v.m + ls;
  const int t = a.tokens[row];
  a.log_prob[row] = t >= 0 && t < a.vocab ? (to_float(((const T*)a.x)[row * a.vocab + t]) - v.m) - ls + (v.s == 0.f ? n - n : 0.f) : 0.f;
  a.entropy[row] = ls - v.u / v.s * kLn2;
  a.normalizer[row] = n;
  a.remainder[row] = (v.m - n) + ls;
}
template <typename T>
__device__ __forceinline__ void finish_best(const Rows& a, long long row, const Sums& v, int place, int j) {
  a.top_values[row * a.top + place] = (to_float(((const T*)a.x)[row * a.vocab + j]) - v.m) - logf(v.s);
  a.top_ids[row * a.top + place] = j;
}

// A block takes a segment of a row, up to 8192 logits, which its threads hold: one pass over memory for the sums and the alternatives.
// Pieces of 16 bytes that lie inside the row are read whole; rows need not begin at such a piece.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) probs_kernel(const __grid_constant__ Rows a) {
  pdl_prologue();
  constexpr int N = Pack<T>::N, NV = kHeld / N;
  __shared__ float maxima[kWarps];
  __shared__ float2 sums[kWarps];
  __shared__ TopShared top;
  const int tid = threadIdx.x, seg = (int)(blockIdx.x % a.segments);
  const long long row = blockIdx.x / a.segments;
  const T* x = (const T*)a.x + row * a.vocab;
  const int off = (int)(((unsigned long long)x / sizeof(T)) % N);     // logits of the row's first piece that belong to the row in front
  const int pieces = (a.vocab + off + N - 1) / N, each = (pieces + a.segments - 1) / a.segments, p0 = seg * each, p1 = min(pieces, p0 + each);
  float f[kHeld];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = p0 + tid + i * kThreads, j = p * N - off;
    float g[N];
    if (p < p1 && j >= 0 && j + N <= a.vocab) {
      unpack<T>(__ldcs((const uint4*)(x + j)), g);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = p < p1 && j + e >= 0 && j + e < a.vocab ? to_float(x[j + e]) : neg_inf();
    }
#pragma unroll
    for (int e = 0; e < N; ++e) f[i * N + e] = g[e];
  }
  Sums v = {kLowest, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kHeld; i += 2) v.m = max3(v.m, f[i], f[i + 1]);
  v.m = block_max(v.m, maxima);
  uint64_t s[2] = {0, 0}, u[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kHeld; i += 2) add_weights(two(f[i], f[i + 1]), two(-v.m, -v.m), s[i / 2 % 2], u[i / 2 % 2]);
  s[0] = add2(s[0], s[1]);
  u[0] = add2(u[0], u[1]);
  v.s = first(s[0]) + second(s[0]);
  v.u = first(u[0]) + second(u[0]);
  block_sums(v.s, v.u, sums);
  const bool whole = a.segments == 1;
  if (tid == 0) {
    if (whole) finish_row<T>(a, row, v);
    else a.sums[blockIdx.x] = v;
  }
  if (TOP) {
    uint2* best = a.best + (long long)blockIdx.x * a.top;
    const int have = max(0, min(a.top, min(a.vocab, p1 * N - off) - max(0, p0 * N - off)));
    if (!whole && tid < a.top && tid >= have) best[tid] = make_uint2(0u, kNobody);
    block_top<kHeld>(top, have, [&](int i) { return order_of(f[i]); },
                     [&](int i) {
                       const int p = p0 + tid + i / N * kThreads, j = p * N - off + i % N;
                       return p < p1 && j >= 0 && j < a.vocab ? j : kNobody;
                     },
                     [&](int place, uint32_t order, int j) {
                       if (whole) finish_best<T>(a, row, v, place, j);
                       else best[place] = make_uint2(order, (unsigned)j);
                     });
  }
}

// Joins the segments of a row, in their order: a block per row where alternatives are wanted, else a warp.
template <typename T>
__device__ __forceinline__ Sums row_sums(const Rows& a, long long row) {
  Sums v = {kLowest, 0.f, 0.f};
  for (int i = threadIdx.x & 31; i < a.segments; i += 32) v = join(v, a.sums[row * a.segments + i]);
  v = warp_join(v);
  // the first lane's for all: the last bit depends on which of two was joined to which, and no alternative's on the thread that has it
  return {__shfl_sync(0xFFFFFFFFu, v.m, 0), __shfl_sync(0xFFFFFFFFu, v.s, 0), __shfl_sync(0xFFFFFFFFu, v.u, 0)};
}
template <typename T>
__global__ void __launch_bounds__(kThreads) probs_join_kernel(const __grid_constant__ Rows a) {
  pdl_prologue();
  const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const Sums v = row_sums<T>(a, row);
  if ((threadIdx.x & 31) == 0) finish_row<T>(a, row, v);
}
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) probs_join_top_kernel(const __grid_constant__ Rows a) {
  pdl_prologue();
  __shared__ TopShared top;
  const long long row = blockIdx.x;
  const Sums v = row_sums<T>(a, row);
  if (threadIdx.x == 0) finish_row<T>(a, row, v);
  uint2 held[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = threadIdx.x + i * kThreads;
    held[i] = c < a.segments * a.top ? a.best[row * a.segments * a.top + c] : make_uint2(0u, kNobody);
  }
  block_top<N>(top, a.top, [&](int i) { return held[i].x; }, [&](int i) { return (int)held[i].y; },
               [&](int place, uint32_t, int j) { finish_best<T>(a, row, v, place, j); });
}

struct Grad {
  const void* x;
  const int* tokens;
  const float *normalizer, *remainder, *entropy, *d_log_prob, *d_entropy, *d_normalizer;
  void* dx;
  int vocab, segments;
};

// The same pieces of the logits and of their gradient, one after another: nothing is held.
template <typename T>
__global__ void __launch_bounds__(kThreads) probs_grad_kernel(const __grid_constant__ Grad a) {
  pdl_prologue();
  constexpr int N = Pack<T>::N, NV = kHeld / N;
  const int tid = threadIdx.x, seg = (int)(blockIdx.x % a.segments);
  const long long row = blockIdx.x / a.segments;
  const T* x = (const T*)a.x + row * a.vocab;
  T* dx = (T*)a.dx + row * a.vocab;
  const int off = (int)(((unsigned long long)x / sizeof(T)) % N);
  const int pieces = (a.vocab + off + N - 1) / N, each = (pieces + a.segments - 1) / a.segments, p0 = seg * each, p1 = min(pieces, p0 + each);
  const int t = a.tokens[row];
  const float n = a.normalizer[row], low = a.remainder[row], h = a.entropy[row], dh = a.d_entropy[row], dl = t >= 0 && t < a.vocab ? a.d_log_prob[row] : 0.f;
  const float c = a.d_normalizer[row] - dl;
  const uint64_t minus_n = two(-n, -n), scaled = two(-low * kLog2e, -low * kLog2e), minus_dh = two(-dh, -dh), others = two(c - dh * (h - low), c - dh * (h - low));
  uint4 held[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = p0 + tid + i * kThreads, j = p * N - off;
    if (p < p1 && j >= 0 && j + N <= a.vocab) held[i] = __ldcs((const uint4*)(x + j));
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = p0 + tid + i * kThreads, j = p * N - off;
    if (p >= p1) break;
    if (j >= 0 && j + N <= a.vocab) {
      float f[N];
      unpack<T>(held[i], f);
      uint4 out;
      T* o = reinterpret_cast<T*>(&out);
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const uint64_t d = two_gradients(add2(two(f[e], f[e + 1]), minus_n), scaled, minus_dh, others);
        f[e] = first(d);
        f[e + 1] = second(d);
      }
      if ((unsigned)t - (unsigned)j < N) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] += j + e == t ? dl : 0.f;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = from_float<T>(f[e]);
      *(uint4*)(dx + j) = out;
    } else {
      for (int e = 0; e < N; ++e)
        if (j + e >= 0 && j + e < a.vocab)
          dx[j + e] = from_float<T>(first(two_gradients(add2(two(to_float(x[j + e]), 0.f), minus_n), scaled, minus_dh, others)) + (j + e == t ? dl : 0.f));
    }
  }
}

// Both at once where the cotangents do not depend on the results: a block has a whole row in its registers, eight pieces of 16 bytes a
// thread, takes the sums of it and writes the gradient, while the next row is on its way to shared memory, each thread's pieces to its
// own place, so that no thread waits for another's. Bound by memory: the logits are read once and the gradient is written (4096 x 30522
// in 32 bits 264 us by the two kernels above, 190 to 201 so, 153 at the rate of a copy; in bf16 128 and 76; 8141 x 8446 in 32 bits 130
// and 84). Blocks of 1024 threads for all rows, of which an SM has room for one, took 178 and 236 us for the last two.
constexpr int kRowThreads = 1024, kRowPieces = 8;

struct Both {
  Rows rows;
  Grad grad;
};
__device__ __forceinline__ void fetch16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, kRowThreads / THREADS) probs_both_kernel(const __grid_constant__ Both a) {
  pdl_prologue();
  constexpr int N = Pack<T>::N, W = THREADS / 32;
  extern __shared__ __align__(16) uint8_t ahead[];
  __shared__ float maxima[W];
  __shared__ float2 sums[W];
  const int tid = threadIdx.x, vocab = a.rows.vocab;
  const uint32_t mine = smem_u32(ahead) + tid * 16;
  auto offset = [&](const T* x) { return (int)(((unsigned long long)x / sizeof(T)) % N); };
  auto inside = [&](int j) { return (unsigned)j <= (unsigned)(vocab - N); };
  // 16-bit data: pieces at a row's ends, which hold logits of its neighbours as well, are fetched whole and what is not the row's goes, but
  // for those at the ends of the logits themselves. (Read one by one, 4096 x 30522 in bf16 267 us instead of 178, with 1024 threads a block; 32-bit data so 206 instead of 197.)
  auto whole = [&](long long row, int j) {
    return N == 4 ? inside(j) : j >= (row == 0 ? 0 : 1 - N) && j <= (row == a.rows.rows - 1 ? vocab - N : vocab - 1);
  };
  auto fetch = [&](long long row) {
    if (row < a.rows.rows) {
      const T* x = (const T*)a.rows.x + row * vocab;
      const int off = offset(x);
#pragma unroll
      for (int i = 0; i < kRowPieces; ++i) {
        const int j = (tid + i * THREADS) * N - off;
        if (whole(row, j)) fetch16(mine + i * THREADS * 16, x + j);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(blockIdx.x);
  for (long long row = blockIdx.x; row < a.rows.rows; row += gridDim.x) {
    const T* x = (const T*)a.rows.x + row * vocab;
    const int off = offset(x);
    const int t = a.rows.tokens[row];
    const float dh = a.grad.d_entropy[row], dn = a.grad.d_normalizer[row], dl = t >= 0 && t < vocab ? a.grad.d_log_prob[row] : 0.f;
    const float at_token = t >= 0 && t < vocab ? to_float(x[t]) : 0.f;
    uint4 held[kRowPieces];
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i) {
      const int j = (tid + i * THREADS) * N - off;
      if (inside(j)) {
        held[i] = *(const uint4*)(ahead + (tid + i * THREADS) * 16);
      } else {
        T e[N];
        const bool fetched = N == 8 && whole(row, j);
        if (fetched) *reinterpret_cast<uint4*>(e) = *(const uint4*)(ahead + (tid + i * THREADS) * 16);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if (j + k < 0 || j + k >= vocab) e[k] = from_float<T>(neg_inf());
          else if (!fetched) e[k] = x[j + k];
        }
        held[i] = *reinterpret_cast<const uint4*>(e);
      }
    }
    fetch(row + gridDim.x);
    Sums v = {kLowest, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i) {
      if (N == 8 && i * THREADS * N >= vocab + off) break;        // (rows leave up to half of the pieces empty)
      float f[N];
      unpack<T>(held[i], f);
#pragma unroll
      for (int k = 0; k < N; k += 2) v.m = max3(v.m, f[k], f[k + 1]);
    }
    v.m = block_max(v.m, maxima);                                     // (a barrier between any two uses of `maxima` and of `sums`)
    const uint64_t minus_max = two(-v.m, -v.m);
    uint64_t s[2] = {0, 0}, u[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i) {
      if (N == 8 && i * THREADS * N >= vocab + off) break;
      float f[N];
      unpack<T>(held[i], f);
#pragma unroll
      for (int k = 0; k < N; k += 2) add_weights(two(f[k], f[k + 1]), minus_max, s[k / 2 % 2], u[k / 2 % 2]);
    }
    s[0] = add2(s[0], s[1]);
    u[0] = add2(u[0], u[1]);
    v.s = first(s[0]) + second(s[0]);
    v.u = first(u[0]) + second(u[0]);
    block_sums(v.s, v.u, sums);
    const float ls = logf(v.s), n = v.s == 0.f ? neg_inf() : v.m + ls, low = (v.m - n) + ls, h = ls - v.u / v.s * kLn2;
    if (tid == 0) {
      a.rows.log_prob[row] = t >= 0 && t < vocab ? (at_token - v.m) - ls + (v.s == 0.f ? n - n : 0.f) : 0.f;
      a.rows.entropy[row] = h;
      a.rows.normalizer[row] = n;
      a.rows.remainder[row] = low;
    }
    const float c = dn - dl;
    const uint64_t scaled = two(-ls * kLog2e, -ls * kLog2e), minus_dh = two(-dh, -dh), others = two(c - dh * (h - ls), c - dh * (h - ls));
    T* dx = (T*)a.grad.dx + row * vocab;
#pragma unroll
    for (int i = 0; i < kRowPieces; ++i) {
      const int j = (tid + i * THREADS) * N - off;
      if (j >= vocab) break;
      float f[N];
      unpack<T>(held[i], f);
      uint4 out;
      T* o = reinterpret_cast<T*>(&out);
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        const uint64_t d = two_gradients(add2(two(f[k], f[k + 1]), minus_max), scaled, minus_dh, others);
        f[k] = first(d);
        f[k + 1] = second(d);
      }
      if ((unsigned)t - (unsigned)j < N) {
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] += j + k == t ? dl : 0.f;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) o[k] = from_float<T>(f[k]);
      if (inside(j)) {
        __stcs((uint4*)(dx + j), out);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (j + k >= 0 && j + k < vocab) dx[j + k] = o[k];
      }
    }
  }
}

constexpr int kJoined = 64 * kThreads;                        // alternatives of a row's segments that the block that joins them holds

// Segments of a row: as few as hold it (a first piece that starts in front of the row counts), and more for few rows, down to 2048
// logits, so that the blocks fill the chip, as long as their alternatives can be joined.
int segments_of(const OperatorLaunch& op) {
  const long long least = ((long long)op.vocab + 8 + kSegment - 1) / kSegment;
  const long long most = std::max<long long>(least, std::min<long long>(op.vocab / 2048, op.top ? kJoined / op.top : op.vocab));
  return (int)std::max<long long>(least, std::min<long long>(most, 2 * kSMs / std::max<long long>(1, op.rows)));
}

template <typename T>
cudaError_t launch_rows(const Rows& a, cudaStream_t stream, int* launches) {
  const dim3 grid((unsigned)(a.rows * a.segments));
  if (cudaError_t e = a.top ? launch_op(probs_kernel<T, true>, grid, kThreads, 0, stream, launches, a) : launch_op(probs_kernel<T, false>, grid, kThreads, 0, stream, launches, a))
    return e;
  if (a.segments == 1) return cudaSuccess;
  if (!a.top) return launch_op(probs_join_kernel<T>, dim3((unsigned)((a.rows + kWarps - 1) / kWarps)), kThreads, 0, stream, launches, a);
  const int each = (a.segments * a.top + kThreads - 1) / kThreads;
  if (each <= 4) return launch_op(probs_join_top_kernel<T, 4>, dim3((unsigned)a.rows), kThreads, 0, stream, launches, a);
  if (each <= 16) return launch_op(probs_join_top_kernel<T, 16>, dim3((unsigned)a.rows), kThreads, 0, stream, launches, a);
  return launch_op(probs_join_top_kernel<T, 64>, dim3((unsigned)a.rows), kThreads, 0, stream, launches, a);
}
template <typename T>
cudaError_t launch_grad(const Grad& a, long long rows, cudaStream_t stream, int* launches) {
  return launch_op(probs_grad_kernel<T>, dim3((unsigned)(rows * a.segments)), kThreads, 0, stream, launches, a);
}

long long row_bytes(const OperatorLaunch& op) { return (long long)op.vocab * (op.type == 0 ? 4 : 2) + 32; }      // with what its ends may share

template <typename T, int THREADS>
cudaError_t launch_both(const Both& a, cudaStream_t stream, int* launches) {
  static bool done[64] = {};
  constexpr size_t smem = (size_t)THREADS * kRowPieces * 16;
  if (cudaError_t e = allow_smem(probs_both_kernel<T, THREADS>, smem, done)) return e;
  const dim3 grid((unsigned)std::min<long long>(a.rows.rows, kSMs * (kRowThreads / THREADS)));
  return launch_op(probs_both_kernel<T, THREADS>, grid, THREADS, smem, stream, launches, a);
}
template <typename T>
cudaError_t launch_both(const OperatorLaunch& op, const Both& a, cudaStream_t stream, int* launches) {
  // the smallest blocks that hold a row: the more of them an SM has, the more of a row's waits another's arithmetic fills
  const long long bytes = row_bytes(op), each = kRowPieces * 16;
  if (bytes <= 256 * each) return launch_both<T, 256>(a, stream, launches);
  if (bytes <= 512 * each) return launch_both<T, 512>(a, stream, launches);
  return launch_both<T, kRowThreads>(a, stream, launches);
}

Rows rows_of(const OperatorLaunch& op, void* const* results, void* const* operands) {
  Rows a = {};
  a.log_prob = (float*)results[0];
  a.entropy = (float*)results[1];
  a.normalizer = (float*)results[2];
  a.remainder = (float*)results[3];
  a.x = operands[0];
  a.tokens = (const int*)operands[1];
  a.vocab = op.vocab;
  a.rows = op.rows;
  return a;
}

}  // namespace

// Rows that a block's registers hold and that give each thread something, and enough of them for every SM to have two.
bool token_log_probs_at_once(const OperatorLaunch& op) {
  const long long bytes = row_bytes(op);
  return op.top == 0 && op.rows >= 2 * kSMs && bytes - 32 >= kRowThreads * 16 && bytes <= kRowThreads * kRowPieces * 16LL;
}

const char* token_log_probs_plan(OperatorLaunch& op) {
  if (op.vocab > (1 << 30)) return "a vocabulary of more than 2^30";
  if (op.kind == OperatorLaunch::TOKEN_LOG_PROBS_BOTH) {
    op.launches = 1;
    return op.rows < (1LL << 31) && token_log_probs_at_once(op) ? nullptr : "internal: rows that do not fit";
  }
  const bool grad = op.kind == OperatorLaunch::TOKEN_LOG_PROBS_GRAD;
  int s = segments_of(op);
  if (op.top && (long long)s * op.top > kJoined) return "more alternatives than this vocabulary's segments leave room for";
  if (op.rows * s >= (1LL << 31)) return "too many logits";
  const bool several = !grad && s > 1;
  op.scratch_bytes = several ? op.rows * s * (12 + 8LL * op.top) + 16 : 0;
  op.launches = several ? 2 : 1;
  return nullptr;
}

cudaError_t launch_token_log_probs(const OperatorLaunch& op, void* const* args, void* scratch, cudaStream_t stream, int* launches) {
  Rows a = rows_of(op, args, args + (op.top ? 6 : 4));
  if (op.top) { a.top_values = (float*)args[4]; a.top_ids = (int*)args[5]; }
  a.top = op.top;
  a.segments = segments_of(op);
  a.best = (uint2*)scratch;
  a.sums = (Sums*)((char*)scratch + op.rows * a.segments * 8LL * op.top);
  if (op.type == 0) return launch_rows<float>(a, stream, launches);
  if (op.type == 1) return launch_rows<__nv_bfloat16>(a, stream, launches);
  return launch_rows<__half>(a, stream, launches);
}

cudaError_t launch_token_log_probs_grad(const OperatorLaunch& op, void* const* args, cudaStream_t stream, int* launches) {
  Grad a = {};
  a.dx = args[0];
  a.x = args[1];
  a.tokens = (const int*)args[2];
  a.normalizer = (const float*)args[3];
  a.remainder = (const float*)args[4];
  a.entropy = (const float*)args[5];
  a.d_log_prob = (const float*)args[6];
  a.d_entropy = (const float*)args[7];
  a.d_normalizer = (const float*)args[8];
  a.vocab = op.vocab;
  a.segments = segments_of(op);
  if (op.type == 0) return launch_grad<float>(a, op.rows, stream, launches);
  if (op.type == 1) return launch_grad<__nv_bfloat16>(a, op.rows, stream, launches);
  return launch_grad<__half>(a, op.rows, stream, launches);
}

cudaError_t launch_token_log_probs_both(const OperatorLaunch& op, void* const* args, cudaStream_t stream, int* launches) {
  Both a = {};
  a.rows = rows_of(op, args, args + 5);
  a.grad.dx = args[4];
  a.grad.d_log_prob = (const float*)args[7];
  a.grad.d_entropy = (const float*)args[8];
  a.grad.d_normalizer = (const float*)args[9];
  if (op.type == 0) return launch_both<float>(op, a, stream, launches);
  if (op.type == 1) return launch_both<__nv_bfloat16>(op, a, stream, launches);
  return launch_both<__half>(op, a, stream, launches);
}

}  // namespace b200
