// Causal attention of whole prompts with an optional sliding window and sinks (custom call b200.window_attention).
//
//   out[b, i, h] = sum_j w_j v_j,  w = softmax_j(scale * q[b, i, h] . k[b, j, h / group])  over j <= i with no window, i - j < window
//   or j < sinks; rows from a sequence's length on are zero.
//
// Sums, maxima and normalisers are held in 32 bits; tiles of keys that no row of a tile of queries sees are not read.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "operators.cuh"

namespace b200 {
namespace {

struct Prompt {
  const void *q, *k, *v;
  const int* lengths;                 // null: all of them are `tokens`
  void* out;
  int batch, tokens, heads, kv_heads, dim, group, window, sinks;
  float scale;                        // of the scores, times log2(e)
  // tensor cores: whether a block's two tiles of queries are two heads (else two tiles of one), units of heads and of queries, all units
  int pairs, head_units, query_units, units;
};

__device__ __forceinline__ int length_of(const Prompt& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.tokens) : a.tokens;
}

// Whether a position is seen; the keys' and values' sums run over these.
__device__ __forceinline__ bool sees(const Prompt& a, int row, int key) {
  return key <= row && (a.window == 0 || row - key < a.window || key < a.sinks);
}

// The kernels multiply whole tiles of values by weights that are zero where a row does not look, and zero times an infinity or a NaN is
// none. They notice by a result that is no finite number, and then this has another look at such rows, a warp at each: where a value
// that the row does not see, but that lay in a tile with what it does, is no finite number (or where `all` asks for it), the row is made
// again from what it sees alone; in f16 also where it sees an infinity, for weights that f16 has no number for are zero beside it too. Nothing is
// spent on it otherwise. Rows that are made again take their time: one prompt of 4096, 8 heads of 128, 89 us; with an infinity at position 4000 13
// ms in bf16, 43 in f16; with one at position 0, which every row sees, 4 (for having looked) and 60; with a NaN there 4 and 7.
constexpr int kReach = 384;           // positions beside its own and beside its window that a row's tiles cover, two tiles of queries together
template <typename T>
__device__ __noinline__ void mend_rows(const Prompt& a, int b, int h, int q0, int rows, int warp, int warps, bool all) {
  const int lane = threadIdx.x & 31, D = a.dim, n = length_of(a, b), kvh = h / a.group;
  const long long stride = (long long)a.kv_heads * D, base = ((long long)b * a.tokens * a.kv_heads + kvh) * D;
  const T *keys = (const T*)a.k + base, *values = (const T*)a.v + base;
  auto finite = [](T v) { return fabsf(to_float(v)) <= 3.4028235e38f; };
  for (int row = q0 + warp; row < min(q0 + rows, n); row += warps) {
    const long long at = (((long long)b * a.tokens + row) * a.heads + h) * D;
    T* out = (T*)a.out + at;
    bool odd = false;
    for (int d = lane; d < D; d += 32) odd |= !finite(out[d]);
    if (!__any_sync(0xFFFFFFFFu, odd)) continue;
    auto hidden = [&](int from, int to) {                          // whether one of these is hidden and not finite
      bool found = false;
      for (int key = max(from, 0); key < min(to, n); ++key)
        if (!sees(a, row, key))
          for (int d = lane; d < D; d += 32) found |= !finite(values[key * stride + d]);
      return __any_sync(0xFFFFFFFFu, found);
    };
    const int start = a.window > 0 ? max(0, row - a.window + 1) : 0, sinks = min(a.sinks, start);
    auto infinite = [&](int from, int to) {                        // whether one of these is an infinity of f16; eight of them a load
      const unsigned pieces = D / 8, total = (unsigned)max(to - from, 0) * pieces;
      bool found = false;
#pragma unroll 8
      for (unsigned p = lane; p < total; p += 32) {
        const uint4 v = *(const uint4*)(values + (from + p / pieces) * stride + p % pieces * 8);
        for (uint32_t w : {v.x, v.y, v.z, v.w}) found |= (w & 0x7FFFu) == 0x7C00u || (w & 0x7FFF0000u) == 0x7C000000u;
      }
      return __any_sync(0xFFFFFFFFu, found);
    };
    const bool seen = std::is_same<T, __half>::value && (infinite(0, sinks) || infinite(start, row + 1));
    if (!all && !seen && !hidden(row + 1, row + kReach) && !hidden(start - kReach, start) && !hidden(sinks, sinks + kReach)) continue;
    float q[8], o[8], m = neg_inf(), l = 0.f;                      // features lane, lane + 32, ...
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[e] = lane + 32 * e < D ? to_float(((const T*)a.q)[at + lane + 32 * e]) * a.scale : 0.f;
      o[e] = 0.f;
    }
    for (int i = 0; i < sinks + row - start + 1; ++i) {
      const long long key = (i < sinks ? i : start + i - sinks) * stride;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < D) s = fmaf(q[e], to_float(keys[key + lane + 32 * e]), s);
      s = warp_sum(s);
      const float top = fmaxf(m, s), ref = top == neg_inf() ? 0.f : top, keep = power(m - ref), p = power(s - ref);
      m = top;
      l = l * keep + p;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < D) o[e] = fmaf(p, to_float(values[key + lane + 32 * e]), o[e] * keep);
    }
    const bool some = l > 0.f || l != l;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < D) out[lane + 32 * e] = from_float<T>(some ? o[e] / l : 0.f);
  }
}

// ---- 32-bit data ---------------------------------------------------------------------------------------
// A block takes 32 or 64 queries of a head, a warp 16 of them, and goes through 32 places of its row of keys at a time: first the sinks that lie
// in front of its first query's window, then from that window's first key on, whichever key that is, so that no tile is half empty. Keys
// and values come by cp.async, a tile ahead. Both products run on the tensor cores by mma.sync (tf32 m16n8k8) in three parts, hi hi + hi
// lo + lo hi, hi a word rounded to the 19 bits that they read and lo what that leaves, rounded likewise; a tile's outputs are added up apart
// and then to the others in 32 bits, since the tensor core cuts its sums. The order of the features within a step of 16 and of the keys
// within a step of 8 is chosen so that fragments are loaded 16 bytes a thread, free of bank conflicts, and so that the scores' fragments
// are the weights'. Bound by the conversions and products, and for few queries by their chain: three prompts of up to 501 tokens, 12 heads of
// 64, window 200 took 76 us on the FMA pipe, 38 with four warps of 16 queries each, 30 with two warps for the same queries. Three of up to 1356, 2
// heads of 72: 195 us with four warps, 128 with eight, two for the same queries; 256 features leave no room for a second half of a tile.
template <int DP>
struct Wide {
  // warps that share their queries, each with its own 32 keys of a tile: two where the tiles leave room for it
  static constexpr int HALVES = DP <= 128 ? 2 : 1, THREADS = DP == 128 ? 256 : 128, ROWS = THREADS / 2 / HALVES, KEYS = 32 * HALVES;
  static constexpr int KP = DP + 16, VP = DP + 4;                    // floats between rows of queries and keys, of values
  static constexpr int STAGE = KEYS * (KP + VP), SMEM = (ROWS * KP + 2 * STAGE) * 4;
  static constexpr int PER_SM = DP == 64 ? 2 : 1;
  static constexpr bool HELD = DP == 64;                             // the queries' parts stay in registers
  static_assert(HALVES == 1 || ROWS * (DP + 2) <= STAGE, "no room for the halves' outputs");
  static_assert((SMEM + 1024) * PER_SM <= 233472, "more than an SM has");
};

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void halves(float v, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(v));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(v - __uint_as_float(hi)));
}
// c[j] += a b[j] for four products side by side: one behind another each would wait for the last.
__device__ __forceinline__ void mma_four(float (&c)[4][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], const float (&b0)[4], const float (&b1)[4]) {
  uint32_t h0[4], l0[4], h1[4], l1[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) { halves(b0[j], h0[j], l0[j]); halves(b1[j], h1[j], l1[j]); }
#pragma unroll
  for (int j = 0; j < 4; ++j) mma_tf32(c[j], lo, h0[j], h1[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) mma_tf32(c[j], hi, l0[j], l1[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) mma_tf32(c[j], hi, h0[j], h1[j]);
}

template <int DP>
__global__ void __launch_bounds__(Wide<DP>::THREADS, Wide<DP>::PER_SM) prompt_wide_kernel(const __grid_constant__ Prompt a) {
  pdl_prologue();
  using C = Wide<DP>;
  constexpr int P = DP / 4, KEYS = C::KEYS;
  extern __shared__ __align__(16) float smem[];
  const int D = a.dim, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane / 4, t = lane % 4, half = warp % C::HALVES, rows = warp / C::HALVES * 16;
  const int h = blockIdx.y, b = blockIdx.z, kvh = h / a.group, n = length_of(a, b);
  const int q0 = (int)(gridDim.x - 1 - blockIdx.x) * C::ROWS, row0 = q0 + rows;           // the rows that see most go first
  const int start = a.window > 0 ? max(0, q0 - a.window + 1) : 0, sinks = min(a.sinks, start), shift = start - sinks;
  const int places = q0 < n ? sinks + min(q0 + C::ROWS, n) - start : 0, tiles = (places + KEYS - 1) / KEYS;
  float *qs = smem, *stages = qs + C::ROWS * C::KP;
  auto copy = [&](float* to, const float* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
  };
  // a thread copies the same four features of every so many rows
  const int c0 = tid % P * 4, r0 = tid / P;
  const long long stride = (long long)a.kv_heads * D, base = ((long long)b * a.tokens * a.kv_heads + kvh) * D + c0;
  auto fetch = [&](int tile) {
    if (tile < tiles) {
      float *ks = stages + (tile & 1) * C::STAGE + r0 * C::KP + c0, *vs = stages + (tile & 1) * C::STAGE + KEYS * C::KP + r0 * C::VP + c0;
#pragma unroll 8
      for (int r = 0; r < KEYS; r += C::THREADS / P) {
        const int place = tile * KEYS + r0 + r;
        const bool there = place < places && c0 < D;
        const long long at = there ? base + (place + (place < sinks ? 0 : shift)) * stride : 0;
        copy(ks + r * C::KP, (const float*)a.k + at, there);
        copy(vs + r * C::VP, (const float*)a.v + at, there);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (tiles) {
    for (int r = r0; r < C::ROWS; r += C::THREADS / P) {
      const bool there = q0 + r < n && c0 < D;
      copy(qs + r * C::KP + c0, (const float*)a.q + (there ? (((long long)b * a.tokens + q0 + r) * a.heads + h) * D + c0 : 0), there);
    }
  }
  fetch(0);
  float m[2] = {neg_inf(), neg_inf()}, l[2] = {0.f, 0.f}, o[DP / 32][4][4];
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[c][e][0] = o[c][e][1] = o[c][e][2] = o[c][e][3] = 0.f;
  // the queries of 16 features, two steps of a product
  auto queries = [&](int c, uint32_t (&hi)[2][4], uint32_t (&lo)[2][4]) {
    const float4 x = *(const float4*)(qs + (rows + g) * C::KP + c * 16 + t * 4), y = *(const float4*)(qs + (rows + g + 8) * C::KP + c * 16 + t * 4);
    halves(x.x, hi[0][0], lo[0][0]); halves(y.x, hi[0][1], lo[0][1]); halves(x.y, hi[0][2], lo[0][2]); halves(y.y, hi[0][3], lo[0][3]);
    halves(x.z, hi[1][0], lo[1][0]); halves(y.z, hi[1][1], lo[1][1]); halves(x.w, hi[1][2], lo[1][2]); halves(y.w, hi[1][3], lo[1][3]);
  };
  uint32_t qh[C::HELD ? DP / 16 : 1][2][4], ql[C::HELD ? DP / 16 : 1][2][4];
  if (C::HELD && tiles) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int c = 0; c < (C::HELD ? DP / 16 : 1); ++c) queries(c, qh[c], ql[c]);
  }
#pragma unroll 1
  for (int tile = 0; tile < tiles; ++tile) {
    fetch(tile + 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const float *ks = stages + (tile & 1) * C::STAGE + half * 32 * C::KP, *vs = stages + (tile & 1) * C::STAGE + KEYS * C::KP + half * 32 * C::VP;
    // the keys of the tile: its sinks, then from `low` to `high`
    const int p0 = tile * KEYS + half * 32, low = max(p0, sinks) + shift, high = p0 + 31 + shift;
    const bool some_sinks = p0 < sinks, hidden = low > row0 + 15 || (a.window > 0 && row0 - high >= a.window && low >= a.sinks);
    if (some_sinks || !hidden) {
      float s[4][4] = {};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c)
        if (c * 16 < D) {
          if (!C::HELD) queries(c, qh[0], ql[0]);
          const int at = C::HELD ? c : 0;
          float k[4][4], add[4][4] = {};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 v = *(const float4*)(ks + (j * 8 + g) * C::KP + c * 16 + t * 4);
            k[0][j] = v.x; k[1][j] = v.y; k[2][j] = v.z; k[3][j] = v.w;
          }
          mma_four(add, qh[at][0], ql[at][0], k[0], k[1]);
          mma_four(add, qh[at][1], ql[at][1], k[2], k[3]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] += add[j][i];
        }
      const bool edge = high > row0 || (a.window > 0 && row0 + 15 - low >= a.window);
      float top[2] = {neg_inf(), neg_inf()};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[j][i] *= a.scale;
          if (edge) {
            const int place = p0 + j * 8 + t * 2 + (i & 1);
            if (!sees(a, row0 + g + i / 2 * 8, place + (place < sinks ? 0 : shift))) s[j][i] = neg_inf();
          }
          top[i / 2] = fmaxf(top[i / 2], s[j][i]);
        }
      uint32_t hi[4][4], lo[4][4];
      float keep[2], ref[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 1));
        top[r] = fmaxf(fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 2)), m[r]);
        ref[r] = top[r] == neg_inf() ? 0.f : top[r];
        keep[r] = power(m[r] - ref[r]);
        l[r] *= keep[r];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = power(s[j][i] - ref[i / 2]);
          l[i / 2] += p[i];
          halves(p[i], hi[j][(i & 1) * 2 + i / 2], lo[j][(i & 1) * 2 + i / 2]);
        }
      }
      if (__any_sync(0xFFFFFFFFu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[c][e][i] *= keep[i / 2];
      }
      m[0] = top[0];
      m[1] = top[1];
#pragma unroll
      for (int c = 0; c < DP / 32; ++c)
        if (c * 32 < D) {
          float add[4][4] = {};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 x = *(const float4*)(vs + (j * 8 + t * 2) * C::VP + c * 32 + g * 4), y = *(const float4*)(vs + (j * 8 + t * 2 + 1) * C::VP + c * 32 + g * 4);
            const float v0[4] = {x.x, x.y, x.z, x.w}, v1[4] = {y.x, y.y, y.z, y.w};
            mma_four(add, hi[j], lo[j], v0, v1);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[c][e][i] += add[e][i];
        }
    }
    __syncthreads();                                                // the tile's place may be filled again
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
    l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
  }
  if (C::HALVES == 2 && tiles) {                                     // the second half's outputs to the first: a lane's words, 32 apart
    float* at = stages + warp / 2 * (16 * (DP + 2)) + lane;
    if (half) {
#pragma unroll
      for (int c = 0; c < DP / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) at[(c * 16 + i) * 32] = o[c][i / 4][i % 4];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (t < 2) at[(DP / 2) * 32 - lane + (g + 8 * r) * 2 + t] = t ? l[r] : m[r];
    }
    __syncthreads();
    if (!half) {
      float mine[2], other[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float* stats = at - lane + (DP / 2) * 32 + (g + 8 * r) * 2;
        const float top = fmaxf(m[r], stats[0]), ref = top == neg_inf() ? 0.f : top;
        mine[r] = power(m[r] - ref);
        other[r] = power(stats[0] - ref);
        l[r] = l[r] * mine[r] + stats[1] * other[r];
      }
#pragma unroll
      for (int c = 0; c < DP / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i / 4][i % 4] = o[c][i / 4][i % 4] * mine[i % 4 / 2] + at[(c * 16 + i) * 32] * other[i % 4 / 2];
    }
  }
  float odd = 0.f;                                                  // NaN where a result is not finite
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row0 + g + r * 8;
    if (half || row >= a.tokens) continue;
    const float inv = row < n && (l[r] > 0.f || l[r] != l[r]) ? 1.f / l[r] : 0.f;
    float* to = (float*)a.out + (((long long)b * a.tokens + row) * a.heads + h) * D + t * 8;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (c * 32 + t * 8 >= D) continue;
        float4 v = {0.f, 0.f, 0.f, 0.f};
        if (row < n) v = {o[c][0][r * 2 + i] * inv, o[c][1][r * 2 + i] * inv, o[c][2][r * 2 + i] * inv, o[c][3][r * 2 + i] * inv};
        odd = fmaf(v.x + v.y + v.z + v.w, 0.f, odd);
        *(float4*)(to + c * 32 + i * 4) = v;
      }
  }
  // (with all rows that are not finite: parts of infinities are no numbers)
  if (__syncthreads_or(odd != odd)) mend_rows<float>(a, b, h, q0, C::ROWS, warp, C::THREADS / 32, true);
}

// ---- 16-bit data on the tensor cores -------------------------------------------------------------------
// A block, one per SM, goes from one tile of 128 queries of a head to another, or takes two of them along that read the same keys: two
// heads that share a key-value head, or two tiles of one head. Warp 8 brings queries and tiles of 128 keys and values by TMA tiled
// copies into 128-byte-swizzled shared memory, a tile or more ahead of warp 9, which issues tcgen05.mma: scores = Q K^T from shared
// memory into tensor memory, then O += P V with the weights P read from tensor memory, where they take the place of the scores.
// Warps 0-7 read the scores, mask them, exponentiate and round the weights to 16 bits (the one rounding beside the result's: the second
// product's operands have 16 bits): four for each tile of queries, a thread a row, or with one tile two threads a row, which agree on
// its maximum. One tile's products run while the other's weights are made; a single tile has two places for its scores instead. The
// first half of a row's weights is multiplied while the second is made. The outputs are scaled to a new maximum only when it has
// grown by more than 2^8 since the last time; the weights are at most 2^8 until then, which no type minds, and the sums are divided
// in the end by a sum that was taken in the same units.
// Two prompts of 4096, 32 heads of 128, window 1024: one tile a block, two blocks an SM 206 us, two tiles a block 185 to 195 (650 TFLOP/s); with
// two threads a row there too 192, with a quarter of the exponentials as polynomials on the FMA pipe 190. The chain of a tile - scores,
// maximum, exponentials, outputs, 4300 cycles of which the tensor core works 2050 for both tiles - is what is left.
// Products of a block run in the order in which its one thread issued them, so that scores may go where the weights of a product in
// front are read.
constexpr int kRows = 128, kMmaThreads = 320;
constexpr float kGrowth = 8.f;

constexpr int kStagePitch = 80;       // bytes between rows of 32 results on their way out

template <int DP, int ITEMS>
struct Mma {
  static constexpr int BLOCKS = DP / 64, BLOCK = kRows * 128, TILE = BLOCKS * BLOCK;      // bytes: a box of 64 features, a tile
  static constexpr int STAGES = DP == 64 ? 4 : DP == 128 ? 2 : 1;
  static constexpr int HALVES = ITEMS == 1 ? 2 : 1, COLS = kRows / HALVES;               // threads of a row, scores of a thread
  static constexpr int SMEM = TILE * (ITEMS + 2 * STAGES) + 1024 + 512 + 4 * kRows * 4 + 8 * 32 * kStagePitch;
  static_assert(SMEM <= 232448, "more than an SM has");
  // columns of the weights of one half of a tile's keys: over the scores of the thread that makes them
  static __device__ __forceinline__ int weights(int half) { return half * (ITEMS == 2 ? 32 : 64); }
};

__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// The values' tile as second operand, its features contiguous: atoms of 64 features x 8 keys, 1024 bytes apart along the keys and a
// box apart along the features.
__device__ __forceinline__ uint64_t values_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)((kRows * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of a thread's lane of tensor memory. Loads are on their way until `loaded` has been passed, and what they give is touched by
// `settle` behind it, so that no use of it can come before.
__device__ __forceinline__ void load32(uint32_t addr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(addr) : "memory");
}
__device__ __forceinline__ void loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void settle(uint32_t* v) {
  asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
// Eight columns scaled in place.
__device__ __forceinline__ void scale8(uint32_t addr, float by) {
  uint32_t v[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(addr) : "memory");
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * by);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void store32(uint32_t addr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
               ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
  uint32_t d;
  if (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// What a block does next: its tiles of queries and the tiles of keys that they visit, those of the sinks in front of the window, then
// the window's.
template <int ITEMS>
struct Unit {
  int b, kvh, n, first, sinks, count;
  int head[ITEMS], q0[ITEMS];
  __device__ __forceinline__ Unit(const Prompt& a, int unit) {
    const int each = a.head_units * a.batch, rest = unit % each, hu = rest % a.head_units;
    const int qu = a.query_units - 1 - unit / each;                  // the rows that see most go first
    b = rest / a.head_units;
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      head[u] = ITEMS == 2 && a.pairs ? hu * 2 + u : hu;
      q0[u] = (ITEMS == 2 && !a.pairs ? qu * 2 + u : qu) * kRows;
    }
    kvh = head[0] / a.group;
    n = length_of(a, b);
    first = a.window > 0 ? max(0, q0[0] - a.window + 1) / kRows : 0;
    sinks = min((int)(((long long)a.sinks + kRows - 1) / kRows), first);
    count = q0[0] >= n ? 0 : sinks + (min(q0[ITEMS - 1] + kRows, n) - 1) / kRows - first + 1;
  }
  __device__ __forceinline__ int key(int i) const { return (i < sinks ? i : first + i - sinks) * kRows; }
};

template <typename T, int DP, int ITEMS>
__global__ void __launch_bounds__(kMmaThreads, 1) prompt_mma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Prompt a,
                                                                    int* __restrict__ error_flag) {
  using C = Mma<DP, ITEMS>;
  constexpr int S = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *qs = smem, *ks = qs + ITEMS * C::TILE, *vs = ks + S * C::TILE;
  uint64_t* bars = (uint64_t*)(vs + S * C::TILE);
  // queries are there, are done with; keys and values likewise, a stage each; scores of a place; weights of a place, two halves, the first
  // with the outputs scaled; outputs of a tile have all products so far, have been read; both threads of a row have spoken; nothing is
  // under way
  constexpr int Q_FULL = 0, Q_EMPTY = 1, K_FULL = 2, K_EMPTY = K_FULL + S, V_FULL = K_EMPTY + S, V_EMPTY = V_FULL + S, S_FULL = V_EMPTY + S, P_FULL = S_FULL + 2,
                PV_DONE = P_FULL + 4, O_EMPTY = PV_DONE + 2, AGREED = O_EMPTY + 2, DRAINED = AGREED + 4, BARRIERS = DRAINED + 1;
  static_assert(BARRIERS * 8 + 12 <= 512, "barriers");
  auto bar = [base = smem_u32(bars)](int k) { return base + 8u * (uint32_t)k; };
  uint32_t* tmem_slot = (uint32_t*)(bars + BARRIERS);
  volatile int *failed = (volatile int*)(tmem_slot + 1), *strange = failed + 1;
  float* said = (float*)((uint8_t*)bars + 512);                      // [parity][half][row]
  uint8_t* stage = (uint8_t*)(said + 4 * kRows);                     // [warp][row][32 results]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, D = a.dim;
  if (tid == 0) {
    // (with two threads a row, the first half's weights are announced by its four warps, and by the four others that the outputs are scaled)
    for (int k = 0; k < BARRIERS; ++k)
      mbar_init(bar(k), k >= P_FULL && k < PV_DONE ? (ITEMS == 1 && (k - P_FULL) % 2 == 0 ? 8 : 4) : k >= O_EMPTY && k < AGREED ? 8 / ITEMS : k >= AGREED && k < DRAINED ? 2 : 1);
    *failed = 0;
    *strange = 0;                                                    // whether a result is not finite
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_prologue();
  // the place of a tile's scores and how often it has been used, by the number of the tile since the block began
  auto place = [](int u, int it) { return ITEMS == 2 ? u : it & 1; };
  auto turn = [](int it) { return ITEMS == 2 ? it & 1 : it >> 1 & 1; };
  auto outputs = [&](int u) { return tmem + 256 + u * DP; };

  if (warp == 8) {
    // ------------------------------ copies (one lane) -----------------------------------------------------------
    if (lane == 0) {
      bool ok = true;
      int it = 0, kt = 0, vt = 0, done = 0;
      for (int unit = blockIdx.x; unit < a.units && ok; unit += gridDim.x) {
        const Unit<ITEMS> w(a, unit);
        if (!w.count) continue;
        const int row = w.b * a.tokens;
        if (done && !(ok = role_wait(bar(Q_EMPTY), (done - 1) & 1, failed))) break;
        expect_bytes(bar(Q_FULL), ITEMS * C::TILE);
#pragma unroll
        for (int u = 0; u < ITEMS; ++u)
#pragma unroll
          for (int c = 0; c < C::BLOCKS; ++c) copy_box(smem_u32(qs) + u * C::TILE + c * C::BLOCK, &tm_q, bar(Q_FULL), c * 64, row + w.q0[u], w.head[u]);
        ++done;
        for (int i = 0; i < w.count; ++i, ++it) {
          const int s = it % S, parity = ((it / S) & 1) ^ 1, k0 = row + w.key(i);
          if (it >= S && !(ok = role_wait(bar(K_EMPTY + s), parity, failed))) break;
          expect_bytes(bar(K_FULL + s), C::TILE);
#pragma unroll
          for (int c = 0; c < C::BLOCKS; ++c) copy_box(smem_u32(ks) + s * C::TILE + c * C::BLOCK, &tm_k, bar(K_FULL + s), c * 64, k0, w.kvh);
          ++kt;
          if (it >= S && !(ok = role_wait(bar(V_EMPTY + s), parity, failed))) break;
          expect_bytes(bar(V_FULL + s), C::TILE);
#pragma unroll
          for (int c = 0; c < C::BLOCKS; ++c) copy_box(smem_u32(vs) + s * C::TILE + c * C::BLOCK, &tm_v, bar(V_FULL + s), c * 64, k0, w.kvh);
          ++vt;
        }
      }
      if (!ok || *failed) {
        // copies that nobody consumed any more: wait for them before the shared memory goes away
        if (done) mbar_wait(bar(Q_FULL), (done - 1) & 1);
        for (int j = max(0, kt - S); j < kt; ++j) mbar_wait(bar(K_FULL + j % S), (j / S) & 1);
        for (int j = max(0, vt - S); j < vt; ++j) mbar_wait(bar(V_FULL + j % S), (j / S) & 1);
      }
    }
  } else if (warp == 9) {
    // ------------------------------ products --------------------------------------------------------------------
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRows >> 4) << 24);
    constexpr uint32_t idesc_s = common | ((uint32_t)(kRows >> 3) << 17), idesc_o = common | (1u << 16) | ((uint32_t)(DP >> 3) << 17);
    const uint64_t d_q = umma_desc(smem_u32(qs)), d_k = umma_desc(smem_u32(ks)), d_v = values_desc(smem_u32(vs));
    bool ok = true;
    auto wait = [&](int k, int parity) {
      ok = __all_sync(0xFFFFFFFFu, ok && role_wait(bar(k), parity, failed));
      after_sync();
    };
    int it = 0, done = 0;
    for (int unit = blockIdx.x; unit < a.units && ok; unit += gridDim.x) {
      const Unit<ITEMS> w(a, unit);
      if (!w.count) continue;
      auto scores = [&](int u, int i) {
        const int j = it + i, s = j % S;
        if (u == 0) wait(K_FULL + s, (j / S) & 1);
        if (ok && elect_one()) {
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk) {
            const uint64_t at = (uint64_t)((kk / 4 * C::BLOCK + kk % 4 * 32) >> 4);
            mma_smem(tmem + place(u, j) * kRows, d_q + (uint64_t)((u * C::TILE) >> 4) + at, d_k + (uint64_t)((s * C::TILE) >> 4) + at, idesc_s, kk > 0);
          }
          commit(bar(S_FULL + place(u, j)));
          if (u == ITEMS - 1) {
            commit(bar(K_EMPTY + s));
            if (i + 1 == w.count) commit(bar(Q_EMPTY));
          }
        }
        __syncwarp();
      };
      auto weighted = [&](int u, int i) {
        const int j = it + i, s = j % S, k0 = w.key(i);
        if (u == 0) {
          wait(V_FULL + s, (j / S) & 1);
          if (ok && k0 + kRows > w.n) {
            // values behind the sequence are not zero times a weight of zero where they are no numbers: they go
            const int gone = k0 + kRows - w.n;
            for (int p = lane; p < C::BLOCKS * gone * 8; p += 32) {
              const int c = p / (gone * 8), r = kRows - gone + p % (gone * 8) / 8;
              *(uint4*)(vs + s * C::TILE + c * C::BLOCK + r * 128 + p % 8 * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
        }
        if (i == 0 && done) wait(O_EMPTY + u, (done - 1) & 1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          wait(P_FULL + 2 * place(u, j) + half, turn(j));
          if (ok && elect_one()) {
#pragma unroll
            for (int kk = half * (kRows / 32); kk < (half + 1) * (kRows / 32); ++kk)
              mma_tmem(outputs(u), tmem + place(u, j) * kRows + C::weights(half) + kk % 4 * 8, d_v + (uint64_t)((s * C::TILE + kk * 2048) >> 4), idesc_o, i > 0 || kk > 0);
            if (half) {
              commit(bar(PV_DONE + u));
              if (u == ITEMS - 1) commit(bar(V_EMPTY + s));
            }
          }
          __syncwarp();
        }
      };
      wait(Q_FULL, done & 1);
#pragma unroll
      for (int u = 0; u < ITEMS; ++u) scores(u, 0);
      for (int i = 0; i < w.count && ok; ++i) {
        if (ITEMS == 1 && i + 1 < w.count) scores(0, i + 1);
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) {
          weighted(u, i);
          if (ITEMS == 2 && i + 1 < w.count) scores(u, i + 1);
        }
      }
      it += w.count;
      ++done;
    }
    if (!ok || *failed) {                                            // tensor memory goes back only when no product is left
      if (elect_one()) commit(bar(DRAINED));
      __syncwarp();
      mbar_wait(bar(DRAINED), 0);
    }
  } else {
    // ------------------------------ rows: weights, then the result ------------------------------------------------
    constexpr int COLS = C::COLS;
    const int quad = warp & 3, upper = warp >> 2, u = ITEMS == 2 ? upper : 0, half = ITEMS == 2 ? 0 : upper, r = quad * 32 + lane;
    const uint32_t mine = (uint32_t)(32 * quad) << 16;
    // f16: weights in units that keep the small ones out of its subnormal range
    constexpr float shift = std::is_same<T, __half>::value ? 6.f : 0.f;
    const uint64_t scale = two(a.scale, a.scale);
    bool ok = true;
    auto wait = [&](int k, int parity) { return ok = __all_sync(0xFFFFFFFFu, role_wait(bar(k), parity, failed)); };
    int it = 0, spoken = 0;
    // what the other thread of the row says for what this one says
    auto exchange = [&](float v, float& other) {
      float* at = said + (spoken & 1) * 2 * kRows;
      at[half * kRows + r] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(AGREED + quad));
      if (!wait(AGREED + quad, spoken & 1)) return false;
      ++spoken;
      other = at[(half ^ 1) * kRows + r];
      return true;
    };
    for (int unit = blockIdx.x; unit < a.units && ok; unit += gridDim.x) {
      const Unit<ITEMS> w(a, unit);
      const int q0 = w.q0[u], row = q0 + r;
      T* out = (T*)a.out + (((long long)w.b * a.tokens + q0 + quad * 32) * a.heads + w.head[u]) * D;
      float m = neg_inf(), l = 0.f;
      for (int i = 0; i < w.count; ++i) {
        const int j = it + i, k0 = w.key(i) + half * COLS;
        const uint32_t t_s = tmem + mine + place(u, j) * kRows;
        if (!wait(S_FULL + place(u, j), turn(j))) break;
        after_sync();
        // The scores are read twice, 32 at a time and the next while these are worked on: once for the maximum, once for the weights. (Held
        // from one to the other, a row's did not stay in registers.)
        constexpr int PARTS = COLS / 32;
        uint32_t held[2][32];
        // masks at the edges only: the last key that the row sees, the first of its window, the sinks
        const bool late = k0 + COLS - 1 > q0, early = a.window > 0 && q0 + kRows - 1 - k0 >= a.window && k0 + COLS > a.sinks;
        // (compares and selects run at half the rate of additions: each case has no more of them than it needs, and what they leave goes
        // back to where the weights' pass reads it)
        auto masked = [&](uint32_t* s, int c) {
          const int most = row - k0 - c, least = row - a.window + 1 - k0 - c, always = a.sinks - k0 - c;
          if (early && always > 0) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k < least && k >= always) s[k] = 0xFF800000u;
          } else if (early) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k < least) s[k] = 0xFF800000u;
          }
          if (late) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k > most) s[k] = 0xFF800000u;
          }
        };
        float top[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
        load32(t_s + half * COLS, held[0]);
#pragma unroll
        for (int c = 0; c < PARTS; ++c) {
          uint32_t* s = held[c & 1];
          loaded();
          settle(s);
          if (c + 1 < PARTS) load32(t_s + half * COLS + (c + 1) * 32, held[(c + 1) & 1]);
          else if (!(late || early)) load32(t_s + half * COLS, held[0]);                    // the first once more, for the weights
          if (late || early) {
            masked(s, c * 32);
            store32(t_s + half * COLS + c * 32, s);
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2) top[k / 2 % 4] = max3(top[k / 2 % 4], __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
        }
        if (late || early) {
          stored();
          load32(t_s + half * COLS, held[0]);
        }
        float best = fmaxf(max3(top[0], top[1], top[2]), top[3]);
        if (ITEMS == 1) {
          float other;
          if (!exchange(best, other)) break;
          best = fmaxf(best, other);
        }
        const bool grown = best > m && (best - m) * a.scale > kGrowth;
        if (__any_sync(0xFFFFFFFFu, grown)) {                          // (of the same rows, so the same in both warps of a row)
          const float now = fmaxf(m, best), keep = m == neg_inf() ? 0.f : power((m - now) * a.scale);
          m = now;
          l *= keep;
          if (i > 0) {
            if (!wait(PV_DONE + u, (j - 1) & 1)) break;
            after_sync();
#pragma unroll 1
            for (int c = half * (DP / 2); c < (ITEMS == 2 ? DP : (half + 1) * (DP / 2)); c += 8) scale8(outputs(u) + mine + c, keep);
          }
        }
        if (ITEMS == 1 && half) {
          // a product adds to all columns of the outputs, so the first one waits for what this thread has scaled of them too, not only for
          // the weights of the other
          stored();
          before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(P_FULL + 2 * place(u, j)));
        }
        const float ref = m == neg_inf() ? 0.f : m * a.scale - shift;
        const uint64_t minus = two(-ref, -ref);
        uint64_t sum[4] = {0, 0, 0, 0};
        uint32_t p[32];
#pragma unroll
        for (int c = 0; c < PARTS; ++c) {
          uint32_t* s = held[c & 1];
          loaded();
          settle(s);
          if (c + 1 < PARTS) load32(t_s + half * COLS + (c + 1) * 32, held[(c + 1) & 1]);
#pragma unroll
          for (int g = 0; g < 32; g += 16) {                            // eight pairs side by side: one after another they are a chain
            uint64_t x[8];
            float y[16];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = fma2(two(s[g + 2 * k], s[g + 2 * k + 1]), scale, minus);
#pragma unroll
            for (int k = 0; k < 8; ++k) { y[2 * k] = power(first(x[k])); y[2 * k + 1] = power(second(x[k])); }
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[k % 4] = add2(sum[k % 4], two(y[2 * k], y[2 * k + 1]));
#pragma unroll
            for (int k = 0; k < 8; ++k) p[c % 2 * 16 + g / 2 + k] = pair16<T>(y[2 * k], y[2 * k + 1]);
          }
          if (c % 2 == 1) {
            // the weights of 64 keys take the place of scores that this thread has read
            const int part = ITEMS == 2 ? c / 2 : half;
            store32(t_s + C::weights(part), p);
            stored();
            // A barrier's parity tells a phase from the next and not from the one after: who waits for the last tile's products below has
            // to have seen those of the tile in front of it, and here the last ones cannot be through yet. (With one tile of queries, scores
            // are issued in front of the last tile's products, so that having them says nothing of those, which wait for the slowest warp.)
            if (c + 1 == PARTS && i > 0 && i + 1 == w.count) wait(PV_DONE + u, (j - 1) & 1);
            before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P_FULL + 2 * place(u, j) + part));
          }
        }
        const uint64_t all = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
        l += first(all) + second(all);
        if (!ok) break;
      }
      if (!ok) break;
      if (w.count) {
        if (ITEMS == 1) {
          float other;
          if (!exchange(l, other)) break;
          l += other;
        }
        it += w.count;
        if (!wait(PV_DONE + u, (it - 1) & 1)) break;
        after_sync();
      }
      const bool some = w.count && row < w.n && (l > 0.f || l != l);      // whether the row has any weight to give
      const float inv = some ? 1.f / l : 0.f;
      uint64_t odd = 0;                                              // NaN where one is not finite
#pragma unroll
      for (int c0 = 0; c0 < (ITEMS == 2 ? DP : DP / 2); c0 += 32) {
        const int c = (ITEMS == 2 ? 0 : half * (DP / 2)) + c0;
        uint32_t o[32];
        if (w.count) {
          load32(outputs(u) + mine + c, o);
          loaded();
          settle(o);
          if (some) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) odd = fma2(two(o[e], o[e + 1]), two(0.f, 0.f), odd);
          }
        }
        // by way of shared memory, so that a store touches eight rows' 64 bytes and not 32 rows' 16: those took 8600 cycles a tile, 4500 so, most of it
        // the wait for the last product
        uint8_t* at = stage + warp * 32 * kStagePitch;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint4 v = {0, 0, 0, 0};
          if (some) {
            v.x = pair16<T>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
            v.y = pair16<T>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            v.z = pair16<T>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
            v.w = pair16<T>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
          }
          *(uint4*)(at + lane * kStagePitch + e * 2) = v;
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int line = e * 8 + lane / 4, col = c + lane % 4 * 8;
          if (q0 + quad * 32 + line < a.tokens && col < D) *(uint4*)(out + (long long)line * a.heads * D + col) = *(const uint4*)(at + line * kStagePitch + lane % 4 * 16);
        }
        __syncwarp();
      }
      if (first(odd) != first(odd) || second(odd) != second(odd)) *strange = 1;
      if (w.count) {
        before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(O_EMPTY + u));
      }
    }
  }
  before_sync();
  __syncthreads();
  if (tid == 0 && *failed) atomicAdd(error_flag, 1);
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  if (!*strange || *failed) return;
  for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
    const Unit<ITEMS> w(a, unit);
#pragma unroll 1
    for (int u = 0; u < ITEMS; ++u) mend_rows<T>(a, w.b, w.head[u], w.q0[u], kRows, warp, kMmaThreads / 32, false);
  }
}

template <int DP>
cudaError_t launch_wide(const Prompt& a, cudaStream_t stream, int* launches) {
  static bool done[64] = {};
  if (cudaError_t e = allow_smem(prompt_wide_kernel<DP>, Wide<DP>::SMEM, done)) return e;
  return launch_op(prompt_wide_kernel<DP>, dim3((unsigned)((a.tokens + Wide<DP>::ROWS - 1) / Wide<DP>::ROWS), (unsigned)a.heads, (unsigned)a.batch), Wide<DP>::THREADS,
                   Wide<DP>::SMEM, stream, launches, a);
}

template <typename T, int DP, int ITEMS>
cudaError_t launch_mma(Prompt a, int* error_flag, cudaStream_t stream, int* launches, const char** why) {
  static bool done[64] = {};
  using C = Mma<DP, ITEMS>;
  if (cudaError_t e = allow_smem(prompt_mma_kernel<T, DP, ITEMS>, C::SMEM, done)) return e;
  // features, tokens of all sequences, heads: boxes of 64 features and 128 tokens of one head; what is outside reads zero
  alignas(64) CUtensorMap maps[3];
  const void* bases[3] = {a.q, a.k, a.v};
  for (int i = 0; i < 3; i++) {
    const unsigned long long heads = (unsigned long long)(i ? a.kv_heads : a.heads), dims[3] = {(unsigned long long)a.dim, (unsigned long long)a.batch * a.tokens, heads},
                             strides[2] = {heads * a.dim * 2, (unsigned long long)a.dim * 2};
    const unsigned box[3] = {64, (unsigned)kRows, 1};
    if (!encode_tensor_map(&maps[i], std::is_same<T, __nv_bfloat16>::value ? 1 : 0, 3, bases[i], dims, strides, box)) {
      *why = "cuTensorMapEncodeTiled refused an operand";
      return cudaErrorInvalidValue;
    }
  }
  const int tiles = (a.tokens + kRows - 1) / kRows;
  a.pairs = ITEMS == 2 && a.group % 2 == 0;
  a.head_units = a.pairs ? a.heads / 2 : a.heads;
  a.query_units = ITEMS == 2 && !a.pairs ? (tiles + 1) / 2 : tiles;
  a.units = a.head_units * a.query_units * a.batch;
  return launch_op(prompt_mma_kernel<T, DP, ITEMS>, dim3((unsigned)std::min(a.units, kSMs)), kMmaThreads, C::SMEM, stream, launches, maps[0], maps[1], maps[2], a,
                   error_flag);
}
template <typename T>
cudaError_t launch_16bit(const Prompt& a, int* error_flag, cudaStream_t stream, int* launches, const char** why) {
  // two tiles of queries a block where that still leaves no SM without one
  const bool two = (long long)a.heads * a.batch * ((a.tokens + kRows - 1) / kRows) >= 2 * kSMs;
  if (a.dim <= 64) return two ? launch_mma<T, 64, 2>(a, error_flag, stream, launches, why) : launch_mma<T, 64, 1>(a, error_flag, stream, launches, why);
  if (a.dim <= 128) return two ? launch_mma<T, 128, 2>(a, error_flag, stream, launches, why) : launch_mma<T, 128, 1>(a, error_flag, stream, launches, why);
  return launch_mma<T, 256, 1>(a, error_flag, stream, launches, why);
}

}  // namespace

const char* window_attention_plan(OperatorLaunch& op) {
  if (op.heads > 65535 || op.batch > 65535) return "more than 65535 heads or sequences";
  if (op.tokens >= (1 << 30)) return "prompts of 2^30 tokens and more";
  if ((long long)op.batch * op.tokens >= (1LL << 31)) return "2^31 tokens and more";
  if ((long long)op.batch * op.heads * ((op.tokens + kRows - 1) / kRows) >= (1LL << 31) - kSMs) return "too many heads and sequences";
  op.scratch_bytes = 0;
  op.launches = 1;
  op.waits = op.type != 0;
  return nullptr;
}

cudaError_t launch_window_attention(const OperatorLaunch& op, void* const* args, void*, int* error_flag, cudaStream_t stream, int* launches,
                                    const char** why) {
  Prompt a = {};
  a.out = args[0];
  a.q = args[1];
  a.k = args[2];
  a.v = args[3];
  a.lengths = op.has_lengths ? (const int*)args[4] : nullptr;
  a.batch = op.batch; a.tokens = op.tokens; a.heads = op.heads; a.kv_heads = op.kv_heads; a.dim = op.dim; a.group = op.heads / op.kv_heads;
  a.window = op.window; a.sinks = op.sinks;
  a.scale = op.scale * kLog2e;
  if (op.type == 0)
    return op.dim <= 64 ? launch_wide<64>(a, stream, launches) : op.dim <= 128 ? launch_wide<128>(a, stream, launches) : launch_wide<256>(a, stream, launches);
  if (op.type == 1) return launch_16bit<__nv_bfloat16>(a, error_flag, stream, launches, why);
  return launch_16bit<__half>(a, error_flag, stream, launches, why);
}

}  // namespace b200
