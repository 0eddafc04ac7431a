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
};

__device__ __forceinline__ int length_of(const Prompt& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.tokens) : a.tokens;
}

// 32-bit data on the FMA pipe: a block takes 64 queries of a head, in tiles of 64 keys. A thread holds 4 x 4 scores and, of the
// outputs, four rows and every sixteenth group of four features.
constexpr int kTile = 64, kScoreRow = kTile + 4;

template <typename T>
__global__ void __launch_bounds__(256) prompt_fma_kernel(const __grid_constant__ Prompt a) {
  pdl_prologue();
  extern __shared__ __align__(16) float smem[];
  const int D = a.dim, P = D + 4, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  float *qs = smem, *ks = qs + kTile * P, *vs = ks + kTile * P, *ss = vs + kTile * P;
  const int h = blockIdx.y, b = blockIdx.z, kvh = h / a.group, n = length_of(a, b);
  const int q0 = (int)(gridDim.x - 1 - blockIdx.x) * kTile;         // the rows that see most go first
  constexpr int N = Pack<T>::N;
  const int pieces = D / N;
  auto load = [&](float* to, const void* from, int row0, int heads, int head, float scale) {
    for (int i = tid; i < kTile * pieces; i += 256) {
      const int row = i / pieces, c = i % pieces * N;
      uint4 v = {0, 0, 0, 0};
      if (row0 + row < n) v = *(const uint4*)((const T*)from + (((long long)b * a.tokens + row0 + row) * heads + head) * D + c);
      float f[N];
      unpack<T>(v, f);
#pragma unroll
      for (int e = 0; e < N; ++e) to[row * P + c + e] = f[e] * scale;
    }
  };
  float m[4], l[4], o[4][4][4];                                     // row, group of features, feature
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = neg_inf();
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
  }
  if (q0 < n) {
    load(qs, a.q, q0, a.heads, h, a.scale);
    const int last = min(q0 + kTile, n), first = a.window > 0 ? max(0, q0 - a.window + 1) : 0;
    for (int k0 = 0; k0 < last; k0 += kTile) {
      if (k0 + kTile <= first && k0 >= a.sinks) continue;
      __syncthreads();
      load(ks, a.k, k0, a.kv_heads, kvh, 1.f);
      load(vs, a.v, k0, a.kv_heads, kvh, 1.f);
      __syncthreads();
      float s[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
      for (int d = 0; d < D; d += 4) {
        float4 q[4], k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = *(const float4*)(qs + (ty * 4 + i) * P + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = *(const float4*)(ks + (tx + 16 * j) * P + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] = fmaf(q[i].x, k[j].x, fmaf(q[i].y, k[j].y, fmaf(q[i].z, k[j].z, fmaf(q[i].w, k[j].w, s[i][j]))));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = q0 + ty * 4 + i;
        float top = neg_inf();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = k0 + tx + 16 * j;
          const bool see = key <= row && key < n && (a.window == 0 || row - key < a.window || key < a.sinks);
          if (!see) s[i][j] = neg_inf();
          top = fmaxf(top, s[i][j]);
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
        const float now = fmaxf(m[i], top), ref = now == neg_inf() ? 0.f : now, keep = exp2f(m[i] - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(s[i][j] - ref);
          sum += p;
          ss[(ty * 4 + i) * kScoreRow + tx + 16 * j] = p;
        }
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
        l[i] = l[i] * keep + sum;
        m[i] = now;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][c][e] *= keep;
      }
      __syncwarp();                                                 // a row's scores stay within a warp
      for (int t = 0; t < kTile; t += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *(const float4*)(ss + (ty * 4 + i) * kScoreRow + t);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int d = (tx + 16 * c) * 4;
          if (d < D) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float4 v = *(const float4*)(vs + (t + u) * P + d);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
                o[i][c][0] = fmaf(w, v.x, o[i][c][0]);
                o[i][c][1] = fmaf(w, v.y, o[i][c][1]);
                o[i][c][2] = fmaf(w, v.z, o[i][c][2]);
                o[i][c][3] = fmaf(w, v.w, o[i][c][3]);
              }
            }
          }
        }
      }
      __syncwarp();
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = q0 + ty * 4 + i;
    if (row >= a.tokens) continue;
    const bool some = row < n && (l[i] > 0.f || l[i] != l[i]);
    T* to = (T*)a.out + (((long long)b * a.tokens + row) * a.heads + h) * D;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = (tx + 16 * c) * 4;
      if (d < D)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[d + e] = from_float<T>(some ? o[i][c][e] / l[i] : 0.f);
    }
  }
}

// ---- 16-bit data on the tensor cores -------------------------------------------------------------------
// A block takes 128 queries of a head in tiles of 128 keys. Warp 4 brings the queries and the tiles of keys and values by TMA tiled
// copies into 128-byte-swizzled shared memory, warp 5 issues tcgen05.mma: scores = Q K^T from shared memory into tensor memory, then
// O += P V with the weights P read from tensor memory, where they take the place of the scores. Warps 0-3 hold a row a thread: they
// read the scores, mask them, exponentiate and round the weights to 16 bits (the one rounding beside the result's: the second
// product's operands have 16 bits), and keep maximum and sum; the first half of a tile's weights is multiplied while the second is
// made. The outputs are scaled to a new maximum only when it has grown by more
// than 2^8 since the last time; the weights are at most 2^8 until then, which no type minds, and the sums are divided in the end by
// a sum that was taken in the same units. Heads of up to 128 features: two blocks an SM, so that one's products run while the other
// exponentiates. Heads of up to 256: one block, and two tiles of scores in tensor memory.
constexpr int kRows = 128, kMmaThreads = 192;
constexpr float kGrowth = 8.f;

template <int DP>
struct Mma {
  static constexpr int BLOCKS = DP / 64, BLOCK = kRows * 128, TILE = BLOCKS * BLOCK;      // bytes: a box of 64 features, a tile
  static constexpr int STAGES = DP == 64 ? 2 : 1;
  static constexpr int SCORES = DP == 256 ? 2 : 1;                   // tiles of scores in tensor memory
  static constexpr int COLUMNS = DP == 256 ? 512 : 256;
  static constexpr int BLOCKS_PER_SM = DP == 256 ? 1 : 2;
  static constexpr int SMEM = TILE * (1 + 2 * STAGES) + 1024 + 256;
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
__device__ __forceinline__ float power(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two floats in a register pair, for the instructions that take both at once.
__device__ __forceinline__ uint64_t two(uint32_t x, uint32_t y) { return (uint64_t)y << 32 | x; }
__device__ __forceinline__ uint64_t two(float x, float y) { return two(__float_as_uint(x), __float_as_uint(y)); }
__device__ __forceinline__ float first(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float second(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The tiles of keys that a tile of queries visits: those of the sinks in front of the window, then the window's.
struct Tiles {
  int sinks, first, count;
  __device__ __forceinline__ Tiles(const Prompt& a, int q0, int n) {
    first = a.window > 0 ? max(0, q0 - a.window + 1) / kRows : 0;
    sinks = min((int)(((long long)a.sinks + kRows - 1) / kRows), first);
    count = sinks + (min(q0 + kRows, n) - 1) / kRows - first + 1;
  }
  __device__ __forceinline__ int key(int i) const { return (i < sinks ? i : first + i - sinks) * kRows; }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kMmaThreads, Mma<DP>::BLOCKS_PER_SM) prompt_mma_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                                                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Prompt a,
                                                                                        int* __restrict__ error_flag) {
  using C = Mma<DP>;
  constexpr int S = C::STAGES, NS = C::SCORES, AHEAD = NS - 1;
  pdl_prologue();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x, b = blockIdx.z, kvh = h / a.group, n = length_of(a, b), D = a.dim;
  const int q0 = (int)(gridDim.y - 1 - blockIdx.y) * kRows;          // the rows that see most go first
  T* out = (T*)a.out + (((long long)b * a.tokens + q0) * a.heads + h) * D;
  const long long pitch = (long long)a.heads * D;
  if (q0 >= n) {
    const uint4 zero = {0, 0, 0, 0};
    for (int i = tid; i < kRows * (D / 8); i += kMmaThreads)
      if (q0 + i / (D / 8) < a.tokens) *(uint4*)(out + i / (D / 8) * pitch + i % (D / 8) * 8) = zero;
    return;
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t *qs = smem, *ks = qs + C::TILE, *vs = ks + S * C::TILE;
  uint64_t* bars = (uint64_t*)(vs + S * C::TILE);
  const uint32_t q_full = smem_u32(bars), k_full = q_full + 8, k_empty = k_full + 8 * S, v_full = k_empty + 8 * S, v_empty = v_full + 8 * S,
                 s_full = v_empty + 8 * S, p_full = s_full + 8 * NS, pv_done = p_full + 16 * NS, drained = pv_done + 8;
  uint32_t* tmem_slot = (uint32_t*)(bars + 3 + 4 * S + 3 * NS);
  volatile int* failed = (volatile int*)(tmem_slot + 1);
  if (tid == 0) {
    for (uint32_t bar = q_full; bar <= drained; bar += 8) mbar_init(bar, bar >= p_full && bar < pv_done ? 4 : 1);
    *failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = *tmem_slot, t_out = tmem + NS * kRows;
  const Tiles tiles(a, q0, n);

  if (warp == 4) {
    // ------------------------------ copies (one lane) -----------------------------------------------------------
    if (lane == 0) {
      bool ok = true;
      int kt = 0, vt = 0;
      const int row = b * a.tokens;
      expect_bytes(q_full, C::TILE);
#pragma unroll
      for (int c = 0; c < C::BLOCKS; ++c) copy_box(smem_u32(qs) + c * C::BLOCK, &tm_q, q_full, c * 64, row + q0, h);
      for (int i = 0; i < tiles.count; ++i) {
        const int s = i % S, parity = ((i / S) & 1) ^ 1, k0 = row + tiles.key(i);
        if (i >= S && !(ok = role_wait(k_empty + 8 * s, parity, failed))) break;
        expect_bytes(k_full + 8 * s, C::TILE);
#pragma unroll
        for (int c = 0; c < C::BLOCKS; ++c) copy_box(smem_u32(ks) + s * C::TILE + c * C::BLOCK, &tm_k, k_full + 8 * s, c * 64, k0, kvh);
        ++kt;
        if (i >= S && !(ok = role_wait(v_empty + 8 * s, parity, failed))) break;
        expect_bytes(v_full + 8 * s, C::TILE);
#pragma unroll
        for (int c = 0; c < C::BLOCKS; ++c) copy_box(smem_u32(vs) + s * C::TILE + c * C::BLOCK, &tm_v, v_full + 8 * s, c * 64, k0, kvh);
        ++vt;
      }
      if (!ok || *failed) {
        // copies that nobody consumed any more: wait for them before the shared memory goes away
        mbar_wait(q_full, 0);
        for (int j = max(0, kt - S); j < kt; ++j) mbar_wait(k_full + 8 * (j % S), (j / S) & 1);
        for (int j = max(0, vt - S); j < vt; ++j) mbar_wait(v_full + 8 * (j % S), (j / S) & 1);
      }
    }
  } else if (warp == 5) {
    // ------------------------------ products --------------------------------------------------------------------
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRows >> 4) << 24);
    constexpr uint32_t idesc_s = common | ((uint32_t)(kRows >> 3) << 17), idesc_o = common | (1u << 16) | ((uint32_t)(DP >> 3) << 17);
    const uint64_t d_q = umma_desc(smem_u32(qs)), d_k = umma_desc(smem_u32(ks)), d_v = values_desc(smem_u32(vs));
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity) {
      ok = __all_sync(0xFFFFFFFFu, ok && role_wait(bar, parity, failed));
      after_sync();
    };
    auto scores = [&](int i) {
      const int s = i % S;
      wait(k_full + 8 * s, (i / S) & 1);
      if (i >= NS) wait(pv_done, (i - NS) & 1);                       // the weights in this place have been read
      if (ok && elect_one()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint64_t at = (uint64_t)((kk / 4 * C::BLOCK + kk % 4 * 32) >> 4);
          mma_smem(tmem + i % NS * kRows, d_q + at, d_k + (uint64_t)((s * C::TILE) >> 4) + at, idesc_s, kk > 0);
        }
        commit(k_empty + 8 * s);
        commit(s_full + 8 * (i % NS));
      }
      __syncwarp();
    };
    wait(q_full, 0);
    for (int i = 0; i < AHEAD && i < tiles.count && ok; ++i) scores(i);
    for (int i = 0; i < tiles.count && ok; ++i) {
      if (i + AHEAD < tiles.count) scores(i + AHEAD);
      if (!ok) break;
      const int s = i % S, k0 = tiles.key(i);
      wait(v_full + 8 * s, (i / S) & 1);
      if (ok && k0 + kRows > n) {
        // values behind the sequence are not zero times a weight of zero where they are no numbers: they go
        const int gone = k0 + kRows - n;
        for (int p = lane; p < C::BLOCKS * gone * 8; p += 32) {
          const int c = p / (gone * 8), r = kRows - gone + p % (gone * 8) / 8;
          *(uint4*)(vs + s * C::TILE + c * C::BLOCK + r * 128 + p % 8 * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        wait(p_full + 16 * (i % NS) + 8 * half, (i / NS) & 1);
        if (ok && elect_one()) {
#pragma unroll
          for (int kk = half * (kRows / 32); kk < (half + 1) * (kRows / 32); ++kk)
            mma_tmem(t_out, tmem + i % NS * kRows + kk * 8, d_v + (uint64_t)((s * C::TILE + kk * 2048) >> 4), idesc_o, i > 0 || kk > 0);
          if (half) {
            commit(v_empty + 8 * s);
            commit(pv_done);
          }
        }
        __syncwarp();
      }
    }
    if (!ok || *failed) {                                            // tensor memory goes back only when no product is left
      if (elect_one()) commit(drained);
      __syncwarp();
      mbar_wait(drained, 0);
    }
  } else {
    // ------------------------------ rows: weights, then the result ------------------------------------------------
    const uint32_t mine = (uint32_t)(32 * warp) << 16;
    const int row = q0 + tid;
    // f16: weights in units that keep the small ones out of its subnormal range
    constexpr float shift = std::is_same<T, __half>::value ? 6.f : 0.f;
    float m = neg_inf(), l = 0.f;
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity) {
      ok = __all_sync(0xFFFFFFFFu, role_wait(bar, parity, failed));
      after_sync();
      return ok;
    };
    for (int i = 0; i < tiles.count; ++i) {
      const int k0 = tiles.key(i);
      const uint32_t t_s = tmem + mine + i % NS * kRows;
      if (!wait(s_full + 8 * (i % NS), (i / NS) & 1)) break;
      uint32_t s[kRows];
#pragma unroll
      for (int c = 0; c < kRows; c += 32) load32(t_s + c, s + c);
      loaded();
#pragma unroll
      for (int c = 0; c < kRows; c += 32) settle(s + c);
      // masks at the edges only: the last key that the row sees, the first of its window, the sinks
      const bool late = k0 + kRows - 1 > q0, early = a.window > 0 && q0 + kRows - 1 - k0 >= a.window && k0 + kRows > a.sinks;
      if (early && k0 < a.sinks) {
        const int least = row - a.window + 1 - k0, always = a.sinks - k0;
#pragma unroll
        for (int k = 0; k < kRows; ++k)
          if (k < least && k >= always) s[k] = 0xFF800000u;
      } else if (early) {
        const int least = row - a.window + 1 - k0;
#pragma unroll
        for (int k = 0; k < kRows; ++k)
          if (k < least) s[k] = 0xFF800000u;
      }
      if (late) {
        const int most = row - k0;
#pragma unroll
        for (int k = 0; k < kRows; ++k)
          if (k > most) s[k] = 0xFF800000u;
      }
      float top[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
      for (int k = 0; k < kRows; k += 2) top[k / 2 % 4] = max3(top[k / 2 % 4], __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
      const float best = fmaxf(max3(top[0], top[1], top[2]), top[3]);
      const bool grown = best > m && (best - m) * a.scale > kGrowth;
      if (__any_sync(0xFFFFFFFFu, grown)) {
        const float now = fmaxf(m, best), keep = m == neg_inf() ? 0.f : power((m - now) * a.scale);
        m = now;
        l *= keep;
        if (i > 0) {
          if (!wait(pv_done, (i - 1) & 1)) break;
#pragma unroll 1
          for (int c = 0; c < DP; c += 32) {
            uint32_t o[32];
            load32(t_out + mine + c, o);
            loaded();
            settle(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            store32(t_out + mine + c, o);
          }
        }
      }
      const float ref = m == neg_inf() ? 0.f : m * a.scale - shift;
      const uint64_t scale = two(a.scale, a.scale), minus = two(-ref, -ref);
      uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t p[32];
#pragma unroll
        for (int k = 0; k < kRows / 2; k += 2) {
          const uint64_t x = fma2(two(s[half * (kRows / 2) + k], s[half * (kRows / 2) + k + 1]), scale, minus);
          const float a0 = power(first(x)), a1 = power(second(x));
          sum[k / 2 % 4] = add2(sum[k / 2 % 4], two(a0, a1));
          p[k / 2] = pair16<T>(a0, a1);
        }
        store32(t_s + half * 32, p);
        stored();
        before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 16 * (i % NS) + 8 * half);
      }
      const uint64_t all = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
      l += first(all) + second(all);
    }
    if (ok && wait(pv_done, (tiles.count - 1) & 1)) {
      const bool some = row < n;
      const float inv = some && (l > 0.f || l != l) ? 1.f / l : 0.f;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        load32(t_out + mine + c, o);
        loaded();
        settle(o);
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (row < a.tokens && c + e < D) {
            uint4 v = {0, 0, 0, 0};
            if (some) {
              v.x = pair16<T>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
              v.y = pair16<T>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
              v.z = pair16<T>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
              v.w = pair16<T>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
            }
            *(uint4*)(out + tid * pitch + c + e) = v;
          }
        }
      }
    }
  }
  before_sync();
  __syncthreads();
  if (tid == 0 && *failed) atomicAdd(error_flag, 1);
  if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLUMNS) : "memory");
}

size_t fma_smem(int dim) { return (size_t)(3 * kTile * (dim + 4) + kTile * kScoreRow) * 4; }

template <typename T>
cudaError_t launch_fma(const Prompt& a, cudaStream_t stream, int* launches) {
  static bool done[64] = {};
  if (cudaError_t e = allow_smem(prompt_fma_kernel<T>, fma_smem(256), done)) return e;
  return launch_op(prompt_fma_kernel<T>, dim3((unsigned)((a.tokens + kTile - 1) / kTile), (unsigned)a.heads, (unsigned)a.batch), 256, fma_smem(a.dim),
                   stream, launches, a);
}

template <typename T, int DP>
cudaError_t launch_mma(const Prompt& a, int* error_flag, cudaStream_t stream, int* launches, const char** why) {
  static bool done[64] = {};
  if (cudaError_t e = allow_smem(prompt_mma_kernel<T, DP>, Mma<DP>::SMEM, done)) return e;
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
  return launch_op(prompt_mma_kernel<T, DP>, dim3((unsigned)a.heads, (unsigned)((a.tokens + kRows - 1) / kRows), (unsigned)a.batch), kMmaThreads, Mma<DP>::SMEM, stream,
                   launches, maps[0], maps[1], maps[2], a, error_flag);
}
template <typename T>
cudaError_t launch_16bit(const Prompt& a, int* error_flag, cudaStream_t stream, int* launches, const char** why) {
  if (a.dim <= 64) return launch_mma<T, 64>(a, error_flag, stream, launches, why);
  if (a.dim <= 128) return launch_mma<T, 128>(a, error_flag, stream, launches, why);
  return launch_mma<T, 256>(a, error_flag, stream, launches, why);
}

}  // namespace

const char* window_attention_plan(OperatorLaunch& op) {
  if (op.heads > 65535 || op.batch > 65535) return "more than 65535 heads or sequences";
  if (op.tokens > 65535 * kTile) return "prompts of more than 65535 tiles of 64 tokens";
  if ((long long)op.batch * op.tokens >= (1LL << 31)) return "2^31 tokens and more";
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
  if (op.type == 0) return launch_fma<float>(a, stream, launches);
  if (op.type == 1) return launch_16bit<__nv_bfloat16>(a, error_flag, stream, launches, why);
  return launch_16bit<__half>(a, error_flag, stream, launches, why);
}

}  // namespace b200
