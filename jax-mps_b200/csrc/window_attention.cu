// Causal attention of whole prompts with an optional sliding window and sinks (custom call b200.window_attention).
//
//   out[b, i, h] = sum_j w_j v_j,  w = softmax_j(scale * q[b, i, h] . k[b, j, h / group])  over j <= i with no window, i - j < window
//   or j < sinks; rows from a sequence's length on are zero.
//
// Sums, maxima and normalisers are held in 32 bits; tiles of keys that no row of a tile of queries sees are not read.
#include <algorithm>

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

size_t fma_smem(int dim) { return (size_t)(3 * kTile * (dim + 4) + kTile * kScoreRow) * 4; }

template <typename T>
cudaError_t launch_fma(const Prompt& a, cudaStream_t stream, int* launches) {
  static bool done[64] = {};
  if (cudaError_t e = allow_smem(prompt_fma_kernel<T>, fma_smem(256), done)) return e;
  return launch_op(prompt_fma_kernel<T>, dim3((unsigned)((a.tokens + kTile - 1) / kTile), (unsigned)a.heads, (unsigned)a.batch), 256, fma_smem(a.dim),
                   stream, launches, a);
}

}  // namespace

const char* window_attention_plan(OperatorLaunch& op) {
  if (op.heads > 65535 || op.batch > 65535) return "more than 65535 heads or sequences";
  if (op.tokens >= (1 << 30)) return "prompts of 2^30 tokens and more";
  op.scratch_bytes = 0;
  op.launches = 1;
  return nullptr;
}

cudaError_t launch_window_attention(const OperatorLaunch& op, void* const* args, void*, int*, cudaStream_t stream, int* launches, const char**) {
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
  if (op.type == 1) return launch_fma<__nv_bfloat16>(a, stream, launches);
  return launch_fma<__half>(a, stream, launches);
}

}  // namespace b200
