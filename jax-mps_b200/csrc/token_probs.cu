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
  float m, s, u;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == neg_inf()) return {m, a.s + b.s, a.u + b.u};
  const float da = a.m - m, db = b.m - m, fa = __expf(da), fb = __expf(db);
  // a side without weight adds nothing, however far it is below (its product with the distance could overflow)
  return {m, fa * a.s + fb * b.s, (fa == 0.f ? 0.f : fa * (a.u + a.s * da)) + (fb == 0.f ? 0.f : fb * (b.u + b.s * db))};
}
template <typename F>
__device__ __forceinline__ Sums block_join(Sums v, F* shared, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, {__shfl_xor_sync(0xFFFFFFFFu, v.m, o), __shfl_xor_sync(0xFFFFFFFFu, v.s, o), __shfl_xor_sync(0xFFFFFFFFu, v.u, o)});
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) shared[warp] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < warps; ++w) v = join(v, shared[w]);
  return v;
}

// Order of the alternatives: larger logits first, equal ones by their number; NaN behind every number, -0 like +0.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0u;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

struct Rows {
  const void* x;
  const int* tokens;
  float *log_prob, *entropy, *normalizer, *remainder, *top_values;
  int* top_ids;
  int vocab, top;
};

// A block per row; the best alternatives one after another, each the first in order behind the one before.
template <typename T>
__global__ void __launch_bounds__(256) probs_simple_kernel(const __grid_constant__ Rows a) {
  pdl_prologue();
  __shared__ Sums shared[8];
  __shared__ unsigned long long best[8];
  const long long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.vocab;
  Sums v = {neg_inf(), 0.f, 0.f};
  for (int j = threadIdx.x; j < a.vocab; j += 256) {
    const float f = to_float(x[j]);
    v = f == neg_inf() ? v : join(v, {f, 1.f, 0.f});
    if (f != f) v.s = f;
  }
  v = block_join(v, shared, 8);
  const float ls = logf(v.s), n = v.m + ls;
  if (threadIdx.x == 0) {
    const int t = a.tokens[row];
    a.log_prob[row] = t >= 0 && t < a.vocab ? (to_float(x[t]) - v.m) - ls : 0.f;
    a.entropy[row] = ls - v.u / v.s;
    a.normalizer[row] = n;
    a.remainder[row] = (v.m - n) + ls;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long mine = 0;
    for (int j = threadIdx.x; j < a.vocab; j += 256) {
      const unsigned long long key = (unsigned long long)order_of(to_float(x[j])) << 32 | (0xFFFFFFFFu - (unsigned)j);
      if (key < last && key > mine) mine = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { const unsigned long long w = __shfl_xor_sync(0xFFFFFFFFu, mine, o); mine = w > mine ? w : mine; }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) mine = best[w] > mine ? best[w] : mine;
    last = mine;
    const int j = (int)(0xFFFFFFFFu - (unsigned)mine);
    if (threadIdx.x == 0) {
      a.top_values[row * a.top + k] = (to_float(x[j]) - v.m) - ls;
      a.top_ids[row * a.top + k] = j;
    }
  }
}

struct Grad {
  const void* x;
  const int* tokens;
  const float *normalizer, *remainder, *entropy, *d_log_prob, *d_entropy, *d_normalizer;
  void* dx;
  int vocab;
};

template <typename T>
__global__ void __launch_bounds__(256) probs_grad_simple_kernel(const __grid_constant__ Grad a) {
  pdl_prologue();
  const long long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.vocab;
  T* dx = (T*)a.dx + row * a.vocab;
  const int t = a.tokens[row];
  const float n = a.normalizer[row], low = a.remainder[row], h = a.entropy[row], dh = a.d_entropy[row], dl = t >= 0 && t < a.vocab ? a.d_log_prob[row] : 0.f;
  const float c = a.d_normalizer[row] - dl;
  for (int j = threadIdx.x; j < a.vocab; j += 256) {
    const float y = (to_float(x[j]) - n) - low, p = __expf(y);
    const float e = p > 0.f ? p * (y + h) : p;
    dx[j] = from_float<T>((j == t ? dl : 0.f) + p * c - dh * e);
  }
}

template <typename T>
cudaError_t launch_rows(const Rows& a, long long rows, cudaStream_t stream, int* launches) {
  return launch_op(probs_simple_kernel<T>, dim3((unsigned)rows), 256, 0, stream, launches, a);
}
template <typename T>
cudaError_t launch_grad(const Grad& a, long long rows, cudaStream_t stream, int* launches) {
  return launch_op(probs_grad_simple_kernel<T>, dim3((unsigned)rows), 256, 0, stream, launches, a);
}

}  // namespace

const char* token_log_probs_plan(OperatorLaunch& op) {
  if (op.rows >= (1LL << 31)) return "2^31 rows and more";
  op.scratch_bytes = 0;
  op.launches = 1;
  return nullptr;
}

cudaError_t launch_token_log_probs(const OperatorLaunch& op, void* const* args, void*, cudaStream_t stream, int* launches) {
  Rows a = {};
  const int results = op.top ? 6 : 4;
  a.log_prob = (float*)args[0];
  a.entropy = (float*)args[1];
  a.normalizer = (float*)args[2];
  a.remainder = (float*)args[3];
  if (op.top) { a.top_values = (float*)args[4]; a.top_ids = (int*)args[5]; }
  a.x = args[results];
  a.tokens = (const int*)args[results + 1];
  a.vocab = op.vocab;
  a.top = op.top;
  if (op.type == 0) return launch_rows<float>(a, op.rows, stream, launches);
  if (op.type == 1) return launch_rows<__nv_bfloat16>(a, op.rows, stream, launches);
  return launch_rows<__half>(a, op.rows, stream, launches);
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
  if (op.type == 0) return launch_grad<float>(a, op.rows, stream, launches);
  if (op.type == 1) return launch_grad<__nv_bfloat16>(a, op.rows, stream, launches);
  return launch_grad<__half>(a, op.rows, stream, launches);
}

}  // namespace b200
