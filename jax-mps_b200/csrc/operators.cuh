// Device and launch helpers of the operator kernels (paged_attention.cu, window_attention.cu, token_probs.cu, pages.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.h"
#include "operators.h"
#include "tc_util.cuh"

namespace b200 {

// Cleared by set_operators_programmatic_launch: plain launches.
extern bool operators_programmatic_launch;

constexpr int kSMs = 148;

namespace {

// With programmatic stream serialization, like every kernel of a plan: each of these kernels begins with pdl_prologue.
template <typename... P, typename... A>
cudaError_t launch_op(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, int* launches, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = operators_programmatic_launch ? 1 : 0;
  if (launches) (*launches)++;
  return launch_kernel(cfg, kernel, std::forward<A>(args)...);
}

// More shared memory than 48 KB has to be asked for, once per kernel and device. It counts as asked for behind the call and not in front of
// it: another client's thread may be about to launch the same kernel.
template <typename K>
cudaError_t allow_smem(K* kernel, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
  if (known && __atomic_load_n(&done[dev], __ATOMIC_ACQUIRE)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && known) __atomic_store_n(&done[dev], true, __ATOMIC_RELEASE);
  return e;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// 16 bytes of T as floats.
template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); };
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[Pack<T>::N]) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < Pack<T>::N; ++i) f[i] = to_float(e[i]);
}

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
// 2^v; denormal results are zero.
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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

}  // namespace
}  // namespace b200
