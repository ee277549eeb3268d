// What the row-wise kernels share (layer_norm.hip, token_probs.hip): the
// element types, and sums and maxima over a wave and a workgroup.
#pragma once
#include <hip/hip_runtime.h>

#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// f32 -> T, to the nearest (ties to even) for the 16-bit types
template <typename T>
__device__ __forceinline__ T from_f(float f) { return (T)f; }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}

// Sum over the workgroup, in every thread.  `tmp`: one float for each wave,
// free again after the call.
__device__ __forceinline__ float block_sum(float v, float* tmp) {
  const int waves = blockDim.x / WAVE;
  v = wave_sum(v);
  if (waves == 1) return v;
  if ((threadIdx.x & (WAVE - 1)) == 0) tmp[threadIdx.x / WAVE] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < waves; ++i) v += tmp[i];
  __syncthreads();
  return v;
}

__device__ __forceinline__ float block_max(float v, float* tmp) {
  const int waves = blockDim.x / WAVE;
  v = wave_max(v);
  if (waves == 1) return v;
  if ((threadIdx.x & (WAVE - 1)) == 0) tmp[threadIdx.x / WAVE] = v;
  __syncthreads();
  v = tmp[0];
  for (int i = 1; i < waves; ++i) v = fmaxf(v, tmp[i]);
  __syncthreads();
  return v;
}

// one case for each element type; F is a macro of the type
#define ROW_TYPE_SWITCH(code, F)                                             \
  switch (code) {                                                            \
    case ROW_BF16: F(bf16_t); break;                                         \
    case ROW_F16: F(f16_t); break;                                           \
    case ROW_F32: F(float); break;                                           \
    default: throw std::runtime_error("row kernels: unknown element type");  \
  }
