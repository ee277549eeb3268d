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

// Over the 64 lanes of a wave, all of them at work; the result in every lane.
// Sixteen lanes are joined through the operands of the instructions
// themselves (a shuffle goes through LDS, at ten times the delay).
template <int CTRL, typename V>
__device__ __forceinline__ V other_lane(V v) {
  return __builtin_bit_cast(
      V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf,
                                  true));
}
template <typename V>
__device__ __forceinline__ V lane_of(V v, int lane) {
  return __builtin_bit_cast(
      V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
template <typename V, typename F>
__device__ __forceinline__ V wave_join(V v, F f) {
  v = f(v, other_lane<0xb1>(v));     // lanes 1 0 3 2
  v = f(v, other_lane<0x4e>(v));     // 2 3 0 1
  v = f(v, other_lane<0x141>(v));    // 7 ... 0
  v = f(v, other_lane<0x140>(v));    // 15 ... 0
  return f(f(lane_of(v, 0), lane_of(v, 16)),
           f(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_join(v, [](float a, float b) { return a + b; });
}
// (in the last lane alone)
__device__ __forceinline__ float wave_sum_last(float v) {
#define ROW_STEP(CTRL, ROWS)                                                 \
  v += __builtin_bit_cast(                                                   \
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),      \
                                         CTRL, ROWS, 0xf, false))
  ROW_STEP(0x111, 0xf);    // from the lane 1, 2, 4, 8 before in the row of 16
  ROW_STEP(0x112, 0xf);
  ROW_STEP(0x114, 0xf);
  ROW_STEP(0x118, 0xf);
  ROW_STEP(0x142, 0xa);    // the rows' last lanes to the next rows
  ROW_STEP(0x143, 0xc);
#undef ROW_STEP
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_join(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ int wave_max(int v) {
  return wave_join(v, [](int a, int b) { return max(a, b); });
}
__device__ __forceinline__ int wave_min(int v) {
  return wave_join(v, [](int a, int b) { return min(a, b); });
}
__device__ __forceinline__ int wave_sum(int v) {
  return wave_join(v, [](int a, int b) { return a + b; });
}

// What the lanes of a wave have written to LDS, or read from it, before this is
// done for those that read, or write, it afterwards.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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

// The largest of three, NaN left aside.  (fmaxf of loaded values takes two
// more instructions each, which make them canonical.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// 16 bytes of a row.  A row may begin at any element, so these loads and
// stores ask for no more than an element's alignment.
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef u32x4 __attribute__((aligned(2))) u32x4_any;

template <typename T>
struct Pack {
  static constexpr int N = 16 / sizeof(T);
  u32x4 raw;

  __device__ __forceinline__ void load(const T* p) {
    __builtin_memcpy(&raw, p, 16);
  }
  // of what is read once: 6.8 instead of 6.1 TB/s over 512 MB
  __device__ __forceinline__ void load_once(const T* p) {
    raw = __builtin_nontemporal_load((const u32x4_any*)p);
  }
  __device__ __forceinline__ void store(T* p) const {
    __builtin_memcpy(p, &raw, 16);
  }
  __device__ __forceinline__ void store_once(T* p) const {
    __builtin_nontemporal_store(raw, (u32x4_any*)p);
  }
  // The compiler forgets what it knows of the elements, so that it takes
  // them apart again where they are used again, instead of holding them in
  // 32 bits each from one use to the other.
  __device__ __forceinline__ void forget() { asm volatile("" : "+v"(raw)); }
  __device__ __forceinline__ void fill(float v) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = from_f<T>(v);
    __builtin_memcpy(&raw, t, 16);
  }
  // (bf16 by hand: the compiler would otherwise turn what is done with the
  // values back into steps of 16 bits, with a rounding after each)
  __device__ __forceinline__ void get(float* v) const {
    if constexpr (__is_same(T, bf16_t)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(raw[i] << 16);
        v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
      }
    } else {
      T t[N];
      __builtin_memcpy(t, &raw, 16);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)t[i];
    }
  }
  __device__ __forceinline__ void set(const float* v) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = from_f<T>(v[i]);
    __builtin_memcpy(&raw, t, 16);
  }
};

// one case for each element type; F is a macro of the type
#define ROW_TYPE_SWITCH(code, F)                                             \
  switch (code) {                                                            \
    case ROW_BF16: F(bf16_t); break;                                         \
    case ROW_F16: F(f16_t); break;                                           \
    case ROW_F32: F(float); break;                                           \
    default: throw std::runtime_error("row kernels: unknown element type");  \
  }
