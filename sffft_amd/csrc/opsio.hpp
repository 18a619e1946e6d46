// Loads, stores and conversions that the sequence-mixing operators share. Activations are fp32 or
// bf16 (uint16_t bit patterns); arithmetic is fp32. Rounding to bf16 is to nearest even.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sffft {
namespace ops {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// two values to bf16 in one dword
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(uint16_t* p, float x) { *p = (uint16_t)pack_bf16(x, x); }

// __syncthreads with its wait for LDS written out: at the head of a loop the compiler weakened the one it inserts to
// none, with LDS writes of the loop's end still outstanding. (0xc07f: lgkmcnt 0, the other counters not waited for.)
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// N consecutive elements as fp32; p aligned to them
template <int N>
__device__ __forceinline__ void load(const float* p, float (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = p[i];
  }
}
template <int N>
__device__ __forceinline__ void load(const uint16_t* p, float (&x)[N]) {
  if constexpr (N % 4 == 0) {
    uint32_t w[N / 2];
    if constexpr (N % 8 == 0) {
#pragma unroll
      for (int i = 0; i < N / 2; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + 2 * i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; i += 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p + 2 * i);
        w[i] = v.x, w[i + 1] = v.y;
      }
    }
#pragma unroll
    for (int i = 0; i < N / 2; i++) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f32(p[i]);
  }
}
template <int N>
__device__ __forceinline__ void store(float* p, const float (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = x[i];
  }
}
template <int N>
__device__ __forceinline__ void store(uint16_t* p, const float (&x)[N]) {
  if constexpr (N % 4 == 0) {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; i++) w[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    if constexpr (N % 8 == 0) {
#pragma unroll
      for (int i = 0; i < N / 2; i += 4)
        *reinterpret_cast<uint4*>(p + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; i += 2) *reinterpret_cast<uint2*>(p + 2 * i) = make_uint2(w[i], w[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) put(p + i, x[i]);
  }
}

}  // namespace ops
}  // namespace sffft
