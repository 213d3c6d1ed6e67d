// The 32x32 matrix instructions of each operand type and the conversions to and
// from fp32, shared by the GEMM-shaped kernels.
#pragma once

#include "sp_common.h"

namespace sp {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

template <typename T>
struct Mfma;

template <>
struct Mfma<_Float16> {
  using frag = half8;
  static constexpr int V = 8;       // elements per 16-byte lane load
  static constexpr int KSTEP = 16;  // reduction indices per step (2 halves x V)
  __device__ static __forceinline__ void mma(const frag& a, const frag& b, floatx16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Mfma<__bf16> {
  using frag = bf16x8;
  static constexpr int V = 8;
  static constexpr int KSTEP = 16;
  __device__ static __forceinline__ void mma(const frag& a, const frag& b, floatx16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Mfma<float> {
  using frag = float4v;
  static constexpr int V = 4;
  static constexpr int KSTEP = 8;
  __device__ static __forceinline__ void mma(const frag& a, const frag& b, floatx16& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[0], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[1], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[2], b[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[3], b[3], c, 0, 0, 0);
  }
};

__device__ __forceinline__ float to_f32(_Float16 v) { return float(v); }
__device__ __forceinline__ float to_f32(__bf16 v) { return float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float v) { return _Float16(v); }
template <>
__device__ __forceinline__ __bf16 from_f32<__bf16>(float v) { return __bf16(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

}  // namespace sp
