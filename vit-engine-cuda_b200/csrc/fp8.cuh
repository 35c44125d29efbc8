// Shared by the FP8 operators (quantize_fp8.cu, gemm_fp8.cu): element types,
// vector loads widened to fp32, and the code of one block.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "vitb200.h"

namespace vitb200 {

// Columns (and, for weights, rows) that share one scale.
constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;        // largest e4m3 magnitude
constexpr float kFp8AmaxFloor = 1e-30f; // blocks below this are scaled as if they reached it

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Four consecutive elements, aligned to their total size (16 or 8 bytes).
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 t = *reinterpret_cast<const float4*>(p);
  v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
}
__device__ __forceinline__ void load4(const __half* p, float (&v)[4]) {
  const uint2 t = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&t.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 t = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(t.x << 16), v[1] = __uint_as_float(t.x & 0xffff0000u);
  v[2] = __uint_as_float(t.y << 16), v[3] = __uint_as_float(t.y & 0xffff0000u);
}

__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  uint2 t;
  T* e = reinterpret_cast<T*>(&t);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<uint2*>(p) = t;
}

// Largest magnitude of a lane's values, as the bits of |v|: unsigned order is
// the order of the magnitudes, with infinity above every number and NaN above
// infinity, so that one NaN marks its whole block instead of being skipped.
__device__ __forceinline__ uint32_t abs_bits_max(const float (&v)[4], uint32_t m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// The codes of a block with largest magnitude a: e4m3(448 * x / a), each
// quotient rounded once. A 16-bit x makes 448 * x exact, and such quotients
// often lie midway between two codes (a a power of two, say), so x times a
// rounded reciprocal would pick the wrong neighbour. Division by Markstein's
// step instead: with y = 1 / a correctly rounded, q0 = n * y,
// q = q0 + (n - q0 * a) * y is the correctly rounded n / a (the remainder is
// exact in one FMA) as long as nothing leaves the normal range, which dividing
// both by a's power of two ensures. Four operations an element instead of a
// general division's ten.
struct Fp8Scale {
  float a1;  // a / 2^e in [1, 2)
  float y;   // 1 / a1
  float k;   // 448 / 2^e, exact

  __device__ __forceinline__ explicit Fp8Scale(float a) {
    const uint32_t bits = __float_as_uint(a);
    const int e = static_cast<int>(bits >> 23) - 127;
    a1 = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
    y = __frcp_rn(a1);
    k = __uint_as_float((static_cast<uint32_t>(135 - e) << 23) | 0x600000u);
    if (e == 128) {  // infinity: finite values become 0; NaN: all values NaN
      a1 = 1.f;
      k = 1.f;
      y = (bits & 0x7fffffu) ? __uint_as_float(0x7fc00000u) : 0.f;
    }
  }
  __device__ __forceinline__ float value(float x) const {
    const float n = x * k;
    const float q0 = n * y;
    return fmaf(fmaf(-q0, a1, n), y, q0);
  }
  // Four codes, the first in the lowest byte.
  __device__ __forceinline__ uint32_t codes(const float (&v)[4]) const {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(value(v[0]), value(v[1])),
                                                 __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(value(v[2]), value(v[3])),
                                                 __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
};

// The block's magnitude as the scale uses it.
__device__ __forceinline__ float fp8_amax(uint32_t bits) {
  const float a = __uint_as_float(bits);
  return a < kFp8AmaxFloor ? kFp8AmaxFloor : a;  // NaN stays NaN
}

}  // namespace vitb200
