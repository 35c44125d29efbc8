// Shared by the FP8 operators (quantize_fp8.cu, gemm_fp8.cu): element types,
// vector loads widened to fp32, and the code of one block.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <string.h>

#include <type_traits>

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

// How rows are read: element by element, in aligned vectors of which a lane's is
// inside the row or not, or in vectors that are all inside (whose checks and
// zeros would be a third of a LayerNorm's instructions).
enum Fp8Rows : int { kScalarRows = 0, kVectorRows = 1, kFullRows = 2 };

// PER consecutive elements, 16 bytes, as they lie in memory: what a lane loads.
template <typename T>
struct Lane16 {
  static constexpr int PER = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void clear() { w = make_uint4(0, 0, 0, 0); }
  // The first min(n, PER) elements from p on, the rest zero.
  template <int ROWS>
  __device__ __forceinline__ void load(const T* p, int n) {
    if constexpr (ROWS == kFullRows) {
      w = *reinterpret_cast<const uint4*>(p);
    } else if constexpr (ROWS == kVectorRows) {
      clear();
      if (n > 0) w = *reinterpret_cast<const uint4*>(p);
    } else {
      T e[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) e[i] = i < n ? p[i] : from_f32<T>(0.f);
      memcpy(&w, e, sizeof(w));
    }
  }
  __device__ __forceinline__ void widen(float2 (&v)[PER / 2]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) {
      if constexpr (sizeof(T) == 4)
        v[i] = make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
      else if constexpr (std::is_same_v<T, __half>)
        v[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      else
        v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    }
  }
};

// Largest magnitude of a lane's values, as the bits of |v|: their unsigned order
// is the order of the magnitudes, with infinity above every number and NaN above
// infinity, and the maximum of three propagates NaN, so that one NaN marks its
// whole block instead of being skipped.
template <int N>
__device__ __forceinline__ uint32_t abs_bits_max(const float2 (&v)[N]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[i].x), "f"(v[i].y));
  return __float_as_uint(m) & 0x7fffffffu;
}

// The codes of a block with largest magnitude a: e4m3(448 * x / a), each
// quotient rounded once. A 16-bit x makes 448 * x exact, and such quotients
// often lie midway between two codes (a a power of two, say), so x times a
// rounded reciprocal would pick the wrong neighbour. Division by Markstein's
// step instead: with y = 1 / a correctly rounded, q0 = n * y,
// q = q0 + (n - q0 * a) * y is the correctly rounded n / a (the remainder is
// exact in one FMA) as long as nothing leaves the normal range, which dividing
// both by a's power of two ensures: four operations an element, two when paired,
// instead of a general division's ten.
struct Fp8Scale {
  float a1;  // a / 2^e in [1, 2)
  float k;   // 448 / 2^e, exact
  float y;   // 1 / a1

  // a1 and k; infinity and NaN (exponent 255) divide by one.
  __device__ __forceinline__ explicit Fp8Scale(float a) {
    const uint32_t bits = __float_as_uint(a);
    const bool finite = bits < 0x7f800000u;
    a1 = finite ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : 1.f;
    // 448 = 1.75 * 2^8: exponent 8 - e, biased 262 - (bits >> 23)
    k = finite ? __uint_as_float(((262u << 23) - (bits & 0x7f800000u)) | 0x600000u) : 1.f;
  }
  // 1 / a1; for infinity 0, so that finite values become 0, and for NaN NaN.
  static __device__ __forceinline__ float reciprocal(float a) {
    const uint32_t bits = __float_as_uint(a);
    if (bits >= 0x7f800000u) return bits == 0x7f800000u ? 0.f : a;
    return __frcp_rn(__uint_as_float((bits & 0x7fffffu) | 0x3f800000u));
  }
  __device__ __forceinline__ float2 value(float2 x) const {
    const float2 n = mul2(x, splat2(k));
    const float2 q0 = mul2(n, splat2(y));
    return fma2(fma2(q0, splat2(-a1), n), splat2(y), q0);
  }
  // Four codes, the first in the lowest byte.
  __device__ __forceinline__ uint32_t codes(float2 v0, float2 v1) const {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(value(v0), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(value(v1), __NV_SATFINITE, __NV_E4M3);
    return __byte_perm(lo, hi, 0x5410);
  }
  // The codes of a lane's values, in memory order.
  template <int N>
  __device__ __forceinline__ void store(uint8_t* q, const float2 (&v)[N]) const {
    if constexpr (N == 2)
      *reinterpret_cast<uint32_t*>(q) = codes(v[0], v[1]);
    else
      *reinterpret_cast<uint2*>(q) = make_uint2(codes(v[0], v[1]), codes(v[2], v[3]));
  }
};

// The block's magnitude as the scale uses it.
__device__ __forceinline__ float fp8_amax(uint32_t bits) {
  const float a = __uint_as_float(bits);
  return a < kFp8AmaxFloor ? kFp8AmaxFloor : a;  // NaN stays NaN
}

}  // namespace vitb200
