// Shared by the three forms of cross_attention (cross_attention.cu: 128-row tiles
// on tcgen05; cross_attention_rows.cu: 64-row tiles; cross_attention_token.cu: up to
// 16 rows per key head).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <limits>
#include <type_traits>

#include "common.cuh"
#include "engine.h"
#include "vitb200.h"

namespace vitb200 {

constexpr int kCrossMaxSplit = 8;  // CTAs that share an item's keys: a portable cluster
constexpr int kTokenRows = 16;     // rows per key head the token form takes
constexpr float kLog2e = 1.44269504088896340736f;

// The softmax scale in log2 units. Masked scores are infinite, and infinity times
// zero is NaN: the smallest float in place of zero moves no score by more than 5e-7.
inline float cross_scale(float scale) {
  const float c = scale * kLog2e;
  return c == 0.f ? std::numeric_limits<float>::denorm_min() : c;
}

// Probabilities are exponentials lifted by 2^kLift: the largest of a row is near
// 2^kLift instead of 1, and O and the sum it is divided by are lifted alike. bf16 has
// fp32's range. fp16 ends at 2^16 and 2^-25: at 1, tens of thousands of keys whose
// probabilities lie below that would be lost for the product with V while the sum
// counts them; at 2^15 they may be 2^-40 of the largest.
template <typename T>
constexpr float kLift = std::is_same_v<T, __half> ? 15.f : 0.f;

// Exponents are x * c - m in one FMA where m is the rounded product of the largest x,
// so all of a row's are off by that rounding, up to 2^-24 |m|, which the quotient o =
// O / l does not see. Past this m it would leave the range of fp16 or of the exponent:
// such a row's products are rounded, or the largest x subtracted first.
constexpr float kHugeScore = 1048576.f;
// (m - 15 would be rounded as coarsely, so the lift is added by itself.)
__device__ __forceinline__ float huge_exponent(float x, float c, float m, float up) {
  return __fadd_rn(__fsub_rn(__fmul_rn(x, c), m), up);
}

struct CrossTokenArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* parts;     // workspace of the streaming form
  const int* lens;  // [B] or null
  int B, Tq, Tk, kv_heads;
  int group;   // query heads per key head
  int rows;    // group * Tq <= 16
  float c;     // scale * log2(e)
  int64_t q_row, q_batch, k_row, k_batch, v_row, v_batch, o_row;
};
int cross_attention_rows_prepare_device();
int cross_attention_rows_launch(const CrossProblem& p, cudaStream_t s);

int cross_attention_token_prepare_device();
// Bytes of workspace its launch needs (0 where a CTA per key head does).
size_t cross_attention_token_workspace(const CrossProblem& p);
int cross_attention_token_launch(const CrossProblem& p, cudaStream_t s);

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Floats of a partial result, in this CTA's shared memory or a peer's.
__device__ __forceinline__ float ld_partial(uint32_t addr, bool remote) {
  float v;
  if (remote)
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_partial4(uint32_t addr, bool remote) {
  if (remote) return ld_shared_cluster_f4(addr);
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// D += A B of one warp: 16 x 16 by 16 x 8, fp32 sums.
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                            uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The two values of a packed pair.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t p) {
  if constexpr (std::is_same_v<T, __half>)
    return __half22float2(*reinterpret_cast<const __half2*>(&p));
  else
    return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}

// Sixteen bytes from global to shared memory, past L1; zeros where `inside` is
// false (the address is not read then).
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool inside) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(inside ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace vitb200
