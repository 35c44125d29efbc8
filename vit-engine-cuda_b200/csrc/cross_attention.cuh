// Shared by the two forms of cross_attention (cross_attention.cu: row tiles on
// tcgen05; cross_attention_token.cu: up to 16 rows per key head).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "engine.h"
#include "vitb200.h"

namespace vitb200 {

constexpr int kCrossMaxSplit = 8;  // CTAs that share an item's keys: a portable cluster
constexpr int kTokenRows = 16;     // rows per key head the token form takes
constexpr float kLog2e = 1.44269504088896340736f;

struct CrossTokenArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const int* lens;  // [B] or null
  int Tq, Tk, kv_heads;
  int group;   // query heads per key head
  int rows;    // group * Tq <= 16
  int nsplit;  // CTAs per key head
  float c;     // scale * log2(e)
  int64_t q_row, q_batch, k_row, k_batch, v_row, v_batch, o_row;
};
int cross_attention_token_prepare_device();
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

// Sixteen bytes that are read once: past L1.
__device__ __forceinline__ uint4 ld_stream(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

}  // namespace vitb200
