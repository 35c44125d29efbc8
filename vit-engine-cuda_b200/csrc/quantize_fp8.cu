// FP8 operand preparation: e4m3 codes with one fp32 scale per block, from
// rows as they are (quantize_fp8) or through a LayerNorm (layernorm_fp8).
//
//   a = max |x| over the block, scale = a / 448, code = e4m3(448 * x / a)
//
// A block is 128 columns of one row (activations) or 128 x 128 (weights); the
// last block of a row or column may be smaller. All three kernels read every
// element once, hold it in registers while the block's maximum is found, and
// write one byte: they are bound by HBM traffic.
#include <algorithm>

#include "engine.h"
#include "fp8.cuh"

namespace vitb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// The four columns of lane `lane` in the block starting at c0, widened to
// fp32; columns from K on read as zero. VEC: whole vectors (K % 4 == 0 and the
// rows aligned to four elements), so a lane's columns are all inside or all
// outside.
template <typename T, bool VEC>
__device__ __forceinline__ void load_lane(const T* row, int c, int K, float (&v)[4]) {
  if constexpr (VEC) {
    if (c < K) {
      load4(row + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i < K ? to_f32(row[c + i]) : 0.f;
  }
}

// 1 x 128 blocks: a warp holds a block, four columns a lane, and takes UNROLL
// consecutive blocks of the matrix at a time so that their loads are in flight
// together. `redux` finds a block's maximum in one instruction.
template <typename T, bool VEC, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int kb,
                         uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scales) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t blocks = rows * kb;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps * UNROLL;
  for (int64_t b0 = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * UNROLL;
       b0 < blocks; b0 += step) {
    float v[UNROLL][4];
    int64_t r = b0 / kb;
    int g = static_cast<int>(b0 - r * kb);
    const int64_t r0 = r;
    const int g0 = g;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (r < rows) load_lane<T, VEC>(x + r * ldx, g * kFp8Block + 4 * lane, K, v[u]);
      if (++g == kb) g = 0, ++r;
    }
    r = r0, g = g0;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (r < rows) {  // uniform over the warp
        const float a = fp8_amax(__reduce_max_sync(0xffffffffu, abs_bits_max(v[u], 0)));
        const uint32_t codes = Fp8Scale(a).codes(v[u]);
        const int c = g * kFp8Block + 4 * lane;
        if (c < K) *reinterpret_cast<uint32_t*>(q + r * ldq + c) = codes;
        if (lane == 0) scales[r * kb + g] = a / kFp8Max;
      }
      if (++g == kb) g = 0, ++r;
    }
  }
}

// 128 x 128 blocks: a CTA holds a block (16 rows a warp, 64 values a thread).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    quantize_blocks_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int kb,
                           uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scales,
                           int64_t blocks) {
  __shared__ uint32_t part[2][kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  constexpr int kRows = kFp8Block / kWarps;
  int turn = 0;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x, turn ^= 1) {
    const int64_t rb = b / kb;
    const int g = static_cast<int>(b - rb * kb);
    const int64_t r0 = rb * kFp8Block + warp;
    const int c = g * kFp8Block + 4 * lane;
    float v[kRows][4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = r0 + i * kWarps;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = 0.f;
      if (r < rows) load_lane<T, VEC>(x + r * ldx, c, K, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) m = abs_bits_max(v[i], m);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) part[turn][warp] = m;
    __syncthreads();  // `part` alternates: the next block's writes cannot meet these reads
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = max(m, part[turn][w]);
    const float a = fp8_amax(m);
    const Fp8Scale s(a);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = r0 + i * kWarps;
      if (r < rows && c < K) *reinterpret_cast<uint32_t*>(q + r * ldq + c) = s.codes(v[i]);
    }
    if (threadIdx.x == 0) scales[b] = a / kFp8Max;
  }
}

// Sum over the WARPS warps that share a row; every thread gets it.
template <int WARPS>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += part[w];
  }
  return v;
}

// LayerNorm and 1 x 128 blocks in one pass: WARPS warps hold a row of up to
// WARPS * GROUPS blocks (block g in warp g % WARPS), so x is read once, the
// variance is the mean of squared deviations, and y never reaches memory.
template <typename T, bool VEC, int WARPS, int GROUPS>
__global__ void __launch_bounds__(kThreads)
    layernorm_fp8_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                         const float* __restrict__ beta, float eps, int64_t rows, int K, int kb,
                         uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scales) {
  static_assert(WARPS == 1 || WARPS == kWarps, "a row per warp or per CTA");
  __shared__ float part[2][kWarps];
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kRowsPerCta = kWarps / WARPS;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int first = WARPS == 1 ? 0 : warp;  // this warp's first block of the row
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + (WARPS == 1 ? warp : 0);
       r < rows; r += static_cast<int64_t>(gridDim.x) * kRowsPerCta) {
    float v[GROUPS][4];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i)
      load_lane<T, VEC>(x + r * ldx, (first + i * WARPS) * kFp8Block + 4 * lane, K, v[i]);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) sum += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
    const float mean = row_sum<WARPS>(sum, part[0]) / static_cast<float>(K);
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const int c = (first + i * WARPS) * kFp8Block + 4 * lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i][j] = c + j < K ? v[i][j] - mean : 0.f;
        sq = fmaf(v[i][j], v[i][j], sq);
      }
    }
    const float var = row_sum<WARPS>(sq, part[1]) / static_cast<float>(K);
    const float rstd = 1.f / sqrtf(var + eps);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const int g = first + i * WARPS;
      if (g >= kb) break;  // uniform over the warp
      const int c = g * kFp8Block + 4 * lane;
      float ga[4], be[4];
      load_lane<float, VEC>(gamma, c, K, ga);
      load_lane<float, VEC>(beta, c, K, be);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = fmaf(v[i][j] * rstd, ga[j], be[j]);
      const float a = fp8_amax(__reduce_max_sync(0xffffffffu, abs_bits_max(v[i], 0)));
      const uint32_t codes = Fp8Scale(a).codes(v[i]);
      if (c < K) *reinterpret_cast<uint32_t*>(q + r * ldq + c) = codes;
      if (lane == 0) scales[r * kb + g] = a / kFp8Max;
    }
  }
}

// Rows too wide for a CTA's registers: the same three steps, x read again
// (from L2) for each.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
    layernorm_fp8_wide_kernel(const T* __restrict__ x, int64_t ldx,
                              const float* __restrict__ gamma, const float* __restrict__ beta,
                              float eps, int64_t rows, int K, int kb, uint8_t* __restrict__ q,
                              int64_t ldq, float* __restrict__ scales) {
  __shared__ float part[2][kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * ldx;
    float v[4];
    float sum = 0.f;
    for (int g = warp; g < kb; g += kWarps) {
      load_lane<T, VEC>(row, g * kFp8Block + 4 * lane, K, v);
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
    const float mean = row_sum<kWarps>(sum, part[0]) / static_cast<float>(K);
    float sq = 0.f;
    for (int g = warp; g < kb; g += kWarps) {
      const int c = g * kFp8Block + 4 * lane;
      load_lane<T, VEC>(row, c, K, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = c + j < K ? v[j] - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float var = row_sum<kWarps>(sq, part[1]) / static_cast<float>(K);
    const float rstd = 1.f / sqrtf(var + eps);
    for (int g = warp; g < kb; g += kWarps) {
      const int c = g * kFp8Block + 4 * lane;
      float ga[4], be[4];
      load_lane<T, VEC>(row, c, K, v);
      load_lane<float, VEC>(gamma, c, K, ga);
      load_lane<float, VEC>(beta, c, K, be);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c + j < K ? fmaf((v[j] - mean) * rstd, ga[j], be[j]) : 0.f;
      const float a = fp8_amax(__reduce_max_sync(0xffffffffu, abs_bits_max(v, 0)));
      const uint32_t codes = Fp8Scale(a).codes(v);
      if (c < K) *reinterpret_cast<uint32_t*>(q + r * ldq + c) = codes;
      if (lane == 0) scales[r * kb + g] = a / kFp8Max;
    }
  }
}

// CTAs for `work` CTA-sized pieces: enough to fill the GPU eight deep, the
// kernels stride over the rest.
unsigned grid_for(int64_t work) {
  return static_cast<unsigned>(
      std::max<int64_t>(1, std::min<int64_t>(work, static_cast<int64_t>(device_num_sms()) * 8)));
}

template <typename T>
bool vector_rows(const T* x, int64_t ldx, int K) {
  return K % 4 == 0 && ldx % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0;
}

template <typename T, bool VEC>
int quantize_typed(const T* x, int64_t rows, int K, int64_t ldx, int block_rows, uint8_t* q,
                   int64_t ldq, float* scales, cudaStream_t s) {
  const int kb = (K + kFp8Block - 1) / kFp8Block;
  if (block_rows == 1) {
    constexpr int kUnroll = 4;
    const int64_t per_cta = kWarps * kUnroll;
    return launch_kernel(quantize_rows_kernel<T, VEC, kUnroll>,
                         dim3(grid_for((rows * kb + per_cta - 1) / per_cta)), dim3(kThreads), 0, s,
                         1, x, ldx, rows, K, kb, q, ldq, scales);
  }
  const int64_t blocks = (rows + kFp8Block - 1) / kFp8Block * kb;
  return launch_kernel(quantize_blocks_kernel<T, VEC>, dim3(grid_for(blocks)), dim3(kThreads), 0,
                       s, 1, x, ldx, rows, K, kb, q, ldq, scales, blocks);
}

template <typename T, bool VEC>
int layernorm_typed(const T* x, int64_t rows, int K, int64_t ldx, const float* gamma,
                    const float* beta, float eps, uint8_t* q, int64_t ldq, float* scales,
                    cudaStream_t s) {
  const int kb = (K + kFp8Block - 1) / kFp8Block;
  auto go = [&](auto kernel, int rows_per_cta) {
    return launch_kernel(kernel, dim3(grid_for((rows + rows_per_cta - 1) / rows_per_cta)),
                         dim3(kThreads), 0, s, 1, x, ldx, gamma, beta, eps, rows, K, kb, q, ldq,
                         scales);
  };
  // The narrowest form that holds the row: registers, not work, differ.
  if (kb <= 2) return go(layernorm_fp8_kernel<T, VEC, 1, 2>, kWarps);
  if (kb <= 6) return go(layernorm_fp8_kernel<T, VEC, 1, 6>, kWarps);
  if (kb <= 2 * kWarps) return go(layernorm_fp8_kernel<T, VEC, kWarps, 2>, 1);
  if (kb <= 8 * kWarps) return go(layernorm_fp8_kernel<T, VEC, kWarps, 8>, 1);
  return go(layernorm_fp8_wide_kernel<T, VEC>, 1);
}

template <typename F>
int with_type(int type, F&& f) {
  switch (type) {
    case VITB200_F32: return f(static_cast<const float*>(nullptr));
    case VITB200_F16: return f(static_cast<const __half*>(nullptr));
    case VITB200_BF16: return f(static_cast<const __nv_bfloat16*>(nullptr));
    default: return VITB200_E_INVALID_ARG;
  }
}

}  // namespace

int quantize_fp8_launch(const void* x, int type, int64_t rows, int K, int64_t ldx, int block_rows,
                        uint8_t* q, int64_t ldq, float* scales, cudaStream_t s) {
  return with_type(type, [&](auto tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    const T* p = static_cast<const T*>(x);
    return vector_rows(p, ldx, K)
               ? quantize_typed<T, true>(p, rows, K, ldx, block_rows, q, ldq, scales, s)
               : quantize_typed<T, false>(p, rows, K, ldx, block_rows, q, ldq, scales, s);
  });
}

int layernorm_fp8_launch(const void* x, int type, int64_t rows, int K, int64_t ldx,
                         const float* gamma, const float* beta, float eps, uint8_t* q, int64_t ldq,
                         float* scales, cudaStream_t s) {
  return with_type(type, [&](auto tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    const T* p = static_cast<const T*>(x);
    const bool vec = vector_rows(p, ldx, K) && reinterpret_cast<uintptr_t>(gamma) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(beta) % 16 == 0;
    return vec ? layernorm_typed<T, true>(p, rows, K, ldx, gamma, beta, eps, q, ldq, scales, s)
               : layernorm_typed<T, false>(p, rows, K, ldx, gamma, beta, eps, q, ldq, scales, s);
  });
}

}  // namespace vitb200

using namespace vitb200;

namespace {

// Argument checks the two entry points share; 1 = nothing to do.
int check_quantize(const void* x, int type, int64_t rows, int K, int64_t ldx, const uint8_t* q,
                   int64_t ldq, const float* scales) {
  if (rows < 0 || K < 1 || K > (1 << 30) || ldx < K || ldq < K) return VITB200_E_INVALID_ARG;
  if (type < VITB200_F32 || type > VITB200_BF16) return VITB200_E_INVALID_ARG;
  if (ldq % 16 != 0 || reinterpret_cast<uintptr_t>(q) % 16 != 0) return VITB200_E_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(x) % (type == VITB200_F32 ? 4 : 2) != 0)
    return VITB200_E_ALIGNMENT;
  if (rows == 0) return 1;
  return x && q && scales ? 0 : VITB200_E_INVALID_ARG;
}

}  // namespace

extern "C" int vitb200_quantize_fp8(const void* x, int x_type, int64_t rows, int K, int64_t ldx,
                                    int block_rows, uint8_t* q, int64_t ldq, float* scales,
                                    void* stream) {
  try {
    if (block_rows != 1 && block_rows != kFp8Block) return VITB200_E_INVALID_ARG;
    if (int st = check_quantize(x, x_type, rows, K, ldx, q, ldq, scales)) return st > 0 ? 0 : st;
    if (int st = vitb200_init()) return st;
    return quantize_fp8_launch(x, x_type, rows, K, ldx, block_rows, q, ldq, scales,
                               static_cast<cudaStream_t>(stream));
  } catch (...) {
    return VITB200_E_INVALID_ARG;
  }
}

extern "C" int vitb200_layernorm_fp8(const void* x, int x_type, int64_t rows, int K, int64_t ldx,
                                     const float* gamma, const float* beta, float eps, uint8_t* q,
                                     int64_t ldq, float* scales, void* stream) {
  try {
    if (int st = check_quantize(x, x_type, rows, K, ldx, q, ldq, scales)) return st > 0 ? 0 : st;
    if (!gamma || !beta) return VITB200_E_INVALID_ARG;
    if (int st = vitb200_init()) return st;
    return layernorm_fp8_launch(x, x_type, rows, K, ldx, gamma, beta, eps, q, ldq, scales,
                                static_cast<cudaStream_t>(stream));
  } catch (...) {
    return VITB200_E_INVALID_ARG;
  }
}
