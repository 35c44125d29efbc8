// FP8 operand preparation: e4m3 codes with one fp32 scale per block, from
// rows as they are (quantize_fp8) or through a LayerNorm (layernorm_fp8).
//
//   a = max |x| over the block, scale = a / 448, code = e4m3(448 * x / a)
//
// A block is 128 columns of one row (activations) or 128 x 128 (weights); the
// last block of a row or column may be smaller. The kernels read every element
// once, hold it in registers while the block's maximum is found, and write one
// byte: the bound is HBM traffic.
#include <algorithm>

#include "engine.h"
#include "fp8.cuh"

namespace vitb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// A lane holds PER = 16 bytes' worth of elements, a warp 32 * PER columns: one
// block of 128 fp32 columns, or two of a 16-bit type (one per half warp).
template <typename T>
struct Warp {
  static constexpr int PER = Lane16<T>::PER;
  static constexpr int kCols = 32 * PER;
  static constexpr int kBlocks = kCols / kFp8Block;
  static constexpr int kLanes = 32 / kBlocks;  // lanes of a block
  // The lanes that share this lane's block.
  static __device__ __forceinline__ uint32_t mask(int lane) {
    return kBlocks == 1 ? 0xffffffffu : (lane < 16 ? 0x0000ffffu : 0xffff0000u);
  }
};

// The scale work of N warp-loads: a block's reciprocal and scale cost some thirty
// instructions, as much as the rest of its work, so lane u of a block's lanes
// computes load u's for all of them; `get` hands load u's back by a shuffle.
template <typename T, int N>
struct WarpScales {
  float a[N];
  float y, scale;  // lane u of the block's lanes: of load u

  __device__ __forceinline__ void find(const uint32_t (&bits)[N], int lane) {
    const int l = lane % Warp<T>::kLanes;
#pragma unroll
    for (int u = 0; u < N; ++u)
      a[u] = fp8_amax(__reduce_max_sync(Warp<T>::mask(lane), bits[u]));
    float mine = a[0];
#pragma unroll
    for (int u = 1; u < N; ++u) mine = l == u ? a[u] : mine;
    y = Fp8Scale::reciprocal(mine);
    scale = mine / kFp8Max;
  }
  __device__ __forceinline__ Fp8Scale get(int u, int lane) const {
    Fp8Scale s(a[u]);
    s.y = __shfl_sync(0xffffffffu, y, (lane & ~(Warp<T>::kLanes - 1)) + u);
    return s;
  }
};

// 1 x 128 blocks: a warp takes N loads along a row (the last of a row may hold
// fewer blocks), whose elements stay in their own type until they are coded. A
// lane's loads are in flight together, and `redux` finds a block's maximum in one
// instruction.
template <typename T, int ROWS, int N>
__global__ void __launch_bounds__(kThreads)
    quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int kb,
                         int per_row, uint8_t* __restrict__ q, int64_t ldq,
                         float* __restrict__ scales) {
  using W = Warp<T>;
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t pieces = rows * per_row;  // N loads each
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  for (int64_t p = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); p < pieces;
       p += step) {
    const int64_t r = per_row == 1 ? p : p / per_row;
    const int c0 = static_cast<int>(p - r * per_row) * (N * W::kCols) + W::PER * lane;
    const T* row = x + r * ldx + c0;
    Lane16<T> raw[N];
#pragma unroll
    for (int u = 0; u < N; ++u) raw[u].template load<ROWS>(row + u * W::kCols, K - c0 - u * W::kCols);
    uint32_t bits[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float2 v[W::PER / 2];
      raw[u].widen(v);
      bits[u] = abs_bits_max(v);
    }
    WarpScales<T, N> ws;
    ws.find(bits, lane);
    uint8_t* to = q + r * ldq + c0;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const Fp8Scale s = ws.get(u, lane);
      float2 v[W::PER / 2];
      raw[u].widen(v);
      if (ROWS == kFullRows || c0 + u * W::kCols < K) s.store(to + u * W::kCols, v);
    }
    const int g = (c0 - W::PER * lane) / kFp8Block + (lane % W::kLanes) * W::kBlocks +
                  lane / W::kLanes;
    if (lane % W::kLanes < N && g < kb) scales[r * kb + g] = ws.scale;
  }
}

// 128 x 128 blocks: a CTA holds a block, in its own type until it is coded. Loads,
// maximum and stores overlap only between CTAs. Three an SM for 16-bit rows read in 16-byte
// pieces: 4096 x 4096 bf16 12.4 us, 4.1 TB/s, against 12.8 with two or four CTAs and
// 17 with 256 threads (768 x 768, less than a block an SM: 2.6 against 2.3). Rows
// read value by value spill with three, 4096 x 4095 19.1 us against 15.4. A thread
// holds 32 registers of an fp32 block, so two (4096 x 4096: 17.6 us).
constexpr int kBlockThreads = 512;
template <typename T, int ROWS>
__global__ void __launch_bounds__(kBlockThreads, sizeof(T) == 2 && ROWS != kScalarRows ? 3 : 2)
    quantize_blocks_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int kb,
                           uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scales,
                           int64_t blocks) {
  using W = Warp<T>;
  constexpr int kW = kBlockThreads / 32;
  constexpr int kStep = kW * W::kBlocks;         // rows the CTA covers with one load a lane
  constexpr int N = kFp8Block / kStep;
  __shared__ uint32_t part[2][kW];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int turn = 0;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x, turn ^= 1) {
    const int64_t rb = b / kb;
    const int g = static_cast<int>(b - rb * kb);
    const int64_t r0 = rb * kFp8Block + warp * W::kBlocks + lane / W::kLanes;
    const int c = g * kFp8Block + W::PER * (lane % W::kLanes);
    const T* at = x + r0 * ldx + c;
    Lane16<T> raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      raw[i].template load<ROWS>(at + i * kStep * ldx, r0 + i * kStep < rows ? K - c : 0);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float2 v[W::PER / 2];
      raw[i].widen(v);
      m = max(m, abs_bits_max(v));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) part[turn][warp] = m;
    __syncthreads();  // `part` alternates: the next block's writes cannot meet these reads
    m = __reduce_max_sync(0xffffffffu, part[turn][lane % kW]);
    const float a = fp8_amax(m);
    Fp8Scale s(a);
    s.y = Fp8Scale::reciprocal(a);
    uint8_t* to = q + r0 * ldq + c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float2 v[W::PER / 2];
      raw[i].widen(v);
      if (r0 + i * kStep < rows && c < K) s.store(to + i * kStep * ldq, v);
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

// A lane's values minus the mean, zero outside the row; returns sq plus the sum
// of their squares.
template <int ROWS, int P>
__device__ __forceinline__ float2 centre(float2 (&v)[P], float mean, int c, int K, float2 sq) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    v[i] = add2(v[i], splat2(-mean));
    if (ROWS != kFullRows) {
      if (c + (ROWS == kVectorRows ? 0 : 2 * i) >= K) v[i].x = 0.f;
      if (c + (ROWS == kVectorRows ? 0 : 2 * i + 1) >= K) v[i].y = 0.f;
    }
    sq = fma2(v[i], v[i], sq);
  }
  return sq;
}

// v * rstd * gamma + beta (gamma and beta read as zero outside the row).
template <int ROWS, int P>
__device__ __forceinline__ void affine(float2 (&v)[P], float rstd, const float* gamma,
                                       const float* beta, int c, int K) {
#pragma unroll
  for (int i = 0; i < P; i += 2) {
    Lane16<float> g, b;
    float2 gv[2], bv[2];
    g.template load<ROWS>(gamma + c + 2 * i, K - c - 2 * i);
    b.template load<ROWS>(beta + c + 2 * i, K - c - 2 * i);
    g.widen(gv);
    b.widen(bv);
    v[i] = fma2(mul2(v[i], splat2(rstd)), gv[0], bv[0]);
    v[i + 1] = fma2(mul2(v[i + 1], splat2(rstd)), gv[1], bv[1]);
  }
}

// LayerNorm and 1 x 128 blocks in one pass: WARPS warps hold a row of up to
// WARPS * N warp-loads (warp w those from w * N on), so x is read once, the
// variance is the mean of squared deviations, and y never reaches memory. A row's
// chain of two sums, maxima and codes is long next to its loads, so what counts is
// how many rows an SM has under way: with a row per warp, four CTAs (50432 x 768
// fp32: 35 us, 5.5 TB/s; before rows had a form without checks 40, with three CTAs
// 42, with two and the next row's loads ahead 44); with a row per CTA the next row's
// loads go ahead (8192 x 4096 bf16: 43 us).
template <typename T, int ROWS, int WARPS, int N>
__global__ void __launch_bounds__(kThreads, WARPS == 1 ? (N * Lane16<T>::PER > 24 ? 3 : 4)
                                                  : (N >= 4 ? 2 : 4))
    layernorm_fp8_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                         const float* __restrict__ beta, float eps, int64_t rows, int K, int kb,
                         uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ scales) {
  static_assert(WARPS == 1 || WARPS == kWarps, "a row per warp or per CTA");
  using W = Warp<T>;
  __shared__ float part[2][kWarps];
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kRowsPerCta = kWarps / WARPS;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int col0 = WARPS == 1 ? 0 : warp * N * W::kCols;  // this warp's first column
  const int c0 = col0 + W::PER * lane;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRowsPerCta;
  int64_t r = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + (WARPS == 1 ? warp : 0);
  constexpr bool kAhead = WARPS > 1;
  Lane16<T> next[N];
  auto fetch = [&](int64_t row) {
    if (ROWS == kFullRows && row >= rows) return;  // uniform over the row's warps
    const T* at = x + row * ldx + c0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      next[i].template load<ROWS>(at + i * W::kCols, row < rows ? K - c0 - i * W::kCols : 0);
  };
  if (kAhead) fetch(r);
  for (; r < rows; r += step) {
    if (!kAhead) fetch(r);
    float2 v[N][W::PER / 2];
#pragma unroll
    for (int i = 0; i < N; ++i) next[i].widen(v[i]);
    if (kAhead) fetch(r + step);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < W::PER / 2; ++j) sum = add2(sum, v[i][j]);
    const float mean = row_sum<WARPS>(sum.x + sum.y, part[0]) / static_cast<float>(K);
    float2 sq = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) sq = centre<ROWS>(v[i], mean, c0 + i * W::kCols, K, sq);
    const float var = row_sum<WARPS>(sq.x + sq.y, part[1]) / static_cast<float>(K);
    const float rstd = 1.f / sqrtf(var + eps);
    uint32_t bits[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      affine<ROWS>(v[i], rstd, gamma, beta, c0 + i * W::kCols, K);
      bits[i] = abs_bits_max(v[i]);
    }
    WarpScales<T, N> ws;
    ws.find(bits, lane);
    uint8_t* to = q + r * ldq + c0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Fp8Scale s = ws.get(i, lane);
      if (ROWS == kFullRows || c0 + i * W::kCols < K) s.store(to + i * W::kCols, v[i]);
    }
    const int g = col0 / kFp8Block + (lane % W::kLanes) * W::kBlocks + lane / W::kLanes;
    if (lane % W::kLanes < N && g < kb) scales[r * kb + g] = ws.scale;
  }
}

// Rows too wide for a CTA's registers: the same three steps, x read again
// (from L2) for each.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kThreads)
    layernorm_fp8_wide_kernel(const T* __restrict__ x, int64_t ldx,
                              const float* __restrict__ gamma, const float* __restrict__ beta,
                              float eps, int64_t rows, int K, int kb, uint8_t* __restrict__ q,
                              int64_t ldq, float* __restrict__ scales) {
  using W = Warp<T>;
  __shared__ float part[2][kWarps];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int first = (threadIdx.x >> 5) * W::kCols;  // this warp's first column
  constexpr int kStep = kWarps * W::kCols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * ldx;
    Lane16<T> raw;
    float2 v[W::PER / 2];
    float2 sum = make_float2(0.f, 0.f);
    for (int b = first; b < K; b += kStep) {
      const int c = b + W::PER * lane;
      raw.template load<ROWS>(row + c, K - c);
      raw.widen(v);
#pragma unroll
      for (int j = 0; j < W::PER / 2; ++j) sum = add2(sum, v[j]);
    }
    const float mean = row_sum<kWarps>(sum.x + sum.y, part[0]) / static_cast<float>(K);
    float2 sq = make_float2(0.f, 0.f);
    for (int b = first; b < K; b += kStep) {
      const int c = b + W::PER * lane;
      raw.template load<ROWS>(row + c, K - c);
      raw.widen(v);
      sq = centre<ROWS>(v, mean, c, K, sq);
    }
    const float var = row_sum<kWarps>(sq.x + sq.y, part[1]) / static_cast<float>(K);
    const float rstd = 1.f / sqrtf(var + eps);
    for (int b = first; b < K; b += kStep) {
      const int c = b + W::PER * lane;
      raw.template load<ROWS>(row + c, K - c);
      raw.widen(v);
      centre<ROWS>(v, mean, c, K, sq);
      affine<ROWS>(v, rstd, gamma, beta, c, K);
      const uint32_t bits[1] = {abs_bits_max(v)};
      WarpScales<T, 1> ws;
      ws.find(bits, lane);
      const Fp8Scale s = ws.get(0, lane);
      if (c < K) s.store(q + r * ldq + c, v);
      const int g = b / kFp8Block + lane / W::kLanes;
      if (lane % W::kLanes == 0 && g < kb) scales[r * kb + g] = ws.scale;
    }
  }
}

// CTAs for `work` CTA-sized pieces: enough to fill the GPU eight deep, the
// kernels stride over the rest.
unsigned grid_for(int64_t work) {
  return static_cast<unsigned>(
      std::max<int64_t>(1, std::min<int64_t>(work, static_cast<int64_t>(device_num_sms()) * 8)));
}

// Whole 16-byte loads: rows aligned to them, and K a multiple.
template <typename T>
bool vector_rows(const T* x, int64_t ldx, int K) {
  constexpr int kPer = Lane16<T>::PER;
  return K % kPer == 0 && ldx % kPer == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
}

template <typename T, int ROWS>
int quantize_typed(const T* x, int64_t rows, int K, int64_t ldx, int block_rows, uint8_t* q,
                   int64_t ldq, float* scales, cudaStream_t s) {
  using W = Warp<T>;
  const int kb = (K + kFp8Block - 1) / kFp8Block;
  if (block_rows != 1) {
    const int64_t blocks = (rows + kFp8Block - 1) / kFp8Block * kb;
    return launch_kernel(quantize_blocks_kernel<T, ROWS>, dim3(grid_for(blocks)),
                         dim3(kBlockThreads), 0, s, 1, x, ldx, rows, K, kb, q, ldq, scales, blocks);
  }
  auto go = [&](auto kernel, int n) {
    const int per_row = (K + n * W::kCols - 1) / (n * W::kCols);
    const int64_t ctas = (rows * per_row + kWarps - 1) / kWarps;
    return launch_kernel(kernel, dim3(grid_for(ctas)), dim3(kThreads), 0, s, 1, x, ldx, rows, K, kb,
                         per_row, q, ldq, scales);
  };
  // `n` loads a warp; rows that they fill exactly need no checks.
  auto rows_of = [&](auto n) {
    constexpr int N = decltype(n)::value;
    if (ROWS == kVectorRows && K % (N * W::kCols) == 0)
      return go(quantize_rows_kernel<T, kFullRows, N>, N);
    return go(quantize_rows_kernel<T, ROWS, N>, N);
  };
  // The loads that a warp takes share the work on the scales, but those past a row's end
  // are empty: six where they fill rows exactly, else four, and one where the matrix would
  // leave SMs without work (50432 rows with one, four, six loads: 768 columns fp32 49.7,
  // 38.3, 30.2 us; 1536 bf16 68.9, 53.5, 43.5; 512 fp32 with one, four 33.9, 21.4).
  const int loads = (K + W::kCols - 1) / W::kCols;
  const int64_t fill = static_cast<int64_t>(device_num_sms()) * 4 * kWarps;
  if (loads == 1 || rows * loads <= fill) return rows_of(std::integral_constant<int, 1>{});
  if (loads % 6 != 0 || rows * (loads / 6) <= fill)
    return rows_of(std::integral_constant<int, 4>{});
  return rows_of(std::integral_constant<int, 6>{});
}

template <typename T, int ROWS>
int layernorm_typed(const T* x, int64_t rows, int K, int64_t ldx, const float* gamma,
                    const float* beta, float eps, uint8_t* q, int64_t ldq, float* scales,
                    cudaStream_t s) {
  using W = Warp<T>;
  const int kb = (K + kFp8Block - 1) / kFp8Block;
  auto go = [&](auto kernel, int rows_per_cta) {
    return launch_kernel(kernel, dim3(grid_for((rows + rows_per_cta - 1) / rows_per_cta)),
                         dim3(kThreads), 0, s, 1, x, ldx, gamma, beta, eps, rows, K, kb, q, ldq,
                         scales);
  };
  auto form = [&](auto warps, auto n) {
    constexpr int WARPS = decltype(warps)::value, N = decltype(n)::value;
    if (ROWS == kVectorRows && K == WARPS * N * W::kCols)
      return go(layernorm_fp8_kernel<T, kFullRows, WARPS, N>, kWarps / WARPS);
    return go(layernorm_fp8_kernel<T, ROWS, WARPS, N>, kWarps / WARPS);
  };
  // The narrowest form that holds the row: registers, not work, differ (24 values a lane
  // against 32: 50432 x 768 fp32 34.6 and 53.2 us, x 512 33.3 and 43.1).
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, kWarps> all{};
  const int loads = (K + W::kCols - 1) / W::kCols;
  if (loads == 1) return form(one, one);
  if (loads <= 3) return form(one, std::integral_constant<int, 3>{});
  if (loads <= 24 / W::PER) return form(one, std::integral_constant<int, 24 / W::PER>{});
  if (loads <= 32 / W::PER) return form(one, std::integral_constant<int, 32 / W::PER>{});
  if (loads <= kWarps) return form(all, one);
  if (loads <= 2 * kWarps) return form(all, std::integral_constant<int, 2>{});
  if (loads <= 4 * kWarps) return form(all, std::integral_constant<int, 4>{});
  if (loads <= 32 / W::PER * kWarps) return form(all, std::integral_constant<int, 32 / W::PER>{});
  return go(layernorm_fp8_wide_kernel<T, ROWS>, 1);
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
               ? quantize_typed<T, kVectorRows>(p, rows, K, ldx, block_rows, q, ldq, scales, s)
               : quantize_typed<T, kScalarRows>(p, rows, K, ldx, block_rows, q, ldq, scales, s);
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
    return vec ? layernorm_typed<T, kVectorRows>(p, rows, K, ldx, gamma, beta, eps, q, ldq, scales, s)
               : layernorm_typed<T, kScalarRows>(p, rows, K, ldx, gamma, beta, eps, q, ldq, scales, s);
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
  if (reinterpret_cast<uintptr_t>(x) % (type == VITB200_F32 ? 4 : 2) != 0 ||
      reinterpret_cast<uintptr_t>(scales) % 4 != 0)
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
    if (reinterpret_cast<uintptr_t>(gamma) % 4 != 0 || reinterpret_cast<uintptr_t>(beta) % 4 != 0)
      return VITB200_E_ALIGNMENT;
    if (int st = vitb200_init()) return st;
    return layernorm_fp8_launch(x, x_type, rows, K, ldx, gamma, beta, eps, q, ldq, scales,
                                static_cast<cudaStream_t>(stream));
  } catch (...) {
    return VITB200_E_INVALID_ARG;
  }
}
