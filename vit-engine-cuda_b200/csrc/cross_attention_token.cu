// cross_attention (see cross_attention.cu for the operator) for up to 16 rows per
// key head: single tokens, and short prompts of few heads.
//
// Nothing is reused here, so the bound is reading K and V once from HBM; the
// 128-row tiles of the tcgen05 kernel would spend their set-up and hand-overs on
// rows that do not exist (192 key heads x 197 keys: 16 us there). A warp instead
// takes 16 keys at a time straight from global memory into the registers of
// mma.sync m16n8k16 (16 rows; the legacy tensor path is far from its limit at one
// product per loaded fragment), with its own running maximum, sum and output, and
// no barrier until the end:
//  * S = Q K^T: a lane's 16-byte load is eight neighbouring columns of one key.
//    The order in which the columns enter the sum is free, so these eight serve as
//    the B fragments of two products, with Q's fragments loaded in the same order.
//  * O = P V: the sum runs over keys, so a fragment needs two keys' values of one
//    column. A lane loads the same eight columns of its four keys and pairs them
//    with byte permutes; column j of each eight forms the j-th product's eight
//    output columns.
// A key head's keys are shared out over the CTAs of a cluster and their warps; the
// partial results meet in shared memory, in a fixed order.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "cross_attention.cuh"
#include "engine.h"

namespace vitb200 {

namespace {

constexpr int kTokenWarps = 8;
constexpr int kTokenThreads = 32 * kTokenWarps;
// Keys a warp takes at a time: K and V of 16 keys are 32 (D = 64) or 64 registers
// of loads in flight beside O's 32 or 64; 32 keys spill.
constexpr int kStep = 16;

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

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Sum of the two values of a packed pair.
template <typename T>
__device__ __forceinline__ float pair_sum(uint32_t p) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
    return f.x + f.y;
  }
  return __uint_as_float(p << 16) + __uint_as_float(p & 0xffff0000u);
}

// Floats of a warp's or CTA's partial result: [rows][D + 4], then m and l, rounded
// up to 16 bytes (the next result's rows are stored and read as float4).
template <int D>
constexpr int kPartPitch = D + 4;
template <int D>
__host__ __device__ constexpr int part_floats(int rows) {
  return (rows * (kPartPitch<D> + 2) + 3) / 4 * 4;
}
static_assert(kPartPitch<64> % 4 == 0 && kPartPitch<128> % 4 == 0, "16-byte rows");

// Adds the partial results of `count` sources, `at(p)` the shared-memory address
// of source p's: eight columns from `col` of row r, and the row's maximum and sum.
template <int D, typename At>
__device__ __forceinline__ void join_row(int count, At&& at, int rows, int r, int col, float& M,
                                         float& L, float (&o)[8], bool remote) {
  M = -INFINITY;
  for (int p = 0; p < count; ++p)
    M = fmaxf(M, ld_partial(at(p) + 4u * (rows * kPartPitch<D> + r), remote));
  const float ref = M == -INFINITY ? 0.f : M;
  L = 0.f;
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = 0.f;
  for (int p = 0; p < count; ++p) {
    const float f = ex2_approx(ld_partial(at(p) + 4u * (rows * kPartPitch<D> + r), remote) - ref);
    L = fmaf(ld_partial(at(p) + 4u * (rows * (kPartPitch<D> + 1) + r), remote), f, L);
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      const float4 t = ld_partial4(at(p) + 4u * (r * kPartPitch<D> + col + q), remote);
      o[q] = fmaf(t.x, f, o[q]), o[q + 1] = fmaf(t.y, f, o[q + 1]);
      o[q + 2] = fmaf(t.z, f, o[q + 2]), o[q + 3] = fmaf(t.w, f, o[q + 3]);
    }
  }
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kTokenThreads, D == 64 ? 2 : 1)
    cross_attention_token_kernel(const CrossTokenArgs a) {
  constexpr int kTiles = kStep / 8;    // S products' key tiles
  constexpr int kPairs = kStep / 16;   // P V products' key sums
  constexpr int kE = D / 32;           // 16-byte loads of a key row's quarter lanes
  constexpr int kH = D / 64;           // 128-byte spans of a value row
  extern __shared__ __align__(16) float part[];  // [warps] partial results, then the CTA's

  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;  // row (and g + 8), key or column of a fragment
  const int c = lane & 3;
  const int split = static_cast<int>(blockIdx.x) % a.nsplit;
  const int item = static_cast<int>(blockIdx.x) / a.nsplit;
  const int b = item / a.kv_heads;
  const int hk = item - b * a.kv_heads;
  int len = a.Tk;
  if (a.lens != nullptr) len = max(0, min(a.Tk, __ldg(a.lens + b)));
  const int steps = (len + kStep - 1) / kStep;
  const int step0 = static_cast<int>(static_cast<int64_t>(steps) * split / a.nsplit);
  const int step1 = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / a.nsplit);

  // Q fragments of rows g and g + 8: 16 bytes of each 32 columns, two products.
  uint4 q[2][kE];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    const int t = r / a.group;
    const uint16_t* row = a.q + b * a.q_batch + t * a.q_row +
                          (static_cast<int64_t>(hk) * a.group + (r - t * a.group)) * D + 8 * c;
#pragma unroll
    for (int e = 0; e < kE; ++e)
      q[h][e] = r < a.rows ? __ldg(reinterpret_cast<const uint4*>(row + 32 * e))
                           : make_uint4(0, 0, 0, 0);
  }

  const uint16_t* kp = a.k + b * a.k_batch + static_cast<int64_t>(hk) * D + 8 * c;
  const uint16_t* vp = a.v + b * a.v_batch + static_cast<int64_t>(hk) * D + 8 * g;
  uint4 kf[kTiles][kE], vf[kPairs][4][kH];
  // Keys past the length are read as zeros: a value there may be NaN, and zero
  // times NaN is not zero.
  auto load_k = [&](int key0) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int key = key0 + 8 * t + g;
#pragma unroll
      for (int e = 0; e < kE; ++e)
        kf[t][e] = key < len ? ld_stream(kp + key * a.k_row + 32 * e) : make_uint4(0, 0, 0, 0);
    }
  };
  auto load_v = [&](int key0) {
#pragma unroll
    for (int p = 0; p < kPairs; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * p + 2 * c + (i & 1) + 8 * (i >> 1);
#pragma unroll
        for (int h = 0; h < kH; ++h)
          vf[p][i][h] = key < len ? ld_stream(vp + key * a.v_row + 64 * h) : make_uint4(0, 0, 0, 0);
      }
  };

  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  int step = step0 + warp;
  if (step < step1) {
    load_k(step * kStep);
    load_v(step * kStep);
  }
  for (; step < step1; step += kTokenWarps) {
    const int key0 = step * kStep;
    float s[kTiles][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t qa[4] = {word(q[0][e], 2 * u), word(q[1][e], 2 * u),
                                  word(q[0][e], 2 * u + 1), word(q[1][e], 2 * u + 1)};
          mma_16x8x16<T>(s[t], qa, word(kf[t][e], 2 * u), word(kf[t][e], 2 * u + 1));
        }
    }
    const bool more = step + kTokenWarps < step1;
    if (more) load_k(key0 + kTokenWarps * kStep);  // lands during the rest of the step
    // Scores in log2 units; lane holds keys 8 t + 2 c + {0, 1} of rows g and g + 8.
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[t][i] = key0 + 8 * t + 2 * c + (i & 1) < len ? s[t][i] * a.c : -INFINITY;
    bool grew = false;
    float old[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = m[h];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) top = max3(top, s[t][2 * h], s[t][2 * h + 1]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      old[h] = m[h];
      grew |= top > m[h];
      m[h] = top;
    }
    const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
    if (__any_sync(0xffffffffu, grew)) {
      const float f0 = ex2_approx(old[0] - ref[0]), f1 = ex2_approx(old[1] - ref[1]);
      l[0] *= f0;
      l[1] *= f1;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) o[j][0] *= f0, o[j][1] *= f0, o[j][2] *= f1, o[j][3] *= f1;
    }
    uint32_t p[kPairs][4];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w = pack2<T>(ex2_approx(s[t][2 * h] - ref[h]),
                                    ex2_approx(s[t][2 * h + 1] - ref[h]));
        l[h] += pair_sum<T>(w);  // the probabilities as V sees them
        p[t / 2][2 * (t & 1) + h] = w;
      }
#pragma unroll
    for (int pr = 0; pr < kPairs; ++pr)
#pragma unroll
      for (int h = 0; h < kH; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
          const uint32_t b0 = __byte_perm(word(vf[pr][0][h], j / 2), word(vf[pr][1][h], j / 2), sel);
          const uint32_t b1 = __byte_perm(word(vf[pr][2][h], j / 2), word(vf[pr][3][h], j / 2), sel);
          mma_16x8x16<T>(o[8 * h + j], p[pr], b0, b1);
        }
    if (more) load_v(key0 + kTokenWarps * kStep);
  }

  // The warp's partial result. Product j of span h gave columns 64 h + 8 n + j,
  // n = 2 c + {0, 1}.
  const int rows = a.rows;
  float* mine = part + warp * part_floats<D>(rows);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (r >= rows) continue;
    float* row = mine + r * kPartPitch<D>;
#pragma unroll
    for (int x = 0; x < kH; ++x)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4*>(row + 64 * x + 8 * (2 * c + n) + j) =
              make_float4(o[8 * x + j][2 * h + n], o[8 * x + j + 1][2 * h + n],
                          o[8 * x + j + 2][2 * h + n], o[8 * x + j + 3][2 * h + n]);
    if (c == 0) {
      mine[rows * kPartPitch<D> + r] = m[h];
      mine[rows * (kPartPitch<D> + 1) + r] = l[h];
    }
  }
  __syncthreads();

  constexpr int kChunks = D / 8;
  const uint32_t base = smem_addr(part);
  const uint32_t stride = 4u * part_floats<D>(rows);
  auto finish = [&](int r, int col, float L, const float (&v)[8]) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (len > 0) {
      const float inv = 1.f / L;
      w = make_uint4(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv),
                     pack2<T>(v[4] * inv, v[5] * inv), pack2<T>(v[6] * inv, v[7] * inv));
    }
    const int t = r / a.group;
    const int64_t row = (static_cast<int64_t>(b) * a.Tq + t) * a.o_row +
                        (static_cast<int64_t>(hk) * a.group + (r - t * a.group)) * D;
    *reinterpret_cast<uint4*>(a.o + row + col) = w;
  };
  // Warps first, then (with a cluster) CTAs, whose results follow the warps'.
  float* cta = part + kTokenWarps * part_floats<D>(rows);
  for (int x = threadIdx.x; x < rows * kChunks; x += kTokenThreads) {
    const int r = x / kChunks, col = 8 * (x - r * kChunks);
    float M, L, v[8];
    join_row<D>(kTokenWarps, [&](int p) { return base + stride * p; }, rows, r, col, M, L, v, false);
    if (a.nsplit == 1) {
      finish(r, col, L, v);
    } else {
      float* to = cta + r * kPartPitch<D> + col;
      *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
      if (col == 0) {
        cta[rows * kPartPitch<D> + r] = M;
        cta[rows * (kPartPitch<D> + 1) + r] = L;
      }
    }
  }
  if (a.nsplit == 1) return;
  __syncwarp();
  cluster_sync_all();
  for (int x = split * kTokenThreads + static_cast<int>(threadIdx.x); x < rows * kChunks;
       x += a.nsplit * kTokenThreads) {
    const int r = x / kChunks, col = 8 * (x - r * kChunks);
    float M, L, v[8];
    join_row<D>(
        a.nsplit,
        [&](int p) { return mapa_shared(base + stride * kTokenWarps, static_cast<uint32_t>(p)); },
        rows, r, col, M, L, v, true);
    finish(r, col, L, v);
  }
  __syncwarp();
  cluster_sync_all();  // no CTA exits while its result may be read
}

namespace {

template <typename T, int D>
int token_smem(int rows) {
  return (kTokenWarps + 1) * part_floats<D>(rows) * 4;
}

template <typename T, int D>
int launch_token(const CrossTokenArgs& args, int64_t items, cudaStream_t s) {
  CrossTokenArgs a = args;
  // Enough CTAs to fill the GPU, each with a step for every warp at least.
  const int64_t slots = static_cast<int64_t>(device_num_sms()) * (D == 64 ? 2 : 1);
  const int64_t steps = (a.Tk + kStep - 1) / kStep;
  a.nsplit = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>({slots / items, steps / kTokenWarps, kCrossMaxSplit})));
  return launch_kernel(cross_attention_token_kernel<T, D>,
                       dim3(static_cast<unsigned>(items * a.nsplit)), dim3(kTokenThreads),
                       static_cast<size_t>(token_smem<T, D>(a.rows)), s,
                       static_cast<unsigned>(a.nsplit), a);
}

}  // namespace

int cross_attention_token_prepare_device() {
  auto one = [](auto kernel, int bytes) {
    return cuda_status(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  };
  using bf16 = __nv_bfloat16;
  if (int st = one(cross_attention_token_kernel<__half, 64>, token_smem<__half, 64>(16))) return st;
  if (int st = one(cross_attention_token_kernel<bf16, 64>, token_smem<bf16, 64>(16))) return st;
  if (int st = one(cross_attention_token_kernel<__half, 128>, token_smem<__half, 128>(16)))
    return st;
  return one(cross_attention_token_kernel<bf16, 128>, token_smem<bf16, 128>(16));
}

int cross_attention_token_launch(const CrossProblem& p, cudaStream_t s) {
  CrossTokenArgs a = {};
  a.q = static_cast<const uint16_t*>(p.q);
  a.k = static_cast<const uint16_t*>(p.k);
  a.v = static_cast<const uint16_t*>(p.v);
  a.o = static_cast<uint16_t*>(p.o);
  a.lens = p.lens;
  a.Tq = p.Tq;
  a.Tk = p.Tk;
  a.kv_heads = p.kv_heads;
  a.group = p.heads / p.kv_heads;
  a.rows = a.group * p.Tq;
  a.q_row = p.q_row;
  a.q_batch = p.q_batch;
  a.k_row = p.k_row;
  a.k_batch = p.k_batch;
  a.v_row = p.v_row;
  a.v_batch = p.v_batch;
  a.o_row = static_cast<int64_t>(p.heads) * p.D;
  a.c = p.scale * kLog2e;
  const int64_t items = static_cast<int64_t>(p.B) * p.kv_heads;
  if (items > INT32_MAX / kCrossMaxSplit) return VITB200_E_UNSUPPORTED;
  if (p.type == VITB200_BF16)
    return p.D == 64 ? launch_token<__nv_bfloat16, 64>(a, items, s)
                     : launch_token<__nv_bfloat16, 128>(a, items, s);
  return p.D == 64 ? launch_token<__half, 64>(a, items, s) : launch_token<__half, 128>(a, items, s);
}

}  // namespace vitb200
