// cross_attention (see cross_attention.cu for the operator) for up to 16 rows per
// key head: single tokens, and short prompts of few heads.
//
// Nothing is reused here, so the bound is reading K and V once from HBM; the
// 128-row tiles of the tcgen05 kernel would spend their set-up and hand-overs on
// rows that do not exist (192 key heads x 197 keys: 16 us there). A warp instead
// takes 16 keys at a time, through shared memory of its own lanes, to mma.sync
// m16n8k16, with keys (then output columns) as the product's 16 rows and eight query
// rows as its columns, with its own running maxima, sums and output, and no barrier
// until the end. (The legacy tensor path is far from its limit at one product or two
// per loaded fragment; query rows as the product's 16 rows take twice the products
// and registers.)
//  * S^T = K Q^T: a lane's 16-byte load is eight neighbouring columns of one key.
//    The order in which the columns enter the sum is free, so these eight serve as
//    fragments of two products, with Q's fragments loaded in the same order.
//  * O^T = V^T P^T: the sum runs over keys, so a fragment needs two keys' values of
//    one column. A lane loads the same eight columns of its four keys and pairs them
//    with byte permutes, two columns a product; P^T's fragments are S^T's
//    transposed by movmatrix.
//
// A step is 16 keys of one key head of one image. Either a CTA takes a key head of
// an image (its warps the steps in turn, their results joined in shared memory),
// or, where that would leave SMs idle, the steps of all images form one list per
// key head, which as many CTAs as the head gets cut into equal parts, whatever the
// images' lengths: the parts of an image that several CTAs share go to a workspace,
// and a second kernel adds them in order. Neighbouring CTAs take the same part for
// neighbouring heads, whose keys lie side by side: one list of all heads would
// read 256-byte pieces far apart. (Sharing a key head over a cluster
// needs no workspace, but 16 clusters of 8 one-per-SM CTAs do not fit the GPU at
// once, and images of different lengths finish at different times: 2 x 8 heads x
// 32768 keys ran at 2.6 TB/s.)
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "cross_attention.cuh"
#include "engine.h"

namespace vitb200 {

namespace {

constexpr int kStep = 16;  // keys a warp takes at a time
// Steps in flight, in shared memory: each lane copies the 16-byte pieces that it
// will itself read as fragments into places of its own, so the ring needs no
// barrier and has no bank conflicts.
template <int D>
constexpr int kPieces = 2 * kStep * D * 2 / (32 * 16);  // per lane and step, K and V

// Eight warps and three steps in flight: up to 192 KB per SM. The streaming form
// was also measured with CTAs of four warps, two or three an SM and two or three
// steps in flight (2 x 8 heads x 32768 keys: 72 us against 66).
template <int D>
struct TokenCfg {
  static constexpr int kWarps = 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStages = 3;
  static constexpr int kPerSm = D == 64 ? 2 : 1;
  static constexpr int kRingBytes = kStages * kPieces<D> * 16 * kThreads;
};

// The 8 x 8 matrix of 16-bit values a warp holds as fragments, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
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

// Joins a few partial results: eight columns from `col` of row r, the row's
// maximum and sum; `at(p)` is the address of source p's first float.
template <int D, typename At>
__device__ __forceinline__ void join_row(int count, At&& at, int rows, int r, int col, float& M,
                                         float& L, float (&o)[8]) {
  M = -INFINITY;
  for (int p = 0; p < count; ++p) M = fmaxf(M, at(p)[rows * kPartPitch<D> + r]);
  const float ref = M == -INFINITY ? 0.f : M;
  L = 0.f;
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = 0.f;
  for (int p = 0; p < count; ++p) {
    const float* src = at(p);
    const float f = ex2_approx(src[rows * kPartPitch<D> + r] - ref);
    L = fmaf(src[rows * (kPartPitch<D> + 1) + r], f, L);
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      const float4 t = *reinterpret_cast<const float4*>(src + r * kPartPitch<D> + col + q);
      o[q] = fmaf(t.x, f, o[q]), o[q + 1] = fmaf(t.y, f, o[q + 1]);
      o[q + 2] = fmaf(t.z, f, o[q + 2]), o[q + 3] = fmaf(t.w, f, o[q + 3]);
    }
  }
}

// Writes eight output columns of a row: v / L (zeros for an image without keys).
template <typename T, int D>
__device__ __forceinline__ void put_row(const CrossTokenArgs& a, int b, int hk, int r, int col,
                                        bool keys, float L, const float (&v)[8]) {
  uint4 w = make_uint4(0, 0, 0, 0);
  if (keys) {
    const float inv = 1.f / L;
    w = make_uint4(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv),
                   pack2<T>(v[4] * inv, v[5] * inv), pack2<T>(v[6] * inv, v[7] * inv));
  }
  const int t = r / a.group;
  const int64_t row = (static_cast<int64_t>(b) * a.Tq + t) * a.o_row +
                      (static_cast<int64_t>(hk) * a.group + (r - t * a.group)) * D;
  *reinterpret_cast<uint4*>(a.o + row + col) = w;
}

__device__ __forceinline__ int keys_of(const CrossTokenArgs& a, int b) {
  return a.lens == nullptr ? a.Tk : max(0, min(a.Tk, __ldg(a.lens + b)));
}

__device__ __forceinline__ int steps_of(const CrossTokenArgs& a, int b) {
  return (keys_of(a, b) + kStep - 1) / kStep;
}

// A key head's list of steps, image by image, is cut into as many equal parts as
// it has CTAs, none of them empty (the grid goes by the longest possible images):
// the first `rem` parts have base + 1 steps, the others base.
struct Parts {
  int total, n, base, rem;
  __device__ __forceinline__ Parts() {}
  __device__ __forceinline__ Parts(int total_, int ctas) : total(total_) {
    n = min(total, ctas);
    base = n > 0 ? total / n : 0;
    rem = n > 0 ? total - base * n : 0;
  }
  __device__ __forceinline__ int begin(int i) const { return i * base + min(i, rem); }
  __device__ __forceinline__ int holder(int step) const {  // the part that holds a step
    const int high = rem * (base + 1);
    return step < high ? step / (base + 1) : rem + (step - high) / base;
  }
};

// By a warp: the steps of images 0 .. end - 1, and the last image among them that
// begins at or before step `want` and has keys, with the steps before it.
struct Place {
  int total, before, b;
};
__device__ __forceinline__ Place place_of(const CrossTokenArgs& a, int end, int want, int lane) {
  if (a.lens == nullptr) {
    const int per = steps_of(a, 0);
    const int b = want / per;
    return {end * per, b * per, b};
  }
  Place p{0, 0, 0};
  for (int b0 = 0; b0 < end; b0 += 32) {
    const int b = b0 + lane;
    const int mine = b < end ? steps_of(a, b) : 0;
    int sum = mine;  // of the images up to this lane's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += t;
    }
    const int start = p.total + sum - mine;
    const uint32_t here = __ballot_sync(0xffffffffu, mine > 0 && start <= want);
    if (here != 0) {
      const int src = 31 - __clz(here);
      p.b = b0 + src;
      p.before = __shfl_sync(0xffffffffu, start, src);
    }
    p.total += __shfl_sync(0xffffffffu, sum, 31);
  }
  return p;
}

}  // namespace

// STREAM: the CTA works through its part of a head's list; else through a key
// head of an image.
template <typename T, int D, int NT, bool STREAM>
__global__ void __launch_bounds__(TokenCfg<D>::kThreads, TokenCfg<D>::kPerSm)
    cross_attention_token_kernel(const CrossTokenArgs a) {
  constexpr int kTokenWarps = TokenCfg<D>::kWarps;
  constexpr int kTokenThreads = TokenCfg<D>::kThreads;
  constexpr int kStages = TokenCfg<D>::kStages;
  constexpr int kE = D / 32;           // 16-byte pieces of a key row that a lane takes
  constexpr int kH = D / 64;           // 128-byte spans of a value row
  static_assert(2 * kE + 4 * kH == kPieces<D>, "pieces of a step");
  // The ring; between segments the warps' partial results.
  extern __shared__ __align__(16) float smem[];
  __shared__ Place place;

  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;  // row (and g + 8) or column of a fragment
  const int c = lane & 3;
  const int rows = a.rows;

  int b, hk;
  int step0 = 0;  // of the segment, within its key head
  int left = 0;   // steps of the part that are left
  if constexpr (STREAM) {
    const int ctas = static_cast<int>(gridDim.x) / a.kv_heads;  // per head
    const int i = static_cast<int>(blockIdx.x) / a.kv_heads;
    hk = static_cast<int>(blockIdx.x) - i * a.kv_heads;
    if (warp == 0) {
      const int total = place_of(a, a.B, 0, lane).total;
      const Parts parts(total, ctas);
      Place p = place_of(a, a.B, parts.begin(min(i, max(parts.n - 1, 0))), lane);
      if (lane == 0) place = p;
    }
    __syncthreads();
    const Place p = place;
    const Parts parts(p.total, ctas);
    if (i >= parts.n) return;
    left = parts.begin(i + 1) - parts.begin(i);
    b = p.b;
    step0 = parts.begin(i) - p.before;
  } else {
    b = static_cast<int>(blockIdx.x) / a.kv_heads;
    hk = static_cast<int>(blockIdx.x) - b * a.kv_heads;
  }

  while (true) {
    const int len = keys_of(a, b);
    const int steps = (len + kStep - 1) / kStep;
    const int step1 = STREAM ? min(steps, step0 + left) : steps;

    // Q fragments of rows 8 n + g: 16 bytes of each 32 columns, two products.
    uint4 q[NT][kE];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + g;
      const int t = r / a.group;
      const uint16_t* row = a.q + b * a.q_batch + t * a.q_row +
                            (static_cast<int64_t>(hk) * a.group + (r - t * a.group)) * D + 8 * c;
#pragma unroll
      for (int e = 0; e < kE; ++e)
        q[n][e] = r < rows ? __ldg(reinterpret_cast<const uint4*>(row + 32 * e))
                           : make_uint4(0, 0, 0, 0);
    }

    const uint16_t* kp = a.k + b * a.k_batch + static_cast<int64_t>(hk) * D + 8 * c;
    const uint16_t* vp = a.v + b * a.v_batch + static_cast<int64_t>(hk) * D + 8 * g;
    // This lane's pieces: K's 2 * kE (keys g, g + 8), then V's 4 * kH (keys 2 c,
    // 2 c + 1 and eight further), of each stage.
    uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;
    const uint32_t ring_addr = smem_addr(ring);
    // Keys past the length are read as zeros: a value there may be NaN, and zero
    // times NaN is not zero. One group of copies a step, empty past the last.
    auto fetch = [&](int step, int stage) {
      if (step < step1) {
        const int key0 = step * kStep;
        uint32_t to = ring_addr + static_cast<uint32_t>(stage * kPieces<D> * kTokenThreads * 16);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int key = key0 + 8 * t + g;
          const uint16_t* row = kp + (key < len ? key : 0) * a.k_row;
#pragma unroll
          for (int e = 0; e < kE; ++e, to += kTokenThreads * 16)
            copy_async16(to, row + 32 * e, key < len);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 2 * c + (i & 1) + 8 * (i >> 1);
          const uint16_t* row = vp + (key < len ? key : 0) * a.v_row;
#pragma unroll
          for (int h = 0; h < kH; ++h, to += kTokenThreads * 16)
            copy_async16(to, row + 64 * h, key < len);
        }
      }
      copy_async_commit();
    };

    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];  // of rows 8 n + 2 c + {0, 1}; l of this lane's keys
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    int step = step0 + warp;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(step + i * kTokenWarps, i);
    int stage = 0;
    for (; step < step1; step += kTokenWarps) {
      const int key0 = step * kStep;
      // The stage that the previous step has read takes the last step in flight.
      fetch(step + (kStages - 1) * kTokenWarps, stage == 0 ? kStages - 1 : stage - 1);
      copy_async_wait<kStages - 1>();
      const uint4* kf = ring + stage * kPieces<D> * kTokenThreads;
      const uint4* vf = kf + 2 * kE * kTokenThreads;
      if (++stage == kStages) stage = 0;
      // Scores of keys g and g + 8 (s[0..1], s[2..3]) for rows 8 n + 2 c + {0, 1}.
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const uint4 k0 = kf[e * kTokenThreads], k1 = kf[(kE + e) * kTokenThreads];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t ka[4] = {word(k0, 2 * u), word(k1, 2 * u), word(k0, 2 * u + 1),
                                  word(k1, 2 * u + 1)};
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma_16x8x16<T>(s[n], ka, word(q[n][e], 2 * u), word(q[n][e], 2 * u + 1));
        }
      }
      const bool in0 = key0 + g < len, in1 = key0 + 8 + g < len;
      bool grew = false;
      float f[NT][2], ref[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[n][i] = in0 ? s[n][i] * a.c : -INFINITY;  // log2 units
          s[n][2 + i] = in1 ? s[n][2 + i] * a.c : -INFINITY;
          float top = max3(m[n][i], s[n][i], s[n][2 + i]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          grew |= top > m[n][i];
          ref[n][i] = top == -INFINITY ? 0.f : top;
          f[n][i] = ex2_approx(m[n][i] - ref[n][i]);
          m[n][i] = top;
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          l[n][0] *= f[n][0];
          l[n][1] *= f[n][1];
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[n][j][0] *= f[n][0], o[n][j][1] *= f[n][1];
            o[n][j][2] *= f[n][0], o[n][j][3] *= f[n][1];
          }
        }
      }
      uint32_t p[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // (the lift comes last: where scores are huge, ref - 15 would be rounded)
          float e0 = s[n][2 * i] - ref[n][0], e1 = s[n][2 * i + 1] - ref[n][1];
          if constexpr (kLift<T> != 0.f) e0 += kLift<T>, e1 += kLift<T>;
          const uint32_t w = pack2<T>(ex2_approx(e0), ex2_approx(e1));
          const float2 seen = unpack2<T>(w);  // the probabilities as V sees them
          l[n][0] += seen.x;
          l[n][1] += seen.y;
          p[n][i] = transpose_8x8(w);
        }
#pragma unroll
      for (int h = 0; h < kH; ++h) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = vf[(i * kH + h) * kTokenThreads];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // columns 64 h + 8 g + 2 j + {0, 1}
          const uint32_t va[4] = {__byte_perm(word(v[0], j), word(v[1], j), 0x5410u),
                                  __byte_perm(word(v[0], j), word(v[1], j), 0x7632u),
                                  __byte_perm(word(v[2], j), word(v[3], j), 0x5410u),
                                  __byte_perm(word(v[2], j), word(v[3], j), 0x7632u)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16x8x16<T>(o[n][4 * h + j], va, p[n][0], p[n][1]);
        }
      }
    }
    copy_async_wait<0>();
    __syncthreads();  // every warp has left the ring: its bytes take the partial results

    // The warp's partial result.
    float* mine = smem + warp * part_floats<D>(rows);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 8 * n + 2 * c + i;
        l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 4);
        l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 8);
        l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], 16);
        if (r >= rows) continue;
        float* row = mine + r * kPartPitch<D> + 8 * g;
#pragma unroll
        for (int j = 0; j < D / 16; j += 2)
          *reinterpret_cast<float4*>(row + 64 * (j / 4) + 2 * (j % 4)) =
              make_float4(o[n][j][i], o[n][j][2 + i], o[n][j + 1][i], o[n][j + 1][2 + i]);
        if (g == 0) {
          mine[rows * kPartPitch<D> + r] = m[n][i];
          mine[rows * (kPartPitch<D> + 1) + r] = l[n][i];
        }
      }
    __syncthreads();

    // Joined over the warps: the output where the segment is all of the image,
    // else a part in the workspace. A CTA has at most one segment that goes on from
    // an earlier CTA's (slot 0) and one that begins an image without ending it
    // (slot 1).
    constexpr int kChunks = D / 8;
    const bool whole = !STREAM || (step0 == 0 && step1 == steps);
    float* slot = nullptr;
    if constexpr (STREAM)
      slot = a.parts +
             (2 * static_cast<int64_t>(blockIdx.x) + (step0 == 0 ? 1 : 0)) * part_floats<D>(rows);
    for (int x = threadIdx.x; x < rows * kChunks; x += kTokenThreads) {
      const int r = x / kChunks, col = 8 * (x - r * kChunks);
      float M, L, v[8];
      join_row<D>(kTokenWarps, [&](int p) { return smem + p * part_floats<D>(rows); }, rows, r, col,
                  M, L, v);
      if (whole) {
        put_row<T, D>(a, b, hk, r, col, len > 0, L, v);
      } else {
        float* to = slot + r * kPartPitch<D> + col;
        *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
        if (col == 0) {
          slot[rows * kPartPitch<D> + r] = M;
          slot[rows * (kPartPitch<D> + 1) + r] = L;
        }
      }
    }
    if constexpr (!STREAM) return;
    left -= step1 - step0;
    if (left == 0) return;
    __syncthreads();  // the results have been read: the next segment's copies may land
    step0 = 0;
    do
      if (++b == a.B) return;  // (steps are left, so an image with keys follows)
    while (keys_of(a, b) == 0);
  }
}

// Adds the parts of the images that several CTAs of the streaming kernel shared,
// in the order of their keys, and writes zeros for images without keys. One CTA per
// image and key head; `ctas` is that kernel's CTAs per head.
constexpr int kJoinThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
    cross_attention_join_kernel(const CrossTokenArgs a, int ctas) {
  __shared__ int total_before[2];
  __shared__ float row_inv[kTokenRows];
  extern __shared__ float factors[];  // [parts][rows]: 2^(m - M)
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int b = static_cast<int>(blockIdx.x) / a.kv_heads;
  const int hk = static_cast<int>(blockIdx.x) - b * a.kv_heads;
  const int steps = steps_of(a, b);
  if (warp < 2) {
    const int t = place_of(a, warp == 0 ? a.B : b, 0, lane).total;
    if (lane == 0) total_before[warp] = t;
  }
  __syncthreads();
  const Parts parts(total_before[0], ctas);
  const int begin = total_before[1];  // this image's first step
  int first = 0, count = 0;
  if (steps > 0) {
    first = parts.holder(begin);
    count = parts.holder(begin + steps - 1) - first + 1;
    if (count == 1) return;  // its CTA has written the output
  }
  const int rows = a.rows;
  // Part p: the first CTA began the image, the others went on with it.
  const int64_t stride = 2 * static_cast<int64_t>(a.kv_heads) * part_floats<D>(rows);
  const float* part0 = a.parts + first * stride + 2 * hk * part_floats<D>(rows);
  auto part = [&](int p) { return part0 + p * stride + (p == 0 ? part_floats<D>(rows) : 0); };
  // A row's maximum and sum over the parts, a lane per part.
  for (int r = warp; r < rows; r += kJoinThreads / 32) {
    float M = -INFINITY;
    for (int p = lane; p < count; p += 32) M = fmaxf(M, part(p)[rows * kPartPitch<D> + r]);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (M == -INFINITY) M = 0.f;
    float L = 0.f;
    for (int p = lane; p < count; p += 32) {
      const float f = ex2_approx(part(p)[rows * kPartPitch<D> + r] - M);
      factors[p * rows + r] = f;
      L = fmaf(part(p)[rows * (kPartPitch<D> + 1) + r], f, L);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) row_inv[r] = 1.f / L;
  }
  __syncthreads();
  // Four columns a thread; where that leaves threads over, groups of them take
  // every `groups`-th part and their sums meet in shared memory.
  constexpr int kQuads = D / 4;
  __shared__ float4 sums[kJoinThreads];
  const int cells = rows * kQuads;
  const int groups = max(1, kJoinThreads / cells);
  auto put = [&](int cell, float4 o) {
    const int r = cell / kQuads, col = 4 * (cell - r * kQuads);
    const float inv = count > 0 ? row_inv[r] : 0.f;
    const int t = r / a.group;
    const int64_t row = (static_cast<int64_t>(b) * a.Tq + t) * a.o_row +
                        (static_cast<int64_t>(hk) * a.group + (r - t * a.group)) * D;
    *reinterpret_cast<uint2*>(a.o + row + col) =
        make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
  };
  const int group = groups > 1 ? static_cast<int>(threadIdx.x) / cells : 0;
  for (int x = threadIdx.x - group * cells; x < cells && group < groups; x += kJoinThreads) {
    const int r = x / kQuads, col = 4 * (x - r * kQuads);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = group; p < count; p += groups) {
      const float4 t = *reinterpret_cast<const float4*>(part(p) + r * kPartPitch<D> + col);
      const float f = factors[p * rows + r];
      o.x = fmaf(t.x, f, o.x), o.y = fmaf(t.y, f, o.y);
      o.z = fmaf(t.z, f, o.z), o.w = fmaf(t.w, f, o.w);
    }
    if (groups == 1)
      put(x, o);
    else
      sums[threadIdx.x] = o;
  }
  if (groups == 1) return;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < cells) {
    float4 o = sums[threadIdx.x];
    for (int q = 1; q < groups; ++q) {
      const float4 t = sums[q * cells + threadIdx.x];
      o.x += t.x, o.y += t.y, o.z += t.z, o.w += t.w;
    }
    put(threadIdx.x, o);
  }
}

namespace {

template <int D>
int token_smem(int rows) {
  using C = TokenCfg<D>;
  return std::max(C::kRingBytes, C::kWarps * part_floats<D>(rows) * 4);
}

// CTAs per key head of the streaming form for this problem, or 0 where a CTA per
// image and key head does. Fitted: an SM reads 46 GB/s, the GPU 5.2 TB/s; streaming
// spreads the steps evenly, but finding its place in the list, further ramps and the
// second kernel cost some 12 us. Both sides measured: 32 images x 8 heads x 2048
// keys, D = 128, 55 us with a CTA each and 68 streaming; 2 x 8 x 32768, 367 and 66.
template <int D>
int stream_ctas(int B, int kv_heads, int Tk) {
  const int64_t items = static_cast<int64_t>(B) * kv_heads;
  const int64_t sms = device_num_sms();
  const int64_t slots = sms * TokenCfg<D>::kPerSm;
  const int64_t steps = (static_cast<int64_t>(Tk) + kStep - 1) / kStep;
  const double bytes = static_cast<double>(steps) * kStep * D * 4;  // of an image's key head
  const double waves = static_cast<double>((items + slots - 1) / slots);
  const double per_sm =
      static_cast<double>(std::min<int64_t>(TokenCfg<D>::kPerSm, (items + sms - 1) / sms));
  const double alone_us = waves * bytes * per_sm / 46e3;
  const double stream_us = static_cast<double>(items) * bytes / 5.2e6 + 12.0;
  if (alone_us <= stream_us) return 0;
  if (B * steps > INT32_MAX) return 0;  // the list is counted in 32 bits
  // A step a warp at least: the parts that are joined later cost time too.
  return static_cast<int>(std::min(slots / kv_heads, B * steps / TokenCfg<D>::kWarps));
}

template <typename T, int D, int NT>
int launch_token(const CrossTokenArgs& a, cudaStream_t s) {
  const int64_t items = static_cast<int64_t>(a.B) * a.kv_heads;
  const int ctas = stream_ctas<D>(a.B, a.kv_heads, a.Tk);
  if (ctas == 0)
    return launch_kernel(cross_attention_token_kernel<T, D, NT, false>,
                         dim3(static_cast<unsigned>(items)), dim3(TokenCfg<D>::kThreads),
                         static_cast<size_t>(token_smem<D>(a.rows)), s, 1, a);
  if (int st = launch_kernel(cross_attention_token_kernel<T, D, NT, true>,
                             dim3(static_cast<unsigned>(ctas) * static_cast<unsigned>(a.kv_heads)),
                             dim3(TokenCfg<D>::kThreads),
                             static_cast<size_t>(token_smem<D>(a.rows)), s, 1, a))
    return st;
  return launch_kernel(cross_attention_join_kernel<T, D>, dim3(static_cast<unsigned>(items)),
                       dim3(kJoinThreads), static_cast<size_t>(ctas) * a.rows * sizeof(float), s, 1,
                       a, ctas);
}

template <typename T, int D, int NT>
int allow_smem() {
  if (int st = cuda_status(cudaFuncSetAttribute(cross_attention_token_kernel<T, D, NT, false>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                token_smem<D>(8 * NT))))
    return st;
  return cuda_status(cudaFuncSetAttribute(cross_attention_token_kernel<T, D, NT, true>,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          token_smem<D>(8 * NT)));
}

// f(type, head size, tiles of eight rows) as types and constants.
template <typename F>
int with_token_form(int type, int D, int rows, F&& f) {
  auto sized = [&](auto tag, auto d) {
    return rows <= 8 ? f(tag, d, std::integral_constant<int, 1>{})
                     : f(tag, d, std::integral_constant<int, 2>{});
  };
  auto typed = [&](auto tag) {
    return D == 64 ? sized(tag, std::integral_constant<int, 64>{})
                   : sized(tag, std::integral_constant<int, 128>{});
  };
  return type == VITB200_BF16 ? typed(__nv_bfloat16{}) : typed(__half{});
}

}  // namespace

int cross_attention_token_prepare_device() {
  for (int type : {VITB200_F16, VITB200_BF16})
    for (int D : {64, 128})
      for (int rows : {8, kTokenRows})
        if (int st = with_token_form(type, D, rows, [](auto tag, auto d, auto nt) {
              return allow_smem<decltype(tag), decltype(d)::value, decltype(nt)::value>();
            }))
          return st;
  return 0;
}

size_t cross_attention_token_workspace(const CrossProblem& p) {
  const int rows = p.heads / p.kv_heads * p.Tq;
  const int ctas = p.kv_heads * (p.D == 64 ? stream_ctas<64>(p.B, p.kv_heads, p.Tk)
                                           : stream_ctas<128>(p.B, p.kv_heads, p.Tk));
  const int floats = p.D == 64 ? part_floats<64>(rows) : part_floats<128>(rows);
  return static_cast<size_t>(2) * ctas * floats * sizeof(float);
}

int cross_attention_token_launch(const CrossProblem& p, cudaStream_t s) {
  CrossTokenArgs a = {};
  a.q = static_cast<const uint16_t*>(p.q);
  a.k = static_cast<const uint16_t*>(p.k);
  a.v = static_cast<const uint16_t*>(p.v);
  a.o = static_cast<uint16_t*>(p.o);
  a.parts = static_cast<float*>(p.workspace);
  a.lens = p.lens;
  a.B = p.B;
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
  if (static_cast<int64_t>(p.B) * p.kv_heads > INT32_MAX) return VITB200_E_UNSUPPORTED;
  return with_token_form(p.type, p.D, a.rows, [&](auto tag, auto d, auto nt) {
    return launch_token<decltype(tag), decltype(d)::value, decltype(nt)::value>(a, s);
  });
}

}  // namespace vitb200
