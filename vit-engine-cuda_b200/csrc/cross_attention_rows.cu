// cross_attention (see cross_attention.cu for the operator) for short prompts: tiles
// of 64 packed rows (a key head's G query heads x Tq queries) on mma.sync.
//
// A tcgen05 CTA has an SM to itself (512 TMEM columns, 168 registers a thread of
// 384) and runs one dependent chain of S, softmax and P V per 128 rows; with 61 rows
// and five key tiles most of its time is set-up and waiting (384 image-heads of 61 x
// 577: 36 us). Here a CTA has four warps of 16 rows each, an SM up to four CTAs (two for
// D = 128), and they hide each other's chains. The legacy tensor path's lower rate, and
// K and V read again for every 64 rows, matter from the sizes on where the tcgen05
// kernel's set-up is small.
//
// Key tiles of 64 come through a two-deep ring in shared memory (16-byte chunks,
// XOR-swizzled by row: ldmatrix reads eight rows without bank conflicts, transposed
// for V). A launch with too few CTAs shares the key tiles out over a cluster; the
// partial results are joined in a fixed order through distributed shared memory.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "cross_attention.cuh"
#include "engine.h"

namespace vitb200 {

namespace {

constexpr int kRowsThreads = 128;
constexpr int kTileRows = 64;
constexpr int kTileKeys = 64;

template <int D>
struct RowsCfg {
  static constexpr int kChunks = D * 2 / 16;             // 16-byte chunks of a row
  static constexpr int kTile = kTileKeys * D * 2;        // bytes of a Q, K or V tile
  static constexpr int kSmem = 5 * kTile;                // Q, two of K, two of V
  static constexpr int kPerSm = D == 64 ? 4 : 2;
  // The partial result [64][D + 4] floats, then m and l, over the K and V ring.
  static constexpr int kPitch = D + 4;
  static_assert((kTileRows * (kPitch + 2)) * 4 <= 4 * kTile, "partial results fit the ring");
};

struct CrossRowsArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const int* lens;
  int Tq, Tk, kv_heads;
  int group;   // query heads per key head
  int rows;    // group * Tq
  int tiles;   // row tiles per image and key head
  int nsplit;  // CTAs that share a row tile's keys
  float c;     // |scale| * log2(e)
  int negate;  // scale < 0
  int64_t q_row, q_batch, k_row, k_batch, v_row, v_batch, o_row;
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Byte offset of chunk `ch` of row `row` in a tile.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int row, int ch) {
  return static_cast<uint32_t>(row * (D * 2) + 16 * (ch ^ (row & 7)));
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kRowsThreads, RowsCfg<D>::kPerSm)
    cross_attention_rows_kernel(const CrossRowsArgs a) {
  using C = RowsCfg<D>;
  extern __shared__ __align__(128) uint8_t smem_rows[];
  griddep_wait();
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int split = static_cast<int>(blockIdx.x) % a.nsplit;  // = rank in the cluster
  const int item = static_cast<int>(blockIdx.x) / a.nsplit;
  const int bh = item / a.tiles;
  const int row0 = (item - bh * a.tiles) * kTileRows;  // first packed row
  const int b = bh / a.kv_heads;
  const int hk = bh - b * a.kv_heads;
  int len = a.Tk;
  if (a.lens != nullptr) len = max(0, min(a.Tk, __ldg(a.lens + b)));
  const int all = (len + kTileKeys - 1) / kTileKeys;
  const int j0 = static_cast<int>(static_cast<int64_t>(all) * split / a.nsplit);
  const int j1 = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.nsplit);

  const uint32_t sq = smem_addr(smem_rows);
  const uint32_t sk = sq + C::kTile, sv = sk + 2 * C::kTile;
  const uint16_t* kp = a.k + b * a.k_batch + static_cast<int64_t>(hk) * D;
  const uint16_t* vp = a.v + b * a.v_batch + static_cast<int64_t>(hk) * D;
  // Keys past the length arrive as zeros: a value there may be NaN.
  auto fetch = [&](int j, int stage) {
    if (j < j1) {
#pragma unroll
      for (int i = 0; i < kTileKeys * C::kChunks / kRowsThreads; ++i) {
        const int x = i * kRowsThreads + static_cast<int>(threadIdx.x);
        const int r = x / C::kChunks, ch = x - r * C::kChunks;
        const int key = j * kTileKeys + r;
        const bool in = key < len;
        const int64_t at = in ? key : 0;
        const uint32_t to = stage * C::kTile + chunk_at<D>(r, ch);
        copy_async16(sk + to, kp + at * a.k_row + 8 * ch, in);
        copy_async16(sv + to, vp + at * a.v_row + 8 * ch, in);
      }
    }
    copy_async_commit();
  };
  // Output row of packed row r.
  auto q_offset = [&](int r, int64_t row, int64_t batch) {
    const int t = r / a.group;
    return b * batch + t * row + (static_cast<int64_t>(hk) * a.group + (r - t * a.group)) * D;
  };
#pragma unroll
  for (int i = 0; i < kTileRows * C::kChunks / kRowsThreads; ++i) {
    const int x = i * kRowsThreads + static_cast<int>(threadIdx.x);
    const int r = x / C::kChunks, ch = x - r * C::kChunks;
    const bool in = row0 + r < a.rows;
    copy_async16(sq + chunk_at<D>(r, ch),
                 a.q + q_offset(in ? row0 + r : 0, a.q_row, a.q_batch) + 8 * ch, in);
  }
  fetch(j0, 0);  // Q travels with the first tile

  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  // Rows g and g + 8: the largest score so far, the sum of this lane's exponentials.
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  bool huge = false;  // some m * c of the warp's rows is past kHugeScore
  uint32_t q[D / 16][4];
  const int sub = lane >> 3, sr = lane & 7;  // ldmatrix: this lane's matrix and row
  for (int j = j0; j < j1; ++j) {
    const int stage = (j - j0) & 1;
    fetch(j + 1, stage ^ 1);
    copy_async_wait<1>();
    __syncthreads();
    if (j == j0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        ldmatrix_x4(q[kk], sq + chunk_at<D>(warp * 16 + (sub & 1) * 8 + sr, 2 * kk + (sub >> 1)));
    }
    const uint32_t k_tile = sk + stage * C::kTile, v_tile = sv + stage * C::kTile;
    float s[kTileKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kTileKeys / 8; n += 2) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      s[n + 1][0] = s[n + 1][1] = s[n + 1][2] = s[n + 1][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t kb[4];
        ldmatrix_x4(kb, k_tile + chunk_at<D>(8 * n + (sub >> 1) * 8 + sr, 2 * kk + (sub & 1)));
        mma_16x8x16<T>(s[n], q[kk], kb[0], kb[1]);
        mma_16x8x16<T>(s[n + 1], q[kk], kb[2], kb[3]);
      }
    }
    if (a.negate) {  // a negative scale: its magnitude, and the scores turned round
#pragma unroll
      for (int n = 0; n < kTileKeys / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = -s[n][i];
    }
    const int valid = len - j * kTileKeys;
    if (valid < kTileKeys) {
#pragma unroll
      for (int n = 0; n < kTileKeys / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (8 * n + 2 * c + (i & 1) >= valid) s[n][i] = -INFINITY;
    }
    bool grew = false;
    float f[2], ref[2];  // ref: m in log2 units
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = s[0][2 * h];
      top = fmaxf(top, s[0][2 * h + 1]);
#pragma unroll
      for (int n = 1; n < kTileKeys / 8; ++n) top = max3(top, s[n][2 * h], s[n][2 * h + 1]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, m[h]);
      grew |= top > m[h];
      f[h] = ex2_approx((m[h] - (top == -INFINITY ? 0.f : top)) * a.c);
      m[h] = top;
      ref[h] = top == -INFINITY ? 0.f : top * a.c;
    }
    if (__any_sync(0xffffffffu, grew)) {
      huge = __any_sync(0xffffffffu, fmaxf(fabsf(ref[0]), fabsf(ref[1])) > kHugeScore);
      l[0] *= f[0];
      l[1] *= f[1];
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        o[n][0] *= f[0], o[n][1] *= f[0], o[n][2] *= f[1], o[n][3] *= f[1];
    }
    if (huge) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool row = fabsf(ref[h]) > kHugeScore;
        const float off = row ? m[h] : 0.f;
        if (row) ref[h] = 0.f;
#pragma unroll
        for (int n = 0; n < kTileKeys / 8; ++n) s[n][2 * h] -= off, s[n][2 * h + 1] -= off;
      }
    }
    ref[0] -= kLift<T>, ref[1] -= kLift<T>;
#pragma unroll
    for (int kk = 0; kk < kTileKeys / 16; ++kk) {
      uint32_t p[4];  // the scores' layout is the product's: keys 16 kk + 2 c + {0, 1, 8, 9}
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* x = &s[2 * kk + (i >> 1)][2 * (i & 1)];
        const float e0 = ex2_approx(fmaf(x[0], a.c, -ref[i & 1]));
        const float e1 = ex2_approx(fmaf(x[1], a.c, -ref[i & 1]));
        l[i & 1] += e0 + e1;
        p[i] = pack2<T>(e0, e1);
      }
#pragma unroll
      for (int n = 0; n < D / 8; n += 2) {
        uint32_t vb[4];
        ldmatrix_x4_trans(vb,
                          v_tile + chunk_at<D>(16 * kk + (sub & 1) * 8 + sr, n + (sub >> 1)));
        mma_16x8x16<T>(o[n], p, vb[0], vb[1]);
        mma_16x8x16<T>(o[n + 1], p, vb[2], vb[3]);
      }
    }
    __syncthreads();  // the tile has been read: the next copies may land
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }
  copy_async_wait<0>();

  // (Stored as they lie in registers: through shared memory, in 16-byte pieces, the
  // rows' addresses cost more than the wider stores save, 88 against 80 us at 300
  // heads of 2224 rows.)
  if (a.nsplit == 1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row0 + warp * 16 + g + 8 * h;
      if (r >= a.rows) continue;
      const float inv = len > 0 ? 1.f / l[h] : 0.f;
      uint16_t* to = a.o + q_offset(r, a.o_row, static_cast<int64_t>(a.Tq) * a.o_row) + 2 * c;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<uint32_t*>(to + 8 * n) =
            len > 0 ? pack2<T>(o[n][2 * h] * inv, o[n][2 * h + 1] * inv) : 0u;
    }
    return;
  }

  // Several CTAs: partial results in shared memory (a CTA without tiles leaves an
  // empty one), each CTA joins and writes a share of the rows.
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem_rows + C::kTile);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = warp * 16 + g + 8 * h;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2*>(part + r * C::kPitch + 8 * n + 2 * c) =
          make_float2(o[n][2 * h], o[n][2 * h + 1]);
    if (c == 0) {
      part[kTileRows * C::kPitch + r] = m[h] * a.c;
      part[kTileRows * (C::kPitch + 1) + r] = l[h];
    }
  }
  __syncwarp();
  cluster_sync_all();
  const uint32_t mine = smem_addr(part);
  const int rows = min(kTileRows, a.rows - row0);
  for (int x = split * kRowsThreads + static_cast<int>(threadIdx.x); x < rows * (D / 8);
       x += a.nsplit * kRowsThreads) {
    const int r = x / (D / 8), col = 8 * (x - r * (D / 8));
    float M = -INFINITY, L = 0.f, v[8] = {};
    for (int p = 0; p < a.nsplit; ++p)
      M = fmaxf(M, ld_partial(mapa_shared(mine, p) + 4u * (kTileRows * C::kPitch + r), true));
    if (M == -INFINITY) M = 0.f;
    for (int p = 0; p < a.nsplit; ++p) {
      const uint32_t src = mapa_shared(mine, static_cast<uint32_t>(p));
      const float w = ex2_approx(ld_partial(src + 4u * (kTileRows * C::kPitch + r), true) - M);
      L = fmaf(ld_partial(src + 4u * (kTileRows * (C::kPitch + 1) + r), true), w, L);
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 t = ld_partial4(src + 4u * (r * C::kPitch + col + i), true);
        v[i] = fmaf(t.x, w, v[i]), v[i + 1] = fmaf(t.y, w, v[i + 1]);
        v[i + 2] = fmaf(t.z, w, v[i + 2]), v[i + 3] = fmaf(t.w, w, v[i + 3]);
      }
    }
    uint4 w = make_uint4(0, 0, 0, 0);
    if (len > 0) {
      const float inv = 1.f / L;
      w = make_uint4(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv),
                     pack2<T>(v[4] * inv, v[5] * inv), pack2<T>(v[6] * inv, v[7] * inv));
    }
    *reinterpret_cast<uint4*>(
        a.o + q_offset(row0 + r, a.o_row, static_cast<int64_t>(a.Tq) * a.o_row) + col) = w;
  }
  __syncwarp();
  cluster_sync_all();  // no CTA exits while its result may be read
}

namespace {

template <typename T, int D>
int launch_rows(const CrossRowsArgs& args, int B, cudaStream_t s) {
  using C = RowsCfg<D>;
  CrossRowsArgs a = args;
  const int64_t items = static_cast<int64_t>(B) * a.kv_heads * a.tiles;
  if (items > INT32_MAX / kCrossMaxSplit) return VITB200_E_UNSUPPORTED;
  const int64_t slots = static_cast<int64_t>(device_num_sms()) * C::kPerSm;
  const int64_t key_tiles = (static_cast<int64_t>(a.Tk) + kTileKeys - 1) / kTileKeys;
  // Up to a CTA per slot, with two key tiles each at least.
  a.nsplit = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({slots / items, key_tiles / 2, kCrossMaxSplit})));
  while (a.nsplit > 1 && cluster_slots(cross_attention_rows_kernel<T, D>, C::kSmem, kRowsThreads,
                                       a.nsplit) < items)
    --a.nsplit;
  return launch_kernel(cross_attention_rows_kernel<T, D>,
                       dim3(static_cast<unsigned>(items * a.nsplit)), dim3(kRowsThreads), C::kSmem,
                       s, static_cast<unsigned>(a.nsplit), a);
}

template <typename T, int D>
int allow_smem() {
  return cuda_status(cudaFuncSetAttribute(cross_attention_rows_kernel<T, D>,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          RowsCfg<D>::kSmem));
}

}  // namespace

int cross_attention_rows_prepare_device() {
  if (int st = allow_smem<__half, 64>()) return st;
  if (int st = allow_smem<__half, 128>()) return st;
  if (int st = allow_smem<__nv_bfloat16, 64>()) return st;
  return allow_smem<__nv_bfloat16, 128>();
}

int cross_attention_rows_launch(const CrossProblem& p, cudaStream_t s) {
  CrossRowsArgs a = {};
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
  a.tiles = (a.rows + kTileRows - 1) / kTileRows;
  a.q_row = p.q_row;
  a.q_batch = p.q_batch;
  a.k_row = p.k_row;
  a.k_batch = p.k_batch;
  a.v_row = p.v_row;
  a.v_batch = p.v_batch;
  a.o_row = static_cast<int64_t>(p.heads) * p.D;
  a.c = cross_scale(fabsf(p.scale));
  a.negate = p.scale < 0.f;
  if (p.type == VITB200_BF16)
    return p.D == 64 ? launch_rows<__nv_bfloat16, 64>(a, p.B, s)
                     : launch_rows<__nv_bfloat16, 128>(a, p.B, s);
  return p.D == 64 ? launch_rows<__half, 64>(a, p.B, s) : launch_rows<__half, 128>(a, p.B, s);
}

}  // namespace vitb200
