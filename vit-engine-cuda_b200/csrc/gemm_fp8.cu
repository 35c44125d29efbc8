// FP8 matrix product with one fp32 scale per block of 128:
//
//   Y[m][n] = epilogue( sum_kb xs[m][kb] * ws[n / 128][kb]
//                       * sum_{k in block kb} X[m][k] * W[n][k] )
//
// X[M][K], W[N][K] e4m3 (PyTorch Linear layout), X scaled per row and 128
// columns, W per 128 x 128 block; epilogue = bias, erf-GELU, residual, in that
// order, in fp32 and rounded once to the output's type.
//
// The scales change every 128 columns of K, so the tensor core may only sum
// one block at a time: a K block is four tcgen05.mma.kind::f8f6f4 (K = 32) into
// a fresh TMEM accumulator, which the epilogue warps read back and add, times
// the block's two scales, to fp32 sums in registers. (That also bounds the
// tensor core's truncating accumulation to four steps.) A 128 x 128 block takes
// 256 cycles on the tensor core, and its read-back 128 cycles of TMEM bandwidth
// and 128 issue slots of FMAs per scheduler: both fit under the products when
// they overlap, which is what the double-buffered accumulators are for.
//
// Two kernels:
//  * gemm_fp8_pair_kernel, for outputs of many tiles: persistent, 256 x 256
//    tiles on a CTA pair (tcgen05 cta_group::2). One SM's 128 x 256 half needs
//    32 KB of operands per K block and 512 cycles, so shared memory feeds the
//    tensor core at half its bandwidth; a single-CTA 128 x 128 tile would need
//    all of it.
//  * gemm_fp8_tile_kernel, for the rest: one 128 x BN tile per cluster of
//    `ksplit` CTAs that share the K blocks out; their partial sums meet in
//    distributed shared memory, added in split order, so results do not depend
//    on timing and no workspace is needed.
// Every wait is bounded (device error word).
#include <algorithm>
#include <type_traits>

#include "engine.h"
#include "fp8.cuh"

namespace vitb200 {

namespace {

constexpr int kBM = 128;          // rows of X per CTA
constexpr int kBK = kFp8Block;    // one K block: 128 bytes, one swizzle span
constexpr int kTmemAll = 512;
constexpr int kThreads = 384;     // control warpgroup + two epilogue warpgroups
constexpr int kABytes = kBM * kBK;

struct Fp8GemmArgs {
  int64_t M;
  int N;
  int num_kb;
  int num_n_tiles;
  int num_tiles;
  int ksplit;         // tile kernel: CTAs that share a tile's K blocks
  int a_rows;         // tile kernel: rows of the X box (M rounded up to 8, at most 128)
  const float* xs;    // [M][num_kb]
  int64_t ldxs;
  const float* ws;    // [ceil(N / 128)][num_kb]
  int64_t ldws;
  const float* bias;  // [N] or null
  const void* residual;
  int64_t ldr;
  void* out;
  int64_t ldo;
  int gelu;
  int vec_xs;         // rows of X's scales take four at a time
  int tma_out;        // the result goes out through tmap_out
  int tma_res;        // the residual comes in through tmap_res
  int vec;            // tile kernel: out, residual and bias take four columns at a time
  int* err;
};

// D[tmem] (+)= A * B^T, kind::f8f6f4 (e4m3 operands, fp32 accumulator).
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// e4m3 is format 0 of this kind, as f16 is of kind::f16: the same descriptor bits.
constexpr uint32_t make_idesc_f8(int M, int N) { return make_idesc_f16(M, N); }

// Lane 0 waits; the verdict is broadcast so that the warp stays converged.
__device__ __forceinline__ bool warp_wait8(uint64_t* bar, uint32_t parity, int* err, int code,
                                           int lane) {
  int ok = 1;
  if (lane == 0) ok = mbar_wait(bar, parity, err, code) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// Bounded wait on the way out, whatever the error word says: asynchronous work
// in flight has to land before the CTA exits.
__device__ __forceinline__ void drain_wait8(uint64_t* bar, uint32_t parity, int* err) {
  const uint32_t addr = smem_addr(bar);
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(addr, parity)) {
    if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
      report_error(err, kErrDrain);
      return;
    }
  }
}

// sum[i] += s * (column i of the accumulator at taddr), 16 columns at a time,
// each load in flight while the previous 16 are added; `release` runs as soon as
// the last has arrived. (Loads of 32 columns spilled and ran 3 % slower.)
template <int COLS, typename Release>
__device__ __forceinline__ void drain_block(uint32_t taddr, float s, float2 (&sum)[COLS / 2],
                                            Release&& release) {
  const float2 s2 = splat2(s);
  uint32_t r[2][16];
  tmem_ld_issue_x16(taddr, r[0]);
#pragma unroll
  for (int i = 0; i < COLS / 16; ++i) {
    uint32_t(&t)[16] = r[i & 1];
    tmem_ld_wait_x16(t);
    if (i + 1 < COLS / 16)
      tmem_ld_issue_x16(taddr + static_cast<uint32_t>(16 * (i + 1)), r[(i + 1) & 1]);
    else
      release();
#pragma unroll
    for (int c = 0; c < 8; ++c)
      sum[8 * i + c] =
          fma2(s2, make_float2(__uint_as_float(t[2 * c]), __uint_as_float(t[2 * c + 1])),
               sum[8 * i + c]);
  }
}

// ---------------------------------------------------------------- CTA pair
constexpr int kPairBN = 256;
constexpr int kWgCols = kPairBN / 2;             // columns of a tile an epilogue warpgroup owns
constexpr int kPairBRows = kPairBN / 2;
constexpr int kPairStageBytes = kABytes + kPairBRows * kBK;
// Five stages: six measure the same (319-342 us against 324-343 in the long run at 16384
// x 4096 x 4096 with GELU) and leave L1 too small for the scales' lines.
constexpr int kPairStages = 5;
constexpr int kPairBufs = kTmemAll / kPairBN;
// Per epilogue warp: one slab of the result or residual.
constexpr int kSlabBytes = 32 * 128;
constexpr int kPairSmem = kPairStages * kPairStageBytes + 8 * kSlabBytes + 1024;
static_assert(kPairSmem <= 227 * 1024, "shared memory");
// 384 threads launched at 168 registers; the control warpgroup drops to 56 and
// the epilogue warpgroups (128 sums and two loads of 16 a thread) rise to 224:
// 128 * 56 + 256 * 224 = 384 * 168. build.py checks that ptxas allocated 168.
// Four epilogue warpgroups of 64 columns (104 registers) measured 322-357 us when two
// took 317-322.
constexpr uint32_t kPairCtrlRegs = 56;
constexpr uint32_t kPairEpiRegs = 224;
static_assert(128 * kPairCtrlRegs + 256 * kPairEpiRegs == kThreads * 168, "register split");

// A slab is 32 rows of 128 bytes: the 16-byte chunk q of row r lies where the
// 128-byte swizzle of the tensor map that stores it puts it, which also keeps a
// lane writing its own row free of bank conflicts.
__device__ __forceinline__ int slab_at(int r, int q) { return r * 128 + 16 * (q ^ (r & 7)); }
template <typename T>
constexpr int kSlabCols = 128 / sizeof(T);

template <typename T>
__device__ __forceinline__ void add_chunk(const uint8_t* p, float* v) {
  const uint4 t = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&t);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) v[i] = to_f32(e[i]) + v[i];
}
template <typename T>
__device__ __forceinline__ void put_chunk(uint8_t* p, const float* v) {
  uint4 t;
  T* e = reinterpret_cast<T*>(&t);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<uint4*>(p) = t;
}

// Epilogue of a warp's slab (lane i = row m_base + i, columns n0..), warp-
// collective. `slab` is the warp's buffer, `res_bar` its residual barrier.
template <typename T>
__device__ __forceinline__ void finish_slab(const Fp8GemmArgs& a, int64_t m_base, int lane, int n0,
                                            float2* v, uint8_t* slab,
                                            const CUtensorMap* tmap_out,
                                            const CUtensorMap* tmap_res, uint64_t* res_bar,
                                            uint32_t& res_phase) {
  constexpr int kCols = kSlabCols<T>;
  constexpr int kPer = 16 / sizeof(T);  // columns per 16-byte chunk
  const int64_t m = m_base + lane;
  if (a.tma_res && lane == 0) {
    bulk_wait_group_read<0>();  // the previous slab's store has read the buffer
    mbar_arrive_expect_tx(res_bar, kSlabBytes);
    tma_load_2d(slab, tmap_res, res_bar, n0, static_cast<int>(m_base));
  }
  if (a.bias != nullptr) {
    if (n0 + kCols <= a.N && (reinterpret_cast<uintptr_t>(a.bias) & 15) == 0) {
#pragma unroll
      for (int j = 0; j < kCols / 4; ++j) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(a.bias + n0) + j);
        v[2 * j] = add2(v[2 * j], make_float2(b.x, b.y));
        v[2 * j + 1] = add2(v[2 * j + 1], make_float2(b.z, b.w));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) {
        v[j].x += n0 + 2 * j < a.N ? __ldg(a.bias + n0 + 2 * j) : 0.f;
        v[j].y += n0 + 2 * j + 1 < a.N ? __ldg(a.bias + n0 + 2 * j + 1) : 0.f;
      }
    }
  }
  if (a.gelu) {
#pragma unroll
    for (int j = 0; j < kCols / 2; ++j) v[j] = gelu_erf2(v[j]);
  }
  if (a.tma_res) {
    if (!mbar_wait(res_bar, res_phase, a.err, kErrWaitFull)) drain_wait8(res_bar, res_phase, a.err);
    res_phase ^= 1u;
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q)
      add_chunk<T>(slab + slab_at(lane, q), reinterpret_cast<float*>(v + q * kPer / 2));
    __syncwarp();
  } else if (a.residual != nullptr && m < a.M) {
    const T* r = static_cast<const T*>(a.residual) + m * a.ldr + n0;
#pragma unroll
    for (int j = 0; j < kCols / 2; ++j) {
      if (n0 + 2 * j < a.N) v[j].x = to_f32(r[2 * j]) + v[j].x;
      if (n0 + 2 * j + 1 < a.N) v[j].y = to_f32(r[2 * j + 1]) + v[j].y;
    }
  }
  if (a.tma_out) {
    if (!a.tma_res) {
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
    }
#pragma unroll
    for (int q = 0; q < 8; ++q)
      put_chunk<T>(slab + slab_at(lane, q), reinterpret_cast<const float*>(v + q * kPer / 2));
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(tmap_out, slab, n0, static_cast<int>(m_base));
      bulk_commit_group();
    }
  } else if (m < a.M) {
    T* o = static_cast<T*>(a.out) + m * a.ldo + n0;
#pragma unroll
    for (int j = 0; j < kCols / 2; ++j) {
      if (n0 + 2 * j < a.N) o[2 * j] = from_f32<T>(v[j].x);
      if (n0 + 2 * j + 1 < a.N) o[2 * j + 1] = from_f32<T>(v[j].y);
    }
  }
}

__device__ __forceinline__ void prefetch_l1(const void* p) {
  asm volatile("prefetch.global.L1 [%0];" ::"l"(p));
}

// A row's scales of K blocks kb .. kb + 3 (those past the last are not read).
__device__ __forceinline__ float4 load_scales(const float* xs, int kb, int num_kb, int vec) {
  if (vec && kb + 4 <= num_kb) return __ldg(reinterpret_cast<const float4*>(xs + kb));
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (kb < num_kb) v.x = __ldg(xs + kb);
  if (kb + 1 < num_kb) v.y = __ldg(xs + kb + 1);
  if (kb + 2 < num_kb) v.z = __ldg(xs + kb + 2);
  if (kb + 3 < num_kb) v.w = __ldg(xs + kb + 3);
  return v;
}

// Output tile `t`: bands of kBandN column tiles, row block by row block with the band's
// columns running fastest, so that the tiles in flight share few rows of X and W in L2.
constexpr int kBandN = 8;
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& m, int& n) {
  const int band = t / (m_tiles * kBandN);
  const int width = min(kBandN, n_tiles - band * kBandN);
  const int rem = t - band * m_tiles * kBandN;
  m = rem / width;
  n = band * kBandN + rem - m * width;
}

}  // namespace

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_x,
                         const __grid_constant__ CUtensorMap tmap_w,
                         const __grid_constant__ CUtensorMap tmap_out,
                         const __grid_constant__ CUtensorMap tmap_res, const Fp8GemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kPairStages];
  // A K block's products are done: its stage is free and its accumulator full.
  // One barrier serves producer and epilogue, so a block costs one commit. The
  // epilogue cannot fall a turn of the ring behind: block s + kPairStages needs
  // an accumulator that every warp has drained after block s.
  __shared__ __align__(8) uint64_t done_bar[kPairStages];
  __shared__ __align__(8) uint64_t acc_empty_bar[kPairBufs];
  __shared__ __align__(8) uint64_t mma_done_bar;
  __shared__ __align__(8) uint64_t res_bar[8];
  __shared__ uint32_t tmem_slot;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int* err = a.err;
  const uint32_t rank = cluster_ctarank();  // rank 0 issues the pair's MMAs
  const bool leader = rank == 0;
  const int unit = static_cast<int>(blockIdx.x >> 1);
  const int num_units = static_cast<int>(gridDim.x >> 1);
  const uint32_t raw = smem_addr(smem_raw);
  uint8_t* ring = smem_raw + (((raw + 1023u) & ~1023u) - raw);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&done_bar[s], 1);
    }
    for (int b = 0; b < kPairBufs; ++b) {
      mbar_init(&acc_empty_bar[b], 16);  // every epilogue warp of both CTAs
    }
    mbar_init(&mma_done_bar, 1);
    for (int i = 0; i < 8; ++i) mbar_init(&res_bar[i], 1);
    fence_barrier_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  cluster_sync_all();  // the peer's barriers exist before any remote use
  if (warp == 1) {
    tmem_alloc_pair(&tmem_slot, kTmemAll);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int num_kb = a.num_kb;
  const int m_tiles = a.num_tiles / a.num_n_tiles;

  if (warp < 4) {
    setmaxnreg_dec<kPairCtrlRegs>();
    if (warp == 0 && elect_one()) {
      // ------------------------------------------------------------ TMA
      int stage = 0;
      uint32_t phase = 0;
      int64_t issued = 0;
      bool ok = true;
      for (int t = unit; t < a.num_tiles && ok; t += num_units) {
        int mb, nb;
        tile_at(t, m_tiles, a.num_n_tiles, mb, nb);
        const int x_row = mb * 2 * kBM + static_cast<int>(rank) * kBM;
        const int w_row = nb * kPairBN + static_cast<int>(rank) * kPairBRows;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&done_bar[stage], phase ^ 1u, err, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          uint8_t* sx = ring + stage * kPairStageBytes;
          // Both CTAs' copies complete on the leader's barrier.
          const uint32_t full_leader = mapa_shared(smem_addr(&full_bar[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * kPairStageBytes);
          tma_load_2d_pair(sx, &tmap_x, full_leader, kb * kBK, x_row);
          tma_load_2d_pair(sx + kABytes, &tmap_w, full_leader, kb * kBK, w_row);
          ++issued;
          if (++stage == kPairStages) stage = 0, phase ^= 1u;
        }
      }
      // Every copy issued lands before the CTAs can exit.
      if (leader) {
        for (int s = 0; s < kPairStages; ++s)
          if (issued > s) {
            const int64_t fills = (issued - s + kPairStages - 1) / kPairStages;
            drain_wait8(&full_bar[s], static_cast<uint32_t>((fills - 1) & 1), err);
          }
      }
    } else if (warp == 1 && leader && elect_one()) {
      // ------------------------------------------------------------ MMA
      constexpr uint32_t kIdesc = make_idesc_f8(2 * kBM, kPairBN);
      int stage = 0;
      uint32_t phase = 0;
      uint32_t seq = 0;  // K blocks so far: accumulator seq % 2, its use seq / 2
      bool ok = true;
      for (int t = unit; t < a.num_tiles && ok; t += num_units) {
        for (int kb = 0; kb < num_kb; ++kb, ++seq) {
          const int buf = static_cast<int>(seq % kPairBufs);
          const uint32_t use = seq / kPairBufs;
          if (!mbar_wait(&acc_empty_bar[buf], (use & 1u) ^ 1u, err, kErrWaitAccEmpty) ||
              !mbar_wait(&full_bar[stage], phase, err, kErrWaitFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem_base + static_cast<uint32_t>(buf * kPairBN);
          const uint32_t sx = smem_addr(ring + stage * kPairStageBytes);
          const uint64_t dx = make_sdesc_kmajor(sx, kBK);
          const uint64_t dw = make_sdesc_kmajor(sx + kABytes, kBK);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 32 columns = 32 bytes = +2 in the address field
            umma_f8_pair(d, dx + 2 * kk, dw + 2 * kk, kIdesc, kk ? 1u : 0u);
          umma_commit_both(&done_bar[stage]);
          if (++stage == kPairStages) stage = 0, phase ^= 1u;
        }
      }
      // Every MMA issued finishes before TMEM is released.
      umma_commit_pair(smem_addr(&mma_done_bar));
      drain_wait8(&mma_done_bar, 0, err);
    }
  } else {
    setmaxnreg_inc<kPairEpiRegs>();
    // ------------------------------------------------------------ epilogue
    // Warpgroup wg owns the tile's columns [128 wg, 128 wg + 128), one W scale
    // block; a thread owns one row, so a block's scale is one number a thread.
    const int wg = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                               static_cast<uint32_t>(wg * kWgCols);
    uint8_t* slab = ring + kPairStages * kPairStageBytes + (warp - 4) * kSlabBytes;
    uint32_t res_phase = 0;
    uint32_t seq = 0;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = unit; t < a.num_tiles && ok; t += num_units) {
      int mb, nb;
      tile_at(t, m_tiles, a.num_n_tiles, mb, nb);
      const int64_t m_base = static_cast<int64_t>(mb) * 2 * kBM + rank * kBM + quarter * 32;
      const int n_base = nb * kPairBN + wg * kWgCols;
      // Tiles at the edges: warps whose rows or columns lie outside read nothing.
      const bool live = m_base < a.M && n_base < a.N;
      const float* xs = a.xs + (m_base + lane < a.M ? m_base + lane : a.M - 1) * a.ldxs;
      const float* ws = a.ws + static_cast<int64_t>(live ? n_base / kFp8Block : 0) * a.ldws;
      float2 sum[kWgCols / 2];
#pragma unroll
      for (int c = 0; c < kWgCols / 2; ++c) sum[c] = make_float2(0.f, 0.f);
      if (a.bias != nullptr && n_base + 4 * lane < a.N) prefetch_l1(a.bias + n_base + 4 * lane);
      float4 sx = load_scales(xs, 0, num_kb, a.vec_xs), sx_next = sx;
      float sw = __ldg(ws);
      for (int kb = 0; kb < num_kb; ++kb, ++seq) {
        const int buf = static_cast<int>(seq % kPairBufs);
        const int u = kb & 3;
        if (u == 0) {
          sx = sx_next;
          sx_next = load_scales(xs, kb + 4, num_kb, a.vec_xs);
        }
        const float s = sw * (u & 2 ? (u & 1 ? sx.w : sx.z) : (u & 1 ? sx.y : sx.x));
        sw = __ldg(ws + (kb + 1 < num_kb ? kb + 1 : kb));
        if (!mbar_wait(&done_bar[stage], phase, err, kErrWaitAccFull)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        auto release = [&] {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (leader)
              mbar_arrive(&acc_empty_bar[buf]);
            else
              mbar_arrive_remote(mapa_shared(smem_addr(&acc_empty_bar[buf]), 0));
          }
        };
        if (live)
          drain_block<kWgCols>(lane_base + static_cast<uint32_t>(buf * kPairBN), s, sum, release);
        else
          release();
        if (++stage == kPairStages) stage = 0, phase ^= 1u;
      }
      if (!ok) break;
      if (live) {
        // One copy of the slab code: the sums move down by a slab after each.
        constexpr int kCols = kSlabCols<T>;
#pragma unroll 1
        for (int n0 = n_base; n0 < n_base + kWgCols; n0 += kCols) {
          if (n0 < a.N)
            finish_slab<T>(a, m_base, lane, n0, sum, slab, &tmap_out, &tmap_res,
                           &res_bar[warp - 4], res_phase);
#pragma unroll
          for (int c = 0; c < (kWgCols - kCols) / 2; ++c) sum[c] = sum[c + kCols / 2];
        }
      }
    }
    if (a.tma_out && lane == 0) bulk_wait_group<0>();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemAll);
  }
}

// ---------------------------------------------------------------- one tile
namespace {

template <int BN>
struct TileCfg {
  static constexpr int kBBytes = BN * kBK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = BN == 128 ? 6 : 8;
  static constexpr int kPitch = BN + 4;  // floats per row of the partial sums
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kBufs = 4;        // accumulators in TMEM
  static constexpr int kTmem = kBufs * BN;
  static constexpr int kWgCols = BN / 2; // columns per epilogue warpgroup
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static_assert(kBM * kPitch * 4 <= kStages * kStageBytes, "partial sums fit the ring");
};

}  // namespace

template <typename T, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap tmap_x,
                         const __grid_constant__ CUtensorMap tmap_w, const Fp8GemmArgs a) {
  using Cfg = TileCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[Cfg::kStages];
  __shared__ __align__(8) uint64_t empty_bar[Cfg::kStages];
  __shared__ __align__(8) uint64_t acc_full_bar[Cfg::kBufs];
  __shared__ __align__(8) uint64_t acc_empty_bar[Cfg::kBufs];
  __shared__ __align__(8) uint64_t mma_done_bar;
  __shared__ uint32_t tmem_slot;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int* err = a.err;
  const int ksplit = a.ksplit;
  const int tile = static_cast<int>(blockIdx.x) / ksplit;
  const int split = static_cast<int>(blockIdx.x) - tile * ksplit;  // = rank in the cluster
  const int mb = tile / a.num_n_tiles;
  const int nb = tile - mb * a.num_n_tiles;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.num_kb) * split / ksplit);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.num_kb) * (split + 1) / ksplit);
  const uint32_t raw = smem_addr(smem_raw);
  uint8_t* ring = smem_raw + (((raw + 1023u) & ~1023u) - raw);

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < Cfg::kBufs; ++b) {
      mbar_init(&acc_full_bar[b], 1);
      mbar_init(&acc_empty_bar[b], 8);
    }
    mbar_init(&mma_done_bar, 1);
    fence_barrier_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, Cfg::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int64_t m_tile = static_cast<int64_t>(mb) * kBM;
  float* part = reinterpret_cast<float*>(ring);  // [128][kPitch] once the ring is idle

  if (warp == 0 && elect_one()) {
    // -------------------------------------------------------------- TMA
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    const uint32_t bytes = static_cast<uint32_t>(a.a_rows * kBK + Cfg::kBBytes);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(&empty_bar[stage], phase ^ 1u, err, kErrWaitEmpty)) break;
      uint8_t* sx = ring + stage * Cfg::kStageBytes;
      mbar_arrive_expect_tx(&full_bar[stage], bytes);
      tma_load_2d(sx, &tmap_x, &full_bar[stage], kb * kBK, static_cast<int>(m_tile));
      tma_load_2d(sx + kABytes, &tmap_w, &full_bar[stage], kb * kBK, nb * BN);
      ++issued;
      if (++stage == Cfg::kStages) stage = 0, phase ^= 1u;
    }
    for (int s = 0; s < Cfg::kStages; ++s)
      if (issued > s) {
        const int fills = (issued - s + Cfg::kStages - 1) / Cfg::kStages;
        drain_wait8(&full_bar[s], static_cast<uint32_t>((fills - 1) & 1), err);
      }
  } else if (warp == 1 && elect_one()) {
    // -------------------------------------------------------------- MMA
    // With a_rows < 128 the rows of the X tile past the box hold whatever was
    // there: they only reach output rows that do not exist.
    constexpr uint32_t kIdesc = make_idesc_f8(kBM, BN);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const uint32_t seq = static_cast<uint32_t>(kb - kb0);
      const int buf = static_cast<int>(seq % Cfg::kBufs);
      if (!mbar_wait(&acc_empty_bar[buf], ((seq / Cfg::kBufs) & 1u) ^ 1u, err, kErrWaitAccEmpty) ||
          !mbar_wait(&full_bar[stage], phase, err, kErrWaitFull))
        break;
      tc_fence_after();
      const uint32_t d = tmem_base + static_cast<uint32_t>(buf * BN);
      const uint32_t sx = smem_addr(ring + stage * Cfg::kStageBytes);
      const uint64_t dx = make_sdesc_kmajor(sx, kBK);
      const uint64_t dw = make_sdesc_kmajor(sx + kABytes, kBK);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        umma_f8(d, dx + 2 * kk, dw + 2 * kk, kIdesc, kk ? 1u : 0u);
      umma_commit(&empty_bar[stage]);
      umma_commit(&acc_full_bar[buf]);
      if (++stage == Cfg::kStages) stage = 0, phase ^= 1u;
    }
    umma_commit(&mma_done_bar);
    drain_wait8(&mma_done_bar, 0, err);
  } else if (warp >= 4) {
    // -------------------------------------------------------------- sums
    const int wg = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int64_t m = m_tile + row;
    const int n_base = nb * BN + wg * Cfg::kWgCols;
    const bool live = m_tile + quarter * 32 < a.M && n_base < a.N;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                               static_cast<uint32_t>(wg * Cfg::kWgCols);
    const float* xs = a.xs + (m < a.M ? m : a.M - 1) * a.ldxs;
    const float* ws = a.ws + static_cast<int64_t>(live ? n_base / kFp8Block : 0) * a.ldws;
    float2 sum[Cfg::kWgCols / 2];
#pragma unroll
    for (int c = 0; c < Cfg::kWgCols / 2; ++c) sum[c] = make_float2(0.f, 0.f);
    float s = __ldg(xs + kb0) * __ldg(ws + kb0);
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const uint32_t seq = static_cast<uint32_t>(kb - kb0);
      const int buf = static_cast<int>(seq % Cfg::kBufs);
      const int next = kb + 1 < kb1 ? kb + 1 : kb;
      const float xs_next = __ldg(xs + next), ws_next = __ldg(ws + next);
      if (!warp_wait8(&acc_full_bar[buf], (seq / Cfg::kBufs) & 1u, err, kErrWaitAccFull, lane)) {
        ok = false;
        break;
      }
      tc_fence_after();
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty_bar[buf]);
      };
      if (live)
        drain_block<Cfg::kWgCols>(lane_base + static_cast<uint32_t>(buf * BN), s, sum, release);
      else
        release();
      s = xs_next * ws_next;
    }
    // The last block's accumulator is complete, so every product has read the
    // ring and every copy into it has landed: its bytes take the partial sums.
    // After an error they may still be in flight; nothing is written then.
    if (ok && live) {
      fence_proxy_async_smem();
#pragma unroll
      for (int c = 0; c < Cfg::kWgCols; c += 4)
        *reinterpret_cast<float4*>(part + row * Cfg::kPitch + wg * Cfg::kWgCols + c) =
            make_float4(sum[c / 2].x, sum[c / 2].y, sum[c / 2 + 1].x, sum[c / 2 + 1].y);
    }
  }
  __syncwarp();
  tc_fence_before();
  if (ksplit > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmem);
  }

  // Every CTA of the cluster finishes a share of the tile's rows, adding the
  // partial sums in split order; four columns a thread.
  const int rows = static_cast<int>(a.M - m_tile < kBM ? a.M - m_tile : kBM);
  const uint32_t part_addr = smem_addr(part);
  constexpr int kQuads = BN / 4;
  for (int i = split * kThreads + static_cast<int>(threadIdx.x); i < rows * kQuads;
       i += ksplit * kThreads) {
    const int r = i / kQuads;
    const int c = 4 * (i - r * kQuads);
    const int n = nb * BN + c;
    if (n >= a.N) continue;
    const uint32_t at = part_addr + static_cast<uint32_t>((r * Cfg::kPitch + c) * 4);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < ksplit; ++p) {
      const float4 t = ksplit > 1 ? ld_shared_cluster_f4(mapa_shared(at, static_cast<uint32_t>(p)))
                                  : *reinterpret_cast<const float4*>(part + r * Cfg::kPitch + c);
      v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
    }
    const int64_t m = m_tile + r;
    const T* res = static_cast<const T*>(a.residual);
    T* out = static_cast<T*>(a.out) + m * a.ldo + n;
    if (a.vec) {  // N % 4 == 0: the four columns exist
      if (a.bias != nullptr) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(a.bias + n));
        v[0] += b.x, v[1] += b.y, v[2] += b.z, v[3] += b.w;
      }
      if (a.gelu) {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const float2 g = gelu_erf2(make_float2(v[j], v[j + 1]));
          v[j] = g.x, v[j + 1] = g.y;
        }
      }
      if (res != nullptr) {
        float rv[4];
        load4(res + m * a.ldr + n, rv);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = rv[j] + v[j];
      }
      store4(out, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (n + j >= a.N) break;
        float y = v[j];
        if (a.bias != nullptr) y += __ldg(a.bias + n + j);
        if (a.gelu) y = gelu_erf2(make_float2(y, 0.f)).x;
        if (res != nullptr) y = to_f32(res[m * a.ldr + n + j]) + y;
        out[j] = from_f32<T>(y);
      }
    }
  }
  if (ksplit > 1) cluster_sync_all();  // no CTA exits while its sums may be read
}

// ---------------------------------------------------------------- host side
namespace {

template <typename F>
int with_out_type(int type, F&& f) {
  switch (type) {
    case VITB200_F32: return f(float{});
    case VITB200_F16: return f(__half{});
    case VITB200_BF16: return f(__nv_bfloat16{});
    default: return VITB200_E_INVALID_ARG;
  }
}

int codes_map(CUtensorMap* map, const uint8_t* q, int64_t rows, int K, int64_t ld, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld)};
  const uint32_t box[2] = {kBK, static_cast<uint32_t>(box_rows)};
  return encode_tmap_typed(map, 2, q, dims, strides, box, 1, 2);
}

bool aligned(const void* p, int64_t ld_bytes, int to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && ld_bytes % to == 0;
}

template <typename T>
int launch_pair(const Fp8GemmProblem& p, Fp8GemmArgs& a, cudaStream_t s) {
  CUtensorMap tx, tw, to, tr;
  if (int st = codes_map(&tx, p.x, p.M, p.K, p.ldx, kBM)) return st;
  if (int st = codes_map(&tw, p.w, p.N, p.K, p.ldw, kPairBRows)) return st;
  a.num_n_tiles = (p.N + kPairBN - 1) / kPairBN;
  a.num_tiles = static_cast<int>((p.M + 2 * kBM - 1) / (2 * kBM)) * a.num_n_tiles;
  // 32 x 32 slabs through tensor maps where rows are 16-byte aligned.
  auto slab_map = [&](CUtensorMap* map, const void* base, int64_t ld) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)};
    const uint64_t strides[1] = {static_cast<uint64_t>(ld) * sizeof(T)};
    const uint32_t box[2] = {kSlabCols<T>, 32};
    return encode_tmap_typed(map, 2, base, dims, strides, box, 1, sizeof(T) == 2);
  };
  to = tr = tx;
  a.tma_out = aligned(p.out, p.ldo * sizeof(T), 16);
  a.tma_res = p.residual != nullptr && aligned(p.residual, p.ldr * sizeof(T), 16);
  if (a.tma_out)
    if (int st = slab_map(&to, p.out, p.ldo)) return st;
  if (a.tma_res)
    if (int st = slab_map(&tr, p.residual, p.ldr)) return st;
  const int pairs = std::min(a.num_tiles, device_num_sms() / 2);
  return launch_kernel(gemm_fp8_pair_kernel<T>, dim3(2 * static_cast<unsigned>(pairs)),
                       dim3(kThreads), kPairSmem, s, 2, tx, tw, to, tr, a);
}

template <typename T, int BN>
int launch_tile(const Fp8GemmProblem& p, Fp8GemmArgs& a, int ksplit, cudaStream_t s) {
  CUtensorMap tx, tw;
  a.a_rows = static_cast<int>(std::min<int64_t>(kBM, (p.M + 7) / 8 * 8));
  if (int st = codes_map(&tx, p.x, p.M, p.K, p.ldx, a.a_rows)) return st;
  if (int st = codes_map(&tw, p.w, p.N, p.K, p.ldw, BN)) return st;
  a.num_n_tiles = (p.N + BN - 1) / BN;
  a.num_tiles = static_cast<int>((p.M + kBM - 1) / kBM) * a.num_n_tiles;
  a.ksplit = ksplit;
  a.vec = p.N % 4 == 0 && aligned(p.out, p.ldo * sizeof(T), 4 * sizeof(T)) &&
          (p.residual == nullptr || aligned(p.residual, p.ldr * sizeof(T), 4 * sizeof(T))) &&
          (p.bias == nullptr || aligned(p.bias, 0, 16));
  return launch_kernel(gemm_fp8_tile_kernel<T, BN>,
                       dim3(static_cast<unsigned>(a.num_tiles) * static_cast<unsigned>(ksplit)),
                       dim3(kThreads), TileCfg<BN>::kSmem, s, static_cast<unsigned>(ksplit), tx, tw,
                       a);
}

template <typename Kernel>
int allow_smem(Kernel kernel, int bytes) {
  return cuda_status(
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

constexpr int kMaxSplit = 8;  // portable cluster size

// The K split that makes a launch of the tile kernel shortest: 0.27 us a K block
// with 64 columns and 0.34 with 128, and for joining a cluster's sums 0.8 us, 0.1 a
// CTA and up to 1.5 for a full tile's rows (fitted to splits 1..8 of eight shapes; 8
// x 4096 x 4096 takes 12.1, 8.5 us with 64 columns split 1, 2 ways and 8.9, 7.0 with
// 128 split 2, 4 ways; 577 x 1024 x 1024 5.9 and 10.5, 7.0 and 11.1). Only splits whose clusters
// all fit the GPU at once: the others run a second wave (64 x 4096 x 1024, 64
// columns, 16 clusters of 8: 10.7 us, of 4: 6.1).
struct TilePlan {
  int ksplit;
  double us;
};
template <typename T, int BN>
TilePlan plan_tile(int64_t tiles, int num_kb, int64_t M) {
  const int sms = device_num_sms();
  const double block_us = BN == 64 ? 0.27 : 0.34;
  TilePlan best = {1, static_cast<double>((tiles + sms - 1) / sms) * num_kb * block_us};
  for (int d = 2; d <= std::min(kMaxSplit, num_kb) && tiles * d <= sms; ++d) {
    const double us = (num_kb + d - 1) / d * block_us + 0.8 + 0.1 * d +
                      1.5 * static_cast<double>(std::min<int64_t>(M, kBM)) / kBM;
    if (us < best.us && cluster_slots(gemm_fp8_tile_kernel<T, BN>, TileCfg<BN>::kSmem, kThreads,
                                      d) >= tiles)
      best = {d, us};
  }
  return best;
}

}  // namespace

int gemm_fp8_prepare_device() {
  auto one = [](auto tag) {
    using T = decltype(tag);
    if (int st = allow_smem(gemm_fp8_pair_kernel<T>, kPairSmem)) return st;
    if (int st = allow_smem(gemm_fp8_tile_kernel<T, 64>, TileCfg<64>::kSmem)) return st;
    return allow_smem(gemm_fp8_tile_kernel<T, 128>, TileCfg<128>::kSmem);
  };
  if (int st = one(float{})) return st;
  if (int st = one(__half{})) return st;
  return one(__nv_bfloat16{});
}

int gemm_fp8_launch(const Fp8GemmProblem& p, cudaStream_t s) {
  Fp8GemmArgs a = {};
  a.M = p.M;
  a.N = p.N;
  a.num_kb = (p.K + kFp8Block - 1) / kFp8Block;
  a.xs = p.xs;
  a.ldxs = p.ldxs;
  a.ws = p.ws;
  a.ldws = p.ldws;
  a.bias = p.bias;
  a.residual = p.residual;
  a.ldr = p.ldr;
  a.out = p.out;
  a.ldo = p.ldo;
  a.gelu = p.gelu;
  a.vec_xs = aligned(p.xs, p.ldxs * 4, 16);
  a.err = device_error_word();
  const int64_t pair_tiles = (p.M + 2 * kBM - 1) / (2 * kBM) * ((p.N + kPairBN - 1) / kPairBN);
  const int64_t m_tiles = (p.M + kBM - 1) / kBM;
  const int64_t tiles64 = m_tiles * ((p.N + 63) / 64), tiles128 = m_tiles * ((p.N + 127) / 128);
  if (std::max(pair_tiles, tiles64) > INT32_MAX / kMaxSplit) return VITB200_E_UNSUPPORTED;
  return with_out_type(p.out_type, [&](auto tag) {
    using T = decltype(tag);
    // One wave of 128 x 128 tiles, else pairs (tile and pair form: 117 tiles, 1664 x 1024 x
    // 1152, 7.8 and 10.6 us; 144, 1152 x 4096 x 2048, 17.4 and 24.6; 160, 2500 x 4096 x 1024,
    // 32.7 and 22.3; 395 of 50432 x 768 x 96 21.7 and 16.3).
    if (tiles128 > device_num_sms()) return launch_pair<T>(p, a, s);
    const TilePlan narrow = plan_tile<T, 64>(tiles64, a.num_kb, p.M);
    const TilePlan wide = plan_tile<T, 128>(tiles128, a.num_kb, p.M);
    return narrow.us <= wide.us ? launch_tile<T, 64>(p, a, narrow.ksplit, s)
                                : launch_tile<T, 128>(p, a, wide.ksplit, s);
  });
}

}  // namespace vitb200

using namespace vitb200;

extern "C" int vitb200_gemm_fp8(const uint8_t* X, int64_t ldx, const float* x_scales, int64_t ldxs,
                                const uint8_t* W, int64_t ldw, const float* w_scales, int64_t ldws,
                                const float* bias, const void* residual, int64_t ldr, void* out,
                                int64_t ldo, int out_type, int64_t M, int K, int N, int gelu,
                                void* stream) {
  try {
    if (M < 0 || M > INT32_MAX - 256 || N < 0 || N > INT32_MAX - 256 || K < 1 ||
        K > INT32_MAX - 256 || out_type < VITB200_F32 || out_type > VITB200_BF16)
      return VITB200_E_INVALID_ARG;
    const int64_t kb = (static_cast<int64_t>(K) + kFp8Block - 1) / kFp8Block;
    if (ldx < K || ldw < K || ldxs < kb || ldws < kb || ldo < N || (residual && ldr < N))
      return VITB200_E_INVALID_ARG;
    if (M == 0 || N == 0) return 0;
    if (!X || !W || !x_scales || !w_scales || !out) return VITB200_E_INVALID_ARG;
    const int es = out_type == VITB200_F32 ? 4 : 2;
    if (!aligned(X, ldx, 16) || !aligned(W, ldw, 16) || !aligned(x_scales, 0, 4) ||
        !aligned(w_scales, 0, 4) || !aligned(bias, 0, 4) || !aligned(out, 0, es) ||
        !aligned(residual, 0, es))
      return VITB200_E_ALIGNMENT;
    if (int st = vitb200_init()) return st;
    Fp8GemmProblem p = {};
    p.x = X;
    p.w = W;
    p.xs = x_scales;
    p.ws = w_scales;
    p.bias = bias;
    p.residual = residual;
    p.out = out;
    p.M = M;
    p.ldx = ldx;
    p.ldw = ldw;
    p.ldxs = ldxs;
    p.ldws = ldws;
    p.ldr = ldr;
    p.ldo = ldo;
    p.N = N;
    p.K = K;
    p.gelu = gelu != 0;
    p.out_type = out_type;
    return gemm_fp8_launch(p, static_cast<cudaStream_t>(stream));
  } catch (...) {
    return VITB200_E_INVALID_ARG;
  }
}
