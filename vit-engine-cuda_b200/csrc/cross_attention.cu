// Attention of queries to an encoder's states of another length:
//
//   o[b][t][h] = softmax_s(q[b][t][h] . k[b][s][h / G] * scale) v[b][s][h / G]
//
// over keys s < len[b], bf16 or fp16, head size D = 64 or 128, G = heads /
// kv_heads query heads to a key head. No key: o = 0.
//
// The rows a key head serves (G heads x Tq queries) are packed into tiles of up
// to 128 rows, so a group of heads reads its keys once. A CTA runs two streams,
// each with a softmax warpgroup (one row a thread), a score accumulator S and an
// output accumulator O in TMEM:
//  * two row tiles: both streams go over all key tiles and share the K and V
//    copies;
//  * one row tile: the streams take the even and the odd key tiles and their
//    results are joined at the end.
// Either way unit u = (stream u % 2, key tile) runs S = Q K^T, softmax, O += P V,
// and while one stream's softmax runs the tensor core works for the other. P
// overwrites S in TMEM as 16-bit pairs and is the A operand from there; V is the
// N-major B operand as it lies in memory, no transposition.
//
// O stays in TMEM over all key tiles. With m the maximum that a row's
// exponentials refer to, a new maximum within 2^8 of it leaves m as it is (P then
// reaches at most 256, sums in fp32); only a larger one rescales O and the sum,
// which after the first tiles is rare. The quotient o = O / l is the same.
//
// A launch with too few rows to fill the GPU shares the key tiles out over a
// cluster of CTAs, joined in a fixed order through distributed shared memory: no
// workspace, results independent of timing.
// Every wait is bounded (device error word).
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cross_attention.cuh"
#include "engine.h"

namespace vitb200 {

namespace {

constexpr int kRows = 128;       // rows of a tile
constexpr int kKeys = 128;       // keys of a tile
constexpr int kThreads = 384;    // control warpgroup + two softmax warpgroups
constexpr int kHalf = 64;                        // columns of one 128-byte swizzle span
constexpr int kHalfBytes = kRows * kHalf * 2;    // 128 rows x 64 columns
constexpr float kRescale = 8.f;                  // log2 of the largest P

template <int D>
struct Cfg {
  static constexpr int kHalves = D / kHalf;
  static constexpr int kTile = kHalves * kHalfBytes;  // a Q, K or V tile
  static constexpr int kKSlots = D == 64 ? 4 : 2;
  static constexpr int kVSlots = D == 64 ? 4 : 3;
  static constexpr int kSmem = (2 + kKSlots + kVSlots) * kTile + 1024;
  // 384 threads launched at 168 registers (build.py checks that ptxas allocated
  // 168), shared out between control and softmax warpgroups. D = 128 waits on the
  // issuing thread, which spills below 104 (575 us against 558 in the long run at 4 x 16
  // heads x 4096 x 4500); D = 64 takes either (427-433 at 4 x 16 x 4096 x 4096).
  static constexpr uint32_t kCtrlRegs = D == 64 ? 56 : 104;
  static constexpr uint32_t kSoftRegs = D == 64 ? 224 : 200;
  static_assert(128 * kCtrlRegs + 256 * kSoftRegs == kThreads * 168, "register split");
  // Partial results of both streams, joined at the end: [2][128][D + 4] floats
  // (the pad keeps a thread-per-row store free of bank conflicts), then m and l.
  static constexpr int kPitch = D + 4;
  static constexpr int kStatsAt = 2 * kRows * kPitch;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  static_assert((kStatsAt + 4 * kRows) * 4 <= kSmem - 1024, "partial results fit");
};

struct CrossArgs {
  int Tq, Tk;
  int kv_heads;    // key heads as the row tiles see them
  int group;       // query heads packed into a row tile
  int tile_t;      // queries per row tile (G * tile_t <= 128 rows)
  int nq;          // row tiles per (image, key head)
  int nsplit;      // CTAs per work item
  int kv_div;      // packed key heads per key head (1 where groups are packed)
  float c;         // scale * log2(e)
  const int* lens; // [B] or null
  uint16_t* o;     // [B][Tq][heads * D]
  int64_t o_row;   // heads * D
  int* err;
};

// S and P V instruction descriptors: fp32 accumulator, A and B f16 (0) or bf16
// (1); V is N-major (bit 16).
template <typename T>
constexpr uint32_t idesc(int N, bool b_n_major) {
  const uint32_t f = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return make_idesc_f16(kRows, N) | (f << 7) | (f << 10) | (b_n_major ? 1u << 16 : 0u);
}

// N-major tile of [keys][64 columns] rows of 128 bytes under the 128-byte
// swizzle: 8-key atoms 1024 bytes apart, the next 64 columns `halves` bytes on.
__device__ __forceinline__ uint64_t sdesc_nmajor(uint32_t saddr, uint32_t half_bytes) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(half_bytes >> 4) << 16) |
         (uint64_t(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ bool warp_wait_x(uint64_t* bar, uint32_t parity, int* err, int code,
                                            int lane) {
  int ok = 1;
  if (lane == 0) ok = mbar_wait(bar, parity, err, code) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

__device__ __forceinline__ void drain_wait_x(uint64_t* bar, uint32_t parity, int* err) {
  const uint32_t addr = smem_addr(bar);
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(addr, parity)) {
    if (globaltimer_ns() - t0 > kWaitTimeoutNs) {
      report_error(err, kErrDrain);
      return;
    }
  }
}

// A work item: a key head of an image and one or two of its row tiles.
struct Item {
  int b, hk, tile0, tiles;
};
__device__ __forceinline__ Item item_at(const CrossArgs& a, int i) {
  const int groups = (a.nq + 1) / 2;
  Item it;
  const int bh = i / groups;
  it.b = bh / a.kv_heads;
  it.hk = bh - it.b * a.kv_heads;
  it.tile0 = 2 * (i - bh * groups);
  it.tiles = min(2, a.nq - it.tile0);
  return it;
}

// Output row of packed row r of tile `tile`, or -1 past the last query.
__device__ __forceinline__ int64_t out_row(const CrossArgs& a, const Item& it, int tile, int r,
                                           int D) {
  const int tl = r / a.group;
  const int t = tile * a.tile_t + tl;
  if (tl >= a.tile_t || t >= a.Tq) return -1;
  return (static_cast<int64_t>(it.b) * a.Tq + t) * a.o_row +
         (static_cast<int64_t>(it.hk) * a.group + (r - tl * a.group)) * D;
}

}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    cross_attention_kernel(const __grid_constant__ CUtensorMap tmap_q,
                           const __grid_constant__ CUtensorMap tmap_k,
                           const __grid_constant__ CUtensorMap tmap_v, const CrossArgs a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full;
  __shared__ __align__(8) uint64_t k_full[C::kKSlots], k_empty[C::kKSlots];
  __shared__ __align__(8) uint64_t v_full[C::kVSlots], v_empty[C::kVSlots];
  __shared__ __align__(8) uint64_t s_full[2], p_half[2], p_full[2], pv_done[2];
  __shared__ __align__(8) uint64_t tail_go, tail_bar;
  __shared__ __align__(8) uint64_t mma_done;
  __shared__ uint32_t tmem_slot;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int* err = a.err;
  const uint32_t raw = smem_addr(smem_raw);
  uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* sq = base;
  uint8_t* sk = base + 2 * C::kTile;
  uint8_t* sv = sk + C::kKSlots * C::kTile;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int i = 0; i < C::kKSlots; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < C::kVSlots; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_half[i], 4);  // one arrival per warp of the stream's warpgroup
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(&tail_go, 1);
    mbar_init(&tail_bar, 1);
    mbar_init(&mma_done, 1);
    fence_barrier_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int split = static_cast<int>(blockIdx.x) % a.nsplit;  // = rank in the cluster
  const Item it = item_at(a, static_cast<int>(blockIdx.x) / a.nsplit);
  int len = a.Tk;
  if (a.lens != nullptr) len = max(0, min(a.Tk, __ldg(a.lens + it.b)));
  // This CTA's key tiles [j0, j0 + nk) of the image's `all`.
  const int all = (len + kKeys - 1) / kKeys;
  const int j0 = static_cast<int>(static_cast<int64_t>(all) * split / a.nsplit);
  const int nk = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.nsplit) - j0;
  const bool shared_keys = it.tiles == 2;  // two row tiles: every key tile is two units
  const int units = shared_keys ? 2 * nk : nk;
  // V's rows past the last key, inside its tile, may hold anything: P is zero
  // there, but zero times NaN is not. (Rows past Tk arrive as zeros.)
  const int tail_keys = len - (all - 1) * kKeys;
  const bool fix_tail = nk > 0 && j0 + nk == all && len < a.Tk && tail_keys < kKeys;

  if (warp < 4) {
    setmaxnreg_dec<C::kCtrlRegs>();
    if (warp == 0 && nk > 0 && elect_one()) {
      // -------------------------------------------------------------- TMA
      mbar_arrive_expect_tx(&q_full, static_cast<uint32_t>(it.tiles * C::kHalves * a.group *
                                                           a.tile_t * kHalf * 2));
      for (int i = 0; i < it.tiles; ++i)
        for (int h = 0; h < C::kHalves; ++h)
          tma_load_5d(sq + i * C::kTile + h * kHalfBytes, &tmap_q, &q_full, h * kHalf, 0,
                      (it.tile0 + i) * a.tile_t, it.hk, it.b);
      int k_issued = 0, v_issued = 0;
      auto load = [&](uint8_t* ring, int slots, uint64_t* full, uint64_t* empty,
                      const CUtensorMap* map, int j, int& issued) -> bool {
        const int s = j % slots;
        if (!mbar_wait(&empty[s], ((j / slots) & 1) ^ 1u, err, kErrWaitEmpty)) return false;
        mbar_arrive_expect_tx(&full[s], C::kTile);
        for (int h = 0; h < C::kHalves; ++h)
          tma_load_4d(ring + s * C::kTile + h * kHalfBytes, map, &full[s], h * kHalf,
                      (j0 + j) * kKeys, it.hk / a.kv_div, it.b);
        ++issued;
        return true;
      };
      // Order of use: K runs one tile ahead of V.
      bool ok = load(sk, C::kKSlots, k_full, k_empty, &tmap_k, 0, k_issued);
      for (int j = 0; j < nk && ok; ++j) {
        if (j + 1 < nk) ok = load(sk, C::kKSlots, k_full, k_empty, &tmap_k, j + 1, k_issued);
        if (ok) ok = load(sv, C::kVSlots, v_full, v_empty, &tmap_v, j, v_issued);
      }
      if (fix_tail) mbar_arrive(&tail_go);
      // Every copy issued lands before the CTA can exit.
      drain_wait_x(&q_full, 0, err);
      for (int s = 0; s < C::kKSlots; ++s)
        if (k_issued > s)
          drain_wait_x(&k_full[s], ((k_issued - 1 - s) / C::kKSlots) & 1, err);
      for (int s = 0; s < C::kVSlots; ++s)
        if (v_issued > s)
          drain_wait_x(&v_full[s], ((v_issued - 1 - s) / C::kVSlots) & 1, err);
    } else if (warp == 1 && nk > 0 && elect_one()) {
      // -------------------------------------------------------------- MMA
      // One thread issues everything, and its own instructions between products of
      // 64 cycles show: loops are unrolled, ring positions are counters, and a tile's
      // barriers are waited on once. SHARED: two units (streams) per key tile.
      constexpr uint32_t kIdescS = idesc<T>(kKeys, false);
      constexpr uint32_t kIdescPV = idesc<T>(D, true);
      const uint64_t dq0 = make_sdesc_kmajor(smem_addr(sq), 128);
      const uint64_t dk0 = make_sdesc_kmajor(smem_addr(sk), 128);
      const uint64_t dv0 = sdesc_nmajor(smem_addr(sv), kHalfBytes);
      constexpr uint64_t kTileStep = C::kTile >> 4, kHalfStep = kHalfBytes >> 4;
      auto run = [&](auto shared) {
        constexpr bool SHARED = decltype(shared)::value;
        int ks = 0, vs = 0;           // ring positions
        uint32_t kph = 0, vph = 0;    // and their phases
        auto issue_s = [&](int i) -> bool {
          if ((!SHARED || i == 0) && !mbar_wait(&k_full[ks], kph, err, kErrWaitFull)) return false;
          tc_fence_after();
          const uint64_t dq = dq0 + (SHARED && i ? kTileStep : 0);
          const uint64_t dk = dk0 + static_cast<uint32_t>(ks) * kTileStep;
          const uint32_t d = tmem + i * kKeys;
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 16 columns = 32 bytes = +2
              umma_f16(d, dq + h * kHalfStep + 2 * kk, dk + h * kHalfStep + 2 * kk, kIdescS,
                       h + kk ? 1u : 0u);
          umma_commit(&s_full[i]);
          if (!SHARED || i == 1) {  // the tile's last use
            umma_commit(&k_empty[ks]);
            if (++ks == C::kKSlots) ks = 0, kph ^= 1u;
          }
          return true;
        };
        auto issue_pv = [&](int i, int n, bool last) -> bool {
          if (!SHARED || i == 0) {
            if (!mbar_wait(&v_full[vs], vph, err, kErrWaitFull)) return false;
            if (last && fix_tail && !mbar_wait(&tail_bar, 0, err, kErrWaitFull)) return false;
          }
          const uint64_t dv = dv0 + static_cast<uint32_t>(vs) * kTileStep;
          const uint32_t d = tmem + 2 * kKeys + i * D;
          const uint32_t p = tmem + i * kKeys;
          // The first half of the keys while the exponentials of the second run; 16
          // keys a product: 2048 bytes of V, 8 columns of P.
          if (!mbar_wait(&p_half[i], n & 1, err, kErrWaitAccFull)) return false;
          tc_fence_after();
          const int steps = last ? (tail_keys + 15) / 16 : kKeys / 16;
          if (steps == 8) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f16_tmem_a(d, p + 8 * kk, dv + 128 * kk, kIdescPV, kk ? 1u : (n ? 1u : 0u));
            if (!mbar_wait(&p_full[i], n & 1, err, kErrWaitAccFull)) return false;
            tc_fence_after();
#pragma unroll
            for (int kk = 4; kk < 8; ++kk)
              umma_f16_tmem_a(d, p + 8 * kk, dv + 128 * kk, kIdescPV, 1u);
          } else {
            for (int kk = 0; kk < min(4, steps); ++kk)
              umma_f16_tmem_a(d, p + 8 * kk, dv + 128 * kk, kIdescPV, n || kk ? 1u : 0u);
            if (!mbar_wait(&p_full[i], n & 1, err, kErrWaitAccFull)) return false;
            tc_fence_after();
            for (int kk = 4; kk < steps; ++kk)
              umma_f16_tmem_a(d, p + 8 * kk, dv + 128 * kk, kIdescPV, 1u);
          }
          umma_commit(&pv_done[i]);
          if (!SHARED || i == 1) {
            umma_commit(&v_empty[vs]);
            if (++vs == C::kVSlots) vs = 0, vph ^= 1u;
          }
          return true;
        };
        bool ok = mbar_wait(&q_full, 0, err, kErrWaitFull);
        // S(u + 2) overwrites P(u): it is issued after the product that reads P(u),
        // and one thread's products run in order.
        if (ok) ok = issue_s(0);
        if (ok && units > 1) ok = issue_s(1);
        for (int u = 0; u < units && ok; u += 2) {
          const int n = u >> 1;
          const int j = j0 + (SHARED ? n : u);  // key tile of unit u
          ok = issue_pv(0, n, j == all - 1);
          if (ok && u + 2 < units) ok = issue_s(0);
          if (!ok || u + 1 >= units) break;
          ok = issue_pv(1, n, (SHARED ? j : j + 1) == all - 1);
          if (ok && u + 3 < units) ok = issue_s(1);
        }
      };
      if (shared_keys)
        run(std::true_type{});
      else
        run(std::false_type{});
      umma_commit(&mma_done);
      drain_wait_x(&mma_done, 0, err);
    } else if (warp == 2 && fix_tail) {
      // ------------------------------------------------------------- tail
      // Not before the copy is issued: until then the slot's barrier may be a
      // whole turn of the ring behind, and its parity would say nothing.
      const int j = nk - 1, s = j % C::kVSlots;
      if (warp_wait_x(&tail_go, 0, err, kErrWaitFull, lane) &&
          warp_wait_x(&v_full[s], (j / C::kVSlots) & 1, err, kErrWaitFull, lane)) {
        uint4* v = reinterpret_cast<uint4*>(sv + s * C::kTile);
        constexpr int kRow16 = 8;  // 16-byte chunks of a 128-byte row
        for (int h = 0; h < C::kHalves; ++h)
          for (int c = tail_keys * kRow16 + lane; c < kKeys * kRow16; c += 32)
            v[h * (kHalfBytes / 16) + c] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail_bar);
      }
    }
    __syncwarp();
  }

  // Softmax state of this thread's row, kept past the role split.
  const bool joined = a.nsplit > 1 || !shared_keys;  // rows have several partial results
  if (warp >= 4) {
    setmaxnreg_inc<C::kSoftRegs>();
    // ---------------------------------------------------------------- softmax
    const int i = (warp - 4) >> 2;  // stream
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_col = lanes + i * kKeys;
    const uint32_t o_col = lanes + 2 * kKeys + i * D;
    const int mine = (units + 1 - i) / 2;  // units of this stream
    const float c = a.c;
    float m = -INFINITY, l = 0.f;
    // Past this, m is huge (cross_attention.cuh), and the warp takes the way through the
    // rescaling for every tile. (Rows past the packed ones hold whatever was in shared
    // memory.) Having that way costs D = 64 3 % (411 to 422 us at 4 x 16 x 4096 x 4096),
    // D = 128 nothing; subtracting the largest score first, for every row, 9 and 8 %.
    const float huge = r < a.group * a.tile_t ? kHugeScore : INFINITY;
    bool ok = true;
    for (int n = 0; n < mine; ++n) {
      const int j = j0 + (shared_keys ? n : 2 * n + i);
      // Every lane waits: that is quicker than one lane and a broadcast. S(n) was
      // issued after the stream's product n - 1, so that one is in O as well.
      ok = mbar_wait(&s_full[i], n & 1, err, kErrWaitAccFull) &&
           (n == 0 || mbar_wait(&pv_done[i], (n - 1) & 1, err, kErrWaitAccFull));
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float s[kKeys];
#pragma unroll
      for (int h = 0; h < 4; ++h) tmem_ld_issue_x32(s_col + 32 * h, s + 32 * h);
      tmem_ld_wait_x32(s);
#pragma unroll
      for (int h = 1; h < 4; ++h) tmem_ld_landed_x32(s + 32 * h);
      const int valid = len - j * kKeys;
      if (valid < kKeys) {
        const float out = c < 0.f ? INFINITY : -INFINITY;
#pragma unroll
        for (int x = 0; x < kKeys; ++x)
          if (x >= valid) s[x] = out;
      }
      // The largest s * c (the smallest s where c is negative).
      float e0 = s[0], e1 = s[1], e2 = s[2], e3 = s[3];
      if (c >= 0.f) {
#pragma unroll
        for (int x = 4; x + 8 <= kKeys; x += 8) {
          e0 = max3(e0, s[x], s[x + 4]), e1 = max3(e1, s[x + 1], s[x + 5]);
          e2 = max3(e2, s[x + 2], s[x + 6]), e3 = max3(e3, s[x + 3], s[x + 7]);
        }
        e0 = max3(e0, s[kKeys - 4], s[kKeys - 3]);
        e1 = max3(e1, s[kKeys - 2], s[kKeys - 1]);
        e0 = fmaxf(max3(e0, e1, e2), e3);
      } else {
#pragma unroll
        for (int x = 4; x + 8 <= kKeys; x += 8) {
          e0 = min3(e0, s[x], s[x + 4]), e1 = min3(e1, s[x + 1], s[x + 5]);
          e2 = min3(e2, s[x + 2], s[x + 6]), e3 = min3(e3, s[x + 3], s[x + 7]);
        }
        e0 = min3(e0, s[kKeys - 4], s[kKeys - 3]);
        e1 = min3(e1, s[kKeys - 2], s[kKeys - 1]);
        e0 = fminf(min3(e0, e1, e2), e3);
      }
      const float top = e0 * c;
      // (P may pass the largest seen by 2^kRescale: that much less lift for fp16.)
      constexpr float kUp = kLift<T> > kRescale ? kLift<T> - kRescale : 0.f;
      if (n == 0) m = top;
      if (__any_sync(0xffffffffu, top - m > kRescale || fabsf(m) > huge)) {
        float f = 1.f;
        if (top - m > kRescale) {
          f = ex2_approx(m - top);
          m = top;
        }
        l *= f;
#pragma unroll 1
        for (int h = 0; h < D && n > 0; h += 32) {
          float t[32];
          tmem_ld_32x32b_x32(o_col + h, t);
#pragma unroll
          for (int x = 0; x < 32; ++x) t[x] *= f;
          tmem_st_32x32b_x32(o_col + h, t);
        }
        tmem_wait_st();
        if (__any_sync(0xffffffffu, fabsf(m) > huge)) {
          // The scores again, 32 at a time. Half h of P takes columns read by then.
          const float ref = m == -INFINITY ? 0.f : m;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            float p[32];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float t[32];
              __syncwarp();
              tmem_ld_32x32b_x32(s_col + 64 * h + 32 * q, t);
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                const float u = fabsf(m) > huge ? huge_exponent(t[x], c, ref, kUp)
                                                : fmaf(t[x], c, kUp > 0.f ? kUp - ref : -ref);
                t[x] = 64 * h + 32 * q + x < valid ? ex2_approx(u) : 0.f;
              }
#pragma unroll
              for (int x = 0; x < 32; x += 2) {
                sum = add2(sum, make_float2(t[x], t[x + 1]));
                p[16 * q + x / 2] = __uint_as_float(pack2<T>(t[x], t[x + 1]));
              }
            }
            tmem_st_32x32b_x32(s_col + 32 * h, p);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(h == 0 ? &p_half[i] : &p_full[i]);
          }
          l += sum.x + sum.y;
          continue;
        }
      }
      // All scores -inf so far: 2^(-inf - 0) = 0, not NaN.
      const float ref = m == -INFINITY ? 0.f : m;
      const float2 c2 = splat2(c), r2 = splat2(kUp > 0.f ? kUp - ref : -ref);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float p[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          const float2 t = fma2(make_float2(s[64 * h + 2 * x], s[64 * h + 2 * x + 1]), c2, r2);
          const float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
          sum = add2(sum, e);
          p[x] = __uint_as_float(pack2<T>(e.x, e.y));
        }
        tmem_st_32x32b_x32(s_col + 32 * h, p);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(h == 0 ? &p_half[i] : &p_full[i]);
      }
      l += sum.x + sum.y;
    }
    if (ok && mine > 0)
      ok = warp_wait_x(&pv_done[i], (mine - 1) & 1, err, kErrWaitAccFull, lane);
    tc_fence_after();
    if (ok && !joined) {
      // Two row tiles, all keys here: this thread's row is complete.
      const int64_t row = out_row(a, it, it.tile0 + i, r, D);
      const float inv = 1.f / l;
#pragma unroll 1
      for (int h = 0; h < D; h += 32) {
        float t[32];
        if (len > 0) {
          __syncwarp();
          tmem_ld_32x32b_x32(o_col + h, t);
        }
        if (row >= 0) {
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (len > 0)
              w = make_uint4(pack2<T>(t[x] * inv, t[x + 1] * inv),
                             pack2<T>(t[x + 2] * inv, t[x + 3] * inv),
                             pack2<T>(t[x + 4] * inv, t[x + 5] * inv),
                             pack2<T>(t[x + 6] * inv, t[x + 7] * inv));
            *reinterpret_cast<uint4*>(a.o + row + h + x) = w;
          }
        }
      }
    } else if (ok) {
      // Leave the partial result in shared memory: this stream's products have
      // read the tiles there, the other's may not have, so wait for it too. A
      // stream without units leaves an empty result.
      const int theirs = (units + i) / 2;
      if (theirs > 0)
        ok = warp_wait_x(&pv_done[1 - i], (theirs - 1) & 1, err, kErrWaitAccFull, lane);
      if (ok) {
        fence_proxy_async_smem();
        float* part = reinterpret_cast<float*>(base);
        float* mine_at = part + (i * kRows + r) * C::kPitch;
#pragma unroll 1
        for (int h = 0; h < D; h += 32) {
          float t[32];
          if (mine > 0) {
            __syncwarp();
            tmem_ld_32x32b_x32(o_col + h, t);
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) t[x] = 0.f;
          }
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            *reinterpret_cast<float4*>(mine_at + h + x) =
                make_float4(t[x], t[x + 1], t[x + 2], t[x + 3]);
        }
        part[C::kStatsAt + i * kRows + r] = m;
        part[C::kStatsAt + 2 * kRows + i * kRows + r] = l;
      }
    }
  }

  tc_fence_before();
  if (a.nsplit > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (!joined) return;

  // Join the partial results (the softmax warps: the control warps gave their
  // registers up), eight columns a thread, the rows shared out over
  // the cluster: o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p. Row tile i of
  // two has one result per CTA (stream i); a single row tile has two.
  const int streams = shared_keys ? 1 : 2;
  constexpr int kChunks = D / 8;
  const uint32_t part = smem_addr(base);
  constexpr int kJoiners = kThreads - 128;
  for (int x = split * kJoiners + static_cast<int>(threadIdx.x) - 128;
       warp >= 4 && x < it.tiles * kRows * kChunks; x += a.nsplit * kJoiners) {
    const int col = 8 * (x % kChunks);
    const int tr = x / kChunks;
    const int tile = tr / kRows, r = tr - tile * kRows;
    const int64_t row = out_row(a, it, it.tile0 + tile, r, D);
    if (row < 0) continue;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (len > 0) {
      auto peer = [&](int p, int at) {  // float `at` of partial result p's CTA
        const uint32_t addr = part + static_cast<uint32_t>(at) * 4u;
        return a.nsplit > 1 ? mapa_shared(addr, static_cast<uint32_t>(p / streams)) : addr;
      };
      auto slot = [&](int p) { return (shared_keys ? tile : p % streams) * kRows + r; };
      const int parts = a.nsplit * streams;
      float M = -INFINITY;
      for (int p = 0; p < parts; ++p)
        M = fmaxf(M, ld_partial(peer(p, C::kStatsAt + slot(p)), a.nsplit > 1));
      if (M == -INFINITY) M = 0.f;
      float L = 0.f, o[8] = {};
      for (int p = 0; p < parts; ++p) {
        const float f = ex2_approx(ld_partial(peer(p, C::kStatsAt + slot(p)), a.nsplit > 1) - M);
        L = fmaf(ld_partial(peer(p, C::kStatsAt + 2 * kRows + slot(p)), a.nsplit > 1), f, L);
#pragma unroll
        for (int q = 0; q < 8; q += 4) {
          const float4 t =
              ld_partial4(peer(p, slot(p) * C::kPitch + col + q), a.nsplit > 1);
          o[q] = fmaf(t.x, f, o[q]), o[q + 1] = fmaf(t.y, f, o[q + 1]);
          o[q + 2] = fmaf(t.z, f, o[q + 2]), o[q + 3] = fmaf(t.w, f, o[q + 3]);
        }
      }
      const float inv = 1.f / L;
      w = make_uint4(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv),
                     pack2<T>(o[4] * inv, o[5] * inv), pack2<T>(o[6] * inv, o[7] * inv));
    }
    *reinterpret_cast<uint4*>(a.o + row + col) = w;
  }
  __syncwarp();
  if (a.nsplit > 1) cluster_sync_all();  // no CTA exits while its results may be read
}

// ---------------------------------------------------------------- host side
namespace {

// A key head's G query heads packed into row tiles; groups too large for a tile (or that
// would waste half of one) run head by head, every query head with its own copy of the
// key head.
struct RowTiles {
  int group, kv_heads, tile_t, nq;
  int64_t items;
};
RowTiles row_tiles(const CrossProblem& p) {
  const int G = p.heads / p.kv_heads;
  const bool pack = G <= kRows / 2 || kRows % G == 0;
  RowTiles t;
  t.group = pack ? G : 1;
  t.kv_heads = pack ? p.kv_heads : p.heads;
  t.tile_t = std::min(kRows / t.group, p.Tq);
  t.nq = (p.Tq + t.tile_t - 1) / t.tile_t;
  t.items = static_cast<int64_t>(p.B) * t.kv_heads * ((t.nq + 1) / 2);
  return t;
}

template <typename T, int D>
int launch_tiles(const CrossProblem& p, cudaStream_t s) {
  using C = Cfg<D>;
  CrossArgs a = {};
  a.Tq = p.Tq;
  a.Tk = p.Tk;
  a.lens = p.lens;
  a.o = static_cast<uint16_t*>(p.o);
  a.o_row = static_cast<int64_t>(p.heads) * D;
  a.c = cross_scale(p.scale);
  a.err = device_error_word();
  const RowTiles t = row_tiles(p);
  a.group = t.group;
  a.kv_heads = t.kv_heads;
  a.tile_t = t.tile_t;
  a.nq = t.nq;
  const int64_t items = t.items;
  if (items > INT32_MAX / kCrossMaxSplit) return VITB200_E_UNSUPPORTED;
  const int key_tiles = std::max(1, (p.Tk + kKeys - 1) / kKeys);
  // The largest cluster of which `items` fit the GPU at once.
  a.nsplit = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({device_num_sms() / items, key_tiles, kCrossMaxSplit})));
  while (a.nsplit > 1 &&
         cluster_slots(cross_attention_kernel<T, D>, C::kSmem, kThreads, a.nsplit) < items)
    --a.nsplit;

  CUtensorMap tq, tk, tv;
  const uint64_t es = 2;
  {
    const uint64_t dims[5] = {D, static_cast<uint64_t>(a.group), static_cast<uint64_t>(p.Tq),
                              static_cast<uint64_t>(a.kv_heads), static_cast<uint64_t>(p.B)};
    const uint64_t strides[4] = {D * es, static_cast<uint64_t>(p.q_row) * es,
                                 static_cast<uint64_t>(a.group) * D * es,
                                 static_cast<uint64_t>(p.B == 1 ? p.q_row * p.Tq : p.q_batch) * es};
    const uint32_t box[5] = {kHalf, static_cast<uint32_t>(a.group),
                             static_cast<uint32_t>(a.tile_t), 1, 1};
    if (int st = encode_tmap_typed(&tq, 5, p.q, dims, strides, box, 1, 1)) return st;
  }
  // (One image has no batch stride; a map wants a real one.)
  auto kv_map = [&](CUtensorMap* map, const void* t, int64_t row, int64_t batch) {
    if (p.B == 1) batch = row * p.Tk;
    const uint64_t dims[4] = {D, static_cast<uint64_t>(p.Tk), static_cast<uint64_t>(p.kv_heads),
                              static_cast<uint64_t>(p.B)};
    const uint64_t strides[3] = {static_cast<uint64_t>(row) * es, D * es,
                                 static_cast<uint64_t>(batch) * es};
    const uint32_t box[4] = {kHalf, kKeys, 1, 1};
    return encode_tmap_typed(map, 4, t, dims, strides, box, 1, 1);
  };
  if (int st = kv_map(&tk, p.k, p.k_row, p.k_batch)) return st;
  if (int st = kv_map(&tv, p.v, p.v_row, p.v_batch)) return st;
  a.kv_div = p.heads / p.kv_heads / a.group;
  return launch_kernel(cross_attention_kernel<T, D>,
                       dim3(static_cast<unsigned>(items * a.nsplit)), dim3(kThreads), C::kSmem, s,
                       static_cast<unsigned>(a.nsplit), tq, tk, tv, a);
}

template <typename F>
int with_head(int type, int D, F&& f) {
  auto typed = [&](auto tag) {
    if (D == 64) return f(tag, std::integral_constant<int, 64>{});
    return f(tag, std::integral_constant<int, 128>{});
  };
  return type == VITB200_BF16 ? typed(__nv_bfloat16{}) : typed(__half{});
}

}  // namespace

int cross_attention_prepare_device() {
  for (int type : {VITB200_F16, VITB200_BF16})
    for (int D : {64, 128}) {
      const int st = with_head(type, D, [](auto tag, auto d) {
        return cuda_status(cudaFuncSetAttribute(cross_attention_kernel<decltype(tag), d.value>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                Cfg<d.value>::kSmem));
      });
      if (st) return st;
    }
  if (int st = cross_attention_rows_prepare_device()) return st;
  return cross_attention_token_prepare_device();
}

namespace {
bool token_form(const CrossProblem& p) {
  return static_cast<int64_t>(p.heads / p.kv_heads) * p.Tq <= kTokenRows;
}
// The 64-row and the tcgen05 form by fitted times, in us (bf16, 1 to 384 image-heads of 20
// to 192 rows x 257 to 16384 keys, both head sizes: over 444 such calls the choice is
// 0.6 % slower than the faster form on average, 29 % at worst). 64 image-heads, D = 64 and 128:
// 64 rows x 257 keys 7 and 10 us against 10 and 11; 128 x 2048 24 and 38 against 16 and 21.
// 384 x 61 x 577, D = 64: 21 against 33; 300 x 2224 x 64, D = 64: 80 against 134.
double ceil_of(double a, double b) { return std::ceil(a / b); }

// A CTA of the 64-row form takes `alone` a key tile, an SM `full` for each of its CTAs.
double rows_form_us(const CrossProblem& p) {
  const bool d64 = p.D == 64;
  const double alone = d64 ? 0.71 : 1.25, full = d64 ? 0.576 : 0.94, setup = d64 ? 0.48 : 0.98;
  const double sms = device_num_sms(), per_sm = d64 ? 4 : 2;
  const double ctas = static_cast<double>(p.B) * p.kv_heads *
                      ceil_of(static_cast<double>(p.heads / p.kv_heads) * p.Tq, 64);
  const double tiles = ceil_of(p.Tk, 64);
  const double split = std::max(1.0, std::min<double>({std::floor(sms * per_sm / ctas),
                                                       std::floor(tiles / 2), kCrossMaxSplit}));
  const double share = ceil_of(tiles, split), each = ctas * split / sms;
  return 5.0 + (split > 1 ? (d64 ? 1.4 : 1.3) : 0.0) +
         std::max(ceil_of(each, per_sm) * (setup + share * alone),
                  (each <= per_sm ? std::ceil(each) : each) * (setup + share * full));
}

// A CTA of the tcgen05 form has an SM; joining partial results goes by their number.
double tile_form_us(const CrossProblem& p) {
  const bool d64 = p.D == 64;
  const RowTiles t = row_tiles(p);
  const double sms = device_num_sms(), ctas = static_cast<double>(t.items);
  const double tiles = ceil_of(p.Tk, kKeys);
  const double split =
      std::max(1.0, std::min<double>({std::floor(sms / ctas), tiles, kCrossMaxSplit}));
  const double key_tile = t.nq > 1 ? (d64 ? 1.75 : 2.4) : (d64 ? 0.84 : 1.17);
  const double parts = split * (t.nq > 1 ? 1 : 2);
  const double rows = std::min<double>(static_cast<double>(t.group) * p.Tq, 2 * kRows);
  return 3.0 + ceil_of(ctas * split, sms) *
                   ((d64 ? 5.6 : 6.3) + ceil_of(tiles, split) * key_tile +
                    (parts > 1 ? (d64 ? 0.044 : 0.09) * rows * parts / 16 : 0.0));
}

// A batch that shares one image (stride 0) has no tensor map, which the tcgen05 form
// copies by: the 64-row form reads by address.
bool shared_image(const CrossProblem& p) {
  return p.B > 1 && (p.q_batch == 0 || p.k_batch == 0 || p.v_batch == 0);
}
bool rows_form(const CrossProblem& p) {
  const int64_t rows = static_cast<int64_t>(p.heads / p.kv_heads) * p.Tq;
  if (rows > INT32_MAX / 2) return false;  // counted in 32 bits there
  if (shared_image(p)) return true;
  return static_cast<int64_t>(p.B) * p.kv_heads * ((rows + 63) / 64) <=
             INT32_MAX / kCrossMaxSplit &&
         rows_form_us(p) <= tile_form_us(p);
}
}  // namespace

size_t cross_attention_workspace(const CrossProblem& p) {
  return token_form(p) ? cross_attention_token_workspace(p) : 0;
}

int cross_attention_launch(const CrossProblem& p, cudaStream_t s) {
  if (token_form(p)) return cross_attention_token_launch(p, s);
  if (rows_form(p)) return cross_attention_rows_launch(p, s);
  if (shared_image(p)) return VITB200_E_UNSUPPORTED;
  return with_head(p.type, p.D, [&](auto tag, auto d) {
    return launch_tiles<decltype(tag), d.value>(p, s);
  });
}

}  // namespace vitb200

using namespace vitb200;

namespace {

// Sizes of the operator; a status where they make none.
int cross_sizes(int type, int B, int Tq, int Tk, int heads, int kv_heads, int head_dim,
                CrossProblem* p) {
  if (type != VITB200_F16 && type != VITB200_BF16) return VITB200_E_INVALID_ARG;
  if (B < 0 || Tq < 0 || Tk < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0)
    return VITB200_E_INVALID_ARG;
  if (head_dim != 64 && head_dim != 128) return VITB200_E_UNSUPPORTED;
  if (Tq > INT32_MAX - 256 || Tk > INT32_MAX - 256 || heads > 65535) return VITB200_E_UNSUPPORTED;
  p->type = type;
  p->B = B;
  p->Tq = Tq;
  p->Tk = Tk;
  p->heads = heads;
  p->kv_heads = kv_heads;
  p->D = head_dim;
  return 0;
}

}  // namespace

extern "C" size_t vitb200_cross_attention_workspace_bytes(int B, int Tq, int Tk, int heads,
                                                          int kv_heads, int head_dim) {
  try {
    CrossProblem p = {};
    if (cross_sizes(VITB200_BF16, B, Tq, Tk, heads, kv_heads, head_dim, &p) || B == 0 || Tq == 0 ||
        Tk == 0)
      return 0;
    return cross_attention_workspace(p);
  } catch (...) {
    return 0;
  }
}

extern "C" int vitb200_cross_attention(const void* q, const void* k, const void* v, void* o,
                                       int type, int B, int Tq, int Tk, int heads, int kv_heads,
                                       int head_dim, int64_t q_row, int64_t q_batch, int64_t k_row,
                                       int64_t k_batch, int64_t v_row, int64_t v_batch,
                                       const int* kv_lens, float scale, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  try {
    CrossProblem p = {};
    if (int st = cross_sizes(type, B, Tq, Tk, heads, kv_heads, head_dim, &p)) return st;
    const int64_t wq = static_cast<int64_t>(heads) * head_dim;
    const int64_t wk = static_cast<int64_t>(kv_heads) * head_dim;
    if (q_row < wq || k_row < wk || v_row < wk || q_batch < 0 || k_batch < 0 || v_batch < 0)
      return VITB200_E_INVALID_ARG;
    if (B == 0 || Tq == 0) return 0;
    if (!q || !o || (Tk > 0 && (!k || !v))) return VITB200_E_INVALID_ARG;
    for (const void* t : {q, k, v, static_cast<const void*>(o), static_cast<const void*>(workspace)})
      if (reinterpret_cast<uintptr_t>(t) % 16 != 0) return VITB200_E_ALIGNMENT;
    for (int64_t st : {q_row, q_batch, k_row, k_batch, v_row, v_batch})
      if (st % 8 != 0) return VITB200_E_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(kv_lens) % 4 != 0) return VITB200_E_ALIGNMENT;
    if (int st = vitb200_init()) return st;
    if (Tk == 0)
      return cuda_status(cudaMemsetAsync(o, 0, static_cast<size_t>(B) * Tq * wq * 2,
                                         static_cast<cudaStream_t>(stream)));
    const size_t need = cross_attention_workspace(p);
    if (need > 0 && (!workspace || workspace_bytes < need)) return VITB200_E_WORKSPACE;
    p.q = q;
    p.k = k;
    p.v = v;
    p.o = o;
    p.lens = kv_lens;
    p.q_row = q_row;
    p.q_batch = q_batch;
    p.k_row = k_row;
    p.k_batch = k_batch;
    p.v_row = v_row;
    p.v_batch = v_batch;
    p.scale = scale;
    p.workspace = workspace;
    return cross_attention_launch(p, static_cast<cudaStream_t>(stream));
  } catch (...) {
    return VITB200_E_INVALID_ARG;
  }
}
