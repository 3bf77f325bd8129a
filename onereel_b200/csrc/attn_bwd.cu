// Packed variable-length scene attention, backward, bf16 in / fp32 accumulate / bf16 out, for sm_100a.
//
// With S = scale q k^T, P = exp(S - lse) (recomputed from the forward's log-sum-exp), o = P v and incoming gradients
// dO of o and dL of lse:
//   delta_i = sum_d dO_id o_id - dL_i        dP = dO v^T        dS = P * (dP - delta)
//   dq = scale dS k        dk = scale dS^T q        dv = P^T dO
// delta and lse * log2(e) come from a first, memory-bound kernel ([heads, nq] pairs). The main kernel has two kinds of
// work items, both a block of up to 128 rows of one head that stays resident while tiles of 128 rows stream past it:
//   kDkv: K / V rows resident, the q / dO rows that read them stream:  S^T = K q^T, dP^T = V dO^T,
//         dV += P^T dO, dK += dS^T q. Its ranges are every query range that reads the rows, so key ranges that several
//         segments share are summed in fp32 in a fixed order.
//   kDq:  q / dO rows resident, their K / V rows stream:               S = q K^T, dP = dO V^T, dQ += dS K.
// S and dP are computed twice (seven products of the size of S instead of five). In exchange nothing is added across
// CTAs: no atomics, no fp32 dQ in memory, the same bits on every run.
//
// A CTA has the forward's roles: warp 0 streams tiles by TMA, warp 1 owns TMEM and issues MMAs (kDq: those of S and dP;
// warp 3 those of dQ), warps 2-3 (kDq: warp 2) prepare each tile (row statistics of streamed queries; zeros in the
// shared-memory rows past a range's end, so that what lies there - other segments, or NaN in rows no segment owns -
// enters no product), warps 4-11 hold P and dS as fragments of two rows of a 16-lane block each and write them back to
// TMEM as bf16, the A operand of the accumulating MMAs.
//
// kDkv, tiles of 128 queries. TMEM columns: S^T / P^T [0,128), dP^T / dS^T [128,256), dV [256,256+D), dK [256+D,256+2D):
// all 512 at D = 128. While the compute warps work on P(j) the tensor pipe runs dK(j-1) and dP(j); while they work on
// dS(j), dV(j) and S(j+1). P is handed over in two halves, so dV begins under the second half's exponentials.
// kDq, tiles of 64 keys, taken by turns by two groups of four compute warps: a step (loads, exponentials, dS) is mostly
// latency, and each group's hides in the other's. TMEM columns, per group: S [0,128), dP [128,256), dS [256,320) (bf16);
// dQ [320,320+D), q [448,..) as a bf16 A operand: from TMEM a 64-column MMA takes 32 clocks instead of the 48 that
// reading both operands from shared memory costs (dO has no TMEM left). S and dP of a group's next tile are issued once
// it has read them, dQ when dS is there.
//
// delta. do . o~ with the forward's bf16 o~ (P rounded, then o rounded) is off by some e_i, the same for all keys of
// query i. In dq_i it adds e_i sum_j P k, one more error of the size of dS's roundings. In the dk it adds up: sum_j dS_ij
// should be 0 and becomes -e_i, so that sums of dk over keys - the gradient of a key bias - came out twice as far from
// float64 as with exact attention. So the kDq blocks, which see all keys of their queries, also sum P dP in fp32 and
// publish delta_i = sum_j P dP - dL; the kDkv blocks wait for it. Items are drawn by a ticket with the kDq items first:
// whoever holds a kDkv item knows that every kDq item is being computed or done, and kDq items wait for nothing. Where
// one tile holds all keys of its queries (at most 64: then dS is a small difference of large terms; two keys: dq 0.0040
// off in the 2-norm instead of 0.0024) a kDq block uses its own sum as well.
//
// Rounded to bf16 are P and dS, the A operands of the accumulating products (one rounding of each in dv, dq and dk), and the
// gradients as they are stored; scores, exponentials, delta and the accumulators are fp32.
//
// What bounds it (figures: forward excluded, 5 products of useful work). 16 heads of 128, 22516 x 48212 rows in segments
// of up to 14438 keys: 6.7 ms, 0.90 PFLOP/s useful and 1.26 computed, with the clock down at 1.7 GHz under the power cap:
// the seven products run at 0.92 of the rate at which a library product is sustained under that cap. 16 heads of 64,
// 3 x 2048 rows: 279 us; a tile costs the compute warps as much as at D = 128 (exponentials, TMEM loads and barriers of
// some 1200 clocks per 64 keys), in which its MMAs take 450.
//
// Every mbarrier wait is bounded as in the forward: a stuck pipeline sets the error word and winds down. The compute warps'
// waits have one verdict per warp, and their last barrier one for all eight, so that no warp waits there for another that has
// given up (0.7 % of the time at D = 128, 2 % at D = 64).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>
#include <initializer_list>
#include <new>
#include <type_traits>
#include <vector>

#include "orl_common.h"
#include "ptx.cuh"
#include "tensor_map.cuh"

namespace orl {

using BwdWork = orl_attn_bwd_work;
static_assert(sizeof(BwdWork) == 32, "backward work item layout");
constexpr int kDkv = ORL_ATTN_BWD_KV, kDq = ORL_ATTN_BWD_Q;
constexpr float kLog2e = 1.4426950408889634f;

constexpr int kDkvRows = 128, kDqRows = 64;             // rows of a streamed tile
constexpr int kWholeKeys = ORL_ATTN_BWD_WHOLE;          // segments of so few keys take delta from their tile
static_assert(kWholeKeys <= kDqRows, "a whole segment is one tile");

template <int D>
struct BwdCfg {
  static constexpr int kChunks = D / 64;              // 128-byte swizzle columns per row
  static constexpr int kTileBytes = 128 * D * 2;      // one 128-row bf16 tile
  static constexpr int kChunkBytes = 128 * 128;       // one 128-row x 64-column chunk
  // kDkv: resident tiles K, V; rings of streamed tiles T1 = dO and T0 = q (S of tile j + 1 is issued before dK of tile
  // j, so q is loaded two tiles ahead of its release).
  static constexpr int kStages0 = D == 64 ? 4 : 3;
  static constexpr int kStages1 = D == 64 ? 4 : 2;
  static constexpr int kROff = 0;
  static constexpr int kT1Off = 2 * kTileBytes;
  static constexpr int kT0Off = kT1Off + kStages1 * kTileBytes;
  static constexpr int kStatOff = kT0Off + kStages0 * kTileBytes;
  static constexpr int kStatBytes = 2 * 4 * 36 * 4;   // lse2, delta: four groups of 32 columns, padded (see stat_at)
  // kDq: dO resident, a ring of pairs of 64-row tiles K, V
  static constexpr int kPairOff = kTileBytes;
  static constexpr int kHalfBytes = kTileBytes / 2;
  static constexpr int kHalfChunk = kChunkBytes / 2;
  static constexpr int kPairStages = D == 64 ? 8 : 6;
  static constexpr int kMaxStages = 8;
  static constexpr int kBarOff = kStatOff + 2 * kStatBytes;
  static constexpr int kBarR = 0;                       // resident tiles landed
  static constexpr int kBarQ = 1;                       // kDq: q in TMEM
  static constexpr int kBarT0 = 2;                      // streamed tiles landed, per stage (kDq: the pair)
  static constexpr int kBarT1 = kBarT0 + kMaxStages;
  static constexpr int kBarAux = kBarT1 + kStages1;     // streamed tiles landed and prepared, per T0 stage
  static constexpr int kBarE0 = kBarAux + kMaxStages;   // stage free
  static constexpr int kBarE1 = kBarE0 + kMaxStages;
  static constexpr int kBarS = kBarE1 + kStages1;       // S computed; kDq: S and dP, per group
  static constexpr int kBarDp = kBarS + 2;              // kDkv: dP computed
  static constexpr int kBarP = kBarDp + 1;              // kDkv: half of P stored (two); kDq: S and dP read, per group
  static constexpr int kBarDs = kBarP + 2;              // dS stored; kDq: per group
  static constexpr int kBarDone = kBarDs + 2;
  static constexpr int kBarDrain = kBarDone + 1;
  static constexpr int kBarDrain1 = kBarDrain + 1;      // kDq: of the thread that issues S and dP
  static constexpr int kNumBars = kBarDrain1 + 1;
  static constexpr int kSmemBytes = kBarOff + kNumBars * 8 + 16;
  static constexpr uint32_t kTmemCols = 512;
  static constexpr uint32_t kColDv = 256, kColDk = 256 + D;       // kDkv (S at 0, dP at 128)
  static constexpr uint32_t kColDp = 128, kColDs = 256, kColDq = 320, kColQ = 448;                // kDq (S at 0)
  static_assert(kPairOff + kPairStages * 2 * kHalfBytes <= kStatOff, "ring of pairs");
  static_assert(kPairStages <= kMaxStages && kStages0 <= kMaxStages, "rings");
  static_assert(kStatOff % 16 == 0 && kBarOff % 8 == 0, "alignment");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// Where the statistic of streamed row c lies: a thread of the compute warps needs columns 8r + 2 cq + {0, 1}, here 32
// consecutive floats of group cq (eight 16-byte loads); groups 36 floats apart fall into different banks.
__device__ __forceinline__ int stat_at(int c) { return 36 * ((c >> 1) & 3) + 2 * (c >> 3) + (c & 1); }

// position in a ring of n stages: stage s, parity ph of its current use
struct Ring {
  int n, s = 0, ph = 0;
  __device__ explicit Ring(int n_) : n(n_) {}
  __device__ void next() {
    if (++s == n) {
      s = 0;
      ph ^= 1;
    }
  }
};

constexpr int kBwdThreads = 384;
constexpr int kAuxThreads = 64;
// register split as in the forward: 4 x 32 x 120 + 8 x 32 x 192 = 384 x 168
constexpr int kBwdLaunchRegs = 168, kBwdRegsLow = 120, kBwdRegsHigh = 192;
static_assert(4 * kBwdRegsLow + 8 * kBwdRegsHigh == 12 * kBwdLaunchRegs, "register split must add up to the launch total");

__device__ __forceinline__ void bwd_drain_wait(uint32_t bar, uint32_t parity, int* err) {
  const unsigned long long t0 = global_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (global_ns() - t0 > kWaitLimitNs) {
      atomicOr(err, kErrTimeoutDrain);
      return;
    }
  }
}

struct BwdShared {
  uint8_t* smem;         // 1024-aligned tile area
  uint32_t sbase;        // its shared-window address
  uint32_t bar0;         // address of barrier 0
  volatile int* abort_flag;
  __device__ uint32_t bar(int i) const { return bar0 + 8u * i; }
};

// the tiles of an item's ranges in order: each range cut into tiles of kRows rows, the last one of a range shorter
template <int kRows>
struct TileWalk {
  const int2* ranges;
  int left;              // ranges not yet begun
  int row, rest;         // next row and rows left in the current range
  __device__ TileWalk(const int2* r, int n) : ranges(r), left(n), row(0), rest(0) {}
  // moves to the next tile: its first row, its rows in the return value
  __device__ int next(int& first) {
    while (rest <= 0) {
      if (left == 0) return 0;
      const int2 r = __ldg(ranges++);
      --left;
      row = r.x;
      rest = r.y;
    }
    first = row;
    const int n = min(kRows, rest);
    row += kRows;
    rest -= kRows;
    return n;
  }
};

// ---------------------------------------------------------------------------------------------- TMA producer
// rows [y, y + 64 boxes) of head columns x0.. into a tile of that many 64-row boxes
template <int D, int kBoxes>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x0, int y,
                                          uint64_t pol) {
  constexpr int kBox = 64 * 128;
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll
    for (int b = 0; b < kBoxes; ++b)
      tma_load_2d(dst + (c * kBoxes + b) * kBox, map, bar, x0 + 64 * c, y + 64 * b, pol);
}

template <int D>
__device__ __forceinline__ void bwd_produce_dkv(const BwdShared& sh, const CUtensorMap* tm_q, const CUtensorMap* tm_k,
                                                const CUtensorMap* tm_v, const CUtensorMap* tm_do, const BwdWork& wi,
                                                const int2* ranges, int* err) {
  using C = BwdCfg<D>;
  const uint64_t pol_r = policy_evict_first(), pol_t = policy_evict_last();
  const int x0 = wi.head * D;
  mbar_expect_tx(sh.bar(C::kBarR), 2 * C::kTileBytes);
  load_tile<D, 2>(sh.sbase + C::kROff, tm_k, sh.bar(C::kBarR), x0, wi.row0, pol_r);
  load_tile<D, 2>(sh.sbase + C::kROff + C::kTileBytes, tm_v, sh.bar(C::kBarR), x0, wi.row0, pol_r);
  TileWalk<kDkvRows> walk(ranges, wi.n_ranges);
  const int n0 = C::kStages0;
  Ring a(n0), b(C::kStages1);
  int issued0 = 0, issued1 = 0;
  for (int j = 0; j < wi.n_tiles; ++j, a.next(), b.next()) {
    int y = 0;
    walk.next(y);
    bool ok = j < n0 || mbar_wait(sh.bar(C::kBarE0 + a.s), a.ph ^ 1, sh.abort_flag);
    if (ok) {
      mbar_expect_tx(sh.bar(C::kBarT0 + a.s), C::kTileBytes);
      load_tile<D, 2>(sh.sbase + C::kT0Off + a.s * C::kTileBytes, tm_q, sh.bar(C::kBarT0 + a.s), x0, y, pol_t);
      issued0 = j + 1;
      ok = j < C::kStages1 || mbar_wait(sh.bar(C::kBarE1 + b.s), b.ph ^ 1, sh.abort_flag);
    }
    if (!ok) {
      atomicOr(err, kErrTimeoutLoad);
      break;
    }
    mbar_expect_tx(sh.bar(C::kBarT1 + b.s), C::kTileBytes);
    load_tile<D, 2>(sh.sbase + C::kT1Off + b.s * C::kTileBytes, tm_do, sh.bar(C::kBarT1 + b.s), x0, y, pol_t);
    issued1 = j + 1;
  }
  if (*sh.abort_flag) {
    // wind down: every copy this thread started must land before the CTA's shared memory is released
    bwd_drain_wait(sh.bar(C::kBarR), 0, err);
    for (int j = issued0 > n0 ? issued0 - n0 : 0; j < issued0; ++j)
      bwd_drain_wait(sh.bar(C::kBarT0 + j % n0), (j / n0) & 1, err);
    for (int j = issued1 > C::kStages1 ? issued1 - C::kStages1 : 0; j < issued1; ++j)
      bwd_drain_wait(sh.bar(C::kBarT1 + j % C::kStages1), (j / C::kStages1) & 1, err);
  }
}

template <int D>
__device__ __forceinline__ void bwd_produce_dq(const BwdShared& sh, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                                               const CUtensorMap* tm_do, const BwdWork& wi, const int2* ranges,
                                               int* err) {
  using C = BwdCfg<D>;
  const uint64_t pol = policy_evict_last();
  const int x0 = wi.head * D;
  mbar_expect_tx(sh.bar(C::kBarR), C::kTileBytes);
  load_tile<D, 2>(sh.sbase + C::kROff, tm_do, sh.bar(C::kBarR), x0, wi.row0, policy_evict_first());
  TileWalk<kDqRows> walk(ranges, wi.n_ranges);
  Ring a(C::kPairStages);
  int issued = 0;
  for (int u = 0; u < wi.n_tiles; ++u, a.next()) {
    int y = 0;
    walk.next(y);
    if (u >= C::kPairStages && !mbar_wait(sh.bar(C::kBarE0 + a.s), a.ph ^ 1, sh.abort_flag)) {
      atomicOr(err, kErrTimeoutLoad);
      break;
    }
    const uint32_t dst = sh.sbase + C::kPairOff + a.s * 2 * C::kHalfBytes, bar = sh.bar(C::kBarT0 + a.s);
    mbar_expect_tx(bar, 2 * C::kHalfBytes);
    load_tile<D, 1>(dst, tm_k, bar, x0, y, pol);
    load_tile<D, 1>(dst + C::kHalfBytes, tm_v, bar, x0, y, pol);
    issued = u + 1;
  }
  if (*sh.abort_flag) {
    bwd_drain_wait(sh.bar(C::kBarR), 0, err);
    for (int u = issued > C::kPairStages ? issued - C::kPairStages : 0; u < issued; ++u)
      bwd_drain_wait(sh.bar(C::kBarT0 + u % C::kPairStages), (u / C::kPairStages) & 1, err);
  }
}

// ---------------------------------------------------------------------------------------------- tile preparation
constexpr uint32_t kDeltaPending = 0x7fd1d1d1u;          // a NaN no arithmetic gives
__device__ __forceinline__ uint32_t load_relaxed(const float* p) {
  uint32_t v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// 64 threads (kDq: 32) wait for each streamed tile and hand it on prepared, so that the issuing thread has one wait for it.
// kDkv: the statistics of its query rows (lse2 = +inf past the end, so P = 0 there) into one of two slots, zeros
// over the shared-memory rows past the end.
template <int D>
__device__ __forceinline__ void bwd_prepare_dkv(const BwdShared& sh, const BwdWork& wi, const int2* ranges,
                                                const float2* __restrict__ stats, const float* __restrict__ delta,
                                                long long nq, int t, int* err) {
  using C = BwdCfg<D>;
  const long long h0 = static_cast<long long>(wi.head) * nq;
  // (lse2, delta) of a query row, once its kDq block has published it
  auto row_stats = [&](long long row, bool& ok) {
    float2 x = __ldg(stats + h0 + row);
    const unsigned long long t0 = global_ns();
    uint32_t bits = load_relaxed(delta + h0 + row);
    while (ok && bits == kDeltaPending) {
      if (*sh.abort_flag || global_ns() - t0 > kWaitLimitNs) {
        *sh.abort_flag = 1;
        ok = false;
      }
      bits = load_relaxed(delta + h0 + row);
    }
    x.y = __uint_as_float(bits);
    return x;
  };
  TileWalk<kDkvRows> walk(ranges, wi.n_ranges);
  const int n0 = C::kStages0;
  Ring a(n0), b(C::kStages1), free(n0);                  // free: two tiles behind, whose dK released the slot
  for (int j = 0; j < wi.n_tiles; ++j, a.next(), b.next()) {
    int row = 0;
    const int valid = walk.next(row);
    float2 x = make_float2(INFINITY, 0.f), y = x;
    bool ok = true;
    if (t < valid) x = row_stats(row + t, ok);
    if (t + 64 < valid) y = row_stats(row + t + 64, ok);
    if (ok && j >= 2) {
      ok = mbar_wait(sh.bar(C::kBarE0 + free.s), free.ph, sh.abort_flag);
      free.next();
    }
    ok = ok && mbar_wait(sh.bar(C::kBarT0 + a.s), a.ph, sh.abort_flag) &&
         mbar_wait(sh.bar(C::kBarT1 + b.s), b.ph, sh.abort_flag);
    if (!ok) {
      if (t == 0) atomicOr(err, kErrTimeoutLoad);
      return;
    }
    float* dst = reinterpret_cast<float*>(sh.smem + C::kStatOff + (j & 1) * C::kStatBytes);
    dst[stat_at(t)] = -x.x;                              // negated, as they are added
    dst[stat_at(t + 64)] = -y.x;
    dst[144 + stat_at(t)] = -x.y;
    dst[144 + stat_at(t + 64)] = -y.y;
    if (valid < kDkvRows) {
      for (int c = 0; c < 2 * C::kChunks; ++c) {         // T0's chunks, then T1's
        uint8_t* chunk = sh.smem + (c < C::kChunks ? C::kT0Off + a.s * C::kTileBytes + c * C::kChunkBytes
                                                   : C::kT1Off + b.s * C::kTileBytes + (c - C::kChunks) * C::kChunkBytes);
        for (int o = valid * 128 + t * 16; o < C::kChunkBytes; o += kAuxThreads * 16)
          *reinterpret_cast<uint4*>(chunk + o) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_async_smem();
    }
    mbar_arrive(sh.bar(C::kBarAux + a.s));
  }
}

// kDq: zeros over K's rows past the range (the columns of S and dP past the end are masked, but dS K sums over K's rows)
template <int D>
__device__ __forceinline__ void bwd_prepare_dq(const BwdShared& sh, const BwdWork& wi, const int2* ranges, int t,
                                               int* err) {
  using C = BwdCfg<D>;
  TileWalk<kDqRows> walk(ranges, wi.n_ranges);
  Ring a(C::kPairStages);
  for (int u = 0; u < wi.n_tiles; ++u, a.next()) {
    int row = 0;
    const int valid = walk.next(row);
    if (!mbar_wait(sh.bar(C::kBarT0 + a.s), a.ph, sh.abort_flag)) {
      if (t == 0) atomicOr(err, kErrTimeoutLoad);
      return;
    }
    if (valid < kDqRows) {
      uint8_t* k = sh.smem + C::kPairOff + a.s * 2 * C::kHalfBytes;
      for (int c = 0; c < C::kChunks; ++c)
        for (int o = valid * 128 + t * 16; o < C::kHalfChunk; o += 32 * 16)
          *reinterpret_cast<uint4*>(k + c * C::kHalfChunk + o) = make_uint4(0u, 0u, 0u, 0u);
      fence_async_smem();
    }
    mbar_arrive(sh.bar(C::kBarAux + a.s));
  }
}

// ---------------------------------------------------------------------------------------------- MMA issuer
// Descriptors are built once per tile and stepped by a constant: building one per MMA costs the issuing thread more
// (67 clocks measured per MMA) than the MMA takes (64 clocks at N = 128), stepping them 20. A wait costs it about 80
// clocks even when there is nothing to wait for, so waits for tiles stand before those for the compute warps.

__device__ __forceinline__ void bwd_mma_end(const BwdShared& sh, bool ok, int bar_done, int bar_drain, int* err) {
  if (ok) {
    mma_commit(sh.bar(bar_done));
  } else {
    atomicOr(err, kErrTimeoutMma);
    mma_commit(sh.bar(bar_drain));
    bwd_drain_wait(sh.bar(bar_drain), 0, err);
  }
}

template <int D>
__device__ __forceinline__ void bwd_mma_dkv(const BwdShared& sh, uint32_t tmem, const BwdWork& wi, int* err) {
  using C = BwdCfg<D>;
  constexpr uint32_t kIdescS = idesc_bf16(128, 128, false, false);
  constexpr uint32_t kIdescA = idesc_bf16(128, D, false, true);
  constexpr uint64_t kStep = C::kTileBytes >> 4;         // descriptor step from one tile to the next
  const int n = wi.n_tiles;
  auto wait = [&](int bar, int phase) { return mbar_wait(sh.bar(bar), phase & 1, sh.abort_flag); };
  const uint64_t k0 = smem_desc_sw128(sh.sbase + C::kROff, 16, 1024), v0 = k0 + kStep;
  const uint64_t q0 = smem_desc_sw128(sh.sbase + C::kT0Off, 16, 1024), o0 = smem_desc_sw128(sh.sbase + C::kT1Off, 16, 1024);
  const uint64_t qt0 = smem_desc_sw128(sh.sbase + C::kT0Off, C::kChunkBytes, 1024);     // the same tiles MN-major
  const uint64_t ot0 = smem_desc_sw128(sh.sbase + C::kT1Off, C::kChunkBytes, 1024);
  // D[col] = R * T^T, both K-major
  auto product = [&](uint32_t d, uint64_t r, uint64_t t) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint64_t off = ((kk >> 2) * C::kChunkBytes + (kk & 3) * 32) >> 4;
      mma_ss(d, r + off, t + off, kIdescS, kk > 0 ? 1u : 0u);
    }
  };
  // D[col] (+)= A * T, A bf16 in TMEM, T MN-major; 16-row steps [lo, hi) of the contraction
  auto accumulate = [&](uint32_t d, uint32_t a, uint64_t t, int lo, int hi, bool acc) {
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      if (kk >= lo && kk < hi) mma_ts(d, a + kk * 8, t + ((kk * 2048) >> 4), kIdescA, (acc || kk > 0) ? 1u : 0u);
  };
  Ring a(C::kStages0), b(C::kStages1);        // tile j; nx: tile j + 1
  Ring nx(a.n);
  nx.next();
  bool ok = wait(C::kBarR, 0) && wait(C::kBarAux, 0);
  if (ok) {
    tc_fence_after();
    product(tmem, k0, q0);
    mma_commit(sh.bar(C::kBarS));
  }
  for (int j = 0; ok && j < n; ++j) {
    // dP overwrites dS of tile j - 1, whose dK MMA was issued before
    product(tmem + 128, v0, o0 + b.s * kStep);
    mma_commit(sh.bar(C::kBarDp));
    ok = wait(C::kBarP, j);
    if (!ok) break;
    tc_fence_after();
    accumulate(tmem + C::kColDv, tmem, ot0 + b.s * kStep, 0, 4, j > 0);
    if (j + 1 < n) ok = wait(C::kBarAux + nx.s, nx.ph);
    ok = ok && wait(C::kBarP + 1, j);
    if (!ok) break;
    tc_fence_after();
    accumulate(tmem + C::kColDv, tmem, ot0 + b.s * kStep, 4, 8, true);
    if (j + 1 < n) {                                     // over P of this tile, whose dV MMA was issued before
      product(tmem, k0, q0 + nx.s * kStep);
      mma_commit(sh.bar(C::kBarS));
    }
    mma_commit(sh.bar(C::kBarE1 + b.s));
    ok = wait(C::kBarDs, j);
    if (!ok) break;
    tc_fence_after();
    accumulate(tmem + C::kColDk, tmem + 128, qt0 + a.s * kStep, 0, 8, j > 0);
    mma_commit(sh.bar(C::kBarE0 + a.s));
    a.next();
    b.next();
    nx.next();
  }
  bwd_mma_end(sh, ok, C::kBarDone, C::kBarDrain, err);
}

// kDq has two issuing threads, one for S and dP and one for dQ. One thread for all three was never waiting for anything but
// its own instructions (900 clocks of waits that were met and of issuing per 64 keys, in which the MMAs take 450 at D = 64
// and 900 at D = 128). What orders them is what the compute warps have read and written.
template <int D>
__device__ __forceinline__ void bwd_mma_dq_scores(const BwdShared& sh, uint32_t tmem, const BwdWork& wi, int* err) {
  using C = BwdCfg<D>;
  constexpr uint32_t kIdescS = idesc_bf16(128, 64, false, false);
  constexpr uint64_t kStep = (2 * C::kHalfBytes) >> 4;
  auto wait = [&](int bar, int phase) { return mbar_wait(sh.bar(bar), phase & 1, sh.abort_flag); };
  const uint64_t o0 = smem_desc_sw128(sh.sbase + C::kROff, 16, 1024);
  const uint64_t k0 = smem_desc_sw128(sh.sbase + C::kPairOff, 16, 1024), v0 = k0 + (C::kHalfBytes >> 4);
  Ring a(C::kPairStages);
  bool ok = wait(C::kBarQ, 0) && wait(C::kBarR, 0);
  for (int u = 0; ok && u < wi.n_tiles; ++u, a.next()) {
    // into the columns of tile u - 2 once that has been read
    ok = wait(C::kBarAux + a.s, a.ph) && (u < 2 || wait(C::kBarP + (u & 1), (u >> 1) - 1));
    if (!ok) break;
    tc_fence_after();
    const uint32_t d = tmem + 64 * (u & 1);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
      mma_ts(d, tmem + C::kColQ + kk * 8, k0 + a.s * kStep + (((kk >> 2) * C::kHalfChunk + (kk & 3) * 32) >> 4), kIdescS,
             kk > 0 ? 1u : 0u);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
      mma_ss(d + C::kColDp, o0 + (((kk >> 2) * C::kChunkBytes + (kk & 3) * 32) >> 4),
             v0 + a.s * kStep + (((kk >> 2) * C::kHalfChunk + (kk & 3) * 32) >> 4), kIdescS, kk > 0 ? 1u : 0u);
    mma_commit(sh.bar(C::kBarS + (u & 1)));
  }
  if (!ok) atomicOr(err, kErrTimeoutMma);
  mma_commit(sh.bar(C::kBarDrain1));
  bwd_drain_wait(sh.bar(C::kBarDrain1), 0, err);
}

template <int D>
__device__ __forceinline__ void bwd_mma_dq_acc(const BwdShared& sh, uint32_t tmem, const BwdWork& wi, int* err) {
  using C = BwdCfg<D>;
  constexpr uint32_t kIdescA = idesc_bf16(128, D, false, true);
  constexpr uint64_t kStep = (2 * C::kHalfBytes) >> 4;
  const uint64_t kt0 = smem_desc_sw128(sh.sbase + C::kPairOff, C::kHalfChunk, 1024);    // K MN-major
  Ring a(C::kPairStages);
  bool ok = true;
  for (int u = 0; u < wi.n_tiles; ++u, a.next()) {
    ok = mbar_wait(sh.bar(C::kBarDs + (u & 1)), (u >> 1) & 1, sh.abort_flag);
    if (!ok) break;
    tc_fence_after();
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      mma_ts(tmem + C::kColDq, tmem + C::kColDs + 32 * (u & 1) + kk * 8, kt0 + a.s * kStep + ((kk * 2048) >> 4), kIdescA,
             (u > 0 || kk > 0) ? 1u : 0u);
    mma_commit(sh.bar(C::kBarE0 + a.s));
  }
  bwd_mma_end(sh, ok, C::kBarDone, C::kBarDrain, err);
}

// ---------------------------------------------------------------------------------------------- P and dS
// whether ok holds for all eight compute warps (each with one verdict of its own, see mbar_wait_warp): all 256
// threads get here
__device__ __forceinline__ bool all_compute_warps(bool ok) {
  uint32_t all;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u)
      : "memory");
  return all != 0;
}

// two consecutive fp32 values of a fragment (one row, two columns) as a pair for the f32x2 instructions, which halve the
// issue slots of the arithmetic around the exponentials
__device__ __forceinline__ F2 f2_of(const uint32_t* x) { return f2(__uint_as_float(x[0]), __uint_as_float(x[1])); }

// Thread layout of the .16x256b / .16x128b TMEM shapes: warp sw owns lanes 32 (sw % 4) + 16 (sw / 4) + [0, 16); its
// thread holds the rows lane / 4 and lane / 4 + 8 of that block, register 4r + 2i + e of a 64-column load: row i,
// column 8r + 2 (lane % 4) + e.
struct BwdThread {
  int cq, row;           // lane % 4; tile row of the first of the two rows
  uint32_t lane_off;     // TMEM lane field
  __device__ BwdThread(int sw, int lane)
      : cq(lane & 3),
        row(32 * (sw & 3) + 16 * (sw >> 2) + (lane >> 2)),
        lane_off(static_cast<uint32_t>(32 * (sw & 3) + 16 * (sw >> 2)) << 16) {}
};

// Gradient rows go out through shared memory (the tiles there are done with): written as bf16 pairs at a pitch that
// spreads a warp's eight rows over all banks, then one bulk copy per row of D values. (Stored from the registers, 4 bytes
// per lane, they cost a block 4 us.)
template <int D>
struct BwdOut {
  static constexpr int kPitch = 2 * D + 16;             // bytes
  static constexpr int kBytes = 128 * kPitch;
};

// accumulator columns times f into staging slot i
template <int D>
__device__ __forceinline__ void bwd_stage(const BwdShared& sh, uint32_t acc, const BwdThread& th, float f, int i) {
  uint8_t* row = sh.smem + i * BwdOut<D>::kBytes + th.row * BwdOut<D>::kPitch + 4 * th.cq;
#pragma unroll
  for (int ch = 0; ch < D / 64; ++ch) {
    uint32_t o[32];
    tmem_ld_16x256b_x8(acc + th.lane_off + 64 * ch, o);
    tmem_wait_ld();
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      uint8_t* at = row + 128 * ch + 16 * r;
      *reinterpret_cast<uint32_t*>(at) = pack_bf16x2(__uint_as_float(o[4 * r + 0]) * f, __uint_as_float(o[4 * r + 1]) * f);
      *reinterpret_cast<uint32_t*>(at + 8 * BwdOut<D>::kPitch) =
          pack_bf16x2(__uint_as_float(o[4 * r + 2]) * f, __uint_as_float(o[4 * r + 3]) * f);
    }
  }
}

// the n staged tensors' rows to dst[0..n): 256 threads, one row copy each while there are rows; nothing unless all of them
// got here with ok
template <int D>
__device__ __forceinline__ void bwd_flush(const BwdShared& sh, const BwdWork& wi, int n, __nv_bfloat16* dst0,
                                          __nv_bfloat16* dst1, int heads, bool ok, int* err) {
  fence_async_smem();
  if (!all_compute_warps(ok)) {
    atomicOr(err, kErrTimeoutSoftmax);
    return;
  }
  const int t = threadIdx.x - 128, i = t >> 7, r = t & 127;
  if (i < n && r < wi.rows) {
    __nv_bfloat16* dst = i == 0 ? dst0 : dst1;
    bulk_store(dst + ((static_cast<long long>(wi.row0) + r) * heads + wi.head) * D,
               sh.sbase + i * BwdOut<D>::kBytes + r * BwdOut<D>::kPitch, 2 * D);
    bulk_commit();
    bulk_wait_read<0>();                                // shared memory outlives the copies
  }
}

// rows no product reaches (keys no query reads, queries without keys): zero gradients
template <int D>
__device__ __forceinline__ void bwd_zero(const BwdThread& th, const BwdWork& wi, __nv_bfloat16* __restrict__ dst,
                                         int heads) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (th.row + 8 * i >= wi.rows) continue;
    __nv_bfloat16* o = dst + (static_cast<long long>(wi.row0) + th.row + 8 * i) * heads * D + wi.head * D + 2 * th.cq;
    for (int col = 0; col < D; col += 8) *reinterpret_cast<uint32_t*>(o + col) = 0u;
  }
}

template <int D>
__device__ __forceinline__ void bwd_compute_dkv(const BwdShared& sh, uint32_t tmem, const BwdThread& th,
                                                const BwdWork& wi, float scale, __nv_bfloat16* __restrict__ dk,
                                                __nv_bfloat16* __restrict__ dv, int heads, int* err) {
  using C = BwdCfg<D>;
  const float scale_log2 = scale * kLog2e;
  const uint32_t s_addr = tmem + th.lane_off, dp_addr = s_addr + 128;
  const F2 sc = f2(scale_log2, scale_log2);
  Ring a(C::kStages0);
  bool ok = true;
  uint32_t p[64];                               // scores, then P in fp32
  for (int j = 0; j < wi.n_tiles; ++j, a.next()) {
    ok = mbar_wait_warp(sh.bar(C::kBarAux + a.s), a.ph, sh.abort_flag);
    if (!ok) break;
    // statistics of columns 8r + 2 cq + {0, 1}, two r per load, read before the wait for S (dP)
    const float4* st = reinterpret_cast<const float4*>(sh.smem + C::kStatOff + (j & 1) * C::kStatBytes) + 9 * th.cq;
    float4 c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = st[i];
    ok = mbar_wait_warp(sh.bar(C::kBarS), j & 1, sh.abort_flag);
    if (!ok) break;
    tc_fence_after();
    tmem_ld_16x256b_x8(s_addr, p);
    tmem_ld_16x256b_x8(s_addr + 64, p + 32);
    tmem_wait_ld();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[16];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float4 c4 = c[4 * h + (r >> 1)];
        const F2 l = (r & 1) ? f2(c4.z, c4.w) : f2(c4.x, c4.y);
        uint32_t* x = p + 4 * (8 * h + r);
        const float2 u = f2_split(ffma2(f2_of(x), sc, l)), v = f2_split(ffma2(f2_of(x + 2), sc, l));
        const float a0 = ex2(u.x), a1 = ex2(u.y), b0 = ex2(v.x), b1 = ex2(v.y);
        x[0] = __float_as_uint(a0);
        x[1] = __float_as_uint(a1);
        x[2] = __float_as_uint(b0);
        x[3] = __float_as_uint(b1);
        w[2 * r] = pack_bf16x2(a0, a1);
        w[2 * r + 1] = pack_bf16x2(b0, b1);
      }
      tmem_st_16x128b_x8(s_addr + 32 * h, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(sh.bar(C::kBarP + h));
    }
    ok = mbar_wait_warp(sh.bar(C::kBarDp), j & 1, sh.abort_flag);
    if (!ok) break;
    tc_fence_after();
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = st[36 + i];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t d[32], w[16];
      tmem_ld_16x256b_x8(dp_addr + 64 * h, d);
      tmem_wait_ld();
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float4 c4 = c[4 * h + (r >> 1)];
        const F2 l = (r & 1) ? f2(c4.z, c4.w) : f2(c4.x, c4.y);
        const uint32_t* x = p + 4 * (8 * h + r);
        const float2 u = f2_split(fmul2(f2_of(x), fadd2(f2_of(d + 4 * r), l)));
        const float2 v = f2_split(fmul2(f2_of(x + 2), fadd2(f2_of(d + 4 * r + 2), l)));
        w[2 * r] = pack_bf16x2(u.x, u.y);
        w[2 * r + 1] = pack_bf16x2(v.x, v.y);
      }
      // dS words of half h go over the dP columns [32 h, 32 h + 32), which half 0 has loaded
      tmem_st_16x128b_x8(dp_addr + 32 * h, w);
    }
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(sh.bar(C::kBarDs));
  }
  if (ok) ok = mbar_wait_warp(sh.bar(C::kBarDone), 0, sh.abort_flag);
  static_assert(2 * BwdOut<D>::kBytes <= C::kStatOff, "staging");
  if (ok) {
    tc_fence_after();
    bwd_stage<D>(sh, tmem + C::kColDv, th, 1.f, 0);
    bwd_stage<D>(sh, tmem + C::kColDk, th, scale, 1);
  }
  bwd_flush<D>(sh, wi, 2, dv, dk, heads, ok, err);
}

__device__ __forceinline__ float quad_add(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

template <int D>
__device__ __forceinline__ void bwd_compute_dq(const BwdShared& sh, uint32_t tmem, const BwdThread& th,
                                               const BwdWork& wi, const int2* ranges, float scale,
                                               const __nv_bfloat16* __restrict__ q, const float2* __restrict__ stats,
                                               const float* __restrict__ dlse, float* __restrict__ delta_out,
                                               long long nq, __nv_bfloat16* __restrict__ dq, int heads, int* err) {
  using C = BwdCfg<D>;
  const int sw = (threadIdx.x >> 5) - 4, lane = threadIdx.x & 31;
  const int grp = sw >> 2;                      // tiles grp, grp + 2, ...
  const uint32_t lanes = static_cast<uint32_t>(32 * (sw & 3)) << 16;
  {
    // q rows into TMEM, one row per thread, half of its columns per group; rows past the block are zeros
    constexpr int kWords = D / 4;
    const int r = 32 * (sw & 3) + lane;
    const __nv_bfloat16* src = q + ((static_cast<long long>(wi.row0) + r) * heads + wi.head) * D + grp * (D / 2);
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 x = r < wi.rows ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0u, 0u, 0u, 0u);
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
    if constexpr (D == 128) tmem_st32(tmem + C::kColQ + kWords * grp + lanes, w);
    else tmem_st16(tmem + C::kColQ + kWords * grp + lanes, w);
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(sh.bar(C::kBarQ));
  }
  const float scale_log2 = scale * kLog2e;
  // this thread's four rows: lane / 4 + 8 i of its warp's 32 TMEM lanes, i = 2 h + (register pair) of 16-lane block h
  float lse2[4], delta[4], dl[4], pdp[4];      // pdp: this thread's part of sum_j P dP
  const int row = 32 * (sw & 3) + (lane >> 2);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row + 8 * i;
    const float2 x = r < wi.rows ? __ldg(stats + static_cast<long long>(wi.head) * nq + wi.row0 + r)
                                 : make_float2(INFINITY, 0.f);
    lse2[i] = x.x;
    delta[i] = x.y;
    dl[i] = dlse != nullptr && r < wi.rows ? __ldg(dlse + static_cast<long long>(wi.head) * nq + wi.row0 + r) : 0.f;
    pdp[i] = 0.f;
  }
  const F2 sc = f2(scale_log2, scale_log2);
  const uint32_t s_addr = tmem + 64 * grp + lanes, dp_addr = s_addr + C::kColDp, ds_addr = tmem + C::kColDs + 32 * grp + lanes;
  constexpr uint32_t kBlock = 16u << 16;        // TMEM lane offset of the second 16-lane block
  TileWalk<kDqRows> walk(ranges, wi.n_ranges);
  int skip = 0;
  if (grp == 1) walk.next(skip);
  Ring before(C::kPairStages);                  // stage of this group's previous tile
  if (grp == 1) before.next();
  bool ok = true;
  for (int u = grp; u < wi.n_tiles; u += 2) {
    const int valid = walk.next(skip);
    walk.next(skip);
    ok = mbar_wait_warp(sh.bar(C::kBarS + grp), (u >> 1) & 1, sh.abort_flag);
    if (!ok) break;
    tc_fence_after();
    uint32_t p[2][32], d[2][32];
#pragma unroll
    for (int h = 0; h < 2; ++h) tmem_ld_16x256b_x8(s_addr + h * kBlock, p[h]);
#pragma unroll
    for (int h = 0; h < 2; ++h) tmem_ld_16x256b_x8(dp_addr + h * kBlock, d[h]);
    tmem_wait_ld();
    tc_fence_before();
    mbar_arrive(sh.bar(C::kBarP + grp));
    uint32_t w[2][16];
    // P, P dP with its row sums and dS, two columns per instruction. At D = 64, where the compute warps set the pace, one
    // block of code without branches, so that the arithmetic of some columns runs under the exponentials of others (dq of
    // 3 x 2048 rows, 16 heads: 164 -> 153 us); not for the last tile of a range, nor for segments whose delta is their
    // tile's, nor for D = 128: there the tensor pipe sets the pace, and dq of the scenes' layer went from 3050 to 3290 us.
    if (D == 64 && valid == kDqRows && !wi.whole) {
      F2 sum[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float l = -lse2[2 * h + (r & 1)], y = -delta[2 * h + (r & 1)];
          const float2 e = f2_split(ffma2(f2_of(&p[h][2 * r]), sc, f2(l, l)));
          const F2 pr = f2(ex2(e.x), ex2(e.y)), t = fmul2(pr, f2_of(&d[h][2 * r]));
          F2& x = sum[2 * h + (r & 1)];
          x = fadd2(x, t);
          const float2 ds = f2_split(ffma2(f2(y, y), pr, t));              // P dP - delta P
          w[h][r] = pack_bf16x2(ds.x, ds.y);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = f2_split(sum[i]);
        pdp[i] += x.x + x.y;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float l = -lse2[2 * h + (r & 1)];
          const float2 x = f2_split(ffma2(f2_of(&p[h][2 * r]), sc, f2(l, l)));
          p[h][2 * r] = __float_as_uint(ex2(x.x));
          p[h][2 * r + 1] = __float_as_uint(ex2(x.y));
        }
      if (valid < kDqRows) {
        // keys past the range add nothing, whatever their rows held
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (8 * (i >> 2) + 2 * th.cq + (i & 1) >= valid) p[h][i] = d[h][i] = 0u;
      }
      // d <- P dP and its row sums, two columns per instruction
      F2 sum[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
      F2 t[2][16];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          t[h][r] = fmul2(f2_of(&p[h][2 * r]), f2_of(&d[h][2 * r]));
          F2& x = sum[2 * h + (r & 1)];
          x = fadd2(x, t[h][r]);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = f2_split(sum[i]);
        if (wi.whole) delta[i] = quad_add(x.x + x.y) - dl[i];
        pdp[i] += x.x + x.y;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float y = -delta[2 * h + (r & 1)];
          const float2 ds = f2_split(ffma2(f2(y, y), f2_of(&p[h][2 * r]), t[h][r]));      // P dP - delta P
          w[h][r] = pack_bf16x2(ds.x, ds.y);
        }
    }
    if (u >= 2) {
      // dS goes over that of tile u - 2: its dQ is done when its stage is free
      ok = mbar_wait_warp(sh.bar(C::kBarE0 + before.s), before.ph, sh.abort_flag);
      if (!ok) break;
      before.next();
      before.next();
      tc_fence_after();
    }
    tmem_st_16x128b_x8(ds_addr, w[0]);
    tmem_st_16x128b_x8(ds_addr + kBlock, w[1]);
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(sh.bar(C::kBarDs + grp));
  }
  if (ok) {
    // both groups' sums meet in shared memory; group 0 publishes the rows' delta
    float* meet = reinterpret_cast<float*>(sh.smem + C::kStatOff);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pdp[i] = quad_add(pdp[i]);
      if (grp == 1 && th.cq == 0) meet[row + 8 * i] = pdp[i];
    }
  }
  asm volatile("bar.sync 1, 256;" ::: "memory");         // by every compute warp, whatever its verdict
  if (ok && grp == 0 && th.cq == 0) {
    const float* meet = reinterpret_cast<const float*>(sh.smem + C::kStatOff);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row + 8 * i;
      if (r >= wi.rows) continue;
      const float x = pdp[i] + meet[r] - dl[i];
      const uint32_t bits = x == x ? __float_as_uint(x) : 0x7fffffffu;      // any NaN but the pending mark
      asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(delta_out + static_cast<long long>(wi.head) * nq +
                                                               wi.row0 + r),
                   "r"(bits)
                   : "memory");
    }
  }
  if (ok) ok = mbar_wait_warp(sh.bar(C::kBarDone), 0, sh.abort_flag);
  if (ok) {
    tc_fence_after();
    bwd_stage<D>(sh, tmem + C::kColDq, th, scale, 0);
  }
  bwd_flush<D>(sh, wi, 1, dq, dq, heads, ok, err);
}

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                    const __nv_bfloat16* __restrict__ q,
                    const BwdWork* __restrict__ work, const int2* __restrict__ ranges,
                    const float2* __restrict__ stats, float* __restrict__ delta, int* __restrict__ ticket,
                    const float* __restrict__ dlse, __nv_bfloat16* __restrict__ dq,
                    __nv_bfloat16* __restrict__ dk,
                    __nv_bfloat16* __restrict__ dv, long long nq, int heads, float scale, int* __restrict__ err,
                    const int* __restrict__ n_items_dev) {
  using C = BwdCfg<D>;
  // the tiles need a 1024-byte boundary, which dynamic shared memory without static shared memory before it has
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  BwdShared sh;
  sh.smem = smem_raw;
  sh.sbase = smem_u32(sh.smem);
  if (sh.sbase & 1023u) {
    if (threadIdx.x == 0) atomicOr(err, kErrPlan);
    return;
  }
  sh.bar0 = sh.sbase + C::kBarOff;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sh.smem + C::kBarOff + C::kNumBars * 8);
  sh.abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 32 * 2) {
    tma_prefetch_map(&tm_q);
    tma_prefetch_map(&tm_k);
    tma_prefetch_map(&tm_v);
    tma_prefetch_map(&tm_do);
  }
  volatile int* drawn = reinterpret_cast<volatile int*>(tmem_slot + 2);
  if (threadIdx.x == 0) *drawn = atomicAdd(ticket, 1);
  __syncthreads();
  const int item = *drawn;
  // a grid sized by an upper bound (work list planned on the device): CTAs past the planned count have no item
  if (n_items_dev != nullptr && item >= __ldg(n_items_dev)) return;
  const BwdWork wi = work[item];
  const bool dkv = wi.kind == kDkv;

  if (threadIdx.x == 0) {
    mbar_init(sh.bar(C::kBarR), 1);
    mbar_init(sh.bar(C::kBarQ), 256);
    for (int s = 0; s < C::kMaxStages; ++s) {
      mbar_init(sh.bar(C::kBarT0 + s), 1);
      mbar_init(sh.bar(C::kBarAux + s), dkv ? kAuxThreads : 32);
      mbar_init(sh.bar(C::kBarE0 + s), 1);
    }
    for (int s = 0; s < C::kStages1; ++s) {
      mbar_init(sh.bar(C::kBarT1 + s), 1);
      mbar_init(sh.bar(C::kBarE1 + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sh.bar(C::kBarS + i), 1);
      mbar_init(sh.bar(C::kBarP + i), dkv ? 256 : 128);
      mbar_init(sh.bar(C::kBarDs + i), dkv ? 256 : 128);
    }
    mbar_init(sh.bar(C::kBarDp), 1);
    mbar_init(sh.bar(C::kBarDone), 1);
    mbar_init(sh.bar(C::kBarDrain), 1);
    mbar_init(sh.bar(C::kBarDrain1), 1);
    *sh.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int2* rg = ranges + wi.range0;

  if (warp < 4) {
    // warpgroup 0 returns registers at one program point (all four warps), then splits into its roles
    regs_dec<kBwdRegsLow>();
    if (wi.n_tiles > 0) {
      if (warp == 0) {
        if (elect_one()) {
          if (dkv) bwd_produce_dkv<D>(sh, &tm_q, &tm_k, &tm_v, &tm_do, wi, rg, err);
          else bwd_produce_dq<D>(sh, &tm_k, &tm_v, &tm_do, wi, rg, err);
        }
      } else if (warp == 1) {
        if (elect_one()) {
          if (dkv) bwd_mma_dkv<D>(sh, tmem, wi, err);
          else bwd_mma_dq_scores<D>(sh, tmem, wi, err);
        }
      } else if (dkv) {
        bwd_prepare_dkv<D>(sh, wi, rg, stats, delta, nq, threadIdx.x - 64, err);
      } else if (warp == 2) {
        bwd_prepare_dq<D>(sh, wi, rg, threadIdx.x - 64, err);
      } else if (elect_one()) {
        bwd_mma_dq_acc<D>(sh, tmem, wi, err);
      }
    }
  } else {
    regs_inc<kBwdRegsHigh>();
    const BwdThread th(warp - 4, lane);
    if (wi.n_tiles == 0) {
      if (dkv) {
        bwd_zero<D>(th, wi, dk, heads);
        bwd_zero<D>(th, wi, dv, heads);
      } else {
        bwd_zero<D>(th, wi, dq, heads);
      }
    } else if (dkv) {
      bwd_compute_dkv<D>(sh, tmem, th, wi, scale, dk, dv, heads, err);
    } else {
      bwd_compute_dq<D>(sh, tmem, th, wi, rg, scale, q, stats, dlse, delta, nq, dq, heads, err);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------- row statistics
// stats[h][row] = (lse * log2 e, sum_d dO o - dL), and delta[h][row] marked as pending, the ticket as undrawn. Memory
// bound: dO and o are read once, 16 bytes per thread, D / 8 lanes per (row, head); a block covers 32 rows x 8 heads and
// writes its pairs through shared memory, so that the head-major statistics are written in runs of 32 rows.
template <int D>
__global__ void __launch_bounds__(256) attn_bwd_stats_kernel(const __nv_bfloat16* __restrict__ out,
                                                             const __nv_bfloat16* __restrict__ dout,
                                                             const float* __restrict__ lse,
                                                             const float* __restrict__ dlse,
                                                             float2* __restrict__ stats, float* __restrict__ pending,
                                                             int* __restrict__ ticket, long long nq, int heads) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *ticket = 0;
  constexpr int kLanes = D / 8;                 // lanes per (row, head)
  constexpr int kPer = 256 / kLanes;            // (row, head) pairs per pass: 8 heads x kPer / 8 rows
  __shared__ float delta[8][33];
  const int t = threadIdx.x, g = t / kLanes, l = t % kLanes;
  const long long row0 = 32ll * blockIdx.x;
  const int h0 = 8 * blockIdx.y;
  const int h = h0 + g % 8;
#pragma unroll
  for (int i = 0; i < 32 / (kPer / 8); ++i) {
    const int r = i * (kPer / 8) + g / 8;
    const long long row = row0 + r;
    float sum = 0.f;
    if (row < nq && h < heads) {
      const long long at = (row * heads + h) * D + 8 * l;
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(out + at));
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(dout + at));
      const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[e]));
        const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y[e]));
        sum += u.x * v.x + u.y * v.y;
      }
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (l == 0) delta[g % 8][r] = sum;
  }
  __syncthreads();
  const int hh = h0 + (t >> 5);
  const long long row = row0 + (t & 31);
  if (hh < heads && row < nq) {
    const long long at = static_cast<long long>(hh) * nq + row;
    float d = delta[t >> 5][t & 31];
    if (dlse != nullptr) d -= dlse[at];
    stats[at] = make_float2(lse[at] * kLog2e, d);
    pending[at] = __uint_as_float(kDeltaPending);
  }
}

// ------------------------------------------------------------------------------------------------ host side

template <int D>
static int launch_attn_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout,
                           const float* lse, const float* dlse, void* dq, void* dk, void* dv, long long nq,
                           long long nk, int heads, float scale, const BwdWork* work, int n_items, const int2* ranges,
                           float* scratch, int* err, cudaStream_t stream, const int* n_items_dev) {
  using C = BwdCfg<D>;
  // an empty side has no tiles to load: its maps only need a valid address
  if (nk == 0) k = v = q;
  if (nq == 0) q = dout = k;
  const long long rq = nq > 0 ? nq : nk, rk = nk > 0 ? nk : nq;
  CUtensorMap mq, mk, mv, mdo;
  const long long w = static_cast<long long>(heads) * D;
  int rc;
  if ((rc = make_rows_map(&mq, q, rq, w, w, 64)) != ORL_OK) return rc;
  if ((rc = make_rows_map(&mdo, dout, rq, w, w, 64)) != ORL_OK) return rc;
  if ((rc = make_rows_map(&mk, k, rk, w, w, 64)) != ORL_OK) return rc;
  if ((rc = make_rows_map(&mv, v, rk, w, w, 64)) != ORL_OK) return rc;
  static std::mutex mu;
  static bool attr_set[kMaxDevices] = {};
  static int launch_regs = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return ORL_ERR_LAUNCH;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!attr_set[dev]) {
      if (cudaFuncSetAttribute(attn_bwd_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) !=
          cudaSuccess)
        return ORL_ERR_LAUNCH;
      cudaFuncAttributes fa{};
      if (cudaFuncGetAttributes(&fa, attn_bwd_kernel<D>) != cudaSuccess) return ORL_ERR_LAUNCH;
      launch_regs = fa.numRegs;
      attr_set[dev] = true;
    }
  }
  // as in the forward: a build with another register count could leave the split's increase waiting, so it never runs
  if (launch_regs != kBwdLaunchRegs) return ORL_ERR_UNSUPPORTED;
  // scratch: the ticket (16 bytes), the pairs, delta
  int* ticket = reinterpret_cast<int*>(scratch);
  float2* stats = reinterpret_cast<float2*>(scratch + 4);
  float* delta = scratch + 4 + 2 * static_cast<long long>(heads) * nq;
  const dim3 grid(static_cast<unsigned>(std::max<long long>(1, (nq + 31) / 32)), static_cast<unsigned>((heads + 7) / 8));
  attn_bwd_stats_kernel<D><<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(out),
                                                     static_cast<const __nv_bfloat16*>(dout), lse, dlse, stats, delta,
                                                     ticket, nq, heads);
  if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
  attn_bwd_kernel<D><<<n_items, kBwdThreads, C::kSmemBytes, stream>>>(
      mq, mk, mv, mdo, static_cast<const __nv_bfloat16*>(q), work, ranges, stats, delta, ticket, dlse,
      static_cast<__nv_bfloat16*>(dq), static_cast<__nv_bfloat16*>(dk),
      static_cast<__nv_bfloat16*>(dv), nq, heads, scale, err, n_items_dev);
  return cudaGetLastError() == cudaSuccess ? ORL_OK : ORL_ERR_LAUNCH;
}

static bool bwd_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int check_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout, const float* lse,
                     void* dq, void* dk, void* dv, long long nq, long long nk, int heads, int head_dim, float scale,
                     const void* stats, const int* err) {
  if (nq < 0 || nk < 0 || nq > 0x7fffffffLL || nk > 0x7fffffffLL || heads <= 0 || !(scale > 0.f) || err == nullptr)
    return ORL_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return ORL_ERR_UNSUPPORTED;
  if (static_cast<long long>(heads) * head_dim > 0x7fffffffLL) return ORL_ERR_ARG;
  if (stats == nullptr) return ORL_ERR_ARG;
  if (nq > 0 && (q == nullptr || out == nullptr || dout == nullptr || lse == nullptr || dq == nullptr))
    return ORL_ERR_ARG;
  if (nk > 0 && (k == nullptr || v == nullptr || dk == nullptr || dv == nullptr)) return ORL_ERR_ARG;
  for (const void* p : {q, k, v, out, dout, static_cast<const void*>(dq), static_cast<const void*>(dk),
                        static_cast<const void*>(dv), stats})
    if (!bwd_aligned(p)) return ORL_ERR_ALIGN;
  return ORL_OK;
}

// Work list of the backward, on the host. Key rows are cut at every start and end of a segment's keys: inside one of
// the resulting intervals all rows are read by the same segments.
struct BwdPlan {
  std::vector<BwdWork> items;
  std::vector<int2> ranges;
};

static int plan_bwd(const int32_t* q_start, const int32_t* q_len, const int32_t* k_start, const int32_t* k_len,
                    int n_seg, int heads, long long nq, long long nk, BwdPlan& plan) {
  struct Block {
    int row0, rows, kind, range0, n_ranges, n_tiles, whole;
  };
  std::vector<Block> blocks;
  std::vector<int> by_q;                                  // segments with query rows, by first row
  for (int i = 0; i < n_seg; ++i) {
    if (q_len[i] < 0 || k_len[i] < 0 || q_start[i] < 0 || k_start[i] < 0) return ORL_ERR_ARG;
    if (static_cast<long long>(q_start[i]) + q_len[i] > nq || static_cast<long long>(k_start[i]) + k_len[i] > nk)
      return ORL_ERR_ARG;
    if (q_len[i] > 0) by_q.push_back(i);
  }
  auto cut = [&](long long lo, long long hi, int kind, int range0, int n_ranges, int n_tiles, bool whole) {
    for (long long r = lo; r < hi; r += 128)
      blocks.push_back({static_cast<int>(r), static_cast<int>(std::min<long long>(128, hi - r)), kind, range0, n_ranges,
                        n_tiles, whole ? 1 : 0});
  };
  // queries: one range of keys per segment; rows of no segment get zeros
  std::sort(by_q.begin(), by_q.end(), [&](int a, int b) { return q_start[a] < q_start[b]; });
  long long at = 0;
  for (int i : by_q) {
    if (q_start[i] < at) return ORL_ERR_ARG;              // two segments share a query row
    cut(at, q_start[i], kDq, 0, 0, 0, false);
    plan.ranges.push_back({k_start[i], k_len[i]});
    cut(q_start[i], static_cast<long long>(q_start[i]) + q_len[i], kDq, static_cast<int>(plan.ranges.size()) - 1, 1,
        (k_len[i] + kDqRows - 1) / kDqRows, k_len[i] > 0 && k_len[i] <= kWholeKeys);
    at = static_cast<long long>(q_start[i]) + q_len[i];
  }
  cut(at, nq, kDq, 0, 0, 0, false);
  // keys: the elementary intervals, each with the query ranges of the segments that cover it (in segment order)
  std::vector<long long> cuts = {0, nk};
  for (int i = 0; i < n_seg; ++i)
    if (q_len[i] > 0 && k_len[i] > 0) {
      cuts.push_back(k_start[i]);
      cuts.push_back(static_cast<long long>(k_start[i]) + k_len[i]);
    }
  std::sort(cuts.begin(), cuts.end());
  cuts.erase(std::unique(cuts.begin(), cuts.end()), cuts.end());
  for (size_t c = 0; c + 1 < cuts.size(); ++c) {
    const int range0 = static_cast<int>(plan.ranges.size());
    int n = 0;
    long long tiles = 0;
    for (int i = 0; i < n_seg; ++i)
      if (q_len[i] > 0 && k_len[i] > 0 && k_start[i] <= cuts[c] &&
          static_cast<long long>(k_start[i]) + k_len[i] >= cuts[c + 1]) {
        plan.ranges.push_back({q_start[i], q_len[i]});
        tiles += (q_len[i] + kDkvRows - 1) / kDkvRows;
        ++n;
      }
    if (tiles > 0x7fffffffLL || plan.ranges.size() > 0x7ffffff0u) return ORL_ERR_CAPACITY;
    cut(cuts[c], cuts[c + 1], kDkv, range0, n, static_cast<int>(tiles), false);
  }
  // the queries' items first (the keys' wait for their delta), longest first
  std::vector<int> order(blocks.size());
  for (size_t i = 0; i < order.size(); ++i) order[i] = static_cast<int>(i);
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) {
    const Block &x = blocks[a], &y = blocks[b];
    return x.kind != y.kind ? x.kind == kDq : x.n_tiles > y.n_tiles;
  });
  if (static_cast<long long>(blocks.size()) * heads > 0x3fffffffLL) return ORL_ERR_CAPACITY;
  plan.items.reserve(blocks.size() * heads);
  for (size_t lo = 0; lo < order.size();) {
    // blocks of the same kind and ranges: head by head, so that concurrent CTAs share the streamed tiles in L2
    size_t hi = lo + 1;
    auto same = [&](const Block& a, const Block& b) {
      return a.kind == b.kind && a.range0 == b.range0 && a.n_ranges == b.n_ranges;
    };
    while (hi < order.size() && same(blocks[order[lo]], blocks[order[hi]])) ++hi;
    for (int h = 0; h < heads; ++h)
      for (size_t x = lo; x < hi; ++x) {
        const Block& b = blocks[order[x]];
        plan.items.push_back({b.row0, b.rows, h, b.kind, b.range0, b.n_ranges, b.n_tiles, b.whole});
      }
    lo = hi;
  }
  return ORL_OK;
}

}  // namespace orl

using namespace orl;

extern "C" int orl_attn_bwd_plan(const int32_t* q_start, const int32_t* q_len, const int32_t* k_start,
                                 const int32_t* k_len, int n_seg, int heads, long long nq, long long nk,
                                 orl_attn_bwd_work* work, int work_capacity, int32_t* ranges, int ranges_capacity,
                                 int* n_ranges) {
  if (n_seg < 0 || heads <= 0 || nq < 0 || nk < 0 || nq > 0x7fffffffLL || nk > 0x7fffffffLL || n_ranges == nullptr)
    return ORL_ERR_ARG;
  if (n_seg > 0 && (q_start == nullptr || q_len == nullptr || k_start == nullptr || k_len == nullptr))
    return ORL_ERR_ARG;
  try {
    BwdPlan plan;
    const int rc = plan_bwd(q_start, q_len, k_start, k_len, n_seg, heads, nq, nk, plan);
    if (rc != ORL_OK) return rc;
    const int n = static_cast<int>(plan.items.size());
    *n_ranges = static_cast<int>(plan.ranges.size());
    if (n == 0) return 0;
    if (work == nullptr || work_capacity < n || (ranges == nullptr && *n_ranges > 0) || ranges_capacity < *n_ranges)
      return -n - 1000;                                   // caller sizes the buffers
    std::copy(plan.items.begin(), plan.items.end(), work);
    for (int i = 0; i < *n_ranges; ++i) {
      ranges[2 * i] = plan.ranges[i].x;
      ranges[2 * i + 1] = plan.ranges[i].y;
    }
    return n;
  } catch (const std::bad_alloc&) {
    return ORL_ERR_CAPACITY;
  }
}

extern "C" int orl_attn_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout,
                            const float* lse, const float* dlse, void* dq, void* dk, void* dv, long long nq,
                            long long nk, int heads, int head_dim, float scale, const orl_attn_bwd_work* work_dev,
                            int n_items, const int32_t* ranges_dev, float* stats_dev, int* err_dev,
                            void* stream_ptr) {
  const int rc = check_bwd(q, k, v, out, dout, lse, dq, dk, dv, nq, nk, heads, head_dim, scale, stats_dev, err_dev);
  if (rc != ORL_OK) return rc;
  if (n_items < 0 || (n_items > 0 && work_dev == nullptr)) return ORL_ERR_ARG;
  if (n_items == 0) return ORL_OK;
  auto launch = head_dim == 64 ? launch_attn_bwd<64> : launch_attn_bwd<128>;
  return launch(q, k, v, out, dout, lse, dlse, dq, dk, dv, nq, nk, heads, scale, work_dev, n_items,
                reinterpret_cast<const int2*>(ranges_dev), stats_dev, err_dev,
                static_cast<cudaStream_t>(stream_ptr), nullptr);
}

// ------------------------------------------------------------------------------------------------ device plan
// orl_attn_bwd_cu: cu_seqlens on the device, the work list planned there. Keys of different segments do
// not overlap, so a segment's key rows have one query range and its query rows one key range: ranges[i] = segment
// i's query range, ranges[n_seg + i] its key range. Rows before the first and after the last segment get zeros.
// Every block ranks the segments for itself and writes its share of the items (one block took 30 us to write the 12000
// items of two scenes of 22000 rows and 16 heads).
// Scratch: a 32-byte header (slot 0: item count), the items, then the ranges.
namespace orl {

constexpr int kBwdPlanMaxSeg = 4096;

__global__ void __launch_bounds__(1024)
    attn_bwd_plan_kernel(const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k, int n_seg, int heads,
                         long long nq, long long nk, BwdWork* __restrict__ work, int2* __restrict__ ranges,
                         long long capacity, int* __restrict__ err) {
  // groups: n_seg dkv, n_seg dq, then the rows outside the segments (dkv before / after, dq before / after)
  extern __shared__ int plan_smem[];
  const int n_grp = 2 * n_seg + 4;
  int* s_row = plan_smem;                   // [n_grp] first row
  int* s_len = s_row + n_grp;               // [n_grp] rows
  int* s_tiles = s_len + n_grp;             // [n_grp] streamed tiles
  int* s_grp = s_tiles + n_grp;             // [n_grp] group at each rank
  int* s_end = s_grp + n_grp;               // [n_grp] end of each rank's items
  __shared__ int bad, total, n_ranked;
  const int t = threadIdx.x;
  if (t == 0) bad = total = n_ranked = 0;
  __syncthreads();
  for (int i = t; i < n_seg; i += blockDim.x) {
    const long long q0 = cu_q[i], q1 = cu_q[i + 1], k0 = cu_k[i], k1 = cu_k[i + 1];
    if (q0 < 0 || q1 < q0 || q1 > nq || k0 < 0 || k1 < k0 || k1 > nk) bad = 1;
    const int lq = static_cast<int>(q1 - q0), lk = static_cast<int>(k1 - k0);
    s_row[i] = static_cast<int>(k0);
    s_len[i] = lk;
    s_tiles[i] = (lq + kDkvRows - 1) / kDkvRows;
    s_row[n_seg + i] = static_cast<int>(q0);
    s_len[n_seg + i] = lq;
    s_tiles[n_seg + i] = (lk + kDqRows - 1) / kDqRows;
    if (blockIdx.x == 0) {
      ranges[i] = make_int2(static_cast<int>(q0), lq);
      ranges[n_seg + i] = make_int2(static_cast<int>(k0), lk);
    }
  }
  if (t < 4) {
    const int32_t* cu = t < 2 ? cu_k : cu_q;
    const long long n = t < 2 ? nk : nq;
    const int first = cu[0], last = cu[n_seg];
    if (first < 0 || first > n || last < 0 || last > n) bad = 1;
    const int lo = (t & 1) ? last : 0;
    s_row[2 * n_seg + t] = lo;
    s_len[2 * n_seg + t] = (t & 1) ? static_cast<int>(n - lo) : first;
    s_tiles[2 * n_seg + t] = 0;
  }
  __syncthreads();
  if (bad) {
    if (t == 0 && blockIdx.x == 0) {
      work[0].row0 = 0;
      atomicOr(err, kErrPlan);
    }
    return;
  }
  auto is_dkv = [&](int g) { return g < n_seg || (g >= 2 * n_seg && g < 2 * n_seg + 2); };
  // the queries' items first (the keys' wait for their delta), longest first
  auto cost = [&](int g) { return static_cast<long long>(s_tiles[g]) + (is_dkv(g) ? 0 : 1ll << 32); };
  auto items = [&](int g) { return heads * ((s_len[g] + 127) >> 7); };
  for (int g = t; g < n_grp; g += blockDim.x) {
    if (s_len[g] == 0) continue;
    const long long cg = cost(g);
    int rank = 0, before = 0;
    for (int x = 0; x < n_grp; ++x) {
      if (s_len[x] == 0) continue;
      const long long cx = cost(x);
      if (cx > cg || (cx == cg && x < g)) {
        ++rank;
        before += items(x);
      }
    }
    s_grp[rank] = g;
    s_end[rank] = before + items(g);
    atomicAdd(&n_ranked, 1);
    atomicAdd(&total, items(g));
  }
  __syncthreads();
  const int n = total, m = n_ranked;
  if (static_cast<long long>(n) + 1 > capacity) {
    if (t == 0 && blockIdx.x == 0) {
      work[0].row0 = 0;
      atomicOr(err, kErrPlan);
    }
    return;
  }
  for (int it = blockIdx.x * blockDim.x + t; it < n; it += gridDim.x * blockDim.x) {
    int lo = 0, hi = m - 1;                 // first rank whose items end after it
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_end[mid] > it) hi = mid; else lo = mid + 1;
    }
    const int g = s_grp[lo];
    const int chunks = (s_len[g] + 127) >> 7;
    const int r = it - (lo > 0 ? s_end[lo - 1] : 0);
    const int h = r / chunks, c = r - h * chunks;
    BwdWork w;
    w.row0 = s_row[g] + 128 * c;
    w.rows = min(128, s_len[g] - 128 * c);
    w.head = h;
    w.kind = is_dkv(g) ? kDkv : kDq;
    w.range0 = g < 2 * n_seg ? g : 0;
    w.n_ranges = s_tiles[g] > 0 ? 1 : 0;
    w.n_tiles = s_tiles[g];
    const int keys = g >= n_seg && g < 2 * n_seg ? s_len[g - n_seg] : 0;
    w.whole = keys > 0 && keys <= kWholeKeys ? 1 : 0;
    work[1 + it] = w;
  }
  if (t == 0 && blockIdx.x == 0) work[0].row0 = n;
}

}  // namespace orl

extern "C" long long orl_attn_bwd_cu_scratch(long long nq, long long nk, int n_seg, int heads) {
  if (nq < 0 || nk < 0 || n_seg < 0 || heads <= 0) return ORL_ERR_ARG;
  // every group of rows may end in a short block: n_seg + 2 groups on each side
  const long long items = heads * ((nq + 127) / 128 + (nk + 127) / 128 + 2ll * (n_seg + 2));
  return 32 * (1 + items) + 16ll * n_seg;
}

extern "C" int orl_attn_bwd_cu(const void* q, const void* k, const void* v, const void* out, const void* dout,
                               const float* lse, const float* dlse, void* dq, void* dk, void* dv, long long nq,
                               long long nk, int heads, int head_dim, float scale, const int32_t* cu_q_dev,
                               const int32_t* cu_k_dev, int n_seg, void* scratch_dev, long long scratch_bytes,
                               float* stats_dev, int* err_dev, void* stream_ptr) {
  const int rc = check_bwd(q, k, v, out, dout, lse, dq, dk, dv, nq, nk, heads, head_dim, scale, stats_dev, err_dev);
  if (rc != ORL_OK) return rc;
  if (n_seg < 0 || cu_q_dev == nullptr || cu_k_dev == nullptr || scratch_dev == nullptr) return ORL_ERR_ARG;
  if (!bwd_aligned(scratch_dev)) return ORL_ERR_ALIGN;
  if (n_seg > kBwdPlanMaxSeg) return ORL_ERR_CAPACITY;
  const long long need = orl_attn_bwd_cu_scratch(nq, nk, n_seg, heads);
  if (scratch_bytes < need) return ORL_ERR_CAPACITY;
  const long long items = (need - 32 - 16ll * n_seg) / 32;
  if (items > 0x3fffffffLL) return ORL_ERR_CAPACITY;
  if (nq == 0 && nk == 0) return ORL_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const int smem = 20 * (2 * n_seg + 4);
  static std::mutex mu;
  static bool attr_set[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return ORL_ERR_LAUNCH;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!attr_set[dev]) {
      if (cudaFuncSetAttribute(attn_bwd_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               20 * (2 * kBwdPlanMaxSeg + 4)) != cudaSuccess)
        return ORL_ERR_LAUNCH;
      attr_set[dev] = true;
    }
  }
  BwdWork* work = static_cast<BwdWork*>(scratch_dev);
  int2* ranges = reinterpret_cast<int2*>(work + 1 + items);
  const int blocks = static_cast<int>(std::min<long long>(64, (items + 1023) / 1024));
  attn_bwd_plan_kernel<<<blocks, 1024, smem, stream>>>(cu_q_dev, cu_k_dev, n_seg, heads, nq, nk, work, ranges, 1 + items,
                                                  err_dev);
  if (cudaGetLastError() != cudaSuccess) return ORL_ERR_LAUNCH;
  auto launch = head_dim == 64 ? launch_attn_bwd<64> : launch_attn_bwd<128>;
  return launch(q, k, v, out, dout, lse, dlse, dq, dk, dv, nq, nk, heads, scale, work + 1, static_cast<int>(items),
                ranges, stats_dev, err_dev, stream, reinterpret_cast<const int*>(work));
}
