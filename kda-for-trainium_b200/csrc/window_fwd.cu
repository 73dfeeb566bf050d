// Forward of the sliding-window attention with sinks (head_dim 128, bf16) on
// tcgen05.  Query i sees key j <= i where i - j < window or j < sinks:
//   S = Q K^T,  P = 2^(S scale log2e - m),  O = P V / rowsum(P)
// with m a running reference of each row's scores: it only moves when a score
// exceeds it by more than 2^8, because weights up to 256 are as exact in bf16
// and their sum in fp32 as weights up to 1.
//
// Work unit = (batch, query head, 256 query rows as two 128-row tiles); one
// persistent CTA per SM.  Per unit the K and V blocks of its window (and those
// with sinks before it) pass through a 3-slot TMA ring, K_0, K_1, V_0, K_2, V_1,
// ..., and serve both tiles.  A tile skips the blocks that none of its rows sees.
//
// 640 threads: warp 0 TMA producer, warp 1 MMA issuer of S (allocates TMEM), warp 3
// of P V, warps 4-11 / 12-19 softmax of tile 0 / 1: warp w reads TMEM lanes
// 32 (w % 4), 64 of a row's 128 keys per thread.
// P stays in TMEM, as bf16, and is the P V product's A operand there: 64 KB a step
// of two tiles that are neither stored to shared memory nor read back from it (the
// TMEM operand beside shared-memory ones runs at the full rate: 2,048 cycles for
// the step's four products).  With P's columns of their own, one region is left for
// S, which the tiles take in turn: S_0(j), S_1(j), S_0(j+1), ...; a tile's S is
// issued as soon as the other has copied its S into registers, so the tiles run
// half a step apart and one exponentiates while the other stores.  An issuer's wait
// stalls behind its own queued MMAs, hence one for S and one for P V: neither's next
// wait ends before its last product anyway.
// The two warps that share a row agree on its reference with one bar.red a step
// (did a score exceed it?) and exchange maxima only when one did.
// V is read as stored (MN-major B).
// TMEM columns: S [0,128), P_0 [128,192), P_1 [192,256), O_0 [256,384), O_1 [384,512).
// Shared memory: Q_0 | Q_1 | outgoing O_0 | O_1 | ring (3 x 32 KB) | row exchange.
// 1.16 ms at S32768 W2048 of 32 heads (1.07 TFLOP on visible pairs: 923 TFLOP/s, 0.54
// of the measured bf16 rate; 1.14 to 1.19 from box to box): a step of two tiles takes about 3,250 cycles, of
// which the tensor core works 2,048 and the exponentials' pipe 2,048; the rest is the
// latency of a tile's chain (wait, TMEM load, maximum, exponentials, store).  With P
// through shared memory, S_t of each tile its own: 1.43 ms.  One of eight pairs by
// a polynomial instead of ex2: 1 % faster, one of four 4 % slower; not kept.  One
// tile a unit for calls that leave SMs idle: no faster.
// All mbarrier waits are bounded (common.cuh); every TMA load targets one CTA.
#include <math.h>

#include "launch.cuh"
#include "window.cuh"

KDA_DEFINE_ERROR_WORD(window_fwd)

namespace kda {
namespace {

constexpr int kSlots = 3;
constexpr int kRowWarps = 16;
constexpr int kThreads = 128 + 32 * kRowWarps;
// Registers per thread: at launch (what the compiler reports for 640 threads), and
// after the control warpgroup has given some to the four of row warps.
constexpr int kRegsLaunch = 96, kRegsCtl = 64, kRegsRow = 104;
static_assert(128 * kRegsCtl + 32 * kRowWarps * kRegsRow <= kThreads * kRegsLaunch, "register split");
constexpr int kPairBarrier = 2;  // named barriers 2 .. 9: the two warps of a (tile, 32 rows)
constexpr int kHalfBarrier = 10;  // 10 .. 13: the four warps of a (tile, 64 columns)

struct FwdParams {
  int B, S, QH, KH, rep;
  int npairs;  // 256-row units per head
  int window, sinks;
  float scale_log2;  // softmax scale * log2(e)
  float* lse;        // [B][QH][S] or null: each row's log2-sum-exp of the scaled scores
};

struct Smem {
  static constexpr uint32_t kQ = 0, kOut = 2 * kTile, kRing = 4 * kTile;
  static constexpr uint32_t kExchange = 7 * kTile;  // 1 KB, fp32 [tile][row]: maxima and sums of two warps' halves
  static constexpr uint32_t kBars = kExchange + 1024;
  static constexpr uint32_t kNumBars = 24;
  static constexpr size_t kBytes = 1024 + kBars + kNumBars * 8;
  static_assert(kBytes > 116 * 1024 && kBytes <= 227 * 1024, "shared memory budget");
};

// A unit and the key blocks it visits: [0, ns) (sinks), then [ns + skip, nb + skip).
struct Unit {
  int b, h, q0;
  int nb, ns, skip;
};
__device__ __forceinline__ Unit unit_at(const FwdParams& p, int u) {
  const int heads = p.B * p.QH;
  const int level = u / heads, bh = u - level * heads;
  const int qp = p.npairs - 1 - level;  // the last units, which see the most, first
  Unit c;
  c.b = bh / p.QH;
  c.h = bh - c.b * p.QH;
  c.q0 = qp * 2 * kBlk;
  const int all = (p.S + kBlk - 1) / kBlk;
  const int last = min(2 * qp + 2, all);
  const int first = max(0, c.q0 - p.window + 1) / kBlk;
  c.ns = min((p.sinks + kBlk - 1) / kBlk, first);
  c.nb = c.ns + last - first;
  c.skip = first - c.ns;
  return c;
}
__device__ __forceinline__ int key_block(const Unit& c, int j) { return j < c.ns ? j : j + c.skip; }
// The unit's blocks that any row of a tile sees: j < sinks and from <= j < to.
struct Seen {
  int sinks, from, to;
  __device__ __forceinline__ bool at(int j) const { return j < sinks || (j >= from && j < to); }
};
__device__ __forceinline__ Seen tile_sees(const FwdParams& p, const Unit& c, int t) {
  const int q0 = c.q0 + t * kBlk;
  if (q0 >= p.S) return {0, 0, 0};
  const int first = max(0, q0 - p.window + 1) / kBlk;  // >= the unit's, which goes by tile 0
  // blocks [0, sink blocks) of key order that lie in the walk: those before ns, and
  // where the window reaches down to them, the ones from ns on
  const int sinks = (p.sinks + kBlk - 1) / kBlk, to = q0 / kBlk + 1 - c.skip;
  return {min(max(c.ns, sinks - c.skip), to), max(first, c.ns + c.skip) - c.skip, to};
}

// Ring items of a unit: K_0, K_1, V_0, K_2, V_1, ..., K_{nb-1}, V_{nb-2}, V_{nb-1};
// `base` counts the items of earlier units.  Item x lives in slot x % 3.
__device__ __forceinline__ uint32_t item_k(uint32_t base, int j) {
  return base + (j == 0 ? 0u : 2u * static_cast<uint32_t>(j) - 1u);
}
__device__ __forceinline__ uint32_t item_v(uint32_t base, int j, int nb) {
  return base + (j == nb - 1 ? 2u * static_cast<uint32_t>(nb) - 1u : 2u * static_cast<uint32_t>(j) + 2u);
}
__device__ __forceinline__ uint32_t item_slot(uint32_t x) { return x % kSlots; }
__device__ __forceinline__ uint32_t item_par(uint32_t x) { return (x / kSlots) & 1u; }

__global__ void __launch_bounds__(kThreads, 1)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                      const FwdParams p, unsigned* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem::kBars);
  uint64_t* slot_full = bars;      // [2][2] the nth K, the nth V landed: at n % 2 (each issuer waits for its own in turn)
  uint64_t* slot_free = bars + 4;  // [3] the MMAs that read it are done
  uint64_t* s_free = bars + 9;     // S copied out (8 warps); one phase per S, of either tile
  // [2], per tile; one phase per block that the tile sees
  uint64_t* s_ready = bars + 7;    // S in TMEM
  uint64_t* p_ready = bars + 11;   // P in TMEM (8 warps)
  uint64_t* pv_done = bars + 13;   // O += P V done
  // [2], one phase per unit in which the tile has rows
  uint64_t* o_free = bars + 15;    // O read out (8 warps)
  uint64_t* q_full = bars + 19;    // Q landed
  uint64_t* drain = bars + 17;     // [2] once
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 21);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 21; ++i) {
      const bool rows = i == 9 || i == 11 || i == 12 || i == 15 || i == 16;
      mbar_init(bars + i, rows ? kRowWarps / 2 : 1);
    }
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmO);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();  // the next launch may start
  pdl_wait();     // the one before is done
  const uint32_t tmem = *tmem_holder;
  const int units = p.B * p.QH * p.npairs;

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsCtl));
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      bool ok = true;
      uint32_t base = 0, loads[2] = {0u, 0u};  // items of earlier units; loads of K and V issued
      int qs[2] = {0, 0};
      uint32_t seen[2] = {0u, 0u};   // blocks each tile has seen
      auto load_item = [&](const int kv, uint32_t x, const CUtensorMap* m, int g, int j, int b) -> bool {
        const uint32_t s = item_slot(x);
        uint64_t* full = &slot_full[2 * kv + (loads[kv] & 1u)];
        if (x >= kSlots && !mbar_wait(&slot_free[s], item_par(x) ^ 1u, err, kErrWaitEmpty)) return false;
        mbar_arrive_expect_tx(full, kTile);
        load_tile(smem + Smem::kRing + s * kTile, m, full, g, j * kBlk, b);
        ++loads[kv];
        return true;
      };
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const Unit c = unit_at(p, u);
        const int g = c.h / p.rep;
        const Seen sees[2] = {tile_sees(p, c, 0), tile_sees(p, c, 1)};
        // Q of a tile that has rows, once its last S is done
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (sees[t].to > 0) {
            if (ok && seen[t] > 0) ok = mbar_wait(&s_ready[t], (seen[t] - 1u) & 1u, err, kErrWaitEmpty);
            if (!ok) break;
            mbar_arrive_expect_tx(&q_full[t], kTile);
            load_tile(smem + Smem::kQ + t * kTile, &tmQ, &q_full[t], c.h, c.q0 + t * kBlk, c.b);
            ++qs[t];
          }
        if (!ok) break;
        ok = load_item(0, item_k(base, 0), &tmK, g, key_block(c, 0), c.b);
        for (int j = 0; j < c.nb && ok; ++j) {
          if (j + 1 < c.nb) ok = load_item(0, item_k(base, j + 1), &tmK, g, key_block(c, j + 1), c.b);
          if (ok) ok = load_item(1, item_v(base, j, c.nb), &tmV, g, key_block(c, j), c.b);
#pragma unroll
          for (int t = 0; t < 2; ++t) seen[t] += sees[t].at(j) ? 1u : 0u;
        }
        base += 2u * static_cast<uint32_t>(c.nb);
      }
      // no copy may still be writing shared memory when the CTA exits
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (qs[t] > 0) mbar_drain(&q_full[t], static_cast<uint32_t>(qs[t] - 1) & 1u);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t uses = (loads[i >> 1] + 1u - (i & 1u)) >> 1;
        if (uses > 0) mbar_drain(&slot_full[i], (uses - 1u) & 1u);
      }
    }
    __syncwarp();
  } else if (warp < 4) {
    // ------------------------------- MMA issuers: S (warp 1) and P V (warp 3)
    if (warp == 1 || warp == 3) {
      const bool one = elect_one();
      const uint32_t ring = smem_u32(smem) + Smem::kRing, qs = smem_u32(smem) + Smem::kQ;
      const bool is_s = warp == 1;
      uint32_t base = 0;           // ring items of earlier units
      uint32_t items = 0;          // K (or V) so far
      uint32_t ns = 0;             // S so far, of both tiles
      uint32_t np[2] = {0u, 0u};   // a tile's P V so far
      uint32_t un[2] = {0u, 0u};   // and its units
      bool ok = true, any = false;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const Unit c = unit_at(p, u);
        const Seen sees[2] = {tile_sees(p, c, 0), tile_sees(p, c, 1)};
        bool begins[2] = {true, true};
        for (int j = 0; j < c.nb && ok; ++j) {
          const uint32_t x = is_s ? item_k(base, j) : item_v(base, j, c.nb), slot = item_slot(x);
          const uint32_t tile = ring + slot * kTile;
          bool seen = false;
          ok = warp_wait(&slot_full[(is_s ? 0 : 2) + (items & 1u)], (items >> 1) & 1u, err, kErrWaitFull);
          ++items;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || !sees[t].at(j)) continue;
            if (is_s) {  // Q landed, the last S copied out
              if (begins[t]) ok = warp_wait(&q_full[t], un[t] & 1u, err, kErrWaitFull);
              if (ok && ns > 0) ok = warp_wait(s_free, (ns - 1u) & 1u, err, kErrWaitAccumFree);
              if (!ok) continue;
              tc_fence_after();
              if (one) {
                mma_kk(tmem, qs + t * kTile, tile);
                umma_commit(&s_ready[t]);
              }
              ++ns;
            } else {  // P written, the last unit's O read
              ok = warp_wait(&p_ready[t], np[t] & 1u, err, kErrWaitFull);
              if (ok && begins[t] && un[t] > 0) ok = warp_wait(&o_free[t], (un[t] - 1u) & 1u, err, kErrWaitAccumFree);
              if (!ok) continue;
              tc_fence_after();
              if (one) {
                mma_tm(tmem + 256 + t * kBlk, tmem + 128 + t * 64, tile, begins[t]);
                umma_commit(&pv_done[t]);
              }
              ++np[t];
            }
            un[t] += begins[t] ? 1u : 0u;
            begins[t] = false;
            seen = any = true;
          }
          if (one && seen) umma_commit(&slot_free[slot]);  // once this thread's MMAs have read the item
          else if (one && ok) mbar_arrive(&slot_free[slot]);
        }
        base += 2u * static_cast<uint32_t>(c.nb);
      }
      if (one && any) {
        // every issued MMA must finish before TMEM is released
        umma_commit(&drain[is_s ? 0 : 1]);
        mbar_drain(&drain[is_s ? 0 : 1], 0u);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsRow));
    const int t = (warp - 4) >> 3;          // tile
    const int half = ((warp - 4) >> 2) & 1;  // keys (and columns of O) [64 half, + 64)
    const int quad = warp & 3;
    const int r = quad * 32 + lane;  // query row of this thread (TMEM lane)
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t scol = lanes + 64 * half;
    const uint32_t pcol = lanes + 128 + 64 * t + 32 * half;
    const uint32_t ocol = lanes + 256 + t * kBlk + 64 * half;
    uint8_t* tile = smem + Smem::kOut + t * kTile + half * kHalf;
    const uint32_t row = smem_u32(tile) + static_cast<uint32_t>(r * 128);
    const uint32_t rsw = static_cast<uint32_t>(r & 7);
    float* xch = reinterpret_cast<float*>(smem + Smem::kExchange) + t * kBlk + r;
    const int pair = kPairBarrier + t * 4 + quad, quarter = kHalfBarrier + t * 2 + half;
    const bool elected = quad == 0 && lane == 0;  // issues this (tile, half)'s output
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    uint32_t n = 0;   // blocks seen so far
    bool ok = true, stored = false;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const Unit c = unit_at(p, u);
      const int qpos = c.q0 + t * kBlk + r;
      if (c.q0 + t * kBlk >= p.S) continue;  // no rows (both halves alike)
      const Seen sees = tile_sees(p, c, t);
      if (stored) {  // the last unit's output has left its tile
        if (elected) bulk_wait_read_all();
        ok = bar_and(quarter, 128, ok);
        if (!ok) break;
      }
      float m = -INFINITY, l = 0.f;
      bool first = true;
      // A wait that expires does not leave the loop by itself: its warp meets its
      // partner at the next pair barrier (or the unit's end) and both leave there.
      bool s_there = false;  // S is known to be ready
      for (int j = sees.sinks > 0 ? 0 : sees.from; j < sees.to; j = j + 1 >= sees.sinks ? max(j + 1, sees.from) : j + 1) {
        const uint32_t par = n & 1u;
        const int k0 = key_block(c, j) * kBlk + 64 * half;  // this thread's first key
        if (ok && !s_there) ok = warp_wait(&s_ready[t], par, err, kErrWaitAccum);
        tc_fence_after();
        uint32_t s[64];
        tmem_ld_32x32b_x32(scol, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_ld_32x32b_x32(scol + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
        tmem_ld_wait();
        tc_fence_before();
        if (ok) mbar_arrive_warp(s_free);
        // keys [k0, k0 + hi) are not after the query; of those, keys before k0 + old
        // only as sinks.  The test is on the tile's first and last row: most blocks
        // are visible whole.
        const int q0 = c.q0 + t * kBlk;
        if (k0 + 63 > q0 || (k0 + p.window < q0 + kBlk && k0 + 64 > p.sinks)) {
          const int hi = qpos + 1 - k0, old = qpos + 1 - p.window - k0, sink = min(hi, p.sinks - k0);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t live = range_mask(old - 32 * w, hi - 32 * w) | range_mask(0, sink - 32 * w);
            if (live != 0xffffffffu)
#pragma unroll
              for (int i = 0; i < 32; ++i) s[32 * w + i] = (live >> i) & 1u ? s[32 * w + i] : 0xff800000u;  // -inf
          }
        }
        float mx;
        {
          float a[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) a[k] = fmaxf(__uint_as_float(s[k]), __uint_as_float(s[k + 4]));
#pragma unroll
          for (int i = 8; i < 64; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = fmax3(a[k], __uint_as_float(s[i + k]), __uint_as_float(s[i + 4 + k]));
          mx = fmaxf(fmax3(a[0], a[1], a[2]), a[3]) * p.scale_log2;
        }
        // a score above the reference by 2^8 anywhere in these 32 rows (or a wait
        // that expired): both warps exchange their maxima and move the reference
        if (bar_or(pair, 64, !ok || mx > m + 8.f)) {
          if (half == 1) *xch = mx;
          ok = bar_and(pair, 64, ok);
          if (!ok) break;
          if (half == 0) *xch = fmaxf(m, fmaxf(mx, *xch));
          bar_sync(pair, 64);
          const float m_new = *xch;
          const float f = m_new == -INFINITY ? 1.f : exp2_approx(m - m_new);
          m = m_new;
          l *= f;
          if (!first) {
            // O += P V of the last block must be done before O is rescaled
            ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], par ^ 1u, err, kErrWaitAccum));
            if (ok) {
              tc_fence_after();
#pragma unroll 1
              for (int k = 0; k < 64; k += 16) {
                uint32_t o[16];
                tmem_ld_32x32b_x16(ocol + k, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st_32x32b_x16(ocol + k, o);
              }
              tmem_st_wait();
              tc_fence_before();
            }
          }
        }
        const bool p_free = first || __all_sync(0xffffffffu, mbar_test(&pv_done[t], par ^ 1u));
        const float mb = m == -INFINITY ? 0.f : m;
        const float2 nm2 = make_float2(-mb, -mb);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 a = __ffma2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), sc2, nm2);
          const float2 e = make_float2(exp2_approx(a.x), exp2_approx(a.y));
          sum[i & 1] = __fadd2_rn(sum[i & 1], e);
          s[i] = pack_bf16x2(e.x, e.y);  // the weights meet V as bf16, the tensor core's operand type
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        // P's columns are free once O += P V of the last block is done
        if (ok && !p_free) ok = warp_wait(&pv_done[t], par ^ 1u, err, kErrWaitAccum);
        if (ok) {
          tmem_st_32x32b_x16(pcol, *reinterpret_cast<const uint32_t(*)[16]>(&s[0]));
          tmem_st_32x32b_x16(pcol + 16, *reinterpret_cast<const uint32_t(*)[16]>(&s[16]));
          s_there = __all_sync(0xffffffffu, mbar_test(&s_ready[t], par ^ 1u));
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive_warp(&p_ready[t]);
        }
        first = false;
        ++n;
      }
      // O / l to bf16, through shared memory, out by TMA (rows past S are not written)
      if (ok) ok = mbar_wait(&pv_done[t], (n - 1u) & 1u, err, kErrWaitAccum);
      ok = bar_and(quarter, 128, ok);
      // the two halves' sums: half 1 hands its over, half 0 answers with the whole
      if (half == 1) *xch = l;
      ok = bar_and(pair, 64, ok);
      if (!ok) break;
      if (half == 0) {
        l += *xch;
        *xch = l;
        if (p.lse && qpos < p.S)
          p.lse[(static_cast<int64_t>(c.b) * p.QH + c.h) * p.S + qpos] = (m == -INFINITY ? 0.f : m) + __log2f(l);
      }
      bar_sync(pair, 64);
      if (half == 1) l = *xch;
      tc_fence_after();
      const float inv = 1.0f / l;
      uint32_t o[64];
      tmem_ld_32x32b_x32(ocol, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
      tmem_ld_32x32b_x32(ocol + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive_warp(&o_free[t]);
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = pack_bf16x2(__uint_as_float(o[8 * v + 2 * k]) * inv, __uint_as_float(o[8 * v + 2 * k + 1]) * inv);
        st_shared_v4(row + ((static_cast<uint32_t>(v) ^ rsw) << 4), w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async_smem();
      bar_sync(quarter, 128);
      if (elected) {
        tma_store_4d(&tmO, tile, 64 * half, c.h, c.q0 + t * kBlk, c.b);
        bulk_commit();
      }
      stored = true;
    }
    if (elected) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

}  // namespace

kda_status gqa_window_check(const char* op, int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, int64_t window,
                            int64_t sinks) {
  KDA_CHECK_ARG(B > 0 && S > 0 && QH > 0 && KH > 0 && QH % KH == 0, "%s: bad sizes B=%lld S=%lld QH=%lld KH=%lld", op,
                (long long)B, (long long)S, (long long)QH, (long long)KH);
  KDA_CHECK_ARG(window > 0 && sinks >= 0, "%s: window must be positive and sinks not negative, got %lld and %lld", op,
                (long long)window, (long long)sinks);
  KDA_CHECK_SUPPORTED(D == kD, "%s: head_dim must be 128, got %lld", op, (long long)D);
  KDA_CHECK_SUPPORTED(S < (1ll << 24) && QH <= 65535 && B <= 65535 && B * S < (1ll << 31) / QH,
                      "%s: too many rows (B=%lld S=%lld QH=%lld)", op, (long long)B, (long long)S, (long long)QH);
  return KDA_OK;
}

bool head_rows_ok(const void* p, const int64_t* s, int64_t n0, int64_t n1, int64_t n2) {
  const int64_t n[3] = {n0, n1, n2};
  bool ok = (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (n[i] == 1 || (s[i] >= 0 && s[i] % 8 == 0));
  return ok;
}

kda_status tmap_head_rows(CUtensorMap* m, const void* base, int64_t B, int64_t S, int64_t H, const int64_t* strides) {
  const uint64_t dims[4] = {static_cast<uint64_t>(kD), static_cast<uint64_t>(H), static_cast<uint64_t>(S),
                            static_cast<uint64_t>(B)};
  const uint64_t st[3] = {static_cast<uint64_t>(H > 1 ? strides[2] : kD) * 2,
                          static_cast<uint64_t>(S > 1 ? strides[1] : kD) * 2,
                          static_cast<uint64_t>(B > 1 ? strides[0] : kD) * 2};
  const uint32_t box[4] = {64, 1, static_cast<uint32_t>(kBlk), 1};
  return make_tmap_bf16(m, base, 4, dims, st, box);
}

}  // namespace kda

using namespace kda;

extern "C" kda_status kda_gqa_window_bf16(const void* q, const void* k, const void* v, void* out, float* lse,
                                          int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, int64_t window,
                                          int64_t sinks, const int64_t* q_strides, const int64_t* k_strides,
                                          const int64_t* v_strides, void* stream) {
  const char* op = "gqa_window";
  kda_status s;
  if ((s = gqa_window_check(op, B, S, QH, KH, D, window, sinks)) != KDA_OK) return s;
  KDA_CHECK_ARG(q && k && v && out && q_strides && k_strides && v_strides, "%s: null pointer", op);
  const int64_t dense[3] = {S * QH * kD, QH * kD, kD};
  KDA_CHECK_SUPPORTED(head_rows_ok(q, q_strides, B, S, QH) && head_rows_ok(k, k_strides, B, S, KH) &&
                          head_rows_ok(v, v_strides, B, S, KH) && head_rows_ok(out, dense, B, S, QH),
                      "%s: pointers and rows must be 16-byte aligned", op);
  FwdParams p{};
  p.B = static_cast<int>(B);
  p.S = static_cast<int>(S);
  p.QH = static_cast<int>(QH);
  p.KH = static_cast<int>(KH);
  p.rep = static_cast<int>(QH / KH);
  p.npairs = static_cast<int>((S + 2 * kBlk - 1) / (2 * kBlk));
  p.window = static_cast<int>(window < S ? window : S);
  p.sinks = static_cast<int>(sinks < S ? sinks : S);
  p.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(kD)));
  p.lse = lse;
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, window_fwd_kernel) != cudaSuccess) return launch_status("gqa_window: attributes");
    KDA_CHECK_SUPPORTED(fa.numRegs == kRegsLaunch, "%s: kernel compiled to %d registers/thread, its split needs %d", op,
                        fa.numRegs, kRegsLaunch);
    if (cudaFuncSetAttribute(window_fwd_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(Smem::kBytes)) != cudaSuccess)
      return launch_status("gqa_window: cudaFuncSetAttribute");
    attr_set[dev].store(true, std::memory_order_release);
  }
  // the encoder is a driver call that needs a current context: a thread that has
  // not used the device yet (autograd's) gets it here
  cudaSetDevice(dev);
  CUtensorMap tq, tk, tv, to;
  if ((s = tmap_head_rows(&tq, q, B, S, QH, q_strides)) != KDA_OK) return s;
  if ((s = tmap_head_rows(&tk, k, B, S, KH, k_strides)) != KDA_OK) return s;
  if ((s = tmap_head_rows(&tv, v, B, S, KH, v_strides)) != KDA_OK) return s;
  if ((s = tmap_head_rows(&to, out, B, S, QH, dense)) != KDA_OK) return s;
  const int64_t units = B * QH * p.npairs;
  const int grid = static_cast<int>(units < num_sms() ? units : num_sms());
  return launch_after("gqa_window", window_fwd_kernel, dim3(grid), kThreads, Smem::kBytes,
                      static_cast<cudaStream_t>(stream), tq, tk, tv, to, p, kda_err_ptr_window_fwd());
}
