// Forward of causal attention over packed sequences (head_dim 128, bf16) on tcgen05.
// In each sequence, query i sees key j <= i:
//   S = Q K^T,  P = 2^(S scale log2e - m),  O = P V / rowsum(P)
// with m a running reference of each row's scores: it only moves when a score exceeds it
// by more than 2^8, because weights up to 256 are as exact in bf16 and their sum in fp32
// as weights up to 1.
//
// Work unit = two tiles of 128 query rows that see the same keys: the same block of two
// heads of a group where its heads are even in number, else two consecutive blocks of a
// head.  (Heads first because both tiles then have rows at every block: a short sequence
// has one block only.)  One tile where there are no more such units than SMs.  Units come
// from the plan's tables, those with the most keys first; the persistent CTAs, one per SM,
// take them in turn.  A unit's K and V blocks pass through rings of 3 and 2 tiles and serve
// both tiles.
//
// A tile of a sequence's last block also holds rows of whatever lies behind it.  Such
// query rows are computed and not stored, and never move a row's reference, so a
// sequence's results do not depend on its neighbours; such keys lie after every query and
// their scores are replaced; and such rows of V, which a weight of zero would still
// multiply (0 x NaN), are overwritten with zeros between their arrival and their use.
//
// 640 threads: warp 0 loads Q and K, warp 2 V (and clears those rows), warp 1 issues S
// (and allocates TMEM), warp 3 P V, warps 4-11 / 12-19 softmax of tile 0 / 1: warp w reads
// TMEM lanes 32 (w % 4), 64 of a row's 128 keys per thread.
// P stays in TMEM, as bf16, and is the P V product's A operand there.  One region is left
// for S, which the tiles take in turn: a tile's S is issued as soon as the other has
// copied its S into registers, so the tiles run half a step apart and one exponentiates
// while the other stores.  The two warps that share a row agree on its reference with one
// bar.red a step and exchange maxima only when a score exceeded it.
// V is read as stored (MN-major B); rows of O leave from registers.
// TMEM columns: S [0,128), P_0 [128,192), P_1 [192,256), O_0 [256,384), O_1 [384,512).
// Shared memory: Q_0 | Q_1 | K ring (3 x 32 KB) | V ring (2 x 32 KB) | row exchange.
// 464 us for one sequence of 8,192 tokens, 32 heads (0.55 TFLOP on visible pairs: 1,185
// TFLOP/s, 0.72 of the measured bf16 rate), 352 us for 24 of 16,384 together (1,027).  A step
// of two tiles takes about 3,070 cycles, of which the tensor core works 2,048 and the
// exponentials' pipe 2,048: the rest is the latency of a tile's chain (wait, TMEM load,
// maximum, agreement, exponentials, store).  Without maximum and agreement after a unit's
// first block, which needs a second launch for units whose weights then overflow, 4 to 5 %
// faster; not kept.  Calls that last are held by the power limit: 32,768 tokens take 7.6 ms.
// All mbarrier waits are bounded (common.cuh); every TMA load targets one CTA.
#include <math.h>

#include "launch.cuh"
#include "packed.cuh"
#include "window.cuh"

KDA_DEFINE_ERROR_WORD(packed_fwd)
KDA_DEFINE_ERROR_WORD(packed_fwd_plan)  // a plan for other rows: later calls' waits do not read it

namespace kda {
namespace {

constexpr int kKSlots = 3, kVSlots = 2;
constexpr int kRowWarps = 16;
constexpr int kThreads = 128 + 32 * kRowWarps;
// Registers per thread: at launch (what the compiler reports for 640 threads), and
// after the control warpgroup has given some to the four of row warps.
constexpr int kRegsLaunch = 96, kRegsCtl = 64, kRegsRow = 104;
static_assert(128 * kRegsCtl + 32 * kRowWarps * kRegsRow <= kThreads * kRegsLaunch, "register split");
constexpr int kPairBarrier = 2;   // named barriers 2 .. 9: the two warps of a (tile, 32 rows)

// What a unit's two tiles are: two blocks of a head, a block of two heads, or (one tile) a block of one.
enum Mode { kBlocks, kHeads, kOne };

struct FwdParams {
  PlanView plan;
  int tokens, QH, rep;
  int mode;          // what a unit's tiles are
  int per;           // units of a block (or of two)
  int zero_rest;     // rows of no sequence: zeros, or left as they are
  float scale_log2;  // softmax scale * log2(e)
  __nv_bfloat16* out;  // [tokens][QH][128]
  float* lse;          // [QH][tokens] or null: each row's log2-sum-exp of the scaled scores
  unsigned* plan_err;
};

struct Smem {
  static constexpr uint32_t kQ = 0, kK = 2 * kTile, kV = kK + kKSlots * kTile;
  static constexpr uint32_t kExchange = kV + kVSlots * kTile;  // 1 KB, fp32 [tile][row]: maxima and sums of two warps' halves
  static constexpr uint32_t kBars = kExchange + 1024;
  static constexpr uint32_t kNumBars = 28;
  static constexpr size_t kBytes = 1024 + kBars + kNumBars * 8;
  static_assert(kBytes > 116 * 1024 && kBytes <= 227 * 1024, "shared memory budget");
};

// A unit: tile t is block `block[t]` of head `head[t]`, and sees key blocks [0, to[t])
// (none where the tile has no rows); nb: of either.
struct Unit {
  int start, len;
  int block[2], head[2], to[2];
  int nb;
};
__device__ __forceinline__ int num_units(const FwdParams& p) {
  return (p.mode == kBlocks ? p.plan.head->pairs : p.plan.head->blocks) * p.per;
}
__device__ __forceinline__ Unit unit_at(const FwdParams& p, int u) {
  const int e = u / p.per, h = u - e * p.per;
  const Block b = (p.mode == kBlocks ? p.plan.pairs : p.plan.sorted)[e];
  Unit c;
  c.start = b.x;
  c.len = b.y;
  c.block[0] = b.z;
  c.block[1] = p.mode == kBlocks ? b.z + 1 : b.z;
  c.head[0] = p.mode == kHeads ? 2 * h : h;
  c.head[1] = p.mode == kHeads ? 2 * h + 1 : h;
  c.to[0] = b.z + 1;
  c.to[1] = p.mode == kHeads ? b.z + 1 : p.mode == kBlocks && (b.z + 1) * kBlk < b.y ? b.z + 2 : 0;
  c.nb = max(c.to[0], c.to[1]);
  return c;
}

__global__ void __launch_bounds__(kThreads, 1)
    packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const FwdParams p, unsigned* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem::kBars);
  // per slot of a ring, one phase per use; every waiter waits for all of them in turn
  uint64_t* k_full = bars;         // [3] K landed
  uint64_t* k_free = bars + 3;     // [3] the S that read it are done
  uint64_t* v_full = bars + 6;     // [2] V landed, rows of others cleared
  uint64_t* v_free = bars + 8;     // [2] the P V that read it are done
  uint64_t* v_landed = bars + 10;  // a V tile to clear landed; one phase each
  uint64_t* s_free = bars + 11;    // S copied out (8 warps); one phase per S, of either tile
  // [2], per tile; one phase per block that the tile sees
  uint64_t* s_ready = bars + 12;   // S in TMEM
  uint64_t* p_ready = bars + 14;   // P in TMEM (8 warps)
  uint64_t* pv_done = bars + 16;   // O += P V done
  // [2], one phase per unit in which the tile has rows
  uint64_t* q_full = bars + 18;    // Q landed
  uint64_t* q_free = bars + 20;    // its last S is done
  uint64_t* o_free = bars + 22;    // O read out (8 warps)
  uint64_t* drain = bars + 24;     // [2] once
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 26);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 26; ++i) {
      const bool rows = i == 11 || i == 14 || i == 15 || i == 22 || i == 23;
      mbar_init(bars + i, rows ? kRowWarps / 2 : 1);
    }
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
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
  const bool fits = plan_ok(p.plan, p.tokens, p.plan_err);
  const int units = fits ? num_units(p) : 0;

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsCtl));
  if (warp == 0) {
    // ------------------------------------------------------- producer of Q and K
    if (lane == 0) {
      bool ok = true;
      int ks = 0, slot = 0, lap = 0;  // loads of K issued; slot of the next, and its use of that slot
      int qs[2] = {0, 0};
      for (int k = 0, u = blockIdx.x; u < units && ok; u = unit_of_round(++k)) {
        const Unit c = unit_at(p, u);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (c.to[t] > 0 && ok) {
            if (qs[t] > 0) ok = mbar_wait(&q_free[t], static_cast<uint32_t>(qs[t] - 1) & 1u, err, kErrWaitEmpty);
            if (!ok) break;
            mbar_arrive_expect_tx(&q_full[t], kTile);
            load_tile(smem + Smem::kQ + t * kTile, &tmQ, &q_full[t], c.head[t], c.start + c.block[t] * kBlk, 0);
            ++qs[t];
          }
        const int g = c.head[0] / p.rep;
        for (int j = 0; j < c.nb && ok; ++j) {
          if (lap > 0) ok = mbar_wait(&k_free[slot], static_cast<uint32_t>(lap - 1) & 1u, err, kErrWaitEmpty);
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[slot], kTile);
          load_tile(smem + Smem::kK + slot * kTile, &tmK, &k_full[slot], g, c.start + j * kBlk, 0);
          ++ks;
          if (++slot == kKSlots) {
            slot = 0;
            ++lap;
          }
        }
      }
      // no copy may still be writing shared memory when the CTA exits
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (qs[t] > 0) mbar_drain(&q_full[t], static_cast<uint32_t>(qs[t] - 1) & 1u);
#pragma unroll
      for (int s = 0; s < kKSlots; ++s) {
        const int uses = (ks + kKSlots - 1 - s) / kKSlots;
        if (uses > 0) mbar_drain(&k_full[s], static_cast<uint32_t>(uses - 1) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------- producer of V
    bool ok = true;
    int vs = 0, cleared = 0;       // loads; of those, to v_landed
    int direct0 = -1, direct1 = -1;  // a slot's last load if it was not: its phase of v_full
    for (int k = 0, u = blockIdx.x; u < units && ok; u = unit_of_round(++k)) {
      const Unit c = unit_at(p, u);
      const int g = c.head[0] / p.rep;
      for (int j = 0; j < c.nb && ok; ++j, ++vs) {
        const int slot = vs & 1;
        uint8_t* tile = smem + Smem::kV + slot * kTile;
        if (vs >= kVSlots) ok = warp_wait(&v_free[slot], static_cast<uint32_t>((vs >> 1) - 1) & 1u, err, kErrWaitEmpty);
        if (!ok) break;
        const int rows = c.len - j * kBlk;  // of this sequence
        uint64_t* landed = rows < kBlk ? v_landed : &v_full[slot];
        if (lane == 0) {
          mbar_arrive_expect_tx(landed, kTile);
          load_tile(tile, &tmV, landed, g, c.start + j * kBlk, 0);
        }
        __syncwarp();
        (slot == 0 ? direct0 : direct1) = rows < kBlk ? -1 : vs >> 1;
        if (rows < kBlk) {
          // whatever lies behind the sequence must not meet its weights of zero
          ++cleared;
          ok = warp_wait(v_landed, static_cast<uint32_t>(cleared - 1) & 1u, err, kErrWaitFull);
          if (!ok) break;
          for (int i = rows * 8 + lane; i < kBlk * 8; i += 32) {
            st_shared_v4(smem_u32(tile) + i * 16, 0u, 0u, 0u, 0u);
            st_shared_v4(smem_u32(tile) + kHalf + i * 16, 0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[slot]);
        }
      }
    }
    if (lane == 0) {
      if (cleared > 0) mbar_drain(v_landed, static_cast<uint32_t>(cleared - 1) & 1u);
      if (direct0 >= 0) mbar_drain(&v_full[0], static_cast<uint32_t>(direct0) & 1u);
      if (direct1 >= 0) mbar_drain(&v_full[1], static_cast<uint32_t>(direct1) & 1u);
    }
    __syncwarp();
  } else if (warp < 4) {
    // ------------------------------- MMA issuers: S (warp 1) and P V (warp 3)
    const bool one = elect_one();
    const uint32_t base = smem_u32(smem);
    const bool is_s = warp == 1;
    int slot = 0;
    uint32_t lap = 0;            // of the next item in its ring
    uint32_t ns = 0;             // S so far, of both tiles
    uint32_t np[2] = {0u, 0u};   // a tile's P V so far
    uint32_t un[2] = {0u, 0u};   // and its units
    bool ok = true, any = false;
    for (int k = 0, u = blockIdx.x; u < units && ok; u = unit_of_round(++k)) {
      const Unit c = unit_at(p, u);
      for (int j = 0; j < c.nb && ok; ++j) {
        const uint32_t tile = base + (is_s ? Smem::kK : Smem::kV) + slot * kTile;
        ok = warp_wait(&(is_s ? k_full : v_full)[slot], lap & 1u, err, kErrWaitFull);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || j >= c.to[t]) continue;
          if (is_s) {  // Q landed, the last S copied out
            if (j == 0) ok = warp_wait(&q_full[t], un[t] & 1u, err, kErrWaitFull);
            if (ok && ns > 0) ok = warp_wait(s_free, (ns - 1u) & 1u, err, kErrWaitAccumFree);
            if (!ok) continue;
            tc_fence_after();
            if (one) {
              mma_kk(tmem, base + Smem::kQ + t * kTile, tile);
              umma_commit(&s_ready[t]);
              if (j + 1 == c.to[t]) umma_commit(&q_free[t]);
            }
            ++ns;
          } else {  // P written, the last unit's O read
            ok = warp_wait(&p_ready[t], np[t] & 1u, err, kErrWaitFull);
            if (ok && j == 0 && un[t] > 0) ok = warp_wait(&o_free[t], (un[t] - 1u) & 1u, err, kErrWaitAccumFree);
            if (!ok) continue;
            tc_fence_after();
            if (one) {
              mma_tm(tmem + 256 + t * kBlk, tmem + 128 + t * 64, tile, j == 0);
              umma_commit(&pv_done[t]);
            }
            ++np[t];
          }
          un[t] += j == 0 ? 1u : 0u;
          any = true;
        }
        if (one && ok) umma_commit(&(is_s ? k_free : v_free)[slot]);  // once this thread's MMAs have read the item
        __syncwarp();
        if (++slot == (is_s ? kKSlots : kVSlots)) {
          slot = 0;
          ++lap;
        }
      }
    }
    if (one && any) {
      // every issued MMA must finish before TMEM is released
      umma_commit(&drain[is_s ? 0 : 1]);
      mbar_drain(&drain[is_s ? 0 : 1], 0u);
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
    float* xch = reinterpret_cast<float*>(smem + Smem::kExchange) + t * kBlk + r;
    const int pair = kPairBarrier + t * 4 + quad;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    uint32_t n = 0;   // blocks seen so far
    bool ok = true;
    for (int k = 0, u = blockIdx.x; u < units && ok; u = unit_of_round(++k)) {
      const Unit c = unit_at(p, u);
      const int to = t == 0 ? c.to[0] : c.to[1], block = t == 0 ? c.block[0] : c.block[1];
      const int head = t == 0 ? c.head[0] : c.head[1];
      if (to == 0) continue;  // no rows (both halves alike)
      const int qpos = block * kBlk + r;  // in the sequence
      // A row of another sequence never moves a reference: NaN and -inf + inf compare false.
      const float room = qpos < c.len ? 8.f : INFINITY;
      float m = -INFINITY, l = 0.f;
      // A wait that expires does not leave the loop by itself: its warp meets its
      // partner at the next pair barrier (or the unit's end) and both leave there.
      bool s_there = false;  // S is known to be ready
      for (int j = 0; j < to; ++j) {
        const uint32_t par = n & 1u;
        if (ok && !s_there) ok = warp_wait(&s_ready[t], par, err, kErrWaitAccum);
        tc_fence_after();
        uint32_t s[64];
        tmem_ld_32x32b_x32(scol, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_ld_32x32b_x32(scol + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
        tmem_ld_wait();
        tc_fence_before();
        if (ok) mbar_arrive_warp(s_free);
        if (j + 1 == to) {  // the diagonal: keys [0, hi) of this thread's are not after the query
          const int hi = r + 1 - 64 * half;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t live = range_mask(0, hi - 32 * w);
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
        if (bar_or(pair, 64, !ok || mx > m + room)) {
          if (half == 1) *xch = mx;
          ok = bar_and(pair, 64, ok);
          if (!ok) break;
          if (half == 0) *xch = fmaxf(m, fmaxf(mx, *xch));
          bar_sync(pair, 64);
          const float m_new = *xch;
          const float f = m_new == -INFINITY ? 1.f : exp2_approx(m - m_new);
          m = m_new;
          l *= f;
          if (j > 0) {
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
        const bool p_free = j == 0 || __all_sync(0xffffffffu, mbar_test(&pv_done[t], par ^ 1u));
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
          s_there = j + 1 < to && __all_sync(0xffffffffu, mbar_test(&s_ready[t], par ^ 1u));
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive_warp(&p_ready[t]);
        }
        ++n;
      }
      if (ok) ok = warp_wait(&pv_done[t], (n - 1u) & 1u, err, kErrWaitAccum);
      // the two halves' sums: half 1 hands its over, half 0 answers with the whole
      if (half == 1) *xch = l;
      ok = bar_and(pair, 64, ok);
      if (!ok) break;
      if (half == 0) {
        l += *xch;
        *xch = l;
        if (p.lse && qpos < c.len)
          p.lse[static_cast<int64_t>(head) * p.tokens + c.start + qpos] = (m == -INFINITY ? 0.f : m) + __log2f(l);
      }
      bar_sync(pair, 64);
      if (half == 1) l = *xch;
      tc_fence_after();
      const float inv = 1.0f / l;
      const int row0 = block * kBlk + quad * 32;
      __nv_bfloat16* dst = p.out + (static_cast<int64_t>(c.start + row0) * p.QH + head) * kD + 64 * half;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t o[32], w[16];
        tmem_ld_32x32b_x32(ocol + 32 * k, o);
        tmem_ld_wait();
        if (k == 1) {
          tc_fence_before();
          mbar_arrive_warp(&o_free[t]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[i] = pack_bf16x2(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
        store_rows(w, dst + 32 * k, static_cast<int64_t>(p.QH) * kD, c.len - row0);
      }
    }
    if (fits && p.zero_rest) {
      const PlanHead& h = *p.plan.head;
      const int64_t at = static_cast<int64_t>(blockIdx.x) * (32 * kRowWarps) + threadIdx.x - 128;
      const int64_t count = static_cast<int64_t>(gridDim.x) * (32 * kRowWarps);
      zero_rest(p.out, h.first, h.last, p.tokens, static_cast<int64_t>(p.QH) * kD * 2, at, count);
      if (p.lse) {
        const int64_t rest = h.first + p.tokens - h.last;
        for (int64_t i = at; i < rest * p.QH; i += count) {
          const int64_t head = i / rest, row = i - head * rest;
          p.lse[head * p.tokens + (row < h.first ? row : row - h.first + h.last)] = 0.f;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" kda_status kda_gqa_packed_bf16(const void* q, const void* k, const void* v, const void* plan,
                                          size_t plan_size, void* out, float* lse, int zero_rest, int64_t tokens,
                                          int64_t QH, int64_t KH, int64_t D, const int64_t* q_strides,
                                          const int64_t* k_strides, const int64_t* v_strides, void* stream) {
  const char* op = "gqa_packed";
  kda_status s;
  int64_t sequences = 0;
  if ((s = gqa_packed_check(op, tokens, QH, KH, D, plan, plan_size, &sequences)) != KDA_OK) return s;
  KDA_CHECK_ARG(q && k && v && out && q_strides && k_strides && v_strides, "%s: null pointer", op);
  const int64_t qs[3] = {0, q_strides[0], q_strides[1]}, ks[3] = {0, k_strides[0], k_strides[1]},
                vs[3] = {0, v_strides[0], v_strides[1]};
  KDA_CHECK_SUPPORTED(head_rows_ok(q, qs, 1, tokens, QH) && head_rows_ok(k, ks, 1, tokens, KH) &&
                          head_rows_ok(v, vs, 1, tokens, KH) && (reinterpret_cast<uintptr_t>(out) & 15u) == 0 &&
                          (reinterpret_cast<uintptr_t>(lse) & 3u) == 0,
                      "%s: pointers and rows must be 16-byte aligned", op);
  const int64_t most = plan_blocks(tokens, sequences);
  FwdParams p{};
  p.plan = plan_view(plan, most);
  p.tokens = static_cast<int>(tokens);
  p.QH = static_cast<int>(QH);
  p.rep = static_cast<int>(QH / KH);
  p.zero_rest = zero_rest;
  p.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(kD)));
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.plan_err = kda_err_ptr_packed_fwd_plan();
  const int64_t units = (tokens / kBlk + (sequences < tokens ? sequences : tokens)) * QH;
  KDA_CHECK_SUPPORTED(units < (1ll << 30), "%s: too many rows (tokens=%lld QH=%lld sequences=%lld)", op,
                      (long long)tokens, (long long)QH, (long long)sequences);
  // One tile where that gives no CTA a second unit (`units` is a bound; the blocks are counted on the
  // device): a tile that does not wait for the other's turns takes less time.  One sequence of
  // 1,024 tokens, 16 heads 18.1 us, 20.9 with two; 1,500 of 12 heads 23.3 and 27.5.
  p.mode = units <= num_sms() ? kOne : p.rep % 2 == 0 ? kHeads : kBlocks;
  p.per = static_cast<int>(p.mode == kHeads ? QH / 2 : QH);
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, packed_fwd_kernel) != cudaSuccess) return launch_status("gqa_packed: attributes");
    KDA_CHECK_SUPPORTED(fa.numRegs == kRegsLaunch, "%s: kernel compiled to %d registers/thread, its split needs %d", op,
                        fa.numRegs, kRegsLaunch);
    if (cudaFuncSetAttribute(packed_fwd_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(Smem::kBytes)) != cudaSuccess)
      return launch_status("gqa_packed: cudaFuncSetAttribute");
    attr_set[dev].store(true, std::memory_order_release);
  }
  // the encoder is a driver call that needs a current context: a thread that has
  // not used the device yet (autograd's) gets it here
  cudaSetDevice(dev);
  CUtensorMap tq, tk, tv;
  if ((s = tmap_head_rows(&tq, q, 1, tokens, QH, qs)) != KDA_OK) return s;
  if ((s = tmap_head_rows(&tk, k, 1, tokens, KH, ks)) != KDA_OK) return s;
  if ((s = tmap_head_rows(&tv, v, 1, tokens, KH, vs)) != KDA_OK) return s;
  const int grid = static_cast<int>(units < num_sms() ? units : num_sms());
  return launch_after(op, packed_fwd_kernel, dim3(grid), kThreads, Smem::kBytes, static_cast<cudaStream_t>(stream), tq,
                      tk, tv, p, kda_err_ptr_packed_fwd());
}
