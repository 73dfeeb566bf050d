// Backward of causal attention over packed sequences (head_dim 128, bf16) on tcgen05:
// P and dS live on chip, one 128 x 128 block at a time.
//
// In each sequence, query i sees key j <= i.  With
//   P = 2^(Q K^T scale log2e - lse),  dP = dO V^T,  dS = P (dP - di),
//   di = rowsum(dO * O)
// two kernels compute, block by block,
//   packed_dkv_kernel  dV_j = sum P^T dO, dK_j = scale sum dS^T Q over the query
//                      blocks (of all heads of the group) from key block j on
//   packed_dq_kernel   dQ_i = scale sum dS K over the key blocks up to query block i
// Each sum stays in TMEM until it is whole, so nothing is added through global memory,
// and the results do not depend on timing.  S and dP are computed twice (7 products a
// block pair instead of 5): added into an fp32 buffer, dQ's shares are 64 KB a block
// pair, which the L2 takes at 2.3 TB/s.
//
// P^T, dS^T and dS are written to TMEM as bf16, each thread's into the columns of S
// that it has read, and are the A operand of their products there.
//
// The last tile of a sequence also holds rows of whatever lies behind it.  Their scores'
// results are replaced by zeros; and where such rows are the long side of a product (Q and
// dO in dK and dV, K in dQ), zeros that meet them would still give 0 x NaN, so the row
// warps clear them in shared memory before they report the step's P or dS.
//
// Both kernels: 640 threads -- warp 0 TMA producer, warps 1-3 MMA issuers (warp 1
// allocates TMEM), warps 4-19 row warps: warp w reads TMEM lanes 32 (w % 4), columns
// 32 ((w - 4) / 4), i.e. 32 values of one row per thread, four warps on each SM
// partition to cover each other's latencies.  An issuer's mbarrier wait stalls
// behind its own queued MMAs, so products that wait for different things have
// issuers of their own (S and dV from one warp: 9 % slower).
// An mbarrier tells phases apart by parity only.  A barrier that may complete again
// before a waiter has looked is one of a pair (p_ready, ds_ready, s_ready), and
// every waiter waits for the phases in turn.
// Operand tiles are two 16 KB halves of 64 columns, 128-byte rows, 128-byte swizzle,
// loaded once and read K-major where their rows index M or N and MN-major where their
// rows index K.
// All mbarrier waits are bounded (common.cuh); every TMA load targets one CTA.
#include <math.h>

#include <algorithm>

#include "launch.cuh"
#include "packed.cuh"
#include "window.cuh"

KDA_DEFINE_ERROR_WORD(packed_bwd)
KDA_DEFINE_ERROR_WORD(packed_bwd_plan)  // a plan for other rows: later calls' waits do not read it

#define KDA_PB_TRY(expr)                  \
  do {                                    \
    const kda_status s_ = (expr);         \
    if (s_ != KDA_OK) return s_;          \
  } while (0)

namespace kda {
namespace {

constexpr int kRowWarps = 16;
constexpr int kThreads = 128 + 32 * kRowWarps;

struct BwdParams {
  PlanView plan;
  int tokens, QH, KH, rep;
  int64_t sp;         // rows per head of nlse and ndi: whole blocks, in the order of the buffer
  int zero_rest;      // rows of no sequence: zeros, or left as they are
  float sl2;          // softmax scale * log2(e)
  float scale;
  const float* nlse;  // [QH][sp]: -lse
  const float* ndi;   // [QH][sp]: -rowsum(dout * out)
  float* partial;     // [2 x CTAs][2][128 d][128 keys] fp32: dV_j, dK_j (unscaled) of cut walks
  int4* pieces;       // [2 x CTAs] beside them: block, kv head, steps of the share, of the walk
  unsigned* counter;  // join items taken
  int ctas;           // of dkv
  __nv_bfloat16* dq;  // [tokens][QH][128]
  __nv_bfloat16* dk;  // [tokens][KH][128]
  __nv_bfloat16* dv;
  unsigned* plan_err;
};

// Seven tiles, then small things.
struct Smem {
  // dkv: K_j | V_j | Q (two buffers) | dO (two)
  // dq:  Q | dO | K (three buffers) | V (two)
  static constexpr uint32_t kLse = 7 * kTile;             // dkv: [2][128] floats
  static constexpr uint32_t kDi = kLse + 1024;            // dkv: [2][128] floats
  static constexpr uint32_t kBars = kDi + 1024;
  static constexpr uint32_t kNumBars = 24;
  static constexpr uint32_t kFirst = kBars + kNumBars * 8;  // dkv: the run's first piece and its length
  static constexpr size_t kBytes = kFirst + 64;
  static_assert(kBytes > 116 * 1024 && kBytes <= 227 * 1024, "shared memory budget");
};

// A piece of a CTA's run: steps [it0, it0 + n) of the walk of key block e (of the plan's
// natural order) for kv head g, which has `walk` steps, nq (the query blocks from its own
// to its sequence's last) for each head.
struct Piece {
  Block b;
  int e, g, it0, n, walk, nq;
};
__device__ __forceinline__ void set_block(const BwdParams& p, Piece* c) {
  c->b = p.plan.natural[c->e];
  c->nq = ((c->b.y + kBlk - 1) >> 7) - c->b.z;
  c->walk = p.rep * c->nq;
}
// The piece at step x of the concatenated walks (block after block, each for every kv
// head; x < their number), of at most `most` steps.
__device__ __forceinline__ Piece piece_at(const BwdParams& p, int64_t x, int64_t most) {
  Piece c;
  int lo = 0, hi = p.plan.head->blocks;  // the last key block whose walks start at or before x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.plan.before[mid] * p.QH <= x) lo = mid;
    else hi = mid;
  }
  c.e = lo;
  set_block(p, &c);
  const int64_t y = x - p.plan.before[lo] * p.QH;
  c.g = static_cast<int>(y / c.walk);
  c.it0 = static_cast<int>(y - static_cast<int64_t>(c.g) * c.walk);
  c.n = static_cast<int>(min(most, static_cast<int64_t>(c.walk - c.it0)));
  return c;
}
// The step at which a run starts that has x of the walks' cost before it, where a walk
// costs its steps and kWalkCost before the first of them (loads without a step beside them,
// results on their way out: by steps alone the CTA with the short walks at a sequence's end
// worked 270,000 cycles at S4096 of 16 heads, the others 200,000; with 1 to 3: 212,000).
constexpr int kWalkCost = 2;
__device__ __forceinline__ int64_t step_at_cost(const BwdParams& p, int64_t x) {
  auto cost_before = [&](int e) { return p.plan.before[e] * p.QH + static_cast<int64_t>(e) * p.KH * kWalkCost; };
  int lo = 0, hi = p.plan.head->blocks;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cost_before(mid) <= x) lo = mid;
    else hi = mid;
  }
  Piece c;
  c.e = lo;
  set_block(p, &c);
  const int64_t y = x - cost_before(lo);
  const int64_t g = y / (c.walk + kWalkCost), in = y - g * (c.walk + kWalkCost);
  return p.plan.before[lo] * p.QH + g * c.walk + (in > kWalkCost ? in - kWalkCost : 0);
}
// The piece after c, of at most `most` steps: the next walk from its start.
__device__ __forceinline__ Piece piece_after(const BwdParams& p, const Piece& c, int most) {
  Piece d = c;
  if (++d.g == p.KH) {
    d.g = 0;
    ++d.e;
    set_block(p, &d);
  }
  d.it0 = 0;
  d.n = min(most, d.walk);
  return d;
}
// Rows from `rows` on of a tile become zeros, by the 512 threads of the row warps, which
// fence them to the tensor core's reads afterwards.
__device__ __forceinline__ void clear_rows(uint32_t tile, int rows, int thread) {
  for (int i = rows * 8 + thread; i < kBlk * 8; i += 32 * kRowWarps) {
    st_shared_v4(tile + i * 16, 0u, 0u, 0u, 0u);
    st_shared_v4(tile + kHalf + i * 16, 0u, 0u, 0u, 0u);
  }
}

// ---------------------------------------------------------------- dK and dV
// A step is one (head, query block) of a key block's walk.  Walks are of all lengths, up
// to rep x the blocks of the sequence, and there may be few, so the CTAs (one per SM,
// persistent) each take an equal run of the concatenated walks.  Where a run
// cuts a walk, its dV_j and dK_j are fp32 partial sums, which the row warps of the
// dQ kernel add in order.
//   S^T = K_j Q^T, P^T (row warps, key rows; 32 queries per thread, kept in
//   registers as fp32, bf16 for the product), dP^T = V_j dO^T, dV_j += P^T dO,
//   dS^T = P^T (dP^T - di) (from the unrounded P^T), dK_j += dS^T Q
// S^T(n) lies in region n % 2 and dP^T(n) in the other; P^T(n) and dS^T(n) replace
// S^T(n) column by column.  S^T(n+1) is issued as soon as the row warps have copied
// dP^T(n), dV(n) and dK(n) as soon as they have written P^T(n) and dS^T(n), and
// dP^T(n+1) once both are done with the region it overwrites.
// A step takes about 3,050 cycles, the row warps' chain: wait, TMEM load, 16,384
// exponentials (1,024 cycles of their pipe), store, wait, load, store.  The tensor
// core works 2,048 of them.  A walk costs some 8,000 cycles more: 3,000 to 4,000 until its
// results have left (stores and the exchanges before them), the first loads of K, V and dO
// behind the last products.  133 us at S4096 of 16 heads, 103 at 12 sequences of 8,192 tokens.
// With dS^T through shared memory, which lets dP^T run a step ahead, a call is 6 % slower
// (a product with both operands there needs all of its bandwidth); with the next walk's K
// loaded a walk ahead, or results out before the first dS, it is no faster.
// TMEM columns: regions [0,128), [128,256), dV [256,384), dK [384,512).
__global__ void __launch_bounds__(kThreads, 1)
    packed_dkv_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                      const BwdParams p, unsigned* err) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr uint32_t kK = 0, kV = kTile, kQ = 2 * kTile, kDO = 4 * kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem::kBars);
  // one phase per piece
  uint64_t* k_full = bars + 0;      // K_j landed
  uint64_t* v_full = bars + 1;      // V_j landed
  uint64_t* dkv_ready = bars + 2;   // every MMA of the piece done: dV_j, dK_j final (2 issuers)
  uint64_t* acc_free = bars + 3;    // dV_j, dK_j read out of TMEM (16 warps)
  // [2] one phase per use of the buffers of step n, n % 2
  uint64_t* q_full = bars + 4;      // Q, nlse, ndi landed
  uint64_t* q_free = bars + 6;      // dK(n) done: Q read, dS^T read, and the rows are past nlse, ndi
  uint64_t* do_full = bars + 8;     // dO landed
  uint64_t* do_free = bars + 10;    // dV(n) done: P^T read
  // one phase per step n of the run
  uint64_t* s_ready = bars + 12;    // S^T(n) in TMEM
  uint64_t* dp_ready = bars + 13;   // dP^T(n) in TMEM
  uint64_t* dp_free = bars + 14;    // dP^T(n) read out (16 warps)
  uint64_t* p_ready = bars + 15;    // [2] P^T(n) in TMEM (16 warps): the rows may be a step ahead of dV
  uint64_t* ds_ready = bars + 17;   // dS^T(n) in TMEM (16 warps)
  uint64_t* drain = bars + 18;      // [3] once
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 21);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 21; ++i)
      mbar_init(bars + i, i == 3 || (i >= 14 && i <= 17) ? kRowWarps : i == 2 ? 2 : 1);
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmDO);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  int* first_s = reinterpret_cast<int*>(smem + Smem::kFirst);
  if (warp == 3 && lane == 0) {
    const PlanHead& head = *p.plan.head;
    const bool fits = plan_matches(p.plan, p.tokens);
    const int64_t total = fits ? head.steps * p.QH : 0;
    const int64_t cost = fits ? total + static_cast<int64_t>(head.blocks) * p.KH * kWalkCost : 0;
    // Fewer than CTAs: the first ones take one each, so that a walk's shares follow one
    // another.  (A run between two walks may still be empty.)
    const int64_t ctas = min(static_cast<int64_t>(gridDim.x), cost), cta = blockIdx.x;
    const int64_t x = cta < ctas ? step_at_cost(p, cost * cta / ctas) : 0;
    const int64_t end = cta + 1 < ctas ? step_at_cost(p, cost * (cta + 1) / ctas) : cta < ctas ? total : 0;
    Piece c{};
    if (end > x) c = piece_at(p, x, end - x);
    first_s[0] = c.e, first_s[1] = c.g, first_s[2] = c.it0, first_s[3] = c.n, first_s[4] = c.walk, first_s[5] = c.nq;
    first_s[6] = static_cast<int>(end - x);
    first_s[8] = c.b.x, first_s[9] = c.b.y, first_s[10] = c.b.z, first_s[11] = c.b.w;
    // no share of a cut walk here, until the row warps say so (which they may not reach)
    p.pieces[2 * blockIdx.x] = p.pieces[2 * blockIdx.x + 1] = make_int4(0, 0, 0, 0);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  // every role walks the run's pieces; n0: steps of the earlier ones
  Piece c = {make_int4(first_s[8], first_s[9], first_s[10], first_s[11]),
             first_s[0], first_s[1], first_s[2], first_s[3], first_s[4], first_s[5]};
  const int run = first_s[6];  // 0 where there are fewer steps than CTAs
  int n0 = 0;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      bool ok = run > 0;
      int ks = 0, vs = 0, qs = 0, dos = 0;  // loads issued
      while (ok) {
        int h = c.g * p.rep + c.it0 / c.nq, q = c.it0 % c.nq;  // head; query block of the walk
        for (int i = 0; i < c.n; ++i) {
          const int n = n0 + i;
          const uint32_t pprev = static_cast<uint32_t>(n - 1) & 1u;
          const uint32_t use = static_cast<uint32_t>((n >> 1) - 1) & 1u;  // phase of step n - 2 in its buffers
          const int s0 = c.b.x + (c.b.z + q) * kBlk;
          const int nb = n & 1;
          const int64_t row = h * p.sp + static_cast<int64_t>(c.b.w + c.b.z + q) * kBlk;
          if (n >= 2) ok = mbar_wait(&q_free[nb], use, err, kErrWaitEmpty);
          if (!ok) break;
          mbar_arrive_expect_tx(&q_full[nb], kTile + 2 * kBlk * 4);
          load_tile(smem + kQ + nb * kTile, &tmQ, &q_full[nb], h, s0, 0);
          if (n == 0) {
            pdl_wait();     // nlse, ndi are written by the launch before this one
            pdl_trigger();  // and complete before any CTA of the launch after this one starts
          }
          bulk_load_1d(smem + Smem::kLse + nb * kBlk * 4, p.nlse + row, kBlk * 4, &q_full[nb]);
          bulk_load_1d(smem + Smem::kDi + nb * kBlk * 4, p.ndi + row, kBlk * 4, &q_full[nb]);
          ++qs;
          if (i == 0) {
            // K_j once the previous piece's last S is done, V_j once its last dP is
            if (n > 0) ok = mbar_wait(s_ready, pprev, err, kErrWaitEmpty);
            if (!ok) break;
            mbar_arrive_expect_tx(k_full, kTile);
            load_tile(smem + kK, &tmK, k_full, c.g, c.b.x + c.b.z * kBlk, 0);
            ++ks;
            if (n > 0) ok = mbar_wait(dp_ready, pprev, err, kErrWaitEmpty);
            if (!ok) break;
            mbar_arrive_expect_tx(v_full, kTile);
            load_tile(smem + kV, &tmV, v_full, c.g, c.b.x + c.b.z * kBlk, 0);
            ++vs;
          }
          // dO(n - 2) has been read: by dV, and by dP before the dK of above
          if (n >= 2) ok = mbar_wait(&do_free[nb], use, err, kErrWaitEmpty);
          if (!ok) break;
          mbar_arrive_expect_tx(&do_full[nb], kTile);
          load_tile(smem + kDO + nb * kTile, &tmDO, &do_full[nb], h, s0, 0);
          ++dos;
          if (++q == c.nq) {
            q = 0;
            ++h;
          }
        }
        n0 += c.n;
        if (n0 >= run) break;
        c = piece_after(p, c, run - n0);
      }
      if (run == 0) pdl_wait();  // this launch does not end before the one before it has
      // no copy may still be writing shared memory when the CTA exits
      if (ks > 0) mbar_drain(k_full, static_cast<uint32_t>(ks - 1) & 1u);
      if (vs > 0) mbar_drain(v_full, static_cast<uint32_t>(vs - 1) & 1u);
      for (int t = 0; t < 2; ++t) {
        const int uses = (qs + 1 - t) >> 1, douses = (dos + 1 - t) >> 1;
        if (uses > 0) mbar_drain(&q_full[t], static_cast<uint32_t>(uses - 1) & 1u);
        if (douses > 0) mbar_drain(&do_full[t], static_cast<uint32_t>(douses - 1) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // -------------------------------------------------- issuer of dK and dP^T
    const bool one = elect_one();
    const uint32_t base = smem_u32(smem);
    bool ok = run > 0, any = false;
    int pieces = 0;
    // dP^T(n) into the columns of step n - 1's S^T, once dV(n - 1) and dK(n - 1) have
    // read the P^T and dS^T there
    auto issue_dp = [&](int n, bool first) -> bool {
      const uint32_t nb = static_cast<uint32_t>(n) & 1u, ob = nb ^ 1u;
      const uint32_t prev = static_cast<uint32_t>((n - 1) >> 1) & 1u;
      if (first && !warp_wait(v_full, static_cast<uint32_t>(pieces) & 1u, err, kErrWaitFull)) return false;
      if (!warp_wait(&do_full[nb], static_cast<uint32_t>(n >> 1) & 1u, err, kErrWaitFull)) return false;
      if (n > 0 && !(warp_wait(&do_free[ob], prev, err, kErrWaitAccumFree) &&
                     warp_wait(&q_free[ob], prev, err, kErrWaitAccumFree)))
        return false;
      tc_fence_after();
      if (one) {
        mma_kk(tmem + ob * 128, base + kV, base + kDO + nb * kTile);
        umma_commit(dp_ready);
      }
      __syncwarp();
      return any = true;
    };
    while (ok) {
      for (int i = 0; i < c.n && ok; ++i) {
        const int n = n0 + i;
        const uint32_t nb = static_cast<uint32_t>(n) & 1u;
        ok = issue_dp(n, i == 0);
        // dK_j += dS^T(n) Q(n) (the first of a piece once the last piece's sums are read)
        if (ok && i == 0 && pieces > 0)
          ok = warp_wait(acc_free, static_cast<uint32_t>(pieces - 1) & 1u, err, kErrWaitAccumFree);
        if (ok) ok = warp_wait(ds_ready, nb, err, kErrWaitFull);
        if (!ok) break;
        tc_fence_after();
        if (one) {
          mma_tm_pairs(tmem + 384, tmem + nb * 128 + 16, base + kQ + nb * kTile, i == 0);
          umma_commit(&q_free[nb]);
          if (i + 1 == c.n) umma_commit(dkv_ready);
        }
        __syncwarp();
      }
      if (!ok) break;
      n0 += c.n;
      ++pieces;
      if (n0 >= run) break;
      c = piece_after(p, c, run - n0);
    }
    if (one && any) {
      // every issued MMA must finish before TMEM is released
      umma_commit(&drain[0]);
      mbar_drain(&drain[0], 0u);
    }
    __syncwarp();
  } else if (warp < 4) {
    // ------------------------------------ issuers of dV (warp 2) and S^T (warp 3)
    const bool one = elect_one();
    const uint32_t base = smem_u32(smem);
    bool ok = run > 0, any = false;
    int pieces = 0;
    while (ok) {
      for (int i = 0; i < c.n && ok; ++i) {
        const int n = n0 + i;
        const uint32_t nb = static_cast<uint32_t>(n) & 1u, use = static_cast<uint32_t>(n >> 1) & 1u;
        if (warp == 3) {
          // S^T(n) into the columns that dP^T(n - 1) has been read from
          if (i == 0) ok = warp_wait(k_full, static_cast<uint32_t>(pieces) & 1u, err, kErrWaitFull);
          if (ok) ok = warp_wait(&q_full[nb], use, err, kErrWaitFull);
          if (ok && n > 0) ok = warp_wait(dp_free, nb ^ 1u, err, kErrWaitAccumFree);
          if (!ok) break;
          tc_fence_after();
          if (one) {
            mma_kk(tmem + nb * 128, base + kK, base + kQ + nb * kTile);
            umma_commit(s_ready);
          }
        } else {
          // dV_j += P^T(n) dO(n) (the first of a piece once the last piece's sums are read)
          if (i == 0 && pieces > 0)
            ok = warp_wait(acc_free, static_cast<uint32_t>(pieces - 1) & 1u, err, kErrWaitAccumFree);
          if (ok) ok = warp_wait(&do_full[nb], use, err, kErrWaitFull);
          if (ok) ok = warp_wait(&p_ready[nb], use, err, kErrWaitFull);
          if (!ok) break;
          tc_fence_after();
          if (one) {
            mma_tm_pairs(tmem + 256, tmem + nb * 128, base + kDO + nb * kTile, i == 0);
            umma_commit(&do_free[nb]);
            if (i + 1 == c.n) umma_commit(dkv_ready);
          }
        }
        __syncwarp();
        any = true;
      }
      if (!ok) break;
      n0 += c.n;
      ++pieces;
      if (n0 >= run) break;
      c = piece_after(p, c, run - n0);
    }
    if (one && any) {
      umma_commit(&drain[warp - 1]);
      mbar_drain(&drain[warp - 1], 0u);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------- row warps
    const int grp = (warp - 4) >> 2;        // queries [32 grp, + 32) of the block
    const int kr = (warp & 3) * 32 + lane;  // key row of this thread (TMEM lane)
    const uint32_t col = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float2 sl2 = make_float2(p.sl2, p.sl2);
    // dV_j (groups 0, 1) and dK_j (2, 3) of a piece, 64 columns a thread, once its
    // MMAs are done: bf16 (dK times the softmax scale), or the fp32 share of a cut
    // walk.  Called after the next piece's first step, whose MMAs run meanwhile.
    auto finish = [&](const Piece& c, int piece) -> bool {
      if (!warp_wait(dkv_ready, static_cast<uint32_t>(piece) & 1u, err, kErrWaitAccum)) return false;
      tc_fence_after();
      const bool cut = c.n < c.walk;
      const int which = grp >> 1;
      const int slot = 2 * static_cast<int>(blockIdx.x) + (c.it0 == 0 ? 1 : 0);
      // [slot][dV, dK][d][key]: a warp writes 32 keys of one d, a 128-byte line
      float* part = p.partial + ((static_cast<int64_t>(slot) * 2 + which) * kD + (grp & 1) * 64) * kBlk + kr;
      if (cut && warp == 4 && lane == 0) p.pieces[slot] = make_int4(c.e, c.g, c.n, c.walk);
      const float f = which == 0 ? 1.f : p.scale;
      const int k0 = c.b.z * kBlk + (warp & 3) * 32;
      __nv_bfloat16* dst = (which == 0 ? p.dv : p.dk) +
                           (static_cast<int64_t>(c.b.x + k0) * p.KH + c.g) * kD + (grp & 1) * 64;
      uint32_t r[64];
      tmem_ld_32x32b_x32(col + 256 + grp * 64, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
      tmem_ld_32x32b_x32(col + 256 + grp * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive_warp(acc_free);
      if (cut) {
#pragma unroll
        for (int q = 0; q < 64; ++q) part[q * kBlk] = __uint_as_float(r[q]);
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w[16];
#pragma unroll
          for (int q = 0; q < 16; ++q)
            w[q] = pack_bf16x2(__uint_as_float(r[32 * half + 2 * q]) * f, __uint_as_float(r[32 * half + 2 * q + 1]) * f);
          store_rows(w, dst + 32 * half, static_cast<int64_t>(p.KH) * kD, c.b.y - k0);
        }
      }
      return true;
    };
    bool ok = run > 0;
    int pieces = 0;
    Piece last = c;  // the piece before this one
    while (ok) {
      // live queries of this key row: from the key itself up to the sequence's last;
      // none when the key is past it
      const int qlo = c.b.z * kBlk + kr, qhi = c.b.y;
      int q = c.it0 % c.nq;  // query block of the walk
      for (int i = 0; i < c.n; ++i) {
        const int n = n0 + i;
        const uint32_t par = static_cast<uint32_t>(n) & 1u;
        const int s0 = (c.b.z + q) * kBlk + 32 * grp;  // this thread's first query
        const int own = c.b.y - (c.b.z + q) * kBlk;      // rows of the query block that are the sequence's
        const uint32_t live = range_mask(qlo - s0, qhi - s0);
        // S^T(n) here, overwritten by P^T(n) and dS^T(n); dP^T(n) in the other region
        const uint32_t scol = col + par * 128 + 32 * grp, dpcol = col + (par ^ 1u) * 128 + 32 * grp;
        const float4* nlse_s = reinterpret_cast<const float4*>(smem + Smem::kLse) + par * 32 + 8 * grp;
        const float4* ndi_s = reinterpret_cast<const float4*>(smem + Smem::kDi) + par * 32 + 8 * grp;
        q = q + 1 == c.nq ? 0 : q + 1;
        ok = warp_wait2(s_ready, par, &q_full[par], static_cast<uint32_t>(n >> 1) & 1u, err, kErrWaitAccum);
        if (!ok) break;
        tc_fence_after();
        float2 e[16];  // P^T: 2^(s scale log2e - lse[q])
        uint32_t w[16];
        {
          uint32_t s[32];
          tmem_ld_32x32b_x32(scol, s);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 l = nlse_s[q];
            const float2 a = __ffma2_rn(make_float2(__uint_as_float(s[4 * q]), __uint_as_float(s[4 * q + 1])), sl2,
                                        make_float2(l.x, l.y));
            const float2 b = __ffma2_rn(make_float2(__uint_as_float(s[4 * q + 2]), __uint_as_float(s[4 * q + 3])), sl2,
                                        make_float2(l.z, l.w));
            e[2 * q] = make_float2(exp2_approx(a.x), exp2_approx(a.y));
            e[2 * q + 1] = make_float2(exp2_approx(b.x), exp2_approx(b.y));
          }
        }
        keep_live(live, e);
        pack16(e, w);
        tmem_st_32x32b_x16(scol, w);
        if (own < kBlk) {
          // S^T(n) has read Q; dP^T(n) may be reading dO, whose rows here only reach
          // columns that are replaced
          ok = warp_wait(&do_full[par], static_cast<uint32_t>(n >> 1) & 1u, err, kErrWaitAccum);
          if (!ok) break;
          clear_rows(smem_u32(smem) + kQ + par * kTile, own, threadIdx.x - 128);
          clear_rows(smem_u32(smem) + kDO + par * kTile, own, threadIdx.x - 128);
          fence_proxy_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive_warp(&p_ready[par]);
        // dS^T = P^T (dP^T - di[q])
        ok = warp_wait(dp_ready, par, err, kErrWaitAccum);
        if (!ok) break;
        tc_fence_after();
        {
          uint32_t d[32];
          tmem_ld_32x32b_x32(dpcol, d);
          tmem_ld_wait();
          tc_fence_before();
          mbar_arrive_warp(dp_free);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 l = ndi_s[q];
            e[2 * q] = __fmul2_rn(e[2 * q], __fadd2_rn(make_float2(__uint_as_float(d[4 * q]), __uint_as_float(d[4 * q + 1])),
                                                       make_float2(l.x, l.y)));
            e[2 * q + 1] =
                __fmul2_rn(e[2 * q + 1], __fadd2_rn(make_float2(__uint_as_float(d[4 * q + 2]), __uint_as_float(d[4 * q + 3])),
                                                    make_float2(l.z, l.w)));
          }
        }
        keep_live(live, e);
        pack16(e, w);
        tmem_st_32x32b_x16(scol + 16, w);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive_warp(ds_ready);
        if (i == 0 && pieces > 0) ok = finish(last, pieces - 1);
        if (!ok) break;
      }
      n0 += c.n;
      ++pieces;
      last = c;
      if (n0 >= run) break;
      c = piece_after(p, c, run - n0);
    }
    if (ok) finish(last, pieces - 1);
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ----------------------------------------------------------------------- dQ
// Unit = (query block, query head); one persistent CTA per SM.  Per key
// block the unit sees: S = Q K^T, dP = dO V^T, dS = P (dP - di) (row warps, query
// rows; 32 keys per thread, lse and di one register each), dQ += dS K.
// dS(n), in bf16, takes the columns of the S(n) that its thread has read, and is
// dQ's operand there.  dP(n + 1) is issued as soon as the rows have copied step n,
// S(n + 2) (two regions) when dQ(n) has read dS(n); units follow one another
// without a gap.
// A step takes about 2,500 cycles over a launch, the row warps' chain again (1,024 of
// them the exponentials' pipe); the tensor core works 1,536.  96 us at S4096 of 16 heads.
// TMEM columns: S [0,128) and [256,384), dP [128,256), dQ [384,512).
struct Unit {
  Block b;
  int h;  // query head
  int n;  // key blocks
};
__device__ __forceinline__ Unit dq_unit(const BwdParams& p, int u) {
  Unit c;
  const int e = u / p.QH;  // the query blocks that see the most first
  c.h = u - e * p.QH;
  c.b = p.plan.sorted[e];
  c.n = c.b.z + 1;
  return c;
}

// dk and dv of the walks that were cut: the shares of a walk (one at the start
// of its run's CTA and the next ones'), added in order.  The row warps that have no
// unit left take the items -- (CTA, dV or dK, 32 keys, 32 of d) -- one by one from
// a counter, so the CTAs that had one unit fewer do most of it; which warp takes an
// item makes no difference to its sum.  Nothing is joined once a wait has expired, here
// or in the launch before: shares may be missing.
__device__ __forceinline__ void join_cut_walks(const BwdParams& p, const unsigned* err) {
  const int lane = threadIdx.x & 31;
  const bool failed = *reinterpret_cast<const volatile unsigned*>(err) != 0u;
  for (;;) {
    unsigned item = 0;
    if (lane == 0) {
      item = atomicAdd(p.counter, 1u);
      if (failed) item = 0xffffffffu;
    }
    item = __shfl_sync(0xffffffffu, item, 0);
    if (item >= 32u * static_cast<unsigned>(p.ctas)) return;
    const int cta = static_cast<int>(item >> 5), which = (item >> 4) & 1, k0 = ((item >> 2) & 3) * 32, d0 = (item & 3) * 32;
    const int4 w = p.pieces[2 * cta + 1];
    if (w.z == 0) continue;
    float v[32];  // d0 + e of key k0 + lane
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = 0.f;
    int steps = w.z;
    for (int slot = 2 * cta + 1; slot >= 0; slot = next_share(p.pieces, 2 * p.ctas, slot, w.w, &steps)) {
      const float* src = p.partial + ((static_cast<int64_t>(slot) * 2 + which) * kD + d0) * kBlk + k0 + lane;
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] += src[e * kBlk];
    }
    const float f = which == 0 ? 1.f : p.scale;
    const Block b = p.plan.natural[w.x];
    const int kpos = b.z * kBlk + k0 + lane;
    if (kpos >= b.y) continue;
    uint4* dst = reinterpret_cast<uint4*>((which == 0 ? p.dv : p.dk) +
                                          (static_cast<int64_t>(b.x + kpos) * p.KH + w.y) * kD + d0);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      dst[u] = make_uint4(pack_bf16x2(v[8 * u] * f, v[8 * u + 1] * f), pack_bf16x2(v[8 * u + 2] * f, v[8 * u + 3] * f),
                          pack_bf16x2(v[8 * u + 4] * f, v[8 * u + 5] * f), pack_bf16x2(v[8 * u + 6] * f, v[8 * u + 7] * f));
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    packed_dq_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                     const BwdParams p, unsigned* err) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr uint32_t kQ = 0, kDO = kTile, kK = 2 * kTile, kV = 5 * kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem::kBars);
  // one phase per unit
  uint64_t* q_full = bars + 0;      // Q landed
  uint64_t* do_full = bars + 1;     // dO landed
  uint64_t* dq_ready = bars + 2;    // dQ final
  uint64_t* dq_free = bars + 3;     // dQ read out of TMEM (16 warps)
  // one phase per step n of the CTA ([m]: per use of buffer n % m)
  uint64_t* k_full = bars + 4;      // [3] K landed
  uint64_t* k_free = bars + 7;      // [3] dQ(n) done: K and dS read
  uint64_t* v_full = bars + 10;     // [2] V landed
  uint64_t* s_ready = bars + 12;    // [2] S(n) in TMEM
  uint64_t* dp_ready = bars + 14;   // dP(n) in TMEM
  uint64_t* sp_free = bars + 15;    // S(n), dP(n) read out (16 warps)
  uint64_t* ds_ready = bars + 16;   // [2] dS(n) in TMEM (16 warps): the rows may be a step ahead of dQ
  uint64_t* v_free = bars + 18;     // [2] dP(n) done: V read
  uint64_t* drain = bars + 20;      // [2] once
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 22);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 22; ++i) mbar_init(bars + i, i == 3 || (i >= 15 && i <= 17) ? kRowWarps : 1);
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmDO);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  // the plan is older than the launch before this one
  const int units = plan_matches(p.plan, p.tokens) ? p.plan.head->blocks * p.QH : 0;
  int n = 0;   // steps so far
  int uc = 0;  // units so far

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      bool ok = true;
      int qs = 0, dos = 0, vs = 0, ks = 0;  // loads issued
      for (int r = 0, u = blockIdx.x; u < units && ok; u = unit_of_round(++r)) {
        const Unit c = dq_unit(p, u);
        const int g = c.h / p.rep;
        for (int j = 0; j < c.n && ok; ++j, ++n) {
          const int kb = n % 3, vb = n & 1;
          const int k0 = c.b.x + j * kBlk;
          // A barrier tells phases apart by parity: every S is waited for in turn, before
          // anything of step n is loaded, so that neither an earlier nor a later phase is
          // taken for the one that Q waits for.
          if (n >= 2) ok = mbar_wait(&s_ready[vb], static_cast<uint32_t>((n >> 1) - 1) & 1u, err, kErrWaitEmpty);
          if (!ok) break;
          if (j == 0) {  // Q once the last unit's last S is done
            if (n > 0) ok = mbar_wait(&s_ready[vb ^ 1], static_cast<uint32_t>((n - 1) >> 1) & 1u, err, kErrWaitEmpty);
            if (!ok) break;
            mbar_arrive_expect_tx(q_full, kTile);
            load_tile(smem + kQ, &tmQ, q_full, c.h, c.b.x + c.b.z * kBlk, 0);
            ++qs;
          }
          if (n >= 3) ok = mbar_wait(&k_free[kb], static_cast<uint32_t>(n / 3 - 1) & 1u, err, kErrWaitEmpty);
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[kb], kTile);
          load_tile(smem + kK + kb * kTile, &tmK, &k_full[kb], g, k0, 0);
          ++ks;
          if (j == 0) {  // dO once the last unit's last dP is done
            if (n > 0) ok = mbar_wait(&v_free[vb ^ 1], static_cast<uint32_t>((n - 1) >> 1) & 1u, err, kErrWaitEmpty);
            if (!ok) break;
            mbar_arrive_expect_tx(do_full, kTile);
            load_tile(smem + kDO, &tmDO, do_full, c.h, c.b.x + c.b.z * kBlk, 0);
            ++dos;
          }
          if (n >= 2) ok = mbar_wait(&v_free[vb], static_cast<uint32_t>((n >> 1) - 1) & 1u, err, kErrWaitEmpty);
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[vb], kTile);
          load_tile(smem + kV + vb * kTile, &tmV, &v_full[vb], g, k0, 0);
          ++vs;
        }
      }
      // no copy may still be writing shared memory when the CTA exits
      if (qs > 0) mbar_drain(q_full, static_cast<uint32_t>(qs - 1) & 1u);
      if (dos > 0) mbar_drain(do_full, static_cast<uint32_t>(dos - 1) & 1u);
      for (int t = 0; t < 3; ++t) {
        const int uses = (ks + 2 - t) / 3, vuses = (vs + 1 - t) >> 1;
        if (uses > 0) mbar_drain(&k_full[t], static_cast<uint32_t>(uses - 1) & 1u);
        if (t < 2 && vuses > 0) mbar_drain(&v_full[t], static_cast<uint32_t>(vuses - 1) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // -------------------------------------------------------- issuer of dP
    const bool one = elect_one();
    const uint32_t base = smem_u32(smem);
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u = unit_of_round(++uc)) {
      const Unit c = dq_unit(p, u);
      for (int j = 0; j < c.n; ++j, ++n) {
        const uint32_t nb = static_cast<uint32_t>(n) & 1u;
        if (j == 0) ok = warp_wait(do_full, static_cast<uint32_t>(uc) & 1u, err, kErrWaitFull);
        if (ok) ok = warp_wait(&v_full[nb], static_cast<uint32_t>(n >> 1) & 1u, err, kErrWaitFull);
        if (ok && n > 0) ok = warp_wait(sp_free, nb ^ 1u, err, kErrWaitAccumFree);
        if (!ok) break;
        tc_fence_after();
        if (one) {
          mma_kk(tmem + 128, base + kDO, base + kV + nb * kTile);
          umma_commit(dp_ready);
          umma_commit(&v_free[nb]);
        }
        __syncwarp();
      }
    }
    if (one && n > 0) {
      // every issued MMA must finish before TMEM is released
      umma_commit(&drain[0]);
      mbar_drain(&drain[0], 0u);
    }
    __syncwarp();
  } else if (warp == 2) {
    // --------------------------------------------------- issuer of dQ and S
    // dQ(n), then S(n + 2) into the columns of its dS; S runs two steps ahead.
    const bool one = elect_one();
    const uint32_t base = smem_u32(smem);
    bool ok = true;
    int su = blockIdx.x, sj = 0, sn = 0, sc = 0;  // the next S: its unit, step in it, step and unit of the CTA
    Unit s_unit = su < units ? dq_unit(p, su) : Unit{};
    auto issue_s = [&]() -> bool {
      if (su >= units) return true;
      const int kb = sn % 3;
      if (sj == 0 && !warp_wait(q_full, static_cast<uint32_t>(sc) & 1u, err, kErrWaitFull)) return false;
      if (!warp_wait(&k_full[kb], static_cast<uint32_t>(sn / 3) & 1u, err, kErrWaitFull)) return false;
      if (sn >= 2 && !warp_wait(&k_free[(sn - 2) % 3], static_cast<uint32_t>((sn - 2) / 3) & 1u, err, kErrWaitAccumFree))
        return false;
      tc_fence_after();
      if (one) {
        mma_kk(tmem + (sn & 1) * 256, base + kQ, base + kK + kb * kTile);
        umma_commit(&s_ready[sn & 1]);
      }
      __syncwarp();
      ++sn;
      if (++sj == s_unit.n) {
        sj = 0;
        su = unit_of_round(++sc);
        if (su < units) s_unit = dq_unit(p, su);
      }
      return true;
    };
    ok = issue_s() && issue_s();
    for (int u = blockIdx.x; u < units && ok; u = unit_of_round(++uc)) {
      const Unit c = dq_unit(p, u);
      for (int j = 0; j < c.n && ok; ++j, ++n) {
        // dQ += dS(n) K (the first of a unit once the last unit's dQ is read)
        const int kb = n % 3;
        if (j == 0 && uc > 0) ok = warp_wait(dq_free, static_cast<uint32_t>(uc - 1) & 1u, err, kErrWaitAccumFree);
        if (ok) ok = warp_wait(&ds_ready[n & 1], static_cast<uint32_t>(n >> 1) & 1u, err, kErrWaitFull);
        if (!ok) break;
        tc_fence_after();
        if (one) {
          mma_tm_pairs(tmem + 384, tmem + (n & 1) * 256, base + kK + kb * kTile, j == 0);
          umma_commit(&k_free[kb]);
          if (j + 1 == c.n) umma_commit(dq_ready);
        }
        __syncwarp();
        ok = issue_s();
      }
    }
    if (one && sn > 0) {
      umma_commit(&drain[1]);
      mbar_drain(&drain[1], 0u);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------------------------------------------------- row warps
    const int grp = (warp - 4) >> 2;       // keys (and columns of dQ) [32 grp, + 32)
    const int r = (warp & 3) * 32 + lane;  // query row of this thread (TMEM lane)
    const uint32_t col = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 32 * grp;
    const float2 sl2 = make_float2(p.sl2, p.sl2);
    // dQ of a unit, once its MMAs are done.  Called after the next unit's first step,
    // whose MMAs run meanwhile.
    auto finish = [&](const Unit& c, int unit) -> bool {
      if (!warp_wait(dq_ready, static_cast<uint32_t>(unit) & 1u, err, kErrWaitAccum)) return false;
      tc_fence_after();
      uint32_t o[32], w[16];
      tmem_ld_32x32b_x32(col + 384, o);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive_warp(dq_free);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        w[i] = pack_bf16x2(__uint_as_float(o[2 * i]) * p.scale, __uint_as_float(o[2 * i + 1]) * p.scale);
      const int s0 = c.b.z * kBlk + (warp & 3) * 32;
      store_rows(w, p.dq + (static_cast<int64_t>(c.b.x + s0) * p.QH + c.h) * kD + 32 * grp,
                 static_cast<int64_t>(p.QH) * kD, c.b.y - s0);
      return true;
    };
    auto row_at = [&](const Unit& c) -> int64_t {
      return c.h * p.sp + static_cast<int64_t>(c.b.w + c.b.z) * kBlk + r;
    };
    bool ok = true;
    int64_t at = static_cast<int>(blockIdx.x) < units ? row_at(dq_unit(p, blockIdx.x)) : 0;
    // of the next unit, so that it does not wait for them.  They are complete: every CTA
    // of the launch before this one waited for their launch before it let this one start.
    float nl = 0.f, nd = 0.f;
    if (static_cast<int>(blockIdx.x) < units) {
      nl = __ldcg(p.nlse + at);
      nd = __ldcg(p.ndi + at);
    }
    Unit last = {};  // the unit before this one
    for (int u = blockIdx.x; u < units && ok; u = unit_of_round(++uc)) {
      const Unit c = dq_unit(p, u);
      const int qpos = c.b.z * kBlk + r;
      const float2 nlse = make_float2(nl, nl), ndi = make_float2(nd, nd);
      const int next = unit_of_round(uc + 1);
      if (next < units) {
        at = row_at(dq_unit(p, next));
        nl = __ldcg(p.nlse + at);
        nd = __ldcg(p.ndi + at);
      }
      for (int j = 0; j < c.n; ++j, ++n) {
        const uint32_t par = static_cast<uint32_t>(n) & 1u;
        const int k0 = j * kBlk + 32 * grp;  // this thread's first key
        // keys [k0, k0 + hi) are not after the query
        const uint32_t live = range_mask(0, qpos < c.b.y ? qpos + 1 - k0 : 0);
        ok = warp_wait2(&s_ready[par], static_cast<uint32_t>(n >> 1) & 1u, dp_ready, par, err, kErrWaitAccum);
        if (!ok) break;
        tc_fence_after();
        {
          uint32_t s[32], d[32];
          tmem_ld_32x32b_x32(col + par * 256, s);
          tmem_ld_32x32b_x32(col + 128, d);
          tmem_ld_wait();
          tc_fence_before();
          mbar_arrive_warp(sp_free);
          float2 e[16];
  #pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float2 a = __ffma2_rn(make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1])), sl2, nlse);
            const float2 t = __fadd2_rn(make_float2(__uint_as_float(d[2 * q]), __uint_as_float(d[2 * q + 1])), ndi);
            e[q] = __fmul2_rn(make_float2(exp2_approx(a.x), exp2_approx(a.y)), t);
          }
          keep_live(live, e);
          uint32_t w[16];
          pack16(e, w);
          tmem_st_32x32b_x16(col + par * 256, w);
          // S(n) has read K
          if ((j + 1) * kBlk > c.b.y) {
            clear_rows(smem_u32(smem) + kK + (n % 3) * kTile, c.b.y - j * kBlk, threadIdx.x - 128);
            fence_proxy_async_smem();
          }
          tmem_st_wait();
          tc_fence_before();
        }
        mbar_arrive_warp(&ds_ready[par]);
        if (j == 0 && uc > 0) ok = finish(last, uc - 1);
        if (!ok) break;
      }
      if (!ok) break;
      last = c;
    }
    if (ok && uc > 0) ok = finish(last, uc - 1);
    pdl_wait();  // the shares are written by the launch before this one
    if (ok) join_cut_walks(p, err);
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Before the products: -rowsum(dout * out) and -lse of every query row, in whole blocks
// (zeros behind a sequence's last row) so that a block's 512 bytes load aligned; and zeros
// in the gradients' rows of no sequence.  dout, out [tokens][QH][128]; 16 lanes take four
// consecutive rows of a head, 8 values of each per lane, all loads issued first.
constexpr int kRowsEach = 4;
constexpr int kRowThreads = 256;
__global__ void __launch_bounds__(kRowThreads) packed_rows_kernel(const __nv_bfloat16* __restrict__ dout,
                                                                  const __nv_bfloat16* __restrict__ out,
                                                                  const float* __restrict__ lse,
                                                                  float* __restrict__ ndi, float* __restrict__ nlse,
                                                                  const BwdParams p) {
  pdl_trigger();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.counter = 0u;
  if (!plan_ok(p.plan, p.tokens, p.plan_err)) return;
  const int lane = threadIdx.x & 15;
  // (block e, four rows of it, h), h fastest
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 16) + (threadIdx.x >> 4);
  const int64_t quad = i / p.QH;
  const int h = static_cast<int>(i - quad * p.QH);
  const int e = static_cast<int>(quad / (kBlk / kRowsEach));
  const int r = static_cast<int>(quad % (kBlk / kRowsEach)) * kRowsEach;
  if (e < p.plan.head->blocks) {  // whole half-warps alike
    const Block b = p.plan.natural[e];
    const int own = b.y - b.z * kBlk - r;  // of the four rows and those after them, the sequence's
    const int64_t row0 = b.x + b.z * kBlk + r;
    uint4 a[kRowsEach], o[kRowsEach];
#pragma unroll
    for (int k = 0; k < kRowsEach; ++k) {
      a[k] = o[k] = make_uint4(0u, 0u, 0u, 0u);
      if (k < own) {
        const int64_t row = (row0 + k) * p.QH + h;
        a[k] = __ldg(reinterpret_cast<const uint4*>(dout + row * kD) + lane);
        o[k] = __ldg(reinterpret_cast<const uint4*>(out + row * kD) + lane);
      }
    }
    const float l = lane < kRowsEach && lane < own ? -lse[static_cast<int64_t>(h) * p.tokens + row0 + lane] : 0.f;
    const unsigned mask = 0xffffu << (threadIdx.x & 16);
    float acc[kRowsEach];
#pragma unroll
    for (int k = 0; k < kRowsEach; ++k) {
      float fa[8], fo[8];
      unpack_bf16x8(a[k], fa);
      unpack_bf16x8(o[k], fo);
      acc[k] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[k] = fmaf(fa[j], fo[j], acc[k]);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) acc[k] += __shfl_xor_sync(mask, acc[k], d);
    }
    if (lane < kRowsEach) {
      const float v = lane == 0 ? acc[0] : lane == 1 ? acc[1] : lane == 2 ? acc[2] : acc[3];
      const int64_t at = h * p.sp + static_cast<int64_t>(e) * kBlk + r + lane;
      ndi[at] = -v;
      nlse[at] = l;
    }
  }
  if (p.zero_rest) {
    const PlanHead& g = *p.plan.head;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
    const int64_t count = static_cast<int64_t>(gridDim.x) * kRowThreads;
    zero_rest(p.dq, g.first, g.last, p.tokens, static_cast<int64_t>(p.QH) * kD * 2, at, count);
    zero_rest(p.dk, g.first, g.last, p.tokens, static_cast<int64_t>(p.KH) * kD * 2, at, count);
    zero_rest(p.dv, g.first, g.last, p.tokens, static_cast<int64_t>(p.KH) * kD * 2, at, count);
  }
}

inline size_t al256(size_t n) { return (n + 255) & ~size_t(255); }

// The most blocks that `tokens` rows of so many sequences can have, and how many CTAs
// share their walks.
int64_t most_blocks(int64_t tokens, int64_t sequences) { return tokens / kBlk + std::min(sequences, tokens); }
int64_t dkv_ctas(int64_t blocks, int64_t QH) {
  return std::min<int64_t>(num_sms(), std::min<int64_t>(blocks, 1024) * (std::min<int64_t>(blocks, 1024) + 1) / 2 * QH);
}

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" size_t kda_gqa_packed_backward_workspace_size(int64_t tokens, size_t plan_size, int64_t QH, int64_t KH,
                                                         int64_t D) {
  if (tokens <= 0 || tokens >= (1ll << 24) || QH <= 0 || KH <= 0 || QH % KH || D != kD || QH > 65535) return 0;
  const int64_t sequences = plan_sequences(tokens, plan_size);
  if (sequences == 0) return 0;
  const int64_t blocks = most_blocks(tokens, sequences);
  return 2 * al256(static_cast<size_t>(QH) * blocks * kBlk * 4) +
         static_cast<size_t>(dkv_ctas(blocks, QH)) * (4 * kBlk * kD * 4 + 32) + 16;
}

extern "C" kda_status kda_gqa_packed_backward_bf16(const void* dout, const void* q, const void* k, const void* v,
                                                   const void* out, const float* lse, const void* plan,
                                                   size_t plan_size, void* dq, void* dk, void* dv, int zero_rest,
                                                   int64_t tokens, int64_t QH, int64_t KH, int64_t D,
                                                   const int64_t* q_strides, const int64_t* k_strides,
                                                   const int64_t* v_strides, void* workspace, size_t workspace_bytes,
                                                   void* stream) {
  const char* op = "gqa_packed_backward";
  int64_t sequences = 0;
  KDA_PB_TRY(gqa_packed_check(op, tokens, QH, KH, D, plan, plan_size, &sequences));
  KDA_CHECK_ARG(dout && q && k && v && out && lse && dq && dk && dv && q_strides && k_strides && v_strides,
                "%s: null pointer", op);
  const int64_t qs[3] = {0, q_strides[0], q_strides[1]}, ks[3] = {0, k_strides[0], k_strides[1]},
                vs[3] = {0, v_strides[0], v_strides[1]};
  const int64_t dense_q[3] = {0, QH * kD, kD}, dense_k[3] = {0, KH * kD, kD};
  KDA_CHECK_SUPPORTED(head_rows_ok(q, qs, 1, tokens, QH) && head_rows_ok(k, ks, 1, tokens, KH) &&
                          head_rows_ok(v, vs, 1, tokens, KH) && head_rows_ok(dout, dense_q, 1, tokens, QH) &&
                          head_rows_ok(out, dense_q, 1, tokens, QH) && head_rows_ok(dq, dense_q, 1, tokens, QH) &&
                          head_rows_ok(dk, dense_k, 1, tokens, KH) && head_rows_ok(dv, dense_k, 1, tokens, KH) &&
                          (reinterpret_cast<uintptr_t>(lse) & 3u) == 0,
                      "%s: pointers and rows must be 16-byte aligned", op);
  const size_t need = kda_gqa_packed_backward_workspace_size(tokens, plan_size, QH, KH, D);
  KDA_CHECK_ARG(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes required, got %zu", op, need,
                workspace_bytes);
  KDA_CHECK_SUPPORTED((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "%s: workspace must be 16-byte aligned",
                      op);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t blocks = most_blocks(tokens, sequences), ctas = dkv_ctas(blocks, QH);
  // the longest run of a CTA, and the most units of a launch
  const int64_t deep = tokens / kBlk + 1;
  KDA_CHECK_SUPPORTED((deep * (deep + 1) / 2 + blocks) * QH < (1ll << 30) * ctas && blocks * QH < (1ll << 30),
                      "%s: too many rows (tokens=%lld QH=%lld sequences=%lld)", op, (long long)tokens, (long long)QH,
                      (long long)sequences);
  const size_t rows = al256(static_cast<size_t>(QH) * blocks * kBlk * 4);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  float* ndi = reinterpret_cast<float*>(w);
  float* nlse = reinterpret_cast<float*>(w + rows);
  BwdParams p{};
  p.plan = plan_view(plan, plan_blocks(tokens, sequences));
  p.tokens = static_cast<int>(tokens);
  p.QH = static_cast<int>(QH);
  p.KH = static_cast<int>(KH);
  p.rep = static_cast<int>(QH / KH);
  p.sp = blocks * kBlk;
  p.zero_rest = zero_rest;
  p.scale = 1.0f / sqrtf(static_cast<float>(kD));
  p.sl2 = p.scale * 1.4426950408889634f;
  p.nlse = nlse;
  p.ndi = ndi;
  p.partial = reinterpret_cast<float*>(w + 2 * rows);
  p.pieces = reinterpret_cast<int4*>(p.partial + ctas * 4 * kBlk * kD);
  p.counter = reinterpret_cast<unsigned*>(p.pieces + 2 * ctas);
  p.ctas = static_cast<int>(ctas);
  p.dq = static_cast<__nv_bfloat16*>(dq);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  p.plan_err = kda_err_ptr_packed_bwd_plan();
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    constexpr int bytes = static_cast<int>(Smem::kBytes);
    if (cudaFuncSetAttribute(packed_dkv_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        cudaFuncSetAttribute(packed_dq_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return launch_status("gqa_packed_backward: cudaFuncSetAttribute");
    attr_set[dev].store(true, std::memory_order_release);
  }
  // An ordinary launch: the next one's producers read the plan and load operands, and it
  // writes to the workspace, without waiting for this one.
  const int64_t groups = blocks * (kBlk / kRowsEach) * QH;
  packed_rows_kernel<<<dim3(static_cast<unsigned>((groups + kRowThreads / 16 - 1) / (kRowThreads / 16))), kRowThreads, 0,
                       st>>>(static_cast<const __nv_bfloat16*>(dout), static_cast<const __nv_bfloat16*>(out), lse, ndi,
                             nlse, p);
  KDA_PB_TRY(launch_status("gqa_packed_backward: rows"));
  // after a launch, which makes the device's context current in a thread that
  // has not used it yet (autograd's); the encoder is a driver call and needs one
  CUtensorMap tk, tv, tq, tdo;
  KDA_PB_TRY(tmap_head_rows(&tk, k, 1, tokens, KH, ks));
  KDA_PB_TRY(tmap_head_rows(&tv, v, 1, tokens, KH, vs));
  KDA_PB_TRY(tmap_head_rows(&tq, q, 1, tokens, QH, qs));
  KDA_PB_TRY(tmap_head_rows(&tdo, dout, 1, tokens, QH, dense_q));
  KDA_PB_TRY(launch_after("gqa_packed_backward: dk, dv", packed_dkv_kernel, dim3(static_cast<unsigned>(ctas)), kThreads,
                          Smem::kBytes, st, tk, tv, tq, tdo, p, kda_err_ptr_packed_bwd()));
  return launch_after("gqa_packed_backward: dq", packed_dq_kernel,
                      dim3(static_cast<unsigned>(std::min<int64_t>(blocks * QH, num_sms()))), kThreads, Smem::kBytes,
                      st, tk, tv, tq, tdo, p, kda_err_ptr_packed_bwd());
}
