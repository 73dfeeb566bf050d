// Grouped-query attention of one new token per request against a 4-bit key/value cache
// (layout: q4.cuh; head_dim 128).
//
// With n = lengths[b] cached tokens (the new one among them), query head h sees the keys
// j < n where j >= n - window or j < sinks:
//   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = q . k_j log2e / sqrt(128)
//
// Every block of 16 tokens with a visible one is read once (1,152 bytes for K and as many for V
// at groups of 64) for up to 16 query heads of its group.  That is the floor: 88.7 us for 64
// requests of 100 to 16,384 tokens, 32 query and 8 kv heads, which take 123.  Between the two lies a
// warp's chain from codes to products (integer pipe 59 %, issue 55 %, DRAM 54 %).  So codes become
// operands with little arithmetic, and steps and lows are applied to sums.  With x = step c + low, over a group G of channels
//   sum_G q x       = step sum_G q c + low sum_G q
//   sum_t p_t x_td  = sum_t (p_t step_t) c_td + sum_t p_t low_t
// The bits of a number below 2^-13 are linear in fp16: a byte in each half of a word is
// (c + 16 c') 2^-24 of two neighbouring codes as it stands, its low nibble c 2^-24.  So these
// two are operands, q' / 16 and q - q' / 16 what meets them in K, and in V the difference of
// the two sums is 16 times the second channel's: 4.5 integer operations for 8 codes.
// (As bf16 16 + code, the 16s subtracted from the sums: 241 us for 64 requests; as fp16
// code - 8 by one more multiply-add a pair: 194; a nibble each, a block at a time: 151;
// two blocks at a time: 139, and 124 for two kv heads together.)
// The other operands are fp16 then, with ranges of their own: q times a power of two per head
// that brings its largest value to 2^14 .. 2^15, and P' = p step times one per head that keeps it below
// 2^15 and was last chosen where the largest so far became 2^6 .. 2^7, in the manner of the running
// maximum.  fp16's last bit is 2^-24, so a weight times step is held to 2^-11 of itself or, where it is
// small, 2^-31 of the head's largest: between the groups of a head, whose channels are different
// outputs, steps may differ by 2^18 before the smaller's are off by more than bf16's rounding.  (The
// largest at 1 .. 2: 1.4 to 2.5 % off at 2^16, where rounding the result is 0.17 %.)
//
// The products are transposed so that the few query heads are the narrow side of the
// m16n8k16 matrix instruction:
//   S^T (16 keys x 8 heads)  = K q^T          O^T (128 x 8 heads) += V^T P^T
// The running maximum moves only when a score exceeds it by 2^8, room for which fp32 sums and the
// scale of the fp16 weights leave; so a block usually needs no exchange between lanes.
//
// A walk is a request's blocks of a kv head.  Short ones: a cluster of 1 to 16 CTAs for each; the
// blocks go to their warps in turn, each through a ring of bulk copies of its own, and the
// warps join through shared memory, the CTAs through the cluster's: one launch.
// Long ones: the walks, one behind the other, are cut into equal runs, one for each CTA
// (lengths are ragged and known on the device only); a run's blocks go to the CTA's warps in
// turn, the rings run on across the ends of walks.  Where a walk ends, or the run does, the
// warps join: a whole walk's output leaves, a cut one's share goes to the workspace, and a
// second launch joins the shares in the order of the walk.  The order of summation is fixed
// in both.
#include <cuda_fp16.h>
#include <math.h>

#include "launch.cuh"
#include "q4.cuh"
#include "window.cuh"

KDA_DEFINE_ERROR_WORD(q4_decode)
KDA_DEFINE_ERROR_WORD(q4_decode_length)  // a length past the cache: later calls' waits do not read it

namespace kda {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kRow = kD + 4;       // floats of a head's share: the output row, maximum, sum
constexpr int kLeast = kWarps;      // chunks of a CTA's run, where there are as many
constexpr unsigned kFull = 0xffffffffu;
// Weights are held as 2^(s - m - kUnder): a weight is 2^8 at most, so that sums of up to 2^24 values of any
// size stay finite in fp32, as the output is.  (Values below 2^-94 of the largest weight lose bits.)
constexpr int kUnder = 32;
constexpr int kTop = 126;           // P' is scaled by 2^kTop at most
constexpr int kWTop = 6;            // where the scale is chosen, a head's largest P' becomes 2^kWTop or twice that:
                                    // a weight may then grow by 2^8, as the reference lets it, within fp16

struct DecodeParams {
  const __nv_bfloat16* q;
  const uint8_t *k, *v;
  __nv_bfloat16* out;        // [B][QH][128]
  const int* lengths;
  int64_t q_b, q_h;          // element strides
  int64_t k_b, k_h, v_b, v_h;  // byte strides
  int cache_len, window, sinks;
  int B, QH, rep;
  int parts;                 // groups of 8 NT query heads per kv head; 0: two kv heads together
  int walks;                 // of a request
  float scale_log2;
  float* shares;             // [2 x CTAs][8 NT][kRow]
  int2* pieces;              // [2 x CTAs]: walk, chunks of the share (0: none)
  unsigned* length_err;
};

// Walk hp of a request: its (first) kv head and its query heads, which follow one another.
struct Heads {
  int kv, first, n;
};
__device__ __forceinline__ Heads heads_of(const DecodeParams& p, int most, int hp) {
  if (p.parts == 0) return {2 * hp, 2 * hp * p.rep, 2 * p.rep};
  const int g = hp / p.parts, part = hp - g * p.parts;
  return {g, g * p.rep + part * most, min(most, p.rep - part * most)};
}

// A request's visible tokens as chunks of PER blocks of each of the walk's kv heads: `ns` over
// blocks [0, sb) (sinks), then those over [first, end).
struct Walk {
  int n, ns, sb, first, end;
  int len, start;
};
template <int PER>
__device__ __forceinline__ Walk walk_of(const DecodeParams& p, int b) {
  Walk w;
  w.len = max(0, min(__ldg(p.lengths + b), p.cache_len));  // the cache's end is the end (reported elsewhere)
  w.start = max(0, w.len - p.window);
  w.first = w.start >> 4;
  w.end = (w.len + kQ4Tokens - 1) >> 4;
  w.sb = min((min(p.sinks, w.start) + kQ4Tokens - 1) >> 4, w.first);
  w.ns = (w.sb + PER - 1) / PER;
  w.n = w.ns + (w.end - w.first + PER - 1) / PER;
  return w;
}
// Chunk x's first block, and whether it has a second one.
template <int PER>
__device__ __forceinline__ int block_of(const Walk& w, int x) {
  return x < w.ns ? PER * x : w.first + PER * (x - w.ns);
}
__device__ __forceinline__ bool second_of(const Walk& w, int x, int block) { return block + 1 < (x < w.ns ? w.sb : w.end); }

// Where a run stands: chunk x of walk (b, hp).
struct Cursor {
  int b, hp, x;
  Walk w;
};
// `by` chunks on, over the ends of walks (those of requests without tokens are empty).
template <int PER>
__device__ __forceinline__ void move(const DecodeParams& p, Cursor* c, int by) {
  c->x += by;
  while (c->x >= c->w.n) {
    c->x -= c->w.n;
    if (++c->hp == p.walks) {
      c->hp = 0;
      do {
        if (++c->b >= p.B) return;  // past the last walk: not read
        c->w = walk_of<PER>(p, c->b);
      } while (c->w.n == 0);
    }
  }
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
constexpr uint32_t kEven = 0x000f000fu;
constexpr float kUnit = 16777216.f;  // 2^24
constexpr int kQTop = 14;            // q's operands: a head's largest |q| becomes 2^14 to 2^15
// Bytes 0 and 2 (second: 1 and 3) of a word, in its halves.
__device__ __forceinline__ uint32_t bytes_of(uint32_t w, int second) {
  return second ? __byte_perm(w, 0u, 0x4341) : w & 0x00ff00ffu;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The exponent field of a float that is not negative, within [lo, hi]; and 2^(e - 127).
__device__ __forceinline__ int exponent(float x, int lo, int hi) {
  return min(max(static_cast<int>(__float_as_uint(x) >> 23), lo), hi);
}
__device__ __forceinline__ float power(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }
template <int N>
__device__ __forceinline__ void ld_shared_n(uint32_t addr, uint32_t (&r)[N]) {
  if constexpr (N == 1) {
    r[0] = ld_shared(addr);
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
  } else {
    const uint4 v = ld_shared_v4(addr);
    r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
  }
}
__device__ __forceinline__ float step_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float low_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// The weight of a share with maximum m among shares whose maximum is mm.  One that saw
// nothing finite has sums of zeros, which may be added as they are, or of NaN, which must be.
__device__ __forceinline__ float share_weight(float m, float mm) { return m == -INFINITY ? 1.f : exp2_approx(m - mm); }

// a / b, neither negative; most fit in 32 bits, where a division takes a fifth of the time.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? static_cast<unsigned>(a) / static_cast<unsigned>(b) : a / b;
}

// Whether the warps' shares lie without gaps between rows: with groups of 32 and 8 heads two CTAs find no
// room on an SM otherwise.  (64 requests of 1 to 8,192 tokens: 4 query heads for each of 8 kv heads, two
// together, 110 us with gaps, 87 without; 8 148 and 135.  Elsewhere gaps are up to 5 % faster.)
constexpr bool compact_rows(int nt, int group, int warps) { return nt == 1 && group == 32 && warps == 8; }

// NT: groups of 8 query heads a CTA works on.  PAIR: two kv heads of at most 4 query heads each;
// a tile of 16 rows of the matrix instruction is then 8 tokens of either, and of S^T the two
// quarters count in which rows and columns are of one kv head: a lane's two values instead of
// four for the same codes, half of the work between the products (64 requests, 4 query heads for
// each of 8 kv heads: 139 us without, 124 with).
// CLUSTER: no runs; the CTAs of a cluster share one walk; grid (cluster size, walks, B).
template <int NT, int GROUP, int STAGES, bool PAIR, bool CLUSTER, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, NT == 1 && WARPS == 8 ? 2 : 1)
    q4_decode_kernel(const DecodeParams p, unsigned* err) {
  constexpr int H = 8 * NT, THREADS = 32 * WARPS;
  constexpr int NG = 128 / GROUP;                       // pairs of a token
  constexpr int RUNS = 4 / NG;                          // 32-channel runs of a group
  constexpr uint32_t kBlock = q4_block_bytes(GROUP);
  constexpr uint32_t kStage = 4 * kBlock;               // a chunk's blocks of K, then of V
  constexpr int PER = PAIR ? 1 : 2;                     // blocks of a chunk, of each kv head
  constexpr int ROWS = PAIR ? 1 : 2;                    // tokens of a lane in a tile of S^T
  static_assert(!PAIR || (NT == 1 && !CLUSTER), "8 columns, runs");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[WARPS][STAGES];
  __shared__ int64_t sums[WARPS];
  __shared__ int first_b;
  __shared__ int64_t first_x;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int r = lane >> 2, c4 = lane & 3;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(&full[warp][s], 1);
    fence_mbar_init();
  }
  pdl_trigger();
  pdl_wait();

  Cursor at;  // of the piece in work
  int run, cta = 0, rank = 0, size = 1;
  if constexpr (CLUSTER) {
    rank = static_cast<int>(cluster_ctarank());
    size = static_cast<int>(gridDim.x);
    at.b = blockIdx.z;
    at.hp = blockIdx.y;
    at.x = 0;
    at.w = walk_of<PER>(p, at.b);
    run = at.w.n;
    if (threadIdx.x == 0 && rank == 0 && at.hp == 0 && __ldg(p.lengths + at.b) > p.cache_len)
      atomicOr(p.length_err, static_cast<unsigned>(kErrRange));
    if (run == 0) {  // no tokens
      const Heads hs = heads_of(p, H, at.hp);
      uint4* out = reinterpret_cast<uint4*>(p.out + (static_cast<int64_t>(at.b) * p.QH + hs.first) * kD);
      if (rank == 0)
        for (int i = threadIdx.x; i < hs.n * (kD / 8); i += THREADS) out[i] = make_uint4(0u, 0u, 0u, 0u);
      return;
    }
  } else {
    if (threadIdx.x == 0) p.pieces[2 * blockIdx.x] = p.pieces[2 * blockIdx.x + 1] = make_int2(0, 0);
    // The run: chunks [r0, r1) of all walks.  Each thread counts the requests [b0, b1).
    const int heads = p.walks;
    const int each = (p.B + THREADS - 1) / THREADS;
    const int b0 = min(static_cast<int>(threadIdx.x) * each, p.B), b1 = min(b0 + each, p.B);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += walk_of<PER>(p, b).n;
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(kFull, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += sums[w];
      total += sums[w];
    }
    total *= heads;
    const int ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total / kLeast > 0 ? total / kLeast : 1));
    cta = static_cast<int>(blockIdx.x);
    // equal runs: [total c / ctas, total (c + 1) / ctas)
    const int64_t each_run = divide(total, ctas);
    const unsigned longer = static_cast<unsigned>(total - each_run * ctas), n_ctas = static_cast<unsigned>(ctas);
    const int64_t r0 = cta * each_run + longer * static_cast<unsigned>(cta) / n_ctas;
    const int64_t r1 = (cta + 1) * each_run + longer * static_cast<unsigned>(cta + 1) / n_ctas;
    run = cta < ctas ? static_cast<int>(r1 - r0) : 0;
    if (run > 0 && before * heads <= r0 && r0 < (before + mine) * heads) {
      int64_t x = before;
      int b = b0, n = walk_of<PER>(p, b).n;
      while (n == 0 || (x + n) * heads <= r0) {
        x += n;
        n = walk_of<PER>(p, ++b).n;
      }
      first_b = b;
      first_x = r0 - x * heads;
    }
    __syncthreads();
    // outputs of requests without tokens, and lengths past the cache
    for (int b = cta; b < p.B; b += gridDim.x) {
      const int n = __ldg(p.lengths + b);
      if (threadIdx.x == 0 && n > p.cache_len) atomicOr(p.length_err, static_cast<unsigned>(kErrRange));
      if (n <= 0)
        for (int i = threadIdx.x; i < p.QH * (kD / 8); i += THREADS)
          reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(b) * p.QH * kD)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if (run == 0) return;
    at.b = first_b;
    at.w = walk_of<PER>(p, at.b);
    at.hp = static_cast<int>(divide(first_x, at.w.n));
    at.x = static_cast<int>(first_x - static_cast<int64_t>(at.hp) * at.w.n);
  }

  // this warp's chunks: first, first + stride, ... of the run
  const int first = rank * WARPS + warp, stride = CLUSTER ? size * WARPS : WARPS;
  uint8_t* ring = smem + warp * (STAGES * kStage);
  Cursor ahead = at;  // of the next load
  if (CLUSTER) ahead.x = first;
  else if (warp > 0) move<PER>(p, &ahead, warp);
  int loads = 0;
  // Loads one behind the other in a walk are `stride` chunks apart: `left` of them, of so many bytes.
  int left = 0;
  uint32_t bytes = 0;
  const uint8_t *kp = nullptr, *vp = nullptr;
  auto load = [&]() {
    if (first + loads * stride >= run) return;
    if (left == 0) {
      if (!CLUSTER && loads > 0) move<PER>(p, &ahead, 0);
      const int g = heads_of(p, H, ahead.hp).kv, block = block_of<PER>(ahead.w, ahead.x);
      const int whole = ahead.x < ahead.w.ns ? ahead.w.sb / PER : ahead.w.ns + (ahead.w.end - ahead.w.first) / PER;
      left = max(1, (whole - ahead.x + stride - 1) / stride);
      bytes = ahead.x < whole ? PER * kBlock : kBlock;
      const int64_t off = static_cast<int64_t>(block) * kBlock;
      kp = p.k + ahead.b * p.k_b + g * p.k_h + off;
      vp = p.v + ahead.b * p.v_b + g * p.v_h + off;
    }
    const int s = loads % STAGES;
    if (lane == 0) {
      uint8_t* dst = ring + s * kStage;
      mbar_arrive_expect_tx(&full[warp][s], PAIR ? 4 * kBlock : 2 * bytes);
      bulk_load_1d(dst, kp, bytes, &full[warp][s]);
      bulk_load_1d(dst + 2 * kBlock, vp, bytes, &full[warp][s]);
      if (PAIR) {  // the second kv head's
        bulk_load_1d(dst + kBlock, kp + p.k_h, kBlock, &full[warp][s]);
        bulk_load_1d(dst + 3 * kBlock, vp + p.v_h, kBlock, &full[warp][s]);
      }
    }
    ++loads;
    --left;
    kp += PER * stride * kBlock;
    vp += PER * stride * kBlock;
    ahead.x += stride;
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load();

  // [WARPS][held][kRow], in the rings' place at the end where they leave no room for it.  (COMPACT:
  // [WARPS][held][kD], columns exchanged so that the heads which a warp writes at once meet different
  // banks, then each row's maximum and sum.)
  float* parts = reinterpret_cast<float*>(smem + (WARPS == 16 ? 0 : WARPS * STAGES * kStage));
  const int held = PAIR ? 2 * p.rep : min(p.rep, H);
  constexpr bool COMPACT = compact_rows(NT, GROUP, WARPS);
  constexpr int kPart = COMPACT ? kD : kRow;
  auto top_at = [&](int i) { return COMPACT ? WARPS * held * kD + 2 * i : i * kRow + kD; };  // of row i's maximum, sum
  auto swap = [](int i) { return COMPACT ? (i & 6) << 2 : 0; };
  bool ok = true;
  int done = 0;       // this warp's chunks
  int piece_at = 0;   // the piece's first chunk in the run
  while (piece_at < run) {
    const int left = run - piece_at;
    const int n = min(left, at.w.n - at.x);  // chunks of the piece
    const Heads hs = heads_of(p, H, at.hp);
    const int h0 = hs.first, nh = hs.n;
    // the place among them of column h of a tile, or nh: of none
    auto head_at = [&](int h) { return PAIR ? ((h & 3) < p.rep ? (h >> 2) * p.rep + (h & 3) : nh) : h; };

    // q^T operands: for run g and step s of its two, head lane / 4, channels of this lane's
    // word: (2 s, 2 s + 4) less a sixteenth of (2 s + 1, 2 s + 5), and the latter, times a
    // power of two; and for the heads of
    // this lane's accumulators, 2 (lane % 4) + {0, 1}, the sums over groups and the factor
    // that makes scores of the products
    uint32_t qf[NT][4][2][2];
    float qsum[NT][NG][2], sl2[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int h = head_at(t * 8 + r);
      float f[4][8], top = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 w = h < nh ? __ldg(reinterpret_cast<const uint4*>(p.q + at.b * p.q_b +
                                                                      static_cast<int64_t>(h0 + h) * p.q_h + 32 * k) + c4)
                               : make_uint4(0u, 0u, 0u, 0u);
        unpack_bf16x8(w, f[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[k][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
      // 2^14 and not 1: what f0 brings up, `back` does not have to, which then is finite below |q| = 2^121
      const int ex = exponent(top, 1 + kQTop, 253);
      const float f0 = power(254 + kQTop - ex);
      float sum[NG];
#pragma unroll
      for (int j = 0; j < NG; ++j) sum[j] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f1 = f0 * 0.0625f;
          qf[t][k][i >> 1][i & 1] = (i & 1) ? pack_f16x2(f[k][i] * f1, f[k][i + 4] * f1)
                                            : pack_f16x2(fmaf(f[k][i + 1], -f1, f[k][i] * f0),
                                                         fmaf(f[k][i + 5], -f1, f[k][i + 4] * f0));
          sum[k / RUNS] += (f[k][i] + f[k][i + 4]) * (f0 / kUnit);  // in the products' unit
        }
      const float back = power(ex) * (p.scale_log2 * (kUnit / (1 << kQTop)));
      sl2[t][0] = __shfl_sync(kFull, back, 8 * c4);
      sl2[t][1] = __shfl_sync(kFull, back, 8 * c4 + 4);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        sum[j] += __shfl_xor_sync(kFull, sum[j], 1);
        sum[j] += __shfl_xor_sync(kFull, sum[j], 2);
        qsum[t][j][0] = __shfl_sync(kFull, sum[j], 8 * c4);
        qsum[t][j][1] = __shfl_sync(kFull, sum[j], 8 * c4 + 4);
      }
    }
    float nm[NT][2];                // -m - kUnder, or zero where that is infinite
    float m[NT][2], l[NT][2];       // heads 8 t + 2 (lane % 4) + {0, 1}; l: this lane's keys only
    int vs[NT][2];                  // P' = 2^(vs - 127) p step
    float lows[NT][NG][2];          // sums of p low, this lane's keys only
    // run, step: channels 32 run + 4 (lane / 4) + 2 step, of P' c 2^-24, and + 1, of P' (c + 16 c') 2^-24
    float o[NT][4][2][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      nm[t][0] = nm[t][1] = 0.f;
      l[t][0] = l[t][1] = 0.f;
      vs[t][0] = vs[t][1] = 127 + kTop;
#pragma unroll
      for (int j = 0; j < NG; ++j) lows[t][j][0] = lows[t][j][1] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int s = 0; s < 2; ++s) o[t][k][s][0] = o[t][k][s][1] = o[t][k][s][2] = o[t][k][s][3] = 0.f;
    }

    // chunks [xa, xb) are visible whole
    const int xa = at.w.ns + ((at.w.start & (kQ4Tokens - 1)) != 0);
    const int xb = at.w.ns + (at.w.len - at.w.first * kQ4Tokens) / (PER * kQ4Tokens);
    const int x_end = at.x + n;
    for (int x = at.x + first + done * stride - piece_at; ok && x < x_end; ++done, x += stride) {
      __syncwarp();  // every lane is done with the stage refilled here
      load();
      const int s = done % STAGES;
      if (!warp_wait(&full[warp][s], static_cast<uint32_t>(done / STAGES) & 1u, err, kErrWaitFull)) {
        ok = false;
        break;
      }
      const bool whole = x >= xa && x < xb;
      const uint32_t ks = smem_u32(ring) + s * kStage, vb = ks + 2 * kBlock;
      // Tile i of the two: block i, the tokens of this lane's accumulators its r and r + 8; or
      // (PAIR) tokens 8 i on of one block of two kv heads, this lane's r of the head of its columns.
      bool see[2][ROWS];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < ROWS; ++c) see[i][c] = true;
      if (!whole) {
        const int block = block_of<PER>(at.w, x);
        const bool two = PAIR || second_of(at.w, x, block);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < ROWS; ++c) {
            const int tok = PAIR ? block * kQ4Tokens + 8 * i + r : (block + i) * kQ4Tokens + r + 8 * c;
            see[i][c] = (i == 0 || two) && tok < at.w.len && (tok >= at.w.start || tok < p.sinks);
          }
      }
      // rows r and r + 8 of tile i, and the pairs of this lane's tokens, in a block of K or of V
      auto row_at = [&](uint32_t base, int i, int c) {
        return base + (PAIR ? c * kBlock + (8 * i + r) * 64 : i * kBlock + (r + 8 * c) * 64);
      };
      auto pairs_at = [&](uint32_t base, int i, int c) {
        return base + kQ4Codes + (PAIR ? (c4 >> 1) * kBlock + (8 * i + r) * NG * 4 : i * kBlock + (r + 8 * c) * NG * 4);
      };

      float sc[2][NT][2 * ROWS];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t chunk = (c4 ^ ((r >> 1) & 3)) << 4;  // chunk lane % 4 of tokens r (+ 8)
        const uint4 k0 = ld_shared_v4(row_at(ks, i, 0) + chunk), k1 = ld_shared_v4(row_at(ks, i, 1) + chunk);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
        uint32_t pr[ROWS][NG];
#pragma unroll
        for (int c = 0; c < ROWS; ++c) ld_shared_n<NG>(pairs_at(ks, i, c), pr[c]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 2 * ROWS; ++c) sc[i][t][c] = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float acc[NT][4];
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
          for (int k = j * RUNS; k < (j + 1) * RUNS; ++k)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              const uint32_t b0 = bytes_of(w0[k], st), b1 = bytes_of(w1[k], st);
              const uint32_t a[4] = {b0 & kEven, b1 & kEven, b0, b1};
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_f16(acc[t], a, qf[t][k][st][0], qf[t][k][st][1]);
            }
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < 2 * ROWS; ++c) {
              const float dot = PAIR ? (c4 < 2 ? acc[t][c] : acc[t][c + 2]) : acc[t][c];
              sc[i][t][c] = fmaf(step_of(pr[c >> 1][j]), dot, fmaf(low_of(pr[c >> 1][j]), qsum[t][j][c & 1], sc[i][t][c]));
            }
        }
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < 2 * ROWS; ++c)
              if (!see[i][c >> 1]) sc[i][t][c] = -INFINITY;
      }
      // the highest of this lane's scores of head c
      auto most = [&](int t, int c) {
        return PAIR ? fmaxf(sc[0][t][c], sc[1][t][c])
                    : fmaxf(fmax3(sc[0][t][c], sc[0][t][(c + 2) % (2 * ROWS)], sc[1][t][c]), sc[1][t][(c + 2) % (2 * ROWS)]);
      };
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          grow |= most(t, c) * sl2[t][c] > m[t][c] + 8.f;
      if (__any_sync(kFull, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = most(t, c) * sl2[t][c];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, d));
            const float ref = fmaxf(mx, m[t][c]) + kUnder;
            mx = ref - kUnder;  // what the weights go by, after ref's rounding
            // nothing finite yet: keep the (empty) sums as they are
            const float f = mx == -INFINITY ? 1.f : exp2_approx(m[t][c] - mx);
            // what the old sums lose, P' gains, rounded up: however often m moves, the scale does not fall behind
            const int up = min(127 + kTop - vs[t][c], __float2int_ru(fminf(mx - m[t][c], 1000.f)));
            const float fo = mx == -INFINITY ? 1.f : exp2_approx(m[t][c] - mx + static_cast<float>(up));
            vs[t][c] += mx == -INFINITY ? 0 : up;
            m[t][c] = mx;
            nm[t][c] = mx == -INFINITY ? 0.f : -ref;
            l[t][c] *= f;
#pragma unroll
            for (int j = 0; j < NG; ++j) lows[t][j][c] *= f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int st = 0; st < 2; ++st) {
                o[t][k][st][c] *= fo;
                o[t][k][st][c + 2] *= fo;
              }
          }
      }
      float e[2][NT][2 * ROWS];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 2 * ROWS; ++c) {
            e[i][t][c] = exp2_approx(fmaf(sc[i][t][c], sl2[t][c & 1], nm[t][c & 1]));
            l[t][c & 1] += e[i][t][c];
          }
      // P' = p step 2^vs, which meets the codes as fp16, the tensor core's operand type
      uint32_t pp[2][NT][NG][ROWS];
      float top = 0.f;
      auto load_pairs = [&](int i, uint32_t (&pr)[ROWS][NG]) {
#pragma unroll
        for (int c = 0; c < ROWS; ++c) {
          ld_shared_n<NG>(pairs_at(vb, i, c), pr[c]);
          if (!whole) {
#pragma unroll
            for (int j = 0; j < NG; ++j)  // whatever is there must not meet its weight of zero
              if (!see[i][c]) pr[c][j] = 0u;
          }
        }
      };
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t pr[ROWS][NG];
        load_pairs(i, pr);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float v[2] = {power(vs[t][0]), power(vs[t][1])};
#pragma unroll
          for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int c = 0; c < ROWS; ++c) {
              const float step = step_of(pr[c][j]), low = low_of(pr[c][j]);
              const float p0 = e[i][t][2 * c] * v[0] * step, p1 = e[i][t][2 * c + 1] * v[1] * step;
              lows[t][j][0] = fmaf(e[i][t][2 * c], low, lows[t][j][0]);
              lows[t][j][1] = fmaf(e[i][t][2 * c + 1], low, lows[t][j][1]);
              top = fmax3(top, p0, p1);
              pp[i][t][j][c] = pack_f16x2(p0, p1);
            }
        }
      }
      if (__any_sync(kFull, top > 32768.f)) {
        uint32_t pr[2][ROWS][NG];
#pragma unroll
        for (int i = 0; i < 2; ++i) load_pairs(i, pr[i]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float v[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float high = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int d = 0; d < ROWS; ++d) high = fmaxf(high, e[i][t][2 * d + c] * step_of(pr[i][d][j]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) high = fmaxf(high, __shfl_xor_sync(kFull, high, d));
            const int to = min(vs[t][c], 254 + kWTop - exponent(high, 127 - kTop + kWTop, 230));
            const float f = exp2_approx(static_cast<float>(to - vs[t][c]));
            vs[t][c] = to;
            v[c] = power(to);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int st = 0; st < 2; ++st) {
                o[t][k][st][c] *= f;
                o[t][k][st][c + 2] *= f;
              }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
              for (int c = 0; c < ROWS; ++c) {
                const float step = step_of(pr[i][c][j]);
                pp[i][t][j][c] = pack_f16x2(e[i][t][2 * c] * v[0] * step, e[i][t][2 * c + 1] * v[1] * step);
              }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // tokens 2 (lane % 4) + {0, 1} of a tile's first 8 rows and of the others: their chunk
        // r / 2, of which this lane takes half of each word: channels 32 run + 4 r + {0 .. 3}
        const uint32_t in = c4 * 128 + (((r >> 1) ^ c4) << 4);
        const uint32_t col = vb + in + (PAIR ? i * 512 : i * kBlock), other = col + (PAIR ? kBlock : 512);
        const uint4 va = ld_shared_v4(col), vc = ld_shared_v4(col + 64), vd = ld_shared_v4(other),
                    ve = ld_shared_v4(other + 64);
        const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vc.x, vc.y, vc.z, vc.w},
                       wc[4] = {vd.x, vd.y, vd.z, vd.w}, wd[4] = {ve.x, ve.y, ve.z, ve.w};
        const uint32_t pick = (r & 1) ? 0x7632u : 0x5410u;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          uint32_t pb[NT][2];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            // (PAIR: the rows of the other kv head weigh nothing)
            pb[t][0] = transpose8x8(PAIR && c4 >= 2 ? 0u : pp[i][t][j][0]);
            pb[t][1] = transpose8x8(PAIR && c4 < 2 ? 0u : pp[i][t][j][ROWS - 1]);
          }
#pragma unroll
          for (int k = j * RUNS; k < (j + 1) * RUNS; ++k) {
            const uint32_t lo = __byte_perm(wa[k], wb[k], pick), hi = __byte_perm(wc[k], wd[k], pick);
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              const uint32_t b0 = bytes_of(lo, st), b1 = bytes_of(hi, st);
              const uint32_t a[4] = {b0 & kEven, b0, b1 & kEven, b1};
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_f16(o[t][k][st], a, pb[t][0], pb[t][1]);
            }
          }
        }
      }
    }

    // the piece's end: this warp's share, then all of them
    if (WARPS == 16) __syncthreads();  // the rings are read
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = head_at(t * 8 + 2 * c4 + c);
        float sum = l[t][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(kFull, sum, d);
        float add[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          add[j] = lows[t][j][c];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) add[j] += __shfl_xor_sync(kFull, add[j], d);
        }
        if (h < nh) {
          float* dst = parts + (warp * held + h) * kPart;
          const float f0 = power(254 - vs[t][c]) * kUnit, f1 = f0 * 0.0625f;  // vs >= 32: 2^119 at most
          if (r == 0) {
            float* top = parts + top_at(warp * held + h);
            top[0] = m[t][c];
            top[1] = sum;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int st = 0; st < 2; ++st)
              *reinterpret_cast<float2*>(dst + ((32 * k + 4 * r + 2 * st) ^ swap(warp * held + h))) =
                  make_float2(fmaf(o[t][k][st][c], f0, add[k / RUNS]),
                              fmaf(o[t][k][st][c + 2] - o[t][k][st][c], f1, add[k / RUNS]));
        }
      }
    __syncthreads();
    const bool cut = n < at.w.n;  // (never in a cluster)
    float* joined = WARPS == 16 ? parts + WARPS * held * kRow : reinterpret_cast<float*>(smem);  // rings are read
    const int slot = 2 * cta + (at.x == 0 ? 1 : 0);
    for (int i = threadIdx.x; i < nh * (kD / 4); i += THREADS) {  // four columns of a head
      const int h = i / (kD / 4), d = i % (kD / 4) * 4;
      float mw[WARPS], mm = -INFINITY, ll = 0.f;
      float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        mw[w] = parts[top_at(w * held + h)];
        mm = fmaxf(mm, mw[w]);
      }
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float* src = parts + (w * held + h) * kPart;
        const float f = share_weight(mw[w], mm);
        const float4 v = *reinterpret_cast<const float4*>(src + (d ^ swap(w * held + h)));
        ll += f * parts[top_at(w * held + h) + 1];
        oo.x += f * v.x, oo.y += f * v.y, oo.z += f * v.z, oo.w += f * v.w;
      }
      if (cut || size > 1) {
        float* dst = size > 1 ? joined + h * kRow : p.shares + (static_cast<int64_t>(slot) * H + h) * kRow;
        *reinterpret_cast<float4*>(dst + d) = oo;
        if (d == 0) {
          dst[kD] = mm;
          dst[kD + 1] = ll;
        }
      } else {
        *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(at.b) * p.QH + h0 + h) * kD + d) =
            make_uint2(pack_bf16x2(oo.x / ll, oo.y / ll), pack_bf16x2(oo.z / ll, oo.w / ll));
      }
    }
    if (cut && threadIdx.x == 0) p.pieces[slot] = make_int2(at.b * p.walks + at.hp, n);
    if (CLUSTER && size > 1) {
      cluster_sync_all();
      const uint32_t base = smem_u32(joined);
      for (int i = rank * THREADS + threadIdx.x; i < nh * (kD / 4); i += size * THREADS) {
        const int h = i / (kD / 4), d = i % (kD / 4) * 4;
        float mm = -INFINITY, ll = 0.f;
        float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < size; ++c) mm = fmaxf(mm, ld_cluster_f32(mapa_shared(base + (h * kRow + kD) * 4, c)));
#pragma unroll 4
        for (int c = 0; c < size; ++c) {
          const uint32_t src = mapa_shared(base + h * kRow * 4, c);
          const float f = share_weight(ld_cluster_f32(src + kD * 4), mm);
          const float4 v = ld_cluster_f32x4(src + d * 4);
          ll += f * ld_cluster_f32(src + kD * 4 + 4);
          oo.x += f * v.x, oo.y += f * v.y, oo.z += f * v.z, oo.w += f * v.w;
        }
        *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(at.b) * p.QH + h0 + h) * kD + d) =
            make_uint2(pack_bf16x2(oo.x / ll, oo.y / ll), pack_bf16x2(oo.z / ll, oo.w / ll));
      }
      cluster_sync_all();  // a CTA's sums are read until here
    }
    __syncthreads();  // parts are free
    piece_at += n;
    if (!CLUSTER && piece_at < run) move<PER>(p, &at, n);
  }
  if (!ok && lane == 0) {  // no copy may still be writing shared memory when the CTA exits
    for (int i = max(0, loads - STAGES); i < loads; ++i)
      mbar_drain(&full[warp][i % STAGES], static_cast<uint32_t>(i / STAGES) & 1u);
  }
}

// The shares of cut walks, added in the order of the walk.  Block x: the walk that CTA x
// began and did not end; y: a head of its; 8 warps take the shares in turn.
template <int H>
__global__ void __launch_bounds__(kThreads) q4_join_kernel(const DecodeParams p, int ctas) {
  __shared__ __align__(16) float parts[kWarps][kRow];
  pdl_trigger();
  pdl_wait();
  // What may be this walk's is asked for at once, whether or not it is: the piece, the next
  // ones, and the shares' maxima (a share's memory is there in any case).
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y;
  const int x = static_cast<int>(blockIdx.x);
  // share i: slot 2 x + 1, then 2 (x + 1), 2 (x + 2), ..., while they are of this walk
  auto share = [&](int i) {
    const int slot = i == 0 ? 2 * x + 1 : 2 * min(x + i, ctas - 1);
    return p.shares + (static_cast<int64_t>(slot) * H + h) * kRow;
  };
  const int2 w = p.pieces[2 * x + 1];
  int2 next = p.pieces[2 * min(x + 1 + lane, ctas - 1)];
  float mm = share(lane)[kD];
  const int b = w.x / p.walks;
  const Heads hs = heads_of(p, H, w.x - b * p.walks);
  if (w.y == 0 || h >= hs.n) return;
  int count = 1;
  for (;;) {
    const unsigned others = ~__ballot_sync(kFull, x + count + lane < ctas && next.y > 0 && next.x == w.x);
    count += others ? __ffs(static_cast<int>(others)) - 1 : 32;
    if (others) break;
    next = p.pieces[2 * min(x + count + lane, ctas - 1)];
  }
  if (lane >= count) mm = -INFINITY;
  for (int i = lane + 32; i < count; i += 32) mm = fmaxf(mm, share(i)[kD]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(kFull, mm, d));
  float ll = 0.f;
  float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < count; i += kWarps) {
    const float* src = share(i);
    const float f = share_weight(src[kD], mm);
    const float4 v = reinterpret_cast<const float4*>(src)[lane];
    ll += f * src[kD + 1];
    oo.x += f * v.x, oo.y += f * v.y, oo.z += f * v.z, oo.w += f * v.w;
  }
  reinterpret_cast<float4*>(parts[warp])[lane] = oo;
  if (lane == 0) parts[warp][kD + 1] = ll;
  __syncthreads();
  if (threadIdx.x < kD) {
    const int d = threadIdx.x;
    float l2 = 0.f, o2 = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      l2 += parts[i][kD + 1];
      o2 += parts[i][d];
    }
    p.out[(static_cast<int64_t>(b) * p.QH + hs.first + h) * kD + d] = __float2bfloat16_rn(o2 / l2);
  }
}

// cluster: CTAs that share a walk, or 0: runs over `ctas` CTAs and a second launch.
template <int NT, int GROUP, bool PAIR, bool CLUSTER, int WARPS = kWarps>
kda_status launch_decode(const DecodeParams& p, int ctas, int cluster, cudaStream_t st) {
  // rings of the depth that leaves two CTAs an SM (one where a group has more than 8 heads; a
  // cluster's short walks are 1 to 3 % faster with 3 stages there than with 4)
  constexpr int kStages = NT == 1 ? 2 : CLUSTER ? 3 : 4;
  constexpr int H = 8 * NT;
  constexpr int kRing = WARPS * kStages * 4 * q4_block_bytes(GROUP);
  constexpr int kRows = WARPS * (compact_rows(NT, GROUP, WARPS) ? kD + 2 : kRow) * 4;
  static_assert((WARPS + 1) * H * kRow * 4 <= kRing, "shares in the rings' place");
  auto bytes = [](int held) { return static_cast<size_t>(kRing + (WARPS == 16 ? 0 : held * kRows)); };
  // an SM's 228 KB hold each CTA's static part (barriers and the run's place) and 1 KB of the system's too
  constexpr int kStatic = (WARPS * kStages * 8 + WARPS * 8 + 16 + 127) / 128 * 128;
  static_assert(kRing + (WARPS == 16 ? 0 : H * kRows) + kStatic + 1024 <= (NT == 1 && WARPS == 8 ? 114 : 228) * 1024,
                "shared memory budget");
  auto* kernel = q4_decode_kernel<NT, GROUP, kStages, PAIR, CLUSTER, WARPS>;
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes(H))) !=
            cudaSuccess ||
        (CLUSTER && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess))
      return launch_status("gqa_decode_q4: cudaFuncSetAttribute");
    attr_set[dev].store(true, std::memory_order_release);
  }
  const int held = PAIR ? 2 * p.rep : p.rep < H ? p.rep : H;  // query heads of a walk
  if (CLUSTER) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(cluster), static_cast<unsigned>(p.walks), static_cast<unsigned>(p.B));
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = bytes(held);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kernel, p, kda_err_ptr_q4_decode());
    return launch_status("gqa_decode_q4");
  }
  const kda_status s = launch_after("gqa_decode_q4", kernel, dim3(static_cast<unsigned>(ctas)), kThreads, bytes(held), st,
                                    p, kda_err_ptr_q4_decode());
  if (s != KDA_OK) return s;
  return launch_after("gqa_decode_q4: join", q4_join_kernel<H>, dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(held)),
                      kThreads, 0, st, p, ctas);
}
// CTAs that share a walk, of so many warps; 0: runs.
struct Cluster {
  int64_t ctas, warps;
};
template <int GROUP>
kda_status launch_group(const DecodeParams& p, int ctas, const Cluster& c, cudaStream_t st) {
  const int cluster = static_cast<int>(c.ctas);
  if (cluster > 0)
    return c.warps == 16 ? launch_decode<1, GROUP, false, true, 16>(p, ctas, cluster, st)
           : p.rep > 8   ? launch_decode<2, GROUP, false, true>(p, ctas, cluster, st)
                         : launch_decode<1, GROUP, false, true>(p, ctas, cluster, st);
  if (p.rep > 8) return launch_decode<2, GROUP, false, false>(p, ctas, 0, st);
  return p.parts == 0 ? launch_decode<1, GROUP, true, false>(p, ctas, 0, st)
                      : launch_decode<1, GROUP, false, false>(p, ctas, 0, st);
}

int decode_ctas(int64_t rep) { return num_sms() * (rep > 8 ? 1 : 2); }

// As many CTAs as have room at once (`room`) and find a chunk for each warp, up to 8 (of 8 with
// an SM to each CTA, 16 clusters do not fit: 8 requests of 2,048 tokens, 16 query heads for each of
// 2 kv heads, 16.5 us with them, 9.8 with 4); 16, two to an SM, up to a quarter of the GPU (one
// request of 8,192 tokens and 4 query heads for each of 2 kv heads 8.1 us, of 8 9.8; 8 kv heads 10.7
// and 10.4).  Clusters save the second launch and the ends of walks within a run, where several
// short ones meet; but they take their time by the longest walk, so that runs are for long
// ones, sooner where clusters leave SMs idle.  32 query and 8 kv heads, us with runs and so:
//   1 request of 1,024 tokens 10.3, 6.2; 8,192 11.8, 10.5; 32,768 (8 chunks a warp) 17.7, 20.2
//   3 of 2,048 10.7, 8.2; 16,384 21.6, 21.0; 32,768 (16) 32.5, 36.7
//   16 of 2,048 19.2, 13.5; 8,192 (16) 40.3, 36.9; 64 of 128 12.3, 9.7; 4,096 (16) 68.2, 67.7;
//   16 of 1 to 8,192 48.1, 34.8; 64 of 1 to 4,096 64.8, 51.2; 32 of 1 to 8,192 (32) 52.7, 62.9
// Thousands of walks of equal, short lengths are the exception: 1,024 of 512 tokens 166, 199
// (of 1 to 512 186, 163).
Cluster cluster_of(int64_t walks, int64_t chunks, int64_t room, bool two_an_sm, int64_t warps) {
  int64_t c = 1;
  while (c < (two_an_sm ? 16 : 8) && c * warps < chunks &&
         2 * c * walks <= (c == 8 ? room / 4 : c == 4 && !two_an_sm ? room * 3 / 4 : room))
    c *= 2;
  const int64_t most = 2 * c * walks < room ? 4 : 4 * c * walks < 3 * room ? 8 : 16;  // chunks of a warp
  return {chunks <= most * c * warps ? c : 0, warps};
}
// CTAs of 16 warps take an SM each: where 8 warps would share SMs two by two all the same, or more
// warps work at once, or a cluster is spared.  1 request of 8,192 tokens 10.6 us, 9.6 so; 16,384 (runs
// otherwise) 14.5, 13.1; 3 of 2,048 8.2, 7.7; 16 of 512 7.7, 6.6; of 4,096 20.9, 19.3; but 1 of 2,048
// 6.7, 7.4.  (More than 8 query heads need the registers of 8 warps.)
Cluster cluster_for(int64_t walks, int64_t chunks, int64_t rep) {
  const Cluster c8 = cluster_of(walks, chunks, decode_ctas(rep), rep <= 8, 8);
  if (rep > 8 || c8.ctas == 16 || chunks <= 8) return c8;
  const Cluster c16 = cluster_of(walks, chunks, num_sms(), false, 16);
  if (walks > num_sms() || c16.ctas == 0) return c8;
  const bool more = c8.ctas == 0 || (chunks - 1) / (16 * c16.ctas) < (chunks - 1) / (8 * c8.ctas);
  return more || c16.ctas == 1 || c8.ctas * walks > num_sms() ? c16 : c8;
}

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" size_t kda_gqa_decode_q4_workspace_size(int64_t QH, int64_t KH) {
  if (QH <= 0 || KH <= 0 || QH % KH || QH > 65535) return 0;
  const int64_t rep = QH / KH;
  return static_cast<size_t>(2 * decode_ctas(rep)) * (sizeof(int2) + (rep > 8 ? 16 : 8) * kRow * 4);
}

extern "C" kda_status kda_gqa_decode_q4(const void* q, const void* k_cache, const void* v_cache, const int* lengths,
                                        void* out, int64_t B, int64_t blocks, int64_t QH, int64_t KH, int64_t D,
                                        int64_t group, int64_t window, int64_t sinks, const int64_t* q_strides,
                                        const int64_t* k_cache_strides, const int64_t* v_cache_strides,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "gqa_decode_q4";
  KDA_CHECK_ARG(B > 0 && blocks > 0 && QH > 0 && KH > 0 && QH % KH == 0,
                "%s: bad sizes B=%lld blocks=%lld QH=%lld KH=%lld", op, (long long)B, (long long)blocks, (long long)QH,
                (long long)KH);
  KDA_CHECK_ARG(window > 0 && sinks >= 0, "%s: window must be positive and sinks not negative, got %lld and %lld", op,
                (long long)window, (long long)sinks);
  KDA_CHECK_SUPPORTED(D == kD, "%s: head_dim must be 128, got %lld", op, (long long)D);
  KDA_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: group must be 32, 64 or 128, got %lld", op,
                (long long)group);
  KDA_CHECK_SUPPORTED(B <= 65535 && QH <= 65535 && blocks < (1ll << 26) && B * QH < (1ll << 31),
                      "%s: too large (B=%lld QH=%lld blocks=%lld)", op, (long long)B, (long long)QH, (long long)blocks);
  KDA_CHECK_ARG(q && k_cache && v_cache && lengths && out && q_strides && k_cache_strides && v_cache_strides,
                "%s: null pointer", op);
  const int64_t qs[3] = {q_strides[0], q_strides[1], 0};
  KDA_CHECK_SUPPORTED(head_rows_ok(q, qs, B, QH, 1) && q4_cache_ok(k_cache, k_cache_strides, B, KH) &&
                          q4_cache_ok(v_cache, v_cache_strides, B, KH) && (reinterpret_cast<uintptr_t>(out) & 15u) == 0,
                      "%s: pointers and blocks must be 16-byte aligned", op);
  const size_t need = kda_gqa_decode_q4_workspace_size(QH, KH);
  KDA_CHECK_ARG(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes required, got %zu", op, need,
                workspace_bytes);
  KDA_CHECK_SUPPORTED((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "%s: workspace must be 16-byte aligned",
                      op);
  DecodeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lengths = lengths;
  p.q_b = B > 1 ? q_strides[0] : 0;
  p.q_h = QH > 1 ? q_strides[1] : 0;
  p.k_b = B > 1 ? k_cache_strides[0] : 0, p.k_h = KH > 1 ? k_cache_strides[1] : 0;
  p.v_b = B > 1 ? v_cache_strides[0] : 0, p.v_h = KH > 1 ? v_cache_strides[1] : 0;
  const int64_t T = blocks * kQ4Tokens;
  p.cache_len = static_cast<int>(T);
  p.window = static_cast<int>(window < T ? window : T);
  p.sinks = static_cast<int>(sinks < T ? sinks : T);
  p.B = static_cast<int>(B);
  p.QH = static_cast<int>(QH);
  p.rep = static_cast<int>(QH / KH);
  p.parts = p.rep > 8 ? (p.rep + 15) / 16 : 1;
  const int64_t tokens = p.window + static_cast<int64_t>(p.sinks) < T ? p.window + static_cast<int64_t>(p.sinks) : T;
  const Cluster cluster = cluster_for(B * KH * p.parts, (tokens + 31) / 32 + (tokens < T ? 2 : 0), p.rep);
  // Runs: two kv heads together take less work for each token, and more of it at the end of each
  // walk and share of one (4 query heads of 8 kv heads, us without and with: 8 requests of 8,192
  // tokens 25.1, 26.7; 16 40.6, 41.1; 32 69.2, 67.1; 64 126, 119; 2 of 32,768 24.5, 25.3; 8
  // 66.4, 65.9; 32 229, 219).  Lengths are not known here, the room for them is.
  if (cluster.ctas == 0 && p.rep <= 4 && KH % 2 == 0 && (B * KH >= 512 || B * KH * T >= (1ll << 21))) p.parts = 0;
  p.walks = static_cast<int>(p.parts == 0 ? KH / 2 : KH * p.parts);
  p.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(kD)));
  const int ctas = decode_ctas(p.rep);
  p.pieces = static_cast<int2*>(workspace);
  p.shares = reinterpret_cast<float*>(p.pieces + 2 * ctas);
  p.length_err = kda_err_ptr_q4_decode_length();
  // the longest run, and the number of walks
  KDA_CHECK_SUPPORTED(B * p.walks < (1ll << 31) && B * p.walks < (1ll << 30) * ctas / blocks,
                      "%s: too large (B=%lld KH=%lld blocks=%lld)", op, (long long)B, (long long)KH, (long long)blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return group == 32   ? launch_group<32>(p, ctas, cluster, st)
         : group == 64 ? launch_group<64>(p, ctas, cluster, st)
                       : launch_group<128>(p, ctas, cluster, st);
}
