// Grouped-query attention of one new token per request against a 4-bit key/value cache
// (layout: q4.cuh; head_dim 128).
//
// With n = lengths[b] cached tokens (the new one among them), query head h sees the keys
// j < n where j >= n - window or j < sinks:
//   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = q . k_j log2e / sqrt(128)
//
// HBM-bound: every block of 16 tokens with a visible one is read once (1,152 bytes for K and
// as many for V at groups of 64) for up to 16 query heads of its group.  At 4 bits the codes
// are also the most arithmetic: some 14 warp instructions for each token of a head, of 25
// that an SM has while it reads one.  So codes become operands without arithmetic on values:
// (word & 0x00780078) | 0x41804180 is a pair of bf16 16 + code, exactly, and steps, lows and
// the 16 are applied to sums.  With x = step c + low, over a group G of channels
//   sum_G q x       = step sum_G q (16 + c) + (low - 16 step) sum_G q
//   sum_t p_t x_td  = sum_t (p_t step_t)(16 + c_td) - 16 sum_t (p_t step_t) + sum_t p_t low_t
// where p_t step_t, rounded to bf16 as the operand that meets V's codes, is summed by the
// tensor core as well (a row of ones), so that the 16s cancel to the last bits of fp32.  (The
// nibble at the top of the mantissa, not its end, where the number would be 128 + code: the
// tensor core's sums are cut off, not rounded, and an output that averages 130,000 tokens
// was 0.0045 off in relative L2, with 16 0.0020.)
//
// The products are transposed so that the few query heads are the narrow side of the
// m16n8k16 matrix instruction:
//   S^T (16 keys x 8 heads)  = K q^T          O^T (128 x 8 heads) += V^T P^T
// The running maximum moves only when a score exceeds it by 2^8, which fp32 sums and bf16
// weights hold exactly as well; so a block usually needs no exchange between lanes.
//
// The blocks of all (request, kv head) walks, one behind the other, are cut into equal runs,
// one for each CTA (lengths are ragged and known on the device only); a run's blocks go to the
// CTA's warps in turn, each through a ring of bulk copies of its own that runs on across the
// ends of walks.  Where a walk ends, or the run does, the warps join through shared memory:
// a whole walk's output leaves, a cut one's share goes to the workspace, and a second launch
// joins the shares in the order of the walk: one fixed order of summation.
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
constexpr int kLeast = 2 * kWarps;  // blocks of a CTA's run, where there are as many
constexpr unsigned kFull = 0xffffffffu;

struct DecodeParams {
  const __nv_bfloat16* q;
  const uint8_t *k, *v;
  __nv_bfloat16* out;        // [B][QH][128]
  const int* lengths;
  int64_t q_b, q_h;          // element strides
  int64_t k_b, k_h, v_b, v_h;  // byte strides
  int64_t cache_len;
  int64_t window, sinks;
  int B, QH, KH, rep, parts;  // parts: groups of 8 NT query heads per kv head
  float scale_log2;
  float* shares;             // [2 x CTAs][8 NT][kRow]
  int4* pieces;              // [2 x CTAs]: walk, 0, blocks of the share, of the walk
  unsigned* length_err;
};

// The blocks of a request's walk: [0, ns) (sinks), then [ns + skip, n + skip).
struct Walk {
  int n, ns, skip;
  int64_t len, start;
};
__device__ __forceinline__ Walk walk_of(const DecodeParams& p, int b) {
  Walk w;
  int64_t n = __ldg(p.lengths + b);
  if (n > p.cache_len) n = p.cache_len;  // the cache's end is the end (reported where outputs of no token are)
  if (n < 0) n = 0;
  w.len = n;
  w.start = n > p.window ? n - p.window : 0;
  const int64_t sinks = p.sinks < w.start ? p.sinks : w.start;
  const int first = static_cast<int>(w.start / kQ4Tokens), end = static_cast<int>((n + kQ4Tokens - 1) / kQ4Tokens);
  w.ns = min(static_cast<int>((sinks + kQ4Tokens - 1) / kQ4Tokens), first);
  w.skip = first - w.ns;
  w.n = w.ns + end - first;
  return w;
}

// Where a run stands: block x of walk (b, hp), hp = kv head * parts + part.
struct Cursor {
  int b, hp, x;
  Walk w;
};
// `by` blocks on, over the ends of walks (those of requests without tokens are empty).
__device__ __forceinline__ void move(const DecodeParams& p, Cursor* c, int by) {
  c->x += by;
  while (c->x >= c->w.n) {
    c->x -= c->w.n;
    if (++c->hp == p.KH * p.parts) {
      c->hp = 0;
      do {
        if (++c->b >= p.B) return;  // past the last walk: not read
        c->w = walk_of(p, c->b);
      } while (c->w.n == 0);
    }
  }
}
__device__ __forceinline__ int64_t block_of(const Cursor& c) { return c.x < c.w.ns ? c.x : c.x + c.w.skip; }

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
// Nibbles I and I + 4 of a word as bf16 16 + code.
template <int I>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  return ((I == 0 ? w << 3 : w >> (4 * I - 3)) & 0x00780078u) | 0x41804180u;
}
__device__ __forceinline__ float step_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float low_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// The weight of a share with maximum m among shares whose maximum is mm.  One that saw
// nothing finite has sums of zeros, which may be added as they are, or of NaN, which must be.
__device__ __forceinline__ float share_weight(float m, float mm) { return m == -INFINITY ? 1.f : exp2_approx(m - mm); }

// A run's start in blocks, of `total` over `ctas`.
__device__ __forceinline__ int64_t run_at(int64_t total, int c, int ctas) { return total * c / ctas; }

// NT: groups of 8 query heads a CTA works on.
template <int NT, int GROUP, int STAGES>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) q4_decode_kernel(const DecodeParams p, unsigned* err) {
  constexpr int H = 8 * NT;
  constexpr int NG = 128 / GROUP;                       // pairs of a token
  constexpr int RUNS = 4 / NG;                          // 32-channel runs of a group
  constexpr uint32_t kBlock = q4_block_bytes(GROUP);    // of K; V's lies behind it in a stage
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kWarps][STAGES];
  __shared__ int64_t sums[kWarps];
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
  if (threadIdx.x == 0) p.pieces[2 * blockIdx.x] = p.pieces[2 * blockIdx.x + 1] = make_int4(0, 0, 0, 0);

  // The run: blocks [r0, r1) of all walks.  Each thread counts the requests [b0, b1).
  const int heads = p.KH * p.parts;
  const int each = (p.B + kThreads - 1) / kThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * each, p.B), b1 = min(b0 + each, p.B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += walk_of(p, b).n;
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
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  total *= heads;
  const int ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total / kLeast > 0 ? total / kLeast : 1));
  const int cta = static_cast<int>(blockIdx.x);
  const int64_t r0 = cta < ctas ? run_at(total, cta, ctas) : 0, r1 = cta < ctas ? run_at(total, cta + 1, ctas) : 0;
  const int run = static_cast<int>(r1 - r0);
  if (run > 0 && before * heads <= r0 && r0 < (before + mine) * heads) {
    int64_t x = before;
    int b = b0, n = walk_of(p, b).n;
    while (n == 0 || (x + n) * heads <= r0) {
      x += n;
      n = walk_of(p, ++b).n;
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
      for (int i = threadIdx.x; i < p.QH * (kD / 8); i += kThreads)
        reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(b) * p.QH * kD)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (run == 0) return;

  Cursor at;  // of the piece in work
  at.b = first_b;
  at.w = walk_of(p, at.b);
  at.hp = static_cast<int>(first_x / at.w.n);
  at.x = static_cast<int>(first_x - static_cast<int64_t>(at.hp) * at.w.n);

  // this warp's blocks: warp, warp + kWarps, ... of the run
  const uint32_t ring = smem_u32(smem) + warp * (STAGES * 2 * kBlock);
  Cursor ahead = at;  // of the next load
  if (warp > 0) move(p, &ahead, warp);
  int loads = 0;
  auto load = [&]() {
    if (warp + loads * kWarps >= run) return;
    const int s = loads % STAGES;
    if (lane == 0) {
      const int g = ahead.hp / p.parts;
      const int64_t off = block_of(ahead) * kBlock;
      mbar_arrive_expect_tx(&full[warp][s], 2 * kBlock);
      uint8_t* dst = smem + warp * (STAGES * 2 * kBlock) + s * 2 * kBlock;
      bulk_load_1d(dst, p.k + ahead.b * p.k_b + g * p.k_h + off, kBlock, &full[warp][s]);
      bulk_load_1d(dst + kBlock, p.v + ahead.b * p.v_b + g * p.v_h + off, kBlock, &full[warp][s]);
    }
    ++loads;
    if (warp + loads * kWarps < run) move(p, &ahead, kWarps);
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load();

  float* parts = reinterpret_cast<float*>(smem + kWarps * STAGES * 2 * kBlock);  // [kWarps][min(rep, H)][kRow]
  const int held = min(p.rep, H);
  bool ok = true;
  int done = 0;       // this warp's blocks
  int piece_at = 0;   // the piece's first block in the run
  while (piece_at < run) {
    const int left = run - piece_at;
    const int n = min(left, at.w.n - at.x);  // blocks of the piece
    const int g = at.hp / p.parts, part = at.hp - g * p.parts;
    const int h0 = g * p.rep + part * H;  // first query head
    const int nh = min(H, p.rep - part * H);

    // q^T operands: for run g and step s of its two, head lane / 4, channels of this lane's
    // word: (2 s, 2 s + 4) and (2 s + 1, 2 s + 5); and the sums over groups of the heads of
    // this lane's accumulators, 2 (lane % 4) + {0, 1}
    uint32_t qf[NT][4][2][2];
    float qsum[NT][NG][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int h = t * 8 + r;
      float sum[NG];
#pragma unroll
      for (int j = 0; j < NG; ++j) sum[j] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 w = h < nh ? __ldg(reinterpret_cast<const uint4*>(p.q + at.b * p.q_b +
                                                                      static_cast<int64_t>(h0 + h) * p.q_h + 32 * k) + c4)
                               : make_uint4(0u, 0u, 0u, 0u);
        qf[t][k][0][0] = __byte_perm(w.x, w.z, 0x5410);
        qf[t][k][0][1] = __byte_perm(w.x, w.z, 0x7632);
        qf[t][k][1][0] = __byte_perm(w.y, w.w, 0x5410);
        qf[t][k][1][1] = __byte_perm(w.y, w.w, 0x7632);
        float f[8];
        unpack_bf16x8(w, f);
        sum[k / RUNS] += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        sum[j] += __shfl_xor_sync(kFull, sum[j], 1);
        sum[j] += __shfl_xor_sync(kFull, sum[j], 2);
        qsum[t][j][0] = __shfl_sync(kFull, sum[j], 8 * c4);
        qsum[t][j][1] = __shfl_sync(kFull, sum[j], 8 * c4 + 4);
      }
    }
    float m[NT][2], l[NT][2];       // heads 8 t + 2 (lane % 4) + {0, 1}; l: this lane's keys only
    float lows[NT][NG][2];          // sums of p low, this lane's keys only
    float ones[NT][NG][4];          // sums of p step (the same in every row)
    float o[NT][4][2][4];           // run, step: channels 32 run + 4 (lane / 4) + 2 step (+ 1)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        lows[t][j][0] = lows[t][j][1] = 0.f;
        ones[t][j][0] = ones[t][j][1] = ones[t][j][2] = ones[t][j][3] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int s = 0; s < 2; ++s) o[t][k][s][0] = o[t][k][s][1] = o[t][k][s][2] = o[t][k][s][3] = 0.f;
    }

    for (; ok && warp + done * kWarps < piece_at + n; ++done) {
      const int x = at.x + warp + done * kWarps - piece_at;
      __syncwarp();  // every lane is done with the stage refilled here
      load();
      const int s = done % STAGES;
      if (!warp_wait(&full[warp][s], static_cast<uint32_t>(done / STAGES) & 1u, err, kErrWaitFull)) {
        ok = false;
        break;
      }
      const uint32_t ks = ring + s * 2 * kBlock, vs = ks + kBlock;
      const int64_t tok = (x < at.w.ns ? x : x + at.w.skip) * static_cast<int64_t>(kQ4Tokens);
      // tokens of this lane's accumulators: r and r + 8
      bool see0 = true, see1 = true;
      const bool whole = tok + kQ4Tokens <= at.w.len && (tok >= at.w.start || tok + kQ4Tokens <= p.sinks);
      if (!whole) {
        const int64_t t0 = tok + r, t1 = t0 + 8;
        see0 = t0 < at.w.len && (t0 >= at.w.start || t0 < p.sinks);
        see1 = t1 < at.w.len && (t1 >= at.w.start || t1 < p.sinks);
      }

      float sc[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
      {
        const uint32_t row = ks + r * 64 + ((c4 ^ ((r >> 1) & 3)) << 4);  // chunk lane % 4 of tokens r and r + 8
        const uint4 k0 = ld_shared_v4(row), k1 = ld_shared_v4(row + 512);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          float acc[NT][4];
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
          for (int k = j * RUNS; k < (j + 1) * RUNS; ++k)
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              const uint32_t a[4] = {st ? codes2<2>(w0[k]) : codes2<0>(w0[k]), st ? codes2<2>(w1[k]) : codes2<0>(w1[k]),
                                     st ? codes2<3>(w0[k]) : codes2<1>(w0[k]), st ? codes2<3>(w1[k]) : codes2<1>(w1[k])};
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_bf16(acc[t], a, qf[t][k][st][0], qf[t][k][st][1]);
            }
          const uint32_t p0 = ld_shared(ks + kQ4Codes + (r * NG + j) * 4);
          const uint32_t p1 = ld_shared(ks + kQ4Codes + ((r + 8) * NG + j) * 4);
          const float s0 = step_of(p0), s1 = step_of(p1);
          const float z0 = fmaf(-16.f, s0, low_of(p0)), z1 = fmaf(-16.f, s1, low_of(p1));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sc[t][0] = fmaf(s0, acc[t][0], fmaf(z0, qsum[t][j][0], sc[t][0]));
            sc[t][1] = fmaf(s0, acc[t][1], fmaf(z0, qsum[t][j][1], sc[t][1]));
            sc[t][2] = fmaf(s1, acc[t][2], fmaf(z1, qsum[t][j][0], sc[t][2]));
            sc[t][3] = fmaf(s1, acc[t][3], fmaf(z1, qsum[t][j][1], sc[t][3]));
          }
        }
      }
      if (!whole) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (!see0) sc[t][0] = sc[t][1] = -INFINITY;
          if (!see1) sc[t][2] = sc[t][3] = -INFINITY;
        }
      }
      bool grow = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) grow |= fmaxf(sc[t][c], sc[t][c + 2]) * p.scale_log2 > m[t][c] + 8.f;
      if (__any_sync(kFull, grow)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(sc[t][c], sc[t][c + 2]) * p.scale_log2;
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, d));
            mx = fmaxf(mx, m[t][c]);
            // nothing finite yet: keep the (empty) sums as they are
            const float f = mx == -INFINITY ? 1.f : exp2_approx(m[t][c] - mx);
            m[t][c] = mx;
            l[t][c] *= f;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
              lows[t][j][c] *= f;
              ones[t][j][c] *= f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int st = 0; st < 2; ++st) {
                o[t][k][st][c] *= f;
                o[t][k][st][c + 2] *= f;
              }
          }
      }
      float e[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float mm = m[t][c & 1] == -INFINITY ? 0.f : m[t][c & 1];
          e[t][c] = exp2_approx(fmaf(sc[t][c], p.scale_log2, -mm));
        }
        l[t][0] += e[t][0] + e[t][2];
        l[t][1] += e[t][1] + e[t][3];
      }
      // tokens 2 (lane % 4) + {0, 1} and 8 on: their chunk r / 2, of which this lane takes half
      // of each word: channels 32 run + 4 r + {0 .. 3}
      const uint32_t col = vs + c4 * 128 + (((r >> 1) ^ c4) << 4);
      const uint4 va = ld_shared_v4(col), vb = ld_shared_v4(col + 64), vc = ld_shared_v4(col + 512),
                  vd = ld_shared_v4(col + 576);
      const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w},
                     wc[4] = {vc.x, vc.y, vc.z, vc.w}, wd[4] = {vd.x, vd.y, vd.z, vd.w};
      const uint32_t pick = (r & 1) ? 0x7632u : 0x5410u;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        uint32_t p0 = ld_shared(vs + kQ4Codes + (r * NG + j) * 4);
        uint32_t p1 = ld_shared(vs + kQ4Codes + ((r + 8) * NG + j) * 4);
        if (!see0) p0 = 0u;  // whatever is there must not meet its weight of zero
        if (!see1) p1 = 0u;
        const float s0 = step_of(p0), s1 = step_of(p1), z0 = low_of(p0), z1 = low_of(p1);
        uint32_t pb[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          lows[t][j][0] = fmaf(e[t][0], z0, fmaf(e[t][2], z1, lows[t][j][0]));
          lows[t][j][1] = fmaf(e[t][1], z0, fmaf(e[t][3], z1, lows[t][j][1]));
          // weight times step meets the codes as bf16, the tensor core's operand type
          pb[t][0] = transpose8x8(pack_bf16x2(e[t][0] * s0, e[t][1] * s0));
          pb[t][1] = transpose8x8(pack_bf16x2(e[t][2] * s1, e[t][3] * s1));
        }
        const uint32_t one[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_bf16(ones[t][j], one, pb[t][0], pb[t][1]);
#pragma unroll
        for (int k = j * RUNS; k < (j + 1) * RUNS; ++k) {
          const uint32_t lo = __byte_perm(wa[k], wb[k], pick), hi = __byte_perm(wc[k], wd[k], pick);
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const uint32_t a[4] = {st ? codes2<2>(lo) : codes2<0>(lo), st ? codes2<3>(lo) : codes2<1>(lo),
                                   st ? codes2<2>(hi) : codes2<0>(hi), st ? codes2<3>(hi) : codes2<1>(hi)};
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_bf16(o[t][k][st], a, pb[t][0], pb[t][1]);
          }
        }
      }
    }

    // the piece's end: this warp's share, then all of them
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = t * 8 + 2 * c4 + c;
        float sum = l[t][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(kFull, sum, d);
        float add[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          add[j] = lows[t][j][c];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) add[j] += __shfl_xor_sync(kFull, add[j], d);
          add[j] = fmaf(-16.f, ones[t][j][c], add[j]);
        }
        if (h < nh) {
          float* dst = parts + (warp * held + h) * kRow;
          if (r == 0) {
            dst[kD] = m[t][c];
            dst[kD + 1] = sum;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int st = 0; st < 2; ++st)
              *reinterpret_cast<float2*>(dst + 32 * k + 4 * r + 2 * st) =
                  make_float2(o[t][k][st][c] + add[k / RUNS], o[t][k][st][c + 2] + add[k / RUNS]);
        }
      }
    __syncthreads();
    const bool cut = n < at.w.n;
    const int slot = 2 * cta + (at.x == 0 ? 1 : 0);
    for (int i = threadIdx.x; i < nh * kD; i += kThreads) {
      const int h = i / kD, d = i - h * kD;
      float mm = -INFINITY, ll = 0.f, oo = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, parts[(w * held + h) * kRow + kD]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* src = parts + (w * held + h) * kRow;
        const float f = share_weight(src[kD], mm);
        ll += f * src[kD + 1];
        oo += f * src[d];
      }
      if (cut) {
        float* dst = p.shares + (static_cast<int64_t>(slot) * H + h) * kRow;
        dst[d] = oo;
        if (d == 0) {
          dst[kD] = mm;
          dst[kD + 1] = ll;
        }
      } else {
        p.out[(static_cast<int64_t>(at.b) * p.QH + h0 + h) * kD + d] = __float2bfloat16_rn(oo / ll);
      }
    }
    if (cut && threadIdx.x == 0) p.pieces[slot] = make_int4(at.b * heads + at.hp, 0, n, at.w.n);
    __syncthreads();  // parts are free
    piece_at += n;
    if (piece_at < run) move(p, &at, n);
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
  const int4 w = p.pieces[2 * blockIdx.x + 1];
  if (w.z == 0) return;
  const int heads = p.KH * p.parts;
  const int b = w.x / heads, hp = w.x - b * heads, g = hp / p.parts, part = hp - g * p.parts;
  const int h = blockIdx.y;
  if (h >= min(H, p.rep - part * H)) return;
  int steps = w.z, count = 1;  // shares: slots 2 x + 1, 2 (x + 1), 2 (x + 2), ...
  for (int slot = 2 * blockIdx.x + 1;; ++count) {
    slot = next_share(p.pieces, 2 * ctas, slot, w.w, &steps);
    if (slot < 0) break;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto share = [&](int i) {
    const int slot = i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i);
    return p.shares + (static_cast<int64_t>(slot) * H + h) * kRow;
  };
  float mm = -INFINITY;
  for (int i = warp; i < count; i += kWarps) mm = fmaxf(mm, share(i)[kD]);
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
  if (lane == 0) {
    parts[warp][kD] = mm;
    parts[warp][kD + 1] = ll;
  }
  __syncthreads();
  if (threadIdx.x < kD) {
    const int d = threadIdx.x;
    float m2 = -INFINITY, l2 = 0.f, o2 = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m2 = fmaxf(m2, parts[i][kD]);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float f = share_weight(parts[i][kD], m2);
      l2 += f * parts[i][kD + 1];
      o2 += f * parts[i][d];
    }
    p.out[(static_cast<int64_t>(b) * p.QH + g * p.rep + part * H + h) * kD + d] = __float2bfloat16_rn(o2 / l2);
  }
}

template <int NT, int GROUP>
kda_status launch_decode(const DecodeParams& p, int ctas, cudaStream_t st) {
  // rings of the depth that leaves two CTAs an SM (one where a group has more than 8 heads)
  constexpr int kStages = NT == 1 ? (GROUP == 32 ? 3 : 4) : 6;
  constexpr int H = 8 * NT;
  constexpr size_t kMost = kWarps * (kStages * 2 * q4_block_bytes(GROUP) + H * kRow * 4);
  static_assert(kMost <= (NT == 1 ? 112 : 226) * 1024, "shared memory budget");
  auto* kernel = q4_decode_kernel<NT, GROUP, kStages>;
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMost)) !=
        cudaSuccess)
      return launch_status("gqa_decode_q4: cudaFuncSetAttribute");
    attr_set[dev].store(true, std::memory_order_release);
  }
  const size_t smem = kWarps * (kStages * 2 * q4_block_bytes(GROUP) + (p.rep < H ? p.rep : H) * kRow * 4);
  const kda_status s = launch_after("gqa_decode_q4", kernel, dim3(static_cast<unsigned>(ctas)), kThreads, smem, st, p,
                                    kda_err_ptr_q4_decode());
  if (s != KDA_OK) return s;
  return launch_after("gqa_decode_q4: join", q4_join_kernel<H>,
                      dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(p.rep < H ? p.rep : H)), kThreads, 0, st, p,
                      ctas);
}

int decode_ctas(int64_t rep) { return num_sms() * (rep > 8 ? 1 : 2); }

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" size_t kda_gqa_decode_q4_workspace_size(int64_t QH, int64_t KH) {
  if (QH <= 0 || KH <= 0 || QH % KH || QH > 65535) return 0;
  const int64_t rep = QH / KH;
  return static_cast<size_t>(2 * decode_ctas(rep)) * (16 + (rep > 8 ? 16 : 8) * kRow * 4);
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
  p.cache_len = blocks * kQ4Tokens;
  p.window = window < p.cache_len ? window : p.cache_len;
  p.sinks = sinks < p.cache_len ? sinks : p.cache_len;
  p.B = static_cast<int>(B);
  p.QH = static_cast<int>(QH);
  p.KH = static_cast<int>(KH);
  p.rep = static_cast<int>(QH / KH);
  p.parts = p.rep > 8 ? (p.rep + 15) / 16 : 1;
  p.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(kD)));
  const int ctas = decode_ctas(p.rep);
  p.pieces = static_cast<int4*>(workspace);
  p.shares = reinterpret_cast<float*>(p.pieces + 2 * ctas);
  p.length_err = kda_err_ptr_q4_decode_length();
  // the longest run, and the number of walks
  KDA_CHECK_SUPPORTED(B * KH * p.parts < (1ll << 31) && B * KH * p.parts < (1ll << 31) * ctas / blocks,
                      "%s: too large (B=%lld KH=%lld blocks=%lld)", op, (long long)B, (long long)KH, (long long)blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.rep > 8)
    return group == 32   ? launch_decode<2, 32>(p, ctas, st)
           : group == 64 ? launch_decode<2, 64>(p, ctas, st)
                         : launch_decode<2, 128>(p, ctas, st);
  return group == 32   ? launch_decode<1, 32>(p, ctas, st)
         : group == 64 ? launch_decode<1, 64>(p, ctas, st)
                       : launch_decode<1, 128>(p, ctas, st);
}
