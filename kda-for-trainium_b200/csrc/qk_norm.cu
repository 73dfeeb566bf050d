// Per-head RMS norm of queries and keys with the position rotation in the same
// pass: forward, backward, and the forward that appends to a key/value cache.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps),  n_d = x_d r g_d
//   y_d       = n_d cos_d - n_{d+D/2} sin_d          (d < D/2; angle = position
//   y_{d+D/2} = n_d sin_d + n_{d+D/2} cos_d           x theta^(-2d/D), read from
//                                                     a table [P][D/2][cos, sin])
// Backward, dn = dy rotated by the negated angle and t = g dn:
//   dx = r t - x r^3 mean(x t),   dg = sum over rows of x r dn
//
// HBM-bound streams: every row is read once and written once.  A row of D
// values belongs to D / (2 VE) lanes (VE = values per 16 bytes); each lane
// holds VE values of the first half and the VE it is rotated with, so the
// rotation needs no exchange and the two loads and stores are 16 bytes wide;
// the sums over the row are shuffles among those lanes.  All arithmetic is
// fp32; bf16 rows are rounded once, when they are stored.
#include <algorithm>

#include "launch.cuh"

KDA_DEFINE_ERROR_WORD(qk_norm)

namespace kda {
namespace {

constexpr int kThreads = 256;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void st_stream(void* p, uint4 v) {
  asm volatile("st.global.cs.v4.b32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// The 16 bytes of a lane as pairs of fp32 values (for the packed f32x2
// instructions, two values per issue slot) and back.
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void unpack(const uint4 v, float2 (&f)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[4]) {
    return make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y),
                      pack_bf16x2(f[3].x, f[3].y));
  }
};
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void unpack(const uint4 v, float2 (&f)[2]) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&f)[2]) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                      __float_as_uint(f[1].y));
  }
};

// A strided [B][S][H][D] operand (rows of D contiguous values); strides in elements.
struct Rows {
  const void* p;
  int64_t sb, ss, sh;
};
struct RowsOut {
  void* p;
  int64_t sb, ss, sh;
};

struct FwdParams {
  Rows q, k, v;
  RowsOut qo, ko, vo;
  const float *gq, *gk;
  const float* table;        // [P][D/2][2]
  const int* positions;      // [B][S] or null: 0 .. S-1
  const int* lengths;        // append: [B], tokens already in the cache (negative: idle slot)
  int64_t table_len, cache_len;
  int B, S, QH, KH;
  int hp;                    // heads per item
  unsigned cq, ck;           // items of a token's queries, of its keys (append: and of its values)
  float eps;
};

template <int LPR>
__device__ __forceinline__ float row_sum(float s) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  return s;
}

template <int N>
__device__ __forceinline__ void load_f32x2(const float* p, float2 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
    f[2 * i] = make_float2(v.x, v.y);
    f[2 * i + 1] = make_float2(v.z, v.w);
  }
}

// N pairs of cosines and sines from the table's interleaved (cos, sin).
template <int N>
__device__ __forceinline__ void load_angles(const float* p, float2 (&c)[N], float2 (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
    c[i] = make_float2(v.x, v.z);
    s[i] = make_float2(v.y, v.w);
  }
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg(float2 v) { return make_float2(-v.x, -v.y); }

// One group of LPR lanes per item = up to hp heads of one token (queries, keys
// or values), U rows at a time, whose loads are issued before anything waits.
// The norm's weights and the token's angles fold into four coefficients per
// pair of values once per item:
//   y0 = r (x0 g0 cos - x1 g1 sin),  y1 = r (x0 g0 sin + x1 g1 cos)
template <typename T, int D, int U, bool kAppend>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const FwdParams p, unsigned* err) {
  constexpr int VE = Vec<T>::kN;
  constexpr int LPR = D / (2 * VE);
  pdl_trigger();  // the next launch may start
  pdl_wait();     // the one before is done: what it wrote is there, what it read may be written
  const int lane = threadIdx.x % LPR;  // owns values [VE lane, + VE) of both halves
  const unsigned nc = p.cq + p.ck * (kAppend ? 2 : 1);
  const unsigned item = (blockIdx.x * static_cast<unsigned>(kThreads) + threadIdx.x) / LPR;
  const bool live = item < static_cast<unsigned>(p.B) * static_cast<unsigned>(p.S) * nc;  // idle groups keep up the shuffles
  const unsigned tok = live ? item / nc : 0;
  unsigned c = live ? item - tok * nc : 0;
  const int b = static_cast<int>(tok / static_cast<unsigned>(p.S));
  const int s = static_cast<int>(tok - static_cast<unsigned>(b) * static_cast<unsigned>(p.S));
  const int kind = c < p.cq ? 0 : c < p.cq + p.ck ? 1 : 2;
  c -= kind == 0 ? 0 : kind == 1 ? p.cq : p.cq + p.ck;
  const Rows in = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
  const RowsOut out = kind == 0 ? p.qo : kind == 1 ? p.ko : p.vo;
  const int h0 = static_cast<int>(c) * p.hp;
  const int nh = live ? min(p.hp, (kind == 0 ? p.QH : p.KH) - h0) : 0;
  const T* src = static_cast<const T*>(in.p) + b * in.sb + s * in.ss + h0 * in.sh + lane * VE;

  int64_t pos = s, row = s;  // table row; row of the output
  bool idle = false;         // append: a slot without a request
  if (kAppend) {
    const int len = __ldg(p.lengths + b);
    idle = len < 0;
    pos = idle ? 0 : static_cast<int64_t>(len) + s;
    row = kind == 0 ? s : pos;
  } else if (p.positions) {
    pos = __ldg(p.positions + static_cast<int64_t>(b) * p.S + s);
  }
  // a position outside the table (or the cache) is reported and gives NaN; nothing is read or appended there
  const bool bad = pos < 0 || pos >= p.table_len || (kAppend && pos >= p.cache_len);
  if (bad && live && lane == 0) atomicOr(err, static_cast<unsigned>(kErrRange));
  T* dst = static_cast<T*>(out.p) + b * out.sb + row * out.ss + h0 * out.sh + lane * VE;
  const bool write = !kAppend || kind == 0 || !(bad || idle);

  constexpr int N = VE / 2;
  float2 k00[N], k01[N], k10[N], k11[N];  // y0 = r (x0 k00 + x1 k01), y1 = r (x0 k10 + x1 k11)
  {
    float2 cs[N], sn[N], g0[N], g1[N];
    const float* g = kind == 0 ? p.gq : p.gk;
    load_angles(p.table + ((bad ? 0 : pos) * (D / 2) + lane * VE) * 2, cs, sn);
    load_f32x2(g + lane * VE, g0);
    load_f32x2(g + D / 2 + lane * VE, g1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      k00[i] = __fmul2_rn(g0[i], cs[i]);
      k01[i] = neg(__fmul2_rn(g1[i], sn[i]));
      k10[i] = __fmul2_rn(g0[i], sn[i]);
      k11[i] = __fmul2_rn(g1[i], cs[i]);
      if (bad) k00[i] = k10[i] = both(__int_as_float(0x7fffffff));
    }
  }
  // all groups of a warp make hp / U rounds (the shuffles need every lane)
  for (int h = 0; h < p.hp; h += U) {
    uint4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      lo[u] = hi[u] = make_uint4(0u, 0u, 0u, 0u);
      if (h + u < nh) {
        lo[u] = ld_stream(src + (h + u) * in.sh);
        hi[u] = ld_stream(src + (h + u) * in.sh + D / 2);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float2 x0[N], x1[N];
      Vec<T>::unpack(lo[u], x0);
      Vec<T>::unpack(hi[u], x1);
      float2 ss = both(0.f);
#pragma unroll
      for (int i = 0; i < N; ++i) ss = __ffma2_rn(x0[i], x0[i], __ffma2_rn(x1[i], x1[i], ss));
      const float2 r = both(rsqrtf(row_sum<LPR>(ss.x + ss.y) * (1.0f / D) + p.eps));
      if (h + u >= nh || !write) continue;  // after the shuffles
      if (!kAppend || kind != 2) {          // (values go to the cache as they are)
        float2 y0[N], y1[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          y0[i] = __fmul2_rn(r, __ffma2_rn(x0[i], k00[i], __fmul2_rn(x1[i], k01[i])));
          y1[i] = __fmul2_rn(r, __ffma2_rn(x0[i], k10[i], __fmul2_rn(x1[i], k11[i])));
        }
        lo[u] = Vec<T>::pack(y0);
        hi[u] = Vec<T>::pack(y1);
        if (kAppend && idle) lo[u] = hi[u] = make_uint4(0u, 0u, 0u, 0u);
      }
      st_stream(dst + (h + u) * out.sh, lo[u]);
      st_stream(dst + (h + u) * out.sh + D / 2, hi[u]);
    }
  }
}

struct BwdParams {
  Rows x[2], dy[2];          // q, k and the gradients of their rotated rows
  RowsOut dx[2];
  const float* g[2];
  const float* table;
  const int* positions;
  int64_t table_len;
  int B, S;
  int H[2];
  int hp[2];                 // heads per item
  int blocks[2];             // CTAs of the queries, of the keys
  float* partial;            // [blocks[0] + blocks[1]][D]: each CTA's share of dg
  float eps;
};

// CTAs [0, blocks[0]) walk the queries, the others the keys; a group of LPR
// lanes takes up to hp heads of a token, one after the other.  Each thread sums its
// columns of dg over all its rows in registers; the CTA's sums go to `partial` in a
// fixed order, so the result does not depend on timing.
// The registers that dg takes leave two CTAs of 8 warps per SM, too few to cover the
// memory's latency with loads into registers (B2 S4096 of 40 heads: 51 us, two rows at
// a time), so the rows come through a ring of 4 per thread in shared memory, 64 KB a
// CTA: 45 us, 5.6 TB/s (6 rows: 46; three CTAs with rings of 3, which spill: 66).
constexpr int kRing = 4;
constexpr size_t kRingBytes = kRing * 4 * kThreads * 16;
constexpr int kBwdHeads = 4;  // heads per item (8: 46 us)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_bwd_kernel(const BwdParams p, unsigned* err) {
  constexpr int VE = Vec<T>::kN;
  constexpr int LPR = D / (2 * VE);
  constexpr int kGroups = kThreads / LPR;
  extern __shared__ __align__(16) uint8_t norm_ring[];
  __shared__ __align__(8) float red[kThreads / 32][D];
  pdl_trigger();  // the join may take its place while this runs
  pdl_wait();     // the launch before this one is done
  const int lane = threadIdx.x % LPR;
  const int w = static_cast<int>(blockIdx.x) < p.blocks[0] ? 0 : 1;
  const int block = static_cast<int>(blockIdx.x) - (w ? p.blocks[0] : 0);
  const Rows xr = p.x[w], dyr = p.dy[w];
  const RowsOut dxr = p.dx[w];
  const int H = p.H[w], hp = p.hp[w];
  const unsigned nc = static_cast<unsigned>((H + hp - 1) / hp);
  const unsigned items = static_cast<unsigned>(p.B) * static_cast<unsigned>(p.S) * nc;
  constexpr int N = VE / 2;
  float2 g0[N], g1[N], a0[N], a1[N];
  load_f32x2(p.g[w] + lane * VE, g0);
  load_f32x2(p.g[w] + D / 2 + lane * VE, g1);
#pragma unroll
  for (int i = 0; i < N; ++i) a0[i] = a1[i] = both(0.f);

  // Every group of a warp makes the same number of rounds (the shuffles need all
  // lanes).  Rows come through a ring in shared memory, kRing - 1 of them on their way
  // while one is worked on; a thread copies what it reads itself, so nothing is
  // synchronised but its own copies.
  struct Item {
    const T *xs, *ds;
    T* dst;
    int nh;
    int64_t pos;
  };
  const unsigned step = static_cast<unsigned>(p.blocks[w]) * kGroups;
  auto locate = [&](unsigned base) -> Item {
    const unsigned item = base + threadIdx.x / LPR;
    const bool live = item < items;
    const unsigned tok = live ? item / nc : 0;
    const int h0 = live ? static_cast<int>(item - tok * nc) * hp : 0;
    const int b = static_cast<int>(tok / static_cast<unsigned>(p.S));
    const int s = static_cast<int>(tok - static_cast<unsigned>(b) * static_cast<unsigned>(p.S));
    Item c;
    c.nh = live ? min(hp, H - h0) : 0;
    c.xs = static_cast<const T*>(xr.p) + b * xr.sb + s * xr.ss + h0 * xr.sh + lane * VE;
    c.ds = static_cast<const T*>(dyr.p) + b * dyr.sb + s * dyr.ss + h0 * dyr.sh + lane * VE;
    c.dst = static_cast<T*>(dxr.p) + b * dxr.sb + s * dxr.ss + h0 * dxr.sh + lane * VE;
    c.pos = p.positions ? __ldg(p.positions + tok) : s;
    return c;
  };
  const unsigned base0 = static_cast<unsigned>(block) * kGroups;
  const uint32_t ring = smem_u32(norm_ring) + threadIdx.x * 16;
  unsigned abase = base0;  // the next row to ask for: its item, row of the item
  int ah = 0;
  Item a = locate(base0);
  auto ask = [&](int stage) {
    if (abase < items) {
      const bool there = ah < a.nh;
      const int64_t row = there ? ah : 0;
      const uint32_t to = ring + stage * (4 * kThreads * 16);
      cp_async16(to, a.xs + row * xr.sh, there);
      cp_async16(to + kThreads * 16, a.xs + row * xr.sh + D / 2, there);
      cp_async16(to + 2 * kThreads * 16, a.ds + row * dyr.sh, there);
      cp_async16(to + 3 * kThreads * 16, a.ds + row * dyr.sh + D / 2, there);
      if (++ah == hp) {
        ah = 0;
        abase += step;
        if (abase < items) a = locate(abase);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) ask(i);
  int stage = 0;
  for (unsigned base = base0; base < items; base += step) {
    const Item c = locate(base);
    const bool bad = c.pos < 0 || c.pos >= p.table_len;
    if (bad && c.nh > 0 && lane == 0) atomicOr(err, static_cast<unsigned>(kErrRange));
    float2 cs[N], sn[N];
    load_angles(p.table + ((bad ? 0 : c.pos) * (D / 2) + lane * VE) * 2, cs, sn);
    if (bad) {  // the position's rows come out as NaN
#pragma unroll
      for (int i = 0; i < N; ++i) cs[i] = both(__int_as_float(0x7fffffff));
    }
    for (int h = 0; h < hp; ++h) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
      float2 x0[N], x1[N], y0[N], y1[N];
      const uint32_t at = ring + stage * (4 * kThreads * 16);
      Vec<T>::unpack(ld_shared16(at), x0);
      Vec<T>::unpack(ld_shared16(at + kThreads * 16), x1);
      Vec<T>::unpack(ld_shared16(at + 2 * kThreads * 16), y0);
      Vec<T>::unpack(ld_shared16(at + 3 * kThreads * 16), y1);
      float2 ss = both(0.f), xt = both(0.f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        // dn = the rotation's transpose applied to dy
        const float2 n0 = __ffma2_rn(y0[i], cs[i], __fmul2_rn(y1[i], sn[i]));
        const float2 n1 = __ffma2_rn(y1[i], cs[i], neg(__fmul2_rn(y0[i], sn[i])));
        y0[i] = n0;
        y1[i] = n1;
        ss = __ffma2_rn(x0[i], x0[i], __ffma2_rn(x1[i], x1[i], ss));
        xt = __ffma2_rn(x0[i], __fmul2_rn(n0, g0[i]), __ffma2_rn(x1[i], __fmul2_rn(n1, g1[i]), xt));
      }
      ask(stage == 0 ? kRing - 1 : stage - 1);  // into the row before's place
      stage = stage + 1 == kRing ? 0 : stage + 1;
      const float rs = rsqrtf(row_sum<LPR>(ss.x + ss.y) * (1.0f / D) + p.eps);
      const float2 r = both(rs);
      // dx = r t - x r^3 mean(x t)
      const float2 k = both(-row_sum<LPR>(xt.x + xt.y) * (1.0f / D) * rs * rs * rs);
      if (h >= c.nh) continue;  // after the shuffles; no row, no share of dg
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float2 m0 = __fmul2_rn(r, y0[i]), m1 = __fmul2_rn(r, y1[i]);
        a0[i] = __ffma2_rn(x0[i], m0, a0[i]);
        a1[i] = __ffma2_rn(x1[i], m1, a1[i]);
        x0[i] = __ffma2_rn(m0, g0[i], __fmul2_rn(x0[i], k));
        x1[i] = __ffma2_rn(m1, g1[i], __fmul2_rn(x1[i], k));
      }
      st_stream(c.dst + h * dxr.sh, Vec<T>::pack(x0));
      st_stream(c.dst + h * dxr.sh + D / 2, Vec<T>::pack(x1));
    }
  }
  // the groups of a warp, then the warps of the CTA
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a0[i].x += __shfl_xor_sync(kFull, a0[i].x, o);
      a0[i].y += __shfl_xor_sync(kFull, a0[i].y, o);
      a1[i].x += __shfl_xor_sync(kFull, a1[i].x, o);
      a1[i].y += __shfl_xor_sync(kFull, a1[i].y, o);
    }
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) < LPR)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      *reinterpret_cast<float2*>(&red[warp][lane * VE + 2 * i]) = a0[i];
      *reinterpret_cast<float2*>(&red[warp][D / 2 + lane * VE + 2 * i]) = a1[i];
    }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) sum += red[i][d];
    p.partial[static_cast<int64_t>(blockIdx.x) * D + d] = sum;
  }
}

// dg[d] = sum of the CTAs' shares.  One CTA per 32 columns of dgq or dgk: 32
// row slices of 32 lanes, joined in shared memory.
__global__ void __launch_bounds__(1024) dg_join_kernel(const float* __restrict__ partial, float* __restrict__ dgq,
                                                       float* __restrict__ dgk, int D, int bq, int bk) {
  __shared__ float red[32][33];
  pdl_wait();  // the rows' kernel is done
  const int col = blockIdx.x * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  const int w = blockIdx.y;
  const int n = w ? bk : bq;
  const float* src = partial + (w ? static_cast<int64_t>(bq) * D : 0) + col;
  float s = 0.f;
#pragma unroll 4
  for (int i = slice; i < n; i += 32) s += src[static_cast<int64_t>(i) * D];
  red[slice][threadIdx.x & 31] = s;
  __syncthreads();
  s = red[threadIdx.x & 31][slice];  // lane = slice, warp = column
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  if ((threadIdx.x & 31) == 0) (w ? dgk : dgq)[blockIdx.x * 32 + slice] = s;
}

// cos and sin of position x theta^(-2 f / D), angles in double precision.
__global__ void __launch_bounds__(256) rope_table_any_kernel(float2* __restrict__ tab, int64_t n, int half,
                                                             double log2_theta) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t pos = i / half;
  const int f = static_cast<int>(i - pos * half);
  double sn, cs;
  sincos(static_cast<double>(pos) * exp2(-static_cast<double>(f) / half * log2_theta), &sn, &cs);
  tab[i] = make_float2(static_cast<float>(cs), static_cast<float>(sn));
}

constexpr int kFwdRows = 4;  // rows whose loads a group has in flight

// Heads per item: two rounds of `rows` where the rows fill the GPU many times
// over, so that the token's angles and the weights (as many load instructions
// as four bf16 rows) are paid once for both; one round otherwise.  Measured,
// forward B8 S4096 of 40 heads, 1 / 2 / 4 / 8 rounds: 120 / 109 / 140 / 127 us
// (few, short-lived items keep the reads of a CTA close together); fp32 B3 S1001 of
// 16 heads, 1 / 2 rounds: 4.8 / 5.0 us.
int heads_per_item(int64_t tokens, int64_t heads, int64_t lanes, int rows) {
  return tokens * heads * lanes >= 16 * 512ll * num_sms() ? 2 * rows : rows;
}

template <typename T, int D, int U, bool kAppend>
kda_status launch_fwd_u(FwdParams& p, int hp, cudaStream_t st) {
  constexpr int LPR = D / (2 * Vec<T>::kN);
  p.hp = hp;
  p.cq = static_cast<unsigned>((p.QH + hp - 1) / hp);
  p.ck = static_cast<unsigned>((p.KH + hp - 1) / hp);
  const int64_t items = static_cast<int64_t>(p.B) * p.S * (p.cq + p.ck * (kAppend ? 2 : 1));
  KDA_CHECK_SUPPORTED(items * LPR < (1ll << 32), "qk_norm_rope: too many rows (%lld tokens)", (long long)p.B * p.S);
  const int64_t grid = (items * LPR + kThreads - 1) / kThreads;
  return launch_after(kAppend ? "qk_norm_rope_append" : "qk_norm_rope", norm_rope_kernel<T, D, U, kAppend>,
                      dim3(static_cast<unsigned>(grid)), kThreads, 0, st, p, kda_err_ptr_qk_norm());
}

template <typename T, int D, bool kAppend>
kda_status launch_fwd_d(FwdParams& p, cudaStream_t st) {
  constexpr int LPR = D / (2 * Vec<T>::kN);
  const int64_t tokens = static_cast<int64_t>(p.B) * p.S;
  // few rows: one per group of lanes, so that all of them load at once
  if (tokens * (p.QH + p.KH) * LPR <= 512ll * num_sms()) return launch_fwd_u<T, D, 1, kAppend>(p, 1, st);
  return launch_fwd_u<T, D, kFwdRows, kAppend>(
      p, heads_per_item(tokens, p.QH + p.KH, LPR, kFwdRows), st);
}

template <typename T, bool kAppend>
kda_status launch_fwd(FwdParams& p, int64_t D, cudaStream_t st) {
  switch (D) {
    case 64: return launch_fwd_d<T, 64, kAppend>(p, st);
    case 128: return launch_fwd_d<T, 128, kAppend>(p, st);
    default: return launch_fwd_d<T, 256, kAppend>(p, st);
  }
}

// The backward's items and CTAs: one CTA per round of work up to eight per SM;
// beyond that the two that are resident on each SM, shared between queries and
// keys in proportion to their rows.  A CTA per round / resident CTAs: 777 tokens of
// 9 heads of 256 6.7 / 8.4 us, 2048 of 24 heads of 128 11.3 / 12.8, 8192 of 10 (five
// rounds per SM) 19.2 / 20.6, 8192 of 40 (17 per SM: the shares of dg) 60 / 45.
void bwd_split(int64_t tokens, int64_t QH, int64_t KH, int64_t D, bool f32, int (&hp)[2], int (&blocks)[2]) {
  const int64_t lanes = D / (f32 ? 8 : 16);
  const int64_t groups = kThreads / lanes;
  const int64_t heads[2] = {QH, KH};
  int64_t rounds[2];
  for (int w = 0; w < 2; ++w) {
    hp[w] = kBwdHeads;
    rounds[w] = (tokens * ((heads[w] + hp[w] - 1) / hp[w]) + groups - 1) / groups;
  }
  const bool few = rounds[0] + rounds[1] <= 8ll * num_sms();
  for (int w = 0; w < 2; ++w) {
    const int64_t share = std::max<int64_t>(1, 2ll * num_sms() * heads[w] / (QH + KH));
    blocks[w] = static_cast<int>(few ? rounds[w] : std::min(rounds[w], share));
  }
}

template <typename T, int D>
kda_status launch_bwd_d(const BwdParams& p, float* dgq, float* dgk, cudaStream_t st) {
  const int64_t most = static_cast<int64_t>(p.B) * p.S *
                       std::max((p.H[0] + p.hp[0] - 1) / p.hp[0], (p.H[1] + p.hp[1] - 1) / p.hp[1]);
  KDA_CHECK_SUPPORTED(most < (1ll << 31), "qk_norm_rope_backward: too many rows (%lld tokens)", (long long)p.B * p.S);
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(norm_rope_bwd_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kRingBytes)) != cudaSuccess)
      return launch_status("qk_norm_rope_backward: cudaFuncSetAttribute");
    attr_set[dev].store(true, std::memory_order_release);
  }
  const kda_status s = launch_after("qk_norm_rope_backward", norm_rope_bwd_kernel<T, D>,
                                    dim3(static_cast<unsigned>(p.blocks[0] + p.blocks[1])), kThreads, kRingBytes, st, p,
                                    kda_err_ptr_qk_norm());
  if (s != KDA_OK) return s;
  return launch_after("qk_norm_rope_backward: dg", dg_join_kernel, dim3(D / 32, 2), 1024, 0, st, p.partial, dgq, dgk, D,
                      p.blocks[0], p.blocks[1]);
}

template <typename T>
kda_status launch_bwd(const BwdParams& p, int64_t D, float* dgq, float* dgk, cudaStream_t st) {
  switch (D) {
    case 64: return launch_bwd_d<T, 64>(p, dgq, dgk, st);
    case 128: return launch_bwd_d<T, 128>(p, dgq, dgk, st);
    default: return launch_bwd_d<T, 256>(p, dgq, dgk, st);
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// every row of [n0][n1][n2] starts on 16 bytes (an axis of one entry may have any stride)
bool rows_ok(const void* p, const int64_t* s, int64_t n0, int64_t n1, int64_t n2, int es) {
  return al16(p) && (n0 == 1 || s[0] * es % 16 == 0) && (n1 == 1 || s[1] * es % 16 == 0) &&
         (n2 == 1 || s[2] * es % 16 == 0);
}

kda_status common_check(const char* op, int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, float eps) {
  KDA_CHECK_ARG(B > 0 && S > 0 && QH > 0 && KH > 0, "%s: bad sizes B=%lld S=%lld QH=%lld KH=%lld", op, (long long)B,
                (long long)S, (long long)QH, (long long)KH);
  KDA_CHECK_ARG(eps >= 0.f, "%s: eps must not be negative", op);
  KDA_CHECK_SUPPORTED(D == 64 || D == 128 || D == 256, "%s: head_dim must be 64, 128 or 256, got %lld", op,
                      (long long)D);
  KDA_CHECK_SUPPORTED(B < (1ll << 31) && S < (1ll << 31) && B * S < (1ll << 31) && QH <= 65535 && KH <= 65535,
                      "%s: too many rows (B=%lld S=%lld QH=%lld KH=%lld)", op, (long long)B, (long long)S,
                      (long long)QH, (long long)KH);
  return KDA_OK;
}

}  // namespace
}  // namespace kda

using namespace kda;

#define KDA_TRY_QK(expr)         \
  do {                           \
    const kda_status s_ = (expr); \
    if (s_ != KDA_OK) return s_; \
  } while (0)

extern "C" kda_status kda_rope_table_f32(float* table, int64_t length, int64_t D, double theta, void* stream) {
  KDA_CHECK_ARG(table && length > 0 && D > 0 && D % 2 == 0 && theta > 0.0,
                "rope_table: bad arguments length=%lld D=%lld theta=%g", (long long)length, (long long)D, theta);
  KDA_CHECK_SUPPORTED(length <= (1ll << 38) / D, "rope_table: too many positions (%lld)", (long long)length);
  const int64_t n = length * (D / 2);
  rope_table_any_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<float2*>(table), n, static_cast<int>(D / 2), log2(theta));
  return launch_status("rope_table");
}

extern "C" kda_status kda_qk_norm_rope(const void* q, const void* k, const float* gq, const float* gk,
                                       const float* table, int64_t table_len, const int* positions, float eps,
                                       void* q_out, void* k_out, int64_t B, int64_t S, int64_t QH, int64_t KH,
                                       int64_t D, const int64_t* q_strides, const int64_t* k_strides, int f32,
                                       void* stream) {
  const char* op = "qk_norm_rope";
  KDA_TRY_QK(common_check(op, B, S, QH, KH, D, eps));
  KDA_CHECK_ARG(q && k && gq && gk && table && q_out && k_out && q_strides && k_strides, "%s: null pointer", op);
  KDA_CHECK_ARG(table_len > 0 && (positions || table_len >= S), "%s: table of %lld positions for %lld tokens", op,
                (long long)table_len, (long long)S);
  const int es = f32 ? 4 : 2;
  KDA_CHECK_SUPPORTED(rows_ok(q, q_strides, B, S, QH, es) && rows_ok(k, k_strides, B, S, KH, es) && al16(gq) &&
                          al16(gk) && al16(table) && al16(q_out) && al16(k_out),
                      "%s: pointers and rows must be 16-byte aligned", op);
  FwdParams p{};
  p.q = {q, q_strides[0], q_strides[1], q_strides[2]};
  p.k = {k, k_strides[0], k_strides[1], k_strides[2]};
  p.qo = {q_out, S * QH * D, QH * D, D};
  p.ko = {k_out, S * KH * D, KH * D, D};
  p.gq = gq;
  p.gk = gk;
  p.table = table;
  p.table_len = table_len;
  p.positions = positions;
  p.eps = eps;
  p.B = static_cast<int>(B);
  p.S = static_cast<int>(S);
  p.QH = static_cast<int>(QH);
  p.KH = static_cast<int>(KH);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return f32 ? launch_fwd<float, false>(p, D, st) : launch_fwd<__nv_bfloat16, false>(p, D, st);
}

extern "C" kda_status kda_qk_norm_rope_append_bf16(const void* q, const void* k, const void* v, const float* gq,
                                                   const float* gk, const float* table, int64_t table_len,
                                                   const int* lengths, float eps, void* q_out, void* k_cache,
                                                   void* v_cache, int64_t cache_len, int64_t B, int64_t S, int64_t QH,
                                                   int64_t KH, int64_t D, const int64_t* q_strides,
                                                   const int64_t* k_strides, const int64_t* v_strides,
                                                   const int64_t* k_cache_strides, const int64_t* v_cache_strides,
                                                   void* stream) {
  const char* op = "qk_norm_rope_append";
  KDA_TRY_QK(common_check(op, B, S, QH, KH, D, eps));
  KDA_CHECK_ARG(q && k && v && gq && gk && table && lengths && q_out && k_cache && v_cache && q_strides && k_strides &&
                    v_strides && k_cache_strides && v_cache_strides,
                "%s: null pointer", op);
  KDA_CHECK_ARG(table_len > 0 && cache_len > 0, "%s: empty table or cache", op);
  KDA_CHECK_SUPPORTED(rows_ok(q, q_strides, B, S, QH, 2) && rows_ok(k, k_strides, B, S, KH, 2) &&
                          rows_ok(v, v_strides, B, S, KH, 2) && rows_ok(k_cache, k_cache_strides, B, cache_len, KH, 2) &&
                          rows_ok(v_cache, v_cache_strides, B, cache_len, KH, 2) && al16(gq) && al16(gk) && al16(table) &&
                          al16(q_out),
                      "%s: pointers and rows must be 16-byte aligned", op);
  FwdParams p{};
  p.q = {q, q_strides[0], q_strides[1], q_strides[2]};
  p.k = {k, k_strides[0], k_strides[1], k_strides[2]};
  p.v = {v, v_strides[0], v_strides[1], v_strides[2]};
  p.qo = {q_out, S * QH * D, QH * D, D};
  p.ko = {k_cache, k_cache_strides[0], k_cache_strides[1], k_cache_strides[2]};
  p.vo = {v_cache, v_cache_strides[0], v_cache_strides[1], v_cache_strides[2]};
  p.gq = gq;
  p.gk = gk;
  p.table = table;
  p.table_len = table_len;
  p.cache_len = cache_len;
  p.lengths = lengths;
  p.eps = eps;
  p.B = static_cast<int>(B);
  p.S = static_cast<int>(S);
  p.QH = static_cast<int>(QH);
  p.KH = static_cast<int>(KH);
  return launch_fwd<__nv_bfloat16, true>(p, D, static_cast<cudaStream_t>(stream));
}

extern "C" size_t kda_qk_norm_rope_backward_workspace_size(int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D,
                                                           int f32) {
  if (B <= 0 || S <= 0 || QH <= 0 || KH <= 0 || (D != 64 && D != 128 && D != 256)) return 0;
  int hp[2], blocks[2];
  bwd_split(B * S, QH, KH, D, f32 != 0, hp, blocks);
  return static_cast<size_t>(blocks[0] + blocks[1]) * D * 4;
}

extern "C" kda_status kda_qk_norm_rope_backward(const void* dq_out, const void* dk_out, const void* q, const void* k,
                                                const float* gq, const float* gk, const float* table,
                                                int64_t table_len, const int* positions, float eps, void* dq, void* dk,
                                                float* dgq, float* dgk, int64_t B, int64_t S, int64_t QH, int64_t KH,
                                                int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                                                int f32, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "qk_norm_rope_backward";
  KDA_TRY_QK(common_check(op, B, S, QH, KH, D, eps));
  KDA_CHECK_ARG(dq_out && dk_out && q && k && gq && gk && table && dq && dk && dgq && dgk && q_strides && k_strides,
                "%s: null pointer", op);
  KDA_CHECK_ARG(table_len > 0 && (positions || table_len >= S), "%s: table of %lld positions for %lld tokens", op,
                (long long)table_len, (long long)S);
  const int es = f32 ? 4 : 2;
  KDA_CHECK_SUPPORTED(rows_ok(q, q_strides, B, S, QH, es) && rows_ok(k, k_strides, B, S, KH, es) && al16(dq_out) &&
                          al16(dk_out) && al16(gq) && al16(gk) && al16(table) && al16(dq) && al16(dk),
                      "%s: pointers and rows must be 16-byte aligned", op);
  const size_t need = kda_qk_norm_rope_backward_workspace_size(B, S, QH, KH, D, f32);
  KDA_CHECK_ARG(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes required, got %zu", op, need,
                workspace_bytes);
  KDA_CHECK_SUPPORTED(al16(workspace), "%s: workspace must be 16-byte aligned", op);
  BwdParams p{};
  const int64_t H[2] = {QH, KH};
  const void* x[2] = {q, k};
  const void* dy[2] = {dq_out, dk_out};
  void* dx[2] = {dq, dk};
  const int64_t* xs[2] = {q_strides, k_strides};
  const float* g[2] = {gq, gk};
  for (int w = 0; w < 2; ++w) {
    p.x[w] = {x[w], xs[w][0], xs[w][1], xs[w][2]};
    p.dy[w] = {dy[w], S * H[w] * D, H[w] * D, D};
    p.dx[w] = {dx[w], S * H[w] * D, H[w] * D, D};
    p.g[w] = g[w];
    p.H[w] = static_cast<int>(H[w]);
  }
  p.table = table;
  p.table_len = table_len;
  p.positions = positions;
  p.eps = eps;
  p.B = static_cast<int>(B);
  p.S = static_cast<int>(S);
  bwd_split(B * S, QH, KH, D, f32 != 0, p.hp, p.blocks);
  p.partial = static_cast<float*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return f32 ? launch_bwd<float>(p, D, dgq, dgk, st) : launch_bwd<__nv_bfloat16>(p, D, dgq, dgk, st);
}
