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
#include "common.cuh"

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

// The 16 bytes of a lane as fp32 values and back.
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void unpack(const uint4 v, float (&f)[8]) { unpack_bf16x8(v, f); }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void unpack(const uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
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
  int cq, ck;                // head chunks of a token's queries, of its keys (append: and of its values)
  float eps;
};

template <int LPR>
__device__ __forceinline__ float row_sum(float s) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  return s;
}

template <int N>
__device__ __forceinline__ void load_f32(const float* p, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
    f[4 * i] = v.x;
    f[4 * i + 1] = v.y;
    f[4 * i + 2] = v.z;
    f[4 * i + 3] = v.w;
  }
}

// One group of LPR lanes per item = U heads of one token (all queries, all
// keys or all values): the U rows' loads are issued before anything waits.
template <typename T, int D, int U, bool kAppend>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const FwdParams p, unsigned* err) {
  constexpr int VE = Vec<T>::kN;
  constexpr int LPR = D / (2 * VE);
  const int lane = threadIdx.x % LPR;  // owns values [VE lane, + VE) of both halves
  const int nc = p.cq + p.ck * (kAppend ? 2 : 1);
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / LPR;
  const bool live = item < static_cast<int64_t>(p.B) * p.S * nc;  // whole groups; idle ones keep up the shuffles
  const int64_t tok = live ? item / nc : 0;
  int c = live ? static_cast<int>(item - tok * nc) : 0;
  const int b = static_cast<int>(tok / p.S);
  const int s = static_cast<int>(tok - static_cast<int64_t>(b) * p.S);
  const int kind = c < p.cq ? 0 : c < p.cq + p.ck ? 1 : 2;
  c -= kind == 0 ? 0 : kind == 1 ? p.cq : p.cq + p.ck;
  const Rows in = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
  const RowsOut out = kind == 0 ? p.qo : kind == 1 ? p.ko : p.vo;
  const int h0 = c * U;
  const int nh = min(U, (kind == 0 ? p.QH : p.KH) - h0);

  const T* src = static_cast<const T*>(in.p) + b * in.sb + s * in.ss + h0 * in.sh + lane * VE;
  uint4 lo[U], hi[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (live && u < nh) {
      lo[u] = ld_stream(src + u * in.sh);
      hi[u] = ld_stream(src + u * in.sh + D / 2);
    }

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
  const bool write = live && (!kAppend || kind == 0 || !(bad || idle));

  if (kAppend && kind == 2) {  // values go to the cache as they are
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (write && u < nh) {
        st_stream(dst + u * out.sh, lo[u]);
        st_stream(dst + u * out.sh + D / 2, hi[u]);
      }
  }
  float cs[2 * VE], g0[VE], g1[VE];
  const float* g = kind == 0 ? p.gq : p.gk;
  load_f32(p.table + ((bad ? 0 : pos) * (D / 2) + lane * VE) * 2, cs);
  load_f32(g + lane * VE, g0);
  load_f32(g + D / 2 + lane * VE, g1);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool on = live && u < nh && kind != 2;
    float x0[VE], x1[VE];
    Vec<T>::unpack(on ? lo[u] : make_uint4(0u, 0u, 0u, 0u), x0);
    Vec<T>::unpack(on ? hi[u] : make_uint4(0u, 0u, 0u, 0u), x1);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VE; ++i) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
    const float r = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + p.eps);
    float y0[VE], y1[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float n0 = x0[i] * r * g0[i], n1 = x1[i] * r * g1[i];
      y0[i] = n0 * cs[2 * i] - n1 * cs[2 * i + 1];
      y1[i] = n0 * cs[2 * i + 1] + n1 * cs[2 * i];
      if (bad) y0[i] = y1[i] = __int_as_float(0x7fffffff);
      if (kAppend && idle) y0[i] = y1[i] = 0.f;
    }
    if (write && on) {
      st_stream(dst + u * out.sh, Vec<T>::pack(y0));
      st_stream(dst + u * out.sh + D / 2, Vec<T>::pack(y1));
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
  int blocks[2];             // CTAs of the queries, of the keys
  float* partial;            // [blocks[0] + blocks[1]][D]: each CTA's share of dg
  float eps;
};

// CTAs [0, blocks[0]) walk the queries, the others the keys; a group of LPR
// lanes takes U heads of a token at a time.  Each thread sums its columns of
// dg over all its rows in registers; the CTA's sums go to `partial` in a fixed
// order, so the result does not depend on timing.
template <typename T, int D, int U>
__global__ void __launch_bounds__(kThreads) norm_rope_bwd_kernel(const BwdParams p, unsigned* err) {
  constexpr int VE = Vec<T>::kN;
  constexpr int LPR = D / (2 * VE);
  constexpr int kGroups = kThreads / LPR;
  __shared__ float red[kThreads / 32][D];
  const int lane = threadIdx.x % LPR;
  const int w = static_cast<int>(blockIdx.x) < p.blocks[0] ? 0 : 1;
  const int block = static_cast<int>(blockIdx.x) - (w ? p.blocks[0] : 0);
  const Rows xr = p.x[w], dyr = p.dy[w];
  const RowsOut dxr = p.dx[w];
  const int H = p.H[w];
  const int nc = (H + U - 1) / U;
  const int64_t items = static_cast<int64_t>(p.B) * p.S * nc;
  float g0[VE], g1[VE], a0[VE], a1[VE];
  load_f32(p.g[w] + lane * VE, g0);
  load_f32(p.g[w] + D / 2 + lane * VE, g1);
#pragma unroll
  for (int i = 0; i < VE; ++i) a0[i] = a1[i] = 0.f;

  // every group of a warp makes the same number of rounds (the shuffles need all lanes)
  const int64_t step = static_cast<int64_t>(p.blocks[w]) * kGroups;
  for (int64_t base = static_cast<int64_t>(block) * kGroups; base < items; base += step) {
    const int64_t item = base + threadIdx.x / LPR;
    const bool live = item < items;
    const int64_t tok = live ? item / nc : 0;
    const int h0 = live ? static_cast<int>(item - tok * nc) * U : 0;
    const int nh = min(U, H - h0);
    const int b = static_cast<int>(tok / p.S);
    const int s = static_cast<int>(tok - static_cast<int64_t>(b) * p.S);
    const T* xs = static_cast<const T*>(xr.p) + b * xr.sb + s * xr.ss + h0 * xr.sh + lane * VE;
    const T* ds = static_cast<const T*>(dyr.p) + b * dyr.sb + s * dyr.ss + h0 * dyr.sh + lane * VE;
    T* dst = static_cast<T*>(dxr.p) + b * dxr.sb + s * dxr.ss + h0 * dxr.sh + lane * VE;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 xl[U], xh[U], dl[U], dh[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      xl[u] = xh[u] = dl[u] = dh[u] = zero;
      if (live && u < nh) {
        xl[u] = ld_stream(xs + u * xr.sh);
        xh[u] = ld_stream(xs + u * xr.sh + D / 2);
        dl[u] = ld_stream(ds + u * dyr.sh);
        dh[u] = ld_stream(ds + u * dyr.sh + D / 2);
      }
    }
    int64_t pos = s;
    if (p.positions) pos = __ldg(p.positions + tok);
    const bool bad = pos < 0 || pos >= p.table_len;
    if (bad && live && lane == 0) atomicOr(err, static_cast<unsigned>(kErrRange));
    float cs[2 * VE];
    load_f32(p.table + ((bad ? 0 : pos) * (D / 2) + lane * VE) * 2, cs);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x0[VE], x1[VE], y0[VE], y1[VE];
      Vec<T>::unpack(xl[u], x0);
      Vec<T>::unpack(xh[u], x1);
      Vec<T>::unpack(dl[u], y0);
      Vec<T>::unpack(dh[u], y1);
      float ss = 0.f, xt = 0.f;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        // dn = the rotation's transpose applied to dy
        const float n0 = y0[i] * cs[2 * i] + y1[i] * cs[2 * i + 1];
        const float n1 = y1[i] * cs[2 * i] - y0[i] * cs[2 * i + 1];
        y0[i] = bad ? __int_as_float(0x7fffffff) : n0;
        y1[i] = bad ? __int_as_float(0x7fffffff) : n1;
        ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
        xt = fmaf(x0[i], y0[i] * g0[i], fmaf(x1[i], y1[i] * g1[i], xt));
      }
      const float r = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + p.eps);
      const float k = row_sum<LPR>(xt) * (1.0f / D) * r * r;  // dx = r (t - x r^2 mean(x t))
      const bool on = live && u < nh;
      float o0[VE], o1[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        o0[i] = r * (y0[i] * g0[i] - x0[i] * k);
        o1[i] = r * (y1[i] * g1[i] - x1[i] * k);
        if (on) {  // a row that is not there has r = 1 / sqrt(eps), infinite for eps = 0
          a0[i] = fmaf(x0[i] * r, y0[i], a0[i]);
          a1[i] = fmaf(x1[i] * r, y1[i], a1[i]);
        }
      }
      if (on) {
        st_stream(dst + u * dxr.sh, Vec<T>::pack(o0));
        st_stream(dst + u * dxr.sh + D / 2, Vec<T>::pack(o1));
      }
    }
  }
  // the groups of a warp, then the warps of the CTA
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      a0[i] += __shfl_xor_sync(kFull, a0[i], o);
      a1[i] += __shfl_xor_sync(kFull, a1[i], o);
    }
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) < LPR)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      red[warp][lane * VE + i] = a0[i];
      red[warp][D / 2 + lane * VE + i] = a1[i];
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

// Forward CTAs take U heads of a token per group of lanes.
constexpr int kFwdHeads = 4;
constexpr int kBwdHeads = 2;

template <typename T, int D, bool kAppend>
kda_status launch_fwd_d(FwdParams& p, cudaStream_t st) {
  constexpr int LPR = D / (2 * Vec<T>::kN);
  p.cq = (p.QH + kFwdHeads - 1) / kFwdHeads;
  p.ck = (p.KH + kFwdHeads - 1) / kFwdHeads;
  const int64_t items = static_cast<int64_t>(p.B) * p.S * (p.cq + p.ck * (kAppend ? 2 : 1));
  const int64_t grid = (items * LPR + kThreads - 1) / kThreads;
  norm_rope_kernel<T, D, kFwdHeads, kAppend>
      <<<static_cast<unsigned>(grid), kThreads, 0, st>>>(p, kda_err_ptr_qk_norm());
  return launch_status(kAppend ? "qk_norm_rope_append" : "qk_norm_rope");
}

template <typename T, bool kAppend>
kda_status launch_fwd(FwdParams& p, int64_t D, cudaStream_t st) {
  switch (D) {
    case 64: return launch_fwd_d<T, 64, kAppend>(p, st);
    case 128: return launch_fwd_d<T, 128, kAppend>(p, st);
    default: return launch_fwd_d<T, 256, kAppend>(p, st);
  }
}

// CTAs of the backward: four per SM, shared between queries and keys in
// proportion to their rows, no more than there are rounds of work.
void bwd_blocks(int64_t tokens, int64_t QH, int64_t KH, int64_t D, bool f32, int (&blocks)[2]) {
  const int64_t groups = kThreads / (D / (f32 ? 8 : 16));
  const int64_t total = 4ll * num_sms();
  const int64_t heads[2] = {QH, KH};
  for (int w = 0; w < 2; ++w) {
    const int64_t rounds = (tokens * ((heads[w] + kBwdHeads - 1) / kBwdHeads) + groups - 1) / groups;
    int64_t n = total * heads[w] / (QH + KH);
    if (n < 1) n = 1;
    blocks[w] = static_cast<int>(rounds < n ? rounds : n);
  }
}

template <typename T, int D>
kda_status launch_bwd_d(const BwdParams& p, float* dgq, float* dgk, cudaStream_t st) {
  norm_rope_bwd_kernel<T, D, kBwdHeads>
      <<<static_cast<unsigned>(p.blocks[0] + p.blocks[1]), kThreads, 0, st>>>(p, kda_err_ptr_qk_norm());
  const kda_status s = launch_status("qk_norm_rope_backward");
  if (s != KDA_OK) return s;
  dg_join_kernel<<<dim3(D / 32, 2), 1024, 0, st>>>(p.partial, dgq, dgk, D, p.blocks[0], p.blocks[1]);
  return launch_status("qk_norm_rope_backward: dg");
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
// every row starts on 16 bytes
bool rows_ok(const void* p, const int64_t* s, int es) {
  return al16(p) && s[0] * es % 16 == 0 && s[1] * es % 16 == 0 && s[2] * es % 16 == 0;
}

kda_status common_check(const char* op, int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, float eps) {
  KDA_CHECK_ARG(B > 0 && S > 0 && QH > 0 && KH > 0, "%s: bad sizes B=%lld S=%lld QH=%lld KH=%lld", op, (long long)B,
                (long long)S, (long long)QH, (long long)KH);
  KDA_CHECK_ARG(eps >= 0.f, "%s: eps must not be negative", op);
  KDA_CHECK_SUPPORTED(D == 64 || D == 128 || D == 256, "%s: head_dim must be 64, 128 or 256, got %lld", op,
                      (long long)D);
  KDA_CHECK_SUPPORTED(B <= (1ll << 31) - 1 && S <= (1ll << 31) - 1 && QH <= 65535 && KH <= 65535 &&
                          B * S <= (1ll << 36) / (QH + 2 * KH),
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

extern "C" kda_status kda_rope_table_f32(float* table, int64_t length, int64_t D, float theta, void* stream) {
  KDA_CHECK_ARG(table && length > 0 && D > 0 && D % 2 == 0 && theta > 0.f,
                "rope_table: bad arguments length=%lld D=%lld theta=%g", (long long)length, (long long)D, theta);
  KDA_CHECK_SUPPORTED(length <= (1ll << 38) / D, "rope_table: too many positions (%lld)", (long long)length);
  const int64_t n = length * (D / 2);
  rope_table_any_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<float2*>(table), n, static_cast<int>(D / 2), log2(static_cast<double>(theta)));
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
  KDA_CHECK_SUPPORTED(rows_ok(q, q_strides, es) && rows_ok(k, k_strides, es) && al16(gq) && al16(gk) && al16(table) &&
                          al16(q_out) && al16(k_out),
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
  KDA_CHECK_SUPPORTED(rows_ok(q, q_strides, 2) && rows_ok(k, k_strides, 2) && rows_ok(v, v_strides, 2) &&
                          rows_ok(k_cache, k_cache_strides, 2) && rows_ok(v_cache, v_cache_strides, 2) && al16(gq) &&
                          al16(gk) && al16(table) && al16(q_out),
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
  int blocks[2];
  bwd_blocks(B * S, QH, KH, D, f32 != 0, blocks);
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
  KDA_CHECK_SUPPORTED(rows_ok(q, q_strides, es) && rows_ok(k, k_strides, es) && al16(dq_out) && al16(dk_out) &&
                          al16(gq) && al16(gk) && al16(table) && al16(dq) && al16(dk),
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
  bwd_blocks(B * S, QH, KH, D, f32 != 0, p.blocks);
  p.partial = static_cast<float*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return f32 ? launch_bwd<float>(p, D, dgq, dgk, st) : launch_bwd<__nv_bfloat16>(p, D, dgq, dgk, st);
}
