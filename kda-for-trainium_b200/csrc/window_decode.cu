// Grouped-query attention of one new token per request against a key/value
// cache, with a sliding window and sinks (head_dim 128, bf16).
//
// With n = lengths[b] cached tokens (the new one among them), query head h sees
// the keys j < n where j >= n - window or j < sinks:
//   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = q . k_j log2e / sqrt(128)
//
// HBM-bound: every visible key and value row is read once, 256 bytes each, for
// up to 16 query heads of its group (once more for each 16 beyond).  The visible keys are numbered through
// (x < ns: the sinks before the window, then the window) and cut into tiles of
// 16; a cluster of CTAs shares the tiles of one (request, kv head), and every
// warp streams its own tiles through a private cp.async ring, so the loop has
// no CTA barrier.  The products are transposed so that the few query heads are
// the narrow side of the m16n8k16 matrix instruction:
//   S^T (16 keys x 8 heads)  = K q^T          O^T (128 x 8 heads) += V^T P^T
// (8 heads padded would fill half of an m16 tile with the heads as rows; the
// tcgen05 shapes start at 64 rows and gain nothing at a few flops per byte).
// P^T goes from the accumulator's layout to the operand's with movmatrix.  The
// running maximum moves only when a score exceeds it by 2^8, which fp32 sums
// and bf16 weights (up to 256, relative rounding unchanged) hold exactly as
// well; so a tile usually needs no exchange between lanes.  At the end the
// warps join through shared memory, the CTAs of a cluster through distributed
// shared memory: one launch, no workspace, one fixed order of summation.
#include <math.h>

#include "window.cuh"

KDA_DEFINE_ERROR_WORD(window_decode)

namespace kda {
namespace {

constexpr int kWarps = 8;  // 192 KB of rings in one CTA per SM (4 warps, two CTAs: 148 against 143 us at 64 requests)
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 3;
constexpr int kKeys = 16;                        // keys per warp tile
constexpr uint32_t kRow = kD * 2;                // bytes of a key row
constexpr uint32_t kStage = 2 * kKeys * kRow;    // K and V rows of a tile
constexpr uint32_t kRing = kStages * kStage;     // per warp
constexpr size_t kSmem = kWarps * kRing;
constexpr unsigned kFull = 0xffffffffu;

struct DecodeParams {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* out;        // [B][QH][128]
  const int* lengths;
  int64_t q_b, q_h;          // element strides
  int64_t k_b, k_t, k_h;
  int64_t v_b, v_t, v_h;
  int64_t cache_len;
  int QH, KH, rep, parts;    // parts: groups of 8 NT query heads per kv head
  int64_t window, sinks;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
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
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// What a warp or CTA hands on: per head the running maximum, the sum, and the
// unnormalised output row.
template <int H>
struct Partial {
  float m[H], l[H];
  float o[H][kD];
};

// NT: groups of 8 query heads a CTA works on.  Grid (cluster size, KH * parts, B).
template <int NT>
__global__ void __launch_bounds__(kThreads) window_decode_kernel(const DecodeParams p, unsigned* err) {
  constexpr int H = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  static_assert(sizeof(Partial<H>) * (kWarps + 1) <= kSmem, "the partials reuse the rings");
  // The launch before this one may still be running, and the one after it may start:
  // their prologues overlap (append and decode of one request, a layer: 9.3 -> 8.6 us).
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int nsplit = static_cast<int>(cluster_nctarank());
  const int split = static_cast<int>(cluster_ctarank());
  const int b = blockIdx.z;
  const int g = static_cast<int>(blockIdx.y) / p.parts;
  const int part = static_cast<int>(blockIdx.y) - g * p.parts;
  const int h0 = g * p.rep + part * H;               // first query head
  const int nh = min(H, p.rep - part * H);

  int64_t n = __ldg(p.lengths + b);
  if (n > p.cache_len) {                             // reported; the cache's end is the end
    if (threadIdx.x == 0) atomicOr(err, static_cast<unsigned>(kErrRange));
    n = p.cache_len;
  }
  if (n < 0) n = 0;
  const int64_t start = n > p.window ? n - p.window : 0;
  const int ns = static_cast<int>(p.sinks < start ? p.sinks : start);
  const int nv = static_cast<int>(n - start) + ns;   // visible keys
  const int64_t skip = start - ns;                   // key of x >= ns: x + skip
  const int tiles = (nv + kKeys - 1) / kKeys;
  const int first = split * kWarps + warp, stride = nsplit * kWarps;

  const uint32_t ring = smem_u32(smem) + warp * kRing;
  const __nv_bfloat16* kb = p.k + b * p.k_b + g * p.k_h + (lane & 15) * 8;
  const __nv_bfloat16* vb = p.v + b * p.v_b + g * p.v_h + (lane & 15) * 8;
  // rows of 16 units of 16 bytes; unit u of row r sits at u ^ (r & 7)
  auto load = [&](int tile, int stage) {
    const uint32_t dst = ring + stage * kStage;
#pragma unroll
    for (int i = 0; i < kKeys / 2; ++i) {
      const int r = (lane >> 4) + 2 * i;
      const int x = tile * kKeys + r;
      const bool in = x < nv;
      const int64_t key = in ? (x < ns ? x : x + skip) : 0;
      const uint32_t off = r * kRow + (((lane & 15) ^ (r & 7)) << 4);
      cp_async16(dst + off, kb + key * p.k_t, in);
      cp_async16(dst + kKeys * kRow + off, vb + key * p.v_t, in);
    }
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (first + s * stride < tiles) load(first + s * stride, s);
    cp_async_commit();
  }

  // q^T operands (16 x 8 per step): head lane / 4, columns 2 (lane % 4) + {0, 1} and + 8
  uint32_t qf[NT][kD / 16][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int h = t * 8 + (lane >> 2);
    const __nv_bfloat16* qr = p.q + b * p.q_b + static_cast<int64_t>(h0 + h) * p.q_h + (lane & 3) * 2;
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk) {
      qf[t][kk][0] = h < nh ? __ldg(reinterpret_cast<const unsigned*>(qr + kk * 16)) : 0u;
      qf[t][kk][1] = h < nh ? __ldg(reinterpret_cast<const unsigned*>(qr + kk * 16 + 8)) : 0u;
    }
  }
  float m[NT][2], l[NT][2];        // heads 8 t + 2 (lane % 4) + {0, 1}; l: this lane's keys only
  float o[NT][kD / 16][4];         // rows 16 i + lane / 4 (+ 8) of O^T
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int i = 0; i < kD / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
  }

  int stage = 0;
  for (int tile = first; tile < tiles; tile += stride) {
    const int ahead = tile + (kStages - 1) * stride;
    __syncwarp();  // every lane is done with the stage refilled here
    if (ahead < tiles) load(ahead, stage == 0 ? kStages - 1 : stage - 1);
    cp_async_commit();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t ks = ring + stage * kStage, vs = ks + kKeys * kRow;
    stage = stage + 1 == kStages ? 0 : stage + 1;

    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
    // K rows (16 keys x 16 columns): matrices (keys 0-7, 8-15) x (columns 0-7, 8-15)
    const int kr = lane & 15;
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk) {
      uint32_t a[4];
      ldsm_x4(ks + kr * kRow + (((2 * kk + (lane >> 4)) ^ (kr & 7)) << 4), a);
#pragma unroll
      for (int t = 0; t < NT; ++t) mma_bf16(s[t], a, qf[t][kk][0], qf[t][kk][1]);
    }
    // keys of this lane: lane / 4 and + 8; those past the end see nothing
    const int x0 = tile * kKeys + (lane >> 2);
    if (tile + 1 == tiles) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (x0 >= nv) s[t][0] = s[t][1] = -INFINITY;
        if (x0 + 8 >= nv) s[t][2] = s[t][3] = -INFINITY;
      }
    }
    bool grow = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) grow |= fmaxf(s[t][c], s[t][c + 2]) * p.scale_log2 > m[t][c] + 8.f;
    if (__any_sync(kFull, grow)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(s[t][c], s[t][c + 2]) * p.scale_log2;
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, d));
          mx = fmaxf(mx, m[t][c]);
          // nothing finite yet: keep the (empty) sums as they are
          const float f = mx == -INFINITY ? 1.f : exp2_approx(m[t][c] - mx);
          m[t][c] = mx;
          l[t][c] *= f;
#pragma unroll
          for (int i = 0; i < kD / 16; ++i) {
            o[t][i][c] *= f;
            o[t][i][c + 2] *= f;
          }
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float e[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float mm = m[t][c & 1] == -INFINITY ? 0.f : m[t][c & 1];
        e[c] = exp2_approx(fmaf(s[t][c], p.scale_log2, -mm));
      }
      l[t][0] += e[0] + e[2];
      l[t][1] += e[1] + e[3];
      // the weights meet V as bf16, the tensor core's operand type
      pb[t][0] = transpose8x8(pack_bf16x2(e[0], e[1]));
      pb[t][1] = transpose8x8(pack_bf16x2(e[2], e[3]));
    }
    // V^T (16 columns x 16 keys): matrices (columns 0-7, 8-15) x (keys 0-7, 8-15), each stored by key
    const int vr = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
    for (int i = 0; i < kD / 16; ++i) {
      uint32_t a[4];
      ldsm_x4_t(vs + vr * kRow + (((2 * i + ((lane >> 3) & 1)) ^ (vr & 7)) << 4), a);
#pragma unroll
      for (int t = 0; t < NT; ++t) mma_bf16(o[t][i], a, pb[t][0], pb[t][1]);
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings are free: partials go there

  Partial<H>* parts = reinterpret_cast<Partial<H>*>(smem);
  {
    Partial<H>& mine = parts[1 + warp];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[t][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(kFull, sum, d);
        const int h = t * 8 + (lane & 3) * 2 + c;
        if (lane < 4) {
          mine.m[h] = m[t][c];
          mine.l[h] = sum;
        }
#pragma unroll
        for (int i = 0; i < kD / 16; ++i) {
          mine.o[h][i * 16 + (lane >> 2)] = o[t][i][c];
          mine.o[h][i * 16 + (lane >> 2) + 8] = o[t][i][c + 2];
        }
      }
  }
  __syncthreads();
  // join `count` partials (of warps, then of CTAs) at head h, column d
  auto weight = [](float mw, float mm) { return mw == -INFINITY ? 0.f : exp2_approx(mw - mm); };
  for (int i = threadIdx.x; i < H * kD; i += kThreads) {
    const int h = i / kD, d = i - h * kD;
    float mm = -INFINITY, ll = 0.f, oo = 0.f;
#pragma unroll
    for (int w = 1; w <= kWarps; ++w) mm = fmaxf(mm, parts[w].m[h]);
#pragma unroll
    for (int w = 1; w <= kWarps; ++w) {
      const float f = weight(parts[w].m[h], mm);
      ll += f * parts[w].l[h];
      oo += f * parts[w].o[h][d];
    }
    parts[0].o[h][d] = oo;
    if (d == 0) {
      parts[0].m[h] = mm;
      parts[0].l[h] = ll;
    }
  }
  cluster_sync_all();
  const uint32_t base = smem_u32(&parts[0]);
  const uint32_t off_l = static_cast<uint32_t>(offsetof(Partial<H>, l)), off_o = static_cast<uint32_t>(offsetof(Partial<H>, o));
  for (int i = split * kThreads + threadIdx.x; i < nh * kD; i += nsplit * kThreads) {
    const int h = i / kD;
    float mm = -INFINITY, ll = 0.f, oo = 0.f;
    for (int r = 0; r < nsplit; ++r) mm = fmaxf(mm, ld_cluster_f32(mapa_shared(base, r) + 4 * h));
    for (int r = 0; r < nsplit; ++r) {
      const uint32_t rb = mapa_shared(base, r);
      const float f = weight(ld_cluster_f32(rb + 4 * h), mm);
      ll += f * ld_cluster_f32(rb + off_l + 4 * h);
      oo += f * ld_cluster_f32(rb + off_o + 4 * i);
    }
    // no visible key: zeros
    p.out[(static_cast<int64_t>(b) * p.QH + h0) * kD + i] = __float2bfloat16_rn(nv > 0 ? oo / ll : 0.f);
  }
  cluster_sync_all();  // a CTA's partial is read until here
}

template <int NT>
kda_status launch_decode(const DecodeParams& p, int64_t B, int cluster, cudaStream_t st) {
  auto* kernel = window_decode_kernel<NT>;
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem)) !=
        cudaSuccess)
      return launch_status("gqa_window_decode: cudaFuncSetAttribute");
    attr_set[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster), static_cast<unsigned>(p.KH * p.parts), static_cast<unsigned>(B));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
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
  cudaLaunchKernelEx(&cfg, kernel, p, kda_err_ptr_window_decode());
  return launch_status("gqa_window_decode");
}

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" kda_status kda_gqa_window_decode_bf16(const void* q, const void* k_cache, const void* v_cache,
                                                 const int* lengths, void* out, int64_t B, int64_t T, int64_t QH,
                                                 int64_t KH, int64_t D, int64_t window, int64_t sinks,
                                                 const int64_t* q_strides, const int64_t* k_strides,
                                                 const int64_t* v_strides, void* stream) {
  const char* op = "gqa_window_decode";
  KDA_CHECK_ARG(B > 0 && T > 0 && QH > 0 && KH > 0 && QH % KH == 0, "%s: bad sizes B=%lld T=%lld QH=%lld KH=%lld", op,
                (long long)B, (long long)T, (long long)QH, (long long)KH);
  KDA_CHECK_ARG(window > 0 && sinks >= 0, "%s: window must be positive and sinks not negative, got %lld and %lld", op,
                (long long)window, (long long)sinks);
  KDA_CHECK_SUPPORTED(D == kD, "%s: head_dim must be 128, got %lld", op, (long long)D);
  KDA_CHECK_SUPPORTED(B <= 65535 && QH <= 65535 && T < (1ll << 30), "%s: too large (B=%lld QH=%lld T=%lld)", op,
                      (long long)B, (long long)QH, (long long)T);
  KDA_CHECK_ARG(q && k_cache && v_cache && lengths && out && q_strides && k_strides && v_strides, "%s: null pointer",
                op);
  const int64_t qs[3] = {q_strides[0], q_strides[1], 0};
  KDA_CHECK_SUPPORTED(head_rows_ok(q, qs, B, QH, 1) && head_rows_ok(k_cache, k_strides, B, T, KH) &&
                          head_rows_ok(v_cache, v_strides, B, T, KH) && (reinterpret_cast<uintptr_t>(out) & 15u) == 0,
                      "%s: pointers and rows must be 16-byte aligned", op);
  DecodeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k_cache);
  p.v = static_cast<const __nv_bfloat16*>(v_cache);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lengths = lengths;
  p.q_b = q_strides[0];
  p.q_h = q_strides[1];
  p.k_b = k_strides[0];
  p.k_t = k_strides[1];
  p.k_h = k_strides[2];
  p.v_b = v_strides[0];
  p.v_t = v_strides[1];
  p.v_h = v_strides[2];
  p.cache_len = T;
  p.QH = static_cast<int>(QH);
  p.KH = static_cast<int>(KH);
  p.rep = static_cast<int>(QH / KH);
  p.window = window < T ? window : T;
  p.sinks = sinks < T ? sinks : T;
  p.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(kD)));
  const bool wide = p.rep > 8;
  p.parts = wide ? (p.rep + 15) / 16 : 1;
  // CTAs per (request, kv head): up to four per SM, so that requests of ragged
  // lengths even out, each with two tiles per warp at least at the longest
  // visible length.  Eight at most: one request of 4,100 keys and 8 kv heads takes
  // 9.7 us with clusters of 8, 15.5 us with 16 (a whole GPC has to be free).
  const int64_t units = B * KH * p.parts;
  const int64_t keys = p.window + p.sinks < T ? p.window + p.sinks : T;
  int cluster = 1;
  while (cluster < 8 && units * cluster < 4ll * num_sms() && keys >= 2ll * cluster * kWarps * kKeys * 2) cluster *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return wide ? launch_decode<2>(p, B, cluster, st) : launch_decode<1>(p, B, cluster, st);
}
