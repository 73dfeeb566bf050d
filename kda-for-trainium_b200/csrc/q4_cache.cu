// Writing and reading back the 4-bit key/value cache (layout: q4.cuh).
//
// Append, per (token, head) row of k and of v and per group of channels:
//   low = min x,  step = bf16((max x - low) / 15),  code = round((x - low) / step)
// low is one of the bf16 inputs, so it is exact.  The operations are single fp32 ones in
// this order: x - low, times the fp32 reciprocal of step, rounded to nearest even, at most
// 15; (max - low) times the fp32 1/15.  A step below 2^-126 becomes zero (every value reads
// back as low).  A group with an infinity or a NaN, or wider than fp32 holds, reads back as NaN.
//
// 16 lanes take a row, 8 channels each (one 16-byte load, one 4-byte store of codes), a
// group's minimum and maximum by exchanges of bf16 pairs.  Bandwidth-bound: 656 bytes a
// row of k and v; 20.4 us for 18,700 tokens of 8 heads, floor 15.0; 92 for 100,000, floor 80.
// Reading back, of buffers that do not stay in the L2: 54.5 us for 131,072 tokens of 8 heads, floor
// 52.5; 15.9 for 32,768, floor 13.1.  (12.5 for those again and again into one buffer, 13.7 with codes
// converted one by one: the integer pipe was full.)
#include <cuda_fp16.h>

#include "launch.cuh"
#include "q4.cuh"

KDA_DEFINE_ERROR_WORD(q4_cache)

namespace kda {
namespace {

constexpr int kThreads = 256;

struct AppendParams {
  const __nv_bfloat16 *k, *v;
  uint8_t *k_cache, *v_cache;
  const int* offsets;  // [B + 1] rows of each request, or null: `per` rows each
  const int* lengths;  // [B] tokens cached already; below zero: an idle slot
  unsigned rows;       // tokens in k and v
  unsigned per;
  int64_t k_b, k_t, k_h, v_b, v_t, v_h;  // element strides
  int64_t kc_b, kc_h, vc_b, vc_h;        // byte strides
  int64_t cache_len;
  int B, KH;
  int heads;           // of a CTA
};

__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// One row's 8 channels of this lane: codes (the word's nibbles) and the group's (step, low).
template <int GROUP>
__device__ __forceinline__ void quantise(const uint4 x, unsigned mask, uint32_t* word, uint32_t* pair) {
  uint32_t lo = min2(min2(x.x, x.y), min2(x.z, x.w)), hi = max2(max2(x.x, x.y), max2(x.z, x.w));
  lo ^= 0x80008000u;  // the least is the negative of the largest -x, so one word holds both
  uint32_t most = max2(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
#pragma unroll
  for (int d = 1; d < GROUP / 8; d <<= 1) most = max2(most, __shfl_xor_sync(mask, most, d));
  const float nlow = __uint_as_float(most << 16), high = __uint_as_float(most & 0xffff0000u);
  float step = __bfloat162float(__float2bfloat16_rn(__fmul_rn(__fadd_rn(high, nlow), 1.0f / 15.0f)));
  if (step < 1.1754943508222875e-38f) step = 0.f;
  if (step > 3.3895313892515355e38f) step = __uint_as_float(0x7fc00000u);  // an infinity, or past bf16's largest
  const float inv = step > 0.f ? __frcp_rn(step) : 0.f;  // NaN: zero codes beside a NaN pair
  // Adding 2^23 rounds to a whole number (ties to even), left in the low mantissa bits; the
  // shifted sum of the eight bit patterns is the word, and eight times 2^23's pattern shifted.
  // No code is past 15: step is off by 2^-8 of itself at most, and (max - low) / step then
  // below 15.06.
  float f[8];
  unpack_bf16x8(x, f);
  uint32_t w = 0u - 0x4b000000u * 0x11111111u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 t = __fadd2_rn(make_float2(f[2 * i], f[2 * i + 1]), make_float2(nlow, nlow));
    // __fmul_rn, not __fmul2_rn, which the compiler may fuse with the addition: a product that
    // rounds to a tie would then be rounded as what it was before
    t = __fadd2_rn(make_float2(__fmul_rn(t.x, inv), __fmul_rn(t.y, inv)), make_float2(8388608.f, 8388608.f));
    w += __float_as_uint(t.x) * (1u << (8 * i)) + __float_as_uint(t.y) * (16u << (8 * i));
  }
  *word = w;
  *pair = __byte_perm(__float_as_uint(step), most ^ 0x8000u, 0x5432);
}

// The request that row `row` belongs to: the last one whose first row is not after it, 16 at
// a time by the 16 lanes of `mask` (l: which of them).
__device__ __forceinline__ int request_of(const int* offsets, int B, int row, int l, unsigned mask) {
  int lo = 0, n = B;  // among [lo, lo + n)
  while (n > 1) {
    const int step = (n + 15) >> 4;
    const bool in = l == 0 || (l * step < n && __ldg(offsets + lo + l * step) <= row);
    const int last = 31 - __clz(static_cast<int>((__ballot_sync(mask, in) & mask) >> (threadIdx.x & 16)));
    n = min(step, n - last * step);
    lo += last * step;
  }
  return lo;
}

// A CTA takes 16 tokens, 16 lanes each, and p.heads of their heads one after the other, k and v
// together: the first head's loads are issued first, and while they are under way each token's
// request is looked up, once for all heads; the next head's loads are issued before a head is
// quantised.  (A CTA of 16 (token, head) pairs, nothing under way while they are quantised: 27.2 us
// for 18,700 tokens of 8 heads against 20.4, 134 for 100,000 against 92, 2.1 for 64 against 1.8.)
constexpr int kItems = kThreads / 16;
template <int GROUP>
__global__ void __launch_bounds__(kThreads) q4_append_kernel(const AppendParams p, unsigned* err) {
  pdl_trigger();
  pdl_wait();
  const int l = threadIdx.x & 15;
  const unsigned mask = 0xffffu << (threadIdx.x & 16);
  const unsigned i = blockIdx.x * kItems + (threadIdx.x >> 4);  // < 2^31
  const unsigned row = min(i, p.rows - 1);
  const int h0 = blockIdx.y * p.heads;
  int left = min(p.heads, p.KH - h0);
  const unsigned of = p.offsets ? 0u : row / p.per, in = row - of * p.per;
  const __nv_bfloat16* k = p.k + of * p.k_b + in * p.k_t + h0 * p.k_h + 8 * l;
  const __nv_bfloat16* v = p.v + of * p.v_b + in * p.v_t + h0 * p.v_h + 8 * l;
  uint4 xk = *reinterpret_cast<const uint4*>(k), xv = *reinterpret_cast<const uint4*>(v);
  int b = static_cast<int>(of);
  int64_t at = in;
  bool write = i < p.rows;
  if (p.offsets) {
    b = request_of(p.offsets, p.B, static_cast<int>(row), l, mask);
    const int first = __ldg(p.offsets + b);
    write = write && static_cast<int>(row) >= first && static_cast<int>(row) < __ldg(p.offsets + b + 1);  // of some request
    at = static_cast<int64_t>(row) - first;
  }
  const int cached = __ldg(p.lengths + b);
  write = write && cached >= 0;  // not an idle slot
  const int64_t pos = cached + at;
  if (write && pos >= p.cache_len) {
    if (l == 0) atomicOr(err, static_cast<unsigned>(kErrRange));
    write = false;
  }
  if (!write) return;  // (all 16 lanes of the row)
  const int t = static_cast<int>(pos) & (kQ4Tokens - 1);
  const int64_t block = (pos >> 4) * q4_block_bytes(GROUP);
  const uint32_t code_at = q4_word(t, l & 3, l >> 2);
  const uint32_t pair_at = kQ4Codes + (t * (128 / GROUP) + l / (GROUP / 8)) * 4;
  uint8_t* kd = p.k_cache + b * p.kc_b + h0 * p.kc_h + block;
  uint8_t* vd = p.v_cache + b * p.vc_b + h0 * p.vc_h + block;
  for (;;) {
    const uint4 yk = xk, yv = xv;
    if (--left > 0) {
      k += p.k_h, v += p.v_h;
      xk = *reinterpret_cast<const uint4*>(k), xv = *reinterpret_cast<const uint4*>(v);
    }
    uint32_t kw, kp, vw, vp;
    quantise<GROUP>(yk, mask, &kw, &kp);
    quantise<GROUP>(yv, mask, &vw, &vp);
    *reinterpret_cast<uint32_t*>(kd + code_at) = kw;
    *reinterpret_cast<uint32_t*>(vd + code_at) = vw;
    if (l % (GROUP / 8) == 0) {
      *reinterpret_cast<uint32_t*>(kd + pair_at) = kp;
      *reinterpret_cast<uint32_t*>(vd + pair_at) = vp;
    }
    if (left <= 0) break;
    kd += p.kc_h, vd += p.vc_h;
  }
}

// A warp reads a block; 16 lanes write a token's row of values, 16 bytes each.
template <int GROUP>
__global__ void __launch_bounds__(kThreads) q4_read_kernel(const uint8_t* __restrict__ cache, int64_t c_b,
                                                           int64_t c_h, __nv_bfloat16* __restrict__ out,
                                                           int64_t all, int64_t blocks, int KH) {
  pdl_trigger();
  pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (i >= all) return;
  const int64_t bh = i / blocks, block = i - bh * blocks;
  const int64_t b = bh / KH;
  const int h = static_cast<int>(bh - b * KH);
  const int l = threadIdx.x & 15, half = (threadIdx.x >> 4) & 1;
  const uint8_t* src = cache + b * c_b + h * c_h + block * q4_block_bytes(GROUP);
  uint32_t w[8], pair[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int t = 2 * k + half;
    w[k] = __ldg(reinterpret_cast<const uint32_t*>(src + q4_word(t, l & 3, l >> 2)));
    pair[k] = __ldg(reinterpret_cast<const uint32_t*>(src + kQ4Codes + (t * (128 / GROUP) + l / (GROUP / 8)) * 4));
  }
  __nv_bfloat16* dst = out + ((b * blocks + block) * kQ4Tokens * KH + h) * 128 + 8 * l;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float step = __uint_as_float(pair[k] << 16), low = __uint_as_float(pair[k] & 0xffff0000u);
    // nibbles j and j + 4 as fp16 1024 + code (j even), 1024 + 16 code (odd), exactly
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u = (((j < 2 ? w[k] : w[k] >> 8) & (j % 2 == 0 ? 0x000f000fu : 0x00f000f0u)) | 0x64006400u);
      const __half2 h = *reinterpret_cast<const __half2*>(&u);
      const float2 c = __half22float2(j % 2 == 0 ? __hadd2(h, __float2half2_rn(-1024.f))
                                                 : __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-64.f)));
      f[j] = fmaf(c.x, step, low);  // code * step is exact in fp32
      f[j + 4] = fmaf(c.y, step, low);
    }
    *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(2 * k + half) * KH * 128) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
}

template <int GROUP>
kda_status launch_append(AppendParams p, cudaStream_t st) {
  const unsigned groups = (p.rows + kItems - 1) / kItems;
  // heads are split over as many CTAs as the GPU has room for (8 an SM): 4,096 tokens of 8 heads 6.6 us,
  // 7.9 with a head to each CTA; 18,700 20.4 and 30.7
  const int64_t splits = static_cast<int64_t>(num_sms()) * 8 / groups;
  const int n = static_cast<int>(splits < 1 ? 1 : splits < p.KH ? splits : p.KH);
  p.heads = (p.KH + n - 1) / n;
  return launch_after("kv_append_q4", q4_append_kernel<GROUP>, dim3(groups, (p.KH + p.heads - 1) / p.heads), kThreads,
                      0, st, p, kda_err_ptr_q4_cache());
}

}  // namespace
}  // namespace kda

using namespace kda;

extern "C" size_t kda_q4_block_bytes(int64_t group) {
  return group == 32 || group == 64 || group == 128 ? q4_block_bytes(static_cast<int>(group)) : 0;
}

extern "C" kda_status kda_kv_append_q4(const void* k, const void* v, const int* offsets, const int* lengths,
                                       void* k_cache, void* v_cache, int64_t tokens, int64_t B, int64_t blocks,
                                       int64_t KH, int64_t D, int64_t group, const int64_t* k_strides,
                                       const int64_t* v_strides, const int64_t* k_cache_strides,
                                       const int64_t* v_cache_strides, void* stream) {
  const char* op = "kv_append_q4";
  KDA_CHECK_ARG(tokens > 0 && B > 0 && blocks > 0 && KH > 0 && (offsets || tokens % B == 0),
                "%s: bad sizes tokens=%lld B=%lld blocks=%lld KH=%lld", op, (long long)tokens, (long long)B,
                (long long)blocks, (long long)KH);
  KDA_CHECK_SUPPORTED(D == 128, "%s: head_dim must be 128, got %lld", op, (long long)D);
  KDA_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: group must be 32, 64 or 128, got %lld", op,
                (long long)group);
  KDA_CHECK_SUPPORTED(B < (1ll << 24) && KH <= 65535 && blocks < (1ll << 26) && tokens < (1ll << 31) &&
                          tokens * KH < (1ll << 31),
                      "%s: too large (tokens=%lld B=%lld blocks=%lld KH=%lld)", op, (long long)tokens, (long long)B,
                      (long long)blocks, (long long)KH);
  KDA_CHECK_ARG(k && v && lengths && k_cache && v_cache && k_strides && v_strides && k_cache_strides &&
                    v_cache_strides,
                "%s: null pointer", op);
  const int64_t n0 = offsets ? 1 : B, n1 = offsets ? tokens : tokens / B;
  auto rows_ok = [&](const void* p, const int64_t* s) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (n0 == 1 || (s[0] > 0 && s[0] % 8 == 0)) &&
           (n1 == 1 || (s[1] > 0 && s[1] % 8 == 0)) && (KH == 1 || (s[2] > 0 && s[2] % 8 == 0));
  };
  KDA_CHECK_SUPPORTED(rows_ok(k, k_strides) && rows_ok(v, v_strides) &&
                          q4_cache_ok(k_cache, k_cache_strides, B, KH) && q4_cache_ok(v_cache, v_cache_strides, B, KH),
                      "%s: pointers and rows must be 16-byte aligned", op);
  AppendParams p{};
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.offsets = offsets;
  p.lengths = lengths;
  p.rows = static_cast<unsigned>(tokens);
  p.per = static_cast<unsigned>(n1);
  p.k_b = n0 > 1 ? k_strides[0] : 0, p.k_t = n1 > 1 ? k_strides[1] : 0, p.k_h = KH > 1 ? k_strides[2] : 0;
  p.v_b = n0 > 1 ? v_strides[0] : 0, p.v_t = n1 > 1 ? v_strides[1] : 0, p.v_h = KH > 1 ? v_strides[2] : 0;
  p.kc_b = B > 1 ? k_cache_strides[0] : 0, p.kc_h = KH > 1 ? k_cache_strides[1] : 0;
  p.vc_b = B > 1 ? v_cache_strides[0] : 0, p.vc_h = KH > 1 ? v_cache_strides[1] : 0;
  p.cache_len = blocks * kQ4Tokens;
  p.B = static_cast<int>(B);
  p.KH = static_cast<int>(KH);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return group == 32 ? launch_append<32>(p, st) : group == 64 ? launch_append<64>(p, st) : launch_append<128>(p, st);
}

extern "C" kda_status kda_kv_read_q4(const void* cache, void* out, int64_t B, int64_t blocks, int64_t KH, int64_t D,
                                     int64_t group, const int64_t* cache_strides, void* stream) {
  const char* op = "kv_read_q4";
  KDA_CHECK_ARG(B > 0 && blocks > 0 && KH > 0, "%s: bad sizes B=%lld blocks=%lld KH=%lld", op, (long long)B,
                (long long)blocks, (long long)KH);
  KDA_CHECK_SUPPORTED(D == 128, "%s: head_dim must be 128, got %lld", op, (long long)D);
  KDA_CHECK_ARG(group == 32 || group == 64 || group == 128, "%s: group must be 32, 64 or 128, got %lld", op,
                (long long)group);
  KDA_CHECK_SUPPORTED(B < (1ll << 24) && KH <= 65535 && blocks < (1ll << 26) && B * KH < (1ll << 33) / blocks,
                      "%s: too large (B=%lld blocks=%lld KH=%lld)", op, (long long)B, (long long)blocks, (long long)KH);
  KDA_CHECK_ARG(cache && out && cache_strides, "%s: null pointer", op);
  KDA_CHECK_SUPPORTED(q4_cache_ok(cache, cache_strides, B, KH) && (reinterpret_cast<uintptr_t>(out) & 15u) == 0,
                      "%s: pointers and blocks must be 16-byte aligned", op);
  const int64_t all = B * KH * blocks;
  const dim3 grid(static_cast<unsigned>((all + kThreads / 32 - 1) / (kThreads / 32)));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t* c = static_cast<const uint8_t*>(cache);
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
  const int64_t cb = B > 1 ? cache_strides[0] : 0, ch = KH > 1 ? cache_strides[1] : 0;
  const int kh = static_cast<int>(KH);
  if (group == 32) return launch_after(op, q4_read_kernel<32>, grid, kThreads, 0, st, c, cb, ch, o, all, blocks, kh);
  if (group == 64) return launch_after(op, q4_read_kernel<64>, grid, kThreads, 0, st, c, cb, ch, o, all, blocks, kh);
  return launch_after(op, q4_read_kernel<128>, grid, kThreads, 0, st, c, cb, ch, o, all, blocks, kh);
}
