// Shared by the sliding-window attention kernels (window_fwd.cu, window_bwd.cu,
// window_decode.cu): tiles, tensor-core products of whole tiles, barriers of row
// warps, and the entry points' checks.
#pragma once

#include "common.cuh"

namespace kda {

constexpr int kD = 128;                    // head dim
constexpr int kBlk = 128;                  // rows of a block of queries or keys
constexpr uint32_t kTile = kBlk * kD * 2;  // 32 KB: two halves of 64 columns, 128-byte rows, 128-byte swizzle
constexpr uint32_t kHalf = kTile / 2;

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// The same, returning the AND of every thread's `ok`.  Named barriers have no
// time limit, so a warp whose bounded wait expired still joins the next one of
// its group, with false, and all of them stop there together.
__device__ __forceinline__ bool bar_and(int id, int threads, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.and.pred p, %2, %3, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(ok ? 1u : 0u), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
// The OR of every thread's predicate.
__device__ __forceinline__ bool bar_or(int id, int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, %3, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(v ? 1u : 0u), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
// For warps that run as one and issue from one elected lane (uniform control flow
// keeps descriptors in uniform registers: a product issues in fewer cycles).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// Their waits, every lane's: one lane's alone would diverge, which costs far more
// (20 % of the backward).  warp_wait2: both barriers are asked before either answer
// is needed.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}
__device__ __forceinline__ bool warp_wait2(uint64_t* b1, uint32_t p1, uint64_t* b2, uint32_t p2, unsigned* err,
                                           unsigned code) {
  const bool a = mbar_try_wait(b1, p1), b = mbar_try_wait(b2, p2);
  if (__all_sync(0xffffffffu, a && b)) return true;
  return __all_sync(0xffffffffu, mbar_wait(b1, p1, err, code) && mbar_wait(b2, p2, err, code));
}
// Whether a phase is complete, without waiting: asked early, so that the answer's
// latency (200 cycles and more beside the tensor core's operand reads) is hidden.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return r != 0;
}
// Every committed bulk store of this thread has read its shared memory.
__device__ __forceinline__ void bulk_wait_read_all() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, const void* src, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns, as the x32 forms in common.cuh.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Bits [a, b) of a 32-bit word (empty when a >= b); a, b may lie outside [0, 32].
__device__ __forceinline__ uint32_t range_mask(int a, int b) {
  a = a < 0 ? 0 : a;
  b = b > 32 ? 32 : b;
  if (a >= b) return 0u;
  const uint32_t hi = b >= 32 ? 0xffffffffu : ((1u << b) - 1u);
  return hi & ~((1u << a) - 1u);
}

// Bounded wait at the end, also after an error elsewhere: what is in flight
// must land before shared memory and TMEM go.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > kWaitLimitNs) return;
}

constexpr uint32_t kIdKK = idesc_bf16_f32(kBlk, kBlk, 0, 0);  // K-major A, K-major B
constexpr uint32_t kIdKM = idesc_bf16_f32(kBlk, kBlk, 0, 1);  // K-major A, MN-major B
// Descriptors of a tile read K-major (rows = M or N, 64-element halves along K:
// K step kk at (kk / 4) halves + (kk % 4) x 32 bytes) and MN-major (rows = K: K
// step kk at kk x 16 rows x 128 bytes, the two 64-element MN atoms 16 KB apart).
__device__ __forceinline__ uint64_t kmajor(uint32_t tile) { return smem_desc_sw128(tile, 16, 1024); }
__device__ __forceinline__ uint64_t mnmajor(uint32_t tile) { return smem_desc_sw128(tile, kHalf, 1024); }
__device__ __forceinline__ uint64_t kmajor_step(int kk) {
  return static_cast<uint64_t>(((kk >> 2) * kHalf + (kk & 3) * 32) >> 4);
}
__device__ __forceinline__ uint64_t mnmajor_step(int kk) { return static_cast<uint64_t>(kk * 128); }
// D (+)= A B with A in TMEM: lane = row of A, 32-bit column = two of its columns
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D = A B^T with both read K-major: 128 x (16 n16) x 128, from the first 16 n16 rows of B
__device__ __forceinline__ void mma_kk(uint32_t d, uint32_t a, uint32_t b, int n16 = 8) {
  const uint64_t da = kmajor(a), db = kmajor(b);
  const uint32_t id = kIdKK - (static_cast<uint32_t>(8 - n16) << 18);  // bits 17 to 22: N / 8
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) umma_bf16(d, da + kmajor_step(kk), db + kmajor_step(kk), id, kk != 0 ? 1u : 0u);
}
// D (+)= A B with A (bf16 pairs, 64 columns) in TMEM and B MN-major
__device__ __forceinline__ void mma_tm(uint32_t d, uint32_t a, uint32_t b, bool first) {
  const uint64_t db = mnmajor(b);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) umma_bf16_ts(d, a + 8 * kk, db + mnmajor_step(kk), kIdKM, (!first || kk != 0) ? 1u : 0u);
}
// with A's K steps in pairs 32 columns apart, [0, 16), [32, 48), ... of 128; the first k16
// of them
__device__ __forceinline__ void mma_tm_pairs(uint32_t d, uint32_t a, uint32_t b, bool first, int k16 = 8) {
  const uint64_t db = mnmajor(b);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    if (kk < k16)
      umma_bf16_ts(d, a + 32 * (kk >> 1) + 8 * (kk & 1), db + mnmajor_step(kk), kIdKM, (!first || kk != 0) ? 1u : 0u);
}
// The shares of a walk that is cut between CTAs: the first in slot 2 c + 1 of the CTA c
// that began it, the others in slots 2 (c + 1), 2 (c + 2), ...  The slot after `slot`,
// or -1 where the walk has all its steps (`steps` so far; advanced) or its records end:
// a launch whose wait expired leaves some of them empty.
__host__ __device__ __forceinline__ int next_share(const int4* pieces, int slots, int slot, int walk, int* steps) {
  if (*steps >= walk) return -1;
  const int next = (slot | 1) + 1;
  if (next >= slots) return -1;
  const int n = pieces[next].z;
  if (n <= 0) return -1;
  *steps += n < walk - *steps ? n : walk - *steps;
  return next;
}
// 128 rows x 128 columns as two halves
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int head, int row, int b) {
  tma_load_4d(dst, m, bar, 0, head, row, b);
  tma_load_4d(dst + kHalf, m, bar, 64, head, row, b);
}

// The entry points' size checks; whether the strided rows of [n0][n1][n2] start on 16
// bytes; the TMA map of [B][S][H][128] rows with element strides of batch, token and
// head (128-row boxes of 64 columns; rows past S read as zeros).  In both an axis of one
// entry may have any stride.
kda_status gqa_window_check(const char* op, int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, int64_t window,
                            int64_t sinks);
bool head_rows_ok(const void* p, const int64_t* strides, int64_t n0, int64_t n1, int64_t n2);
kda_status tmap_head_rows(CUtensorMap* m, const void* base, int64_t B, int64_t S, int64_t H, const int64_t* strides);

}  // namespace kda
