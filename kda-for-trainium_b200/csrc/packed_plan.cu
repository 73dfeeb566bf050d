// The plan of a buffer of packed sequences: tables of their 128-row blocks, built on the
// device from the offsets, once for all the calls on that buffer (every layer's forward
// and backward).
//
// One CTA.  Bound by latency: a scan over the sequences, a binary search for each block's
// sequence and a counting sort by the block's place, 3.7 us for 24 sequences of 16,384
// tokens.  The tables hold the same values every time; only the order of blocks at the
// same place in `sorted` and `pairs` may differ, which moves work between CTAs and changes
// no result.
#include "launch.cuh"
#include "packed.cuh"

KDA_DEFINE_ERROR_WORD(packed_plan)

namespace kda {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = kThreads;  // places from here on share the first bin: they are sorted no further
constexpr unsigned kFull = 0xffffffffu;

// The sums over the threads before this one, and over all.
__device__ __forceinline__ int64_t scan_block(int64_t v, int64_t* warp_sums, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t sum = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(kFull, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int64_t w = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(kFull, w, d);
      if (lane >= d) w += o;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *total = warp_sums[31];
  const int64_t before = (warp > 0 ? warp_sums[warp - 1] : 0) + sum - v;
  __syncthreads();  // warp_sums may be used again
  return before;
}

// The bin of place z: the last places first.
__device__ __forceinline__ int bin_of(int z) { return kBins - 1 - min(z, kBins - 1); }

__global__ void __launch_bounds__(kThreads) packed_plan_kernel(const int* __restrict__ offsets, int sequences,
                                                               int tokens, uint8_t* plan, int64_t most,
                                                               unsigned* err) {
  __shared__ int bins[2][kBins];  // all blocks, those at even places
  __shared__ int64_t sums[32];
  pdl_trigger();
  pdl_wait();
  PlanHead* head = reinterpret_cast<PlanHead*>(plan);
  Block* natural = reinterpret_cast<Block*>(plan + 32);
  Block* sorted = natural + most;
  Block* pairs = sorted + most;
  int64_t* before = reinterpret_cast<int64_t*>(pairs + most);
  int64_t* seq_steps = before + most;
  int* seq_block = reinterpret_cast<int*>(seq_steps + sequences);

  bins[0][threadIdx.x] = bins[1][threadIdx.x] = 0;
  bool bad = false;
  int blocks = 0;
  int64_t steps = 0;
  for (int s0 = 0; s0 < sequences; s0 += kThreads) {
    const int s = s0 + threadIdx.x;
    int n = 0;
    if (s < sequences) {
      const int a = offsets[s], b = offsets[s + 1];
      if (a < 0 || b < a || b > tokens) bad = true;
      else n = (b - a + 127) >> 7;
    }
    if (__syncthreads_or(bad)) break;  // no table is read or written past its end
    // both sums in one scan: blocks (below 2^24 together) beneath steps (below 2^35)
    int64_t all;
    const int64_t at = scan_block((static_cast<int64_t>(n) * (n + 1) / 2) << 24 | n, sums, &all);
    if (s < sequences) {
      seq_block[s] = blocks + static_cast<int>(at & 0xffffff);
      seq_steps[s] = steps + (at >> 24);
    }
    blocks += static_cast<int>(all & 0xffffff);
    steps += all >> 24;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) {
      atomicOr(err, static_cast<unsigned>(kErrRange));
      *head = PlanHead{kPlanMagic, 0, 0, 0, 0, tokens, 0};
    }
    return;
  }
  // each block's sequence: the last one whose block 0 is not after it
  for (int e = threadIdx.x; e < blocks; e += kThreads) {
    int lo = 0, hi = sequences;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (seq_block[mid] <= e) lo = mid;
      else hi = mid;
    }
    const int start = offsets[lo], len = offsets[lo + 1] - start, base = seq_block[lo];
    const int64_t z = e - base, n = (len + 127) >> 7;
    natural[e] = make_int4(start, len, static_cast<int>(z), base);
    before[e] = seq_steps[lo] + z * n - z * (z - 1) / 2;
    atomicAdd(&bins[0][bin_of(static_cast<int>(z))], 1);
    if ((z & 1) == 0) atomicAdd(&bins[1][bin_of(static_cast<int>(z))], 1);
  }
  __syncthreads();
  // the bins' first places, of both in one scan
  int64_t all;
  const int64_t at = scan_block(static_cast<int64_t>(bins[1][threadIdx.x]) << 32 | bins[0][threadIdx.x], sums, &all);
  bins[0][threadIdx.x] = static_cast<int>(at & 0xffffffff);
  bins[1][threadIdx.x] = static_cast<int>(at >> 32);
  __syncthreads();
  for (int e = threadIdx.x; e < blocks; e += kThreads) {
    const Block b = natural[e];
    sorted[atomicAdd(&bins[0][bin_of(b.z)], 1)] = b;
    if ((b.z & 1) == 0) pairs[atomicAdd(&bins[1][bin_of(b.z)], 1)] = b;
  }
  if (threadIdx.x == 0)
    *head = PlanHead{kPlanMagic, blocks, static_cast<int>(all >> 32), offsets[0], offsets[sequences], tokens, steps};
}

}  // namespace

kda_status gqa_packed_check(const char* op, int64_t tokens, int64_t QH, int64_t KH, int64_t D, const void* plan,
                            size_t bytes, int64_t* sequences) {
  KDA_CHECK_ARG(tokens > 0 && QH > 0 && KH > 0 && QH % KH == 0, "%s: bad sizes tokens=%lld QH=%lld KH=%lld", op,
                (long long)tokens, (long long)QH, (long long)KH);
  KDA_CHECK_SUPPORTED(D == 128, "%s: head_dim must be 128, got %lld", op, (long long)D);
  KDA_CHECK_SUPPORTED(tokens < (1ll << 24) && QH <= 65535 && tokens < (1ll << 31) / QH,
                      "%s: too many rows (tokens=%lld QH=%lld)", op, (long long)tokens, (long long)QH);
  KDA_CHECK_ARG(plan, "%s: null pointer", op);
  KDA_CHECK_SUPPORTED((reinterpret_cast<uintptr_t>(plan) & 15u) == 0, "%s: the plan must be 16-byte aligned", op);
  const int64_t n = plan_sequences(tokens, bytes);
  KDA_CHECK_ARG(n > 0, "%s: a plan of %zu bytes is not one for %lld rows", op, bytes, (long long)tokens);
  *sequences = n;
  return KDA_OK;
}

}  // namespace kda

using namespace kda;

extern "C" size_t kda_packed_plan_size(int64_t tokens, int64_t sequences) {
  if (tokens <= 0 || sequences <= 0 || tokens >= (1ll << 24) || sequences >= (1ll << 24)) return 0;
  return static_cast<size_t>(plan_bytes(tokens, sequences));
}

extern "C" kda_status kda_packed_plan(const int* offsets, int64_t sequences, int64_t tokens, void* plan,
                                      size_t plan_bytes_, void* stream) {
  const char* op = "packed_plan";
  KDA_CHECK_ARG(tokens > 0 && sequences > 0, "%s: bad sizes tokens=%lld sequences=%lld", op, (long long)tokens,
                (long long)sequences);
  KDA_CHECK_SUPPORTED(tokens < (1ll << 24) && sequences < (1ll << 24), "%s: too large (tokens=%lld sequences=%lld)",
                      op, (long long)tokens, (long long)sequences);
  KDA_CHECK_ARG(offsets && plan, "%s: null pointer", op);
  KDA_CHECK_ARG(plan_bytes_ == static_cast<size_t>(plan_bytes(tokens, sequences)),
                "%s: a plan of %lld bytes required, got %zu", op, (long long)plan_bytes(tokens, sequences), plan_bytes_);
  KDA_CHECK_SUPPORTED((reinterpret_cast<uintptr_t>(plan) & 15u) == 0, "%s: the plan must be 16-byte aligned", op);
  return launch_after(op, packed_plan_kernel, dim3(1), kThreads, 0, static_cast<cudaStream_t>(stream), offsets,
                      static_cast<int>(sequences), static_cast<int>(tokens), static_cast<uint8_t*>(plan),
                      plan_blocks(tokens, sequences), kda_err_ptr_packed_plan());
}
