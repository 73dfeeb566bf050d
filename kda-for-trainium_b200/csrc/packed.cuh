// Shared by the kernels of attention over packed sequences (packed_plan.cu,
// packed_fwd.cu, packed_bwd.cu): the plan's layout.
//
// Sequence s is the rows [offsets[s], offsets[s + 1]) of one buffer of tokens.  Work is
// cut into blocks of 128 rows that start where their sequence starts, so a tile holds
// one sequence's rows, then (in a sequence's last block) rows that belong to others.
#pragma once

#include "common.cuh"

namespace kda {

struct PlanHead {
  int magic;
  int blocks;        // of all sequences
  int pairs;         // of those, the ones at an even place in their sequence
  int first, last;   // the rows that belong to sequences
  int tokens;        // rows of the buffer
  int64_t steps;     // (query block, key block) pairs of one head with a visible pair
};
constexpr int kPlanMagic = 0x6b647031;

// A block: its sequence's first row and length, its place in the sequence, and the
// place of the sequence's block 0 among all blocks in the order of the buffer.
//   x start, y length, z place, w block 0
using Block = int4;

// A plan in memory: the head, then `most` of each.
struct PlanView {
  const PlanHead* head;
  const Block* natural;     // in the order of the buffer
  const Block* sorted;      // those with the most keys before them first
  const Block* pairs;       // the sorted ones at even places
  const int64_t* before;    // natural order: steps of the key blocks before this one, a key
                            // block's steps being the query blocks from its own to the sequence's last
};
inline __host__ __device__ int64_t plan_blocks(int64_t tokens, int64_t sequences) { return tokens / 128 + sequences; }
// head | natural | sorted | pairs | before | per sequence: steps before it (8 bytes), block 0 (4, even count)
inline __host__ __device__ int64_t plan_bytes(int64_t tokens, int64_t sequences) {
  return 32 + 56 * plan_blocks(tokens, sequences) + 8 * sequences + 4 * (sequences + (sequences & 1));
}
// The sequences that a plan of so many bytes was made for; 0: none.  (Two sequences more
// are 136 bytes more.)
inline int64_t plan_sequences(int64_t tokens, size_t bytes) {
  const int64_t have = bytes < (size_t(1) << 40) ? static_cast<int64_t>(bytes) : 0, none = plan_bytes(tokens, 0);
  if (have <= none) return 0;
  int64_t n = (have - none) / 136 * 2;
  if (plan_bytes(tokens, n) != have) ++n;
  return plan_bytes(tokens, n) == have ? n : 0;
}
inline __host__ __device__ PlanView plan_view(const void* plan, int64_t most) {
  const uint8_t* p = static_cast<const uint8_t*>(plan);
  PlanView v;
  v.head = reinterpret_cast<const PlanHead*>(p);
  v.natural = reinterpret_cast<const Block*>(p + 32);
  v.sorted = v.natural + most;
  v.pairs = v.sorted + most;
  v.before = reinterpret_cast<const int64_t*>(v.pairs + most);
  return v;
}

// Whether the plan was made for a buffer of this many rows; if not, nothing is done and
// (plan_ok) the error word says so.
__device__ __forceinline__ bool plan_matches(const PlanView& v, int tokens) {
  return v.head->magic == kPlanMagic && v.head->tokens == tokens;
}
__device__ __forceinline__ bool plan_ok(const PlanView& v, int tokens, unsigned* err) {
  const bool ok = plan_matches(v, tokens);
  if (!ok && threadIdx.x == 0) atomicOr(err, static_cast<unsigned>(kErrRange));
  return ok;
}

// A CTA's kth unit of a table sorted by length: the rounds go through the CTAs in alternating
// directions, so that none has the longest of every round (S8192 of 32 heads, where a round
// spans nine lengths: the CTAs work 590,000 to 782,000 cycles without, 670,000 to 713,000 with).
__device__ __forceinline__ int unit_of_round(int k) {
  const int g = static_cast<int>(gridDim.x), b = static_cast<int>(blockIdx.x);
  return k * g + ((k & 1) != 0 ? g - 1 - b : b);
}

// Zeros in the rows of [tokens][row_bytes] that belong to no sequence, by `count`
// threads of which this one is the `at`th.
__device__ __forceinline__ void zero_rest(void* base, int first, int last, int tokens, int64_t row_bytes, int64_t at,
                                          int64_t count) {
  uint4* p = static_cast<uint4*>(base);
  const int64_t per = row_bytes / 16, head = first * per, tail = (tokens - last) * per;
  for (int64_t i = at; i < head; i += count) p[i] = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t i = at; i < tail; i += count) p[last * per + i] = make_uint4(0u, 0u, 0u, 0u);
}

// The entry points' size checks; *sequences: what a plan of `bytes` for `tokens` rows
// was made for.
kda_status gqa_packed_check(const char* op, int64_t tokens, int64_t QH, int64_t KH, int64_t D, const void* plan,
                            size_t bytes, int64_t* sequences);

}  // namespace kda
