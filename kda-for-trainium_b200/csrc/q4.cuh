// The 4-bit key/value cache: its layout, shared by the kernels that write it (q4_cache.cu)
// and attend to it (q4_decode.cu).
//
// A cache is [B][KH][blocks] blocks of 16 tokens of one head.  A value is
//   code * step + low,   code 0 .. 15, step and low bf16, one pair for each group of
// 32, 64 or 128 channels of a token.  A block is 16 rows of 64 bytes of codes, then
// [16 tokens][128 / group] pairs (step, low).
//
// A row's 16-byte chunk c holds, for g = 0 .. 3, the word of channels 32 g + 8 c .. + 7, the
// first in the low nibble: a lane of the matrix instruction then finds its operand columns of
// all four 32-channel runs in one chunk, and every k16 step lies in one run, so steps of any
// group size are applied to whole sums instead of every code.  Chunk c of token t lies at
// place c ^ ((t >> 1) & 3): lanes that read one chunk of tokens 0, 2, 4 and 6 then meet
// different banks of shared memory.
#pragma once

#include "common.cuh"

namespace kda {

constexpr int kQ4Tokens = 16;                    // of a block
constexpr uint32_t kQ4Codes = kQ4Tokens * 64;    // bytes of codes

inline __host__ __device__ constexpr uint32_t q4_block_bytes(int group) { return kQ4Codes + kQ4Tokens * (128 / group) * 4; }
// Byte of the 32-bit word of run g, chunk c of token t in its block.
__device__ __forceinline__ uint32_t q4_word(int t, int c, int g) {
  return static_cast<uint32_t>(t * 64 + ((c ^ ((t >> 1) & 3)) << 4) + g * 4);
}

// Whether a cache's blocks start on 16 bytes ([B][KH], strides in bytes; an axis of one
// entry may have any stride).
inline bool q4_cache_ok(const void* p, const int64_t* strides, int64_t B, int64_t KH) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (B == 1 || (strides[0] > 0 && strides[0] % 16 == 0)) &&
         (KH == 1 || (strides[1] > 0 && strides[1] % 16 == 0));
}

}  // namespace kda
