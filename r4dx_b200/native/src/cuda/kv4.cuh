// The 4-bit paged KV cache: what its writer, its reader and the attentions over it share.
//
// A pool is uint8 [blocks][kv heads][2 (keys, values)][9 D], D = 64, 128 or 256, a block 16 tokens of a sequence.  Every 64 channels
// of a row are a group: codes n of 4 bits, a scale s and a low end lo (the group's minimum), both bf16; a value is n s + lo.  4.5 bits
// a value: 64 channels a group keep the pairs at an eighth of the codes, and each kernel's work per group small.
//   bytes 0 .. 8 D:    code words, eight consecutive channels of a token each, the first in the lowest bits; word w (channels
//                      8 w ..) of token t lies at Word
//   bytes 8 D .. 9 D:  [16 tokens][D / 64 groups] pairs (s in the lower half, lo in the upper)
// Keys and values of a head's block are one run of 18 D bytes: one copy brings both to shared memory.
//
// The order of the words is the one in which the decode kernel's lanes hold tensor-core fragments, with the swizzles that give each of
// its shared-memory loads all banks:
//   keys    lane (g, c) of a warp has tokens g and g + 8, of every 32 channels 8 c .. 8 c + 7: its words of a token lie side by side
//   values  lane (g, c) has tokens 2 c, 2 c + 1 (+ 8), of every 64 channels 8 g .. 8 g + 7
#pragma once
#include "common.cuh"

namespace r4dxb {
namespace kv4 {

constexpr int kBlock = 16;          // tokens
constexpr int kGroup = 64;          // channels that share a scale
constexpr float kLimit = 32768.f;   // values saturate here: what the codes stand for (n s + lo) then fits fp16

template <int D>
struct Shape {
  static_assert(D == 64 || D == 128 || D == 256, "head dimensions of the 4-bit cache");
  static constexpr int kGroups = D / kGroup;
  static constexpr int kWords = D / 8;               // code words of a token
  static constexpr int kCodeBytes = 8 * D;           // of a block's keys or values
  static constexpr int kPart = 9 * D;
  static constexpr int kRun = 18 * D;                // keys and values of a block
};

// Place (in 32-bit words) of word w of token t in its block.
template <int D, bool VALUES>
__host__ __device__ __forceinline__ int Word(int t, int w) {
  if constexpr (VALUES) {
    const int g = w & 7, j = w >> 3, p = t >> 1;
    if constexpr (D == 256) return t * 32 + (g ^ (t & 6)) * 4 + j;
    if constexpr (D == 128) return p * 32 + (g ^ (t & 6)) * 4 + (t & 1) * 2 + j;
    return p * 16 + (g ^ ((p & 2) << 1)) * 2 + (t & 1);
  } else {
    const int c = w & 3, j = w >> 2;
    if constexpr (D == 256) return t * 32 + ((j >> 2) ^ (t & 1)) * 16 + c * 4 + (j & 3);
    return t * (D / 8) + c * (D / 32) + j;
  }
}

// A sequence's block table: which block of the pool holds a token, -1 where none does (a position or a table entry out of range: such
// a row is not written, and attention over it or its read-back gives NaN).
struct Table {
  const int* entries;
  int length;           // of a table
  int pool;             // blocks
  __device__ __forceinline__ int BlockAt(int index) const {
    if (index < 0 || index >= length) return -1;
    const int b = __ldg(entries + index);
    return b >= 0 && b < pool ? b : -1;
  }
};

}  // namespace kv4
}  // namespace r4dxb
