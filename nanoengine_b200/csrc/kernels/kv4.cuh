// Rows of a key / value cache held in 4 bits.  A page holds, for every kv head, the codes of its tokens (D / 2 bytes each), then their scales (a byte per
// group of 32 neighbouring dims).  Scale byte b = 8 e + m stands for (8 + m) 2^(e - 19), code c for (c - 8) scale; a word of 8 dims keeps those of even
// place in its low half and the others in its high half, lowest first.
#pragma once
#include "ptx.cuh"

namespace ne {

// bf16 bits of a scale byte: (1 + m / 8) 2^(e - 16), no zero and no infinity among them
__device__ __forceinline__ uint32_t kv4_scale_bits(uint32_t b) { return (b << 4) + 0x3780u; }

__device__ __forceinline__ uint32_t hmul2_bf16(uint32_t a, uint32_t b) {
  uint32_t d; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d;
}
__device__ __forceinline__ uint32_t hfma2_bf16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d; asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c)); return d;
}

// Nibbles i of both halves of a word as a pair of bf16 16 + c: the nibble becomes the upper four of bf16's seven mantissa bits under the exponent of 16.
template <int kNibble> __device__ __forceinline__ uint32_t kv4_pair_raw(uint32_t w) {
  constexpr int sh = 4 * kNibble - 3;
  const uint32_t x = sh < 0 ? w << (-sh & 31) : w >> (sh & 31);
  return (x & 0x00780078u) | 0x41804180u;
}
// (16 + c) s - 24 s = (c - 8) s.  Exact: 24 s has six significant bits, (c - 8) s seven, and the fused product rounds once.
template <int kNibble> __device__ __forceinline__ uint32_t kv4_pair(uint32_t w, uint32_t s2, uint32_t m24s2) {
  return hfma2_bf16(kv4_pair_raw<kNibble>(w), s2, m24s2);
}
__device__ __forceinline__ uint32_t kv4_minus24(uint32_t s2) { return hmul2_bf16(s2, 0xC1C0C1C0u); }

// The 8 dims of a word, in order, as four bf16 pairs.
__device__ __forceinline__ uint4 kv4_word(uint32_t w, uint32_t scale_byte) {
  const uint32_t s2 = kv4_scale_bits(scale_byte) * 0x00010001u, z = kv4_minus24(s2);
  return make_uint4(kv4_pair<0>(w, s2, z), kv4_pair<1>(w, s2, z), kv4_pair<2>(w, s2, z), kv4_pair<3>(w, s2, z));
}

}  // namespace ne
