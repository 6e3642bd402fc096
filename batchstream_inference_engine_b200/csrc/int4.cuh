// The 4-bit cache: its rows, and what turns their codes into bf16.
//
// A group is 32 consecutive dims of one token and kv head, with one scale s: a bf16 number
// of at most 4 significant bits and either sign.  Its codes n = 0 .. 15 stand for
// s (n - 8): 4 bits times 4 bits, so every value is exactly a bf16 number, and attention
// over the cache is attention over the bf16 cache that holds these numbers.
//
// The append takes s = -x / 8 for the element x of the largest magnitude (of two of either
// sign the negative one), the magnitude rounded up to 4 bits, and n = rint(x / s) + 8, at
// most 15.  So values are off by |s| / 2 at most, and by |s| where an element on the other
// side is beyond 7.5 |s|: one of the 16 codes is lost to no side, and the step is an
// eighth of the largest element instead of a seventh.
//
// Pools are [.., num_blocks, bs, 9 D / 16] bytes: a block of bs tokens is its codes, D / 2
// bytes a token, then its scales, D / 32 bf16 a token.  The codes of 8 dims are a 32-bit
// word (little-endian), dim 2i in nibble i and dim 2i + 1 in nibble i + 4: one shift and one
// mask leave neighbours in the halves of a register.
#pragma once

#include "common.cuh"

namespace bsb {

constexpr int kInt4Group = 32;

// Bytes of a token's codes, of its scales, and of both.
__host__ __device__ constexpr int int4_code_bytes(int D) { return D / 2; }
__host__ __device__ constexpr int int4_scale_bytes(int D) { return D / 16; }
__host__ __device__ constexpr int int4_row_bytes(int D) { return D / 2 + D / 16; }

// Values of a word: bf16 pairs (2i, 2i + 1) in v[i].  `scale`: s in both halves, `shift`:
// -136 s.  A code in the mantissa's low bits below the exponent of 128 is 128 + n, and
// (128 + n) s - 136 s has one rounding, of a bf16 number.  136 s is one too: 17 times 4 bits
// are 8 bits.
__device__ __forceinline__ uint32_t int4_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t int4_shift(uint32_t scale) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(scale), "r"(0xc308c308u));  // -136
  return d;
}
__device__ __forceinline__ uint32_t int4_raw(uint32_t w, int i) {  // 128 + n of dims 2i, 2i + 1
  uint32_t d;  // (one instruction; with two immediates the compiler makes it two)
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(w >> (4 * i)), "r"(0x000f000fu), "r"(0x43004300u));
  return d;
}
__device__ __forceinline__ void int4_values(uint32_t w, uint32_t scale, uint32_t shift,
                                            uint32_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = int4_fma(int4_raw(w, i), scale, shift);
}

// Values of a word in fp32, dims in order.
__device__ __forceinline__ void int4_floats(uint32_t w, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = scale * (static_cast<float>((w >> (4 * i)) & 15u) - 8.f);
    v[2 * i + 1] = scale * (static_cast<float>((w >> (4 * i + 16)) & 15u) - 8.f);
  }
}

__device__ __forceinline__ float int4_scale_float(uint16_t bits) {
  return __uint_as_float(static_cast<uint32_t>(bits) << 16);
}

}  // namespace bsb
