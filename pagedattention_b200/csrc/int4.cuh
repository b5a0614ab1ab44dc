// The 4-bit page format and the register arithmetic on its codes.
//
// A row (one token of one kv head) is cut into groups of 64 elements; a group
// holds its minimum `lo` and a scale s = T((hi - lo) / 15), both of the rows'
// 16-bit type T, and a code c = rint((x - lo) / s) in 0..15 per element, which
// stands for lo + s c.  A page of block_size rows is
//
//   codes   block_size x D/2 bytes
//   pairs   block_size x D/64 (s, lo)
//
// that is block_size * D * 9/16 bytes, contiguous, a multiple of 16.
//
// Codes are stored as 32-bit words of 8 consecutive elements, element i in
// nibble i / 2 + 4 (i % 2): the low nibbles of the word's two 16-bit halves are
// elements 0 and 1, so that a mask gives two neighbouring elements in one pair
// of 16-bit lanes.  Where a word goes follows the fragments of the decode's
// matrix instructions, so that every lane reads its codes of 8 tokens with one
// contiguous, conflict-free load:
//   keys    row-major rows of D/2 bytes; within a row, chunk c of 4 holds the
//           words of elements 16 c .. 16 c + 15 of every group (D/64 x 2 words)
//   values  tiles of 8 tokens, 4 D bytes each: [octet o of 8][token pair of 4]
//           [token parity of 2][group] words of elements 8 o .. 8 o + 7
#pragma once

#include <cstdint>

#include "ptx.cuh"

namespace pab {

constexpr int kInt4Group = 64;

// Bytes of one row: its codes and its (scale, minimum) pairs.
__host__ __device__ constexpr int int4_row_bytes(int D) { return D / 2 + D / kInt4Group * 4; }

// Byte offset in a page of the code word of elements 64 g + 8 o .. + 7 (group
// g, octet o) of row r.
__host__ __device__ __forceinline__ int int4_key_word(int D, int r, int g, int o) {
  return r * (D / 2) + (o >> 1) * (D / 8) + g * 8 + (o & 1) * 4;
}
__host__ __device__ __forceinline__ int int4_value_word(int D, int r, int g, int o) {
  return (r >> 3) * (4 * D) + (((o * 4 + ((r & 7) >> 1)) * 2 + (r & 1)) * (D / kInt4Group) + g) * 4;
}
// Byte offset in a page of `bs` rows of group g's (scale, minimum) of row r.
__host__ __device__ __forceinline__ int int4_pair(int D, int bs, int r, int g) {
  return bs * (D / 2) + (r * (D / kInt4Group) + g) * 4;
}

// Two 16-bit values of one register.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// N consecutive 32-bit words of shared memory (aligned to min(N, 4) words).
template <int N>
__device__ __forceinline__ void ld_shared_words(uint32_t addr, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                   : "r"(addr + i * 4));
  }
}

// (x & mask) | bits, one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}

// Nibble m of both 16-bit halves of w as it stands: the pair r[m] is two fp16
// subnormals c * 2^-24 (m even) or c * 2^-20 (m odd), exact, for the price of a
// mask.  What they are multiplied with carries the powers of two.
__device__ __forceinline__ void int4_raw_pairs(uint32_t w, uint32_t (&r)[4]) {
  const uint32_t v = w >> 8;
  r[0] = w & 0x000f000fu;
  r[1] = w & 0x00f000f0u;
  r[2] = v & 0x000f000fu;
  r[3] = v & 0x00f000f0u;
}

// Nibble m of both 16-bit halves of w as the fp16 pair r[m], the odd nibbles with
// the even ones below them, which saves an instruction of five; sums of the two
// differ by what the odd one contributes.  Everything here is exact.
//   plain    even c 2^-24; odd c 2^-20 + c' 2^-24
//   CENTRED  even c - 8; odd (c - 8) + (c' - 8) / 16.  A byte OR-ed under the
//            exponent of 1024 reads as 1024 + c' + 16 c.
template <bool CENTRED>
__device__ __forceinline__ void int4_value_pairs(uint32_t w, uint32_t (&r)[4]) {
  if constexpr (!CENTRED) {
    r[0] = w & 0x000f000fu;
    r[1] = w & 0x00ff00ffu;
    r[3] = __byte_perm(w, 0u, 0x4341);
    r[2] = r[3] & 0x000f000fu;
    return;
  }
  const __half2 base = __float2half2_rn(1032.f);
  const __half2 sixteenth = __float2half2_rn(0.0625f), off = __float2half2_rn(-72.5f);
  uint32_t t[4];
  t[0] = and_or(w, 0x000f000fu, 0x64006400u);
  t[1] = and_or(w, 0x00ff00ffu, 0x64006400u);
  t[3] = __byte_perm(w, 0x64646464u, 0x4341);
  t[2] = t[3] & 0xff0fff0fu;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const __half2 x = *reinterpret_cast<const __half2*>(&t[m]);
    const __half2 y = m & 1 ? __hfma2(x, sixteenth, off) : __hsub2(x, base);
    r[m] = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// Maximum of two pairs of T.
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t max2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max2<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Nibble m of both halves of w as the pair r[m] of exact values c (0..15) of T.
template <typename T>
__device__ __forceinline__ void int4_codes(uint32_t w, uint32_t (&r)[4]);
template <>
__device__ __forceinline__ void int4_codes<__half>(uint32_t w, uint32_t (&r)[4]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const uint32_t t = and_or(w >> (4 * m), 0x000f000fu, 0x64006400u);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&t), __float2half2_rn(1024.f));
    r[m] = *reinterpret_cast<const uint32_t*>(&y);
  }
}
template <>
__device__ __forceinline__ void int4_codes<__nv_bfloat16>(uint32_t w, uint32_t (&r)[4]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const uint32_t t = and_or(w >> (4 * m), 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 y =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&t), __floats2bfloat162_rn(128.f, 128.f));
    r[m] = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// a * b + c of two pairs of T, one rounding.
template <typename T>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c);
template <>
__device__ __forceinline__ uint32_t fma2<__half>(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
template <>
__device__ __forceinline__ uint32_t fma2<__nv_bfloat16>(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// (scale, value of code 8) of a (scale, minimum) pair.
template <typename T>
__device__ __forceinline__ float2 int4_centre(uint32_t pair) {
  const float2 f = unpack2<T>(pair);
  return make_float2(f.x, fmaf(8.f, f.x, f.y));
}

}  // namespace pab
