// Layout of the 4-bit paged K/V cache and the conversions its kernels share.
//
// A page holds 64 positions of one K/V head in 72 D contiguous bytes (D = 64, 128 or 256
// values per row), keys first, so that either half is one copy:
//   [ 0 D, 32 D)  key codes     [slab][64 tokens][piece t < 4][SD / 8 bytes]
//   [32 D, 36 D)  key scales    [64 tokens][D / 16]           e4m3
//   [36 D, 68 D)  value codes   [slab][32 token pairs][g < 8][token of the pair][SD / 16 bytes]
//   [68 D, 72 D)  value scales  [32 token pairs][D / 16][token of the pair]   e4m3
// A slab is SD = min(D, 128) values.  The orders are those in which a warp's m16n8k16
// fragments want them, so one wide shared-memory load per token gives a lane all that it
// needs of a row and no two lanes meet in a bank:
//   key byte (t, 4 w + i)  = value 32 w + 4 t + i (low half), value 32 w + 16 + 4 t + i (high half):
//       the two halves of a converted f16x2 carry two scales that are neighbours in memory;
//   value byte (g, block b) = value 16 b + g (low half), value 16 b + 8 + g (high half):
//       a row's bytes are its own (two tokens never share a byte, so rows can be written in
//       any order); a lane joins the two tokens of a pair with two ALU operations per word.
// An element is e2m1 * scale * 2^exp (exp per cache, for K and V).  e2m1 times e4m3 has at
// most six significant bits, at most 2688 and is a multiple of 2^-10: exact in f16.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace moet {
namespace kv4 {

constexpr int kPage = 64;   // positions per page

template <int D> struct Lay {
  static constexpr int SD = D < 128 ? D : 128;       // values per slab
  static constexpr int NS = D / SD;                  // slabs
  static constexpr int NB = D / 16;                  // scale blocks per row
  static constexpr int KC = 0, KS = 32 * D, VC = 36 * D, VS = 68 * D;
  static constexpr int kHalfBytes = 36 * D, kPageBytes = 72 * D;
  static constexpr int kSlabBytes = kPage * SD / 2;  // codes of a slab
};

// four bytes of two e2m1 codes each -> four f16x2 (low code in the low half)
MOET_DEVICE void e2m1x8_to_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}
// four e4m3 bytes -> two f16x2
MOET_DEVICE void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 h0, h1;\nmov.b32 {h0, h1}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, h0;\ncvt.rn.f16x2.e4m3x2 %1, h1;\n}\n"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
// products of f16 pairs keep their subnormals (no .ftz)
MOET_DEVICE uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The two tokens of a pair (words a, b of four blocks' bytes) -> codes of values g and g + 8.
MOET_DEVICE void join_pair(uint32_t a, uint32_t b, uint32_t& g0, uint32_t& g8) {
  g0 = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u);
  g8 = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
}

template <typename T16> MOET_DEVICE float to_f32(T16 x);
template <> MOET_DEVICE float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> MOET_DEVICE float to_f32(__half x) { return __half2float(x); }

MOET_DEVICE float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// Smallest e >= -100 with amax <= 127 * 2^e; 0 for amax = 0 (finite amax >= 0).
MOET_DEVICE int exp_for_127(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (!(amax > 0.f)) return 0;
  // amax = 1.m * 2^x = (1.m / 2) 2^(x+1): 127 * 2^(x-6) holds it iff 1.m <= 127 / 64
  const int x = (int)(u >> 23) - 127;
  return max(-100, x - 6 + ((u & 0x7FFFFFu) > 0x7E0000u ? 1 : 0));
}

}  // namespace kv4
}  // namespace moet
