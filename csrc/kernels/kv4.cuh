// Layout of the 4-bit paged K/V cache and the conversions its kernels share.
//
// A page holds 64 positions of one K/V head in 72 D contiguous bytes (D = 64, 128 or 256
// values per row), keys first, so that either half is one copy:
//   [ 0 D, 32 D)  key codes     [slab][64 tokens][piece t < 4][SD / 8 bytes]
//   [32 D, 36 D)  key scales    [64 tokens][D / 16]           e4m3
//   [36 D, 68 D)  value codes   [slab][32 token pairs][piece g < 8][token of the pair][SD / 16 bytes]
//   [68 D, 72 D)  value scales  [32 token pairs][D / 16][token of the pair]   e4m3
// A slab is SD = min(D, 128) values.  A piece is what one lane of a warp needs of a row in the
// m16n8k16 fragments (the order of the values within a product's depth, or of its rows, is
// free), chosen so that it takes few scales:
//   key piece t:   SD = 128: byte i = value 32 t + i (low half), 32 t + 16 + i (high half): two
//                  blocks, whose scales are the two halves of one f16x2;
//                  SD = 64:  byte i = value 16 t + i, 16 t + 8 + i: one block;
//   value piece g: byte i = value E g + i, E g + E / 2 + i, E = SD / 8 (one block, or half of
//                  one); a row's bytes are its own (two tokens never share a byte, so rows can be
//                  written in any order), and a lane joins the two tokens of a pair with two ALU
//                  operations per word; their scales are one f16x2.
// An element is e2m1 * scale * 2^exp (exp per cache, for K and V).  e2m1 times e4m3 has at
// most six significant bits, at most 2688 and is a multiple of 2^-10: exact in f16.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

#include <cmath>

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

// SMs of the current device: grids, plans and the rules that choose between forms go by it
inline int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// four bytes of two e2m1 codes each -> four f16x2 (low code in the low half)
MOET_DEVICE void e2m1x8_to_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}
// two e4m3 bytes (the low half of w) -> f16x2
MOET_DEVICE uint32_t e4m3x2_to_f16(uint16_t w) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(w));
  return d;
}
// 2 or 4 words, from 8- or 16-byte aligned memory
template <int W> MOET_DEVICE void load_words(const uint8_t* p, uint32_t (&c)[W]) {
  if constexpr (W == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    c[0] = v.x, c[1] = v.y, c[2] = v.z, c[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    c[0] = v.x, c[1] = v.y;
  }
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

MOET_DEVICE uint32_t pack_f16x2(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
MOET_DEVICE float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two 16-bit values as floats, and back
template <typename T16> MOET_DEVICE float2 unpack2(uint32_t v);
template <> MOET_DEVICE float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <> MOET_DEVICE float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
template <typename T16> MOET_DEVICE uint32_t round2(float a, float b);
template <> MOET_DEVICE uint32_t round2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <> MOET_DEVICE uint32_t round2<__half>(float a, float b) { return pack_f16x2(a, b); }

template <typename T16> MOET_DEVICE float to_f32(T16 x);
template <> MOET_DEVICE float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> MOET_DEVICE float to_f32(__half x) { return __half2float(x); }

// the scale bytes of a lane's key codes, as they are held (two, or one with SD = 64): `row` = the
// token's scales, sl the slab, t the piece; and the f16x2 they stand for
template <int D> MOET_DEVICE uint16_t raw_key_scales(const uint8_t* row, int sl, int t) {
  if constexpr (Lay<D>::SD == 128) return *reinterpret_cast<const uint16_t*>(row + sl * 8 + 2 * t);
  return row[t];
}
template <int D> MOET_DEVICE uint32_t key_scales_f16(uint16_t raw) {
  return e4m3x2_to_f16(Lay<D>::SD == 128 ? raw : (uint16_t)(raw | raw << 8));
}
// of a lane's value codes, one per token of the pair: `row` = the pair's scales, g the piece
template <int D> MOET_DEVICE uint16_t raw_value_scales(const uint8_t* row, int sl, int g) {
  return *reinterpret_cast<const uint16_t*>(row + 2 * (Lay<D>::SD == 128 ? sl * 8 + g : g >> 1));
}
template <int D> MOET_DEVICE uint32_t key_scales(const uint8_t* row, int sl, int t) {
  return key_scales_f16<D>(raw_key_scales<D>(row, sl, t));
}
template <int D> MOET_DEVICE uint32_t value_scales(const uint8_t* row, int sl, int g) {
  return e4m3x2_to_f16(raw_value_scales<D>(row, sl, g));
}

// The grid's threads fetch `bytes` from p on into L2, a line each as far as they reach.  A prefetch uses
// no value, so it may come before the wait for the kernel that is still writing there.
MOET_DEVICE void grid_prefetch(const void* p, long long bytes) {
  const long long at = ((long long)(blockIdx.x + gridDim.x * blockIdx.y) * blockDim.x + threadIdx.x) * 128;
  if (at < bytes) prefetch_l2(static_cast<const uint8_t*>(p) + at);
}

// Positions of a sequence that a table of W pages can hold: a length out of range is taken as the nearest in range.
MOET_DEVICE int held_length(int len, int W) { return max(0, min(len, W * kPage)); }
// Sequence b of a batch with T rows: reports a length out of range, and row offsets that are out of range or order
// (they are pulled back into the rows).  Once a call.
MOET_DEVICE void check_sequence(const int* cu_q, const int* seq_lens, int b, int T, int W, int* status) {
  const int c0 = cu_q[b], c1 = cu_q[b + 1], len = seq_lens[b];
  if (c0 < 0 || c1 < c0 || c1 > T || len != held_length(len, W)) set_status(status, kBadIndex);
}
MOET_DEVICE void blank_row(long long row, void* out, float* lse, int heads, int D) {
  uint4* p = static_cast<uint4*>(out) + row * heads * (D / 8);
  for (int e = threadIdx.x; e < heads * (D / 8); e += blockDim.x) p[e] = make_uint4(0, 0, 0, 0);
  if (lse)
    for (int e = threadIdx.x; e < heads; e += blockDim.x) lse[row * heads + e] = -INFINITY;
}
// Output rows of no sequence, in front of the first offset and past the last (a batch padded to a captured size): zeros,
// and a log-sum-exp of -inf.  The grid's blocks share them out; the first rows go to the last blocks.
MOET_DEVICE void blank_rows(int first, int last, int T, void* out, float* lse, int heads, int D) {
  first = max(0, min(first, T)), last = max(first, min(last, T));
  for (int i = gridDim.x - 1 - blockIdx.x; i < first + T - last; i += gridDim.x)
    blank_row(i < first ? i : last + i - first, out, lse, heads, D);
}

MOET_DEVICE float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// What a product of a query and a key is multiplied by (scale * log2(e) * 2^k_exp), as a factor and a power of two:
// with a row's own power, 2^-118 to 2^119, either may leave f32's range while their product is in it.
struct ScoreScale {
  float factor; int exp;
};
inline ScoreScale score_scale(double scale, int k_exp) {
  int e = 0;
  const double f = std::frexp(scale * 1.4426950408889634, &e);
  return {(float)f, e + k_exp};
}
MOET_DEVICE float row_factor(const ScoreScale& s, int row_exp) {
  return pow2f(max(-126, min(127, s.exp + row_exp))) * s.factor;
}

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
