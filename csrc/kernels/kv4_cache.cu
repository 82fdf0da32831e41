// The 4-bit paged K/V cache: rows quantised as they are written, page bounds, rows read back.
//
// A row of D values is quantised in blocks of 16: scale byte s8 = e4m3(amax / 6 * 2^-exp),
// element = the e2m1 value nearest to x / (s8 * 2^exp), ties to the even code.  The quotient
// is corrected by its exact residual (x - y s is exact in one fma), so a value that lies
// midway between two codes is seen as exactly midway and the codes are those of the
// definition; for 16-bit inputs every other quotient is at least 2^-17 away from a tie.
// NaN is held as 0 and infinities as the largest value; both set the status word.
//
// Page bounds (for choosing pages, kv4_select.cu): per page and head, hi = ceil(max k / e),
// lo = floor(min k / e) over the page's 64 rows as they are held, e = 2^n the smallest power
// of two with max |k| <= 127 e.  A second launch recomputes them for every page that the
// rows touched, so they are at all times a function of the page's bytes.
#include "kv4.cuh"
#include "torch_glue.h"

#include <type_traits>

namespace moet {
namespace kv4 {

struct Rows {                     // [T, H, D] rows, inner stride 1
  const void* p; long long tok, head;
};
struct AppendArgs {
  Rows k, v;
  const long long* slots; int T, H; long long n_slots;
  uint8_t* pages; float k_inv, v_inv;     // 2^-exp
  int* status;
};

template <typename T16, bool VEC>
MOET_DEVICE void load16(const T16* p, uint32_t (&w)[8]) {
  if (VEC) {
    const uint4 a = ldg_stream_u4(p), b = ldg_stream_u4(p + 8);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
  }
}
template <typename T16> constexpr uint32_t kInf16 = std::is_same<T16, __half>::value ? 0x7C00u : 0x7F80u;

// The scale byte of 16 values, and the values over the scale (what the codes are rounded from) in x.
// The largest magnitude is found on the 16-bit patterns, which also shows what is not finite.
template <typename T16> MOET_DEVICE uint32_t scale_of(const uint32_t (&w)[8], float (&x)[16], float inv_exp, bool& bad) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
    const float2 f = unpack2<T16>(w[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
  top = max(top >> 16, top & 0xFFFFu);
  float amax = unpack2<T16>(top).x;
  if (top >= kInf16<T16>) {                              // NaN counts as 0, an infinity as a value past every scale
    bad = true;
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -3e38f), 3e38f);
      amax = fmaxf(amax, fabsf(x[i]));
    }
  }
  const float want = __fmul_rn(__fdiv_rn(amax, 6.f), inv_exp);
  const uint32_t s8 = f32_to_e4m3(fminf(want, 448.f));
  const float s = __fdiv_rn(e4m3_to_f32((uint8_t)s8), inv_exp);     // inv_exp is a power of two: exact
  if (want > 448.f) {                                    // saturated: 6 s is the largest that can be held
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = fminf(fmaxf(x[i], -8.f * s), 8.f * s);
  }
  if (s8 == 0) {
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = copysignf(0.f, x[i]);
  } else {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float y = __fmul_rn(x[i], r);
      x[i] = copysignf(__fmaf_rn(__fmaf_rn(-y, s, x[i]), r, y), x[i]);      // -0 stays -0
    }
  }
  return s8;
}
// codes of values a[0..3] in the low halves of a word's bytes, of b[0..3] in the high halves
MOET_DEVICE uint32_t codes4(const float* a, const float* b) {
  uint32_t r;
  asm("{\n.reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %5, %1;\ncvt.rn.satfinite.e2m1x2.f32 b1, %6, %2;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %7, %3;\ncvt.rn.satfinite.e2m1x2.f32 b3, %8, %4;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n}\n"
      : "=r"(r) : "f"(a[0]), "f"(a[1]), "f"(a[2]), "f"(a[3]), "f"(b[0]), "f"(b[1]), "f"(b[2]), "f"(b[3]));
  return r;
}

// One thread per (row, block of 16).  Bound by memory in a prompt (4 D bytes read and 1.125 D
// written per row and head), by the launch in a decode step.  B200, 8 heads of 128: 8183 rows 14 us
// (3.1 TB/s: four loads of 16 bytes per thread are in flight, and a short grid ends with their latency);
// 32 rows 4 us.  Rows that do not start on 16 bytes are read value by value (VEC false): written and
// read back, 8183 rows take 38 us instead of 32.
template <int D, typename T16, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(AppendArgs a) {
  using L = Lay<D>;
  pdl_entry();
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = idx / L::NB;
  const int b = (int)(idx % L::NB), bs = b % (L::SD / 16), slab = b / (L::SD / 16);
  const int tok = (int)((uint32_t)row / (uint32_t)a.H), h = (int)row - tok * a.H;      // rows are counted in 31 bits
  const bool there = row < (long long)a.T * a.H;
  bool bad = false;
  const long long slot = there ? a.slots[tok] : -1;
  if (slot >= a.n_slots) set_status(a.status, kBadIndex);
  const bool live = slot >= 0 && slot < a.n_slots;
  const int j = (int)(slot % kPage);                                   // position in its page
  uint8_t* page = a.pages + ((slot / kPage) * a.H + h) * (long long)L::kPageBytes;
  uint32_t xw[8], yw[8];
  float x[16], y[16];
#pragma unroll
  for (int i = 0; i < 8; i++) xw[i] = yw[i] = 0;
  if (there) {                           // without waiting for the slot
    load16<T16, VEC>((const T16*)a.k.p + tok * a.k.tok + h * a.k.head + b * 16, xw);
    load16<T16, VEC>((const T16*)a.v.p + tok * a.v.tok + h * a.v.head + b * 16, yw);
  }
  const uint32_t k8 = scale_of<T16>(xw, x, a.k_inv, bad), v8 = scale_of<T16>(yw, y, a.v_inv, bad);
  uint8_t* kc = page + L::KC + slab * L::kSlabBytes + j * (L::SD / 2);
  uint8_t* vc = page + L::VC + slab * L::kSlabBytes + (j >> 1) * L::SD + (j & 1) * (L::SD / 16);
  if constexpr (L::SD == 128) {
    // key piece: this block's codes and its neighbour's; each of the two lanes stores one half
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t w[4], o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = codes4(x + 4 * i, zero);
      o[i] = __shfl_xor_sync(0xffffffffu, w[i], 1);
    }
    if (live) {
      const bool odd = b & 1;
      *reinterpret_cast<uint2*>(kc + bs * 8) = odd ? make_uint2(o[2] | w[2] << 4, o[3] | w[3] << 4)
                                                   : make_uint2(w[0] | o[0] << 4, w[1] | o[1] << 4);
      *reinterpret_cast<uint2*>(vc + bs * 16) = make_uint2(codes4(y, y + 8), codes4(y + 4, y + 12));
    }
  } else if (live) {
    *reinterpret_cast<uint2*>(kc + bs * 8) = make_uint2(codes4(x, x + 8), codes4(x + 4, x + 12));
    *reinterpret_cast<uint32_t*>(vc + (2 * bs) * 8) = codes4(y, y + 4);
    *reinterpret_cast<uint32_t*>(vc + (2 * bs + 1) * 8) = codes4(y + 8, y + 12);
  }
  if (live) {
    page[L::KS + j * L::NB + b] = (uint8_t)k8;
    page[L::VS + (j >> 1) * (2 * L::NB) + 2 * b + (j & 1)] = (uint8_t)v8;
    if (bad) set_status(a.status, kBadValue);
  }
}

struct BoundsArgs {
  const long long* slots; int T, H; long long n_slots; int win;
  const uint8_t* pages; int8_t* bounds; float* unit; float k_mul;     // k_mul = 2^k_exp
};

// A warp per touched page and head.  The block looks at `win` slots and lists the last of each run in one
// page; max and min are taken in f16, where the held values are exact.  Bound by the page's own latency
// (its keys are read once more, out of L2).  B200, 8 heads of 128: 32 pages 3 us, 8183 rows (131 pages) 9 us.
template <int D>
__global__ void __launch_bounds__(64) kv4_bounds_kernel(BoundsArgs a) {
  using L = Lay<D>;
  pdl_entry();
  __shared__ int list[64], count;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y;
  if ((int)threadIdx.x < a.win) {
    const int i = blockIdx.x * a.win + threadIdx.x;
    if (i < a.T) {
      const long long s = a.slots[i], n = i + 1 < a.T ? a.slots[i + 1] : -1;
      if (s >= 0 && s < a.n_slots && (n < 0 || n / kPage != s / kPage)) list[atomicAdd(&count, 1)] = (int)(s / kPage);
    }
  }
  __syncthreads();
  const int n = count, t = lane & 3;
  constexpr int W = L::SD / 32;                    // 32-bit words of a piece
  for (int e = warp; e < n; e += 2) {
    const long long page = list[e];
    const uint8_t* base = a.pages + (page * a.H + h) * (long long)L::kPageBytes;
    __half2 hi[L::NS][W][4], lo[L::NS][W][4];
    const __half2 ninf = __float2half2_rn(-65504.f), pinf = __float2half2_rn(65504.f);
#pragma unroll
    for (int i = 0; i < L::NS * W * 4; i++) (&hi[0][0][0])[i] = ninf, (&lo[0][0][0])[i] = pinf;
#pragma unroll
    for (int j = lane >> 2; j < kPage; j += 8) {
#pragma unroll
      for (int sl = 0; sl < L::NS; sl++) {
        uint32_t c[W];
        load_words<W>(base + L::KC + sl * L::kSlabBytes + j * (L::SD / 2) + t * (L::SD / 8), c);
        const uint32_t s = key_scales<D>(base + L::KS + j * L::NB, sl, t);
#pragma unroll
        for (int w = 0; w < W; w++) {
          uint32_t r[4];
          e2m1x8_to_f16(c[w], r);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t m = mul_f16x2(r[i], s);
            const __half2 x = *reinterpret_cast<const __half2*>(&m);
            hi[sl][w][i] = __hmax2(hi[sl][w][i], x);
            lo[sl][w][i] = __hmin2(lo[sl][w][i], x);
          }
        }
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < L::NS * W * 4; i++) {
      __half2 &p = (&hi[0][0][0])[i], &q = (&lo[0][0][0])[i];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        p = __hmax2(p, __shfl_xor_sync(0xffffffffu, p, o));
        q = __hmin2(q, __shfl_xor_sync(0xffffffffu, q, o));
      }
      amax = fmaxf(amax, fmaxf(fmaxf(__low2float(p), __high2float(p)), -fminf(__low2float(q), __high2float(q))));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int ex = exp_for_127(amax);
    const float inv = pow2f(-ex);
    int8_t* out = a.bounds + (page * a.H + h) * (long long)(2 * D);
    if (lane < 4) {
#pragma unroll
      for (int sl = 0; sl < L::NS; sl++)
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
          for (int half = 0; half < 2; half++) {
            uint32_t ph = 0, pl = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float x = half ? __high2float(hi[sl][w][i]) : __low2float(hi[sl][w][i]);
              const float y = half ? __high2float(lo[sl][w][i]) : __low2float(lo[sl][w][i]);
              ph |= (uint32_t)(uint8_t)(int8_t)(int)ceilf(x * inv) << (8 * i);
              pl |= (uint32_t)(uint8_t)(int8_t)(int)floorf(y * inv) << (8 * i);
            }
            const int d = sl * L::SD + (L::SD / 4) * t + (L::SD / 8) * half + 4 * w;
            *reinterpret_cast<uint32_t*>(out + d) = ph;
            *reinterpret_cast<uint32_t*>(out + D + d) = pl;
          }
      if (lane == 0) a.unit[page * a.H + h] = amax > 0.f ? pow2f(ex) * a.k_mul : 1.f;
    }
  }
}

// the low (or, shift 4, the high) codes of four bytes as two f16x2, in order
MOET_DEVICE void values4(uint32_t w, int shift, uint32_t& a, uint32_t& b) {
  uint32_t t = (w >> shift) & 0x0F0F0F0Fu;
  t |= t >> 4;                                             // bytes 0 and 2 now hold two codes each
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %2;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b2;\n}\n" : "=r"(a), "=r"(b) : "r"(t));
}
// values of f16 pairs in the output's type
template <typename T16> MOET_DEVICE uint32_t out2(uint32_t v);
template <> MOET_DEVICE uint32_t out2<__half>(uint32_t v) { return v; }
template <> MOET_DEVICE uint32_t out2<__nv_bfloat16>(uint32_t v) {
  const float2 f = unpack2<__half>(v);
  return pack_bf16x2(f.x, f.y);
}
// a scale times 2^exp, in both halves: every product with a code is exact in f16 (exp in [-14, 4])
MOET_DEVICE uint32_t scale2(uint8_t s8, float mul) {
  const __half2 h = __float2half2_rn(e4m3_to_f32(s8) * mul);
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct ReadArgs {
  const long long* slots; int T, H; long long n_slots;
  const uint8_t* pages; float k_mul, v_mul;
  void *k, *v;                          // [T, H, D] contiguous
  int* status;
};

// One thread per (row, half block of 8): one 16-byte store for the key, one for the value, a warp's
// stores contiguous.  A row that is skipped (slot < 0) reads as zeros.  A row costs two loads one after
// the other (its slot, its codes): a thread takes U rows at once where there are rows enough.
// Bound by memory (1.125 D bytes read, 4 D written): 32768 rows of 8 heads of 128 take 32 us on B200,
// 5.4 TB/s, 83 % of the measured copy rate.
template <int D, typename T16, int U>
__global__ void __launch_bounds__(256) kv4_read_kernel(ReadArgs a) {
  using L = Lay<D>;
  pdl_entry();
  const int part = threadIdx.x % (2 * L::NB), b = part >> 1, half = part & 1;     // the same for every row
  const int bs = b % (L::SD / 16), slab = b / (L::SD / 16);
  constexpr int kRows = 256 / (2 * L::NB);                                        // of a block, at a time
  const uint32_t row0 = blockIdx.x * (uint32_t)(kRows * U) + threadIdx.x / (2 * L::NB), rows = (uint32_t)a.T * a.H;
  long long slot[U];
  int h[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t row = row0 + u * kRows, tok = row / (uint32_t)a.H;
    h[u] = (int)(row - tok * a.H);
    slot[u] = row < rows ? a.slots[tok] : -1;
  }
  uint32_t kw[U][2], vw[U][2];
  uint8_t k8[U], v8[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    kw[u][0] = kw[u][1] = vw[u][0] = vw[u][1] = 0;
    k8[u] = v8[u] = 0;
    if (slot[u] >= a.n_slots) set_status(a.status, kBadIndex);
    if (slot[u] >= 0 && slot[u] < a.n_slots) {
      const int j = (int)(slot[u] % kPage);
      const uint8_t* page = a.pages + ((slot[u] / kPage) * a.H + h[u]) * (long long)L::kPageBytes;
      const uint8_t* kc = page + L::KC + slab * L::kSlabBytes + j * (L::SD / 2);
      const uint8_t* vc = page + L::VC + slab * L::kSlabBytes + (j >> 1) * L::SD + (j & 1) * (L::SD / 16);
      load_words<2>(kc + (L::SD == 128 ? (bs >> 1) * 16 + half * 8 : bs * 8), kw[u]);
      if constexpr (L::SD == 128) load_words<2>(vc + bs * 16, vw[u]);
      else vw[u][0] = *reinterpret_cast<const uint32_t*>(vc + (2 * bs + half) * 8);
      k8[u] = page[L::KS + j * L::NB + b];
      v8[u] = page[L::VS + (j >> 1) * (2 * L::NB) + 2 * b + (j & 1)];
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t row = row0 + u * kRows;
    if (row >= rows) return;
    const uint32_t ks = scale2(k8[u], a.k_mul), vs = scale2(v8[u], a.v_mul);
    // SD = 128: a piece's low codes are one block's, its high codes the next block's; SD = 64: its two halves
    const int up = 4 * (L::SD == 128 ? b & 1 : half);
    uint32_t x[4], y[4];
    values4(kw[u][0], up, x[0], x[1]);
    values4(kw[u][1], up, x[2], x[3]);
    if constexpr (L::SD == 128) {
      values4(vw[u][0], 4 * half, y[0], y[1]);
      values4(vw[u][1], 4 * half, y[2], y[3]);
    } else {
      values4(vw[u][0], 0, y[0], y[1]);
      values4(vw[u][0], 4, y[2], y[3]);
    }
    const long long at = (long long)row * D + b * 16 + half * 8;
    *reinterpret_cast<uint4*>((T16*)a.k + at) = make_uint4(out2<T16>(mul_f16x2(x[0], ks)), out2<T16>(mul_f16x2(x[1], ks)),
                                                           out2<T16>(mul_f16x2(x[2], ks)), out2<T16>(mul_f16x2(x[3], ks)));
    *reinterpret_cast<uint4*>((T16*)a.v + at) = make_uint4(out2<T16>(mul_f16x2(y[0], vs)), out2<T16>(mul_f16x2(y[1], vs)),
                                                           out2<T16>(mul_f16x2(y[2], vs)), out2<T16>(mul_f16x2(y[3], vs)));
  }
}

static int dim_of(const torch::Tensor& pages) { return (int)(pages.size(2) / 72); }

}  // namespace kv4
}  // namespace moet

using namespace moet;
using namespace moet::kv4;

void kv4_append_launch(torch::Tensor k, torch::Tensor v, torch::Tensor slots, torch::Tensor pages, torch::Tensor bounds,
                       torch::Tensor unit, int64_t k_exp, int64_t v_exp, torch::Tensor status) {
  const int T = (int)slots.size(0), H = (int)pages.size(1), D = dim_of(pages);
  auto stream = at::cuda::getCurrentCUDAStream();
  AppendArgs a;
  a.k = {k.data_ptr(), k.stride(0), k.stride(1)};
  a.v = {v.data_ptr(), v.stride(0), v.stride(1)};
  a.slots = (const long long*)slots.data_ptr();
  a.T = T; a.H = H; a.n_slots = pages.size(0) * kPage;
  a.pages = (uint8_t*)pages.data_ptr();
  a.k_inv = std::ldexp(1.f, (int)-k_exp); a.v_inv = std::ldexp(1.f, (int)-v_exp);
  a.status = (int*)status.data_ptr();
  bool vec = true;                       // 16-byte loads need every row to start on 16 bytes
  for (const torch::Tensor* x : {&k, &v})
    vec = vec && ((uintptr_t)x->data_ptr() % 16 == 0) && x->stride(0) % 8 == 0 && x->stride(1) % 8 == 0;
  const long long threads = (long long)T * H * (D / 16);
  const dim3 grid((unsigned)((threads + 255) / 256));
  auto go = [&](auto dim, auto t) {
    constexpr int DD = decltype(dim)::value;
    using T16 = decltype(t);
    if (vec) launch_k(kv4_append_kernel<DD, T16, true>, grid, dim3(256), 0, stream, a);
    else launch_k(kv4_append_kernel<DD, T16, false>, grid, dim3(256), 0, stream, a);
    // Long runs in one page (prompts) want a long window, pages of one row each (decode steps) a short one, and the
    // call does not say which it has: few rows may be either, more than 4096 are prompts.  us of an append with win =
    // 2 / 8 / 64, 8 heads of 128, cold, B200: one prompt's rows, 256: 11.4 / 11.4 / 11.3, 1024: 15.3 / 13.4 / 13.4, 2048: 21.5 /
    // 15.4 / 15.4, 8183: 54.4 / 29.8 / 25.6; rows of a page each, 32: 13 / 19.5 / 48, 512: 19.5 / 23.6 / 87, 2048: 42 / 44 / 118.
    const int win = T > 4096 ? 64 : T >= 1024 ? 8 : 2;
    BoundsArgs c{a.slots, T, H, a.n_slots, win, a.pages, (int8_t*)bounds.data_ptr(),
                 (float*)unit.data_ptr(), std::ldexp(1.f, (int)k_exp)};
    launch_k(kv4_bounds_kernel<DD>, dim3((T + c.win - 1) / c.win, H), dim3(64), 0, stream, c);
  };
  auto by_type = [&](auto dim) {
    if (k.scalar_type() == at::kHalf) go(dim, __half{});
    else go(dim, __nv_bfloat16{});
  };
  if (D == 64) by_type(std::integral_constant<int, 64>{});
  else if (D == 128) by_type(std::integral_constant<int, 128>{});
  else by_type(std::integral_constant<int, 256>{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void kv4_read_launch(torch::Tensor slots, torch::Tensor pages, int64_t k_exp, int64_t v_exp, torch::Tensor k,
                     torch::Tensor v, torch::Tensor status) {
  const int T = (int)slots.size(0), H = (int)pages.size(1), D = dim_of(pages);
  auto stream = at::cuda::getCurrentCUDAStream();
  ReadArgs a{(const long long*)slots.data_ptr(), T, H, pages.size(0) * kPage, (const uint8_t*)pages.data_ptr(),
             std::ldexp(1.f, (int)k_exp), std::ldexp(1.f, (int)v_exp), k.data_ptr(), v.data_ptr(),
             (int*)status.data_ptr()};
  const long long threads = (long long)T * H * (D / 8);
  // Four rows a thread where one row each would be two or more full waves (32768 rows x 8 heads: 41 us with
  // one, 37 with four, cold); below that more threads hide the same latency (1574 rows, D = 64: 8.1 and 8.3).
  const int per = threads >= 2ll * sm_count() * 2048 ? 4 : 1;
  const dim3 grid((unsigned)((threads + 256 * per - 1) / (256 * per)));
  auto launch = [&](auto dim, auto t, auto u) {
    launch_k(kv4_read_kernel<decltype(dim)::value, decltype(t), decltype(u)::value>, grid, dim3(256), 0, stream, a);
  };
  auto by_type = [&](auto dim, auto u) {
    if (k.scalar_type() == at::kHalf) launch(dim, __half{}, u);
    else launch(dim, __nv_bfloat16{}, u);
  };
  auto go = [&](auto dim) {
    if (per == 4) by_type(dim, std::integral_constant<int, 4>{});
    else by_type(dim, std::integral_constant<int, 1>{});
  };
  if (D == 64) go(std::integral_constant<int, 64>{});
  else if (D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 256>{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
