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

template <typename T16> MOET_DEVICE uint32_t pack2(float a, float b);
template <> MOET_DEVICE uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <> MOET_DEVICE uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <typename T16, bool VEC>
MOET_DEVICE void load16(const T16* p, float (&x)[16]) {
  T16 h[16];
  if (VEC) {
    reinterpret_cast<uint4*>(h)[0] = ldg_stream_u4(p);
    reinterpret_cast<uint4*>(h)[1] = ldg_stream_u4(p + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++) h[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 16; i++) x[i] = to_f32(h[i]);
}

// The block's scale byte, and its values over the scale (what a code is rounded from) in x.
MOET_DEVICE uint32_t scale_of(float (&x)[16], float inv_exp, bool& bad, float& s) {
  float amax = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    odd |= !(fabsf(x[i]) <= 3.3895314e38f);      // NaN or infinite (bf16's largest finite value)
    amax = fmaxf(amax, fabsf(x[i]));
  }
  if (odd) {
    bad = true;
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -3e38f), 3e38f);
      amax = fmaxf(amax, fabsf(x[i]));
    }
  }
  const float want = fminf(__fmul_rn(__fdiv_rn(amax, 6.f), inv_exp), 448.f);
  const uint32_t s8 = f32_to_e4m3(want);
  s = __fdiv_rn(e4m3_to_f32((uint8_t)s8), inv_exp);     // inv_exp is a power of two: exact
  if (s8 == 0) {
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = copysignf(0.f, x[i]);
  } else {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float c = fminf(fmaxf(x[i], -8.f * s), 8.f * s);    // beyond 6 s all the same; keeps the fma finite
      const float y = __fmul_rn(c, r);
      x[i] = __fmaf_rn(__fmaf_rn(-y, s, c), r, y);
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
// written per row and head), by the launch in a decode step.
template <int D, typename T16, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(AppendArgs a) {
  using L = Lay<D>;
  pdl_entry();
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = idx / L::NB;
  const int b = (int)(idx % L::NB), bs = b % (L::SD / 16), slab = b / (L::SD / 16);
  const int tok = (int)(row / a.H), h = (int)(row % a.H);
  bool live = row < (long long)a.T * a.H, bad = false;
  const long long slot = live ? a.slots[tok] : -1;
  if (slot >= a.n_slots) set_status(a.status, kBadIndex);
  live = slot >= 0 && slot < a.n_slots;
  const int j = (int)(slot % kPage);                                   // position in its page
  uint8_t* page = a.pages + ((slot / kPage) * a.H + h) * (long long)L::kPageBytes;
  float x[16], y[16], s;
#pragma unroll
  for (int i = 0; i < 16; i++) x[i] = y[i] = 0.f;
  if (live) {
    load16<T16, VEC>((const T16*)a.k.p + tok * a.k.tok + h * a.k.head + b * 16, x);
    load16<T16, VEC>((const T16*)a.v.p + tok * a.v.tok + h * a.v.head + b * 16, y);
  }
  const uint32_t k8 = scale_of(x, a.k_inv, bad, s), v8 = scale_of(y, a.v_inv, bad, s);
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

// A warp per touched page and head.  The block looks at `win` slots and lists the last of each
// run in one page; max and min are taken in f16, where the held values are exact.
template <int D>
__global__ void __launch_bounds__(256) kv4_bounds_kernel(BoundsArgs a) {
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
  for (int e = warp; e < n; e += 8) {
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

// four bytes' low codes and high codes
MOET_DEVICE void values4(uint32_t w, float* lo, float* hi) {
  uint32_t r[4];
  e2m1x8_to_f16(w, r);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
    lo[i] = f.x, hi[i] = f.y;
  }
}

struct ReadArgs {
  const long long* slots; int T, H; long long n_slots;
  const uint8_t* pages; float k_mul, v_mul;
  void *k, *v;                          // [T, H, D] contiguous
  int* status;
};

// One thread per (row, block of 16); a row that is skipped (slot < 0) reads as zeros.
template <int D, typename T16>
__global__ void __launch_bounds__(256) kv4_read_kernel(ReadArgs a) {
  using L = Lay<D>;
  pdl_entry();
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = idx / L::NB;
  if (row >= (long long)a.T * a.H) return;
  const int b = (int)(idx % L::NB), bs = b % (L::SD / 16), slab = b / (L::SD / 16);
  const int tok = (int)(row / a.H), h = (int)(row % a.H);
  const long long slot = a.slots[tok];
  if (slot >= a.n_slots) set_status(a.status, kBadIndex);
  const bool live = slot >= 0 && slot < a.n_slots;
  float x[16], y[16];
#pragma unroll
  for (int i = 0; i < 16; i++) x[i] = y[i] = 0.f;
  if (live) {
    const int j = (int)(slot % kPage);
    const uint8_t* page = a.pages + ((slot / kPage) * a.H + h) * (long long)L::kPageBytes;
    const float ks = e4m3_to_f32(page[L::KS + j * L::NB + b]) * a.k_mul;
    const float vs = e4m3_to_f32(page[L::VS + (j >> 1) * (2 * L::NB) + 2 * b + (j & 1)]) * a.v_mul;
    const uint8_t* kc = page + L::KC + slab * L::kSlabBytes + j * (L::SD / 2);
    const uint8_t* vc = page + L::VC + slab * L::kSlabBytes + (j >> 1) * L::SD + (j & 1) * (L::SD / 16);
    if constexpr (L::SD == 128) {
      uint32_t c[4];
      load_words<4>(kc + (bs >> 1) * 16, c);
#pragma unroll
      for (int w = 0; w < 4; w++) {      // this block's codes are the low or the high halves
        float lo[4], hi[4];
        values4(c[w], lo, hi);
#pragma unroll
        for (int i = 0; i < 4; i++) x[4 * w + i] = ((b & 1) ? hi[i] : lo[i]) * ks;
      }
      load_words<2>(vc + bs * 16, *reinterpret_cast<uint32_t(*)[2]>(c));
      values4(c[0], y, y + 8);
      values4(c[1], y + 4, y + 12);
    } else {
      uint32_t c[2];
      load_words<2>(kc + bs * 8, c);
      values4(c[0], x, x + 8);
      values4(c[1], x + 4, x + 12);
      values4(*reinterpret_cast<const uint32_t*>(vc + (2 * bs) * 8), y, y + 4);
      values4(*reinterpret_cast<const uint32_t*>(vc + (2 * bs + 1) * 8), y + 8, y + 12);
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] *= ks;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) y[i] *= vs;
  }
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; i++) o[i] = pack2<T16>(x[2 * i], x[2 * i + 1]);
  uint4* dst = reinterpret_cast<uint4*>((T16*)a.k + row * D + b * 16);
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
#pragma unroll
  for (int i = 0; i < 8; i++) o[i] = pack2<T16>(y[2 * i], y[2 * i + 1]);
  dst = reinterpret_cast<uint4*>((T16*)a.v + row * D + b * 16);
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
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
    BoundsArgs c{a.slots, T, H, a.n_slots, T >= 4096 ? 64 : 8, a.pages, (int8_t*)bounds.data_ptr(),
                 (float*)unit.data_ptr(), std::ldexp(1.f, (int)k_exp)};
    launch_k(kv4_bounds_kernel<DD>, dim3((T + c.win - 1) / c.win, H), dim3(256), 0, stream, c);
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
  const long long threads = (long long)T * H * (D / 16);
  const dim3 grid((unsigned)((threads + 255) / 256));
  auto go = [&](auto dim) {
    constexpr int DD = decltype(dim)::value;
    if (k.scalar_type() == at::kHalf) launch_k(kv4_read_kernel<DD, __half>, grid, dim3(256), 0, stream, a);
    else launch_k(kv4_read_kernel<DD, __nv_bfloat16>, grid, dim3(256), 0, stream, a);
  };
  if (D == 64) go(std::integral_constant<int, 64>{});
  else if (D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 256>{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
