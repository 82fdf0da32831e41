// Attention of many query rows per sequence (prompt chunks) over the 4-bit paged K/V cache, on
// the tcgen05 tensor cores.  The mathematics and the layout of a batch are kv4_attend.cu's.
//
// A block takes two tiles of 128 rows ((token, head of the group) pairs of one K/V head; one
// tile with D = 256) and walks over the keys.  Per step of 64 keys and tile
//   S = Q K^T   f16 x f16 -> f32 in tensor memory,
//   P = exp2(S c - m), over S as f16 (the A operand of the second product),
//   O += P V    f32 in tensor memory.
// Roles: four warps convert keys and values from 4 bits into f16 operands in shared memory
// (exact, kv4.cuh), once for both tiles; four warps per tile hold a row per thread and do the
// softmax, 64 keys at a step; one warp issues the products.  Each tile has two S buffers, so its
// next scores are computed under its softmax; the order of issue is S0' PV0 S1' PV1 (' = next step).
//
// The running maximum is only moved when a row's scores exceed it by 2^8: O is rescaled a few times
// per row, not per block.  Weights are P = 2^7 exp2(score - maximum) <= 2^15 in f16: a weight of a long
// tail is off by at most 2^-32 of the row's largest (2^-11 of itself down to 2^-21 of that); sums stay in
// f32.  A chunk of 2048 rows over 16384 keys takes 579 us so, 588 if the maximum moves at 2^6 and 607 at 2^4.  Operands are
// in the no-swizzle core-matrix order; the orders of values (depth of S, columns of O) are the
// ones the cache's pieces give, so every 16-byte store of the conversion is one core-matrix row
// and a warp's stores fill whole matrices without bank conflicts.
//
// B200, 2048 x 4 rows, 8 heads of 128, 16384 keys: 551 us for the kernel (575 with the join and the launches,
// 896 TFLOP/s, 54 % of the measured bf16 rate; 128 registers, 256 bytes of spills a thread).  The tensor path is busy 60 % of the time (64 keys a step
// read Q and K from shared memory at three quarters of the product's own rate), exp2 46 %, the ALU
// 34 %; the rest is the chain score, softmax, product of a step.  Measured and not taken: a warp per tile that
// issues the products (570 us), eight warps that convert (586), 128 keys a step with one S
// buffer per tile (601), two threads per row (748).
#include "kv4.cuh"
#include "tcgen05.cuh"
#include "torch_glue.h"

#include <algorithm>
#include <tuple>

// Tries of a bounded wait, and of the wait for the softmax's weights.  Constants (as an argument they cost the kernel
// 3 %: registers); the test of waits that run out builds this file with its own.
#ifndef MOET_KV4_TRIES
#define MOET_KV4_TRIES tc::kWaitTries
#define MOET_KV4_P_TRIES tc::kWaitTries
#endif

namespace moet {
namespace kv4 {

struct PromptArgs {
  const void* q; long long q_tok; int q_head;
  const int *cu_q, *seq_lens, *table; int B, W, T, H, G, max_q, window;
  const uint8_t* pages; int n_pages;
  ScoreScale scale;
  float v_mul;
  void* out; float* lse;
  int whole, splits;                  // tiles that a block takes whole; stretches of keys of each of the others, at most
  float* part;                        // the stretches' outputs, maxima and sums
  int* status;
};

template <int D> struct PromptCfg {
  static constexpr int BK = D == 256 ? 64 : 128;            // keys converted at a time
  static constexpr int SK = 64, HALVES = BK / SK;           // keys of a softmax step: one page
  static constexpr int TILES = D == 256 ? 1 : 2;            // row tiles per block
  static constexpr int kSoftWarps = 4 * TILES, kWarps = kSoftWarps + 5;   // + conversion, + products
  static constexpr int kQBytes = 128 * D * 2, kKBytes = BK * D * 2;   // one operand tile; V's is K's size
  static constexpr int kOCol = 256;    // tensor memory: S of tile t and step n at 128 t + 64 (n & 1), P over it; O at 256 + D t
};

template <int D> struct PromptSmem {
  using C = PromptCfg<D>;
  uint8_t q[C::TILES][C::kQBytes];
  uint8_t k[2][C::kKBytes];
  uint8_t v[2][C::kKBytes];
  float row_scale[C::TILES * 128];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], pv_done[2], o_full[2], done;
  uint32_t tmem;
  const int* holes;                    // the sequence's table row where a page is missing, else null
};

namespace pr {
MOET_DEVICE uint32_t idesc_f16(int M, int N) { return 1u << 4 | (uint32_t)(N >> 3) << 17 | (uint32_t)(M >> 4) << 24; }
// One product, issued by the warp's elected lane (`lead`); the operands are the same in every lane,
// so that they stay in uniform registers.
MOET_DEVICE void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead) : "memory");
}
MOET_DEVICE void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead) : "memory");
}
MOET_DEVICE void commit(uint32_t lead, uint64_t* bar) {
  asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n"
               "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n"
               ::"r"(tc::smem_addr(bar)), "r"(lead) : "memory");
}
MOET_DEVICE uint32_t elect() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r;
}
#define KV4_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define KV4_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
MOET_DEVICE void ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : KV4_R8(r, 0), KV4_R8(r, 8), KV4_R8(r, 16), KV4_R8(r, 24) : "r"(addr));
}
MOET_DEVICE void st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
      ::KV4_W8(r, 0), KV4_W8(r, 8), KV4_W8(r, 16), KV4_W8(r, 24), "r"(addr) : "memory");
}
MOET_DEVICE void st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
      ::KV4_W8(r, 0), KV4_W8(r, 8), "r"(addr) : "memory");
}
MOET_DEVICE void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
MOET_DEVICE void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_addr(bar)) : "memory");
}
// x * c + b on a pair
MOET_DEVICE void fma2(float& x, float& y, float c, float b) {
  asm("{\n.reg .b64 u, v, w;\nmov.b64 u, {%0, %1};\nmov.b64 v, {%2, %2};\nmov.b64 w, {%3, %3};\n"
      "fma.rn.ftz.f32x2 u, u, v, w;\nmov.b64 {%0, %1}, u;\n}\n" : "+f"(x), "+f"(y) : "f"(c), "f"(b));
}
MOET_DEVICE void add2(float& x, float& y, float a, float b) {
  asm("{\n.reg .b64 u, v;\nmov.b64 u, {%0, %1};\nmov.b64 v, {%2, %3};\nadd.rn.ftz.f32x2 u, u, v;\nmov.b64 {%0, %1}, u;\n}\n"
      : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
MOET_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
}  // namespace pr

// Keys of a stretch, at least.  us with 128 / 256 / 512, 8 K/V heads, 4 rows per token, B200: 128 tokens of 1000 keys,
// D = 128: 26.4 / 25.9 / 28.9, D = 64: 20.8 / 19.5 / 22.2; 70 tokens, D = 256: 24.4 / 24.0 / 27.8; 4 sequences of 40
// tokens and 700 keys, D = 64: 17.7 / 18.1 / 20.4.
constexpr int kMinStretch = 256;
constexpr float kSlack = 8.f, kLift = 7.f;       // in powers of two; together 15, as f16 holds

// where the part of one stretch of a tile's keys lies: rows x D outputs, then the rows' maxima and sums
template <int D> MOET_DEVICE long long prompt_part(const PromptArgs& a, int entry, int split) {
  return ((long long)entry * a.splits + split) * (PromptCfg<D>::TILES * 128 * (D + 2));
}

// Entry of the grid's order: a row tile of a sequence and K/V head, the last rows (the longest stretches of keys) of every
// sequence and head first.
template <int D> struct PromptTile {
  int b, h, back;                     // back: tiles of the sequence behind this one
  int c0, all, nq, p0;                // first row, rows, rows within max_q, position of the first row
  int rows, tile, row0, live;         // query rows; tile (< 0: none), its first row and rows
  int p_first, p_last;                // positions of its first and last row
  int from, to, splits;               // its key blocks [from, to), and the stretches they are shared out over
  MOET_DEVICE PromptTile(const PromptArgs& a, int entry) {
    constexpr int RT = PromptCfg<D>::TILES * 128, BK = PromptCfg<D>::BK;
    b = entry % a.B, h = entry / a.B % a.H, back = entry / (a.B * a.H);
    c0 = max(0, min(a.cu_q[b], a.T)), all = max(0, max(0, min(a.cu_q[b + 1], a.T)) - c0);
    nq = min(all, a.max_q);                                // the tiles that there are: rows past them are reported
    p0 = held_length(a.seq_lens[b], a.W) - all;
    rows = nq * a.G;
    tile = (rows + RT - 1) / RT - 1 - back;
    row0 = tile * RT, live = min(rows - row0, RT);
    p_first = p0 + row0 / a.G, p_last = p0 + (row0 + live - 1) / a.G;
    from = a.window > 0 ? max(0, p_first - a.window + 1) / BK : 0;
    to = p_last < 0 ? from : p_last / BK + 1;
    splits = entry < a.whole ? 1 : max(1, min(a.splits, (to - from) * BK / kMinStretch));
  }
};

// scores of keys j0 .. that the row at position p does not see -> -inf
template <int N> MOET_DEVICE void hide(uint32_t (&u)[N], int j0, int p, int window) {
#pragma unroll
  for (int k = 0; k < N; k++)
    if (j0 + k > p || (window > 0 && j0 + k <= p - window)) u[k] = 0xFF800000u;
}

template <int D, typename T16>
__global__ void __launch_bounds__(PromptCfg<D>::kWarps * 32, 1) kv4_prompt_kernel(PromptArgs a) {
  using L = Lay<D>;
  using C = PromptCfg<D>;
  constexpr int BK = C::BK, TILES = C::TILES, E2 = L::SD / 8;      // E2: f16 pairs of a key piece
  constexpr uint32_t kQSbo = 16 * D, kKSbo = 16 * D, kVSbo = 16 * BK;   // bytes from 8 rows to the next 8
  extern __shared__ __align__(128) uint8_t smem_raw[];
  PromptSmem<D>& sm = *reinterpret_cast<PromptSmem<D>*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_entry();

  const int entry = (int)blockIdx.x < a.whole ? blockIdx.x : a.whole + (int)(blockIdx.x - a.whole) / a.splits;
  const int split = (int)blockIdx.x < a.whole ? 0 : (int)(blockIdx.x - a.whole) % a.splits;
  const PromptTile<D> tl(a, entry);
  const int b = tl.b, h = tl.h, c0 = tl.c0, rows = tl.rows, p0 = tl.p0, splits = tl.splits;
  blank_rows(a.cu_q[0], a.cu_q[a.B], a.T, a.out, a.lse, a.H * a.G, D);
  if (h == 0 && tl.back == 0 && split == 0) {
    if (tid == 0) check_sequence(a.cu_q, a.seq_lens, b, a.T, a.W, a.status);
    if (tl.all > tl.nq) {
      if (tid == 0) set_status(a.status, kBadSize);
      for (int i = tl.nq; i < tl.all; i++) blank_row(c0 + i, a.out, a.lse, a.H * a.G, D);
    }
  }
  if (tl.tile < 0 || split >= splits) return;
  const int row0 = tl.row0, live = tl.live, p_first = tl.p_first, p_last = tl.p_last;
  const int ntile = (live + 127) / 128;
  const int per = (tl.to - tl.from + splits - 1) / splits;
  const int kb0 = min(tl.to, tl.from + split * per), kb1 = min(tl.to, kb0 + per);
  const int nkb = kb1 - kb0;
  const int steps = nkb > 0 ? min(p_last / C::SK + 1, kb1 * C::HALVES) - kb0 * C::HALVES : 0;   // softmax steps

  // ---- pages of this stretch that some row sees and that are not in the pool: reported, and hidden step by step.  Looked
  // for once, in front: flags that the conversion passes on with every step cost D = 256 14 %, D = 128 1 %.
  constexpr int KP = BK / kPage;
  const int page0 = max(kb0 * KP, a.window > 0 ? max(0, p_first - a.window + 1) / kPage : 0);
  const int page1 = nkb > 0 ? min(kb1 * KP, p_last / kPage + 1) : 0;
  auto in_pool = [&](int phys) { return (uint32_t)phys < (uint32_t)a.n_pages; };
  bool missing = false;
  for (int x = page0 + tid; x < page1; x += C::kWarps * 32) missing |= !in_pool(a.table[(long long)b * a.W + x]);
  if (tid == 0) sm.holes = nullptr;

  // ---- queries as f16 operands (bf16 rows scaled to at most 512), barriers, tensor memory
  if (warp == 0) tc::tmem_alloc(&sm.tmem, 512);
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&sm.k_full[i], 128);
      tc::mbar_init(&sm.v_full[i], 128);
      tc::mbar_init(&sm.k_empty[i], 1);
      tc::mbar_init(&sm.v_empty[i], 1);
      tc::mbar_init(&sm.s_full[i][0], 1);
      tc::mbar_init(&sm.s_full[i][1], 1);
      tc::mbar_init(&sm.p_full[i][0], 128);
      tc::mbar_init(&sm.p_full[i][1], 128);
      tc::mbar_init(&sm.pv_done[i], 1);
      tc::mbar_init(&sm.o_full[i], 1);
    }
    tc::mbar_init(&sm.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int it = tid; it < TILES * 128 * 4; it += C::kWarps * 32) {   // kWarps * 32 is a multiple of 4: lanes stay together
    const int r = it >> 2, t = it & 3, row = row0 + r;
    const bool on = r < live;
    const T16* src = (const T16*)a.q + (long long)(c0 + (on ? row / a.G : 0)) * a.q_tok +
                     (long long)(h * a.G + (on ? row % a.G : 0)) * a.q_head;
    float v[L::NS][2 * E2], amax = 0.f;
#pragma unroll
    for (int sl = 0; sl < L::NS; sl++)
#pragma unroll
      for (int x = 0; x < 2 * E2 / 8; x++) {
        const uint4 y = on ? *reinterpret_cast<const uint4*>(src + sl * L::SD + t * 2 * E2 + x * 8) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float2 f = unpack2<T16>(w[k]);
          v[sl][8 * x + 2 * k] = f.x, v[sl][8 * x + 2 * k + 1] = f.y;
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
    float mul = 1.f;
    int e = 0;                                             // the row is held times 2^-e
    if (!std::is_same<T16, __half>::value) {
      const uint32_t quad = 0xFu << (lane & 28);
      amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 2));
      e = amax > 0.f ? max(-110, min(119, (int)(__float_as_uint(amax) >> 23) - 127 - 8)) : 0;
      mul = pow2f(-e);
    }
    // the scale's sign goes to the row, so that scores only grow; above 0, so that -inf stays what it is
    if (t == 0) sm.row_scale[r] = fmaxf(fabsf(row_factor(a.scale, e)), 1e-30f);
    mul = copysignf(mul, a.scale.factor);
    uint8_t* dst = sm.q[r >> 7] + ((r & 127) >> 3) * kQSbo + (r & 7) * 16;
#pragma unroll
    for (int sl = 0; sl < L::NS; sl++)
#pragma unroll
      for (int c = 0; c < E2 / 4; c++) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = pack_f16x2(v[sl][4 * c + k] * mul, v[sl][E2 + 4 * c + k] * mul);
        *reinterpret_cast<uint4*>(dst + (sl * (L::SD / 8) + t * (E2 / 4) + c) * 128) = make_uint4(w[0], w[1], w[2], w[3]);
      }
  }
  tc::fence_proxy_async_smem();
  tc::fence_before();
  const bool holes = __syncthreads_or(missing);
  if (holes) {
    if (tid == 0) {
      sm.holes = a.table + (long long)b * a.W;
      set_status(a.status, kBadIndex);
    }
    __syncthreads();
  }
  tc::fence_after();
  const uint32_t tmem = sm.tmem;
  bool ok = true;

  if (warp < C::kSoftWarps) {
    // ---- softmax: thread = row; its scores of a step all in registers
    const int t = warp >> 2, r = t * 128 + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_at = tmem + lanes + C::kOCol + t * D;
    const int row = row0 + r, p = p0 + min(row, rows - 1) / a.G;
    const int pt_first = holes ? -1 : p0 + (row0 + t * 128) / a.G;     // with holes, every step is looked at key by key
    const int pt_last = p0 + min(row0 + t * 128 + 127, rows - 1) / a.G;
    const float cs = sm.row_scale[r];
    // the reference is the product m + rest, exactly: the largest score's own difference is 0 at any size
    float m = -INFINITY, rest = 0.f, l = 0.f;
    if (t < ntile) {
      for (int i = 0; i < steps && ok; i++) {
        constexpr int SK = C::SK;
        const int j0 = kb0 * BK + i * SK;
        const uint32_t s_at = tmem + lanes + t * 128 + (i & 1) * SK;
        ok = tc::mbar_wait(&sm.s_full[t][i & 1], (i >> 1) & 1, MOET_KV4_TRIES);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc::fence_after();
        uint32_t u[SK / 32][32];
#pragma unroll
        for (int c = 0; c < SK / 32; c++) pr::ld32(s_at + c * 32, u[c]);
        const bool edge = j0 + SK - 1 > pt_first || (a.window > 0 && j0 <= pt_last - a.window);
        tc::tmem_wait_ld();
        // the row's largest score; where it exceeds the reference by kSlack (or there is none yet) the reference moves
        float top = -INFINITY, top1 = -INFINITY;
        int pe = p;
        if (edge && sm.holes && !in_pool(sm.holes[j0 / kPage])) pe = -1;     // nobody sees a page that is not there
#pragma unroll
        for (int c = 0; c < SK / 32; c++) {
          if (edge) hide<32>(u[c], j0 + c * 32, pe, a.window);
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            top = pr::max3(top, __uint_as_float(u[c][k]), __uint_as_float(u[c][k + 1]));
            top1 = pr::max3(top1, __uint_as_float(u[c][k + 2]), __uint_as_float(u[c][k + 3]));
          }
        }
        top = fmaxf(top, top1);
        const float raw = top;
        top *= cs;
        const bool move = m == -INFINITY ? top > -INFINITY : top > m + kSlack;
        if (__any_sync(0xffffffffu, move)) {
          const float f = !move ? 1.f : m == -INFINITY ? 0.f : fast_exp2(m - top);
          if (move) m = top, rest = __fmaf_rn(raw, cs, -top);
          l *= f;
          // Once the product before is in O.  A wait by parity is right only if the phase before has ended:
          // these scores were issued after the product of two steps ago.
          if (i > 0) {
            ok = tc::mbar_wait(&sm.pv_done[t], (i - 1) & 1, MOET_KV4_TRIES);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
              uint32_t u[32];
              pr::ld32(o_at + c * 32, u);
              tc::tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; k++) u[k] = __float_as_uint(__uint_as_float(u[k]) * f);
              pr::st32(o_at + c * 32, u);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int c = 0; c < SK / 32; c++) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float x = __uint_as_float(u[c][k]), y = __uint_as_float(u[c][k + 1]);
            pr::fma2(x, y, cs, -ref);
            pr::add2(x, y, kLift - rest, kLift - rest);
            x = fast_exp2(x), y = fast_exp2(y);
            pr::add2(s0, s1, x, y);
            pk[k / 2] = pack_f16x2(x, y);
          }
          pr::st16(s_at + c * 16, pk);       // P takes the columns of the scores
        }
        l += s0 + s1;
        pr::wait_st();
        tc::fence_before();
        pr::arrive(&sm.p_full[t][i & 1]);   // one per buffer: a warp may end its next step before the last warp ends this one
      }
      // ---- output
      if (nkb > 0 && ok) {
        ok = tc::mbar_wait(&sm.o_full[t], 0, MOET_KV4_TRIES);      // its own barrier: pv_done may still be two phases back
        if (!__all_sync(0xffffffffu, ok)) ok = false;
      }
      if (ok) {
        tc::fence_after();
        const float inv = l > 0.f ? __fdividef(a.v_mul, l) : l;
        float* part = nullptr;
        if (splits > 1) {
          part = a.part + prompt_part<D>(a, entry - a.whole, split);
          part[TILES * 128 * D + r] = m;
          part[TILES * 128 * (D + 1) + r] = l;
        }
        const long long at = (long long)(c0 + row / a.G) * a.H * a.G + h * a.G + row % a.G;
        const bool on = r < live;
        constexpr int E = L::SD / 8;         // values of a lane's piece; column (i, g) of a slab = value E g + i
#pragma unroll
        for (int sl = 0; sl < L::NS; sl++)
#pragma unroll
          for (int part_i = 0; part_i < E / 8; part_i++) {      // 64 columns: values i = 8 part_i .. + 7 of all pieces
            uint32_t u[2][32];
            if (nkb > 0) {
              pr::ld32(o_at + sl * L::SD + part_i * 64, u[0]);
              pr::ld32(o_at + sl * L::SD + part_i * 64 + 32, u[1]);
              tc::tmem_wait_ld();
            } else {
#pragma unroll
              for (int k = 0; k < 64; k++) u[k >> 5][k & 31] = 0;
            }
            if (on) {
#pragma unroll
              for (int g = 0; g < 8; g++) {
                float x[8];
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = __uint_as_float(u[(k * 8 + g) >> 5][(k * 8 + g) & 31]);
                if (part) {                  // as it is: the join divides
                  if (nkb > 0) {
                    float4* to4 = reinterpret_cast<float4*>(part + r * D + sl * L::SD + E * g + part_i * 8);
                    to4[0] = make_float4(x[0], x[1], x[2], x[3]);
                    to4[1] = make_float4(x[4], x[5], x[6], x[7]);
                  }
                  continue;
                }
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] *= inv;
                *reinterpret_cast<uint4*>((T16*)a.out + at * D + sl * L::SD + E * g + part_i * 8) =
                    make_uint4(round2<T16>(x[0], x[1]), round2<T16>(x[2], x[3]), round2<T16>(x[4], x[5]),
                               round2<T16>(x[6], x[7]));
              }
            }
          }
        if (on && a.lse && !part) a.lse[at] = l == 0.f ? -INFINITY : (m + (__log2f(l) - kLift)) * 0.6931471805599453f;
      }
    }
  } else if (warp < C::kSoftWarps + 4) {
    // ---- keys and values from 4 bits to f16 operands; codes are fetched a block ahead
    const int dt = tid - C::kSoftWarps * 32;
    constexpr int KI = BK * 4 * L::NS / 128;                 // key pieces per thread: 4
    constexpr int W = L::SD / 32;                            // 32-bit words of a key piece
    const int kt = (dt >> 3) & 3, kj = (dt & 7) | (dt >> 5) << 3;   // piece, token (of 32): 8 neighbours store one core matrix
    constexpr int OCT = BK / 8;                              // octets of tokens
    const int vg = dt & 7, vo = (dt >> 3) % OCT, vsl = (dt >> 3) / OCT;
    uint32_t kc[KI][W], vc[4][W];
    uint16_t ks[KI], vs[4];                                  // scales as they are held: converting waits for the load
    // pages of a key block, looked up two blocks ahead (the look-up is a load of its own): -1 for none
    int ahead[KP], page[KP];                                 // of the block after the next one, of the next one
    auto look_up = [&](int kb, int (&to)[KP]) {
#pragma unroll
      for (int i = 0; i < KP; i++) {
        const int x = kb * KP + i;
        to[i] = x >= page0 && x < page1 ? a.table[(long long)b * a.W + x] : -1;
      }
    };
    auto at = [&](int phys) -> const uint8_t* {
      return in_pool(phys) ? a.pages + ((long long)phys * a.H + h) * L::kPageBytes : nullptr;
    };
    auto fetch_k = [&](int kb) {
#pragma unroll
      for (int i = 0; i < KI; i++) {
        const int sl = i * 32 / BK, j = i * 32 % BK + kj;    // BK = 64: two tokens per slab
        const uint8_t* pg = at(page[i * 32 % BK / kPage]);
        const int jj = j % kPage;
        ks[i] = 0;
        if (pg && kb * BK + j <= p_last) {
          load_words<W>(pg + L::KC + sl * L::kSlabBytes + jj * (L::SD / 2) + kt * (L::SD / 8), kc[i]);
          ks[i] = raw_key_scales<D>(pg + L::KS + jj * L::NB, sl, kt);
        } else {
#pragma unroll
          for (int w = 0; w < W; w++) kc[i][w] = 0;
        }
      }
    };
    auto fetch_v = [&](int kb) {
      const uint8_t* pg = at(vo / 8 ? page[KP - 1] : page[0]);
      const int pair0 = vo % 8 * 4;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        vs[x] = 0;
        const int j = kb * BK + vo * 8 + 2 * x;
        if (pg && j <= p_last) {
          load_words<W>(pg + L::VC + vsl * L::kSlabBytes + (pair0 + x) * L::SD + vg * (L::SD / 8), vc[x]);
          vs[x] = raw_value_scales<D>(pg + L::VS + (pair0 + x) * (2 * L::NB), vsl, vg);
          if (j == p_last) vs[x] &= 0xFFu;                   // the pair's second token is past the rows
        } else {
#pragma unroll
          for (int w = 0; w < W; w++) vc[x][w] = 0;
        }
      }
    };
    look_up(kb0, page);
    look_up(kb0 + 1, ahead);
    fetch_k(kb0);
    fetch_v(kb0);
    for (int i = 0; i < nkb && ok; i++) {
      const int st = i & 1;
      if (i >= 2) ok = tc::mbar_wait(&sm.k_empty[st], ((i >> 1) - 1) & 1, MOET_KV4_TRIES);
      if (!ok) break;
#pragma unroll
      for (int x = 0; x < KI; x++) {
        const int sl = x * 32 / BK, j = x * 32 % BK + kj;
        const uint32_t f16s = key_scales_f16<D>(ks[x]);
        uint8_t* dst = sm.k[st] + (j >> 3) * kKSbo + (j & 7) * 16 + (sl * (L::SD / 8) + kt * (E2 / 4)) * 128;
#pragma unroll
        for (int w = 0; w < W; w++) {
          uint32_t f[4];
          e2m1x8_to_f16(kc[x][w], f);
          *reinterpret_cast<uint4*>(dst + w * 128) = make_uint4(mul_f16x2(f[0], f16s), mul_f16x2(f[1], f16s),
                                                               mul_f16x2(f[2], f16s), mul_f16x2(f[3], f16s));
        }
      }
      tc::fence_proxy_async_smem();
      pr::arrive(&sm.k_full[st]);
#pragma unroll
      for (int x = 0; x < KP; x++) page[x] = ahead[x];
      fetch_k(kb0 + i + 1);
      look_up(kb0 + i + 2, ahead);
      if (i >= 2) ok = tc::mbar_wait(&sm.v_empty[st], ((i >> 1) - 1) & 1, MOET_KV4_TRIES);
      if (!ok) break;
      // values: a thread has 8 tokens of its piece: per value one 16-byte row of a core matrix
      uint8_t* dst = sm.v[st] + vsl * (L::SD / 8) * kVSbo + vo * 128 + vg * 16;
      constexpr int WV = W / 2;                              // words per token
      uint32_t fs[4];
#pragma unroll
      for (int x = 0; x < 4; x++) fs[x] = e4m3x2_to_f16(vs[x]);
#pragma unroll
      for (int w = 0; w < WV; w++) {
        uint32_t lo[4][4], hi[4][4];                         // [pair][value]
#pragma unroll
        for (int x = 0; x < 4; x++) {
          uint32_t c0w, c8w;
          join_pair(vc[x][w], vc[x][WV + w], c0w, c8w);
          e2m1x8_to_f16(c0w, lo[x]);
          e2m1x8_to_f16(c8w, hi[x]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int n = 4 * w + k;
          *reinterpret_cast<uint4*>(dst + n * kVSbo) = make_uint4(mul_f16x2(lo[0][k], fs[0]), mul_f16x2(lo[1][k], fs[1]),
                                                                 mul_f16x2(lo[2][k], fs[2]), mul_f16x2(lo[3][k], fs[3]));
          *reinterpret_cast<uint4*>(dst + (E2 / 2 + n) * kVSbo) = make_uint4(
              mul_f16x2(hi[0][k], fs[0]), mul_f16x2(hi[1][k], fs[1]), mul_f16x2(hi[2][k], fs[2]), mul_f16x2(hi[3][k], fs[3]));
        }
      }
      tc::fence_proxy_async_smem();
      pr::arrive(&sm.v_full[st]);
      fetch_v(kb0 + i + 1);
    }
  } else {
    // ---- products: the whole warp waits, one lane issues
    const uint32_t lead = pr::elect();
    const uint32_t id_s = pr::idesc_f16(128, C::SK), id_o = pr::idesc_f16(128, D);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q0 = tc::smem_desc(tc::smem_addr(sm.q[0]), 128, kQSbo), k0 = tc::smem_desc(tc::smem_addr(sm.k[0]), 128, kKSbo),
                   v0 = tc::smem_desc(tc::smem_addr(sm.v[0]), 128, kVSbo);
    // a descriptor moves on by its address in 16-byte steps: 256 bytes per depth of 16; a half is 64
    // rows of K (8 groups) and 8 chunks of V's depth
    auto scores = [&](int t, int n) {
      const int st = n / C::HALVES & 1, half = n % C::HALVES;
      const uint64_t qa = q0 + (uint32_t)t * (C::kQBytes >> 4);
      const uint64_t ka = k0 + (uint32_t)st * (C::kKBytes >> 4) + (uint32_t)half * (8 * kKSbo >> 4);
#pragma unroll
      for (int k = 0; k < D / 16; k++) pr::mma_ss(lead, tm + t * 128 + (n & 1) * C::SK, qa + k * 16, ka + k * 16, id_s, k > 0);
      pr::commit(lead, &sm.s_full[t][n & 1]);
      if (t == ntile - 1 && half == C::HALVES - 1) pr::commit(lead, &sm.k_empty[st]);
    };
    auto outputs = [&](int t, int n) {
      const int st = n / C::HALVES & 1, half = n % C::HALVES;
      const uint64_t va = v0 + (uint32_t)st * (C::kKBytes >> 4) + (uint32_t)half * (8 * 128 >> 4);
#pragma unroll
      for (int k = 0; k < C::SK / 16; k++)
        pr::mma_ts(lead, tm + C::kOCol + t * D, tm + t * 128 + (n & 1) * C::SK + k * 8, va + k * 16, id_o, n > 0 || k > 0);
      pr::commit(lead, &sm.pv_done[t]);
      if (n == steps - 1) pr::commit(lead, &sm.o_full[t]);
      if (t == ntile - 1 && half == C::HALVES - 1) pr::commit(lead, &sm.v_empty[st]);
    };
    if (steps > 0) {
      ok = tc::mbar_wait(&sm.k_full[0], 0, MOET_KV4_TRIES);
      tc::fence_after();
      for (int t = 0; t < ntile && ok; t++) scores(t, 0);
    }
    for (int n = 0; n < steps && ok; n++) {
      const int nx = n + 1, kb = n / C::HALVES, kx = nx / C::HALVES;
      if (nx < steps && nx % C::HALVES == 0) ok = tc::mbar_wait(&sm.k_full[kx & 1], (kx >> 1) & 1, MOET_KV4_TRIES);
      if (ok && n % C::HALVES == 0) ok = tc::mbar_wait(&sm.v_full[kb & 1], (kb >> 1) & 1, MOET_KV4_TRIES);
      for (int t = 0; t < ntile && ok; t++) {
        if (nx < steps) {                      // under this tile's softmax; its P of two steps before has been read
          if (n > 0) ok = tc::mbar_wait(&sm.pv_done[t], (n - 1) & 1, MOET_KV4_TRIES);
          if (!ok) break;
          tc::fence_after();
          scores(t, nx);
        }
        ok = tc::mbar_wait(&sm.p_full[t][n & 1], (n >> 1) & 1, MOET_KV4_P_TRIES);
        if (!ok) break;
        tc::fence_after();
        outputs(t, n);
      }
    }
    // Where a wait ran out (here or in another warp) nobody has waited for the last products: none may still read
    // shared memory or write tensor memory when the block gives them back.  With the full limit; it costs no time.
    __syncwarp();
    pr::commit(lead, &sm.done);
    if (!tc::mbar_wait(&sm.done, 0)) ok = false;
  }
  __syncwarp();
  if (!ok) set_status(a.status, kTimeout);
  tc::fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after();
    tc::tmem_relinquish();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins a tile's stretches, in their order: a thread per 8 values of a row.
template <int D, typename T16>
__global__ void __launch_bounds__(256) kv4_prompt_join_kernel(PromptArgs a) {
  constexpr int RT = PromptCfg<D>::TILES * 128;
  pdl_entry();
  const PromptTile<D> tl(a, a.whole + blockIdx.y);
  const int it = blockIdx.x * 256 + threadIdx.x, r = it / (D / 8), d = it % (D / 8) * 8;
  const int row = tl.row0 + r;
  if (tl.tile < 0 || row >= tl.rows || tl.splits == 1) return;      // one stretch: its block has written the rows
  const float* p = a.part + prompt_part<D>(a, blockIdx.y, 0);
  constexpr int PF = RT * (D + 2);
  float M = -INFINITY;
  for (int s = 0; s < tl.splits; s++) M = fmaxf(M, p[s * PF + RT * D + r]);
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll 2
  for (int s = 0; s < tl.splits; s++) {
    const float m = p[s * PF + RT * D + r], l = p[s * PF + RT * (D + 1) + r];
    if (m == -INFINITY && l == 0.f) continue;          // a stretch of which the row saw nothing
    const float w = m == -INFINITY ? 1.f : fast_exp2(m - M);   // NaN sums have no maximum
    const float4 y = *reinterpret_cast<const float4*>(p + s * PF + r * D + d), z = *reinterpret_cast<const float4*>(p + s * PF + r * D + d + 4);
    x[0] += w * y.x, x[1] += w * y.y, x[2] += w * y.z, x[3] += w * y.w;
    x[4] += w * z.x, x[5] += w * z.y, x[6] += w * z.z, x[7] += w * z.w;
    sum += w * l;
  }
  const float inv = sum > 0.f ? __fdividef(a.v_mul, sum) : sum;
  const long long at = (long long)(tl.c0 + row / a.G) * a.H * a.G + tl.h * a.G + row % a.G;
  *reinterpret_cast<uint4*>((T16*)a.out + at * D + d) =
      make_uint4(round2<T16>(x[0] * inv, x[1] * inv), round2<T16>(x[2] * inv, x[3] * inv),
                 round2<T16>(x[4] * inv, x[5] * inv), round2<T16>(x[6] * inv, x[7] * inv));
  if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : (M + (__log2f(sum) - kLift)) * 0.6931471805599453f;
}

static int64_t prompt_tiles(int64_t T, int64_t G, int64_t D, int64_t max_q) {
  const int64_t rt = D == 256 ? 128 : 256;
  return (std::min(max_q, T) * G + rt - 1) / rt;
}

}  // namespace kv4
}  // namespace moet

using namespace moet;
using namespace moet::kv4;

// {tiles taken whole, stretches of keys of each of the others, floats of `part`}.  Tiles that fill all SMs
// are taken whole.  The rest (all, where there are fewer tiles than SMs) would leave SMs idle: its keys
// are split so that the last wave is even, unless four or more waves come before it.  The number of stretches
// comes from the table's width (or the window) and is the most there can be; each tile takes as many as its own
// keys fill with kMinStretch keys or more, and the blocks of the others leave at once.
// us whole / with the rest split, 8 heads x 4 rows, warm: 2048 tokens and 16384 keys (256 tiles), D = 64: 471 / 450, D = 128:
// 551 / 542, D = 256 (512 tiles): 1190 / 1099; 1300 tokens, 8192 keys (168 tiles): 268 / 194; 1250 tokens, 32768 keys: 1112 / 674.
std::tuple<int64_t, int64_t, int64_t> kv4_prompt_plan(int64_t T, int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_q,
                                                      int64_t W, int64_t window) {
  const int64_t sms = sm_count();
  const int64_t n = prompt_tiles(T, G, D, max_q) * H * B, rest = n % sms;
  const int64_t rt = D == 256 ? 128 : 256, keys = window > 0 ? std::min(W * kPage, window + (rt + G - 1) / G) : W * kPage;
  if (rest == 0 || n >= 4 * sms) return {n, 1, 0};
  int64_t best = 1;
  if (n < sms) {
    best = std::min<int64_t>({sms / n, keys / kMinStretch, 64});
  } else {
    for (int64_t s = 2; s <= std::min<int64_t>(keys / kMinStretch, 8); s++) {       // waves of stretches / s, 3 % for a split
      const auto cost = [&](int64_t x) { return (double)((rest * x + sms - 1) / sms) / x + 0.03 * (x - 1); };
      if (cost(s) < cost(best)) best = s;
    }
  }
  if (best <= 1) return {n, 1, 0};
  return {n - rest, best, rest * best * rt * (D + 2)};
}

void kv4_prompt_launch(torch::Tensor q, torch::Tensor cu_q, torch::Tensor seq_lens, torch::Tensor table,
                       torch::Tensor pages, double scale, int64_t max_q, int64_t window, int64_t k_exp, int64_t v_exp,
                       torch::Tensor out, c10::optional<torch::Tensor> lse, int64_t whole,
                       int64_t splits, c10::optional<torch::Tensor> part, torch::Tensor status) {
  PromptArgs a;
  const int D = (int)(pages.size(2) / 72);
  a.T = (int)q.size(0); a.H = (int)pages.size(1); a.G = (int)(q.size(1) / a.H);
  a.B = (int)seq_lens.size(0); a.W = (int)table.size(1);
  a.q = q.data_ptr(); a.q_tok = q.stride(0); a.q_head = (int)q.stride(1);
  a.cu_q = (const int*)cu_q.data_ptr(); a.seq_lens = (const int*)seq_lens.data_ptr();
  a.table = (const int*)table.data_ptr(); a.max_q = (int)std::min<int64_t>(max_q, a.T); a.window = (int)window;
  a.pages = (const uint8_t*)pages.data_ptr(); a.n_pages = (int)pages.size(0);
  a.scale = score_scale(scale, (int)k_exp);
  a.v_mul = std::ldexp(1.f, (int)v_exp);
  a.out = out.data_ptr(); a.lse = (float*)opt_ptr(lse);
  a.status = (int*)status.data_ptr();
  const int64_t n = prompt_tiles(a.T, a.G, D, max_q) * a.H * a.B, rest = n - whole;
  a.whole = (int)whole; a.splits = (int)splits;
  a.part = (float*)opt_ptr(part);
  TORCH_CHECK(n < (int64_t)1 << 30 && (rest == 0 || a.part), "kv4: too much work for one call, or no workspace");
  auto stream = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto dim, auto t) {
    constexpr int DD = decltype(dim)::value;
    using T16 = decltype(t);
    using C = PromptCfg<DD>;
    const dim3 grid((unsigned)(whole + rest * splits));
    moet_allow_max_smem(kv4_prompt_kernel<DD, T16>);
    launch_k(kv4_prompt_kernel<DD, T16>, grid, dim3(C::kWarps * 32), sizeof(PromptSmem<DD>), stream, a);
    if (rest > 0)         // fewer tiles than SMs
      launch_k(kv4_prompt_join_kernel<DD, T16>, dim3(C::TILES * 128 * DD / 8 / 256, (unsigned)rest), dim3(256), 0, stream, a);
  };
  auto by_type = [&](auto dim) {
    if (q.scalar_type() == at::kHalf) go(dim, __half{});
    else go(dim, __nv_bfloat16{});
  };
  if (D == 64) by_type(std::integral_constant<int, 64>{});
  else if (D == 128) by_type(std::integral_constant<int, 128>{});
  else by_type(std::integral_constant<int, 256>{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
