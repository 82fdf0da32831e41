// Attention of a few query rows per sequence over the 4-bit paged K/V cache (layout: kv4.cuh):
// decode tokens, verify rows, and tokens that have chosen their pages.
//
//   out = softmax(scale q k^T) v over positions j <= p (j > p - window), p the row's position.
//
// Transposed products keep the small side small: S^T = K Q^T takes 16 tokens as the M side of
// m16n8k16 and 8 query rows as the N side, O^T = V^T P^T 16 values and 8 rows, so a head group
// of up to 8 rows pads nothing.  Keys and values are converted in registers (e2m1 -> f16, times
// the block's e4m3 scale: exact, kv4.cuh) straight into the A fragments; P goes from the
// accumulator layout to a B fragment by one 8x8 transpose per tile.  Queries are held as f16:
// bf16 rows are scaled by a power of two to at most 512 first, which leaves their 8
// significant bits whole down to 2^-23 of the row's maximum.  P <= 1 is rounded to f16 (11
// bits, three more than a bf16 output has); maxima, sums and outputs stay in 32 bits.
//
// What bounds it is the cache's bytes (a long context), so each warp streams its own units
// (64 positions; 32 with D = 256) through a private ring of bulk copies, one contiguous copy
// per unit, with no block-wide barrier inside a tile.  Work is split evenly: the units of all
// (sequence, row tile, head) tiles lie on one line, each block takes an equal stretch of it,
// and a tile that several blocks share is joined by the last of them to arrive, in block
// order (the order of arrival changes nothing in the result).
#include "kv4.cuh"
#include "tcgen05.cuh"
#include "torch_glue.h"

namespace moet {
namespace kv4 {

constexpr int kWarps = 4;
constexpr int kMaxSeqs = 4096;

struct AttendArgs {
  const void* q; long long q_tok; int q_head;
  const int *cu_q, *seq_lens, *table; int B, W;         // table [B, W]
  const int* sel; int budget;                           // [T, H, budget] or null
  int T, H, G, window;
  const uint8_t* pages; int n_pages;
  float scale_log2;                                     // scale * log2(e) * 2^k_exp
  float v_mul;                                          // 2^v_exp
  void* out; float* lse;                                // [T, H * G, D], [T, H * G] or null
  float* part; int* counters;
  int min_units;
  int* status;
};

MOET_DEVICE void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
MOET_DEVICE uint32_t transpose_8x8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
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
MOET_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_addr(bar)), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(tc::smem_addr(dst)), "l"(src), "r"(bytes), "r"(tc::smem_addr(bar)) : "memory");
}
template <typename T16> MOET_DEVICE float2 unpack2(uint32_t v);
template <> MOET_DEVICE float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <> MOET_DEVICE float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
template <typename T16> MOET_DEVICE uint32_t round2(float a, float b);
template <> MOET_DEVICE uint32_t round2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <> MOET_DEVICE uint32_t round2<__half>(float a, float b) { return pack_f16x2(a, b); }

// A unit of work: 64 (or 32) positions of one tile (sequence, row tile, head).
struct Unit {
  int b, h, row0, rows, tok0, p0;   // tile: rows [row0, row0 + count) of the sequence's; first token, its position
  int x, n;                         // unit index in the tile, units of the tile
  int page, tile;                   // logical page (or entry of the choice), counter of the tile
};

template <int D> struct StepCfg {
  static constexpr int UT = D == 256 ? 32 : 64;                      // positions of a unit
  static constexpr int PU = kPage / UT;
  static constexpr int kUnitBytes = UT / kSub * Lay<D>::kSubBytes;   // 4608, 9216, 9216
  static constexpr int kStages = D == 64 ? 4 : 2;
};

constexpr int kMaxBlocks = 3;       // blocks per SM, at most

template <int D, int NT> struct StepSmem {
  using C = StepCfg<D>;
  static constexpr int RT = 8 * NT;
  static constexpr int kRedStride = D + 4;                           // rows 4 banks apart: stores of a quad do not meet
  uint8_t ring[kWarps][C::kStages][C::kUnitBytes];
  float red[RT * kRedStride];
  float wm[kWarps][RT], wl[kWarps][RT];
  float fm[RT], fl[RT];
  uint64_t bar[kWarps][C::kStages];
  int start[kWarps][C::kStages];
  int scan[kWarps];
  int last;
};

// start of sequence b's rows; an offset outside the rows is pulled back into them
MOET_DEVICE int row_start(const AttendArgs& a, int b) { return max(0, min(a.cu_q[b], a.T)); }

// units of sequence b with all its pages: (tiles, units per tile)
template <int D, int NT>
MOET_DEVICE void seq_units(const AttendArgs& a, int b, int& tiles, int& n, int& page0) {
  const int nq = max(0, row_start(a, b + 1) - row_start(a, b));
  const int len = max(0, min(a.seq_lens[b], a.W * kPage));
  tiles = (nq * a.G + 8 * NT - 1) / (8 * NT);
  page0 = a.window > 0 ? max(0, len - nq - a.window + 1) / kPage : 0;
  n = max(1, (len + kPage - 1) / kPage - page0) * StepCfg<D>::PU;    // an empty sequence's rows are still written
}

template <int D, int NT>
MOET_DEVICE Unit find_unit(const AttendArgs& a, const int* pre, int u) {
  constexpr int RT = 8 * NT, PU = StepCfg<D>::PU;
  Unit r;
  if (a.sel) {
    const int nc = (a.G + RT - 1) / RT;
    r.n = a.budget * PU;
    const int th = u / r.n;
    r.x = u - th * r.n;
    r.tile = th;
    const int chunk = th % nc;
    r.h = (th / nc) % a.H;
    r.tok0 = th / (nc * a.H);
    int lo = 0, hi = a.B;                       // last b with cu_q[b] <= tok0
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (pre[m] <= r.tok0) lo = m; else hi = m;
    }
    r.b = lo;
    r.row0 = chunk * RT;
    r.rows = a.G;
    r.p0 = r.tok0 < pre[lo + 1] ? min(a.seq_lens[lo], a.W * kPage) - pre[lo + 1] + r.tok0 : -1;   // -1: no sequence's
    r.page = r.x / PU;
    return r;
  }
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= u) lo = m; else hi = m;
  }
  int tiles, page0;
  seq_units<D, NT>(a, lo, tiles, r.n, page0);
  const int rem = u - pre[lo], th = rem / r.n;
  r.b = lo;
  r.x = rem - th * r.n;
  r.h = th % a.H;
  const int tile = th / a.H, c0 = row_start(a, lo), nq = row_start(a, lo + 1) - c0;
  r.row0 = tile * RT;
  r.rows = nq * a.G;
  r.tok0 = c0;
  r.p0 = min(a.seq_lens[lo], a.W * kPage) - nq;
  r.page = page0 + r.x / PU;
  r.tile = ((int)((long long)c0 * a.G / RT) + lo + tile) * a.H + r.h;
  return r;
}

template <int D, int NT, typename T16>
__global__ void __launch_bounds__(kWarps * 32, 2) kv4_attend_kernel(AttendArgs a) {
  using L = Lay<D>;
  using C = StepCfg<D>;
  using S = StepSmem<D, NT>;
  constexpr int RT = S::RT, NSTG = C::kStages, KW = D / 32;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  int* pre = reinterpret_cast<int*>(smem_raw + sizeof(S));            // [B + 1]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int i = 0; i < NSTG; i++) tc::mbar_init(&sm.bar[warp][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_entry();

  // the line of units: prefix sums over the sequences (all pages), or over nothing (chosen pages)
  int total;
  if (a.sel) {
    for (int i = tid; i <= a.B; i += kWarps * 32) pre[i] = row_start(a, i);
    total = a.T * a.H * ((a.G + RT - 1) / RT) * a.budget * C::PU;
  } else {
    int run = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWarps * 32) {
      const int b = b0 + tid;
      int mine = 0;
      if (b < a.B) {
        int tiles, n, page0;
        seq_units<D, NT>(a, b, tiles, n, page0);
        mine = tiles * a.H * n;
      }
      int x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) sm.scan[warp] = x;
      __syncthreads();
      int before = run;
      for (int w = 0; w < warp; w++) before += sm.scan[w];
      if (b < a.B) pre[b] = before + x - mine;
      for (int w = 0; w < kWarps; w++) run += sm.scan[w];
      __syncthreads();
    }
    if (tid == 0) pre[a.B] = run;
    total = run;
  }
  __syncthreads();
  const int per = max((int)(((long long)total + gridDim.x - 1) / gridDim.x), a.min_units);
  const int u0 = (int)min((long long)blockIdx.x * per, (long long)total), u1 = min(u0 + per, total);
  if (u0 >= u1) return;

  // ---- this warp's units u0 + warp + 4 i through its ring
  const int mine = (u1 - u0 - warp + kWarps - 1) / kWarps;
  const uint8_t* my_src = nullptr;       // of unit (batch of 32) + lane
  int my_start = -1;
  uint32_t phase = 0;
  bool dead = false;
  auto issue = [&](int i) {
    if (i >= mine) return;
    if ((i & 31) == 0) {                 // look up the next 32 units, one per lane
      my_start = -1;
      if (i + lane < mine) {
        const Unit r = find_unit<D, NT>(a, pre, u0 + warp + kWarps * (i + lane));
        int page = r.page;
        bool bad = false;
        const int row_last = min(r.row0 + RT, r.rows) - 1;
        const int p_last = r.p0 + (a.sel ? 0 : row_last / a.G);        // the tile's last position
        if (a.sel) page = a.sel[((long long)r.tok0 * a.H + r.h) * a.budget + page];
        const int st = page * kPage + (r.x % C::PU) * C::UT;
        if (page >= 0 && page < a.W && st <= p_last) {
          const int phys = a.table[(long long)r.b * a.W + page];
          bad = phys < 0 || phys >= a.n_pages;
          if (!bad) {
            my_start = st;
            my_src = a.pages + ((long long)phys * a.H + r.h) * L::kPageBytes + (r.x % C::PU) * C::kUnitBytes;
          }
        } else {
          bad = page >= a.W;
        }
        if (bad) set_status(a.status, kBadIndex);
      }
    }
    const int st = i % NSTG;
    if (lane == (i & 31)) {
      sm.start[warp][st] = dead ? -1 : my_start;
      if (my_start >= 0 && !dead) bulk_load(sm.ring[warp][st], my_src, C::kUnitBytes, &sm.bar[warp][st]);
    }
    __syncwarp();
  };
#pragma unroll 1
  for (int i = 0; i < NSTG; i++) issue(i);

  int i = 0;                             // next own unit
  for (int cur = u0; cur < u1;) {
    const Unit tl = find_unit<D, NT>(a, pre, cur);
    const int first = cur - tl.x, seg_end = min(u1, first + tl.n);     // tile = [first, first + n)

    // ---- queries: B fragments of rows n * 8 + g, positions of accumulator columns n * 8 + 2 t, + 1
    uint32_t qf[NT][KW][2][2];
    float cs[NT][2];
    int pc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int r = tl.row0 + n * 8 + g;
      const bool live = r < tl.rows;
      const int tok = tl.tok0 + (a.sel ? 0 : r / a.G), head = tl.h * a.G + (a.sel ? r : r % a.G);
      const T16* qp = (const T16*)a.q + (long long)(live ? tok : 0) * a.q_tok + (long long)(live ? head : 0) * a.q_head;
      float v[KW][8];
      float amax = 0.f;
#pragma unroll
      for (int w = 0; w < KW; w++) {
        // 8-byte loads: the host checks that rows start on 8 bytes
        const uint2 lo = live ? *reinterpret_cast<const uint2*>(qp + 32 * w + 4 * t) : make_uint2(0, 0);
        const uint2 hi = live ? *reinterpret_cast<const uint2*>(qp + 32 * w + 16 + 4 * t) : make_uint2(0, 0);
        const float2 a0 = unpack2<T16>(lo.x), a1 = unpack2<T16>(lo.y), b0 = unpack2<T16>(hi.x), b1 = unpack2<T16>(hi.y);
        v[w][0] = a0.x, v[w][1] = a0.y, v[w][2] = a1.x, v[w][3] = a1.y;
        v[w][4] = b0.x, v[w][5] = b0.y, v[w][6] = b1.x, v[w][7] = b1.y;
#pragma unroll
        for (int k = 0; k < 8; k++) amax = fmaxf(amax, fabsf(v[w][k]));
      }
      float mul = 1.f, back = 1.f;
      if (sizeof(T16) == 2 && !std::is_same<T16, __half>::value) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e = amax > 0.f ? max(-110, min(110, (int)(__float_as_uint(amax) >> 23) - 127 - 8)) : 0;
        mul = pow2f(-e), back = pow2f(e);
      }
#pragma unroll
      for (int w = 0; w < KW; w++) {
        qf[n][w][0][0] = pack_f16x2(v[w][0] * mul, v[w][4] * mul);
        qf[n][w][0][1] = pack_f16x2(v[w][1] * mul, v[w][5] * mul);
        qf[n][w][1][0] = pack_f16x2(v[w][2] * mul, v[w][6] * mul);
        qf[n][w][1][1] = pack_f16x2(v[w][3] * mul, v[w][7] * mul);
      }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        cs[n][c] = __shfl_sync(0xffffffffu, back, (2 * t + c) * 4) * a.scale_log2;
        const int rc = min(tl.row0 + n * 8 + 2 * t + c, tl.rows - 1);
        pc[n][c] = tl.p0 + (a.sel ? 0 : rc / a.G);
      }
    }
    const int row_last = min(tl.row0 + RT, tl.rows) - 1;
    const int p_first = tl.p0 + (a.sel ? 0 : tl.row0 / a.G), p_last = tl.p0 + (a.sel ? 0 : row_last / a.G);

    float o[D / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; d++) o[d][n][0] = o[d][n][1] = o[d][n][2] = o[d][n][3] = 0.f;
    }

    for (; u0 + warp + kWarps * i < seg_end; i++) {
      const int st = i % NSTG, start = sm.start[warp][st];
      if (start >= 0 && !dead) {
        if (!tc::mbar_wait(&sm.bar[warp][st], (phase >> st) & 1)) {
          set_status(a.status, kTimeout);
          dead = true;
        }
        phase ^= 1u << st;
      }
      if (start >= 0 && !dead) {
#pragma unroll 1
        for (int sb = 0; sb < C::UT / kSub; sb++) {
          const uint8_t* sub = sm.ring[warp][st] + sb * L::kSubBytes;
          const int s0 = start + sb * kSub;
          // S^T: two tiles of 16 tokens
          float s[2][NT][4];
#pragma unroll
          for (int mt = 0; mt < 2; mt++) {
#pragma unroll
            for (int n = 0; n < NT; n++) s[mt][n][0] = s[mt][n][1] = s[mt][n][2] = s[mt][n][3] = 0.f;
            const int j0 = mt * 16 + g, j1 = j0 + 8;
#pragma unroll
            for (int sl = 0; sl < L::NS; sl++) {
              constexpr int W = L::SD / 32;
              uint32_t c0[W], c1[W], f0[W], f1[W];
              const uint8_t* kc = sub + L::KC + sl * (kSub * L::SD / 2) + t * (L::SD / 8);
              const uint8_t* ks = sub + L::KS + sl * (L::SD / 16);
              if (W == 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(kc + j0 * (L::SD / 2));
                const uint4 y = *reinterpret_cast<const uint4*>(kc + j1 * (L::SD / 2));
                c0[0] = x.x, c0[1] = x.y, c0[W - 2] = x.z, c0[W - 1] = x.w;
                c1[0] = y.x, c1[1] = y.y, c1[W - 2] = y.z, c1[W - 1] = y.w;
                const uint2 p = *reinterpret_cast<const uint2*>(ks + j0 * L::NB);
                const uint2 q = *reinterpret_cast<const uint2*>(ks + j1 * L::NB);
                e4m3x4_to_f16(p.x, f0[0], f0[1]);
                e4m3x4_to_f16(p.y, f0[W - 2], f0[W - 1]);
                e4m3x4_to_f16(q.x, f1[0], f1[1]);
                e4m3x4_to_f16(q.y, f1[W - 2], f1[W - 1]);
              } else {
                const uint2 x = *reinterpret_cast<const uint2*>(kc + j0 * (L::SD / 2));
                const uint2 y = *reinterpret_cast<const uint2*>(kc + j1 * (L::SD / 2));
                c0[0] = x.x, c0[1] = x.y, c1[0] = y.x, c1[1] = y.y;
                e4m3x4_to_f16(*reinterpret_cast<const uint32_t*>(ks + j0 * L::NB), f0[0], f0[1]);
                e4m3x4_to_f16(*reinterpret_cast<const uint32_t*>(ks + j1 * L::NB), f1[0], f1[1]);
              }
#pragma unroll
              for (int w = 0; w < W; w++) {
                uint32_t x[4], y[4];
                e2m1x8_to_f16(c0[w], x);
                e2m1x8_to_f16(c1[w], y);
#pragma unroll
                for (int k = 0; k < 4; k++) x[k] = mul_f16x2(x[k], f0[w]), y[k] = mul_f16x2(y[k], f1[w]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                  const uint32_t(&q)[2][2] = qf[n][sl * W + w];
                  mma_f16_16816(s[mt][n], x[0], y[0], x[1], y[1], q[0][0], q[0][1]);
                  mma_f16_16816(s[mt][n], x[2], y[2], x[3], y[3], q[1][0], q[1][1]);
                }
              }
            }
          }
          // online softmax over the 32 tokens, in powers of two
          const bool edge = s0 + kSub - 1 > p_first || (a.window > 0 && s0 <= p_last - a.window);
          uint32_t pf[2][NT][2];
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float mx[2] = {m[n][0], m[n][1]};
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
              for (int k = 0; k < 4; k++) {
                float x = s[mt][n][k] * cs[n][k & 1];
                if (edge) {
                  const int j = s0 + mt * 16 + g + (k >> 1) * 8, p = pc[n][k & 1];
                  if (j > p || (a.window > 0 && j <= p - a.window)) x = -INFINITY;
                }
                s[mt][n][k] = x;
                mx[k & 1] = fmaxf(mx[k & 1], x);
              }
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], off));
            }
            const float ref0 = mx[0] == -INFINITY ? 0.f : mx[0], ref1 = mx[1] == -INFINITY ? 0.f : mx[1];
            if (__any_sync(0xffffffffu, mx[0] != m[n][0] || mx[1] != m[n][1])) {
              const float a0 = fast_exp2(m[n][0] - ref0), a1 = fast_exp2(m[n][1] - ref1);
              l[n][0] *= a0, l[n][1] *= a1;
#pragma unroll
              for (int d = 0; d < D / 16; d++) o[d][n][0] *= a0, o[d][n][1] *= a1, o[d][n][2] *= a0, o[d][n][3] *= a1;
              m[n][0] = mx[0], m[n][1] = mx[1];
            }
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
              float p[4];
#pragma unroll
              for (int k = 0; k < 4; k++) p[k] = fast_exp2(s[mt][n][k] - ((k & 1) ? ref1 : ref0));
              l[n][0] += p[0] + p[2], l[n][1] += p[1] + p[3];
              pf[mt][n][0] = transpose_8x8(pack_f16x2(p[0], p[1]));
              pf[mt][n][1] = transpose_8x8(pack_f16x2(p[2], p[3]));
            }
          }
          // O^T += V^T P^T
#pragma unroll
          for (int mt = 0; mt < 2; mt++) {
            const int pa = mt * 8 + t, pb = pa + 4;                 // token pairs 2 pa, 2 pa + 1 and 2 pb, 2 pb + 1
            uint32_t keep_a = 0xFFFFFFFFu, keep_b = 0xFFFFFFFFu;
            if (edge) {      // what lies past the rows may be anything: its scales (NaN, maybe) are put to 0
              keep_a = (s0 + 2 * pa <= p_last ? 0xFFFFu : 0u) | (s0 + 2 * pa + 1 <= p_last ? 0xFFFF0000u : 0u);
              keep_b = (s0 + 2 * pb <= p_last ? 0xFFFFu : 0u) | (s0 + 2 * pb + 1 <= p_last ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int sl = 0; sl < L::NS; sl++) {
              constexpr int PB = L::SD / 16, W = PB / 4;            // words per token and piece
              uint32_t xa[2][W], xb[2][W], sa[PB], sb2[PB];
              const uint8_t* vc = sub + L::VC + sl * (kSub * L::SD / 2) + g * (2 * PB);
              const uint8_t* vs = sub + L::VS + sl * (2 * PB);
              if (W == 2) {
                const uint4 x = *reinterpret_cast<const uint4*>(vc + pa * (16 * PB));
                const uint4 y = *reinterpret_cast<const uint4*>(vc + pb * (16 * PB));
                xa[0][0] = x.x, xa[0][W - 1] = x.y, xa[1][0] = x.z, xa[1][W - 1] = x.w;
                xb[0][0] = y.x, xb[0][W - 1] = y.y, xb[1][0] = y.z, xb[1][W - 1] = y.w;
                const uint4 p = *reinterpret_cast<const uint4*>(vs + pa * (2 * L::NB));
                const uint4 q = *reinterpret_cast<const uint4*>(vs + pb * (2 * L::NB));
                e4m3x4_to_f16(p.x, sa[0], sa[1]);
                e4m3x4_to_f16(p.y, sa[2], sa[3]);
                e4m3x4_to_f16(p.z, sa[PB - 4], sa[PB - 3]);
                e4m3x4_to_f16(p.w, sa[PB - 2], sa[PB - 1]);
                e4m3x4_to_f16(q.x, sb2[0], sb2[1]);
                e4m3x4_to_f16(q.y, sb2[2], sb2[3]);
                e4m3x4_to_f16(q.z, sb2[PB - 4], sb2[PB - 3]);
                e4m3x4_to_f16(q.w, sb2[PB - 2], sb2[PB - 1]);
              } else {
                const uint2 x = *reinterpret_cast<const uint2*>(vc + pa * (16 * PB));
                const uint2 y = *reinterpret_cast<const uint2*>(vc + pb * (16 * PB));
                xa[0][0] = x.x, xa[1][0] = x.y, xb[0][0] = y.x, xb[1][0] = y.y;
                const uint2 p = *reinterpret_cast<const uint2*>(vs + pa * (2 * L::NB));
                const uint2 q = *reinterpret_cast<const uint2*>(vs + pb * (2 * L::NB));
                e4m3x4_to_f16(p.x, sa[0], sa[1]);
                e4m3x4_to_f16(p.y, sa[2], sa[3]);
                e4m3x4_to_f16(q.x, sb2[0], sb2[1]);
                e4m3x4_to_f16(q.y, sb2[2], sb2[3]);
              }
              if (edge) {
#pragma unroll
                for (int k = 0; k < PB; k++) sa[k] &= keep_a, sb2[k] &= keep_b;
              }
#pragma unroll
              for (int w = 0; w < W; w++) {
                uint32_t ca, ca8, cb, cb8, va[4], va8[4], vb[4], vb8[4];
                join_pair(xa[0][w], xa[1][w], ca, ca8);
                join_pair(xb[0][w], xb[1][w], cb, cb8);
                e2m1x8_to_f16(ca, va);
                e2m1x8_to_f16(ca8, va8);
                e2m1x8_to_f16(cb, vb);
                e2m1x8_to_f16(cb8, vb8);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                  const int blk = 4 * w + k;
                  const uint32_t f0 = mul_f16x2(va[k], sa[blk]), f1 = mul_f16x2(va8[k], sa[blk]);
                  const uint32_t f2 = mul_f16x2(vb[k], sb2[blk]), f3 = mul_f16x2(vb8[k], sb2[blk]);
#pragma unroll
                  for (int n = 0; n < NT; n++)
                    mma_f16_16816(o[sl * PB + blk][n], f0, f1, f2, f3, pf[mt][n][0], pf[mt][n][1]);
                }
              }
            }
          }
        }
      }
      __syncwarp();                 // every lane has read the stage
      issue(i + NSTG);
    }

    // ---- join the four warps, in warp order
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
        if (g == 0) {
          sm.wm[warp][n * 8 + 2 * t + c] = m[n][c];
          sm.wl[warp][n * 8 + 2 * t + c] = l[n][c];
        }
      }
    __syncthreads();
    float f[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int r = n * 8 + 2 * t + c;
        float M = -INFINITY, sum = 0.f;
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, sm.wm[w][r]);
        const float ref = M == -INFINITY ? 0.f : M;
        for (int w = 0; w < kWarps; w++) sum += sm.wl[w][r] * fast_exp2(sm.wm[w][r] - ref);
        f[n][c] = fast_exp2(m[n][c] - ref);
        if (warp == 0 && g == 0) sm.fm[r] = M, sm.fl[r] = sum;
      }
    for (int w = 0; w < kWarps; w++) {
      if (warp == w) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int d = 0; d < D / 16; d++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
              float* p = &sm.red[(n * 8 + 2 * t + (k & 1)) * S::kRedStride + d * 16 + g + (k >> 1) * 8];
              const float x = o[d][n][k] * f[n][k & 1];
              *p = w ? *p + x : x;
            }
      }
      __syncthreads();
    }

    // ---- a whole tile is finished here; a shared one by the last block that arrives
    bool final = seg_end - cur == tl.n;
    constexpr int kPart = RT * (D + 2);
    if (!final) {
      float* pt = a.part + ((long long)blockIdx.x * 2 + (first >= u0 ? 1 : 0)) * kPart;
      for (int e = tid; e < RT * D / 4; e += kWarps * 32) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        __stcg(reinterpret_cast<float4*>(pt + r * D + d), *reinterpret_cast<const float4*>(&sm.red[r * S::kRedStride + d]));
      }
      if (tid < RT) {
        __stcg(pt + RT * D + tid, sm.fm[tid]);
        __stcg(pt + RT * D + RT + tid, sm.fl[tid]);
      }
      __threadfence();
      __syncthreads();
      const int c0 = first / per, c1 = (first + tl.n - 1) / per;
      if (tid == 0) {
        const int was = atomicAdd(&a.counters[tl.tile], 1);
        sm.last = was == c1 - c0;
        if (sm.last) a.counters[tl.tile] = 0;
      }
      __syncthreads();
      if (sm.last) {
        __threadfence();
        auto at = [&](int c) { return a.part + ((long long)c * 2 + (first >= c * per ? 1 : 0)) * kPart; };
        if (tid < RT) {
          float M = -INFINITY, sum = 0.f;
          for (int c = c0; c <= c1; c++) M = fmaxf(M, __ldcg(at(c) + RT * D + tid));
          const float ref = M == -INFINITY ? 0.f : M;
          for (int c = c0; c <= c1; c++)
            sum += __ldcg(at(c) + RT * D + RT + tid) * fast_exp2(__ldcg(at(c) + RT * D + tid) - ref);
          sm.fm[tid] = M;
          sm.fl[tid] = sum;
        }
        __syncthreads();
        for (int e = tid; e < RT * D / 4; e += kWarps * 32) {
          const int r = e / (D / 4), d = e % (D / 4) * 4;
          const float ref = sm.fm[r] == -INFINITY ? 0.f : sm.fm[r];
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int c = c0; c <= c1; c++) {
            const float* p = at(c);
            const float w = fast_exp2(__ldcg(p + RT * D + r) - ref);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(p + r * D + d));
            sum.x += w * x.x, sum.y += w * x.y, sum.z += w * x.z, sum.w += w * x.w;
          }
          *reinterpret_cast<float4*>(&sm.red[r * S::kRedStride + d]) = sum;
        }
        __syncthreads();
        final = true;
      }
    }
    if (final) {
      for (int e = tid; e < RT * D / 8; e += kWarps * 32) {
        const int r = e / (D / 8), d = e % (D / 8) * 8, row = tl.row0 + r;
        if (row < tl.rows) {
          const int tok = tl.tok0 + (a.sel ? 0 : row / a.G), head = tl.h * a.G + (a.sel ? row : row % a.G);
          const float inv = sm.fl[r] > 0.f ? __fdividef(a.v_mul, sm.fl[r]) : (sm.fl[r] == 0.f ? 0.f : sm.fl[r]);
          const float* x = &sm.red[r * S::kRedStride + d];
          *reinterpret_cast<uint4*>((T16*)a.out + ((long long)tok * a.H * a.G + head) * D + d) =
              make_uint4(round2<T16>(x[0] * inv, x[1] * inv), round2<T16>(x[2] * inv, x[3] * inv),
                         round2<T16>(x[4] * inv, x[5] * inv), round2<T16>(x[6] * inv, x[7] * inv));
        }
      }
      if (a.lse && tid < RT && tl.row0 + tid < tl.rows) {
        const int row = tl.row0 + tid;
        const int tok = tl.tok0 + (a.sel ? 0 : row / a.G), head = tl.h * a.G + (a.sel ? row : row % a.G);
        a.lse[(long long)tok * a.H * a.G + head] =
            sm.fl[tid] == 0.f ? -INFINITY : (sm.fm[tid] + __log2f(sm.fl[tid])) * 0.6931471805599453f;
      }
    }
    __syncthreads();
    cur = seg_end;
  }
  if (dead) {        // copies that are still in flight must not outlive the block's shared memory
    for (int k = 0; k < NSTG; k++) tc::mbar_wait(&sm.bar[warp][k], (phase >> k) & 1);
  }
}

static int sm_count() {
  static int n = [] {
    int dev = 0, v = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    return v > 0 ? v : 148;
  }();
  return n;
}

// query rows of a tile / 8: the fewest that hold a sequence's rows, as the registers allow
static int row_tiles(int64_t rows, int D) { return rows <= 8 ? 1 : (rows <= 16 || D == 256) ? 2 : 4; }

}  // namespace kv4
}  // namespace moet

using namespace moet;
using namespace moet::kv4;

// (floats of `part`, ints of `counters`) that kv4_attend needs; counters start as zeros and are
// left as zeros.
std::tuple<int64_t, int64_t> kv4_attend_workspace(int64_t T, int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_q,
                                                  bool chosen) {
  const int64_t rt = 8 * row_tiles(chosen ? G : max_q * G, (int)D);
  const int64_t tiles = chosen ? T * H * ((G + rt - 1) / rt) : (T * G / rt + B + 1) * H;
  return {(int64_t)sm_count() * kMaxBlocks * 2 * rt * (D + 2), tiles};
}

void kv4_attend(torch::Tensor q, torch::Tensor cu_q, torch::Tensor seq_lens, torch::Tensor table, torch::Tensor pages,
                c10::optional<torch::Tensor> sel, double scale, int64_t max_q, int64_t window, int64_t k_exp,
                int64_t v_exp, torch::Tensor out, c10::optional<torch::Tensor> lse, torch::Tensor part,
                torch::Tensor counters, torch::Tensor status) {
  const int T = (int)q.size(0), H = (int)pages.size(1), D = (int)(pages.size(2) / 72), G = (int)(q.size(1) / H);
  const int B = (int)seq_lens.size(0), W = (int)table.size(1);
  const bool chosen = sel.has_value() && sel->defined();
  TORCH_CHECK(B <= kMaxSeqs, "kv4_attend: at most ", kMaxSeqs, " sequences, got ", B);
  const int nt = row_tiles(chosen ? G : max_q * G, D);
  AttendArgs a;
  a.q = q.data_ptr(); a.q_tok = q.stride(0); a.q_head = (int)q.stride(1);
  a.cu_q = (const int*)cu_q.data_ptr(); a.seq_lens = (const int*)seq_lens.data_ptr();
  a.table = (const int*)table.data_ptr(); a.B = B; a.W = W;
  a.sel = chosen ? (const int*)sel->data_ptr() : nullptr;
  a.budget = chosen ? (int)sel->size(2) : 0;
  a.T = T; a.H = H; a.G = G; a.window = (int)window;
  a.pages = (const uint8_t*)pages.data_ptr(); a.n_pages = (int)pages.size(0);
  a.scale_log2 = (float)(scale * 1.4426950408889634 * std::ldexp(1.0, (int)k_exp));
  a.v_mul = std::ldexp(1.f, (int)v_exp);
  a.out = out.data_ptr(); a.lse = (float*)opt_ptr(lse);
  a.part = (float*)part.data_ptr(); a.counters = (int*)counters.data_ptr();
  a.min_units = kWarps;
  a.status = (int*)status.data_ptr();
  if (T == 0 || B == 0) return;
  // the unit line is counted in 32 bits
  const int64_t line = chosen ? (int64_t)T * H * ((G + 8 * nt - 1) / (8 * nt)) * a.budget * 2
                              : ((int64_t)T * G / (8 * nt) + B) * H * W * 2;
  TORCH_CHECK(line < (int64_t)1 << 31, "kv4_attend: too much work for one call (", line, " units)");
  auto stream = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto dim, auto n, auto t) {
    constexpr int DD = decltype(dim)::value, NT = decltype(n)::value;
    using T16 = decltype(t);
    const size_t smem = sizeof(StepSmem<DD, NT>) + (B + 1) * sizeof(int);
    const int blocks = std::max(1, std::min(2, (int)(227 * 1024 / (smem + 1024))));
    moet_allow_max_smem(kv4_attend_kernel<DD, NT, T16>);
    launch_k(kv4_attend_kernel<DD, NT, T16>, dim3(sm_count() * blocks), dim3(kWarps * 32), smem, stream, a);
  };
  auto by_type = [&](auto dim, auto n) {
    if (q.scalar_type() == at::kHalf) go(dim, n, __half{});
    else go(dim, n, __nv_bfloat16{});
  };
  auto by_rows = [&](auto dim) {
    constexpr int DD = decltype(dim)::value;
    if (nt == 1) by_type(dim, std::integral_constant<int, 1>{});
    else if (nt == 2) by_type(dim, std::integral_constant<int, 2>{});
    else if constexpr (DD != 256) by_type(dim, std::integral_constant<int, 4>{});
  };
  if (D == 64) by_rows(std::integral_constant<int, 64>{});
  else if (D == 128) by_rows(std::integral_constant<int, 128>{});
  else by_rows(std::integral_constant<int, 256>{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
