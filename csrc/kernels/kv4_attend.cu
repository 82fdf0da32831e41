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
// significant bits whole down to 2^-23 of the row's maximum.  P <= 2^14 is rounded to f16 (11
// bits, three more than a bf16 output has); references, sums and outputs stay in 32 bits.  exp2,
// log2 and the division are the hardware's approximations (2^-21 or better, against P's 2^-11).
//
// What bounds it is the cache's bytes (a long context), so each warp streams its own units
// (pages) through a private ring of bulk copies, one for a page's keys and one for its
// values, with no block-wide barrier inside a tile.  Work is split evenly: the units of all
// (sequence, row tile, head) tiles lie on one line and each block takes an equal stretch of
// it.  A tile that lies within one block is finished there; of the others each block leaves
// its part (maxima, sums, unnormalised outputs), and kv4_join_kernel adds the parts up in
// block order.  A split tile is named by the block in which it begins, so the join needs no
// counters and its grid is the first one's.
//
// B200: 32 sequences with 362 k positions together, 8 heads of 128, 8 rows each: 94 us, 4.5 TB/s (68 % of the
// measured copy rate); not the bytes but the instructions of the conversion bound it there (IPC 2.2 of
// 4, ALU pipe 50 %, tensor 25 %, DRAM 55 %).  One sequence of 1000 positions: 8 us, a chain of
// schedule, page look-up, one page per warp and join.
#include "kv4.cuh"
#include "tcgen05.cuh"
#include "torch_glue.h"

namespace moet {
namespace kv4 {

constexpr int kWarps = 4;

struct AttendArgs {
  const void* q; long long q_tok; int q_head;
  const int *cu_q, *seq_lens, *table; int B, W;         // table [B, W]
  const int* sel; int budget;                           // [T, H, budget] or null
  int T, H, G, window;
  const uint8_t* pages; int n_pages;
  ScoreScale scale;
  float v_mul;                                          // 2^v_exp
  void* out; float* lse;                                // [T, H * G, D], [T, H * G] or null
  float* part; int* split;                              // parts: two per block; split: kSplitInts per block
  int min_units;
  uint32_t tries;                                       // of a wait for a copy, before it gives up
  int* status;
};
// What a block notes of the tile that begins in it and goes on past it:
// {parts (0: none), head, first row, rows, first token}
constexpr int kSplitInts = 8;

MOET_DEVICE void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
MOET_DEVICE uint32_t transpose_8x8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// two f32 operations in one instruction
MOET_DEVICE void mul2(float& x, float& y, float a, float b) {
  asm("{\n.reg .b64 u, v;\nmov.b64 u, {%0, %1};\nmov.b64 v, {%2, %3};\nmul.rn.ftz.f32x2 u, u, v;\nmov.b64 {%0, %1}, u;\n}\n"
      : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
MOET_DEVICE void sub2(float& x, float& y, float a, float b) {
  asm("{\n.reg .b64 u, v;\nmov.b64 u, {%0, %1};\nmov.b64 v, {%2, %3};\nadd.rn.ftz.f32x2 u, u, v;\nmov.b64 {%0, %1}, u;\n}\n"
      : "+f"(x), "+f"(y) : "f"(-a), "f"(-b));
}
// What a row's weights exp2(s - reference) refer to: 14 below its largest score, so that the weights use f16's range up to
// 2^14 and those of a long tail, down to 2^-28 of the largest, keep all their bits.  Scores that are too large for
// the difference to be near 14 in f32 refer to the largest itself.
MOET_DEVICE float reference(float top) { return fabsf(top) < 1048576.f ? top - 14.f : top; }
MOET_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_addr(bar)), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(tc::smem_addr(dst)), "l"(src), "r"(bytes), "r"(tc::smem_addr(bar)) : "memory");
}

// A unit of work: a page of one tile (sequence, row tile, head).
struct Unit {
  int b, h, row0, rows, tok0, p0;   // tile: rows [row0, row0 + count) of the sequence's; first token, its position
  int x, n;                         // unit index in the tile, units of the tile: kTileCost empty ones, then its pages
  int page;                         // logical page (or entry of the choice)
};

// A tile's queries, join and output take a block as long as about this many of its pages;
// counted as empty units in front of them, so that many short tiles do not all fall to one block.
// B200, 32 sequences, one of them of two positions: without it the block that got its eight one-page
// tiles ended after 120 us, the others after 87.
constexpr int kTileCost = 8;

// A unit is one page of a tile.  Its keys and its values are two copies, each into a slot of
// its own; a warp takes TS tokens per softmax step.
template <int D, int NT> struct StepCfg {
  static constexpr int kSlots = D == 256 ? 2 : 3;                    // 2304, 4608 or 9216 bytes each
  static constexpr int kRed = D == 256 || NT == 2 ? 1 : 2;                     // buffers in which the warps are joined
  static constexpr int TS = NT == 1 ? 64 : 32;                       // as the registers allow
};

constexpr int kMaxBlocks = 4;       // blocks per SM, at most
template <int D, int NT> constexpr int blocks_per_sm() { return D <= 128 && NT <= 2 ? 3 : 2; }   // by registers

template <int D, int NT> struct StepSmem {
  using C = StepCfg<D, NT>;
  static constexpr int RT = 8 * NT;
  static constexpr int kRedStride = D + 4;                           // rows 4 banks apart: stores of a quad do not meet
  uint8_t ring[kWarps][C::kSlots][Lay<D>::kHalfBytes];
  static constexpr int kQStride = D + 8;
  __align__(16) uint16_t q[RT * kQStride];                           // the next tile's queries
  float red[C::kRed][RT * kRedStride];
  float wm[kWarps][RT], wl[kWarps][RT];
  float fm[RT], fl[RT];
  uint64_t bar[kWarps][C::kSlots];
  int start[kWarps][C::kSlots];
  int scan[kWarps];
};

// start of sequence b's rows; an offset outside the rows is pulled back into them
MOET_DEVICE int row_start(const AttendArgs& a, int b) { return max(0, min(a.cu_q[b], a.T)); }

// units of sequence b with all its pages: (tiles, units per tile)
template <int D, int NT>
MOET_DEVICE void seq_units(const AttendArgs& a, int b, int& tiles, int& n, int& page0) {
  const int nq = max(0, row_start(a, b + 1) - row_start(a, b));
  const int len = held_length(a.seq_lens[b], a.W);
  tiles = (nq * a.G + 8 * NT - 1) / (8 * NT);
  page0 = a.window > 0 ? max(0, len - nq - a.window + 1) / kPage : 0;
  n = max(1, (len + kPage - 1) / kPage - page0) + kTileCost;      // an empty sequence's rows are still written
}

template <int D, int NT>
MOET_DEVICE Unit find_unit(const AttendArgs& a, const int* pre, int u) {
  constexpr int RT = 8 * NT;
  Unit r;
  if (a.sel) {
    const int nc = (a.G + RT - 1) / RT;
    r.n = a.budget + kTileCost;
    const int th = u / r.n;
    r.x = u - th * r.n;
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
    r.p0 = r.tok0 >= pre[lo] && r.tok0 < pre[lo + 1] ? held_length(a.seq_lens[lo], a.W) - pre[lo + 1] + r.tok0 : -1;   // -1: no sequence's
    r.page = r.x - kTileCost;
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
  r.p0 = held_length(a.seq_lens[lo], a.W) - nq;
  r.page = page0 + r.x - kTileCost;
  return r;
}

// where value d of a row lies in the accumulators' order [M tile][half][g]
template <int D> MOET_DEVICE int column(int d) {
  constexpr int SD = Lay<D>::SD, E = SD / 8;
  const int sl = d / SD, g = d % SD / E, half = d % E / (E / 2), i = d % (E / 2);
  return (sl * (E / 2) + i) * 16 + half * 8 + g;
}

template <int D, int NT> constexpr int part_floats() { return 8 * NT * (D + 2); }

MOET_DEVICE long long out_row(const AttendArgs& a, int h, int row, int tok0) {
  const int tok = tok0 + (a.sel ? 0 : row / a.G), head = h * a.G + (a.sel ? row : row % a.G);
  return (long long)tok * a.H * a.G + head;
}
// N neighbouring values x of an output row (unnormalised, with the row's sum)
template <typename T16, int N>
MOET_DEVICE void store_row(const AttendArgs& a, int h, int row, int tok0, int d, int D, const float (&x)[N], float sum) {
  const float inv = sum > 0.f ? __fdividef(a.v_mul, sum) : sum;      // 0: nothing was seen; NaN stays
  uint32_t w[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; k++) w[k] = round2<T16>(x[2 * k] * inv, x[2 * k + 1] * inv);
  T16* p = (T16*)a.out + out_row(a, h, row, tok0) * D + d;
  if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
MOET_DEVICE void store_lse(const AttendArgs& a, int h, int row, int tok0, float m, float sum) {
  if (a.lse) a.lse[out_row(a, h, row, tok0)] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * 0.6931471805599453f;
}

template <int D, int NT, typename T16>
__global__ void __launch_bounds__(kWarps * 32, blocks_per_sm<D, NT>()) kv4_attend_kernel(AttendArgs a) {
  using L = Lay<D>;
  using C = StepCfg<D, NT>;
  using S = StepSmem<D, NT>;
  constexpr int RT = S::RT, NSLOT = C::kSlots, TS = C::TS, MT = TS / 16, KW = D / 32;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  int* pre = reinterpret_cast<int*>(smem_raw + sizeof(S));            // [B + 1]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int i = 0; i < NSLOT; i++) tc::mbar_init(&sm.bar[warp][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // what is read first is fetched into L2 while the kernel before still runs
  grid_prefetch(a.seq_lens, a.B * 4ll);
  grid_prefetch(a.cu_q, a.B * 4ll);
  grid_prefetch(a.table, (long long)a.B * a.W * 4);
  grid_prefetch(a.q, ((long long)(a.T - 1) * a.q_tok + (a.H * a.G - 1ll) * a.q_head + D) * 2);
  pdl_entry();

  const int rows0 = a.cu_q[0], rows1 = a.cu_q[a.B];

  // the line of units: prefix sums over the sequences (all pages), or over nothing (chosen pages)
  int total;
  if (a.sel) {
    for (int i = tid; i <= a.B; i += kWarps * 32) pre[i] = row_start(a, i);
    total = a.T * a.H * ((a.G + RT - 1) / RT) * (a.budget + kTileCost);
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
  int* split = a.split + blockIdx.x * kSplitInts;
  if (tid == 0) split[0] = 0;
  if (blockIdx.x == gridDim.x - 1)       // the last block, which has the least to do
    for (int b = tid; b < a.B; b += kWarps * 32) check_sequence(a.cu_q, a.seq_lens, b, a.T, a.W, a.status);
  if (!a.sel) blank_rows(rows0, rows1, a.T, a.out, a.lse, a.H * a.G, D);     // chosen pages: such a row is a tile that sees nothing
  if (u0 >= u1) return;

  // ---- queries come by way of shared memory, a tile ahead
  auto stage_q = [&](const Unit& tl) {
    for (int e = tid; e < RT * D / 8; e += kWarps * 32) {
      const int r = e / (D / 8), d = e % (D / 8) * 8, row = tl.row0 + r;
      const bool live = row < tl.rows;
      const int tok = tl.tok0 + (a.sel || !live ? 0 : row / a.G), head = tl.h * a.G + (!live ? 0 : a.sel ? row : row % a.G);
      const T16* src = (const T16*)a.q + (long long)tok * a.q_tok + (long long)head * a.q_head + d;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"      // rows past the tile's: zeros
                   ::"r"(tc::smem_addr(&sm.q[r * S::kQStride + d])), "l"(src), "r"(live ? 16 : 0) : "memory");
    }
  };
  Unit tl = find_unit<D, NT>(a, pre, u0);
  stage_q(tl);

  // ---- this warp's units u0 + warp + 4 i through its ring
  const int mine = (u1 - u0 - warp + kWarps - 1) / kWarps;
  const uint8_t* my_src = nullptr;       // of unit (batch of 32) + lane
  int my_start = -1;
  uint32_t phase = 0;
  bool dead = false;
  int next = 0, next_slot = 0;           // the half to be issued (keys of unit next / 2, or its values) and its slot
  auto issue = [&]() {
    const int i = next >> 1;
    if (i >= mine) return;
    if ((next & 63) == 0) {              // look up the next 32 units, one per lane
      my_start = -1;
      if (i + lane < mine) {
        const Unit r = find_unit<D, NT>(a, pre, u0 + warp + kWarps * (i + lane));
        int page = r.page;
        bool bad = false;
        const int row_last = min(r.row0 + RT, r.rows) - 1;
        const int p_last = r.p0 + (a.sel ? 0 : row_last / a.G);        // the tile's last position
        const bool real = r.x >= kTileCost;
        if (a.sel && real) page = a.sel[((long long)r.tok0 * a.H + r.h) * a.budget + page];
        if (real && page >= 0 && page < a.W && page * kPage <= p_last) {
          const int phys = a.table[(long long)r.b * a.W + page];
          bad = phys < 0 || phys >= a.n_pages;
          if (!bad) {
            my_start = page * kPage;
            my_src = a.pages + ((long long)phys * a.H + r.h) * L::kPageBytes;
          }
        } else {
          bad = real && page >= a.W;
        }
        if (bad) set_status(a.status, kBadIndex);
      }
    }
    if (lane == (i & 31)) {
      sm.start[warp][next_slot] = dead ? -1 : my_start;
      if (my_start >= 0 && !dead)
        bulk_load(sm.ring[warp][next_slot], my_src + (next & 1) * L::kHalfBytes, L::kHalfBytes, &sm.bar[warp][next_slot]);
    }
    next++;
    next_slot = next_slot + 1 == NSLOT ? 0 : next_slot + 1;
    __syncwarp();
  };
#pragma unroll 1
  for (int k = 0; k < NSLOT; k++) issue();
  int slot = 0;                          // the half that comes next
  // Wait for half x (of this warp's halves, in order).  If its copy does not come in time the warp computes
  // nothing more, and waits here for what it has in flight: a copy must not outlive the block's shared memory.
  auto arrived = [&](int k, int x) {     // k: the half's slot
    if (dead) return;
    // one answer for the warp: its lanes go on to matrix instructions and shuffles, or none does
    if (__all_sync(0xffffffffu, tc::mbar_wait(&sm.bar[warp][k], (phase >> k) & 1, a.tries))) {
      phase ^= 1u << k;
      return;
    }
    set_status(a.status, kTimeout);
    dead = true;
    for (; x < next; x++)
      if (sm.start[warp][x % NSLOT] >= 0) tc::mbar_wait(&sm.bar[warp][x % NSLOT], (phase >> x % NSLOT) & 1);
    __syncwarp();
  };

  int i = 0;                             // next own unit
  for (int cur = u0; cur < u1;) {
    const int first = cur - tl.x + kTileCost, end = cur - tl.x + tl.n, seg_end = min(u1, end);   // pages: [first, end)
    if (seg_end <= first) break;                                       // the tile begins in the next block
    Unit after = tl;
    if (seg_end < u1) after = find_unit<D, NT>(a, pre, seg_end);

    // ---- queries: B fragments of rows n * 8 + g, positions of accumulator columns n * 8 + 2 t, + 1
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    uint32_t qf[NT][KW][2][2];
    float cs[NT][2];
    int pc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      float v[D / 4];                     // of each slab, piece t's values
      float amax = 0.f;
#pragma unroll
      for (int x = 0; x < D / 32; x++) {
        constexpr int PER = L::SD / 32;   // 16-byte loads per slab
        const int d = x / PER * L::SD + t * (L::SD / 4) + x % PER * 8;
        const uint4 y = *reinterpret_cast<const uint4*>(&sm.q[(n * 8 + g) * S::kQStride + d]);
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float2 f = unpack2<T16>(w[k]);
          v[8 * x + 2 * k] = f.x, v[8 * x + 2 * k + 1] = f.y;
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      float mul = 1.f;
      int e = 0;                            // queries are held times 2^-e
      if (sizeof(T16) == 2 && !std::is_same<T16, __half>::value) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        e = amax > 0.f ? max(-110, min(119, (int)(__float_as_uint(amax) >> 23) - 127 - 8)) : 0;
        mul = pow2f(-e);
      }
#pragma unroll
      for (int w = 0; w < KW; w++)
#pragma unroll
        for (int k = 0; k < 4; k++) {      // byte k of word w: a code in its low half, one in its high half
          constexpr int WS = L::SD / 32, HALF = L::SD / 8;
          const int lo = w / WS * (L::SD / 4) + w % WS * 4 + k;
          qf[n][w][k >> 1][k & 1] = pack_f16x2(v[lo] * mul, v[lo + HALF] * mul);
        }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        cs[n][c] = row_factor(a.scale, __shfl_sync(0xffffffffu, e, (2 * t + c) * 4));
        const int rc = min(tl.row0 + n * 8 + 2 * t + c, tl.rows - 1);
        pc[n][c] = tl.p0 + (a.sel ? 0 : rc / a.G);
      }
    }
    __syncthreads();
    if (seg_end < u1) stage_q(after);
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
      const int ks = slot, vs_ = ks + 1 == NSLOT ? 0 : ks + 1, start = sm.start[warp][ks];
      slot = vs_ + 1 == NSLOT ? 0 : vs_ + 1;
      if (start >= 0) arrived(ks, 2 * i);
      const uint8_t *keys = sm.ring[warp][ks], *values = sm.ring[warp][vs_];
#pragma unroll 1
      for (int st = 0; st < kPage / TS; st++) {
        const int s0 = start + st * TS;
        if (start >= 0 && !dead) {
          // S^T: tiles of 16 tokens
          float s[MT][NT][4];
#pragma unroll
          for (int mt = 0; mt < MT; mt++) {
#pragma unroll
            for (int n = 0; n < NT; n++) s[mt][n][0] = s[mt][n][1] = s[mt][n][2] = s[mt][n][3] = 0.f;
            const int j0 = st * TS + mt * 16 + g, j1 = j0 + 8;
#pragma unroll
            for (int sl = 0; sl < L::NS; sl++) {
              constexpr int W = L::SD / 32;
              uint32_t c0[W], c1[W];
              const uint8_t* kc = keys + L::KC + sl * L::kSlabBytes + t * (L::SD / 8);
              load_words<W>(kc + j0 * (L::SD / 2), c0);
              load_words<W>(kc + j1 * (L::SD / 2), c1);
              const uint32_t f0 = key_scales<D>(keys + L::KS + j0 * L::NB, sl, t);
              const uint32_t f1 = key_scales<D>(keys + L::KS + j1 * L::NB, sl, t);
#pragma unroll
              for (int w = 0; w < W; w++) {
                uint32_t x[4], y[4];
                e2m1x8_to_f16(c0[w], x);
                e2m1x8_to_f16(c1[w], y);
#pragma unroll
                for (int k = 0; k < 4; k++) x[k] = mul_f16x2(x[k], f0), y[k] = mul_f16x2(y[k], f1);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                  const uint32_t(&q)[2][2] = qf[n][sl * W + w];
                  mma_f16_16816(s[mt][n], x[0], y[0], x[1], y[1], q[0][0], q[0][1]);
                  mma_f16_16816(s[mt][n], x[2], y[2], x[3], y[3], q[1][0], q[1][1]);
                }
              }
            }
          }
          // online softmax over the step's tokens, in powers of two
          const bool edge = s0 + TS - 1 > p_first || (a.window > 0 && s0 <= p_last - a.window);
          uint32_t pf[MT][NT][2];
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
              mul2(s[mt][n][0], s[mt][n][1], cs[n][0], cs[n][1]);
              mul2(s[mt][n][2], s[mt][n][3], cs[n][0], cs[n][1]);
            }
            if (edge) {
#pragma unroll
              for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                  const int j = s0 + mt * 16 + g + (k >> 1) * 8, p = pc[n][k & 1];
                  if (j > p || (a.window > 0 && j <= p - a.window)) s[mt][n][k] = -INFINITY;
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
              for (int k = 0; k < 4; k++) mx[k & 1] = fmaxf(mx[k & 1], s[mt][n][k]);
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], off));
              mx[c] = fmaxf(m[n][c], reference(mx[c]));
            }
            const float ref0 = mx[0] == -INFINITY ? 0.f : mx[0], ref1 = mx[1] == -INFINITY ? 0.f : mx[1];
            if (__any_sync(0xffffffffu, mx[0] != m[n][0] || mx[1] != m[n][1])) {
              const float a0 = fast_exp2(m[n][0] - ref0), a1 = fast_exp2(m[n][1] - ref1);
              l[n][0] *= a0, l[n][1] *= a1;
#pragma unroll
              for (int d = 0; d < D / 16; d++) mul2(o[d][n][0], o[d][n][1], a0, a1), mul2(o[d][n][2], o[d][n][3], a0, a1);
              m[n][0] = mx[0], m[n][1] = mx[1];
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
              float (&p)[4] = s[mt][n];
              sub2(p[0], p[1], ref0, ref1);
              sub2(p[2], p[3], ref0, ref1);
#pragma unroll
              for (int k = 0; k < 4; k++) p[k] = fast_exp2(p[k]);
              l[n][0] += p[0] + p[2], l[n][1] += p[1] + p[3];
              pf[mt][n][0] = transpose_8x8(pack_f16x2(p[0], p[1]));
              pf[mt][n][1] = transpose_8x8(pack_f16x2(p[2], p[3]));
            }
          }
          if (st == kPage / TS - 1) {
            __syncwarp();           // every lane has read the keys
            issue();
          }
          if (st == 0) arrived(vs_, 2 * i + 1);
          // O^T += V^T P^T
#pragma unroll
          for (int mt = 0; mt < MT; mt++) {
            const int pa = st * (TS / 2) + mt * 8 + t, pb = pa + 4;                 // token pairs 2 pa, 2 pa + 1 and 2 pb, 2 pb + 1
            uint32_t keep_a = 0xFFFFFFFFu, keep_b = 0xFFFFFFFFu;
            if (edge) {      // what lies past the rows may be anything: its scales (NaN, maybe) are put to 0
              keep_a = (start + 2 * pa <= p_last ? 0xFFFFu : 0u) | (start + 2 * pa + 1 <= p_last ? 0xFFFF0000u : 0u);
              keep_b = (start + 2 * pb <= p_last ? 0xFFFFu : 0u) | (start + 2 * pb + 1 <= p_last ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int sl = 0; sl < L::NS; sl++) {
              constexpr int PB = L::SD / 16, W = PB / 4;            // bytes and words per token and piece
              uint32_t xa[2 * W], xb[2 * W];                        // the pair's first token, then its second
              const uint8_t* vc = values + sl * L::kSlabBytes + g * (2 * PB);
              load_words<2 * W>(vc + pa * (16 * PB), xa);
              load_words<2 * W>(vc + pb * (16 * PB), xb);
              const uint8_t* vs = values + (L::VS - L::VC);
              const uint32_t fa = value_scales<D>(vs + pa * (2 * L::NB), sl, g) & keep_a;
              const uint32_t fb = value_scales<D>(vs + pb * (2 * L::NB), sl, g) & keep_b;
#pragma unroll
              for (int w = 0; w < W; w++) {
                uint32_t ca, ca8, cb, cb8, va[4], va8[4], vb[4], vb8[4];
                join_pair(xa[w], xa[W + w], ca, ca8);
                join_pair(xb[w], xb[W + w], cb, cb8);
                e2m1x8_to_f16(ca, va);
                e2m1x8_to_f16(ca8, va8);
                e2m1x8_to_f16(cb, vb);
                e2m1x8_to_f16(cb8, vb8);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                  const uint32_t f0 = mul_f16x2(va[k], fa), f1 = mul_f16x2(va8[k], fa);
                  const uint32_t f2 = mul_f16x2(vb[k], fb), f3 = mul_f16x2(vb8[k], fb);
#pragma unroll
                  for (int n = 0; n < NT; n++)
                    mma_f16_16816(o[sl * PB + 4 * w + k][n], f0, f1, f2, f3, pf[mt][n][0], pf[mt][n][1]);
                }
              }
            }
          }
        } else if (st == kPage / TS - 1) {
          __syncwarp();             // every lane has read the slot's start, which the next unit overwrites
          issue();
        }
      }
      __syncwarp();                 // every lane has read the values
      issue();
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
#pragma unroll
    for (int round = 0; round < kWarps / C::kRed; round++) {
      if (warp / C::kRed == round) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int d = 0; d < D / 16; d++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
              float* p = &sm.red[warp % C::kRed][(n * 8 + 2 * t + (k & 1)) * S::kRedStride + d * 16 + (k >> 1) * 8 + g];
              const float x = o[d][n][k] * f[n][k & 1];
              *p = round ? *p + x : x;
            }
      }
      __syncthreads();
    }

    // ---- a whole tile is finished here; of a shared one the block leaves its part
    if (first >= u0 && seg_end == end) {
      for (int e = tid; e < RT * D / 8; e += kWarps * 32) {
        const int r = e / (D / 8), d = e % (D / 8) * 8;
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int c = column<D>(d + k);
          x[k] = sm.red[0][r * S::kRedStride + c];
          if (C::kRed == 2) x[k] += sm.red[C::kRed - 1][r * S::kRedStride + c];
        }
        if (tl.row0 + r < tl.rows) store_row<T16, 8>(a, tl.h, tl.row0 + r, tl.tok0, d, D, x, sm.fl[r]);
      }
      if (tid < RT && tl.row0 + tid < tl.rows) store_lse(a, tl.h, tl.row0 + tid, tl.tok0, sm.fm[tid], sm.fl[tid]);
    } else {
      float* pt = a.part + ((long long)blockIdx.x * 2 + (first >= u0 ? 1 : 0)) * part_floats<D, NT>();
      for (int e = tid; e < RT * D / 4; e += kWarps * 32) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int c = column<D>(d + k);
          x[k] = sm.red[0][r * S::kRedStride + c];
          if (C::kRed == 2) x[k] += sm.red[C::kRed - 1][r * S::kRedStride + c];
        }
        *reinterpret_cast<float4*>(pt + r * D + d) = make_float4(x[0], x[1], x[2], x[3]);
      }
      if (tid < RT) {
        pt[RT * D + tid] = sm.fm[tid];
        pt[RT * D + RT + tid] = sm.fl[tid];
      }
      if (tid == 0 && first >= u0) {          // it begins here: the join of block blockIdx.x
        split[0] = (end - 1) / per - (int)blockIdx.x + 1;
        split[1] = tl.h, split[2] = tl.row0, split[3] = tl.rows, split[4] = tl.tok0;
      }
    }
    __syncthreads();
    cur = seg_end;
    tl = after;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Joins the tile that begins in block blockIdx.x and goes on: 32 columns per block, the parts
// shared out over groups of threads.
template <int D, int NT, typename T16>
__global__ void __launch_bounds__(256) kv4_join_kernel(AttendArgs a) {
  constexpr int RT = 8 * NT, ITEMS = RT * 8, GROUPS = 256 / ITEMS, PF = part_floats<D, NT>();
  __shared__ float fm[RT], fl[RT];
  __shared__ float4 sum[GROUPS][ITEMS];
  pdl_entry();
  const int c0 = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int* split = a.split + c0 * kSplitInts;
  const int parts = split[0];
  if (parts == 0) return;
  const int h = split[1], row0 = split[2], rows = split[3], tok0 = split[4];
  // part p: the tail of block c0's stretch, then the head of each next block's
  auto at = [&](int p) { return a.part + ((long long)(c0 + p) * 2 + (p == 0 ? 1 : 0)) * PF; };
  for (int r = warp; r < RT; r += 8) {
    float M = -INFINITY, l = 0.f;
    for (int p = lane; p < parts; p += 32) {
      const float* x = at(p) + RT * D + r;
      const float m = __ldcg(x), s = __ldcg(x + RT), hi = fmaxf(M, m);
      if (hi != -INFINITY) l = l * fast_exp2(M - hi) + s * fast_exp2(m - hi);
      else l += s;                              // 0, or NaN from a row that has one
      M = hi;
    }
    const float top = warp_max(M);
    l = warp_sum(l * (top == -INFINITY ? 1.f : fast_exp2(M - top)));
    if (lane == 0) fm[r] = top, fl[r] = l;
  }
  __syncthreads();
  const int it = tid % ITEMS, grp = tid / ITEMS, r = it / 8, d = blockIdx.y * 32 + it % 8 * 4;
  const float ref = fm[r] == -INFINITY ? 0.f : fm[r];
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int p = grp; p < parts && grp < GROUPS; p += GROUPS) {     // 24 rows leave the last 64 threads over
    const float w = fast_exp2(__ldcg(at(p) + RT * D + r) - ref);
    const float4 y = __ldcg(reinterpret_cast<const float4*>(at(p) + r * D + d));
    x.x += w * y.x, x.y += w * y.y, x.z += w * y.z, x.w += w * y.w;
  }
  if (grp < GROUPS) sum[grp][it] = x;
  __syncthreads();
  if (grp || row0 + r >= rows) return;
#pragma unroll
  for (int k = 1; k < GROUPS; k++) {
    const float4 y = sum[k][it];
    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
  }
  const float v[4] = {x.x, x.y, x.z, x.w};
  store_row<T16, 4>(a, h, row0 + r, tok0, d, D, v, fl[r]);
  if (blockIdx.y == 0 && it % 8 == 0) store_lse(a, h, row0 + r, tok0, fm[r], fl[r]);
}

// query rows of a tile / 8: the fewest that hold a sequence's rows, as the registers allow.  B200, 8 sequences
// of 30000, 8 heads of 128, 24 rows: 209 us in two tiles of 16, which convert every page twice, 124 in one of 24.
static int row_tiles(int64_t rows, int D) {
  return rows <= 8 ? 1 : (rows <= 16 || D == 256) ? 2 : rows <= 24 ? 3 : 4;
}

}  // namespace kv4
}  // namespace moet

using namespace moet;
using namespace moet::kv4;

// floats of `part` and ints of `split` that kv4_attend needs (their contents do not matter)
std::tuple<int64_t, int64_t> kv4_attend_workspace(int64_t G, int64_t D, int64_t max_q, bool chosen) {
  const int64_t rt = 8 * row_tiles(chosen ? G : max_q * G, (int)D), blocks = (int64_t)sm_count() * kMaxBlocks;
  return {blocks * 2 * rt * (D + 2), blocks * kSplitInts};
}

void kv4_attend_launch(torch::Tensor q, torch::Tensor cu_q, torch::Tensor seq_lens, torch::Tensor table,
                       torch::Tensor pages, c10::optional<torch::Tensor> sel, double scale, int64_t max_q,
                       int64_t window, int64_t k_exp, int64_t v_exp, torch::Tensor out,
                       c10::optional<torch::Tensor> lse, torch::Tensor part, torch::Tensor split, int64_t tries,
                       torch::Tensor status) {
  const int T = (int)q.size(0), H = (int)pages.size(1), D = (int)(pages.size(2) / 72), G = (int)(q.size(1) / H);
  const int B = (int)seq_lens.size(0), W = (int)table.size(1);
  const bool chosen = sel.has_value() && sel->defined();
  const int nt = row_tiles(chosen ? G : max_q * G, D);
  AttendArgs a;
  a.q = q.data_ptr(); a.q_tok = q.stride(0); a.q_head = (int)q.stride(1);
  a.cu_q = (const int*)cu_q.data_ptr(); a.seq_lens = (const int*)seq_lens.data_ptr();
  a.table = (const int*)table.data_ptr(); a.B = B; a.W = W;
  a.sel = chosen ? (const int*)sel->data_ptr() : nullptr;
  a.budget = chosen ? (int)sel->size(2) : 0;
  a.T = T; a.H = H; a.G = G; a.window = (int)window;
  a.pages = (const uint8_t*)pages.data_ptr(); a.n_pages = (int)pages.size(0);
  a.scale = score_scale(scale, (int)k_exp);
  a.v_mul = std::ldexp(1.f, (int)v_exp);
  a.out = out.data_ptr(); a.lse = (float*)opt_ptr(lse);
  a.part = (float*)part.data_ptr(); a.split = (int*)split.data_ptr();
  a.min_units = kWarps;
  a.tries = (uint32_t)tries;
  a.status = (int*)status.data_ptr();
  // the unit line is counted in 32 bits
  const int64_t line = chosen ? (int64_t)T * H * ((G + 8 * nt - 1) / (8 * nt)) * (a.budget + kTileCost)
                              : ((int64_t)T * G / (8 * nt) + B) * H * (W + kTileCost);
  TORCH_CHECK(line < (int64_t)1 << 31, "kv4: too much work for one call");
  auto stream = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto dim, auto n, auto t) {
    constexpr int DD = decltype(dim)::value, NT = decltype(n)::value;
    using T16 = decltype(t);
    const size_t smem = sizeof(StepSmem<DD, NT>) + (B + 1) * sizeof(int);
    const int blocks = std::max(1, std::min(blocks_per_sm<DD, NT>(), (int)(227 * 1024 / (smem + 1024))));
    moet_allow_max_smem(kv4_attend_kernel<DD, NT, T16>);
    launch_k(kv4_attend_kernel<DD, NT, T16>, dim3(sm_count() * blocks), dim3(kWarps * 32), smem, stream, a);
    launch_k(kv4_join_kernel<DD, NT, T16>, dim3(sm_count() * blocks, DD / 32), dim3(256), 0, stream, a);
  };
  auto by_type = [&](auto dim, auto n) {
    if (q.scalar_type() == at::kHalf) go(dim, n, __half{});
    else go(dim, n, __nv_bfloat16{});
  };
  auto by_rows = [&](auto dim) {
    constexpr int DD = decltype(dim)::value;
    if (nt == 1) by_type(dim, std::integral_constant<int, 1>{});
    else if (nt == 2) by_type(dim, std::integral_constant<int, 2>{});
    else if constexpr (DD != 256) {
      if (nt == 3) by_type(dim, std::integral_constant<int, 3>{});
      else by_type(dim, std::integral_constant<int, 4>{});
    }
  };
  if (D == 64) by_rows(std::integral_constant<int, 64>{});
  else if (D == 128) by_rows(std::integral_constant<int, 128>{});
  else by_rows(std::integral_constant<int, 256>{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
