// Choosing the pages that a query attends to, per token and K/V head.
//
// The score of a page estimates the largest product of the head's query rows with the page's
// keys, from the page bounds that kv4_cache.cu keeps (hi, lo in units e):
//   score = max over the head's rows of f e sum_d (max(r_d, 0) hi_d + min(r_d, 0) lo_d),
// r = round(q / f), f the smallest power of two with max |q| <= 127 f.  It is an upper bound for
// the rounded query f r; a product of q itself lies at most f / 2 sum_d max |k_d| above it (with
// pages of equal keys and D = 128, 6 random queries in 100 do).  The scale is taken as positive.
// The sum is an integer below 2^24 (D <= 256 products of 7-bit numbers), f and e are powers of two:
// the score is exact in f32 whatever the order of the additions (queries between 2^-90 and 2^100),
// so every rank and every replay of a step makes the same choice.  Ties go to the lowest page.
//
// Two launches.  Scores: the sum over d is one int8 matrix product of depth 2 D, [r+ | r-] by
// [hi | lo]; a warp holds 16 pages' bounds as A fragments (16-byte loads, straight from
// memory: each byte is used by one block per token tile) and walks over the rows' B fragments
// in shared memory.  Bound by the bounds' bytes (2 D per page and head) in a decode step, by
// the int8 product in a prompt chunk.  Choice: a warp (long rows: a block) per (token, head) finds
// the threshold over the ordered bits and writes the pages in order.
//
// B200, 8 heads of 128: 1024 tokens x 8 rows over 512 pages, scores 68 us (252 int8 TOP/s: the per-token
// maximum, in 32-bit integers and floats, costs as much issue as the products); 32 tokens x 8 rows over
// 1.1 M positions, scores 14 us (its 35 MB of bounds are 2.5 TB/s: three dependent loads, then one wave).
#include "kv4.cuh"
#include "torch_glue.h"

#include <type_traits>

namespace moet {
namespace kv4 {

struct SelectArgs {
  const void* q; long long q_tok; int q_head;
  const int *cu_q, *seq_lens, *table; int B, W, T, H, G, max_q;
  int gp, tpc;                        // rows reserved per token (a power of two or a multiple of 8), tokens per block
  int tiles, chunks, span;            // token tiles per sequence; chunks of 128 pages, in spans of so many per block
  const int8_t* bounds; const float* unit; int n_pages;
  float* score; int first, last, budget;
  int* pages;
  int* status;
};

constexpr int kScoreWarps = 8, kScoreRows = 64;     // rows per block: 8 n-tiles

MOET_DEVICE void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// first row and row count of a sequence, the position of its first row
MOET_DEVICE void seq_rows(const SelectArgs& a, int b, int& c0, int& nq, int& p0) {
  c0 = max(0, min(a.cu_q[b], a.T));
  nq = max(0, max(0, min(a.cu_q[b + 1], a.T)) - c0);
  p0 = held_length(a.seq_lens[b], a.W) - nq;
}
// pages of a row at position p that compete for a place: [first, n - last), n = p / 64 + 1
MOET_DEVICE int rivals_end(const SelectArgs& a, int p) { return p < 0 ? 0 : p / kPage + 1 - a.last; }

// d as a float without the conversion pipe: |d| <= 256 * 127^2 < 2^22
MOET_DEVICE float small_int(int d) { return __int_as_float(0x4B400000 + d) - 12582912.f; }

// GP: rows reserved per token, 1, 2, 4 or 8; 16 stands for a multiple of 8 (a.gp).
template <int D, int GP, typename T16>
__global__ void __launch_bounds__(kScoreWarps * 32) kv4_score_kernel(SelectArgs a) {
  constexpr int KB = 2 * D, STRIDE = KB + 64;       // rows 64 bytes apart in the banks: 16-byte reads do not meet
  constexpr int CH = KB / 64;                       // 16-byte pieces of a lane per page
  constexpr int kChunk = kScoreWarps * 16;
  __shared__ __align__(16) int8_t rows[kScoreRows * STRIDE];
  __shared__ float unit_q[kScoreRows];
  grid_prefetch(a.seq_lens, a.B * 4ll);
  grid_prefetch(a.cu_q, a.B * 4ll);
  grid_prefetch(a.table, (long long)a.B * a.W * 4);
  grid_prefetch(a.q, ((long long)(a.T - 1) * a.q_tok + (a.H * a.G - 1ll) * a.q_head + D) * 2);
  pdl_entry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int spans = (a.chunks + a.span - 1) / a.span;
  const int h = blockIdx.y, chunk0 = blockIdx.x % spans * a.span, bt = blockIdx.x / spans;
  const int b = bt / a.tiles, tile = bt % a.tiles;
  int c0, nq, p0;
  seq_rows(a, b, c0, nq, p0);
  const int i0 = tile * a.tpc, ntok = min(a.tpc, min(nq, a.max_q) - i0);
  if (ntok <= 0) return;
  const int end = rivals_end(a, p0 + i0 + ntok - 1);       // the last token's
  if (chunk0 * kChunk >= end) return;
  if (p0 + i0 + ntok - 1 < a.budget * kPage) return;       // every token takes all its pages

  // 16 pages per warp and chunk; the first ones come while the rows are converted
  uint4 x[2][CH];
  float u[2];
  int phys[2];
  auto look_up = [&](int pg) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int page = pg + g + 8 * i;
      phys[i] = page < end ? a.table[(long long)b * a.W + page] : 0;      // end <= W
    }
  };
  auto row_of = [&](int i) {
    if (phys[i] < 0 || phys[i] >= a.n_pages) {
      set_status(a.status, kBadIndex);
      phys[i] = 0;
    }
    return ((long long)phys[i] * a.H + h) * KB;
  };
  auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int8_t* p = a.bounds + row_of(i) + t * 16;
#pragma unroll
      for (int c = 0; c < CH; c++) x[i][c] = *reinterpret_cast<const uint4*>(p + c * 64);
      u[i] = a.unit[(long long)phys[i] * a.H + h];
    }
  };
  look_up(chunk0 * kChunk + warp * 16);
  fetch();
  const bool more = a.span > 1;
  if (more) look_up((chunk0 + 1) * kChunk + warp * 16);

  // ---- rows: r = round(q / f) as [max(r, 0) | min(r, 0)]; a place without a row repeats the token's first
  const int gp = GP == 16 ? a.gp : GP, nrows = ntok * gp;
  constexpr int E = D / 32;                                // values per lane
  for (int r = warp; r < ((nrows + 7) & ~7); r += kScoreWarps) {
    const int ti = min(r / gp, ntok - 1), gi = r % gp < a.G ? r % gp : 0;
    float v[E], amax = 0.f;
    T16 raw[E];
    const T16* p = (const T16*)a.q + (long long)(c0 + i0 + ti) * a.q_tok + (long long)(h * a.G + gi) * a.q_head + lane * E;
    if constexpr (E == 8) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (E == 4) *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    else *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int e = 0; e < E; e++) {
      float y = to_f32(raw[e]);
      y = y != y ? 0.f : fminf(fmaxf(y, -3.4028235e38f), 3.4028235e38f);
      v[e] = y;
      amax = fmaxf(amax, fabsf(y));
    }
    amax = warp_max(amax);
    const int ex = exp_for_127(amax);
    const float inv = pow2f(-ex);
    int8_t pos[E], neg[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int y = __float2int_rn(v[e] * inv);
      pos[e] = (int8_t)max(y, 0);
      neg[e] = (int8_t)min(y, 0);
    }
    using Word = std::conditional_t<E == 8, uint2, std::conditional_t<E == 4, uint32_t, uint16_t>>;
    *reinterpret_cast<Word*>(rows + r * STRIDE + lane * E) = *reinterpret_cast<const Word*>(pos);
    *reinterpret_cast<Word*>(rows + r * STRIDE + D + lane * E) = *reinterpret_cast<const Word*>(neg);
    if (lane == 0) unit_q[r] = pow2f(ex);
  }
  __syncthreads();

  const int wide = gp / 8;                                 // n-tiles of one token, GP = 16
  const int ntiles = (nrows + 7) / 8, chunk1 = min(chunk0 + a.span, a.chunks);
  const long long tstep = (long long)a.H * a.W;
  for (int chunk = chunk0; chunk < chunk1; chunk++) {
    const int pg = chunk * kChunk + warp * 16;
    if (pg >= end) return;
    if (chunk > chunk0) {
      fetch();
      if (chunk + 1 < chunk1) look_up(pg + kChunk);
    }
    if (chunk + 1 < chunk1) {                              // the next chunk's bounds on their way to L2
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int8_t* p = a.bounds + row_of(i);
        if (t * 128 < KB) prefetch_l2(p + t * 128);
      }
    }
    const bool in0 = pg + g < end, in1 = pg + g + 8 < end;
    float* out = a.score + ((long long)(c0 + i0) * a.H + h) * a.W + pg + g;     // + token * H * W
    float best0 = -INFINITY, best1 = -INFINITY;
    int left = wide, ti = GP == 1 ? 2 * t : GP == 2 ? t : GP == 4 ? t >> 1 : 0;   // this lane's token in the n-tile
    out += ti * tstep;
    for (int n = 0; n < ntiles; n++) {
      int d[4] = {0, 0, 0, 0};
      const int8_t* rp = rows + (n * 8 + g) * STRIDE + t * 16;
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const uint4 y = *reinterpret_cast<const uint4*>(rp + c * 64);
        mma_s8_16832(d, x[0][c].x, x[1][c].x, x[0][c].y, x[1][c].y, y.x, y.y);
        mma_s8_16832(d, x[0][c].z, x[1][c].z, x[0][c].w, x[1][c].w, y.z, y.w);
      }
      const float2 f = *reinterpret_cast<const float2*>(&unit_q[n * 8 + 2 * t]);
      // (page g, row 2t), (g, 2t+1), (g + 8, 2t), (g + 8, 2t + 1); the page's unit is positive and comes last
      float m0 = small_int(d[0]) * f.x, m1 = small_int(d[2]) * f.x;
      const float s0 = small_int(d[1]) * f.y, s1 = small_int(d[3]) * f.y;
      if constexpr (GP == 1) {
        if (ti < ntok) {
          if (in0) out[0] = m0 * u[0];
          if (in1) out[8] = m1 * u[1];
        }
        if (ti + 1 < ntok) {
          if (in0) out[tstep] = s0 * u[0];
          if (in1) out[tstep + 8] = s1 * u[1];
        }
        ti += 8, out += 8 * tstep;
        continue;
      }
      m0 = fmaxf(m0, s0), m1 = fmaxf(m1, s1);
      if constexpr (GP >= 4) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
      }
      if constexpr (GP >= 8) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
      }
      if constexpr (GP == 16) {
        m0 = best0 = fmaxf(best0, m0);
        m1 = best1 = fmaxf(best1, m1);
        if (--left > 0) continue;                          // the token goes on in the next n-tile
        left = wide, best0 = best1 = -INFINITY;
      }
      const bool mine = ti < ntok && (GP == 2 || (GP == 4 ? (t & 1) == 0 : t == 0));
      if (mine && in0) out[0] = m0 * u[0];
      if (mine && in1) out[8] = m1 * u[1];
      constexpr int kTok = GP == 2 ? 4 : GP == 4 ? 2 : 1;   // tokens of an n-tile
      ti += kTok, out += kTok * tstep;
    }
  }
}

MOET_DEVICE uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f == 0.f ? 0.f : f);  // -0 and 0 are one score
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// The row's sequence, first row, position and pages; the choice when all pages fit, and the pages that are always taken.
struct Pick {
  int n, end, want;         // pages; rivals are [first, end), `want` of them are taken (more than that: n > budget)
  int* out;
};
MOET_DEVICE void check_batch(const SelectArgs& a) {      // by the last block
  if (blockIdx.x == gridDim.x - 1)
    for (int b = threadIdx.x; b < a.B; b += blockDim.x) check_sequence(a.cu_q, a.seq_lens, b, a.T, a.W, a.status);
}
MOET_DEVICE Pick pick_row(const SelectArgs& a, int tok, int h, int tid, int threads) {
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (max(0, min(a.cu_q[mid], a.T)) <= tok) lo = mid; else hi = mid;
  }
  int c0, nq, p0;
  seq_rows(a, lo, c0, nq, p0);
  const int p = tok >= c0 && tok - c0 < nq ? p0 + tok - c0 : -1;       // -1: no sequence's
  Pick r;
  r.n = p < 0 ? 0 : p / kPage + 1;
  r.out = a.pages + ((long long)tok * a.H + h) * a.budget;
  r.end = r.n - a.last;
  r.want = 0;
  if (r.n <= a.budget) {
    for (int i = tid; i < a.budget; i += threads) r.out[i] = i < r.n ? i : -1;
    return r;
  }
  if (tok - c0 >= a.max_q) {         // its scores were not computed
    for (int i = tid; i < a.budget; i += threads) r.out[i] = -1;
    if (tid == 0) set_status(a.status, kBadSize);
    return r;
  }
  r.want = a.budget - a.first - a.last;
  for (int i = tid; i < a.first; i += threads) r.out[i] = i;
  for (int i = tid; i < a.last; i += threads) r.out[a.budget - a.last + i] = r.end + i;
  return r;
}

// A warp per (token, head), its keys in registers: up to 32 K pages.  The threshold is found bit by
// bit from the highest bit in which the keys differ, and stops as soon as just `want` keys reach it.
// Bound by the chain of votes (a step per bit over the warp's keys).
template <int K>
__global__ void __launch_bounds__(128) kv4_pick_warp_kernel(SelectArgs a) {
  pdl_entry();
  check_batch(a);
  const int lane = threadIdx.x & 31;
  const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (id >= (long long)a.T * a.H) return;
  const int tok = (int)(id / a.H), h = (int)(id % a.H);
  const Pick r = pick_row(a, tok, h, lane, 32);
  if (r.want == 0) return;
  const float* row = a.score + id * a.W;
  uint32_t key[K], top = 0, low = 0xFFFFFFFFu;
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int i = a.first + 32 * k + lane;
    key[k] = i < r.end ? order_bits(__ldg(row + i)) : 0;       // 0 lies below every score
    if (i < r.end) top = max(top, key[k]), low = min(low, key[k]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  uint32_t t = top;
  int above = -1;                                              // keys >= t, once that is known to be `want`
  if (top != low) {
    int bit = 31 - __clz(top ^ low);
    t = top >> bit >> 1 << bit << 1;                           // the bits they share
    for (; bit >= 0; bit--) {
      const uint32_t cand = t | 1u << bit;
      int n = 0;
#pragma unroll
      for (int k = 0; k < K; k++) n += key[k] >= cand;
      n = __reduce_add_sync(0xffffffffu, n);
      if (n >= r.want) t = cand;
      if (n == r.want) {
        above = n;
        break;
      }
    }
  }
  int ties = 0;                                                // places for keys that equal t
  if (above < 0) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < K; k++) n += key[k] > t;
    ties = r.want - __reduce_add_sync(0xffffffffu, n);
  }
  int at = a.first;
  const uint32_t below = (1u << lane) - 1;
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int i = a.first + 32 * k + lane;
    bool take = i < r.end && (above >= 0 ? key[k] >= t : key[k] > t);
    if (ties > 0) {
      const bool eq = i < r.end && key[k] == t;
      const uint32_t be = __ballot_sync(0xffffffffu, eq);
      take |= eq && __popc(be & below) < ties;
      ties -= min(ties, __popc(be));
    }
    const uint32_t b = __ballot_sync(0xffffffffu, take);
    if (take) r.out[at + __popc(b & below)] = i;
    at += __popc(b);
  }
}

constexpr int kPickThreads = 128;

// A block per (token, head) for longer rows, or few of them: four passes of a radix search over the row in memory, which L2
// holds.  8 tokens x 8 heads over 2048 pages: 6 us (B200), the passes one after the other.
__global__ void __launch_bounds__(kPickThreads) kv4_pick_kernel(SelectArgs a) {
  pdl_entry();
  check_batch(a);
  __shared__ uint32_t hist[256];
  __shared__ int scan[kPickThreads / 32][2];
  __shared__ uint32_t prefix_s;
  __shared__ int remain_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tok = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const Pick r = pick_row(a, tok, h, tid, kPickThreads);
  const int end = r.end, want = r.want;
  int* out = r.out;
  if (want == 0) return;
  const float* row = a.score + ((long long)tok * a.H + h) * a.W;
  uint32_t prefix = 0, mask = 0;
  int remain = want;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kPickThreads) hist[i] = 0;
    __syncthreads();
    for (int i = a.first + tid; i < end; i += kPickThreads) {
      const uint32_t k = order_bits(row[i]);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (warp == 0) {       // the bin, from the top, in which the count reaches `remain`
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) c[i] = hist[255 - (lane * 8 + i)], sum += c[i];
      uint32_t before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      before -= sum;
      if ((int)before < remain && (int)(before + sum) >= remain) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if ((int)before < remain && (int)(before + c[i]) >= remain) {
            prefix_s = prefix | (uint32_t)(255 - (lane * 8 + i)) << shift;
            remain_s = remain - (int)before;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    prefix = prefix_s;
    remain = remain_s;
    mask |= 255u << shift;
  }
  // take what is above the threshold, and the first `remain` that equal it, in page order
  int above = 0, equal = 0;                                // taken so far
  for (int i0 = a.first; i0 < end; i0 += kPickThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < end ? order_bits(row[i]) : 0;
    const bool gt = i < end && k > prefix, eq = i < end && k == prefix;
    const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) scan[warp][0] = __popc(bg), scan[warp][1] = __popc(be);
    __syncthreads();
    int ng = above, ne = equal;
    for (int w = 0; w < warp; w++) ng += scan[w][0], ne += scan[w][1];
    for (int w = 0; w < kPickThreads / 32; w++) above += scan[w][0], equal += scan[w][1];
    const uint32_t below = (1u << lane) - 1;
    ng += __popc(bg & below), ne += __popc(be & below);
    if (gt || (eq && ne < remain)) out[a.first + ng + min(ne, remain)] = i;
    __syncthreads();
  }
}

}  // namespace kv4
}  // namespace moet

using namespace moet;
using namespace moet::kv4;

void kv4_select_launch(torch::Tensor q, torch::Tensor cu_q, torch::Tensor seq_lens, torch::Tensor table,
                       torch::Tensor bounds, torch::Tensor unit, int64_t max_q, int64_t first, int64_t last,
                       torch::Tensor score, torch::Tensor pages, torch::Tensor status) {
  SelectArgs a;
  const int D = (int)q.size(2);
  a.T = (int)q.size(0); a.H = (int)bounds.size(1); a.G = (int)(q.size(1) / a.H);
  a.B = (int)seq_lens.size(0); a.W = (int)table.size(1);
  a.q = q.data_ptr(); a.q_tok = q.stride(0); a.q_head = (int)q.stride(1);
  a.cu_q = (const int*)cu_q.data_ptr(); a.seq_lens = (const int*)seq_lens.data_ptr();
  a.table = (const int*)table.data_ptr();
  a.bounds = (const int8_t*)bounds.data_ptr(); a.unit = (const float*)unit.data_ptr(); a.n_pages = (int)bounds.size(0);
  a.score = (float*)score.data_ptr(); a.first = (int)first; a.last = (int)last; a.budget = (int)pages.size(2);
  a.pages = (int*)pages.data_ptr();
  a.status = (int*)status.data_ptr();
  a.gp = 1;
  while (a.gp < a.G && a.gp < 8) a.gp *= 2;
  if (a.G > 8) a.gp = (a.G + 7) / 8 * 8;
  a.tpc = kScoreRows / a.gp;
  a.max_q = (int)std::min<int64_t>(max_q, a.T);
  a.tiles = (a.max_q + a.tpc - 1) / a.tpc;
  a.chunks = (a.W + kScoreWarps * 16 - 1) / (kScoreWarps * 16);
  // As many chunks per block as leave four blocks per SM: a block converts its rows once per span.  us with
  // 2 / 4 / 8 per SM, cold, choice included: 32 tokens over 1.1 M positions 36 / 34 / 36, 1024 tokens over
  // 512 pages 89 / 89 / 99.
  const int64_t per_chunk = (int64_t)a.B * a.tiles * a.H;
  a.span = (int)std::max<int64_t>(1, std::min<int64_t>(a.chunks, per_chunk * a.chunks / (4 * sm_count())));
  const int64_t blocks = (int64_t)a.B * a.tiles * ((a.chunks + a.span - 1) / a.span);
  TORCH_CHECK(blocks < (int64_t)1 << 31 && (int64_t)a.T * a.H < (int64_t)1 << 31, "kv4: too much work for one call");
  auto stream = at::cuda::getCurrentCUDAStream();
  const dim3 grid((unsigned)blocks, a.H), block(kScoreWarps * 32);
  auto launch = [&](auto dim, auto gp, auto t) {
    launch_k(kv4_score_kernel<decltype(dim)::value, decltype(gp)::value, decltype(t)>, grid, block, 0, stream, a);
  };
  auto by_type = [&](auto dim, auto gp) {
    if (q.scalar_type() == at::kHalf) launch(dim, gp, __half{});
    else launch(dim, gp, __nv_bfloat16{});
  };
  auto go = [&](auto dim) {
    if (a.gp == 1) by_type(dim, std::integral_constant<int, 1>{});
    else if (a.gp == 2) by_type(dim, std::integral_constant<int, 2>{});
    else if (a.gp == 4) by_type(dim, std::integral_constant<int, 4>{});
    else if (a.gp == 8) by_type(dim, std::integral_constant<int, 8>{});
    else by_type(dim, std::integral_constant<int, 16>{});
  };
  if (a.W > a.budget) {               // else every token takes all its pages
    if (D == 64) go(std::integral_constant<int, 64>{});
    else if (D == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
  }
  const dim3 warps((unsigned)(((int64_t)a.T * a.H + 3) / 4)), four(128);
  // A warp per row, except for more than 512 pages (32 keys a lane) with fewer than two rows per SM, where the
  // latency of one row counts.  us of a whole choice, warp / block, 8 heads, back to back on B200: 32 tokens, 400
  // pages 18.9 / 19.5, 700 pages 26.1 / 22.0; 64 tokens, 700 pages 36.6 / 37.6; 512 tokens, 1000 pages 156 / 165.
  const bool few = a.W > 512 && (int64_t)a.T * a.H < 2 * sm_count();
  if (a.W <= 256) launch_k(kv4_pick_warp_kernel<8>, warps, four, 0, stream, a);
  else if (a.W <= 512) launch_k(kv4_pick_warp_kernel<16>, warps, four, 0, stream, a);
  else if (a.W <= 1024 && !few) launch_k(kv4_pick_warp_kernel<32>, warps, four, 0, stream, a);
  else launch_k(kv4_pick_kernel, dim3((unsigned)((int64_t)a.T * a.H)), dim3(kPickThreads), 0, stream, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
