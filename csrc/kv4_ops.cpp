// Entry points of the 4-bit paged K/V cache (vllm_moet_b200/ops/kv4.py): argument checks, outputs
// and workspaces; the launches are in csrc/kernels/kv4_*.cu.
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <string>

using at::Tensor;
using c10::optional;

void kv4_append_launch(Tensor k, Tensor v, Tensor slots, Tensor pages, Tensor bounds, Tensor unit, int64_t k_exp,
                       int64_t v_exp, Tensor status);
void kv4_read_launch(Tensor slots, Tensor pages, int64_t k_exp, int64_t v_exp, Tensor k, Tensor v, Tensor status);
void kv4_select_launch(Tensor q, Tensor cu_q, Tensor seq_lens, Tensor table, Tensor bounds, Tensor unit, int64_t max_q,
                       int64_t first, int64_t last, Tensor score, Tensor pages, Tensor status);
std::tuple<int64_t, int64_t> kv4_attend_workspace(int64_t G, int64_t D, int64_t max_q, bool chosen);
void kv4_attend_launch(Tensor q, Tensor cu_q, Tensor seq_lens, Tensor table, Tensor pages, optional<Tensor> sel,
                       double scale, int64_t max_q, int64_t window, int64_t k_exp, int64_t v_exp, Tensor out,
                       optional<Tensor> lse, Tensor part, Tensor split, int64_t tries, Tensor status);
void kv4_prompt_launch(Tensor q, Tensor cu_q, Tensor seq_lens, Tensor table, Tensor pages, double scale, int64_t max_q,
                       int64_t window, int64_t k_exp, int64_t v_exp, Tensor out, optional<Tensor> lse, int64_t whole,
                       int64_t splits, optional<Tensor> part, Tensor status);
std::tuple<int64_t, int64_t, int64_t> kv4_prompt_plan(int64_t T, int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_q,
                                                      int64_t W, int64_t window);

namespace {

struct Cache {
  int64_t n, H, D;
};

// Numbers enter a message as text: a stream that formats them itself crashes where the interpreter's
// C++ runtime and this module's have different locale tables.
std::string num(int64_t x) { return std::to_string(x); }

Cache check_cache(const Tensor& pages, const Tensor& bounds, const Tensor& unit, const Tensor& status, int64_t k_exp,
                  int64_t v_exp) {
  TORCH_CHECK(pages.is_cuda() && pages.is_contiguous() && pages.scalar_type() == at::kByte && pages.dim() == 3 &&
                  pages.size(0) >= 1 && pages.size(1) >= 1 && pages.size(1) <= 65535,      // heads are a grid's second dimension
              "kv4: pages must be a contiguous uint8 CUDA tensor [pages, kv_heads <= 65535, 72 * head_dim]");
  const Cache c{pages.size(0), pages.size(1), pages.size(2) / 72};
  TORCH_CHECK(pages.size(2) == 72 * c.D && (c.D == 64 || c.D == 128 || c.D == 256),
              "kv4: head_dim must be 64, 128 or 256");
  TORCH_CHECK(bounds.device() == pages.device() && bounds.is_contiguous() && bounds.scalar_type() == at::kChar &&
                  bounds.numel() == c.n * c.H * 2 * c.D && unit.device() == pages.device() && unit.is_contiguous() &&
                  unit.scalar_type() == at::kFloat && unit.numel() == c.n * c.H &&
                  status.device() == pages.device() && status.scalar_type() == at::kInt && status.numel() == 1,
              "kv4: bounds int8 [pages, kv_heads, 2, head_dim], unit f32 [pages, kv_heads] or status int32 [1] do not fit");
  TORCH_CHECK(k_exp >= -14 && k_exp <= 4 && v_exp >= -14 && v_exp <= 4, "kv4: k_exp and v_exp must lie in [-14, 4]");
  return c;
}

bool half_type(const Tensor& x) { return x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf; }

void check_slots(const Tensor& slots, const Tensor& pages) {
  TORCH_CHECK(slots.device() == pages.device() && slots.scalar_type() == at::kLong && slots.dim() == 1 &&
                  slots.is_contiguous(),
              "kv4: slots must be a contiguous int64 tensor [rows] on the cache's device");
}

// the batch's row count per K/V head group; q's rows made to start on 16 bytes
int64_t check_batch(Tensor& q, const Tensor& cu_q, const Tensor& seq_lens, const Tensor& table, const Tensor& pages,
                    const Cache& c, int64_t& max_q) {
  TORCH_CHECK(q.device() == pages.device() && half_type(q) && q.dim() == 3 && q.size(2) == c.D,
              "kv4: q must be bf16 or f16 [rows, heads, ", num(c.D), "] on the cache's device");
  TORCH_CHECK(q.size(1) >= c.H && q.size(1) % c.H == 0, "kv4: q's heads must be a multiple of the ", num(c.H), " K/V heads");
  const auto int32_on = [&](const Tensor& x, int64_t dim) {
    return x.device() == pages.device() && x.scalar_type() == at::kInt && x.dim() == dim && x.is_contiguous();
  };
  TORCH_CHECK(int32_on(seq_lens, 1) && seq_lens.size(0) <= 4096,
              "kv4: seq_lens must be a contiguous int32 tensor of at most 4096 sequences on the cache's device");
  const int64_t B = seq_lens.size(0);
  TORCH_CHECK(int32_on(cu_q, 1) && cu_q.size(0) == B + 1, "kv4: cu_q must be a contiguous int32 tensor [", num(B + 1), "]");
  TORCH_CHECK(int32_on(table, 2) && table.size(0) == B && table.size(1) >= 1 && table.size(1) <= (1 << 24),
              "kv4: block_table must be a contiguous int32 tensor [", num(B), ", pages >= 1]");
  TORCH_CHECK(q.size(0) == 0 || B > 0, "kv4: rows without a sequence");
  TORCH_CHECK(q.size(0) < (int64_t)1 << 31, "kv4: too many rows");
  if (max_q < 0) max_q = q.size(0);
  TORCH_CHECK(max_q >= 1 || q.size(0) == 0, "kv4: max_q must be at least 1");
  if (q.stride(2) != 1 || q.stride(0) % 8 || q.stride(1) % 8 || (uintptr_t)q.data_ptr() % 16)
    q = q.clone(at::MemoryFormat::Contiguous);      // the kernels copy rows 16 bytes at a time
  return q.size(1) / c.H;
}

// Parts of split tiles, kept per stream (calls on one stream run one after the other).  A captured
// graph owns its workspace.  Never freed: destructors would run after the CUDA context.
std::pair<Tensor, Tensor> workspace(const Tensor& like, int64_t floats, int64_t ints) {
  static auto* kept = new std::map<std::pair<int, void*>, std::pair<Tensor, Tensor>>();
  static std::mutex mu;
  const auto stream = c10::cuda::getCurrentCUDAStream();
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  C10_CUDA_CHECK(cudaStreamIsCapturing(stream, &capturing));
  const auto make = [&](int64_t f, int64_t n) {
    return std::make_pair(at::empty({f}, like.options().dtype(at::kFloat)), at::empty({n}, like.options().dtype(at::kInt)));
  };
  if (capturing != cudaStreamCaptureStatusNone) return make(floats, ints);
  std::lock_guard<std::mutex> lock(mu);
  auto& w = (*kept)[{like.get_device(), (void*)stream.stream()}];
  if (!w.first.defined()) w = make(floats, ints);
  if (w.first.numel() < floats || w.second.numel() < ints)
    w = make(std::max(floats, w.first.numel()), std::max(ints, w.second.numel()));
  return w;
}

}  // namespace

void kv4_append(Tensor k, Tensor v, Tensor slots, Tensor pages, Tensor bounds, Tensor unit, Tensor status, int64_t k_exp,
                int64_t v_exp) {
  const Cache c = check_cache(pages, bounds, unit, status, k_exp, v_exp);
  check_slots(slots, pages);
  const int64_t T = slots.size(0);
  for (const Tensor* x : {&k, &v})
    TORCH_CHECK(x->device() == pages.device() && x->dim() == 3 && x->size(0) == T && x->size(1) == c.H &&
                    x->size(2) == c.D && (T == 0 || x->stride(2) == 1) && half_type(*x) && x->scalar_type() == k.scalar_type(),
                "kv4: k and v must be bf16 or f16 [", num(T), ", ", num(c.H), ", ", num(c.D),
                "] of one type, inner stride 1, on the cache's device");
  TORCH_CHECK(T * c.H < (int64_t)1 << 31, "kv4: too many rows for one call");
  if (T == 0) return;
  const c10::cuda::CUDAGuard guard(pages.device());
  kv4_append_launch(k, v, slots, pages, bounds, unit, k_exp, v_exp, status);
}

std::tuple<Tensor, Tensor> kv4_read(Tensor slots, at::ScalarType dtype, Tensor pages, Tensor bounds, Tensor unit,
                                    Tensor status, int64_t k_exp, int64_t v_exp) {
  const Cache c = check_cache(pages, bounds, unit, status, k_exp, v_exp);
  check_slots(slots, pages);
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf, "kv4: read gives bf16 or f16");
  TORCH_CHECK(slots.size(0) * c.H < (int64_t)1 << 31, "kv4: too many rows for one call");
  const c10::cuda::CUDAGuard guard(pages.device());
  const auto opt = pages.options().dtype(dtype);
  Tensor k = at::empty({slots.size(0), c.H, c.D}, opt), v = at::empty({slots.size(0), c.H, c.D}, opt);
  if (slots.size(0)) kv4_read_launch(slots, pages, k_exp, v_exp, k, v, status);
  return {k, v};
}

Tensor kv4_select(Tensor q, Tensor cu_q, Tensor seq_lens, Tensor table, int64_t budget, int64_t first, int64_t last,
                  int64_t max_q, Tensor pages, Tensor bounds, Tensor unit, Tensor status) {
  const Cache c = check_cache(pages, bounds, unit, status, 0, 0);
  const c10::cuda::CUDAGuard guard(pages.device());
  const int64_t G = check_batch(q, cu_q, seq_lens, table, pages, c, max_q);
  TORCH_CHECK(first >= 0 && last >= 1 && first + last <= budget && budget < (1 << 24),
              "kv4: need first >= 0, last >= 1 and first + last <= budget, got ", num(first), ", ", num(last), ", ", num(budget));
  TORCH_CHECK(G <= 64, "kv4: select takes at most 64 query heads per K/V head, got ", num(G));
  const int64_t T = q.size(0), W = table.size(1);
  Tensor chosen = at::empty({T, c.H, budget}, seq_lens.options());
  Tensor score = at::empty({W > budget ? T * c.H * W : 0}, unit.options());
  if (T) kv4_select_launch(q, cu_q, seq_lens, table, bounds, unit, max_q, first, last, score, chosen, status);
  return chosen;
}

// Query rows of one sequence and K/V head above which attention runs on the tcgen05 kernel, which
// converts each key and value once for 256 rows (128 with D = 256) where the other does for 32 (16).
// us, other / tcgen05, 8 K/V heads, B200: 8 sequences of 30000, D = 128: 32 rows 211 / 215, 40 rows
// 391 / 216; D = 256: 32 rows 317 / 377, 40 rows 458 / 380; 32 sequences of 4000, D = 64: 64 rows 126 / 132.
int64_t prompt_rows(int64_t D) { return D == 64 ? 64 : 32; }

std::tuple<Tensor, optional<Tensor>> kv4_attend(Tensor q, Tensor cu_q, Tensor seq_lens, Tensor table, double scale,
                                                int64_t max_q, int64_t window, optional<Tensor> chosen, bool return_lse,
                                                Tensor pages, Tensor bounds, Tensor unit, Tensor status, int64_t k_exp,
                                                int64_t v_exp, int64_t tries) {
  const Cache c = check_cache(pages, bounds, unit, status, k_exp, v_exp);
  TORCH_CHECK(tries >= 0 && tries <= 1 << 22, "kv4: a wait takes 0 to 2^22 tries");
  const c10::cuda::CUDAGuard guard(pages.device());
  const int64_t G = check_batch(q, cu_q, seq_lens, table, pages, c, max_q);
  TORCH_CHECK(window >= 0 && window < (int64_t)1 << 31, "kv4: window must be >= 0");
  if (window >= table.size(1) * 64) window = 0;     // hides nothing; so position - window stays well within 32 bits
  const int64_t T = q.size(0);
  if (chosen.has_value())
    TORCH_CHECK(chosen->device() == pages.device() && chosen->scalar_type() == at::kInt && chosen->is_contiguous() &&
                    chosen->dim() == 3 && chosen->size(0) == T && chosen->size(1) == c.H && chosen->size(2) >= 1,
                "kv4: pages must be a contiguous int32 tensor [", num(T), ", ", num(c.H), ", n >= 1] on the cache's device");
  Tensor out = at::empty({T, q.size(1), c.D}, q.options());
  optional<Tensor> lse;
  if (return_lse) lse = at::empty({T, q.size(1)}, unit.options());
  if (T) {
    if (!chosen.has_value() && max_q * G > prompt_rows(c.D)) {
      const auto [whole, splits, floats] = kv4_prompt_plan(T, seq_lens.size(0), c.H, G, c.D, max_q, table.size(1), window);
      optional<Tensor> part;
      if (floats) part = workspace(pages, floats, 0).first;
      kv4_prompt_launch(q, cu_q, seq_lens, table, pages, scale, max_q, window, k_exp, v_exp, out, lse, whole, splits, part,
                        status);
    } else {
      const auto [floats, ints] = kv4_attend_workspace(G, c.D, max_q, chosen.has_value());
      auto [part, split] = workspace(pages, floats, ints);
      kv4_attend_launch(q, cu_q, seq_lens, table, pages, chosen, scale, max_q, window, k_exp, v_exp, out, lse, part, split,
                        tries, status);
    }
  }
  return {out, lse};
}

void register_kv4(pybind11::module& m) {
  m.def("kv4_append", &kv4_append);
  m.def("kv4_read", [](Tensor slots, py::object dtype, Tensor pages, Tensor bounds, Tensor unit, Tensor status, int64_t k_exp,
                       int64_t v_exp) {
    return kv4_read(slots, torch::python::detail::py_object_to_dtype(dtype), pages, bounds, unit, status, k_exp, v_exp);
  });
  m.def("kv4_select", &kv4_select);
  m.def("kv4_attend", &kv4_attend);
}
