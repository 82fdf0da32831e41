// Test-only native module `moet_testkit`: kernels that validate hardware paths
// but serve no model (built beside the product library, never imported by it).
#include <torch/extension.h>

void tc_gemm_test(torch::Tensor a, torch::Tensor sa, torch::Tensor b, torch::Tensor sb, torch::Tensor out,
                  torch::Tensor status, int64_t stage);
void kv4_prompt_wait_test(torch::Tensor q, torch::Tensor cu_q, torch::Tensor seq_lens, torch::Tensor table,
                          torch::Tensor pages, int64_t max_q, torch::Tensor out, torch::Tensor status);

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("tc_gemm_test", &tc_gemm_test, "one-CTA tcgen05 block-scaled e4m3 GEMM through TMEM (validation)");
  m.def("kv4_prompt_wait_test", &kv4_prompt_wait_test, "prompt attention of the 4-bit cache, giving up at once");
}
