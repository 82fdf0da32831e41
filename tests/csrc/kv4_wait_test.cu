// The prompt kernel of the 4-bit cache with short waits: the warp that issues the products gives up its first wait
// for weights, with products in flight, and every other warp runs out of tries after it.
#define MOET_KV4_TRIES 1024
#define MOET_KV4_P_TRIES 0
#define kv4_prompt_launch kv4_prompt_wait_launch
#define kv4_prompt_plan kv4_prompt_wait_plan
#include "kv4_prompt.cu"

// one stretch per tile; status is set, the outputs mean nothing
void kv4_prompt_wait_test(torch::Tensor q, torch::Tensor cu_q, torch::Tensor seq_lens, torch::Tensor table,
                          torch::Tensor pages, int64_t max_q, torch::Tensor out, torch::Tensor status) {
  const int64_t H = pages.size(1), D = pages.size(2) / 72, G = q.size(1) / H;
  const int64_t whole = moet::kv4::prompt_tiles(q.size(0), G, D, max_q) * H * seq_lens.size(0);
  kv4_prompt_wait_launch(q, cu_q, seq_lens, table, pages, 0.1, max_q, 0, -6, -6, out, c10::nullopt, whole, 1, c10::nullopt,
                         status);
}
