// Attention over the paged 4-bit cache: which kernel a call takes.
#include "kv4_attn.hpp"

namespace flk {

// Up to 16 query-head rows a kv head take the decode kernel.
static bool few_rows(uint32_t max_q, uint32_t n_heads, uint32_t n_kv_heads) {
  return (uint64_t)max_q * (n_heads / n_kv_heads) <= 16;
}

uint64_t kv4_attn_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys, uint32_t n_heads,
                           uint32_t n_kv_heads, uint32_t head_dim, uint32_t window,
                           uint32_t n_sinks) {
  const auto plan = few_rows(max_q, n_heads, n_kv_heads) ? kv4_decode_plan : kv4_prefill_plan;
  return plan(n_seqs, max_q, max_n_keys, n_heads, n_kv_heads, head_dim, window, n_sinks).ws_bytes;
}

hipError_t launch_kv4_attn(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  const bool few = few_rows(a.max_q, a.n_heads, a.s.n_kv_heads);
  const Kv4SplitPlan p = (few ? kv4_decode_plan : kv4_prefill_plan)(
      a.n_seqs, a.max_q, a.max_n_keys, a.n_heads, a.s.n_kv_heads, a.s.head_dim, a.window,
      a.n_sinks);
  return few ? launch_kv4_decode(a, p, ws, st) : launch_kv4_prefill(a, p, ws, st);
}

}  // namespace flk
