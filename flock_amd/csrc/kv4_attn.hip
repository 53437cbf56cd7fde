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
  return (few_rows(max_q, n_heads, n_kv_heads) ? kv4_decode_ws_bytes : kv4_prefill_ws_bytes)(
      n_seqs, max_q, max_n_keys, n_heads, n_kv_heads, head_dim, window, n_sinks);
}

bool kv4_attn_fits(const Kv4AttnArgs& a) {
  return few_rows(a.max_q, a.n_heads, a.s.n_kv_heads) ? kv4_decode_fits(a) : kv4_prefill_fits(a);
}

hipError_t launch_kv4_attn(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  return (few_rows(a.max_q, a.n_heads, a.s.n_kv_heads) ? launch_kv4_decode : launch_kv4_prefill)(
      a, ws, st);
}

}  // namespace flk
