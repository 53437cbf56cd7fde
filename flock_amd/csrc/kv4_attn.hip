// Attention over the paged 4-bit cache: which kernel a call takes.
#include "kv4_attn.hpp"

namespace flk {

// Up to 48 query-head rows a kv head take the decode kernel, in chunks of 16: the prompt
// kernel's 128-row tiles cost the same for a few rows as for many. us, decode kernel / prompt
// kernel, 64 sequences of up to 16000 keys / 16 of up to 4000 / one of 131072: 16 rows 180 /
// 762, 24 / 40.5, 35 / 78; 32 rows 326 / 745, 38 / 41.6, 53 / 79; 48 rows 481 / 819, 50 / 48.6,
// 73 / 95; 64 rows 605 / 822, 60 / 50, 90 / 96.
static bool few_rows(uint32_t max_q, uint32_t n_heads, uint32_t n_kv_heads) {
  return (uint64_t)max_q * (n_heads / n_kv_heads) <= 48;
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
