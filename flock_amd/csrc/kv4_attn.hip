// Attention over the paged 4-bit cache: which kernel a call takes.
#include <algorithm>

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

// A call whose sequences may be prompts and single tokens: those of up to this many queries (8
// query-head rows, one column tile) take the decode kernel in a launch of their own, for in the
// prompt kernel each of their workgroups would go through a long context alone. 0: one launch.
// us, prompt kernel / both: a 2048-token prompt with 31 single tokens of up to 16384 keys 578 /
// 143, with another of 131072 beside them 598 / 169; a 512-token chunk with 31 of up to 4000
// 142 / 105, of 2000 83 / 77; with 7 of up to 8000 132 / 120, of 4000 80 / 84, of 2000 55 / 66;
// chunks alone 5 more (113 / 118). So from contexts of more than 2048 keys on.
constexpr uint32_t kMixedTiles = 64;
static uint32_t mixed_q(uint32_t n_seqs, uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                        uint32_t window, uint32_t n_sinks) {
  const uint32_t q = 8 / (n_heads / n_kv_heads);
  return n_seqs > 1 && kv4_max_tiles(max_n_keys, q, window, n_sinks) > kMixedTiles ? q : 0;
}
static uint32_t mixed_q(const Kv4AttnArgs& a) {
  return mixed_q(a.n_seqs, a.max_n_keys, a.n_heads, a.s.n_kv_heads, a.window, a.n_sinks);
}
static Kv4AttnArgs few_of(const Kv4AttnArgs& a, uint32_t q) {
  Kv4AttnArgs few = a;
  few.max_q = few.q_to = q;
  return few;
}

uint64_t kv4_attn_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys, uint32_t n_heads,
                           uint32_t n_kv_heads, uint32_t head_dim, uint32_t window,
                           uint32_t n_sinks) {
  if (few_rows(max_q, n_heads, n_kv_heads))
    return kv4_decode_ws_bytes(n_seqs, max_q, max_n_keys, n_heads, n_kv_heads, head_dim, window,
                               n_sinks);
  const uint64_t bytes = kv4_prefill_ws_bytes(n_seqs, max_q, max_n_keys, n_heads, n_kv_heads,
                                              head_dim, window, n_sinks);
  const uint32_t q = mixed_q(n_seqs, max_n_keys, n_heads, n_kv_heads, window, n_sinks);
  if (q == 0) return bytes;
  return std::max(bytes, kv4_decode_ws_bytes(n_seqs, q, max_n_keys, n_heads, n_kv_heads, head_dim,
                                             window, n_sinks));
}

bool kv4_attn_fits(const Kv4AttnArgs& a) {
  if (few_rows(a.max_q, a.n_heads, a.s.n_kv_heads)) return kv4_decode_fits(a);
  const uint32_t q = mixed_q(a);
  return kv4_prefill_fits(a) && (q == 0 || kv4_decode_fits(few_of(a, q)));
}

hipError_t launch_kv4_attn(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  if (few_rows(a.max_q, a.n_heads, a.s.n_kv_heads)) return launch_kv4_decode(a, ws, st);
  const uint32_t q = mixed_q(a);
  if (q == 0) return launch_kv4_prefill(a, ws, st);
  // (One workspace: the launches follow each other.)
  const hipError_t e = launch_kv4_decode(few_of(a, q), ws, st);
  if (e != hipSuccess) return e;
  Kv4AttnArgs many = a;
  many.q_from = q + 1;
  return launch_kv4_prefill(many, ws, st);
}

}  // namespace flk
