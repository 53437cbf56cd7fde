// Log probabilities of tokens, their alternatives, and sampling: arguments, launches.
#pragma once

#include "common.hpp"

namespace flk {

constexpr uint32_t kMaxTop = 64;  // alternatives of a row: one a lane

struct TokenArgs {
  const float* logits;
  uint64_t ld;                // floats from one row to the next
  uint32_t n_rows, n_vocab, n_top;
  // flk_token_logprobs
  const uint32_t* tokens;     // null: no logprob
  float *logprob, *entropy;   // null: not wanted
  uint32_t* top_ids;
  float* top_logprobs;
  // flk_sample (uniform not null)
  const float *temperature, *top_p, *min_p, *uniform;
  const uint32_t* top_k;
  uint32_t* token;
};
uint64_t tokens_need(uint32_t n_rows, uint32_t n_vocab, uint32_t n_top);
uint64_t tokens_ws_bytes(uint32_t n_rows, uint32_t n_vocab, uint32_t n_top);
hipError_t launch_tokens(const TokenArgs& a, void* ws, hipStream_t st);

}  // namespace flk
