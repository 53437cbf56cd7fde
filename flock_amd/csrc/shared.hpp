// Decode attention of sequences that share prefixes: arguments, groups, launches.
#pragma once

#include "common.hpp"

namespace flk {

struct SharedArgs {
  const float *q, *kcache, *vcache;
  const uint64_t *prefix_row, *seq_row_off;
  const uint32_t *n_prefix, *seq_off, *n_keys;
  float* o;
  uint32_t n_groups, n_seqs, max_prefix, max_n_keys, n_heads, n_kv_heads, head_dim;
  bool step;  // the layer's step: n_keys[b] = 0 is an idle sequence
};

// What a sequence sees.
struct SharedSeq {
  uint32_t prefix, own;
  uint64_t prefix_row;
  bool refused, idle;
};

// The group of sequence b, by every thread of a workgroup: the one whose range holds it.
// Offsets that fall, or pass n_seqs, refuse the whole call (NaN), so that no sequence is
// in two groups.
template <int kThreads>
__device__ __forceinline__ SharedSeq shared_seq(const SharedArgs& a, uint32_t b) {
  __shared__ uint32_t s_group, s_bad;
  if (threadIdx.x == 0) s_group = 0xffffffffu, s_bad = 0;
  __syncthreads();
  for (uint32_t g = threadIdx.x; g < a.n_groups; g += kThreads) {
    const uint32_t lo = a.seq_off[g], hi = a.seq_off[g + 1];
    if (lo > hi || hi > a.n_seqs) s_bad = 1;
    if (lo <= b && b < hi) s_group = g;
  }
  __syncthreads();
  SharedSeq s{};
  const uint32_t g = s_group;
  s.own = a.n_keys[b];
  if (g < a.n_groups) s.prefix = a.n_prefix[g], s.prefix_row = a.prefix_row[g];
  s.refused = s_bad || s.own > a.max_n_keys || s.prefix > a.max_prefix;
  s.idle = !s.refused && a.step && s.own == 0;
  return s;
}

uint64_t shared_ws_bytes(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                         uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                         uint32_t head_dim);
// fused: the step's raw rows and gains (null: attention alone), q rows q_stride floats
// apart, k and v rows kv_stride.
hipError_t launch_shared(const SharedArgs& a, const DecodeFused* fused, uint32_t q_stride,
                         uint32_t kv_stride, void* ws, hipStream_t st);
hipError_t launch_shared_prologue(const SharedArgs& a, const DecodeFused& f, uint32_t q_stride,
                                  uint32_t kv_stride, hipStream_t st);

}  // namespace flk
