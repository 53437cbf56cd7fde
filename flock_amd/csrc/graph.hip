// Device-side bookkeeping of a replayable decode step: the embedding gather
// (embed.wgsl) and the position / token-log advance.
#include "common.hpp"

namespace flk {

// embed.wgsl:52-75: one workgroup per token, threads over 4-element groups;
// each element is q * scale (one rounding). An id past the vocabulary writes
// zeros instead of reading outside the matrix.
__global__ __launch_bounds__(256) void embed_kernel(const int8_t* __restrict__ qs,
                                                    const uint16_t* __restrict__ scales,
                                                    const uint32_t* __restrict__ ids,
                                                    uint32_t vocab, uint32_t hidden,
                                                    float* __restrict__ out) {
  const uint32_t tok = blockIdx.x;
  const uint32_t row = ids[tok];
  const bool ok = row < vocab;
  const uint32_t r = ok ? row : 0;
  const uint32_t nb = hidden / 32;
  float* o = out + (size_t)tok * hidden;
  for (uint32_t g = threadIdx.x; g < hidden / 4; g += 256) {
    const uint16_t h = scales[(size_t)r * nb + g / 8];
    float s;
    if ((h & 0x7c00u) == 0x7c00u)
      s = (h & 0x8000u) ? -3.40282347e38f : 3.40282347e38f;
    else
      s = (float)__builtin_bit_cast(_Float16, h);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(qs + (size_t)r * hidden + 4 * g);
    float4 v;
    v.x = (float)((int32_t)(w << 24) >> 24) * s;
    v.y = (float)((int32_t)(w << 16) >> 24) * s;
    v.z = (float)((int32_t)(w << 8) >> 24) * s;
    v.w = (float)((int32_t)w >> 24) * s;
    if (!ok) v = make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<float4*>(o)[g] = v;
  }
}

hipError_t launch_embed(const int8_t* qs, const uint16_t* scales, const uint32_t* ids,
                        uint32_t n_tokens, uint32_t vocab, uint32_t hidden, float* out,
                        hipStream_t st) {
  hipLaunchKernelGGL(embed_kernel, dim3(n_tokens), dim3(256), 0, st, qs, scales, ids, vocab,
                     hidden, out);
  return hipGetLastError();
}

// state = {n_keys, cursor}: the position word every captured decode call
// reads, and where the next logged token goes.
__global__ void advance_kernel(uint32_t* state, uint32_t delta, const uint32_t* value,
                               uint32_t* log, uint32_t log_len) {
  state[0] += delta;
  const uint32_t c = state[1];
  if (log != nullptr && value != nullptr && c < log_len) {
    log[c] = *value;
    state[1] = c + 1;
  }
}

hipError_t launch_advance(uint32_t* state, uint32_t delta, const uint32_t* value, uint32_t* log,
                          uint32_t log_len, hipStream_t st) {
  hipLaunchKernelGGL(advance_kernel, dim3(1), dim3(1), 0, st, state, delta, value, log, log_len);
  return hipGetLastError();
}

// One workgroup: its time is the launch's, and the cursor moves when all have read it.
__global__ __launch_bounds__(256) void advance_seqs_kernel(AdvanceSeqs a) {
  const uint32_t c = *a.cursor;
  __syncthreads();
  if (threadIdx.x == 0) *a.cursor = c + 1;
  for (uint32_t b = threadIdx.x; b < a.n_seqs; b += 256) {
    const uint32_t t = a.token[b], n = a.n_keys[b];
    bool stop = t == 0xffffffffu;
    for (uint32_t i = 0; i < a.n_stops; i++) stop |= t == a.stops[i];
    a.n_keys[b] = n == 0 || stop ? 0 : n + 1;
    if (c < a.log_len) {
      const size_t at = (size_t)c * a.n_seqs + b;
      a.token_log[at] = t;
      if (a.logprob_log != nullptr) a.logprob_log[at] = a.logprob[b];
    }
    if (a.uniform != nullptr && c < a.log_len && c + 1 < a.log_len)
      a.uniform[b] = a.uniform_log[(size_t)(c + 1) * a.n_seqs + b];
  }
}

hipError_t launch_advance_seqs(const AdvanceSeqs& a, hipStream_t st) {
  hipLaunchKernelGGL(advance_seqs_kernel, dim3(1), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace flk
