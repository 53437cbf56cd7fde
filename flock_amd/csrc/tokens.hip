// Log probabilities of given tokens with entropy and top alternatives, and sampling from
// the alternatives.
//
// For a row x with largest value m (held c times) and R = sum of exp(x - m) over the
// others, log sum exp x = m + log(c + R); with c and R apart, log1p keeps the small
// logarithms of a row that is nearly sure. Entropy is log(c + R) + sum exp(x - m) (m - x)
// / (c + R), whose terms are all positive. Alternatives are ordered by 64-bit keys: the
// value's bits in an order of unsigned numbers, then the id from the top down, so that
// ties go to the lowest id and no two keys are equal.
//
// One workgroup a row.
#include "tokens.hpp"

namespace flk {

constexpr int kTokenThreads = 256;

// Larger values have larger keys; 0 for what is no alternative (-infinity, NaN).
__device__ __forceinline__ uint64_t token_key(float x, uint32_t id) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 as 0
  const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x > -INFINITY ? (uint64_t)order << 32 | (0xffffffffu - id) : 0;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __builtin_bit_cast(float, order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint32_t key_id(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// A row's sums: largest value, how often, the other weights and their spread.
struct RowSums {
  float m, count, rest, spread;
  __device__ __forceinline__ double log_total() const {  // log(count + rest)
    return log1p((double)(count - 1.f) + (double)rest);
  }
  __device__ __forceinline__ bool none() const { return !(m > -INFINITY && m < INFINITY); }
  __device__ __forceinline__ float logprob(float x) const {
    if (none() || isnan(rest)) return __builtin_nanf("");
    return (float)((double)x - (double)m - log_total());
  }
  __device__ __forceinline__ float entropy() const {
    if (none() || isnan(rest)) return __builtin_nanf("");
    return (float)(log_total() + (double)spread / ((double)count + (double)rest));
  }
};

// The token that a row's settings and its number choose among its keys (descending; 0:
// none), by one thread.
__device__ __forceinline__ uint32_t choose(const TokenArgs& a, uint32_t row, const uint64_t* keys) {
  const float t = a.temperature ? a.temperature[row] : 1.f, u = a.uniform[row];
  const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
  const uint32_t k = a.top_k ? a.top_k[row] : a.n_top;
  const bool ok = t >= 0.f && t < INFINITY && k >= 1 && k <= a.n_top && top_p > 0.f && min_p >= 0.f &&
                  min_p <= 1.f && u >= 0.f && u < 1.f;
  if (!ok || keys[0] == 0) return 0xffffffffu;
  if (t == 0.f) return key_id(keys[0]);
  const float x0 = key_value(keys[0]);
  auto weight = [&](uint32_t i) {
    const float x = key_value(keys[i]);
    return x == x0 ? 1.0 : exp(((double)x - (double)x0) / (double)t);
  };
  double all = 0;
  for (uint32_t i = 0; i < k && keys[i]; i++) all += weight(i);
  double kept = 0, sum = 0;
  uint32_t n = 0;
  for (uint32_t i = 0; i < k && keys[i]; i++) {
    const double w = weight(i);
    if (!(sum < (double)top_p * all) || w < (double)min_p || w == 0) break;
    sum += w, kept = sum, n = i + 1;
  }
  sum = 0;
  for (uint32_t i = 0; i < n; i++) {
    sum += weight(i);
    if (sum > (double)u * kept) return key_id(keys[i]);
  }
  return key_id(keys[n - 1]);
}

__global__ __launch_bounds__(kTokenThreads) void token_rows_kernel(TokenArgs a) {
  constexpr int kWaves = kTokenThreads / 64;
  __shared__ float s_f[3][kWaves];
  __shared__ uint64_t s_key[kWaves];
  __shared__ uint64_t s_top[kMaxTop];
  const uint32_t row = blockIdx.x;
  const float* x = a.logits + row * a.ld;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = -INFINITY;
  for (uint32_t i = threadIdx.x; i < a.n_vocab; i += kTokenThreads) m = fmaxf(m, x[i]);
  for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, shfl_xor(m, s));
  if (lane == 0) s_f[0][wave] = m;
  __syncthreads();
  for (int w = 0; w < kWaves; w++) m = fmaxf(m, s_f[0][w]);
  __syncthreads();
  float count = 0.f, rest = 0.f, spread = 0.f;
  for (uint32_t i = threadIdx.x; i < a.n_vocab; i += kTokenThreads) {
    const float v = x[i];
    if (v == m) {
      count += 1.f;
    } else if (!(v == -INFINITY)) {
      const float e = expf(v - m);
      rest += e;
      spread += e * (m - v);
    }
  }
  for (int s = 1; s < 64; s <<= 1) {
    count += shfl_xor(count, s);
    rest += shfl_xor(rest, s);
    spread += shfl_xor(spread, s);
  }
  if (lane == 0) s_f[0][wave] = count, s_f[1][wave] = rest, s_f[2][wave] = spread;
  __syncthreads();
  count = rest = spread = 0.f;
  for (int w = 0; w < kWaves; w++)
    count += s_f[0][w], rest += s_f[1][w], spread += s_f[2][w];
  const RowSums sums{m, count, rest, spread};
  uint64_t last = ~0ull;
  for (uint32_t k = 0; k < a.n_top; k++) {
    uint64_t best = 0;
    for (uint32_t i = threadIdx.x; i < a.n_vocab; i += kTokenThreads) {
      const uint64_t key = token_key(x[i], i);
      if (key < last && key > best) best = key;
    }
    for (int s = 1; s < 64; s <<= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, s, kWave);
      if (other > best) best = other;
    }
    __syncthreads();
    if (lane == 0) s_key[wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; w++)
      if (s_key[w] > best) best = s_key[w];
    last = best;
    if (threadIdx.x == 0) s_top[k] = best;
  }
  __syncthreads();
  if (a.uniform == nullptr) {
    for (uint32_t k = threadIdx.x; k < a.n_top; k += kTokenThreads) {
      const uint64_t key = s_top[k];
      a.top_ids[(size_t)row * a.n_top + k] = key ? key_id(key) : 0xffffffffu;
      a.top_logprobs[(size_t)row * a.n_top + k] = key ? sums.logprob(key_value(key)) : -INFINITY;
    }
  }
  if (threadIdx.x != 0) return;
  uint32_t token = 0xffffffffu;
  if (a.uniform != nullptr) {
    token = choose(a, row, s_top);
    a.token[row] = token;
  } else if (a.tokens != nullptr) {
    token = a.tokens[row];
  }
  if (a.logprob != nullptr)
    a.logprob[row] = token < a.n_vocab ? sums.logprob(x[token]) : __builtin_nanf("");
  if (a.entropy != nullptr) a.entropy[row] = sums.entropy();
}

uint64_t tokens_ws_bytes(uint32_t, uint32_t, uint32_t) { return 0; }

hipError_t launch_tokens(const TokenArgs& a, void*, hipStream_t st) {
  hipLaunchKernelGGL(token_rows_kernel, dim3(a.n_rows), dim3(kTokenThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace flk
