// Pieces of the attention kernels over the paged 4-bit cache: codes to f16, q and
// the weights in two f16 parts, which keys a row sees.
#pragma once

#include "kv4.hpp"

namespace flk {

constexpr float kLog2e = 1.44269504088896340736f;

// Four packed pairs of a dword's eight codes as (c - 8) * d, d a pair of scales: pair i
// is nibbles i and i + 4. A masked nibble under 0x6400 is the f16 1024 + c (or 1024 +
// 16 c, a bit position higher): no shift for the second, and no rounding anywhere.
__device__ __forceinline__ halfx2 as_half2(uint32_t v) { return __builtin_bit_cast(halfx2, v); }
__device__ __forceinline__ uint32_t as_u32(halfx2 v) { return __builtin_bit_cast(uint32_t, v); }
template <int J>
__device__ __forceinline__ halfx2 kv4_pair(uint32_t w, halfx2 d) {
  const uint32_t x = J >= 2 ? w >> 8 : w;
  halfx2 c;
  if constexpr (J & 1) {
    const halfx2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const halfx2 off = {(_Float16)-72.f, (_Float16)-72.f};
    c = __builtin_elementwise_fma(as_half2((x & 0x00f000f0u) | 0x64006400u), sixteenth, off);
  } else {
    const halfx2 off = {(_Float16)-1032.f, (_Float16)-1032.f};
    c = as_half2((x & 0x000f000fu) | 0x64006400u) + off;
  }
  return c * d;
}

union Half8 {
  uint32_t u[4];
  halfx8 h;
};

__device__ __forceinline__ halfx2 pack_half2(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 v = {a, b};
  return __builtin_convertvector(v, halfx2);
}

// A power of two that brings a row's largest |q| to 2^14 .. 2^15, and its inverse:
// the row's two f16 parts then hold 22 bits of every element down to 2^-39 of the
// largest. Rows below 2^-112 keep the largest factor (their scores are 0 next to 1);
// infinities stay infinite, and their second part is NaN.
struct RowScale {
  float up, down;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  const uint32_t e = max((__builtin_bit_cast(uint32_t, amax) >> 23) & 255u, 15u);
  return {__builtin_bit_cast(float, (268u - e) << 23), __builtin_bit_cast(float, (e - 14u) << 23)};
}

// Weights are exp2(score - reference + kBias), at most 2^15: the second parts of
// weights down to 2^-14 of the largest are then normal f16 numbers. The reference
// moves when a score passes it by more than kSlack.
constexpr float kBias = 10.f, kSlack = 5.f;

struct Kv4Seq {
  uint32_t q0, nq, n_keys;
  bool refused;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs& a, uint32_t b) {
  Kv4Seq s;
  s.q0 = min(a.q_off[b], a.n_tokens);
  const uint32_t q1 = min(a.q_off[b + 1], a.n_tokens);
  s.nq = q1 > s.q0 ? q1 - s.q0 : 0;
  s.n_keys = a.n_keys[b];
  s.refused = s.n_keys > a.max_n_keys || s.nq > a.max_q;
  return s;
}

// Pieces that a row tile's key tiles are cut into: as few as leave none more than
// `most` tiles, then as equal as they come.
struct Kv4Pieces {
  uint32_t n, per;
};
__device__ __forceinline__ Kv4Pieces kv4_pieces(uint32_t tiles, uint32_t most) {
  const uint32_t n = max(1u, (tiles + most - 1) / most);
  return {n, (tiles + n - 1) / n};
}

// Key tiles that a row tile of `queries` queries may have, from the call's bounds.
inline uint32_t kv4_max_tiles(uint32_t max_n_keys, uint32_t queries, uint32_t window,
                              uint32_t n_sinks) {
  const uint64_t all = ((uint64_t)max_n_keys + kKv4Tile - 1) / kKv4Tile;
  if (window == 0) return (uint32_t)all;
  const uint64_t seen = ((uint64_t)window + queries + kKv4Tile - 2) / kKv4Tile + 1 +
                        ((uint64_t)n_sinks + kKv4Tile - 1) / kKv4Tile;
  return (uint32_t)(seen < all ? seen : all);
}

// The two kernels' plans, from the call's bounds alone (lengths are on the device).
struct Kv4SplitPlan {
  uint32_t rows;       // query-head rows of a row tile
  uint32_t row_tiles;  // row tiles of a (sequence, kv head)
  uint32_t most;       // key tiles of a piece, at most
  uint32_t splits;     // pieces that a row tile may have
  uint64_t ws_bytes;
};
Kv4SplitPlan kv4_decode_plan(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                             uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                             uint32_t window, uint32_t n_sinks);
hipError_t launch_kv4_decode(const Kv4AttnArgs& a, const Kv4SplitPlan& p, void* ws,
                             hipStream_t st);

}  // namespace flk
