// Pieces of the attention kernels over the paged 4-bit cache: codes to f16, q and
// the weights in two f16 parts, which keys a row sees.
#pragma once

#include "kv4.hpp"

namespace flk {

constexpr double kLog2e = 1.44269504088896340736;

// Four packed pairs of a dword's eight codes as (c - 8) * d, d a pair of scales: pair i
// is nibbles i and i + 4. A masked nibble under 0x6400 is the f16 1024 + c (or 1024 +
// 16 c, a bit position higher): no shift for the second, and no rounding anywhere.
__device__ __forceinline__ halfx2 as_half2(uint32_t v) { return __builtin_bit_cast(halfx2, v); }
__device__ __forceinline__ uint32_t as_u32(halfx2 v) { return __builtin_bit_cast(uint32_t, v); }
// (w & mask) | bits in one instruction: its two constants do not both fit as literals,
// so the compiler makes two of it unless they are held in registers.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(bits));
  return r;
}
template <int J>
__device__ __forceinline__ halfx2 kv4_pair(uint32_t w, halfx2 d) {
  const uint32_t x = J >= 2 ? w >> 8 : w;
  halfx2 c;
  if constexpr (J & 1) {
    const halfx2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const halfx2 off = {(_Float16)-72.f, (_Float16)-72.f};
    c = __builtin_elementwise_fma(as_half2(and_or(x, 0x00f000f0u, 0x64006400u)), sixteenth, off);
  } else {
    const halfx2 off = {(_Float16)-1032.f, (_Float16)-1032.f};
    c = as_half2(and_or(x, 0x000f000fu, 0x64006400u)) + off;
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

// x + s * (one half of a pair of f16), in one instruction.
template <int HI>
__device__ __forceinline__ float mix_fma(halfx2 h, float s, float x) {
  float r;
  if constexpr (HI)
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(r) : "v"(h), "v"(s), "v"(x));
  else
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(s), "v"(x));
  return r;
}

// The second f16 parts of two values whose first are hi (x - hi is exact in f32). With
// s = 0 in place of -1 the first parts again: a lane that holds one of the two picks it
// by s.
__device__ __forceinline__ halfx2 rest_half2(float a, float b, halfx2 hi, float s = -1.f) {
  return pack_half2(mix_fma<0>(hi, s, a), mix_fma<1>(hi, s, b));
}

// A power of two that brings a row's largest |q| to 2^14 .. 2^15, and its inverse. Two f16
// parts are off by at most 2^-23 of an element from 2^-2 on (2^-16 of the largest at most),
// and by 2^-25, half of the second part's last subnormal bit, of smaller ones: 2^-39 of the
// largest, which is what counts in a sum over the row. Rows below 2^-97 keep the largest factor (their scores are 0 next to 1);
// infinities stay infinite, and their second part is NaN.
struct RowScale {
  float up, down;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  const uint32_t e = max((__builtin_bit_cast(uint32_t, amax) >> 23) & 255u, 30u);
  return {__builtin_bit_cast(float, (268u - e) << 23), __builtin_bit_cast(float, (e - 14u) << 23)};
}

// Weights are exp2(score - reference + kBias): 2^10 for the reference's own key, at most 2^15.
// Two f16 parts are off by at most 2^-23 of a weight down to 2^-12 of the largest (as above,
// from 2^-2 on), and by 2^-25, which is 2^-35 of the largest, below: n keys of them by n 2^-35
// of the largest |v|, also where their scores are equal and the errors do not average out
// (2^20 keys: 3e-5). The reference moves when a score passes it by more than kSlack.
constexpr float kBias = 10.f, kSlack = 5.f;

struct Kv4Seq {
  uint32_t q0, nq, n_keys;
  bool refused;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs& a, uint32_t b) {
  Kv4Seq s;
  s.q0 = min(a.q_off[b], a.n_tokens);
  const uint32_t end = a.q_off[b + 1], q1 = min(end, a.n_tokens);
  s.nq = q1 > s.q0 ? q1 - s.q0 : 0;
  if (s.nq < a.q_from || s.nq > a.q_to) s.nq = 0;
  s.n_keys = a.n_keys[b];
  // (Of rows behind n_tokens the cache has no keys, and positions count from the last.)
  s.refused = s.n_keys > a.max_n_keys || s.nq > a.max_q || end > a.n_tokens;
  return s;
}

// Which keys of a tile the rows of a row tile see, in 32 bits: a key `off` into the
// tile and a row `delta` positions behind the row tile's first.
struct Kv4Mask {
  int causal, window, sinks;
  __device__ __forceinline__ bool sees(int off, int delta) const {
    return causal + off <= delta && (window + off > delta || off < sinks);
  }
};
__device__ __forceinline__ int clamp30(int64_t x) {
  return (int)(x < -(1 << 30) ? -(1 << 30) : x > (1 << 30) ? 1 << 30 : x);
}
// The keys that a row tile at positions first .. last sees: its tiles, and which of
// them every row sees whole.
struct Kv4Span {
  Kv4Tiles tiles;
  int64_t first;
  uint32_t window, n_sinks;
  uint32_t before, from, sinks;  // whole: below `before`, and from `from` or below `sinks`
  __device__ __forceinline__ Kv4Span(int64_t first_, int64_t last, uint32_t window_,
                                     uint32_t n_sinks_)
      : tiles(kv4_tiles(first_, last, window_, n_sinks_)),
        first(first_),
        window(window_),
        n_sinks(n_sinks_) {
    before = first < 0 ? 0u : (uint32_t)((first + 1) / kKv4Tile);
    const int64_t w = last - (int64_t)window + kKv4Tile;  // ceil((last - window + 1) / 32)
    from = window == 0 || w < 0 ? 0u : (uint32_t)(w / kKv4Tile);
    sinks = n_sinks / kKv4Tile;
  }
  __device__ __forceinline__ bool whole(uint32_t tile) const {
    return tile < before && (tile >= from || tile < sinks);
  }
  __device__ __forceinline__ Kv4Mask mask(uint32_t tile) const {
    const int64_t key0 = (int64_t)tile * kKv4Tile;
    return {clamp30(key0 - first), window == 0 ? 1 << 30 : clamp30(key0 - first + window),
            clamp30((int64_t)n_sinks - key0)};
  }
};

// Key tiles that a row tile of `queries` queries may have, from the call's bounds.
inline uint32_t kv4_max_tiles(uint32_t max_n_keys, uint32_t queries, uint32_t window,
                              uint32_t n_sinks) {
  const uint64_t all = ((uint64_t)max_n_keys + kKv4Tile - 1) / kKv4Tile;
  if (window == 0) return (uint32_t)all;
  const uint64_t seen = ((uint64_t)window + queries + kKv4Tile - 2) / kKv4Tile + 1 +
                        ((uint64_t)n_sinks + kKv4Tile - 1) / kKv4Tile;
  return (uint32_t)(seen < all ? seen : all);
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) {  // in a scalar register
  return __builtin_amdgcn_readfirstlane(v);
}

// Tiles of a piece at most: `pieces` pieces for the batch, none cut below `least` tiles.
__device__ __forceinline__ uint32_t kv4_per(uint32_t total, uint32_t pieces, uint32_t least) {
  return max(total / pieces + (total % pieces != 0), least);
}

// Sum over the workgroup of v, and over the threads before this one.
template <int kWaves>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s_wave, uint32_t& before) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t scan = v;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const uint32_t y = __shfl_up(scan, x, kWave);
    if (lane >= x) scan += y;
  }
  if (lane == 63) s_wave[wave] = scan;
  __syncthreads();
  uint32_t total = 0;
  before = scan - v;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  return uniform(total);
}

// Partial results: row r of slot x is at x * rows + r.
struct Kv4Part {
  float* ml;   // pairs (reference, sum)
  float* acc;  // D floats
};

// o of one row from n partial results, i-th at at(i): kThreads threads, D / 4 of them over
// the row's dims and the pieces dealt out to the groups of them. A piece without a visible
// key holds zeros (or NaN, which stay).
template <int D, int kThreads, typename At>
__device__ __forceinline__ void merge_pieces(const Kv4Part& part, uint32_t n, At at, float* dst) {
  constexpr int kLanes = D / 4, kGroups = kThreads / kLanes;
  __shared__ float4 s_acc[kGroups][kLanes];
  __shared__ float s_sum[kGroups];
  const float2* ml = reinterpret_cast<const float2*>(part.ml);
  const uint32_t lane = threadIdx.x & 63, e = threadIdx.x % kLanes, g = threadIdx.x / kLanes;
  float top = -INFINITY;
  for (uint32_t i = lane; i < n; i += 64) top = fmaxf(top, ml[at(i)].x);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, shfl_xor(top, x));
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (uint32_t i = g; i < n; i += kGroups) {
    const size_t p = at(i);
    const float2 x = ml[p];
    const float4 y = reinterpret_cast<const float4*>(part.acc + p * D)[e];
    const float k = x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.x - top);
    sum = fmaf(x.y, k, sum);
    f.x = fmaf(y.x, k, f.x), f.y = fmaf(y.y, k, f.y);
    f.z = fmaf(y.z, k, f.z), f.w = fmaf(y.w, k, f.w);
  }
  s_acc[g][e] = f;
  if (e == 0) s_sum[g] = sum;
  __syncthreads();
  if (g != 0) return;
  for (int i = 1; i < kGroups; i++) {
    const float4 y = s_acc[i][e];
    f.x += y.x, f.y += y.y, f.z += y.z, f.w += y.w;
    sum += s_sum[i];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  reinterpret_cast<float4*>(dst)[e] = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
}

// The same by D / 4 neighbouring threads alone.
template <int D, typename At>
__device__ __forceinline__ void merge_few(const Kv4Part& part, uint32_t n, At at, float* dst) {
  const float2* ml = reinterpret_cast<const float2*>(part.ml);
  const uint32_t e = threadIdx.x % (D / 4);
  float top = -INFINITY;
  for (uint32_t i = 0; i < n; i++) top = fmaxf(top, ml[at(i)].x);
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (uint32_t i = 0; i < n; i++) {
    const size_t p = at(i);
    const float2 x = ml[p];
    const float4 y = reinterpret_cast<const float4*>(part.acc + p * D)[e];
    const float k = x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.x - top);
    sum = fmaf(x.y, k, sum);
    f.x = fmaf(y.x, k, f.x), f.y = fmaf(y.y, k, f.y);
    f.z = fmaf(y.z, k, f.z), f.w = fmaf(y.w, k, f.w);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  reinterpret_cast<float4*>(dst)[e] = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
}

uint64_t kv4_decode_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                             uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                             uint32_t window, uint32_t n_sinks);
hipError_t launch_kv4_decode(const Kv4AttnArgs& a, void* ws, hipStream_t st);
uint64_t kv4_prefill_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                              uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                              uint32_t window, uint32_t n_sinks);
hipError_t launch_kv4_prefill(const Kv4AttnArgs& a, void* ws, hipStream_t st);

// Whether a call's launches and its numbers of tiles (32 bits) hold it.
bool kv4_decode_fits(const Kv4AttnArgs& a);
bool kv4_prefill_fits(const Kv4AttnArgs& a);

}  // namespace flk
