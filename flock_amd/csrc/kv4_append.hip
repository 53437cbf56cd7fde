// New tokens into the paged 4-bit cache (with q/k norm and RoPE before, or as they
// are), and rows of it back as f32.
//
// A block of 32 values x of a head vector: m is its value of largest magnitude
// (the positive one in a tie), d = f16(bf16(m / -8)), c = rint(x / d) limited to
// -8 .. 7, kept as c + 8. The scale is rounded to the eight bits of bf16, an error
// of at most 2^-9 of it, so that (c) * d, three bits (or a power of two) times
// eight, is exact in f16: attention multiplies the stored values themselves. f16
// bounds the scale to 8160, values to 65280; larger finite ones saturate.
// A block with an infinity or a NaN gets d = NaN: all its 32 values read as NaN.
#include <type_traits>

#include "kv4.hpp"

namespace flk {

// Max and min over the lane's half wave (32 lanes), in every lane.
__device__ __forceinline__ void half_wave_range(float v, float& hi, float& lo) {
  hi = lo = v;
  auto step = [&](float a, float b) {
    hi = fmaxf(hi, a);
    lo = fminf(lo, b);
  };
  step(dpp<kDppXor1>(hi), dpp<kDppXor1>(lo));
  step(dpp<kDppXor2>(hi), dpp<kDppXor2>(lo));
  step(dpp<kDppHalfMirror>(hi), dpp<kDppHalfMirror>(lo));
  step(dpp<kDppMirror>(hi), dpp<kDppMirror>(lo));
  float a, b;
  swap_pair<16>(hi, a, b);
  hi = fmaxf(a, b);
  swap_pair<16>(lo, a, b);
  lo = fminf(a, b);
}

// Scale (f16 bits) and code (0 .. 15) of this lane's value in its block of 32 lanes.
__device__ __forceinline__ uint32_t kv4_quantise(float x, uint16_t& scale_bits) {
  float hi, lo;
  half_wave_range(x, hi, lo);
  const uint64_t bad = __ballot(!(fabsf(x) <= 3.40282347e38f));
  const uint32_t bad_half = (threadIdx.x & 32) ? (uint32_t)(bad >> 32) : (uint32_t)bad;
  const float m = hi >= -lo ? hi : lo;
  const float d0 = fminf(fmaxf(m / -8.f, -8160.f), 8160.f);
  const _Float16 h = (_Float16)(float)(__bf16)d0;
  const float d = (float)h;
  const float inv = d == 0.f ? 0.f : 1.f / d;
  const float c = fminf(fmaxf(rintf(x * inv), -8.f), 7.f);
  scale_bits = bad_half ? 0x7e00u : __builtin_bit_cast(uint16_t, h);
  return bad_half ? 8u : (uint32_t)((int)c + 8);
}

// OR over aligned groups of 4 or 8 lanes, in every lane.
template <int N>
__device__ __forceinline__ uint32_t or_lanes(uint32_t v) {
  auto move = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  v |= move(v, std::integral_constant<int, kDppXor1>{});
  v |= move(v, std::integral_constant<int, kDppXor2>{});
  if constexpr (N == 8) v |= move(v, std::integral_constant<int, kDppHalfMirror>{});
  return v;
}

// This lane's value (dim `dim` = 64 * part + lane) of a K or V row into token t of
// the tile. Every lane of the wave calls it.
template <int D>
__device__ __forceinline__ void kv4_store(uint8_t* tile, int t, bool is_k, int dim, float x) {
  const int lane = threadIdx.x & 63;
  uint16_t scale;
  const uint32_t code = kv4_quantise(x, scale);
  if ((lane & 31) == 0) {
    const int b = dim >> 5;
    *reinterpret_cast<uint16_t*>(tile + (is_k ? Kv4<D>::k_scale(t, b) : Kv4<D>::v_scale(t, b))) =
        scale;
  }
  if (is_k) {
    const int u = lane & 7;
    const uint32_t w = or_lanes<8>(code << (4 * ((u >> 1) + 4 * (u & 1))));
    if (u == 0) *reinterpret_cast<uint32_t*>(tile + Kv4<D>::k_dword(t, dim >> 3)) = w;
  } else {
    const uint32_t w = or_lanes<4>(code << (4 * (lane & 3)));
    if ((lane & 3) == 0)
      *reinterpret_cast<uint16_t*>(tile + Kv4<D>::v_word(t, dim >> 2)) = (uint16_t)w;
  }
}

// One workgroup per token, a wave per head vector at a time (as the prologue of the
// f32 caches, whose arithmetic the norm and the rotation share): q heads (norm, RoPE,
// to qn_out), then k heads (norm, RoPE, 4 bits), then v heads (4 bits). NORM false:
// k and v only, as they are. A token whose slot lies outside the pool is not stored.
constexpr int kKv4Threads = 256;

template <int D, bool NORM>
__global__ __launch_bounds__(kKv4Threads) void kv4_append_kernel(Kv4AppendArgs a) {
  __shared__ float2 s_cs[D / 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tok = blockIdx.x, G = a.s.n_kv_heads;
  const uint32_t slot = a.slots[tok];
  const bool stored = slot < a.s.n_pages * a.s.page;
  const uint32_t page_id = slot / a.s.page, in_page = slot % a.s.page;
  const uint32_t n_q = NORM ? a.n_heads : 0, per_tok = n_q + 2 * G;
  auto source = [&](uint32_t idx) {
    if (NORM && idx < n_q) return a.q + (size_t)tok * a.q_stride + (size_t)idx * D;
    if (idx < n_q + G) return a.k + (size_t)tok * a.kv_stride + (size_t)(idx - n_q) * D;
    return a.v + (size_t)tok * a.kv_stride + (size_t)(idx - n_q - G) * D;
  };
  constexpr int kWaves = kKv4Threads / 64, kBatch = 8;
  float e0[kBatch], e1[kBatch];
  auto load_batch = [&](uint32_t base) {
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const float* src = source(min(base + kWaves * i, per_tok - 1));
      e0[i] = src[lane];
      e1[i] = D == 128 ? src[lane + 64] : 0.f;
    }
  };
  float gq0 = 1.f, gq1 = 1.f, gk0 = 1.f, gk1 = 1.f, invf = 0.f;
  if (NORM) invf = a.inv_freq[min((int)threadIdx.x, D / 2 - 1)];
  load_batch(wave);
  if (NORM) {
    gq0 = a.gq[lane], gk0 = a.gk[lane];
    if (D == 128) gq1 = a.gq[lane + 64], gk1 = a.gk[lane + 64];
    if (threadIdx.x < D / 2) s_cs[threadIdx.x] = rope_cos_sin(invf, a.positions[tok]);
    __syncthreads();
  }
  for (uint32_t base = wave; base < per_tok; base += kWaves * kBatch) {
    if (base != (uint32_t)wave) load_batch(base);
    float scale_mine = 0.f;
    if (NORM) {  // as qk_prologue_kernel: lane i forms vector i's 1 / sqrt
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        float p = e0[i] * e0[i];
        if (D == 128) p = p + e1[i] * e1[i];
        p = tree_sum64(p);
        mine = (lane & (kBatch - 1)) == i ? p : mine;
      }
      scale_mine = rsqrt_once(mine / (float)D + a.eps);
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const uint32_t idx = base + kWaves * i;
      if (idx >= per_tok) continue;  // uniform per wave
      float x0 = e0[i], x1 = e1[i];
      const bool is_q = idx < n_q, is_k = !is_q && idx < n_q + G;
      if (NORM && (is_q || is_k)) {
        const float scale = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale_mine), i));
        x0 = (x0 * scale) * (is_q ? gq0 : gk0);
        if (D == 128) x1 = (x1 * scale) * (is_q ? gq1 : gk1);
        head_rope<D>(x0, x1, s_cs, a.pairing, lane);
      }
      if (is_q) {
        float* dst = a.qn_out + ((size_t)tok * n_q + idx) * D;
        dst[lane] = x0;
        if (D == 128) dst[lane + 64] = x1;
      } else if (stored) {
        const uint32_t head = idx - n_q - (is_k ? 0 : G);
        uint8_t* tile = a.pool + kv4_tile_at(page_id, head, in_page, G, a.s.page,
                                             Kv4<D>::kTileBytes);
        const int t = in_page % kKv4Tile;
        kv4_store<D>(tile, t, is_k, lane, x0);
        if (D == 128) kv4_store<D>(tile, t, is_k, lane + 64, x1);
      }
    }
  }
}

hipError_t launch_kv4_append(const Kv4AppendArgs& a, hipStream_t st) {
  const dim3 grid(a.n_tokens), block(kKv4Threads);
  if (a.s.head_dim == 128) {
    if (a.q != nullptr)
      hipLaunchKernelGGL((kv4_append_kernel<128, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((kv4_append_kernel<128, false>), grid, block, 0, st, a);
  } else {
    if (a.q != nullptr)
      hipLaunchKernelGGL((kv4_append_kernel<64, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((kv4_append_kernel<64, false>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}

// ------------------------------------------------------------------- read ----
// A thread per four dims of a token's K and V row of one head: the values of the
// codes, or zeros where the slot lies outside the pool.
template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const uint8_t* __restrict__ pool,
                                                       const uint32_t* __restrict__ slots,
                                                       float* __restrict__ k,
                                                       float* __restrict__ v, uint32_t n_tokens,
                                                       Kv4Shape s) {
  const uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const uint64_t row = id / (D / 4);  // (token, head)
  if (row >= (uint64_t)n_tokens * s.n_kv_heads) return;
  const uint32_t w = (uint32_t)(id % (D / 4));
  const uint32_t tok = (uint32_t)(row / s.n_kv_heads), head = (uint32_t)(row % s.n_kv_heads);
  const uint32_t slot = slots[tok];
  float kx[4] = {0.f, 0.f, 0.f, 0.f}, vx[4] = {0.f, 0.f, 0.f, 0.f};
  if (slot < s.n_pages * s.page) {
    const uint32_t in_page = slot % s.page;
    const uint8_t* tile = pool + kv4_tile_at(slot / s.page, head, in_page, s.n_kv_heads, s.page,
                                             Kv4<D>::kTileBytes);
    const int t = in_page % kKv4Tile, b = w >> 3;
    auto f16 = [&](int at) {
      return (float)__builtin_bit_cast(_Float16, *reinterpret_cast<const uint16_t*>(tile + at));
    };
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(tile + Kv4<D>::k_dword(t, w >> 1));
    const uint32_t vw = *reinterpret_cast<const uint16_t*>(tile + Kv4<D>::v_word(t, w));
    const float ks = f16(Kv4<D>::k_scale(t, b)), vs = f16(Kv4<D>::v_scale(t, b));
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int u = 4 * (w & 1) + j;
      kx[j] = (float)((int)(kw >> (4 * ((u >> 1) + 4 * (u & 1))) & 15) - 8) * ks;
      vx[j] = (float)((int)(vw >> (4 * j) & 15) - 8) * vs;
    }
  }
  *reinterpret_cast<float4*>(k + row * D + 4 * w) = make_float4(kx[0], kx[1], kx[2], kx[3]);
  *reinterpret_cast<float4*>(v + row * D + 4 * w) = make_float4(vx[0], vx[1], vx[2], vx[3]);
}

hipError_t launch_kv4_read(const uint8_t* pool, const uint32_t* slots, float* k, float* v,
                           uint32_t n_tokens, const Kv4Shape& s, hipStream_t st) {
  const uint64_t threads = (uint64_t)n_tokens * s.n_kv_heads * (s.head_dim / 4);
  const dim3 grid((uint32_t)((threads + 255) / 256)), block(256);
  if (s.head_dim == 128)
    hipLaunchKernelGGL(kv4_read_kernel<128>, grid, block, 0, st, pool, slots, k, v, n_tokens, s);
  else
    hipLaunchKernelGGL(kv4_read_kernel<64>, grid, block, 0, st, pool, slots, k, v, n_tokens, s);
  return hipGetLastError();
}

}  // namespace flk
