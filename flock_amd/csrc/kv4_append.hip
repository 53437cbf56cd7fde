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
#include "kv4.hpp"

namespace flk {

// A head vector lies over D / 4 lanes, four neighbouring dims each, so a block of 32 dims is
// eight lanes: the block's range takes three lane steps, its scale is formed once for
// four values, and a lane's codes are packed by a few f32 products (below 2^16: exact).
// A wave takes 256 / D vectors at a time. (A value a lane, with a range over 32 lanes and
// a division each, was VALU-bound: 8192 tokens of 16 / 8 heads of 128 60 us. 48 now, 4.4 TB/s
// of 211 MB, the VALU still busy for 0.92 of it.)

// v of the lane 16, 8, 4, 2 or 1 away, all of them lanes of one vector; 4 only where
// lanes 8 apart hold the same value already (row_ror:4 reads one of the two).
template <int M>
__device__ __forceinline__ float vec_xor(float v) {
  static_assert(M == 8 || M == 4 || M == 2 || M == 1, "vec_xor");
  if constexpr (M == 8) return dpp<kDppRor8>(v);
  if constexpr (M == 4) return dpp<kDppRor4>(v);
  if constexpr (M == 2) return dpp<kDppXor2>(v);
  return dpp<kDppXor1>(v);
}

// The reference's pairwise tree over a vector's squares (strides D / 2 .. 1), in every lane.
template <int D>
__device__ __forceinline__ float vec_tree(const float (&x)[4]) {
  float p[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    p[j] = x[j] * x[j];
    if constexpr (D == 128) p[j] = sum_xor<16>(p[j]);
    p[j] = p[j] + vec_xor<8>(p[j]);
    p[j] = p[j] + vec_xor<4>(p[j]);
    p[j] = p[j] + vec_xor<2>(p[j]);
    p[j] = p[j] + vec_xor<1>(p[j]);
  }
  p[0] = p[0] + p[2];
  p[1] = p[1] + p[3];
  return p[0] + p[1];
}

// RoPE of dims 4 l .. 4 l + 3 of a vector, as head_rope.
template <int D>
__device__ __forceinline__ void vec_rope(float (&x)[4], const float2* cs, int pairing, int l) {
  if (pairing == FLK_ROPE_NORM) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float a = x[j], b = x[j + 1];
      const float2 c = cs[2 * l + j / 2];
      x[j] = rope_rot(a, b, true, c);
      x[j + 1] = rope_rot(b, a, false, c);
    }
  } else {
    const bool first = l < D / 8;
    const int at = 4 * (first ? l : l - D / 8);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float y;
      if constexpr (D == 128) {
        float lo, hi;
        swap_pair<16>(x[j], lo, hi);
        y = (threadIdx.x & 16) ? lo : hi;  // lane i & ~16 holds lo, i | 16 hi
      } else {
        y = vec_xor<8>(x[j]);
      }
      x[j] = rope_rot(x[j], y, first, cs[at + j]);
    }
  }
}

// Dims 4 l .. 4 l + 3 of a K or V row into token t of the tile. Every lane of the wave
// calls it; `store` says which have a row.
template <int D>
__device__ __forceinline__ void kv4_store(uint8_t* tile, int t, bool is_k, int l,
                                          const float (&x)[4], bool store) {
  float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
  hi = fmaxf(hi, dpp<kDppXor1>(hi)), lo = fminf(lo, dpp<kDppXor1>(lo));
  hi = fmaxf(hi, dpp<kDppXor2>(hi)), lo = fminf(lo, dpp<kDppXor2>(lo));
  hi = fmaxf(hi, dpp<kDppHalfMirror>(hi)), lo = fminf(lo, dpp<kDppHalfMirror>(lo));
  constexpr float kMax = 3.40282347e38f;
  const uint64_t bad = __ballot(!(fabsf(x[0]) <= kMax && fabsf(x[1]) <= kMax &&
                                  fabsf(x[2]) <= kMax && fabsf(x[3]) <= kMax));
  const bool none = (bad >> (threadIdx.x & 56)) & 0xff;  // no number in the block
  const float m = hi >= -lo ? hi : lo;
  const float d0 = fminf(fmaxf(m * -0.125f, -8160.f), 8160.f);
  const _Float16 h = (_Float16)(float)(__bf16)d0;
  const float d = (float)h;
  const float inv = d == 0.f || none ? 0.f : 1.f / d;  // (zero codes, 8, for a NaN block)
  float c[4];
#pragma unroll
  for (int j = 0; j < 4; j++)
    c[j] = fminf(fmaxf(rintf((none ? 0.f : x[j]) * inv), -8.f), 7.f) + 8.f;
  uint32_t w;
  if (is_k) {
    // Dims t of eight as nibbles (t >> 1) + 4 (t & 1): this lane's are t = 0 .. 3 or 4 .. 7.
    w = (uint32_t)fmaf(c[2], 16.f, c[0]) | (uint32_t)fmaf(c[3], 16.f, c[1]) << 16;
    w <<= 8 * (l & 1);
  } else {
    w = (uint32_t)fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]);
  }
  const uint32_t both =
      w | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, kDppXor1, 0xF, 0xF, false);
  if (!store) return;
  if ((l & 7) == 0) {
    const int b = l >> 3;
    *reinterpret_cast<uint16_t*>(tile + (is_k ? Kv4<D>::k_scale(t, b) : Kv4<D>::v_scale(t, b))) =
        none ? (uint16_t)0x7e00 : __builtin_bit_cast(uint16_t, h);
  }
  if (is_k) {
    if ((l & 1) == 0) *reinterpret_cast<uint32_t*>(tile + Kv4<D>::k_dword(t, l >> 1)) = both;
  } else {
    *reinterpret_cast<uint16_t*>(tile + Kv4<D>::v_word(t, l)) = (uint16_t)w;
  }
}

// One workgroup per token (as the prologue of the f32 caches, whose arithmetic the norm and
// the rotation share): q heads (norm, RoPE, to qn_out), then k heads (norm, RoPE, 4 bits),
// then v heads (4 bits). NORM false: k and v only, as they are. A token whose slot lies
// outside the pool is not stored.
constexpr int kKv4Threads = 256;

template <int D, bool NORM>
__global__ __launch_bounds__(kKv4Threads) void kv4_append_kernel(Kv4AppendArgs a) {
  __shared__ float2 s_cs[D / 2];
  constexpr int kLanes = D / 4, kVec = 64 / kLanes;  // lanes of a vector, vectors of a wave
  constexpr int kBatch = 4;                          // wave steps that are loaded together
  const int lane = threadIdx.x & 63, l = lane % kLanes;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tok = blockIdx.x, G = a.s.n_kv_heads;
  const uint32_t slot = a.slots[tok];
  const bool stored = slot < a.s.n_pages * a.s.page;
  const uint32_t log_page = 31 - __builtin_clz(a.s.page);
  const uint32_t page_id = slot >> log_page, in_page = slot & (a.s.page - 1);
  const uint32_t n_q = NORM ? a.n_heads : 0, per_tok = n_q + 2 * G;
  const uint32_t my = wave * kVec + lane / kLanes;  // this lane's vector of the first step
  constexpr uint32_t kStride = kKv4Threads / kLanes;
  const float* q_row = NORM ? a.q + (size_t)tok * a.q_stride : nullptr;
  const float* k_row = a.k + (size_t)tok * a.kv_stride;
  const float* v_row = a.v + (size_t)tok * a.kv_stride;
  float x[kBatch][4];
  auto load_batch = [&](uint32_t base) {
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const uint32_t idx = min(base + kStride * i, per_tok - 1);
      const float* src = NORM && idx < n_q ? q_row + (size_t)idx * D
                         : idx < n_q + G   ? k_row + (size_t)(idx - n_q) * D
                                           : v_row + (size_t)(idx - n_q - G) * D;
#pragma unroll
      for (int j = 0; j < 4; j++) x[i][j] = src[4 * l + j];
    }
  };
  float gq[4] = {}, gk[4] = {};
  float invf = 0.f;
  if (NORM) invf = a.inv_freq[min((int)threadIdx.x, D / 2 - 1)];
  load_batch(my);
  if (NORM) {
#pragma unroll
    for (int j = 0; j < 4; j++) gq[j] = a.gq[4 * l + j], gk[j] = a.gk[4 * l + j];
    if (threadIdx.x < D / 2) s_cs[threadIdx.x] = rope_cos_sin(invf, a.positions[tok]);
    __syncthreads();
  }
  uint8_t* page = a.pool + kv4_tile_at(stored ? page_id : 0, 0, in_page, G, a.s.page,
                                       Kv4<D>::kTileBytes);
  const size_t head_bytes = (size_t)(a.s.page / kKv4Tile) * Kv4<D>::kTileBytes;
  const int t = in_page % kKv4Tile;
  // (Waves stay whole: base is the first vector of the wave's step.)
  for (uint32_t base = wave * kVec; base < per_tok; base += kStride * kBatch) {
    if (base != (uint32_t)wave * kVec) load_batch(base + lane / kLanes);
    float scale[kBatch] = {};
    if (NORM) {
      // 1 / sqrt of the batch's means in one f64 sequence: lane i of every four forms step
      // i's and hands it to the other three.
      float mine = 0.f;
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        const float p = vec_tree<D>(x[i]);
        mine = (lane & 3) == i ? p : mine;
      }
      mine = rsqrt_once(mine / (float)D + a.eps);
      scale[0] = dpp<0x00>(mine), scale[1] = dpp<0x55>(mine);
      scale[2] = dpp<0xAA>(mine), scale[3] = dpp<0xFF>(mine);
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const uint32_t first = base + kStride * i, idx = first + lane / kLanes;
      if (first >= per_tok) break;  // uniform per wave
      const bool is_q = idx < n_q, is_k = !is_q && idx < n_q + G;
      float y[4] = {x[i][0], x[i][1], x[i][2], x[i][3]};
      if (NORM && first < n_q + G) {
        float z[4];
#pragma unroll
        for (int j = 0; j < 4; j++) z[j] = (y[j] * scale[i]) * (is_q ? gq[j] : gk[j]);
        vec_rope<D>(z, s_cs, a.pairing, l);
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = is_q || is_k ? z[j] : y[j];
      }
      if (is_q) {
        float* dst = a.qn_out + ((size_t)tok * n_q + idx) * D + 4 * l;
#pragma unroll
        for (int j = 0; j < 4; j++) dst[j] = y[j];
      }
      if (stored && first + kVec > n_q) {
        const uint32_t head = idx - n_q - (is_k ? 0 : G);
        const bool store = !is_q && idx < per_tok;
        kv4_store<D>(page + (store ? head : 0) * head_bytes, t, is_k, l, y, store);
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
// codes, or zeros where the slot lies outside the pool. HBM-bound by what it writes (8192
// tokens of 8 heads of 128: 16.7 us, 4.6 TB/s).
template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const uint8_t* __restrict__ pool,
                                                       const uint32_t* __restrict__ slots,
                                                       float* __restrict__ k,
                                                       float* __restrict__ v, uint32_t n_tokens,
                                                       Kv4Shape s) {
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
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
