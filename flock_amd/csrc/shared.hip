// Decode attention of sequences that share long prefixes: each sequence's token sees its
// group's prefix keys and its own, and the prefix is read once for the group.
//
// f32 keys and values meet q and the softmax weights on f16 matrix products of two parts each:
// x = h + l, h = x rounded to f16 and l = x - h likewise (22 bits), and x y = h h' + h l' +
// l h', all sums in f32. The product left out, l l', is at most 2^-22 of x y. Operands are
// scaled by powers of two first: q by its row's largest, K and V by factors that stay while the
// tiles' largest values suit f16 with them (K's and q's are undone in the score's factor, V's
// at the end).
//
// A workgroup takes a run of tiles, 32 keys each (64 of 64-wide heads) that meet up to 128
// rows of q; four waves of 32 rows, two workgroups a CU. A tile's K and V come through
// registers, are split there and put into LDS, in the order of the matrix operands, once for all
// rows; the next tile's loads are in flight meanwhile, also where a chain ends and the next begins.
// S^T = K Q^T and O^T += V^T P^T on 32x32x16: a column is a row of q, and P^T is taken from the
// S^T accumulators as they lie, because V's keys are put in the order in which a lane holds its
// scores. Waves without rows (a sequence's own keys meet few) only stage.
//
// What bounds it: with few rows, reading K and V; with many, how fast a wave gets through its
// instructions, for a vector instruction of a lone wave takes 7 to 14 cycles and two waves share
// a SIMD. So the split of the next tile stands among the products of the scores, four
// instructions to a product, and a tile is split before its largest values are known. Calls: 16
// sequences over 32k keys (32 rows a kv head) 70 us, of which plan and merge are 13 under a kernel
// trace; 128 over 128k (256 rows in two row tiles) 536 to 557 us, this kernel 537, 769 TFLOP/s of f16
// products, the matrix units busy for 0.46 of the cycles.
#include <algorithm>

#include "shared.hpp"
#include "kv4_attn.hpp"

namespace flk {

// The reference of a row's weights follows the keys, so that those which matter have two parts in
// f16. It rises to a score more than kSlack above it and falls to the largest of a block of 32 keys
// that is more than kDrop below it: that key's weight is 2^-6 at least, and two parts are off by
// 2^-25, 2^-19 of it, or by 2^-22 of themselves. Where it rises far (kFar) and the block's other keys
// have fallen behind by kDrop, these are taken first, against a reference of their own. So a
// key that takes nearly all of the weight and has small values leaves the others as exact as they are
// without it: with such a key 20 nats above 512 others, 5e-7 off in the 2-norm (f32 5e-7), and 1.4e-4
// against the largest score so far alone. A row whose accumulators are kSolid times its sum (of
// values that are 2^16 at most) does not fall: 2^-25 is little beside what it holds. Nor
// does one fall farther than l stays below 2^kRoom by. Ordinary scores (2 nats around their mean)
// rise as often as with the largest score alone, and calls take 0 to 2 % longer; with scores 8
// nats around it -1 to 11 % (32 % without kSolid, whose rows fall and rise in turn).
constexpr float kDrop = 16.f, kFar = 8.f, kSolid = 256.f;
constexpr int kRoom = 60;

typedef float floatx16v __attribute__((ext_vector_type(16)));

constexpr int kShThreads = 256;

// LDS, for each part: K's rows in 16-byte slots of 8 dims, V's (a row a dim: of head_dim / 4
// rows each the dims 0, 1, 2, 3 modulo 4) in slots of 8 keys; slots xored with bits of the row so
// that neighbouring rows of one slot lie in distinct banks.
template <int D>
__device__ __forceinline__ uint32_t sh_k_at(uint32_t key, uint32_t slot) {
  return key * (2 * D) + ((slot ^ (D == 128 ? key & 15 : (key >> 1) & 7)) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t sh_v_at(uint32_t row, uint32_t slot) {
  return row * (8192 / D) + ((slot ^ (D == 128 ? (row >> 2) & 3 : (row >> 1) & 7)) << 4);
}

template <int D>
struct alignas(16) SharedLds {
  static constexpr int kPart = 8192;  // bytes of a tile's part
  uint8_t k[2][2][kPart], v[2][2][kPart];
  float top[2][kShThreads / 64];             // the largest |k| and |v| of a tile, by wave
  alignas(16) uint32_t fit[2][kShThreads / 64];  // how each wave's k and v fit the factors
};
// Values with their factor: none (0), too large for f16, all too small for two parts of it.
constexpr uint32_t kFits = 1, kLarge = 2, kSmall = 4;
__device__ __forceinline__ uint32_t shared_fit(float top, float up) {  // top: of the lane, >= 0
  const float x = top * up;
  const uint64_t large = __ballot(!(x < 65000.f)), fits = __ballot(x >= 256.f);
  const uint64_t some = __ballot(top > 0.f);
  return large ? kLarge : fits ? kFits : some ? kSmall : 0;
}
// Those of a tile: k's in the low half, v's above.
__device__ __forceinline__ uint32_t shared_fits_of(const uint32_t (&of)[kShThreads / 64]) {
  const uint4 fit = *reinterpret_cast<const uint4*>(of);
  return uniform(fit.x | fit.y | fit.z | fit.w);
}
__device__ __forceinline__ bool shared_misfit(uint32_t fits) {
  const uint32_t k = fits & 0xffff, v = fits >> 16;
  return ((k | v) & kLarge) || k == kSmall || v == kSmall;
}

// f16(x s) and f16(y s), and what is left of x s and y s (a difference that is formed exactly),
// rounded likewise; s a power of two.
__device__ __forceinline__ uint32_t first_part(float x, float y, float s) {
  return as_u32(pack_half2(x * s, y * s));
}
__device__ __forceinline__ uint32_t second_part(float x, float y, float s, uint32_t first) {
  const halfx2 h = as_half2(first);
  const halfx2 l = {(_Float16)fmaf(x, s, -(float)h[0]), (_Float16)fmaf(y, s, -(float)h[1])};
  return as_u32(l);
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, xor_lane<1>(v));
  v = fmaxf(v, xor_lane<2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  v = fmaxf(v, dpp<kDppMirror>(v));
  v = max_xor<16>(v);
  return max_xor<32>(v);
}
__device__ __forceinline__ float uniform_f(float v) {  // in a scalar register
  return __builtin_bit_cast(float, uniform(__builtin_bit_cast(uint32_t, v)));
}
__device__ __forceinline__ int exponent(float v) {  // of v >= 0: -127 for 0, 128 for infinity
  return (int)(__builtin_bit_cast(uint32_t, v) >> 23) - 127;
}
__device__ __forceinline__ float power_of_two(int e) {  // 2^e, |e| < 127
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// v, in a way that what is computed from it is not moved out of a loop: the kernel's registers
// are full, and a few instructions a tile cost less than registers held or spilled.
__device__ __forceinline__ uint32_t here(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// What of a tile is known when its loads are sent, and goes with it.
struct SharedTile {
  uint64_t at;            // floats: its first row in the caches
  uint32_t once;          // read by this workgroup alone
  uint32_t keys;          // it holds
  uint32_t row0, n_rows;  // they meet
  uint32_t part;          // where the rows' results go
  uint32_t last;          // of the run's tiles of its chain: 1
};

template <int D>
__global__ __launch_bounds__(kShThreads, 2) void shared_attn_kernel(SharedArgs a, SharedPlan p,
                                                                   float scale_log2e) {
  constexpr int kTile = 4096 / D, kBlocks = kTile / 32, kSteps = D / 16, kOT = D / 32;
  constexpr int kPart = SharedLds<D>::kPart;
  constexpr int kChunks = D / 4;          // float4s of a row
  constexpr int kGroups = 64 / kChunks;   // rows of a load
  __shared__ SharedLds<D> sh;
  const uint32_t G = a.n_kv_heads, m = a.n_heads / G;
  const uint32_t kvh = blockIdx.x % G, run = blockIdx.x / G;
  uint32_t e = uniform(p.run[run].chain), tile = uniform(p.run[run].tile0);
  const uint32_t end = uniform(p.run[run + 1].tile0);
  if (tile == end) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const uint32_t rows = a.n_seqs * m;
  const size_t part0 = kvh * shared_parts(rows, p.max_runs);

  // The chain that tiles are fetched from.
  uint64_t key_row;
  uint32_t n_keys, in_chain;
  SharedTile next;  // the last tile that was sent for
  auto open = [&] {
    typedef const __attribute__((address_space(4))) uint32_t* ConstPtr;
    const ConstPtr c = (ConstPtr)(uintptr_t)(p.chain + e);
    key_row = uniform(c[0]) | (uint64_t)uniform(c[1]) << 32;
    n_keys = uniform(c[2]), next.row0 = uniform(c[3]), next.n_rows = uniform(c[4]);
    in_chain = uniform(tile - c[5]);
    const uint32_t kind = uniform(c[7]);
    next.once = kind & kSharedOnce;
    next.part = uniform(c[6]) == run ? next.row0 + (kind & kSharedOwn ? rows : 0)
                                     : 2 * rows + run * kSharedRows;
  };
  auto advance = [&] {  // next: one tile on
    if (next.last) {
      e++;
      open();
    }
    next.at = ((key_row + (uint64_t)in_chain * kTile) * G + kvh) * D;
    next.keys = uniform(min(n_keys - in_chain * kTile, (uint32_t)kTile));
    next.last = uniform(tile + 1 == end || (in_chain + 1) * kTile >= n_keys ? 1 : 0);
    tile++, in_chain++;
  };

  // Staging: a thread loads chunk c of four rows of K, and of four rows of V that are
  // neighbours in the operands' order of keys: of a 16-key step, lane half h holds the scores of
  // keys 4 h .. (first) and 8 + 4 h .. (second).
  const int c = lane % kChunks, gr = lane / kChunks;
  const int v_step = D == 128 ? wave >> 1 : wave;
  const int v_unit = D == 128 ? (wave & 1) + 2 * gr : gr;
  const uint32_t stride = G * D * 4;  // bytes of a cache row
  const uint32_t k_key = wave * (kTile / 4) + gr, v_key = 16 * v_step + 4 * v_unit;
  // (Rows 2 i, or 4 i, further of K lie 512 i bytes on, their slots xored with 2 i; V's rows of
  // dims j modulo 4 2048 j bytes on.)
  const uint32_t k_to = sh_k_at<D>(k_key, c >> 1) + 8 * (c & 1);
  const uint32_t v_to = sh_v_at<D>(c, 2 * v_step + (v_unit & 1)) + 8 * (v_unit >> 1);
  const uint32_t k_from = sh_k_at<D>(col, h), v_from = sh_v_at<D>(col, h);
  const uint32_t k_off = k_key * stride + 16 * c, v_off = v_key * stride + 16 * c;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  u4 rk[4], rv[4];
  auto fetch = [&](const SharedTile& x) {
    // (Rows behind the last read as zeros: the descriptors end with the tile's last row.)
    const uint32_t bytes = (x.keys - 1) * stride + D * 4;
    const auto ks = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.kcache + x.at), 0,
                                                      bytes, 0x00020000);
    const auto vs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.vcache + x.at), 0,
                                                      bytes, 0x00020000);
    const uint32_t ko = here(k_off), vo = here(v_off);
    if (x.once) {  // not to stay in the caches
#pragma unroll
      for (int i = 0; i < 4; i++)
        rk[i] = __builtin_amdgcn_raw_buffer_load_b128(ks, ko + kGroups * i * stride, 0, 2);
#pragma unroll
      for (int i = 0; i < 4; i++)
        rv[i] = __builtin_amdgcn_raw_buffer_load_b128(vs, vo + i * stride, 0, 2);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        rk[i] = __builtin_amdgcn_raw_buffer_load_b128(ks, ko + kGroups * i * stride, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; i++)
        rv[i] = __builtin_amdgcn_raw_buffer_load_b128(vs, vo + i * stride, 0, 0);
    }
  };
  auto f = [](uint32_t x) { return __builtin_bit_cast(float, x); };
  // The factors of the tile in LDS, 2^k_e and 2^v_e. They stay while a tile's largest values lie
  // in 2^8 .. 2^16 with them, or are 0: then two parts in f16 are off by 2^-25 at most, 2^-33
  // of the largest. So a tile need not be seen as a whole before it is split: each wave
  // notes how its part fits, and the tile is done again if need be.
  int k_e = 0, v_e = 0;
  // The least v_e of the chain's tiles so far that held values other than 0; kNoValues: none did,
  // and the accumulators are 0.
  constexpr int kNoValues = 62;
  int v_low = kNoValues;
  // An eighth of the tile in registers into LDS.
  auto stage_part = [&](int buf, int part, float k_up, float v_up) {
    const int i = part & 3;
    float x, y, z, w;
    if (part < 4)
      x = f(rk[i][0]), y = f(rk[i][1]), z = f(rk[i][2]), w = f(rk[i][3]);
    else
      x = f(rv[0][i]), y = f(rv[1][i]), z = f(rv[2][i]), w = f(rv[3][i]);
    const float up = part < 4 ? k_up : v_up;
    uint2 hi, lo;
    hi.x = first_part(x, y, up), hi.y = first_part(z, w, up);
    lo.x = second_part(x, y, up, hi.x), lo.y = second_part(z, w, up, hi.y);
    uint8_t* at = part < 4 ? &sh.k[0][0][(k_to + buf * (2 * kPart)) ^ (i << 5)] + 512 * i
                           : &sh.v[0][0][v_to + buf * (2 * kPart)] + 2048 * i;
    *reinterpret_cast<uint2*>(at) = hi;
    *reinterpret_cast<uint2*>(at + kPart) = lo;
  };
  auto note_fit = [&](int buf) {
    float k = 0.f, v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        k = fmaxf(k, fabsf(f(rk[i][j])));
        v = fmaxf(v, fabsf(f(rv[i][j])));
      }
    sh.fit[buf][wave] =
        shared_fit(k, power_of_two(k_e)) | shared_fit(v, power_of_two(v_e)) << 16;
  };
  // The factors from the tile in registers, 2^11 .. 2^12 its largest values with them, and
  // the tile into LDS; by all waves. (V's is at most 2^48 of the chain's least, so that
  // accumulators stay finite.) The exponent of V's largest: at 128 it holds an infinity, its
  // rows are NaN, and the factor is as before. (Where every tile's sizes jump by 2^4, a call takes 119 us for 68, 16 sequences
  // over 32k keys, or 767 for 541, 128 over 128k.)
  auto anchor = [&](int buf) {
    float k = 0.f, v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        k = fmaxf(k, fabsf(f(rk[i][j])));
        v = fmaxf(v, fabsf(f(rv[i][j])));
      }
    k = wave_max(k), v = wave_max(v);
    if (lane == 0) sh.top[0][wave] = k, sh.top[1][wave] = v;
    lds_barrier();
    const float4 kt = *reinterpret_cast<const float4*>(sh.top[0]);
    const float4 vt = *reinterpret_cast<const float4*>(sh.top[1]);
    const int ke = exponent(uniform_f(fmaxf(fmaxf(kt.x, kt.y), fmaxf(kt.z, kt.w))));
    const int ve = exponent(uniform_f(fmaxf(fmaxf(vt.x, vt.y), fmaxf(vt.z, vt.w))));
    if (ke != -127 && ke != 128) k_e = max(11 - max(ke, -100), -115);
    if (ve != -127 && ve != 128) v_e = max(min(11 - max(ve, -100), v_low + 48), -115);
#pragma unroll
    for (int i = 0; i < 8; i++) stage_part(buf, i, power_of_two(k_e), power_of_two(v_e));
    lds_barrier();
    return ve;
  };

  // This wave's rows (lanes behind the last repeat it), q in two parts: dims 16 s + 8 h ..
  Half8 qh[kSteps], ql[kSteps];
  float c_s = 0.f;
  auto load_q = [&](uint32_t row0, uint32_t n_rows) {
    const uint32_t l = here(lane), my = row0 + min(wave * 32u + (l & 31), n_rows - 1);
    const float* src = a.q + ((size_t)(my / m) * a.n_heads + kvh * m + my % m) * D + 8 * (l >> 5);
    float x[D / 2], amax = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float4 y = *reinterpret_cast<const float4*>(src + 16 * s + 4 * i);
        x[8 * s + 4 * i] = y.x, x[8 * s + 4 * i + 1] = y.y;
        x[8 * s + 4 * i + 2] = y.z, x[8 * s + 4 * i + 3] = y.w;
      }
#pragma unroll
    for (int i = 0; i < D / 2; i++) amax = fmaxf(amax, fabsf(x[i]));
    amax = max_xor<32>(amax);
    const RowScale rs = row_scale(amax);
    c_s = rs.down * scale_log2e;
#pragma unroll
    for (int i = 0; i < D / 4; i++) {
      const uint32_t hi = first_part(x[2 * i], x[2 * i + 1], rs.up);
      qh[i >> 2].u[i & 3] = hi;
      ql[i >> 2].u[i & 3] = second_part(x[2 * i], x[2 * i + 1], rs.up, hi);
    }
  };

  floatx16v o[kOT];
  float ref = -INFINITY, l = 0.f;
  float under = -INFINITY;  // where the reference falls
  floatx16v scores[kBlocks];
  // The scores of the tile in LDS and, among their products, the next tile's way there.
  auto products = [&](int buf) {
    const int to = buf ^ 1;
    const float k_up = power_of_two(k_e), v_up = power_of_two(v_e);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int kb = i / kSteps, st = i % kSteps;
      floatx16v& s = scores[kb];
      if (st == 0) s = floatx16v{};
      const uint8_t* at = &sh.k[0][0][(k_from + buf * (2 * kPart)) ^ (st << 5)] + kb * (64 * D);
      const halfx8 kh = *reinterpret_cast<const halfx8*>(at);
      const halfx8 kl = *reinterpret_cast<const halfx8*>(at + kPart);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[st].h, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[st].h, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[st].h, s, 0, 0, 0);
      stage_part(to, i, k_up, v_up);
    }
    note_fit(to);
    // (K's operands two steps ahead of the products.)
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < 8; i++) {
#pragma unroll
      for (int j = 0; j < 3; j++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x200, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };
  // 16 keys' values with their weights.
  auto values = [&](int buf, int kb, int ks, Half8 ph, Half8 pl) {
#pragma unroll
    for (int x = 0; x < kOT; x++) {
      const uint8_t* at =
          &sh.v[0][0][(v_from + buf * (2 * kPart)) ^ ((4 * kb + 2 * ks) << 4)] + x * (kPart / kOT);
      const halfx8 vh = *reinterpret_cast<const halfx8*>(at);
      const halfx8 vl = *reinterpret_cast<const halfx8*>(at + kPart);
      o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph.h, o[x], 0, 0, 0);
      o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl.h, o[x], 0, 0, 0);
      o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph.h, o[x], 0, 0, 0);
    }
  };
  // Moves the reference of rows whose scores have left its range.
  auto follow = [&](floatx16v& s, int buf, int kb, float c_t, float top) {
    top = max_xor<32>(top);  // (the row's other keys are in lane + 32)
    // The reference falls no farther than l stays below 2^61 by, and accumulators (l 2^16 2^48 at
    // most) finite.
    auto fall = [&](float to) {
      return fmaxf(to, ref - (float)min(kRoom - exponent(max_xor<32>(l)), 100));
    };
    auto move = [&](float to) {
      const float alpha = to == ref ? 1.f : __builtin_amdgcn_exp2f(ref - to);
      under = to == ref ? under : to - kDrop;
      ref = to;
      if (__ballot(alpha != 1.f && l > 0.f) == 0) return;  // (of accumulators that are 0 as well)
      l *= alpha;
#pragma unroll
      for (int x = 0; x < kOT; x++) o[x] *= alpha;
    };
    // Where a row rises far: the largest of its keys in the block that are far below the top.
    if (__ballot(top > ref + kFar)) {
      const float cut = top > ref + kFar ? (top - kFar) * __builtin_amdgcn_rcpf(c_t) : -INFINITY;
      float low = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; i++) low = fmaxf(low, s[i] < cut ? s[i] : -INFINITY);
      low = max_xor<32>(low) * c_t;
      const bool apart = low < top - kDrop && low > -INFINITY;
      if (__ballot(apart)) {
        const float to = fall(low), limit = apart ? cut : -INFINITY;
        move(apart ? to : ref);
        const float rb = (ref == -INFINITY ? 0.f : ref) - kBias;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
          Half8 ph, pl;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float w[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const float y = s[8 * ks + 2 * i + j];
              const bool is = y < limit;
              w[j] = is ? __builtin_amdgcn_exp2f(fmaf(y, c_t, -rb)) : 0.f;
              s[8 * ks + 2 * i + j] = is ? -INFINITY : y;
              l += w[j];
            }
            ph.u[i] = as_u32(pack_half2(w[0], w[1]));
            pl.u[i] = second_part(w[0], w[1], 1.f, ph.u[i]);
          }
          values(buf, kb, ks, ph, pl);
        }
      }
    }
    float to = fmaxf(ref, top);
    bool falls = top < under && top > -INFINITY;
    if (__ballot(falls)) {
      float size = 0.f;
#pragma unroll
      for (int x = 0; x < kOT; x++)
#pragma unroll
        for (int i = 0; i < 16; i++) size = fmaxf(size, fabsf(o[x][i]));
      if (max_xor<32>(size) >= max_xor<32>(l) * kSolid) under = -INFINITY, falls = false;
      const float down = fall(top);
      to = falls ? down : to;
    }
    move(to);
  };
  auto block = [&](int buf, int kb, float c_t, uint32_t keys) {
    floatx16v& s = scores[kb];
    if (keys < kTile) {
#pragma unroll
      for (int i = 0; i < 16; i++)
        s[i] = kb * 32 + 8 * (i >> 2) + 4 * h + (i & 3) < (int)keys ? s[i] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
    top *= c_t;
    const uint64_t rises = __ballot(top > ref + kSlack), falls = __ballot(top < under);
    if (rises | (uint32_t)(falls & falls >> 32))  // (a row's lanes are i and i + 32)
      follow(s, buf, kb, c_t, top);
    const float rb = (ref == -INFINITY ? 0.f : ref) - kBias;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c_t, -rb));
      l += s[i];
    }
    Half8 ph[2], pl[2];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t hi = as_u32(pack_half2(s[2 * i], s[2 * i + 1]));
      ph[i >> 2].u[i & 3] = hi;
      pl[i >> 2].u[i & 3] = second_part(s[2 * i], s[2 * i + 1], 1.f, hi);
    }
#pragma unroll
    for (int ks = 0; ks < 2; ks++) values(buf, kb, ks, ph[ks], pl[ks]);
    // (V's operands likewise; the first during the weights.)
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < 2 * kOT; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };
  // The rows' results so far: accumulator i of block x is row 8 (i / 4) + 4 h + i % 4 of V's
  // 32 x .., so dim 4 (row % (D / 4)) + row / (D / 4).
  auto store = [&](uint32_t part, uint32_t n_rows, int unit) {
    float lo, hi;
    swap_pair<32>(l, lo, hi);
    const float sum = lo + hi;
    const uint32_t ln = here(lane), row = wave * 32u + (ln & 31);
    if (row >= n_rows) return;
    const size_t at = part0 + part + row;
    if (ln < 32) p.ml[at] = make_float2(ref, sum);
    // (One after the other: their product may overflow. The sum is 0 where every score is below
    // f32's range: weight 0 beside other keys.)
    const float inv = sum == 0.f ? 0.f : 1.f / sum, down = power_of_two(-unit);
    float* dst = p.acc + at * D + 16 * (ln >> 5);
#pragma unroll
    for (int i = 0; i < D / 8; i++) {
      const int r = 8 * (i >> 2) + (i & 3);  // (and 4 h)
      if constexpr (D == 128)
        *reinterpret_cast<float4*>(dst + 4 * r) =
            make_float4(o[0][i] * inv * down, o[1][i] * inv * down, o[2][i] * inv * down,
                        o[3][i] * inv * down);
      else
        *reinterpret_cast<float4*>(dst + 4 * r) =
            make_float4(o[0][i] * inv * down, o[0][i + 8] * inv * down, o[1][i] * inv * down,
                        o[1][i + 8] * inv * down);
    }
  };

  // Two waves share a SIMD, and where both could issue the older one does: its run was done in
  // 388 us of 529, the other's in 470 (128 sequences, 128k keys). So the wave in the second place
  // goes first in every other tile: 548 -> 537 us, and 126 -> 120 of 64-wide heads.
  const bool second = __builtin_amdgcn_s_getreg(4 | 0 << 6 | 3 << 11) & 1;  // HW_ID's wave id
  const uint32_t n = end - tile;
  open();
  next.last = 0;
  advance();
  fetch(next);
  SharedTile staged = next;
  if (wave * 32u < staged.n_rows) load_q(staged.row0, staged.n_rows);
  const int top_v = anchor(0);
  if (n > 1) {
    advance();
    fetch(next);
  }
  for (uint32_t t = 0; t < n;) {  // chains
    const uint32_t n_rows = staged.n_rows, part = staged.part;
    const bool busy = wave * 32u < n_rows;
    if (busy && t > 0) load_q(staged.row0, n_rows);
    ref = under = -INFINITY, l = 0.f;
#pragma unroll
    for (int x = 0; x < kOT; x++) o[x] = floatx16v{};
    v_low = kNoValues;
    int unit = v_e;  // accumulators hold O^T 2^unit
    uint32_t last;
    do {  // their tiles
      const int buf = t & 1;
      if (second && (t & 1))
        __builtin_amdgcn_s_setprio(1);
      else
        __builtin_amdgcn_s_setprio(0);
      const SharedTile now = staged;
      last = now.last;
      if (t + 1 < n) staged = next;
      bool some = top_v != -127, infinite = top_v == 128;
      if (t > 0) {
        const uint32_t fits = shared_fits_of(sh.fit[buf]);
        some = fits >> 16;
        infinite = false;
        if (shared_misfit(fits)) {
          fetch(now);
          infinite = anchor(buf) == 128;
          if (t + 1 < n) fetch(staged);
        }
      }
      // (Behind the run's last tile what is staged is not read.)
      if (busy) {
        products(buf);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) stage_part(buf ^ 1, i, power_of_two(k_e), power_of_two(v_e));
        note_fit(buf ^ 1);
      }
      if (t + 2 < n) {
        advance();
        fetch(next);
      }
      if (v_e != unit || infinite) {
        const float alpha = infinite             ? __builtin_nanf("")
                            : v_low == kNoValues ? 0.f
                                                 : ldexpf(1.f, v_e - unit);
#pragma unroll
        for (int x = 0; x < kOT; x++) o[x] *= alpha;
        unit = v_e;
      }
      if (some) v_low = min(v_low, v_e);
      // (Neither 0 nor infinite: masked scores are -infinity, others may be 0. The least normal
      // number leaves scores next to 0 too; with the largest those that are not lost beside the
      // tile's largest keys overflow as well.)
      if (t % 16 == 0) under = ref - kDrop;  // (what is solid is looked at again)
      const float c_t = fminf(fmaxf(c_s * power_of_two(-k_e), 1.17549435e-38f), 3.40282347e38f);
      if (busy) {
#pragma unroll
        for (int kb = 0; kb < kBlocks; kb++) block(buf, kb, c_t, now.keys);
      }
      lds_barrier();
      t++;
    } while (!last);
    if (busy) store(part, n_rows, unit);
  }
}

// Joins the partial results of rows: o = sum w o_i / sum w, w = l 2^ref. D / 4 threads over a
// row's dims, kGroups of them over its pieces.
template <int D, int kGroups>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a, SharedPlan p) {
  constexpr uint32_t kLanes = D / 4, kRows = 256 / (kLanes * kGroups);
  __shared__ float4 s_acc[kGroups > 1 ? kRows : 1][kGroups][kLanes];
  __shared__ float s_sum[kGroups > 1 ? kRows : 1][kGroups];
  const uint32_t mine = threadIdx.x / (kLanes * kGroups), g = threadIdx.x / kLanes % kGroups;
  const uint32_t e = threadIdx.x % kLanes, all_rows = a.n_seqs * a.n_heads;
  const uint32_t row = min(blockIdx.x * kRows + mine, all_rows - 1);
  const uint32_t b = row / a.n_heads, head = row % a.n_heads, m = a.n_heads / a.n_kv_heads;
  const uint32_t kvh = head / m, at_row = b * m + head % m, rows = a.n_seqs * m;
  const SharedRecord r = p.record[b];
  const bool refused = r.own_n == kSharedRefused || r.prefix_n == kSharedRefused;
  const bool idle = r.own_n == kSharedIdle;
  const uint32_t n = refused || idle ? 0 : r.prefix_n + r.own_n;
  const size_t part0 = kvh * shared_parts(rows, p.max_runs);
  auto at = [&](uint32_t i) {
    if (i == 0 && r.prefix_n > 0) return part0 + at_row;
    if (i < r.prefix_n)
      return part0 + 2 * rows + (size_t)(r.prefix_run + i) * kSharedRows + (at_row - r.row0);
    i -= r.prefix_n;
    if (i == 0) return part0 + rows + at_row;
    return part0 + 2 * rows + (size_t)(r.own_run + i) * kSharedRows + head % m;
  };
  // (The largest weight is below 2: sums reach 2^62, and their product with huge values f32's end.)
  float top = -INFINITY;
  for (uint32_t i = e; i < n; i += kLanes) {
    const float2 ml = p.ml[at(i)];
    top = fmaxf(top, ml.x + (float)exponent(ml.y));
  }
#pragma unroll
  for (uint32_t x = 1; x < kLanes; x <<= 1) top = fmaxf(top, shfl_xor(top, x));
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (uint32_t i = g; i < n; i += kGroups) {
    const size_t x = at(i);
    const float2 ml = p.ml[x];
    const float4 y = reinterpret_cast<const float4*>(p.acc + x * D)[e];
    const float w = ml.y * __builtin_amdgcn_exp2f(ml.x - top);
    sum += w;
    f.x = fmaf(y.x, w, f.x), f.y = fmaf(y.y, w, f.y);
    f.z = fmaf(y.z, w, f.z), f.w = fmaf(y.w, w, f.w);
  }
  if constexpr (kGroups > 1) {
    s_acc[mine][g][e] = f;
    if (e == 0) s_sum[mine][g] = sum;
    __syncthreads();
    if (g != 0) return;
    for (int i = 1; i < kGroups; i++) {
      const float4 y = s_acc[mine][i][e];
      f.x += y.x, f.y += y.y, f.z += y.z, f.w += y.w;
      sum += s_sum[mine][i];
    }
  }
  if (blockIdx.x * kRows + mine >= all_rows) return;
  const float inv = refused ? __builtin_nanf("") : n == 0 ? 0.f : 1.f / sum;
  reinterpret_cast<float4*>(a.o + (size_t)row * D)[e] =
      make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
}

constexpr int kPlanThreads = 256;
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(SharedArgs a, SharedPlan p) {
  shared_plan<kPlanThreads>(a, p);
}

// Workgroups: two a CU, all at once. Calls with 256 / 512 / 1024, us: 64 x 8k step 77 / 59 / 75,
// 16 x 32k 91 / 73 / 80, 128 x 128k 654 / 547 / 564.
constexpr uint32_t kSharedSlots = 512;
// Rows from which a row's pieces are joined by one group of threads: with more rows each has fewer
// pieces, and the GPU is full without dividing them. Whole calls, us, divided / not: 256 rows
// 73 / 78, 1024 59.1 / 60.0, 2048 556 / 555, 6400 129 / 121, 8192 84 / 76.
constexpr uint32_t kMergeRows = 4096;

static SharedPlan plan_of(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                          uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                          uint32_t head_dim, uint64_t* work_out = nullptr) {
  SharedPlan p{};
  p.tile = 4096 / head_dim;
  const uint64_t tile_seqs = kSharedRows / (n_heads / n_kv_heads);
  const uint64_t row_tiles = std::min(n_groups, n_seqs) + n_seqs / tile_seqs;
  auto tiles_of = [&](uint64_t keys) { return (keys + p.tile - 1) / p.tile; };
  const uint64_t tiles = row_tiles * tiles_of(max_prefix) + n_seqs * tiles_of(max_n_keys);
  p.chains = (uint32_t)(row_tiles + n_seqs);
  const uint64_t work = tiles + p.chains;
  p.max_runs = (uint32_t)std::min((uint64_t)std::max(1u, kSharedSlots / n_kv_heads), work);
  if (work_out) *work_out = work;
  return p;
}

static uint64_t list_bytes(const SharedPlan& p, uint32_t n_seqs) {
  return ws_align((p.max_runs + 1ull) * sizeof(SharedRun)) +
         ws_align((uint64_t)p.chains * sizeof(SharedChain)) +
         ws_align((uint64_t)n_seqs * sizeof(SharedRecord));
}
static uint64_t part_rows(const SharedPlan& p, uint32_t n_seqs, uint32_t n_heads,
                          uint32_t n_kv_heads) {
  return n_kv_heads * shared_parts(n_seqs * (n_heads / n_kv_heads), p.max_runs);
}

uint64_t shared_ws_bytes(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                         uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                         uint32_t head_dim) {
  const SharedPlan p = plan_of(n_groups, n_seqs, max_prefix, max_n_keys, n_heads, n_kv_heads,
                               head_dim);
  const uint64_t parts = part_rows(p, n_seqs, n_heads, n_kv_heads);
  return list_bytes(p, n_seqs) + ws_align(parts * 8) + ws_align(parts * head_dim * 4);
}

bool shared_fits(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix, uint32_t max_n_keys,
                 uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim) {
  uint64_t work;
  const SharedPlan p = plan_of(n_groups, n_seqs, max_prefix, max_n_keys, n_heads, n_kv_heads,
                               head_dim, &work);
  return work <= 0xfffffffeull && (uint64_t)p.max_runs * n_kv_heads <= kMaxGroups &&
         shared_parts(n_seqs * (n_heads / n_kv_heads), p.max_runs) <= 0xffffffffull &&
         (uint64_t)n_seqs * n_heads <= kMaxGroups;
}

template <int D>
static hipError_t launch(const SharedArgs& a, const DecodeFused* fused, uint32_t q_stride,
                         uint32_t kv_stride, void* ws, hipStream_t st) {
  SharedPlan p = plan_of(a.n_groups, a.n_seqs, a.max_prefix, a.max_n_keys, a.n_heads,
                         a.n_kv_heads, a.head_dim);
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.run = reinterpret_cast<SharedRun*>(w);
  p.chain = reinterpret_cast<SharedChain*>(w + ws_align((p.max_runs + 1ull) * sizeof(SharedRun)));
  p.record = reinterpret_cast<SharedRecord*>(
      reinterpret_cast<uint8_t*>(p.chain) + ws_align((uint64_t)p.chains * sizeof(SharedChain)));
  w += list_bytes(p, a.n_seqs);
  p.ml = reinterpret_cast<float2*>(w);
  p.acc = reinterpret_cast<float*>(
      w + ws_align(part_rows(p, a.n_seqs, a.n_heads, a.n_kv_heads) * 8));
  hipError_t e;
  if (fused != nullptr) {
    e = launch_shared_prologue(a, p, *fused, q_stride, kv_stride, st);
  } else {
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a, p);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  const float scale = (float)(kLog2e / sqrt((double)D));
  hipLaunchKernelGGL(shared_attn_kernel<D>, dim3(p.max_runs * a.n_kv_heads), dim3(kShThreads), 0,
                     st, a, p, scale);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t rows = a.n_seqs * a.n_heads;
  auto merge = [&](auto kernel, uint32_t groups) {
    const uint32_t per = 1024 / (D * groups);
    hipLaunchKernelGGL(kernel, dim3((rows + per - 1) / per), dim3(256), 0, st, a, p);
  };
  if (rows <= kMergeRows)
    merge(shared_merge_kernel<D, 1024 / D>, 1024 / D);
  else
    merge(shared_merge_kernel<D, 1>, 1);
  return hipGetLastError();
}

hipError_t launch_shared(const SharedArgs& a, const DecodeFused* fused, uint32_t q_stride,
                         uint32_t kv_stride, void* ws, hipStream_t st) {
  return a.head_dim == 128 ? launch<128>(a, fused, q_stride, kv_stride, ws, st)
                           : launch<64>(a, fused, q_stride, kv_stride, ws, st);
}

}  // namespace flk
