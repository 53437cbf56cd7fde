// Log probabilities of given tokens with entropy and top alternatives, and sampling from
// the alternatives. HBM-bound: a row of logits is read once. 2048 rows of 151936: 186 us, 6.7
// TB/s; 256 with 50 alternatives 32 us, 4.8 TB/s; with fewer rows two launches and the
// latency of the alternatives' second look count (64 rows: 14 + 4.6 us, one row 7.5 + 5.4).
//
// For a row x with largest value m (held c times) and R = sum of exp(x - m) over the
// others, log sum exp x = m + log(c + R); with c and R apart, log1p keeps the small
// logarithms of a row that is nearly sure. Entropy is log(c + R) + S / (c + R), S = sum
// exp(x - m) (m - x), whose terms are all positive. Alternatives are ordered by 64-bit
// keys: the value's bits in an order of unsigned numbers, then the id from the top down, so
// that ties go to the lowest id and no two keys are equal.
//
// A wave goes over its part of a row in chunks of 1024 logits with a running m, c, R and S, and
// notes each lane's largest value of each chunk. Alternatives are sought afterwards: the n_top-th
// largest of the workgroup's 256 lanes' maxima is a lower bound of the n_top-th value, few
// more values than n_top reach it, and only the lanes' chunks that hold one are read again.
// What they hold is sorted into the wave's list of 64 keys, one a lane in falling order (a
// bitonic network over the lanes). The waves of a workgroup join in LDS, and the parts of a
// row in a second launch where one workgroup would be too few.
#include "tokens.hpp"

namespace flk {

constexpr int kTokenThreads = 256, kTokenWaves = kTokenThreads / 64;
constexpr uint32_t kChunk = 1024;  // logits of a wave's step: 16 a lane
typedef unsigned long long u64;

// Larger values have larger keys; 0 for what is no alternative (-infinity, NaN).
__device__ __forceinline__ u64 token_key(float x, uint32_t id) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 as 0
  const uint32_t order = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x > -INFINITY ? (u64)order << 32 | (0xffffffffu - id) : 0;
}
__device__ __forceinline__ float key_value(u64 key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __builtin_bit_cast(float, order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint32_t key_id(u64 key) { return 0xffffffffu - (uint32_t)key; }

// ------------------------------------------------------------- lane networks --
// The value of lane ^ M; for M = 16 and 32 the pair (own, other) in any order.
template <int CTRL>
__device__ __forceinline__ uint32_t row_move(uint32_t v) {  // every lane has a source
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
template <int M>
__device__ __forceinline__ uint32_t xor_bits(uint32_t v) {
  if constexpr (M == 1) return row_move<kDppXor1>(v);
  if constexpr (M == 2) return row_move<kDppXor2>(v);
  if constexpr (M == 4) return row_move<0x1B>(row_move<kDppHalfMirror>(v));  // i ^ 7 ^ 3
  return row_move<kDppRor8>(v);
}
// One step of a network: of the two keys of lanes i and i ^ M the lane keeps the larger
// (`large`) or the smaller.
constexpr u64 lanes_without(int bit) {  // lanes whose number lacks `bit` (0: all)
  u64 m = 0;
  for (int i = 0; i < 64; i++)
    if (!(i & bit)) m |= 1ull << i;
  return m;
}
template <int M>
__device__ __forceinline__ u64 keep(u64 key, bool large) {
  u64 a, b;
  if constexpr (M >= 16) {
    const uint32_t lo = (uint32_t)key, hi = (uint32_t)(key >> 32);
    const auto swap = [](uint32_t v) {
      if constexpr (M == 16) return __builtin_amdgcn_permlane16_swap(v, v, false, false);
      else return __builtin_amdgcn_permlane32_swap(v, v, false, false);
    };
    const auto l = swap(lo), h = swap(hi);
    a = (u64)h[0] << 32 | l[0];
    b = (u64)h[1] << 32 | l[1];
  } else {
    a = key;
    b = (u64)xor_bits<M>((uint32_t)(key >> 32)) << 32 | xor_bits<M>((uint32_t)key);
  }
  return (a > b) == large ? a : b;
}
// The steps M, M / 2 .. 1; UP: the bit of lanes that end in rising order (64: none, 0: all).
template <int M, int UP>
__device__ __forceinline__ u64 merge_steps(u64 key) {
  constexpr u64 falling = UP == 0 ? 0 : lanes_without(UP);
  key = keep<M>(key, __builtin_amdgcn_inverse_ballot_w64(~(lanes_without(M) ^ falling)));
  if constexpr (M > 1) return merge_steps<M / 2, UP>(key);
  return key;
}
// 64 keys, one a lane, in rising order.
__device__ __forceinline__ u64 sort_rising(u64 key) {
  key = merge_steps<1, 2>(key);
  key = merge_steps<2, 4>(key);
  key = merge_steps<4, 8>(key);
  key = merge_steps<8, 16>(key);
  key = merge_steps<16, 32>(key);
  return merge_steps<32, 0>(key);
}
// The same of values without NaN.
template <int M, int UP>
__device__ __forceinline__ float merge_values(float v) {
  constexpr u64 falling = UP == 0 ? 0 : lanes_without(UP);
  float a = v, b;
  if constexpr (M >= 16) swap_pair<M>(v, a, b);
  else b = __builtin_bit_cast(float, xor_bits<M>(__builtin_bit_cast(uint32_t, v)));
  v = __builtin_amdgcn_inverse_ballot_w64(~(lanes_without(M) ^ falling)) ? fmaxf(a, b) : fminf(a, b);
  if constexpr (M > 1) return merge_values<M / 2, UP>(v);
  return v;
}
__device__ __forceinline__ float sort_values(float v) {
  v = merge_values<1, 2>(v);
  v = merge_values<2, 4>(v);
  v = merge_values<4, 8>(v);
  v = merge_values<8, 16>(v);
  v = merge_values<16, 32>(v);
  return merge_values<32, 0>(v);
}
__device__ __forceinline__ float join_values(float falling, float rising) {
  return merge_values<32, 64>(fmaxf(falling, rising));
}
// The 64 largest of a falling list and a rising one, falling: the larger of each lane's two
// form a sequence that rises at most once and falls at most once, which the last steps sort.
__device__ __forceinline__ u64 join(u64 falling, u64 rising) {
  return merge_steps<32, 64>(falling > rising ? falling : rising);
}
__device__ __forceinline__ u64 lane_key(u64 key, uint32_t lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(key >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)key, lane);
}
__device__ __forceinline__ float wave_top(float v) {
  v = fmaxf(v, xor_lane<1>(v));
  v = fmaxf(v, xor_lane<2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  v = fmaxf(v, dpp<kDppMirror>(v));
  v = max_xor<16>(v);
  return max_xor<32>(v);
}

// ---------------------------------------------------------------------- sums --
// A row's, or a part's: the largest value, how often, the other weights and their spread.
struct RowSums {
  float m, count, rest, spread;
  // The same against a larger m.
  __device__ __forceinline__ void move(float to) {
    if (!(to > m)) return;
    if (m == -INFINITY) {  // (nothing of weight yet)
      count = 0.f;
    } else {
      const float w = __builtin_amdgcn_exp2f((m - to) * 1.44269504f);
      rest = w * (rest + count);
      spread = fmaf(w, spread, rest * fminf(to - m, 3e38f));  // (0 of what is infinitely far)
      count = 0.f;
    }
    m = to;
  }
  __device__ __forceinline__ void add(RowSums x) {
    const float to = fmaxf(m, x.m);
    move(to), x.move(to);
    count += x.count, rest += x.rest, spread += x.spread;
  }
  __device__ __forceinline__ double log_total() const {  // log(count + rest)
    return log1p((double)(count - 1.f) + (double)rest);
  }
  __device__ __forceinline__ bool none() const {
    return !(m > -INFINITY && m < INFINITY) || isnan(rest);
  }
  __device__ __forceinline__ float logprob(float x) const {
    return none() ? __builtin_nanf("") : (float)((double)x - (double)m - log_total());
  }
  __device__ __forceinline__ float entropy() const {
    return none() ? __builtin_nanf("")
                  : (float)(log_total() + (double)spread / ((double)count + (double)rest));
  }
};

// The sums of 64 lanes with the same m.
__device__ __forceinline__ RowSums wave_sums(RowSums s) {
  s.count = group_sum<64>(s.count);
  s.rest = group_sum<64>(s.rest);
  s.spread = group_sum<64>(s.spread);
  return s;
}
// Those of lanes with different m, in every lane.
__device__ __forceinline__ RowSums wave_join(RowSums s) {
  s.move(wave_top(s.m));
  return wave_sums(s);
}

// The token that a row's settings and its number choose among its keys (a lane each,
// falling; 0: none), by one wave, in 64 bits.
__device__ __forceinline__ u64 choose(const TokenArgs& a, uint32_t row, u64 key, int lane) {
  const float t = a.temperature ? a.temperature[row] : 1.f, u = a.uniform[row];
  const float top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
  const uint32_t k = a.top_k ? a.top_k[row] : a.n_top;
  const u64 first = lane_key(key, 0);
  const bool ok = t >= 0.f && t < INFINITY && k >= 1 && k <= a.n_top && top_p > 0.f &&
                  min_p >= 0.f && min_p <= 1.f && u >= 0.f && u < 1.f;
  if (!ok || first == 0) return 0;
  if (t == 0.f) return first;
  const float x0 = key_value(first), x = key_value(key);
  double w = 0;
  if ((uint32_t)lane < k && key != 0)
    w = x == x0 ? 1.0 : exp(((double)x - (double)x0) / (double)t);
  double sum = w;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const double y = __shfl_up(sum, s, kWave);
    if (lane >= s) sum += y;
  }
  const double all = __shfl(sum, 63, kWave);
  const bool stays = w > 0 && sum - w < (double)top_p * all && w >= (double)min_p;
  const u64 gone = ~__ballot(stays);  // (the first always stays)
  const int n = gone ? __builtin_ctzll(gone) : 64;
  const double kept = __shfl(sum, n - 1, kWave);
  const u64 past = __ballot(lane < n && sum > (double)u * kept);
  return lane_key(key, past ? __builtin_ctzll(past) : n - 1);
}

// What a row's sums and keys give, by one wave.
__device__ __forceinline__ void finish(const TokenArgs& a, uint32_t row, RowSums sums, u64 key,
                                       int lane) {
  if (a.uniform != nullptr) {
    const u64 chosen = choose(a, row, key, lane);
    if (lane == 0) {
      a.token[row] = chosen ? key_id(chosen) : 0xffffffffu;
      if (a.logprob != nullptr)
        a.logprob[row] = chosen ? sums.logprob(key_value(chosen)) : __builtin_nanf("");
    }
    return;
  }
  if ((uint32_t)lane < a.n_top) {
    const size_t at = (size_t)row * a.n_top + lane;
    a.top_ids[at] = key ? key_id(key) : 0xffffffffu;
    a.top_logprobs[at] = key ? sums.logprob(key_value(key)) : -INFINITY;
  }
  if (lane != 0) return;
  if (a.logprob != nullptr) {
    const uint32_t token = a.tokens[row];
    a.logprob[row] = token < a.n_vocab ? sums.logprob(a.logits[row * a.ld + token])
                                       : __builtin_nanf("");
  }
  if (a.entropy != nullptr) a.entropy[row] = sums.entropy();
}

struct TokenParts {
  uint32_t splits;  // parts of a row: one workgroup each
  float4* sums;     // [row][part]
  u64* keys;        // [row][part][n_top], falling
};

typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));  // of a row at any float

// The next larger float (of -infinity the lowest finite).
__device__ __forceinline__ float next_up(float x) {
  const int u = __builtin_bit_cast(int, x + 0.f);
  return x < INFINITY ? __builtin_bit_cast(float, u >= 0 ? u + 1 : u - 1) : __builtin_nanf("");
}

// grid (parts, rows); kSegment: chunks of a wave between two looks at the alternatives
template <bool TOP, bool ENTROPY, uint32_t kSegment>
__global__ __launch_bounds__(kTokenThreads) void token_rows_kernel(TokenArgs a, TokenParts p) {
  struct Lds {
    float top[kSegment][64];     // each lane's largest value of a chunk
    float best[64];              // each lane's largest of a segment, sorted
    uint32_t chunk[64];          // lanes of chunks to look at again: 64 chunk + lane
    u64 key[64 + 256];           // alternatives, with room for four values a lane
  };
  __shared__ Lds s_lds[TOP ? kTokenWaves : 1];
  __shared__ u64 s_list[TOP ? kTokenWaves : 1][64];
  __shared__ float4 s_sums[kTokenWaves];
  const uint32_t row = blockIdx.y, part = blockIdx.x;
  const float* x = a.logits + row * a.ld;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t chunks = (a.n_vocab + kChunk - 1) / kChunk;
  const uint32_t of = p.splits * kTokenWaves, me = part * kTokenWaves + wave;
  const uint32_t c0 = (uint32_t)((u64)chunks * me / of), c1 = (uint32_t)((u64)chunks * (me + 1) / of);
  Lds& lds = s_lds[TOP ? wave : 0];

  // (Without a second look a row need not stay in the caches: 2048 rows of 151936 186 us, 210
  // with ordinary loads. With one, a row that is still there counts: 256 rows 32 us, 36.)
  auto load = [&](uint32_t chunk, uint32_t l, float (&v)[16]) {
    const uint32_t i0 = chunk * kChunk + 4 * l;
    if ((u64)(chunk + 1) * kChunk <= a.n_vocab) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const Float4* from = reinterpret_cast<const Float4*>(x + i0 + 256 * i);
        const Float4 f = TOP ? *from : __builtin_nontemporal_load(from);
        v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const uint32_t id = i0 + 256 * (i >> 2) + (i & 3);
        v[i] = id < a.n_vocab ? x[id] : -INFINITY;
      }
    }
  };
  RowSums s{-INFINITY, 0.f, 0.f, 0.f};
  float best = -INFINITY;  // of the lane, in this segment
  auto take = [&](const float (&v)[16], uint32_t at) {
    float top = v[0];  // (NaN is passed over: it makes the sums NaN)
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, v[i]);
    if constexpr (TOP) {
      lds.top[at][lane] = top;
      best = fmaxf(best, top);
    }
    const bool largest = __ballot(!(top < s.m)) != 0;
    if (largest) s.move(wave_top(top));
    const float m = fmaxf(s.m, -3.40282347e38f);  // (against it -infinity has a weight of 0)
    if (largest) {  // it is in this chunk: counted apart
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float d = m - v[i], e = __builtin_amdgcn_exp2f(d * -1.44269504f);
        s.count += d == 0.f ? 1.f : 0.f;
        s.rest += d == 0.f ? 0.f : e;
        if constexpr (ENTROPY) s.spread = fmaf(e, fminf(d, 3e38f), s.spread);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float d = m - v[i], e = __builtin_amdgcn_exp2f(d * -1.44269504f);
        s.rest += e;
        if constexpr (ENTROPY) s.spread = fmaf(e, fminf(d, 3e38f), s.spread);
      }
    }
  };

  u64 list = 0;                       // falling
  float own = next_up(-INFINITY);     // above the list's n_top-th value
  auto kth = [&](float falling) {     // of 64 values
    return __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, falling), a.n_top - 1));
  };
  // All waves go through as many segments (some of them empty ones), for their barriers.
  const uint32_t per_wave = (chunks + of - 1) / of;
  for (uint32_t g0 = c0, seg = 0; TOP ? seg < per_wave : seg == 0; g0 += kSegment, seg += kSegment) {
    const uint32_t g1 = TOP ? min(g0 + kSegment, max(c1, g0)) : c1;
    float v[16], w[16];
    if (g0 < g1) load(g0, lane, v);
    for (uint32_t c = g0; c < g1; c += 2) {
      if (c + 1 < g1) load(c + 1, lane, w);
      take(v, c - g0);
      if (c + 1 < g1) {
        if (c + 2 < g1) load(c + 2, lane, v);
        take(w, c + 1 - g0);
      }
    }
    if constexpr (TOP) {
      // The n_top-th of the workgroup's 256 lanes' largest values: as many values are not below
      // it, so that none below it is an alternative.
      float sorted = sort_values(best);  // rising
      lds.best[lane] = sorted;
      __syncthreads();
      float all = lds.best[63 - lane];
#pragma unroll
      for (int i = 1; i < kTokenWaves; i++)
        all = join_values(all, s_lds[(wave + i) % kTokenWaves].best[lane]);
      const float bound = kth(all);
      float from = fmaxf(bound, own);
      uint32_t n = 0;  // lanes of chunks to look at again
      auto look = [&] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float v[16];
        uint32_t code = 0;
        if ((uint32_t)lane < n) {
          code = lds.chunk[lane];
          load(g0 + code / 64, code % 64, v);
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) v[i] = __builtin_nanf("");
        }
        const uint32_t id0 = (g0 + code / 64) * kChunk + 4 * (code % 64);
        uint32_t waiting = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const u64 mask = __ballot(v[i] >= from);
          if (mask) {
            const uint32_t before = __builtin_amdgcn_mbcnt_hi(
                (uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
            if (v[i] >= from)
              lds.key[waiting + before] = token_key(v[i], id0 + 256 * (i >> 2) + (i & 3));
            waiting += __popcll(mask);
          }
          if (i % 4 == 3 && (waiting >= 64 || i == 15)) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (uint32_t k = 0; k < waiting; k += 64)
              list = join(list, sort_rising(k + lane < waiting ? lds.key[k + lane] : 0));
            waiting = 0;
          }
        }
        // Ids rise from chunk to chunk, so a later value has to exceed the n_top-th to
        // displace it. (Chunks are looked at whole: within one, ids don't come in order.)
        const u64 last = lane_key(list, a.n_top - 1);
        if (last) own = next_up(key_value(last));
        from = fmaxf(bound, own);
        n = 0;
      };
      for (uint32_t c = g0; c < g1; c++) {
        const bool again = lds.top[c - g0][lane] >= from;
        const u64 mask = __ballot(again);
        if (mask == 0) continue;
        if (n + __popcll(mask) > 64) {
          look();
          c--;  // (with the new bound)
          continue;
        }
        if (again)
          lds.chunk[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                  __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] =
              64 * (c - g0) + lane;
        n += __popcll(mask);
      }
      if (n > 0) look();
      best = -INFINITY;
      __syncthreads();  // s_lds.best is read by all
    }
  }
  s = wave_sums(s);
  if (lane == 0) s_sums[wave] = make_float4(s.m, s.count, s.rest, s.spread);
  if constexpr (TOP) s_list[wave][lane] = list;
  __syncthreads();
  if (wave != 0) return;
  for (int i = 1; i < kTokenWaves; i++) {
    const float4 y = s_sums[i];
    s.add(RowSums{y.x, y.y, y.z, y.w});
    if constexpr (TOP) list = join(list, s_list[TOP ? i : 0][63 - lane]);
  }
  if (p.splits == 1) {
    finish(a, row, s, list, lane);
    return;
  }
  const size_t at = (size_t)row * p.splits + part;
  if (lane == 0) p.sums[at] = make_float4(s.m, s.count, s.rest, s.spread);
  if (TOP && (uint32_t)lane < a.n_top) p.keys[at * a.n_top + lane] = list;
}

// A row's parts, by one workgroup: each wave joins every fourth.
template <bool TOP>
__global__ __launch_bounds__(kTokenThreads) void token_join_kernel(TokenArgs a, TokenParts p) {
  __shared__ u64 s_list[TOP ? kTokenWaves : 1][64];
  const uint32_t row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t at = (size_t)row * p.splits;
  u64 list = 0;
  if constexpr (TOP) {
    const uint32_t from = 63 - lane;  // rising
    auto part = [&](uint32_t i) {
      return from < a.n_top && i < p.splits ? p.keys[(at + i) * a.n_top + from] : 0;
    };
    for (uint32_t i = wave; i < p.splits; i += 4 * kTokenWaves) {
      u64 key[4];
#pragma unroll
      for (int k = 0; k < 4; k++) key[k] = part(i + k * kTokenWaves);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (i + k * kTokenWaves < p.splits) list = join(list, key[k]);
    }
    s_list[wave][lane] = list;
    __syncthreads();
  }
  if (wave != 0) return;
  if constexpr (TOP)
    for (int i = 1; i < kTokenWaves; i++) list = join(list, s_list[TOP ? i : 0][63 - lane]);
  RowSums s{-INFINITY, 0.f, 0.f, 0.f};
  for (uint32_t i = lane; i < p.splits; i += 64) {
    const float4 y = p.sums[at + i];
    s.add(RowSums{y.x, y.y, y.z, y.w});
  }
  finish(a, row, wave_join(s), list, lane);
}

// Rows are cut where a workgroup each would leave CUs idle, into parts of two chunks a wave at
// least. (With alternatives two of their workgroups fit a CU: 512 are one round of the GPU, 1024
// two.) Calls, us, cut into 256 / 512 / 1024 workgroups: 64 rows of 151936 18.8 / 17.6 / 24.7,
// 100 of 50021 16.1 / 15.2 / 19.2; 256 rows of 151936, uncut / in four 32.4 / 40.7. One row, its
// parts of one chunk a wave at least / two / four: 14.2 / 13.1 / 13.5.
constexpr uint32_t kTokenGroups = 512, kTokenLeast = 2;
static uint32_t token_splits(uint32_t n_rows, uint32_t n_vocab) {
  const uint32_t part = kChunk * kTokenWaves * kTokenLeast;
  const uint32_t most = n_vocab / part + (n_vocab % part != 0);
  const uint32_t wanted = n_rows < 256 ? kTokenGroups / n_rows : 1;
  return wanted < most ? wanted : most;
}

static uint64_t parts_bytes(uint64_t parts, uint32_t n_top) {
  return ws_align(parts * sizeof(float4)) + parts * n_top * sizeof(u64);
}
uint64_t tokens_need(uint32_t n_rows, uint32_t n_vocab, uint32_t n_top) {
  const uint32_t splits = token_splits(n_rows, n_vocab);
  return splits == 1 ? 0 : parts_bytes((uint64_t)n_rows * splits, n_top);
}
// For every number of rows up to n_rows.
uint64_t tokens_ws_bytes(uint32_t n_rows, uint32_t n_vocab, uint32_t n_top) {
  const uint64_t most = (uint64_t)n_rows * token_splits(1, n_vocab);
  return most == n_rows ? 0 : parts_bytes(most < kTokenGroups ? most : kTokenGroups, n_top);
}

hipError_t launch_tokens(const TokenArgs& a, void* ws, hipStream_t st) {
  TokenParts p{};
  p.splits = token_splits(a.n_rows, a.n_vocab);
  if (p.splits > 1) {
    p.sums = static_cast<float4*>(ws);
    p.keys = reinterpret_cast<u64*>(static_cast<char*>(ws) +
                                    ws_align((uint64_t)a.n_rows * p.splits * sizeof(float4)));
  }
  // (Grid y holds 65535 rows.)
  for (uint32_t r = 0; r < a.n_rows; r += 65535) {
    TokenArgs b = a;
    b.n_rows = a.n_rows - r < 65535 ? a.n_rows - r : 65535;
    if (r > 0) {
      b.logits += r * a.ld;
      if (b.tokens) b.tokens += r;
      if (b.logprob) b.logprob += r;
      if (b.entropy) b.entropy += r;
      if (b.top_ids) b.top_ids += (size_t)r * a.n_top, b.top_logprobs += (size_t)r * a.n_top;
      if (b.temperature) b.temperature += r;
      if (b.top_k) b.top_k += r;
      if (b.top_p) b.top_p += r;
      if (b.min_p) b.min_p += r;
      if (b.uniform) b.uniform += r, b.token += r;
    }
    const dim3 grid(p.splits, b.n_rows), threads(kTokenThreads);
    // Long segments look again seldom, short ones leave LDS for four workgroups a CU instead of
    // two (34880 and 55360 bytes). us, segments of 40 / 20: 256 rows of 151936, 50 alternatives 32.4 / 37, 600 of 65000
    // 44.3 / 35.1, 2048 of 151936 230 / 222.
    const bool entropy = a.entropy != nullptr, few = a.n_rows < 512;
    const auto kernel =
        a.n_top == 0 ? (entropy ? token_rows_kernel<false, true, 1> : token_rows_kernel<false, false, 1>)
        : few ? (entropy ? token_rows_kernel<true, true, 40> : token_rows_kernel<true, false, 40>)
              : (entropy ? token_rows_kernel<true, true, 20> : token_rows_kernel<true, false, 20>);
    hipLaunchKernelGGL(kernel, grid, threads, 0, st, b, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.splits == 1) return hipSuccess;
  if (a.n_top > 0)
    hipLaunchKernelGGL(token_join_kernel<true>, dim3(a.n_rows), dim3(kTokenThreads), 0, st, a, p);
  else
    hipLaunchKernelGGL(token_join_kernel<false>, dim3(a.n_rows), dim3(kTokenThreads), 0, st, a, p);
  return hipGetLastError();
}

}  // namespace flk
