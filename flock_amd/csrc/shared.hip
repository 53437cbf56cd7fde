// Decode attention of sequences that share long prefixes: each sequence's token sees its
// group's prefix keys and its own, and the prefix is read once for the group.
//
// f32 keys and values meet q and the softmax weights on f16 matrix products of two parts each:
// x = h + l, h = x rounded to f16 and l = x - h likewise (22 bits), and x y = h h' + h l' +
// l h', all sums in f32. The product left out, l l', is at most 2^-22 of x y. Operands are
// scaled by powers of two first: q by its row's largest, K by its tile's largest (both
// undone in the score's factor), V by a factor that moves with its tiles' largest.
//
// An item is 128 rows of q (query heads of one kv head, of as many sequences) and a piece of
// their keys; four waves of 32 rows, two workgroups a CU. A tile of 32 keys (64 of 64-wide
// heads) of K and V comes through registers, is split there and put into LDS, in the order of
// the matrix operands, once for all rows; the next tile's loads are in flight meanwhile. S^T = K
// Q^T and O^T += V^T P^T on 32x32x16: a column is a row of q, and P^T is taken from the S^T
// accumulators as they lie, because V's keys are put in the order in which a lane holds its
// scores. Own keys are items of the sequence's few rows; waves without rows only stage.
#include <algorithm>

#include "shared.hpp"
#include "kv4_attn.hpp"

namespace flk {

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
  float top[2][2][kShThreads / 64];  // the largest |k| and |v| of a tile, by wave
};

// Two f16 parts of four values times s (a power of two), 8 bytes each.
__device__ __forceinline__ void split4(float x, float y, float z, float w, float s, uint2& hi,
                                       uint2& lo) {
  x *= s, y *= s, z *= s, w *= s;
  const halfx2 a = pack_half2(x, y), b = pack_half2(z, w);
  hi = make_uint2(as_u32(a), as_u32(b));
  lo = make_uint2(as_u32(rest_half2(x, y, a)), as_u32(rest_half2(z, w, b)));
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, xor_lane<1>(v));
  v = fmaxf(v, xor_lane<2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  v = fmaxf(v, dpp<kDppMirror>(v));
  v = max_xor<16>(v);
  return max_xor<32>(v);
}
__device__ __forceinline__ float power_of_two(int e) {  // 2^e, |e| < 127
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

template <int D>
__global__ __launch_bounds__(kShThreads, 2) void shared_attn_kernel(SharedArgs a, SharedPlan p,
                                                                   float scale_log2e) {
  constexpr int kTile = 4096 / D, kBlocks = kTile / 32, kSteps = D / 16, kOT = D / 32;
  constexpr int kChunks = D / 4;          // float4s of a row
  constexpr int kGroups = 64 / kChunks;   // rows of a load
  __shared__ SharedLds<D> sh;
  if (blockIdx.x >= *p.n_items) return;
  const SharedItem* it = p.item + blockIdx.x;
  const uint64_t key_row = it->key_row;
  const uint32_t n_keys = it->n_keys, row0 = it->row0, n_rows = it->n_rows, kvh = it->kvh;
  const uint32_t G = a.n_kv_heads, m = a.n_heads / G;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const uint32_t n_tiles = (n_keys + kTile - 1) / kTile;

  // Staging: a thread loads chunk c of four rows of K, and of four rows of V that are
  // neighbours in the operands' order of keys: of a 16-key step, lane half h holds the scores of
  // keys 4 h .. (first) and 8 + 4 h .. (second).
  const int c = lane % kChunks, gr = lane / kChunks;
  const int v_step = D == 128 ? wave >> 1 : wave;
  const int v_unit = D == 128 ? (wave & 1) + 2 * gr : gr;
  const uint32_t stride = G * D * 4;  // bytes of a cache row
  const uint32_t k_key = wave * (kTile / 4) + gr, v_key = 16 * v_step + 4 * v_unit;
  const size_t base = (key_row * G + kvh) * D;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  u4 rk[4], rv[4];
  auto fetch = [&](uint32_t tile) {
    const size_t at = base + (size_t)tile * kTile * G * D;
    const uint32_t keys = min(n_keys - tile * kTile, (uint32_t)kTile);
    const uint32_t bytes = (keys - 1) * stride + D * 4;  // rows behind the last read as zeros
    const auto ks = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.kcache + at), 0, bytes,
                                                      0x00020000);
    const auto vs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.vcache + at), 0, bytes,
                                                      0x00020000);
#pragma unroll
    for (int i = 0; i < 4; i++)
      rk[i] = __builtin_amdgcn_raw_buffer_load_b128(ks, (k_key + kGroups * i) * stride + 16 * c, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; i++)
      rv[i] = __builtin_amdgcn_raw_buffer_load_b128(vs, (v_key + i) * stride + 16 * c, 0, 0);
  };
  auto f = [](uint32_t x) { return __builtin_bit_cast(float, x); };
  auto note_top = [&](int buf) {
    float k = 0.f, v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        k = fmaxf(k, fabsf(f(rk[i][j])));
        v = fmaxf(v, fabsf(f(rv[i][j])));
      }
    k = wave_max(k), v = wave_max(v);
    if (lane == 0) sh.top[buf][0][wave] = k, sh.top[buf][1][wave] = v;
  };
  // K's and V's factors of the tile in registers. V's stays while the tile's largest value
  // lies in 2^7 .. 2^15 with it, so that accumulators seldom change theirs.
  float k_down = 0.f, v_up = 1.f;
  auto stage = [&](int buf, bool first) {
    const float4 kt = *reinterpret_cast<const float4*>(sh.top[buf][0]);
    const float4 vt = *reinterpret_cast<const float4*>(sh.top[buf][1]);
    const RowScale rs = row_scale(fmaxf(fmaxf(kt.x, kt.y), fmaxf(kt.z, kt.w)));
    k_down = rs.down;
    const float top = fmaxf(fmaxf(vt.x, vt.y), fmaxf(vt.z, vt.w)), now = top * v_up;
    if (first || !(now >= 128.f && now < 32768.f)) {
      const int e = (int)((__builtin_bit_cast(uint32_t, top) >> 23) & 255u) - 127;
      const int old = (int)((__builtin_bit_cast(uint32_t, v_up) >> 23) & 255u) - 127;
      // (2^12 .. 2^13; by at most 2^60 up, so that accumulators stay finite.)
      int up = min(12 - max(e, -100), first ? 112 : old + 60);
      if (top == 0.f && !first) up = old;
      v_up = top < INFINITY ? power_of_two(max(up, -115)) : __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint2 hi, lo;
      split4(f(rk[i][0]), f(rk[i][1]), f(rk[i][2]), f(rk[i][3]), rs.up, hi, lo);
      const uint32_t at = sh_k_at<D>(k_key + kGroups * i, c >> 1) + 8 * (c & 1);
      *reinterpret_cast<uint2*>(&sh.k[buf][0][at]) = hi;
      *reinterpret_cast<uint2*>(&sh.k[buf][1][at]) = lo;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      uint2 hi, lo;
      split4(f(rv[0][j]), f(rv[1][j]), f(rv[2][j]), f(rv[3][j]), v_up, hi, lo);
      const uint32_t at = sh_v_at<D>(j * kChunks + c, 2 * v_step + (v_unit & 1)) + 8 * (v_unit >> 1);
      *reinterpret_cast<uint2*>(&sh.v[buf][0][at]) = hi;
      *reinterpret_cast<uint2*>(&sh.v[buf][1][at]) = lo;
    }
  };

  fetch(0);
  // This wave's rows (lanes behind the last repeat it), q in two parts: dims 16 s + 8 h ..
  const bool idle = wave * 32u >= n_rows;
  const uint32_t my = row0 + min(wave * 32u + col, n_rows - 1);
  Half8 qh[kSteps], ql[kSteps];
  float c_s;
  {
    const float* src = a.q + ((size_t)(my / m) * a.n_heads + kvh * m + my % m) * D;
    float x[D / 2], amax = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float4 y = *reinterpret_cast<const float4*>(src + 16 * s + 8 * h + 4 * i);
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
      const float u = x[2 * i] * rs.up, v = x[2 * i + 1] * rs.up;
      const halfx2 hi = pack_half2(u, v);
      qh[i >> 2].u[i & 3] = as_u32(hi);
      ql[i >> 2].u[i & 3] = as_u32(rest_half2(u, v, hi));
    }
  }

  floatx16v o[kOT] = {};
  float ref = -INFINITY, l = 0.f;
  auto block = [&](int buf, int kb, float c_t, uint32_t keys) {
    floatx16v s = {};
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const uint32_t at = sh_k_at<D>(kb * 32 + col, 2 * i + h);
      const halfx8 kh = *reinterpret_cast<const halfx8*>(&sh.k[buf][0][at]);
      const halfx8 kl = *reinterpret_cast<const halfx8*>(&sh.k[buf][1][at]);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[i].h, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[i].h, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[i].h, s, 0, 0, 0);
    }
    if (keys < kTile) {
#pragma unroll
      for (int i = 0; i < 16; i++)
        s[i] = kb * 32 + 8 * (i >> 2) + 4 * h + (i & 3) < (int)keys ? s[i] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
    top *= c_t;
    if (__ballot(top > ref + kSlack)) {
      top = max_xor<32>(top);
      const float nr = fmaxf(ref, top);
      const float alpha = nr == ref ? 1.f : __builtin_amdgcn_exp2f(ref - nr);
      ref = nr;
      l *= alpha;
#pragma unroll
      for (int x = 0; x < kOT; x++) o[x] *= alpha;
    }
    const float rb = (ref == -INFINITY ? 0.f : ref) - kBias;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c_t, -rb));
      l += s[i];
    }
    Half8 ph[2], pl[2];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const halfx2 hi = pack_half2(s[2 * i], s[2 * i + 1]);
      ph[i >> 2].u[i & 3] = as_u32(hi);
      pl[i >> 2].u[i & 3] = as_u32(rest_half2(s[2 * i], s[2 * i + 1], hi));
    }
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int x = 0; x < kOT; x++) {
        const uint32_t at = sh_v_at<D>(32 * x + col, 4 * kb + 2 * ks + h);
        const halfx8 vh = *reinterpret_cast<const halfx8*>(&sh.v[buf][0][at]);
        const halfx8 vl = *reinterpret_cast<const halfx8*>(&sh.v[buf][1][at]);
        o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[ks].h, o[x], 0, 0, 0);
        o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[ks].h, o[x], 0, 0, 0);
        o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[ks].h, o[x], 0, 0, 0);
      }
  };

  note_top(0);
  lds_barrier();
  stage(0, true);
  float unit = v_up;  // of the accumulators
  if (n_tiles > 1) {
    fetch(1);
  }
  float c_t = c_s * k_down, v_now = v_up;
  if (n_tiles > 1) note_top(1);
  lds_barrier();
  for (uint32_t t = 0; t < n_tiles; t++) {
    const int buf = t & 1;
    const float c_now = c_t, u_now = v_now;
    if (t + 1 < n_tiles) {
      stage(buf ^ 1, false);
      c_t = c_s * k_down, v_now = v_up;
      if (t + 2 < n_tiles) fetch(t + 2);
    }
    if (!idle) {
      if (u_now != unit) {  // uniform
        const float alpha = u_now / unit;
#pragma unroll
        for (int x = 0; x < kOT; x++) o[x] *= alpha;
        unit = u_now;
      }
      const uint32_t keys = min(n_keys - t * kTile, (uint32_t)kTile);
#pragma unroll
      for (int kb = 0; kb < kBlocks; kb++) block(buf, kb, c_now, keys);
    }
    if (t + 2 < n_tiles) note_top(buf);
    lds_barrier();
  }
  if (idle || wave * 32u + col >= n_rows) return;
  float lo, hi;
  swap_pair<32>(l, lo, hi);
  l = lo + hi;
  const size_t at = it->part + wave * 32u + col;
  if (h == 0) p.ml[at] = make_float2(ref, l);
  const float inv = 1.f / l, down = 1.f / unit;  // (one after the other: l * unit may overflow)
  float* dst = p.acc + at * D;
  // Accumulator i of block x: row 8 (i / 4) + 4 h + i % 4 of V's 32 x .., so dim 4 (row % (D / 4))
  // + row / (D / 4).
#pragma unroll
  for (int i = 0; i < D / 8; i++) {
    const int r = 8 * (i >> 2) + 4 * h + (i & 3);
    if constexpr (D == 128)
      *reinterpret_cast<float4*>(dst + 4 * r) =
          make_float4(o[0][i] * inv * down, o[1][i] * inv * down, o[2][i] * inv * down,
                      o[3][i] * inv * down);
    else
      *reinterpret_cast<float4*>(dst + 4 * r) =
          make_float4(o[0][i] * inv * down, o[0][i + 8] * inv * down, o[1][i] * inv * down,
                      o[1][i + 8] * inv * down);
  }
}

// Joins the partial results of rows, D / 4 threads a row: o = sum w o_i / sum w, w = l 2^ref.
template <int D>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a, SharedPlan p) {
  constexpr uint32_t kRows = 1024 / D;
  const uint32_t row = blockIdx.x * kRows + threadIdx.x / (D / 4), e = threadIdx.x % (D / 4);
  if (row >= a.n_seqs * a.n_heads) return;
  const uint32_t b = row / a.n_heads, head = row % a.n_heads, G = a.n_kv_heads, m = a.n_heads / G;
  const uint32_t kvh = head / m, j = head % m;
  const SharedRecord r = p.record[b];
  float4* dst = reinterpret_cast<float4*>(a.o + (size_t)row * D) + e;
  if (r.own_n >= kSharedIdle || r.prefix_n == kSharedRefused) {
    const bool idle = r.own_n == kSharedIdle && r.prefix_n != kSharedRefused;
    const float x = idle ? 0.f : __builtin_nanf("");
    *dst = make_float4(x, x, x, x);
    return;
  }
  const uint32_t n = r.prefix_n + r.own_n;
  auto at = [&](uint32_t i) {
    return i < r.prefix_n ? (size_t)r.prefix + i * r.prefix_step + kvh * r.prefix_head + j
                          : (size_t)r.own + ((i - r.prefix_n) * G + kvh) * m + j;
  };
  float top = -INFINITY;
  for (uint32_t i = 0; i < n; i++) top = fmaxf(top, p.ml[at(i)].x);
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (uint32_t i = 0; i < n; i++) {
    const size_t x = at(i);
    const float2 ml = p.ml[x];
    const float4 y = reinterpret_cast<const float4*>(p.acc + x * D)[e];
    const float w = ml.y * __builtin_amdgcn_exp2f(ml.x - top);
    sum += w;
    f.x = fmaf(y.x, w, f.x), f.y = fmaf(y.y, w, f.y);
    f.z = fmaf(y.z, w, f.z), f.w = fmaf(y.w, w, f.w);
  }
  const float inv = n == 0 ? 0.f : 1.f / sum;
  *dst = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
}

constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(SharedArgs a, SharedPlan p) {
  shared_plan<kPlanThreads>(a, p);
}

// Two workgroups a CU.
constexpr uint32_t kSharedSlots = 512;

static SharedPlan plan_of(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                          uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                          uint32_t head_dim, uint64_t* items_out = nullptr) {
  SharedPlan p{};
  const uint64_t G = n_kv_heads, m = n_heads / n_kv_heads;
  p.tile = 4096 / head_dim;
  p.pieces = std::max(1u, kSharedSlots / n_kv_heads);
  const uint64_t rows = (uint64_t)n_seqs * m;
  const uint64_t row_tiles = std::min(n_groups, n_seqs) + rows / kSharedRows;
  auto most = [&](uint64_t keys) {  // pieces that so many keys are cut into
    const uint64_t tiles = (keys + p.tile - 1) / p.tile;
    return (tiles + kSharedLeast - 1) / kSharedLeast;
  };
  // Each piece but a row tile's last has the share of one of `pieces`.
  const uint64_t pre = std::min(p.pieces + row_tiles, row_tiles * most(max_prefix));
  const uint64_t own = std::min((uint64_t)p.pieces + n_seqs, n_seqs * most(max_n_keys));
  const uint64_t items = G * (pre + own);
  p.items = (uint32_t)std::min(items, (uint64_t)0xffffffffu);
  p.parts = G * (std::min(pre * kSharedRows, rows * std::min((uint64_t)p.pieces + 1, most(max_prefix))) +
                 own * m);
  if (items_out) *items_out = items;
  return p;
}

static uint64_t list_bytes(const SharedPlan& p, uint32_t n_seqs) {
  return 256 + ws_align((uint64_t)p.items * sizeof(SharedItem)) +
         ws_align((uint64_t)n_seqs * sizeof(SharedRecord));
}

uint64_t shared_ws_bytes(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                         uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                         uint32_t head_dim) {
  const SharedPlan p = plan_of(n_groups, n_seqs, max_prefix, max_n_keys, n_heads, n_kv_heads,
                               head_dim);
  return list_bytes(p, n_seqs) + ws_align(p.parts * 8) + ws_align(p.parts * head_dim * 4);
}

bool shared_fits(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix, uint32_t max_n_keys,
                 uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim) {
  uint64_t items;
  const SharedPlan p = plan_of(n_groups, n_seqs, max_prefix, max_n_keys, n_heads, n_kv_heads,
                               head_dim, &items);
  return items <= kMaxGroups && p.parts <= 0xffffffffull &&
         (uint64_t)n_seqs * n_heads <= kMaxGroups;
}

template <int D>
static hipError_t launch(const SharedArgs& a, const DecodeFused* fused, uint32_t q_stride,
                         uint32_t kv_stride, void* ws, hipStream_t st) {
  SharedPlan p = plan_of(a.n_groups, a.n_seqs, a.max_prefix, a.max_n_keys, a.n_heads,
                         a.n_kv_heads, a.head_dim);
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.n_items = reinterpret_cast<uint32_t*>(w);
  p.item = reinterpret_cast<SharedItem*>(w + 256);
  p.record = reinterpret_cast<SharedRecord*>(w + 256 + ws_align((uint64_t)p.items * sizeof(SharedItem)));
  w += list_bytes(p, a.n_seqs);
  p.ml = reinterpret_cast<float2*>(w);
  p.acc = reinterpret_cast<float*>(w + ws_align(p.parts * 8));
  hipError_t e;
  if (fused != nullptr) {
    e = launch_shared_prologue(a, p, *fused, q_stride, kv_stride, st);
  } else {
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a, p);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  const float scale = (float)(kLog2e / sqrt((double)D));
  hipLaunchKernelGGL(shared_attn_kernel<D>, dim3(p.items), dim3(kShThreads), 0, st, a, p, scale);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  constexpr uint32_t kRows = 1024 / D;
  hipLaunchKernelGGL(shared_merge_kernel<D>, dim3((a.n_seqs * a.n_heads + kRows - 1) / kRows),
                     dim3(256), 0, st, a, p);
  return hipGetLastError();
}

hipError_t launch_shared(const SharedArgs& a, const DecodeFused* fused, uint32_t q_stride,
                         uint32_t kv_stride, void* ws, hipStream_t st) {
  return a.head_dim == 128 ? launch<128>(a, fused, q_stride, kv_stride, ws, st)
                           : launch<64>(a, fused, q_stride, kv_stride, ws, st);
}

}  // namespace flk
