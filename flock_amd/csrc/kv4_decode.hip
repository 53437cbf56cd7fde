// Attention of a few queries a sequence over the paged 4-bit cache (single tokens,
// drafts), split over the keys. HBM-bound: 9/16 byte a value, each read once for the
// query-head rows of a kv head.
//
// A wave takes 32-key tiles. S^T = K Q^T and O^T += V^T P^T on 16x16x32 f16 MFMA: the
// 16 columns are 8 query-head rows in two f16 parts each (22 bits), so the parts
// ride in columns that the few rows would leave empty. The cache's layout gives each
// lane its operands in 16-byte pieces, and P^T is taken from the S^T accumulators as
// they lie (a lane's scores are of the tokens whose values it holds).
#include "kv4_attn.hpp"

namespace flk {

constexpr int kDecWaves = 4;

template <int D>
struct TileRegs {
  uint4 k[D / 64], v[D / 64], vs;
  uint32_t ks;
};

// Every load of a tile is relative to its first byte, which is uniform: buffer loads
// take that in scalar registers and leave one 32-bit offset a lane for each part.
constexpr int kBufferWord3 = 0x00020000;  // untyped
constexpr int kNonTemporal = 2;
struct TileOffsets {
  int k, ks, v, vs;
};
template <int D>
__device__ __forceinline__ TileOffsets tile_offsets(int lane) {
  const int n = lane & 15, kg = lane >> 4;
  return {(n * 4 + kg) * 16,
          Kv4<D>::kKScale + (n * Kv4<D>::kBlocks + (D == 128 ? kg : kg >> 1)) * 4, lane * 16,
          (kg * Kv4<D>::kBlocks + n * (D / 16) / 32) * 16};
}
template <int D>
__device__ __forceinline__ void load_tile(TileRegs<D>& t, const uint8_t* base,
                                          const TileOffsets& at) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0,
                                                      Kv4<D>::kTileBytes, kBufferWord3);
  auto load16 = [&](int lane_at, int offset) {
    const u4 v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, lane_at, offset, kNonTemporal);
    return make_uint4(v[0], v[1], v[2], v[3]);
  };
#pragma unroll
  for (int c = 0; c < D / 64; c++) t.k[c] = load16(at.k + c * 1024, 0);
  t.ks = __builtin_amdgcn_raw_buffer_load_b32(rsrc, at.ks, 0, kNonTemporal);
  t.vs = load16(at.vs, Kv4<D>::kVScale);
#pragma unroll
  for (int c = 0; c < D / 64; c++) t.v[c] = load16(at.v, Kv4<D>::kV + c * 1024);
}

template <int D, int NT>
__global__ __launch_bounds__(kDecWaves * 64, 4 / NT) void kv4_decode_kernel(
    Kv4AttnArgs a, Kv4SplitPlan plan, Kv4Part part, float scale_log2e) {
  constexpr int kRows = 8 * NT, kSteps = D / 32, kOT = D / 16;
  __shared__ float s_o[kDecWaves][kRows][D + 4];
  __shared__ float s_m[kDecWaves][kRows], s_l[kDecWaves][kRows];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  const uint32_t G = a.s.n_kv_heads, group = a.n_heads / G;
  uint32_t id = blockIdx.x;
  const uint32_t kvh = id % G;
  id /= G;
  const uint32_t rt = id % plan.row_tiles;
  id /= plan.row_tiles;
  const uint32_t b = id % a.n_seqs, split = id / a.n_seqs;

  const Kv4Seq seq = kv4_seq(a, b);
  const uint32_t rows = seq.nq * group;  // of the (sequence, kv head)
  if (seq.refused) {
    if (rt == 0 && split == 0)
      for (uint32_t i = threadIdx.x; i < rows * D; i += blockDim.x) {
        const uint32_t r = i / D;
        a.o[((size_t)(seq.q0 + r / group) * a.n_heads + kvh * group + r % group) * D + i % D] =
            __builtin_nanf("");
      }
    return;
  }
  const uint32_t r0 = rt * kRows;
  if (r0 >= rows) return;
  const uint32_t n_rows = min((uint32_t)kRows, rows - r0);
  const int64_t pos0 = (int64_t)seq.n_keys - seq.nq;
  const int64_t first = pos0 + r0 / group, last = pos0 + (r0 + n_rows - 1) / group;
  const Kv4Span span(first, last, a.window, a.n_sinks);
  const Kv4Pieces pc = kv4_pieces(span.tiles.count(), plan.most);
  if (split >= pc.n) return;
  const uint32_t t0 = split * pc.per, t1 = min(t0 + pc.per, span.tiles.count());

  // q: column col of column tile nt is part col & 1 of row 8 nt + col / 2.
  Half8 q[NT][kSteps];
  float c_s[NT];
  int delta[NT];  // the row's position behind the first
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const uint32_t r = min(r0 + 8 * nt + (col >> 1), rows - 1);
    delta[nt] = (int)(r / group - r0 / group);
    const float4* src = reinterpret_cast<const float4*>(
        a.q + ((size_t)(seq.q0 + r / group) * a.n_heads + kvh * group + r % group) * D +
        kg * (D / 4));
    float x[D / 4];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
      const float4 f = src[i];
      x[4 * i] = f.x, x[4 * i + 1] = f.y, x[4 * i + 2] = f.z, x[4 * i + 3] = f.w;
#pragma unroll
      for (int j = 0; j < 4; j++) amax = fmaxf(amax, fabsf(x[4 * i + j]));
    }
    amax = max_xor<16>(amax);
    amax = max_xor<32>(amax);
    const RowScale rs = row_scale(amax);
    c_s[nt] = rs.down * scale_log2e;
#pragma unroll
    for (int i = 0; i < D / 8; i++) {
      const float u = x[2 * i] * rs.up, v = x[2 * i + 1] * rs.up;
      const halfx2 hi = pack_half2(u, v);
      const halfx2 lo = rest_half2(u, v, hi);
      q[nt][i >> 2].u[i & 3] = as_u32(col & 1 ? lo : hi);
    }
  }

  floatx4v o[NT][kOT] = {};
  float m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) m[nt] = -INFINITY, l[nt] = 0.f;

  const uint32_t log_page = 31 - __builtin_clz(a.s.page);  // 5 .. 8
  const uint32_t* row = a.table + (size_t)b * a.max_blocks;
  const size_t tile_bytes = Kv4<D>::kTileBytes;
  const uint32_t n_it = t0 + wave < t1 ? (t1 - t0 - wave + kDecWaves - 1) / kDecWaves : 0;
  auto index = [&](uint32_t it) { return span.tiles.tile(t0 + wave + it * kDecWaves); };
  // Page ids come through the scalar cache: a vector load would have the wait for it
  // also wait for the tiles in flight.
  auto page_of = [&](uint32_t it) {
    typedef const __attribute__((address_space(4))) uint32_t* ConstPtr;
    return *(ConstPtr)(uintptr_t)(row + (index(it) >> (log_page - 5)));
  };
  auto base_of = [&](uint32_t it, uint32_t id) {
    id = id >= a.s.n_pages ? 0 : id;
    const uint32_t in = index(it) & ((a.s.page >> 5) - 1);
    return a.pool + ((((size_t)id * G + kvh) << (log_page - 5)) + in) * tile_bytes;
  };

  auto work = [&](const TileRegs<D>& t, uint32_t it, bool bad) {
    const bool whole = span.whole(index(it));
    // S^T of the two halves.
    const halfx2 ks = bad ? as_half2(0x7e007e00u) : as_half2(t.ks);
    const halfx2 d0 = {ks[0], ks[0]}, d1 = {ks[1], ks[1]};
    floatx4v s[NT][2] = {};
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(&t.k[0]);
        const uint32_t w = D == 128 ? kw[4 * h + i] : kw[2 * h + i];
        const halfx2 d = h ? d1 : d0;
        Half8 k;
        k.u[0] = as_u32(kv4_pair<0>(w, d));
        k.u[1] = as_u32(kv4_pair<1>(w, d));
        k.u[2] = as_u32(kv4_pair<2>(w, d));
        k.u[3] = as_u32(kv4_pair<3>(w, d));
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
          s[nt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.h, q[nt][i].h, s[nt][h], 0, 0, 0);
      }
    }
    uint4 vs = t.vs;
    Half8 p[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float x[8];
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[i] = s[nt][i >> 2][i & 3];
        x[i] += dpp<kDppXor1>(x[i]);
      }
      if (!whole) {
        const Kv4Mask mask = span.mask(index(it));
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[i] = mask.sees(16 * (i >> 2) + 4 * kg + (i & 3), delta[nt]) ? x[i] : -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; i++) top = fmaxf(top, x[i]);
      top *= c_s[nt];
      if (__ballot(top > m[nt] + kSlack)) {
        top = max_xor<16>(top);
        top = max_xor<32>(top);
        const float nm = fmaxf(m[nt], top);
        const float alpha = nm == m[nt] ? 1.f : __builtin_amdgcn_exp2f(m[nt] - nm);
        m[nt] = nm;
        l[nt] *= alpha;
#pragma unroll
        for (int c = 0; c < kOT; c++) o[nt][c] *= alpha;
      }
      const float mb = (m[nt] == -INFINITY ? 0.f : m[nt]) - kBias;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c_s[nt], -mb));
        l[nt] += x[i];
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const halfx2 hi = pack_half2(x[2 * i], x[2 * i + 1]);
        const halfx2 lo = rest_half2(x[2 * i], x[2 * i + 1], hi);
        p[nt].u[i] = as_u32(col & 1 ? lo : hi);
      }
    }
    if (!whole) {
      // Values of keys that some row does not see: scales that are no numbers (NaN
      // blocks, memory never written) count as 0 in the products, and make NaN of the
      // rows that do see them.
      Half8 flag;
      uint32_t* w = reinterpret_cast<uint32_t*>(&vs);
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const bool lo = (w[i] & 0x7c00u) == 0x7c00u, hi = (w[i] & 0x7c000000u) == 0x7c000000u;
        flag.u[i] = (lo ? 0x3c00u : 0u) | (hi ? 0x3c000000u : 0u);
        w[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
        any |= lo || hi;
      }
      if (__ballot(any)) {
        const Kv4Mask mask = span.mask(index(it));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          Half8 sees;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            sees.u[i] = 0;
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const int u = 2 * i + j;
              if (mask.sees(16 * (u >> 2) + 4 * kg + (u & 3), delta[nt]))
                sees.u[i] |= 0x3c00u << (16 * j);
            }
          }
          floatx4v count = {};
          count = __builtin_amdgcn_mfma_f32_16x16x32_f16(flag.h, sees.h, count, 0, 0, 0);
#pragma unroll
          for (int c = 0; c < kOT; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (count[i] > 0.f) o[nt][c][i] = __builtin_nanf("");
        }
      }
    }
    const halfx2 sv[4] = {as_half2(vs.x), as_half2(vs.y), as_half2(vs.z), as_half2(vs.w)};
#pragma unroll
    for (int c = 0; c < D / 64; c++) {
      const uint32_t w[4] = {t.v[c].x, t.v[c].y, t.v[c].z, t.v[c].w};
      Half8 v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        v[0].u[i] = as_u32(kv4_pair<0>(w[i], sv[i]));
        v[1].u[i] = as_u32(kv4_pair<1>(w[i], sv[i]));
        v[2].u[i] = as_u32(kv4_pair<2>(w[i], sv[i]));
        v[3].u[i] = as_u32(kv4_pair<3>(w[i], sv[i]));
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
          o[nt][4 * c + j] =
              __builtin_amdgcn_mfma_f32_16x16x32_f16(v[j].h, p[nt].h, o[nt][4 * c + j], 0, 0, 0);
    }
  };

  if (n_it > 0) {
    TileRegs<D> x, y;
    const TileOffsets at = tile_offsets<D>(lane);
    uint32_t id_x = page_of(0), id_y = page_of(min(1u, n_it - 1));
    load_tile<D>(x, base_of(0, id_x), at);
    for (uint32_t it = 0; it < n_it; it += 2) {
      // Past the end the last tile is read once more (an L2 hit) and not used.
      const uint32_t n1 = min(it + 1, n_it - 1), n2 = min(it + 2, n_it - 1);
      load_tile<D>(y, base_of(n1, id_y), at);
      const uint32_t id_2 = page_of(n2), id_3 = page_of(min(it + 3, n_it - 1));
      work(x, it, id_x >= a.s.n_pages);
      if (it + 1 >= n_it) break;
      load_tile<D>(x, base_of(n2, id_2), at);
      work(y, it + 1, id_y >= a.s.n_pages);
      id_x = id_2, id_y = id_3;
    }
  }

  // The waves' states into LDS: row 8 nt + col / 2 (both parts added), dims
  // (D / 16) (4 kg + i) + 4 c + j.
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    float sum = sum_xor<16>(l[nt]);
    sum = sum_xor<32>(sum);
    const int r = 8 * nt + (col >> 1);
    if ((col & 1) == 0 && kg == 0) s_m[wave][r] = m[nt], s_l[wave][r] = sum;
#pragma unroll
    for (int c = 0; c < D / 64; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f[j] = o[nt][4 * c + j][i];
          f[j] += dpp<kDppXor1>(f[j]);
        }
        if ((col & 1) == 0)
          *reinterpret_cast<float4*>(&s_o[wave][r][(D / 16) * (4 * kg + i) + 4 * c]) =
              make_float4(f[0], f[1], f[2], f[3]);
      }
  }
  __syncthreads();
  const size_t slot = ((size_t)b * plan.row_tiles + rt) * G + kvh;
  for (uint32_t i = threadIdx.x; i < n_rows * (D / 4); i += blockDim.x) {
    const uint32_t r = i / (D / 4), e = 4 * (i % (D / 4));
    float top = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kDecWaves; w++) top = fmaxf(top, s_m[w][r]);
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWaves; w++) {
      // A wave without a visible key holds zeros (or NaN: kept).
      const float k = s_m[w][r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s_m[w][r] - top);
      const float4 g = *reinterpret_cast<const float4*>(&s_o[w][r][e]);
      f.x = fmaf(g.x, k, f.x), f.y = fmaf(g.y, k, f.y);
      f.z = fmaf(g.z, k, f.z), f.w = fmaf(g.w, k, f.w);
      sum = fmaf(s_l[w][r], k, sum);
    }
    if (pc.n == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      f.x *= inv, f.y *= inv, f.z *= inv, f.w *= inv;
      const uint32_t rr = r0 + r;
      *reinterpret_cast<float4*>(
          a.o + ((size_t)(seq.q0 + rr / group) * a.n_heads + kvh * group + rr % group) * D + e) = f;
    } else {
      const size_t at = (slot * plan.splits + split) * kRows + r;
      if (e == 0) part.ml[2 * at] = top, part.ml[2 * at + 1] = sum;
      *reinterpret_cast<float4*>(part.acc + at * D + e) = f;
    }
  }
}

// Joins the pieces of a row: a workgroup per row, D / 4 threads over its dims and the
// pieces dealt out to the 1024 / D groups of them (a long context has a hundred).
template <int D>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Kv4AttnArgs a, Kv4SplitPlan plan,
                                                        Kv4Part part) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float4 s_acc[kGroups][kLanes];
  __shared__ float s_sum[kGroups];
  const uint32_t G = a.s.n_kv_heads, group = a.n_heads / G;
  const int lane = threadIdx.x & 63;
  const uint32_t r = blockIdx.x % plan.rows, slot = blockIdx.x / plan.rows;
  const uint32_t kvh = slot % G, rt = slot / G % plan.row_tiles, b = slot / G / plan.row_tiles;
  const Kv4Seq seq = kv4_seq(a, b);
  const uint32_t rows = seq.nq * group, r0 = rt * plan.rows, rr = r0 + r;
  if (seq.refused || rr >= rows) return;
  const uint32_t n_rows = min(plan.rows, rows - r0);
  const int64_t pos0 = (int64_t)seq.n_keys - seq.nq;
  const Kv4Tiles tiles = kv4_tiles(pos0 + r0 / group, pos0 + (r0 + n_rows - 1) / group, a.window,
                                   a.n_sinks);
  const uint32_t n = kv4_pieces(tiles.count(), plan.most).n;
  if (n == 1) return;
  const size_t at = (size_t)slot * plan.splits * plan.rows + r;
  const float2* ml = reinterpret_cast<const float2*>(part.ml) + at;
  float top = -INFINITY;
  for (uint32_t i = lane; i < n; i += 64) top = fmaxf(top, ml[(size_t)i * plan.rows].x);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, shfl_xor(top, x));
  const uint32_t e = threadIdx.x % kLanes, g = threadIdx.x / kLanes;
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (uint32_t i = g; i < n; i += kGroups) {
    const float2 x = ml[(size_t)i * plan.rows];
    const float4 y = reinterpret_cast<const float4*>(part.acc + (at + (size_t)i * plan.rows) * D)[e];
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
  float4* dst = reinterpret_cast<float4*>(
      a.o + ((size_t)(seq.q0 + rr / group) * a.n_heads + kvh * group + rr % group) * D);
  dst[e] = make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
}

// Key tiles of a piece: few enough that the pieces of the call's bounds fill the
// 256 CUs with four workgroups each a few times over (sequences are shorter than
// the bound), and two a wave at least.
constexpr uint32_t kDecTarget = 4096, kDecAlone = 1024, kDecFew = 2 * kDecWaves;

Kv4SplitPlan kv4_decode_plan(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                             uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                             uint32_t window, uint32_t n_sinks) {
  Kv4SplitPlan p;
  const uint32_t group = n_heads / n_kv_heads;
  const uint64_t rows = (uint64_t)max_q * group;
  p.rows = rows <= 8 ? 8 : 16;
  p.row_tiles = (uint32_t)((rows + p.rows - 1) / p.rows);
  const uint32_t tiles = kv4_max_tiles(max_n_keys, (p.rows + group - 1) / group + 1, window, n_sinks);
  const uint64_t items = (uint64_t)n_seqs * n_kv_heads * p.row_tiles;
  const uint32_t target = n_seqs == 1 ? kDecAlone : kDecTarget;
  const uint64_t most = (items * tiles + target - 1) / target;
  p.most = (uint32_t)(most < kDecFew ? kDecFew : most > 0xffffffffu ? 0xffffffffu : most);
  p.splits = (tiles + p.most - 1) / p.most;
  p.ws_bytes = p.splits == 1 ? 0
                             : ws_align(items * p.splits * p.rows * 8) +
                                   ws_align(items * p.splits * p.rows * head_dim * 4);
  return p;
}

template <int D>
static hipError_t launch(const Kv4AttnArgs& a, const Kv4SplitPlan& p, void* ws, hipStream_t st) {
  const uint64_t items = (uint64_t)a.n_seqs * a.s.n_kv_heads * p.row_tiles;
  if (items * p.splits > 0x7fffffffull || items * p.rows > 0x7fffffffull)
    return hipErrorInvalidConfiguration;
  const Kv4Part part = kv4_part(ws, p, items);
  const float scale = (float)(1.44269504088896340736 / sqrt((double)D));
  const dim3 grid((uint32_t)(items * p.splits)), block(kDecWaves * 64);
  if (p.rows == 8)
    hipLaunchKernelGGL((kv4_decode_kernel<D, 1>), grid, block, 0, st, a, p, part, scale);
  else
    hipLaunchKernelGGL((kv4_decode_kernel<D, 2>), grid, block, 0, st, a, p, part, scale);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  return launch_kv4_merge(a, p, part, st);
}

hipError_t launch_kv4_merge(const Kv4AttnArgs& a, const Kv4SplitPlan& p, const Kv4Part& part,
                            hipStream_t st) {
  const uint32_t rows = a.n_seqs * a.s.n_kv_heads * p.row_tiles * p.rows;
  if (a.s.head_dim == 128)
    hipLaunchKernelGGL(kv4_merge_kernel<128>, dim3(rows), dim3(256), 0, st, a, p, part);
  else
    hipLaunchKernelGGL(kv4_merge_kernel<64>, dim3(rows), dim3(256), 0, st, a, p, part);
  return hipGetLastError();
}

hipError_t launch_kv4_decode(const Kv4AttnArgs& a, const Kv4SplitPlan& p, void* ws,
                             hipStream_t st) {
  return a.s.head_dim == 128 ? launch<128>(a, p, ws, st) : launch<64>(a, p, ws, st);
}

}  // namespace flk
