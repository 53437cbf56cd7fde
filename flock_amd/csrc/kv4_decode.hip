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

struct Kv4Part {
  float* ml;   // [slot][rows] pairs (m, l)
  float* acc;  // [slot][rows][D]
};

template <int D>
struct TileRegs {
  uint4 k[D / 64], v[D / 64], vs;
  uint32_t ks;
};

__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

template <int D>
__device__ __forceinline__ void load_tile(TileRegs<D>& t, const uint8_t* base, int lane) {
  const int n = lane & 15, kg = lane >> 4;
#pragma unroll
  for (int c = 0; c < D / 64; c++) {
    t.k[c] = load16(base + c * 1024 + (n * 4 + kg) * 16);
    t.v[c] = load16(base + Kv4<D>::kV + c * 1024 + (kg * 16 + n) * 16);
  }
  t.ks = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(
      base + Kv4<D>::kKScale + (n * Kv4<D>::kBlocks + (D == 128 ? kg : kg >> 1)) * 4));
  t.vs = load16(base + Kv4<D>::kVScale + (kg * Kv4<D>::kBlocks + n * (D / 16) / 32) * 16);
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
  const Kv4Tiles tiles = kv4_tiles(first, last, a.window, a.n_sinks);
  const Kv4Pieces pc = kv4_pieces(tiles.count(), plan.most);
  if (split >= pc.n) return;
  const uint32_t t0 = split * pc.per, t1 = min(t0 + pc.per, tiles.count());

  // q: column col of column tile nt is part col & 1 of row 8 nt + col / 2.
  Half8 q[NT][kSteps];
  float c_s[NT];
  int64_t pos[NT];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const uint32_t r = min(r0 + 8 * nt + (col >> 1), rows - 1);
    pos[nt] = pos0 + r / group;
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
      const halfx2 lo = pack_half2(u - (float)hi[0], v - (float)hi[1]);
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
  uint32_t ids = 0;  // lane i: the page of this wave's i-th tile from id_at
  uint32_t id_at = 0;
  const uint32_t n_it = t0 + wave < t1 ? (t1 - t0 - wave + kDecWaves - 1) / kDecWaves : 0;
  auto index = [&](uint32_t it) { return tiles.tile(t0 + wave + it * kDecWaves); };
  auto fetch_ids = [&](uint32_t it) {
    id_at = it;
    ids = row[index(min(it + lane, n_it - 1)) >> (log_page - 5)];
  };
  bool cur_bad = false, nxt_bad = false;
  auto base_of = [&](uint32_t it, bool& bad) {
    uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)ids, (int)(it - id_at));
    bad = id >= a.s.n_pages;
    id = bad ? 0 : id;
    const uint32_t in = index(it) & ((a.s.page >> 5) - 1);
    return a.pool + ((((size_t)id * G + kvh) << (log_page - 5)) + in) * tile_bytes;
  };

  auto work = [&](const TileRegs<D>& t, uint32_t it, bool bad) {
    const uint32_t key0 = index(it) * kKv4Tile;
    const bool whole = (int64_t)key0 + 31 <= first &&
                       (a.window == 0 || (int64_t)key0 > last - (int64_t)a.window ||
                        (uint64_t)key0 + 31 < a.n_sinks);
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
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int64_t key = (int64_t)key0 + 16 * (i >> 2) + 4 * kg + (i & 3);
          x[i] = kv4_sees(pos[nt], key, a.window, a.n_sinks) ? x[i] : -INFINITY;
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
        const halfx2 lo = pack_half2(x[2 * i] - (float)hi[0], x[2 * i + 1] - (float)hi[1]);
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
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          Half8 sees;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            sees.u[i] = 0;
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const int u = 2 * i + j;
              const int64_t key = (int64_t)key0 + 16 * (u >> 2) + 4 * kg + (u & 3);
              if (kv4_sees(pos[nt], key, a.window, a.n_sinks)) sees.u[i] |= 0x3c00u << (16 * j);
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
    fetch_ids(0);
    load_tile<D>(x, base_of(0, cur_bad), lane);
    for (uint32_t it = 0; it < n_it; it += 2) {
      // Past the end the last tile is read once more (an L2 hit) and not used.
      uint32_t nx = min(it + 1, n_it - 1);
      if (nx - id_at >= 64) fetch_ids(nx);
      load_tile<D>(y, base_of(nx, nxt_bad), lane);
      work(x, it, cur_bad);
      if (it + 1 >= n_it) break;
      nx = min(it + 2, n_it - 1);
      if (nx - id_at >= 64) fetch_ids(nx);
      load_tile<D>(x, base_of(nx, cur_bad), lane);
      work(y, it + 1, nxt_bad);
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

// Joins the pieces of a row: a wave per row, lanes over dims.
template <int D>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Kv4AttnArgs a, Kv4SplitPlan plan,
                                                        Kv4Part part) {
  const uint32_t G = a.s.n_kv_heads, group = a.n_heads / G;
  const int lane = threadIdx.x & 63;
  const uint64_t id = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t r = (uint32_t)(id % plan.rows);
  const uint64_t slot = id / plan.rows;
  if (slot >= (uint64_t)a.n_seqs * plan.row_tiles * G) return;
  const uint32_t kvh = (uint32_t)(slot % G), rt = (uint32_t)(slot / G % plan.row_tiles);
  const uint32_t b = (uint32_t)(slot / G / plan.row_tiles);
  const Kv4Seq seq = kv4_seq(a, b);
  const uint32_t rows = seq.nq * group, r0 = rt * plan.rows, rr = r0 + r;
  if (seq.refused || rr >= rows) return;
  const uint32_t n_rows = min(plan.rows, rows - r0);
  const int64_t pos0 = (int64_t)seq.n_keys - seq.nq;
  const Kv4Tiles tiles = kv4_tiles(pos0 + r0 / group, pos0 + (r0 + n_rows - 1) / group, a.window,
                                   a.n_sinks);
  const uint32_t n = kv4_pieces(tiles.count(), plan.most).n;
  if (n == 1) return;
  const size_t at = slot * plan.splits * plan.rows + r;
  float top = -INFINITY;
  for (uint32_t i = lane; i < n; i += 64) top = fmaxf(top, part.ml[2 * (at + (size_t)i * plan.rows)]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, shfl_xor(top, x));
  float sum = 0.f, acc[D / 64] = {};
  for (uint32_t i = 0; i < n; i++) {
    const size_t p = at + (size_t)i * plan.rows;
    const float m = part.ml[2 * p];
    const float k = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
    sum = fmaf(part.ml[2 * p + 1], k, sum);
#pragma unroll
    for (int c = 0; c < D / 64; c++) acc[c] = fmaf(part.acc[p * D + 64 * c + lane], k, acc[c]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float* dst = a.o + ((size_t)(seq.q0 + rr / group) * a.n_heads + kvh * group + rr % group) * D;
#pragma unroll
  for (int c = 0; c < D / 64; c++) dst[64 * c + lane] = acc[c] * inv;
}

// Key tiles of a piece: few enough that the pieces of the call's bounds fill the
// 256 CUs with four workgroups each a few times over (sequences are shorter than
// the bound), and two a wave at least.
constexpr uint32_t kDecTarget = 4096, kDecFew = 2 * kDecWaves;

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
  const uint64_t most = (items * tiles + kDecTarget - 1) / kDecTarget;
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
  if (items * p.splits > 0x7fffffffull || items * p.rows / 4 > 0x7fffffffull)
    return hipErrorInvalidConfiguration;
  Kv4Part part{static_cast<float*>(ws), nullptr};
  part.acc = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) +
                                      ws_align(items * p.splits * p.rows * 8));
  const float scale = (float)(1.44269504088896340736 / sqrt((double)D));
  const dim3 grid((uint32_t)(items * p.splits)), block(kDecWaves * 64);
  if (p.rows == 8)
    hipLaunchKernelGGL((kv4_decode_kernel<D, 1>), grid, block, 0, st, a, p, part, scale);
  else
    hipLaunchKernelGGL((kv4_decode_kernel<D, 2>), grid, block, 0, st, a, p, part, scale);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  hipLaunchKernelGGL(kv4_merge_kernel<D>, dim3((uint32_t)((items * p.rows + 3) / 4)), dim3(256), 0,
                     st, a, p, part);
  return hipGetLastError();
}

hipError_t launch_kv4_decode(const Kv4AttnArgs& a, const Kv4SplitPlan& p, void* ws,
                             hipStream_t st) {
  return a.s.head_dim == 128 ? launch<128>(a, p, ws, st) : launch<64>(a, p, ws, st);
}

}  // namespace flk
