// Attention of a few queries a sequence over the paged 4-bit cache (single tokens,
// drafts), split over the keys. HBM-bound: 9/16 byte a value, each read once for the
// query-head rows of a kv head. 16 / 8 heads of 128: 64 sequences of 1025 to 16385 keys 108 us
// (5.9 TB/s) and 4.6 of merge, one of 131072 28.3 us (5.3 TB/s) and 3.8.
//
// A wave takes 32-key tiles. S^T = K Q^T and O^T += V^T P^T on 16x16x32 f16 MFMA: the
// 16 columns are 8 query-head rows in two f16 parts each, so the parts
// ride in columns that the few rows would leave empty. The cache's layout gives each
// lane its operands in 16-byte pieces, and P^T is taken from the S^T accumulators as
// they lie (a lane's scores are of the tokens whose values it holds). More than 8 rows take
// two column tiles, more than 16 go in chunks of 16, workgroups side by side so that the
// chunks after the first find a piece's tiles in the caches.
#include <algorithm>

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

// The work: each sequence's tiles in equal pieces of at most `per` tiles, a workgroup for
// each piece and kv head. `per` comes from the batch's total on the device, so pieces are
// as many as the GPU wants whether the lengths are equal or far apart; every workgroup
// sums the lengths and finds its piece (of up to 256 sequences). A sequence of several pieces goes through the
// workspace and a merge launch.
constexpr int kDecThreads = kDecWaves * 64;

// Tiles of each of a sequence's kv heads; one at least where it has rows (the run that has
// it writes them: zeros, or NaN for a refused sequence).
__device__ __forceinline__ uint32_t dec_tiles(const Kv4AttnArgs& a, const Kv4Seq& s) {
  if (s.nq == 0) return 0;
  if (s.refused) return 1;
  const int64_t pos0 = (int64_t)s.n_keys - s.nq;
  return max(1u, kv4_tiles(pos0, (int64_t)s.n_keys - 1, a.window, a.n_sinks).count());
}

// Pieces of a batch at `per` tiles, of_thread(per) of them this thread's, `before` in the
// threads before it. Shortest pieces, or rounding up, may make a few more than are resident
// together: then longer ones, in one round of the GPU (16 drafts of 5 onto up to 4000 keys:
// 26.5 us for 30.9).
template <int kWaves, typename OfThread>
__device__ __forceinline__ uint32_t dec_pieces(uint32_t& per, uint32_t resident, uint32_t* s_wave,
                                               uint32_t& before, OfThread of_thread) {
  for (int round = 0;; round++) {
    const uint32_t all = block_scan<kWaves>(of_thread(per), s_wave, before);
    if (all <= resident || all - resident > resident / 2 || round == 3) return all;
    per = max(per + 1, (uint32_t)((uint64_t)per * all / resident));
    __syncthreads();
  }
}

// The pieces of more sequences than a workgroup has threads, by a workgroup of a launch before:
// in every workgroup of the attention a thread's several sequences took longer than its tiles
// (2048 sequences of 250 to 1000 keys: 338 us for 547).
constexpr int kItemThreads = 1024;
__global__ __launch_bounds__(kItemThreads) void kv4_decode_items_kernel(
    Kv4AttnArgs a, uint32_t* first_piece, uint4* items, uint32_t runs, uint32_t pieces,
    uint32_t least, uint32_t resident) {
  __shared__ uint32_t s_wave[2][kItemThreads / 64];
  const uint32_t each = (a.n_seqs + kItemThreads - 1) / kItemThreads;
  const uint32_t my_b = min(threadIdx.x * each, a.n_seqs), my_end = min(my_b + each, a.n_seqs);
  uint32_t tiles = 0, at;
  for (uint32_t x = my_b; x < my_end; x++) tiles += dec_tiles(a, kv4_seq(a, x));
  uint32_t per = kv4_per(block_scan<kItemThreads / 64>(tiles, s_wave[0], at), pieces, least);
  auto pieces_of = [&](uint32_t x, uint32_t n) { return (dec_tiles(a, kv4_seq(a, x)) + n - 1) / n; };
  const uint32_t all =
      dec_pieces<kItemThreads / 64>(per, resident, s_wave[1], at, [&](uint32_t n) {
        uint32_t mine = 0;
        for (uint32_t x = my_b; x < my_end; x++) mine += pieces_of(x, n);
        return mine;
      });
  for (uint32_t x = my_b; x < my_end; x++) {
    const uint32_t n = pieces_of(x, per);
    first_piece[x] = at;
    for (uint32_t i = 0; i < n && at + i < runs; i++) items[at + i] = make_uint4(x, i, n, 0);
    at += n;
  }
  if (threadIdx.x == 0) first_piece[a.n_seqs] = all;
  for (uint32_t i = all + threadIdx.x; i < runs; i += kItemThreads) items[i] = make_uint4(0, 0, 0, 0);
}

// Workgroups a CU: three as far as the registers go (D = 64 with two column tiles keeps one
// in scratch memory for it, outside the loop: 108 us for 116 with two, 64 sequences of up to
// 16000 keys and 16 rows; D = 128 would spill in the loop).
template <int D>
constexpr uint32_t dec_per_cu(int nt) {
  return nt == 1 || D == 64 ? 3 : 2;
}
template <int D, int NT>
__global__ __launch_bounds__(kDecThreads, dec_per_cu<D>(NT)) void kv4_decode_kernel(
    Kv4AttnArgs a, Kv4Part part, uint32_t* first_piece, const uint4* items, uint32_t chunks,
    uint32_t pieces, uint32_t least, uint32_t resident, float scale_log2e) {
  constexpr int kRows = 8 * NT, kSteps = D / 32, kOT = D / 16;
  __shared__ float s_o[kDecWaves][kRows][D + 4];
  __shared__ float s_m[kDecWaves][kRows], s_l[kDecWaves][kRows];
  __shared__ uint32_t s_wave[2][kDecWaves], s_found[3];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  const uint32_t G = a.s.n_kv_heads, group = a.n_heads / G;

  const uint32_t kvh = blockIdx.x % G, chunk = blockIdx.x / G % chunks;
  const uint32_t run = blockIdx.x / G / chunks;
  uint32_t b = 0, piece = run, n_pieces, per;
  if (a.n_seqs > kDecThreads) {
    const uint4 item = items[run];
    b = uniform(item.x), piece = uniform(item.y), n_pieces = uniform(item.z);
    if (n_pieces == 0) return;
  } else if (a.n_seqs == 1) {
    const uint32_t count = uniform(dec_tiles(a, kv4_seq(a, 0)));
    per = kv4_per(count, pieces, least);
    n_pieces = (count + per - 1) / per;
    if (blockIdx.x == 0 && threadIdx.x == 0) first_piece[0] = 0, first_piece[1] = n_pieces;
    if (piece >= n_pieces) return;
  } else {
    // A thread per sequence.
    const uint32_t count = threadIdx.x < a.n_seqs ? dec_tiles(a, kv4_seq(a, threadIdx.x)) : 0;
    uint32_t mine, all, at;
    per = kv4_per(block_scan<kDecWaves>(count, s_wave[0], at), pieces, least);
    all = dec_pieces<kDecWaves>(per, resident, s_wave[1], at, [&](uint32_t n) {
      return mine = (count + n - 1) / n;
    });
    if (blockIdx.x == 0) {  // for the merge
      if (threadIdx.x < a.n_seqs) first_piece[threadIdx.x] = at;
      if (threadIdx.x == 0) first_piece[a.n_seqs] = all;
    }
    if (run >= all) return;
    if (run >= at && run < at + mine) {  // one thread
      s_found[0] = threadIdx.x;
      s_found[1] = run - at;
      s_found[2] = mine;
    }
    __syncthreads();
    b = uniform(s_found[0]), piece = uniform(s_found[1]), n_pieces = uniform(s_found[2]);
  }
  const Kv4Seq seq = kv4_seq(a, b);
  const uint32_t rows = seq.nq * group, r0 = chunk * kRows;
  if (r0 >= rows) return;
  const uint32_t n_rows = min(rows - r0, (uint32_t)kRows);
  if (seq.refused) {  // the first chunk is there for all of its rows
    if (chunk == 0)
      for (uint64_t i = threadIdx.x; i < (uint64_t)rows * D; i += kDecThreads) {
        const uint32_t r = (uint32_t)(i / D);
        a.o[((size_t)(seq.q0 + r / group) * a.n_heads + kvh * group + r % group) * D + i % D] =
            __builtin_nanf("");
      }
    return;
  }
  const int64_t first = (int64_t)seq.n_keys - seq.nq, last = (int64_t)seq.n_keys - 1;
  const Kv4Span span(first, last, a.window, a.n_sinks);
  // Pieces of one length, or one tile less.
  const uint32_t n_tiles = span.tiles.count();
  const uint32_t t0 = (uint32_t)((uint64_t)n_tiles * piece / n_pieces);
  const uint32_t t1 = (uint32_t)((uint64_t)n_tiles * (piece + 1) / n_pieces);

  const float second = col & 1 ? -1.f : 0.f;  // this lane's columns are second parts

  // q: column col of column tile nt is part col & 1 of row 8 nt + col / 2. The rows and
  // the first tile are on their way together.
  float4 qf[NT][D / 16];
  int delta[NT];  // the row's position behind the first
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const uint32_t r = r0 + min((uint32_t)(8 * nt + (col >> 1)), n_rows - 1);
    delta[nt] = (int)(r / group);
    const float4* src = reinterpret_cast<const float4*>(
        a.q + ((size_t)(seq.q0 + r / group) * a.n_heads + kvh * group + r % group) * D +
        kg * (D / 4));
#pragma unroll
    for (int i = 0; i < D / 16; i++) qf[nt][i] = src[i];
  }
  // l: the sums of this lane's weights.
  floatx4v o[NT][kOT] = {};
  float l[NT] = {};
  float m[NT];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) m[nt] = -INFINITY;

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

  TileRegs<D> x, y;
  const TileOffsets at = tile_offsets<D>(lane);
  uint32_t id_x = 0, id_y = 0;
  if (n_it > 0) {
    id_x = page_of(0);
    id_y = page_of(min(1u, n_it - 1));
    load_tile<D>(x, base_of(0, id_x), at);
  }

  Half8 q[NT][kSteps];
  float c_s[NT];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; i++)
      amax = fmaxf(fmaxf(fmaxf(amax, fabsf(qf[nt][i].x)), fabsf(qf[nt][i].y)),
                   fmaxf(fabsf(qf[nt][i].z), fabsf(qf[nt][i].w)));
    amax = max_xor<16>(amax);
    amax = max_xor<32>(amax);
    const RowScale rs = row_scale(amax);
    c_s[nt] = rs.down * scale_log2e;
#pragma unroll
    for (int i = 0; i < D / 8; i++) {
      const float4 f = qf[nt][i >> 1];
      const float u = (i & 1 ? f.z : f.x) * rs.up, v = (i & 1 ? f.w : f.y) * rs.up;
      const halfx2 hi = pack_half2(u, v);
      q[nt][i >> 2].u[i & 3] = as_u32(rest_half2(u, v, hi, second));
    }
  }

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
        p[nt].u[i] = as_u32(rest_half2(x[2 * i], x[2 * i + 1], hi, second));
      }
    }
    if (!whole) {
      // Values of keys that some row does not see: scales from 8192 on, which no append
      // writes but for NaN blocks (memory never written holds anything, and times a code
      // it may be infinite), count as 0 in the products, and make NaN of the rows that do
      // see them.
      Half8 flag;
      uint32_t* w = reinterpret_cast<uint32_t*>(&vs);
      bool any = false;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const bool lo = (w[i] & 0x7000u) == 0x7000u, hi = (w[i] & 0x70000000u) == 0x70000000u;
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
  const size_t slot = (size_t)blockIdx.x * kRows;
  for (uint32_t i = threadIdx.x; i < n_rows * (D / 4); i += kDecThreads) {
    const uint32_t r = i / (D / 4), e = 4 * (i % (D / 4)), rr = r0 + r;
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
    if (n_pieces == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      f.x *= inv, f.y *= inv, f.z *= inv, f.w *= inv;
      *reinterpret_cast<float4*>(
          a.o + ((size_t)(seq.q0 + rr / group) * a.n_heads + kvh * group + rr % group) * D + e) = f;
    } else {
      if (e == 0) part.ml[2 * (slot + r)] = top, part.ml[2 * (slot + r) + 1] = sum;
      *reinterpret_cast<float4*>(part.acc + (slot + r) * D + e) = f;
    }
  }
}

// Joins the pieces of a sequence's row; a workgroup per row.
template <int D, int kThreads>
__global__ __launch_bounds__(kThreads) void kv4_decode_merge_kernel(Kv4AttnArgs a, Kv4Part part,
                                                                    const uint32_t* first_piece,
                                                                    uint32_t rows, uint32_t chunks,
                                                                    uint32_t slot_rows) {
  const uint32_t G = a.s.n_kv_heads, group = a.n_heads / G;
  const uint32_t r = blockIdx.x % rows, item = blockIdx.x / rows, kvh = item % G, b = item / G;
  const uint32_t p0 = first_piece[b], n = first_piece[b + 1] - p0;
  if (n <= 1) return;  // written by the piece itself
  const Kv4Seq seq = kv4_seq(a, b);
  if (r >= seq.nq * group) return;
  merge_pieces<D, kThreads>(
      part, n,
      [&](uint32_t i) {
        return (((size_t)(p0 + i) * chunks + r / slot_rows) * G + kvh) * slot_rows + r % slot_rows;
      },
      a.o + ((size_t)(seq.q0 + r / group) * a.n_heads + kvh * group + r % group) * D);
}

// Pieces that a batch is cut into (over its kv heads), beside one more a sequence at most
// from rounding up. 768 workgroups are resident (three a CU, by the kernel's registers);
// twice as many let the GPU even out a batch, while a single sequence's pieces are equal
// already and two a CU stream as fast. No piece has fewer than 20 tiles: up to 640 keys
// then need no merge launch. us, 64 sequences of up to 16385 keys / one of 131072 / 128
// with a window of 4096: 1024 pieces 127 / 36.3 / 70.5, 1536 120 / 36.3 / 68, 2048 121 /
// 37.3 / 72, 3000 127 / 39 / 77; 512 for the one sequence 34.4; 513 keys in pieces of 8
// tiles 12.1, of 20 9.6.
constexpr uint32_t kDecPieces = 1536, kDecAlone = 512, kDecLeast = 5 * kDecWaves;
struct DecodePlan {
  uint32_t slot_rows;  // rows of a chunk
  uint32_t chunks;     // of a sequence's rows
  uint32_t pieces, least;
  uint32_t resident;   // pieces
  uint32_t runs;       // workgroups of a kv head and chunk
};
static DecodePlan decode_plan(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                              uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                              uint32_t window, uint32_t n_sinks) {
  DecodePlan p;
  const uint32_t rows = max_q * (n_heads / n_kv_heads);
  p.slot_rows = rows <= 8 ? 8 : 16;
  p.chunks = (rows + p.slot_rows - 1) / p.slot_rows;
  p.least = kDecLeast;
  p.pieces = std::max(1u, (n_seqs == 1 ? kDecAlone : kDecPieces) / n_kv_heads / p.chunks);
  const uint32_t per_cu =
      head_dim == 64 ? dec_per_cu<64>(p.slot_rows / 8) : dec_per_cu<128>(p.slot_rows / 8);
  p.resident = std::max(1u, 256 * per_cu / n_kv_heads / p.chunks);
  const uint64_t tiles = kv4_max_tiles(max_n_keys, max_q, window, n_sinks);
  const uint64_t cut = (n_seqs * tiles + p.least - 1) / p.least;  // at most, plus n_seqs
  p.runs = (uint32_t)std::min(std::min((uint64_t)p.pieces, cut) + n_seqs - 1,
                              n_seqs * ((tiles + p.least - 1) / p.least));
  return p;
}

static uint64_t first_bytes(uint32_t n_seqs) { return ws_align(((uint64_t)n_seqs + 1) * 4); }
static uint64_t item_bytes(uint32_t n_seqs, const DecodePlan& p) {
  return n_seqs > (uint32_t)kDecThreads ? ws_align((uint64_t)p.runs * sizeof(uint4)) : 0;
}
static uint64_t slots(const DecodePlan& p, uint32_t n_kv_heads) {
  return (uint64_t)p.runs * p.chunks * n_kv_heads * p.slot_rows;
}

uint64_t kv4_decode_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                             uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                             uint32_t window, uint32_t n_sinks) {
  const DecodePlan p =
      decode_plan(n_seqs, max_q, max_n_keys, n_heads, n_kv_heads, head_dim, window, n_sinks);
  return first_bytes(n_seqs) + item_bytes(n_seqs, p) + ws_align(slots(p, n_kv_heads) * 8) +
         ws_align(slots(p, n_kv_heads) * head_dim * 4);
}

bool kv4_decode_fits(const Kv4AttnArgs& a) {
  const uint32_t G = a.s.n_kv_heads;
  const DecodePlan p =
      decode_plan(a.n_seqs, a.max_q, a.max_n_keys, a.n_heads, G, a.s.head_dim, a.window, a.n_sinks);
  const uint64_t tiles =
      (uint64_t)a.n_seqs * kv4_max_tiles(a.max_n_keys, a.max_q, a.window, a.n_sinks);
  return tiles <= 0xffffffffull && (uint64_t)p.runs * p.chunks * G <= kMaxGroups &&
         (uint64_t)a.n_seqs * a.max_q * a.n_heads <= kMaxGroups;
}

template <int D>
static hipError_t launch(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  const uint32_t G = a.s.n_kv_heads;
  const DecodePlan p =
      decode_plan(a.n_seqs, a.max_q, a.max_n_keys, a.n_heads, G, D, a.window, a.n_sinks);
  uint8_t* w = static_cast<uint8_t*>(ws);
  uint32_t* first_piece = reinterpret_cast<uint32_t*>(w);
  Kv4Part part;
  w += first_bytes(a.n_seqs);
  uint4* items = reinterpret_cast<uint4*>(w);
  w += item_bytes(a.n_seqs, p);
  part.ml = reinterpret_cast<float*>(w);
  part.acc = reinterpret_cast<float*>(w + ws_align(slots(p, G) * 8));
  const float scale = (float)(kLog2e / sqrt((double)D));
  const uint32_t rows = a.max_q * (a.n_heads / G);
  const dim3 grid(p.runs * p.chunks * G), block(kDecThreads);
  if (a.n_seqs > (uint32_t)kDecThreads) {
    hipLaunchKernelGGL(kv4_decode_items_kernel, dim3(1), dim3(kItemThreads), 0, st, a, first_piece,
                       items, p.runs, p.pieces, p.least, p.resident);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.slot_rows == 8)
    hipLaunchKernelGGL((kv4_decode_kernel<D, 1>), grid, block, 0, st, a, part, first_piece, items,
                       p.chunks, p.pieces, p.least, p.resident, scale);
  else
    hipLaunchKernelGGL((kv4_decode_kernel<D, 2>), grid, block, 0, st, a, part, first_piece, items,
                       p.chunks, p.pieces, p.least, p.resident, scale);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.runs <= a.n_seqs) return e;  // no more pieces than sequences: none cut
  const dim3 mgrid(a.n_seqs * G * rows);
  if (p.runs >= 8 * a.n_seqs)  // many pieces a sequence
    hipLaunchKernelGGL((kv4_decode_merge_kernel<D, 256>), mgrid, dim3(256), 0, st, a, part,
                       first_piece, rows, p.chunks, p.slot_rows);
  else
    hipLaunchKernelGGL((kv4_decode_merge_kernel<D, 64>), mgrid, dim3(64), 0, st, a, part,
                       first_piece, rows, p.chunks, p.slot_rows);
  return hipGetLastError();
}

hipError_t launch_kv4_decode(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  return a.s.head_dim == 128 ? launch<128>(a, ws, st) : launch<64>(a, ws, st);
}

}  // namespace flk
