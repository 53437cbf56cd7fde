// Attention of many queries a sequence over the paged 4-bit cache (prompts, chunks).
// MFMA-bound: f16 matrix products of the cache's exact values with q and the weights
// in two f16 parts, twice the plain products' work. 8192 tokens, 16 / 8 heads of 128: 530 us,
// 1037 TFLOP/s of them (a plain product of 8192 x 8192 matrices reaches 1140).
//
// A work item is 128 query-head rows of one kv head and a piece of their key tiles; four
// waves of 32 rows, two workgroups a CU (three of 64-wide heads, which halve LDS and the
// accumulators: 87 us for 96 with two, seven ragged prompts). Every 64 keys the workgroup
// turns the two tiles' codes to f16 in LDS (each code once for 128 rows), into the buffer that
// the step before has read; the next tiles' codes are loaded meanwhile. S^T = K Q^T and
// O^T += V^T P^T on 32x32x16: a column is a row of q, and P^T is taken from the S^T
// accumulators as they lie, because V's keys are put in the order in which a lane holds its
// scores.
#include <algorithm>

#include "kv4_attn.hpp"

namespace flk {

typedef float floatx16v __attribute__((ext_vector_type(16)));

constexpr int kPreRows = 128, kPreThreads = 256, kStep = 64;
// Pieces of a call (over its kv heads): one for each workgroup that is resident; with as many
// row tiles as two a CU anyway, some more than those, so that the heaviest are cut. None has
// fewer than four key tiles. us, 128-wide heads, 2048 tokens / 64 at 32768 / four prompts of
// 500 to 1500 onto up to 3000 / 8192 tokens: 512 pieces 64 / 55.6 / 166 / 545, 640 73 / 69.7 /
// 164 / 525, 1024 74 / 73 / 179 / 559; whole row tiles cut by the call's bounds 107 / 55.7 /
// 251 / 546. 64-wide, 700 tokens / 1500 onto 3000 / 4096: 512 pieces 24.2 / 137 / -, 640 25.4 /
// 153 / 164, 768 25.4 / 117 / 171.
template <int D>
constexpr uint32_t kPreResident = D == 64 ? 3 : 2;  // workgroups a CU
constexpr uint32_t kPreMany = 512, kPreMore = 640, kPreLeast = 4;

// The work: row tiles, those of the last queries first (in a prompt without a window they see the
// most keys), the sequences in turn, each in equal pieces of at most `per` key tiles. Where
// lengths differ or a window evens them out this is no order by weight: seven ragged prompts
// with a window, 143 row tiles of 1 to 35 key tiles, take the time of 55 key tiles as ordered and
// of 37 heaviest first, in a greedy model of 96 workgroups a kv head. As for single tokens, `per` comes from the batch's
// total on the device, and every workgroup finds its piece; of more than kMaxCut row tiles a
// launch before lists them.
constexpr uint32_t kMaxCut = kPreThreads;
// Row tiles of up to this many key tiles (2048 keys, or a window's) are whole where there are
// more than kMaxCut, and without a list up to twice as many. us, a workgroup for every row tile
// that the call's bounds allow / listed whole / listed and cut: 7 prompts of up to 1500 tokens,
// 64-wide, window 1024 (294) 88.5 / 97.5 / 100.4, 20 of up to 2000 (640) 224 / 174 / 179, 100
// (3200) 1597 / 1496 / 1494.
constexpr uint32_t kShortTiles = 64;

struct PrePlan {
  uint32_t row_tiles;  // of a sequence, at most
  uint32_t pieces;     // that the row tiles are cut into (for a kv head); 0: whole
  uint32_t runs;       // workgroups of a kv head
  // More row tiles than kMaxCut: a launch before lists the pieces, of row tiles with rows only.
  bool listed;
  uint32_t many, more;  // from `many` row tiles with rows on, `more` pieces
  uint32_t slots, cuts; // partial results, row tiles that have them: at most
};
// A piece (n = 0: none) and its partial result; of a cut row tile the first of them.
struct alignas(16) PrePiece {
  uint32_t e, cut, n, slot;
};

// Row tile e: its sequence and place, and its key tiles (none: no rows; one at least
// otherwise, of a refused sequence the first row tile alone).
struct PreItem {
  uint32_t b, rt;
};
__device__ __forceinline__ PreItem pre_item(const Kv4AttnArgs& a, const PrePlan& p, uint32_t e) {
  return {e % a.n_seqs, p.row_tiles - 1 - e / a.n_seqs};
}
__device__ __forceinline__ Kv4Tiles pre_tiles(const Kv4AttnArgs& a, const Kv4Seq& seq, uint32_t rt,
                                              uint32_t group) {
  const uint32_t r0 = rt * kPreRows, rows = seq.nq * group;
  const int64_t pos0 = (int64_t)seq.n_keys - seq.nq;
  const uint32_t end = min(r0 + (uint32_t)kPreRows, rows);
  return kv4_tiles(pos0 + r0 / group, pos0 + (end - 1) / group, a.window, a.n_sinks);
}
__device__ __forceinline__ uint32_t pre_count(const Kv4AttnArgs& a, const PrePlan& p, uint32_t e,
                                              uint32_t group) {
  const PreItem i = pre_item(a, p, e);
  const Kv4Seq seq = kv4_seq(a, i.b);
  if (i.rt * kPreRows >= seq.nq * group) return 0;
  if (seq.refused) return i.rt == 0;
  return max(1u, pre_tiles(a, seq, i.rt, group).count());
}

// LDS: K's rows in 16-byte slots of 8 dims, V's (a row a dim) in slots of 8 keys, slots
// xored with bits of the row so that neighbouring rows of one slot lie in distinct banks.
// Byte offsets in one buffer; the xors reach bits 4 .. 7 only, so a lane's other slots are
// its first offset xor a constant.
template <int D>
__device__ __forceinline__ uint32_t k_at(uint32_t key, uint32_t slot) {
  return key * (2 * D) + ((slot ^ (D == 128 ? key & 15 : (key >> 1) & 7)) << 4);
}
__device__ __forceinline__ uint32_t v_at(uint32_t dim, uint32_t slot) {
  return dim * (2 * kStep) + ((slot ^ ((dim >> 1) & 7) ^ ((dim >> 4) & 7)) << 4);
}

template <int D>
struct alignas(16) PreShared {
  uint8_t k[2][kStep * D * 2];
  uint8_t v[2][kStep * D * 2];
  // Slots (keys) of a tile whose V scale is 8192 or more, by [block][g]: a NaN block's, or
  // memory never written behind a sequence. It counts as 0 in LDS, and the rows that see
  // such a key get their NaN from here.
  uint32_t flag[2][2][4];
};

// One thread's share of two tiles, as it lies in the pool.
struct PreRegs {
  uint4 k, v, vs;
  uint32_t ks;
};

template <int D>
__global__ __launch_bounds__(kPreThreads, kPreResident<D>) void kv4_prefill_kernel(
    Kv4AttnArgs a, PrePlan plan, Kv4Part part, uint32_t* first_piece, const PrePiece* list,
    float scale_log2e) {
  constexpr int kSteps = D / 16, kOT = D / 32;
  __shared__ PreShared<D> sh;
  __shared__ uint32_t s_wave[kPreThreads / 64], s_found[3];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const uint32_t G = a.s.n_kv_heads, group = a.n_heads / G;
  const uint32_t kvh = blockIdx.x % G, run = blockIdx.x / G;
  uint32_t e = run, cut = 0, n_pieces = 1, piece_slot = run;
  if (plan.listed) {
    const uint4 x = *reinterpret_cast<const uint4*>(&list[run]);
    e = uniform(x.x), cut = uniform(x.y), n_pieces = uniform(x.z), piece_slot = uniform(x.w);
    if (n_pieces == 0) return;
  } else if (plan.pieces > 0) {
    // A thread per row tile.
    const uint32_t items = a.n_seqs * plan.row_tiles;
    uint32_t at;
    const uint32_t count = threadIdx.x < items ? pre_count(a, plan, threadIdx.x, group) : 0;
    uint32_t per = kv4_per(block_scan<kPreThreads / 64>(count, s_wave, at), plan.pieces, kPreLeast);
    uint32_t mine, all;
    // Rounding up makes more pieces than asked for: where that leaves a few for a second
    // round of the GPU, longer ones.
    for (int round = 0;; round++) {
      __syncthreads();
      mine = (count + per - 1) / per;
      all = block_scan<kPreThreads / 64>(mine, s_wave, at);
      if (all <= plan.pieces || items >= plan.pieces || round == 3) break;
      per = max(per + 1, (uint32_t)((uint64_t)per * all / plan.pieces));
    }
    if (blockIdx.x == 0) {  // for the merge
      if (threadIdx.x < items) first_piece[threadIdx.x] = at;
      if (threadIdx.x == 0) first_piece[items] = all;
    }
    if (run >= all) return;
    if (run >= at && run < at + mine) {  // one thread
      s_found[0] = threadIdx.x;
      s_found[1] = run - at;
      s_found[2] = mine;
    }
    __syncthreads();
    e = uniform(s_found[0]), cut = uniform(s_found[1]), n_pieces = uniform(s_found[2]);
  }
  const uint32_t b = pre_item(a, plan, e).b, rt = pre_item(a, plan, e).rt;
  const Kv4Seq seq = kv4_seq(a, b);
  const uint32_t rows = seq.nq * group;
  const uint32_t r0 = rt * kPreRows;
  if (r0 >= rows) return;
  if (seq.refused) {
    if (rt == 0)
      for (uint64_t i = threadIdx.x; i < (uint64_t)rows * D; i += kPreThreads) {
        const uint32_t r = (uint32_t)(i / D);
        a.o[((size_t)(seq.q0 + r / group) * a.n_heads + kvh * group + r % group) * D + i % D] =
            __builtin_nanf("");
      }
    return;
  }
  const int64_t pos0 = (int64_t)seq.n_keys - seq.nq;
  const Kv4Tiles tiles = pre_tiles(a, seq, rt, group);
  const uint32_t n_tiles = tiles.count();
  const uint32_t t0 = (uint32_t)((uint64_t)n_tiles * cut / n_pieces);
  const uint32_t t1 = (uint32_t)((uint64_t)n_tiles * (cut + 1) / n_pieces);
  const uint32_t n_steps = (t1 - t0 + 1) / 2;

  // This wave's rows.
  const uint32_t w0 = r0 + wave * 32;
  const bool idle = w0 >= rows;
  const uint32_t wl = min(w0 + 31, rows - 1);
  const int64_t first = pos0 + min(w0, rows - 1) / group, last = pos0 + wl / group;
  const Kv4Span span(first, last, a.window, a.n_sinks);
  const uint32_t my = min(w0 + col, rows - 1);  // lanes behind the last row repeat it
  const int delta = (int)(my / group - min(w0, rows - 1) / group);
  const size_t my_at =
      ((size_t)(seq.q0 + my / group) * a.n_heads + kvh * group + my % group) * D;

  // Two parts of q: dims 16 s + 8 h ..
  Half8 qh[kSteps], ql[kSteps];
  float c_s;
  {
    float x[D / 2], amax = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; s++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float4 f = *reinterpret_cast<const float4*>(a.q + my_at + 16 * s + 8 * h + 4 * i);
        x[8 * s + 4 * i] = f.x, x[8 * s + 4 * i + 1] = f.y;
        x[8 * s + 4 * i + 2] = f.z, x[8 * s + 4 * i + 3] = f.w;
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

  // Staging: a thread takes a 16-byte piece of K and one of V of tile `half` of the step
  // (D = 128), or a piece of K or of V (D = 64).
  const uint32_t log_page = 31 - __builtin_clz(a.s.page);
  const uint32_t* row = a.table + (size_t)b * a.max_blocks;
  const int st_tile = D == 128 ? wave >> 1 : wave & 1;
  const int piece = D == 128 ? (int)(threadIdx.x & 127) : lane;
  const bool st_k = D == 128 || wave < 2, st_v = D == 128 || wave >= 2;
  auto tile_of = [&](uint32_t i) { return tiles.tile(min(t0 + i, t1 - 1)); };
  auto page_of = [&](uint32_t i) {
    typedef const __attribute__((address_space(4))) uint32_t* ConstPtr;
    return *(ConstPtr)(uintptr_t)(row + (tile_of(i) >> (log_page - 5)));
  };
  PreRegs rg;
  const int v_n = piece & 15, v_g = (piece >> 4) & 3, v_c = piece >> 6;
  const int v_block = v_n * (D / 16) / 32;
  const int ks_at = Kv4<D>::kKScale +
                    4 * (D == 128 ? piece & 63 : (piece >> 2) * 2 + ((piece >> 1) & 1));
  const int st_half = D == 128 ? piece >> 6 : 0, st_key = D == 128 ? (piece >> 2) & 15 : piece >> 2;
  const uint32_t k_to =
      k_at<D>(32 * st_tile + 16 * st_half + st_key, (D == 128 ? 4 : 2) * (piece & 3));
  auto fetch = [&](uint32_t step, uint32_t page_id) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const bool bad = page_id >= a.s.n_pages;
    const uint32_t in = tile_of(2 * step + st_tile) & ((a.s.page >> 5) - 1);
    const uint8_t* base =
        a.pool + ((((size_t)(bad ? 0 : page_id) * G + kvh) << (log_page - 5)) + in) *
                     (size_t)Kv4<D>::kTileBytes;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0,
                                                        Kv4<D>::kTileBytes, 0x00020000);
    if (st_k) {
      const u4 k = __builtin_amdgcn_raw_buffer_load_b128(rsrc, piece * 16, 0, 0);
      rg.k = make_uint4(k[0], k[1], k[2], k[3]);
      rg.ks = __builtin_amdgcn_raw_buffer_load_b32(rsrc, ks_at, 0, 0);
      if (bad) rg.ks = 0x7e007e00u;
    }
    if (st_v) {
      const u4 v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, piece * 16, Kv4<D>::kV, 0);
      const u4 s = __builtin_amdgcn_raw_buffer_load_b128(
          rsrc, (v_g * Kv4<D>::kBlocks + v_block) * 16, Kv4<D>::kVScale, 0);
      rg.v = make_uint4(v[0], v[1], v[2], v[3]);
      rg.vs = make_uint4(s[0], s[1], s[2], s[3]);
    }
  };
  auto stage = [&](int buf) {
    if (st_k) {
      const uint32_t w[4] = {rg.k.x, rg.k.y, rg.k.z, rg.k.w};
      // D = 128: piece [half][key][part], octet i of the part, one scale. D = 64: [key][part]
      // with two octets of each half.
      const uint32_t lo = rg.ks & 0xffffu, hi = rg.ks >> 16;
      const uint32_t one = D == 128 && st_half ? hi : lo;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const halfx2 d = as_half2((D == 128 || i < 2 ? one : hi) * 0x10001u);
        uint4 x;
        x.x = as_u32(kv4_pair<0>(w[i], d)), x.y = as_u32(kv4_pair<1>(w[i], d));
        x.z = as_u32(kv4_pair<2>(w[i], d)), x.w = as_u32(kv4_pair<3>(w[i], d));
        // (Slots 4 part + i, or 2 part + i % 2 of half i / 2, whose rows lie 16 keys on.)
        const uint32_t at =
            D == 128 ? k_to ^ (i << 4) : (k_to ^ ((i & 1) << 4)) + (i >> 1) * 32 * D;
        *reinterpret_cast<uint4*>(&sh.k[buf][at]) = x;
      }
    }
    if (st_v) {
      uint32_t s[4] = {rg.vs.x, rg.vs.y, rg.vs.z, rg.vs.w};
      const uint32_t w[4] = {rg.v.x, rg.v.y, rg.v.z, rg.v.w};
      uint32_t odd = 0, mask = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) odd |= (s[i] & 0x70007000u) + 0x10001000u;
      if (odd & 0x80008000u) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const bool lo = (s[i] & 0x7000u) == 0x7000u, hi = (s[i] & 0x70000000u) == 0x70000000u;
          s[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
          mask |= (lo ? 1u : 0u) << (2 * i) | (hi ? 2u : 0u) << (2 * i);
        }
      }
      if (v_c == 0 && v_n % (512 / D) == 0)
        reinterpret_cast<uint8_t*>(sh.flag[buf][st_tile])[v_block * 4 + v_g] = (uint8_t)mask;
      // Slots 0 .. 3 are keys 4 g .., slots 4 .. 7 keys 16 + 4 g ..: of a 16-key step, lane
      // half g & 1 holds the scores of keys 4 (g & 1) .. (first) and 8 + 4 (g & 1) ..
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int dim = (D / 16) * v_n + 4 * v_c + j;
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const halfx2 d = as_half2(s[i]);
          x[i] = as_u32(j == 0   ? kv4_pair<0>(w[i], d)
                        : j == 1 ? kv4_pair<1>(w[i], d)
                        : j == 2 ? kv4_pair<2>(w[i], d)
                                 : kv4_pair<3>(w[i], d));
        }
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
          const uint32_t at = v_at(dim, 4 * st_tile + 2 * ks + (v_g & 1)) + 8 * (v_g >> 1);
          *reinterpret_cast<uint2*>(&sh.v[buf][at]) = make_uint2(x[2 * ks], x[2 * ks + 1]);
        }
      }
    }
  };

  const uint32_t k_from = k_at<D>(col, h), v_from = v_at(col, h);
  floatx16v o[kOT] = {};
  float m = -INFINITY, l = 0.f;

  auto block = [&](int buf, int t2, uint32_t tile) {
    const bool whole = span.whole(tile);
    floatx16v s = {};
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const halfx8 k = *reinterpret_cast<const halfx8*>(
          &sh.k[0][(k_from + buf * (kStep * D * 2)) ^ (i << 5)] + t2 * (64 * D));
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[i].h, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[i].h, s, 0, 0, 0);
    }
    // (K's operands two reads ahead of the products.)
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    Kv4Mask mask{};
    if (!whole) {
      mask = span.mask(tile);
#pragma unroll
      for (int i = 0; i < 16; i++)
        s[i] = mask.sees(8 * (i >> 2) + 4 * h + (i & 3), delta) ? s[i] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
    top *= c_s;
    if (__ballot(top > m + kSlack)) {
      top = max_xor<32>(top);
      const float nm = fmaxf(m, top);
      const float alpha = nm == m ? 1.f : __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      l *= alpha;
#pragma unroll
      for (int c = 0; c < kOT; c++) o[c] *= alpha;
    }
    const float mb = (m == -INFINITY ? 0.f : m) - kBias;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c_s, -mb));
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
    for (int ks = 0; ks < 2; ks++) {
      halfx8 v[kOT];
#pragma unroll
      for (int c = 0; c < kOT; c++) {
        v[c] = *reinterpret_cast<const halfx8*>(
            &sh.v[0][(v_from + buf * (kStep * D * 2)) ^ ((4 * t2 + 2 * ks) ^ (2 * c)) << 4] +
            c * (64 * kStep));
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[c], pl[ks].h, o[c], 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < kOT; c++)
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[c], ph[ks].h, o[c], 0, 0, 0);
    }
    const uint32_t* flag = sh.flag[buf][t2];
    uint32_t any = 0;
#pragma unroll
    for (int c = 0; c < kOT; c++) any |= flag[c];
    if (__builtin_amdgcn_readfirstlane(any)) {
#pragma unroll 1
      for (int c = 0; c < kOT; c++) {
        bool hit = false;
#pragma unroll 1
        for (int key = 0; key < 32; key++) {
          const uint32_t bits = flag[c] >> (8 * ((key >> 2) & 3));
          hit |= (bits >> ((key & 3) + 4 * (key >> 4)) & 1) && (whole || mask.sees(key, delta));
        }
#pragma unroll
        for (int cc = 0; cc < kOT; cc++)
          if (cc == c && hit) o[cc] = __builtin_nanf("");
      }
    }
  };

  if (n_steps > 0) {
    uint32_t id_n = page_of(st_tile);
    fetch(0, id_n);
    id_n = page_of(2 + st_tile);
    stage(0);
    fetch(1, id_n);  // past the end: the last tile again
    __syncthreads();
    for (uint32_t st = 0; st < n_steps; st++) {
      const int buf = st & 1;
      id_n = page_of(2 * (st + 2) + st_tile);
      if (st + 1 < n_steps) {
        stage(buf ^ 1);
        fetch(st + 2, id_n);
      }
      if (!idle) {
#pragma unroll
        for (int t2 = 0; t2 < 2; t2++) {
          if (t0 + 2 * st + t2 >= t1) break;
          const uint32_t tile = tiles.tile(t0 + 2 * st + t2);
          // Some row of the wave sees some key: not past its last, not between its first
          // tokens and its window.
          if (tile >= span.tiles.to || (tile >= span.tiles.sinks && tile < span.tiles.from))
            continue;
          block(buf, t2, tile);
        }
      }
      __syncthreads();
    }
  }
  if (idle || w0 + col >= rows) return;
  float lo, hi;
  swap_pair<32>(l, lo, hi);
  l = lo + hi;
  const size_t at = ((size_t)piece_slot * G + kvh) * kPreRows + wave * 32 + col;
  float* dst = n_pieces == 1 ? a.o + my_at : part.acc + at * D;
  const float inv = n_pieces > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
  if (n_pieces > 1 && h == 0) part.ml[2 * at] = m, part.ml[2 * at + 1] = l;
#pragma unroll
  for (int c = 0; c < kOT; c++)
#pragma unroll
    for (int i = 0; i < 4; i++)
      *reinterpret_cast<float4*>(dst + 32 * c + 8 * i + 4 * h) =
          make_float4(o[c][4 * i] * inv, o[c][4 * i + 1] * inv, o[c][4 * i + 2] * inv,
                      o[c][4 * i + 3] * inv);
}

// The list. us, a 2048-token prompt at 32768 beside 31 single tokens / one of 8192: 1117 / 598;
// in workgroups for every row tile that the call's bounds allow, whole, 3372 / 1650 (those
// without rows are started too, and the others may meet on few CUs). One workgroup goes over the
// row tiles of the bounds, not of the lengths, some passes of dependent loads: 512 of them 12 us,
// 65536 (512 sequences, max_q 8192, eight prompts of 1000 tokens in it) 124, 524288 891.
constexpr int kListThreads = 1024;
__device__ __forceinline__ uint32_t pre_pieces(uint32_t count, uint32_t per) {
  return count / per + (count % per != 0);
}
__global__ __launch_bounds__(kListThreads) void kv4_prefill_list_kernel(Kv4AttnArgs a, PrePlan plan,
                                                                        PrePiece* list,
                                                                        PrePiece* cuts) {
  constexpr int kWaves = kListThreads / 64;
  __shared__ uint32_t s_wave[5][kWaves];
  const uint32_t group = a.n_heads / a.s.n_kv_heads, items = a.n_seqs * plan.row_tiles;
  const uint32_t each = (items + kListThreads - 1) / kListThreads;
  const uint32_t e0 = min(threadIdx.x * each, items), e1 = min(e0 + each, items);
  uint32_t tiles = 0, real = 0, at, slot, c;
  for (uint32_t e = e0; e < e1; e++) {
    const uint32_t n = pre_count(a, plan, e, group);
    tiles += n, real += n > 0;
  }
  real = block_scan<kWaves>(real, s_wave[0], at);
  const uint32_t pieces = real >= plan.many ? plan.more : plan.pieces;
  uint32_t per = kv4_per(block_scan<kWaves>(tiles, s_wave[1], at), pieces, kPreLeast), all;
  if (plan.cuts == 0) per = 0xffffffffu;
  for (int round = 0;; round++) {  // as in the attention
    uint32_t mine = 0;
    for (uint32_t e = e0; e < e1; e++) mine += pre_pieces(pre_count(a, plan, e, group), per);
    all = block_scan<kWaves>(mine, s_wave[2], at);
    if (all <= pieces || real >= pieces || plan.cuts == 0 || round == 3) break;
    per = max(per + 1, (uint32_t)((uint64_t)per * all / pieces));
    __syncthreads();
  }
  uint32_t my_slots = 0, my_cuts = 0;
  for (uint32_t e = e0; e < e1; e++) {
    const uint32_t n = pre_pieces(pre_count(a, plan, e, group), per);
    if (n > 1) my_slots += n, my_cuts++;
  }
  block_scan<kWaves>(my_slots, s_wave[3], slot);
  const uint32_t n_cuts = block_scan<kWaves>(my_cuts, s_wave[4], c);
  for (uint32_t e = e0; e < e1; e++) {
    const uint32_t n = pre_pieces(pre_count(a, plan, e, group), per);
    // (Rows of sequences that overlap may be more than the plan's bounds: whole then, or out.)
    const bool cut = n > 1 && slot + n <= plan.slots && c < plan.cuts;
    for (uint32_t i = 0; i < n && at + i < plan.runs; i++)
      list[at + i] = cut ? PrePiece{e, i, n, slot + i} : PrePiece{e, 0, i == 0 ? 1u : 0u, 0};
    if (cut) cuts[c] = {e, 0, n, slot};
    at += n;
    if (n > 1) slot += n, c++;
  }
  for (uint32_t i = all + threadIdx.x; i < plan.runs; i += kListThreads) list[i] = {0, 0, 0, 0};
  for (uint32_t i = n_cuts + threadIdx.x; i < plan.cuts; i += kListThreads) cuts[i] = {0, 0, 0, 0};
}

// Joins the pieces of rows: a workgroup per row, or (FEW pieces) D / 4 threads per row, for
// there may be many rows and nothing to join.
template <int D, bool FEW>
__global__ __launch_bounds__(256) void kv4_prefill_merge_kernel(Kv4AttnArgs a, PrePlan plan,
                                                                Kv4Part part,
                                                                const uint32_t* first_piece,
                                                                const PrePiece* cuts) {
  constexpr uint32_t kRows = FEW ? 1024 / D : 1, kParts = kPreRows / kRows;
  const uint32_t G = a.s.n_kv_heads, group = a.n_heads / G;
  const uint32_t kvh = blockIdx.x / kParts % G, item = blockIdx.x / kParts / G;
  uint32_t e = item, p0, n;
  if (plan.listed)
    e = cuts[item].e, p0 = cuts[item].slot, n = cuts[item].n;
  else
    p0 = first_piece[e], n = first_piece[e + 1] - p0;
  if (n <= 1) return;  // written by the piece itself
  const PreItem i = pre_item(a, plan, e);
  const Kv4Seq seq = kv4_seq(a, i.b);
  const uint32_t r = blockIdx.x % kParts * kRows + (FEW ? threadIdx.x / (D / 4) : 0);
  const uint32_t rr = i.rt * kPreRows + r;
  if (rr >= seq.nq * group) return;
  float* dst = a.o + ((size_t)(seq.q0 + rr / group) * a.n_heads + kvh * group + rr % group) * D;
  auto at = [&](uint32_t x) { return ((size_t)(p0 + x) * G + kvh) * kPreRows + r; };
  if constexpr (FEW)
    merge_few<D>(part, n, at, dst);
  else
    merge_pieces<D, 256>(part, n, at, dst);
}

// n_tokens: 0xffffffff for the workspace of any.
static PrePlan prefill_plan(uint32_t n_seqs, uint32_t n_tokens, uint32_t max_q, uint32_t max_n_keys,
                            uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                            uint32_t window, uint32_t n_sinks) {
  PrePlan p{};
  const uint32_t group = n_heads / n_kv_heads;
  p.row_tiles = (uint32_t)(((uint64_t)max_q * group + kPreRows - 1) / kPreRows);
  const uint64_t items = (uint64_t)n_seqs * p.row_tiles;
  const uint64_t tiles = kv4_max_tiles(max_n_keys, kPreRows / group + 2, window, n_sinks);
  const uint64_t most = (tiles + kPreLeast - 1) / kPreLeast;  // pieces of a row tile
  const uint32_t resident = 256 * (head_dim == 64 ? kPreResident<64> : kPreResident<128>);
  p.many = std::max(1u, kPreMany / n_kv_heads);
  p.more = std::max(1u, kPreMore / n_kv_heads);
  p.pieces = items < p.many || items > kMaxCut ? std::max(1u, resident / n_kv_heads) : p.more;
  if (items > kMaxCut && (items > 2 * kMaxCut || tiles > kShortTiles)) {
    p.listed = true;
    // Row tiles with rows; as many pieces more as the cuts make, each cut row tile being longer
    // than its share of the total.
    const uint64_t real = std::min(items, (uint64_t)n_tokens * group / kPreRows + n_seqs);
    const uint32_t pieces = std::max(p.pieces, p.more);
    p.runs = (uint32_t)std::min(real + pieces - 1, std::min(real * most, (uint64_t)0xffffffffu));
    p.cuts = tiles <= kShortTiles ? 0 : pieces;
    p.slots = 2 * p.cuts;
  } else if (most == 1 || items > kMaxCut) {
    p.pieces = 0;
    p.runs = (uint32_t)items;
  } else {
    p.runs = (uint32_t)std::min(p.pieces + items - 1, items * most);
    p.slots = p.runs;
  }
  return p;
}
static PrePlan prefill_plan(const Kv4AttnArgs& a) {
  return prefill_plan(a.n_seqs, a.n_tokens, a.max_q, a.max_n_keys, a.n_heads, a.s.n_kv_heads,
                      a.s.head_dim, a.window, a.n_sinks);
}

static uint64_t first_bytes(const PrePlan& p) {
  return p.listed ? ws_align(((uint64_t)p.runs + p.cuts) * sizeof(PrePiece))
                  : ws_align((kMaxCut + 1) * 4);
}

uint64_t kv4_prefill_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                              uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                              uint32_t window, uint32_t n_sinks) {
  const PrePlan p = prefill_plan(n_seqs, 0xffffffffu, max_q, max_n_keys, n_heads, n_kv_heads,
                                 head_dim, window, n_sinks);
  if (p.pieces == 0) return 0;
  const uint64_t rows = (uint64_t)p.slots * n_kv_heads * kPreRows;
  return first_bytes(p) + ws_align(rows * 8) + ws_align(rows * head_dim * 4);
}

bool kv4_prefill_fits(const Kv4AttnArgs& a) {
  const uint32_t G = a.s.n_kv_heads;
  const PrePlan p = prefill_plan(a);
  const uint64_t items = (uint64_t)a.n_seqs * p.row_tiles;
  const uint64_t tiles = kv4_max_tiles(a.max_n_keys, a.max_q, a.window, a.n_sinks);
  if (items > kMaxGroups || (uint64_t)p.runs * G > kMaxGroups) return false;
  // (Tiles of every row tile that the bounds allow, whatever q_off holds.)
  return p.pieces == 0 || ((uint64_t)(p.listed ? p.cuts : items) * G * kPreRows <= kMaxGroups &&
                           items * tiles <= 0xffffffffull);
}

template <int D>
static hipError_t launch(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  const uint32_t G = a.s.n_kv_heads;
  const PrePlan p = prefill_plan(a);
  const uint32_t items = a.n_seqs * p.row_tiles, grid = p.runs * G;
  uint32_t* first_piece = nullptr;
  PrePiece *cuts = nullptr, *list = nullptr;
  Kv4Part part{};
  if (p.pieces > 0) {
    uint8_t* w = static_cast<uint8_t*>(ws);
    if (p.listed)
      cuts = reinterpret_cast<PrePiece*>(w), list = cuts + p.cuts;
    else
      first_piece = reinterpret_cast<uint32_t*>(w);
    w += first_bytes(p);
    part.ml = reinterpret_cast<float*>(w);
    part.acc = reinterpret_cast<float*>(w + ws_align((uint64_t)p.slots * G * kPreRows * 8));
  }
  if (p.listed) {
    hipLaunchKernelGGL(kv4_prefill_list_kernel, dim3(1), dim3(kListThreads), 0, st, a, p, list,
                       cuts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const float scale = (float)(kLog2e / sqrt((double)D));
  hipLaunchKernelGGL(kv4_prefill_kernel<D>, dim3(grid), dim3(kPreThreads), 0, st, a, p, part,
                     first_piece, list, scale);
  const hipError_t e = hipGetLastError();
  const uint32_t merged = p.listed ? p.cuts : p.runs > items ? items : 0;
  if (e != hipSuccess || p.pieces == 0 || merged == 0) return e;
  if (!p.listed && p.runs >= 8 * items)  // many pieces a row tile
    hipLaunchKernelGGL((kv4_prefill_merge_kernel<D, false>), dim3(merged * G * kPreRows), dim3(256),
                       0, st, a, p, part, first_piece, cuts);
  else
    hipLaunchKernelGGL((kv4_prefill_merge_kernel<D, true>),
                       dim3(merged * G * (kPreRows * D / 1024)), dim3(256), 0, st, a, p, part,
                       first_piece, cuts);
  return hipGetLastError();
}

hipError_t launch_kv4_prefill(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  return a.s.head_dim == 128 ? launch<128>(a, ws, st) : launch<64>(a, ws, st);
}

}  // namespace flk
