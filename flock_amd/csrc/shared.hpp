// Decode attention of sequences that share prefixes: arguments, the plan of a call's work,
// launches.
#pragma once

#include "common.hpp"

namespace flk {

struct SharedArgs {
  const float *q, *kcache, *vcache;
  const uint64_t *prefix_row, *seq_row_off;
  const uint32_t *n_prefix, *seq_off, *n_keys;
  float* o;
  uint32_t n_groups, n_seqs, max_prefix, max_n_keys, n_heads, n_kv_heads, head_dim;
  bool step;  // the layer's step: n_keys[b] = 0 is an idle sequence
};

// Rows of q that meet the same keys are taken together: the m = n_heads / n_kv_heads query
// heads of a kv head, of every sequence of a group (its row of q is sequence * m + head of the
// kv head), in row tiles of 128, and the m of one sequence for its own keys. An item is a row tile
// and a piece of its keys for one kv head; its partial results are rows `part` .. of them.
constexpr uint32_t kSharedRows = 128;
struct alignas(16) SharedItem {
  uint64_t key_row;  // of the caches
  uint32_t n_keys, row0, n_rows, part, kvh, pad;
};
// Where a sequence's partial results lie: of piece p, kv head h and head j of it at
// prefix + p * prefix_step + h * prefix_head + j and own + (p * n_kv_heads + h) * m + j.
struct alignas(16) SharedRecord {
  uint32_t prefix, prefix_n, prefix_step, prefix_head, own, own_n, pad[2];
};
constexpr uint32_t kSharedRefused = 0xffffffffu, kSharedIdle = 0xfffffffeu;  // counts

struct SharedPlan {
  uint32_t tile;     // keys of a tile
  uint32_t pieces;   // of a kv head's tiles, over all of its row tiles: about so many items
  uint32_t items;    // at most
  uint64_t parts;    // rows of partial results, at most
  uint32_t* n_items;
  SharedItem* item;
  SharedRecord* record;
  float2* ml;        // (reference, sum) of a row
  float* acc;        // its output, normalised
};

constexpr uint32_t kSharedLeast = 2;  // tiles of an item at least, where there are as many

// Sum over the workgroup, and over the threads before this one, in 64 bits.
template <int kWaves>
__device__ __forceinline__ uint64_t shared_scan(uint64_t v, uint64_t* s_wave, uint64_t& before) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t scan = v;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const uint64_t y = __shfl_up((unsigned long long)scan, x, kWave);
    if (lane >= x) scan += y;
  }
  __syncthreads();  // s_wave may still be read
  if (lane == 63) s_wave[wave] = scan;
  __syncthreads();
  uint64_t total = 0;
  before = scan - v;
  for (int w = 0; w < kWaves; w++) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  return total;
}

// The items of a call and the sequences' records, by one workgroup. Lengths come from the
// device, so the pieces are cut by the work there is: `pieces` of them over all row tiles of
// a kv head, each of as many tiles, a row tile's last one shorter. All row tiles of a group
// have the same pieces, neighbours in the list, so that they read a piece's keys at the same time.
template <int kThreads>
__device__ __forceinline__ void shared_plan(const SharedArgs& a, const SharedPlan& p) {
  constexpr int kWaves = kThreads / 64;
  __shared__ uint64_t s_wave[kWaves];
  __shared__ uint32_t s_first[kThreads + 1], s_off[kThreads + 1], s_n[kThreads], s_part[kThreads];
  __shared__ uint32_t s_bad;
  const uint32_t t = threadIdx.x, G = a.n_kv_heads, m = a.n_heads / G;
  auto tiles_of = [&](uint32_t keys) { return keys / p.tile + (keys % p.tile != 0); };
  auto row_tiles = [&](uint32_t seqs) { return (seqs * m + kSharedRows - 1) / kSharedRows; };
  if (t == 0) s_bad = 0;
  __syncthreads();
  uint64_t work = 0, before;
  for (uint32_t g = t; g < a.n_groups; g += kThreads) {
    const uint32_t lo = a.seq_off[g], hi = a.seq_off[g + 1], n = a.n_prefix[g];
    if (lo > hi || hi > a.n_seqs)
      s_bad = 1;
    else if (n <= a.max_prefix)
      work += (uint64_t)row_tiles(hi - lo) * tiles_of(n);
  }
  for (uint32_t b = t; b < a.n_seqs; b += kThreads) {
    const uint32_t n = a.n_keys[b];
    if (n <= a.max_n_keys) work += tiles_of(n);
  }
  work = shared_scan<kWaves>(work, s_wave, before);
  if (s_bad) {  // (seen by all: the sum's barriers)
    for (uint32_t b = t; b < a.n_seqs; b += kThreads)
      p.record[b] = SharedRecord{0, kSharedRefused, 0, 0, 0, kSharedRefused, {0, 0}};
    if (t == 0) *p.n_items = 0;
    return;
  }
  const uint64_t share = (work + p.pieces - 1) / p.pieces;
  const uint32_t per = share > kSharedLeast ? (uint32_t)share : kSharedLeast;
  uint64_t item0 = 0, part0 = 0;

  // The entry of s_first that an item lies in, of n.
  auto find = [&](const uint32_t* first, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
  };
  for (uint32_t g0 = 0; g0 < a.n_groups; g0 += kThreads) {
    const uint32_t n_here = min((uint32_t)kThreads, a.n_groups - g0), g = g0 + t;
    uint32_t lo = 0, hi = 0, n = 0, pieces = 0;
    if (t < n_here) {
      lo = a.seq_off[g], hi = a.seq_off[g + 1], n = a.n_prefix[g];
      if (n <= a.max_prefix && hi > lo) pieces = (tiles_of(n) + per - 1) / per;
    }
    uint64_t at_item, at_part;
    const uint32_t items = pieces * row_tiles(hi - lo) * G;
    const uint64_t all = shared_scan<kWaves>(items, s_wave, at_item);
    const uint64_t parts = shared_scan<kWaves>((uint64_t)pieces * (hi - lo) * m * G, s_wave, at_part);
    s_first[t] = (uint32_t)at_item;
    if (t < n_here) s_off[t] = lo;
    s_n[t] = n > a.max_prefix ? kSharedRefused : pieces;
    s_part[t] = (uint32_t)(part0 + at_part);
    if (t + 1 == n_here) s_off[n_here] = hi;
    __syncthreads();
    for (uint32_t i = t; i < (uint32_t)all; i += kThreads) {
      // (The last group that starts at or before item i: empty ones share its first item.)
      const uint32_t e = find(s_first, n_here, i);
      const uint32_t x = i - s_first[e], kvh = x % G;
      const uint32_t rows = (s_off[e + 1] - s_off[e]) * m, rts = (rows + kSharedRows - 1) / kSharedRows;
      const uint32_t rt = x / G % rts, piece = x / G / rts;
      const uint32_t keys = a.n_prefix[g0 + e], nt = tiles_of(keys);
      const uint32_t t0 = (uint32_t)((uint64_t)nt * piece / s_n[e]);
      const uint32_t t1 = (uint32_t)((uint64_t)nt * (piece + 1) / s_n[e]);
      const uint64_t end = min((uint64_t)t1 * p.tile, (uint64_t)keys);
      SharedItem item;
      item.key_row = a.prefix_row[g0 + e] + (uint64_t)t0 * p.tile;
      item.n_keys = (uint32_t)(end - (uint64_t)t0 * p.tile);
      item.row0 = s_off[e] * m + rt * kSharedRows;
      item.n_rows = min(kSharedRows, rows - rt * kSharedRows);
      item.part = s_part[e] + (piece * G + kvh) * rows + rt * kSharedRows;
      item.kvh = kvh, item.pad = 0;
      p.item[item0 + i] = item;
    }
    for (uint32_t b = s_off[0] + t; b < s_off[n_here]; b += kThreads) {
      const uint32_t e = find(s_off, n_here, b), rows = (s_off[e + 1] - s_off[e]) * m;
      SharedRecord& r = p.record[b];
      r.prefix = s_part[e] + (b - s_off[e]) * m, r.prefix_n = s_n[e];
      r.prefix_step = rows * G, r.prefix_head = rows;
    }
    item0 += all, part0 += parts;
    __syncthreads();
  }
  for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += kThreads) {
    const uint32_t n_here = min((uint32_t)kThreads, a.n_seqs - b0), b = b0 + t;
    uint32_t n = 0, pieces = 0;
    if (t < n_here) {
      n = a.n_keys[b];
      if (n <= a.max_n_keys) pieces = (tiles_of(n) + per - 1) / per;
    }
    uint64_t at_item;
    const uint64_t all = shared_scan<kWaves>((uint64_t)pieces * G, s_wave, at_item);
    const uint32_t part = (uint32_t)(part0 + at_item * m);
    s_first[t] = (uint32_t)at_item, s_n[t] = pieces, s_part[t] = part;
    if (t < n_here) {
      SharedRecord& r = p.record[b];
      r.own = part;
      r.own_n = n > a.max_n_keys ? kSharedRefused : n == 0 && a.step ? kSharedIdle : pieces;
      if (b < a.seq_off[0] || b >= a.seq_off[a.n_groups]) r.prefix_n = 0;
    }
    __syncthreads();
    for (uint32_t i = t; i < (uint32_t)all; i += kThreads) {
      const uint32_t e = find(s_first, n_here, i), x = i - s_first[e];
      const uint32_t kvh = x % G, piece = x / G, keys = a.n_keys[b0 + e], nt = tiles_of(keys);
      const uint32_t t0 = (uint32_t)((uint64_t)nt * piece / s_n[e]);
      const uint32_t t1 = (uint32_t)((uint64_t)nt * (piece + 1) / s_n[e]);
      const uint64_t end = min((uint64_t)t1 * p.tile, (uint64_t)keys);
      SharedItem item;
      item.key_row = a.seq_row_off[b0 + e] + (uint64_t)t0 * p.tile;
      item.n_keys = (uint32_t)(end - (uint64_t)t0 * p.tile);
      item.row0 = (b0 + e) * m, item.n_rows = m;
      item.part = s_part[e] + x * m;
      item.kvh = kvh, item.pad = 0;
      p.item[item0 + i] = item;
    }
    item0 += all, part0 += all * m;
    __syncthreads();
  }
  if (t == 0) *p.n_items = (uint32_t)item0;
}

// What a sequence sees.
struct SharedSeq {
  uint32_t prefix, own;
  bool refused, idle;
};

// The group of sequence b, by every thread of a workgroup: the one whose range holds it.
// Offsets that fall, or pass n_seqs, refuse the whole call (NaN), so that no sequence is
// in two groups.
template <int kThreads>
__device__ __forceinline__ SharedSeq shared_seq(const SharedArgs& a, uint32_t b) {
  __shared__ uint32_t s_group, s_bad;
  if (threadIdx.x == 0) s_group = 0xffffffffu, s_bad = 0;
  __syncthreads();
  for (uint32_t g = threadIdx.x; g < a.n_groups; g += kThreads) {
    const uint32_t lo = a.seq_off[g], hi = a.seq_off[g + 1];
    if (lo > hi || hi > a.n_seqs) s_bad = 1;
    if (lo <= b && b < hi) s_group = g;
  }
  __syncthreads();
  SharedSeq s{};
  const uint32_t g = s_group;
  s.own = a.n_keys[b];
  if (g < a.n_groups) s.prefix = a.n_prefix[g];
  s.refused = s_bad || s.own > a.max_n_keys || s.prefix > a.max_prefix;
  s.idle = !s.refused && a.step && s.own == 0;
  return s;
}

uint64_t shared_ws_bytes(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                         uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                         uint32_t head_dim);
// Whether a call's launches and its numbers of rows and items (32 bits) hold it.
bool shared_fits(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix, uint32_t max_n_keys,
                 uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim);
// fused: the step's raw rows and gains (null: attention alone), q rows q_stride floats
// apart, k and v rows kv_stride.
hipError_t launch_shared(const SharedArgs& a, const DecodeFused* fused, uint32_t q_stride,
                         uint32_t kv_stride, void* ws, hipStream_t st);
// The step's norm, rotation and append, and the plan.
hipError_t launch_shared_prologue(const SharedArgs& a, const SharedPlan& p, const DecodeFused& f,
                                  uint32_t q_stride, uint32_t kv_stride, hipStream_t st);

}  // namespace flk
