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
// heads of a kv head, of every sequence of a group (a row is sequence * m + head of the kv
// head), in row tiles of up to 128 rows of whole sequences, and the m of one sequence for its
// own keys. A chain is a row tile and its keys, in tiles. The tiles of all chains, one after the
// other, are cut into runs of the same work: a run is one workgroup's for one kv head, whatever
// the lengths of the chains in it. Work is counted in tiles, and each chain is one more: to
// read q and to write the results takes about as long (64 sequences of one own key each, a tile
// a chain: 151 us for such a run, and 112 for as many tiles of a prefix).
constexpr uint32_t kSharedRows = 128;
struct alignas(16) SharedChain {
  uint64_t key_row;               // of the caches
  uint32_t n_keys, row0, n_rows;
  uint32_t start;                 // its first tile among all
  uint32_t first_run;             // the run that holds it
  uint32_t kind;                  // kSharedOwn: a sequence's own keys; kSharedOnce: read once
};
constexpr uint32_t kSharedOwn = 1, kSharedOnce = 2;
struct alignas(8) SharedRun {
  uint32_t chain, tile0;  // it ends where the next begins
};
// A sequence's partial results: prefix_n of its prefix (the first by run prefix_run, for a row
// tile whose first row is row0) and own_n of its own keys.
struct alignas(16) SharedRecord {
  uint32_t prefix_run, prefix_n, row0, own_run, own_n, pad[3];
};
constexpr uint32_t kSharedRefused = 0xffffffffu, kSharedIdle = 0xfffffffeu;  // counts

struct SharedPlan {
  uint32_t tile;      // keys of a tile
  uint32_t max_runs;  // of a kv head
  uint32_t chains;    // at most
  SharedRun* run;     // max_runs and one more; those behind the last have no tiles
  SharedChain* chain;
  SharedRecord* record;
  float2* ml;         // (reference, sum) of a partial result's row
  float* acc;         // its output, normalised
};

// Rows of partial results of a kv head: the first piece of every row's prefix, then of its
// own keys; a run that does not begin with a chain has room of its own for the first (only that
// piece is not the chain's first).
__host__ __device__ __forceinline__ uint64_t shared_parts(uint32_t rows, uint32_t runs) {
  return 2ull * rows + (uint64_t)runs * kSharedRows;
}


// The run that holds x of the work, cut into `runs`: run r begins at work * r / runs.
__device__ __forceinline__ uint32_t shared_run_of(uint32_t x, uint32_t work, uint32_t runs) {
  const uint64_t n = ((uint64_t)x + 1) * runs - 1;
  return n >> 32 ? (uint32_t)(n / work) : (uint32_t)n / work;
}
__device__ __forceinline__ uint32_t shared_run_start(uint32_t r, uint32_t work, uint32_t runs) {
  const uint64_t n = (uint64_t)work * r;
  return n >> 32 ? (uint32_t)(n / runs) : (uint32_t)n / runs;
}

// Exclusive sums over the workgroup's threads of two pairs (chains, tiles); the totals come back
// in a and b.
struct SharedPair {
  uint32_t chains, tiles;
};
template <int kWaves>
__device__ __forceinline__ void shared_scan(SharedPair& a, SharedPair& b, uint4* s_wave,
                                            SharedPair& before_a, SharedPair& before_b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint4 v = make_uint4(a.chains, a.tiles, b.chains, b.tiles);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const uint32_t p = __shfl_up(v.x, x, kWave), q = __shfl_up(v.y, x, kWave);
    const uint32_t r = __shfl_up(v.z, x, kWave), s = __shfl_up(v.w, x, kWave);
    if (lane >= x) v.x += p, v.y += q, v.z += r, v.w += s;
  }
  __syncthreads();  // s_wave may still be read
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  before_a = {v.x - a.chains, v.y - a.tiles};
  before_b = {v.z - b.chains, v.w - b.tiles};
  a = b = {0, 0};
  for (int w = 0; w < kWaves; w++) {
    const uint4 y = s_wave[w];
    if (w < wave) {
      before_a.chains += y.x, before_a.tiles += y.y;
      before_b.chains += y.z, before_b.tiles += y.w;
    }
    a.chains += y.x, a.tiles += y.y, b.chains += y.z, b.tiles += y.w;
  }
}

// A call's chains, runs and records, by one workgroup, from the lengths on the device. The chains
// of the groups come first, each group's row tiles one after the other.
template <int kThreads>
__device__ __forceinline__ void shared_plan(const SharedArgs& a, const SharedPlan& p) {
  constexpr int kWaves = kThreads / 64;
  __shared__ uint4 s_wave[kWaves];
  __shared__ uint32_t s_chain[kThreads], s_start[kThreads], s_off[kThreads + 1], s_keys[kThreads];
  __shared__ uint32_t s_bad;
  const uint32_t t = threadIdx.x, m = a.n_heads / a.n_kv_heads;
  const uint32_t tile_seqs = kSharedRows / m;  // sequences of a row tile
  auto tiles_of = [&](uint32_t keys) { return keys / p.tile + (keys % p.tile != 0); };
  auto row_tiles = [&](uint32_t seqs) { return seqs / tile_seqs + (seqs % tile_seqs != 0); };
  struct Group {
    uint32_t lo, hi, keys;  // keys = 0: refused too
    bool refused;
  };
  auto group = [&](uint32_t g) {
    Group x{0, 0, 0, false};
    if (g < a.n_groups) {
      x.lo = a.seq_off[g], x.hi = a.seq_off[g + 1], x.keys = a.n_prefix[g];
      x.refused = x.keys > a.max_prefix;
      if (x.refused) x.keys = 0;
    }
    return x;
  };
  auto group_pair = [&](const Group& x) {
    const uint32_t nt = tiles_of(x.keys), rts = nt ? row_tiles(x.hi - x.lo) : 0;
    return SharedPair{rts, rts * nt};
  };
  auto own_keys = [&](uint32_t b) {  // 0xffffffff: refused
    if (b >= a.n_seqs) return 0u;
    const uint32_t n = a.n_keys[b];
    return n > a.max_n_keys ? kSharedRefused : n;
  };
  auto own_pair = [&](uint32_t n) {
    const uint32_t nt = n == kSharedRefused ? 0 : tiles_of(n);
    return SharedPair{nt > 0, nt};
  };
  if (t == 0) s_bad = 0;
  __syncthreads();
  // Whole sums first; of the first group and sequence of a thread what it has read stays.
  const Group mine = group(t);
  const uint32_t mine_own = own_keys(t);
  SharedPair groups{0, 0}, owns{0, 0}, before_g, before_o;
  for (uint32_t g = t; g < a.n_groups; g += kThreads) {
    const Group x = g == t ? mine : group(g);
    if (x.lo > x.hi || x.hi > a.n_seqs) {
      s_bad = 1;
    } else {
      const SharedPair y = group_pair(x);
      groups.chains += y.chains, groups.tiles += y.tiles;
    }
  }
  for (uint32_t b = t; b < a.n_seqs; b += kThreads) {
    const SharedPair y = own_pair(b == t ? mine_own : own_keys(b));
    owns.chains += y.chains, owns.tiles += y.tiles;
  }
  shared_scan<kWaves>(groups, owns, s_wave, before_g, before_o);
  if (s_bad) {  // (seen by all: the sums' barriers)
    for (uint32_t b = t; b < a.n_seqs; b += kThreads)
      p.record[b] = SharedRecord{0, kSharedRefused, 0, 0, kSharedRefused, {0, 0, 0}};
    for (uint32_t r = t; r <= p.max_runs; r += kThreads) p.run[r] = SharedRun{0, 0};
    return;
  }
  const uint32_t tiles = groups.tiles + owns.tiles;
  const uint32_t work = tiles + groups.chains + owns.chains;
  // (As many as there is work for: a run's one tile at least, or the start of a chain and none.
  // Runs of one / two / three at least, us: 2 sequences over 200 keys 15.6 / 17.4 / 18.9, 8 over
  // 1000 18.9 / 19.4 / 20.7, over 3000 23.0 / 22.6 / 24.5.)
  const uint32_t runs = min(p.max_runs, work);
  for (uint32_t r = runs + t; r <= p.max_runs; r += kThreads) p.run[r] = SharedRun{0, tiles};
  // Tile x (among all) of a chain that c others precede lies at x + c + 1 of the work.
  auto run_of = [&](uint32_t x, uint32_t c) {
    return shared_run_of(x + c + 1, work, runs);
  };

  // The last of n entries that does not begin above x.
  auto find = [&](uint32_t n, uint32_t x, auto begin) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (begin(mid) <= x) lo = mid; else hi = mid;
    }
    return lo;
  };
  // Runs that begin in a range of the work: the chain there, and how many tiles of it are before.
  auto put_runs = [&](uint32_t from, uint32_t to, auto chain_at) {
    for (uint32_t r = t; r < runs; r += kThreads) {
      const uint32_t x = shared_run_start(r, work, runs);
      if (x >= from && x < to) p.run[r] = chain_at(x);
    }
  };
  uint32_t chain0 = 0, tile0 = 0;
  for (uint32_t g0 = 0; g0 < a.n_groups; g0 += kThreads) {
    const uint32_t n_here = min((uint32_t)kThreads, a.n_groups - g0);
    const Group x = g0 == 0 ? mine : group(g0 + t);
    SharedPair here = t < n_here ? group_pair(x) : SharedPair{0, 0}, none{0, 0};
    shared_scan<kWaves>(here, none, s_wave, before_g, before_o);
    s_chain[t] = before_g.chains, s_start[t] = tile0 + before_g.tiles;
    s_keys[t] = x.refused ? kSharedRefused : x.keys;
    if (t < n_here) s_off[t] = x.lo;
    if (t + 1 == n_here) s_off[n_here] = x.hi;
    __syncthreads();
    for (uint32_t i = t; i < here.chains; i += kThreads) {
      // (Of entries without chains, which share the next one's first, find passes all.)
      const uint32_t e = find(n_here, i, [&](uint32_t j) { return s_chain[j]; });
      const uint32_t rt = i - s_chain[e], nt = tiles_of(s_keys[e]);
      const uint32_t seq0 = s_off[e] + rt * tile_seqs, start = s_start[e] + rt * nt;
      SharedChain c;
      c.key_row = a.prefix_row[g0 + e];
      c.n_keys = s_keys[e], c.row0 = seq0 * m;
      c.n_rows = min(tile_seqs, s_off[e + 1] - seq0) * m;
      c.start = start, c.first_run = run_of(start, chain0 + i);
      c.kind = s_off[e + 1] - s_off[e] <= tile_seqs ? kSharedOnce : 0;
      p.chain[chain0 + i] = c;
    }
    for (uint32_t b = s_off[0] + t; b < s_off[n_here]; b += kThreads) {
      const uint32_t e = find(n_here, b, [&](uint32_t j) { return s_off[j]; });
      const uint32_t keys = s_keys[e];
      const uint32_t nt = keys == kSharedRefused ? 0 : tiles_of(keys);
      const uint32_t rt = (b - s_off[e]) / tile_seqs, start = s_start[e] + rt * nt;
      SharedRecord& r = p.record[b];
      r.row0 = (s_off[e] + rt * tile_seqs) * m;
      r.prefix_n = keys == kSharedRefused ? keys : 0;
      if (nt > 0) {
        const uint32_t before = chain0 + s_chain[e] + rt;
        r.prefix_run = run_of(start, before);
        r.prefix_n = run_of(start + nt - 1, before) - r.prefix_run + 1;
      }
    }
    const uint32_t from = tile0 + chain0;
    put_runs(from, from + here.tiles + here.chains, [&](uint32_t x) {
      auto begin = [&](uint32_t j) { return s_start[j] + chain0 + s_chain[j]; };
      const uint32_t e = find(n_here, x, begin), nt = tiles_of(s_keys[e]);
      const uint32_t y = x - begin(e), rt = y / (nt + 1), i = y % (nt + 1);
      return SharedRun{chain0 + s_chain[e] + rt, s_start[e] + rt * nt + (i > 0 ? i - 1 : 0)};
    });
    chain0 += here.chains, tile0 += here.tiles;
    __syncthreads();
  }
  const uint32_t off_0 = a.seq_off[0], off_n = a.seq_off[a.n_groups];
  for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += kThreads) {
    const uint32_t n_here = min((uint32_t)kThreads, a.n_seqs - b0), b = b0 + t;
    const uint32_t n = b0 == 0 ? mine_own : own_keys(b);
    SharedPair here = t < n_here ? own_pair(n) : SharedPair{0, 0}, none{0, 0};
    const uint32_t nt = here.tiles;
    shared_scan<kWaves>(here, none, s_wave, before_g, before_o);
    const uint32_t start = tile0 + before_g.tiles;
    s_chain[t] = before_g.chains, s_start[t] = start;
    if (t < n_here) {
      SharedRecord& r = p.record[b];
      if (b < off_0 || b >= off_n) r.prefix_n = 0;
      r.own_n = n == kSharedRefused ? n : n == 0 && a.step ? kSharedIdle : 0;
      if (nt > 0) {
        const uint32_t before = chain0 + before_g.chains, first = run_of(start, before);
        r.own_run = first;
        r.own_n = run_of(start + nt - 1, before) - first + 1;
        p.chain[chain0 + before_g.chains] =
            SharedChain{a.seq_row_off[b], n, b * m, m, start, first, kSharedOwn | kSharedOnce};
      }
    }
    __syncthreads();
    const uint32_t from = tile0 + chain0;
    put_runs(from, from + here.tiles + here.chains, [&](uint32_t x) {
      auto begin = [&](uint32_t j) { return s_start[j] + chain0 + s_chain[j]; };
      const uint32_t e = find(n_here, x, begin), i = x - begin(e);
      return SharedRun{chain0 + s_chain[e], s_start[e] + (i > 0 ? i - 1 : 0)};
    });
    chain0 += here.chains, tile0 += here.tiles;
    __syncthreads();
  }
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
// Whether a call's launches and its numbers of rows and tiles (32 bits) hold it.
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
