// Block tables and slot maps of a paged cache from request lengths, on the GPU.
//
// Integers only, bound by latency (2048 sequences of 512 blocks: 8 MB and 10.6 us, two
// launches, in both of which a wave waits for the loads of its row eight times in turn). Each
// sequence's row of the table is looked at by one wave, 64 blocks at a time;
// what needs a number over the whole batch (which free page a block takes, where a released
// page goes, where a sequence's tokens start) is a prefix sum in (sequence, block) order. Up
// to 16 sequences, a wave of one workgroup each, count and write in one launch (6.4 us from
// the host, 3.9 of kernel); more are counted by a launch of its own, and every workgroup of
// the second sums the counts of those before it.
//
// The kernels use no blockDim and no private array that the compiler would keep in LDS: it
// takes the workgroup's size for either from the dispatch packet, in host memory, and every
// wave waits for that (25.5 us for 13.2, the same batch).
#include "kv4.hpp"

namespace flk {

// Sequences of a workgroup, a wave each: of the only one, and of many.
constexpr int kAloneWaves = 16, kPlanWaves = 8;

struct PlanCount {
  uint32_t need, drop, fresh;  // blocks to take, blocks to release, new tokens
};

struct PlanSeq {
  uint32_t keys, fresh, pos0;  // pos0: position of the first new token
  // Blocks it holds after the step: below `blocks`, and from `from` on or below `sinks`.
  uint32_t blocks, from, sinks;
  __device__ __forceinline__ bool wants(uint32_t i) const {
    return i < blocks && (i >= from || i < sinks);
  }
};

__device__ __forceinline__ PlanSeq plan_seq(const Kv4PlanArgs& a, uint32_t b) {
  const uint32_t log_page = 31 - __builtin_clz(a.page);
  auto blocks_of = [&](uint32_t n) { return (n >> log_page) + ((n & (a.page - 1)) != 0); };
  PlanSeq s;
  s.keys = a.n_keys[b];
  s.fresh = min(a.n_new[b], s.keys);
  s.pos0 = s.keys - s.fresh;
  // The earliest key that the first new token sees.
  const int64_t first = (int64_t)s.pos0 - a.window + 1;
  s.from = a.window == 0 || first <= 0 ? 0u : (uint32_t)first >> log_page;
  s.blocks = min(blocks_of(s.keys), a.max_blocks);
  s.sinks = blocks_of(a.n_sinks);
  return s;
}

__device__ __forceinline__ uint32_t plan_entry(const Kv4PlanArgs& a, uint32_t b, uint32_t i) {
  return i < a.max_blocks ? a.table_in[(size_t)b * a.max_blocks + i] : kNoPage;
}

// A page whose block has keys that were not stored (their rows lay past max_tokens) is the
// sequence's still, but no entry that attention reads: bit 31, the page and the first such
// key's place in it, halved where the three take more than 32 bits (its even neighbour before
// it then). kNoPage is none of these.
struct PlanMark {
  uint32_t log_page, half;
  __device__ __forceinline__ explicit PlanMark(const Kv4PlanArgs& a)
      : log_page(31 - __builtin_clz(a.page)), half(a.n_pages >= 0x80000000u >> log_page) {}
  __device__ __forceinline__ uint32_t of(uint32_t id, uint32_t key) const {
    return 0x80000000u | id << (log_page - half) | key >> half;
  }
  __device__ __forceinline__ uint32_t page(uint32_t e) const {
    return (e & 0x7fffffffu) >> (log_page - half);
  }
  __device__ __forceinline__ uint32_t key(uint32_t e) const {
    return (e & ((1u << (log_page - half)) - 1)) << half;
  }
};

// Of block i with entry e (an entry past the row is none): its page, whether it takes one or
// gives it back, and whether keys of it from before the step, which its rows see, were stored
// nowhere. Such a block takes no page: with another's, attention would read what that held before.
struct PlanJudged {
  uint32_t id;
  bool need, drop, missing;
};
__device__ __forceinline__ PlanJudged plan_judge(const Kv4PlanArgs& a, const PlanSeq& s, uint32_t i,
                                                 uint32_t e) {
  const PlanMark mark(a);
  const bool marked = e >= 0x80000000u;
  const uint32_t id = marked ? mark.page(e) : e, key0 = i << mark.log_page;
  const bool have = id < a.n_pages, want = s.wants(i);
  // (A window of one token shows a row no key before the step, but for sinks.)
  const bool seen = a.window != 1 || i < s.sinks;
  const bool lacks = seen && key0 + (have && marked ? mark.key(e) : 0) < s.pos0;
  return {id, want && !have && !lacks, have && !want, want && lacks && (!have || marked)};
}

// Whether block i is as it has to be already, which most are.
__device__ __forceinline__ bool plan_settled(const Kv4PlanArgs& a, const PlanSeq& s, uint32_t i,
                                             uint32_t e) {
  return s.wants(i) ? e < a.n_pages : e == kNoPage;
}

__device__ __forceinline__ PlanCount plan_count(const Kv4PlanArgs& a, const PlanSeq& s,
                                                uint32_t b) {
  const int lane = threadIdx.x & 63;
  PlanCount c{0, 0, s.fresh};
  uint32_t next = plan_entry(a, b, lane);
#pragma unroll 1
  for (uint32_t base = 0; base < a.max_blocks; base += 64) {
    const uint32_t e = next;
    next = plan_entry(a, b, base + 64 + lane);
    if (__ballot(!plan_settled(a, s, base + lane, e)) == 0) continue;
    const PlanJudged j = plan_judge(a, s, base + lane, e);
    c.need += __popcll(__ballot(j.need));
    c.drop += __popcll(__ballot(j.drop));
  }
  return c;
}

__global__ __launch_bounds__(kPlanWaves * 64) void kv4_plan_count_kernel(Kv4PlanArgs a,
                                                                         PlanCount* seq_count,
                                                                         PlanCount* wg_count) {
  __shared__ PlanCount s_count[kPlanWaves];
  const int wave = threadIdx.x >> 6;
  const uint32_t b = blockIdx.x * kPlanWaves + wave;
  PlanCount c{0, 0, 0};
  if (b < a.n_seqs) c = plan_count(a, plan_seq(a, b), b);
  if ((threadIdx.x & 63) == 0) {
    s_count[wave] = c;
    if (b < a.n_seqs) seq_count[b] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    PlanCount sum{0, 0, 0};
    for (int w = 0; w < kPlanWaves; w++) {
      sum.need += s_count[w].need;
      sum.drop += s_count[w].drop;
      sum.fresh += s_count[w].fresh;
    }
    wg_count[blockIdx.x] = sum;
    if (blockIdx.x == 0) *a.lost = 0;
  }
}

// Sum over the wave.
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) v += __shfl_xor((int)v, x, kWave);
  return v;
}

// ALONE: the only workgroup, which counts for itself.
template <int W, bool ALONE>
__global__ __launch_bounds__(W * 64) void kv4_plan_kernel(Kv4PlanArgs a,
                                                          const PlanCount* seq_count,
                                                          const PlanCount* wg_count) {
  __shared__ uint32_t s_sum[6];  // needs, drops, new tokens before this workgroup, and in all
  __shared__ PlanCount s_count[W];
  __shared__ uint32_t s_lost;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t b = blockIdx.x * W + wave, n_wgs = (a.n_seqs + W - 1) / W;
  const PlanMark mark(a);
  const uint32_t log_page = mark.log_page;
  if (threadIdx.x == 0) s_lost = 0;
  PlanSeq s{};
  PlanCount own{0, 0, 0};
  uint32_t next = kNoPage;  // the first blocks are on their way while the sums are formed
  if (b < a.n_seqs) {
    next = plan_entry(a, b, lane);
    s = plan_seq(a, b);
    if constexpr (ALONE) {
      own = plan_count(a, s, b);
    } else {
      own.need = seq_count[b].need;
      own.drop = seq_count[b].drop;
      own.fresh = s.fresh;
    }
  }
  if (lane == 0) {
    s_count[wave].need = own.need;
    s_count[wave].drop = own.drop;
    s_count[wave].fresh = own.fresh;
  }
  const uint32_t n_free = min(a.free_in[0], a.n_pages);
  if (!ALONE && wave < 6) {  // a wave for each sum
    const uint32_t* word = reinterpret_cast<const uint32_t*>(wg_count) + wave % 3;
    const uint32_t end = wave < 3 ? blockIdx.x : n_wgs;
    uint32_t sum = 0;
    for (uint32_t w = lane; w < end; w += 64) sum += word[3 * (size_t)w];
    sum = wave_sum(sum);
    if (lane == 0) s_sum[wave] = sum;
  }
  __syncthreads();
  PlanCount at{0, 0, 0}, all{0, 0, 0};
  if (!ALONE) {
    at.need = s_sum[0], at.drop = s_sum[1], at.fresh = s_sum[2];
    all.need = s_sum[3], all.drop = s_sum[4], all.fresh = s_sum[5];
  }
#pragma unroll 1
  for (int w = 0; w < W; w++) {
    const uint32_t need = s_count[w].need, drop = s_count[w].drop, fresh = s_count[w].fresh;
    if (w < wave) at.need += need, at.drop += drop, at.fresh += fresh;
    if (ALONE) all.need += need, all.drop += drop, all.fresh += fresh;
  }
  const uint32_t left = n_free - min(all.need, n_free);  // of the old list

  // Its tokens that got a slot, its blocks that lack earlier keys.
  uint32_t mapped = 0, missing = 0;
  if (b < a.n_seqs) {
    if (lane == 0) {
      a.q_off[b] = at.fresh;
      if (b == a.n_seqs - 1) a.q_off[a.n_seqs] = at.fresh + s.fresh;
    }
    const uint32_t pos0 = s.pos0;
    // Tokens whose rows are within max_tokens.
    const uint32_t rows = min(s.fresh, at.fresh < a.max_tokens ? a.max_tokens - at.fresh : 0);
    // Blocks that the new tokens lie in.
    const uint32_t new_from = s.fresh ? pos0 >> log_page : 0xffffffffu, new_to = s.blocks;
    uint32_t need_at = at.need, drop_at = at.drop;
#pragma unroll 1
    for (uint32_t base = 0; base < a.max_blocks; base += 64) {
      const uint32_t i = base + lane;
      uint32_t e = next;
      next = plan_entry(a, b, i + 64);
      uint32_t id = e;
      if (__ballot(!plan_settled(a, s, i, e))) {
        const PlanJudged j = plan_judge(a, s, i, e);
        const uint64_t needs = __ballot(j.need), drops = __ballot(j.drop);
        const uint64_t below = (1ull << lane) - 1;
        id = j.id < a.n_pages && !j.drop && !j.missing ? j.id : kNoPage;
        // (A block that lacks keys of its page stays marked.)
        e = j.missing && j.id < a.n_pages ? e : id;
        if (j.drop) {
          const uint32_t to = left + drop_at + __popcll(drops & below);
          if (to < a.n_pages) a.free_out[1 + to] = j.id;
        }
        if (j.need) {
          const uint32_t n = need_at + __popcll(needs & below);
          e = id = n < n_free ? a.free_in[n_free - n] : kNoPage;  // n-th from the list's end
        }
        need_at += __popcll(needs);
        drop_at += __popcll(drops);
        missing += __popcll(__ballot(j.missing));
      }
      if (rows < s.fresh && id < a.n_pages) {  // which of them are not stored
        const uint32_t key0 = i << log_page, from = max(pos0 + rows, key0);
        if (from - key0 < a.page) e = mark.of(id, from - key0);
      }
      if (i < a.max_blocks) a.table_out[(size_t)b * a.max_blocks + i] = e;
      // The new tokens that lie in these 64 blocks, block by block.
      const uint32_t blk_end = min(base + 64, new_to);
#pragma unroll 1
      for (uint32_t blk = max(base, new_from); blk < blk_end; blk++) {
        const uint32_t p = max(blk << log_page, pos0);
        const uint32_t n = min(a.page - (p & (a.page - 1)), s.keys - p);
        const uint32_t page_id = __shfl((int)id, (int)(blk - base), kWave);
        const bool ok = page_id < a.n_pages;
        const uint64_t row = (uint64_t)at.fresh + (p - pos0);
#pragma unroll 1
        for (uint32_t x = lane; x < n && row + x < a.max_tokens; x += 64) {
          a.positions[row + x] = p + x;
          a.slots[row + x] = ok ? (page_id << log_page) + (p & (a.page - 1)) + x : kNoPage;
        }
        if (ok && row < a.max_tokens) mapped += (uint32_t)min((uint64_t)n, a.max_tokens - row);
      }
    }
    // Tokens behind the table's last block.
    const uint64_t cap = (uint64_t)a.max_blocks << log_page;
#pragma unroll 1
    for (uint64_t x = max(cap, (uint64_t)pos0) + lane; x < s.keys; x += 64) {
      const uint64_t t = at.fresh + (x - pos0);
      if (t >= a.max_tokens) break;
      a.positions[t] = (uint32_t)x;
      a.slots[t] = kNoPage;
    }
    const uint32_t lost = s.fresh - mapped + missing;
    if (lane == 0 && lost) atomicAdd(&s_lost, lost);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (ALONE) *a.lost = s_lost;
    else if (s_lost) atomicAdd(a.lost, s_lost);
    if (blockIdx.x == 0) a.free_out[0] = min(left + all.drop, a.n_pages);
  }
  // The part of the list that stays, and the map's entries behind the last token.
  const uint32_t id = blockIdx.x * (W * 64) + threadIdx.x, step = n_wgs * (W * 64);
#pragma unroll 1
  for (uint64_t i = id; i < left; i += step) a.free_out[1 + i] = a.free_in[1 + i];
#pragma unroll 1
  for (uint64_t t = all.fresh + id; t < a.max_tokens; t += step) {
    a.positions[t] = 0;
    a.slots[t] = kNoPage;
  }
}

static uint32_t plan_wgs(uint32_t n_seqs) { return (n_seqs + kPlanWaves - 1) / kPlanWaves; }

uint64_t kv4_plan_ws_bytes(uint32_t n_seqs) {
  return ws_align(((uint64_t)n_seqs + plan_wgs(n_seqs)) * sizeof(PlanCount));
}

hipError_t launch_kv4_plan(const Kv4PlanArgs& a, void* ws, hipStream_t st) {
  if (a.n_seqs <= kAloneWaves) {
    hipLaunchKernelGGL((kv4_plan_kernel<kAloneWaves, true>), dim3(1), dim3(kAloneWaves * 64), 0, st,
                       a, nullptr, nullptr);
    return hipGetLastError();
  }
  PlanCount* seq = static_cast<PlanCount*>(ws);
  PlanCount* wg = seq + a.n_seqs;
  const dim3 grid(plan_wgs(a.n_seqs)), block(kPlanWaves * 64);
  hipLaunchKernelGGL(kv4_plan_count_kernel, grid, block, 0, st, a, seq, wg);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((kv4_plan_kernel<kPlanWaves, false>), grid, block, 0, st, a, seq, wg);
  return hipGetLastError();
}

}  // namespace flk
