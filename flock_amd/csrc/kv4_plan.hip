// Block tables and slot maps of a paged cache from request lengths, on the GPU.
//
// Integers only. Each sequence's row of the table is looked at by one wave; what
// needs a number over the whole batch (which free page a block takes, where a
// released page goes, where a sequence's tokens start) is a prefix sum in
// (sequence, block) order: a first launch counts, 16 sequences per workgroup, and
// the second sums the counts of the workgroups before its own.
#include "kv4.hpp"

namespace flk {

constexpr int kPlanWaves = 16;  // sequences of a workgroup, a wave each

struct PlanCount {
  uint32_t need, drop, fresh;  // blocks to take, blocks to release, new tokens
};

struct PlanSeq {
  uint32_t keys, fresh, first;  // first: the earliest key that the new tokens see
};

__device__ __forceinline__ PlanSeq plan_seq(const Kv4PlanArgs& a, uint32_t b) {
  PlanSeq s;
  s.keys = a.n_keys[b];
  s.fresh = min(a.n_new[b], s.keys);
  const int64_t first = (int64_t)s.keys - s.fresh - a.window + 1;
  s.first = first > 0 ? (uint32_t)first : 0u;
  return s;
}

// Whether the sequence holds block i after the step.
__device__ __forceinline__ bool plan_wants(const Kv4PlanArgs& a, const PlanSeq& s, uint32_t i) {
  const uint64_t begin = (uint64_t)i * a.page;
  return begin < s.keys &&
         (a.window == 0 || begin + a.page > s.first || begin < a.n_sinks);
}

// This lane's entry of row b (kNoPage past the row) and what becomes of it.
__device__ __forceinline__ uint32_t plan_entry(const Kv4PlanArgs& a, const PlanSeq& s, uint32_t b,
                                               uint32_t i, bool& need, bool& drop) {
  uint32_t e = i < a.max_blocks ? a.table_in[(size_t)b * a.max_blocks + i] : kNoPage;
  const bool have = e < a.n_pages, want = i < a.max_blocks && plan_wants(a, s, i);
  need = want && !have;
  drop = have && !want;
  return e;
}

__device__ __forceinline__ PlanCount plan_count(const Kv4PlanArgs& a, const PlanSeq& s,
                                                uint32_t b) {
  const int lane = threadIdx.x & 63;
  PlanCount c{0, 0, s.fresh};
  for (uint32_t base = 0; base < a.max_blocks; base += 64) {
    bool need, drop;
    plan_entry(a, s, b, base + lane, need, drop);
    c.need += __popcll(__ballot(need));
    c.drop += __popcll(__ballot(drop));
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

__global__ __launch_bounds__(kPlanWaves * 64) void kv4_plan_kernel(Kv4PlanArgs a,
                                                                   const PlanCount* seq_count,
                                                                   const PlanCount* wg_count) {
  __shared__ uint32_t s_sum[6];          // before this workgroup, and in all
  __shared__ PlanCount s_count[kPlanWaves];
  __shared__ uint32_t s_lost;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t b = blockIdx.x * kPlanWaves + wave;
  if (threadIdx.x < 6) s_sum[threadIdx.x] = 0;
  if (threadIdx.x == 0) s_lost = 0;
  if (lane == 0) s_count[wave] = b < a.n_seqs ? seq_count[b] : PlanCount{0, 0, 0};
  __syncthreads();
  {
    uint32_t before[3] = {0, 0, 0}, all[3] = {0, 0, 0};
    for (uint32_t w = threadIdx.x; w < gridDim.x; w += blockDim.x) {
      const PlanCount c = wg_count[w];
      const uint32_t v[3] = {c.need, c.drop, c.fresh};
      for (int k = 0; k < 3; k++) {
        all[k] += v[k];
        if (w < blockIdx.x) before[k] += v[k];
      }
    }
    for (int k = 0; k < 3; k++) {
      if (before[k]) atomicAdd(&s_sum[k], before[k]);
      if (all[k]) atomicAdd(&s_sum[3 + k], all[k]);
    }
  }
  __syncthreads();
  PlanCount at{s_sum[0], s_sum[1], s_sum[2]};
  for (int w = 0; w < wave; w++) {
    at.need += s_count[w].need;
    at.drop += s_count[w].drop;
    at.fresh += s_count[w].fresh;
  }
  const uint32_t total = s_sum[5];
  const uint32_t n_free = min(a.free_in[0], a.n_pages);
  const uint32_t left = n_free - min(s_sum[3], n_free);  // of the old list

  uint32_t mapped = 0;  // tokens of this sequence that got a slot
  if (b < a.n_seqs) {
    const PlanSeq s = plan_seq(a, b);
    if (lane == 0) {
      a.q_off[b] = at.fresh;
      if (b == a.n_seqs - 1) a.q_off[a.n_seqs] = at.fresh + s.fresh;
    }
    const uint32_t pos0 = s.keys - s.fresh;
    uint32_t need_at = at.need, drop_at = at.drop;
    for (uint32_t base = 0; base < a.max_blocks; base += 64) {
      const uint32_t i = base + lane;
      bool need, drop;
      uint32_t e = plan_entry(a, s, b, i, need, drop);
      const uint64_t below = (1ull << lane) - 1;
      const uint64_t needs = __ballot(need), drops = __ballot(drop);
      if (drop) {
        const uint32_t to = left + drop_at + __popcll(drops & below);
        if (to < a.n_pages) a.free_out[1 + to] = e;
        e = kNoPage;
      }
      if (need) {
        const uint32_t k = need_at + __popcll(needs & below);
        e = k < n_free ? a.free_in[n_free - k] : kNoPage;  // entry n_free - 1 - k of the list
      }
      need_at += __popcll(needs);
      drop_at += __popcll(drops);
      if (i < a.max_blocks) a.table_out[(size_t)b * a.max_blocks + i] = e;
      // The new tokens that lie in these 64 blocks, block by block.
      const uint64_t lo = max((uint64_t)base * a.page, (uint64_t)pos0);
      const uint64_t hi = min((uint64_t)min(base + 64, a.max_blocks) * a.page, (uint64_t)s.keys);
      for (uint64_t p = lo; p < hi;) {
        const uint32_t blk = (uint32_t)(p / a.page);
        const uint64_t end = min((uint64_t)(blk + 1) * a.page, hi);
        const uint32_t page_id = __shfl((int)e, (int)(blk - base), kWave);
        const bool ok = page_id < a.n_pages;
        for (uint64_t x = p + lane; x < end; x += 64) {
          const uint64_t t = at.fresh + (x - pos0);
          if (t >= a.max_tokens) continue;
          a.positions[t] = (uint32_t)x;
          a.slots[t] = ok ? page_id * a.page + (uint32_t)(x - (uint64_t)blk * a.page) : kNoPage;
        }
        if (ok) {
          const uint64_t t0 = at.fresh + (p - pos0), t1 = at.fresh + (end - pos0);
          const uint64_t cap = a.max_tokens;
          mapped += (uint32_t)(min(t1, cap) - min(t0, cap));
        }
        p = end;
      }
    }
    // Tokens behind the table's last block.
    const uint64_t cap = (uint64_t)a.max_blocks * a.page;
    for (uint64_t x = max(cap, (uint64_t)pos0) + lane; x < s.keys; x += 64) {
      const uint64_t t = at.fresh + (x - pos0);
      if (t >= a.max_tokens) break;
      a.positions[t] = (uint32_t)x;
      a.slots[t] = kNoPage;
    }
    if (lane == 0 && mapped != s.fresh) atomicAdd(&s_lost, s.fresh - mapped);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (s_lost) atomicAdd(a.lost, s_lost);
    if (blockIdx.x == 0) a.free_out[0] = min(left + s_sum[4], a.n_pages);
  }
  // The part of the list that stays, and the map's entries behind the last token.
  const uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const uint64_t step = (uint64_t)gridDim.x * blockDim.x;
  for (uint64_t i = id; i < left; i += step) a.free_out[1 + i] = a.free_in[1 + i];
  for (uint64_t t = total + id; t < a.max_tokens; t += step) {
    a.positions[t] = 0;
    a.slots[t] = kNoPage;
  }
}

static uint32_t plan_wgs(uint32_t n_seqs) { return (n_seqs + kPlanWaves - 1) / kPlanWaves; }

uint64_t kv4_plan_ws_bytes(uint32_t n_seqs) {
  return ws_align(((uint64_t)n_seqs + plan_wgs(n_seqs)) * sizeof(PlanCount));
}

hipError_t launch_kv4_plan(const Kv4PlanArgs& a, void* ws, hipStream_t st) {
  PlanCount* seq = static_cast<PlanCount*>(ws);
  PlanCount* wg = seq + a.n_seqs;
  const dim3 grid(plan_wgs(a.n_seqs)), block(kPlanWaves * 64);
  hipLaunchKernelGGL(kv4_plan_count_kernel, grid, block, 0, st, a, seq, wg);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kv4_plan_kernel, grid, block, 0, st, a, seq, wg);
  return hipGetLastError();
}

}  // namespace flk
