// Decode attention of sequences that share long prefixes: each sequence's token sees its
// group's prefix keys and its own.
//
// One workgroup a query head of a sequence: its waves deal out the keys, each with a
// running maximum and sum, and join in LDS.
#include "shared.hpp"

namespace flk {

constexpr int kSharedThreads = 256;

template <int D>
__global__ __launch_bounds__(kSharedThreads) void shared_simple_kernel(SharedArgs a, float scale) {
  constexpr int kWaves = kSharedThreads / 64, kE = D / 64;
  __shared__ float s_m[kWaves], s_l[kWaves], s_acc[kWaves][D];
  const uint32_t h = blockIdx.x, b = blockIdx.y, G = a.n_kv_heads;
  const uint32_t kvh = h / (a.n_heads / G);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const SharedSeq s = shared_seq<kSharedThreads>(a, b);
  const size_t at = ((size_t)b * a.n_heads + h) * D;
  if (s.refused || s.idle) {
    if (threadIdx.x < D) a.o[at + threadIdx.x] = s.refused ? __builtin_nanf("") : 0.f;
    return;
  }
  float q[kE], acc[kE] = {}, m = -INFINITY, l = 0.f;
  for (int e = 0; e < kE; e++) q[e] = a.q[at + lane + 64 * e] * scale;
  const uint64_t own_row = a.seq_row_off[b];
  for (uint64_t i = wave; i < (uint64_t)s.prefix + s.own; i += kWaves) {
    const uint64_t row = i < s.prefix ? s.prefix_row + i : own_row + (i - s.prefix);
    const size_t src = (row * G + kvh) * D + lane;
    float x = 0.f;
    for (int e = 0; e < kE; e++) x = fmaf(q[e], a.kcache[src + 64 * e], x);
    x = group_sum<64>(x);
    const float top = fmaxf(m, x), w = expf(m - top), p = expf(x - top);
    l = fmaf(l, w, p);
    for (int e = 0; e < kE; e++) acc[e] = fmaf(acc[e], w, p * a.vcache[src + 64 * e]);
    m = top;
  }
  if (lane == 0) s_m[wave] = m, s_l[wave] = l;
  for (int e = 0; e < kE; e++) s_acc[wave][lane + 64 * e] = acc[e];
  __syncthreads();
  if (threadIdx.x >= D) return;
  float top = -INFINITY, sum = 0.f, out = 0.f;
  for (int w = 0; w < kWaves; w++) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kWaves; w++) {
    const float k = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - top);
    sum = fmaf(s_l[w], k, sum);
    out = fmaf(s_acc[w][threadIdx.x], k, out);
  }
  a.o[at + threadIdx.x] = sum == 0.f ? 0.f : out / sum;
}

uint64_t shared_ws_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) {
  return 0;
}

hipError_t launch_shared(const SharedArgs& a, const DecodeFused* fused, uint32_t q_stride,
                         uint32_t kv_stride, void*, hipStream_t st) {
  if (fused != nullptr) {
    const hipError_t e = launch_shared_prologue(a, *fused, q_stride, kv_stride, st);
    if (e != hipSuccess) return e;
  }
  const dim3 grid(a.n_heads, a.n_seqs);
  const float scale = (float)(1.0 / sqrt((double)a.head_dim));
  if (a.head_dim == 128)
    hipLaunchKernelGGL(shared_simple_kernel<128>, grid, dim3(kSharedThreads), 0, st, a, scale);
  else
    hipLaunchKernelGGL(shared_simple_kernel<64>, grid, dim3(kSharedThreads), 0, st, a, scale);
  return hipGetLastError();
}

}  // namespace flk
