// Attention over the paged 4-bit cache: one wave per (query, head).
#include "kv4_attn.hpp"

namespace flk {

template <int D>
__global__ __launch_bounds__(64) void kv4_attn_kernel(Kv4AttnArgs a, float scale) {
  __shared__ float s_q[D], s_p[64];
  const uint32_t head = blockIdx.x, i = blockIdx.y, b = blockIdx.z, lane = threadIdx.x;
  const uint32_t q0 = min(a.q_off[b], a.n_tokens), q1 = min(a.q_off[b + 1], a.n_tokens);
  const uint32_t nq = q1 > q0 ? q1 - q0 : 0, n_keys = a.n_keys[b];
  if (n_keys > a.max_n_keys || nq > a.max_q) {  // refused: NaN rows
    for (uint32_t r = i; r < nq; r += a.max_q)
      for (int e = lane; e < D; e += 64)
        a.o[((size_t)(q0 + r) * a.n_heads + head) * D + e] = __builtin_nanf("");
    return;
  }
  if (i >= nq) return;
  const int64_t pos = (int64_t)n_keys - nq + i;
  const uint32_t kvh = head / (a.n_heads / a.s.n_kv_heads);
  const size_t row = ((size_t)(q0 + i) * a.n_heads + head) * D;
  for (int e = lane; e < D; e += 64) s_q[e] = a.q[row + e];
  __syncthreads();
  const Kv4Tiles tiles = kv4_tiles(pos, pos, a.window, a.n_sinks);
  float m = -INFINITY, l = 0.f, acc[D / 64] = {};
  for (uint32_t n = 0; n < tiles.count(); n += 2) {
    const uint32_t ti = n + (lane >> 5);
    const int t = lane & 31;
    float s = -INFINITY;
    if (ti < tiles.count()) {
      const uint32_t key = tiles.tile(ti) * kKv4Tile + t;
      if (kv4_sees(pos, key, a.window, a.n_sinks)) {
        const uint32_t page_id = a.table[(size_t)b * a.max_blocks + key / a.s.page];
        if (page_id < a.s.n_pages) {
          const uint8_t* tile = a.pool + kv4_tile_at(page_id, kvh, key % a.s.page, a.s.n_kv_heads,
                                                     a.s.page, Kv4<D>::kTileBytes);
          s = 0.f;
          for (int o = 0; o < D / 8; o++) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + Kv4<D>::k_dword(t, o));
            const float d = (float)*reinterpret_cast<const _Float16*>(
                tile + Kv4<D>::k_scale(t, o >> 2));
            for (int u = 0; u < 8; u++)
              s = fmaf(s_q[8 * o + u],
                       (float)((int)(w >> (4 * ((u >> 1) + 4 * (u & 1))) & 15) - 8) * d, s);
          }
          s *= scale;
        } else {
          s = __builtin_nanf("");
        }
      }
    }
    float top = s;
    for (int x = 32; x; x >>= 1) top = fmaxf(top, shfl_xor(top, x));
    const float nm = fmaxf(m, top), ref = nm == -INFINITY ? 0.f : nm;
    const float p = __expf(s - ref), alpha = __expf(m - ref);
    m = nm;
    l = l * alpha + p;
    __syncthreads();
    s_p[lane] = p;
    __syncthreads();
    for (int c = 0; c < D / 64; c++) acc[c] *= alpha;
    for (int j = 0; j < 64; j++) {
      if (s_p[j] == 0.f || n + (j >> 5) >= tiles.count()) continue;
      const uint32_t key = tiles.tile(n + (j >> 5)) * kKv4Tile + (j & 31);
      const uint32_t page_id = a.table[(size_t)b * a.max_blocks + key / a.s.page];
      if (page_id >= a.s.n_pages) {
        for (int c = 0; c < D / 64; c++) acc[c] = __builtin_nanf("");
        continue;
      }
      const uint8_t* tile = a.pool + kv4_tile_at(page_id, kvh, key % a.s.page, a.s.n_kv_heads,
                                                 a.s.page, Kv4<D>::kTileBytes);
      for (int c = 0; c < D / 64; c++) {
        const int e = 64 * c + lane;
        const uint32_t w =
            *reinterpret_cast<const uint16_t*>(tile + Kv4<D>::v_word(j & 31, e >> 2));
        const float d =
            (float)*reinterpret_cast<const _Float16*>(tile + Kv4<D>::v_scale(j & 31, e >> 5));
        acc[c] = fmaf(s_p[j], (float)((int)(w >> (4 * (e & 3)) & 15) - 8) * d, acc[c]);
      }
    }
  }
  l = lane_tree<64>(l);
  for (int c = 0; c < D / 64; c++) a.o[row + 64 * c + lane] = l == 0.f ? 0.f : acc[c] / l;
}

// Up to 16 query-head rows a kv head take the decode kernel.
static bool few_rows(uint32_t max_q, uint32_t n_heads, uint32_t n_kv_heads) {
  return (uint64_t)max_q * (n_heads / n_kv_heads) <= 16;
}

uint64_t kv4_attn_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys, uint32_t n_heads,
                           uint32_t n_kv_heads, uint32_t head_dim, uint32_t window,
                           uint32_t n_sinks) {
  if (few_rows(max_q, n_heads, n_kv_heads))
    return kv4_decode_plan(n_seqs, max_q, max_n_keys, n_heads, n_kv_heads, head_dim, window,
                           n_sinks).ws_bytes;
  return 0;
}

hipError_t launch_kv4_attn(const Kv4AttnArgs& a, void* ws, hipStream_t st) {
  if (few_rows(a.max_q, a.n_heads, a.s.n_kv_heads))
    return launch_kv4_decode(a, kv4_decode_plan(a.n_seqs, a.max_q, a.max_n_keys, a.n_heads,
                                                a.s.n_kv_heads, a.s.head_dim, a.window, a.n_sinks),
                             ws, st);
  const float scale = (float)(1.0 / sqrt((double)a.s.head_dim));
  const dim3 grid(a.n_heads, a.max_q, a.n_seqs);
  if (a.s.head_dim == 128)
    hipLaunchKernelGGL(kv4_attn_kernel<128>, grid, dim3(64), 0, st, a, scale);
  else
    hipLaunchKernelGGL(kv4_attn_kernel<64>, grid, dim3(64), 0, st, a, scale);
  return hipGetLastError();
}

}  // namespace flk
