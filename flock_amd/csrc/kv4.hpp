// The paged cache in 4 bits: layout of a tile, scales and codes, launches.
//
// A pool is n_pages pages of `page` tokens (32, 64, 128 or 256); a page holds,
// for each kv head, page / 32 tiles of 32 tokens, 36 D bytes each. A tile lies
// as the matrix cores want it, so that attention loads whole 16-byte pieces and
// moves nothing between lanes (K is operand A of S^T = K Q^T, V^T that of
// O^T = V^T P^T, both 16x16x32):
//   K codes  16 D B  lane (key 16, part 4) of a half tile of 16 tokens: dims
//                    part D/4 .. of token 16 half + key, D/8 bytes. D = 128:
//                    [half][key][part], D = 64: [key][part][half]. In each dword
//                    dim t of its 8 is nibble (t >> 1) + 4 (t & 1): a mask of
//                    0x000f000f then takes two neighbouring dims.
//   K scales  2 D B  [key][block D/32][half] f16
//   V codes  16 D B  [chunk D/64][g 4][n 16][slot 8] 16-bit words: nibble j is dim
//                    D/16 n + 4 chunk + j of token 4 g + slot (slot < 4) or
//                    16 + 4 g + slot - 4: the tokens whose scores lane group g
//                    holds after S^T. Tokens share no byte.
//   V scales  2 D B  [g][block D/32][slot] f16
#pragma once

#include "common.hpp"

namespace flk {

constexpr uint32_t kKv4Tile = 32;  // tokens of a tile
constexpr uint32_t kNoPage = 0xffffffffu;
constexpr uint64_t kMaxGroups = 0xffffff;  // workgroups of 256 threads: a grid has 2^32 at most

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4v __attribute__((ext_vector_type(4)));

template <int D>
struct Kv4 {
  static constexpr int kTileBytes = 36 * D;
  static constexpr int kKScale = 16 * D;
  static constexpr int kV = 18 * D;
  static constexpr int kVScale = 34 * D;
  static constexpr int kBlocks = D / 32;
  // Byte of the dword of K's dims 8 o .. 8 o + 7 of token t, of the scale of
  // block b; of V's word of dims 4 w .. 4 w + 3, and its scale.
  __host__ __device__ static constexpr int k_dword(int t, int o) {
    const int half = t >> 4, key = t & 15;
    return D == 128 ? half * 1024 + key * 64 + o * 4
                    : key * 64 + (o >> 1) * 16 + half * 8 + (o & 1) * 4;
  }
  __host__ __device__ static constexpr int k_scale(int t, int b) {
    return kKScale + 2 * (((t & 15) * kBlocks + b) * 2 + (t >> 4));
  }
  __host__ __device__ static constexpr int v_word(int t, int w) {
    const int g = (t >> 2) & 3, slot = (t & 3) + 4 * (t >> 4);
    const int n = D == 128 ? w >> 1 : w, c = D == 128 ? w & 1 : 0;
    return kV + 2 * (((c * 4 + g) * 16 + n) * 8 + slot);
  }
  __host__ __device__ static constexpr int v_scale(int t, int b) {
    const int g = (t >> 2) & 3, slot = (t & 3) + 4 * (t >> 4);
    return kVScale + 2 * ((g * kBlocks + b) * 8 + slot);
  }
};

// Byte of the tile that holds token `slot % page` of kv head `head`'s page.
__device__ __forceinline__ size_t kv4_tile_at(uint32_t page_id, uint32_t head, uint32_t in_page,
                                              uint32_t n_kv_heads, uint32_t page,
                                              uint32_t tile_bytes) {
  return (((size_t)page_id * n_kv_heads + head) * (page / kKv4Tile) + in_page / kKv4Tile) *
         tile_bytes;
}

// The keys that queries at positions first .. last (signed: a sequence may hold
// fewer keys than it has queries) see, as tiles: `sinks` tiles from the first
// token, then the tiles from `from` up to `to`.
struct Kv4Tiles {
  uint32_t sinks, from, to;
  __device__ __forceinline__ uint32_t count() const { return sinks + to - from; }
  __device__ __forceinline__ uint32_t tile(uint32_t i) const {
    return i < sinks ? i : from + (i - sinks);
  }
};
__device__ __forceinline__ Kv4Tiles kv4_tiles(int64_t first, int64_t last, uint32_t window,
                                              uint32_t n_sinks) {
  if (last < 0) return {0, 0, 0};
  const uint32_t to = (uint32_t)(last / kKv4Tile) + 1;
  const int64_t lo = first - (int64_t)window + 1;
  if (window == 0 || lo <= 0) return {0, 0, to};
  const uint32_t from = min((uint32_t)(lo / kKv4Tile), to);
  const uint64_t s = ((uint64_t)n_sinks + kKv4Tile - 1) / kKv4Tile;
  return {(uint32_t)(s < from ? s : from), from, to};
}

struct Kv4Shape {
  uint32_t n_kv_heads, head_dim, n_pages, page;
};

struct Kv4PlanArgs {
  const uint32_t *n_keys, *n_new, *table_in, *free_in;
  uint32_t *table_out, *free_out, *q_off, *positions, *slots, *lost;
  uint32_t n_seqs, max_blocks, n_pages, max_tokens, page, window, n_sinks;
};
uint64_t kv4_plan_ws_bytes(uint32_t n_seqs);
hipError_t launch_kv4_plan(const Kv4PlanArgs& a, void* ws, hipStream_t st);

struct Kv4AppendArgs {
  const float *q, *k, *v;           // raw rows; q null: k and v are stored as they are
  uint32_t q_stride, kv_stride;     // floats from one token to the next
  const float *gq, *gk, *inv_freq;
  float eps;
  int32_t pairing;
  const uint32_t *positions, *slots;
  float* qn_out;
  uint8_t* pool;
  uint32_t n_tokens, n_heads;
  Kv4Shape s;
};
hipError_t launch_kv4_append(const Kv4AppendArgs& a, hipStream_t st);
hipError_t launch_kv4_read(const uint8_t* pool, const uint32_t* slots, float* k, float* v,
                           uint32_t n_tokens, const Kv4Shape& s, hipStream_t st);

struct Kv4AttnArgs {
  const float* q;
  const uint8_t* pool;
  const uint32_t *table, *n_keys, *q_off;
  float* o;
  uint32_t n_seqs, n_tokens, max_q, max_n_keys, max_blocks, n_heads, window, n_sinks;
  uint32_t q_from, q_to;  // sequences of so many rows are this launch's
  Kv4Shape s;
};
uint64_t kv4_attn_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys, uint32_t n_heads,
                           uint32_t n_kv_heads, uint32_t head_dim, uint32_t window,
                           uint32_t n_sinks);
bool kv4_attn_fits(const Kv4AttnArgs& a);
hipError_t launch_kv4_attn(const Kv4AttnArgs& a, void* ws, hipStream_t st);

}  // namespace flk
