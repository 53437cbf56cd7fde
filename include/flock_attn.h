/*
 * flock_attn.h -- C ABI of libflock_attn.so, the MI355X (gfx950) attention hot
 * path of flock: per-head q/k RMSNorm + RoPE + K/V-cache append, GQA decode
 * attention, causal prefill attention.
 *
 * In the reference every op below is a WGSL compute dispatch whose "ABI" is a
 * binding list plus a uniform struct, encoded by kernels/layer.ts. Each entry
 * point here replaces one such dispatch (cited per function) with the same
 * buffer layouts and the same position semantics:
 *
 *   q, qn, o (decode)     [n_heads][head_dim]                f32
 *   q, qn, o (prefill)    [n_tokens][n_heads][head_dim]      f32
 *   k, v (new rows)       [n_tokens][n_kv_heads][head_dim]   f32
 *   kcache, vcache        [max_keys][n_kv_heads][head_dim]   f32, row = position
 *   GQA map               query head h reads kv head h / (n_heads / n_kv_heads)
 *
 * Conventions (all entry points):
 *   - Pointers named q/k/v/o/kcache/... are DEVICE pointers (flk_alloc, or any
 *     HIP/torch allocation on the current device). Host pointers appear only in
 *     flk_h2d / flk_d2h.
 *   - Every function returns int32 status: FLK_OK (0) or a negative FLK_ERR_*.
 *     Argument checks run on the host BEFORE any launch, so a rejected call
 *     has no side effect (the reference throws from Layer before encoding:
 *     kernels/layer.ts:575, 689-698; lib.ts:504-506). flk_last_error() gives a
 *     message for the calling thread's most recent failure. Nothing throws.
 *   - Launches are asynchronous and ordered on the library's current stream
 *     (flk_set_stream; default: the null stream). flk_sync() waits for it.
 *     The current stream, like the flk_last_error text, belongs to the
 *     calling host thread.
 *   - Split-K kernels need scratch for per-split partial results. The caller
 *     passes it as (ws, ws_bytes), sized with flk_workspace_bytes; it needs no
 *     initialisation and holds nothing between calls. Calls that share one
 *     workspace must be ordered on one stream (concurrent calls race). A call
 *     whose plan has a single split needs none (ws may then be NULL).
 *   - head_dim must be 64 or 128; n_heads must be a multiple of n_kv_heads
 *     with n_heads / n_kv_heads <= 8.
 *   - The attention kernels move 16-byte vectors: q, qn, o, kcache, vcache and
 *     (flk_decode_layer) q_raw, k_raw, v_raw must be 16-byte aligned; a
 *     misaligned pointer is rejected with FLK_ERR_ARG before any launch.
 */
#ifndef FLOCK_ATTN_H
#define FLOCK_ATTN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  FLK_OK = 0,
  FLK_ERR_ARG = -1,          /* bad shape, null pointer, n < 1, ...           */
  FLK_ERR_CACHE_FULL = -2,   /* pos + n_tokens > max_keys (layer.ts:575, 693) */
  FLK_ERR_UNSUPPORTED = -3,  /* head_dim / GQA group outside supported set    */
  FLK_ERR_WORKSPACE = -4,    /* ws null or smaller than flk_workspace_bytes   */
  FLK_ERR_HIP = -5,          /* HIP runtime error (message in flk_last_error) */
};

/* RoPE pairing (lib.ts:517-531): NEOX pairs (j, j + d/2), NORM pairs (2j, 2j+1). */
enum { FLK_ROPE_NEOX = 0, FLK_ROPE_NORM = 1 };

/* ---------------------------------------------------------------- runtime -- */

/* Message for the calling thread's last non-zero status ("" if none). */
const char* flk_last_error(void);
/* Library version string. */
const char* flk_version(void);
/* Number of visible devices (0 when no GPU); never fails. */
int32_t flk_device_count(int32_t* count);
/* Stream for all later launches from the calling thread (hipStream_t; NULL =
 * default; each host thread starts on NULL). Replaces the caller-supplied
 * GPUCommandEncoder of Layer.encode (layer.ts:586-589). */
int32_t flk_set_stream(void* stream);

/* Device memory (storageBuffer / createBuffer, lib.ts:548-566; readBack,
 * lib.ts:575-593). flk_h2d/flk_d2h are synchronous with respect to the host.
 * flk_free waits for the calling thread's library stream -- for the whole
 * device when that thread has switched away from a non-null stream since its
 * last such wait -- then releases the memory with hipFree: call it outside
 * loops that must not stall. While the library stream is capturing a graph it returns
 * FLK_ERR_ARG and frees nothing (free after flk_capture_end). */
int32_t flk_alloc(void** dptr, uint64_t bytes);
int32_t flk_free(void* dptr);
int32_t flk_h2d(void* dst, const void* host_src, uint64_t bytes, uint64_t dst_off);
int32_t flk_d2h(void* host_dst, const void* src, uint64_t bytes, uint64_t src_off);
int32_t flk_memset(void* dst, int32_t value, uint64_t bytes);
/* Wait for all work on the current stream (the mapAsync fence, layer.ts:801-816). */
int32_t flk_sync(void);

/* Workspace for the split-K kernels: bytes needed by any call with at most
 * these sizes (max_seqs: sequences of flk_attn_decode_ragged, else 1). */
uint64_t flk_workspace_bytes(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                             uint32_t max_keys, uint32_t max_queries, uint32_t max_seqs);
/* Bytes one call needs. kind: FLK_CALL_DECODE (flk_attn_decode /
 * flk_decode_layer; n = n_keys), FLK_CALL_PREFILL (n = n_queries, pos0),
 * FLK_CALL_RAGGED (n = max_n_keys, n_seqs). 0 when the call needs no workspace
 * (a single-split plan) or the shape is invalid. flk_attn_prefill also accepts
 * less (down to none) where that holds the partials of its f32 kernel: the call
 * then takes that kernel, which is slower and rounds its sums in another order.
 * So its speed and its last bits depend on which of the two fits. */
enum { FLK_CALL_DECODE = 0, FLK_CALL_PREFILL = 1, FLK_CALL_RAGGED = 2 };
uint64_t flk_call_workspace_bytes(int32_t kind, uint32_t n_heads, uint32_t n_kv_heads,
                                  uint32_t head_dim, uint32_t n, uint32_t pos0, uint32_t n_seqs);

/* -------------------------------------------------------------- unfused ops -- */

/* rmsnorm.wgsl main (rmsnorm.wgsl:41-73; dispatch layer.ts:601-602, 725-726).
 * o[v][i] = x[v][i] / sqrt(mean(x[v]^2) + eps) * g[i] over n_vecs vectors of
 * width n, with the reference's 128-lane strided partial sums and pairwise tree.
 * Bit-exact with rmsnormRef (ops_ref.ts:20-49). Any n >= 1. */
int32_t flk_rmsnorm(const float* x, const float* g, float* o, uint32_t n, uint32_t n_vecs,
                    float eps);

/* rope.wgsl main (rope.wgsl:50-78 with ropeSource, lib.ts:528-531; dispatch
 * layer.ts:607-613). In place on x [n_tokens][n_heads][head_dim]; token t is
 * rotated by position pos0 + t using inv_freq [head_dim/2] (layer.ts:180-186).
 * Bit-exact with ropeRef (ops_ref.ts:65-92) up to libm's cos/sin last bit. */
int32_t flk_rope(float* x, const float* inv_freq, uint32_t n_tokens, uint32_t n_heads,
                 uint32_t head_dim, uint32_t pos0, int32_t pairing);

/* The two copyBufferToBuffer calls of the K/V append (layer.ts:616-622,
 * 737-741): kcache[pos0 .. pos0+n) <- kn, vcache[pos0 .. pos0+n) <- v. */
int32_t flk_kv_append(const float* kn, const float* v, float* kcache, float* vcache,
                      uint32_t n_tokens, uint32_t pos0, uint32_t n_kv_heads,
                      uint32_t head_dim, uint32_t max_keys);

/* ------------------------------------------------------------ fused prologue -- */

/* layer.ts:598-622 (decode) and 722-741 (prefill) in one launch: per-head
 * RMSNorm of q and k with gains gq, gk [head_dim]; RoPE of both at positions
 * pos0 + t; qn_out <- q; kcache/vcache rows pos0 + t <- (k normed+roped, v raw).
 * Bit-identical to flk_rmsnorm + flk_rope + flk_kv_append. */
int32_t flk_qk_prologue(const float* q_raw, const float* k_raw, const float* v_raw,
                        const float* gq, const float* gk, const float* inv_freq, float eps,
                        int32_t pairing, float* qn_out, float* kcache, float* vcache,
                        uint32_t n_tokens, uint32_t pos0, uint32_t n_heads,
                        uint32_t n_kv_heads, uint32_t head_dim, uint32_t max_keys);

/* Extension, no reference counterpart (layer.ts:722-724 projects q, k and v
 * into three buffers): flk_qk_prologue reading raw rows that lie in_stride
 * floats apart from one token to the next -- e.g. q_raw = qkv, k_raw = qkv +
 * n_heads * head_dim, v_raw = k_raw + n_kv_heads * head_dim, in_stride = (n_heads
 * + 2 * n_kv_heads) * head_dim for the output of ONE projection over q|k|v
 * stacked row-wise. in_stride 0 means packed (flk_qk_prologue); otherwise it
 * must be at least n_heads * head_dim. Same results. */
int32_t flk_qk_prologue_strided(const float* q_raw, const float* k_raw, const float* v_raw,
                                uint32_t in_stride, const float* gq, const float* gk,
                                const float* inv_freq, float eps, int32_t pairing,
                                float* qn_out, float* kcache, float* vcache, uint32_t n_tokens,
                                uint32_t pos0, uint32_t n_heads, uint32_t n_kv_heads,
                                uint32_t head_dim, uint32_t max_keys);

/* -------------------------------------------------------------- attention -- */

/* attention.wgsl main (attention.wgsl:58-122; bindings [q, kcache, vcache, o,
 * Dims{n_heads, n_kv_heads, head_dim, n_keys}], dispatch layer.ts:624-630).
 * One query per head attends keys [0, n_keys). No cap on n_keys beyond the
 * cache (the reference's $MAX_KEYS workgroup array, lib.ts:503-508, is gone):
 * split-K flash-decoding -- a split kernel, then a log-sum-exp merge launch
 * ordered after it on the same stream (one launch when the plan has a single
 * split). */
int32_t flk_attn_decode(const float* q, const float* kcache, const float* vcache, float* o,
                        uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                        uint32_t n_keys, void* ws, uint64_t ws_bytes);

/* attention_prefill.wgsl main (attention_prefill.wgsl:75-175; bindings [q,
 * kcache, vcache, o, Dims{n_heads, n_kv_heads, head_dim, n_queries, pos0}],
 * dispatch layer.ts:743-750). Query i (absolute position pos0 + i) attends
 * keys [0, pos0 + i]; the chunk's own rows must already be in the cache.
 * Tiled flash attention on the matrix cores in f32 precision (operands in
 * three bf16 parts; fp32 MFMA for calls of little work), cut over keys where
 * whole q tiles would leave the GPU idle. o may lie over q (the call then
 * takes the fp32 kernel if ws holds its partials). Range: rows whose q or output holds
 * an infinity, a NaN or extreme magnitudes (q from 2^100 or below 2^-110, an
 * output below 2^-108) are formed in plain f32, slowly. A weight below 2^-110
 * of its row's largest is off by up to 2^-134 of that, and a v below 2^-134
 * may count as 0. */
int32_t flk_attn_prefill(const float* q, const float* kcache, const float* vcache, float* o,
                         uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                         uint32_t n_queries, uint32_t pos0, void* ws, uint64_t ws_bytes);

/* Layer.encode's attention slice (layer.ts:571-630) as ONE launch: prologue for
 * the token at position pos (norm + RoPE of q and k, append k/v at row pos),
 * then decode attention over pos + 1 keys. qn_out receives the attention input
 * (layer.ts buf.qn). Cache rows are bit-identical to flk_qk_prologue's. */
int32_t flk_decode_layer(const float* q_raw, const float* k_raw, const float* v_raw,
                         const float* gq, const float* gk, const float* inv_freq, float eps,
                         int32_t pairing, float* qn_out, float* kcache, float* vcache,
                         float* o, uint32_t pos, uint32_t n_heads, uint32_t n_kv_heads,
                         uint32_t head_dim, uint32_t max_keys, void* ws, uint64_t ws_bytes);

/* No counterpart in the reference. For callers that cannot allocate (code
 * under graph capture, serving loops, harnesses that forbid hipMalloc):
 * flk_decode_layer with no workspace argument. The split-K partials go to a
 * static scratch array of 8 MiB that the library holds on each device until
 * the process ends; a call needing more (flk_call_workspace_bytes(
 * FLK_CALL_DECODE, ..., pos + 1, ...) > 8 MiB, i.e. more than ~63 heads of
 * width 128) returns FLK_ERR_WORKSPACE before any launch. Nothing in the
 * array must start at zero: each call's split kernel writes every partial
 * its merge reads. All calls on one device share the array, so calls that
 * overlap on one device (several streams or threads) race: order them on
 * one stream. Same results as flk_decode_layer, bit for bit. */
int32_t flk_decode_layer_noalloc(const float* q_raw, const float* k_raw, const float* v_raw,
                                 const float* gq, const float* gk, const float* inv_freq,
                                 float eps, int32_t pairing, float* qn_out, float* kcache,
                                 float* vcache, float* o, uint32_t pos, uint32_t n_heads,
                                 uint32_t n_kv_heads, uint32_t head_dim, uint32_t max_keys);

/* Extension, no reference counterpart (the reference runs one sequence per
 * Layer, layer.ts:203-204): decode for n_seqs independent sequences in one
 * call. q, o: [n_seqs][n_heads][head_dim]. Sequence b's cache rows start at
 * row seq_row_off[b] of kcache/vcache (rows of n_kv_heads*head_dim floats) and
 * it attends n_keys[b] keys (0: its o rows are zeros). seq_row_off and n_keys
 * are DEVICE arrays (8- and 4-byte aligned), so the library cannot check
 * their contents: rows seq_row_off[b] .. seq_row_off[b] + n_keys[b] - 1 must
 * lie inside kcache and vcache. max_n_keys bounds every n_keys[b] (larger
 * values are clamped to it: such a sequence attends its first max_n_keys
 * rows). Up to 2048 sequences run on persistent workgroups that take
 * the batch's (sequence, split) pieces from a counter kept in the workspace
 * (reset by the call itself); results are the same bits on every call. */
int32_t flk_attn_decode_ragged(const float* q, const float* kcache, const float* vcache,
                               const uint64_t* seq_row_off, const uint32_t* n_keys, float* o,
                               uint32_t n_seqs, uint32_t max_n_keys, uint32_t n_heads,
                               uint32_t n_kv_heads, uint32_t head_dim, void* ws,
                               uint64_t ws_bytes);

/* Extension, no reference counterpart: Layer.encode's attention slice
 * (layer.ts:571-630) for n_seqs independent sequences in one call -- the
 * per-token step of flk_decode_layer applied to every sequence of a batch
 * (the reference runs one sequence per Layer, layer.ts:203-204).
 * q_raw, qn_out, o: [n_seqs][n_heads][head_dim]; k_raw, v_raw:
 * [n_seqs][n_kv_heads][head_dim]. n_keys[b] counts sequence b's keys AFTER
 * this step: its new token sits at position pos_b = n_keys[b] - 1, q and k
 * are normed (gains gq, gk) and rotated at pos_b, k (normed, rotated) and v
 * (raw) are written to cache row seq_row_off[b] + pos_b, and the attention
 * covers the rows seq_row_off[b] .. seq_row_off[b] + pos_b. n_keys[b] == 0
 * marks an idle sequence: its qn and o rows are zeros and nothing is written
 * to the caches. n_keys[b] > max_n_keys (the reference's "KV cache full",
 * layer.ts:575, which the library cannot see on the host: the counts live
 * in device memory) is refused on the device: that sequence's qn and o rows
 * are NaN and nothing is written to the caches. Layouts, alignment,
 * workspace (flk_call_workspace_bytes(FLK_CALL_RAGGED, ...)) and the
 * conditions on seq_row_off are those of flk_attn_decode_ragged. Launches:
 * the prologue (one workgroup per sequence; it also resets the batch's item
 * counters), then flk_attn_decode_ragged's attention and merge. qn and the
 * cache rows are bit-identical to flk_decode_layer's for each sequence. */
int32_t flk_decode_layer_ragged(const float* q_raw, const float* k_raw, const float* v_raw,
                                const float* gq, const float* gk, const float* inv_freq,
                                float eps, int32_t pairing, float* qn_out, float* kcache,
                                float* vcache, const uint64_t* seq_row_off,
                                const uint32_t* n_keys, float* o, uint32_t n_seqs,
                                uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                                uint32_t head_dim, void* ws, uint64_t ws_bytes);

/* ------------------------------------------------------ shared prefixes -- */

/* Extension, no reference counterpart (the reference runs one sequence per
 * Layer, layer.ts:203-204): decode for sequences that share long prefixes --
 * several answers to one prompt, questions about one document -- where the
 * prefix is stored once and read once for all of them.
 *
 *   groups        group g is the sequences seq_off[g] .. seq_off[g + 1] - 1
 *                 ([n_groups + 1], never falling, at most n_seqs). A group may be
 *                 empty; a sequence in none has no prefix.
 *   prefix        group g's is n_prefix[g] rows from row prefix_row[g] of kcache
 *                 and vcache (rows of n_kv_heads * head_dim floats); 0: none
 *   own keys      sequence b's are n_keys[b] rows from row seq_row_off[b], as in
 *                 flk_attn_decode_ragged. They follow the prefix: the newest is at
 *                 position n_prefix[g] + n_keys[b] - 1.
 *
 * All five are DEVICE arrays (prefix_row and seq_row_off 8-byte aligned, the others
 * 4-byte), so that a captured step replays as they change; the rows they name must lie
 * inside kcache and vcache. max_prefix and max_n_keys bound n_prefix and n_keys (their
 * sum is below 2^32, and at least 1) and set the launch shape. What the host cannot
 * see is refused on the device, with NaN rows: a count beyond its bound (the
 * sequence, or the group's), and seq_off that falls or passes n_seqs (every row).
 *
 * q, keys, values and softmax weights enter the matrix products as two f16 parts each,
 * the sums are f32. An element is off by 2^-22 of itself at most, or by the largest of
 * these where that is more:
 *   q        2^-39 of the largest of its row
 *   keys     2^-33 of the largest of the 32 or 64 keys that are read together, and 2^-135
 *   values   the same, and 2^-81 of the largest value before it in the prefix or own keys
 *   weights  2^-19 of the largest weight among the 32 keys around it (or 2^-35 of the sum of
 *            the row's weights, while its result so far is 2^-8 of the largest value or
 *            more), and 2^-85 of that sum
 * So results are as near to exact ones as those of f32 products, also where one key takes
 * nearly all of the weight and has small values. Any finite sizes do, as long as scores
 * are finite: a key whose score overflows to -infinity has no weight, and a row that has no
 * other key, or one whose score overflows to +infinity, is NaN. Where sizes jump by more than
 * 2^3 from some keys to the next a call may take longer. A sequence that sees a NaN or
 * an infinity among its keys or values has NaN in the dims that they reach, and may have
 * it in others of the same head.
 * Results are the same bits on every call. ws: flk_decode_shared_ws_bytes of the same arguments, 256-byte
 * aligned; calls that share one must be ordered on one stream. */
uint64_t flk_decode_shared_ws_bytes(uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                                    uint32_t max_n_keys, uint32_t n_heads, uint32_t n_kv_heads,
                                    uint32_t head_dim);

/* Attention of one query per sequence. q, o: [n_seqs][n_heads][head_dim]. A sequence
 * without any key is zeros. o may be q, but not lie partly over it. */
int32_t flk_attn_decode_shared(const float* q, const float* kcache, const float* vcache,
                               const uint64_t* prefix_row, const uint32_t* n_prefix,
                               const uint32_t* seq_off, const uint64_t* seq_row_off,
                               const uint32_t* n_keys, float* o, uint32_t n_groups,
                               uint32_t n_seqs, uint32_t max_prefix, uint32_t max_n_keys,
                               uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                               void* ws, uint64_t ws_bytes);

/* flk_decode_layer_ragged for such a batch: n_keys[b] counts sequence b's own keys AFTER
 * the step; q and k are normed and rotated at position n_prefix[g] + n_keys[b] - 1, k
 * and v appended at row seq_row_off[b] + n_keys[b] - 1 (no two sequences' the same, and
 * none in a prefix), then the attention above over qn_out. n_keys[b] = 0 is an idle
 * sequence: its qn and o rows are zeros. Nothing is appended for it or for a refused
 * one, whose qn and o rows are NaN. Raw rows lie in_stride floats apart (0: packed), as in
 * flk_qk_prologue_strided. qn_out and o may not overlap. */
int32_t flk_decode_layer_shared(const float* q_raw, const float* k_raw, const float* v_raw,
                                uint32_t in_stride, const float* gq, const float* gk,
                                const float* inv_freq, float eps, int32_t pairing,
                                float* qn_out, float* kcache, float* vcache,
                                const uint64_t* prefix_row, const uint32_t* n_prefix,
                                const uint32_t* seq_off, const uint64_t* seq_row_off,
                                const uint32_t* n_keys, float* o, uint32_t n_groups,
                                uint32_t n_seqs, uint32_t max_prefix, uint32_t max_n_keys,
                                uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                                void* ws, uint64_t ws_bytes);

/* ------------------------------------------------- paged cache in 4 bits -- */

/* Extension, no reference counterpart (the reference keeps one contiguous f32
 * cache per Layer, layer.ts:394-397): a batch's keys and values in 4 bits, in
 * pages that sequences take from a common pool. One step of a layer is
 *
 *   flk_kv4_plan      (once per step, for all layers: tables, positions, slots)
 *   flk_kv4_prologue  (q/k norm + RoPE, k and v into the pool)
 *   flk_kv4_attn      (attention of the step's queries over the pool)
 *
 * all of them from DEVICE arrays of lengths, so that a step can be captured into
 * a graph and replayed.
 *
 *   pool       n_pages * flk_kv4_page_bytes bytes, 16-byte aligned; needs no
 *              initialisation. `page`, the tokens of a page, is 32, 64, 128 or
 *              256; n_pages * page must be below 2^32. Pages hold every kv head.
 *   slot       of a token: page id * page + its place in the page; a value of
 *              n_pages * page or more (0xffffffff) means none
 *   table      [n_seqs][max_blocks] page ids: entry i holds the sequence's
 *              tokens i * page .. i * page + page - 1; n_pages or more
 *              (0xffffffff): no page
 *   n_keys[b]  keys of sequence b AFTER the step (as flk_decode_layer_ragged)
 *   q_off      [n_seqs + 1]: sequence b's new tokens are rows q_off[b] ..
 *              q_off[b + 1] - 1 of q and o, its last ones: the row before
 *              q_off[b + 1] is at position n_keys[b] - 1
 *   window     0: a token sees every key up to its own. w > 0: it sees the last w
 *              keys (its own among them) and the sequence's first n_sinks.
 *
 * Values are kept per 32 neighbouring dims as codes c (0 .. 15) and one scale d:
 * with m the block's value of largest magnitude (the positive one in a tie), d =
 * m / -8 rounded to bf16 and that to f16, c = 8 + x * (1 / d) rounded to the
 * nearest (half to even) and limited to 0 .. 15; the value is (c - 8) * d. Larger
 * magnitudes than 65280 saturate; a block with an infinity or NaN is NaN as a
 * whole. That is 0.5625 bytes a value. */

/* Bytes of a page (0 for an unsupported shape). */
uint64_t flk_kv4_page_bytes(uint32_t n_kv_heads, uint32_t head_dim, uint32_t page);

/* Block tables and slot maps of a step from request lengths. Sequence b has
 * n_keys[b] keys after the step, the last n_new[b] of them new (at most all).
 * It holds block i after the step if i * page < n_keys[b] and, where window > 0,
 * the block has a token that its first new token sees or n_sinks covers. Blocks to
 * hold that table_in has no page for take one if they start with a new token; pages
 * of other blocks go back (all of them for n_keys[b] = 0: a finished sequence; those
 * past the end after tokens were taken back; those that left the window).
 *   A block to hold that starts before the first new token and has no page stays
 * without: its earlier keys were stored nowhere (no page was free in their step, or
 * with a window the sequence was taken back behind the first new token of the step
 * before, to keys whose pages had left it). Rows that see it are NaN, its new tokens
 * have no slot, in every step until one in which all of the block's keys are new.
 * (With window = 1 no row sees an earlier key, so a block behind the sinks takes one.)
 *   Tokens whose rows lie past max_tokens are stored nowhere either: from the first
 * of them on a sequence's blocks keep their pages, but as marked entries, with the
 * same consequences, until a step in which that token and those behind it are new
 * (the same lengths again with more rows, or a step that goes on from it).
 *   free_in, free_out  [1 + n_pages]: a count, then that many free page ids. The
 *     k-th block that takes a page, in order of (sequence, block), takes the k-th
 *     from the end of free_in's list. free_out's list is what is left of it, then
 *     the pages that went back, in the same order: they can be taken in the next
 *     step. The two may not overlap (a caller keeps two and swaps them).
 *   table_out  may be table_in. Entries without a page are 0xffffffff, marked ones
 *     2^31 + (page id * page + place in the page of the first key not stored), the
 *     sum halved from n_pages * page = 2^31 on. Neither is a page to flk_kv4_attn; a
 *     table that the caller writes holds page ids and 0xffffffff.
 *   q_off      [n_seqs + 1] as above
 *   positions, slots  [max_tokens], by row of q: the token's position, and its
 *     slot. Entries behind the last token: position 0, no slot.
 *   lost       [1]: new tokens without a slot: no page was free (a later call with
 *     the same lengths takes what is free then), a block without a page or marked as
 *     above, a position behind the table's last block, or a row past max_tokens; and
 *     one more for each block to hold that lacks keys from before the step. 0 when all
 *     is well: what the step's rows see is stored once its prologue has run.
 * The new tokens of all sequences are below 2^32, n_seqs * max_blocks below 2^31. A
 * page that two rows of table_in hold would go back twice: tables that share pages
 * (flk_kv4_attn reads those too) are the caller's.
 * ws: flk_kv4_plan_ws_bytes, 256-byte aligned. */
uint64_t flk_kv4_plan_ws_bytes(uint32_t n_seqs);
int32_t flk_kv4_plan(const uint32_t* n_keys, const uint32_t* n_new, const uint32_t* table_in,
                     uint32_t* table_out, const uint32_t* free_in, uint32_t* free_out,
                     uint32_t* q_off, uint32_t* positions, uint32_t* slots, uint32_t* lost,
                     uint32_t n_seqs, uint32_t max_blocks, uint32_t n_pages,
                     uint32_t max_tokens, uint32_t page, uint32_t window, uint32_t n_sinks,
                     void* ws, uint64_t ws_bytes);

/* flk_qk_prologue(_strided) onto the pool: q and k of token t normed and rotated
 * at positions[t], q to qn_out, k (in 4 bits, from the same f32 values) and v to
 * slots[t]. A token without a slot is not stored. No slot may come twice.
 * in_stride as in flk_qk_prologue_strided. */
int32_t flk_kv4_prologue(const float* q_raw, const float* k_raw, const float* v_raw,
                         uint32_t in_stride, const float* gq, const float* gk,
                         const float* inv_freq, float eps, int32_t pairing,
                         const uint32_t* positions, const uint32_t* slots, float* qn_out,
                         void* pool, uint32_t n_tokens, uint32_t n_heads, uint32_t n_kv_heads,
                         uint32_t head_dim, uint32_t n_pages, uint32_t page);

/* flk_kv_append onto the pool: rows kn, v [n_tokens][n_kv_heads][head_dim] in 4
 * bits to slots[t]. */
int32_t flk_kv4_append(const float* kn, const float* v, const uint32_t* slots, void* pool,
                       uint32_t n_tokens, uint32_t n_kv_heads, uint32_t head_dim,
                       uint32_t n_pages, uint32_t page);

/* The values at slots[t] as rows k, v [n_tokens][n_kv_heads][head_dim] (16-byte
 * aligned); zeros for a token without a slot. */
int32_t flk_kv4_read(const void* pool, const uint32_t* slots, float* k, float* v,
                     uint32_t n_tokens, uint32_t n_kv_heads, uint32_t head_dim,
                     uint32_t n_pages, uint32_t page);

/* Attention of each sequence's new tokens over its keys in the pool (the rows of
 * this step must be there already). q, o: [n_tokens][n_heads][head_dim] f32; rows
 * that no sequence has are left as they were. max_q bounds every q_off[b + 1] -
 * q_off[b], max_n_keys every n_keys[b] (at most max_blocks * page): they set the
 * launch shape, so near bounds are faster. A sequence beyond either, or with rows
 * behind n_tokens, is refused on the device: its o rows are NaN, as are rows that
 * see a key without a page. A row that sees no key (n_keys[b] below its row count)
 * is zeros. o may be q, but not
 * lie partly over it. Sums are f32, the cache's values enter the matrix
 * products as they are, q and the weights in two f16 parts: off by at most 2^-23 of a q
 * down to 2^-16 of its row's largest and of a weight down to 2^-12 of the largest, by
 * 2^-39 and 2^-35 of the largest below.
 * ws: flk_kv4_attn_ws_bytes of the same arguments, 256-byte aligned; calls that
 * share one must be ordered on one stream. */
uint64_t flk_kv4_attn_ws_bytes(uint32_t n_seqs, uint32_t max_q, uint32_t max_n_keys,
                               uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                               uint32_t window, uint32_t n_sinks);
int32_t flk_kv4_attn(const float* q, const void* pool, const uint32_t* table,
                     const uint32_t* n_keys, const uint32_t* q_off, float* o, uint32_t n_seqs,
                     uint32_t n_tokens, uint32_t max_q, uint32_t max_n_keys,
                     uint32_t max_blocks, uint32_t n_heads, uint32_t n_kv_heads,
                     uint32_t head_dim, uint32_t n_pages, uint32_t page, uint32_t window,
                     uint32_t n_sinks, void* ws, uint64_t ws_bytes);

#ifdef __cplusplus
}
#endif

#endif /* FLOCK_ATTN_H */
