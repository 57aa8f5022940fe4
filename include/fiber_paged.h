/* fiber_paged.h — operators over the paged KV cache for ragged batches of sequences
 * (extern "C", libfiber_cuda.so; conventions and status codes of fiber_cuda.h).
 *
 * fiber_kv_append rotates the new tokens' queries and keys and stores keys and values
 * in the cache; fiber_attn_paged lets every new token attend to its sequence's pages,
 * for chunks of any length and for single tokens. The reference decodes one sequence
 * token by token (src/gpu_ffn.m:488-617), so neither has a counterpart there.
 *
 * Both take the lengths from device memory, so one captured graph serves growing
 * sequences. All calls are enqueued on `stream`; nothing is allocated or synchronized.
 */
#ifndef FIBER_PAGED_H
#define FIBER_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "kv_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (GGUF's numbering). */
#define FIBER_TYPE_F32 0
#define FIBER_TYPE_F16 1
#define FIBER_TYPE_BF16 30

/* One layer of a paged cache: position i of slot s and KV head g starts at element
 *     table[s][i / page_size] * page_stride + g * head_stride + (i % page_size) * pos_stride
 * of the pools (strides in elements, multiples of 8; pools 16-byte aligned). Table
 * entries are read only for pages that hold positions below a sequence's kv_len;
 * an entry outside [0, n_pages) reads as zeros and is not written. */
typedef struct {
    int type;      /* FIBER_TYPE_F16 or FIBER_TYPE_BF16 */
    int head_dim;  /* 64 or 128 */
    int n_kv_heads;
    int page_size; /* 16, 32, 64, 128 or 256 positions */
    int n_pages;   /* pages in each pool */
    int n_slots, max_pages; /* page_table is [n_slots][max_pages]; max_pages * page_size <= 2^31 - 256 */
    int64_t page_stride, head_stride, pos_stride;
    void *k_pool, *v_pool;     /* device */
    const int32_t *page_table; /* device */
} fiber_kv_view_t;

/* The view of layer `layer` of a kv_cache_t (kv_cache.h). */
int fiber_kv_view(const kv_cache_t *kv, int layer, fiber_kv_view_t *out);

/* A ragged batch: sequence s brings tokens q_start[s] .. q_start[s + 1] - 1 (q_start does
 * not decrease, q_start[n_seqs] <= n_tokens) and, with them, has kv_len[s] positions in
 * cache slot slot[s] (slot null: slot s); its token i sits at position
 * kv_len[s] - (q_start[s + 1] - q_start[s]) + i. Tokens at negative positions are not
 * in the cache: they are not stored and attend to nothing (zero output); so do all
 * tokens of a sequence whose slot or kv_len lies outside the table. Rows before q_start[0]
 * and from q_start[n_seqs] on belong to no sequence: neither operator writes them. */
typedef struct {
    int n_seqs, n_tokens; /* n_tokens: rows of the token buffers */
    int max_q;            /* tokens of the longest sequence; picks the kernel, the result does not depend on it */
    const int32_t *q_start; /* device, [n_seqs + 1] */
    const int32_t *kv_len;  /* device, [n_seqs] */
    const int32_t *slot;    /* device, [n_seqs], or null */
} fiber_ragged_t;

/* Rotary positions: (cos, sin) pairs, fp32 [max_pos][dim / 2][2] on the device, applied
 * to the first `dim` values of a head (a multiple of 16): pairs (j, j + dim / 2), or
 * (2 j, 2 j + 1) when `adjacent` is set. Tokens at positions >= max_pos are treated like
 * those at negative positions. */
typedef struct {
    const float *table;
    int max_pos, dim, adjacent;
} fiber_rope_t;

/* Rotate and append. d_q / d_k / d_v: the new tokens' rows (in_type: F32, or the cache's
 * type), heads contiguous, token rows ldq / ldk / ldv elements apart, so the parts of one
 * fused q|k|v row can be passed. Keys are rotated and rounded once into k_pool, values
 * rounded into v_pool, queries rotated into d_q_out (rows of ldo elements, the cache's
 * type; may be d_q when types and row strides agree, and overlaps no other input). d_q and
 * d_q_out null: keys and values only. rope null: no rotation. Rows of all buffers are 16-byte
 * aligned. */
int fiber_kv_append(const fiber_kv_view_t *kv, const fiber_ragged_t *batch, int in_type, const void *d_q,
                    int64_t ldq, const void *d_k, int64_t ldk, const void *d_v, int64_t ldv, int n_heads,
                    const fiber_rope_t *rope, void *d_q_out, int64_t ldo, void *stream);

/* Bytes of workspace fiber_attn_paged needs for this view, batch shape (n_seqs, n_tokens,
 * max_q) and number of query heads on the current device; 0 on bad arguments. */
size_t fiber_attn_paged_workspace(const fiber_kv_view_t *kv, const fiber_ragged_t *batch, int n_heads);

/* Causal softmax attention of the batch's tokens over the cache, which holds their own
 * keys and values already: query head h of a token at position p attends to positions
 * max(0, p - window + 1) .. p (window 0: 0 .. p) of KV head h / (n_heads / n_kv_heads),
 *     out = sum_j softmax_j(scale * q . k_j) v_j,
 * scores, softmax and sums in fp32, probabilities and the output rounded to the cache's
 * type. d_q and d_out: rows of n_heads * head_dim values, ldq / ldo elements apart (16-byte
 * aligned, the cache's type), that do not overlap. Cache positions that a token does not see do not reach its
 * output, whatever bits they hold.
 *   At most 128 query heads per KV head. A launch counts its work in 32 bits, so a batch is refused
 * (FIBER_EARG; fiber_attn_paged_workspace returns 0) from about
 *     (n_tokens * n_heads / 256 + n_seqs * n_kv_heads) * max_pages * page_size = 1.4e11
 * on (half of that for groups of 65 to 127 heads), or, where max_q tokens are at most 16 rows per KV
 * head, (n_tokens * n_heads / 16 + n_seqs * n_kv_heads) * max_pages * page_size = 2.7e11.
 *   d_ws: workspace, zero-filled before its first use and then reused by any calls of one stream
 * (calls that may overlap need one each). The same call on the same data gives the same bits. */
int fiber_attn_paged(const fiber_kv_view_t *kv, const fiber_ragged_t *batch, const void *d_q, int64_t ldq,
                     void *d_out, int64_t ldo, int n_heads, float scale, int window, void *d_ws, size_t ws_bytes,
                     void *stream);

/* Waits for `stream` and reports whether a bounded wait inside a fiber_attn_paged call on this
 * workspace gave up (FIBER_ETIMEOUT), or a call found a decreasing q_start and wrote nothing for its
 * sequences (FIBER_EARG). Zero-fill the workspace before using it again. */
int fiber_attn_paged_status(const void *d_ws, void *stream);

/* Drill, for a program to try out how it takes a call whose waits give up: while `on`, the kernels of
 * the whole process's later calls never reuse a stage of their shared-memory rings, and wait 1e6
 * cycles (about 0.5 ms) instead of 4e9 (about 2 s). A call long enough to need a stage again (about
 * 1,000 positions per SM) ends with FIBER_ETIMEOUT as its status. */
int fiber_attn_paged_drill(int on);

#ifdef __cplusplus
}
#endif
#endif
