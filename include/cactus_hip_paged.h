/* A paged INT8 key/value cache and the attention that reads it, for independent sequences of different lengths.
 *
 * The caches of cactus_hip.h give every sequence one contiguous run of slots and every (token, kv head, 128 dims) its own
 * scale, as the reference's KVCache does (engine_cache.cpp:11-51, kernel.h:18).  Here the tokens of a sequence live in
 * pages of a pool that all sequences share (no counterpart in the reference, whose engine holds one sequence), and a page
 * holds ONE scale per kv head for its keys and one for its values:
 *
 *   k, v            int8  [num_pages][kv_heads][page_size][head_dim]      (page, head): one contiguous run
 *   k_scales, ...   float [num_pages][kv_heads]                           value = int8 * scale; a scale that
 *                                                         is not positive and finite counts as zero
 *   block_tables    int32 [batch][table_width]    page of tokens page_size * i .. of sequence b in entry [b][i]
 *
 * page_size is 16, 32, 64 or 128 and head_dim 64, 128 or 256; all buffers are 16-byte aligned device memory.  The pages a
 * call appends to belong to one sequence each (pages that are only read may be shared).  An entry of block_tables outside
 * [0, num_pages) names no page: nothing is stored there and its tokens are not seen.  Entries past a sequence's last
 * page are not looked at.
 *
 * Rows (q, k, v, outputs) are packed one sequence behind the other: sequence b owns rows cu_seqlens[b] ..
 * cu_seqlens[b + 1] - 1 of `tokens` (device int32 [batch + 1], not decreasing, starting at 0).  cu_seqlens == NULL: one row
 * per sequence (tokens == batch, a decode step).  Rows behind cu_seqlens[batch] are left as they are.  An input row is
 * half [heads][head_dim]; consecutive rows lie `stride` elements apart (a multiple of 8, at least heads * head_dim, below 2^24: q, k
 * and v may be columns of one fused projection); output rows are contiguous, and an output may be q itself where q's rows are too.
 *
 * Visibility, in every attention here: position p sees the keys j <= p of its sequence with
 *     window == 0   or   p - j <= window   or   j < sink
 * which is the sliding window of cactus_hip_attention_f16_dev (kernel_attention.cpp:81-87) plus `sink` leading tokens.  The
 * reference's KVCache window of W slots with S sink tokens (engine_cache.cpp:268-329) is window = W - S, sink = S.  A row
 * that sees nothing becomes zeros.  scale == 0 means 1 / sqrt(head_dim); otherwise it is at most 1e15, of either sign.
 *
 * Calls enqueue on `stream`, allocate nothing, synchronize nothing and may be captured.  They use no library workspace:
 * scratch comes in as `workspace`, so calls on different streams do not meet.  Returns as in cactus_hip.h. */
#ifndef CACTUS_HIP_PAGED_H
#define CACTUS_HIP_PAGED_H

#include "cactus_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cactus_hip_paged_kv {
    int8_t *k, *v;
    float *k_scales, *v_scales;
    size_t num_pages, page_size, kv_heads, head_dim;
} cactus_hip_paged_kv;

/* The rows of one step or prompt chunk into the cache, with everything that happens to them on the way:
 *   k' = rope(rms_norm(k, k_weight)),  q_output = half(rope(rms_norm(q, q_weight)))      in fp32, angles in fp64
 * (k_weight / q_weight half[head_dim], NULL: no norm; q NULL: no queries; the half-split rotation of cactus_rope_f16,
 * kernel_attention.cpp:614-676; theta 0: no rotation), token i of sequence b at position positions[b] + i, where
 * positions[b] (device int32) is the number of tokens it has in the cache; a sequence with a negative position is skipped.
 * The page scale of k' (and of v) is max(|x|)/127, at least 1e-10, over all tokens of the page: a token that does
 * not fit the scale an already started page has raises it, and the page's earlier tokens are requantized
 * (round(q * old / new)).  A page whose first slot this call writes starts afresh, so a page needs no clearing between
 * owners.  Rounding is to nearest even; NaN is stored as 0 and an infinity as +-65504.
 * Requantizing rounds once more: a stored value is off by at most half of every scale its page has had since it was written.
 * Random rows raise a page's scale a few times (relative RMS error in pages of 64, D = 128: 0.9% written in one call, 1.2% a token at a
 * time; 1.6% and 2.0% if the tokens' norms are spread by half), but rows that grow a little with every token raise it every
 * time (0.4% a token: 2.6% in pages of 16, 10% of 64, 21% of 128, against 0.7% in one call).  Smaller pages keep that down;
 * prompts go in whole or in long chunks. */
int cactus_hip_kv_append_paged_f16_dev(const cactus_hip_paged_kv* cache, const int32_t* block_tables, size_t table_width,
                                       const int32_t* positions, const int32_t* cu_seqlens, size_t batch, size_t tokens,
                                       const cactus_half_t* k, size_t k_stride, const cactus_half_t* v, size_t v_stride,
                                       const cactus_half_t* q, size_t q_stride, cactus_half_t* q_output,
                                       size_t num_q_heads, const cactus_half_t* q_weight, const cactus_half_t* k_weight,
                                       float eps, float theta, void* stream);

/* Tokens of the cache as halves, half(int8 * scale): row r of sequence b (cu_seqlens over `rows`, required) is token
 * starts[b] + r.  k_output, v_output half[rows][kv_heads][head_dim]; a token without a page becomes zeros. */
int cactus_hip_kv_read_paged_f16_dev(const cactus_hip_paged_kv* cache, const int32_t* block_tables, size_t table_width,
                                     const int32_t* starts, const int32_t* cu_seqlens, size_t batch, size_t rows,
                                     cactus_half_t* k_output, cactus_half_t* v_output, void* stream);

/* Attention of query rows over the paged cache.  context_lens[b] (device int32): tokens sequence b has in the cache, the
 * rows of this call included (append first); its query row i of n stands at position context_lens[b] - n + i.
 * max_context: an upper bound of context_lens that the caller knows on the host (it decides how a long context is split
 * over workgroups, never which keys are seen; table_width * page_size will do).  num_q_heads is a multiple of the cache's
 * kv_heads.  workspace: device memory of at least cactus_hip_attention_paged_workspace_bytes(same arguments) bytes,
 * 16-byte aligned, contents free (0 bytes: may be NULL); it must not be shared by calls that may overlap. */
size_t cactus_hip_attention_paged_workspace_bytes(const cactus_hip_paged_kv* cache, size_t batch, size_t tokens,
                                                  size_t max_context, size_t num_q_heads, size_t window, size_t sink,
                                                  int one_row_each);
int cactus_hip_attention_paged_f16_dev(const cactus_hip_paged_kv* cache, const int32_t* block_tables, size_t table_width,
                                       const int32_t* context_lens, const int32_t* cu_seqlens, size_t batch, size_t tokens,
                                       size_t max_context, const cactus_half_t* q, size_t q_stride, cactus_half_t* output,
                                       size_t num_q_heads, float scale, size_t window, size_t sink, void* workspace,
                                       size_t workspace_bytes, void* stream);

/* FP16 attention of whole prompts, causal, packed by cu_seqlens (required); row i of a sequence stands at position i.  A
 * key or value row that a query does not see has no influence on it whatever it holds (infinities and NaN included).  A
 * value that it sees and that is not finite is in its output whatever it weighs: an infinity as that infinity, two of different
 * sign and a NaN as NaN. */
int cactus_hip_attention_ragged_f16_dev(const cactus_half_t* q, size_t q_stride, const cactus_half_t* k, size_t k_stride,
                                        const cactus_half_t* v, size_t v_stride, cactus_half_t* output,
                                        const int32_t* cu_seqlens, size_t batch, size_t tokens, size_t num_q_heads,
                                        size_t num_kv_heads, size_t head_dim, float scale, size_t window, size_t sink,
                                        void* stream);

#ifdef __cplusplus
}
#endif
#endif
