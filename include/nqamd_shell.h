/*
 * nqamd_shell.h — C ABI of the decoder-shell kernels that run around the
 * packed linears in batch-1 autoregressive decode (Qwen3 geometry: RMSNorm,
 * per-head q/k RMSNorm, rotate-half RoPE, grouped-query attention over a KV
 * cache, SiLU-gated MLP, untied bf16 output projection, greedy selection).
 *
 * Conventions are those of nqamd.h: device pointers owned by the caller,
 * `stream` is a hipStream_t passed as void*, nothing allocates, frees or
 * synchronises, the return value is an nq_status.
 *
 * Positions live in device memory (`position`, one int32 = the cache row of
 * the first token of the call) so that a captured decode step can be replayed
 * without rebuilding its kernel arguments; nq_greedy_select advances it.
 *
 * KV cache layout, per layer: [kv_heads][max_positions][head_dim] in
 * cache_dtype (F16/BF16/F32). RoPE tables: [max_positions][head_dim / 2] fp32,
 * cos and sin of position * inv_freq[i].
 */
#ifndef NQAMD_SHELL_H
#define NQAMD_SHELL_H

#include <stddef.h>
#include <stdint.h>

#include "nqamd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* out[t, :] = table[ids[t], :] (* scale[0] when scale is not NULL) as fp32.
 * table dtype F32/F16/BF16, hidden % 8 == 0. An id outside [0, vocab) gives a
 * row of NaN (no out-of-range read). Replaces launch_bfloat16_embedding
 * (src/nanoquant/runtime/cuda_kernels.py:620-681). */
int nq_embedding(const int64_t* ids, int64_t tokens, const void* table, int32_t table_dtype,
                 int64_t vocab, int64_t hidden, const float* scale, float* out, void* stream);

/* nq_embedding that also writes, for each output row, the sums of squares of
 * its 16-column groups: slots [tokens][hidden / 16] fp32, hidden % 16 == 0.
 * These are the row statistics the NQ_INPUT_RMSNORM input of
 * nq_linear_batch_fused reads (norm_slots), so the first layer's projections
 * take the embedding's output with the RMSNorm folded in, as later layers take
 * the residual. No reference counterpart: the reference's embedding
 * (src/nanoquant/runtime/cuda_kernels.py:620-681) is followed by a separate
 * RMSNorm. */
int nq_embedding_slots(const int64_t* ids, int64_t tokens, const void* table, int32_t table_dtype,
                       int64_t vocab, int64_t hidden, const float* scale, float* out, float* slots,
                       void* stream);

/* Residual add and RMSNorm, one row per token:
 *   residual[t, :] += delta[t, :]                      (skipped when delta is NULL)
 *   out[t, :] = weight * (residual[t, :] * rsqrt(mean(residual[t, :]^2) + eps))
 * residual fp32 (updated in place), delta F32/F16/BF16, weight F32/F16/BF16,
 * out F32/F16/BF16, hidden % 8 == 0 and hidden <= 16384. Replaces the residual adds of
 * Qwen3DecoderLayer.forward and Qwen3RMSNorm (the reference runs the
 * Transformers shell around its packed linears,
 * src/nanoquant/runtime/transformers_generation.py:84-114). */
int nq_add_rmsnorm(float* residual, const void* delta, int32_t delta_dtype, const void* weight,
                   int32_t weight_dtype, float eps, int64_t tokens, int64_t hidden, void* out,
                   int32_t out_dtype, void* stream);

/* Per-head RMSNorm of q and k (skipped when the weight is NULL), rotate-half
 * RoPE at positions position[0] + t, and the KV-cache append:
 *   q_out[t, h, :]              = rope(norm(q[t, h, :]))          (fp32)
 *   k_cache[g, position + t, :] = rope(norm(k[t, g, :]))          (cache_dtype)
 *   v_cache[g, position + t, :] = v[t, g, :]
 * head_dim is 64, 128 or 256; rows at or beyond max_positions are not
 * written. Replaces launch_decode_rope and launch_cache_prefix_update
 * (src/nanoquant/runtime/cuda_kernels.py:401-447,546-587,715-815) and the
 * q_norm / k_norm of the Qwen3 attention block. */
int nq_qk_norm_rope_cache(const float* q, const float* k, const float* v, int64_t tokens,
                          int32_t q_heads, int32_t kv_heads, int32_t head_dim, const void* q_norm,
                          const void* k_norm, int32_t norm_dtype, float eps, const float* cos_table,
                          const float* sin_table, const int32_t* position, int64_t max_positions,
                          float* q_out, void* k_cache, void* v_cache, int32_t cache_dtype,
                          void* stream);

/* Workspace bytes of nq_attention for `tokens` queries. */
int64_t nq_attention_workspace_bytes(int64_t tokens, int32_t q_heads, int32_t head_dim,
                                     int64_t max_positions);

/* Causal grouped-query attention: query t (at cache row position[0] + t)
 * attends cache rows [0, position[0] + t] of kv head h / (q_heads / kv_heads):
 *   out[t, h, :] = softmax(scaling * q[t, h, :] · K[g, 0..p, :]) · V[g, 0..p, :]
 * q fp32 [tokens, q_heads, head_dim]; out F32/F16/BF16 [tokens, q_heads *
 * head_dim]. Softmax in fp32, in a fixed order (deterministic): a running
 * softmax over a 16-bit cache from two tokens on (three with heads of 256),
 * otherwise 64-row blocks whose partial results are merged in block order.
 * Queries may have any magnitude; infinities and NaN in the cache do what fp32
 * arithmetic does with them for the tokens that see their row. Replaces
 * launch_decode_attention (src/nanoquant/runtime/cuda_kernels.py:448-544),
 * generalised from its pinned one-kv-head, 64-row geometry. */
int nq_attention(const float* q, const void* k_cache, const void* v_cache, int32_t cache_dtype,
                 int64_t tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                 const int32_t* position, int64_t max_positions, float scaling, void* out,
                 int32_t out_dtype, void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of nq_decode_attention. */
int64_t nq_decode_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                            int32_t cache_dtype, int64_t max_positions);

/* One decode token: nq_qk_norm_rope_cache followed by nq_attention with
 * tokens == 1, as two kernels per layer when head_dim * cache element bytes
 * <= 256 and q_heads / kv_heads is 1, 2, 4 or 8 (pass 1: one workgroup per kv
 * head and 64-row cache block rotates its q heads, appends k/v at row
 * position[0] when the block holds it, and attends over the block; pass 2
 * merges the blocks' partial results), otherwise as the two calls. q, k, v are the fp32 projection outputs [q_heads * head_dim],
 * [kv_heads * head_dim] x2; out [q_heads * head_dim]. Replaces the pinned
 * one-token rope / cache update / attention sequence of the reference
 * (src/nanoquant/runtime/cuda_kernels.py:401-544,715-815). */
int nq_decode_attention(const float* q, const float* k, const float* v, int32_t q_heads, int32_t kv_heads,
                        int32_t head_dim, const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps,
                        const float* cos_table, const float* sin_table, const int32_t* position,
                        int64_t max_positions, void* k_cache, void* v_cache, int32_t cache_dtype,
                        float scaling, void* out, int32_t out_dtype, void* workspace,
                        int64_t workspace_bytes, void* stream);

/* Pass 1 of nq_decode_attention alone (the same arguments without the output;
 * the same workspace size): the partial results of every 64-row cache block
 * stay in the workspace, as fp32 (max, sum) pairs [q_heads][blocks][2]
 * followed by each block's output acc / sum in fp16 [q_heads][blocks][head_dim]
 * (a block's output is a weighted mean of V rows: values beyond the fp16 range
 * become infinite), blocks = ceil(max_positions / 64); a block past position[0]
 * holds the neutral partial (max -inf, sum 0, output 0), so a merge may run
 * over every block, weighting block s by sum_s * exp(max_s - max).
 * For a projection whose input merges them
 * (nq_linear_batch_fused with NQ_INPUT_ATTENTION). Only the one-pass form:
 * head_dim * cache element bytes <= 256 and q_heads / kv_heads 1, 2, 4 or 8,
 * otherwise NQ_ERR_UNSUPPORTED. No reference counterpart: the reference's
 * attention returns its output (src/nanoquant/runtime/cuda_kernels.py:715-815). */
int nq_decode_attention_partials(const float* q, const float* k, const float* v, int32_t q_heads,
                                 int32_t kv_heads, int32_t head_dim, const void* q_norm, const void* k_norm,
                                 int32_t norm_dtype, float eps, const float* cos_table, const float* sin_table,
                                 const int32_t* position, int64_t max_positions, void* k_cache, void* v_cache,
                                 int32_t cache_dtype, float scaling, void* workspace, int64_t workspace_bytes,
                                 void* stream);

/* out[i] = silu(gate[i]) * up[i], gate and up fp32, out F32/F16/BF16,
 * n % 8 == 0. Replaces the activation of Qwen3MLP.forward. */
int nq_silu_mul(const float* gate, const float* up, int64_t n, void* out, int32_t out_dtype,
                void* stream);

/* Workspace bytes of nq_output_projection (per-workgroup argmax partials). */
int64_t nq_output_projection_workspace_bytes(int64_t vocab, int64_t hidden);

/* logits[v] = Σ_i weight[v, i] * x[i] for one token: weight BF16 [vocab,
 * hidden] row-major, x F32/BF16 [hidden], fp32 accumulation, hidden % 8 == 0
 * and hidden <= 8192. Also leaves the per-workgroup (max, argmax) partials in
 * the workspace for nq_greedy_select. Replaces
 * launch_bfloat16_output_projection
 * (src/nanoquant/runtime/cuda_kernels.py:588-618,684-712). */
int nq_output_projection(const void* x, int32_t x_dtype, const void* weight, int64_t vocab,
                         int64_t hidden, float* logits, void* workspace, int64_t workspace_bytes,
                         void* stream);

/* Greedy token from the partials of the last nq_output_projection with the
 * same (vocab, hidden): the index of the largest logit, the lowest index on
 * ties (torch.argmax). Writes token_out[0]. When history and step are not
 * NULL, also history[*step] = token (only while *step < history_capacity)
 * and *step += 1; when position is not NULL, *position += 1. Replaces the
 * greedy branch of _sample_tokens
 * (src/nanoquant/runtime/generation.py:240-246). */
int nq_greedy_select(const void* workspace, int64_t vocab, int64_t hidden, int64_t* token_out,
                     int64_t* history, int64_t history_capacity, int32_t* step,
                     int32_t* position, void* stream);

/* nq_greedy_select from `count` partials of another projection (nq_int4_projection). */
int nq_greedy_select_partials(const void* partials, int64_t count, int64_t* token_out, int64_t* history,
                              int64_t history_capacity, int32_t* step, int32_t* position, void* stream);

/* Workspace bytes of nq_int4_projection, whatever the type of x (0: none needed; -1: refused sizes). */
int64_t nq_int4_projection_workspace_bytes(int64_t tokens, int64_t out_features, int64_t in_features, int32_t group);

/* Partials (8 bytes each) that nq_int4_projection leaves for one token. */
int64_t nq_int4_projection_partials(int64_t out_features);

/* Products with 4-bit weights and group scales:
 *   y[t, o] = sum_i scales[o, i / group] * (w[o, i] - zeros[o, i / group]) * x[t, i]
 * x F32/F16/BF16 [tokens, in_features] (1 to 65535 tokens; the form is that of a few: the weights
 * are read once for up to 30 tokens (24 of fp32) with groups of 128, 12 with 64 and 6 with 32); packed
 * [out_features, in_features / 2], byte j of a row holding column 2 j in its low
 * four bits and 2 j + 1 in its high ones, 16-byte aligned; scales F32/F16/BF16 [out_features,
 * ceil(in_features / group)], zeros uint8 of the same shape (NULL: 8), any value
 * from 0 to 255; y F32/F16/BF16 [tokens, out_features]. group 32, 64 or 128,
 * in_features a multiple of 32. x is read to 2^-31 of its largest value in a group where it is fp32 (or of 2^-96), to 2^-23
 * where it has 16 bits (or of 2^-100): its values are exact down to 2^-7 (fp32), 2^-12 (fp16) and
 * 2^-15 (bf16) of that largest one. Sums within a group are exact, those of groups fp32 in a fixed order. A token that
 * holds an infinity or a NaN gives NaN. partials, for one token (NULL: not
 * wanted), get the largest value of each 16 rows for nq_greedy_select_partials.
 * Stands beside nq_output_projection for a weight of a quarter of its bytes
 * (the reference's is bf16: src/nanoquant/runtime/cuda_kernels.py:588-618,684-712). */
int nq_int4_projection(const void* x, int32_t x_dtype, int64_t tokens, const void* packed, const void* scales,
                       int32_t scale_dtype, const uint8_t* zeros, int64_t out_features, int64_t in_features,
                       int32_t group, void* y, int32_t y_dtype, void* partials, void* workspace,
                       int64_t workspace_bytes, void* stream);

/* ---- Serving: ragged batches over an 8-bit paged KV cache ------------------ */

/* An 8-bit paged KV cache and the batch that a call runs on it.
 *
 * A page holds page_size (16, 32, 64 or 128) consecutive cache rows of one
 * sequence: for each kv head K as [page_size][head_dim] and V transposed, as
 * [head_dim][page_size], OCP e4m3 bytes that stand for byte * scale, with one
 * fp32 scale for each page, kv head and K or V ([num_pages][kv_heads]). head_dim
 * is 64, 128 or 256; k_pages and v_pages are 16-byte aligned.
 *
 * The call's tokens lie one sequence after the other: sequence b has tokens
 * [query_starts[b], query_starts[b + 1]) (int32, not decreasing; tokens before
 * the first or behind the last start are nobody's, and their rows of every
 * output stay as they were), at cache rows context_lens[b], context_lens[b] + 1,
 * ... Row r of sequence b lies in page page_table[b][r / page_size] at row
 * r % page_size. Entries of the table behind a sequence's last row are not
 * read. All three arrays are device memory, so that a captured call replays
 * with other lengths. */
typedef struct nq_paged_kv {
    void* k_pages;
    void* v_pages;
    float* k_scales;
    float* v_scales;
    int64_t num_pages;
    int32_t kv_heads;
    int32_t head_dim;
    int32_t page_size;
    int32_t reserved;              /* 0 */
    const int32_t* page_table;     /* [batch][table_pages] */
    int64_t table_pages;
    const int32_t* query_starts;   /* [batch + 1] */
    const int32_t* context_lens;   /* [batch] */
    int64_t batch;
} nq_paged_kv;

/* Per-head RMSNorm of q and k (skipped when both weights are NULL), rotate-half
 * RoPE at each token's cache row, and the append to the paged cache:
 *   q_out[t, h, :] = rope(norm(q[t, h, :]))                     (q_out_dtype)
 *   K row of token t = rope(norm(k[t, g, :])), V row = v[t, g, :], as e4m3(x / scale)
 * A page's scale is the least power of two (from 2^-126 on) that brings all its
 * rows within 448: the larger of the one it has and of what the new rows need;
 * a page whose row 0 is written starts anew. When it grows, the rows before the
 * new ones are rounded to the new scale. Rows behind the new ones stay as they
 * are. Infinities and NaN are stored as NaN and do not count for the scale.
 * q, k, v F32/F16/BF16 of one type, [tokens, heads * head_dim]; tables
 * [rope_positions, head_dim / 2]. A token whose row lies outside the page table
 * or the RoPE tables writes nothing; one whose table entry names no page writes
 * q_out alone. A page that the call writes to belongs to one sequence and stands
 * once in its part of the table. q_out may be q where both have one type.
 * K is normed and rotated in fp64, so a stored byte is the rounding of the exact
 * value. Replaces launch_decode_rope and launch_cache_prefix_update
 * (src/nanoquant/runtime/cuda_kernels.py:401-447,546-587,715-815) for many
 * sequences and pages. */
int nq_paged_append(const void* q, const void* k, const void* v, int32_t dtype, int64_t tokens,
                    int32_t q_heads, const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps,
                    const float* cos_table, const float* sin_table, int64_t rope_positions,
                    const nq_paged_kv* kv, void* q_out, int32_t q_out_dtype, void* stream);

/* nq_paged_append for sequences whose tokens have other positions than cache rows,
 * as after nq_paged_evict: sequence b's tokens are rotated as those at positions
 * rope_starts[b], rope_starts[b] + 1, ... (int32 [batch], device memory; NULL:
 * their cache rows). A token whose position lies outside the RoPE tables writes nothing. */
int nq_paged_append_at(const void* q, const void* k, const void* v, int32_t dtype, int64_t tokens,
                       int32_t q_heads, const void* q_norm, const void* k_norm, int32_t norm_dtype, float eps,
                       const float* cos_table, const float* sin_table, int64_t rope_positions,
                       const nq_paged_kv* kv, const int32_t* rope_starts, void* q_out, int32_t q_out_dtype,
                       void* stream);

/* Workspace bytes of nq_paged_attention (0: none needed; at most 1 GiB), or -1 for
 * sizes that it refuses: among others a grid of 2^32 threads or more, as the
 * append and the log probabilities refuse too (NQ_ERR_SHAPE). */
int64_t nq_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int32_t q_heads, int32_t kv_heads,
                                           int32_t head_dim, int32_t page_size, int64_t table_pages);

/* Causal grouped-query attention of the call's tokens (after nq_paged_append
 * with the same arrays): the token at cache row r attends rows [0, r] of its
 * sequence, kv head h / (q_heads / kv_heads):
 *   out[t, h, :] = softmax(scaling * q[t, h, :] . K) . V
 * q F32/F16/BF16 [tokens, q_heads, head_dim] (F16 and BF16 read exactly, F32 to
 * 2^-23 of every value down to 2^-28 of its head's largest, or of 2^-100, and to
 * 2^-51 of that below); out F32/F16/BF16 [tokens, q_heads * head_dim]; both
 * 16-byte aligned, q_heads a multiple of kv_heads. Scores and softmax in fp32, the
 * weights to 16 bits for 16-bit outputs and 24 for fp32, results joined in a fixed
 * order (deterministic).
 * A token whose row lies outside the page table gives zeros. A table entry in use
 * that names no page counts as NaN rows. NaN in the cache, infinities and NaN in q
 * do what fp32 arithmetic does with them, for the tokens that see them alone; rows
 * that nobody sees may hold anything. Replaces
 * launch_decode_attention (src/nanoquant/runtime/cuda_kernels.py:448-544) for
 * many sequences and pages. */
int nq_paged_attention(const void* q, int32_t q_dtype, int64_t tokens, int32_t q_heads, const nq_paged_kv* kv,
                       float scaling, void* out, int32_t out_dtype, void* workspace, int64_t workspace_bytes,
                       void* stream);

/* Workspace bytes of nq_shared_attention (0: none needed; at most 1 GiB), or -1 for
 * sizes that it refuses. */
int64_t nq_shared_attention_workspace_bytes(int64_t tokens, int64_t batch, int32_t q_heads, int32_t kv_heads,
                                            int32_t head_dim, int32_t page_size, int64_t table_pages,
                                            int64_t shared_rows);

/* nq_paged_attention for sequences that hold the same first rows, which are read
 * once for many query rows of different sequences where each has few of them:
 * the first shared_rows / page_size entries of every sequence's part of the page
 * table stand for the same pages, and the call reads sequence 0's in their
 * place (as many of them as make whole multiples of 64 rows too). What a token sees is what it sees in
 * nq_paged_attention, also where a sequence has fewer rows than that. shared_rows
 * is 0 to page_size * table_pages; it is part of a captured call.
 * lse (fp32 [tokens, q_heads], NULL: not wanted) gets each query row's
 *   lse[t, h] = log sum_j exp(scaling * q[t, h, :] . K_j)
 * over the rows that the token sees; -inf for a token whose row lies outside the
 * page table. Types, layouts and everything else as in nq_paged_attention. */
int nq_shared_attention(const void* q, int32_t q_dtype, int64_t tokens, int32_t q_heads, const nq_paged_kv* kv,
                        int64_t shared_rows, float scaling, void* out, int32_t out_dtype, float* lse,
                        void* workspace, int64_t workspace_bytes, void* stream);

/* The attention that cached rows receive from the call's tokens, summed over the
 * tokens that see them and the q heads of a kv head g:
 *   out[page of j, g, row of j] = old + sum_t sum_h exp(scaling * q[t, h, :] . K_j - lse[t, h])
 * for every row j from `first` on of a sequence that has tokens in the call; old is
 * weights' value there, or 0 for rows that the call itself brought (j >= context_lens[b]),
 * so that pages need no clearing. Nothing else of out is written. weights and out
 * are fp32 [num_pages, kv_heads, page_size] and may be the same; lse as
 * nq_shared_attention left it for the same call. Pages that the rows from `first` on
 * lie in belong to one sequence and stand once in its part of the table; rows before
 * `first` may lie in pages that sequences share. A row whose table entry names no page is left
 * out. q as in nq_paged_attention; a weight is off by about 2^-22 of lse and of its
 * score relative to itself (never above 1 where lse is beyond 710), and NaN where they are. Sums in fp32
 * in a fixed order (deterministic). */
int nq_attention_weights(const void* q, int32_t q_dtype, int64_t tokens, int32_t q_heads, const nq_paged_kv* kv,
                         float scaling, const float* lse, int64_t first, const float* weights, float* out,
                         void* stream);

/* Workspace bytes of nq_paged_evict (0: none needed; -1: refused sizes). */
int64_t nq_paged_evict_workspace_bytes(int64_t batch, int32_t kv_heads, int32_t page_size, int64_t table_pages,
                                       int64_t budget);

/* Cuts every sequence with more than `budget` cached rows to that many. Of such a
 * sequence's n = context_lens[b] rows stay, for each kv head by itself, rows
 * [0, first), rows [n - recent, n) and of those between the
 * budget - first - recent with the greatest weights (nq_attention_weights; fp32
 * [num_pages, kv_heads, page_size]), the lowest row first among equals, NaN above all. They keep
 * their order: row i of the cut sequence is row rows_out[b, g, i] of the old one.
 *   page_table_out [batch, ceil(budget / page_size)]: the first / page_size pages in
 *     front as they were (nothing of them is written: others may share them), then
 *     the pages into[b, :] ([batch, ceil(budget / page_size) - first / page_size])
 *   context_lens_out [batch]: budget
 *   into's pages: the rows' K and V as an append of them in one call would store
 *     them (a page's scale is the least power of two that brings its rows within
 *     448) and their weights; nothing is written behind the last row
 * A sequence with budget rows or fewer keeps its pages and its length; its entries of into are not
 * touched, and rows_out has its rows, then -1. Rows in pages that the
 * table does not name count as NaN; an entry of into that names no page writes nothing but
 * page_table_out. into's pages stand there once, and in no sequence's part of the page table.
 * Values beyond fp32 become NaN. Outputs lie apart from the arrays that the call reads. kv->query_starts is not read and may be NULL.
 * first + recent <= budget. context_lens counts the rows of tokens that a call has just appended too; page_table_out
 * has no entry behind the budget's last page for tokens to come. Keys keep the rotation of their position: the
 * tokens appended next have other positions than cache rows (nq_paged_append_at). */
int nq_paged_evict(const nq_paged_kv* kv, float* weights, const int32_t* into, int64_t budget, int64_t first,
                   int64_t recent, int32_t* page_table_out, int32_t* context_lens_out, int32_t* rows_out,
                   void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of nq_token_logprobs (0: none needed; -1: refused sizes). */
int64_t nq_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int32_t top);

/* For each row of logits (F32/F16/BF16, row_stride >= vocab elements apart):
 *   logprobs[r] = log softmax(logits[r])[tokens[r]]   (NaN for a token outside [0, vocab))
 *   entropy[r]  = -sum p log p over the row, 0 log 0 = 0
 *   top_ids[r, :], top_logprobs[r, :] = the `top` likeliest tokens, likeliest first,
 *     the lowest index first among equals, NaN above all
 * top 0 to 32 (top_ids and top_logprobs may be NULL for 0). Logits of -inf have
 * probability 0; a row that holds NaN or +inf, or -inf alone, has NaN for every
 * log probability and for the entropy. Beside nq_greedy_select for callers that
 * report how likely an answer is; the reference's engine returns tokens alone (src/nanoquant/runtime/generation.py:240-246). */
int nq_token_logprobs(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                      const int64_t* tokens, int32_t top, float* logprobs, float* entropy, int64_t* top_ids,
                      float* top_logprobs, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NQAMD_SHELL_H */
