/*
 * awq_serving.h -- C ABI of the serving operators in the W4A16 AWQ library:
 * many requests that share one paged KV cache held in 4 bits.
 *
 *   awq_serve_page_step       block tables, slots and positions of a step's tokens
 *   awq_serve_page_release    pages of requests that end or shrink go back
 *   awq_serve_kv4_append      RoPE of q and k; k and v quantised and stored
 *   awq_serve_kv4_gather      the values that the cache holds
 *   awq_serve_kv4_attention   attention over the cache
 *   awq_serve_logits          penalties, biases, a grammar's mask, greedy token
 *
 * The reference has one static fp16 cache and one sequence
 * (inference/kv_cache.py:31-67, inference/engine.py:64-147); these have no
 * counterpart there.
 *
 * All pointers are device pointers, `stream` is a hipStream_t (NULL = the
 * legacy default stream).  No entry point allocates, synchronises the host or
 * keeps anything between calls: each can be captured into a HIP graph, and
 * calls on different streams may overlap if their outputs and workspaces
 * differ.  Status codes: awq_w4a16.h.
 *
 * Lengths, tables, slots and positions are read on the device; the host does
 * not see them.  What lies outside its range never moves an access out of a
 * buffer: a token without a valid slot is not stored, a query whose request
 * refers to a page outside the cache gives NaN.  (Bounds that the host gives -- sizes,
 * strides, max_pos -- have to be true of the buffers.)
 *
 * The cache of one layer: uint8 [num_pages, num_kv_heads, block], block =
 * page_size * (head_dim + 8 * head_dim / group_size) bytes.  A block holds one
 * page of one kv head:
 *
 *   K codes   [token][t = 0 .. 3][s = 0 .. head_dim / 32 - 1] 32-bit words: the
 *             word (t, s) holds columns 32 s + 8 t + e, e = 0 .. 7, column e in
 *             the four bits from 4 * (e / 2 + 4 * (e % 2))
 *   V codes   [token / 4][j = 0 .. head_dim / 8 - 1][token % 4] words: columns
 *             8 j + e in the four bits from 4 e
 *   K scales  [token][group] fp16 pairs (scale, zero)
 *   V scales  [token / 4][group][4 scales of token % 4, then 4 zeros] fp16
 *
 * A group is group_size neighbouring columns of one token's head:
 *   zero  = fp16(min), scale = (max - zero) / 15 rounded up to 7 significant
 *   bits (and to fp16's smallest steps below 2^-17), code = round((x - zero) /
 *   scale) to even, 0 where the scale is 0; value = code * scale + zero.
 * code * scale has at most 11 significant bits: it is exact in fp16, and K and
 * V enter the matrix cores without a rounding.
 * Where k or v of a token and head holds a NaN, an infinity or a group that
 * fp16 cannot hold (|min| > 65504, a range over 60480), K's scales and zeros
 * are NaN and V's values 0: every query that sees the token gives NaN, no
 * other does.
 */
#ifndef AWQ_SERVING_H
#define AWQ_SERVING_H

#include <stddef.h>
#include <stdint.h>

#include "awq_w4a16.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations and logits. */
#define AWQ_SERVE_FP16 0
#define AWQ_SERVE_BF16 1
#define AWQ_SERVE_FP32 2

/* Most requests of one call, and the most heads that share a kv head. */
#define AWQ_SERVE_MAX_REQUESTS 4096
#define AWQ_SERVE_MAX_GROUP 64

/* A step's new tokens: request b holds state[b] tokens and adds new_tokens[b],
 * its rows following those of request b - 1 in a batch of `total` rows.
 * state int32 [requests + 1]: the lengths, then the number of free pages; a
 * free page is taken from the end of free_pages (int32 [capacity], as many as can be
 * free at once, the first state[requests] of them free).  block_tables int32 [requests, table_width]:
 * entries of pages that the step takes are written.
 *
 * A request is refused if new_tokens < 0 or length < 0, its rows pass `total`,
 * its tokens pass table_width * page_size, or -- pages being handed out in
 * request order -- the free pages do not suffice for it and all before it that
 * were not refused for the other reasons.  It then keeps its length, takes no
 * page and its rows have slot -1 and position -1.
 *
 * Out: new_state int32 [requests + 1]; query_start int32 [requests + 1] (the
 * requests' first rows, at most `total`; a refused request keeps its rows);
 * slots int32 [total], page * page_size + offset; positions int32 [total];
 * failed int32 [requests], 1 where refused.  Rows behind the last request's have
 * slot -1 and position -1.  No output may overlap an input.  page_size: a power of
 * two of 16 .. 256; total and capacity at most 2^24, table_width * page_size at
 * most 2^30.  One launch. */
int awq_serve_page_step(const int32_t* state, const int32_t* new_tokens, int32_t* block_tables,
                        const int32_t* free_pages, int32_t* new_state, int32_t* query_start, int32_t* slots,
                        int32_t* positions, int32_t* failed, int64_t requests, int64_t total, int64_t table_width,
                        int64_t capacity, int64_t page_size, void* stream);

/* Request b keeps its first min(max(keep[b], 0), length) tokens; the pages past them
 * go onto the end of free_pages in request and page order.  new_state as above.
 * The table's entries stay as they are (those past a length mean nothing). */
int awq_serve_page_release(const int32_t* state, const int32_t* keep, const int32_t* block_tables,
                           int32_t* free_pages, int32_t* new_state, int64_t requests, int64_t table_width,
                           int64_t capacity, int64_t page_size, void* stream);

/* q, k and v of `tokens` rows of a fused projection, qkv [tokens, (num_heads + 2
 * num_kv_heads) * head_dim] with qkv_stride elements from row to row: rotate-half
 * RoPE of q and k in fp32 by cos / sin fp32 [max_pos, head_dim] at the rows'
 * positions (both NULL: no rotation), q_out [tokens, num_heads * head_dim] in
 * qkv's type, k and v quantised into the cache's slots.  A slot outside the
 * cache: nothing is stored.  A position outside 0 .. max_pos - 1: q_out NaN, nothing
 * stored.  Two rows of one slot leave any mixture of theirs (codes of one, scales of the
 * other) in it.  dtype fp16 or bf16; qkv, cos, sin, q_out
 * 16-byte aligned, qkv_stride a multiple of 8.  One launch. */
int awq_serve_kv4_append(const void* qkv, int64_t qkv_stride, void* cache, const int32_t* slots,
                         const int32_t* positions, const void* cos, const void* sin, void* q_out, int64_t tokens,
                         int64_t num_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_pages,
                         int64_t page_size, int64_t group_size, int64_t max_pos, int32_t dtype, void* stream);

/* k, v [tokens, num_kv_heads, head_dim]: code * scale + zero in fp32, rounded once
 * to dtype; NaN where the slot is outside the cache. */
int awq_serve_kv4_gather(const void* cache, const int32_t* slots, void* k, void* v, int64_t tokens,
                         int64_t num_kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
                         int64_t group_size, int32_t dtype, void* stream);

/* softmax(scale * q K^T) V over a paged cache.  Request b has the rows
 * query_start[b] .. query_start[b + 1] - 1 of q [total, num_heads * head_dim]
 * (q_stride elements from row to row) and seq_lens[b] tokens in the cache, the
 * rows' own among them: row i of n stands at position seq_lens[b] - n + i and
 * sees the tokens 0 .. position.  A row that sees none (a negative position) and a
 * row of no request give zeros.  No row is two requests': an entry of query_start below an
 * earlier one counts as that one.  out [total, num_heads * head_dim] in q's type.
 * A row that sees a token past table_width * page_size, or in a page outside the cache, gives NaN.
 * max_query: at least the largest number of rows of a request (it sizes the grid and the
 * workspace; rows past it are NaN).
 * q is scaled by a power of two that brings a row's largest value below 2^8 and held in fp16
 * (to 2^-32 of that value; exact for fp16 rows that are below 2^8 to begin with), the probabilities in two fp16 parts, all sums in
 * fp32.  num_heads a multiple of num_kv_heads, at most AWQ_SERVE_MAX_GROUP
 * times it; scale positive and finite; head_dim 64 or 128, group_size 32, 64 or 128 and at most head_dim.
 * workspace: at least awq_serve_kv4_attention_workspace bytes of any content. */
size_t awq_serve_kv4_attention_workspace(int64_t requests, int64_t total, int64_t max_query, int64_t num_heads,
                                         int64_t num_kv_heads, int64_t head_dim, int64_t table_width,
                                         int64_t page_size);
int awq_serve_kv4_attention(const void* q, int64_t q_stride, const void* cache, const int32_t* block_tables,
                            const int32_t* seq_lens, const int32_t* query_start, void* out, int64_t requests,
                            int64_t total, int64_t max_query, int64_t num_heads, int64_t num_kv_heads,
                            int64_t head_dim, int64_t table_width, int64_t num_pages, int64_t page_size,
                            int64_t group_size, float scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                            void* stream);

/* One step's logits [rows, vocab] (row_stride elements from row to row) after, in this
 * order and in fp32:
 *   repetition  x > 0 ? x / repetition[r] : x * repetition[r]   of every token of the row's history
 *   frequency   x - frequency[r] * n                             n: how often the row generated it
 *   presence    x - presence[r]                                  where n > 0
 *   bias        x + bias_values[i]                               i: the last entry of the row with this token
 *   mask        -inf where bit v % 32 of word v / 32 is 0
 * rounded once to dtype into out [rows, vocab] (contiguous; may be logits itself where that is
 * contiguous).  next_token int64 [rows]: the lowest index of the largest value in
 * out, a NaN counting as the largest; -1 where every value is -inf.
 * The history of row r: tokens [r, 0 .. lengths[r] - 1] of `width` (int64, or int32
 * with token_bytes 4), the first prompt_lens[r] of them the prompt, the rest
 * generated; tokens outside the vocabulary are ignored, lengths count at most `width`.  Biases of row r:
 * entries bias_start[r] .. bias_start[r + 1] - 1 (within 0 .. bias_count) of bias_tokens int32,
 * bias_values fp32.  mask int32 [rows, ceil(vocab / 32)].  repetition, presence and
 * frequency fp32 [rows].  NULL: tokens, lengths and prompt_lens together (then no
 * penalties), each penalty, the three biases together, mask.
 * workspace: awq_serve_logits_workspace bytes of any content, 8-byte aligned.  Two launches. */
size_t awq_serve_logits_workspace(int64_t rows, int64_t vocab);
int awq_serve_logits(const void* logits, int64_t row_stride, void* out, int64_t* next_token, int64_t rows,
                     int64_t vocab, int32_t dtype, const void* tokens, int32_t token_bytes, int64_t width,
                     const int32_t* lengths, const int32_t* prompt_lens, const float* repetition,
                     const float* presence, const float* frequency, const int32_t* bias_start,
                     const int32_t* bias_tokens, const float* bias_values, int64_t bias_count, const int32_t* mask,
                     void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AWQ_SERVING_H */
