/*
 * smeai_paged.h -- C-ABI of the paged key/value cache: a step's block table
 * and slots, writing its keys and values, and attention over the pages.
 *
 * The reference's self-attention (sme_ai_library/include/sme_ai_ops.h:410-455)
 * sees one whole sequence at a time and keeps nothing; a decode step over a
 * running sequence needs the keys and values of the earlier tokens.  These
 * entry points keep them in fixed-size pages shared by all requests.
 *
 * A step of a serving loop over n_req requests, the new tokens of all requests
 * stored behind one another (request i owns rows q_start[i] .. q_start[i+1]):
 *   smeai_paged_plan       lengths -> block table, row offsets, slots, positions
 *   smeai_paged_append     rows of the q/k/v linear -> rotated queries, cache
 *   smeai_paged_attention  queries x pages -> context rows
 *
 * Every pointer is device memory, work is queued on `stream` (a cudaStream_t,
 * NULL = legacy default) of the current device and the calls return without
 * waiting; nothing is allocated, so all three can be captured in a CUDA graph.
 * Status: 0, or a negative code (smeai_q2k.h); smeai_last_error() says why.
 * Values that only the GPU sees (lengths, slots, positions, page numbers) are
 * checked there: one outside its buffer is skipped and reported by bit 1 of
 * smeai_take_device_error; what it would have produced is unspecified.
 */
#ifndef SMEAI_PAGED_H
#define SMEAI_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the cache, the queries and the context (ggml's numbers). */
#define SMEAI_KV_F16 1
#define SMEAI_KV_BF16 30

/* The cache: element d of key head h of the token in slot (page, t), where
 * t < page_size, is k[page * page_stride + h * head_stride + t * token_stride
 * + d]; v likewise.  Strides count elements, are multiples of 8 and do not
 * overlap; k and v are 16-byte aligned.  page_size is a power of two up to
 * 65536, head_dim a multiple of 8 up to 256. */
typedef struct smeai_kv_cache {
  void *k, *v;
  int type;            /* SMEAI_KV_* */
  int page_size;
  int n_kv_heads, head_dim;
  int64_t n_pages;
  int64_t page_stride, head_stride, token_stride;
} smeai_kv_cache;

/* A step's bookkeeping.  Request i holds cached_len[i] tokens in pages
 * block_table[i * ld_table + 0 ..] and brings new_len[i] more.  Requests are
 * served in order: each that needs more pages takes them from free_pages,
 * from index *n_used on.  A request is refused when the pool runs out at or
 * before it and it needs pages, when its length passes max_blocks pages, or
 * when its rows pass n_tokens: its table row stays, its kv_len is 0 and its
 * tokens get no slot.
 *   block_table  entries of the newly taken pages are written, others stay
 *   q_start      [n_req + 1] first row of each request (cut at n_tokens)
 *   kv_len       [n_req] cached + new tokens (0: refused)
 *   slots        [n_tokens] page * page_size + place of each new token; -1
 *                for a refused request's and for rows behind the last token
 *   positions    [n_tokens] the token's place in its sequence; 0 without slot
 *   n_used_out   *n_used plus the pages taken; may be n_used itself
 * The lengths are read before anything is written: kv_len may be cached_len
 * itself, so that one step's result is the next one's input (a refused
 * request's length is then gone), and new_len may lie in q_start or kv_len.
 * n_req is at most 8192; n_tokens may be 0. */
int smeai_paged_plan(const int32_t *cached_len, const int32_t *new_len, int64_t n_req, int page_size,
                     const int32_t *free_pages, int64_t n_free, const int32_t *n_used, int32_t *n_used_out,
                     int32_t *block_table, int64_t ld_table, int64_t max_blocks, int32_t *q_start, int32_t *kv_len,
                     int64_t *slots, int32_t *positions, int64_t n_tokens, void *stream);

/* Rounds a step's keys and values (fp32 rows of n_kv_heads * head_dim values,
 * row strides ld_k and ld_v floats) to the cache's type (nearest even) and
 * writes them into the tokens' slots; rows with slot -1 are left out.  No two
 * rows may have the same slot.  With
 * rope, keys are rotated first, and queries too: rope is [n_rope][head_dim],
 * the cosines of a position's head_dim/2 angles, then their sines; angle i
 * turns elements (2i, 2i+1), or (i, i + head_dim/2) when halves is set.  With
 * q (n_heads * head_dim values a row, stride ld_q), the rotated and rounded
 * queries go to q_out (stride ld_q_out elements), for every row, slot or not.
 * positions is needed with rope only.  q and q_out may be NULL together. */
int smeai_paged_append(const smeai_kv_cache *cache, const float *k, int64_t ld_k, const float *v, int64_t ld_v,
                       const float *q, int64_t ld_q, int n_heads, void *q_out, int64_t ld_q_out, int64_t n_tokens,
                       const int64_t *slots, const int32_t *positions, const float *rope, int64_t n_rope, int halves,
                       void *stream);

/* Attention of each request's new tokens over its kv_len[i] cached tokens
 * (the new ones among them, appended before): for query row r of request i
 * with n = q_start[i+1] - q_start[i], over the keys j < kv_len[i], and with
 * causal only j <= kv_len[i] - n + (r - q_start[i]),
 *   out[r] = sum_j softmax_j(scale * q[r] . k_j) v_j
 * per head; head h reads key head h / (n_heads / n_kv_heads).  A row that sees
 * no key (an empty cache, a refused request) is 0.  q and out hold n_heads *
 * head_dim values of the cache's type a row, row strides ld_q and ld_out
 * elements (multiples of 8), 16-byte aligned; n_tokens rows; out and q do not
 * overlap; rows of out outside q_start[0] .. q_start[n_req] are left as they
 * were.  scale is positive, up to 2e38.  Scores, softmax
 * and the running sums are fp32; the softmax weights are rounded to the
 * cache's type for the tensor cores.  Slots past kv_len are never read, so
 * they may hold anything; a NaN or infinity within reaches the rows of its own
 * request only (with causal, possibly a chunk's rows before it).
 * max_new is the largest number of new tokens of a request (larger ones still
 * come out right, more slowly); a captured call keeps it.
 * workspace: at least smeai_paged_attention_workspace bytes (0, and then NULL
 * will do, when a table row names too few keys for a request ever to be split
 * over CTAs, and for sizes that the call refuses), 256-byte aligned, in use
 * until the call's work is done, by one call at a time; need not be
 * initialised and holds nothing afterwards. */
size_t smeai_paged_attention_workspace(const smeai_kv_cache *cache, int n_heads, int64_t n_tokens, int64_t n_req,
                                       int64_t max_blocks, int64_t max_new);
int smeai_paged_attention(const smeai_kv_cache *cache, const void *q, int64_t ld_q, int n_heads, int64_t n_tokens,
                          const int32_t *q_start, const int32_t *kv_len, int64_t n_req, const int32_t *block_table,
                          int64_t ld_table, int64_t max_blocks, int64_t max_new, float scale, int causal, void *out,
                          int64_t ld_out, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
