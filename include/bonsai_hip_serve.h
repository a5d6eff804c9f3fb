/*
 * bonsai_hip_serve.h -- C ABI of a serving step over a paged KV cache.
 *
 * bonsai_hip.h serves one sequence: its cache is contiguous and a call has one
 * pos0.  The entry points below serve many requests in one step, with the
 * cache in pages of one pool and all bookkeeping on the device:
 *
 *   bh_paged_plan       lengths -> pages taken and given back, slots,
 *                       positions, ragged offsets        (once a step)
 *   bh_kv_store_paged   the step's k / v rows into their slots (a layer)
 *   bh_attention_paged  every request's new queries over its pages (a layer)
 *   bh_token_logprobs   log probabilities of the chosen tokens, entropy,
 *                       the most likely alternatives     (once a step)
 *
 * The reference serves one sequence at a time and has none of these; the
 * conventions are bonsai_hip.h's: device pointers owned by the caller, work
 * enqueued on `stream` of the current device without synchronising, a status
 * code back, the message from bh_last_error().  f32 data; f32 or f16 caches.
 * Nothing depends on data the host cannot see at the call, so every entry
 * point can be captured in a HIP graph and replayed with other lengths.
 *
 * What lies on the device (lengths, tables, slots, tokens) cannot be refused
 * by a status.  No value of it makes a kernel read or write outside the
 * buffers described: each entry point says what it does with bad ones.
 *
 * Workspaces: bh_attention_paged and bh_token_logprobs keep partial results in
 * `workspace` (16-byte aligned, at least the bytes that the _workspace
 * function names).  With workspace = NULL they use the library's per-device
 * scratch, as bh_attention does: calls of one entry point must then not
 * overlap on one device, and the first call outside a capture reserves it.
 * Calls that may overlap (two streams, two captured graphs) each bring their
 * own workspace.
 */
#ifndef BONSAI_HIP_SERVE_H
#define BONSAI_HIP_SERVE_H

#include "bonsai_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A pool of pages of K and V.  Element [page][position][head][dim] lies at
 *   page * page_stride + position * pos_stride + head * head_stride + dim
 * of k and of v (strides in elements, equal for both): a page may hold rows of
 * n_kv * hd as bh_kv_store's cache does, or lie head by head; K and V may share
 * one allocation.  The dimensions nest, in any order: a larger stride is at least
 * what all smaller ones reach, so that no two rows share memory (strides of
 * dimensions of one entry don't count).  page_size is any size from 1; n_pages *
 * page_size < 2^31. */
typedef struct bh_paged_cache {
  void *k, *v;
  int kv_dtype; /* BH_KV_F32 or BH_KV_F16 */
  size_t n_pages, page_size, n_kv, hd;
  size_t page_stride, pos_stride, head_stride;
} bh_paged_cache;

/* ---------------------------------------------------------------------------
 * The plan of a step
 * ------------------------------------------------------------------------- */

#define BH_PAGED_MAX_REQ 4096

/* From the requests' lengths everything the step's other calls read.  Request i
 * holds cached[i] positions in the pages block_table[i][0 ..] and gets
 * n_new[i] new tokens; n_new[i] < 0 releases it.  With W = table_width,
 * P = page_size and have = ceil(cached[i] / P):
 *
 * released  its pages block_table[i][0 .. have) are pushed on the stack of free
 *           pages, requests and blocks in order; kv_len[i] = 0, no tokens.
 * refused   when cached[i] + n_new[i] > W P, or its new pages, counted over the
 *           requests up to it (refused ones included, those too long for the
 *           table not), are more than the stack holds with the released ones
 *           on it, or its new tokens counted so are more than n_tok:
 *           kv_len[i] = 0, no tokens, no pages, its table row as it was.
 *           It holds its cached positions still: cached of the next step is
 *           kv_len[i] where kv_len[i] > 0 or n_new[i] < 0, and as it was
 *           otherwise.  (Refused are those with n_new[i] >= 0 and
 *           kv_len[i] != cached[i] + n_new[i].)
 * otherwise its blocks from `have` on are popped from the stack into
 *           block_table[i], kv_len[i] = cached[i] + n_new[i].
 *
 * q_start: running total of the tokens admitted (n_req + 1 entries).  Token t
 * of request i stands at position p = kv_len[i] - n_new[i] + t - q_start[i]:
 * slots[t] = block_table[i][p / P] * P + p % P, pos[t] = (p, p, p, p) as
 * bh_qk_norm_rope reads it (pos may be NULL).  Tokens from q_start[n_req] on
 * are padding: slot -1, position 0.  n_free_out: pages on the stack now;
 * n_refused (may be NULL): requests refused.
 *
 * A plan that is run again on the same inputs gives the same outputs:
 * n_free and n_free_out are separate words (they may be the same one, for a
 * stack that moves on by itself), and nothing below *n_free on the stack is
 * written.  kv_len must not be cached.  cached[i] < 0 counts as 0, *n_free is
 * clipped to 0 .. n_pages, pages pushed past n_pages are dropped, a released
 * request has no more pages than its table row.  Page numbers are passed on as
 * they are (a page that two requests share is to be released by one of them); a
 * token on a page outside the pool has slot -1.
 * n_req <= BH_PAGED_MAX_REQ. */
typedef struct bh_paged_plan_args {
  const int32_t *cached; /* [n_req]                                  */
  const int32_t *n_new;  /* [n_req]                                  */
  int32_t *block_table;  /* [n_req][table_width]                     */
  int32_t *free_pages;   /* [n_pages], the first *n_free are free     */
  const int32_t *n_free; /* one word                                 */
  int32_t *kv_len;       /* [n_req]                                  */
  int32_t *q_start;      /* [n_req + 1]                              */
  int32_t *slots;        /* [n_tok]                                  */
  int32_t *pos;          /* [n_tok][4] or NULL                       */
  int32_t *n_free_out;   /* one word                                 */
  int32_t *n_refused;    /* one word or NULL                         */
  size_t n_req, n_tok, table_width, page_size, n_pages;
} bh_paged_plan_args;

int bh_paged_plan(const bh_paged_plan_args *args, bh_stream stream);

/* ---------------------------------------------------------------------------
 * The append
 * ------------------------------------------------------------------------- */

/* bh_kv_store into pages: rows k, v [n_tok][n_kv * hd] (f32) to the positions
 * slots[t] = page * page_size + offset of the cache, as f32 or as the f16 bits
 * that bh_kv_store writes.  A slot below 0 or past the pool stores nothing.
 * Slots are distinct, as the plan's are: of two tokens with one slot either
 * may be found there, or parts of both.  No scratch. */
int bh_kv_store_paged(const bh_paged_cache *cache, const float *k, const float *v,
                      const int32_t *slots, size_t n_tok, bh_stream stream);

/* ---------------------------------------------------------------------------
 * Attention
 * ------------------------------------------------------------------------- */

/* bh_attention over pages, for the new tokens of n_req requests at once.
 * Request i's tokens are q_start[i] .. q_start[i + 1] - 1, its query t - th new
 * one stands at p = kv_len[i] - (q_start[i + 1] - q_start[i]) + t and sees the
 * positions 0 .. p of its pages block_table[i]; head hq reads kv head
 * hq / (n_head / n_kv): scores q.k / sqrtf(hd), softmax, probabilities times v.
 * The tokens' own rows are stored already.  What a query does not see, later
 * rows of a page among it, may hold anything.  A query at p < 0 sees nothing
 * and gets zeros.  Tokens of no request are left as they were.
 *
 * q, out: [n_tok][n_head][hd] f32, out is not q; n_tok < 2^24, n_req at most 2^31 -
 * 65536.  Entries of q_start do not decrease (if they do, tokens' results are
 * unspecified, and where requests ask for more than n_tok tokens in all, they may be
 * left as they were) and are clipped to 0 .. n_tok, kv_len to 0 .. table_width *
 * page_size (at most 2^31 - 65536).
 * A table entry outside 0 .. n_pages - 1 among a request's
 * ceil(kv_len / page_size) leaves its positions out, and is written to
 * *bad_page where that is not NULL (the caller presets it).
 *
 * max_new: no request has more new tokens than this (0: n_tok); it steers how
 * the work is laid out, and a wrong one costs time: results agree to rounding
 * whatever it is.  Any hd up to 512 and any
 * n_head that n_kv divides; hd 64, 128 and 256 with strides and pointers of
 * whole 16 bytes run on the matrix cores.  Results agree with 64-bit arithmetic
 * to about 1e-6 of sum w |v|, w being the weights, and are the same bits from call
 * to call on one device.  Scores s are f32, which adds |s| 2^-22 of itself to a
 * weight's error.  The partial sums of q.k, log2(e) q.k, and over an f32 cache the
 * sum of the |v| that a query sees stay below the largest f32.  What is infinite or
 * NaN among the values a query sees makes the dimensions it is in not finite. */
typedef struct bh_attention_paged_args {
  bh_paged_cache cache;
  const float *q;
  float *out;
  const int32_t *q_start;     /* [n_req + 1]            */
  const int32_t *kv_len;      /* [n_req]                */
  const int32_t *block_table; /* [n_req][table_width]   */
  int32_t *bad_page;          /* one word or NULL       */
  size_t n_tok, n_req, n_head, table_width, max_new;
  void *workspace; /* NULL: the library's scratch */
  size_t workspace_bytes;
} bh_attention_paged_args;

int bh_attention_paged(const bh_attention_paged_args *args, bh_stream stream);
/* Bytes of workspace that a call with these arguments needs on the current
 * device; the lengths on the device do not enter (0: none, or bad arguments). */
size_t bh_attention_paged_workspace(const bh_attention_paged_args *args);

/* ---------------------------------------------------------------------------
 * Log probabilities
 * ------------------------------------------------------------------------- */

#define BH_MAX_TOP 32

/* Of each row x [vocab] of logits, with z = x * inv_temp and Z = sum exp(z):
 *   logprob     = z[token] - log Z
 *   entropy     = log Z - sum exp(z) z / Z      (natural logarithm)
 *   top_ids     the n_top ids of the largest logits, largest first, of equal
 *               ones the lowest id first; -0 equals 0
 *   top_logprobs  theirs
 * Rows begin row_stride floats apart.  A logit of -inf has probability 0.  A
 * row with a NaN or +inf among its logits, or with nothing above -inf, has NaN
 * for logprob, entropy and top_logprobs; its top_ids order NaN below every
 * number.  A token >= vocab gives NaN and is written to *bad_id where that is
 * not NULL (the caller presets it), the rest of its row is as any other's.
 * Either of logprob (then tokens too) and entropy may be NULL; with n_top = 0
 * top_ids and top_logprobs are.  n_top <= BH_MAX_TOP and <= vocab; inv_temp is
 * finite and above 0; vocab < 2^31.  Finite logits of a row differ by less than the
 * largest f32 (one further below the largest counts as -inf). */
typedef struct bh_token_logprobs_args {
  const float *x;          /* [n_rows][row_stride]      */
  const uint32_t *tokens;  /* [n_rows] or NULL          */
  float *logprob;          /* [n_rows] or NULL          */
  float *entropy;          /* [n_rows] or NULL          */
  uint32_t *top_ids;       /* [n_rows][n_top] or NULL   */
  float *top_logprobs;     /* [n_rows][n_top] or NULL   */
  uint32_t *bad_id;        /* one word or NULL          */
  size_t n_rows, vocab, row_stride, n_top;
  float inv_temp;
  void *workspace; /* NULL: the library's scratch */
  size_t workspace_bytes;
} bh_token_logprobs_args;

int bh_token_logprobs(const bh_token_logprobs_args *args, bh_stream stream);
/* Bytes of workspace that a call with these arguments needs on the current
 * device (0: none, or bad arguments). */
size_t bh_token_logprobs_workspace(const bh_token_logprobs_args *args);

#ifdef __cplusplus
}
#endif

#endif /* BONSAI_HIP_SERVE_H */
