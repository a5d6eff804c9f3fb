/*
 * bonsai_hip_batch.h -- C ABI of the recurrent layers of many requests at once
 * and of beam search over a paged cache.
 *
 * bonsai_hip_serve.h serves many requests in one step, in the attention layers.
 * The entry points below are that step's other parts:
 *
 *   bh_conv1d_silu_ragged  a recurrent layer's causal conv + SiLU + L2 norms
 *   bh_gdn_ragged          its gated delta rule, one token or a prompt a request
 *   bh_attention_shared    bh_attention_paged of requests that share a prefix,
 *                          the prefix not read by each of them
 *   bh_beam_select         the best continuations of a group's beams
 *   bh_beam_reorder        page tables and state slots put in the new beams' order
 *   bh_kv_copy_paged       the pages of beams that went on more than once (a layer)
 *
 * The reference serves one sequence at a time and has none of these; the
 * conventions are those of bonsai_hip.h and bonsai_hip_serve.h: device pointers
 * owned by the caller, work enqueued on `stream` of the current device without
 * synchronising, a status code back, the message from bh_last_error(), f32 data.
 * Nothing depends on data the host cannot see at the call, so every entry point can
 * be captured in a HIP graph and replayed with other lengths, slots and parents.
 * No value of what lies on the device makes a kernel read or write outside the
 * buffers described.
 *
 * States in slots: a recurrent layer keeps the states of its requests in a pool of
 * slots, slot_stride floats apart.  A step reads request i's state from slot
 * src_slot[i] and leaves the new one in dst_slot[i]; the two may be the same slot.
 * src_slot[i] < 0: the request begins, with a state of zeros.  dst_slot[i] < 0: the
 * new state is not kept.  A slot past the pool is taken as below 0 and written to
 * *bad_slot where that is not NULL (the caller presets it).  A slot that a request
 * with tokens writes is no other's that has tokens, neither to read nor to write
 * (what such requests get is unspecified).  Beams go on from their parents by
 * src_slot = the parent's slot, dst_slot = a slot that no beam reads: no state moves.
 * A request without tokens reads and writes nothing, its slots stay as they were.
 *
 * Tokens of request i are q_start[i] .. q_start[i + 1] - 1, as the plan leaves
 * them; entries do not decrease (if they do, the requests' results are unspecified)
 * and are clipped to 0 .. n_tok.  Rows of no request are left as they were.
 *
 * Workspaces are as in bonsai_hip_serve.h: 16-byte aligned, of the bytes that the
 * _workspace function names; NULL takes the library's per-device scratch, and calls
 * of one entry point must then not overlap on one device.  (bh_attention_shared uses
 * the scratch of bh_attention_paged, bh_beam_select that of bh_token_logprobs.)
 */
#ifndef BONSAI_HIP_BATCH_H
#define BONSAI_HIP_BATCH_H

#include "bonsai_hip_serve.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------
 * Recurrent layers
 * ------------------------------------------------------------------------- */

/* bh_conv1d_silu for ragged requests.  Of request i's inputs x_t (rows of ch
 * channels, x_stride floats apart), preceded by the k - 1 that its slot holds:
 *   y_t[c] = silu(sum_j w[c][j] x_{t - k + 1 + j}[c])
 * and out_t = y_t, but for the first l2_dim channels (a multiple of head_dim; 0:
 * none), of which each group of head_dim is scaled by 1 / max(|group|, eps).  The
 * slot written holds the last k - 1 inputs, [ch][k - 1], oldest first.  out:
 * [n_tok][ch], not x; w: [ch][k], 1 <= k <= 64; k = 1 has no state (state NULL), and
 * no slot is bad then.  max_new is as in bh_gdn_ragged; no form depends on it here.  No
 * scratch. */
typedef struct bh_conv_ragged_args {
  const float *x, *w;
  float *state; /* [n_slots][ch][k - 1] */
  float *out;
  const int32_t *q_start;  /* [n_req + 1]      */
  const int32_t *src_slot; /* [n_req]          */
  const int32_t *dst_slot; /* [n_req]          */
  int32_t *bad_slot;       /* one word or NULL */
  size_t n_tok, n_req, ch, k, l2_dim, head_dim, n_slots, x_stride, slot_stride, max_new;
  float eps;
} bh_conv_ragged_args;

int bh_conv1d_silu_ragged(const bh_conv_ragged_args *args, bh_stream stream);

/* bh_gdn_step for ragged requests: with M = state[slot][h] (s x s, row j
 * contiguous), for each token t of a request and v-head h (q/k head h % h_k)
 *   M *= exp(gate[t][h]);  delta[j] = (v[t][h][j] - M[j].k) beta[t][h];
 *   M[j] += k delta[j];    attn[t][h][j] = (M[j].q) / sqrt(s).
 * q, k: [n_tok][h_k][s], v: [n_tok][h_v][s], a token's heads side by side, tokens
 * q_stride, k_stride, v_stride floats apart (so that they may be parts of one row,
 * as the conv leaves them); gate, beta: [n_tok][h_v]; attn: [n_tok][h_v][s].
 * max_new: no request has more tokens than this (0: n_tok); it steers how the work
 * is laid out, and a wrong one costs time only.
 * Prompts of s = 64 and 128 go by chunks of 64 tokens whose operands keep 22 bits: an
 * output is off by a few 2^-22 of |M[j]| |q| / sqrt(s), the largest of 16 rows j and of what
 * M has been in the chunk, as it has decayed by then; values of later tokens do not enter. */
typedef struct bh_gdn_ragged_args {
  const float *q, *k, *v, *gate, *beta;
  float *state; /* [n_slots][h_v][s][s] */
  float *attn;
  const int32_t *q_start;  /* [n_req + 1]      */
  const int32_t *src_slot; /* [n_req]          */
  const int32_t *dst_slot; /* [n_req]          */
  int32_t *bad_slot;       /* one word or NULL */
  size_t n_tok, n_req, h_k, h_v, s, n_slots, q_stride, k_stride, v_stride, slot_stride, max_new;
  void *workspace; /* NULL: the library's scratch */
  size_t workspace_bytes;
} bh_gdn_ragged_args;

int bh_gdn_ragged(const bh_gdn_ragged_args *args, bh_stream stream);
/* Bytes of workspace that a call with these arguments needs on the current device
 * (0: none, or bad arguments). */
size_t bh_gdn_ragged_workspace(const bh_gdn_ragged_args *args);

/* ---------------------------------------------------------------------------
 * Attention of requests that share a prefix
 * ------------------------------------------------------------------------- */

/* bh_attention_paged where groups of requests have the same keys and values at
 * their first positions, as the beams of one prompt and the users of one system
 * prompt do: results are those of bh_attention_paged on `paged` (to rounding), and
 * the first shared_len[g] positions are read once a tile of 16 to 128 (token, head)
 * rows of all requests of group g.
 *
 * Group g is the requests group_start[g] .. group_start[g + 1] - 1, and group[i]
 * is request i's (a request of group[i] outside 0 .. n_group - 1, or that does not
 * lie among those of its group, is by itself).  The shared positions are read
 * through the pages of the group's first request, whatever that one's kv_len is:
 * the first ceil(shared_len / page_size) entries of its table row are pages, and
 * the other requests' first positions are there too or hold the same.
 * shared_len[g] is clipped to 0 .. table_width * page_size.  A request that does
 * not see all of them with its first new token (kv_len - new tokens < shared_len)
 * is by itself too.  Groups do not overlap (if they do, their requests' results are
 * unspecified).
 *
 * max_group_new: no group has more new tokens than this (0: n_tok); a hint like
 * max_new.  Calls that do not run on the matrix cores run as bh_attention_paged. */
typedef struct bh_attention_shared_args {
  bh_attention_paged_args paged;
  const int32_t *group;       /* [n_req]       */
  const int32_t *group_start; /* [n_group + 1] */
  const int32_t *shared_len;  /* [n_group]     */
  size_t n_group, max_group_new;
} bh_attention_shared_args;

int bh_attention_shared(const bh_attention_shared_args *args, bh_stream stream);
/* Bytes of workspace that a call with these arguments needs on the current
 * device; what lies on the device does not enter (0: none, or bad arguments). */
size_t bh_attention_shared_workspace(const bh_attention_shared_args *args);

/* ---------------------------------------------------------------------------
 * Beam search
 * ------------------------------------------------------------------------- */

#define BH_MAX_BEAMS 32

/* A step's selection.  Row r = g * width + b of logits x (row_stride floats apart)
 * is beam b of group g, of the sum of log probabilities score[r].  With
 * z = x * inv_temp and Z = sum exp(z) of a row, its continuations have
 *   score[r] + z[token] - log Z,
 * and those of a group's beams are ordered by it, largest first, of equal ones the
 * lower row first, then the lower token.  (Compared in f64, before the score is
 * rounded to f32, and a row's own by their logits, of which -0 equals 0; rows of the
 * same bits have the same log Z.  log Z is within 4e-6, commonly 1e-7: continuations of
 * two beams of other bits that are nearer than that may change places.)  The n_best first go to parent (row r), token and
 * score_out, [n_group][n_best].
 * A beam whose score is not finite (-inf: it has ended, or not begun) and a row
 * with a NaN or +inf among its logits or with nothing above -inf have no
 * continuations, and a logit of -inf is none; where there are fewer than n_best,
 * parent is -1, token 0xffffffff and score -inf.
 * width <= BH_MAX_BEAMS, n_best <= BH_MAX_TOP and <= vocab; inv_temp is finite and
 * above 0; vocab < 2^31.  score_out may be score where n_best = width. */
typedef struct bh_beam_select_args {
  const float *x;      /* [n_group * width][row_stride] */
  const float *score;  /* [n_group * width]             */
  int32_t *parent;     /* [n_group][n_best]             */
  uint32_t *token;     /* [n_group][n_best]             */
  float *score_out;    /* [n_group][n_best]             */
  size_t n_group, width, vocab, row_stride, n_best;
  float inv_temp;
  void *workspace; /* NULL: the library's scratch */
  size_t workspace_bytes;
} bh_beam_select_args;

int bh_beam_select(const bh_beam_select_args *args, bh_stream stream);
/* Bytes of workspace that a call with these arguments needs on the current
 * device (0: none, or bad arguments). */
size_t bh_beam_select_workspace(const bh_beam_select_args *args);

/* The beams' storage in the order of the beams selected.  Beam b of group g is row
 * g * width + b of every array below, and goes on from row parent[g * parent_stride
 * + b], one of its group (a value outside the group: it has no parent).
 *
 * Pages.  The first beam of each parent, the heir, gets the parent's table row;
 * each of the others one of the rows whose beam has no children, in order, and
 * copy_from = its parent's heir: bh_kv_copy_paged then copies what it lacks.  No
 * page is taken or given back: a group's rows are to have equally many, as beams of
 * one length have, of which the shared ones stand first in all of them.  copy_from
 * is -1 for heirs and for beams without a parent.  The table is permuted in place.
 *
 * States (all three slot arrays or none): src_slot = dst_slot of the parent (its
 * own without one), which is what the parent's last step wrote, and dst_slot and
 * spare_slot change places.  Before the first selection the beams' states are in
 * dst_slot, or, where a step goes before it, in src_slot, of which spare_slot is a
 * copy; the 2 * n_group * width slots of dst_slot and spare_slot are distinct.
 *
 * No scratch.  The groups' rows of parent share no memory with an output (refused). */
typedef struct bh_beam_reorder_args {
  const int32_t *parent; /* [n_group][parent_stride], of which `width`  */
  int32_t *block_table;  /* [n_group * width][table_width]              */
  int32_t *copy_from;    /* [n_group * width]                           */
  int32_t *src_slot;     /* [n_group * width] or NULL                   */
  int32_t *dst_slot;     /* [n_group * width] or NULL                   */
  int32_t *spare_slot;   /* [n_group * width] or NULL                   */
  size_t n_group, width, parent_stride, table_width;
} bh_beam_reorder_args;

int bh_beam_reorder(const bh_beam_reorder_args *args, bh_stream stream);

/* Positions begin[i] .. end[i] - 1 of request copy_from[i] copied to request i, for
 * each i with copy_from[i] in 0 .. n_req - 1, in the pages of one layer's cache
 * (begin NULL: from 0): the shared positions before begin[i] are there already.
 * begin and end are clipped to 0 .. table_width * page_size.  A block whose page is
 * the same for both, or outside the pool for one of them, stays as it is.  A request
 * that is copied to is not copied from, and a page that is written is read by none
 * (what such pages hold is unspecified).  No scratch. */
typedef struct bh_kv_copy_args {
  bh_paged_cache cache;
  const int32_t *block_table; /* [n_req][table_width] */
  const int32_t *copy_from;   /* [n_req]              */
  const int32_t *begin;       /* [n_req] or NULL      */
  const int32_t *end;         /* [n_req]              */
  size_t n_req, table_width;
} bh_kv_copy_args;

int bh_kv_copy_paged(const bh_kv_copy_args *args, bh_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* BONSAI_HIP_BATCH_H */
