/*
 * ane_serve.h -- serving operators of libane_hip.so on caller-owned device
 * memory: a paged key/value cache held in 8 bits (append, attention, whole or
 * over selected pages, and the tables of its pages), the controls on logits
 * before the next token is chosen, and beam search.  No counterpart in the
 * reference, which evaluates whole windows only (ane/engine.go:954-1038); the
 * model they serve is that of ane_hip.h's decoder, built from the reference's
 * RoPE (ane/train_util.go:183-224) and causal softmax attention
 * (ane/common.go:61-89).
 *
 * Every call is asynchronous on `stream` (a hipStream_t; NULL: the default
 * stream), allocates nothing, keeps no state and may be captured into a HIP
 * graph.  Calls may run at once on several streams and threads as long as
 * they do not write the same memory.  Arguments that the host can see are
 * checked (ANE_ERR_ARG, message in ane_op_last_error()); device-side indexes
 * are checked by the kernels, as each call says, so that no index leads
 * outside the buffers.  `device` is the GPU that holds the buffers; it need
 * not be the current one.
 */
#ifndef ANE_SERVE_H
#define ANE_SERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the cache --------------------------------------------------------------
 * Pages of page_tokens tokens.  Keys and values are e4m3 codes (4 bits of
 * significand, +-448, subnormals down to 2^-9, 0x7f NaN) with one exponent for
 * each page and key/value head: value = code * 2^exp, exp in [-15, 8].  Every
 * value held is then an fp16 number exactly.
 *   k      [pages][kv_heads][page_tokens][head_dim]
 *   v      [pages][kv_heads][page_tokens/16][4][16][head_dim/16][4]: token s
 *          and dimension d of a page at [s/16][s%16/4][d%16][d/16][s%4] (the
 *          order in which the matrix cores take it)
 *   k_exp, v_exp [pages][kv_heads]
 * page_tokens: 16, 32, 64, 128 or 256; head_dim: 64 or 128; kv_heads at most
 * 1024.  k and v are 16-byte aligned.  Pages that no call has written may hold
 * anything, exponents too. */
typedef struct ane_kv8_cache {
  void *k, *v;
  int8_t *k_exp, *v_exp;
  int32_t pages, page_tokens, kv_heads, head_dim;
  int32_t device;
} ane_kv8_cache;

/* The new tokens of a call: nseq sequences, sequence i with rows
 * offsets[i] .. offsets[i+1]-1 of the call's [rows] tensors, the first of them
 * at position start[i] (the tokens it holds already); position p is row
 * p % page_tokens of page table[i][p / page_tokens].  All on the device.
 *
 * At most 65536 sequences, 2^30 rows and 2^30 tokens of a table's row.
 * offsets rise from 0 to at most `rows`; a sequence may have no new rows.
 * What lies outside is not followed: offsets are taken within [0, rows],
 * positions from table_pages * page_tokens on are not taken (their rows belong
 * to no sequence), and a page id outside [0, pages) is a page that is not
 * there: nothing is written to it and its keys do not take part.  Rows of no
 * sequence are left as they are.
 * max_len (tokens of the longest sequence, new ones included) and max_new (its
 * new tokens) size the launches; wrong values cost time, not correctness (an
 * attention's sums are added in as many parts as they make: last bits may
 * differ).  0: not known. */
typedef struct ane_kv8_batch {
  const int32_t *table;   /* [nseq][table_stride], table_pages of each row used */
  const int32_t *start;   /* [nseq] */
  const int32_t *offsets; /* [nseq + 1] */
  int32_t table_stride, table_pages;
  int32_t nseq, rows;
  int32_t max_len, max_new;
} ane_kv8_batch;

/* Rotates the new queries and keys by their positions (pairs (2c, 2c+1):
 * x[2c] cos - x[2c+1] sin, x[2c+1] cos + x[2c] sin, in fp32), writes the
 * queries as fp16 and appends keys and values to the cache.
 *
 * Per page, head and side (K after the rotation, V): the exponent is the
 * smallest in [-15, 8] with max |x| <= 448 * 2^exp over the call's rows of the
 * page (infinities count, and are held, as +-65504 would be; NaN does not
 * count and stays NaN).  Where the page holds rows from before (its row 0 is
 * not this call's), the exponent is at least the old one, and if it rises, the
 * rows before are rounded again from their codes.  Codes are rounded to
 * nearest, ties to even; at exponent 8 they end at +-240, fp16's range.
 * A page may get rows of one sequence only in a call, from one place of its
 * table.
 *
 * q, k, v, q_out: fp16, [rows][heads or kv_heads][head_dim] with element
 * strides between rows and heads; 16-byte aligned, strides multiples of 8.
 * q_out may be q itself (same strides), and shares no memory with q, k and v
 * otherwise.  heads = 0: keys and values only; at most 32768.
 * cos, sin: fp32 [positions][head_dim / 2], 16-byte aligned, positions >=
 * table_pages * page_tokens. */
typedef struct ane_kv8_append_args {
  const uint16_t *q, *k, *v;
  uint16_t *q_out;
  const float *cos, *sin;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, q_out_row, q_out_head;
  int32_t heads, positions;
} ane_kv8_append_args;

int ane_kv8_append(const ane_kv8_cache *cache, const ane_kv8_batch *batch, const ane_kv8_append_args *args,
                   void *stream);

/* Causal attention of the batch's new tokens over the cache, the tokens
 * themselves included (append comes first): the row at position p, query head
 * h, attends to positions 0..p of key/value head h / (heads / kv_heads):
 * out = sum_j softmax_j(scale q . k_j) v_j.  A row without any key, or none of
 * whose scores is above -inf, gives zeros; NaN in a key or value reaches the
 * rows that attend to it and no other.
 *
 * q, out: fp16 [rows][heads][head_dim], 16-byte aligned, strides multiples of
 * 8; out may be q itself (same strides), and shares no memory with it
 * otherwise.  scale > 0, and finite times log2(e) in fp32; heads / kv_heads at
 * most 32.
 * ws: ane_kv8_attend_workspace() bytes of device memory, 16-byte aligned (NULL
 * when that is 0); its contents need not be set, and calls that may overlap
 * need one each. */
typedef struct ane_kv8_attend_args {
  const uint16_t *q;
  uint16_t *out;
  int64_t q_row, q_head, out_row, out_head;
  int32_t heads;
  float scale;
  void *ws;
  int64_t ws_bytes;
} ane_kv8_attend_args;

/* Bytes of workspace for this batch (its sizes count, its device arrays are
 * not looked at), or a negative ANE_ERR_*. */
int64_t ane_kv8_attend_workspace(const ane_kv8_cache *cache, const ane_kv8_batch *batch, int32_t heads);
int ane_kv8_attend(const ane_kv8_cache *cache, const ane_kv8_batch *batch, const ane_kv8_attend_args *args,
                   void *stream);

/* ---- controls on logits -------------------------------------------------------
 * Per row r and token v, with a = the count of v among the row's history[0 ..
 * lengths[r]) and o = its count in history[prompts[r] .. lengths[r]), in fp32,
 * each step rounded:
 *   a > 0: x = x > 0 ? x / repetition[r] : x * repetition[r]
 *   o > 0: x = x - frequency[r] * o, then x = x - presence[r]
 *   x = x + bias[r][v];  mask bit v of row r clear: x = -inf
 * and tokens[r] = the lowest index of the row's largest value (NaN is never
 * chosen; ANE_NO_TOKEN where nothing is above -inf).
 *
 * logits, out: fp32 [rows][vocab] with row strides; out may be logits itself
 * (same stride) or NULL (tokens only), and shares no memory with it otherwise
 * (rows of one may lie between the other's).  history: uint16 [rows][history_row],
 * ids from vocab on are passed over; lengths are taken within [0,
 * history_max], prompts within [0, lengths[r]] (NULL: 0).  repetition,
 * frequency, presence: fp32 [rows] or NULL (1, 0, 0); they need a history (NULL
 * with lengths and history_max = 0: an empty one).  bias: fp32, row stride
 * bias_row (0: one row for all), or NULL.  mask: uint32 words, bit v % 32 of
 * word v / 32, row stride mask_row (0: one for all), or NULL.  tokens: int32
 * [rows] or NULL.  vocab 1..65535, rows at most 65535.  ws as
 * above. */
enum { ANE_NO_TOKEN = 65535 };
typedef struct ane_logits_args {
  const float *logits;
  float *out;
  const uint16_t *history;
  const int32_t *lengths, *prompts;
  const float *repetition, *frequency, *presence, *bias;
  const uint32_t *mask;
  int32_t *tokens;
  int64_t logits_row, out_row, history_row, bias_row, mask_row;
  int32_t rows, vocab, history_max, device;
  void *ws;
  int64_t ws_bytes;
} ane_logits_args;

int64_t ane_control_logits_workspace(int32_t rows, int32_t vocab);
int ane_control_logits(const ane_logits_args *args, void *stream);

/* ---- beam search ---------------------------------------------------------------
 * One step of `requests` searches with `beams` beams each; row r = request *
 * beams + beam.  With x = logits (fp32, or fp16 where half is set) and NaN as
 * -inf:
 *   lse[r] = log sum_v exp(x[r][v])
 *   s(r, v) = scores[r] + (x[r][v] - lse[r]),  key(r, v) = weights[r] * s(r, v)
 * and the request's `beams` candidates of the largest key become its next
 * beams, the best first, equal keys in the order of beam, then token.  A beam
 * that is finished has one candidate, itself: (r, eos) with s = scores[r].  No
 * candidate: keys that are -inf or NaN, rows with scores -inf or NaN, weights
 * that are not above 0, or +inf among their logits.
 * s and keys are 64-bit; lse is the sum of fp32 exponentials, a row's off by at
 * most (19 + 3 sum_v p(v) (max x - x(v))) 2^-24 with p = softmax(x), 2e-6 for
 * logits of normal distribution.  Candidates of two beams whose keys lie closer
 * together than that (times their weights) may change places.
 *   tokens, parents   the candidate's v and r (the row in the call, not within
 *                     the request); ANE_NO_TOKEN and -1 where there are not
 *                     enough candidates
 *   scores_out        s, rounded to fp32 (-inf); may be scores
 *   finished_out      1 where the parent was finished or the token is eos, else
 *                     0 (also where there is no candidate); may be finished
 *   history, lengths  move with their beams, in place: a row gets its parent's
 *                     first lengths[parent] ids, and behind them the token if
 *                     the parent was not finished and there is room; ids from
 *                     the new length on stay as they are.  No candidate: length
 *                     0, ids as they are.  Lengths are taken within [0,
 *                     history_max].
 * weights NULL: 1.  finished NULL with finished_out NULL and eos -1: beams do
 * not finish.  history and lengths NULL: no histories
 * (history NULL, history_max 0, with lengths: empty ones); history_max at most 2^30.
 * beams 1..32, vocab 1..65535, at most 65535 rows.  logits: row stride
 * logits_row; history: uint16, row stride history_row.  Outputs share no memory
 * with each other or with inputs but where said.  ws as above. */
typedef struct ane_beam_args {
  const void *logits;
  const float *scores, *weights;
  const uint8_t *finished;
  int32_t *tokens, *parents;
  float *scores_out;
  uint8_t *finished_out;
  uint16_t *history;
  int32_t *lengths;
  int64_t logits_row, history_row;
  int32_t requests, beams, vocab, eos, history_max, half, device;
  void *ws;
  int64_t ws_bytes;
} ane_beam_args;

int64_t ane_beam_select_workspace(int32_t requests, int32_t beams, int32_t vocab, int32_t half);
int ane_beam_select(const ane_beam_args *args, void *stream);

/* ---- bounds on the keys of a page ------------------------------------------------
 * For each page and key/value head, of the keys it holds: unit, the smallest
 * exponent e >= -30 at which every |k| <= 127 * 2^e, and box [2][head_dim], the
 * largest (first) and smallest key of each dimension in that unit, rounded
 * outwards.  NaN does not count; a dimension without a number has 0 and 0.
 * They are as the last update left them: a fork that cuts a sequence off, or
 * copies a part of a page, leaves those of all the keys that the page (the one
 * copied from) held, no smaller than its own keys', until a token comes to it. */
typedef struct ane_kv8_bounds {
  int8_t *box;  /* [pages][kv_heads][2][head_dim], 16-byte aligned */
  int8_t *unit; /* [pages][kv_heads] */
} ane_kv8_bounds;

/* The bounds of the pages that the batch's new tokens went to (append comes
 * first), of all the sequence's tokens in them. */
int ane_kv8_bound(const ane_kv8_cache *cache, const ane_kv8_bounds *bounds, const ane_kv8_batch *batch, void *stream);

/* For each row of the batch and key/value head, the `count` pages of the row's
 * sequence that its queries may match best.  A query becomes whole numbers z of
 * a power of two 2^f, the smallest f >= -30 with |q| <= 127 * 2^f (to nearest,
 * ties to even; infinities as 65504, NaN as 0); with the page's box and unit
 *   score(page) = max over the group's query heads of
 *                 2^(f + unit) * sum_d z_d * (z_d > 0 ? largest_d : smallest_d)
 * which is exact in fp32, and no smaller than q . k of any key of the page but
 * for the rounding of q.  The first `first` pages and the last `recent` ones up
 * to the row's own position are always taken, then the largest scores, equal
 * ones from the lower page.  Pages that are not there are not taken.
 * A row's own page has bounds of all the call's tokens in it, later ones than the
 * row's too.  With recent >= 1 it is taken whatever they are, and a chunk's rows
 * choose as they would token by token over the same codes; with recent 0 they may
 * choose their own page for the sake of keys that they do not attend to.
 *
 * blocks: int32 [rows][kv_heads][count], the pages' places in the sequence's
 * table, rising, then -1.  Rows of no sequence are left as they are.
 * q as in ane_kv8_attend.  count 1..65536, first and recent >= 0 and together
 * at most count.  ws as above. */
typedef struct ane_kv8_select_args {
  const uint16_t *q;
  int32_t *blocks;
  int64_t q_row, q_head;
  int32_t heads, count, first, recent;
  void *ws;
  int64_t ws_bytes;
} ane_kv8_select_args;

int64_t ane_kv8_select_workspace(const ane_kv8_cache *cache, const ane_kv8_batch *batch, int32_t heads, int32_t count);
int ane_kv8_select(const ane_kv8_cache *cache, const ane_kv8_bounds *bounds, const ane_kv8_batch *batch,
                   const ane_kv8_select_args *args, void *stream);

/* ane_kv8_attend over the pages that `blocks` (as above) names for each row and
 * key/value head, alone: the row at position p attends to the keys at positions
 * 0..p in them.  Places outside [0, table_pages) and pages that are not there
 * take no part; the order of the places does not matter, and a page named twice
 * counts twice. */
int64_t ane_kv8_attend_blocks_workspace(const ane_kv8_cache *cache, const ane_kv8_batch *batch, int32_t heads,
                                        int32_t count);
int ane_kv8_attend_blocks(const ane_kv8_cache *cache, const ane_kv8_batch *batch, const ane_kv8_attend_args *args,
                          const int32_t *blocks, int32_t count, void *stream);

/* ---- the tables of the pages -----------------------------------------------------
 * A pool of pages that the caches of all layers share: page id i is page i of
 * every layer (equal sizes, one device).  refs[i]: how many entries of tables
 * name it; not above 0: free.  bounds: NULL, or one per layer, which then move
 * with their pages (pointers NULL: that layer has none). */
typedef struct ane_kv8_pool {
  const ane_kv8_cache *layers;
  const ane_kv8_bounds *bounds;
  int32_t *refs; /* [pages] */
  int32_t nlayers; /* 1..1024 */
} ane_kv8_pool;

/* Brings the table of nseq sequences (at most 65536, and 2^30 entries and 2^30
 * tokens of a row, here and below) to their next step, with `new` tokens each
 * to come (news[i], or new_tokens where news is NULL; taken within [0, table's
 * room]):
 *  1. sequence i goes on from parents[i] (NULL: itself; outside [0, nseq): it
 *     ends): start[i] = start[parents[i]] (0), taken within [0, table's room],
 *     and its row is the parent's up to the page of its last token, -1 behind.
 *     Smaller starts so cut sequences off, and 0 frees them.  refs follow.
 *  2. A sequence with new tokens writes into the page of its last one, if that
 *     is not full.  Where others hold that page too, it gets a page of its own,
 *     with the tokens held so far (in all layers); the lowest sequence keeps the
 *     page itself if all that hold it (by refs) are such sequences of this call.
 *     A page that is not there stays so.
 *  3. Positions of the new tokens without a page get one.
 * The pages for 2 and 3 are the lowest free ones, in the order of sequence and
 * position.  Where none is left, the entry is -1 (nothing is written there, and
 * its tokens take no part in attention); *missing = the entries that have no
 * page for such tokens, those of 2 that stay without one included.
 *
 * Copies take whole 16-token units; what a page holds behind them stays.
 * A table names a page at most once per sequence. */
typedef struct ane_kv8_fork_args {
  int32_t *table, *start;
  const int32_t *parents, *news;
  int32_t *missing; /* 1 */
  int32_t table_stride, table_pages, nseq, new_tokens;
  void *ws;
  int64_t ws_bytes;
} ane_kv8_fork_args;

int64_t ane_kv8_fork_workspace(const ane_kv8_pool *pool, int32_t nseq, int32_t table_pages);
int ane_kv8_fork(const ane_kv8_pool *pool, const ane_kv8_fork_args *args, void *stream);

/* Brings the U pages that are held (refs above 0) to the ids 0..U-1: those at U
 * and beyond go, in order, to the free ones below U, in order.  moved[i] = where
 * page i is now, -1 if it was free; refs follow, and so do the entries of the
 * table (others outside [0, pages) stay; ones that name a free page become -1).
 * nseq = 0: no table; further tables are the caller's, by `moved`. */
typedef struct ane_kv8_compact_args {
  int32_t *table;
  int32_t *moved; /* [pages] */
  int32_t table_stride, table_pages, nseq;
  void *ws;
  int64_t ws_bytes;
} ane_kv8_compact_args;

int64_t ane_kv8_compact_workspace(const ane_kv8_pool *pool);
int ane_kv8_compact(const ane_kv8_pool *pool, const ane_kv8_compact_args *args, void *stream);

/* Copies the pages src[i] of `from` to the pages dst[i] of `into` (the same pool
 * or another of the same layers, page_tokens, kv_heads and head_dim; pages may
 * differ), i < n: the 16-token units that hold their first tokens[i] tokens
 * (NULL: all; taken within [0, page_tokens]; 0: nothing), exponents and, where
 * both have them, bounds.  n at most 2^24.  Ids outside the pools are passed
 * over.  A page that is written twice, or read and written, holds either; refs
 * are not looked at. */
typedef struct ane_kv8_copy_args {
  const int32_t *src, *dst, *tokens;
  int32_t n;
} ane_kv8_copy_args;

int ane_kv8_copy(const ane_kv8_pool *from, const ane_kv8_pool *into, const ane_kv8_copy_args *args, void *stream);

/* ---- for tests -----------------------------------------------------------------
 * The rows, positions and pages that a work item of the cache kernels takes,
 * by the kernels' own index arithmetic on host arrays: item `item` of tiles of
 * `tile_tokens` tokens (pages = 0), of such tiles with the longest contexts
 * first, at most 64 sequences (2), or of the pages that rows go to (1: as
 * many items as pages may be, 3: an item a row).  out receives {sequence,
 * first row, rows taken, first position, page (-1: not there; 1 and 3 only),
 * items of the batch}; rows taken = 0: the item is empty.  Returns ANE_OK.
 * No GPU is used. */
int ane_debug_kv8_item(const ane_kv8_cache *cache, const ane_kv8_batch *batch, int32_t tile_tokens, int32_t pages,
                       int64_t item, int32_t *out);

/* Whether two tensors [rows][heads][width] share memory, as the operators ask
 * before they refuse an output that overlaps an input: each given as {address,
 * rows, stride of rows, heads, stride of heads, width}, in bytes.  No GPU is
 * used. */
int ane_debug_share_memory(const int64_t *a, const int64_t *b);

/* The form that a call of these sizes takes, by the operators' own rules, so that
 * a test that is to reach a form can ask for it.  No GPU is used, no address
 * followed; ANE_OK, or what the call itself would refuse.
 * select: {tiles of 16 query rows, tokens a block, waves a block, 1: the choice
 *   has a launch of its own, scores that LDS holds}
 * attend, count 0: all pages, else a list of so many: {tiles of 16 rows, tokens
 *   a tile, waves that share its keys, parts of the keys at most, 1: the longest
 *   contexts first, places that a union of lists has masks of (0: a list a
 *   tile)}
 * copy, also of so many pages that a compaction moves: {1: past the caches;
 *   sides (keys or values of a layer) a block of ane_kv8_copy takes}; of the
 *   first 32 layers
 * beam: {loads of a wave of the first launch, threads of the second one, 1:
 *   histories have a launch of their own} */
int ane_debug_kv8_select_form(const ane_kv8_cache *cache, const ane_kv8_batch *batch, int32_t heads, int32_t *out);
int ane_debug_kv8_attend_form(const ane_kv8_cache *cache, const ane_kv8_batch *batch, int32_t heads, int32_t count,
                              int32_t *out);
int ane_debug_kv8_copy_form(const ane_kv8_pool *pool, int32_t pages, int32_t *out);
int ane_debug_beam_form(int32_t requests, int32_t beams, int32_t vocab, int32_t half, int32_t history_max,
                        int32_t *out);

#ifdef __cplusplus
}
#endif
#endif
