/*
 * ane_serve.h -- serving operators of libane_hip.so on caller-owned device
 * memory: a paged key/value cache held in 8 bits (append, attention), and the
 * controls on logits before the next token is chosen.  No counterpart in the
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

#ifdef __cplusplus
}
#endif
#endif
