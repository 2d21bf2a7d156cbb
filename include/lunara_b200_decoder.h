/*
 * lunara_b200_decoder.h -- decoder operators of the kernel library: rotary
 * positions, per-head query/key norms with the rotation in the same pass, a
 * paged key/value cache (append and read), and attention over that cache.
 *
 * lunara_b200.h replaces the reference's launchers one for one; the reference
 * has no counterpart of these, so they carry a prefix of their own. The
 * conventions are those of lunara_b200.h: device pointers owned by the caller,
 * work enqueued on `stream` in the current device context, a lunara_status as
 * return value, messages from lunara_last_error_string(), device errors from
 * lunara_device_error(). Strides are in elements; every innermost (head
 * dimension) stride is 1.
 *
 * The argument structs hold 8-byte fields only, so their layout is the same in
 * every binding.
 *
 * Device error codes: 0x501 a position outside the rotary table, 0x502 a page
 * number outside the cache, 0x503 a position outside the page table, 0x504 a
 * bounded wait of the attention ran out.
 */
#ifndef LUNARA_B200_DECODER_H
#define LUNARA_B200_DECODER_H

#include <stdint.h>

#include "lunara_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache element kind: a lunara_dtype, or 4-bit e2m1 codes (two to a byte, the
 * even element in the low nibble) with one e4m3 scale byte per 16 elements. */
#define LUNARAD_KIND_E2M1 16

/* Or-ed into `dtype` of lunarad_kv_append, lunarad_kv_read and
 * lunarad_paged_attention: output rows of tokens that belong to no sequence are
 * zeroed instead of left alone (for outputs in fresh memory). Refused for tokens
 * without any sequence (batch 0), where no kernel runs. */
#define LUNARAD_ZERO_REST 0x100

/* Pairs that are turned together: (i, i + rot/2) or (2i, 2i + 1). */
typedef enum lunarad_rotary_layout {
  LUNARAD_ROTARY_HALF = 0,
  LUNARAD_ROTARY_INTERLEAVED = 1
} lunarad_rotary_layout;

/* Rotary table: float32 [positions, rot/2, 2] of (cos, sin), contiguous,
 * 16-byte aligned. Each pair (a, b) becomes (a cos - b sin, b cos + a sin);
 * elements from `rot` on pass through. `rot` is even; rot = 0 (table NULL)
 * rotates nothing. */
typedef struct lunarad_rotary_table {
  const float* table;
  int64_t positions;
  int64_t rot;
  int64_t layout;  /* lunarad_rotary_layout */
} lunarad_rotary_table;

/* A [batch, heads, seq, dim] view: element strides of batch, head and seq. */
typedef struct lunarad_view {
  const void* data;
  int64_t batch_stride, head_stride, seq_stride;
} lunarad_view;

/* Rotate X [batch, heads, seq, dim] into Y (Y may be X). positions
 * [batch, seq] int32 or int64 (position_bytes 4 or 8), batch stride 0 when all
 * sequences share them. inverse != 0 turns by the negative angle (the
 * transpose: the gradient of the rotation). A position outside the table
 * records 0x501 and its row is zero-filled. */
typedef struct lunarad_rotary_args {
  lunarad_view x, y;
  const void* positions;
  int64_t position_bytes, position_batch_stride;
  lunarad_rotary_table rotary;
  int64_t batch, heads, seq, dim;
  int64_t inverse;
  int64_t dtype;
} lunarad_rotary_args;
int lunarad_rotary(const lunarad_rotary_args* args, void* stream);

/* Q and K normalised head by head, y = x / sqrt(mean(x^2) + eps) * weight over
 * the head dimension in fp32, then rotated, rounded once; one launch. Weights
 * [dim] in the tensors' dtype or NULL (ones). Outputs may be the inputs. */
typedef struct lunarad_qk_norm_rotary_args {
  lunarad_view q, k, q_out, k_out;
  const void* q_weight;
  const void* k_weight;
  const void* positions;
  int64_t position_bytes, position_batch_stride;
  lunarad_rotary_table rotary;
  int64_t batch, q_heads, k_heads, seq, dim;
  int64_t dtype;
  double eps;
} lunarad_qk_norm_rotary_args;
int lunarad_qk_norm_rotary(const lunarad_qk_norm_rotary_args* args, void* stream);

/* Paged cache: k and v [num_pages, kv_heads, page_size, dim] with free page
 * and head strides and contiguous [page_size, dim] inside; for e2m1 the codes
 * are bytes [.., page_size, dim/2] and the scales [.., page_size, dim/16], both
 * with strides in bytes, and a stored value is code * (scale * gain). */
typedef struct lunarad_cache {
  void* k;
  void* v;
  void* k_scales;
  void* v_scales;
  int64_t k_page_stride, k_head_stride, v_page_stride, v_head_stride;
  int64_t ks_page_stride, ks_head_stride, vs_page_stride, vs_head_stride;
  int64_t num_pages, kv_heads, page_size, dim;
  int64_t kind;  /* lunara_dtype or LUNARAD_KIND_E2M1 */
  double k_gain, v_gain;
} lunarad_cache;

/* Ragged sequences: tokens of all sequences stand one behind the other; those
 * of sequence b are seq_starts[b] .. seq_starts[b + 1] - 1 and are the last
 * ones of its seq_lens[b] positions. Position p of sequence b lies in page
 * page_table[b][p / page_size], slot p % page_size. A token with a negative
 * position (seq_lens[b] below its number of tokens) is padding; tokens before
 * seq_starts[0] and from seq_starts[batch] on belong to no sequence, and their
 * rows are left alone unless LUNARAD_ZERO_REST is given. */
typedef struct lunarad_sequences {
  const int32_t* page_table;  /* [batch, max_pages], row stride table_stride */
  const int32_t* seq_starts;  /* [batch + 1] */
  const int32_t* seq_lens;    /* [batch] */
  int64_t table_stride, max_pages, batch, tokens;
} lunarad_sequences;

/* Write K [tokens, kv_heads, dim] (rotated at its position when a table is
 * given) and V to their slots, and with q_heads > 0 rotate Q [tokens, q_heads,
 * dim] into q_out (which may be Q). Views use head_stride and seq_stride (the
 * token stride); batch_stride is ignored. Into an e2m1 cache K (rotated) and V
 * are multiplied by fp32(1 / gain), each 16 elements get the scale e4m3(amax / 6)
 * (saturating at 448; NaN when an element is NaN), and each element the
 * nearest e2m1 value of element / scale (ties to even, saturating at 6; zeros
 * where the scale is zero); the fp32 arithmetic is uncontracted, one IEEE
 * rounding per operation, so that codes do not depend on the compiler.
 * Padding tokens write nothing and their q_out row is zero. A position
 * outside the table (0x501) or the page table (0x503) and a page outside the
 * cache (0x502) are recorded and treated as padding. Two tokens of one call
 * must not share a slot. */
typedef struct lunarad_kv_append_args {
  lunarad_view k, v, q, q_out;
  const lunarad_cache* cache;
  lunarad_sequences seqs;
  lunarad_rotary_table rotary;
  int64_t q_heads;
  int64_t dtype;  /* of k, v, q, q_out; | LUNARAD_ZERO_REST for q_out */
} lunarad_kv_append_args;
int lunarad_kv_append(const lunarad_kv_append_args* args, void* stream);

/* Read cached keys and values back: k_out, v_out [tokens, kv_heads, dim]
 * contiguous, in the cache's dtype (any lunara_dtype for e2m1). Rows that are
 * padding or lie outside the tables (0x502, 0x503) are zero. */
typedef struct lunarad_kv_read_args {
  void* k_out;
  void* v_out;
  const lunarad_cache* cache;
  lunarad_sequences seqs;
  int64_t dtype;  /* | LUNARAD_ZERO_REST */
} lunarad_kv_read_args;
int lunarad_kv_read(const lunarad_kv_read_args* args, void* stream);

/* O = softmax(Q K^T * scale) V over the cached keys: query token t at position
 * p sees the keys 0..p of its sequence (with window > 0 the last `window` of
 * them). Q and O [tokens, q_heads, dim] (head_stride, seq_stride); query head h
 * reads key head h / (q_heads / kv_heads). fp32 softmax and sums, one rounding
 * of O (16-bit products round the probabilities to the query dtype as
 * well; with an e2m1 cache the products are f16; with many query rows a quarter
 * of the exponentials are off by up to 7.5e-5). A row that sees no key, or whose
 * scores are all -inf, is zero; one with a score of +inf or NaN is NaN. The sums
 * of probabilities times values, before the division by theirs, have to be fp32
 * numbers. Finite values that a row does not see have no influence on it. What
 * the cache holds behind a sequence's end, in other pages and outside every
 * row's window has no influence, NaN included. A value (not a key) that is not
 * finite and that only some of the call's tokens of a sequence see may also
 * reach those that do not. Keys of a page outside the cache (0x502) are left
 * out, and a length outside the page table (0x503) is cut. O may be Q.
 * scale, times the keys' gain of an e2m1 cache and log2(e), is a finite fp32 number.
 * max_q_len: the longest sequence's number of tokens if known (0 = unknown);
 * it only steers the choice of kernels.
 * workspace: device memory of lunarad_paged_attention_workspace() bytes or
 * more (NULL when that is 0), 16-byte aligned, in use until the call's work is
 * done; calls that may run at the same time need one each. Its contents need
 * no preparation. */
typedef struct lunarad_paged_attention_args {
  lunarad_view q, o;
  const lunarad_cache* cache;
  lunarad_sequences seqs;
  int64_t q_heads;
  int64_t window;
  int64_t max_q_len;
  int64_t dtype;  /* | LUNARAD_ZERO_REST */
  double scale;
} lunarad_paged_attention_args;
int lunarad_paged_attention(const lunarad_paged_attention_args* args, void* workspace, int64_t workspace_bytes,
                            void* stream);

/* Workspace bytes that lunarad_paged_attention needs for these arguments on
 * `device`, or -lunara_status. */
int64_t lunarad_paged_attention_workspace(const lunarad_paged_attention_args* args, int device);

#ifdef __cplusplus
}
#endif

#endif /* LUNARA_B200_DECODER_H */
