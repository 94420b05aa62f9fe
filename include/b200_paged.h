/* C-ABI of the serving operators around the fused attention, for sm_100a (B200): rotary positions (forward and gradient),
 * appending new tokens' keys and values to a paged cache, attention of new tokens over that cache, and the handling of
 * the cache's pages.
 *
 * Plain pointers and sizes only; every function returns a tx_dot_status code (b200_dot.h) and tx_paged_last_error()
 * holds the text of this thread's last failure. Calls are asynchronous on `stream` (a cudaStream_t), allocate nothing on
 * the device and keep nothing between calls: workspaces are the caller's, so calls on several streams, from several
 * threads or in several CUDA graphs do not meet anywhere but in the per-device status word that tx_paged_check reads.
 * There is no CPU path: without an sm_100 device every compute entry point returns TXD_ERR_NO_DEVICE.
 */
#ifndef B200_PAGED_H_
#define B200_PAGED_H_

#include <stdint.h>

#include "b200_dot.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TX_ROPE_MAX_PAIRS 128

/* Rotary positions: pair i of the first `rotary_dim` columns of a head is turned by position * turns[i] / 2^64 of a full
 * turn and multiplied by `magnitude`; the other columns pass unchanged. Pairs are columns (i, i + rotary_dim / 2), or
 * (2 i, 2 i + 1) when interleaved. The products of a 64-bit position and the 64-bit fraction wrap at whole turns, so
 * angles are as exact at position 2^31 as at position 1. */
typedef struct tx_rope {
  int32_t rotary_dim; /* even, 2 .. 256, at most the head dimension */
  int32_t interleaved;
  float magnitude;
  int32_t reserved;
  uint64_t turns[TX_ROPE_MAX_PAIRS];
} tx_rope;

/* One tensor [batch, heads, tokens, head_dim] that is turned; strides in elements, head_dim contiguous. `out` may be `in`
 * (with the same strides); apart from that the two may not overlap. */
typedef struct tx_rotary_part {
  const void *in;
  void *out;
  int64_t in_stride[3];  /* batch, head, token */
  int64_t out_stride[3]; /* batch, head, token */
  int32_t heads;
  int32_t reserved;
} tx_rotary_part;

typedef struct tx_rotary_problem {
  int32_t batch, tokens, head_dim;
  int32_t dtype;               /* TXD_F16, TXD_BF16 or TXD_F32 */
  int32_t inverse;             /* 1: turn back; this is the gradient of the forward */
  int32_t positions_64;        /* positions are int64 (1) or int32 (0) */
  int64_t position_stride[2];  /* batch (0: shared), token; in elements */
  int32_t parts;               /* 1 or 2 */
  int32_t reserved;
  tx_rotary_part part[2];
} tx_rotary_problem;

TXD_API int tx_rotary(const tx_rope *rope, const tx_rotary_problem *problem, const void *positions, void *stream);

/* A paged cache as attention and append see it. Position p of sequence b lives in page table[b * table_stride + p / page_size],
 * slot p % page_size. k and v: [num_pages, page_size, kv_heads, head_dim] with head_dim contiguous and the other strides
 * free (multiples of 16 bytes). `kv_lens[b]` counts the cached tokens with the new ones; `cu_q` [batch + 1] holds where
 * each sequence's new tokens start among all new tokens (NULL: one new token for each sequence). Sequence b's new tokens
 * are its last ones: token j of q_len has position kv_lens[b] - q_len + j. cu_q starts at or above zero, never falls and ends at
 * or below the number of new tokens. Where it does not, or a length is negative or beyond the table's row, tx_paged_check
 * reports it: a token with no place in the table is not written, a negative length sees no keys, and beyond that what the
 * call gives for the sequences concerned has no meaning. Table entries that no used position needs are not read; an entry
 * outside [0, num_pages) that is needed reads as zeros, is not written, and is reported by tx_paged_check. */
typedef struct tx_paged_view {
  void *k, *v;
  int64_t k_stride[3], v_stride[3]; /* page, slot, head; in elements */
  const int32_t *table;
  int64_t table_stride;
  const int32_t *kv_lens;
  const int32_t *cu_q;
  int32_t batch, table_width, num_pages, page_size; /* page_size: 16, 32, 64, 128 or 256 */
  int32_t kv_heads, head_dim, dtype, reserved;      /* TXD_F16 or TXD_BF16 */
} tx_paged_view;

/* Writes the new tokens' k (turned, when `rope` is given) and v to their places in the cache and the turned q to q_out
 * (which may be q). q, k, v, q_out: [tokens, heads, head_dim], strides in elements (token, head). `q` may be NULL
 * (q_heads 0). Tokens behind the last sequence are left alone. */
typedef struct tx_append_problem {
  const void *q, *k, *v;
  void *q_out;
  int64_t q_stride[2], k_stride[2], v_stride[2], q_out_stride[2];
  int32_t tokens, q_heads;
} tx_append_problem;

TXD_API int tx_paged_append(const tx_paged_view *cache, const tx_rope *rope, const tx_append_problem *problem, void *stream);

/* Attention of the new tokens over their sequences' cached keys and values (which include their own: append first).
 * Query head h reads key head h / (q_heads / kv_heads). With `causal` new token j sees the keys at positions up to its own,
 * kv_lens[b] - q_len + j, and with `window` > 0 only the last `window` of them; without `causal` it sees all kv_lens[b].
 * A row that sees no key gives zeros and m = -inf (so do the first tokens where kv_lens[b] < q_len: attention allows that, an
 * append reports it). What the cache holds at positions that no row of a sequence sees never
 * matters (it may be NaN); keys and values that some row sees have to be finite.
 * `m` (may be NULL): [tokens, q_heads] fp32, running max + log2(sum) in base 2 as tx_attn_fwd returns it. Rows behind the
 * last sequence are left alone. `max_q` is the caller's bound on the new tokens of one sequence: it decides between the
 * kernels for few and for many rows, not what is computed. Results are the same from run to run, and do not depend on the
 * other sequences of the batch by more than the rounding of a different split. */
typedef struct tx_paged_attn_problem {
  const void *q; /* [tokens, q_heads, head_dim], strides in elements (token, head), multiples of 16 bytes */
  void *out;     /* the same shape and type */
  float *m;
  int64_t q_stride[2], out_stride[2];
  int32_t tokens, q_heads, max_q, causal, window;
  float sm_scale;
} tx_paged_attn_problem;

TXD_API int64_t tx_paged_attention_workspace(const tx_paged_view *cache, const tx_paged_attn_problem *problem);
TXD_API int tx_paged_attention(const tx_paged_view *cache, const tx_paged_attn_problem *problem, void *workspace,
                               int64_t workspace_bytes, void *stream);

/* The pages of a cache and who holds them. k and v: [layers, num_pages, page_bytes]; table: [rows, width], -1 where a row
 * has no page; lens[row]: its tokens; refs[page]: in how many table cells it stands (0: free). All on the device, changed
 * in stream order, without the host. What is wrong with a call is found on the device and reported by tx_paged_check: a
 * row outside the table is passed over by free, truncate and fork; a reserve with such a row, a row listed twice, a negative
 * count, no room in a row or too few free pages does nothing at all (what that means for the step behind it: tx_pages_reserve_lens).
 * `workspace`: tx_pages_workspace(state, n) bytes, 16-byte aligned, of the caller; free again when the call has run. Lists of rows,
 * counts and lengths are not parts of the state's arrays, which change while they are read. */
typedef struct tx_pages_state {
  void *k, *v;
  int64_t page_bytes; /* of one layer's k (or v), a multiple of 16 */
  int32_t *table, *lens, *refs;
  int32_t layers, num_pages, page_size, rows, width, reserved;
} tx_pages_state;

#define TX_PAGES_MAX_LIST 4096 /* rows in one reserve */

TXD_API int64_t tx_pages_workspace(const tx_pages_state *state, int32_t n);
/* Gives the pages of the listed rows back and empties the rows (a row may be listed twice). */
TXD_API int tx_pages_free(const tx_pages_state *state, const int32_t *rows, int32_t n, void *stream);
/* Cuts the listed rows to keep[i] tokens (drafted tokens that were not accepted) and gives the pages behind those back. A row
 * that is no longer than that keeps its length; one listed twice ends at the lesser; a negative keep[i] is passed over.
 * Lengths are shortened by this call, not in lens: a reserve takes the cells behind a row's length for empty. */
TXD_API int tx_pages_truncate(const tx_pages_state *state, const int32_t *rows, const int32_t *keep, int32_t n, void *stream);
/* Row dst[i] becomes what row src[i] was before the call, sharing its pages; what dst[i] held is given back. Sources may be
 * destinations too (a reordering); where a destination is listed twice the last one holds. */
TXD_API int tx_pages_fork(const tx_pages_state *state, const int32_t *dst, const int32_t *src, int32_t n, void *workspace,
                          void *stream);
/* Makes room for counts[i] more tokens in each listed row and adds them to its length: new pages are the lowest free ones,
 * in list order; a partly filled last page that other rows share is copied first (of the listed rows that share it alone,
 * the last keeps it). */
TXD_API int tx_pages_reserve(const tx_pages_state *state, const int32_t *rows, const int32_t *counts, int32_t n,
                             void *workspace, void *stream);
/* The same, and step_lens[i] (device, n values) becomes the new length of row rows[i], or TX_PAGES_REFUSED in all of them where
 * the call did nothing. What follows without the host knowing which it was takes its lengths from there, not from lens:
 * as kv_lens a refused length writes nothing to the cache and sees no key (rows of zeros), and as keep (step_lens - drafted +
 * accepted) it cuts nothing. With lens a step behind a refused reserve would take the last old tokens for its new ones. */
#define TX_PAGES_REFUSED (-(1 << 30)) /* below zero whatever numbers of tokens are added to it */
TXD_API int tx_pages_reserve_lens(const tx_pages_state *state, const int32_t *rows, const int32_t *counts, int32_t n,
                                  int32_t *step_lens, void *workspace, void *stream);
/* Moves pages so that the used ones are the lowest: with U pages in use, those at U and above go to the free ones below, in
 * order, and the table follows. */
TXD_API int tx_pages_compact(const tx_pages_state *state, void *workspace, void *stream);
/* Copies pages src[i] to dst[i] in every layer (host lists). No page may be a destination twice, or source and destination. */
TXD_API int tx_pages_copy(const tx_pages_state *state, const int32_t *src, const int32_t *dst, int32_t n, void *stream);

/* Synchronises `stream` and reports (and clears, in one step) what kernels of this header found on the device since the last
 * check. The word is the device's: a check also reports, and so takes from other threads' checks, what kernels on other
 * streams have found by then; what they find later stays for the next check. */
TXD_API int tx_paged_check(void *stream);

TXD_API uint64_t tx_paged_kernel_launches(void);
TXD_API const char *tx_paged_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* B200_PAGED_H_ */
