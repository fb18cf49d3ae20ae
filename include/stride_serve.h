/* C ABI of the serving operators beside the tensor-core path of libstride_tc.so
 * (MI355X, gfx950): attention over long or bounded contexts, a pool of KV pages that
 * sequences share, and logit processing. The reference has no counterpart; layouts and
 * conventions are those of stride_tc.h: x tiles, logits tiles, the paged KV arena
 * [page][layer][K|V][group][token][dim], launches on `stream` alone (attention one to three of
 * them, fork and copy two, compact three, the others one), errors as return codes with
 * stride_tc_last_error().
 *
 * Nothing here allocates, synchronizes or keeps state: workspaces are the caller's, every
 * launch can be captured in a HIP graph, and each takes its arguments from device memory
 * when it runs, so a replay sees the values of its time. Calls that share a workspace, a
 * pool or token counts are ordered by the caller (one stream, or events), captured graphs
 * among them. Device arrays hold what the caller put there: where a kernel meets an index
 * outside its range it leaves memory alone, as said at each call.
 *
 * Batch invariance: a row's result depends on its own sequence, position and arguments
 * only, whatever the other rows, their order, the placement of pages or the form that a
 * call takes.
 */
#ifndef STRIDE_SERVE_H
#define STRIDE_SERVE_H

#include "stride_tc.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of new rows over the paged bf16 cache, grouped queries. Row j of sequence
 * row_slot[j] at row_pos[j] = p sees position t if t <= p and (window <= 0, or p - t <
 * window, or t < sinks): the last `window` positions and the first `sinks` ones.
 *   out[h] = sum_t w_t V[t],  w = softmax over the visible t of scale * (q[h] . K[t])
 * Weights are rounded to bf16 before they meet V (and their sum is that of the rounded ones),
 * queries to 16 bits, sums are fp32: where stride_tc_attention, which keeps both in fp32, serves
 * the same rows, the two agree to the weights' rounding, not bit for bit.
 * A row that sees nothing (p < 0, as padding rows of a captured batch may have it here, or
 * row_slot[j] < 0) gets zeros, and so does one whose visible scores are all -inf.
 * (stride_tc_qkv has no such rows: padding needs a slot with a page of its own there.) What
 * lies in masked places, NaN and infinities among it, has no influence; what is visible acts
 * as in the formula. A query that is not finite makes its head NaN. Pages wholly outside what
 * any row sees are never read, so their table entries may be anything; a visible position must
 * be held, and one whose entry is negative reads as zeros; slots and entries that are not
 * negative have to be rows of the table and pages of the arena. row_pos is taken as at most
 * max_blocks * page tokens - 1, and 64 * max_pages - 1. Lanes of the last tile behind `rows`
 * are left alone.
 */
typedef struct StrideWindowAttentionParams {
  StrideLanes l;
  const float* q;   /* [row][n_kv * n_q][head_dim] fp32 */
  int64_t q_stride; /* floats from one row to the next, a multiple of 4 */
  uint16_t* out;    /* bf16 x tiles [lt][ct][16][16], out_cols columns */
  StrideKvRef kv;   /* any power-of-two page of 8 tokens or more, a head's part of it up to 2^31 elements */
  const int32_t* row_slot;
  const int32_t* row_pos;
  float* scratch;         /* stride_serve_window_attention_scratch() floats, 16-byte aligned */
  int64_t scratch_floats; /* what `scratch` holds */
  int32_t out_cols;       /* multiple of 16 */
  int32_t max_pages;      /* no row lies beyond position 64 * max_pages - 1 */
  int32_t layer;
  int32_t n_kv;
  int32_t n_q;      /* query heads per KV head, 1 .. 16 */
  int32_t head_dim; /* 32, 64 or 128 */
  int32_t window;   /* <= 0: every position up to the row's own */
  int32_t sinks;    /* >= 0 */
  int32_t runs;     /* a hint that never changes results: at most so many neighbouring rows are
                       of one sequence (1: decode), 0: not known */
  float scale;
} StrideWindowAttentionParams;

int stride_serve_window_attention(const StrideWindowAttentionParams* p, void* stream);

/* Floats of scratch that the call wants (0: none), from every field but the pointers;
 * -1 where the call would be refused. What it says for runs = 0 serves calls with any hint, for
 * another hint calls with that hint. Its contents need no preparation. */
int64_t stride_serve_window_attention_scratch(const StrideWindowAttentionParams* p);

/* A pool of KV pages. table[slot][i] is the page that holds tokens i * page_tokens .. of a
 * sequence, or -1; refs[page] counts the table entries that hold it, and bit page % 32 of
 * free_bits[page / 32] is set where refs is 0. Pages are taken lowest number first, by
 * ascending (item, table index), so that a call's outcome is fixed. Items are device
 * arrays of `n` int32; a slot may come up once in a call as the one to be changed. `kv`
 * carries the table, which these calls write. A page has a power of two of tokens, a head's
 * part of it at most 2^30 bytes.
 *
 * A call whose items break a rule, or that wants more pages than are free, changes nothing
 * and sets a bit of errors[0], which stays set until the caller clears it. Launches that were
 * on their way behind it may meet entries below 0: stride_tc_qkv does not keep such rows.
 */
#define STRIDE_KV_BAD_ITEM 1     /* slot, range, length or page outside its bounds */
#define STRIDE_KV_TWICE 2        /* a slot or page to be changed came up twice, or is a source too */
#define STRIDE_KV_NO_PAGES 4     /* fewer pages are free than the call wants */
#define STRIDE_KV_MISSING 8      /* a position to be moved or copied has no page */
#define STRIDE_KV_BAD_KEEP 16    /* kept positions not ascending from `first` (one rule may be seen late: see below) */
#define STRIDE_KV_BAD_REFS 32    /* a held page's count was not positive: the pool was written from outside */

typedef struct StrideKvPool {
  StrideKvRef kv;
  int32_t* refs;
  uint32_t* free_bits;
  int32_t* errors;    /* [1] */
  int32_t* work;      /* stride_kv_work_ints() int32; contents need no preparation */
  int64_t work_ints;
  int32_t pages;
  int32_t slots;      /* rows of the table, at most 131072 */
  int32_t layers;
  int32_t n_kv;
  int32_t elem_bytes; /* 2: bf16, 4: fp32 */
} StrideKvPool;

int64_t stride_kv_work_ints(int32_t slots, int32_t max_blocks, int32_t pages);

/* table[slot[i]][b] gets a page for every b in [first[i], end[i]) that has none. */
int stride_kv_reserve(const StrideKvPool* p, const int32_t* slot, const int32_t* first, const int32_t* end, int32_t n,
                      void* stream);

/* table[slot[i]][b] is given up for b in [first[i], end[i]); a page without holders is
 * free. Ranges are cut to the table; an item whose slot is out of range is skipped and
 * reported; a slot may come up several times here. */
int stride_kv_release(const StrideKvPool* p, const int32_t* slot, const int32_t* first, const int32_t* end, int32_t n,
                      void* stream);

/* Sequence dst[i] becomes the first length[i] tokens of src[i]: whole pages are shared, a
 * part page is copied to a new one (its tokens below length[i]), and what dst[i] held
 * before is given up. A source may come up often, but is no destination of the same call.
 * Table entries that the source lacks are lacking in the branch. */
int stride_kv_fork(const StrideKvPool* p, const int32_t* src, const int32_t* dst, const int32_t* length, int32_t n,
                   void* stream);

/* Position first[i] + k of slot[i] becomes what keep[i][k] was, for k < count[i], in every
 * layer, K and V, as stored (keys keep the rotation they have). keep[i] ascends strictly
 * from first[i] or above, and count[i] is at most `width`. Pages behind the last kept position are given up, and a page that
 * others hold too is replaced before it is written. With count[i] = 0 nothing is written: the
 * page that first[i] lies in stays, shared or not. A kept position before first[i] + k or
 * behind the table is found before anything changes, as one without a page is. Where a list
 * does not ascend otherwise, which is seen while it is moved, the moved positions of that slot
 * hold some of the slot's old entries; the other slots are right. */
int stride_kv_compact(const StrideKvPool* p, const int32_t* slot, const int32_t* first, const int32_t* count,
                      const int32_t* keep, int64_t keep_stride, int32_t width, int32_t n, void* stream);

/* The first tokens[i] (NULL: all) tokens of page src[i] of `p` go to page dst[i] of `to`
 * (of the same shape: layers, n_kv, head_dim, page tokens, element size), or of `p` itself
 * where `to` is NULL or shares its arena. Counts and tables stay as they are. Destinations
 * differ, and none is a source in the same arena. */
int stride_kv_copy(const StrideKvPool* p, const StrideKvPool* to, const int32_t* src, const int32_t* dst,
                   const int32_t* tokens, int32_t n, void* stream);

/* Logit processing, from lm_full's tiles. For row j of sequence row_slot[j] and token t,
 * with word = counts[slot][t] (bit 31: in the prompt; below: times generated, n):
 *   l1 = word != 0 ? (l > 0 ? l / repetition : l * repetition) : l
 *   l2 = l1 - frequency * n, and - presence where n > 0
 *   l3 = l2 + bias
 *   l4 = allowed ? l3 : -inf
 * each operation rounded to fp32. best[j] becomes the largest l4 above -inf and its token,
 * of equal ones the lowest; (-inf, -1) where nothing is allowed; NaN is never chosen.
 */
typedef struct StrideLogitsParams {
  StrideLanes l;
  const float* logits;     /* tiles [rt][lt][16 rows][16 lanes] */
  float* out;              /* processed tiles (may be `logits`), or NULL; places behind rows or vocab are left alone */
  const int32_t* row_slot; /* NULL with counts NULL */
  const int32_t* counts;   /* [slots][vocab], or NULL: no penalties */
  const uint32_t* seen;    /* [slots][ceil(vocab / 32)]: bit set where counts is not 0 */
  const float* penalties;  /* [rows][3]: repetition (> 0), presence, frequency */
  const int32_t* bias_offsets; /* [rows + 1], or NULL: row j has entries bias_offsets[j] .. bias_offsets[j + 1] - 1, places
                                  of the two arrays below, which the kernel takes as they are */
  const int32_t* bias_tokens;  /* ascending in a row; of equal neighbours the last counts; out of range: ignored */
  const float* bias_values;
  const uint32_t* mask;     /* [masks][ceil(vocab / 32)]: bit set where a token is allowed, or NULL */
  const int32_t* mask_row;  /* [rows]: the row's mask, below 0: none. NULL with mask NULL */
  StrideBestEntry* best;    /* [rows], overwritten */
  uint64_t* scratch;        /* stride_logits_scratch() uint64, zero before the first call; calls leave it zero */
  int32_t vocab;
  int32_t slots;            /* rows of counts and seen; a row whose slot is outside has no penalties */
  int32_t masks;            /* rows of mask; a row whose mask is at or beyond it has none */
} StrideLogitsParams;

int stride_logits_process(const StrideLogitsParams* p, void* stream);
int64_t stride_logits_scratch(int32_t rows);

/* Token counts of sequences. */
typedef struct StrideTokenCounts {
  int32_t* counts; /* [slots][vocab] */
  uint32_t* seen;  /* [slots][ceil(vocab / 32)] */
  int32_t slots;
  int32_t vocab;
} StrideTokenCounts;

/* Token tokens[i * token_stride] of slot[i]: counted once more, or (prompt != 0) marked as
 * in the prompt. Tokens and slots out of range are ignored (-1: no token). */
int stride_logits_record(const StrideTokenCounts* p, const int32_t* slot, const int32_t* tokens, int32_t token_stride,
                         int32_t n, int32_t prompt, void* stream);

/* slot[i] forgets its tokens; src given: it takes over those of src[i] (as they are before
 * the call; a slot to be changed comes up once and is no source). Out of range: skipped. */
int stride_logits_reset(const StrideTokenCounts* p, const int32_t* slot, const int32_t* src, int32_t n, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* STRIDE_SERVE_H */
