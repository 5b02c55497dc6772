/*
 * ecf8_draft.h -- C ABI of the speculative-decoding kernels in libecf8.so:
 * trees of drafted tokens run in one step over a paged KV cache
 * (ecf8_paged.h), verified against the target's probabilities, and what was
 * accepted kept in the cache.
 *
 * None of these replaces a reference interface: the reference runs
 * transformers' generate, one token a step (scripts/inference_llm.py:108-142).
 *
 * Conventions as in ecf8.h: device pointers, stream as void*, ECF8_* status,
 * asynchronous, no allocation.  Deterministic.  Calls with the same trees share
 * their work buffer and have to be ordered, on one stream or by events.
 *
 * In a step that ecf8_paged_plan planned, the new tokens of a sequence are a
 * tree: row 0 is its last accepted token (not in the cache yet), every other
 * row a token drafted to follow an earlier row, its parent.
 */
#ifndef ECF8_DRAFT_H
#define ECF8_DRAFT_H

#include <stdint.h>

#include "ecf8_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Device buffers of the trees of a batch's steps (seqs, rows: the batch's).
 *   masks      [rows]  bit j of a row is set where it reads row j of its
 *                      sequence: its ancestors and itself
 *   parents    [rows]  the planned step's, as they were checked
 *   kept       [seqs]  rows that stay (row 0 and the accepted ones), 0: idle
 *   path       [seqs, max_nodes]  these rows in order, -1 past them
 *   emitted    [seqs, max_nodes]  as many tokens: those accepted and the next
 *                      one, -1 past them
 *   next_token [seqs]  the last of them, -1: idle
 *   work       ecf8_draft_work_bytes bytes, 16-byte aligned, its first 256
 *              bytes zeros before the first plan
 * max_nodes: most rows of a sequence, up to 64; max_children: most rows after
 * one row.  Kernels and launches go by these, not by what a step's trees hold: spare
 * rows make larger tiles (past 128 a group, of less exact probabilities), and each
 * child past the first is a launch of every verification of drawn drafts.
 */
typedef struct ecf8_draft_trees {
  uint64_t *masks;
  int *parents;
  int *kept;
  int *path;
  int64_t *emitted;
  int64_t *next_token;
  void *work;
  int64_t work_bytes;
  int max_nodes;
  int max_children;
} ecf8_draft_trees;

/* Bytes of the work buffer; -1 for sizes outside those of a batch, 1 <=
 * max_nodes <= 64 or 1 <= max_children <= 64. */
int64_t ecf8_draft_work_bytes(int64_t seqs, int64_t rows, int Hq, int Hkv, int max_nodes,
                              int max_children);

/*
 * The trees of the planned step: parents [rows] (device), of each row the row of
 * its sequence that it follows, -1 for row 0.  Fills masks and parents, sets the
 * batch's positions to cached + depth, and plans ecf8_draft_attention.  A
 * sequence with a parent that is not an earlier row (or, of row 0, not -1), or
 * more than max_children rows after one, sets the batch's `refused`; its rows are
 * then on their own: row 0's position, no parents, masks of their own bit.  So
 * does one of more than max_nodes rows, or with rows past the `rows` that parents
 * holds, of which nothing is attended.  Entries past the step's last row are left
 * as they were.  Once for every step that ecf8_paged_plan plans, also for one that
 * it plans a second time: it sets the positions to a chain's.
 */
int ecf8_draft_plan(const ecf8_paged_batch *batch, const ecf8_draft_trees *trees,
                    const int *parents, int64_t rows, void *stream);

/*
 * ecf8_paged_attention's, with trees: row t of sequence s reads the cached
 * positions [0, cached[s]) and position cached[s] + j for every set bit j of its
 * mask (masks may be rewritten after the plan).  A row that reads nothing is
 * zeros.  Probabilities are rounded to bf16 in two parts, to 2^-15, where
 * max_nodes * Hq / Hkv is up to 128, else once.  Trees that were not planned for
 * this step of the batch set `refused`; nothing is written for them.
 */
int ecf8_draft_attention(const void *q, int64_t q_stride, int64_t rows,
                         const ecf8_paged_batch *batch, const ecf8_draft_trees *trees,
                         const void *k_pool, const void *v_pool, int fp8, const float *k_scale,
                         const float *v_scale, void *out, int64_t out_stride, void *stream);

/* Bytes of ecf8_token_probabilities' work buffer. */
#define ECF8_PROBABILITY_CHUNKS 64
int64_t ecf8_probability_work_bytes(int64_t rows);

/*
 * out fp32 [rows, V] (row stride ldo) = softmax(logits / temperature) of rows of
 * bf16 logits (row stride ld), in fp32.  temperature: fp32 [rows] on the device,
 * or NULL for the scalar `common`.  Not above zero: one at the largest logit (ties
 * to the lower index, NaN counts as largest), zero elsewhere.  NaN, or an infinite
 * largest logit, gives a row of NaN.
 */
int ecf8_token_probabilities(const void *logits, int64_t ld, int64_t rows, int64_t V,
                             const float *temperature, float common, float *out, int64_t ldo,
                             void *work, int64_t work_bytes, void *stream);

/*
 * Verification of the planned step's trees: target fp32 [rows, V] are the
 * model's probabilities after each row, tokens int64 [rows] the rows' tokens,
 * accept fp32 [rows] and sample fp32 [seqs] random numbers in [0, 1).  From row
 * 0 on, the children of the last accepted row are tried in order, with w = its
 * target probabilities and Z = 1 at first:
 *   draft = NULL, children are different tokens: child c is accepted if
 *     accept Z < w(c), else w(c) becomes 0 and Z - w(c) the new Z;
 *   draft fp32 [rows, V], children are drawn (independently) from row's q =
 *     draft: accepted if accept q(c) Z < w(c), else max(w / Z - q, 0) becomes
 *     the new w, and its sum Z.
 * The next token is drawn from the last accepted row's w: the first v of which
 * w(0) + ... + w(v) is above sample times the sum; where no w is left, from its
 * target probabilities.  All in 64 bits.  The tokens so emitted are distributed
 * as the target's own.  Fills kept, path, emitted and next_token.
 * rows: those of target, draft and tokens; a step of more rows sets `refused`,
 * and so do tokens outside [0, V), which are never accepted, probabilities
 * whose sum is not above zero and finite (next token -1), and trees that were not
 * planned for this step, of which every sequence is left idle.
 */
int ecf8_draft_verify(const ecf8_paged_batch *batch, const ecf8_draft_trees *trees,
                      const int64_t *tokens, int64_t rows, const float *target, int64_t ld_target,
                      const float *draft, int64_t ld_draft, int64_t V, const float *accept,
                      const float *sample, void *stream);

/*
 * Moves what was accepted together: in each of n_pools pools (an array of device
 * pointers in host memory, read by this call; [pages, Hkv, page_size, 128], bf16
 * or, fp8 != 0, e4m3fn), the row at position cached[s] + path[s][i] goes to
 * cached[s] + i for i < kept[s], as if all were read before any is written.
 * cached: the batch's lengths less the step's rows.  A path that is not ascending
 * from 0 within the sequence's rows sets `refused` and is cut there.  Trees that
 * were planned, but for another step, set it too, and nothing moves.  Once a step: a
 * second call would move what is in its place.
 */
int ecf8_draft_keep(const ecf8_paged_batch *batch, const ecf8_draft_trees *trees,
                    void *const *pools, int n_pools, int fp8, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ECF8_DRAFT_H */
