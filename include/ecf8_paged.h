/*
 * ecf8_paged.h -- C ABI of the ragged-batch kernels in libecf8.so: the
 * bookkeeping of a paged KV cache, the cache write of a step's rows, their
 * attention over the pages, and the causal attention of packed prompts.
 *
 * None of these replaces a reference interface: the reference runs
 * transformers' generate with its dense caches (scripts/inference_llm.py:
 * 108-142) around its decoded weights.
 *
 * Conventions as in ecf8.h: device pointers, stream as void*, ECF8_*
 * status, asynchronous, no allocation.  bf16 tensors are passed as void*
 * (2-byte elements).  Head dimension 128, Hq any multiple of Hkv.
 * Deterministic.
 *
 * A batch holds up to `seqs` sequences.  In a step sequence s has cached[s]
 * tokens in the cache and brings new_tokens[s] more (zero: it is idle).  The
 * new tokens of all sequences are packed: sequence s has rows [starts[s],
 * starts[s + 1]) of the step's activations.
 */
#ifndef ECF8_PAGED_H
#define ECF8_PAGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Device buffers of a batch (int32 unless said otherwise).  A pool holds
 * `pages` pages of page_size (a power of two, at most 1024) positions:
 * [pages, Hkv, page_size, 128], bf16 or e4m3fn.
 *   table      [seqs, width]  the pages of a sequence in order, -1 past owned
 *   owned      [seqs]         pages of a sequence
 *   free_pages [pages]        stack of the free pages, n_free[0] of them
 *   starts     [seqs + 1], lengths [seqs] (cached + new tokens)
 *   slots      [rows]         page * page_size + offset of a packed row's
 *                             position, -1 past the last row
 *   positions  [rows]         its position in its sequence, -1 past the last
 *   refused    [1] or NULL, memory that the device can write (e.g. pinned host
 *              memory): set when a kernel refuses a step's values
 *   work       ecf8_paged_work_bytes bytes, 16-byte aligned: the attention's
 *              schedule (written by ecf8_paged_plan) and partial sums; its first
 *              256 bytes are zeros before the first plan (an empty step)
 */
typedef struct ecf8_paged_batch {
  int *table;
  int *owned;
  int *free_pages;
  int *n_free;
  int *starts;
  int *lengths;
  int *slots;
  int *positions;
  int *refused;
  void *work;
  int64_t work_bytes;
  int seqs;
  int rows;
  int pages;
  int page_size;
  int width;
  int Hq;
  int Hkv;
} ecf8_paged_batch;

/* Bytes of the work buffer for up to `rows` new tokens of `seqs` sequences;
 * -1 for sizes outside 1 <= seqs <= 4096, 1 <= rows <= 262144, Hq a multiple
 * of Hkv. */
int64_t ecf8_paged_work_bytes(int64_t seqs, int64_t rows, int Hq, int Hkv);

/*
 * The bookkeeping of one step, on the device from device lengths:
 *   1. a sequence with release[s] != 0 (release may be NULL) gives its pages
 *      back: pushed on the stack, sequences and their pages in order;
 *   2. a sequence takes pages until it owns ceil((cached + new) / page_size);
 *      it keeps what it owns beyond that.  Pages come off the stack one by
 *      one, sequences in order;
 *   3. starts, lengths, slots, positions and the attention's schedule.
 * A step that cannot be done (negative lengths, a sequence longer than its
 * table row, more rows than `rows`, too few free pages) sets `refused`,
 * changes neither table, owned nor the stack, and plans an empty step: starts
 * and lengths zero, every slot -1.  A step planned again with the same lengths
 * takes no further pages; with release set again, its sequences' pages go back and
 * others come, and what was written to them since is lost.
 */
int ecf8_paged_plan(const ecf8_paged_batch *batch, const int *cached, const int *new_tokens,
                    const int *release, void *stream);

/*
 * For the packed rows of the planned step of the fused projection output qkv
 * bf16 [rows, (Hq + 2*Hkv) * 128] (q heads, then k heads, then v heads):
 *   q, k: RMSNorm over the head (bf16 weights q_norm / k_norm [128]), then
 *         the rotary embedding at the row's position, rotate-half form, cos_t
 *         / sin_t fp32 [table_len, 64];
 *   q -> q_out bf16 [rows, Hq, 128]; k, v -> their pools at the row's slot.
 * fp8 != 0: pools of e4m3fn codes, code = round_nearest_even(x / scale)
 * clamped to +-448, with an fp32 scale per KV head (k_scale / v_scale [Hkv],
 * above zero); fp32 values are rounded once.  Rows without a slot, or past
 * table_len, write nothing.  rows: those of qkv and q_out, at most the
 * batch's; a step of more rows sets `refused` (its first `rows` are written).
 */
int ecf8_paged_qk_norm_rope(const void *qkv, int64_t rows, const ecf8_paged_batch *batch,
                            const void *q_norm, const void *k_norm, float eps, const float *cos_t,
                            const float *sin_t, int64_t table_len, void *q_out, void *k_pool,
                            void *v_pool, int fp8, const float *k_scale, const float *v_scale,
                            void *stream);

/*
 * Attention of the planned step's rows over the pages (the new tokens' keys
 * and values already written): query t of sequence s, at position cached[s] +
 * t, reads positions [0, cached[s] + t].  q bf16, row i's heads at q + i *
 * q_stride elements; scores scaled by 1/sqrt(128); out bf16, row i's heads at
 * out + i * out_stride.  fp8 != 0: e4m3fn pools with scales as above.  fp32
 * scores, softmax statistics and sums; probabilities are rounded to bf16 (in two
 * parts, to 2^-15, for sequences of up to 32 rows of new tokens and heads of a
 * group).
 * rows: those of q and out; max_new: an upper bound of the step's new tokens
 * of any one sequence (the launches depend on both).  A step that exceeds
 * either sets `refused`, and its outputs are incomplete.  So does a `work` that was
 * not planned for a batch of these sizes, of which nothing is read.  Rows past the
 * last sequence are left as they were.
 */
int ecf8_paged_attention(const void *q, int64_t q_stride, int64_t rows,
                         const ecf8_paged_batch *batch,
                         const void *k_pool, const void *v_pool, int fp8, const float *k_scale,
                         const float *v_scale, int64_t max_new, void *out, int64_t out_stride,
                         void *stream);

/*
 * Causal attention of packed prompts without a cache: sequence s has rows
 * [starts[s], starts[s + 1]) (starts: device int32 [seqs + 1], ascending) of
 * q [rows, Hq, 128] and k, v [rows, Hkv, 128] (bf16, row strides in
 * elements, multiples of 8); query t reads rows 0..t of its own sequence.
 * Numerics and out as above, but for the probabilities: rounded to bf16 once in
 * calls of 49152 (rows * Hq) and more, in two parts in smaller ones.  Rows outside
 * every sequence are left as they were.
 */
int ecf8_ragged_attention(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                          const void *v, int64_t v_stride, int64_t rows, const int *starts,
                          int64_t seqs, int Hq, int Hkv, void *out, int64_t out_stride,
                          void *stream);

/* ecf8_ragged_attention; starts that are not ascending, or outside [0, rows],
 * also set refused[0] (memory that the device can write, e.g. pinned host memory).
 * Without it such starts are cut to the rows that there are, and the outputs are
 * incomplete. */
int ecf8_ragged_attention_checked(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                                  const void *v, int64_t v_stride, int64_t rows,
                                  const int *starts, int64_t seqs, int Hq, int Hkv, void *out,
                                  int64_t out_stride, int *refused, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ECF8_PAGED_H */
