/*
 * prefill.h -- C ABI of the MI355X (gfx950) attention of many new tokens a
 * request: whole prompts, chunks of them behind a cached prefix, drafted tokens.
 * Single tokens are gqa_decode.h's.
 *
 * B requests bring T new rows q [T, Hq, 128], in request order: rows
 * cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 are request b's (n of them; without
 * cu_seqlens_q T is B and every request has one). Its keys and values, L of them,
 * are either
 *   paged   k_cache, v_cache [num_blocks, block_size, Hkv, 128] behind block_table
 *           [B, max_blocks] and seq_lens [B] (gqa_decode.h; L = seq_lens[b], which
 *           counts the new tokens, as after kv_cache.h's append), or
 *   packed  rows cu_seqlens_k[b] .. cu_seqlens_k[b + 1] - 1 of k, v [Tk, Hkv, 128].
 * Row i of request b stands at position p = L - n + i, and
 *   out[row, h, :] = sum_j softmax_j(scale * <q[row, h, :], K_j>) . V_j
 * over the keys j <= p (causal), or over all L keys; kv-head h / (Hq / Hkv).
 * fp32 arithmetic of exact products; the softmax weights are rounded to bf16 for the
 * product with V and divided by the sum of the rounded ones; out is rounded to bf16.
 * A value that is not finite, an infinity as well, makes NaN of its dim in every row that
 * sees it. A query that is not finite makes NaN of its whole row, and so do keys whose
 * scores are not finite, but for scores of -infinity beside a finite one (weight 0).
 * lse[row, h] is the natural logarithm of the sum of exp(scale * <q, K_j>), in fp32.
 *
 * Rows without a place get zeros and an lse of -infinity: those of no request (before
 * cu_seqlens_q[0], from cu_seqlens_q[B] on) and those at a negative position (L < n).
 * Paged keys past the table's end (max_blocks * block_size) and in blocks whose id is
 * outside [0, num_blocks) are left out; a row that sees no other key gets zeros and
 * -infinity as well. What lies in cache slots behind a request's end, and in keys and
 * values that a row does not see, has no influence, infinities and NaN included.
 *
 * Launchers are asynchronous on `stream`, allocate nothing, keep nothing between
 * calls, may be captured into graphs, run on the current device and return 0 or a
 * hipError_t code (hipErrorInvalidValue for arguments rejected before any launch). The
 * same call gives the same bits. No reference counterpart.
 */
#ifndef PREFILL_H_
#define PREFILL_H_

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef GQA_DECODE_API
#define GQA_DECODE_API __attribute__((visibility("default")))
#endif

/* Most splits of the key axis, most new rows of a call (T), most requests. */
#define PREFILL_MAX_SPLITS 128
#define PREFILL_MAX_TOKENS (1 << 23)
#define PREFILL_MAX_BATCH (1 << 20)

typedef struct prefill_gqa_args {
  /* Rows [T, Hq, 128] bf16, dims contiguous, any alignment of two bytes; strides in
   * elements, not negative. */
  const uint16_t* q;
  int64_t q_token_stride, q_head_stride;
  /* The caches (paged), or rows [Tk, Hkv, 128] with dims contiguous and strides in
   * elements (packed; strides are multiples of 8 and below 2^27). 16-byte aligned. */
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  uint16_t* out;           /* [T, Hq, 128] contiguous, 16-byte aligned; overlaps no input */
  float* lse;              /* [T, Hq] contiguous, or null */
  const int* cu_seqlens_q; /* [B + 1], null: one row a request */
  const int* block_table;  /* paged */
  const int* seq_lens;     /* paged */
  const int* cu_seqlens_k; /* packed: [B + 1]; null: paged */
  int T, B, Hq, Hkv;
  int num_blocks, block_size, max_blocks; /* paged */
  int Tk;                                 /* packed; up to 2^31 - 65 */
  int causal;
  float scale;
} prefill_gqa_args;

/* num_splits > 0: every request's keys are cut into that many pieces, whose partial
 * results a second launch joins in order (1: no second launch). Paged pieces are equal
 * parts of max_blocks * block_size tokens, whatever of them a request has. 0: chosen from
 * the sizes and the current device's CU count; the host never reads the lengths.
 * Sizes whose launches would have 2^32 threads or more are refused: none with T Hq / 128 +
 * (B + 2) Hkv below 2^23 and, where there is a second launch, T Hq up to 2^26 - 4.
 * workspace: prefill_gqa_workspace_bytes(args, num_splits) bytes (it may be 0), 16-byte
 * aligned, uninitialised; launches that share one must not overlap. */
GQA_DECODE_API int prefill_gqa_launch(const prefill_gqa_args* args, int num_splits,
                                      void* workspace, size_t workspace_bytes,
                                      hipStream_t stream);

GQA_DECODE_API size_t prefill_gqa_workspace_bytes(const prefill_gqa_args* args, int num_splits);

/* The splits that num_splits = 0 takes (from the sizes alone; 0 for invalid sizes). */
GQA_DECODE_API int prefill_gqa_pick_num_splits(const prefill_gqa_args* args);

#ifdef __cplusplus
}
#endif

#endif /* PREFILL_H_ */
