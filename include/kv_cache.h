/*
 * kv_cache.h -- C ABI of the MI355X (gfx950) paged-cache operators: filling the
 * caches that the decode attention of gqa_decode.h and mla_decode.h reads, and
 * a cache of keys and values held in 4 bits with the attention over it.
 *
 * The paged caches and index tensors are those of the attention entry points:
 *   k_cache, v_cache  [num_blocks, block_size, Hkv, 128] bf16 (gqa_decode.h)
 *   kv_cache (MLA)    [num_blocks, block_size, 1, 576]   bf16 (mla_decode.h)
 *   block_table       [B, max_blocks] int32, seq_lens [B] int32
 *
 * The 4-bit cache: E2M1 elements with one power-of-two scale for each 32
 * dims, the MXFP4 format of the OCP Microscaling specification. One array of
 * bytes [num_blocks, Hkv, block_size / 16, 2176]: tiles of 16 tokens of one
 * kv-head, block_size a multiple of 16. Token r (0..15), dim d (0..127) of a
 * tile:
 *   key code    byte   (d / 32) * 256 + r * 16 + (d % 32) / 2
 *   value code  byte   1024 + (r / 4) * 256 + (d / 8) * 16 + (r % 4) * 4 + (d % 8) / 2
 *               (low nibble: even d; sign, then a 3-bit magnitude index of
 *               0, 0.5, 1, 1.5, 2, 3, 4, 6)
 *   key scale   byte   2048 + (d / 32) * 16 + r
 *   value scale byte   2112 + (r / 4) * 16 + (d / 32) * 4 + r % 4
 *               (scale byte e: 2^(e - 127); 255: the 32 values are NaN)
 * 136 bytes a token and kv-head, keys and values together, where the bf16
 * caches take 512.
 *
 * New tokens. A step hands in the rows of T new tokens, in request order.
 * cu_seqlens [B + 1] int32 says where each request's rows start (rows
 * cu_seqlens[b] .. cu_seqlens[b + 1] - 1 are request b's); without it (null) T
 * must be B and every request has one new token. seq_lens counts the new
 * tokens: the last of request b's n rows is at position seq_lens[b] - 1, the
 * first at seq_lens[b] - n. A row that has no place is padding: one at or past
 * cu_seqlens[B], or of a request whose seq_lens[b] is smaller than n (its
 * position would be negative; 0 marks an unused request of a fixed-size
 * batch). Padding writes nothing to a cache, and its row of q_out or of the
 * rows read back is zeros. Rows whose position is past the block table, or
 * whose block id is outside [0, num_blocks), write nothing to the cache either
 * (and read back as zeros); their q_out row is computed. A block that a call
 * writes stands once in the call's table rows: no two of its requests share it,
 * and none lists it twice.
 *
 * Launchers are asynchronous on `stream`, allocate nothing, keep nothing
 * between calls, may be captured into graphs, and return 0 or a hipError_t
 * code (hipErrorInvalidValue for arguments rejected before any launch). They
 * run on the current device. The same call gives the same bits. No reference
 * counterpart: the reference's benches fill their caches with torch.
 */
#ifndef KV_CACHE_H_
#define KV_CACHE_H_

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef GQA_DECODE_API
#define GQA_DECODE_API __attribute__((visibility("default")))
#endif

/* Tokens and bytes of a tile of the 4-bit cache. */
#define KV_MXFP4_TILE_TOKENS 16
#define KV_MXFP4_TILE_BYTES 2176

/* Most new tokens (T) of a call (whose requests are at most 2^30). */
#define KV_MAX_TOKENS (1 << 23)

/* Types of a norm weight. */
#define KV_WEIGHT_BF16 0
#define KV_WEIGHT_FP32 1

/* The arguments of the GQA appends. For every new token t and head h
 *   y = x                                     without a weight, or
 *   y = x / sqrt(mean(x^2) + eps) * weight    the mean over the head's 128 dims,
 * and then, with h = rotary_dim / 2 angle columns cos = table[p][0..h),
 * sin = table[p][h..2h) of the token's rotation position p, pairs of the first
 * rotary_dim dims turn:
 *   (a, b) -> (a cos - b sin, b cos + a sin)
 * pair i being dims (i, i + h), or (2i, 2i + 1) with interleaved != 0; dims from
 * rotary_dim on stay. q goes to q_out, k and the unchanged v to the cache.
 * p is the token's position, or rope_positions[t] if given; a row whose p is
 * outside the table turns into NaN (its first rotary_dim dims). One rounding,
 * to bf16 or to the 4-bit form, at the end. */
typedef struct kv_append_args {
  /* Rows [T, heads, 128] bf16, dims contiguous; strides in elements. q_out may
   * be q itself (the same pointer and strides); otherwise no two of the arrays
   * overlap. Any alignment of two bytes. */
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  int64_t q_token_stride, q_head_stride;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
  int64_t q_out_token_stride, q_out_head_stride;
  /* The bf16 caches (kv_append_launch), 16-byte aligned, or the 4-bit cache
   * (kv_append_mxfp4_launch), 4-byte aligned; the others are ignored. */
  uint16_t* k_cache;
  uint16_t* v_cache;
  uint8_t* mxfp4_cache;
  const int* block_table; /* may be null with B = 0, as may seq_lens */
  const int* seq_lens;
  const int* cu_seqlens;     /* null: one token a request */
  const int* rope_positions; /* [T], null: the tokens' positions */
  /* [table_rows, rotary_dim] fp32: cosines, then sines. Null: no rotation
   * (rotary_dim 0). rotary_dim is a multiple of 16 up to 128. */
  const float* cos_sin;
  const void* q_weight; /* [128], null: no norm */
  const void* k_weight;
  int q_weight_type, k_weight_type; /* KV_WEIGHT_BF16 or KV_WEIGHT_FP32 */
  int T, B, Hq, Hkv, num_blocks, block_size, max_blocks;
  int table_rows, rotary_dim, interleaved;
  float eps;
} kv_append_args;

/* Norm, rotation and append to the bf16 caches. fp32 arithmetic. */
GQA_DECODE_API int kv_append_launch(const kv_append_args* args, hipStream_t stream);

/* The same with the 4-bit cache. A group's scale is the power of two that puts
 * its largest magnitude into (3.5, 7] (at least 2^-126), an element's code the
 * nearest one, ties to the even code; a group that holds an infinity or NaN
 * gets scale 255. Keys are normed and turned in fp64, so the codes are those of
 * the formula, whichever launch wrote them (what is past fp32's range by then
 * counts as its largest value). */
GQA_DECODE_API int kv_append_mxfp4_launch(const kv_append_args* args, hipStream_t stream);

/* The keys and values of the rows that an append with the same T, cu_seqlens,
 * seq_lens and block_table writes, as bf16 [T, Hkv, 128] (contiguous, 16-byte
 * aligned): every value of the 4-bit format is a bf16 value (but those of 2^128
 * and more, under scale bytes 253 and 254, which read as infinities). With seq_lens
 * the requests' lengths and cu_seqlens their running sum, the whole cache. */
GQA_DECODE_API int kv_read_mxfp4_launch(const uint8_t* mxfp4_cache, const int* block_table,
                                        const int* seq_lens, const int* cu_seqlens,
                                        uint16_t* k_out, uint16_t* v_out, int T, int B, int Hkv,
                                        int num_blocks, int block_size, int max_blocks,
                                        hipStream_t stream);

/* The arguments of the MLA append. The latent row c [T, 512] (normed over its
 * 512 dims with c_weight) and the key's rotary part k_pe [T, 64] (turned) go to
 * the cache's 576-dim rows; q_pe [T, h_q, 64] is turned into q_out, which may be
 * the last 64 dims of the absorbed queries [T, h_q, 576]. Norm, rotation,
 * padding and the index tensors as in kv_append_args; the table has 64 columns. */
typedef struct kv_append_mla_args {
  const uint16_t* q_pe;
  const uint16_t* c;
  const uint16_t* k_pe;
  uint16_t* q_out;
  int64_t q_token_stride, q_head_stride;
  int64_t c_token_stride, k_token_stride;
  int64_t q_out_token_stride, q_out_head_stride;
  uint16_t* kv_cache; /* 16-byte aligned */
  const int* block_table;
  const int* seq_lens;
  const int* cu_seqlens;
  const int* rope_positions;
  const float* cos_sin; /* [table_rows, 64] */
  const void* c_weight; /* [512], null: no norm */
  int c_weight_type;
  int T, B, h_q, num_blocks, block_size, max_blocks;
  int table_rows, interleaved;
  float eps;
} kv_append_mla_args;

GQA_DECODE_API int kv_append_mla_launch(const kv_append_mla_args* args, hipStream_t stream);

/* Single-token GQA decode over the 4-bit cache:
 *   out[b, h, :] = softmax_t(scale * <q[b, h, :], K_b[t, kv(h), :]>) . V_b[t, kv(h), :]
 * over t < min(seq_lens[b], max_blocks * block_size), kv(h) = h / (Hq / Hkv),
 * with K and V the values that the cache's codes stand for (V as bf16: of 2^128
 * and more as infinities), in fp32 arithmetic of exact products, rounded once to
 * bf16. (Units of 32 tokens that hold a key of scale byte 253 or 254 take their
 * scores to some 14 bits of the largest product only.) q and out [B, Hq, 128] bf16,
 * contiguous; q, out and the cache 16-byte aligned; out must not overlap q. A
 * request of length 0 gets zeros. Tokens in blocks whose id is outside
 * [0, num_blocks) are left out (a request with no other token gets zeros).
 * B * ceil(max_blocks * block_size / 32) * Hkv * ceil(Hq / Hkv / 16) is at most
 * 2^31 - 1, and so are the bytes of a block (of all heads).
 *
 * num_workgroups > 0: token-balanced. Each workgroup of that grid takes an equal
 * share of the batch's 32-token units, whatever the lengths, and a second launch
 * merges the segments (a request's tokens for up to 16 q-heads of one kv-head)
 * cut at share boundaries, in share order: the bits of a result are those of the
 * lengths, the batch and num_workgroups.
 * num_workgroups <= 0: chosen from the sizes and the current device. Tables of up
 * to 64 units a request (48 where segments are fewer than a quarter of the CUs) keep
 * segments whole, in one launch: a workgroup to each segment if they are no more
 * than the CUs, else shares whose ends are moved to the next segment's start. Wider
 * tables take the token-balanced launch with a workgroup to each CU. The choice, and
 * with it the order of the sums, depends on max_blocks * block_size, not on the
 * lengths: the host never reads seq_lens. Where short requests lie behind a wide
 * table, a max_blocks (and table) cut to the longest saves 1-5 us.
 * workspace: kv_decode_mxfp4_workspace_bytes(B, Hq, Hkv, block_size,
 * max_blocks, num_workgroups) bytes (it may be 0), 16-byte aligned,
 * uninitialised; launches that share one must not overlap. */
GQA_DECODE_API int kv_decode_mxfp4_launch(const uint16_t* q, const uint8_t* mxfp4_cache,
                                          const int* block_table, const int* seq_lens,
                                          uint16_t* out, int B, int Hq, int Hkv, int num_blocks,
                                          int block_size, int max_blocks, float scale,
                                          int num_workgroups, void* workspace,
                                          size_t workspace_bytes, hipStream_t stream);

GQA_DECODE_API size_t kv_decode_mxfp4_workspace_bytes(int B, int Hq, int Hkv, int block_size,
                                                      int max_blocks, int num_workgroups);

#ifdef __cplusplus
}
#endif

#endif /* KV_CACHE_H_ */
