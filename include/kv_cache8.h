/*
 * kv_cache8.h -- C ABI of the MI355X (gfx950) paged cache of keys and values held in 8
 * bits with a scale for each block of 16 tokens and head: append, read-back and
 * single-token decode attention. Index tensors, new tokens, norm, rotation, padding and
 * launch contract are kv_cache.h's.
 *
 * Codes: one array of bytes [num_blocks, Hkv, block_size / 16, 4096]: tiles of 16 tokens
 * of one kv-head, block_size a multiple of 16. Token r (0..15), dim d (0..127) of a tile:
 *   key    byte  (d / 16 % 2) * 1024 + (d / 32) * 256 + r * 16 + d % 16
 *   value  byte  2048 + (d / 4 % 2) * 1024 + (r / 4) * 256 + (d / 8) * 16 + (d % 4) * 4 + r % 4
 * in e4m3 (OCP 8-bit floating point: sign, 4 bits of exponent, 3 of mantissa, bias 7,
 * largest 448, no infinities, NaN 127 and 255).
 * Scales: bytes [num_blocks, Hkv, block_size / 16, 2], for a tile's keys and for its
 * values; byte e (10 to 246) stands for 2^(e - 127). 256 bytes a token and kv-head, and
 * 2 a tile, where the bf16 caches take 512.
 */
#ifndef KV_CACHE8_H_
#define KV_CACHE8_H_

#include "kv_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Tokens and bytes of a tile, scale bytes of a tile. */
#define KV8_TILE_TOKENS 16
#define KV8_TILE_BYTES 4096
#define KV8_TILE_SCALES 2

/* Norm, rotation and append. args as for kv_append_launch, its caches ignored; codes
 * 16-byte, scales 2-byte aligned. Keys are normed and turned in fp64, so that codes are
 * those of the formula.
 *   The new tokens of a tile, keys and values apart, ask for the least scale byte (10 or
 * more) under which their largest finite magnitude is at most 448 (246 at most; what is
 * past 448 under it is held as 448). If the tile has older tokens (slots in front of
 * the first new one) its scale is the larger of that and the present one, and where it
 * grows the older tokens' codes are rounded again under the new scale. Slots behind the
 * new tokens stay as they are. A code is the nearest one, ties to even; infinities and
 * NaN are held as NaN.
 *   A scale thus only grows while a tile fills, and is set anew by a token in slot 0.
 *   Sizes whose launch would have 2^32 threads or more are refused (256 for each kv-head
 * of T / 16 + 2 B tiles, or of T without cu_seqlens, a quarter of that for the values, and
 * 256 for 4 tokens and 16 heads of the queries). */
GQA_DECODE_API int kv8_append_launch(const kv_append_args* args, uint8_t* codes, uint8_t* scales,
                                     hipStream_t stream);

/* Rows as kv_read_mxfp4_launch hands them back, bf16 (exactly). */
GQA_DECODE_API int kv8_read_launch(const uint8_t* codes, const uint8_t* scales,
                                   const int* block_table, const int* seq_lens,
                                   const int* cu_seqlens, uint16_t* k_out, uint16_t* v_out, int T,
                                   int B, int Hkv, int num_blocks, int block_size, int max_blocks,
                                   hipStream_t stream);

/* Single-token GQA decode, as kv_decode_mxfp4_launch (launches, workspace, limits, padding).
 * Codes behind a sequence's end may be anything; scale bytes of tiles in use are 10 to
 * 246. */
GQA_DECODE_API int kv8_decode_launch(const uint16_t* q, const uint8_t* codes,
                                     const uint8_t* scales, const int* block_table,
                                     const int* seq_lens, uint16_t* out, int B, int Hq, int Hkv,
                                     int num_blocks, int block_size, int max_blocks, float scale,
                                     int num_workgroups, void* workspace, size_t workspace_bytes,
                                     hipStream_t stream);

GQA_DECODE_API size_t kv8_decode_workspace_bytes(int B, int Hq, int Hkv, int block_size,
                                                 int max_blocks, int num_workgroups);

#ifdef __cplusplus
}
#endif

#endif /* KV_CACHE8_H_ */
