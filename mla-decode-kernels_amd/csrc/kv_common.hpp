// Layout of the 4-bit paged cache (include/kv_cache.h) and the device helpers
// its kernels and the append kernels share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gqa_device.hpp"
#include "kv_places.hpp"

namespace kv {

using gqa::bf16_hi;
using gqa::bf16_lo;
using gqa::FastDiv;
using gqa::fastdiv;
using gqa::make_fastdiv;

constexpr int kDim = 128;
constexpr int kTileTokens = 16;
constexpr int kTileBytes = 2176;
constexpr int kValueCodes = 1024;   // byte offsets in a tile
constexpr int kKeyScales = 2048;
constexpr int kValueScales = 2112;

// Byte offsets of a token's share of a tile: r the token in the tile, i the
// group of 8 dims (codes: 4 bytes), g the group of 32 dims (scale: 1 byte).
__host__ __device__ constexpr int key_code_at(int r, int i) {
  return (i >> 2) * 256 + r * 16 + (i & 3) * 4;
}
__host__ __device__ constexpr int value_code_at(int r, int i) {
  return kValueCodes + (r >> 2) * 256 + i * 16 + (r & 3) * 4;
}
__host__ __device__ constexpr int key_scale_at(int r, int g) { return kKeyScales + g * 16 + r; }
__host__ __device__ constexpr int value_scale_at(int r, int g) {
  return kValueScales + (r >> 2) * 16 + g * 4 + (r & 3);
}
static_assert(key_code_at(15, 15) + 4 == kValueCodes && value_code_at(15, 15) + 4 == kKeyScales &&
                  key_scale_at(15, 3) + 1 == kValueScales && value_scale_at(15, 3) + 1 == kTileBytes,
              "the four parts fill a tile");

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// 16 bytes at an address that is a multiple of 2 (rows of strided views can
// start anywhere; gfx950 loads and stores them whole at any alignment).
typedef u32x4 u32x4_any __attribute__((aligned(2)));
__device__ __forceinline__ uint4 load16(const uint16_t* p) {
  const u32x4 v = *reinterpret_cast<const u32x4_any*>(p);
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void store16(uint16_t* p, const uint4& v) {
  *reinterpret_cast<u32x4_any*>(p) = u32x4{v.x, v.y, v.z, v.w};
}

__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z); x[5] = bf16_hi(w.z); x[6] = bf16_lo(w.w); x[7] = bf16_hi(w.w);
}
// Two fp32 values as bf16, to nearest even (v_cvt_pk_bf16_f32).
typedef float f32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x, y}, bf16x2_t));
}
// The only rounding of a bf16 append.
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
}

// fp64 -> fp32 rounded to odd: truncated, with the last bit set if anything was
// cut off. A later rounding to fewer than 23 bits then gives what rounding the
// fp64 value itself would have given (no double rounding).
__device__ __forceinline__ float f32_to_odd(double d) {
  const float f = (float)d;
  const double back = (double)f;
  uint32_t u = __float_as_uint(f);
  if (back != d && d == d) {
    if (__builtin_fabs(back) > __builtin_fabs(d)) --u;  // rounded up (from infinity too)
    u |= 1u;
  }
  return __uint_as_float(u);
}

// The place of row t of the new tokens (kv_cache.h), computed by each group of
// kGroup lanes (a power of two, aligned) for its own t; 0 <= t. Every lane of the
// wave calls it. Up to kGroup requests take one round trip to memory, kGroup^2 two.
// The probes of a part of a wave bring along what is needed of the request they
// find (its first row, the next one's, its length): an append of 7255 tokens
// (32Q/8KV) takes 41.0 us so and 42.2 without. A whole wave's t is the same in all
// lanes, so scalar loads fetch that afterwards, in fewer registers: an MLA append
// of 8016 tokens (16 heads) takes 12.6 us so and 12.9 with what the probes bring
// (the same rows again and again).
template <int kGroup>
__device__ __forceinline__ Place find_place(int t, int T, int B, const int* __restrict__ seq_lens,
                                            const int* __restrict__ cu_seqlens, int lane) {
  if (!cu_seqlens) {
    if (t >= B || t >= T) return Place{0, 0, false};
    return place_in(t, t, t, t + 1, seq_lens[t]);
  }
  constexpr bool kBring = kGroup < 64;
  const int sub = lane & (kGroup - 1), shift = lane & ~(kGroup - 1);
  Search s = Search::begin(B);
  int first = cu_seqlens[0], next = 0, len = -1;  // entries lo - 1 and hi, length hi - 1
  // Groups may need different numbers of steps: all lanes stay until all are
  // done (the ballot is the wave's).
  while (__builtin_amdgcn_ballot_w64(!s.done())) {
    const int step = s.step(kGroup), at = s.lo + sub * step;
    const bool probe = at < s.hi;
    const int entry = probe ? cu_seqlens[at] : 0;
    const int its_len = kBring && probe ? seq_lens[at - 1] : -1;
    uint64_t m = __builtin_amdgcn_ballot_w64(probe && entry <= t) >> shift;
    if constexpr (kGroup < 64) m &= (uint64_t(1) << (kGroup & 63)) - 1;
    const int count = __popcll(m);
    const bool below = s.narrow(step, count);
    if constexpr (kBring) {
      const int last = __shfl(entry, shift + max(count - 1, 0), 64);
      const int behind = __shfl(entry, shift + min(count, kGroup - 1), 64);
      const int behind_len = __shfl(its_len, shift + min(count, kGroup - 1), 64);
      if (count > 0) first = last;
      if (below) next = behind, len = behind_len;
    }
  }
  const int b = s.request();
  if (b >= B || t >= T) return Place{0, 0, false};
  if constexpr (!kBring) first = cu_seqlens[b], next = cu_seqlens[b + 1], len = seq_lens[b];
  return place_in(t, b, first, next, len);
}

// The block id of a position, or -1 where the cache has no place for it.
__device__ __forceinline__ int find_block(const Place& p, const int* __restrict__ block_table,
                                          int max_blocks, int num_blocks, const FastDiv& bs_div,
                                          int& slot) {
  slot = 0;
  if (!p.live) return -1;
  const uint32_t lb = fastdiv((uint32_t)p.pos, bs_div);
  slot = p.pos - (int)(lb * bs_div.d);
  if (lb >= (uint32_t)max_blocks) return -1;
  const int id = block_table[(size_t)p.b * max_blocks + lb];
  return (uint32_t)id < (uint32_t)num_blocks ? id : -1;
}

}  // namespace kv
