// Single-token GQA decode over the 8-bit paged cache (include/kv_cache8.h): the plan,
// the walk and the softmax of kv_decode_scan.hpp over e4m3 codes with one power of two
// for a tile's keys and one for its values.
//
// A unit is two 16-token tiles, which the lanes load whole, 32 bytes of keys and 32 of
// values a lane and tile, in the matrix operands' layouts: v_cvt_scalef32_pk_bf16_fp8
// widens two codes exactly, scale and all, and what comes out is the operand. (The values
// lie four tokens of a dim together, so that they need no exchange.) e4m3 codes have 4
// significant bits and the scales end at 2^119, so bf16 holds every value.
//   What bounds it: HBM, at 256 bytes a token and kv-head. 32 requests of 8192 tokens
// (32Q/8KV, blocks of 16: 537 MB) take 86 us, merge launch and all (6.2 TB/s); 64 ragged
// ones up to 32768 (64Q/8KV: 2.1 GB) 331 us (6.5 TB/s); 128 of 777 (205 MB) 38 us (5.4
// TB/s). One request of 512 tokens takes 7.3 us, one launch whose loads wait for each other.
// When a workgroup keeps whole segments is decided as for the 4-bit cache: the rule was
// looked over at these sizes and holds.
#include "kv_cache8.h"
#include "kv_common8.hpp"
#include "kv_decode_scan.hpp"

namespace {

// Eight codes of one scale.
__device__ __forceinline__ bf16x8_t widen8(uint32_t lo, uint32_t hi, float by) {
  const u32x4 w = {
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, by, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, by, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, by, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, by, true))};
  return __builtin_bit_cast(bf16x8_t, w);
}

struct Fp8 {
  // Sums of up to 2^24 weighted values stay in fp32's range under every scale. (What is
  // lost for it are weights below 2^-102 of the largest.)
  static constexpr int kTile = kTile8Bytes, kDown = 24;

  struct Unit {
    u32x4 k[2][2], v[2][2];  // [tile][half]
    uint32_t s[2];           // a tile's scale bytes: keys', values'
    int rest;                // tokens from its first one to the sequence's end
    uint32_t ok;             // bit h: tile h lies in the cache
  };

  struct Lanes {
    uint32_t codes;
  };

  static __device__ __forceinline__ Lanes lanes_of(int lane) { return Lanes{16u * lane}; }

  // Buffer resources that cover one tile (a scalar base, fixed lane offsets). 2: streamed
  // (nt), each byte is read once.
  static __device__ __forceinline__ void load(const DecodeArgs& a, const Spot& s, const Lanes& at,
                                              Unit& u) {
    u.rest = s.rest;
    u.ok = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // An id outside the cache: block 0 is read, no token of it counts.
      const bool in = (uint32_t)s.id[h] < (uint32_t)a.num_blocks;
      u.ok |= in ? 1u << h : 0u;
      const uint64_t at_tile = (uint64_t)(in ? (uint32_t)s.id[h] : 0u) * a.block_bytes + s.off[h];
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(a.cache + at_tile), 0, kTile, 0x00020000);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(a.scales + at_tile / kTile * 2), 0, 2, 0x00020000);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u.k[h][j] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at.codes + 1024 * j, 0, 2));
        u.v[h][j] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at.codes + kValueCodes8 + 1024 * j, 0, 2));
      }
      u.s[h] = __builtin_amdgcn_raw_buffer_load_b16(rs, 0, 0, 0);
    }
  }

  // -infinity for a token that does not count.
  struct Mask {
    f32x4_t bias[2];
  };

  static __device__ __forceinline__ void set_mask(Mask& m, int rest, uint32_t ok, int c, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int valid = ok >> h & 1 ? rest - h * kTileTokens : 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) m.bias[h][e] = 4 * g + e < valid ? 0.f : kNegInf;
    }
  }

  // Codes of tokens that do not count may be anything, NaN included, and so may the
  // scales of a tile without any that does.
  static __device__ __forceinline__ void take_out(Unit& u, int c, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int valid = u.ok >> h & 1 ? u.rest - h * kTileTokens : 0;
      if (valid <= 0) u.s[h] = 0x7f7fu;
      const uint32_t key = c < valid ? ~0u : 0u;
      uint32_t four = 0;  // of the lane's tokens 4g .. 4g + 3
#pragma unroll
      for (int e = 0; e < 4; ++e) four |= 4 * g + e < valid ? 0xffu << (8 * e) : 0u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u.k[h][j] &= key;
        u.v[h][j] &= four;
      }
    }
  }

  static __device__ __forceinline__ void scores(const Unit& u, const Mask& mask, const Query& q,
                                                f32x4_t (&d)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float by = __uint_as_float(u.s[h] << 23);
      d[h] = mask.bias[h];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            widen8(u.k[h][i >> 1][2 * (i & 1)], u.k[h][i >> 1][2 * (i & 1) + 1], by), q.part[i],
            d[h], 0, 0, 0);
    }
  }

  struct Values {
    const Unit& u;
    float by[2];
    __device__ __forceinline__ Values(const Unit& unit, const Mask&)
        : u(unit), by{__uint_as_float(unit.s[0] << 15), __uint_as_float(unit.s[1] << 15)} {}
    // Dims 8c + 2 byte and the next one of the unit's 8 tokens.
    template <class Byte>
    __device__ __forceinline__ void pairs(Byte, u32x4& even, u32x4& odd) const {
      constexpr int j = 2 * Byte::value;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = u.v[h][j >> 2][j & 3], y = u.v[h][j >> 2][(j & 3) + 1];
        const auto widen = [&](uint32_t w, auto upper) {
          return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
                                                  w, by[h], decltype(upper)::value));
        };
        even[2 * h] = widen(x, std::false_type{});
        even[2 * h + 1] = widen(x, std::true_type{});
        odd[2 * h] = widen(y, std::false_type{});
        odd[2 * h + 1] = widen(y, std::true_type{});
      }
    }
  };
};

}  // namespace

extern "C" size_t kv8_decode_workspace_bytes(int B, int Hq, int Hkv, int block_size, int max_blocks,
                                             int num_workgroups) {
  return decode_workspace_bytes<Fp8>(B, Hq, Hkv, block_size, max_blocks, num_workgroups);
}

extern "C" int kv8_decode_launch(const uint16_t* q, const uint8_t* cache, const uint8_t* scales,
                                 const int* block_table, const int* seq_lens, uint16_t* out, int B,
                                 int Hq, int Hkv, int num_blocks, int block_size, int max_blocks,
                                 float scale, int num_workgroups, void* workspace,
                                 size_t workspace_bytes_, hipStream_t stream) {
  if (B > 0 && num_blocks > 0 && (!scales || (reinterpret_cast<uintptr_t>(scales) & 1) != 0))
    return hipErrorInvalidValue;
  return decode_launch<Fp8>(q, cache, scales, block_table, seq_lens, out, B, Hq, Hkv, num_blocks,
                            block_size, max_blocks, scale, num_workgroups, workspace,
                            workspace_bytes_, stream);
}
