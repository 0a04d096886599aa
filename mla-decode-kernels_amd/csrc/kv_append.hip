// Appends to the paged caches (include/kv_cache.h): norm over each head,
// position rotation and the store of the new keys and values, in one pass over
// the step's rows; and the read-back of rows of the 4-bit cache.
//
// What bounds them is the bytes, read once and written once, once there are enough
// of them: 7255 tokens (32Q/8KV, half of each head turned) 180 MB in 35.8 us of GPU
// time, 5.0 TB/s, a plain copy of as many 5.1; below some 500 tokens the chain of latencies
// (request, length, block id, angles), 3-5 us. A wave takes four tokens, 16
// lanes (a DPP row) each, 8 dims a lane, and walks heads: the tokens' places
// and their angles (16 registers) are found once and serve every head. In
// the 4-bit cache four tokens of a request, if they are aligned, are one whole
// 256-byte line of value codes. The 4-bit append of 3880 tokens with norms moves 86 MB
// in 23 us (3.7 TB/s): fp64 costs 2 us of them, the norms 2, the search for places 1.
#include <type_traits>

#include "kv_cache.h"

#include "kv_common.hpp"

namespace {

using namespace kv;
using gqa::dpp_f32;
using gqa::row16_sum;

constexpr int kWaves = 4;  // waves of a workgroup: neighbouring head ranges of the same tokens

// Columns of the rotation of 8 dims [8i, 8i + 8): y = x c + x' s, x' the pair's
// other element, the sign of its sine in s.
struct Turn {
  float c[8], s[8];
  int partner;  // the lane (of the wave) that holds x'
  bool on;      // these dims rotate
};

// How pairs lie: neighbours in a lane, 8 lanes apart (the halves of 128 dims: a
// rotation by 8 within the DPP row, no LDS), or in lane `partner`.
enum Pairs { kInside, kHalfRow, kPartner };

// kLanes lanes hold a row of 8 kLanes dims, of which the first rot turn.
template <int kLanes>
__device__ __forceinline__ Turn load_turn(const float* __restrict__ cos_sin, int rows, int rot,
                                          int interleaved, int p, int lane) {
  Turn t;
  const int i = lane & (kLanes - 1);
  t.on = 8 * i < rot;
  t.partner = lane;
#pragma unroll
  for (int e = 0; e < 8; ++e) t.c[e] = 1.f, t.s[e] = 0.f;
  if (!t.on) return t;
  const int h = rot >> 1;
  // Column of the first pair of these dims, and the number of pairs in them.
  const int col = interleaved ? 4 * i : (8 * i < h ? 8 * i : 8 * i - h);
  if ((uint32_t)p >= (uint32_t)rows) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t.c[e] = t.s[e] = __builtin_nanf("");
  } else {
    const float* row = cos_sin + (size_t)p * rot;
    if (interleaved) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        t.c[2 * e] = t.c[2 * e + 1] = row[col + e];
        const float s = row[h + col + e];
        t.s[2 * e] = -s;
        t.s[2 * e + 1] = s;
      }
    } else {
      const bool first = 8 * i < h;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t.c[e] = row[col + e];
        const float s = row[h + col + e];
        t.s[e] = first ? -s : s;
      }
    }
  }
  if (!interleaved) t.partner = 8 * i < h ? lane + (h >> 3) : lane - (h >> 3);
  return t;
}

__device__ __forceinline__ float half_row(float x) { return dpp_f32<0x128>(x); }
__device__ __forceinline__ double half_row(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, 0x128, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), 0x128, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

// The pair's other elements of x (every lane of the wave calls this).
template <class F>
__device__ __forceinline__ void others(const F (&x)[8], F (&y)[8], const Turn& t, Pairs pairs) {
  if (pairs == kInside) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
  } else if (pairs == kHalfRow) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = half_row(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __shfl(x[e], t.partner, 64);
  }
}

// The mean of the squares of a row of 8 kLanes dims, kLanes lanes each, plus eps.
template <int kLanes>
__device__ __forceinline__ float mean_square(const float (&x)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
  return (kLanes == 16 ? row16_sum(ss) : gqa::wave_sum(ss)) * (1.f / (8 * kLanes)) + eps;
}

// x / sqrt(mean(x^2) + eps) * w. Squares can leave fp32's range on either side (values
// past 1e19, or tiny ones with next to no eps): such a row is taken again times a
// power of two. (Up: eps is below 2^-100 there, so times 2^200 it still fits.)
template <int kLanes>
__device__ __forceinline__ void norm_row(float (&x)[8], const float (&w)[8], float eps) {
  float v = mean_square<kLanes>(x, eps);
  const bool ordinary = v >= 0x1p-100f && v < __builtin_inff();
  if (__builtin_amdgcn_ballot_w64(!ordinary)) {
    const float f = ordinary ? 1.f : v < 1.f ? 0x1p100f : 0x1p-68f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f;
    v = mean_square<kLanes>(x, eps * f * f);
  }
  const float r = rsqrtf(v);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
}

// Norm over the head's 128 dims (16 lanes), then the rotation.
__device__ __forceinline__ void norm_turn(float (&x)[8], bool norm, const float (&w)[8], float eps,
                                          const Turn& t, bool rotate, Pairs pairs) {
  if (norm) norm_row<16>(x, w, eps);
  if (!rotate) return;
  float y[8];
  others(x, y, t, pairs);
  if (!t.on) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = fmaf(x[e], t.c[e], y[e] * t.s[e]);
}

// The same in fp64, for values whose rounding decides on a 4-bit code: bf16
// products are exact, the sum of 128 squares nearly, and what is left is off by
// 2^-50, far less than the chance distance to a border between two codes.
// (gfx950 runs fp64 FMAs at the rate of fp32 ones.)
__device__ __forceinline__ void norm_turn64(float (&x)[8], bool norm, const float (&w)[8],
                                            float eps, const Turn& t, bool rotate, Pairs pairs) {
  double d[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) d[e] = x[e];
  if (norm) {
    double ss = 0.;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fma(d[e], d[e], ss);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) ss += __shfl_xor(ss, o, 64);
    const double r = 1. / sqrt(ss * (1. / kDim) + (double)eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = d[e] * r * (double)w[e];
  }
  if (rotate) {
    double y[8];
    others(d, y, t, pairs);
    if (t.on) {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = fma(d[e], (double)t.c[e], y[e] * (double)t.s[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = f32_to_odd(d[e]);
}

// 8 of a group's 32 values (the other 24 in the quad's other lanes) -> their
// codes, and the group's scale byte. The scale byte is the biased exponent of the
// largest magnitude less 2, plus 1 if its significand is over 1.75: magnitudes
// up to 7 round to 6 or less, those in (7, 8) would be cut to 6, so they take
// the next scale. v_cvt_scalef32_pk_fp4_f32 divides by the scale (its exponent
// field alone counts) and rounds to the nearest code, ties to even.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));
  scale = 255u;
  if (top >= 0x7f800000u) return 0u;
  const int e = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  scale = (uint32_t)max(e, 1);
  const float s = __uint_as_float(scale << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
  return c;
}

// Weights d .. d + 7.
__device__ __forceinline__ void load_weights(const void* p, int type, int d, float (&w)[8]) {
  if (type == KV_WEIGHT_FP32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = static_cast<const float*>(p)[d + e];
  } else {
    unpack8(load16(static_cast<const uint16_t*>(p) + d), w);
  }
}

// Store 8 dims of one key or value row of the 4-bit cache. All lanes of a quad
// call it (they exchange their maxima).
__device__ __forceinline__ void store_mx(const kv_append_args& a, int block, int slot, int head,
                                         int i, bool key, const float (&x)[8]) {
  uint32_t scale;
  const uint32_t code = encode8(x, scale);
  if (block < 0) return;
  uint8_t* tile = a.mxfp4_cache + (((size_t)block * a.Hkv + head) * (a.block_size / kTileTokens) +
                                   slot / kTileTokens) * kTileBytes;
  const int s = slot % kTileTokens;
  *reinterpret_cast<uint32_t*>(tile + (key ? key_code_at(s, i) : value_code_at(s, i))) = code;
  if ((i & 3) == 0)
    tile[key ? key_scale_at(s, i >> 2) : value_scale_at(s, i >> 2)] = (uint8_t)scale;
}

// Heads a wave takes: R of the queries, of the values, and of the keys of the
// bf16 cache; one of the keys of the 4-bit cache, whose fp64 arithmetic on
// several rows at once would take the registers of half the waves. (Append and
// read-back of 3880 tokens: 29.3 us; with the keys one after the other in a loop 29.5 at
// 2 a wave and 32.9 at 4.)
template <bool kMx, int R>
struct Tasks {
  static constexpr int kKeys = kMx ? 1 : R;
  int q, k, v;
  __host__ __device__ Tasks(int Hq, int Hkv)
      : q((Hq + R - 1) / R), k((Hkv + kKeys - 1) / kKeys), v((Hkv + R - 1) / R) {}
};

// Grid: x groups of four tokens, y groups of kWaves tasks (queries, then keys, then
// values).
template <bool kMx, int R>
__global__ __launch_bounds__(64 * kWaves) void kv_append_kernel(kv_append_args a, FastDiv bs_div) {
  const int lane = threadIdx.x & 63;
  const int i = lane & 15;
  const int t = (int)blockIdx.x * 4 + (lane >> 4);
  const Tasks<kMx, R> tasks(a.Hq, a.Hkv);
  const int task = (int)blockIdx.y * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (task >= tasks.q + tasks.k + tasks.v) return;
  const bool is_q = task < tasks.q, is_k = !is_q && task < tasks.q + tasks.k;
  const int h0 = is_q ? task * R
                 : is_k ? (task - tasks.q) * tasks.kKeys
                        : (task - tasks.q - tasks.k) * R;
  const int n = min(is_k ? tasks.kKeys : R, (is_q ? a.Hq : a.Hkv) - h0);
  const bool in = t < a.T;

  // The rows' loads go out first: they need no place.
  const uint16_t* const src = is_q ? a.q : is_k ? a.k : a.v;
  const int64_t st = is_q ? a.q_token_stride : is_k ? a.k_token_stride : a.v_token_stride;
  const int64_t sh = is_q ? a.q_head_stride : is_k ? a.k_head_stride : a.v_head_stride;
  uint4 raw[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    raw[j] = make_uint4(0, 0, 0, 0);
    if (in && j < n) raw[j] = load16(src + t * st + (h0 + j) * sh + 8 * i);
  }

  const Place place = find_place<16>(t, a.T, a.B, a.seq_lens, a.cu_seqlens, lane);
  int slot;
  const int block = find_block(place, a.block_table, a.max_blocks, a.num_blocks, bs_div, slot);

  if (!is_q && !is_k) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (j >= n) break;
      if constexpr (kMx) {
        float x[8];
        unpack8(raw[j], x);
        store_mx(a, block, slot, h0 + j, i, false, x);
      } else if (block >= 0) {
        *reinterpret_cast<uint4*>(
            a.v_cache + (((size_t)block * a.block_size + slot) * a.Hkv + h0 + j) * kDim + 8 * i) =
            raw[j];
      }
    }
    return;
  }

  const bool rotate = a.rotary_dim > 0;
  const Pairs pairs = a.interleaved ? kInside : a.rotary_dim == kDim ? kHalfRow : kPartner;
  Turn turn{};
  if (rotate)
    turn = load_turn<16>(a.cos_sin, a.table_rows, a.rotary_dim, a.interleaved,
                         a.rope_positions && in ? a.rope_positions[t] : place.pos, lane);
  const void* const weight = is_q ? a.q_weight : a.k_weight;
  float w[8] = {};
  if (weight) load_weights(weight, is_q ? a.q_weight_type : a.k_weight_type, 8 * i, w);

  if (kMx && is_k) {
    float x[8];
    unpack8(raw[0], x);
    norm_turn64(x, weight != nullptr, w, a.eps, turn, rotate, pairs);
    store_mx(a, block, slot, h0, i, true, x);
    return;
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    if (j >= n) break;
    float x[8];
    unpack8(raw[j], x);
    norm_turn(x, weight != nullptr, w, a.eps, turn, rotate, pairs);
    if (is_q) {
      if (in)
        store16(a.q_out + t * a.q_out_token_stride + (h0 + j) * a.q_out_head_stride + 8 * i,
                place.live ? pack8(x) : make_uint4(0, 0, 0, 0));
    } else if (block >= 0) {
      *reinterpret_cast<uint4*>(
          a.k_cache + (((size_t)block * a.block_size + slot) * a.Hkv + h0 + j) * kDim + 8 * i) =
          pack8(x);
    }
  }
}

// Eight codes of one scale as bf16 (exact: a code has two significant bits).
__device__ __forceinline__ uint4 decode8(uint32_t code, uint32_t scale) {
  const float s = __uint_as_float(scale << 23);
  return make_uint4(
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 3)));
}

// Grid: x groups of four tokens, y groups of kWaves heads.
__global__ __launch_bounds__(64 * kWaves) void kv_read_mxfp4_kernel(
    const uint8_t* __restrict__ cache, const int* __restrict__ block_table,
    const int* __restrict__ seq_lens, const int* __restrict__ cu_seqlens,
    uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out, int T, int B, int Hkv,
    int num_blocks, int block_size, int max_blocks, FastDiv bs_div) {
  const int lane = threadIdx.x & 63, i = lane & 15;
  const int t = (int)blockIdx.x * 4 + (lane >> 4);
  const int head = (int)blockIdx.y * kWaves + (threadIdx.x >> 6);
  if (head >= Hkv) return;
  const Place place = find_place<16>(t, T, B, seq_lens, cu_seqlens, lane);
  if (t >= T) return;
  int slot;
  const int block = find_block(place, block_table, max_blocks, num_blocks, bs_div, slot);
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (block >= 0) {
    const uint8_t* tile = cache + (((size_t)block * Hkv + head) * (block_size / kTileTokens) +
                                   slot / kTileTokens) * kTileBytes;
    const int s = slot % kTileTokens;
    k = decode8(*reinterpret_cast<const uint32_t*>(tile + key_code_at(s, i)),
                tile[key_scale_at(s, i >> 2)]);
    v = decode8(*reinterpret_cast<const uint32_t*>(tile + value_code_at(s, i)),
                tile[value_scale_at(s, i >> 2)]);
  }
  const size_t at = ((size_t)t * Hkv + head) * kDim + 8 * i;
  *reinterpret_cast<uint4*>(k_out + at) = k;
  *reinterpret_cast<uint4*>(v_out + at) = v;
}

// ------------------------------------------------------------------- MLA

constexpr int kLatent = 512, kRope = 64, kRow = kLatent + kRope;

// A token's rows come in passes of a wave: the latent row (pass 0), then eight
// 64-dim rotary rows at a time, 8 lanes each (queries, then the key). A wave takes
// R passes, whose loads go out together; the token's place and angles are found
// once. Grid: x groups of kWaves tokens, one to each wave, y groups of R passes.
template <int R>
__global__ __launch_bounds__(64 * kWaves) void kv_append_mla_kernel(kv_append_mla_args a,
                                                                    FastDiv bs_div) {
  const int lane = threadIdx.x & 63;
  const int t = (int)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pass0 = (int)blockIdx.y * R;
  const int passes = 1 + (a.h_q + 8) / 8;
  const int i = lane & 7;
  if (t >= a.T) return;
  const auto row_of = [&](int j) { return (pass0 + j - 1) * 8 + (lane >> 3); };

  uint4 raw[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    raw[j] = make_uint4(0, 0, 0, 0);
    const int row = row_of(j);
    if (pass0 + j == 0)
      raw[j] = load16(a.c + t * a.c_token_stride + 8 * lane);
    else if (row < a.h_q)
      raw[j] = load16(a.q_pe + t * a.q_token_stride + row * a.q_head_stride + 8 * i);
    else if (row == a.h_q)
      raw[j] = load16(a.k_pe + t * a.k_token_stride + 8 * i);
  }

  const Place place = find_place<64>(t, a.T, a.B, a.seq_lens, a.cu_seqlens, lane);
  int slot;
  const int block = find_block(place, a.block_table, a.max_blocks, a.num_blocks, bs_div, slot);
  uint16_t* dst = a.kv_cache + ((size_t)max(block, 0) * a.block_size + slot) * kRow;
  Turn turn{};
  if (pass0 + R > 1)
    turn = load_turn<8>(a.cos_sin, a.table_rows, kRope, a.interleaved,
                        a.rope_positions ? a.rope_positions[t] : place.pos, lane);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    if (pass0 + j >= passes) break;
    float x[8];
    unpack8(raw[j], x);
    if (pass0 + j == 0) {
      if (a.c_weight) {
        float w[8];
        load_weights(a.c_weight, a.c_weight_type, 8 * lane, w);
        norm_row<64>(x, w, a.eps);
        raw[j] = pack8(x);
      }
      if (block >= 0) *reinterpret_cast<uint4*>(dst + 8 * lane) = raw[j];
      continue;
    }
    float y[8];
    others(x, y, turn, a.interleaved ? kInside : kPartner);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(x[e], turn.c[e], y[e] * turn.s[e]);
    const int row = row_of(j);
    if (row < a.h_q)
      store16(a.q_out + t * a.q_out_token_stride + row * a.q_out_head_stride + 8 * i,
              place.live ? pack8(x) : make_uint4(0, 0, 0, 0));
    else if (row == a.h_q && block >= 0)
      *reinterpret_cast<uint4*>(dst + kLatent + 8 * i) = pack8(x);
  }
}

// ------------------------------------------------------------------ host

bool bad_weight(const void* w, int type) {
  return w && type != KV_WEIGHT_BF16 && type != KV_WEIGHT_FP32;
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// (Without requests the index tensors are empty and may have no memory; the kernels
// read neither then.)
bool no_index(int B, const int* block_table, const int* seq_lens) {
  return B > 0 && (!block_table || !seq_lens);
}

// Sizes that every append and read shares.
hipError_t check_sizes(int T, int B, bool ragged, int num_blocks, int block_size, int max_blocks) {
  if (T < 0 || T > KV_MAX_TOKENS || B < 0 || num_blocks < 0) return hipErrorInvalidValue;
  if (B > (1 << 30)) return hipErrorInvalidValue;  // the search's steps fit 32 bits
  if (block_size < 1 || max_blocks < 1) return hipErrorInvalidValue;
  if (!ragged && T != B) return hipErrorInvalidValue;
  return hipSuccess;
}

hipError_t check_append(const kv_append_args& a, bool mx) {
  const hipError_t e =
      check_sizes(a.T, a.B, a.cu_seqlens != nullptr, a.num_blocks, a.block_size, a.max_blocks);
  if (e != hipSuccess) return e;
  if (a.Hq < 1 || a.Hkv < 1 || a.Hq > 4096 || a.Hkv > 4096) return hipErrorInvalidValue;
  if (mx && a.block_size % kTileTokens != 0) return hipErrorInvalidValue;
  if (a.rotary_dim < 0 || a.rotary_dim > kDim || a.rotary_dim % 16 != 0)
    return hipErrorInvalidValue;
  if ((a.rotary_dim > 0) != (a.cos_sin != nullptr) || a.table_rows < 0) return hipErrorInvalidValue;
  if (bad_weight(a.q_weight, a.q_weight_type) || bad_weight(a.k_weight, a.k_weight_type))
    return hipErrorInvalidValue;
  if (a.T == 0) return hipSuccess;
  if (!a.q || !a.k || !a.v || !a.q_out || no_index(a.B, a.block_table, a.seq_lens))
    return hipErrorInvalidValue;
  if (a.num_blocks > 0) {
    if (mx ? (!a.mxfp4_cache || misaligned(a.mxfp4_cache, 4))
           : (!a.k_cache || !a.v_cache || misaligned(a.k_cache, 16) || misaligned(a.v_cache, 16)))
      return hipErrorInvalidValue;
  }
  return hipSuccess;
}

template <bool kMx>
int append(const kv_append_args* args, hipStream_t stream) {
  if (!args) return hipErrorInvalidValue;
  const hipError_t e = check_append(*args, kMx);
  if (e != hipSuccess) return e;
  if (args->T == 0) return hipSuccess;
  const kv_append_args a = *args;
  const unsigned groups = (unsigned)((a.T + 3) / 4);
  const FastDiv bs_div = make_fastdiv((uint32_t)a.block_size);
  const auto launch = [&](auto few) {
    constexpr int R = decltype(few)::value;
    const Tasks<kMx, R> tasks(a.Hq, a.Hkv);
    kv_append_kernel<kMx, R>
        <<<dim3(groups, (tasks.q + tasks.k + tasks.v + kWaves - 1) / kWaves), 64 * kWaves, 0,
           stream>>>(a, bs_div);
  };
  // Heads a wave: with 4 a place is found for four rows, with 1 there are four times
  // as many waves to hide its latency. bf16, 32Q/8KV, norms: 128, 512 and 1024 tokens
  // 3.6, 5.4 and 8.9 us with 1, 4.7, 5.5 and 7.9 with 4 (2 and 8 at 7255 tokens: 44.9
  // and 42.2 us, with 4 41.7).
  if ((int64_t)groups * (a.Hq + 2 * a.Hkv) <= 8192)
    launch(std::integral_constant<int, 1>{});
  else
    launch(std::integral_constant<int, 4>{});
  return hipGetLastError();
}

}  // namespace

extern "C" int kv_append_launch(const kv_append_args* args, hipStream_t stream) {
  return append<false>(args, stream);
}

extern "C" int kv_append_mxfp4_launch(const kv_append_args* args, hipStream_t stream) {
  return append<true>(args, stream);
}

extern "C" int kv_read_mxfp4_launch(const uint8_t* mxfp4_cache, const int* block_table,
                                    const int* seq_lens, const int* cu_seqlens, uint16_t* k_out,
                                    uint16_t* v_out, int T, int B, int Hkv, int num_blocks,
                                    int block_size, int max_blocks, hipStream_t stream) {
  const hipError_t e = check_sizes(T, B, cu_seqlens != nullptr, num_blocks, block_size, max_blocks);
  if (e != hipSuccess) return e;
  if (Hkv < 1 || Hkv > 4096 || block_size % kTileTokens != 0) return hipErrorInvalidValue;
  if (T == 0) return hipSuccess;
  if (no_index(B, block_table, seq_lens) || !k_out || !v_out || misaligned(k_out, 16) ||
      misaligned(v_out, 16) || (num_blocks > 0 && (!mxfp4_cache || misaligned(mxfp4_cache, 4))))
    return hipErrorInvalidValue;
  kv_read_mxfp4_kernel<<<dim3((unsigned)((T + 3) / 4), (Hkv + kWaves - 1) / kWaves), 64 * kWaves, 0,
                         stream>>>(mxfp4_cache, block_table, seq_lens, cu_seqlens, k_out, v_out, T,
                                   B, Hkv, num_blocks, block_size, max_blocks,
                                   make_fastdiv(block_size));
  return hipGetLastError();
}

extern "C" int kv_append_mla_launch(const kv_append_mla_args* args, hipStream_t stream) {
  if (!args) return hipErrorInvalidValue;
  const kv_append_mla_args a = *args;
  const hipError_t e =
      check_sizes(a.T, a.B, a.cu_seqlens != nullptr, a.num_blocks, a.block_size, a.max_blocks);
  if (e != hipSuccess) return e;
  if (a.h_q < 1 || a.h_q > 4096 || a.table_rows < 0 || bad_weight(a.c_weight, a.c_weight_type))
    return hipErrorInvalidValue;
  if (a.T == 0) return hipSuccess;
  if (!a.q_pe || !a.c || !a.k_pe || !a.q_out || no_index(a.B, a.block_table, a.seq_lens) ||
      !a.cos_sin ||
      (a.num_blocks > 0 && (!a.kv_cache || misaligned(a.kv_cache, 16))))
    return hipErrorInvalidValue;
  const int passes = 1 + (a.h_q + 8) / 8;  // the latent row, then h_q + 1 rotary rows
  const FastDiv bs_div = make_fastdiv((uint32_t)a.block_size);
  const auto launch = [&](auto many) {
    constexpr int R = decltype(many)::value;
    kv_append_mla_kernel<R><<<dim3((unsigned)(a.T + kWaves - 1) / kWaves, (passes + R - 1) / R),
                              64 * kWaves, 0, stream>>>(a, bs_div);
  };
  // Passes a wave, as the heads of the GQA appends: 16 heads, 128, 1024 and 4096
  // tokens 2.9, 3.5 and 7.5 us with 1, 3.5, 3.9 and 7.1 with 4.
  if ((int64_t)a.T * passes <= 8192)
    launch(std::integral_constant<int, 1>{});
  else
    launch(std::integral_constant<int, 4>{});
  return hipGetLastError();
}
