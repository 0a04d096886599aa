// Single-token GQA decode over the 4-bit paged cache (include/kv_cache.h).
//
// One wave streams a piece of one (request, kv-head): units of 32 tokens, two
// 16-token tiles of the cache, which the lanes load whole (16 bytes of key codes
// and of value codes a lane and tile) and already in the matrix cores' operand
// layouts. A unit, with lane l = (c, g) = (l % 16, l / 16):
//
//   QK^T   S[16 tok x 16 cols] = K . Q^T on 4 v_mfma_f32_16x16x32_bf16: A = the key
//          codes (lane: token c, dims 32g .. +32, 8 of them an instruction) widened
//          exactly by v_cvt_scalef32_pk_bf16_fp4, scale and all, B = the queries as
//          they are. Products are exact and their sums fp32's (off by 8e-8 of the sum
//          of magnitudes at most, measured). v_mfma_scale_f32_16x16x128_f8f6f4 would
//          take codes and scales as they lie in the cache and half the time, but it
//          wants the queries in e4m3 parts, whose lower ends get lost, and adds up
//          neighbouring products with some 14 bits below the largest (off by up to
//          1e-4 of the sum of magnitudes, measured). It is left for units with keys
//          of scale bytes 253 and 254, whose larger codes are past bf16's range.
//          Groups of up to 4 (8) q-heads have every head in four (two) columns.
//   softmax on the C layout: lane (c, g) holds tokens 4g .. 4g+3 of each tile
//          for column c.
//   PV     O^T[128 dims x 16 cols] += V^T . P^T on 8 v_mfma_f32_16x16x32_bf16,
//          contraction slot (g, e): token 4g+e of the first tile, 4g+e-4 of the
//          second, which is where the scores lie (no data crosses lanes) and
//          what a lane loads of the values: 8 dims 8c .. 8c+7 of those 8
//          tokens. v_cvt_scalef32_pk_bf16_fp4 widens them exactly, scale and
//          all. P enters as three bf16 parts, the 24 bits of its fp32 value 8 at a
//          time (nothing is cut off): a head's columns take different parts, so
//          that 1 product does for up to 4 q-heads, 2 for up to 8 and 3 for 16.
//          (Two truncated parts, 16 bits, took 1-4 % less and were off by up to
//          2^-15.)
//          The sum of the weights is one more product, with ones for V^T, so
//          that the weights that are summed are those that were multiplied.
//
// Work is shared out evenly whatever the lengths: all units of the batch in
// (request, kv-head, token) order, an equal run of them to each workgroup and
// within it to each wave. A wave finishes the segments that lie in its run;
// its cut pieces meet in LDS, those that the workgroup's run cuts in the
// workspace, where a second kernel folds them in order.
//
// What bounds it: HBM, at 136 bytes a token and kv-head. 32 requests of 8192 tokens
// (32Q/8KV, blocks of 16: 286 MB) take 48.4 us, merge launch and all (5.9 TB/s); 64
// ragged ones up to 32768 (64Q/8KV, blocks of 64: 1047 MB) 178 us (5.9 TB/s). The same
// launches with the loads alone and no arithmetic took 47 and 164 us. 8 waves a
// workgroup and one workgroup a CU, two waves a SIMD, with one unit (4352 bytes a
// wave) in flight behind the one that is folded: two units ahead 2-10 % slower, 4
// waves and two workgroups a CU 2-4 % slower at these sizes (and 3 % faster at 777
// tokens), three waves a SIMD (168 registers) 5-25 % slower, one buffer whose
// halves are refilled as they are used up 6-8 % slower. A unit costs a wave some 220
// vector instructions with everything around them and 17, 26 or 35 matrix ones
// (groups of up to 4, 8, 16 q-heads); what the two waves of a SIMD do not overlap of
// them is what the wider groups lose.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "gqa_launch.hpp"
#include "kv_cache.h"
#include "kv_decode.hpp"

namespace {

using namespace kv;
using gqa::dpp_f32;
using gqa::exp2_fast;
using gqa::kNegInf;
using gqa::wave_max;
using gqa::wave_sum;
using gqa::xor16_max;
using gqa::xor32_max;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short i16x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

constexpr int kUnit = 32;       // tokens a wave takes at a time
constexpr int kWaves = 8;       // waves of a workgroup
constexpr int kThreads = 64 * kWaves;
static_assert((kWaves & (kWaves - 1)) == 0, "heads are dealt out by masks");
constexpr int kMinUnits = 2;    // units a wave gets before another workgroup joins in

constexpr int kSlice = 4;       // requests a lane keeps the prefix sums of (8 cost 512 requests 0.7 us)

// How the units are shared out.
enum : int {
  kBalanced,    // equal runs to all workgroups, cutting segments (two launches)
  kWhole,       // the same, each workgroup's ends moved to the next segment's start
  kPerSegment,  // a workgroup for each segment, its units dealt out to the waves in turn
};

struct DecodeArgs {
  const uint16_t* q;
  const uint8_t* cache;
  const int* block_table;
  const int* seq_lens;
  uint16_t* out;
  float* states;     // [workgroups][2][heads][kPitch]
  Record* records;   // [workgroups]
  int B, Hq, Hkv, G, chunks;
  int heads;  // the most q-heads of a segment
  int num_blocks, tiles_per_block, max_blocks, capacity;
  uint32_t head_bytes, block_bytes;  // of one head's tiles in a block, of all heads'
  FastDiv tile_div;  // by tiles_per_block
  FastDiv head_div;  // by Hkv * chunks
  FastDiv chunk_div;  // by chunks
  float scale;       // |scale| log2(e)
  uint32_t flip;     // 0x80008000 for a negative scale: the queries change sign
  int mode;
};

// A unit's data in registers.
struct Unit {
  uint4 k[2], v[2];
  uint32_t ks[2], vs[2];
  int rest;     // tokens from its first one to the sequence's end
  uint32_t ok;  // bit h: tile h lies in the cache
};

struct State {
  float m;         // running maximum of the column's raw scores
  f32x4_t o[8];    // o[j][e]: dim 32g + 8e + j of column c
  f32x4_t l;       // sum of the weights (four times the same)
};

struct Query {
  bf16x8_t part[4];  // as RawQuery
};

// The queries of heads h0 .. h0 + nh - 1 of request b, head i in columns i, i + kCols,
// .. (kCols: 4, 8 or 16, the smallest that holds the group's q-heads): lane (c, g) has
// dims 32g + 8i .. +8 in w[i].
struct RawQuery {
  uint4 w[4];
};
template <int kCols>
__device__ __forceinline__ RawQuery load_query(const DecodeArgs& a, int b, int h0, int nh, int c,
                                               int g) {
  const int head = c & (kCols - 1);
  RawQuery r;
#pragma unroll
  for (int part = 0; part < 4; ++part) {
    r.w[part] = make_uint4(0, 0, 0, 0);
    if (head < nh)
      r.w[part] = *reinterpret_cast<const uint4*>(
          a.q + ((size_t)b * a.Hq + h0 + head) * kDim + 32 * g + 8 * part);
  }
  return r;
}

__device__ __forceinline__ uint32_t xor16_umax(uint32_t x) {
  const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return max((uint32_t)p[0], (uint32_t)p[1]);
}
__device__ __forceinline__ uint32_t xor32_umax(uint32_t x) {
  const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max((uint32_t)p[0], (uint32_t)p[1]);
}

// The same as the B operands. A lane with an infinity gets NaN, so that its head's
// result is NaN whatever the keys are.
__device__ __forceinline__ Query query_operands(const RawQuery& r, uint32_t flip) {
  u16x2_t most = {0, 0};
  Query q;
#pragma unroll
  for (int part = 0; part < 4; ++part) {
    const u32x4 w = {r.w[part].x, r.w[part].y, r.w[part].z, r.w[part].w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
    q.part[part] = __builtin_bit_cast(bf16x8_t, w ^ flip);
  }
  if (max((uint32_t)most.x, (uint32_t)most.y) >= 0x7f80u) q.part[0][0] = (__bf16)__builtin_nanf("");
  return q;
}

// Raw scores of two tiles by the scaled instruction, which knows no keys past its
// range: queries in two e4m3 parts, q = 2^E (hi + lo / 16) with one E a head.
__device__ __forceinline__ void far_scores(const Query& q, const uint4 (&k)[2],
                                           const uint32_t (&ks)[2], const f32x4_t (&bias)[2],
                                           f32x4_t (&d)[2]) {
  // Its B operand: lane (c, g) holds dims 16g .. +16, then 64 + 16g .. +16.
  uint32_t w[16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t x = __builtin_bit_cast(u32x4, q.part[i >> 2])[i & 3];
    const uint32_t y = __builtin_bit_cast(u32x4, q.part[2 + (i >> 2)])[i & 3];
    const auto odd = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    const auto half = __builtin_amdgcn_permlane32_swap(odd[0], odd[1], false, false);
    w[i] = half[0];
    w[8 + i] = half[1];
    top = max(max(top, w[i] & 0x7fffu), w[i] >> 16 & 0x7fffu);
    top = max(max(top, w[8 + i] & 0x7fffu), w[8 + i] >> 16 & 0x7fffu);
  }
  top = xor32_umax(xor16_umax(top));
  // E puts the largest into [128, 256); e4m3 ends at 448. (The conversions divide by
  // the exponent of their scale; a head with a NaN gets the scale NaN.)
  const int E = max((int)(top >> 7) - 127 - 7, -118);
  const float s = __uint_as_float((uint32_t)(127 + E) << 23);
  const float s16 = __uint_as_float((uint32_t)(123 + E) << 23);
  i32x8_t hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t x[2] = {w[2 * i], w[2 * i + 1]};
    i16x2_t h = {0, 0}, l = {0, 0};
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2_t, x[0]), s, false);
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2_t, x[1]), s, true);
    hi[i] = __builtin_bit_cast(int, h);
    const f32x2_t b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[i], s, false);
    const f32x2_t b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[i], s, true);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, bf16_lo(x[0]) - b0[0], bf16_hi(x[0]) - b0[1],
                                                 s16, false);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, bf16_lo(x[1]) - b1[0], bf16_hi(x[1]) - b1[1],
                                                 s16, true);
    lo[i] = __builtin_bit_cast(int, l);
  }
  const int scale_hi = top < 0x7f80u ? E + 127 : 255, scale_lo = top < 0x7f80u ? E + 123 : 255;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const i32x8_t a = {(int)k[h].x, (int)k[h].y, (int)k[h].z, (int)k[h].w, 0, 0, 0, 0};
    d[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, hi, bias[h], 4, 0, 0, (int)ks[h], 0,
                                                            scale_hi);
    d[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, lo, d[h], 4, 0, 0, (int)ks[h], 0,
                                                            scale_lo);
  }
}

// Block ids through the constant address space: scalar loads, which do not
// share a counter with the tiles' loads (as gqa_scan_mfma.hpp measured).
typedef const __attribute__((address_space(4))) int* const_ints;

// Where a unit's two tiles are to be found, the block ids on their way: nothing
// looks at them before the unit's loads go out, a unit later, so their latency
// hides behind a fold.
struct Spot {
  int id[2];
  uint32_t off[2];  // the tile's bytes in its block
  int rest;
};

// The segment a walk is in: its table row and the head's place in a block.
struct Segment {
  const_ints table;
  uint32_t head_off;
  int len;
};

__device__ __forceinline__ Segment segment_of(const DecodeArgs& a, int b, int hc, int len) {
  return Segment{(const_ints)(a.block_table + (size_t)b * a.max_blocks),
                 fastdiv((uint32_t)hc, a.chunk_div) * a.head_bytes, len};
}

__device__ __forceinline__ Spot find_unit(const DecodeArgs& a, const Segment& seg, int u) {
  Spot s;
  s.rest = seg.len - u * kUnit;
  uint32_t lb = fastdiv(2 * (uint32_t)u, a.tile_div);
  uint32_t t = 2 * (uint32_t)u - lb * a.tile_div.d;
  s.id[0] = seg.table[lb];
  s.off[0] = seg.head_off + t * kTileBytes;
  // (A second tile past the end: the first one once more, no token of it.)
  if (s.rest > kTileTokens && ++t == a.tile_div.d) t = 0, ++lb;
  s.id[1] = seg.table[lb];
  s.off[1] = seg.head_off + t * kTileBytes;
  return s;
}

// Loads through a buffer resource that covers one tile: a scalar base, fixed
// 32-bit lane offsets, no address arithmetic in vector registers. 2: streamed
// (nt), each byte is read once.
struct Lanes {
  uint32_t codes, ks, vs;  // byte offsets in each part of a tile
};

__device__ __forceinline__ void load_unit(const DecodeArgs& a, const Spot& s, const Lanes& at,
                                          Unit& u) {
  u.rest = s.rest;
  u.ok = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // An id outside the cache: block 0 is read, no token of it counts.
    const bool in = (uint32_t)s.id[h] < (uint32_t)a.num_blocks;
    u.ok |= in ? 1u << h : 0u;
    const uint8_t* p = a.cache + (uint64_t)(in ? (uint32_t)s.id[h] : 0u) * a.block_bytes + s.off[h];
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p), 0, kTileBytes, 0x00020000);
    u.k[h] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, at.codes, 0, 2));
    u.v[h] = __builtin_bit_cast(
        uint4, __builtin_amdgcn_raw_buffer_load_b128(r, at.codes + kValueCodes, 0, 2));
    u.ks[h] = __builtin_amdgcn_raw_buffer_load_b8(r, at.ks + kKeyScales, 0, 0);
    u.vs[h] = __builtin_amdgcn_raw_buffer_load_b32(r, at.vs + kValueScales, 0, 0);
  }
}

// What takes tokens out of a unit, in registers that stay the same while units
// are whole: the C operand of QK^T (-infinity for a token that does not count),
// and bytes that hide the scales of those tokens, which may be anything (255
// would make them NaN), behind the smallest one.
struct Mask {
  f32x4_t bias[2];
  uint32_t ks[2], vs[2];
};

__device__ __forceinline__ void set_mask(Mask& m, int rest, uint32_t ok, int c, int g) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int valid = ok >> h & 1 ? rest - h * kTileTokens : 0;
    m.ks[h] = c < valid ? 0xffu : 0u;
    m.vs[h] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = 4 * g + e < valid;
      m.bias[h][e] = in ? 0.f : kNegInf;
      m.vs[h] |= in ? 0xffu << (8 * e) : 0u;
    }
  }
}

__device__ __forceinline__ uint32_t select_bits(uint32_t mask, uint32_t x, uint32_t y) {
  return (x & mask) | (y & ~mask);
}

// Eight codes of one scale (exact: a code has two significant bits).
__device__ __forceinline__ bf16x8_t widen8(uint32_t codes, float by) {
  const u32x4 w = {
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, by, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, by, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, by, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, by, 3))};
  return __builtin_bit_cast(bf16x8_t, w);
}

// x without the bits of it under `mask`, exactly.
__device__ __forceinline__ float rest_of(float x, uint32_t mask) {
  return x - __uint_as_float(__float_as_uint(x) & mask);
}

// The sum of a head's columns (rotations by 8 and by 4 within the row).
template <int kCols>
__device__ __forceinline__ float sum_columns(float x) {
  if constexpr (kCols < 16) x += dpp_f32<0x128>(x);
  if constexpr (kCols < 8) x += dpp_f32<0x124>(x);
  return x;
}

// Fold a unit into the state.
template <int kCols>
__device__ __forceinline__ void fold_unit(const Unit& u, const Mask& mask, const Query& q, float scale, int c, State& st) {
  constexpr uint32_t kLow16 = 0x05040100u, kHigh16 = 0x07060302u;
  // Scale bytes to exponent fields; the bits around them do not count.
  float vs[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = select_bits(mask.vs[h], u.vs[h], 0x7f7f7f7fu);
    vs[4 * h + 0] = __uint_as_float(w << 23);
    vs[4 * h + 1] = __uint_as_float(w << 15);
    vs[4 * h + 2] = __uint_as_float(w << 7);
    vs[4 * h + 3] = __uint_as_float(w >> 1);
  }
  const uint32_t code[8] = {u.v[0].x, u.v[0].y, u.v[0].z, u.v[0].w,
                            u.v[1].x, u.v[1].y, u.v[1].z, u.v[1].w};
  const auto pairs = [&](auto byte, u32x4& even, u32x4& odd) {
    uint32_t d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      d[e] = __builtin_bit_cast(
          uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[e], vs[e], decltype(byte)::value));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      even[e] = __builtin_amdgcn_perm(d[2 * e + 1], d[2 * e], kLow16);
      odd[e] = __builtin_amdgcn_perm(d[2 * e + 1], d[2 * e], kHigh16);
    }
  };
  const uint32_t ks[2] = {select_bits(mask.ks[0], u.ks[0], 1u),
                          select_bits(mask.ks[1], u.ks[1], 1u)};
  f32x4_t d[2];
  // (255 as well: one NaN key makes all of the unit's heads NaN.)
  if (__builtin_amdgcn_ballot_w64(max(ks[0], ks[1]) >= 253u)) {
    far_scores(q, u.k, ks, mask.bias, d);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t codes[4] = {u.k[h].x, u.k[h].y, u.k[h].z, u.k[h].w};
      const float by = __uint_as_float(ks[h] << 23);
      d[h] = mask.bias[h];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        d[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(codes[i], by), q.part[i], d[h], 0, 0,
                                                       0);
    }
  }
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = d[e >> 2][e & 3];
  __builtin_amdgcn_s_setprio(1);  // (measured: 2-3 % of a long batch)
  float mx = s[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e]);
  mx = xor32_max(xor16_max(mx));
  if (__builtin_amdgcn_ballot_w64(mx > st.m)) {
    const float mn = fmaxf(st.m, mx);
    const float alpha = mn == kNegInf ? 1.f : exp2_fast((st.m - mn) * scale);
    st.m = mn;
    st.l *= alpha;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[j] *= alpha;
  }
  const float ms = st.m == kNegInf ? 0.f : st.m * scale;
  // The weights' parts: the upper 16 bits of each (truncated), then of what that
  // left of them, an exact difference. kParts products; what a column gives to them:
  //   kCols 4   columns 0-3 the first part, 4-7 the second, 8-11 the third, then none;
  //   kCols 8   columns 0-7 the first, then none, 8-15 the second, then the third;
  //   kCols 16  all columns one after the other.
  constexpr uint32_t kUpper = 0xffff0000u;
  constexpr int kParts = kCols == 4 ? 1 : kCols == 8 ? 2 : 3;
  const uint32_t first = c >= kCols ? kUpper : 0u, second = c >= 12 ? ~0u : c >= 8 ? kUpper : 0u;
  float p[kParts][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float w = exp2_fast(fmaf(s[e], scale, -ms));
    p[0][e] = kCols < 16 ? rest_of(w, first) : w;
    if constexpr (kCols == 4) p[0][e] = rest_of(p[0][e], second);
    if constexpr (kCols >= 8) p[1][e] = rest_of(p[0][e], kUpper);
    if constexpr (kCols == 16) p[2][e] = rest_of(p[1][e], kUpper);
  }
  bf16x8_t pb[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const uint32_t some = kCols == 8 && i == 1 && c < 8 ? 0u : ~0u;
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = some & __builtin_amdgcn_perm(__float_as_uint(p[i][2 * e + 1]),
                                          __float_as_uint(p[i][2 * e]), kHigh16);
    pb[i] = __builtin_bit_cast(bf16x8_t, w);
  }
  const auto two_dims = [&](auto byte) {
    constexpr int j = 2 * decltype(byte)::value;
    u32x4 even, odd;
    pairs(byte, even, odd);
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      st.o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, even), pb[i],
                                                        st.o[j], 0, 0, 0);
      st.o[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, odd),
                                                            pb[i], st.o[j + 1], 0, 0, 0);
    }
  };
  const u32x4 one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
  for (int i = 0; i < kParts; ++i)
    st.l = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, one), pb[i], st.l, 0,
                                                   0, 0);
  two_dims(std::integral_constant<int, 0>{});
  two_dims(std::integral_constant<int, 1>{});
  two_dims(std::integral_constant<int, 2>{});
  two_dims(std::integral_constant<int, 3>{});
  __builtin_amdgcn_s_setprio(0);
}

// The q-heads of segment (b, hc): h0 .. h0 + the result - 1.
__device__ __forceinline__ int heads_of(const DecodeArgs& a, int hc, int& h0) {
  const int kv_head = (int)fastdiv((uint32_t)hc, a.chunk_div);
  const int first = (hc - kv_head * a.chunks) * 16;
  h0 = kv_head * a.G + first;
  return min(16, a.G - first);
}

__device__ __forceinline__ int length_of(const DecodeArgs& a, int b) {
  return min(max(((const_ints)a.seq_lens)[b], 0), a.capacity);
}
__device__ __forceinline__ int units_of(int len) { return (int)(((uint32_t)len + kUnit - 1) / kUnit); }

// A place in the line of units: unit u of segment (b, hc), whose request has
// `len` tokens, and the units left from there on (`step` apart in the segment).
struct Walk {
  int b, hc, u, len, units, step;
  uint32_t left;
};

// The next segment (there is one).
__device__ __forceinline__ void next_segment(const DecodeArgs& a, Walk& w) {
  w.u = 0;
  if (++w.hc < a.Hkv * a.chunks) return;
  w.hc = 0;
  do w.len = length_of(a, ++w.b);
  while (w.len == 0);
  w.units = units_of(w.len);
}

// Where the walk's unit lies; then on to the next one. At the end of the run the
// last place stays (its loads are not used).
__device__ __forceinline__ void next_unit(const DecodeArgs& a, Walk& w, Segment& seg, Spot& s) {
  if (w.left == 0) return;
  s = find_unit(a, seg, w.u);
  w.u += w.step;
  if (--w.left > 0 && w.u >= w.units) {
    next_segment(a, w);
    seg = segment_of(a, w.b, w.hc, w.len);
  }
}

// Sums over the lanes up to this one (of values whose total fits 32 bits): within
// each row of 16 by DPP shifts, then the rows' totals.
template <int kShift>
__device__ __forceinline__ uint32_t add_shifted(uint32_t x) {
  return x + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x110 + kShift, 0xF, 0xF, true);
}
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x) {
  x = add_shifted<1>(x);
  x = add_shifted<2>(x);
  x = add_shifted<4>(x);
  x = add_shifted<8>(x);
  const int lane = threadIdx.x & 63;
  const uint32_t r0 = (uint32_t)__builtin_amdgcn_readlane((int)x, 15);
  const uint32_t r1 = (uint32_t)__builtin_amdgcn_readlane((int)x, 31);
  const uint32_t r2 = (uint32_t)__builtin_amdgcn_readlane((int)x, 47);
  return x + (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
}

template <int kCols>
__global__ __launch_bounds__(kThreads, 2) void kv_decode_kernel(DecodeArgs a) {
  extern __shared__ float slots[];  // [kWaves][2][heads][kPitch]
  __shared__ uint32_t prefix[kThreads];
  __shared__ uint32_t wave_total[kWaves];
  __shared__ Record meta[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int Hc = a.Hkv * a.chunks;
  const int wg = blockIdx.x, nwg = gridDim.x;

  // This wave's run of units, in two walks: `at` folds, `ahead` loads. x0 holds
  // the next unit to fold, `next` is the place of the one after it; neither walk
  // stops at a segment's end.
  Walk at{};
  Segment seg{};
  Spot next{};
  const Lanes lanes{16u * lane, (uint32_t)lane, (uint32_t)(16 * g + 4 * (c >> 2))};
  Unit x0, x1;
  RawQuery raw;
  int h0 = 0, nh = 0;  // the q-heads of the segment that raw holds
  if (a.mode == kPerSegment) {
    at.b = (int)fastdiv((uint32_t)wg, a.head_div);
    at.hc = wg - at.b * Hc;
    at.u = wave;
    at.step = kWaves;
    // The queries and the first unit are loaded before the length is known (the
    // table row is there to its end, and an id is looked at before it is used):
    // one memory latency less in a launch that has little else.
    nh = heads_of(a, at.hc, h0);
    raw = load_query<kCols>(a, at.b, h0, nh, c, g);
    if (wave < units_of(a.capacity)) {
      next = find_unit(a, segment_of(a, at.b, at.hc, a.capacity), wave);
      load_unit(a, next, lanes, x0);
    }
    at.len = length_of(a, at.b);
    at.units = units_of(at.len);
    at.left = wave < at.units ? (uint32_t)(at.units - wave + kWaves - 1) / kWaves : 0;
    x0.rest = at.len - wave * kUnit;
  } else {
    // Prefix sums of the requests' units, a slice of them to each lane: up to
    // kSlice each, every wave for itself and in registers; beyond that a slice to
    // each thread of the workgroup, through LDS.
    const bool small = a.B <= 64 * kSlice;
    const int slice = small ? (a.B + 63) / 64 : (a.B + kThreads - 1) / kThreads;
    const int first = (small ? lane : tid) * slice;
    uint32_t sum = 0, upto[kSlice];  // upto: the lane's units with request first + j
    if (small) {
      int lens[kSlice];
#pragma unroll
      for (int j = 0; j < kSlice; ++j)
        if (j < slice) lens[j] = first + j < a.B ? a.seq_lens[first + j] : 0;
#pragma unroll
      for (int j = 0; j < kSlice; ++j) {
        if (j < slice) sum += (uint32_t)units_of(min(max(lens[j], 0), a.capacity));
        upto[j] = sum;
      }
    } else {
      for (int i = 0; i < slice; ++i)
        if (first + i < a.B)
          sum += (uint32_t)units_of(min(max(a.seq_lens[first + i], 0), a.capacity));
    }
    const uint32_t inc = wave_prefix(sum);
    uint32_t base = 0, total = (uint32_t)__builtin_amdgcn_readlane((int)inc, 63);
    if (!small) {
      if (lane == 63) wave_total[wave] = inc;
      __syncthreads();
      total = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t y = wave_total[w];
        if (w < wave) base += y;
        total += y;
      }
      prefix[tid] = base + inc - sum;
      __syncthreads();
      total = (uint32_t)__builtin_amdgcn_readfirstlane((int)total);
    }
    const uint32_t all = total * (uint32_t)Hc;
    // Few units: as many workgroups as give their waves kMinUnits each.
    const uint32_t want = max(1u, (all + kWaves * kMinUnits - 1) / (kWaves * kMinUnits));
    const uint32_t used = min(want, (uint32_t)nwg);
    const uint32_t each = all / used, more = all - each * used;
    uint32_t w0 = (uint32_t)wg * each + min((uint32_t)wg, more);
    uint32_t w1 = (uint32_t)wg < used ? w0 + each + ((uint32_t)wg < more ? 1 : 0) : w0;
    at.step = 1;
    // The places of the workgroup's ends (kWhole: to move them), then of this
    // wave's start. (A segment that holds a whole share leaves it empty.)
    for (int i = a.mode == kWhole && w0 < w1 ? 0 : 2; i < 3; ++i) {
      uint32_t p = i == 0 ? w0 : w1;
      if (i == 1 && w1 == all) continue;
      if (i == 2) {
        const uint32_t share = w1 - w0;
        p = w0 + (uint32_t)((uint64_t)share * wave / kWaves);
        at.left = w0 + (uint32_t)((uint64_t)share * (wave + 1) / kWaves) - p;
        if (at.left == 0) break;
      }
      // Unit p of the line; the request is the one whose prefix sum holds unit
      // p / Hc of a single head.
      const uint32_t x = fastdiv(p, a.head_div);
      uint32_t pre;
      if (small) {
        const uint32_t before = inc - sum;
        const int in = __popcll(__builtin_amdgcn_ballot_w64(before <= x)) - 1;
        uint32_t past = 0, at_past = before;
#pragma unroll
        for (int j = 0; j < kSlice - 1; ++j) {
          const bool over = before + upto[j] <= x;  // (beyond the slice: no, as no unit x)
          past += over ? 1 : 0;
          at_past = over ? before + upto[j] : at_past;
        }
        at.b = in * slice + (int)__builtin_amdgcn_readlane((int)past, in);
        pre = (uint32_t)__builtin_amdgcn_readlane((int)at_past, in);
        at.len = length_of(a, at.b);
        at.units = units_of(at.len);
      } else {
        int found = 0;
#pragma unroll
        for (int j = 0; j < kWaves; ++j)
          found += __popcll(__builtin_amdgcn_ballot_w64(prefix[j * 64 + lane] <= x));
        pre = (uint32_t)__builtin_amdgcn_readfirstlane((int)prefix[found - 1]);
        at.b = __builtin_amdgcn_readfirstlane((found - 1) * slice);
        at.len = length_of(a, at.b);
        at.units = units_of(at.len);
        while (x - pre >= (uint32_t)at.units) {
          pre += (uint32_t)at.units;
          at.len = length_of(a, ++at.b);
          at.units = units_of(at.len);
        }
      }
      const uint32_t rem = p - pre * (uint32_t)Hc;
      at.hc = (int)(rem / (uint32_t)at.units);
      at.u = (int)(rem - (uint32_t)at.hc * (uint32_t)at.units);
      const uint32_t up = at.u > 0 ? (uint32_t)(at.units - at.u) : 0;
      if (i == 0) w0 += up;
      if (i == 1) w1 += up;
    }
  }

  Record mine{0, 0, 0, 0};
  const uint32_t slot_floats = (uint32_t)a.heads * kPitch;
  if (at.left > 0) {
    Walk ahead = at;
    seg = segment_of(a, at.b, at.hc, at.len);
    next_unit(a, ahead, seg, next);
    if (a.mode != kPerSegment) {
      // (The queries first: their conversion waits for no tile.)
      nh = heads_of(a, at.hc, h0);
      raw = load_query<kCols>(a, at.b, h0, nh, c, g);
      load_unit(a, next, lanes, x0);
    }
    next_unit(a, ahead, seg, next);
    Mask mask;
    bool unmasked = false;
    while (true) {
      int k = (int)min((uint32_t)(at.units - at.u), at.left);
      bool starts = at.u == 0, ends = at.u + k == at.units;
      if (a.mode == kPerSegment) {
        k = (int)at.left;
        starts = wave == 0;
        ends = wave == min(at.units, kWaves) - 1;
      }
      const int row = at.b * a.Hq + h0, heads = nh;
      const Query q = query_operands(raw, a.flip);
      at.left -= (uint32_t)k;
      if (at.left > 0) {  // the next segment's queries are on their way meanwhile
        next_segment(a, at);
        nh = heads_of(a, at.hc, h0);
        raw = load_query<kCols>(a, at.b, h0, nh, c, g);
      }
      State st;
      st.m = kNegInf;
      st.l = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) st.o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      // Unit x is folded while the loads of the one after it are in flight.
      const auto step = [&](const Unit& x, Unit& y) {
        load_unit(a, next, lanes, y);
        next_unit(a, ahead, seg, next);
        const bool whole = x.rest >= kUnit && x.ok == 3;
        if (!whole || !unmasked) {
          set_mask(mask, x.rest, x.ok, c, g);
          unmasked = whole;
        }
        fold_unit<kCols>(x, mask, q, a.scale, c, st);
        return --k == 0;
      };
      while (true) {
        if (step(x0, x1)) {
          x0 = x1;
          break;
        }
        if (step(x1, x0)) break;
      }
      if constexpr (kCols < 16) {
        st.l[0] = sum_columns<kCols>(st.l[0]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) st.o[j][e] = sum_columns<kCols>(st.o[j][e]);
      }
      const float l = st.l[0];
      if (starts && ends) {
        if (c < heads) {
          uint16_t* dst = a.out + (size_t)(row + c) * kDim + 32 * g;
          const float r = inverse(l);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = st.o[j][e] * r;
            *reinterpret_cast<uint4*>(dst + 8 * e) = pack8(y);
          }
        }
      } else {
        const int which = starts ? 1 : 0;
        if (which == 0) {
          mine.flags |= kHasA | (ends ? kEndsA : 0);
          mine.row_a = row;
          mine.heads |= heads;
        } else {
          mine.flags |= kHasZ;
          mine.row_z = row;
          mine.heads |= heads << 8;
        }
        if (c < heads) {
          float* dst = slots + (wave * 2 + which) * slot_floats + c * kPitch;
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < 8; j += 4)
              *reinterpret_cast<f32x4_t*>(dst + 32 * g + 8 * e + j) =
                  f32x4_t{st.o[j][e], st.o[j + 1][e], st.o[j + 2][e], st.o[j + 3][e]};
          if (g == 0) {
            dst[kDim] = st.m == kNegInf ? kNegInf : st.m * a.scale;
            dst[kDim + 1] = l;
          }
        }
      }
      if (at.left == 0) break;
    }
  }
  if (lane == 0) meta[wave] = mine;
  __syncthreads();

  // The pieces of a segment cut between waves are neighbours: a run starts
  // at a wave's second piece (Z), or at the first piece of all if the workgroup's
  // run starts inside a segment, and takes the first pieces (A) of the waves
  // after it up to the segment's end. Each head of each run is one wave's, two
  // dims a lane. Bit w of the masks is wave w's.
  const Record m = meta[min(lane, kWaves - 1)];
  const auto bits = [&](int flag) {
    return (uint32_t)__builtin_amdgcn_ballot_w64((m.flags & flag) != 0) & ((1u << kWaves) - 1);
  };
  const uint32_t has_a = bits(kHasA), ends_a = bits(kEndsA), has_z = bits(kHasZ);
  Record rec{0, 0, 0, 0};
  int turn = 0;  // heads handed out so far
  // (A first wave with a cut piece that has no A piece starts at a segment's
  // start, as those in front of it then did, empty or not.)
  const uint32_t any = has_a | has_z;
  uint32_t runs = has_z;  // the waves whose Z starts a run ..
  int which = 1, w = 0;
  if (any && (has_a >> __builtin_ctz(any) & 1)) which = 0;  // .. and the A in front
  while (which == 0 || runs) {
    w = __builtin_ctz(which ? runs : any);
    if (which) runs &= runs - 1;
    // From wave w's piece on: A pieces up to the first that ends its segment.
    const uint32_t behind = which ? ~((2u << w) - 1) : ~((1u << w) - 1);
    const uint32_t last = ends_a & behind;
    const bool ends = last != 0;
    const uint32_t upto = ends ? (last & -last) * 2 - 1 : ~0u;
    const uint32_t as = has_a & behind & upto;  // waves whose A pieces belong to it
    const int row = __builtin_amdgcn_readlane(which ? m.row_z : m.row_a, w);
    const int nh = __builtin_amdgcn_readlane(which ? m.heads >> 8 : m.heads & 255, w);
    const bool to_out = which && ends;
    if (!which) {
      rec.flags |= kHasA | (ends ? kEndsA : 0);
      rec.row_a = row;
      rec.heads = nh;
    } else if (!ends) {
      rec.flags |= kHasZ;
    }
    int h = (wave - turn) & (kWaves - 1);
    turn += nh;
    for (; h < nh; h += kWaves) {
      // Piece i: wave i's A, or piece kWaves: the Z that starts the run. A lane
      // weighs one of them; all rows are read, those of other runs left out.
      const uint32_t live = as | (which ? 1u << kWaves : 0u);
      const auto piece = [&](int i) {
        return slots + (uint32_t)(i == kWaves ? w * 2 + 1 : i * 2) * slot_floats + h * kPitch;
      };
      const int own = min(lane, kWaves);
      const float2 ml = *reinterpret_cast<const float2*>(piece(own) + kDim);
      float2 v[kWaves + 1];
#pragma unroll
      for (int i = 0; i <= kWaves; ++i) v[i] = reinterpret_cast<const float2*>(piece(i))[lane];
      const bool counts = lane <= kWaves && (live >> own & 1);
      const float M = wave_max(counts ? ml.x : kNegInf);
      const float fl = counts && M != kNegInf ? exp2_fast(ml.x - M) : 0.f;
      float L = counts ? ml.y * fl : 0.f, x = 0.f, y = 0.f;
      L = wave_sum(L);
#pragma unroll
      for (int j = 0; j <= kWaves; ++j) {
        const int i = j ? j - 1 : kWaves;  // in the order of the tokens
        const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(fl), i));
        const bool in = live >> i & 1;
        x = fmaf(in ? v[i].x : 0.f, f, x);
        y = fmaf(in ? v[i].y : 0.f, f, y);
      }
      if (to_out) {
        reinterpret_cast<uint32_t*>(a.out + (size_t)(row + h) * kDim)[lane] =
            pack2(x * inverse(L), y * inverse(L));
      } else {
        float* dst = a.states + ((size_t)wg * 2 + which) * slot_floats + h * kPitch;
        reinterpret_cast<float2*>(dst)[lane] = make_float2(x, y);
        if (lane == 0) reinterpret_cast<float2*>(dst + kDim)[0] = make_float2(M, L);
      }
    }
    which = 1;
  }
  if (a.mode == kBalanced && tid == 0) a.records[wg] = rec;

  // Requests without tokens get zeros.
  const bool alone = a.mode == kPerSegment;
  for (int b = alone ? (int)fastdiv((uint32_t)wg, a.head_div) : wg; b < a.B;
       b += alone ? a.B : nwg) {
    if (length_of(a, b) > 0) continue;
    for (int i = tid; i < a.Hq * kDim / 8; i += kThreads)
      reinterpret_cast<uint4*>(a.out + (size_t)b * a.Hq * kDim)[i] = make_uint4(0, 0, 0, 0);
  }
}

struct Shape {
  int G, chunks, heads, capacity, workgroups, mode;
};

// Short sequences keep their segments whole: one launch, no merge, for shares
// that are even only to a segment. Measured on MI355X, 32Q/8KV, block 16, whole
// against balanced: tables of 1000 tokens, 1 to 64 full requests 9.4-18.5 us
// against 10.8-19.9, 8 to 256 of U[1, 1000] 9.6-45.9 against 13.4-46.8; of 2000
// tokens 8, 32 and 64 full requests 13.8, 16.3 and 29.4 against 13.1, 19.2 and
// 29.4, 8 to 256 ragged ones 10.7-63.5 against 12.5-66.6, but a single request
// (8 segments) 13.4 against 12.2 (at 1500 tokens 11.5 against 11.9); of 4000
// tokens 1 and 8 full requests 21.0 and 21.7 against 12.2 and 16.4.
constexpr int kWholeUnits = 64, kFewWholeUnits = 48;
bool keep_whole(int64_t units, int64_t segments, int cus) {
  return units <= (4 * segments >= cus ? kWholeUnits : kFewWholeUnits);
}

bool shape_of(int B, int Hq, int Hkv, int num_blocks, int block_size, int max_blocks,
              int num_workgroups, Shape& s) {
  if (B < 0 || B > (1 << 20) || Hq < 1 || Hkv < 1 || Hq > 4096 || Hq % Hkv != 0) return false;
  if (num_blocks < 0 || block_size < 1 || block_size % kTileTokens != 0 || max_blocks < 1)
    return false;
  const int64_t cap = num_blocks == 0 ? 0 : (int64_t)block_size * max_blocks;
  s.G = Hq / Hkv;
  s.chunks = (s.G + 15) / 16;
  // Token positions and the batch's units fit 31 bits.
  if (cap > INT32_MAX - kUnit || B * ((cap + kUnit - 1) / kUnit) > INT32_MAX / (Hkv * s.chunks))
    return false;
  if ((int64_t)B * Hq > (int64_t(1) << 28)) return false;
  if ((int64_t)block_size / kTileTokens * kTileBytes * Hkv > INT32_MAX) return false;
  s.heads = std::min(s.G, 16);
  s.capacity = (int)cap;
  s.workgroups = num_workgroups;
  s.mode = kBalanced;
  if (num_workgroups <= 0) {
    s.workgroups = gqa::device_cu_count();
    const int64_t segments = (int64_t)B * Hkv * s.chunks;
    if (keep_whole((cap + kUnit - 1) / kUnit, segments, s.workgroups))
      s.mode = segments <= s.workgroups ? kPerSegment : kWhole;
    if (s.mode == kPerSegment) s.workgroups = (int)segments;
  }
  return s.workgroups <= (1 << 22);
}

size_t workspace_bytes(const Shape& s) {
  if (s.mode != kBalanced) return 0;
  return (size_t)s.workgroups * (sizeof(Record) + 2 * (size_t)s.heads * kPitch * sizeof(float));
}

}  // namespace

extern "C" size_t kv_decode_mxfp4_workspace_bytes(int B, int Hq, int Hkv, int block_size,
                                                  int max_blocks, int num_workgroups) {
  Shape s;
  if (!shape_of(B, Hq, Hkv, 1, block_size, max_blocks, num_workgroups, s) || s.workgroups < 1)
    return 0;
  return workspace_bytes(s);
}

extern "C" int kv_decode_mxfp4_launch(const uint16_t* q, const uint8_t* mxfp4_cache,
                                      const int* block_table, const int* seq_lens, uint16_t* out,
                                      int B, int Hq, int Hkv, int num_blocks, int block_size,
                                      int max_blocks, float scale, int num_workgroups,
                                      void* workspace, size_t workspace_bytes_, hipStream_t stream) {
  Shape s;
  if (!shape_of(B, Hq, Hkv, num_blocks, block_size, max_blocks, num_workgroups, s))
    return hipErrorInvalidValue;
  if (!isfinite(scale)) return hipErrorInvalidValue;
  if (B == 0) return hipSuccess;
  if (s.workgroups < 1) return hipErrorInvalidValue;
  const auto bad = [](const void* p, uintptr_t to) {
    return !p || (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0;
  };
  if (bad(q, 16) || bad(out, 16) || !block_table || !seq_lens ||
      (num_blocks > 0 && bad(mxfp4_cache, 16)))
    return hipErrorInvalidValue;
  const size_t need = workspace_bytes(s);
  if (need > 0 && (bad(workspace, 16) || workspace_bytes_ < need)) return hipErrorInvalidValue;
  DecodeArgs a{};
  a.q = q;
  a.cache = mxfp4_cache;
  a.block_table = block_table;
  a.seq_lens = seq_lens;
  a.out = out;
  a.records = static_cast<Record*>(workspace);
  a.states = need ? reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                             sizeof(Record) * s.workgroups)
                  : nullptr;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = s.G;
  a.chunks = s.chunks;
  a.heads = s.heads;
  a.num_blocks = num_blocks;
  a.tiles_per_block = block_size / kTileTokens;
  a.max_blocks = max_blocks;
  a.capacity = s.capacity;
  a.head_bytes = (uint32_t)a.tiles_per_block * kTileBytes;
  a.block_bytes = a.head_bytes * (uint32_t)Hkv;
  a.tile_div = make_fastdiv((uint32_t)a.tiles_per_block);
  a.head_div = make_fastdiv((uint32_t)(Hkv * s.chunks));
  a.chunk_div = make_fastdiv((uint32_t)s.chunks);
  // (A scale of 0 weighs all tokens alike; the smallest normal does as well and
  // keeps 0 * infinity out of the kernel.)
  a.scale = std::max(fabsf(scale) * gqa::kLog2e, 1.17549435e-38f);
  a.flip = scale < 0.f ? 0x80008000u : 0u;
  a.mode = s.mode;
  const size_t lds = (size_t)kWaves * 2 * s.heads * kPitch * sizeof(float);
  const auto kernel = s.G > 8   ? kv_decode_kernel<16>
                      : s.G > 4 ? kv_decode_kernel<8>
                                : kv_decode_kernel<4>;
  if (lds > 65536) {  // more than the default share of a CU's 160 KiB
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  kernel<<<s.workgroups, kThreads, lds, stream>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || s.mode != kBalanced) return e;
  const MergeArgs m{a.records, a.states, out, (uint32_t)s.heads * kPitch};
  return launch_decode_merge(m, s.workgroups, s.heads, stream);
}
