// Append to the 8-bit paged cache and its read-back (include/kv_cache8.h).
//
// The queries are normed and turned as in kv_append.hip, four tokens a wave. Keys and
// values go by tiles, because a tile's new tokens share a scale. A wave loads rows 16 lanes
// a token, 8 dims a lane. A tile's keys take a workgroup, four slots a wave: they are
// normed and turned in fp64, whose values for all 16 slots would take a wave more than the
// registers of a third of the waves (187 of them; 128 with spills); the waves' largest
// magnitudes meet in LDS. A tile's values take a wave: a lane's 8 dims of 4 slots are two
// whole 16-byte pieces of the tile. What the tile held before is only read where it has to
// be: its scale if it has older tokens, the values' pieces that new tokens share with
// others, and all older codes if the scale grows.
//   What bounds it: for a step of single tokens, latency (a request's rows and length, its
// block, the rows, the older tile: 128 requests, 32Q/8KV, 6.4 us and the read-back of their
// tiles 4.3); for prompts, HBM and the fp64 of the norm and the rotation together: 4900
// tokens of 7 ragged requests (137 MB) 31 us, 4.5 TB/s, their read-back (49 MB) 9.6 us.
// A wave for a tile's keys took 43 us there.
#include <algorithm>
#include <type_traits>

#include "kv_cache8.h"
#include "kv_common8.hpp"
#include "kv_rows.hpp"

namespace {

using namespace kv;
using gqa::wave_max;

constexpr int kWaves = 4;

typedef short i16x2_t __attribute__((ext_vector_type(2)));

// Request b's tiles stand from cu_seqlens[b] / 16 + 2b on in the launch's line of tiles,
// which holds those of the requests in front whatever their positions (n tokens touch at
// most (n + 14) / 16 + 1 tiles) and needs no sum over them.
__host__ __device__ constexpr int64_t tiles_bound(int64_t rows, int64_t B) {
  return rows / kTileTokens + 2 * B;
}

// A tile's new tokens: slots from .. to - 1 of tile `tile` of request b, slot s being
// row row0 + s of the step.
struct TileStep {
  int b, tile, from, to, row0;
};

// (The probes of the last round bring along the request's rows and length: up to 64
// requests take one round trip to memory.)
__device__ __forceinline__ TileStep find_tile(const kv_append_args& a, int unit) {
  const int lane = threadIdx.x & 63;
  TileStep s{0, 0, 0, 0, 0};
  int first, end, tokens, before;
  if (!a.cu_seqlens) {
    s.b = unit;
    first = unit, end = unit + 1, before = unit;
    tokens = __builtin_amdgcn_readfirstlane(a.seq_lens[unit]);
  } else {
    int lo = -1, hi = a.B;  // request lo's tiles start at or before `unit`, hi's do not
    first = end = tokens = before = 0;
    while (hi - lo > 1) {
      const int step = (hi - lo - 1 + 63) / 64, at = lo + 1 + lane * step;
      int from = 0, to = 0, n = 0;
      if (at < hi) from = a.cu_seqlens[at], to = a.cu_seqlens[at + 1], n = a.seq_lens[at];
      const int start = (int)tiles_bound(min(max(from, 0), a.T), at);
      const int count = __popcll(__builtin_amdgcn_ballot_w64(at < hi && start <= unit));
      hi = min(hi, lo + 1 + count * step);
      if (count > 0) {
        lo += 1 + (count - 1) * step;
        first = __builtin_amdgcn_readlane(from, count - 1);
        end = __builtin_amdgcn_readlane(to, count - 1);
        tokens = __builtin_amdgcn_readlane(n, count - 1);
        before = __builtin_amdgcn_readlane(start, count - 1);
      }
    }
    s.b = lo;
    if (lo < 0) return s;
  }
  // Row t of the request is at position len - (next - t), if that is not negative.
  const int64_t next = end, len = tokens;
  const int64_t t0 = max(max((int64_t)first, next - len), int64_t(0)), t1 = min(next, (int64_t)a.T);
  if (t0 >= t1) return s;
  const int64_t p0 = len - (next - t0), p1 = len - (next - t1);  // positions p0 .. p1 - 1
  const int64_t tile = p0 / kTileTokens + (unit - before), start = tile * kTileTokens;
  s.tile = (int)tile;
  s.row0 = (int)(start + next - len);
  s.from = (int)max(p0 - start, int64_t(0));
  s.to = (int)min(p1 - start, (int64_t)kTileTokens);
  return s;
}

// x as it is held: what is not finite becomes NaN.
__device__ __forceinline__ float held(float x) {
  return __builtin_isfinite(x) ? x : __builtin_nanf("");
}

// The scale byte for a largest magnitude: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_for(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)min(max(e, kScale8Least), kScale8Most);
}

// Four values as codes (v_cvt_scalef32_pk_fp8_f32 divides by the scale's power of two and
// rounds to the nearest code, ties to even).
__device__ __forceinline__ uint32_t encode4(float x, float y, float z, float w, float s) {
  i16x2_t c = {0, 0};
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, x, y, s, false);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, z, w, s, true);
  return __builtin_bit_cast(uint32_t, c);
}
// Four codes under a new scale.
__device__ __forceinline__ uint32_t again4(uint32_t codes, float from, float to) {
  const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, from, false);
  const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, from, true);
  return encode4(a[0], a[1], b[0], b[1], to);
}
__device__ __forceinline__ float power(uint32_t byte) { return __uint_as_float(byte << 23); }

struct Launch {
  uint8_t* codes;
  uint8_t* scales;
  unsigned k_blocks, v_blocks;  // workgroups of the keys, of the values
  unsigned q_groups;            // of the queries of 4 tokens
  unsigned units;
  FastDiv tile_div, head_div, group_div;
};

// R heads of the queries of four tokens.
template <int R>
__device__ __forceinline__ void turn_queries(const kv_append_args& a, int t, int h0, int lane) {
  const int i = lane & 15, n = min(R, a.Hq - h0);
  const bool in = t < a.T;
  uint4 raw[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    raw[j] = make_uint4(0, 0, 0, 0);
    if (in && j < n) raw[j] = load16(a.q + t * a.q_token_stride + (h0 + j) * a.q_head_stride + 8 * i);
  }
  const Place place = find_place<16>(t, a.T, a.B, a.seq_lens, a.cu_seqlens, lane);
  const bool rotate = a.rotary_dim > 0;
  const Pairs pairs = a.interleaved ? kInside : a.rotary_dim == kDim ? kHalfRow : kPartner;
  Turn turn{};
  if (rotate)
    turn = load_turn<16>(a.cos_sin, a.table_rows, a.rotary_dim, a.interleaved,
                         a.rope_positions && in ? a.rope_positions[t] : place.pos, lane);
  float w[8] = {};
  if (a.q_weight) load_weights(a.q_weight, a.q_weight_type, 8 * i, w);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    if (j >= n) break;
    float x[8];
    unpack8(raw[j], x);
    norm_turn(x, a.q_weight != nullptr, w, a.eps, turn, rotate, pairs);
    if (in)
      store16(a.q_out + t * a.q_out_token_stride + (h0 + j) * a.q_out_head_stride + 8 * i,
              place.live ? pack8(x) : make_uint4(0, 0, 0, 0));
  }
}

constexpr float kMost = 0x1.cp127f;  // 448 * 2^119

// The largest finite magnitude of a row's values in this lane, at least `top`.
__device__ __forceinline__ float larger(const float (&x)[8], float top) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float m = __builtin_fabsf(x[e]);
    top = fmaxf(top, m < __builtin_inff() ? m : 0.f);
  }
  return top;
}

// What does not fit a code as it is: infinities, and magnitudes past 448 under the largest
// scale.
__device__ __forceinline__ void bring_in(float (&x)[8]) {
  bool any = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) any |= !(__builtin_fabsf(x[e]) <= kMost);
  if (!__builtin_amdgcn_ballot_w64(any)) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = held(x[e]);
    x[e] = y > kMost ? kMost : y < -kMost ? -kMost : y;
  }
}

// A tile's place in the cache: its number among all, or -1.
__device__ __forceinline__ int64_t place_of(const kv_append_args& a, const Launch& g,
                                            const TileStep& s, int head) {
  const uint32_t lb = fastdiv((uint32_t)s.tile, g.tile_div);
  if (lb >= (uint32_t)a.max_blocks) return -1;
  const int id = __builtin_amdgcn_readfirstlane(a.block_table[(size_t)s.b * a.max_blocks + lb]);
  if ((uint32_t)id >= (uint32_t)a.num_blocks) return -1;
  return ((int64_t)id * a.Hkv + head) * g.tile_div.d + (s.tile - lb * g.tile_div.d);
}

// The keys of a tile of a head, a wave to each four slots: lane (i, group) of wave w has
// dims 8i .. +8 of slot 4w + group.
struct KeyShare {
  float top[kWaves];
  uint32_t old;
};

__device__ __forceinline__ void append_keys(const kv_append_args& a, const Launch& g, int unit,
                                            int head, int wave, int lane, KeyShare& share) {
  const TileStep s = find_tile(a, unit);
  if (s.from >= s.to) return;
  const int i = lane & 15, slot = 4 * wave + (lane >> 4);
  const bool valid = slot >= s.from && slot < s.to;
  const bool busy = 4 * wave < s.to && 4 * wave + 4 > s.from;  // the wave has a token
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (valid)
    raw = load16(a.k + (s.row0 + slot) * a.k_token_stride + head * a.k_head_stride + 8 * i);
  const bool rotate = a.rotary_dim > 0;
  Turn turn{};
  if (busy && rotate) {
    const int pos = !valid             ? 0
                    : a.rope_positions ? a.rope_positions[s.row0 + slot]
                                       : s.tile * kTileTokens + slot;
    turn = load_turn<16>(a.cos_sin, a.table_rows, a.rotary_dim, a.interleaved, pos, lane);
  }
  const int64_t at = place_of(a, g, s, head);
  if (at < 0) return;
  uint8_t* const tile = g.codes + at * kTile8Bytes;
  uint8_t* const scale_at = g.scales + 2 * at;
  const bool older = s.from > 0;
  uint32_t old = 0;
  if (older && wave == 0) old = min((uint32_t)*scale_at, (uint32_t)kScale8Most);
  float x[8];
  unpack8(raw, x);
  if (busy) {
    float w[8] = {};
    if (a.k_weight) load_weights(a.k_weight, a.k_weight_type, 8 * i, w);
    norm_turn64(x, a.k_weight != nullptr, w, a.eps, turn, rotate,
                a.interleaved ? kInside : a.rotary_dim == kDim ? kHalfRow : kPartner);
  }
  const float top = wave_max(valid ? larger(x, 0.f) : 0.f);
  if (lane == 0) share.top[wave] = top;
  if (lane == 0 && wave == 0) share.old = old;
  __syncthreads();
  const uint32_t need = scale_for(fmaxf(fmaxf(share.top[0], share.top[1]),
                                        fmaxf(share.top[2], share.top[3])));
  old = share.old;
  const uint32_t byte = older ? max(need, old) : need;
  const float by = power(byte), was = power(old);
  bring_in(x);
  if (valid)
    *reinterpret_cast<uint2*>(tile + key8_at(slot, 8 * i)) =
        make_uint2(encode4(x[0], x[1], x[2], x[3], by), encode4(x[4], x[5], x[6], x[7], by));
  // Older tokens under a scale that grows: wave w < 2 takes half w of each group of 32 dims,
  // lane (token i, group) 16 dims.
  if (older && byte > old && wave < 2 && i < s.from) {
    u32x4* const p = reinterpret_cast<u32x4*>(tile + 1024 * wave + 16 * lane);
    const u32x4 c = *p;
    *p = u32x4{again4(c[0], was, by), again4(c[1], was, by), again4(c[2], was, by),
                 again4(c[3], was, by)};
  }
  if (wave == 0 && lane == 0) *scale_at = (uint8_t)byte;
}

// The values of a tile of a head, by one wave: lane (i, group) has dims 8i .. +8 of slots
// 4 group .. +4, which are two pieces of 16 bytes of the tile.
__device__ __forceinline__ void append_values(const kv_append_args& a, const Launch& g, int unit,
                                              int head, int lane) {
  const TileStep s = find_tile(a, unit);
  if (s.from >= s.to) return;
  const int i = lane & 15, group = lane >> 4, g0 = 4 * group;
  uint4 raw[4];
  uint32_t fresh = 0, before = 0;  // bytes of a dword: new tokens, older ones
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    raw[p] = make_uint4(0, 0, 0, 0);
    if (g0 + p >= s.from && g0 + p < s.to) {
      raw[p] = load16(a.v + (s.row0 + g0 + p) * a.v_token_stride + head * a.v_head_stride + 8 * i);
      fresh |= 0xffu << (8 * p);
    }
    before |= g0 + p < s.from ? 0xffu << (8 * p) : 0u;
  }
  const int64_t at = place_of(a, g, s, head);
  if (at < 0) return;
  uint8_t* const scale_at = g.scales + 2 * at + 1;
  u32x4* const piece = reinterpret_cast<u32x4*>(g.codes + at * kTile8Bytes + kValueCodes8 +
                                                    group * 256 + i * 16);
  constexpr int kOther = 1024 / 16;  // the second piece
  const bool older = s.from > 0;
  uint32_t old = 0;
  if (older) old = min((uint32_t)*scale_at, (uint32_t)kScale8Most);
  const bool mixed = fresh != 0 && fresh != ~0u;
  u32x4 kept[2] = {};
  if (mixed) kept[0] = piece[0], kept[1] = piece[kOther];

  // (A slot without a new token has zeros.)
  float top = 0.f;
  float x[4][8];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    unpack8(raw[p], x[p]);
    top = larger(x[p], top);
  }
  const uint32_t need = scale_for(wave_max(top));
  const uint32_t byte = older ? max(need, old) : need;
  const bool grows = older && byte > old;
  const float by = power(byte), was = power(old);
  if (grows && before != 0 && !mixed) kept[0] = piece[0], kept[1] = piece[kOther];
#pragma unroll
  for (int p = 0; p < 4; ++p) bring_in(x[p]);
  if (fresh != 0 || (grows && before != 0)) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      u32x4 c;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        uint32_t o = kept[j][d];
        if (grows) o = (o & ~before) | (again4(o, was, by) & before);
        const int e = 4 * j + d;
        c[d] = (encode4(x[0][e], x[1][e], x[2][e], x[3][e], by) & fresh) | (o & ~fresh);
      }
      piece[kOther * j] = c;
    }
  }
  if (lane == 0) *scale_at = (uint8_t)byte;
}

// Workgroups: the keys', one to a tile of a head, then those of the values, a wave to a
// tile of a head, then the queries'. (The longest chains of latencies first: 4900 tokens
// 31.2 us, with the queries first 32.6.)
template <int R>
__global__ __launch_bounds__(64 * kWaves) void kv8_append_kernel(kv_append_args a, Launch g) {
  __shared__ KeyShare share;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  unsigned block = blockIdx.x;
  if (block < g.k_blocks) {
    const uint32_t unit = fastdiv(block, g.head_div);
    append_keys(a, g, (int)unit, (int)(block - unit * g.head_div.d), wave, lane, share);
    return;
  }
  block -= g.k_blocks;
  if (block < g.v_blocks) {
    const uint32_t task = block * kWaves + wave, unit = fastdiv(task, g.head_div);
    if (unit < g.units) append_values(a, g, (int)unit, (int)(task - unit * g.head_div.d), lane);
    return;
  }
  block -= g.v_blocks;
  const uint32_t tokens = fastdiv(block, g.group_div);
  const int h0 = ((int)(block - tokens * g.q_groups) * kWaves + wave) * R;
  if (h0 < a.Hq) turn_queries<R>(a, (int)tokens * 4 + (lane >> 4), h0, lane);
}

// Eight codes as bf16.
__device__ __forceinline__ uint4 decode8(uint32_t lo, uint32_t hi, float by) {
  return make_uint4(
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, by, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, by, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, by, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, by, true)));
}

// Grid: x groups of four tokens, y groups of kWaves heads; 16 lanes a token, 8 dims a lane.
__global__ __launch_bounds__(64 * kWaves) void kv8_read_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
    const int* __restrict__ block_table, const int* __restrict__ seq_lens,
    const int* __restrict__ cu_seqlens, uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out,
    int T, int B, int Hkv, int num_blocks, int block_size, int max_blocks, FastDiv bs_div) {
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
    const size_t at =
        ((size_t)block * Hkv + head) * (block_size / kTileTokens) + slot / kTileTokens;
    const uint8_t* const tile = codes + at * kTile8Bytes;
    const int s = slot % kTileTokens;
    const uint32_t both = *reinterpret_cast<const uint16_t*>(scales + 2 * at);
    const uint2 kc = *reinterpret_cast<const uint2*>(tile + key8_at(s, 8 * i));
    // The token's byte of each dim's four.
    const u32x4* const piece =
        reinterpret_cast<const u32x4*>(tile + kValueCodes8 + (s >> 2) * 256 + i * 16);
    const u32x4 lo = piece[0], hi = piece[1024 / 16];
    const uint32_t pick = 0x0c0c0000u | (uint32_t)(s & 3) * 0x0101u + 0x0400u;
    const auto four = [&](const u32x4& x) {
      const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], pick);
      const uint32_t b = __builtin_amdgcn_perm(x[3], x[2], pick);
      return a | (b << 16);
    };
    k = decode8(kc.x, kc.y, power(both & 255));
    v = decode8(four(lo), four(hi), power(both >> 8));
  }
  const size_t at = ((size_t)t * Hkv + head) * kDim + 8 * i;
  *reinterpret_cast<uint4*>(k_out + at) = k;
  *reinterpret_cast<uint4*>(v_out + at) = v;
}

// ------------------------------------------------------------------ host

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

bool sizes_fit(int T, int B, bool ragged, int Hkv, int num_blocks, int block_size, int max_blocks) {
  if (T < 0 || T > KV_MAX_TOKENS || B < 0 || B > (1 << 20) || num_blocks < 0) return false;
  if (Hkv < 1 || Hkv > 4096) return false;
  if (block_size < 1 || block_size % kTileTokens != 0 || max_blocks < 1) return false;
  return ragged || T == B;
}

bool bad_weight(const void* w, int type) {
  return w && type != KV_WEIGHT_BF16 && type != KV_WEIGHT_FP32;
}

}  // namespace

extern "C" int kv8_append_launch(const kv_append_args* args, uint8_t* codes, uint8_t* scales,
                                 hipStream_t stream) {
  if (!args) return hipErrorInvalidValue;
  const kv_append_args a = *args;
  if (!sizes_fit(a.T, a.B, a.cu_seqlens != nullptr, a.Hkv, a.num_blocks, a.block_size, a.max_blocks))
    return hipErrorInvalidValue;
  if (a.Hq < 1 || a.Hq > 4096) return hipErrorInvalidValue;
  if (a.rotary_dim < 0 || a.rotary_dim > kDim || a.rotary_dim % 16 != 0) return hipErrorInvalidValue;
  if ((a.rotary_dim > 0) != (a.cos_sin != nullptr) || a.table_rows < 0) return hipErrorInvalidValue;
  if (bad_weight(a.q_weight, a.q_weight_type) || bad_weight(a.k_weight, a.k_weight_type))
    return hipErrorInvalidValue;
  if (a.T == 0) return hipSuccess;
  if (!a.q || !a.k || !a.v || !a.q_out) return hipErrorInvalidValue;
  if (a.B > 0 && (!a.block_table || !a.seq_lens)) return hipErrorInvalidValue;
  if (a.num_blocks > 0 && (!codes || !scales || misaligned(codes, 16) || misaligned(scales, 2)))
    return hipErrorInvalidValue;
  Launch g{};
  g.codes = codes;
  g.scales = scales;
  const int64_t units = a.cu_seqlens ? tiles_bound(a.T, a.B) : a.T;
  const int64_t groups = (a.T + 3) / 4;
  g.units = (unsigned)units;
  g.tile_div = make_fastdiv((uint32_t)(a.block_size / kTileTokens));
  g.head_div = make_fastdiv((uint32_t)a.Hkv);
  // Heads of the queries a wave: as in kv_append.hip.
  const int R = groups * a.Hq <= 4096 ? 1 : 4;
  g.q_groups = (unsigned)((a.Hq + R * kWaves - 1) / (R * kWaves));
  g.group_div = make_fastdiv(g.q_groups);
  const int64_t k_blocks = units * a.Hkv, v_blocks = (k_blocks + kWaves - 1) / kWaves;
  const int64_t blocks = k_blocks + v_blocks + groups * g.q_groups;
  if (blocks * 64 * kWaves > UINT32_MAX) return hipErrorInvalidValue;  // (threads of a launch)
  g.k_blocks = (unsigned)k_blocks;
  g.v_blocks = (unsigned)v_blocks;
  if (R == 1)
    kv8_append_kernel<1><<<(unsigned)blocks, 64 * kWaves, 0, stream>>>(a, g);
  else
    kv8_append_kernel<4><<<(unsigned)blocks, 64 * kWaves, 0, stream>>>(a, g);
  return hipGetLastError();
}

extern "C" int kv8_read_launch(const uint8_t* codes, const uint8_t* scales, const int* block_table,
                               const int* seq_lens, const int* cu_seqlens, uint16_t* k_out,
                               uint16_t* v_out, int T, int B, int Hkv, int num_blocks,
                               int block_size, int max_blocks, hipStream_t stream) {
  if (!sizes_fit(T, B, cu_seqlens != nullptr, Hkv, num_blocks, block_size, max_blocks))
    return hipErrorInvalidValue;
  if (T == 0) return hipSuccess;
  if ((B > 0 && (!block_table || !seq_lens)) || !k_out || !v_out || misaligned(k_out, 16) ||
      misaligned(v_out, 16))
    return hipErrorInvalidValue;
  if (num_blocks > 0 && (!codes || !scales || misaligned(codes, 16) || misaligned(scales, 2)))
    return hipErrorInvalidValue;
  kv8_read_kernel<<<dim3((unsigned)((T + 3) / 4), (Hkv + kWaves - 1) / kWaves), 64 * kWaves, 0,
                    stream>>>(codes, scales, block_table, seq_lens, cu_seqlens, k_out, v_out, T, B,
                              Hkv, num_blocks, block_size, max_blocks,
                              make_fastdiv((uint32_t)block_size));
  return hipGetLastError();
}
