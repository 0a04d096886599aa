// Attention of many new tokens a request (include/prefill.h).
//
// The rows of a workgroup are (token, q-head) pairs of one request and one kv-head,
// heads fastest, so that a group's heads share every key that is read and a tile of
// rows spans few tokens (which is little waste along the diagonal). A wave holds 32
// rows. Keys and values come in tiles through LDS, copied there directly
// (global_load_lds, no registers), and both products run on v_mfma_f32_32x32x16_bf16
// with the rows along the lanes, lane l = (r, h) = (l % 32, l / 32) for row r:
//
//   S^T [keys x rows] = K . Q^T    A = keys from LDS (16 bytes a lane), B = the queries,
//          which stay in registers. A lane has half of its row's scores (keys
//          8i + 4h .. +4 of 32), so the row's maximum costs one exchange of halves.
//   O^T [128 dims x rows] += V^T . P^T    A = values, read transposed from LDS
//          (ds_read_tr16_b64); B = the weights where the scores lie: contraction slot
//          (h, e) of 16 keys is key 4h + e (e < 4) or 4 + 4h + e, no data crosses
//          lanes. Factors of a row (its rescaling, 1 / l) are one register.
//
// Rows that see only part of a tile (the diagonal, the end) take a second form of the
// step, in which scores are masked and values that are not finite enter only the rows
// that see them.
//   The softmax takes one pass: scores are held against a row's reference maximum, which
// is moved (and sums rescaled) only where a tile exceeds it by 2^8, so that the sums stay
// in fp32's range and most steps rescale nothing. The weights enter the second product
// as bf16 (off by up to 2^-8 of themselves each); the sum they are divided by is of the
// rounded weights, in fp32, so that an equal error of all of them cancels. Log-sum-exps, and
// what splits weigh against each other, are of the fp32 weights.
//   Weights of two bf16 parts (off by 2^-16) take 16 matrix instructions more a step: a
// prompt of 16384 tokens 2756 us for 1876, 13 prompts and chunks 568 for 401, 32 packed prompts
// 262 for 213, one of 100 tokens 8.9 for 8.2; a request's 5 drafts behind 32000 keys 38 for 36
// and 30 of them 62 for 45, where nothing hides a step's products. All forms round alike, so
// that a request's rows come out the same whatever else is in the call (in the same splits).
//
// Tiles of 64 keys: 32 matrix instructions a wave and step, 1024 cycles of a SIMD, on
// 32 KB read from LDS. 8 waves, two to a SIMD, share a tile and run half a step apart, so
// that one's products cover the other's softmax (128 KB of LDS, keys copied three tiles
// ahead); or 4 waves with 64 KB, two such workgroups to a CU, which start and end apart and
// cost less where rows or keys are few. 16 rows a wave (16x16x32) would read twice the
// LDS per product.
//   What bounds it:
//   - a long prompt: the matrix rate and LDS. 16384 tokens (32Q/8KV, causal, 2199 GFLOP)
//     take 1.80-1.91 ms, 1.15-1.22 PFLOP/s; a library product of 8192^3 reaches 1.29 on the
//     same card. The matrix units are busy 62 % of the cycles, at some 1.8 GHz, and LDS some
//     70 %: 32 rows a wave read 128 bytes a cycle and CU for products at full rate, which is
//     all it gives. (64 rows a wave would read half, on 512 registers and one wave a SIMD,
//     whose softmax would have to go between its own products.)
//   - prompts of some 500 tokens (64Q/8KV, 32 of them, packed: 209-217 us, 0.6 PFLOP/s): starts
//     and ends of workgroups 5 tiles long (of some 29000 cycles 15000 are in the loop).
//   - drafts over long caches: HBM (16 requests, 454 MB: 93-105 us, 4.6 TB/s, the merge of the
//     splits with it).
//   - a prompt of 100 tokens (8.4 us): the chain of its loads.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "gqa_device.hpp"
#include "gqa_launch.hpp"
#include "prefill.h"

namespace {

using gqa::exp2_fast;
using gqa::FastDiv;
using gqa::fastdiv;
using gqa::kNegInf;
using gqa::make_fastdiv;
using gqa::xor32_max;
using gqa::xor32_sum;

constexpr int kDim = 128;
constexpr int kRows = 32;        // rows of a wave
constexpr int kRowBytes = 256;   // of a key or value
constexpr int kChunk = 16;       // bytes a lane copies
constexpr int kKeys = 64;        // of a tile

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
typedef u32x4_t u32x4_any __attribute__((aligned(2)));
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;
typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
typedef const __attribute__((address_space(4))) int* const_ints;

struct Args {
  const uint16_t* q;
  int64_t q_token_stride, q_head_stride;
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_token_bytes, k_head_bytes, v_token_bytes, v_head_bytes;
  int64_t block_bytes;  // paged
  uint32_t block_bytes32, token_bytes32;
  int tile_blocks, tile_slots;  // a tile's keys in whole blocks, and the slots over
  uint16_t* out;
  float* lse;
  float* states;  // [T * Hq][splits][kDim]: unnormalised sums, then [T * Hq][splits] of (m, l)
  float2* sums;
  const int* cu_q;    // (null: request b has row b; then any array in its place)
  int row_mask;       // -1, without cu_q 0
  const int* lens;    // paged: seq_lens; packed: cu_seqlens_k
  const int* ends;    // packed: the same from its second entry on
  const int* block_table;
  int T, B, Hq, Hkv, G;
  int num_blocks, block_size, max_blocks, capacity, Tk;
  int causal, splits, split_tiles;
  int sorted;  // the requests with the most keys go first
  float scale;    // |scale| log2(e)
  uint32_t flip;  // 0x80008000 for a negative scale: the queries change sign
  FastDiv group_div, bs_div, head_div;
};

__device__ __forceinline__ uint32_t pack2(float x, float y) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{x, y}, bf16x2_t));
}

// ------------------------------------------------------- which rows a workgroup has

// Segment j = 1 .. B is request j - 1; segments 0 and B + 1 are the rows in front of
// the first request and behind the last, which have no place. Segment j starts at row
// first(j) of the step and at tile first(j) * G / rows + j of the launch: an upper
// bound of the tiles in front of it that needs no sum over the requests.
struct Rows {
  int b;             // request, -1: none
  int first, n;      // its rows of the step
  int row0, rows;    // the workgroup's rows (token, head) of it: row0 .. row0 + rows - 1
  int from, length;  // its first key (packed), its keys
};

// (The last round of probes holds the first rows of the segment and of the next one: up to
// 62 requests take one round trip to memory. Its loads leave together: indexes are kept in
// the arrays, and there are no branches.)
template <int kTileRows, bool kPackedKeys>
__device__ __forceinline__ Rows find_rows(const Args& a, int unit) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = a.B + 2;  // the tile of segment lo is at or before `unit`, hi's is not
  int first = 0, next = a.T;  // first(lo), first(hi)
  int from = 0, length = 0;   // keys of lo
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 63) / 64, at = lo + 1 + lane * step;
    const int segment = min(at, a.B + 1), request = max(min(at, a.B) - 1, 0);
    const int start = a.cu_q[(segment - 1) & a.row_mask];
    const int held = a.lens[request], end = kPackedKeys ? a.ends[request] : 0;
    const int e = min(max(a.row_mask != 0 ? start : segment - 1, 0), a.T);
    const bool before = at < hi && e * a.G / kTileRows + at <= unit;
    const int key = kPackedKeys ? min(max(held, 0), a.Tk) : 0;
    const int keys = kPackedKeys ? max(min(end, a.Tk) - key, 0) : max(held, 0);
    const int count = __popcll(__builtin_amdgcn_ballot_w64(before));
    if (lo + 1 + count * step < hi && count < 64) {
      hi = lo + 1 + count * step;
      next = __builtin_amdgcn_readlane(e, count);
    }
    if (count > 0) {
      lo += 1 + (count - 1) * step;
      first = __builtin_amdgcn_readlane(e, count - 1);
      from = __builtin_amdgcn_readlane(key, count - 1);
      length = __builtin_amdgcn_readlane(keys, count - 1);
    }
  }
  Rows r;
  r.b = lo >= 1 && lo <= a.B ? lo - 1 : -1;
  r.first = first;
  r.from = from;
  r.length = length;
  r.n = max(next - r.first, 0);
  r.row0 = (unit - (r.first * a.G / kTileRows + lo)) * kTileRows;
  // (Negative for cu_seqlens out of order alone.)
  r.rows = r.row0 < 0 ? 0 : min(max(r.n * a.G - r.row0, 0), kTileRows);
  return r;
}

// The same for few requests (Args::sorted): those with the most keys go first (and of each
// request the later tiles, which see more), as the last workgroups of a launch run beside
// idle CUs. A lane has a segment; `place` counts tiles in that order and leaves no gaps.
template <int kTileRows, bool kPackedKeys>
__device__ __forceinline__ Rows find_rows_sorted(const Args& a, int place) {
  const int lane = threadIdx.x & 63, segments = a.B + 2;
  const int segment = min(lane, a.B + 1), request = min(max(segment - 1, 0), max(a.B - 1, 0));
  const int start = a.cu_q[max(segment - 1, 0) & a.row_mask];
  const int stop = a.cu_q[min(segment, a.B) & a.row_mask];
  const int held = a.lens[request], end = kPackedKeys ? a.ends[request] : 0;
  const auto within = [&](int row) { return min(max(row, 0), a.T); };
  const int first = segment == 0 ? 0 : within(a.row_mask != 0 ? start : segment - 1);
  const int next = segment > a.B ? a.T : within(a.row_mask != 0 ? stop : segment);
  const int n = lane < segments ? max(next - first, 0) : 0;
  const int tiles = (n * a.G + kTileRows - 1) / kTileRows;
  const bool real = segment >= 1 && segment <= a.B;
  const int key = kPackedKeys && real ? min(max(held, 0), a.Tk) : 0;
  const int keys = !real ? 0 : kPackedKeys ? max(min(end, a.Tk) - key, 0) : max(held, 0);
  int before = 0;  // tiles of the segments in front
  for (int j = 0; j < segments; ++j) {
    const int other = __builtin_amdgcn_readlane(keys, j);
    const int more = __builtin_amdgcn_readlane(tiles, j);
    before += other > keys || (other == keys && j < lane) ? more : 0;
  }
  const uint64_t here = __builtin_amdgcn_ballot_w64(place >= before && place - before < tiles);
  Rows r{-1, 0, 0, 0, 0, 0, 0};
  if (here == 0) return r;
  const int s = __builtin_ctzll(here);
  r.b = s >= 1 && s <= a.B ? s - 1 : -1;
  r.first = __builtin_amdgcn_readlane(first, s);
  r.n = __builtin_amdgcn_readlane(n, s);
  r.from = __builtin_amdgcn_readlane(key, s);
  r.length = __builtin_amdgcn_readlane(keys, s);
  const int ahead = place - __builtin_amdgcn_readlane(before, s);
  r.row0 = (__builtin_amdgcn_readlane(tiles, s) - 1 - ahead) * kTileRows;
  r.rows = min(r.n * a.G - r.row0, kTileRows);
  return r;
}

// ------------------------------------------------------------ tiles from memory to LDS

// lane x's 16 bytes at src + offset land at LDS byte address lds + 16 x (lds uniform;
// one wait state between the write of M0 and its use). Inline assembly, so that the
// compiler does not tie its LDS reads to these copies; they are awaited by hand.
// kStream: each byte is read once (nt).
template <bool kStream>
__device__ __forceinline__ void copy16(const uint8_t* src, uint32_t offset, uint32_t lds) {
  if constexpr (kStream)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(offset), "s"(src), "s"(lds)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(offset), "s"(src), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ void copy16(const uint8_t* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(src), "s"(lds)
               : "memory", "m0");
}

// At most kInFlight of this wave's copies are left, and its LDS accesses are done.
template <int kInFlight>
__device__ __forceinline__ void await_copies() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(kInFlight) : "memory");
}
// All waves are there, their LDS accesses done, and no access to memory moves across.
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

// The change of a phase, where nobody hands over LDS data.
__device__ __forceinline__ void change_over() { asm volatile("s_barrier" : : : "memory"); }

// x is there before what follows in the order of the program.
template <class T>
__device__ __forceinline__ void settle(T& x) {
  asm volatile("" : "+v"(x));
}

// The results of matrix instructions before this are there after it. A vector instruction
// may read one 11 wait states after its matrix instruction at the earliest. The compiler
// sees to that, but it was found to count only the longer of two ways from one to the
// other where a branch may skip instructions between them; so no branch stands between a
// matrix instruction and this.
__device__ __forceinline__ void matrix_done(f32x16_t& x) {
  asm volatile("s_nop 15" : "+v"(x));
}
template <int kN>
__device__ __forceinline__ void matrix_done(f32x16_t (&x)[kN], f32x16_t (&o)[4]) {
  if constexpr (kN == 2)
    asm volatile("s_nop 15"
                 : "+v"(x[0]), "+v"(x[1]), "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]));
  else
    asm volatile("s_nop 15" : "+v"(x[0]), "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]));
}

// How keys are found. kPaged: the keys of a tile that a wave copies share a block, so one
// scalar block id serves them; kGather: blocks of any size; kPacked: rows.
enum Source { kPaged, kGather, kPacked };

// The keys of one (request, kv-head): n of them.
struct Keys {
  const uint8_t* k;
  const uint8_t* v;
  const_ints table;
  int n, last_block;
};

template <Source kSource>
__device__ __forceinline__ Keys keys_of(const Args& a, const Rows& r, int kv_head) {
  Keys s{};
  if constexpr (kSource == kPacked) {
    s.n = r.length;
    s.k = a.k + r.from * a.k_token_bytes + kv_head * a.k_head_bytes;
    s.v = a.v + r.from * a.v_token_bytes + kv_head * a.v_head_bytes;
  } else {
    s.n = min(r.length, a.capacity);
    s.k = a.k + kv_head * a.k_head_bytes;
    s.v = a.v + kv_head * a.v_head_bytes;
    s.table = (const_ints)(a.block_table + (size_t)r.b * a.max_blocks);
    s.last_block = s.n > 0 ? (int)fastdiv((uint32_t)s.n - 1, a.bs_div) : 0;
  }
  return s;
}

// The byte offset of key `key` (paged; an id outside the cache: block 0).
__device__ __forceinline__ int64_t paged_offset(const Args& a, const Keys& s, int key) {
  const uint32_t lb = fastdiv((uint32_t)key, a.bs_div);
  const uint32_t id = (uint32_t)s.table[lb];
  return (id < (uint32_t)a.num_blocks ? id : 0u) * a.block_bytes +
         (int64_t)(key - (int)(lb * a.bs_div.d)) * a.k_token_bytes;
}

// A walk through the tiles that copies a wave's kRun rows of each, of the keys and later of
// the values. Rows behind the last key are any of the cache's, or the last one's.
//   A copy takes 4 rows. The rows' bytes from the run's first, and the 16-byte chunk of its
// row that belongs where a lane writes, are in a register for each copy.
//   kPaged: the run's block and slot are kept and moved on (kKeys = `tile_blocks` blocks and
// `tile_slots`), the block's id is loaded a tile ahead, and the offset found for the keys
// serves the values.
template <Source kSource, bool kStream, int kRun>
struct Feed {
  static constexpr int kCopies = kRun / 4;
  uint32_t k_at[kCopies], v_at[kCopies];  // a lane's byte (kGather: from its own row's start)
  int key;                                // the run's first key in the next tile of keys
  int block, slot, id;                    // kPaged: its block, slot in it, the block's id
  int64_t at;                             // kPaged: its offset in the tile before

  __device__ __forceinline__ void begin(const Args& a, const Keys& s, int tile, int run, int lane) {
    const uint32_t row = (lane >> 4) & 3, chunk = lane & 15;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const uint32_t r = 4 * i + row;
      k_at[i] = (chunk ^ ((4 * (run / 4 + i) + row) & 15)) * kChunk;
      v_at[i] = (chunk ^ (row << 2)) * kChunk;
      if (kSource != kGather) {
        k_at[i] += r * (uint32_t)a.k_token_bytes;
        v_at[i] += r * (uint32_t)a.v_token_bytes;
      }
    }
    key = tile * kKeys + run;
    if constexpr (kSource == kPaged) {
      block = (int)fastdiv((uint32_t)key, a.bs_div);
      slot = key - block * (int)a.bs_div.d;
      id = s.table[min(block, s.last_block)];
    }
  }

  // Copies the run's keys of the next tile to `lds` on.
  __device__ __forceinline__ void keys(const Args& a, const Keys& s, uint32_t lds) {
    if constexpr (kSource == kPaged) {
      const uint32_t b = (uint32_t)id < (uint32_t)a.num_blocks ? (uint32_t)id : 0u;
      at = (int64_t)((uint64_t)b * a.block_bytes32 + (uint32_t)slot * a.token_bytes32);
      const uint8_t* const from = s.k + at;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy16<kStream>(from, k_at[i], lds + i * 4 * kRowBytes);
      block += a.tile_blocks;
      slot += a.tile_slots;
      if (slot >= (int)a.bs_div.d) slot -= (int)a.bs_div.d, ++block;
      id = s.table[min(block, s.last_block)];
    } else {
      copy_rows(a, s, s.k, key, a.k_token_bytes, k_at, lds);
    }
    key += kKeys;
  }
  // The same of the values of the tile whose keys were copied last.
  __device__ __forceinline__ void values(const Args& a, const Keys& s, uint32_t lds) {
    if constexpr (kSource == kPaged) {
      const uint8_t* const from = s.v + at;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy16<kStream>(from, v_at[i], lds + i * 4 * kRowBytes);
    } else {
      copy_rows(a, s, s.v, key - kKeys, a.v_token_bytes, v_at, lds);
    }
  }

 private:
  __device__ __forceinline__ void copy_rows(const Args& a, const Keys& s, const uint8_t* src,
                                            int first, int64_t token_bytes,
                                            const uint32_t (&lane_at)[kCopies], uint32_t lds) {
    const uint32_t row = (threadIdx.x >> 4) & 3;
    const int last = s.n - 1;
    if (kSource == kPacked && first + kRun <= s.n) {
      const uint8_t* const from = src + first * token_bytes;
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        copy16<kStream>(from, lane_at[i], lds + i * 4 * kRowBytes);
      return;
    }
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const uint32_t to = lds + i * 4 * kRowBytes;
      if constexpr (kSource == kGather) {
        int64_t from[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) from[r] = paged_offset(a, s, min(first + 4 * i + r, last));
        const int64_t lo = row & 1 ? from[1] : from[0], hi = row & 1 ? from[3] : from[2];
        copy16(src + (row & 2 ? hi : lo) + lane_at[i], to);
      } else {  // (rows behind the last one: the last one's)
        const int from = min(first, last);
        const uint32_t r = 4 * i + row;
        const uint32_t over = r - min(r, (uint32_t)(last - from));
        copy16<kStream>(src + from * token_bytes, lane_at[i] - over * (uint32_t)token_bytes, to);
      }
    }
  }
};

// ------------------------------------------------------------------------ a wave's work

constexpr float kSlack = 8.f;
// Weights are 2^-kDown of the usual, so that sums of 2^24 weighted values of any magnitude
// stay in fp32's range, by kSlack as well. (What is lost for it are weights below 2^-94 of
// the reference's.)
constexpr float kDown = 32.f, kUp = 0x1p32f;

struct State {
  float m;           // reference of the row's weights (a raw score)
  float l, fine;     // their sums in this half: as they are multiplied, and in fp32
  f32x16_t o[4];     // o[d][i]: dim 32d + 8(i / 4) + 4h + i % 4
};

// LDS layout of a tile: rows of 256 bytes whose 16-byte chunks are permuted, for keys by
// the row's last four bits (32 rows read at one chunk hit all banks), for values by its
// last two (a transposed read takes 64 bytes of 4 rows).
struct Lanes {
  uint32_t k[8];  // the lane's 16 bytes of key l % 32 at each step
  uint32_t v[4];  // the lane's 8 bytes of values, dims 32d ..
};

__device__ __forceinline__ Lanes lanes_of(int lane, uint32_t keys, uint32_t values) {
  const int j = lane & 15, g = lane >> 4, h = lane >> 5;
  Lanes at;
#pragma unroll
  for (int step = 0; step < 8; ++step)
    at.k[step] = keys + (lane & 31) * kRowBytes + ((h ^ j) ^ (2 * step)) * kChunk;
#pragma unroll
  for (int d = 0; d < 4; ++d)
    at.v[d] = values + (4 * h + (j >> 2)) * kRowBytes +
              (((4 * d + 2 * (g & 1) + ((j & 3) >> 1)) ^ ((j >> 2) << 2)) * kChunk) + 8 * (j & 1);
  return at;
}

__device__ __forceinline__ bf16x8_t lds_key(uint32_t addr) {
  return __builtin_bit_cast(bf16x8_t, *(const lds_u32x4_t*)(uintptr_t)addr);
}
__device__ __forceinline__ bf16x8_t lds_values(uint32_t addr) {
  const bf16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t*)(uintptr_t)addr);
  const bf16x4_t y =
      __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t*)(uintptr_t)(addr + 8 * kRowBytes));
  return bf16x8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
}

__device__ __forceinline__ f32x16_t mfma(bf16x8_t x, bf16x8_t y, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
}

// The raw scores of a tile: s[b][i] is key 32b + 8(i / 4) + 4h + i % 4 of it.
template <int kBlocks>
__device__ __forceinline__ void scores(uint32_t slot, const Lanes& at, const bf16x8_t (&q)[8],
                                       f32x16_t (&s)[kBlocks]) {
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
  for (int step = 0; step < 8; ++step) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
      s[b] = mfma(lds_key(at.k[step] + (slot + b * 32 * kRowBytes)), q[step], s[b]);
  }
}

// Takes out the keys that the lane's row does not see: those from `seen` on, counted from
// the tile's first, and those not in `in`.
template <int kBlocks>
__device__ __forceinline__ void take_out(f32x16_t (&s)[kBlocks], int seen, uint64_t in) {
  const int h4 = (threadIdx.x & 32) >> 3;  // 4h
  const int below = seen - h4;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[b][i] = 32 * b + 8 * (i / 4) + i % 4 < below ? s[b][i] : kNegInf;
  if (~in == 0) return;
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const uint32_t mine = (uint32_t)(in >> (32 * b + h4));
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[b][i] = mine >> (8 * (i / 4) + i % 4) & 1 ? s[b][i] : kNegInf;
  }
}

// A row's reference as weights are held against it, in units of log2.
__device__ __forceinline__ float reference(float m, float scale) {
  return m == kNegInf ? 0.f : fmaf(m, scale, kDown);
}

// The weights of a tile as matrix operands, rounded to bf16 (off by 2^-8 of each at most);
// their sum is taken of what is multiplied, so that rows of equal values come out exact. The
// sum of the fp32 weights, for log-sum-exps and splits, is taken beside it with kFine, which
// the loop over whole tiles has a form of its own for: 32 additions a lane and step cost a
// prompt of 16384 tokens 2 % and a branch around them 4 chunks 2 %. (The few tiles that are
// seen in part have them always.)
template <int kBlocks, bool kFine>
__device__ __forceinline__ void soften(const f32x16_t (&s)[kBlocks], float scale, State& st,
                                       uint32_t (&p)[kBlocks * 8]) {
  float mx = s[0][0];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
  mx = xor32_max(mx);
  // The reference is the maximum so far, or up to 2^kSlack of weight below it: weights of
  // more than 1 do no harm, and a row's reference is seldom moved after its first tiles.
  if (__builtin_amdgcn_ballot_w64(!((mx - st.m) * scale <= kSlack))) {
    const float m = fmaxf(st.m, mx);
    const float alpha = m == kNegInf ? 1.f : exp2_fast((st.m - m) * scale);
    const bool first = __builtin_amdgcn_ballot_w64(st.m != kNegInf) == 0;
    st.m = m;
    if (!first) {  // (else there is nothing yet)
      st.l *= alpha;
      if constexpr (kFine) st.fine *= alpha;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[d][i] *= alpha;
    }
  }
  const float ms = reference(st.m, scale);
  float sum = 0.f;
  const bf16x2_t ones = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = exp2_fast(fmaf(s[b][2 * i], scale, -ms));
      const float y = exp2_fast(fmaf(s[b][2 * i + 1], scale, -ms));
      if constexpr (kFine) sum += x + y;
      p[8 * b + i] = pack2(x, y);
      st.l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, p[8 * b + i]), ones, st.l,
                                             false);
    }
  if constexpr (kFine) st.fine += sum;
}

template <int kWords>
__device__ __forceinline__ bf16x8_t weights_of(const uint32_t (&p)[kWords], int t) {
  return __builtin_bit_cast(bf16x8_t, u32x4_t{p[4 * t], p[4 * t + 1], p[4 * t + 2], p[4 * t + 3]});
}

template <int kBlocks>
__device__ __forceinline__ void accumulate(uint32_t slot, const Lanes& at,
                                           const uint32_t (&p)[kBlocks * 8], State& st) {
#pragma unroll
  for (int t = 0; t < 2 * kBlocks; ++t)
#pragma unroll
    for (int d = 0; d < 4; ++d)
      st.o[d] = mfma(lds_values(at.v[d] + (slot + t * 16 * kRowBytes)), weights_of(p, t), st.o[d]);
}

// The scores of a first tile, operands read eight ahead.
template <int kBlocks>
__device__ __forceinline__ void first_scores(uint32_t slot, const Lanes& at,
                                             const bf16x8_t (&q)[8], f32x16_t (&s)[kBlocks]) {
  constexpr int kMatrix = 0x008, kRead = 0x100;
  scores(slot, at, q, s);
  __builtin_amdgcn_sched_group_barrier(kRead, 8, 0);
#pragma unroll
  for (int i = 0; i < 8 * kBlocks - 8; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMatrix, 8, 0);
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) matrix_done(s[b]);
}

// Both products of a step, the tile's weights with its values and the next tile's keys with
// the queries, in one run of matrix instructions whose operands are read from LDS six ahead
// (read one ahead, as the compiler has it, they wait some 100 of 130 cycles each).
__device__ __forceinline__ void products(uint32_t slot, uint32_t next_slot, const Lanes& at,
                                         const bf16x8_t (&q)[8], const uint32_t (&p)[16],
                                         f32x16_t (&s)[2], State& st) {
  accumulate<2>(slot, at, p, st);
  scores(next_slot, at, q, s);
  constexpr int kMatrix = 0x008, kRead = 0x100;
  __builtin_amdgcn_sched_group_barrier(kRead, 12, 0);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMatrix, 6, 0);
  matrix_done(s, st.o);
}

// Whether 16 bytes of values hold an infinity or NaN.
__device__ __forceinline__ bool not_finite(u32x4_t w) {
  u16x2_t most = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
  return max((uint32_t)most.x, (uint32_t)most.y) >= 0x7f80u;
}

// The product of a last tile.
__device__ __forceinline__ void last_product(uint32_t slot, const Lanes& at,
                                             const uint32_t (&p)[16], State& st) {
  constexpr int kMatrix = 0x008, kRead = 0x100;
  accumulate<2>(slot, at, p, st);
  __builtin_amdgcn_sched_group_barrier(kRead, 12, 0);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMatrix, 6, 0);
#pragma unroll
  for (int d = 0; d < 4; ++d) matrix_done(st.o[d]);
}

// Values that are not finite, in tiles that some row does not see whole, where a weight of
// 0 would make NaN of them for that row: they are replaced by 0 in LDS, and the first key
// with one is kept for each dim. A row that sees it gets NaN in that dim in the end.
struct Spoilt {
  int key[kDim];
  int any;
};

__device__ __forceinline__ void begin_spoilt(Spoilt& x) {
  if (threadIdx.x < kDim) x.key[threadIdx.x] = INT32_MAX;
  if (threadIdx.x == 0) x.any = 0;
}

// The 16 bytes of LDS at `at`: dims 8 chunk .. +8 of key `key`.
__device__ __forceinline__ void clean(const Args& a, const Keys& s, bool strange, uint32_t at,
                                      int key, int chunk, Spoilt& spoilt) {
  u32x4_t w = *(const lds_u32x4_t*)(uintptr_t)at;
  if (!not_finite(w)) return;
  bool counts = key < s.n;
  if (counts && strange)
    counts = (uint32_t)s.table[fastdiv((uint32_t)key, a.bs_div)] < (uint32_t)a.num_blocks;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t bits = 0x7f80u << (16 * (e & 1));
    if ((w[e / 2] & bits) != bits) continue;
    w[e / 2] &= e & 1 ? 0xffffu : 0xffff0000u;
    if (counts) {
      atomicMin(&spoilt.key[8 * chunk + e], key);
      spoilt.any = 1;
    }
  }
  *(lds_u32x4_t*)(uintptr_t)at = w;
}

// The row that sees the keys below `seen`.
__device__ __forceinline__ void spoil(const Spoilt& spoilt, int seen, State& st) {
  if (!spoilt.any) return;
  const int h4 = (threadIdx.x & 32) >> 3;  // 4h
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (spoilt.key[32 * d + 8 * (i / 4) + h4 + i % 4] < seen) st.o[d][i] = __builtin_nanf("");
}

// What is not finite as NaN. Finite values do not overflow, so it comes of values that are not,
// whose tile the row sees whole: they were multiplied, and infinities may have stayed such.
__device__ __forceinline__ float number(float x) { return fmaf(x, 0.f, x); }

// The natural logarithm of a sum of weights held against `ref` (2^-kDown of the usual).
__device__ __forceinline__ float log_sum(float ref, float sum) {
  return sum == 0.f ? kNegInf : ((ref - kDown) + __log2f(sum * kUp)) * gqa::kLn2;
}

// A row's result: to out and lse, or to the states of split `split`. A split's sums of values
// are brought from the rounded weights' sum to the fp32 weights', by which the splits are
// weighed against each other.
__device__ __forceinline__ void store_row(const Args& a, int row, int split, const State& st,
                                          bool valid) {
  const int h = (threadIdx.x >> 5) & 1;
  const float m = st.m, l = st.l;
  const f32x16_t(&o)[4] = st.o;
  if (a.splits > 1) {
    if (!valid) return;
    const float f = st.fine / l;
    const size_t at = (size_t)row * a.splits + split;
    float* dst = a.states + at * kDim;
    if (!(m == kNegInf && l == 0.f))  // (else nobody reads it)
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f32x4_t*>(dst + 32 * d + 2 * i + 4 * h) =
            f32x4_t{o[d][i] * f, o[d][i + 1] * f, o[d][i + 2] * f, o[d][i + 3] * f};
    if (h == 0) a.sums[at] = make_float2(m == kNegInf ? kNegInf : reference(m, a.scale), st.fine);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = a.out + (size_t)row * kDim;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      uint32_t x[2], y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[e] = pack2(number(o[d][i + 2 * e] * inv), number(o[d][i + 2 * e + 1] * inv));
        y[e] = pack2(number(o[d][i + 4 + 2 * e] * inv), number(o[d][i + 4 + 2 * e + 1] * inv));
      }
      // Half h gets all 8 dims of group i / 4 + h.
      const auto p0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
      const auto p1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
      if (valid)
        *reinterpret_cast<u32x4_t*>(dst + 32 * d + 2 * i + 8 * h) =
            u32x4_t{p0[0], p1[0], p0[1], p1[1]};
    }
  if (a.lse && valid && h == 0) a.lse[row] = log_sum(reference(m, a.scale), st.fine);
}

// The arguments that a workgroup's start needs, in registers from here on: the compiler loads
// each where it is first used, otherwise, and waits for it there.
__device__ __forceinline__ void fetch(const FastDiv& f) {
  asm volatile("" : : "s"(f.d), "s"(f.mul), "s"(f.shift));
}
template <Source kSource>
__device__ __forceinline__ void fetch(const Args& a, int units) {
  asm volatile("" : : "s"(units), "s"(a.cu_q), "s"(a.row_mask), "s"(a.lens), "s"(a.T), "s"(a.B),
               "s"(a.G), "s"(a.Hkv), "s"(a.causal), "s"(a.sorted), "s"(a.k), "s"(a.v), "s"(a.k_head_bytes),
               "s"(a.v_head_bytes), "s"(a.k_token_bytes), "s"(a.v_token_bytes));
  if constexpr (kSource == kPacked)
    asm volatile("" : : "s"(a.ends), "s"(a.Tk));
  else
    asm volatile("" : : "s"(a.block_table), "s"(a.num_blocks), "s"(a.max_blocks), "s"(a.capacity),
                 "s"(a.split_tiles));
  if constexpr (kSource == kPaged)
    asm volatile("" : : "s"(a.block_bytes32), "s"(a.token_bytes32), "s"(a.tile_blocks),
                 "s"(a.tile_slots));
  asm volatile("" : : "s"(a.q), "s"(a.q_token_stride), "s"(a.q_head_stride), "s"(a.flip),
               "s"(a.scale), "s"(a.lse), "s"(a.splits));
  fetch(a.head_div);
  fetch(a.group_div);
  if constexpr (kSource != kPacked) fetch(a.bs_div);
}

// What a workgroup works on, and this lane's row of it.
struct Work {
  Rows rows;
  Keys keys;
  int kv_head, split;
  bool valid;         // the lane's row is one
  int token, head;    // of the lane's row: the request's token, the q-head
  int seen;           // keys that the row sees
  int most;           // that any row sees
  int t0, t1;         // this split's tiles of kKeys keys
  int whole;          // of those the ones that all rows see whole
  int full, part;     // the ones that this wave's rows see whole, and at all
  bool strange;       // a block id outside the cache among them
};

// Rows row_wave * 32 .. +32 of the workgroup's tile of kTileRows are this wave's.
template <int kTileRows, Source kSource>
__device__ __forceinline__ Work begin(const Args& a, int units, int row_wave) {
  const int lane = threadIdx.x & 63;
  Work w{};
  // Later tiles of rows see more keys: they go first.
  const int from_end = (int)fastdiv(blockIdx.x, a.head_div);
  w.kv_head = (int)blockIdx.x - from_end * a.Hkv;
  w.split = blockIdx.y;
  w.rows = a.sorted
               ? find_rows_sorted<kTileRows, kSource == kPacked>(a, from_end)
               : find_rows<kTileRows, kSource == kPacked>(a, units - 1 - from_end);
  if (w.rows.rows == 0) return w;
  const int mine = row_wave * kRows + (lane & 31);
  w.valid = mine < w.rows.rows;
  const uint32_t row = (uint32_t)(w.rows.row0 + min(mine, w.rows.rows - 1));
  w.token = (int)fastdiv(row, a.group_div);
  w.head = w.kv_head * a.G + (int)(row - (uint32_t)w.token * a.G);
  if (w.rows.b < 0) return w;

  w.keys = keys_of<kSource>(a, w.rows, w.kv_head);
  const int length = w.rows.length;
  // Keys that a row sees: those up to its position, all, or none without a place.
  const auto seen_by = [&](int token) {
    const int p = length - w.rows.n + token;
    return p < 0 ? 0 : a.causal ? min(p + 1, w.keys.n) : w.keys.n;
  };
  const auto seen_at = [&](int r) {
    return __builtin_amdgcn_readfirstlane(
        seen_by((int)fastdiv((uint32_t)(w.rows.row0 + r), a.group_div)));
  };
  w.seen = seen_by(w.token);
  const int first = row_wave * kRows, end = min(first + kRows, w.rows.rows);
  w.most = seen_at(w.rows.rows - 1);
  // Paged: splits of equal numbers of keys for all requests, those of the longest that the
  // table holds (short requests leave the later ones empty); packed, where nobody knows it:
  // of equal parts of each request.
  const int all = (w.most + kKeys - 1) / kKeys;
  const int each = kSource == kPacked ? (all + a.splits - 1) / a.splits : a.split_tiles;
  w.t0 = (int)min((int64_t)w.split * each, (int64_t)all);
  w.t1 = min(w.t0 + each, all);
  w.whole = min(max(seen_at(0) / kKeys, w.t0), w.t1);
  if (first < end) {
    w.full = min(max(seen_at(first) / kKeys, w.t0), w.t1);
    w.part = min(max((seen_at(end - 1) + kKeys - 1) / kKeys, w.full), w.t1);
  } else {
    w.full = w.part = w.t0;
  }
  return w;
}

// Looks for block ids outside the cache (there should be none); with one, every tile asks
// for its own. All waves meet here.
template <int kThreads, Source kSource>
__device__ __forceinline__ void look_at_blocks(const Args& a, Work& w) {
  if constexpr (kSource == kPacked) {
    __syncthreads();
  } else {
    const int b0 = (int)fastdiv((uint32_t)w.t0 * kKeys, a.bs_div);
    const int b1 = (int)fastdiv((uint32_t)min(w.t1 * kKeys, w.most) - 1, a.bs_div);
    const int* table = a.block_table + (size_t)w.rows.b * a.max_blocks;
    bool bad = false;
    for (int i = b0 + (int)threadIdx.x; i <= b1; i += kThreads)
      bad |= (uint32_t)table[i] >= (uint32_t)a.num_blocks;
    w.strange = __builtin_amdgcn_readfirstlane(__syncthreads_or(bad)) != 0;
    if (w.strange) w.full = w.whole = w.t0;
  }
}

// The keys of tile `tile` that lie in blocks of the cache.
__device__ __forceinline__ uint64_t keys_in_cache(const Args& a, const Work& w, int tile) {
  if (!w.strange) return ~0ull;
  const int key = min(tile * kKeys + (int)(threadIdx.x & (kKeys - 1)), w.keys.n - 1);
  const int id = w.keys.table[fastdiv((uint32_t)key, a.bs_div)];
  return __builtin_amdgcn_ballot_w64((uint32_t)id < (uint32_t)a.num_blocks);
}

// Whether the lane's row sees a key of this split at all, of one whose scores were all
// -infinity if they were there. (The whole wave calls this.)
__device__ __forceinline__ bool sees_keys(const Args& a, const Work& w, bool asked) {
  const bool some = asked && w.seen > w.t0 * kKeys;
  if (!w.strange || __builtin_amdgcn_ballot_w64(some) == 0) return some;
  bool in_cache = false;
  for (int tile = w.t0; tile < w.t1; ++tile) {
    const uint64_t in = keys_in_cache(a, w, tile);
    const int n = w.seen - tile * kKeys;
    in_cache |= n > 0 && (in << (kKeys - min(max(n, 1), kKeys))) != 0;
  }
  return some && in_cache;
}

// The queries of the lane's row as matrix operands.
__device__ __forceinline__ void load_queries(const Args& a, const Work& w, bf16x8_t (&q)[8]) {
  const uint16_t* src = a.q + (w.rows.first + w.token) * a.q_token_stride +
                        w.head * a.q_head_stride + ((threadIdx.x >> 5) & 1) * 8;
#pragma unroll
  for (int step = 0; step < 8; ++step)
    q[step] = __builtin_bit_cast(
        bf16x8_t, (u32x4_t)(*reinterpret_cast<const u32x4_any*>(src + 16 * step)));
}

// Turns the queries' signs for a negative scale. A row with an infinity gets NaN, so that its
// result is NaN whatever the keys are (0 times a query that is not finite is NaN).
__device__ __forceinline__ void settle_queries(bf16x8_t (&q)[8], uint32_t flip) {
  const bf16x2_t none = {(__bf16)0.f, (__bf16)0.f};
  float x = 0.f;
#pragma unroll
  for (int step = 0; step < 8; ++step) {
    const u32x4_t w = __builtin_bit_cast(u32x4_t, q[step]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t two = w[i];  // (A bit cast of the element itself takes the vector's first.)
      x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two), none, x, false);
    }
  }
  if (flip != 0)
#pragma unroll
    for (int step = 0; step < 8; ++step)
      q[step] = __builtin_bit_cast(bf16x8_t, __builtin_bit_cast(u32x4_t, q[step]) ^ flip);
  if (x != x) q[0][0] = (__bf16)__builtin_nanf("");
}

__device__ __forceinline__ void clear(State& st) {
  st.m = kNegInf;
  st.l = st.fine = 0.f;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) st.o[d][i] = 0.f;
}

// ---------------------------------------------------------------- many rows a request

// Waves of 32 rows share tiles of 64 keys. A wave alternates between the softmax of a tile
// (vector instructions) and the products of it with the values and of the next tile's keys
// with the queries (matrix instructions, 32 of 32 cycles).
//   Eight waves: the two of a SIMD, 0-3 and 4-7, are half a step apart, held there by a
// barrier at each change, so that one keeps the matrix cores busy while the other does its
// softmax.
//   Four waves: two workgroups to a CU, which hide each other's starts and ends.
constexpr uint32_t kSlotBytes = kKeys * kRowBytes;
// Tiles of keys, and of values, in flight or in use. In phases, the first waves' step i has
// its softmax in phase 2i and its products in 2i + 1, the others' one phase later: keys of
// tile i are read in phases 2i - 1 and 2i, values in 2i + 1 and 2i + 2. A wave copies the
// keys of tile i + 3 and the values of i + 2 in its softmax of step i, phase 2i at the
// earliest, over keys i - 1 and values i - 2, which were read up to phase 2i - 2. It
// awaits the keys of i + 2 and the values of i + 1 at the end of its products of step i,
// phase 2i + 2 at the latest, and they are first read in phase 2i + 3.
//   Four waves are in step: softmax of step i copies keys i + 2 over keys i and values i + 1
// over values i - 1, which were read in the products of step i - 1; they are awaited at the
// end of the products of step i.
constexpr int slots_of(int waves) { return waves == 8 ? 4 : 2; }
constexpr uint32_t lds_of(int waves) { return 2 * slots_of(waves) * kSlotBytes + sizeof(Spoilt); }

template <int kWaves, Source kSource, bool kStream>
__global__ __launch_bounds__(64 * kWaves, 2) void prefill_kernel(Args a, int units) {
  extern __shared__ __align__(256) float lds[];
  constexpr int kSlots = slots_of(kWaves), kRun = kKeys / kWaves;
  Spoilt& spoilt = *reinterpret_cast<Spoilt*>(lds + 2 * kSlots * kSlotBytes / sizeof(float));
  constexpr int kAhead = kWaves == 8 ? 2 : 1;  // steps that values are copied ahead, keys one more
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  fetch<kSource>(a, units);
  begin_spoilt(spoilt);
  Work w = begin<kRows * kWaves, kSource>(a, units, wave);
  if (w.rows.rows == 0) return;
  const uint32_t keys0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) float*)lds;
  const uint32_t values0 = keys0 + kSlots * kSlotBytes;
  const auto slot_of = [&](int tile) { return ((tile - w.t0) & (kSlots - 1)) * kSlotBytes; };
  // A wave copies a run of kRun rows of a tile.
  const uint32_t mine = wave * kRun * kRowBytes;
  Feed<kSource, kStream, kRun> feed;
  const auto copy_keys = [&](int tile) __attribute__((always_inline)) {
    if (tile < w.t1) feed.keys(a, w.keys, keys0 + slot_of(tile) + mine);
  };
  const auto copy_values = [&](int tile) __attribute__((always_inline)) {
    if (tile < w.t1) feed.values(a, w.keys, values0 + slot_of(tile) + mine);
  };
  // What this wave copied of the values of a tile that not all rows see whole.
  const auto look_over = [&](int tile) __attribute__((always_inline)) {
    if (tile < w.whole || tile >= w.t1) return;
    const int row = (lane >> 4) & 3;
#pragma unroll
    for (int i = 0; i < kRun; i += 4)
      clean(a, w.keys, w.strange, values0 + slot_of(tile) + mine + i * kRowBytes + lane * kChunk,
            tile * kKeys + wave * kRun + i + row, (lane & 15) ^ (row << 2), spoilt);
  };

  State st;
  clear(st);
  const bool fine = a.lse != nullptr || a.splits > 1;
  if (w.t0 < w.t1) {
    feed.begin(a, w.keys, w.t0, wave * kRun, lane);
    copy_keys(w.t0);
    copy_values(w.t0);
    copy_keys(w.t0 + 1);
    if constexpr (kAhead == 2) {
      copy_values(w.t0 + 1);
      copy_keys(w.t0 + 2);
    }
  }
  bf16x8_t q[8];
  load_queries(a, w, q);
  const Lanes at = lanes_of(lane, keys0, values0);
  if (w.t0 < w.t1) {
    look_at_blocks<64 * kWaves, kSource>(a, w);
    await_copies<0>();
    look_over(w.t0);
    meet();
    settle_queries(q, a.flip);
    f32x16_t s[2];
    int tile = w.t0;
    if (tile < w.part) first_scores(0u, at, q, s);
    const bool late = kWaves == 8 && wave >= 4;
    if (kWaves == 4 || late) meet();

    // (Values before keys: their offsets are those of the keys copied last.)
    const auto refill = [&](int tile) __attribute__((always_inline)) {
      copy_values(tile + kAhead);
      copy_keys(tile + kAhead + 1);
    };
    // The end of a step's products: what the next step's read has arrived.
    const auto arrive = [&](int tile) __attribute__((always_inline)) {
      if (kAhead == 2 && tile + 3 < w.t1)
        await_copies<kRun / 2>();  // (those of this step's refill stay in flight)
      else
        await_copies<0>();
      look_over(tile + 1);
      meet();
    };
    // A step whose tile all rows see; the tile is in slot kSlot.
    const auto step = [&](auto slot, auto sum) __attribute__((always_inline)) {
      constexpr uint32_t kHere = decltype(slot)::value * kSlotBytes;
      constexpr uint32_t kNext = (decltype(slot)::value + 1) % kSlots * kSlotBytes;
      refill(tile);
      uint32_t p[16];
      soften<2, decltype(sum)::value>(s, a.scale, st, p);
      settle(st.l);
#pragma unroll
      for (int i = 0; i < 16; ++i) settle(p[i]);
      if constexpr (kWaves == 8) change_over();
      // (Of no use behind the last tile, and of no harm.)
      products(kHere, kNext, at, q, p, s, st);
      arrive(tile);
      return ++tile < w.full;
    };
    const auto steps = [&](auto sum) __attribute__((always_inline)) {
      while (tile < w.full) {
        if (!step(std::integral_constant<int, 0>{}, sum)) break;
        if (!step(std::integral_constant<int, 1>{}, sum)) break;
        if constexpr (kSlots == 4) {
          if (!step(std::integral_constant<int, 2>{}, sum)) break;
          if (!step(std::integral_constant<int, 3>{}, sum)) break;
        }
      }
    };
    if (fine)
      steps(std::true_type{});
    else
      steps(std::false_type{});
    // Tiles that some rows see in part; behind the last one are no scores to take.
    const auto part_step = [&](auto last) __attribute__((always_inline)) {
      refill(tile);
      uint32_t p[16];
      take_out<2>(s, w.seen - tile * kKeys, keys_in_cache(a, w, tile));
      soften<2, true>(s, a.scale, st, p);
      settle(st.l);
      settle(st.fine);
#pragma unroll
      for (int i = 0; i < 16; ++i) settle(p[i]);
      if constexpr (kWaves == 8) change_over();
      if constexpr (decltype(last)::value)
        last_product(slot_of(tile), at, p, st);
      else
        products(slot_of(tile), slot_of(tile + 1), at, q, p, s, st);
      arrive(tile);
      ++tile;
    };
    while (tile + 1 < w.part) part_step(std::false_type{});
    if (tile < w.part) part_step(std::true_type{});
    for (; tile < w.t1; ++tile) {
      refill(tile);
      if constexpr (kWaves == 8) change_over();
      arrive(tile);
    }
    if (kWaves == 8 && !late) change_over();
  }
  st.l = xor32_sum(st.l);
  st.fine = xor32_sum(st.fine);
  if (w.t0 < w.t1) {
    spoil(spoilt, w.seen, st);
    // Keys, but scores of -infinity alone (infinite keys): 0 / 0. Another split may have others,
    // so the split says so by a sum of 1 under a reference of -infinity.
    if (sees_keys(a, w, st.m == kNegInf && st.l == 0.f))
      st.l = st.fine = a.splits > 1 ? 1.f : __builtin_nanf("");
  }
  store_row(a, (w.rows.first + w.token) * a.Hq + w.head, w.split, st, w.valid);
}

// Joins the splits of a row, a wave each: a DPP row of 16 lanes takes every fourth split, 8
// dims a lane, with a state of its own and the next two splits' loads in flight; the four
// meet at the end, in the same order every time. (A split's (m, l) of (-infinity, 0) has no
// keys, of (-infinity, 1) scores of -infinity alone, which give NaN if no split has others; a
// NaN has an l of NaN, whatever its m.)
constexpr int kMergeWaves = 4;
__global__ __launch_bounds__(64 * kMergeWaves) void prefill_merge_kernel(Args a) {
  const int row = (int)blockIdx.x * kMergeWaves +
                  __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (row >= a.T * a.Hq) return;
  const int lane = threadIdx.x & 63, i = lane & 15;
  struct Piece {
    float2 ml;
    f32x4_t v[2];
  };
  const auto load = [&](int s) {
    const size_t at = (size_t)row * a.splits + min(s, a.splits - 1);
    const float* src = a.states + at * kDim + 8 * i;
    return Piece{a.sums[at],
                 {reinterpret_cast<const f32x4_t*>(src)[0],
                  reinterpret_cast<const f32x4_t*>(src)[1]}};
  };
  float m = kNegInf, l = 0.f;
  f32x4_t x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  bool hopeless = false;
  int s = lane >> 4;
  Piece next = load(s), after = load(s + 4);
  for (int s0 = 0; s0 < a.splits; s0 += 4, s += 4) {
    const Piece now = next;
    next = after;
    after = load(s + 8);
    if (s >= a.splits || (now.ml.x == kNegInf && now.ml.y == 0.f)) continue;
    const float top = fmaxf(m, now.ml.x), ref = top == kNegInf ? 0.f : top;
    const float old = m == kNegInf ? 0.f : exp2_fast(m - ref);
    const float f = now.ml.x == kNegInf ? 1.f : exp2_fast(now.ml.x - ref);
    const bool all_infinite = now.ml.x == kNegInf && now.ml.y == 1.f;
    hopeless |= all_infinite;
    m = top;
    l = fmaf(l, old, all_infinite ? 0.f : now.ml.y * f);
    x[0] = x[0] * old + now.v[0] * f;
    x[1] = x[1] * old + now.v[1] * f;
  }
  const float top = xor32_max(gqa::xor16_max(m));
  const float f = m == kNegInf ? (l == 0.f ? 0.f : 1.f) : exp2_fast(m - top);
  float sum = xor32_sum(gqa::xor16_sum(l * f));
  if (top == kNegInf && __builtin_amdgcn_ballot_w64(hopeless) != 0) sum = __builtin_nanf("");
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = number(xor32_sum(gqa::xor16_sum(x[e >> 2][e & 3] * f)) * inv);
  if (lane < 16)
    reinterpret_cast<u32x4_t*>(a.out + (size_t)row * kDim)[i] =
        u32x4_t{pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7])};
  if (a.lse && lane == 0) a.lse[row] = log_sum(top, sum);
}

// ---------------------------------------------------------------------------- host

bool misaligned(const void* p, uintptr_t to) {
  return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0;
}

bool sizes_fit(const prefill_gqa_args& p) {
  if (p.T < 0 || p.T > PREFILL_MAX_TOKENS || p.B < 0 || p.B > PREFILL_MAX_BATCH) return false;
  if (p.Hq < 1 || p.Hkv < 1 || p.Hq > 4096 || p.Hq % p.Hkv != 0) return false;
  if ((int64_t)p.T * p.Hq > (1 << 30)) return false;
  if (!p.cu_seqlens_q && p.T != p.B) return false;
  if (p.cu_seqlens_k) {
    if (p.Tk < 0 || p.Tk > INT32_MAX - 64) return false;
  } else {
    if (p.num_blocks < 0 || p.block_size < 1 || p.max_blocks < 1) return false;
    // Keys of a request in 31 bits, a block's bytes in 32.
    if ((int64_t)p.block_size * p.max_blocks > INT32_MAX - 64) return false;
    if ((int64_t)p.block_size * p.Hkv * kRowBytes > UINT32_MAX) return false;
  }
  return true;
}

// The tiles of `rows` rows that the launch has room for, over all requests.
int64_t units_of(const prefill_gqa_args& p, int rows) {
  return (int64_t)p.T * (p.Hq / p.Hkv) / rows + p.B + 2;
}

struct Plan {
  int waves, splits;
};

// Eight waves a workgroup for long work, four for the rest. us with 8 and with 4 (32Q/8KV):
// one prompt of 16384 tokens 1790, 1895; 4 chunks of some 640 tokens over some 3900 keys (with
// 40 us of read-back) 227, 241; 13 prompts and chunks of some 1000 behind some 1500 409, 416;
// one prompt of 2048 tokens 55, 54 and of 1024 tokens 31, 28; 32 prompts of some 500 tokens
// (64 q-heads) 229, 223.
//   Splits: workgroups for two of four waves to a CU, while each has 112 keys or more, and
// no fewer than a request has new tokens (of a whole prompt, later splits are for few rows).
// One row behind 32000 keys 556 us with 1 split, 47 with 16, 35 with 32; 8 requests of 8
// drafts behind 4000 keys 77, 36 (4), 31 (8), 39 (16); 256 tokens behind 16000 keys 311, 107
// (4), 81 (8), 95 (16); a prompt of 600 tokens 20, 26 (2). Where a request's rows are one
// workgroup's, so that the longest request ends last, more of them while they keep 1500
// keys: 16 requests of up to 5 drafts behind up to 16000 keys (64 q-heads) 106 (4), 95 (8),
// 108 (16); 64 of up to 2 behind up to 8000 217 (1), 201 (4), 226 (16).
Plan plan_of(const prefill_gqa_args& p, int num_splits) {
  const int cus = gqa::device_cu_count();
  const int64_t B = std::max(p.B, 1), rows = (int64_t)p.T * (p.Hq / p.Hkv);
  const int64_t keys = p.cu_seqlens_k ? p.Tk / B : (int64_t)p.block_size * p.max_blocks;
  Plan plan{4, num_splits};
  if (keys >= 1024 && rows >= 2048 * B && rows / (8 * kRows) * p.Hkv > cus) plan.waves = 8;
  // Blocks of 8, 24, ..: the 8 keys that each of eight waves copies share a block, 16 do not.
  if (!p.cu_seqlens_k && p.block_size % 16 == 8) plan.waves = 8;
  if (num_splits > 0) return plan;
  plan.splits = 1;
  const int64_t work = std::max(rows / (kRows * plan.waves), B) * p.Hkv;
  const int64_t least = std::max<int64_t>(112, p.T / B);
  while (plan.splits < 32 && work * plan.splits * 2 <= 2 * cus && keys >= least * plan.splits * 2)
    plan.splits *= 2;
  if (!p.cu_seqlens_k && rows <= kRows * plan.waves * B)
    while (plan.splits < 32 && work * plan.splits * 2 <= 8 * cus && keys >= 1500 * plan.splits * 2)
      plan.splits *= 2;
  return plan;
}

size_t states_bytes(const prefill_gqa_args& p, int splits) {
  return splits > 1 ? (size_t)p.T * p.Hq * splits * (kDim * sizeof(float) + sizeof(float2)) : 0;
}

// A launch has fewer than 2^32 threads in a dimension.
bool launches_fit(const prefill_gqa_args& p, const Plan& plan) {
  const int64_t most = UINT32_MAX, rows = (int64_t)p.T * p.Hq;
  if (units_of(p, kRows * plan.waves) * p.Hkv * 64 * plan.waves > most) return false;
  return plan.splits == 1 || (rows + kMergeWaves - 1) / kMergeWaves * 64 * kMergeWaves <= most;
}

using Kernel = void (*)(Args, int);

hipError_t launch(const Args& a, const prefill_gqa_args& p, int waves, hipStream_t stream) {
  const int64_t units = units_of(p, kRows * waves);
  // A prompt of 4096 tokens, 32Q/8KV: 133 us in blocks of 16 or 24, 223 in blocks of 12 and
  // 235 in blocks of 15, whose ids are found row by row.
  const int source = p.cu_seqlens_k                        ? kPacked
                     : p.block_size % (kKeys / waves) == 0 ? kPaged
                                                           : kGather;
  static constexpr Kernel kernels[3][3] = {
      {prefill_kernel<4, kPaged, false>, prefill_kernel<4, kGather, false>,
       prefill_kernel<4, kPacked, false>},
      {prefill_kernel<4, kPaged, true>, prefill_kernel<4, kGather, false>,
       prefill_kernel<4, kPacked, true>},
      {prefill_kernel<8, kPaged, false>, prefill_kernel<8, kGather, false>,
       prefill_kernel<8, kPacked, false>}};
  // Rows of one workgroup a request, on average: nobody else reads most of the keys. (Drafts, 16
  // requests of up to 5 rows behind up to 16000 keys, 64Q/8KV, 454 MB: 107 us with nt, 119
  // without; 60 single rows behind up to 4000 keys, 32Q/8KV, 114, 126; with a chunk of 512
  // rows behind 8000 among them 197, 201, of 1500 behind 16000 560, 522.)
  const bool once = (int64_t)p.T * a.G <= (int64_t)kRows * waves * p.B;
  const Kernel kernel = kernels[waves == 8 ? 2 : once][source];
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize,
                                           lds_of(waves));
  if (e != hipSuccess) return e;
  kernel<<<dim3((unsigned)(units * p.Hkv), a.splits), 64 * waves, lds_of(waves), stream>>>(
      a, (int)units);
  return hipGetLastError();
}

}  // namespace

extern "C" int prefill_gqa_pick_num_splits(const prefill_gqa_args* args) {
  if (!args || !sizes_fit(*args)) return 0;
  return plan_of(*args, 0).splits;
}

extern "C" size_t prefill_gqa_workspace_bytes(const prefill_gqa_args* args, int num_splits) {
  if (!args || !sizes_fit(*args) || num_splits < 0 || num_splits > PREFILL_MAX_SPLITS) return 0;
  return states_bytes(*args, plan_of(*args, num_splits).splits);
}

extern "C" int prefill_gqa_launch(const prefill_gqa_args* args, int num_splits, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  if (!args || !sizes_fit(*args)) return hipErrorInvalidValue;
  const prefill_gqa_args p = *args;
  if (num_splits < 0 || num_splits > PREFILL_MAX_SPLITS || !isfinite(p.scale))
    return hipErrorInvalidValue;
  if (p.q_token_stride < 0 || p.q_head_stride < 0) return hipErrorInvalidValue;
  const bool packed = p.cu_seqlens_k != nullptr;
  if (packed) {
    for (const int64_t s : {p.k_token_stride, p.k_head_stride, p.v_token_stride, p.v_head_stride})
      if (s < 0 || s % 8 != 0 || s >= (1 << 27)) return hipErrorInvalidValue;
  }
  if (p.T == 0) return hipSuccess;
  if (!p.q || !p.out || misaligned(p.out, 16)) return hipErrorInvalidValue;
  const bool any = packed ? p.Tk > 0 : p.num_blocks > 0;
  if (any && (!p.k || !p.v || misaligned(p.k, 16) || misaligned(p.v, 16)))
    return hipErrorInvalidValue;
  if (!packed && p.B > 0 && (!p.block_table || !p.seq_lens)) return hipErrorInvalidValue;
  const Plan plan = plan_of(p, num_splits);
  if (!launches_fit(p, plan)) return hipErrorInvalidValue;
  const size_t need = states_bytes(p, plan.splits);
  if (need > 0 && (!workspace || misaligned(workspace, 16) || workspace_bytes < need))
    return hipErrorInvalidValue;

  Args a{};
  a.q = p.q, a.q_token_stride = p.q_token_stride, a.q_head_stride = p.q_head_stride;
  a.k = reinterpret_cast<const uint8_t*>(p.k), a.v = reinterpret_cast<const uint8_t*>(p.v);
  if (packed) {
    a.k_token_bytes = 2 * p.k_token_stride, a.k_head_bytes = 2 * p.k_head_stride;
    a.v_token_bytes = 2 * p.v_token_stride, a.v_head_bytes = 2 * p.v_head_stride;
    a.Tk = p.Tk;
  } else {
    a.k_token_bytes = a.v_token_bytes = (int64_t)p.Hkv * kRowBytes;
    a.k_head_bytes = a.v_head_bytes = kRowBytes;
    a.block_bytes = a.k_token_bytes * p.block_size;
    a.block_bytes32 = (uint32_t)a.block_bytes, a.token_bytes32 = (uint32_t)a.k_token_bytes;
    a.tile_blocks = kKeys / p.block_size, a.tile_slots = kKeys % p.block_size;
    a.num_blocks = p.num_blocks, a.block_size = p.block_size, a.max_blocks = p.max_blocks;
    a.capacity = p.num_blocks > 0 ? p.block_size * p.max_blocks : 0;
    a.block_table = p.block_table;
    a.bs_div = make_fastdiv((uint32_t)p.block_size);
    const int64_t tiles = ((int64_t)a.capacity + kKeys - 1) / kKeys;
    a.split_tiles = (int)((tiles + plan.splits - 1) / plan.splits);
  }
  a.out = p.out, a.lse = p.lse;
  if (need > 0) {
    a.states = static_cast<float*>(workspace);
    a.sums = reinterpret_cast<float2*>(a.states + (size_t)p.T * p.Hq * plan.splits * kDim);
  }
  // (Arrays that the search may read an entry of, whatever it makes of it: without
  // cu_seqlens_q there is a request, without a request cu_seqlens_q.)
  a.lens = packed ? p.cu_seqlens_k : p.B > 0 ? p.seq_lens : p.cu_seqlens_q;
  a.ends = packed && p.B > 0 ? p.cu_seqlens_k + 1 : a.lens;
  a.cu_q = p.cu_seqlens_q ? p.cu_seqlens_q : a.lens;
  a.row_mask = p.cu_seqlens_q ? -1 : 0;
  a.T = p.T, a.B = p.B, a.Hq = p.Hq, a.Hkv = p.Hkv, a.G = p.Hq / p.Hkv;
  a.causal = p.causal != 0, a.splits = plan.splits;
  // (A scale of 0 weighs all keys alike; the smallest normal does as well and keeps
  // 0 * infinity out of the kernel.)
  a.scale = std::max(fabsf(p.scale) * gqa::kLog2e, 1.17549435e-38f);
  a.flip = p.scale < 0.f ? 0x80008000u : 0u;
  // 4 chunks of up to 1024 rows over up to 8000 keys (with 30 us of read-back) 220 us, in the
  // requests' own order 221 to 265. One request, or one workgroup a request, has nothing to
  // put in order, and for more requests looking through all of them costs prompts more than it
  // gives: in order and not, 17 prompts 16, 17 us (up to 200 tokens) and 89, 86 (1000), 32 139,
  // 122 (1000), 62 37, 24 (100), where 62 chunks of up to 100 behind up to 3000 take 116, 142.
  a.sorted = p.B >= 2 && p.B <= 16 && (int64_t)p.T * a.G > (int64_t)kRows * plan.waves * p.B;
  a.group_div = make_fastdiv((uint32_t)a.G);
  a.head_div = make_fastdiv((uint32_t)p.Hkv);
  const hipError_t e = launch(a, p, plan.waves, stream);
  if (e != hipSuccess || plan.splits == 1) return e;
  prefill_merge_kernel<<<(unsigned)((p.T * p.Hq + kMergeWaves - 1) / kMergeWaves),
                         64 * kMergeWaves, 0, stream>>>(a);
  return hipGetLastError();
}
