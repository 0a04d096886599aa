// The second launch of the token-balanced 4-bit decode (kv_decode.hip): segments cut
// between workgroups.
#include "kv_decode.hpp"

namespace {

using namespace kv;
using gqa::exp2_fast;
using gqa::kNegInf;
using gqa::xor16_max;
using gqa::xor16_sum;
using gqa::xor32_max;
using gqa::xor32_sum;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// The workgroup whose first piece ends a cut segment folds it, from the one whose
// last piece starts it. A wave to a head; a row of 16 lanes takes every fourth piece,
// 8 dims a lane, with a state of its own, and the four rows meet at the end. One chain
// of latencies (records, states, the sum over the rows), so what shortens it is few
// instructions on a wave that has its SIMD to itself. Against 16 waves on one CU that
// share a segment's heads and pieces and meet in LDS: 4 requests of 2048 tokens 11.4 us
// in all for 12.3, a ragged batch of 64 (64Q/8KV) 167.6 for 168.8; one request of 32768
// (32 pieces to a segment) 17.0 for 16.6.
constexpr int kMergeWaves = 4;
__global__ __launch_bounds__(64 * kMergeWaves) void kv_decode_merge_kernel(MergeArgs a) {
  const int wg = blockIdx.x, lane = threadIdx.x & 63;
  // Lane i reads record wg - i: the workgroup's own, and those in front.
  const Record r = a.records[max(wg - lane, 0)];
  const int flags = __builtin_amdgcn_readfirstlane(r.flags);
  const int h = (int)blockIdx.y * kMergeWaves +
                __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if ((flags & (kHasA | kEndsA)) != (kHasA | kEndsA)) return;
  if (h >= __builtin_amdgcn_readfirstlane(r.heads)) return;
  const int row = __builtin_amdgcn_readfirstlane(r.row_a) + h;
  uint64_t hit = __builtin_amdgcn_ballot_w64(lane > 0 && lane <= wg && (r.flags & kHasZ) != 0);
  int base = wg;
  while (!hit) {
    base -= 64;
    if (base < 0) return;
    hit = __builtin_amdgcn_ballot_w64(lane <= base &&
                                      (a.records[max(base - lane, 0)].flags & kHasZ) != 0);
  }
  const int from = base - (int)__builtin_ctzll(hit);
  // (Shares go to the first workgroups, so all from `from` to wg have a piece: a Z,
  // then As.)
  const int n = wg - from + 1, i = lane & 15;
  const float* const states = a.states + (size_t)from * 2 * a.slot_floats + h * kPitch;
  struct Piece {
    float2 ml;
    f32x4_t v[2];
  };
  const auto load = [&](int p) {
    const float* s =
        states + (size_t)(p == 0 ? 1u : 2 * (uint32_t)min(p, n - 1)) * a.slot_floats;
    return Piece{*reinterpret_cast<const float2*>(s + kDim),
                 {reinterpret_cast<const f32x4_t*>(s + 8 * i)[0],
                  reinterpret_cast<const f32x4_t*>(s + 8 * i)[1]}};
  };
  float M = kNegInf, L = 0.f;
  f32x4_t x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  int p = lane >> 4;
  Piece next = load(p), after = load(p + 4);
  for (int p0 = 0; p0 < n; p0 += 4, p += 4) {
    const Piece now = next;
    next = after;
    after = load(p + 8);
    if (p >= n) break;  // (these rows are done)
    const float m = fmaxf(M, now.ml.x), ref = m == kNegInf ? 0.f : m;
    const float old = exp2_fast(M - ref), f = exp2_fast(now.ml.x - ref);
    M = m;
    L = fmaf(L, old, now.ml.y * f);
    x[0] = x[0] * old + now.v[0] * f;
    x[1] = x[1] * old + now.v[1] * f;
  }
  const float top = xor32_max(xor16_max(M));
  const float f = M == kNegInf ? 0.f : exp2_fast(M - top);
  L = xor32_sum(xor16_sum(L * f));
  const float inv = inverse(L);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = xor32_sum(xor16_sum(x[e >> 2][e & 3] * f)) * inv;
  if (lane < 16) reinterpret_cast<uint4*>(a.out + (size_t)row * kDim)[i] = pack8(y);
}

}  // namespace

hipError_t kv::launch_decode_merge(const MergeArgs& args, int workgroups, int heads,
                                   hipStream_t stream) {
  kv_decode_merge_kernel<<<dim3(workgroups, (heads + kMergeWaves - 1) / kMergeWaves),
                           64 * kMergeWaves, 0, stream>>>(args);
  return hipGetLastError();
}
