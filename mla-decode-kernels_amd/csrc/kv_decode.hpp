// What the two kernels of the 4-bit decode (kv_decode.hip, kv_decode_merge.hip) share:
// the states of pieces of segments that the shares' ends cut, and their records.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_common.hpp"

namespace kv {

constexpr int kPitch = 132;  // floats of a head's state: acc [128], m, l, pad

constexpr int kHasA = 1, kEndsA = 2, kHasZ = 4;  // pieces of a share (Record::flags)

// A wave's or a workgroup's cut pieces: what they are, their first row of out
// (request and q-head) and the number of its rows. (Rows and not segments: whoever
// folds them has nothing to divide.)
struct Record {
  int flags, row_a, row_z, heads;  // heads: of A, and of Z from bit 8 on
};

// What a row is multiplied by in the end, 1 / l; a segment without a single token
// gets zeros. (One quotient a lane: its fp32 rounding is nothing to bf16's.)
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

struct MergeArgs {
  const Record* records;
  const float* states;
  uint16_t* out;
  uint32_t slot_floats;
};

// Fold the cut segments of `workgroups` shares of segments of up to `heads` q-heads.
hipError_t launch_decode_merge(const MergeArgs& args, int workgroups, int heads,
                               hipStream_t stream);

}  // namespace kv
