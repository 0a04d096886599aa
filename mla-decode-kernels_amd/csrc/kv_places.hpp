// Where a step's new tokens go: the integer rules of include/kv_cache.h, for the
// kernels and, compiled for the host, for their test.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

namespace kv {

// The number of entries of cu_seqlens[1..B] that are <= t, which is the request
// of row t, by a search that probes `group` entries a step: entry
// lo + i * step by probe i < group if it is below hi. Entries out of order give
// some number in [0, B].
struct Search {
  int lo, hi;  // entries below lo are <= t, those from hi on are not

  KV_HD static Search begin(int B) { return {1, B + 1}; }
  KV_HD bool done() const { return lo >= hi; }
  KV_HD int step(int group) const {
    const int s = (hi - lo + group - 1) / group;
    return s > 1 ? s : 1;
  }
  // `count` of the probes were <= t. The entries next to the range go with it:
  // entry lo - 1 becomes probe count - 1's if count > 0, entry hi probe count's if
  // this says so.
  KV_HD bool narrow(int step, int count) {
    const int end = lo + count * step;
    const bool below = end < hi;
    if (below) hi = end;
    if (count > 0) lo += (count - 1) * step + 1;
    if (step == 1) hi = lo;
    return below;
  }
  KV_HD int request() const { return lo - 1; }
};

struct Place {
  int b, pos;
  bool live;  // else padding
};

// Row t as number t - first of request b's n = next - first rows.
KV_HD Place place_in(int t, int b, int first, int next, int len) {
  // (A request shorter than its rows: those in front have no place.)
  if (t < first || t >= next || len < next - t) return Place{b, 0, false};
  return Place{b, len - (next - t), true};
}

}  // namespace kv
