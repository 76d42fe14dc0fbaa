// How a batch of rows goes to workgroups in policy_loss.hip.  Host code without HIP: the including file has ceil_div.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace rlpyt {
namespace {

constexpr int kGroupV = 128;        // longest row of the lane groups
// And of a wave.  (Rows of 4 to 8 KB by workgroups of 256: 16384 x 3000 in bf16 78 us instead of 67, 60000 219 instead of 175,
// as a workgroup waits for its one lane that works out the row's terms; 256 rows 17.7 instead of 19.6.)
constexpr int kWaveBytes = 8192;

struct LossPlan {
  int P, part;                      // P > 0: rows split into P parts of `part` elements
  int64_t partials;                 // rows of the [., 4] table of partial sums
  int64_t groups(int64_t N) const { return P > 0 ? N * P : partials; }   // workgroups
};
inline int group_lanes(int64_t V) { return V <= 32 ? 8 : 16; }
// Rows of a group.  262144 x 18 in f32 takes 49 us by one row each and 35 by four, 8192 x 18 18.4 and 19.1 (fewer
// workgroups, and what a lane does for a row is not hidden behind others).
inline int group_rows(int64_t N) { return N >= 32768 ? 4 : 1; }

// A row goes to a group of lanes, a wave or a workgroup (256 KB at most) whose registers hold it, unless the row is long and
// the rows are few: then it is split into parts of at least 8 KB so that there are about 1024 workgroups.  (Held against split,
// log-probabilities: 16 x 32000 bf16 5.5 and 7.9 us, 128 x 60000 f32 10.0 and 12.3, 64 x 131072 bf16 12.4 and 11.1; losses: 192 x
// 32000 f32 24 and 31.5, 64 x 131072 bf16 35 and 28.)
inline LossPlan plan_of(int64_t N, int64_t V, int size) {
  LossPlan q = {0, 0, N};
  if (N == 0) return q;
  if (V <= kGroupV) {
    q.partials = ceil_div(N, 256 / group_lanes(V) * group_rows(N));
    return q;
  }
  if (V * size <= kWaveBytes) {
    q.partials = ceil_div(N, 4);
    return q;
  }
  const bool held = V * size <= 256 * 1024;
  if (held && (N >= 128 || V * size <= 128 * 1024)) return q;
  const int64_t least = ceil_div(V * size, 8 * 1024), want = std::max<int64_t>(held ? 1 : 4, ceil_div(1024, N));
  const int64_t P = std::min(least, want);
  q.part = (int)(ceil_div(ceil_div(V, P), 8) * 8);
  q.P = (int)ceil_div(V, q.part);
  return q;
}

// A launch holds less than 2^32 threads: large batches go in slices of rows.
inline int64_t slice_rows(const LossPlan& q) { return q.P > 0 ? std::max<int64_t>(1, ((int64_t)1 << 22) / q.P) : (int64_t)1 << 21; }

}  // namespace
}  // namespace rlpyt
