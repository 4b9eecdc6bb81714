// What the two forms of the attention over a paged 16-bit cache share: the
// request, the rows of a kv head, and the passes that follow them.
//
// A kv head's query rows are taken together: packed row r = i * group + g is
// query row i of head kvh * group + g, r < R = max_q_len * group, so that K and
// V are read once for all of them.
#pragma once

#include "paged.cuh"

namespace llmx_b200 {

constexpr float kPagedLog2e = 1.4426950408889634f;
constexpr float kPagedLn2 = 0.6931471805599453f;

// The tokens [lo, hi) that query row i of a sequence sees (empty: lo >= hi).
struct Visible {
  int lo, hi;
};
__device__ __forceinline__ Visible row_visible(const AttnArgs &a, int i, int ql, int kl) {
  Visible v{0, 0};
  if (i >= ql) return v;
  const int diag = i + kl - ql;  // i, kl and ql are at most 2^30
  v.hi = a.causal ? min(kl, diag + 1) : kl;
  v.lo = a.window >= 0 ? max(0, diag - a.window) : 0;  // window is at most 2^30
  return v;
}

// The token whose ALiBi bias is a row's largest: biases are taken as slope *
// (j - ref), which leaves the softmax as it is and keeps the bits of positions
// far into a sequence; the log-sum-exp gets slope * ref back.
__device__ __forceinline__ int alibi_ref(const Visible &v, float slope) { return slope >= 0.f ? v.hi - 1 : v.lo; }

}  // namespace llmx_b200
