// What the two forms of the attention over a paged 16-bit cache share: the
// request, the rows of a kv head, and the passes that follow them.
//
// A kv head's query rows are taken together: packed row r = i * group + g is
// query row i of head kvh * group + g, r < R = max_q_len * group, so that K and
// V are read once for all of them.
#pragma once

#include <atomic>

#include "paged.cuh"

namespace llmx_b200 {

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

// The tensor-core form (attn_paged_tc.cu): which requests it takes, how a
// request is cut (part_bytes of partial results with a workspace), and the
// launch.  ctr: an int for the work counter, or NULL; stat: nullable
// [B * Hkv][R], log2 of each packed row's sum of 2^score.
struct PagedTcPlan {
  int M, n_mblocks, n_whole, piece, parts, n_work;
  bool on_device;  // the device cuts, by the lengths that it has
  size_t part_bytes;
};
bool paged_tc_supports(const AttnArgs &a);
PagedTcPlan plan_paged_tc(const AttnArgs &a, bool have_ws);
cudaError_t launch_paged_tc(const AttnArgs &a, const PagedArgs &c, const PagedTcPlan &p, int *ctr, float *part, float *stat,
                            cudaStream_t s);

// Key weights of a chunk from the rows' sums (paged_weights.cu), after the
// attention that wrote them.
bool paged_weights_supports(const AttnArgs &a);
cudaError_t launch_paged_weights(const AttnArgs &a, const PagedArgs &c, const float *stat, float decay, cudaStream_t s);

// Allows a kernel `bytes` of dynamic shared memory on the current device, once a
// device (the attribute belongs to the device that is current).  The
// flags are one for each kernel: the template's argument is the kernel itself.
template <auto kKernel>
cudaError_t allow_smem(size_t bytes) {
  static std::atomic<bool> done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev].load())) return e;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true);
  return e;
}

// A launch that may be set up while the kernel before it still runs (it waits
// for that kernel itself).
template <typename K, typename... Args>
cudaError_t launch_paged_after(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, const Args &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace llmx_b200
