// What the tensor-core kernels over a paged 16-bit cache share (attn_paged_tc.cu,
// paged_weights.cu): what rows of a tile see, and TMA loads of 128 tokens from
// their pages.
#pragma once

#include "paged_attn.cuh"
#include "sm100_fmha.cuh"

namespace llmx_b200 {
namespace {

// The tokens that rows [m0, m0 + n) of a sequence see: some row [lo, hi), every
// row [all_lo, all_hi).
struct RowsSee {
  int lo, hi, all_lo, all_hi;
};
__device__ __forceinline__ RowsSee rows_see(const AttnArgs &a, int m0, int n, int ql, int kl) {
  RowsSee s{0, 0, 0, 0};
  const int i0 = m0 / a.group;
  if (i0 >= ql) return s;
  const int i1 = min(ql - 1, (m0 + n - 1) / a.group);
  const Visible f = row_visible(a, i0, ql, kl), l = row_visible(a, i1, ql, kl);
  s.lo = f.lo;
  s.hi = max(0, l.hi);
  s.all_lo = l.lo;
  s.all_hi = f.hi;
  return s;
}
// Whether some row of them does not see the whole block.
__device__ __forceinline__ bool partly(const RowsSee &s, int n0) { return n0 < s.all_lo || n0 + kBN > s.all_hi; }

// A block of 128 tokens comes as 128 / box TMA boxes of `box` = gcd(page_size,
// 128) tokens, each inside one page; lane i has box i.  Where it lies for the
// block at n0: behind the sequence's length, and where the table points outside
// the cache, the page index n_pages, which is outside the tensor map: such a box
// is filled with zeros, nothing is read, and the byte count stays the same.
struct BoxPlace {
  int page, row;
};
__device__ __forceinline__ BoxPlace box_place(const PagedArgs &c, int box, int b, int kl, int n0) {
  const int lane = threadIdx.x % 32;
  BoxPlace p{c.n_pages, 0};
  const int j = n0 + lane * box;
  if (lane < kBN / box && j < kl) {
    const int slot = j / c.page_size;
    const int id = paged_page(c, b, slot);
    if (id >= 0) {
      p.page = id;
      p.row = j - slot * c.page_size;
    }
  }
  return p;
}
// Issues the boxes by a whole warp, counted on `bar`: a tile of 64-column chunks.
template <int D>
__device__ __forceinline__ void load_boxes(uint8_t *dst, const CUtensorMap *tm, uint64_t *bar, int box, int kvh,
                                           const BoxPlace &p) {
  const int lane = threadIdx.x % 32;
  if (lane == 0) mbar_arrive_expect_tx(bar, 128 * D * 2);
  __syncwarp();
  if (lane < kBN / box)
    for (int c = 0; c < D / 64; ++c) tma_load_4d(dst + c * 128 * 128 + lane * box * 128, tm, bar, c * 64, p.row, kvh, p.page);
}

// ------------------------------------------------------------------- maps
CUtensorMapDataType map_type(int dtype) {
  return dtype == LLMX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

bool make_map(CUtensorMap *m, const void *base, int dtype, const cuuint64_t (&dims)[4], const long long (&st)[3],
              const cuuint32_t (&box)[4]) {
  EncodeTiledFn enc = encode_tiled();
  if (enc == nullptr) return false;
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    strides[i] = (cuuint64_t)st[i] * 2u;
    // A dimension of extent 1 is never stepped along; give it any legal stride.
    if (dims[i + 1] <= 1 && (strides[i] == 0 || strides[i] >= (1ULL << 40))) strides[i] = 16;
  }
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return enc(m, map_type(dtype), 4, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// [.., 64 channels] x heads x rows of q: one box is a tile's packed rows.
bool make_q_map(CUtensorMap *m, const AttnArgs &a, int M) {
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.H, (cuuint64_t)a.Sq, (cuuint64_t)a.B};
  const long long st[3] = {a.qs[2], a.qs[1], a.qs[0]};
  const cuuint32_t box[4] = {64, (cuuint32_t)a.group, (cuuint32_t)(M / a.group), 1};
  return make_map(m, a.q, a.dtype, dims, st, box);
}
// Tokens x kv heads x pages of K or V.
bool make_page_map(CUtensorMap *m, const PagedArgs &c, const void *base, const long long *s, int dtype, int box_rows) {
  const cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)c.page_size, (cuuint64_t)c.Hkv, (cuuint64_t)c.n_pages};
  const long long st[3] = {s[2], s[1], s[0]};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  return make_map(m, base, dtype, dims, st, box);
}

}  // namespace
}  // namespace llmx_b200
