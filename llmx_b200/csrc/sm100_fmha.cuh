// What the tensor-core attention kernels share (attn_sm100.cu: dense K / V;
// attn_paged_tc.cu: K / V in pages): the tile sizes, the MMA issue order of a
// pair of query tiles, the softmax of one 128-key block and the epilogue's
// transpose.  The scheme is described at the head of attn_sm100.cu.
#pragma once

#include <cuda.h>

#include <mutex>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace llmx_b200 {
namespace {

using namespace sm100;

constexpr int kBM = 128;       // query rows per tile
constexpr int kTiles = 2;      // query tiles per CTA
constexpr int kBN = 128;       // keys per KV block
constexpr int kThreads = 384;  // 2 softmax warpgroups + MMA / TMA warpgroup
constexpr int kMmaWarp = 8;
constexpr int kTmaWarp = 9;
// Register split (setmaxnreg, multiples of 8): the CTA launches with 384 x 168;
// the MMA / TMA warpgroup drops to 64 and the softmax warpgroups grow to 216:
// 128 * 64 + 256 * 216 = 63488 <= 384 * 168 = 64512.
constexpr uint32_t kRegsControl = 64;
constexpr uint32_t kRegsSoftmax = 216;
static_assert(128 * kRegsControl + 256 * kRegsSoftmax <= kThreads * 168, "register split exceeds the launch");
constexpr uint64_t kTimeoutNs = 1000000000ull;
constexpr int kSchedSlots = 4;
constexpr int kSchedConsumers = 1 + 8;  // the MMA thread + one lane per softmax warp
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Lazy rescale: the running max moves (and O is rescaled) only when a block
// raises it by more than this many log2 units, so P <= 2^threshold.  bf16 P
// has the fp32 exponent range and O / l accumulate in fp32, so 2^64; fp16 P
// must stay below 65504, so 2^15.
template <typename T>
constexpr float rescale_threshold() {
  return std::is_same<T, __nv_bfloat16>::value ? 64.0f : 15.0f;
}

template <int D>
struct Cfg {
  static constexpr int kChunks = D / 64;          // 128-byte wide column chunks of a tile
  static constexpr int kChunkBytes = 128 * 128;   // 128 rows x 128 bytes
  static constexpr int kTileBytes = 128 * D * 2;  // one 128-row tile of 16-bit elements
  static constexpr int kStages = D == 128 ? 2 : 3;
  static constexpr int kQOff = 0;
  static constexpr int kKOff = kQOff + kTiles * kTileBytes;
  static constexpr int kVOff = kKOff + kStages * kTileBytes;
  // ALiBi operands of the extra QK^T step (K-major, no swizzle, 4 KB used
  // of 8 KB each): A' per query tile, B' shared.
  static constexpr int kXOff = kVOff + kStages * kTileBytes;
  static constexpr int kXBytes = 8192;
  static constexpr int kBarOff = kXOff + 3 * kXBytes;
  static constexpr int kSmemBytes = kBarOff + 1024 + 1024;  // barriers + alignment slack
  static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
  static constexpr uint32_t kTmemS0 = 0, kTmemS1 = 128;
  static constexpr uint32_t kTmemO0 = 256, kTmemO1 = 256 + D;
  static constexpr uint32_t kTmemCols = 512;
};

template <typename B>
__device__ __forceinline__ void set_abort(B *bars, unsigned int *err) {
  bars->abort_flag = 1;
  raise_error(err, kDevErrTimeout);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  }
}

// Key-block range of the CTA: blocks [n_start, n_start + nb*kBN).
struct BlockRange {
  int n_start, nb;
};

// First key of the j-th block processed.  With ALiBi the blocks go last to
// first, as the reference's main loop does (single_mha_kernel.cuh:295-296):
// the bias slope * key grows with the key, so the first block processed
// holds the row's largest biases, the running max is set there, and later
// blocks rarely raise it (each raise rescales O).
template <bool kReverse>
__device__ __forceinline__ int block_n0(const BlockRange &br, int j) {
  return br.n_start + (kReverse ? br.nb - 1 - j : j) * kBN;
}

// ALiBi folded into QK^T (no soft-cap): one more K = 16 step adds
// beta * c to S[r][c], beta = slope / sm_scale, c = the key's column in its
// 128-key block.  A'_t (128 x 16, per query tile) holds beta as three 16-bit
// parts in columns 0-2 of every row; B' (128 x 16) holds c in columns 0-2 of
// row c.  Integers below 256 are exact in both 16-bit types and the products
// are exact in fp32, so S' = S + beta * c to fp32 rounding.  The softmax then
// treats ALiBi like the plain path plus slope * (n0 + kv_offset) per block.
// Byte offset of element (r, k) in the no-swizzle K-major layout used for
// A' and B': 8-row x 16-byte core matrices, 128 bytes apart along K,
// 256 bytes apart between 8-row groups.
__device__ __forceinline__ int x_offset(int r, int k) {
  return (r >> 3) * 256 + (k >> 3) * 128 + (r & 7) * 16 + (k & 7) * 2;
}

// ---------------------------------------------------------------- MMA role
// MMAs of one work item.  kv_base: key blocks of earlier items (ring
// position); blk_base0 / blk_base1: key blocks of earlier items on tile 0 /
// tile 1 (s_full, p_full, o_done complete once per block of their tile);
// tile_it: earlier items (q_full phase).  The last QK^T on each Q buffer is
// followed by a commit to q_empty, so the next item's Q load starts while
// this item finishes.  Tile 1 takes part in all nb blocks; tile 0 (the
// earlier rows) in nb0 of them: the first nb0 in forward order, the last
// nb0 in reverse order (kReverse: the key blocks go last to first, so tile
// 0's blocks, the lowest keys, come at the end).
template <int D, bool kBF16, bool kFold, bool kReverse, typename B>
__device__ bool mma_tile(uint8_t *smem, B *bars, uint32_t tmem, int nb, int nb0, int tile_it, int kv_base,
                         int blk_base0, int blk_base1) {
  using C = Cfg<D>;
  constexpr uint32_t idesc_qk = idesc_f16(128, kBN, kBF16, false);
  constexpr uint32_t idesc_pv = idesc_f16(128, D, kBF16, true);
  const uint32_t q_base = smem_u32(smem + C::kQOff);
  const uint32_t k_base = smem_u32(smem + C::kKOff);
  const uint32_t v_base = smem_u32(smem + C::kVOff);
  const uint32_t x_base = smem_u32(smem + C::kXOff);
  auto wait = [&](uint64_t *bar, uint32_t par) {
    return mbar_wait_or_abort(bar, par, kTimeoutNs, &bars->abort_flag);
  };

  // Descriptors are built per call from an opaque base plus the step's
  // offset in the 14-bit address field (shared addresses < 256 KB, so the
  // field never carries): the compiler would otherwise keep every stage's
  // descriptors live in registers across the whole loop.
  // S_t = Q_t K^T over D in steps of 16 (32 bytes inside a 128-byte chunk).
  auto issue_qk = [&](int t, int s) {
    const uint32_t d_tmem = tmem + (t ? C::kTmemS1 : C::kTmemS0);
    uint64_t da = smem_desc_sw128(q_base + t * C::kTileBytes, 16, 1024);
    uint64_t db = smem_desc_sw128(k_base + s * C::kTileBytes, 16, 1024);
    asm volatile("" : "+l"(da), "+l"(db));
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint64_t off = (uint64_t)(((kk / 4) * C::kChunkBytes + (kk % 4) * 32) >> 4);
      mma_ss(d_tmem, da + off, db + off, idesc_qk, kk > 0 ? 1u : 0u);
    }
    if constexpr (kFold) {
      // S_t += A'_t B'^T: + beta * c for key column c (the ALiBi slope over sm_scale).
      uint64_t dx = smem_desc_noswz(x_base + t * C::kXBytes, 128, 256);
      uint64_t dk = smem_desc_noswz(x_base + 2 * C::kXBytes, 128, 256);
      asm volatile("" : "+l"(dx), "+l"(dk));
      mma_ss(d_tmem, dx, dk, idesc_qk, 1u);
    }
  };
  // O_t (+)= P_t V over the 128 keys in steps of 16 (P: 8 TMEM columns per
  // step; V: 16 rows of 128 bytes per step, MN-major, 64-column chunks 16 KB apart).
  auto issue_pv = [&](int t, int s, bool acc) {
    const uint32_t d_tmem = tmem + (t ? C::kTmemO1 : C::kTmemO0);
    const uint32_t p_tmem = tmem + (t ? C::kTmemS1 : C::kTmemS0);
    uint64_t db = smem_desc_sw128(v_base + s * C::kTileBytes, C::kChunkBytes, 1024);
    asm volatile("" : "+l"(db));
#pragma unroll
    for (int kk = 0; kk < kBN / 16; ++kk)
      mma_ts(d_tmem, p_tmem + kk * 8, db + (uint64_t)((kk * 16 * 128) >> 4), idesc_pv, (acc || kk > 0) ? 1u : 0u);
  };

  // Tile 0 works on blocks j in [lo0, hi0) of the item's sequence.
  const int lo0 = kReverse ? nb - nb0 : 0, hi0 = kReverse ? nb : nb0;
  const uint32_t qpar = tile_it & 1;
  const int s0 = kv_base % C::kStages;
  if (!wait(&bars->k_full[s0], (kv_base / C::kStages) & 1)) return false;
  if (lo0 == 0) {
    if (!wait(&bars->q_full[0], qpar)) return false;
    tc_fence_after();
    issue_qk(0, s0);
    tc_commit(&bars->s_full[0]);
    if (hi0 == 1) tc_commit(&bars->q_empty[0]);
  }
  if (!wait(&bars->q_full[1], qpar)) return false;
  tc_fence_after();
  issue_qk(1, s0);
  tc_commit(&bars->s_full[1]);
  tc_commit(&bars->k_empty[s0]);
  if (nb == 1) tc_commit(&bars->q_empty[1]);
  for (int j = 0; j < nb; ++j) {
    const int g = kv_base + j;
    const int sv = g % C::kStages;
    const int sk = (g + 1) % C::kStages;
    const bool more = j + 1 < nb;
    if (!wait(&bars->v_full[sv], (g / C::kStages) & 1)) return false;
    if (j >= lo0 && j < hi0) {
      if (!wait(&bars->p_full[0], (blk_base0 + j - lo0) & 1)) return false;
      tc_fence_after();
      issue_pv(0, sv, j > lo0);
      tc_commit(&bars->o_done[0]);
    }
    if (more && !wait(&bars->k_full[sk], ((g + 1) / C::kStages) & 1)) return false;
    if (j + 1 >= lo0 && j + 1 < hi0) {
      // Tile 0's first block in reverse order: its Q load is awaited here.
      if (j + 1 == lo0 && !wait(&bars->q_full[0], qpar)) return false;
      tc_fence_after();
      issue_qk(0, sk);
      tc_commit(&bars->s_full[0]);
      if (j + 2 == hi0) tc_commit(&bars->q_empty[0]);
    }
    if (!wait(&bars->p_full[1], (blk_base1 + j) & 1)) return false;
    tc_fence_after();
    issue_pv(1, sv, j > 0);
    tc_commit(&bars->o_done[1]);
    tc_commit(&bars->v_empty[sv]);
    if (more) {
      issue_qk(1, sk);
      tc_commit(&bars->s_full[1]);
      tc_commit(&bars->k_empty[sk]);
      if (j + 2 == nb) tc_commit(&bars->q_empty[1]);
    }
    if (bars->abort_flag) return false;
  }
  return true;
}

// head_dim 256: one tile (attn_sm100.cu describes the scheme).
struct Cfg256 {
  static constexpr int D = 256;
  static constexpr int kChunks = D / 64;
  static constexpr int kChunkBytes = 128 * 128;
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kQOff = 0;
  static constexpr int kKOff = kTileBytes;
  static constexpr int kVOff = 2 * kTileBytes;
  static constexpr int kXOff = 3 * kTileBytes;  // A' (8 KB) then B' (8 KB)
  static constexpr int kXBytes = 8192;
  static constexpr int kBarOff = kXOff + 2 * kXBytes;
  static constexpr int kSmemBytes = kBarOff + 1024 + 1024;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
  static constexpr uint32_t kTmemS0 = 0, kTmemS1 = 128, kTmemO = 256, kTmemCols = 512;
};

// MMAs of one item: QK(g0), QK(g0 + 1), then per block PV(g), QK(g + 2).
// Block g's scores live in S_(g & 1); s_full / p_full of a buffer complete
// once per block that uses it (phase g >> 1), and o_done alike: with one
// barrier for both, the last wait of an item could find two phases completed,
// and a wait for the parity of the older one then never returns.
struct Mma256Bars {
  uint64_t *q_full, *q_empty, *k_full, *k_empty, *v_full, *v_empty;
  uint64_t *s_full, *p_full, *o_done;  // [2] each
  volatile int *abort_flag;
};
template <bool kBF16, bool kFold>
__device__ bool mma_256(uint8_t *smem, const Mma256Bars &bars, uint32_t tmem, int nb, int tile_it, int g0) {
  using C = Cfg256;
  constexpr int D = C::D;
  constexpr uint32_t idesc_qk = idesc_f16(128, kBN, kBF16, false);
  constexpr uint32_t idesc_pv = idesc_f16(128, D, kBF16, true);
  const uint32_t q_base = smem_u32(smem + C::kQOff);
  const uint32_t k_base = smem_u32(smem + C::kKOff);
  const uint32_t v_base = smem_u32(smem + C::kVOff);
  const uint32_t x_base = smem_u32(smem + C::kXOff);
  auto wait = [&](uint64_t *bar, uint32_t par) {
    return mbar_wait_or_abort(bar, par, kTimeoutNs, bars.abort_flag);
  };
  auto issue_qk = [&](int buf) {
    const uint32_t d_tmem = tmem + (buf ? C::kTmemS1 : C::kTmemS0);
    uint64_t da = smem_desc_sw128(q_base, 16, 1024);
    uint64_t db = smem_desc_sw128(k_base, 16, 1024);
    asm volatile("" : "+l"(da), "+l"(db));
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint64_t off = (uint64_t)(((kk / 4) * C::kChunkBytes + (kk % 4) * 32) >> 4);
      mma_ss(d_tmem, da + off, db + off, idesc_qk, kk > 0 ? 1u : 0u);
    }
    if constexpr (kFold) {
      uint64_t dx = smem_desc_noswz(x_base, 128, 256);
      uint64_t dk = smem_desc_noswz(x_base + C::kXBytes, 128, 256);
      asm volatile("" : "+l"(dx), "+l"(dk));
      mma_ss(d_tmem, dx, dk, idesc_qk, 1u);
    }
  };
  auto issue_pv = [&](int buf, bool acc) {
    const uint32_t d_tmem = tmem + C::kTmemO;
    const uint32_t p_tmem = tmem + (buf ? C::kTmemS1 : C::kTmemS0);
    uint64_t db = smem_desc_sw128(v_base, C::kChunkBytes, 1024);
    asm volatile("" : "+l"(db));
#pragma unroll
    for (int kk = 0; kk < kBN / 16; ++kk)
      mma_ts(d_tmem, p_tmem + kk * 8, db + (uint64_t)((kk * 16 * 128) >> 4), idesc_pv, (acc || kk > 0) ? 1u : 0u);
  };
  // QK^T of block g (its K is in the single K slot).
  auto qk_block = [&](int g, bool last) {
    if (!wait(bars.k_full, g & 1)) return false;
    tc_fence_after();
    issue_qk(g & 1);
    tc_commit(&bars.s_full[g & 1]);
    tc_commit(bars.k_empty);
    if (last) tc_commit(bars.q_empty);
    return true;
  };
  if (!wait(bars.q_full, tile_it & 1)) return false;
  if (!qk_block(g0, nb == 1)) return false;
  if (nb > 1 && !qk_block(g0 + 1, nb == 2)) return false;
  for (int j = 0; j < nb; ++j) {
    const int g = g0 + j;
    if (!wait(bars.v_full, g & 1) || !wait(&bars.p_full[g & 1], (g >> 1) & 1)) return false;
    tc_fence_after();
    issue_pv(g & 1, j > 0);
    tc_commit(&bars.o_done[g & 1]);
    tc_commit(bars.v_empty);
    if (j + 2 < nb && !qk_block(g + 2, j + 3 == nb)) return false;
    if (*bars.abort_flag) return false;
  }
  return true;
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The soft-cap of the paged cache's kernels, tanh(v * in) * out + add, right to 2^-20
// of itself.  For |z| <= 1/2, z = v * in, it is z P(z^2), P of degree 4, fitted to
// tanh(z) / z by iteratively reweighted least squares on z times the error (2^-24);
// above, tanh is 1 - 2 / (1 + e^2|z|) by two special-function instructions.  Taken for
// a small z that form's error, 2^-22, does not shrink with z, and a large cap makes it
// an error of the score: 0.09 at a cap of 1e6.
constexpr float kCapSmall = 0.5f;
struct SoftCap {
  float in, out, k[5];  // the coefficients times out
  __device__ __forceinline__ SoftCap(float cap_in, float cap_out) : in(cap_in), out(cap_out) {
    constexpr float c[5] = {0.9999999403953552f, -0.3333277702331543f, 0.13320571184158325f, -0.05276213213801384f,
                            0.016737567260861397f};
#pragma unroll
    for (int i = 0; i < 5; ++i) k[i] = c[i] * cap_out;
  }
  __device__ __forceinline__ float operator()(float v, float add) const {
    const float z = __fmul_rn(v, in), w = __fmul_rn(z, z);
    float p = fmaf(k[4], w, k[3]);
    p = fmaf(p, w, k[2]);
    p = fmaf(p, w, k[1]);
    p = fmaf(p, w, k[0]);
    return fabsf(z) <= kCapSmall ? fmaf(z, p, add) : large(z, add);
  }
  // The same bits for a pair of raw scores; kSmall: both are (|v * in| <= 1/2).
  template <bool kSmall>
  __device__ __forceinline__ uint64_t pair(uint64_t v, uint64_t add) const;
  __device__ __forceinline__ float large(float z, float add) const {
    float u;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(u) : "f"(ex2_approx(fabsf(z) * (2.f * kLog2e)) + 1.f));
    return fmaf(copysignf(fmaf(-2.f, u, 1.f), z), out, add);
  }
};

// Score of column c (0..127 inside the block) in log2 units, before masking.
// kFast (the paged cache's kernels): SoftCap instead of tanhf.
template <bool kAlibi, bool kSoftcap, bool kFast = false>
__device__ __forceinline__ float score2(uint32_t raw, int c, float scale2, float slope2, float jf, float cap_in,
                                        float cap_out) {
  const float v = __uint_as_float(raw);
  float y = kSoftcap ? (kFast ? SoftCap(cap_in, cap_out)(v, 0.f) : tanhf(v * cap_in) * cap_out) : v * scale2;
  if (kAlibi) y = fmaf(slope2, (float)c, fmaf(slope2, jf, y));
  return y;
}

// Three-input max (sm_100 max.f32 with three sources).
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Columns of 32 raw scores (c0..c0+31) outside the row's visible interval
// [lo, hi) become -inf, in place: one bit test and one select per column.
// Used when the score transform maps -inf to -inf (no soft-cap), so the max
// and exponent passes then run unmasked (2^-inf = 0).
__device__ __forceinline__ void mask_chunk(uint32_t (&v)[32], int c0, int lo, int hi) {
  const int a = min(max(lo - c0, 0), 32), e = min(max(hi - c0, 0), 32);
  const uint32_t below_e = e >= 32 ? 0xffffffffu : ((1u << e) - 1u);
  const uint32_t below_a = a >= 32 ? 0xffffffffu : ((1u << a) - 1u);
  const uint32_t vis = below_e & ~below_a;
#pragma unroll
  for (int c = 0; c < 32; ++c) v[c] = (vis & (1u << c)) ? v[c] : 0xff800000u;
}

// Max of 32 scores (columns c0..c0+31), four independent chains.
template <bool kAlibi, bool kSoftcap, bool kMask, bool kFast = false>
__device__ __forceinline__ float chunk_max(const uint32_t (&v)[32], int c0, int lo, int hi, float scale2,
                                           float slope2, float jf, float cap_in, float cap_out) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = -CUDART_INF_F;
  if constexpr (!kAlibi) {
    // Without ALiBi the score transform is increasing (scale2 > 0, tanh), so
    // the row max is the transform of the raw max: one max per column.
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      float y0 = __uint_as_float(v[c]), y1 = __uint_as_float(v[c + 1]);
      if (kMask) {
        y0 = (c0 + c >= lo && c0 + c < hi) ? y0 : -CUDART_INF_F;
        y1 = (c0 + c + 1 >= lo && c0 + c + 1 < hi) ? y1 : -CUDART_INF_F;
      }
      m[(c >> 1) & 3] = fmax3(m[(c >> 1) & 3], y0, y1);
    }
    const float raw = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    return raw == -CUDART_INF_F ? raw : score2<false, kSoftcap, kFast>(__float_as_uint(raw), 0, scale2, 0.f, 0.f, cap_in, cap_out);
  } else {
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      float y0 = score2<kAlibi, kSoftcap, kFast>(v[c], c0 + c, scale2, slope2, jf, cap_in, cap_out);
      float y1 = score2<kAlibi, kSoftcap, kFast>(v[c + 1], c0 + c + 1, scale2, slope2, jf, cap_in, cap_out);
      if (kMask) {
        y0 = (c0 + c >= lo && c0 + c < hi) ? y0 : -CUDART_INF_F;
        y1 = (c0 + c + 1 >= lo && c0 + c + 1 < hi) ? y1 : -CUDART_INF_F;
      }
      m[(c >> 1) & 3] = fmax3(m[(c >> 1) & 3], y0, y1);
    }
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  }
}

// p = 2^(score - m) for 32 columns, packed in pairs into pk[0..15];
// returns the sum of the unrounded p (four independent chains).
template <typename T, bool kAlibi, bool kSoftcap, bool kMask, bool kFast = false>
__device__ __forceinline__ float chunk_exp(const uint32_t (&v)[32], uint32_t (&pk)[16], int c0, int lo, int hi,
                                           float scale2, float slope2, float jf, float cap_in, float cap_out,
                                           float m) {
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    float y0 = score2<kAlibi, kSoftcap, kFast>(v[c], c0 + c, scale2, slope2, jf, cap_in, cap_out);
    float y1 = score2<kAlibi, kSoftcap, kFast>(v[c + 1], c0 + c + 1, scale2, slope2, jf, cap_in, cap_out);
    if (kMask) {
      y0 = (c0 + c >= lo && c0 + c < hi) ? y0 : -CUDART_INF_F;
      y1 = (c0 + c + 1 >= lo && c0 + c + 1 < hi) ? y1 : -CUDART_INF_F;
    }
    const float p0 = ex2_approx(y0 - m), p1 = ex2_approx(y1 - m);
    s[(c >> 1) & 3] += p0 + p1;
    pk[c / 2] = pack2<T>(p0, p1);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Packed fp32 pairs (sm_100 f32x2 arithmetic): two lanes of work per
// instruction for the scale-and-subtract and the running sum of the plain
// (and folded-ALiBi) exponent pass.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// p = 2^(v * scale2 - m) for 32 raw scores (masked ones already -inf),
// packed in pairs into pk[0..15]; returns the sum of the unrounded p.
template <typename T>
__device__ __forceinline__ float chunk_exp_plain2(const uint32_t (&v)[32], uint32_t (&pk)[16], float scale2, float m) {
  uint64_t acc0 = f2(0.f, 0.f), acc1 = f2(0.f, 0.f);
  const uint64_t sc = f2(scale2, scale2), nm = f2(-m, -m);
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    float y0, y1;
    f2_split(fma2(f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), sc, nm), y0, y1);
    const float p0 = ex2_approx(y0), p1 = ex2_approx(y1);
    if ((c >> 1) & 1)
      acc1 = add2(acc1, f2(p0, p1));
    else
      acc0 = add2(acc0, f2(p0, p1));
    pk[c / 2] = pack2<T>(p0, p1);
  }
  float a, b, cc, d;
  f2_split(acc0, a, b);
  f2_split(acc1, cc, d);
  return (a + b) + (cc + d);
}

// Small scores need no special function, so that a soft-cap whose scores stay below
// half of it (the usual case) leaves those units to the softmax's own exponentials.  A
// warp takes 32 columns this way at a time where all of them are small enough, which
// decides the time only, no bit (the columns may be of rows or tokens that count for
// nothing): one sequence of 32,768 tokens, 4,096 queries, 32 heads over 8 of 128, 2.85 ms
// against 4.95 ms (which a cap of 2 on unit scores still takes), 1.73 ms without a cap.
template <bool kSmall>
__device__ __forceinline__ uint64_t SoftCap::pair(uint64_t v, uint64_t add) const {
  const uint64_t z = mul2(v, f2(in, in)), w = mul2(z, z);
  uint64_t p = fma2(f2(k[4], k[4]), w, f2(k[3], k[3]));
  p = fma2(p, w, f2(k[2], k[2]));
  p = fma2(p, w, f2(k[1], k[1]));
  p = fma2(p, w, f2(k[0], k[0]));
  p = fma2(z, p, add);
  if constexpr (kSmall) return p;
  float z0, z1, p0, p1, a0, a1;
  f2_split(z, z0, z1);
  f2_split(p, p0, p1);
  f2_split(add, a0, a1);
  return f2(fabsf(z0) <= kCapSmall ? p0 : large(z0, a0), fabsf(z1) <= kCapSmall ? p1 : large(z1, a1));
}
// The largest size of 32 raw scores (a NaN does not count: it stays one in P too).
__device__ __forceinline__ float chunk_size(const uint32_t (&v)[32]) {
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 32; c += 2)
    m[(c >> 1) & 3] = fmax3(m[(c >> 1) & 3], fabsf(__uint_as_float(v[c])), fabsf(__uint_as_float(v[c + 1])));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// chunk_exp with a soft-cap (masked ones are replaced after it).
template <typename T, bool kMask, bool kSmall>
__device__ __forceinline__ float chunk_exp_cap(const uint32_t (&v)[32], uint32_t (&pk)[16], int c0, int lo, int hi,
                                               const SoftCap &cap, float m) {
  uint64_t acc0 = f2(0.f, 0.f), acc1 = f2(0.f, 0.f);
  const uint64_t nm = f2(-m, -m);
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    float y0, y1;
    f2_split(cap.pair<kSmall>(f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), nm), y0, y1);
    if (kMask) {
      y0 = (c0 + c >= lo && c0 + c < hi) ? y0 : -CUDART_INF_F;
      y1 = (c0 + c + 1 >= lo && c0 + c + 1 < hi) ? y1 : -CUDART_INF_F;
    }
    const float p0 = ex2_approx(y0), p1 = ex2_approx(y1);
    if ((c >> 1) & 1)
      acc1 = add2(acc1, f2(p0, p1));
    else
      acc0 = add2(acc0, f2(p0, p1));
    pk[c / 2] = pack2<T>(p0, p1);
  }
  float a, b, cc, d;
  f2_split(acc0, a, b);
  f2_split(acc1, cc, d);
  return (a + b) + (cc + d);
}

// One KV block of one row: load S (128 columns, one TMEM round trip), row
// max, the rescale decision, P = 2^(s - m) written back over S as 16-bit
// pairs, and the running sum.  kMask selects the per-column interval test;
// the two variants are separate code paths.  kShift: P is taken 2^kShift times
// as large (and l with it), so that small weights keep fp16's bits.
template <typename T, bool kAlibi, bool kSoftcap, bool kMask, int kShift = 0, bool kFast = false>
__device__ __forceinline__ void softmax_block(uint32_t tS, int n0, int kv_offset, int lo, int hi, float scale2,
                                              float slope2,
                                              float cap_in, float cap_out, float &m_used, float &l, float &alpha,
                                              bool &rescale) {
  const float kNegInf = -CUDART_INF_F;
  const float jf = (float)(n0 + kv_offset);
  // An opaque per-block copy of the slope keeps the compiler from hoisting
  // 128 per-column products slope * c out of the block loop into registers.
  float sl = slope2;
  asm volatile("" : "+f"(sl));
  // ALiBi without soft-cap is folded into S (the per-column part beta * c,
  // see x_offset); what is left is one constant per block, added to the max
  // and taken out of the exponent's offset.  kCol: per-column bias here.
  constexpr bool kFold = kAlibi && !kSoftcap;
  constexpr bool kCol = kAlibi && !kFold;
  const float off = kFold ? sl * jf : 0.f;
  uint32_t sr[4][32];
#pragma unroll
  for (int q = 0; q < 4; ++q) tmem_ld32(tS + q * 32, sr[q]);
  tmem_wait_ld();
#pragma unroll
  for (int q = 0; q < 4; ++q) reg_fence32(sr[q]);
  // Without soft-cap the mask is applied once, to the raw scores; with it,
  // after the transform in both passes (tanh(-inf) is not -inf).
  constexpr bool kMaskRaw = kMask && !kSoftcap;
  constexpr bool kMaskPass = kMask && kSoftcap;
  if constexpr (kMaskRaw) {
#pragma unroll
    for (int q = 0; q < 4; ++q) mask_chunk(sr[q], q * 32, lo, hi);
  }
  float mx = kNegInf;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    mx = fmaxf(mx, chunk_max<kCol, kSoftcap, kMaskPass, kFast>(sr[q], q * 32, lo, hi, scale2, sl, jf, cap_in, cap_out));
  if constexpr (kFold) mx += off;  // -inf stays -inf
  // Fresh names for the raw scores: pass 2 recomputes each transformed
  // score instead of keeping pass 1's values alive next to the raw row.
#pragma unroll
  for (int q = 0; q < 4; ++q) reg_fence32(sr[q]);
  const float m_new = fmaxf(m_used, mx);
  if (m_used == kNegInf) {
    m_used = m_new;  // nothing accumulated yet: O and l are zero
  } else if (m_new > m_used + (rescale_threshold<T>() - (float)kShift)) {
    alpha = ex2_approx(m_used - m_new);
    m_used = m_new;
    rescale = true;
  }
  const float m_eff = ((m_used == kNegInf) ? 0.f : m_used) - (float)kShift;
  float psum = 0.f;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t pk[16];
    if constexpr (!kCol && !kSoftcap)
      psum += chunk_exp_plain2<T>(sr[q], pk, scale2, m_eff - off);
    else if constexpr (kFast && !kAlibi) {
      const SoftCap cap(cap_in, cap_out);
      psum += __all_sync(0xffffffffu, chunk_size(sr[q]) * cap_in <= kCapSmall)
                  ? chunk_exp_cap<T, kMaskPass, true>(sr[q], pk, q * 32, lo, hi, cap, m_eff)
                  : chunk_exp_cap<T, kMaskPass, false>(sr[q], pk, q * 32, lo, hi, cap, m_eff);
    } else
      psum += chunk_exp<T, kCol, kSoftcap, kMaskPass, kFast>(sr[q], pk, q * 32, lo, hi, scale2, sl, jf, cap_in, cap_out,
                                                    m_eff - off);
    tmem_st16(tS + q * 16, pk);
  }
  l = l * alpha + psum;
}

// 4 x 4 transpose of 16-byte pieces inside each group of four lanes: on
// entry u[j] is piece j of this lane's row, on exit u[k] is piece (lane % 4)
// of row k of the group.  Two rounds of exchanges with lane ^ 2 and lane ^ 1,
// each swapping the two pieces whose index bit differs from the lane's.
__device__ __forceinline__ void xchg_unit(uint4 &dst, const uint4 &src, int mask) {
  dst.x = __shfl_xor_sync(0xffffffffu, src.x, mask);
  dst.y = __shfl_xor_sync(0xffffffffu, src.y, mask);
  dst.z = __shfl_xor_sync(0xffffffffu, src.z, mask);
  dst.w = __shfl_xor_sync(0xffffffffu, src.w, mask);
}
__device__ __forceinline__ void transpose_units4(uint4 (&u)[4]) {
  const int i = threadIdx.x & 3;
  const bool b1 = (i >> 1) & 1, b0 = i & 1;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint4 send = b1 ? u[k] : u[k | 2];
    uint4 recv;
    xchg_unit(recv, send, 2);
    if (b1)
      u[k] = recv;
    else
      u[k | 2] = recv;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint4 send = b0 ? u[2 * k] : u[2 * k + 1];
    uint4 recv;
    xchg_unit(recv, send, 1);
    if (b0)
      u[2 * k] = recv;
    else
      u[2 * k + 1] = recv;
  }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

}  // namespace
}  // namespace llmx_b200
