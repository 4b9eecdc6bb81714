// Attention over the 4-bit key/value cache (include/llmx_attn.h): decode and
// short query blocks, one pass over the tiles.
//
// Mathematics.  A cached value is n s + m with a 4-bit n and s, m of its
// (token, 64-channel group).  Neither K nor V is dequantised:
//   q . K_j  = sum_h s_jh (q_h . n_jh) + m_jh sum(q_h)
//   sum_j p_j V_j = sum_j (p_j s_jh) (n_jh - 8) + sum_j p_j (m_jh + 8 s_jh)
// so the matrix products run on the integers themselves, which fp16 holds
// exactly, and the affine part is a few fp32 operations per token and group.
//   * K: the nibbles of a word are 4 + 4 bytes after two ANDs and a shift, and
//     go as they are into the integer tensor product (m16n8k32, u8 x s8, exact
//     in 32 bits).  q is a 16-bit integer of its row's largest value (steps of
//     1/32512), its high and low byte two products.  What its rounding leaves of
//     a group's sum, times 8, is where the product starts: the rounding then
//     meets n - 8 and not n.
//   * V: a nibble OR-ed into 1024 (0x6400) and 1032 (or 1152 = 1024 + 128 for
//     bits 4-7) subtracted is n - 8 (16 (n - 8)), two operations per two
//     values.  Centred, because the tensor core's fp32 accumulation would
//     otherwise carry a mean of 7.5 through the whole sequence that cancels
//     only at the end.
//   * p s is rounded to fp16 (2^-11 relative at most), after a scale by a power
//     of two that brings the largest s seen so far to [2^7, 2^8).  Scores, p,
//     the softmax sums and the affine part stay fp32.
//
// Shape.  S^T = K q^T with 16 tokens as rows and 8 columns of (head, query row)
// pairs of one kv head; O^T += V^T P^T (m16n8k16, fp16) with channels as rows.
// The cache's tile layout is the order of these fragments, so K and V go from
// linear copies in shared memory to registers to the tensor core; P^T changes
// from the accumulator's layout to the operand's with one 8x8 transpose
// (movmatrix) per 8 tokens and group.  mma.sync and not tcgen05: the operands
// are made in registers, 8 columns are all there are in a decode, and the
// products are not what bounds the pass (the tensor pipe is a quarter filled).
//
// Work.  A unit is one (sequence, kv head, block of pairs); its tokens are cut
// into steps of one or two tiles.  Short units have a worker each.  Of longer
// ones the steps of all, end to end, are dealt to the resident workers in equal
// shares: sequences of any lengths finish together.  With many units a worker
// is a warp, which copies its tiles into its own ring in shared memory (one
// bulk copy a tile, issued ahead across unit boundaries); with few it is a CTA,
// whose warps take every fourth step and are merged in shared memory (COOP;
// plan_kv4() chooses).  A worker writes the result of a unit that it has whole.
// Of a unit that several share each writes a partial result (at most two a
// worker, so the workspace does not grow with the sequences), and a second
// kernel merges them.
//
// Measured on one B200 (bytes of the visible cache, q and o): 64 sequences of
// 256-4096 tokens, 32 heads of 128, ALiBi: 126-135 us from box to box, 4.8-5.1
// TB/s (0.73-0.78 of the copy rate); 32 sequences of 1001-8191 tokens, 32 heads
// on 8: 47 us, 3.6 TB/s; 131071 tokens, 32 heads on 8: 41 us, 3.7 TB/s.  Nothing
// is full: DRAM 0.48-0.65 of its peak, issue slots 0.54-0.60, the integer pipe
// that unpacks the nibbles 0.41-0.59.  A tile's scores, softmax and output
// product are one chain of results, and at 16 warps an SM (128 registers) a warp
// mostly waits for its own last one.  More warps with fewer registers (20 of 96)
// ran 15-25% slower, fewer with more (12 of 168) 4-8%.  With 8 pairs a warp at
// head_dim 128 the registers do not hold all: 28 bytes are spilled and 100 read
// back by warps, 60 and 92 by CTAs.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "kv4.cuh"
#include "sm100_ptx.cuh"

namespace llmx_b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum of a row moves only when a score passes it by this
// much (log2): p reaches 2^6 at most, and p s at most 2^14 in fp16.
constexpr float kLazyMax = 6.f;
constexpr float kQTop = 32512.f;  // 127 * 256: q's largest value as an integer
// The largest weight times the largest step that its row sees stays in
// [2^7, 2^8) (times 2^6 under a lazy maximum): fp16 then keeps 11 bits of
// weights down to 2^-21 of the largest.  Steps count from 2^-40 on (smaller
// ones lose bits from 2^-61 on), and a centre m + 8 s counts as a step of 2^-20
// of it: this keeps the sums of scaled weights, and of these times the centres,
// inside fp32.
constexpr int kStepExp = 7;
constexpr float kCentreStep = 0x1p-20f;
constexpr int kMinStepExp = -40;
constexpr int kMaxStepExp = 125;
// A weight below 2^-126 is 0 and missing from its row's sum as well.  bf16 has
// steps up to 2^125, which would leave the weights 8 binades; their products
// with the steps take a factor of 2^-kFarShift there, so that the weights keep
// 48 (and reach 2^93 beside the smallest steps).
constexpr int kFarShift = 40;
constexpr uint64_t kWaitNs = 1000000000ull;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 4-bit integers (one a byte) times the bytes of q, exact in 32 bits.
__device__ __forceinline__ void imma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from the columns' starting values x (even) and y (odd).
__device__ __forceinline__ void imma16832_first(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1, int x, int y) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(x), "r"(y));
}

// 8x8 transpose of 16-bit elements across the warp: lane (g, t) gives row g,
// columns 2t, 2t + 1 and gets row 2t, 2t + 1 of column g.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// (x & mask) | bits in one operation.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
  return r;
}

// (n - 8) of the nibbles in bits 0-3 of both halves; 16 (n - 8) of bits 4-7.
__device__ __forceinline__ uint32_t centred_lo(uint32_t z) {
  const uint32_t u = and_or(z, 0x000f000fu, 0x64006400u), c = 0x64086408u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t centred_hi(uint32_t z) {
  const uint32_t u = and_or(z, 0x00f000f0u, 0x64006400u), c = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float pow2i(int e) {  // 2^e for e in [-126, 127]
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Tokens that row i sees: [lo, hi).
__device__ __forceinline__ void row_range(const AttnArgs &a, int i, int ql, int kl, int &lo, int &hi) {
  const int diag = i + kl - ql;
  hi = a.causal ? max(0, min(kl, diag + 1)) : kl;
  lo = a.window >= 0 ? max(0, diag - a.window) : 0;
}

// ALiBi counts from the token of the row's largest bias, which changes no weight:
// slope j itself would take the scores' last bits with it far into a sequence
// (2^-7 of 158,000 at a slope of 0.84 and 131,072 tokens).  The log-sum-exp gets
// slope times this token back.
__device__ __forceinline__ int bias_origin(float slope, int lo, int hi) { return slope > 0.f ? hi - 1 : lo; }

// The tokens of sequence b that its rows see between them, as steps of W
// tiles from a 16-token boundary (rows' ranges move one way: the first row's
// begin to the last row's end).
struct Span {
  int first, steps;
  int blocks;  // of R pairs (a power of two)
};
template <int W>
__device__ __forceinline__ Span span_of(const AttnArgs &a, int R, int ql, int kl) {
  Span s = {0, 0, 0};
  if (ql > 0 && kl > 0) {
    int lo, hi, x;
    row_range(a, 0, ql, kl, lo, x);
    row_range(a, ql - 1, ql, kl, x, hi);
    s.first = lo & ~15;
    if (hi > lo) {
      s.steps = (hi - s.first + 16 * W - 1) / (16 * W);
      s.blocks = (ql * a.group + R - 1) >> (31 - __clz(R));
    }
  }
  return s;
}

// A launch's part of the batch and its shares.
struct Work {
  int b0, nb;      // sequences
  int R;           // pairs of a block
  int workers;     // warps (CTAs, where a CTA's warps work together) that take a share, at most
  int min_steps;   // a share is at least this long, unless units are shorter
  int units;       // at most
  int split;       // 0: shares end where units end
};
constexpr int kMaxSlice = 512;

// Shares: worker w of `n` (below 2^16) has the steps [begin(w), begin(w + 1)) of
// `total` (below 2^31, which the host sees to), begin(w) = floor(total w / n)
// without a 64-bit division.
__device__ __forceinline__ uint32_t share_begin(uint32_t total, int w, int n) {
  const uint32_t each = total / n, rest = total - each * n;
  return each * w + rest * w / n;
}
// The share of a step: an estimate (within one of it, n being small), put right.
__device__ __forceinline__ int share_of(uint32_t total, uint32_t step, int n) {
  int w = min(n - 1, (int)__fdividef((float)step * (float)n, (float)total));
  while (w > 0 && share_begin(total, w, n) > step) --w;
  while (w < n - 1 && share_begin(total, w + 1, n) <= step) ++w;
  return w;
}
__device__ __forceinline__ int share_count(const Work &wk, uint32_t total) {
  const uint32_t n = max(total / wk.min_steps, min(total, (uint32_t)wk.units));
  return (int)min(max(n, 1u), (uint32_t)wk.workers);
}

// Steps of all units before each sequence of the slice, prefix[nb] their sum,
// and the sequences' query and key lengths.
// Called by all of the CTA's kThreads threads; ends with a barrier.
template <int W>
__device__ __forceinline__ void scan_steps(const AttnArgs &a, const Work &wk, uint32_t *prefix, int2 *lens, uint32_t *tmp) {
  const int tid = threadIdx.x, lane = tid % 32;
  const int per = (wk.nb + kThreads - 1) / kThreads;
  uint32_t sum = 0;
  for (int i = tid * per; i < min(wk.nb, (tid + 1) * per); ++i) {
    const int b = wk.b0 + i;
    prefix[i] = sum;
    lens[i] = make_int2(clamp_len(a.q_lens, b, a.Sq), clamp_len(a.kv_lens, b, a.Skv));
    const Span sp = span_of<W>(a, wk.R, lens[i].x, lens[i].y);
    sum += (uint32_t)sp.steps * sp.blocks * a.Hkv;
  }
  uint32_t up = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, up, off);
    if (lane >= off) up += x;
  }
  if (lane == 31) tmp[tid / 32] = up;
  __syncthreads();
  uint32_t before = up - sum;
  for (int w = 0; w < tid / 32; ++w) before += tmp[w];
  for (int i = tid * per; i < min(wk.nb, (tid + 1) * per); ++i) prefix[i] += before;
  if (tid == kThreads - 1) prefix[wk.nb] = before + sum;
  __syncthreads();
}

// Where a step of the slice lies.
struct Place {
  int b, ql, kl;   // sequence
  int kvh, block;  // unit
  int first;       // first token of the unit's steps
  int at, steps;   // step in its unit, and the unit's steps
};
template <int W>
__device__ __forceinline__ Place place_of(const AttnArgs &a, const Work &wk, const uint32_t *prefix, const int2 *lens, uint32_t step) {
  int lo = 0, hi = wk.nb - 1;  // the last sequence that begins at or before the step
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (prefix[mid] <= step) lo = mid;
    else hi = mid - 1;
  }
  Place p;
  p.b = wk.b0 + lo;
  p.ql = lens[lo].x;
  p.kl = lens[lo].y;
  const Span sp = span_of<W>(a, wk.R, p.ql, p.kl);
  const uint32_t rest = step - prefix[lo];
  const int unit = (int)(rest / (uint32_t)sp.steps);
  p.first = sp.first;
  p.steps = sp.steps;
  p.at = (int)(rest - (uint32_t)unit * sp.steps);
  p.kvh = unit / sp.blocks;
  p.block = unit - p.kvh * sp.blocks;
  return p;
}

__device__ __forceinline__ uint32_t word_of(const uint4 &u, int i) {
  return i == 0 ? u.x : (i == 1 ? u.y : (i == 2 ? u.z : u.w));
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}

// The K words of group h: [token g, g + 8][8-channel word] from this lane's
// place in a tile (layout: word x = (r G + h) 2 + w).
template <int G>
__device__ __forceinline__ void lds_k(uint32_t (&k)[2][2], uint32_t addr, int h) {
  if constexpr (G == 1) {
    const uint4 u = lds16(addr);
    k[0][0] = u.x;
    k[0][1] = u.y;
    k[1][0] = u.z;
    k[1][1] = u.w;
  } else {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int x = (r * G + h) * 2;
      asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                   : "=r"(k[r][0]), "=r"(k[r][1])
                   : "r"(addr + x / 4 * 512 + x % 4 * 4));
    }
  }
}

// The parameter words of one token's K or V.
template <int G>
__device__ __forceinline__ void lds_params(uint32_t (&w)[G], uint32_t addr) {
  if constexpr (G == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  } else if constexpr (G == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  } else {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr));
  }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&f)[4]) {
  const float x[8] = {f[0], f[1], f[2], f[3], 0.f, 0.f, 0.f, 0.f};
  const uint4 u = pack8<T>(x);
  *reinterpret_cast<uint2 *>(p) = make_uint2(u.x, u.y);
}

// One contiguous tile, global -> this CTA's shared memory, counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Sizes of one variant: 8 columns, SLOTS tiles side by side in them.  With few
// pairs (8 / SLOTS or less) the columns hold the pairs SLOTS times, once per
// tile: q is 0 in the columns of the other tiles, so the
// products of all tiles add up in one accumulator without mixing, and the
// whole softmax part runs once for SLOTS tiles.
//
// NQ = 2: a thread works on columns 2t and 2t + 1, two pairs.  NQ = 1, for
// fewer pairs still: one pair has both, with the low byte of q in the odd one.
template <int D, int NQ, int SLOTS, bool COOP>
struct Shape {
  static constexpr int G = D / kKv4Group;
  static constexpr int kCols = 8;
  static constexpr int kTileCols = kCols / SLOTS;          // columns of one tile
  static constexpr int R = kTileCols / (NQ == 1 ? 2 : 1);  // pairs a warp takes
  static constexpr int kTile = 18 * D;
  static constexpr int W = D == 256 ? 1 : 2;  // tiles of a step: copied and waited for together
  static constexpr int kStages = D == 64 ? 4 : (D == 128 ? 2 : 3);
  static constexpr int kMinCtas = G <= 2 ? 4 : 3;
  static constexpr int kRing = kStages * W * kTile;
  static constexpr int kQFrag = G * 2 * 32 * 16;
  static constexpr int kRows = kCols * (5 + 2 * G) * 4;  // factor, slope, lo, hi, origin, sums and starts of the groups
  // Each warp's ring; q and its columns, of each warp or of all; as many
  // zeros as q for the other tiles' columns; lengths and prefix sums.
  static constexpr int kZeros = SLOTS > 1 ? kQFrag : 0;
  static constexpr int kSmem = kWarps * kRing + (COOP ? 1 : kWarps) * (kQFrag + kRows) + kZeros;
  static constexpr int kMergeRow = D + 4;  // floats of a row in the ring when warps are merged
  static_assert(W % SLOTS == 0, "a step holds whole groups of tiles");
  static_assert(R * kMergeRow * 4 <= kRing, "a warp's result fits its ring");
};

template <typename T, int D, int NQ, int SLOTS, bool COOP>
__global__ void __launch_bounds__(kThreads, Shape<D, NQ, SLOTS, COOP>::kMinCtas)
    kv4_attn_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Kv4Args c, const __grid_constant__ Work wk,
                    float *part_o, float *part_lse) {
  using Sh = Shape<D, NQ, SLOTS, COOP>;
  constexpr int G = Sh::G, R = Sh::R, kStages = Sh::kStages, W = Sh::W, kCols = Sh::kCols;
  // The other column of a lone pair takes what fp16 leaves of its weights: free,
  // and of use where the output has fp16's own 11 bits.
  constexpr bool kLow = NQ == 1 && std::is_same<T, __half>::value;
  constexpr int kFar = std::is_same<T, __nv_bfloat16>::value ? kFarShift : 0;  // fp16 steps stay below 2^16
  constexpr int kTileCols = Sh::kTileCols, kColStep = NQ == 1 ? 2 : 1;  // pair r of a tile has column r * kColStep
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t sm_full[kWarps][kStages];
  __shared__ uint32_t sm_tmp[kWarps];
  __shared__ float sm_m[kWarps][R], sm_l[kWarps][R];  // with COOP: each warp's references and sums
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int g = lane >> 2, t = lane & 3;
  unsigned char *own = smem + warp * Sh::kRing;
  unsigned char *q_at0 = smem + kWarps * Sh::kRing + (COOP ? 0 : warp) * (Sh::kQFrag + Sh::kRows);
  uint4 *q_own = reinterpret_cast<uint4 *>(q_at0);
  float *row_f = reinterpret_cast<float *>(q_at0 + Sh::kQFrag);
  float *row_slope = row_f + kCols;
  int *row_lo = reinterpret_cast<int *>(row_f + 2 * kCols), *row_hi = row_lo + kCols;
  int *row_origin = row_lo + 2 * kCols;
  float *row_qs = row_f + 5 * kCols;                           // [G][kCols]
  int *row_begin = reinterpret_cast<int *>(row_qs + G * kCols);  // [G][kCols]
  unsigned char *zeros = smem + Sh::kSmem - Sh::kZeros;
  int2 *lens = reinterpret_cast<int2 *>(smem + Sh::kSmem);               // [nb]
  uint32_t *prefix = reinterpret_cast<uint32_t *>(lens + wk.nb);         // [nb + 1]

  // The merge kernel may be set up while this one runs.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(&sm_full[warp][i], W);
    sm100::fence_mbar_init();
  }
  for (int i = tid; i < Sh::kZeros / 16; i += kThreads) reinterpret_cast<uint4 *>(zeros)[i] = make_uint4(0u, 0u, 0u, 0u);
  scan_steps<W>(a, wk, prefix, lens, sm_tmp);

  // Neighbouring shares go to different CTAs, so that few of them spread over the SMs.
  const int worker = COOP ? blockIdx.x : warp * gridDim.x + blockIdx.x;
  const uint32_t total = prefix[wk.nb];

  // Rows that see nothing, past their sequence's or in one without a visible
  // key, are 0.
  for (int i = warp * gridDim.x + blockIdx.x; i < wk.nb; i += kWarps * gridDim.x) {
    const int b = wk.b0 + i;
    const int r0 = prefix[i + 1] == prefix[i] ? 0 : lens[i].x;
    for (long long e = lane; e < (long long)(a.Sq - r0) * a.H * (D / 8); e += 32) {
      const int d = (int)(e % (D / 8)) * 8, h = (int)(e / (D / 8) % a.H), r = r0 + (int)(e / (D / 8) / a.H);
      T *op = static_cast<T *>(a.o) + b * a.os[0] + r * a.os[1] + h * a.os[2] + d;
#pragma unroll
      for (int x = 0; x < 8; ++x) op[x] = Elem<T>::from_f(0.f);
      if (a.lse != nullptr && d == 0) a.lse[((long long)b * a.H + h) * a.Sq + r] = -CUDART_INF_F;
    }
  }
  if (total == 0) return;

  uint32_t begin, end;
  if (wk.split) {
    const int n = share_count(wk, total);
    if (worker >= n) return;
    begin = share_begin(total, worker, n);
    end = share_begin(total, worker + 1, n);
  } else if (wk.units <= wk.workers) {
    // Whole units, one for each worker.
    const int per_seq = wk.units / wk.nb, i = worker / per_seq, unit = worker - i * per_seq;
    if (i >= wk.nb) return;
    const Span sp = span_of<W>(a, wk.R, lens[i].x, lens[i].y);
    if (unit >= sp.blocks * a.Hkv) return;
    begin = prefix[i] + (uint32_t)unit * sp.steps;
    end = begin + sp.steps;
  } else {
    // Whole units: a share ends with the unit that holds its last step.
    auto snap = [&](uint32_t step) {
      if (step >= total) return total;
      const Place pl = place_of<W>(a, wk, prefix, lens, step);
      return pl.at == 0 ? step : step - pl.at + pl.steps;
    };
    begin = snap(share_begin(total, worker, wk.workers));
    end = snap(share_begin(total, worker + 1, wk.workers));
  }
  // Steps of the share; this warp takes those with index k0 + kEvery i.
  const int mine = (int)(end - begin);
  constexpr int kEvery = COOP ? kWarps : 1;
  const int k0 = COOP ? warp : 0;

  // Steps in the order of the shares; with ALiBi a unit's last tokens come
  // first: the bias grows with the token, so the maxima are there from the
  // start and rarely move.
  const bool reverse = a.alibi != nullptr;
  const int tpp = c.page_size >> 4;
  const uint32_t ring = sm100::smem_u32(own);
  uint64_t *bar = &sm_full[warp][0];

  // Lane W j + u of the warp keeps where tile u of its step (n 32 / W + j)
  // lies, and issues its copy.  Bit W j + u of `bad`: the page of that tile is
  // outside the cache.
  constexpr int kBatch = 32 / W;
  // A warp on its own runs ahead into the next unit; warps together stop at
  // the unit's end, `last`, where the rings serve the merge.
  const unsigned char *where = nullptr;
  uint32_t bad_now = 0, bad_issue = 0;
  int last = mine, locate_from = 0;
  auto locate = [&](int first) {
    const int i = first + lane / W;
    where = nullptr;
    bool bad = false;
    if (k0 + kEvery * i < last) {
      const Place pl = place_of<W>(a, wk, prefix, lens, begin + k0 + kEvery * i);
      const int tile = (pl.first >> 4) + W * (reverse ? pl.steps - 1 - pl.at : pl.at) + lane % W;
      if (tile * 16 < pl.kl) {
        const int page = tile / tpp;
        const long long off = kv4_page_offset(c, pl.b, page);
        bad = off < 0;
        if (!bad) where = c.data + pl.kvh * c.head_stride + off + (long long)(tile - page * tpp) * Sh::kTile;
      }
    }
    bad_issue = __ballot_sync(0xffffffffu, bad);
  };
  auto issue = [&](int i, int stage) {
    if (lane / W == (i - locate_from) % kBatch) {
      if (where != nullptr) {
        sm100::mbar_arrive_expect_tx(bar + stage, Sh::kTile);
        bulk_load(ring + (W * stage + lane % W) * Sh::kTile, where, Sh::kTile, bar + stage);
      } else {
        sm100::mbar_arrive(bar + stage);
      }
    }
  };
  if constexpr (!COOP) {
    locate(0);
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (i < mine) issue(i, i);
  }

  // Where this lane's column finds q for tile `sl`: in its own tile's columns,
  // elsewhere zeros.
  const int my_slot = SLOTS > 1 ? 2 * t / kTileCols : 0;  // tile of this lane's accumulator columns 2t, 2t + 1
  uint32_t q_at[SLOTS];
#pragma unroll
  for (int sl = 0; sl < SLOTS; ++sl)
    q_at[sl] = (SLOTS > 1 && g / kTileCols != sl ? sm100::smem_u32(zeros) : sm100::smem_u32(q_own)) + lane * 16;

  uint32_t at = ring, phase = 0;
  uint64_t wait_ns = kWaitNs;
  int stage = 0;
  int mine_done = 0;  // steps that this warp has taken
  for (int done = 0, n_steps; done < mine; done += n_steps) {
    // ---- the next unit, or the share's part of it
    const Place pl = place_of<W>(a, wk, prefix, lens, begin + done);
    const int b = pl.b, kvh = pl.kvh, r0 = pl.block * R, ql = pl.ql, kl = pl.kl, first = pl.first;
    const int rows = ql * a.group;  // pair r: query row r / group, head r % group of the kv head
    n_steps = min(mine - done, pl.steps - pl.at);
    const int before = mine_done;
    if constexpr (COOP) {
      // The warp's steps of this unit: indexes i from `before` on with k0 + kEvery i < last.
      last = done + n_steps;
      locate_from = before;
      locate(before);
#pragma unroll
      for (int i = 0; i < kStages; ++i)
        if (k0 + kEvery * (before + i) < last) issue(before + i, (stage + i) % kStages);
    }
    // Tokens [lo_in, hi_in) are seen by all rows of the block.
    int lo_in = 0, hi_in = 0;
    {
      int x;
      row_range(a, r0 / a.group, ql, kl, x, hi_in);
      row_range(a, (min(r0 + R, rows) - 1) / a.group, ql, kl, lo_in, x);
    }

    // q as 16-bit integers of its row's largest value, high and low byte, in
    // the order of the operand fragments; with the factor that undoes the
    // scale and the sums of the groups.  A lane takes 16 channels of a pair.
    // An infinity makes the factor NaN, a NaN the sums.
    __syncwarp();
    constexpr int kLanes = D / 16, kPass = 32 / kLanes;  // lanes of a pair, pairs side by side
#pragma unroll
    for (int p0 = COOP ? warp * kPass : 0; p0 < R; p0 += COOP ? kWarps * kPass : kPass) {
      const int pr = p0 + lane / kLanes, sub = lane % kLanes, r = r0 + pr;
      const bool here = R % kPass == 0 || pr < R, live = here && r < rows;
      const int i = r / a.group, h0 = kvh * a.group + r % a.group;
      uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
      if (live) {
        const T *p = static_cast<const T *>(a.q) + b * a.qs[0] + i * a.qs[1] + h0 * a.qs[2] + 16 * sub;
        if (c.vec) {
          raw[0] = reinterpret_cast<const uint4 *>(p)[0];
          raw[1] = reinterpret_cast<const uint4 *>(p)[1];
        } else {
          const unsigned short *e = reinterpret_cast<const unsigned short *>(p);
          uint32_t u[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) u[x] = (uint32_t)e[2 * x] | ((uint32_t)e[2 * x + 1] << 16);
          raw[0] = make_uint4(u[0], u[1], u[2], u[3]);
          raw[1] = make_uint4(u[4], u[5], u[6], u[7]);
        }
      }
      float f[2][8], top = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        unpack8<T>(raw[w], f[w]);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          top = fmaxf(top, fabsf(f[w][x]));
          sum += f[w][x];
        }
      }
#pragma unroll
      for (int off = 1; off < kLanes; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float up = top > 0.f ? fminf(kQTop / top, 0x1p126f) : 0.f;
      const float scale = a.softcap > 0.f ? a.sm_scale / a.softcap : a.sm_scale * kLog2e;
      const int h = sub >> 2, tt = sub & 3;
      float left = 0.f;  // of the group's sum, in steps
      if (here) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t hi8[2] = {0u, 0u}, lo8[2] = {0u, 0u};
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            // A word's even channels are the low nibbles of its bytes (the
            // first half of the 32 the product sums over), the odd ones the high.
            const int v = __float2int_rn(f[w][x] * up);
            left += fmaf(f[w][x], up, -(float)v);
            hi8[x & 1] |= (uint32_t)((v + 128) >> 8 & 255) << (8 * (x >> 1));
            lo8[x & 1] |= (uint32_t)(v & 255) << (8 * (x >> 1));
          }
#pragma unroll
          for (int sl = 0; sl < SLOTS; ++sl) {
            const int col = sl * kTileCols + pr * kColStep;
            uint4 *dst = q_own + (((col >> 3) * G + h) * 2 + w) * 32 + 4 * (col & 7) + tt;
            dst[0] = make_uint4(hi8[0], hi8[1], lo8[0], lo8[1]);
            if constexpr (NQ == 1) dst[4] = make_uint4(lo8[0], lo8[1], 0u, 0u);
          }
        }
      }
      left += __shfl_xor_sync(0xffffffffu, left, 1);
      left += __shfl_xor_sync(0xffffffffu, left, 2);
      if (here) {
#pragma unroll
        for (int sl = 0; sl < SLOTS; ++sl) {
          const int col = sl * kTileCols + pr * kColStep;
          if (tt == 0) {
            row_qs[h * kCols + col] = sum * scale;
            // The low byte's columns start with it; with NQ = 1 those are the odd ones.
            row_begin[h * kCols + col + kColStep - 1] = __float2int_rn(8.f * left);
            if constexpr (NQ == 1) row_begin[h * kCols + col] = 0;
          }
          if (sub == 0) {
            int lo, hi;
            row_range(a, live ? i : ql - 1, ql, kl, lo, hi);  // a column without a row goes with the last one
            row_f[col] = up > 0.f ? scale / up : (top > 0.f ? CUDART_NAN_F : 0.f);
            const float slope = live && a.alibi != nullptr ? a.alibi[h0] * kLog2e : 0.f;
            row_slope[col] = slope;
            row_origin[col] = bias_origin(slope, lo, hi);
            row_lo[col] = lo;
            row_hi[col] = hi;
          }
        }
      }
    }
    if constexpr (COOP) __syncthreads();
    else __syncwarp();

    // Weights are kept as 2^(S - ref) with one reference per row: the running
    // maximum less a power of two that brings the largest step times the
    // largest weight into fp16's upper range (kStepExp).
    float o[G][4][4];
    float l[NQ], aff[NQ][G], ref[NQ];
    // What a score starts from: minus its row's reference, which with a
    // soft-cap comes off behind the tanh.  0 while there is none.
    float start[NQ], after[NQ];
    int step_exp[NQ];                    // of the steps that the row has seen
    bool fresh = true;                   // some row has no reference yet (the same in all lanes)
    float limit = 0.f, next_step = 0.f;  // a score above `limit` or a step from `next_step` on moves the references
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[h][i][x] = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      l[q] = start[q] = after[q] = 0.f;
      ref[q] = -CUDART_INF_F;
      step_exp[q] = kMinStepExp;
#pragma unroll
      for (int h = 0; h < G; ++h) aff[q][h] = 0.f;
    }

    // SLOTS tiles at shared address `at`, tokens tok0 ..  PART: some row does
    // not see all of their tokens; bit u of `lost`: tile u has no page.
    auto compute = [&](uint32_t at, int tok0, uint32_t lost, auto part_tag) {
      constexpr bool PART = decltype(part_tag)::value;
      const uint32_t mine_at = at + my_slot * Sh::kTile;  // the tile of this lane's columns
      const int tok = tok0 + 16 * my_slot + g;
      // ---- scores, less the rows' references
      float s[2][NQ];
      {
        // High and low byte of q; with NQ = 1 columns 2t and 2t + 1 of one.
        constexpr int B = NQ == 1 ? 1 : 2;
        int acc[G][B][4];
#pragma unroll
        for (int sl = 0; sl < SLOTS; ++sl)
#pragma unroll
          for (int h = 0; h < G; ++h) {
            uint32_t kw[2][2];  // [token g, g + 8][word]
            lds_k<G>(kw, at + sl * Sh::kTile + lane * 16, h);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t a0 = kw[0][w] & 0x0f0f0f0fu, a2 = (kw[0][w] >> 4) & 0x0f0f0f0fu;
              const uint32_t a1 = kw[1][w] & 0x0f0f0f0fu, a3 = (kw[1][w] >> 4) & 0x0f0f0f0fu;
              const uint4 qw = lds16(q_at[sl] + (h * 2 + w) * 512);
              if (w == 0 && sl == 0) {
                const int2 begin = *reinterpret_cast<const int2 *>(&row_begin[h * kCols + 2 * t]);
                if constexpr (B == 2) imma16832_first(acc[h][0], a0, a1, a2, a3, qw.x, qw.y, 0, 0);
                imma16832_first(acc[h][B - 1], a0, a1, a2, a3, B == 2 ? qw.z : qw.x, B == 2 ? qw.w : qw.y, begin.x, begin.y);
              } else {
                imma16832(acc[h][0], a0, a1, a2, a3, qw.x, qw.y);
                if constexpr (B == 2) imma16832(acc[h][B - 1], a0, a1, a2, a3, qw.z, qw.w);
              }
            }
          }
        float2 kp[2][G];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t par[G];
          lds_params<G>(par, mine_at + G * 1024 + (g + 8 * r) * (8 * G));
#pragma unroll
          for (int h = 0; h < G; ++h) kp[r][h] = kv4_unpack_param<T>(par[h]);
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const float fac = row_f[2 * t + q];
          float qs[G];
#pragma unroll
          for (int h = 0; h < G; ++h) qs[h] = row_qs[h * kCols + 2 * t + q];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float dot = 0.f, off = start[q];
#pragma unroll
            for (int h = 0; h < G; ++h) {
              const int sum = NQ == 1 ? acc[h][0][2 * r] * 256 + acc[h][0][2 * r + 1]
                                      : acc[h][0][2 * r + q] * 256 + acc[h][B - 1][2 * r + q];
              dot = h == 0 ? kp[r][h].x * (float)sum : fmaf(kp[r][h].x, (float)sum, dot);
              off = fmaf(kp[r][h].y, qs[h], off);
            }
            s[r][q] = fmaf(dot, fac, off);
          }
        }
      }
      if (a.softcap > 0.f) {
        const float cap2 = a.softcap * kLog2e;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int q = 0; q < NQ; ++q) s[r][q] = fmaf(tanhf(s[r][q]), cap2, after[q]);
      }
      if (a.alibi != nullptr) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const float slope = row_slope[2 * t + q], dist = (float)(tok - row_origin[2 * t + q]);
#pragma unroll
          for (int r = 0; r < 2; ++r) s[r][q] = fmaf(slope, dist + 8.f * r, s[r][q]);
        }
      }
      uint32_t vis = 0;  // bit r NQ + q; only with PART
      if constexpr (PART) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const int lo = row_lo[2 * t + q], hi = row_hi[2 * t + q];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int j = tok + 8 * r;
            if (j >= lo && j < hi && !(lost >> my_slot & 1u)) vis |= 1u << r * NQ + q;
            else s[r][q] = -CUDART_INF_F;
          }
        }
      }
      // ---- V's steps and centres; a token that no row sees may hold anything
      float sv[2][G], cv[2][G];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t par[G];
        lds_params<G>(par, mine_at + G * 1024 + (g + 8 * r) * (8 * G) + 4 * G);
        bool dead = false;
        if constexpr (PART) {
          dead = true;
#pragma unroll
          for (int q = 0; q < NQ; ++q) dead = dead && !(vis >> r * NQ + q & 1u);
        }
#pragma unroll
        for (int h = 0; h < G; ++h) {
          float2 p = kv4_unpack_param<T>(par[h]);
          if (dead) p = make_float2(0.f, 0.f);
          sv[r][h] = p.x;
          cv[r][h] = fmaf(8.f, p.x, p.y);
        }
      }
      // ---- the references move, with everything accumulated, when a score
      // passes its row's maximum by kLazyMax or a larger step turns up
      float most = -CUDART_INF_F, smax = 0.f, cmax = 0.f;
#pragma unroll
      for (int q = 0; q < NQ; ++q) most = max3(most, s[0][q], s[1][q]);
#pragma unroll
      for (int h = 0; h < G; ++h) {
        smax = max3(smax, sv[0][h], sv[1][h]);
        cmax = max3(cmax, fabsf(cv[0][h]), fabsf(cv[1][h]));
      }
      if (__any_sync(0xffffffffu, fresh || most > limit || smax >= next_step || cmax * kCentreStep >= next_step)) {
        uint32_t bits[2] = {0u, 0u};  // the largest finite step of each token
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < G; ++h) {
            const uint32_t x = __float_as_uint(fmaxf(sv[r][h], fabsf(cv[r][h]) * kCentreStep));
            bits[r] = max(bits[r], x < 0x7f800000u ? x : 0u);
          }
        bool missing = false;
        int least = kMaxStepExp, largest = kMinStepExp;  // exponents of this thread's rows
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          // Of the tokens that the row sees: a large step that it does not
          // see must not push its weights out of fp16.
          uint32_t top = max(!PART || (vis >> q & 1u) ? bits[0] : 0u, !PART || (vis >> NQ + q & 1u) ? bits[1] : 0u);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
          const int new_exp = max(step_exp[q], min(kMaxStepExp, (int)(top >> 23) - 127));
          const float old_room = (float)(kStepExp + kFar - step_exp[q]), new_room = (float)(kStepExp + kFar - new_exp);
          step_exp[q] = new_exp;
          least = min(least, new_exp);
          largest = max(largest, new_exp);
          const bool none = ref[q] == -CUDART_INF_F;
          const float shift = none ? 0.f : ref[q];
          float v = fmaxf(s[0][q], s[1][q]) + shift;
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
          const float m = none ? v : fmaxf(ref[q] + old_room, v);
          const float now = m == -CUDART_INF_F ? m : m - new_room;
          // In two halves: steps 2^126 apart still add up in the sum of weights.
          const float root = none ? 1.f : exp2_fast(0.5f * (ref[q] - now)), al = root * root;
          const float back = now == -CUDART_INF_F ? 0.f : shift - now;
          ref[q] = now;
          missing |= now == -CUDART_INF_F;
          const float minus = now == -CUDART_INF_F ? 0.f : -now;
          start[q] = a.softcap > 0.f ? 0.f : minus;
          after[q] = minus;
          s[0][q] += back;
          s[1][q] += back;
          l[q] = l[q] * root * root;
#pragma unroll
          for (int h = 0; h < G; ++h) {
            aff[q][h] *= al;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[h][i][q] *= al;
              o[h][i][2 + q] *= al;
              if constexpr (kLow) {
                o[h][i][1] *= al;
                o[h][i][3] *= al;
              }
            }
          }
        }
        // The lower of two rows' thresholds: at worst the references are looked at more often.
        limit = kLazyMax + (float)(kStepExp + kFar - largest);
        next_step = pow2i(least + 1);
        fresh = __any_sync(0xffffffffu, missing);
      }
      // ---- weights
      uint32_t pf[G][2];
      {
        float p[2][NQ];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            p[r][q] = exp2_fast(s[r][q]);
            l[q] += p[r][q];
          }
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float w[2] = {0.f, 0.f};
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
              w[q] = (kFar > 0 ? p[r][q] * pow2i(-kFar) : p[r][q]) * sv[r][h];
              if constexpr (PART) {
                const bool ok = vis >> r * NQ + q & 1u;
                if (!ok) w[q] = 0.f;
                aff[q][h] += ok ? p[r][q] * cv[r][h] : 0.f;
              } else {
                aff[q][h] = fmaf(p[r][q], cv[r][h], aff[q][h]);
              }
            }
            if constexpr (kLow) w[1] = w[0] - __half2float(__float2half_rn(w[0]));
            pf[h][r] = transpose8x8(pack_half2(w[0], w[1]));
          }
      }
      // ---- O^T += V^T P^T, each tile with its own columns
#pragma unroll
      for (int sl = 0; sl < SLOTS; ++sl) {
        const uint32_t tile = at + sl * Sh::kTile + G * 512;
        uint4 vw[G];
#pragma unroll
        for (int i = 0; i < G; ++i) vw[i] = lds16(tile + i * 512 + lane * 16);
#pragma unroll
        for (int h = 0; h < G; ++h) {
          uint32_t w[4], pb[2];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = word_of(vw[(k * G + h) / 4], (k * G + h) % 4);
#pragma unroll
          for (int r = 0; r < 2; ++r) pb[r] = SLOTS == 1 || g / kTileCols == sl ? pf[h][r] : 0u;
#pragma unroll
          for (int part16 = 0; part16 < 2; ++part16) {
            uint32_t z0 = __byte_perm(w[0], w[1], part16 ? 0x7632 : 0x5410);
            uint32_t z1 = __byte_perm(w[2], w[3], part16 ? 0x7632 : 0x5410);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t a0 = centred_lo(z0), a1 = centred_hi(z0), a2 = centred_lo(z1), a3 = centred_hi(z1);
              mma16816(o[h][2 * part16 + half], a0, a1, a2, a3, pb[0], pb[1]);
              z0 >>= 8;
              z1 >>= 8;
            }
          }
        }
      }
    };

    // Steps [whole_lo, whole_lo + whole) of the unit lie inside what every row sees.
    const int whole_lo = max(0, (lo_in - first + 16 * W - 1) / (16 * W));
    const int whole = max(0, (hi_in - first) / (16 * W) - whole_lo);
    for (int k; (k = k0 + kEvery * mine_done) < done + n_steps; ++mine_done) {
      // A copy that does not arrive in a second (never seen to happen) sets
      // the error word; the warp goes on without waiting again.
      if (!sm100::mbar_wait(bar + stage, phase, wait_ns)) {
        raise_error(a.err, kDevErrTimeout);
        wait_ns = 0;
      }
      const int in_batch = (mine_done - locate_from) % kBatch;
      if (in_batch == 0) bad_now = bad_issue;
      const int order = pl.at + k - done;
      const int st = reverse ? pl.steps - 1 - order : order;
      const int tok0 = first + 16 * W * st;
      const uint32_t lost = bad_now >> (in_batch * W) & ((1u << W) - 1u);
#pragma unroll
      for (int u = 0; u < W; u += SLOTS) {
        if ((unsigned)(st - whole_lo) < (unsigned)whole && lost == 0)
          compute(at + u * Sh::kTile, tok0 + 16 * u, 0u, std::false_type{});
        else
          compute(at + u * Sh::kTile, tok0 + 16 * u, lost >> u, std::true_type{});
      }
      const int next = mine_done + kStages;
      if ((next - locate_from) % kBatch == 0) locate(next);
      __syncwarp();  // the warp has read the stage
      if (k0 + kEvery * next < last) issue(next, stage);
      at += W * Sh::kTile;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
        at = ring;
      }
    }

    // What the log-sum-exp of pair `pr` gets back.
    auto origin_bias = [&](int h0, int pr) {
      return a.alibi != nullptr ? a.alibi[h0] * (float)row_origin[pr * kColStep] : 0.f;
    };

    // ---- the unit's result: sums over the tokens (lanes with the same t hold
    // the same rows), then over the tiles' columns
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[q] += __shfl_xor_sync(0xffffffffu, l[q], off);
#pragma unroll
        for (int h = 0; h < G; ++h) aff[q][h] += __shfl_xor_sync(0xffffffffu, aff[q][h], off);
      }
      float out[G][8];
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float even = o[h][i][q], odd = o[h][i][2 + q];
          if constexpr (kLow) {
            even += o[h][i][1];
            odd += o[h][i][3];
          }
          out[h][2 * i] = fmaf(even, pow2i(kFar), aff[q][h]);
          out[h][2 * i + 1] = fmaf(odd, 0.0625f * pow2i(kFar), aff[q][h]);
        }
      float m = ref[q], sum = l[q];
      if constexpr (SLOTS == 2) {
        const float other = __shfl_xor_sync(0xffffffffu, m, 2);
        const float both = fmaxf(m, other);
        // Columns that saw no finite score add nothing, unless their sum is a NaN.
        const float root = m == -CUDART_INF_F ? (sum == sum ? 0.f : 1.f) : exp2_fast(0.5f * (m - both)), wt = root * root;
        m = both;
        sum = sum * root * root;
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            out[h][x] = wt == 0.f ? 0.f : out[h][x] * wt;
            out[h][x] += __shfl_xor_sync(0xffffffffu, out[h][x], 2);
          }
      }
      const int pr = (2 * t + q) % kTileCols / kColStep, r = r0 + pr;
      if constexpr (COOP) {
        if (my_slot == 0 && r < rows) {
          float *dst = reinterpret_cast<float *>(own) + pr * Sh::kMergeRow + 8 * g;
#pragma unroll
          for (int h = 0; h < G; ++h) {
            *reinterpret_cast<float4 *>(dst + 64 * h) = make_float4(out[h][0], out[h][1], out[h][2], out[h][3]);
            *reinterpret_cast<float4 *>(dst + 64 * h + 4) = make_float4(out[h][4], out[h][5], out[h][6], out[h][7]);
          }
          if (g == 0) {
            sm_m[warp][pr] = m;
            sm_l[warp][pr] = sum;
          }
        }
      } else if (my_slot == 0 && r < rows) {
        const bool none = sum == 0.f;
        const float inv = 1.f / sum;
        const float lse = none ? -CUDART_INF_F : (m == -CUDART_INF_F ? sum : (m + log2f(sum)) * kLn2);
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int x = 0; x < 8; ++x) out[h][x] = none ? 0.f : out[h][x] * inv;
        const int i = r / a.group, h0 = kvh * a.group + r % a.group;
        if (n_steps == pl.steps) {
          T *op = static_cast<T *>(a.o) + b * a.os[0] + i * a.os[1] + h0 * a.os[2] + 8 * g;
#pragma unroll
          for (int h = 0; h < G; ++h) {
            if (c.vec) {
              *reinterpret_cast<uint4 *>(op + 64 * h) = pack8<T>(out[h]);
            } else {
#pragma unroll
              for (int x = 0; x < 8; ++x) op[64 * h + x] = Elem<T>::from_f(out[h][x]);
            }
          }
          if (a.lse != nullptr && g == 0) a.lse[((long long)b * a.H + h0) * a.Sq + i] = lse + origin_bias(h0, pr);
        } else {
          // Slot 1 for the unit that begins in this share, slot 0 for the
          // one that began before it.
          const long long row = ((long long)worker * 2 + (pl.at == 0 ? 1 : 0)) * R + pr;
          float *dst = part_o + row * D + 8 * g;
#pragma unroll
          for (int h = 0; h < G; ++h) {
            *reinterpret_cast<float4 *>(dst + 64 * h) = make_float4(out[h][0], out[h][1], out[h][2], out[h][3]);
            *reinterpret_cast<float4 *>(dst + 64 * h + 4) = make_float4(out[h][4], out[h][5], out[h][6], out[h][7]);
          }
          if (g == 0) part_lse[row] = lse;
        }
      }
    }
    if constexpr (COOP) {
      // The warps' sums, four channels a thread.
      __syncthreads();
      const int live = min(R, rows - r0);
      for (int e = tid; e < live * (D / 4); e += kThreads) {
        const int pr = e / (D / 4), d = e % (D / 4) * 4;
        float mw[kWarps], top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          mw[w] = sm_m[w][pr];
          top = fmaxf(top, mw[w]);
        }
        float sum = 0.f;
        float4 ov = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float lw = sm_l[w][pr];
          // A warp that saw no finite score adds nothing, unless its sum is a NaN.
          if (mw[w] == -CUDART_INF_F && lw == lw) continue;
          const float root = mw[w] == -CUDART_INF_F ? 1.f : exp2_fast(0.5f * (mw[w] - top)), wt = root * root;
          const float4 x = *reinterpret_cast<const float4 *>(smem + w * Sh::kRing + (pr * Sh::kMergeRow + d) * 4);
          sum = fmaf(lw * root, root, sum);
          ov.x = fmaf(x.x, wt, ov.x);
          ov.y = fmaf(x.y, wt, ov.y);
          ov.z = fmaf(x.z, wt, ov.z);
          ov.w = fmaf(x.w, wt, ov.w);
        }
        const bool none = sum == 0.f;
        const float inv = none ? 0.f : 1.f / sum;
        const float lse = none ? -CUDART_INF_F : (top == -CUDART_INF_F ? sum : (top + log2f(sum)) * kLn2);
        ov = make_float4(ov.x * inv, ov.y * inv, ov.z * inv, ov.w * inv);
        const int r = r0 + pr, i = r / a.group, h0 = kvh * a.group + r % a.group;
        if (n_steps == pl.steps) {
          T *op = static_cast<T *>(a.o) + b * a.os[0] + i * a.os[1] + h0 * a.os[2] + d;
          if (c.vec) {
            const float f[4] = {ov.x, ov.y, ov.z, ov.w};
            store4<T>(op, f);
          } else {
            op[0] = Elem<T>::from_f(ov.x);
            op[1] = Elem<T>::from_f(ov.y);
            op[2] = Elem<T>::from_f(ov.z);
            op[3] = Elem<T>::from_f(ov.w);
          }
          if (a.lse != nullptr && d == 0) a.lse[((long long)b * a.H + h0) * a.Sq + i] = lse + origin_bias(h0, pr);
        } else {
          const long long row = ((long long)worker * 2 + (pl.at == 0 ? 1 : 0)) * R + pr;
          *reinterpret_cast<float4 *>(part_o + row * D + d) = ov;
          if (d == 0) part_lse[row] = lse;
        }
      }
      // The next unit's copies come after these reads and writes.
      sm100::fence_proxy_async_smem();
      __syncthreads();
    }
  }
  if (wait_ns == 0) {
    // Copies may still be in flight: they get a last second each before the
    // shared memory goes to another CTA.  (Both parities: which one is due
    // differs from stage to stage.)
    for (int st = 0; st < kStages; ++st)
      for (uint32_t ph = 0; ph < 2; ++ph) sm100::mbar_wait(bar + st, ph, kWaitNs);
  }
}

// O = sum_s exp(lse_s - lse) O_s over the shares of a unit that several workers
// have.  A warp per output row, or with many shares a CTA of PARTS warps, which
// take every PARTS-th one.  A lane has D / 32 channels; eight shares are read at
// a time, before their weights are known: what this kernel takes is the latency
// of a few loads in a row.
constexpr int kAtOnce = 8;
template <typename T, int D, int W, int PARTS>
__global__ void __launch_bounds__(PARTS > 1 ? PARTS * 32 : kThreads) kv4_merge_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Work wk,
                                                             const float *part_o, const float *part_lse) {
  constexpr int E = D / 32;
  __shared__ float sm_m[PARTS], sm_l[PARTS], sm_o[PARTS][PARTS > 1 ? D : 1];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t out_row = PARTS > 1 ? blockIdx.x : blockIdx.x * kWarps + warp;  // (below 2^31: direct_fits())
  const uint32_t query = out_row / a.H;
  const int h = (int)(out_row - query * a.H), n = (int)(query / a.Sq), i = (int)(query - n * a.Sq), b = wk.b0 + n;
  int w0 = 0, used = 0, R = wk.R, r = 0;
  if (n < wk.nb) {
    // Steps before this sequence, and of all.
    uint32_t before = 0, all = 0;
    for (int x = lane; x < wk.nb; x += 32) {
      const Span sp = span_of<W>(a, R, clamp_len(a.q_lens, wk.b0 + x, a.Sq), clamp_len(a.kv_lens, wk.b0 + x, a.Skv));
      const uint32_t s = (uint32_t)sp.steps * sp.blocks * a.Hkv;
      all += s;
      if (x < n) before += s;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    const int ql = clamp_len(a.q_lens, b, a.Sq);
    const Span sp = span_of<W>(a, R, ql, clamp_len(a.kv_lens, b, a.Skv));
    if (i < ql && sp.steps > 0) {  // the others are 0 already
      const int shares = share_count(wk, all);
      r = i * a.group + h % a.group;
      const uint32_t first = before + (uint32_t)(h / a.group * sp.blocks + r / R) * sp.steps;
      w0 = share_of(all, first, shares);
      used = share_of(all, first + sp.steps - 1, shares) - w0 + 1;
    }
  }
  // Every thread waits for the shares to be written, also where there is
  // nothing to do, so that this kernel ends after them.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (used <= 1) return;  // one worker had the unit whole
  float m = -CUDART_INF_F, sum = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s0 = PARTS > 1 ? warp : 0; s0 < used; s0 += kAtOnce * PARTS) {
    float l[kAtOnce], x[kAtOnce][E];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int s = s0 + u * PARTS;
      l[u] = -CUDART_INF_F;
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = 0.f;
      if (s < used) {
        const long long row = ((long long)(w0 + s) * 2 + (s == 0 ? 1 : 0)) * R + r % R;
        l[u] = part_lse[row];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 v = *reinterpret_cast<const float2 *>(part_o + row * D + lane * E + e);
          x[u][e] = v.x;
          x[u][e + 1] = v.y;
        }
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) top = fmaxf(top, l[u]);
    const float al = m == -CUDART_INF_F ? 0.f : expf(m - top);
    m = top;
    sum *= al;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= al;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float w = l[u] == -CUDART_INF_F ? 0.f : expf(l[u] - top);  // a NaN goes on into the sum
      sum += w;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(w, x[u][e], o[e]);
    }
  }
  if constexpr (PARTS > 1) {
    if (lane == 0) {
      sm_m[warp] = m;
      sm_l[warp] = sum;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_o[warp][lane * E + e] = o[e];
    __syncthreads();
    if (warp != 0) return;
    m = sm_m[0];
#pragma unroll
    for (int w = 1; w < PARTS; ++w) m = fmaxf(m, sm_m[w]);
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < PARTS; ++w) {
      const float wt = sm_m[w] == -CUDART_INF_F ? (sm_l[w] == sm_l[w] ? 0.f : 1.f) : expf(sm_m[w] - m);
      sum = fmaf(sm_l[w], wt, sum);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(sm_o[w][lane * E + e], wt, o[e]);
    }
  }
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  T *op = static_cast<T *>(a.o) + b * a.os[0] + i * a.os[1] + h * a.os[2] + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = Elem<T>::from_f(o[e] * inv);
  if (a.lse != nullptr && lane == 0) {
    float bias = 0.f;
    if (a.alibi != nullptr) {
      int lo, hi;
      row_range(a, i, clamp_len(a.q_lens, b, a.Sq), clamp_len(a.kv_lens, b, a.Skv), lo, hi);
      bias = a.alibi[h] * (float)bias_origin(a.alibi[h], lo, hi);
    }
    a.lse[((long long)b * a.H + h) * a.Sq + i] = none ? -CUDART_INF_F : m + logf(sum) + bias;
  }
}

struct Plan {
  int rows;        // (head, query row) pairs of one kv head
  int variant;     // 0: 2 pairs, 1: 4 pairs, 2: 8 pairs a worker
  int R, tiles;    // pairs of a block, tiles of a step
  bool coop;       // a CTA's warps share units
  int ctas;        // of one launch
  int nb;          // sequences of one launch
  bool shared;     // several workers may have to share a unit
  int per_unit;    // about so many
  size_t ws_bytes;
};

Plan plan_kv4(const AttnArgs &a) {
  Plan p;
  p.rows = a.group * a.Sq;
  p.variant = a.D == 256 ? 2 : (p.rows <= 2 ? 0 : (p.rows <= 4 ? 1 : 2));
  p.R = 2 << p.variant;
  p.tiles = a.D == 256 ? 1 : 2;
  // Tokens that a sequence's rows can see between them.
  long long span = a.Skv;
  if (a.window >= 0) span = std::min<long long>(span, (long long)a.window + a.Sq + 15);
  const long long steps = (span + 15 + 16 * p.tiles - 1) / (16 * p.tiles);
  const long long per_seq = (long long)a.Hkv * ((p.rows + p.R - 1) / p.R);
  // (direct_fits() keeps one sequence's steps below 2^31.)
  p.nb = (int)std::min<long long>(std::min(a.B, kMaxSlice), std::max<long long>(1, 0x7fffffffLL / (per_seq * steps)));
  const long long units = p.nb * per_seq, most = units * steps;
  // (At head_dim 256 only two fit beside the lengths of more than 256 sequences,
  // and a third of the shares then comes after the others.  Launches of 256
  // sequences instead cost another start and merge: 512 sequences of 1024-2048
  // tokens, 8 heads on 2, 141 us against 167, but 300 of 512-1024 88 against 78,
  // so it is left.)
  const int resident = a.num_sms * (a.D <= 128 ? 4 : 3);
  // Short sequences: a unit has one worker, which saves the merge's launch and
  // the second part of a share.  Longer ones are shared out; with many units by
  // warps, with few by CTAs (equal at about a third of the resident CTAs at
  // head_dim 128, half of them at 64, all at 256).  Measured, us, 4 heads on each
  // kv head, head_dim 128, half to all of the given tokens a sequence, whole /
  // shared by CTAs / shared by warps:
  //   256 units  600: 13.3 / 17.9 / 18.7   2000: 23 / 27.9 / 27.6    4000: 41 / 36.1 / 35.9
  //   512 units  600: 18.1 / 26.1 / 25.8   2000: 37.5 / 40.1 / 38.0  4000: 59.9 / 59.9 / 56.2
  // and whole by warps / shared by warps:
  //   1024 units  300: 17.4 / 25.6   600: 27.9 / 32.1   1200: 47.8 / 43.4
  // The rule shares earlier than these would, since one long sequence among short
  // ones has to wait for a single worker.
  const bool few = units <= resident;
  const bool whole = steps <= (few ? 32 + units / 10 : 20);
  p.coop = few && (whole || units * (a.D == 256 ? 1 : (a.D == 128 ? 3 : 2)) <= resident);
  p.shared = !whole;
  p.ctas = (int)std::min<long long>(resident, p.shared || !p.coop ? (most + kWarps - 1) / kWarps : units);
  const long long workers = (long long)p.ctas * (p.coop ? 1 : kWarps);
  p.per_unit = (int)std::min<long long>(workers, (workers + units - 1) / units);
  p.ws_bytes = p.shared ? (size_t)workers * 2 * p.R * (a.D + 1) * sizeof(float) : 0;
  return p;
}

template <typename T, int D, int NQ, int SLOTS, bool COOP>
cudaError_t launch_variant(const AttnArgs &a, const Kv4Args &c, const Plan &p, bool split, void *ws, cudaStream_t s) {
  using Sh = Shape<D, NQ, SLOTS, COOP>;
  const int smem = Sh::kSmem + p.nb * 12 + 4;
  // The limit on dynamic shared memory is the most that any slice takes, the same
  // value from every call: host threads that launch at the same time cannot
  // lower it for one another, in whatever order they come.  Once for each
  // device, since setting it costs a microsecond a launch.
  constexpr int most = Sh::kSmem + kMaxSlice * 12 + 4;
  static std::atomic<bool> allowed[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // (48 KB without the attribute, the kernel's static part, under 1 KB, among them.)
  if (most > 47 * 1024 && (dev < 0 || dev >= 64 || !allowed[dev].load())) {
    e = cudaFuncSetAttribute(kv4_attn_kernel<T, D, NQ, SLOTS, COOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) allowed[dev].store(true);
  }
  const size_t workers = (size_t)p.ctas * (COOP ? 1 : kWarps);
  float *part_o = static_cast<float *>(ws);
  float *part_lse = split ? part_o + workers * 2 * p.R * D : nullptr;
  for (int b0 = 0; b0 < a.B; b0 += p.nb) {
    Work wk;
    wk.b0 = b0;
    wk.nb = std::min(p.nb, a.B - b0);
    wk.R = p.R;
    wk.workers = (int)workers;
    // A share of CTAs has at least two steps a warp.  Measured, us with 4 / 8 /
    // 16 / 32 steps, 32 heads on 8 of 128: 1 sequence of 2048 tokens 8.9 / 9.4 /
    // 10.8 / 13.8, of 8192 12.0 / 11.4 / 12.5 / 14.4, 4 of 8192 19.3 / 19.4 /
    // 16.7 / 19.6, 16 of 2048 20.2 / 20.2 / 16.6 / 19.5; 1 of 16384, 16 heads on 4
    // of 64: 12.0 / 10.6 / 10.9 / 12.2.
    wk.min_steps = COOP ? 2 * kWarps : 1;
    wk.units = (int)std::min<long long>(0x7fffffff, (long long)wk.nb * a.Hkv * ((p.rows + p.R - 1) / p.R));
    wk.split = split ? 1 : 0;
    kv4_attn_kernel<T, D, NQ, SLOTS, COOP><<<p.ctas, kThreads, smem, s>>>(a, c, wk, part_o, part_lse);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    if (!split) continue;
    // The merge's launch overlaps the shares; it waits for them itself.
    // Warps of a row by its shares.  Measured, us of the whole call with 1 / 4 / 8
    // warps, 32 heads on 8 of 128: 5 shares 20.1 / 20.1 / 23.7 (16 sequences of
    // 2048 tokens), 10 41.3 / 40.9 / 47.2 (32 of 4096), 19 21.9 / 19.4 / 19.4 (4 of
    // 8192), 64 16.2 / 11.7 / 11.4 (1 of 8192), 74 29.8 / 19.4 / 17.7 (1 of 32768).
    const int parts = p.per_unit > 32 ? 8 : (p.per_unit > 8 ? 4 : 1);
    const long long out_rows = (long long)wk.nb * a.Sq * a.H;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(parts > 1 ? out_rows : (out_rows + kWarps - 1) / kWarps));
    cfg.blockDim = dim3(parts > 1 ? parts * 32 : kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const auto merge = parts == 8 ? kv4_merge_kernel<T, D, Sh::W, 8>
                                  : (parts == 4 ? kv4_merge_kernel<T, D, Sh::W, 4> : kv4_merge_kernel<T, D, Sh::W, 1>);
    e = cudaLaunchKernelEx(&cfg, merge, a, wk, (const float *)part_o, (const float *)part_lse);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T, int D, bool COOP>
cudaError_t launch_coop(const AttnArgs &a, const Kv4Args &c, const Plan &p, bool split, void *ws, cudaStream_t s) {
  if constexpr (D < 256) {
    if (p.variant == 0) return launch_variant<T, D, 1, 2, COOP>(a, c, p, split, ws, s);
    if (p.variant == 1) return launch_variant<T, D, 2, 2, COOP>(a, c, p, split, ws, s);
  }
  return launch_variant<T, D, 2, 1, COOP>(a, c, p, split, ws, s);
}

template <typename T, int D>
cudaError_t launch_d(const AttnArgs &a, const Kv4Args &c, const Plan &p, bool split, void *ws, cudaStream_t s) {
  return p.coop ? launch_coop<T, D, true>(a, c, p, split, ws, s) : launch_coop<T, D, false>(a, c, p, split, ws, s);
}

template <typename T>
cudaError_t launch_kv4_attn(const AttnArgs &a, const Kv4Args &c, const Plan &p, bool split, void *ws, cudaStream_t s) {
  switch (a.D) {
    case 64: return launch_d<T, 64>(a, c, p, split, ws, s);
    case 128: return launch_d<T, 128>(a, c, p, split, ws, s);
    case 256: return launch_d<T, 256>(a, c, p, split, ws, s);
  }
  return cudaErrorNotSupported;
}

// The expanded form: K and V of every sequence as dense 16-bit rows in the
// workspace, followed by the prefill's own workspace.
size_t expanded_rows_bytes(const AttnArgs &a) {
  return ((size_t)a.B * a.Skv * a.Hkv * a.D * 2 + 255) / 256 * 256;
}

// The prefill request over rows at `ws`; false where the prefill cannot run it.
bool expanded_request(const AttnArgs &a, unsigned char *ws, AttnArgs *e) {
  *e = a;
  e->k = ws;
  e->v = ws + expanded_rows_bytes(a);
  for (long long *st : {e->ks, e->vs}) {
    st[2] = a.D;
    st[1] = (long long)a.D * a.Hkv;
    st[0] = st[1] * a.Skv;
  }
  return a.Sq > 1 && sm100_supports(*e);
}

// Which form AUTO takes, by what both were measured to cost on B200 (us):
//   direct    8 + 0.0005 a 16-token tile, kv head and block of 8 pairs (twice
//             that at head_dim 256): the unpacking is done again for each block
//   expanded  10 + the expansion's bytes at 5.5 TB/s + 1.95 a block of 128 keys
//             and wave of work items (256 query rows of a head; 128 at head_dim
//             256): the prefill's items do not share their keys' axis
// e.g. 2 sequences of 8192 tokens, 32 heads of 128 on 8 kv heads: 64 query rows
// 129 against 142 us, 128 rows 242 against 142; one of 65536 tokens: 64 rows
// 456 against 989, 512 rows 3517 against 992.  The expanded rows may take
// kExpandedBytes at most: max_kv_len may be far above the lengths in use.
constexpr double kExpandedBytes = 4294967296.0;
bool expanded_is_faster(const AttnArgs &a) {
  const double wide = a.D == 256 ? 2.0 : 1.0;
  double span = a.Skv;
  if (a.window >= 0) span = std::min<double>(span, (double)a.window + a.Sq + 15);
  const double blocks = ((double)a.group * a.Sq + 7) / 8;
  const double direct = 8 + 0.0005 * wide * a.B * a.Hkv * std::floor(blocks) * (span / 16);
  const double rows = (double)a.B * a.Skv * a.Hkv * a.D;
  const double item_rows = a.D == 256 ? 128 : 256;
  const double waves = std::ceil((double)a.B * a.H * std::ceil(a.Sq / item_rows) / a.num_sms);
  const double expanded = 10 + rows * 5.125 / 5.5e6 + 1.95 * waves * (span / 128);
  return 4 * rows <= kExpandedBytes && expanded < direct;
}

// The direct form counts steps and output rows in 31 bits.
bool direct_fits(const AttnArgs &a) {
  const double pairs = (double)a.group * a.Sq;
  return ((double)a.Skv / 16 + 2) * a.Hkv * (pairs / 2 + 1) < 2147483647.0 &&
         (double)std::min(a.B, kMaxSlice) * a.Sq * a.H < 2147483647.0;
}

// Whether the request runs expanded; `s` gets the refusal of a forced form.
bool use_expanded(const AttnArgs &a, int algo, llmx_status *s) {
  AttnArgs e;
  // Any 256-byte aligned address stands for the workspace here.
  const bool can = expanded_request(a, reinterpret_cast<unsigned char *>(uintptr_t(256)), &e);
  *s = LLMX_OK;
  if (algo == LLMX_ALGO_TCGEN05 && !can)
    *s = record_error(LLMX_ERR_UNSUPPORTED,
                      "kv4: TCGEN05 needs max_q_len > 1, sm_scale > 0 and 16-byte aligned rows of q and o");
  const bool direct = direct_fits(a);
  const bool expand = can && (algo == LLMX_ALGO_TCGEN05 || (algo == LLMX_ALGO_AUTO && (!direct || expanded_is_faster(a))));
  if (*s == LLMX_OK && !expand && !direct)
    *s = record_error(LLMX_ERR_UNSUPPORTED,
                      "kv4: too many query rows for the direct form (max_kv_len / 16 * n_heads * max_q_len / 2 must stay below 2^31)");
  return expand;
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

llmx_status bad(const char *msg) { return record_error(LLMX_ERR_INVALID_ARGUMENT, msg); }

llmx_status check(const llmx_attn_params *p, const llmx_kv4_cache *c, AttnArgs *a, Kv4Args *k) {
  llmx_status s = validate_without_kv(p, a);
  if (s != LLMX_OK) return s;
  s = validate_kv4(c, p->batch, k);
  if (s != LLMX_OK) return s;
  if (p->dtype != c->dtype) return bad("kv4: q must have the cache's dtype");
  if (p->n_kv_heads != c->n_kv_heads || p->head_dim != c->head_dim)
    return bad("kv4: n_kv_heads and head_dim must be the cache's");
  if ((long long)p->max_kv_len > (long long)c->max_pages * c->page_size)
    return bad("kv4: max_kv_len must be at most max_pages * page_size");
  if (p->kv_offset != 0 || p->kv_total != 0) return bad("kv4: key shards (kv_offset, kv_total) are not supported");
  if (p->algo == LLMX_ALGO_SIMT) return record_error(LLMX_ERR_UNSUPPORTED, "kv4: algo must be AUTO, DECODE or TCGEN05");
  if (((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->o)) & 1u) != 0)
    return bad("kv4: q and o must be aligned to their elements");
  const int64_t extent[3] = {p->batch, p->max_q_len, p->n_heads};
  for (int i = 0; i < 3; ++i)
    if (p->o_stride[i] == 0 && extent[i] > 1) return bad("kv4: rows of o must not overlap (stride 0)");
  k->vec = al16(p->q) && al16(p->o);
  for (int i = 0; i < 3; ++i) k->vec = k->vec && p->q_stride[i] % 8 == 0 && p->o_stride[i] % 8 == 0;
  a->window = std::min(a->window, 1 << 30);  // past every length; keeps the ranges inside 32 bits
  return LLMX_OK;
}

}  // namespace
}  // namespace llmx_b200

using namespace llmx_b200;

extern "C" llmx_status llmx_kv4_attn_workspace_size(const llmx_attn_params *p, const llmx_kv4_cache *c, size_t *bytes) {
  AttnArgs a;
  Kv4Args k;
  const llmx_status s = check(p, c, &a, &k);
  if (s != LLMX_OK) return s;
  if (bytes == nullptr) return bad("bytes is NULL");
  unsigned int *err = nullptr;
  int sms = 0;
  if (current_device_info(&err, &sms) == LLMX_OK) a.num_sms = sms;
  llmx_status refused;
  const bool expand = use_expanded(a, p->algo, &refused);
  if (refused != LLMX_OK) return refused;
  *bytes = expand ? 2 * expanded_rows_bytes(a) + kSm100WorkspaceBytes : plan_kv4(a).ws_bytes;
  return LLMX_OK;
}

extern "C" llmx_status llmx_kv4_attn_fwd(const llmx_attn_params *p, const llmx_kv4_cache *c, void *stream) {
  AttnArgs a;
  Kv4Args k;
  llmx_status s = check(p, c, &a, &k);
  if (s != LLMX_OK) return s;
  s = current_device_info(&a.err, &a.num_sms);
  if (s != LLMX_OK) return s;
  k.err = a.err;
  if (p->workspace != nullptr && !al16(p->workspace)) return bad("workspace must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  llmx_status refused;
  bool expand = use_expanded(a, p->algo, &refused);
  const size_t rows = expanded_rows_bytes(a);
  if (expand && (p->workspace == nullptr || p->workspace_bytes < 2 * rows + kSm100WorkspaceBytes)) {
    // AUTO then takes the direct form, which needs no workspace, where that can run.
    if (p->algo != LLMX_ALGO_AUTO || !direct_fits(a))
      return record_error(LLMX_ERR_WORKSPACE_TOO_SMALL,
                          "kv4: the expanded form needs the workspace that llmx_kv4_attn_workspace_size gives");
    expand = false;
  }
  if (expand) {
    unsigned char *ws = static_cast<unsigned char *>(p->workspace);
    AttnArgs e;
    expanded_request(a, ws, &e);
    llmx_kv4_rows r{};
    r.batch = a.B;
    r.max_rows = a.Skv;
    r.k = ws;
    r.v = ws + rows;
    for (int i = 0; i < 3; ++i) {
      r.k_stride[i] = e.ks[i];
      r.v_stride[i] = e.vs[i];
    }
    r.lens = a.kv_lens;
    // The prefill reads whole blocks of 128 keys: what a block holds behind a
    // sequence is multiplied by 0 and so has to be finite.
    cudaError_t err = launch_kv4_load(k, r, a.dtype, 128, st);
    e.expanded = 1;
    if (err == cudaSuccess) err = launch_sm100(e, ws + 2 * rows, kSm100WorkspaceBytes, st);
    if (err != cudaSuccess)
      return record_error(LLMX_ERR_CUDA, (std::string("launch failed: ") + cudaGetErrorString(err)).c_str());
    return LLMX_OK;
  }
  if (refused != LLMX_OK) return refused;
  const Plan plan = plan_kv4(a);
  const bool split = plan.shared && p->workspace != nullptr && p->workspace_bytes >= plan.ws_bytes;
  const cudaError_t e = a.dtype == LLMX_FP16 ? launch_kv4_attn<__half>(a, k, plan, split, p->workspace, st)
                                             : launch_kv4_attn<__nv_bfloat16>(a, k, plan, split, p->workspace, st);
  if (e != cudaSuccess) return record_error(LLMX_ERR_CUDA, (std::string("launch failed: ") + cudaGetErrorString(e)).c_str());
  return LLMX_OK;
}
