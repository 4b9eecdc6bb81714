// Attention over the 4-bit key/value cache (include/llmx_attn.h): decode and
// short query blocks, one pass over the tiles.
//
// Mathematics.  A cached value is n s + m with a 4-bit n and s, m of its
// (token, 64-channel group).  Neither K nor V is dequantised:
//   q . K_j  = sum_h s_jh (q_h . n_jh) + m_jh sum(q_h)
//   sum_j p_j V_j = sum_j (p_j s_jh) (n_jh - 8) + sum_j p_j (m_jh + 8 s_jh)
// so the matrix products run on the integers themselves, which fp16 holds
// exactly, and the affine part is a few fp32 operations per token and group.
//   * K: a nibble masked in place is the fp16 subnormal n 2^-24 (bits 0-3) or
//     16 n 2^-24 (bits 4-7; q carries the 1/16), one AND per two values.
//     q is scaled by a power of two per row to fit fp16: 11 bits of it are
//     kept, all that fp16 and bf16 have.
//   * V: a nibble OR-ed into 1024 (0x6400) and 1032 (or 1152 = 1024 + 128 for
//     bits 4-7) subtracted is n - 8 (16 (n - 8)), two operations per two
//     values.  Centred, because the tensor core's fp32 accumulation would
//     otherwise carry a mean of 7.5 through the whole sequence that cancels
//     only at the end.
//   * p s is rounded to fp16 (2^-12 relative), after a scale by a power of two
//     that brings the largest s seen so far to [2^7, 2^8).  Scores, p, the
//     softmax sums and the affine part stay fp32.
//
// Shape.  S^T = K q^T as mma m16n8k16 with 16 tokens as rows and 8 (head,
// query row) pairs of one kv head as columns; O^T += V^T P^T with channels as
// rows.  The cache's tile layout is the order of these fragments, so K and V
// go from 16-byte global loads to registers to the tensor core, without
// shared memory; P^T changes from the accumulator's layout to the operand's
// with one 8x8 transpose (movmatrix) per 8 tokens and group.  mma.sync and not
// tcgen05: the operands are made in registers, 8 columns are all there are in
// a decode, and the pass is bound by the cache's bytes, not by the products.
//
// A CTA takes a range of tokens of one (sequence, kv head, block of 8 * NT
// pairs); its warps take every fourth tile and are merged at the end, and the
// ranges (splits) by a second kernel as in attn_decode.cu.
#include <algorithm>
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
// The largest weight times the largest step stays in [2^7, 2^8) (times 2^6
// under a lazy maximum): fp16 then keeps 11 bits of weights down to 2^-21 of
// the largest.  Steps count from 2^-40 on (smaller ones lose bits from 2^-61
// on), which keeps the sums of scaled weights inside fp32.
constexpr int kStepExp = 7;
constexpr int kMinStepExp = -40;
constexpr int kMaxStepExp = 125;
constexpr uint64_t kWaitNs = 1000000000ull;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// (n - 8) of the nibbles in bits 0-3 of both halves; 16 (n - 8) of bits 4-7.
__device__ __forceinline__ uint32_t centred_lo(uint32_t z) {
  const uint32_t u = (z & 0x000f000fu) | 0x64006400u, c = 0x64086408u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t centred_hi(uint32_t z) {
  const uint32_t u = (z & 0x00f000f0u) | 0x64006400u, c = 0x64806480u;
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

struct SplitPlan {
  int rows;       // (head, query row) pairs of one kv head
  int nt;         // columns of 8 pairs a CTA takes
  int row_blocks;
  int chunk;      // tokens per split, a multiple of 64
  int n_splits;
  size_t ws_bytes;
};

// Tokens that row i sees: [lo, hi).
__device__ __forceinline__ void row_range(const AttnArgs &a, int i, int ql, int kl, int &lo, int &hi) {
  const int diag = i + kl - ql;
  hi = a.causal ? max(0, min(kl, diag + 1)) : kl;
  lo = a.window >= 0 ? max(0, diag - a.window) : 0;
}

// First token of split 0 of a sequence: the first one that its row 0 sees,
// on a 16-token tile.  Later rows see none before it.
__device__ __forceinline__ int first_token(const AttnArgs &a, int ql, int kl) {
  int lo, hi;
  row_range(a, 0, ql, kl, lo, hi);
  return lo & ~15;
}

__device__ __forceinline__ uint32_t word_of(const uint4 &u, int i) {
  return i == 0 ? u.x : (i == 1 ? u.y : (i == 2 ? u.z : u.w));
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}

// One contiguous tile, global -> this CTA's shared memory, counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
               : "memory");
}

// Sizes of one variant: 8 * NT pairs of head_dim D.
template <int D, int NT>
struct Shape {
  static constexpr int G = D / kKv4Group;
  static constexpr int R = 8 * NT;
  static constexpr int LDO = D + 4;  // padded row of the merge buffer
  static constexpr int kTile = 18 * D;
  static constexpr int kStages = D == 64 ? 6 : (D == 128 ? 4 : 3);
  // q fragments and row factors stay in registers where they are few.
  static constexpr bool kQRegs = NT * G <= 2;
  static constexpr int kMinCtas = NT * G <= 2 ? 4 : (NT * G <= 4 ? 3 : 2);
  static constexpr size_t kRing = (size_t)kWarps * kStages * kTile;
  static constexpr size_t kMerge = (size_t)kWarps * R * LDO * sizeof(float);
  static constexpr size_t kRingOrMerge = kRing > kMerge ? kRing : kMerge;
  static constexpr size_t kQFrag = (size_t)NT * G * 2 * 32 * 16;
  static constexpr size_t kSmem = kRingOrMerge + kQFrag;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, Shape<D, NT>::kMinCtas)
    kv4_attn_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ Kv4Args c, int chunk, int n_splits,
                    int row_blocks, float *part_o, float *part_lse) {
  using Sh = Shape<D, NT>;
  constexpr int G = Sh::G, R = Sh::R, LDO = Sh::LDO, kStages = Sh::kStages;
  extern __shared__ __align__(128) unsigned char smem[];
  float *sm_o = reinterpret_cast<float *>(smem);                              // [kWarps][R][LDO], after the loop
  __half *sm_q = reinterpret_cast<__half *>(smem + Sh::kRingOrMerge);         // fragments of q
  __shared__ float sm_f[R], sm_qs[G][R], sm_slope[R];
  __shared__ int sm_lo[R], sm_hi[R];
  __shared__ float sm_m[kWarps][R], sm_l[kWarps][R];
  __shared__ uint64_t sm_full[kWarps][kStages];

  // The combine kernel may be set up while this one runs.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int split = blockIdx.x;
  const int kvh = blockIdx.y / row_blocks;
  const int r0 = blockIdx.y % row_blocks * R;
  const int b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int g = lane >> 2, t = lane & 3;
  const int rows = a.group * a.Sq;  // pair r: query row r / group, head r % group of the kv head

  const int ql = clamp_len(a.q_lens, b, a.Sq);
  const int kl = clamp_len(a.kv_lens, b, a.Skv);

  // Tokens of this split that some row of the block sees, and the ones
  // [lo_in, hi_in) that all of its rows see (the rows' ranges move one way:
  // the last row's begin, the first row's end).
  int t_lo = 0, t_hi = 0, lo_in = 0, hi_in = 0;
  {
    const int i0 = r0 / a.group, i1 = min(min(r0 + R, rows) - 1, ql * a.group - 1) / a.group;
    if (i0 < ql && kl > 0) {
      int lo0, hi1;
      row_range(a, i0, ql, kl, lo0, hi_in);
      row_range(a, i1, ql, kl, lo_in, hi1);
      const int s0 = first_token(a, ql, kl) + split * chunk;
      t_lo = max(lo0, s0);
      t_hi = min(hi1, s0 + chunk);
    }
  }

  if (t_lo >= t_hi && n_splits > 1) {
    // Nothing here; a row whose range of splits holds this one skips it.
    for (int r = tid; r < R && r0 + r < rows; r += kThreads) {
      const int i = (r0 + r) / a.group, h = kvh * a.group + (r0 + r) % a.group;
      part_lse[(((long long)split * a.B + b) * a.Sq + i) * a.H + h] = -CUDART_INF_F;
    }
    return;
  }

  // Weights are kept as 2^(S - ref) with one reference per row: the running
  // maximum less a power of two that brings the largest step times the
  // largest weight into fp16's upper range (kRoom below).
  float o[NT][G][4][4];
  float l[NT][2], aff[NT][2][G], ref[NT][2];
  int step_exp = kMinStepExp;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][h][i][x] = 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      l[n][q] = 0.f;
      ref[n][q] = -CUDART_INF_F;
#pragma unroll
      for (int h = 0; h < G; ++h) aff[n][q][h] = 0.f;
    }
  }

  if (t_lo < t_hi) {
    const int tile0 = t_lo >> 4, tile1 = (t_hi + 15) >> 4;
    const int tpp = c.page_size >> 4;
    const unsigned char *base = c.data + kvh * c.head_stride;
    const int mine = tile1 - tile0 > warp ? (tile1 - tile0 - warp + kWarps - 1) / kWarps : 0;  // tiles of this warp
    const uint32_t ring = sm100::smem_u32(smem) + warp * kStages * Sh::kTile;

    // Lane i of the warp keeps where its tile (32 n + i) lies, and issues
    // its copy.  Bit i of `bad`: that tile's page is outside the cache.
    long long where = -1;
    uint32_t bad_now = 0, bad_issue = 0;
    auto locate = [&](int first) {
      const int idx = first + lane;
      where = -1;
      if (idx < mine) {
        const int tile = tile0 + warp + idx * kWarps;
        const int page = tile / tpp;
        where = kv4_page_offset(c, b, page);
        if (where >= 0) where += (long long)(tile - page * tpp) * Sh::kTile;
      }
      bad_issue = __ballot_sync(0xffffffffu, idx < mine && where < 0);
    };
    auto issue = [&](int i, int stage) {
      if (lane == i % 32 && where >= 0) {
        sm100::mbar_arrive_expect_tx(&sm_full[warp][stage], Sh::kTile);
        bulk_load(ring + stage * Sh::kTile, base + where, Sh::kTile, &sm_full[warp][stage]);
      }
    };
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kStages; ++i) sm100::mbar_init(&sm_full[warp][i], 1);
      sm100::fence_mbar_init();
    }
    locate(0);
    bad_now = bad_issue;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (i < mine) issue(i, i);

    // Query rows to fp16, scaled by a power of two, in the order of the
    // operand fragments, with the factor that undoes the scale and the sums
    // of their groups.  Lane l holds D / 32 consecutive channels.
    constexpr int E = D / 32;
    for (int r = warp; r < R; r += kWarps) {
      const bool live = r0 + r < rows && (r0 + r) / a.group < ql;
      float x[E];
      float top = 0.f, sum = 0.f;
      int lo = 0, hi = 0;
      float slope = 0.f;
      if (live) {
        const int i = (r0 + r) / a.group, h = kvh * a.group + (r0 + r) % a.group;
        const T *p = static_cast<const T *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = Elem<T>::to_f(p[e]);
        row_range(a, i, ql, kl, lo, hi);
        if (a.alibi != nullptr) slope = a.alibi[h] * kLog2e;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!live) x[e] = 0.f;
        top = fmaxf(top, fabsf(x[e]));
        sum += x[e];
      }
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
#pragma unroll
      for (int off = 1; off < 32 / G; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      // top in [2^ex, 2^(ex + 1)) goes to [2^14, 2^15).
      const int ex = max(-112, (int)(__float_as_uint(top) >> 23) - 127);
      const float up = pow2i(min(126, 14 - ex));
      const float scale = a.softcap > 0.f ? a.sm_scale / a.softcap : a.sm_scale * kLog2e;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane * E + e, p = d & 7;
        // Channels 0..7 of a word go to halves 0, 2, 4, 6, 1, 3, 5, 7 of the
        // fragment; the odd ones meet nibbles that are 16 times too large.
        const int at = ((((r >> 3) * G + (d >> 6)) * 2 + ((d >> 3) & 1)) * 32 + 4 * (r & 7) + ((d >> 4) & 3)) * 8 +
                       (p & 3) * 2 + (p >> 2);
        sm_q[at] = __float2half_rn(x[e] * (p & 1 ? up * 0.0625f : up));
      }
      if (lane == 0) {
        // 2^24 for the subnormals, 2^(ex - 14) for the scaling.
        sm_f[r] = scale * 0x1p24f * pow2i(max(-126, ex - 14));
        sm_lo[r] = lo;
        sm_hi[r] = hi;
        sm_slope[r] = slope;
      }
      if (lane % (32 / G) == 0) sm_qs[lane / (32 / G)][r] = sum * scale;
    }
    __syncthreads();

    uint4 qf[Sh::kQRegs ? NT * G * 2 : 1];
    float2 fac_r[Sh::kQRegs ? NT : 1], qs_r[Sh::kQRegs ? NT * G : 1];
    const uint32_t q_at = sm100::smem_u32(sm_q) + lane * 16;
    if constexpr (Sh::kQRegs) {
#pragma unroll
      for (int i = 0; i < NT * G * 2; ++i) qf[i] = lds16(q_at + i * 512);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        fac_r[n] = *reinterpret_cast<const float2 *>(&sm_f[n * 8 + 2 * t]);
#pragma unroll
        for (int h = 0; h < G; ++h) qs_r[n * G + h] = *reinterpret_cast<const float2 *>(&sm_qs[h][n * 8 + 2 * t]);
      }
    }

    // One tile at shared address `at`, tokens tok0 ..  PART: some row does
    // not see all of its tokens.
    auto compute = [&](uint32_t at, int tok0, auto part_tag) {
      constexpr bool PART = decltype(part_tag)::value;
      uint32_t par[2][2 * G];  // parameters of tokens g, g + 8: [K groups, V groups]
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t q = at + G * 1024 + (g + 8 * r) * (8 * G);
        if constexpr (G == 1) {
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(par[r][0]), "=r"(par[r][1]) : "r"(q));
        } else {
#pragma unroll
          for (int i = 0; i < G / 2; ++i) {
            const uint4 u = lds16(q + i * 16);
            par[r][4 * i] = u.x;
            par[r][4 * i + 1] = u.y;
            par[r][4 * i + 2] = u.z;
            par[r][4 * i + 3] = u.w;
          }
        }
      }
      // Scores, less the rows' references.
      float s[NT][4];
      {
        float acc[NT][G][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < G; ++h)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[n][h][x] = 0.f;
        uint4 kw[G];
#pragma unroll
        for (int i = 0; i < G; ++i) kw[i] = lds16(at + i * 512 + lane * 16);
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int x0 = h * 2 + w, x1 = (G + h) * 2 + w;
            uint32_t k0 = word_of(kw[x0 / 4], x0 % 4), k1 = word_of(kw[x1 / 4], x1 % 4);
            uint32_t af[2][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              af[half][0] = k0 & 0x000f000fu;
              af[half][1] = k1 & 0x000f000fu;
              af[half][2] = k0 & 0x00f000f0u;
              af[half][3] = k1 & 0x00f000f0u;
              k0 >>= 8;
              k1 >>= 8;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint4 qw;
              if constexpr (Sh::kQRegs) qw = qf[(n * G + h) * 2 + w];
              else qw = lds16(q_at + ((n * G + h) * 2 + w) * 512);
              mma16816(acc[n][h], af[0][0], af[0][1], af[0][2], af[0][3], qw.x, qw.y);
              mma16816(acc[n][h], af[1][0], af[1][1], af[1][2], af[1][3], qw.z, qw.w);
            }
          }
        float2 kp[2][G];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < G; ++h) kp[r][h] = kv4_unpack_param<T>(par[r][h]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float2 fac, qs[G];
          if constexpr (Sh::kQRegs) {
            fac = fac_r[n];
#pragma unroll
            for (int h = 0; h < G; ++h) qs[h] = qs_r[n * G + h];
          } else {
            fac = *reinterpret_cast<const float2 *>(&sm_f[n * 8 + 2 * t]);
#pragma unroll
            for (int h = 0; h < G; ++h) qs[h] = *reinterpret_cast<const float2 *>(&sm_qs[h][n * 8 + 2 * t]);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              // With a soft-cap the reference comes off behind the tanh.
              float off = a.softcap > 0.f || ref[n][q] == -CUDART_INF_F ? 0.f : -ref[n][q];
              float dot = kp[r][0].x * acc[n][0][2 * r + q];
              off = fmaf(kp[r][0].y, q ? qs[0].y : qs[0].x, off);
#pragma unroll
              for (int h = 1; h < G; ++h) {
                dot = fmaf(kp[r][h].x, acc[n][h][2 * r + q], dot);
                off = fmaf(kp[r][h].y, q ? qs[h].y : qs[h].x, off);
              }
              s[n][2 * r + q] = fmaf(dot, q ? fac.y : fac.x, off);
            }
        }
      }
      if (a.softcap > 0.f) {
        const float cap2 = a.softcap * kLog2e;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            s[n][x] = fmaf(tanhf(s[n][x]), cap2, ref[n][x & 1] == -CUDART_INF_F ? 0.f : -ref[n][x & 1]);
      }
      if (a.alibi != nullptr) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float2 sl = *reinterpret_cast<const float2 *>(&sm_slope[n * 8 + 2 * t]);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            s[n][x] = fmaf(x & 1 ? sl.y : sl.x, (float)(tok0 + g + 8 * (x >> 1)), s[n][x]);
        }
      }
      uint32_t vis = 0xffffffffu;
      if constexpr (PART) {
        vis = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int2 lo = *reinterpret_cast<const int2 *>(&sm_lo[n * 8 + 2 * t]);
          const int2 hi = *reinterpret_cast<const int2 *>(&sm_hi[n * 8 + 2 * t]);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = tok0 + g + 8 * (x >> 1);
            if (j >= max(x & 1 ? lo.y : lo.x, t_lo) && j < min(x & 1 ? hi.y : hi.x, t_hi)) vis |= 1u << (n * 4 + x);
            else s[n][x] = -CUDART_INF_F;
          }
        }
      }
      // V's steps and centres; a token that no row sees may hold anything.
      float sv[2][G], cv[2][G];
      float smax = 0.f;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int h = 0; h < G; ++h) {
          float2 p = kv4_unpack_param<T>(par[r][G + h]);
          if (PART && (vis & (0x33333333u << (2 * r))) == 0) p = make_float2(0.f, 0.f);
          sv[r][h] = p.x;
          cv[r][h] = fmaf(8.f, p.x, p.y);
          smax = fmaxf(smax, p.x);
        }
      }
      // The references move, with everything accumulated, when a score
      // passes its row's maximum by kLazyMax or a larger step turns up.
      const float limit = kLazyMax + (float)(kStepExp - step_exp);
      float most = s[0][0];
      bool first = false;  // a row without a reference so far
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) most = fmaxf(most, s[n][x]);
        first |= ref[n][0] == -CUDART_INF_F || ref[n][1] == -CUDART_INF_F;
      }
      if (__any_sync(0xffffffffu, first || most > limit || smax >= pow2i(step_exp + 1))) {
        uint32_t bits = 0;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < G; ++h) {
            const uint32_t u = __float_as_uint(sv[r][h]);
            bits = max(bits, u < 0x7f800000u ? u : 0u);
          }
        const int new_exp = max(step_exp, min(kMaxStepExp, (int)(__reduce_max_sync(0xffffffffu, bits) >> 23) - 127));
        const float old_room = (float)(kStepExp - step_exp), new_room = (float)(kStepExp - new_exp);
        step_exp = new_exp;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const bool none = ref[n][q] == -CUDART_INF_F;
            const float shift = none ? 0.f : ref[n][q];
            float v = fmaxf(s[n][q], s[n][2 + q]) + shift;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
            const float m = none ? v : fmaxf(ref[n][q] + old_room, v);
            const float now = m == -CUDART_INF_F ? m : m - new_room;
            const float al = none ? 1.f : exp2_fast(ref[n][q] - now);
            const float back = now == -CUDART_INF_F ? 0.f : shift - now;
            ref[n][q] = now;
            s[n][q] += back;
            s[n][2 + q] += back;
            l[n][q] *= al;
#pragma unroll
            for (int h = 0; h < G; ++h) {
              aff[n][q][h] *= al;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[n][h][i][q] *= al;
                o[n][h][i][2 + q] *= al;
              }
            }
          }
      }
      // Weights.
      uint32_t pf[NT][G][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float p[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          p[x] = exp2_fast(s[n][x]);
          l[n][x & 1] += p[x];
        }
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float w[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              w[q] = p[2 * r + q] * sv[r][h];
              float f = p[2 * r + q] * cv[r][h];
              if constexpr (PART) {
                const bool ok = vis >> (n * 4 + 2 * r + q) & 1u;
                w[q] = ok ? w[q] : 0.f;
                f = ok ? f : 0.f;
                aff[n][q][h] += f;
              } else {
                aff[n][q][h] = fmaf(p[2 * r + q], cv[r][h], aff[n][q][h]);
              }
            }
            pf[n][h][r] = transpose8x8(pack_half2(w[0], w[1]));
          }
      }
      // O^T += V^T P^T.
      uint4 vw[G];
#pragma unroll
      for (int i = 0; i < G; ++i) vw[i] = lds16(at + G * 512 + i * 512 + lane * 16);
#pragma unroll
      for (int h = 0; h < G; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) w[sl] = word_of(vw[(sl * G + h) / 4], (sl * G + h) % 4);
#pragma unroll
        for (int part16 = 0; part16 < 2; ++part16) {
          uint32_t z0 = __byte_perm(w[0], w[1], part16 ? 0x7632 : 0x5410);
          uint32_t z1 = __byte_perm(w[2], w[3], part16 ? 0x7632 : 0x5410);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t a0 = centred_lo(z0), a1 = centred_hi(z0), a2 = centred_lo(z1), a3 = centred_hi(z1);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(o[n][h][2 * part16 + half], a0, a1, a2, a3, pf[n][h][0], pf[n][h][1]);
            z0 >>= 8;
            z1 >>= 8;
          }
        }
      }
    };

    const int full_lo = max(lo_in, t_lo), full_hi = min(hi_in, t_hi);
    int stage = 0;
    uint32_t parity = 0;  // bit s: parity of stage s's next phase
    for (int i = 0; i < mine; ++i) {
      if (i % 32 == 0) bad_now = bad_issue;
      if (!(bad_now >> (i % 32) & 1u)) {
        const bool ok = sm100::mbar_wait(&sm_full[warp][stage], parity >> stage & 1u, kWaitNs);
        if (!__all_sync(0xffffffffu, ok)) {
          // Never seen to happen: the copy did not arrive in a second.  The
          // copies in flight get as long again before the CTA goes on.
          raise_error(a.err, kDevErrTimeout);
          for (int k = 0; k < kStages && i + k < mine; ++k) {
            const int st = (stage + k) % kStages;
            if (!(bad_now >> ((i + k) % 32) & 1u)) sm100::mbar_wait(&sm_full[warp][st], parity >> st & 1u, kWaitNs);
          }
          break;
        }
        parity ^= 1u << stage;
        const int tok0 = (tile0 + warp + i * kWarps) << 4;
        if (tok0 >= full_lo && tok0 + 16 <= full_hi) compute(ring + stage * Sh::kTile, tok0, std::false_type{});
        else compute(ring + stage * Sh::kTile, tok0, std::true_type{});
      }
      const int next = i + kStages;
      if (next % 32 == 0) locate(next);
      __syncwarp();  // the warp has read the stage
      if (next < mine) issue(next, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  }

  // Sums over the tokens of the warp (lanes with the same t hold the same rows).
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[n][q] += __shfl_xor_sync(0xffffffffu, l[n][q], off);
#pragma unroll
        for (int h = 0; h < G; ++h) aff[n][q][h] += __shfl_xor_sync(0xffffffffu, aff[n][q][h], off);
      }
    }
  __syncthreads();  // every warp is through with its ring
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = n * 8 + 2 * t + q;
      if (g == 0) {
        sm_m[warp][r] = ref[n][q];
        sm_l[warp][r] = l[n][q];
      }
      float *dst = sm_o + (warp * R + r) * LDO;
#pragma unroll
      for (int h = 0; h < G; ++h) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = o[n][h][i][q] + aff[n][q][h];
          v[2 * i + 1] = fmaf(o[n][h][i][2 + q], 0.0625f, aff[n][q][h]);
        }
        float4 *d4 = reinterpret_cast<float4 *>(dst + 64 * h + 8 * g);
        d4[0] = make_float4(v[0], v[1], v[2], v[3]);
        d4[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  __syncthreads();

  // Merge the warps.
  for (int e = tid; e < R * D; e += kThreads) {
    const int r = e / D, d = e % D;
    if (r0 + r >= rows) break;
    float top = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w][r]);
    float lsum = 0.f, ov = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float wt = sm_m[w][r] == -CUDART_INF_F ? 0.f : exp2f(sm_m[w][r] - top);
      // A warp that saw no finite score adds nothing, unless its sum is a NaN.
      lsum += wt == 0.f ? (sm_l[w][r] == sm_l[w][r] ? 0.f : sm_l[w][r]) : sm_l[w][r] * wt;
      ov += wt == 0.f ? 0.f : sm_o[(w * R + r) * LDO + d] * wt;
    }
    const bool none = lsum == 0.f;
    const float inv = none ? 0.f : 1.f / lsum;
    const float lse = none ? -CUDART_INF_F : (top == -CUDART_INF_F ? lsum : (top + log2f(lsum)) * kLn2);
    const int i = (r0 + r) / a.group, h = kvh * a.group + (r0 + r) % a.group;
    if (n_splits == 1) {
      static_cast<T *>(a.o)[b * a.os[0] + i * a.os[1] + h * a.os[2] + d] = Elem<T>::from_f(ov * inv);
      if (a.lse != nullptr && d == 0) a.lse[((long long)b * a.H + h) * a.Sq + i] = lse;
    } else {
      const long long row = (((long long)split * a.B + b) * a.Sq + i) * a.H + h;
      part_o[row * D + d] = ov * inv;
      if (d == 0) part_lse[row] = lse;
    }
  }
}

// O = sum_s exp(lse_s - lse) O_s over the splits; a warp per output row.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_combine_kernel(AttnArgs a, int chunk, int n_splits, const float *part_o,
                                                          const float *part_lse) {
  constexpr int E = D / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the splits are written
  const int lane = threadIdx.x % 32;
  const long long n_rows = (long long)a.B * a.Sq * a.H;
  const long long row = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= n_rows) return;
  const int h = (int)(row % a.H), i = (int)(row / a.H % a.Sq), b = (int)(row / a.H / a.Sq);
  const int ql = clamp_len(a.q_lens, b, a.Sq), kl = clamp_len(a.kv_lens, b, a.Skv);
  int used = 0;
  if (i < ql && kl > 0) {
    int lo, hi;
    row_range(a, i, ql, kl, lo, hi);
    const int s0 = first_token(a, ql, kl);
    if (hi > lo) used = min(n_splits, (hi - s0 + chunk - 1) / chunk);
  }
  float top = -CUDART_INF_F;
  for (int s = lane; s < used; s += 32) top = fmaxf(top, part_lse[s * n_rows + row]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  float sum = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s = 0; s < used; ++s) {
    const float ls = part_lse[s * n_rows + row];
    if (ls == -CUDART_INF_F) continue;
    const float w = expf(ls - top);  // a NaN goes on into the sum
    sum += w;
    const float *p = part_o + (s * n_rows + row) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(w, p[e], o[e]);
  }
  const bool none = sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  T *op = static_cast<T *>(a.o) + b * a.os[0] + i * a.os[1] + h * a.os[2] + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = Elem<T>::from_f(o[e] * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[((long long)b * a.H + h) * a.Sq + i] = none ? -CUDART_INF_F : top + logf(sum);
}

template <int D>
constexpr int max_nt() {
  return D == 64 ? 4 : (D == 128 ? 4 : 2);
}

SplitPlan plan_kv4(const AttnArgs &a, size_t ws_available) {
  SplitPlan p;
  p.rows = a.group * a.Sq;
  const int G = a.D / kKv4Group;
  const int most = a.D == 256 ? 2 : 4;
  p.nt = p.rows <= 8 ? 1 : (p.rows <= 16 || most == 2 ? 2 : 4);
  p.row_blocks = (p.rows + 8 * p.nt - 1) / (8 * p.nt);
  const long long units = (long long)a.B * a.Hkv * p.row_blocks;
  const long long slots = (long long)a.num_sms * (p.nt * G <= 2 ? 4 : (p.nt * G <= 4 ? 3 : 2));
  // Tokens that a sequence's rows can see between them.
  long long span = a.Skv;
  if (a.window >= 0) span = std::min<long long>(span, (long long)a.window + a.Sq + 16);
  // One wave of CTAs where that leaves each 128 tokens at least; splits of
  // 1024 tokens where there is more than a wave of work anyway (sequences
  // differ in length, so equal shares cannot be dealt from here).
  long long n = std::max<long long>(1, slots / units);
  n = std::min(n, (span + 127) / 128);
  if (units > slots / 2) n = std::max(n, (span + 1023) / 1024);
  long long chunk = ((span + n - 1) / n + 63) / 64 * 64;
  p.chunk = (int)chunk;
  p.n_splits = (int)((span + chunk - 1) / chunk);
  p.ws_bytes = p.n_splits > 1 ? (size_t)p.n_splits * a.B * a.Sq * a.H * (a.D + 1) * sizeof(float) : 0;
  if (p.n_splits > 1 && ws_available < p.ws_bytes) {
    p.n_splits = 1;
    p.chunk = (int)((span + 63) / 64 * 64);
  }
  return p;
}

template <typename T, int D, int NT>
cudaError_t launch_nt(const AttnArgs &a, const Kv4Args &c, const SplitPlan &p, void *ws, cudaStream_t s) {
  constexpr size_t smem = Shape<D, NT>::kSmem;
  if (smem > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(kv4_attn_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  float *part_o = nullptr, *part_lse = nullptr;
  const long long n_rows = (long long)a.B * a.Sq * a.H;
  if (p.n_splits > 1) {
    part_o = static_cast<float *>(ws);
    part_lse = part_o + (size_t)p.n_splits * n_rows * D;
  }
  const dim3 grid(p.n_splits, a.Hkv * p.row_blocks, a.B);
  kv4_attn_kernel<T, D, NT><<<grid, kThreads, smem, s>>>(a, c, p.chunk, p.n_splits, p.row_blocks, part_o, part_lse);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.n_splits == 1) return e;
  // The combine's launch overlaps the splits; it waits for them itself.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((n_rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_combine_kernel<T, D>, a, p.chunk, p.n_splits, (const float *)part_o,
                            (const float *)part_lse);
}

template <typename T, int D>
cudaError_t launch_d(const AttnArgs &a, const Kv4Args &c, const SplitPlan &p, void *ws, cudaStream_t s) {
  if (p.nt == 1) return launch_nt<T, D, 1>(a, c, p, ws, s);
  if constexpr (max_nt<D>() >= 2) {
    if (p.nt == 2) return launch_nt<T, D, 2>(a, c, p, ws, s);
  }
  if constexpr (max_nt<D>() >= 4) {
    if (p.nt == 4) return launch_nt<T, D, 4>(a, c, p, ws, s);
  }
  return cudaErrorNotSupported;
}

template <typename T>
cudaError_t launch_kv4_attn(const AttnArgs &a, const Kv4Args &c, const SplitPlan &p, void *ws, cudaStream_t s) {
  switch (a.D) {
    case 64: return launch_d<T, 64>(a, c, p, ws, s);
    case 128: return launch_d<T, 128>(a, c, p, ws, s);
    case 256: return launch_d<T, 256>(a, c, p, ws, s);
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

// From this many (head, query row) pairs of a kv head on AUTO expands.
constexpr int kExpandRows = 256;

// Whether the request runs expanded; `s` gets the refusal of a forced form.
bool use_expanded(const AttnArgs &a, int algo, llmx_status *s) {
  AttnArgs e;
  // Any 256-byte aligned address stands for the workspace here.
  const bool can = expanded_request(a, reinterpret_cast<unsigned char *>(uintptr_t(256)), &e);
  *s = LLMX_OK;
  if (algo == LLMX_ALGO_TCGEN05 && !can)
    *s = record_error(LLMX_ERR_UNSUPPORTED,
                      "kv4: TCGEN05 needs max_q_len > 1, sm_scale > 0 and 16-byte aligned rows of q and o");
  return can && (algo == LLMX_ALGO_TCGEN05 || (algo == LLMX_ALGO_AUTO && (long long)a.group * a.Sq >= kExpandRows));
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
  if ((long long)a->group * a->Sq > 0x3fffffffLL || (long long)a->Hkv * ((a->group * (long long)a->Sq + 7) / 8) > 65535)
    return bad("kv4: too many query rows for one call");
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
  *bytes = expand ? 2 * expanded_rows_bytes(a) + kSm100WorkspaceBytes : plan_kv4(a, SIZE_MAX).ws_bytes;
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
  if (use_expanded(a, p->algo, &refused)) {
    const size_t rows = expanded_rows_bytes(a);
    unsigned char *ws = static_cast<unsigned char *>(p->workspace);
    if (ws == nullptr || p->workspace_bytes < 2 * rows + kSm100WorkspaceBytes)
      return record_error(LLMX_ERR_WORKSPACE_TOO_SMALL,
                          "kv4: the expanded form needs the workspace that llmx_kv4_attn_workspace_size gives");
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
    if (err == cudaSuccess) err = launch_sm100(e, ws + 2 * rows, kSm100WorkspaceBytes, st);
    if (err != cudaSuccess)
      return record_error(LLMX_ERR_CUDA, (std::string("launch failed: ") + cudaGetErrorString(err)).c_str());
    return LLMX_OK;
  }
  if (refused != LLMX_OK) return refused;
  const SplitPlan plan = plan_kv4(a, p->workspace != nullptr ? p->workspace_bytes : 0);
  const cudaError_t e = a.dtype == LLMX_FP16 ? launch_kv4_attn<__half>(a, k, plan, p->workspace, st)
                                             : launch_kv4_attn<__nv_bfloat16>(a, k, plan, p->workspace, st);
  if (e != cudaSuccess) return record_error(LLMX_ERR_CUDA, (std::string("launch failed: ") + cudaGetErrorString(e)).c_str());
  return LLMX_OK;
}
