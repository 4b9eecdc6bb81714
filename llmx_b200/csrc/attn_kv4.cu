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

namespace llmx_b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum of a row moves only when a score passes it by this
// much (log2): p reaches 2^6 at most, and p s at most 2^14 in fp16.
constexpr float kLazyMax = 6.f;
constexpr int kStepExp = 7;      // the largest s is scaled to [2^7, 2^8)
constexpr int kMinStepExp = -100;

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

// One lane's share of a tile of 16 tokens.
template <int G>
struct Tile {
  uint4 k[G], v[G];
  uint32_t par[2][2 * G];  // [token g, g + 8][K groups, V groups]
};

template <int G>
__device__ __forceinline__ void load_tile(Tile<G> &t, const unsigned char *p, int lane) {
#pragma unroll
  for (int i = 0; i < G; ++i) t.k[i] = ld_stream16(p + i * 512 + lane * 16);
#pragma unroll
  for (int i = 0; i < G; ++i) t.v[i] = ld_stream16(p + G * 512 + i * 512 + lane * 16);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const unsigned char *q = p + G * 1024 + ((lane >> 2) + 8 * r) * (8 * G);
    if constexpr (G == 1) {
      const uint2 u = *reinterpret_cast<const uint2 *>(q);
      t.par[r][0] = u.x;
      t.par[r][1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < G / 2; ++i) {
        const uint4 u = ld_stream16(q + i * 16);
        t.par[r][4 * i] = u.x;
        t.par[r][4 * i + 1] = u.y;
        t.par[r][4 * i + 2] = u.z;
        t.par[r][4 * i + 3] = u.w;
      }
    }
  }
}

__device__ __forceinline__ uint32_t word_of(const uint4 &u, int i) {
  return i == 0 ? u.x : (i == 1 ? u.y : (i == 2 ? u.z : u.w));
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_attn_kernel(AttnArgs a, Kv4Args c, int chunk, int n_splits, int row_blocks,
                                                            float *part_o, float *part_lse) {
  constexpr int G = D / kKv4Group;
  constexpr int R = 8 * NT;
  constexpr int LDO = D + 4;
  extern __shared__ __align__(16) unsigned char smem[];
  __half *sm_q = reinterpret_cast<__half *>(smem);            // [R][D]
  float *sm_o = reinterpret_cast<float *>(smem);              // [kWarps][R][LDO], after the loop
  __shared__ float sm_f[R], sm_qs[R][G];
  __shared__ float sm_m[kWarps][R], sm_l[kWarps][R];

  const int split = blockIdx.x;
  const int kvh = blockIdx.y / row_blocks;
  const int r0 = blockIdx.y % row_blocks * R;
  const int b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int g = lane >> 2, t = lane & 3;
  const int rows = a.group * a.Sq;  // pair r: query row r / group, head r % group of the kv head

  const int ql = clamp_len(a.q_lens, b, a.Sq);
  const int kl = clamp_len(a.kv_lens, b, a.Skv);

  // Tokens of this split that some row of the block sees.
  int t_lo = 0, t_hi = 0;
  {
    const int i0 = r0 / a.group, i1 = min(min(r0 + R, rows) - 1, ql * a.group - 1) / a.group;
    if (i0 < ql && kl > 0) {
      int lo0, hi0, lo1, hi1;
      row_range(a, i0, ql, kl, lo0, hi0);
      row_range(a, i1, ql, kl, lo1, hi1);
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

  float o[NT][G][4][4];
  float l[NT][2], aff[NT][2][G], mx[NT][2];
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
      mx[n][q] = -CUDART_INF_F;
#pragma unroll
      for (int h = 0; h < G; ++h) aff[n][q][h] = 0.f;
    }
  }

  if (t_lo < t_hi) {
    // Query rows to fp16, scaled by a power of two, with the factor that
    // undoes it and the sums of their groups.  Lane l holds D / 32
    // consecutive channels.
    constexpr int E = D / 32;
    for (int r = warp; r < R; r += kWarps) {
      const bool live = r0 + r < rows && (r0 + r) / a.group < ql;
      float x[E];
      float top = 0.f, sum = 0.f;
      if (live) {
        const int i = (r0 + r) / a.group, h = kvh * a.group + (r0 + r) % a.group;
        const T *p = static_cast<const T *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = Elem<T>::to_f(p[e]);
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
      for (int e = 0; e < E; ++e) sm_q[r * D + lane * E + e] = __float2half_rn(x[e] * up);
      // 2^24 for the subnormals, 2^(ex - 14) for the scaling.
      if (lane == 0) sm_f[r] = scale * 0x1p24f * pow2i(max(-126, ex - 14));
      if (lane % (32 / G) == 0) sm_qs[r][lane / (32 / G)] = sum * scale;
    }
    __syncthreads();

    // Operand fragments of q: 4 registers per 16 channels and column block.
    uint32_t qf[NT][G][2][4];
    float fac[NT][2], qs[NT][2][G], slope[NT][2];
    int lo[NT][2], hi[NT][2];
    int lo_in = 0, hi_in = 0x7fffffff;  // tokens in [lo_in, hi_in) are seen by every row
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const __half *qr = sm_q + (n * 8 + g) * D;
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint4 u = *reinterpret_cast<const uint4 *>(qr + 64 * h + 16 * t + 8 * w);
          const uint32_t sixteenth = 0x2c002c00u;  // 2^-4, twice
          const __half2 s16 = *reinterpret_cast<const __half2 *>(&sixteenth);
          qf[n][h][w][0] = __byte_perm(u.x, u.z, 0x5410);  // channels 0, 4
          uint32_t x1 = __byte_perm(u.x, u.z, 0x7632);     // channels 1, 5
          qf[n][h][w][2] = __byte_perm(u.y, u.w, 0x5410);  // channels 2, 6
          uint32_t x3 = __byte_perm(u.y, u.w, 0x7632);     // channels 3, 7
          const __half2 y1 = __hmul2(*reinterpret_cast<const __half2 *>(&x1), s16);
          const __half2 y3 = __hmul2(*reinterpret_cast<const __half2 *>(&x3), s16);
          qf[n][h][w][1] = *reinterpret_cast<const uint32_t *>(&y1);
          qf[n][h][w][3] = *reinterpret_cast<const uint32_t *>(&y3);
        }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = n * 8 + 2 * t + q;
        fac[n][q] = sm_f[r];
#pragma unroll
        for (int h = 0; h < G; ++h) qs[n][q][h] = sm_qs[r][h];
        const bool live = r0 + r < rows && (r0 + r) / a.group < ql;
        lo[n][q] = hi[n][q] = 0;
        if (live) row_range(a, (r0 + r) / a.group, ql, kl, lo[n][q], hi[n][q]);
        slope[n][q] = a.alibi != nullptr && live ? a.alibi[kvh * a.group + (r0 + r) % a.group] * kLog2e : 0.f;
      }
    }
    {
      // Rows of the block in order: the last one's lo and the first one's hi.
      const int i0 = r0 / a.group, i1 = min(min(r0 + R, rows) - 1, ql * a.group - 1) / a.group;
      int x;
      row_range(a, i1, ql, kl, lo_in, x);
      row_range(a, i0, ql, kl, x, hi_in);
    }

    const int tile0 = t_lo >> 4, tile1 = (t_hi + 15) >> 4;
    const int tpp = c.page_size >> 4;
    const unsigned char *base = c.data + kvh * c.head_stride;
    const int mine = tile1 - tile0 > warp ? (tile1 - tile0 - warp + kWarps - 1) / kWarps : 0;  // tiles of this warp

    // Lane i of the warp keeps where its tile (32 n + i) lies.
    auto locate = [&](int first) -> long long {
      const int idx = first + lane;
      if (idx >= mine) return -1;
      const int tile = tile0 + warp + idx * kWarps;
      const int page = tile / tpp;
      const long long off = kv4_page_offset(c, b, page);
      return off < 0 ? -1 : off + (long long)(tile - page * tpp) * kv4_tile_bytes(D);
    };

    auto compute = [&](const Tile<G> &tl, int tok0) {
      // Scores.
      float s[NT][4];
      {
        float acc[NT][G][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < G; ++h)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[n][h][x] = 0.f;
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int x0 = h * 2 + w, x1 = (G + h) * 2 + w;
            uint32_t k0 = word_of(tl.k[x0 / 4], x0 % 4), k1 = word_of(tl.k[x1 / 4], x1 % 4);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma16816(acc[n][h], k0 & 0x000f000fu, k1 & 0x000f000fu, k0 & 0x00f000f0u, k1 & 0x00f000f0u,
                         qf[n][h][w][2 * half], qf[n][h][w][2 * half + 1]);
              k0 >>= 8;
              k1 >>= 8;
            }
          }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float2 p[G];
#pragma unroll
          for (int h = 0; h < G; ++h) p[h] = kv4_unpack_param<T>(tl.par[r][h]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float dot = 0.f, off = 0.f;
#pragma unroll
              for (int h = 0; h < G; ++h) {
                dot = fmaf(p[h].x, acc[n][h][2 * r + q], dot);
                off = fmaf(p[h].y, qs[n][q][h], off);
              }
              s[n][2 * r + q] = fmaf(dot, fac[n][q], off);
            }
        }
      }
      if (a.softcap > 0.f) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][x] = tanhf(s[n][x]) * (a.softcap * kLog2e);
      }
      if (a.alibi != nullptr) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][x] = fmaf(slope[n][x & 1], (float)(tok0 + g + 8 * (x >> 1)), s[n][x]);
      }
      // Masks, only where the tile is not seen whole by every row.
      const bool part = tok0 < max(lo_in, t_lo) || tok0 + 16 > min(hi_in, t_hi);
      uint32_t vis = 0xffffffffu;
      if (part) {
        vis = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = tok0 + g + 8 * (x >> 1);
            const bool ok = j >= max(lo[n][x & 1], t_lo) && j < min(hi[n][x & 1], t_hi);
            if (ok) vis |= 1u << (n * 4 + x);
            else s[n][x] = -CUDART_INF_F;
          }
      }
      // V's parameters; a token that no row sees may hold anything.
      float sv[2][G], cv[2][G];
      uint32_t sbits = 0;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool dead = part && (vis & (0x33333333u << (2 * r))) == 0;
#pragma unroll
        for (int h = 0; h < G; ++h) {
          float2 p = kv4_unpack_param<T>(tl.par[r][G + h]);
          if (dead) p = make_float2(0.f, 0.f);
          sv[r][h] = p.x;
          cv[r][h] = fmaf(8.f, p.x, p.y);
          const uint32_t u = __float_as_uint(p.x);
          sbits = max(sbits, u < 0x7f800000u ? u : 0u);
        }
      }
      // Running maxima: moved, with everything accumulated, when a score
      // passes one by kLazyMax or a larger step turns up.
      bool move = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < 2; ++q) move |= fmaxf(s[n][q], s[n][2 + q]) > mx[n][q] + kLazyMax;
      move |= (int)(sbits >> 23) - 127 > step_exp;
      if (__any_sync(0xffffffffu, move)) {
        const int top = (int)(__reduce_max_sync(0xffffffffu, sbits) >> 23) - 127;
        const int new_exp = max(step_exp, top);
        const float down = step_exp - new_exp < -126 ? 0.f : pow2i(step_exp - new_exp);
        step_exp = new_exp;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float v = fmaxf(s[n][q], s[n][2 + q]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
            const float m = fmaxf(mx[n][q], v);
            const float al = m == -CUDART_INF_F ? 1.f : exp2_fast(mx[n][q] - m);
            mx[n][q] = m;
            l[n][q] *= al;
#pragma unroll
            for (int h = 0; h < G; ++h) {
              aff[n][q][h] *= al;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[n][h][i][q] *= al * down;
                o[n][h][i][2 + q] *= al * down;
              }
            }
          }
      }
      // Weights.
      const float vs = pow2i(kStepExp - step_exp);
      uint32_t pf[NT][G][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float p[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float m = mx[n][x & 1];
          p[x] = exp2_fast(s[n][x] - (m == -CUDART_INF_F ? 0.f : m));
          l[n][x & 1] += p[x];
        }
#pragma unroll
        for (int h = 0; h < G; ++h)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float w[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const bool ok = !part || (vis >> (n * 4 + 2 * r + q) & 1u);
              w[q] = ok ? p[2 * r + q] * (sv[r][h] * vs) : 0.f;
              aff[n][q][h] += ok ? p[2 * r + q] * cv[r][h] : 0.f;
            }
            pf[n][h][r] = transpose8x8(pack_half2(w[0], w[1]));
          }
      }
      // O^T += V^T P^T.
#pragma unroll
      for (int h = 0; h < G; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) w[sl] = word_of(tl.v[(sl * G + h) / 4], (sl * G + h) % 4);
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

    long long where = locate(0);
    Tile<G> cur, nxt;
    bool have = false, have_next = false;
    auto fetch = [&](int i, Tile<G> &dst) -> bool {
      if (i >= mine) return false;
      if (i > 0 && i % 32 == 0) where = locate(i);
      const long long off = __shfl_sync(0xffffffffu, where, i % 32);
      if (off < 0) return false;
      load_tile<G>(dst, base + off, lane);
      return true;
    };
    have = fetch(0, cur);
    for (int i = 0; i < mine; ++i) {
      have_next = fetch(i + 1, nxt);
      if (have) compute(cur, (tile0 + warp + i * kWarps) << 4);
      cur = nxt;
      have = have_next;
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
  __syncthreads();  // q in shared memory has been read
  {
    const float unscale = pow2i(step_exp - kStepExp);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = n * 8 + 2 * t + q;
        if (g == 0) {
          sm_m[warp][r] = mx[n][q];
          sm_l[warp][r] = l[n][q];
        }
        float *dst = sm_o + (warp * R + r) * LDO;
#pragma unroll
        for (int h = 0; h < G; ++h) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[2 * i] = fmaf(o[n][h][i][q], unscale, aff[n][q][h]);
            v[2 * i + 1] = fmaf(o[n][h][i][2 + q], unscale * 0.0625f, aff[n][q][h]);
          }
          float4 *d4 = reinterpret_cast<float4 *>(dst + 64 * h + 8 * g);
          d4[0] = make_float4(v[0], v[1], v[2], v[3]);
          d4[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
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
      // A warp that saw no finite maximum adds nothing, unless its sum is a NaN.
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
  return D == 64 ? 4 : (D == 128 ? 2 : 1);
}

SplitPlan plan_kv4(const AttnArgs &a, size_t ws_available) {
  SplitPlan p;
  p.rows = a.group * a.Sq;
  const int most = a.D == 64 ? 4 : (a.D == 128 ? 2 : 1);
  p.nt = p.rows <= 8 || most == 1 ? 1 : (p.rows <= 16 || most == 2 ? 2 : 4);
  p.row_blocks = (p.rows + 8 * p.nt - 1) / (8 * p.nt);
  const long long units = (long long)a.B * a.Hkv * p.row_blocks;
  // Tokens that a sequence's rows can see between them.
  long long span = a.Skv;
  if (a.window >= 0) span = std::min<long long>(span, (long long)a.window + a.Sq + 16);
  int chunk = 1024;
  while (chunk > 64 && units * ((span + chunk - 1) / chunk) < 4LL * a.num_sms) chunk /= 2;
  p.chunk = chunk;
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
  constexpr size_t o_bytes = (size_t)kWarps * 8 * NT * (D + 4) * sizeof(float);
  constexpr size_t q_bytes = (size_t)8 * NT * D * sizeof(__half);
  constexpr size_t smem = o_bytes > q_bytes ? o_bytes : q_bytes;
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
  kv4_combine_kernel<T, D><<<(unsigned)((n_rows + 3) / 4), 128, 0, s>>>(a, p.chunk, p.n_splits, part_o, part_lse);
  return cudaGetLastError();
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
