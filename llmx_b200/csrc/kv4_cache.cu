// Writing rows of K and V into the 4-bit cache and reading them back.
//
// A warp takes one tile of 16 tokens of one kv head, lane (g, t) the words that
// the layout gives it: 16 channels of K of tokens g and g + 8 per group, 8
// channels of V of tokens 2t, 2t + 1, 2t + 8, 2t + 9.  Dense rows are moved 16
// bytes a lane in whole 32-byte sectors, a whole tile in 16-byte words; of a
// tile that the rows cover in part only the words of their tokens are written.
// Both are bound by HBM: 4 + 1.125 bytes per (K, V) pair of values.
//
// Few rows (a decode step's new token, a short tail) leave such warps idle or
// alone on their SMs; there a thread takes 8 channels of one row of K and of V.
#include <string>

#include "kv4.cuh"

namespace llmx_b200 {
namespace {

constexpr int kRowThreads = 128;
// From this many tiles on a warp takes a whole tile.  Measured, us of a store, a
// warp a tile / a thread 8 channels, at 256, 512, 1024 and 2048 tiles: head_dim
// 64 2.8 / 2.6, 3.0 / 3.1, 3.5 / 3.7, 4.6 / 5.7; 128 3.7 / 3.0, 3.7 / 3.7,
// 4.7 / 5.8, 6.7 / 9.5; 256 6.6 / 3.8, 6.7 / 5.8, 7.4 / 9.6, 12.9 / 17.2.
constexpr int kManyTiles = 1024;

struct RowArgs {
  const void *k, *v;
  long long ks[3], vs[3];
  const int *start, *lens;
  int B, S, pad;
};

// 8 consecutive channels.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_row8(const T *p) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4 *>(p);
  } else {
    const unsigned short *e = reinterpret_cast<const unsigned short *>(p);
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (uint32_t)e[2 * i] | ((uint32_t)e[2 * i + 1] << 16);
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_row8(T *p, const float (&f)[8]) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4 *>(p) = pack8<T>(f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = Elem<T>::from_f(f[i]);
  }
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

// Minimum and maximum of values two at a time, both halves apart; a NaN goes on.
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  using P = typename Pair<T>::type;
  const P r = __hmin2_nan(*reinterpret_cast<const P *>(&a), *reinterpret_cast<const P *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  using P = typename Pair<T>::type;
  const P r = __hmax2_nan(*reinterpret_cast<const P *>(&a), *reinterpret_cast<const P *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}

template <typename T>
__device__ __forceinline__ T round_up_to(float r);
template <>
__device__ __forceinline__ __half round_up_to<__half>(float r) { return __float2half_ru(r); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_up_to<__nv_bfloat16>(float r) { return __float2bfloat16_ru(r); }

// (min, -max) of the channels of N 16-byte pieces, packed.
template <typename T, int N>
__device__ __forceinline__ uint32_t low_high(const uint4 (&raw)[N]) {
  uint32_t lo = raw[0].x, hi = raw[0].x;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      lo = min2<T>(lo, w[x]);
      hi = max2<T>(hi, w[x]);
    }
  }
  // The halves of lo and hi against each other: (lo, -hi) of one half with that of the other.
  return min2<T>(__byte_perm(lo, hi, 0x5410) ^ 0x80000000u, __byte_perm(lo, hi, 0x7632) ^ 0x80000000u);
}

// A group's parameter word (s, m) from its packed (min, -max).
template <typename T>
__device__ __forceinline__ uint32_t param_of(uint32_t low_neg_high) {
  const uint32_t hi_bits = (low_neg_high >> 16) ^ 0x8000u;
  const unsigned short lo16 = (unsigned short)low_neg_high, hi16 = (unsigned short)hi_bits;
  const float lo = Elem<T>::to_f(*reinterpret_cast<const T *>(&lo16));
  const float range = Elem<T>::to_f(*reinterpret_cast<const T *>(&hi16)) - lo;
  // A range that is not finite gives a step that is a NaN.
  const T st = round_up_to<T>(range < CUDART_INF_F ? __fdiv_rn(range, 15.f) : CUDART_NAN_F);
  unsigned short s16 = *reinterpret_cast<const unsigned short *>(&st);
  // At the end of the type 15 s + m, which passes the maximum by up to 15 of s's
  // last bits, would round to infinity (from the largest number and half its last
  // bit on).  The next s below is under range / 15, so 15 s + m then is not past
  // the maximum, which stays within half a step: 15 last bits of s are at most
  // 15 2^-7 s, and the quotients below 15.5.
  constexpr float kInfinite = std::is_same<T, __half>::value ? 65520.f : 0x1.ffp127f;
  if (fmaf(15.f, Elem<T>::to_f(st), lo) >= kInfinite) --s16;
  return (uint32_t)s16 | ((uint32_t)lo16 << 16);
}
// 1 / s, 0 for s = 0, or -1 where codes_any() has to divide: between these
// bounds neither the reciprocal nor the products in codes()
// leave fp32's normal range.
__device__ __forceinline__ float inverse_of(float s) {
  return s > 0x1p-100f && s < 0x1p100f ? __frcp_rn(s) : (s == 0.f ? 0.f : -1.f);
}

// Parameter words and reciprocal steps of N groups, of which the L lanes that
// differ in the lane bits from FIRST on have a part each (packed (min, -max) in
// v): the lanes reduce them so that each ends with its share of the groups,
// computes those alone, and hands them round.  `own(j, param)` is called by one
// lane for each group j.
template <typename T, int N, int L, int FIRST, typename Own>
__device__ __forceinline__ void finish_groups(uint32_t (&v)[N], uint32_t (&param)[N], float (&inv)[N], int lane, Own own) {
  constexpr int kMine = N > L ? N / L : 1, kSame = N < L ? L / N : 1;  // groups of a lane, lanes of a group
  int cur = N;
#pragma unroll
  for (int off = L / 2 * FIRST; off >= FIRST; off /= 2) {
    const bool upper = (lane & off) != 0;
    if (cur > 1) {
      cur /= 2;
#pragma unroll
      for (int j = 0; j < N / 2; ++j)
        if (j < cur) {
          const uint32_t keep = upper ? v[j + cur] : v[j], send = upper ? v[j] : v[j + cur];
          v[j] = min2<T>(keep, __shfl_xor_sync(0xffffffffu, send, off));
        }
    } else {
      v[0] = min2<T>(v[0], __shfl_xor_sync(0xffffffffu, v[0], off));
    }
  }
  const int li = lane / FIRST % L;
  uint32_t p[kMine];
  float iv[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    p[j] = param_of<T>(v[j]);
    iv[j] = inverse_of(kv4_unpack_param<T>(p[j]).x);
    if (li % kSame == 0) own(li * kMine / kSame + j, p[j]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int from = lane % FIRST + j * kSame / kMine * FIRST + lane / (FIRST * L) * (FIRST * L);
    param[j] = __shfl_sync(0xffffffffu, p[j % kMine], from);
    inv[j] = __shfl_sync(0xffffffffu, iv[j % kMine], from);
  }
}

// x - m of the two halves of a register, straight from 16 bits.
template <typename T>
__device__ __forceinline__ void minus2(uint32_t x, float m, float &lo, float &hi) {
  if constexpr (std::is_same<T, __half>::value) {
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.f16 %0, l, %3;\n\tsub.rn.f32.f16 %1, h, %3;}"
        : "=f"(lo), "=f"(hi)
        : "r"(x), "f"(m));
  } else {
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.bf16 %0, l, %3;\n\tsub.rn.f32.bf16 %1, h, %3;}"
        : "=f"(lo), "=f"(hi)
        : "r"(x), "f"(m));
  }
}

// The code word of 8 channels.  The quotient is the correctly rounded one
// (Markstein: a product with the rounded reciprocal and one step with the
// exact remainder), without the division; adding 1.5 * 2^23 rounds it to the
// nearest even integer in the low bits, and sums of those times 16^i make the
// word.
template <typename T>
__device__ __forceinline__ uint32_t codes(const uint4 &raw, uint32_t param, float inv) {
  const float2 sm = kv4_unpack_param<T>(param);
  float d[8];
  minus2<T>(raw.x, sm.y, d[0], d[1]);
  minus2<T>(raw.y, sm.y, d[2], d[3]);
  minus2<T>(raw.z, sm.y, d[4], d[5]);
  minus2<T>(raw.w, sm.y, d[6], d[7]);
  uint32_t word = 0u - 0x4b400000u * 0x11111111u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = d[i] * inv;
    const float r = fmaf(fmaf(-q, sm.x, d[i]), inv, q);
    word += __float_as_uint(r + 12582912.f) << (4 * i);
  }
  return word;
}
// The same for any step: outside the bounds above it divides, and a step that
// is a NaN gives 0 (the group reads back as NaN).
template <typename T>
__device__ __noinline__ uint32_t codes_any(uint4 raw, uint32_t param, float inv) {
  if (inv >= 0.f) return codes<T>(raw, param, inv);
  float f[8];
  unpack8<T>(raw, f);
  const float2 sm = kv4_unpack_param<T>(param);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = sm.x > 0.f ? __fdiv_rn(f[i] - sm.y, sm.x) : 0.f;
    word |= (uint32_t)min(15, __float2int_rn(q)) << (4 * i);
  }
  return word;
}

template <typename T>
__device__ __forceinline__ void dequantise8(uint32_t code, uint32_t param, float (&f)[8]) {
  const float2 p = kv4_unpack_param<T>(param);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = fmaf((float)((code >> (4 * i)) & 15u), p.x, p.y);
}

// The tile that a warp takes: its place, and the row that its first token is.
struct TileAt {
  int b, h, len;
  long long row0;          // row of token 0 (negative: the rows begin inside the tile)
  unsigned char *tile;     // null where no page holds it
};
__device__ __forceinline__ TileAt tile_at(const Kv4Args &a, const RowArgs &r) {
  TileAt t;
  t.b = blockIdx.y;
  const int warp = threadIdx.x / 32;
  const uint32_t idx = blockIdx.x * (kRowThreads / 32) + warp;
  t.h = (int)(idx % (uint32_t)a.Hkv);
  t.len = clamp_len(r.lens, t.b, r.S);
  const long long start = r.start ? (long long)r.start[t.b] : 0;
  const long long tile = (start >> 4) + idx / (uint32_t)a.Hkv;
  t.row0 = tile * 16 - start;
  t.tile = nullptr;
  // A row of the call lies in the tile.  (Without one, which a first tile that
  // begins before row 0 can be, the table holds nothing for it.)
  if (t.len > 0 && t.row0 < t.len) {
    const long long pos = tile * 16;
    if (pos >= 0 && pos < (long long)a.max_pages * a.page_size) {
      const int p = (int)pos / a.page_size, in = (int)pos - p * a.page_size;
      const long long off = kv4_page_offset(a, t.b, p);
      if (off >= 0) t.tile = a.data + off + t.h * a.head_stride + (long long)(in >> 4) * kv4_tile_bytes(a.D);
    } else {
      raise_error(a.err, kDevErrBadPage);
    }
  }
  return t;
}
__device__ __forceinline__ bool row_here(const TileAt &t, int tok) {
  return t.row0 + tok >= 0 && t.row0 + tok < t.len;
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kRowThreads, D == 256 ? 2 : 4) kv4_store_kernel(const __grid_constant__ Kv4Args a,
                                                                const __grid_constant__ RowArgs r) {
  constexpr int G = D / kKv4Group;
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  const TileAt at = tile_at(a, r);
  if (at.tile == nullptr) return;
  const bool whole = at.row0 >= 0 && at.row0 + 16 <= at.len;
  const T *k = static_cast<const T *>(r.k) + at.b * r.ks[0] + at.h * r.ks[2];
  const T *v = static_cast<const T *>(r.v) + at.b * r.vs[0] + at.h * r.vs[2];
  uint4 kr[2][G][2], vr[4][G][1];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = g + 8 * i;
    const T *p = k + (at.row0 + tok) * r.ks[1] + 16 * t;
    const bool here = whole || row_here(at, tok);
#pragma unroll
    for (int h = 0; h < G; ++h)
#pragma unroll
      for (int w = 0; w < 2; ++w) kr[i][h][w] = here ? load_row8<T, VEC>(p + 64 * h + 8 * w) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tok = 2 * t + (i & 1) + 8 * (i >> 1);
    const T *p = v + (at.row0 + tok) * r.vs[1] + 8 * g;
    const bool here = whole || row_here(at, tok);
#pragma unroll
    for (int h = 0; h < G; ++h) vr[i][h][0] = here ? load_row8<T, VEC>(p + 64 * h) : make_uint4(0u, 0u, 0u, 0u);
  }
  // Groups: (i, h) of K over the lanes t, of V over the lanes g.
  uint32_t kp[2 * G], vp[4 * G], x[2 * G], y[4 * G];
  float ki[2 * G], vi[4 * G];
  unsigned char *par = at.tile + 16 * D;
#pragma unroll
  for (int j = 0; j < 2 * G; ++j) x[j] = low_high<T, 2>(kr[j / G][j % G]);
#pragma unroll
  for (int j = 0; j < 4 * G; ++j) y[j] = low_high<T, 1>(vr[j / G][j % G]);
  finish_groups<T, 2 * G, 4, 1>(x, kp, ki, lane, [&](int j, uint32_t param) {
    const int tok = g + 8 * (j / G);
    if (whole || row_here(at, tok)) *reinterpret_cast<uint32_t *>(par + (tok * 2 * G + j % G) * 4) = param;
  });
  finish_groups<T, 4 * G, 8, 4>(y, vp, vi, lane, [&](int j, uint32_t param) {
    const int tok = 2 * t + (j / G & 1) + 8 * (j / G >> 1);
    if (whole || row_here(at, tok)) *reinterpret_cast<uint32_t *>(par + (tok * 2 * G + G + j % G) * 4) = param;
  });
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 4 * G; ++j) odd = odd || vi[j] < 0.f || ki[j / 2] < 0.f;
  uint32_t kw[4 * G], vw[4 * G];
  if (!__any_sync(0xffffffffu, odd)) {
#pragma unroll
    for (int j = 0; j < 4 * G; ++j) {
      kw[j] = codes<T>(kr[j / 2 / G][j / 2 % G][j % 2], kp[j / 2], ki[j / 2]);
      vw[j] = codes<T>(vr[j / G][j % G][0], vp[j], vi[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4 * G; ++j) {
      kw[j] = codes_any<T>(kr[j / 2 / G][j / 2 % G][j % 2], kp[j / 2], ki[j / 2]);
      vw[j] = codes_any<T>(vr[j / G][j % G][0], vp[j], vi[j]);
    }
  }
  unsigned char *kd = at.tile + lane * 16, *vd = kd + 8 * D;
  if (whole) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      *reinterpret_cast<uint4 *>(kd + 512 * i) = make_uint4(kw[4 * i], kw[4 * i + 1], kw[4 * i + 2], kw[4 * i + 3]);
      *reinterpret_cast<uint4 *>(vd + 512 * i) = make_uint4(vw[4 * i], vw[4 * i + 1], vw[4 * i + 2], vw[4 * i + 3]);
    }
  } else {
#pragma unroll
    for (int x = 0; x < 4 * G; ++x) {
      const int ki = x / (2 * G), vi = x / G;  // the token of word x
      if (row_here(at, g + 8 * ki)) *reinterpret_cast<uint32_t *>(kd + x / 4 * 512 + x % 4 * 4) = kw[x];
      if (row_here(at, 2 * t + (vi & 1) + 8 * (vi >> 1))) *reinterpret_cast<uint32_t *>(vd + x / 4 * 512 + x % 4 * 4) = vw[x];
    }
  }
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv4_load_kernel(const __grid_constant__ Kv4Args a,
                                                               const __grid_constant__ RowArgs r) {
  constexpr int G = D / kKv4Group;
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  const TileAt at = tile_at(a, r);
  const long long end = r.pad > 0 ? min((long long)r.S, ((long long)at.len + r.pad - 1) / r.pad * r.pad) : r.S;
  if (at.row0 >= end) return;
  T *k = static_cast<T *>(const_cast<void *>(r.k)) + at.b * r.ks[0] + at.h * r.ks[2];
  T *v = static_cast<T *>(const_cast<void *>(r.v)) + at.b * r.vs[0] + at.h * r.vs[2];
  uint32_t kw[4 * G], vw[4 * G];
  const unsigned char *par = at.tile + 16 * D;
  if (at.tile != nullptr) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint4 u = ld_stream16(at.tile + 512 * i + lane * 16), w = ld_stream16(at.tile + 8 * D + 512 * i + lane * 16);
      kw[4 * i] = u.x;
      kw[4 * i + 1] = u.y;
      kw[4 * i + 2] = u.z;
      kw[4 * i + 3] = u.w;
      vw[4 * i] = w.x;
      vw[4 * i + 1] = w.y;
      vw[4 * i + 2] = w.z;
      vw[4 * i + 3] = w.w;
    }
  }
  // K: lanes t and t ^ 1 swap a word, so that each store of the two covers a
  // whole 32-byte sector.
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int tok = g + 8 * i;
    const bool held = at.tile != nullptr && row_here(at, tok);
    const bool wanted = at.row0 + tok >= 0 && at.row0 + tok < end;
    T *p = k + (at.row0 + tok) * r.ks[1] + 32 * (t >> 1) + 8 * (t & 1);
#pragma unroll
    for (int h = 0; h < G; ++h) {
      const uint32_t w0 = kw[(i * G + h) * 2], w1 = kw[(i * G + h) * 2 + 1];
      const uint32_t other = __shfl_xor_sync(0xffffffffu, t & 1 ? w0 : w1, 1);
      const uint32_t word[2] = {t & 1 ? other : w0, t & 1 ? w1 : other};
      uint32_t param = held ? *reinterpret_cast<const uint32_t *>(par + (tok * 2 * G + h) * 4) : 0u;
      if (r.pad > 0 && held) {
        const uint32_t of_v = *reinterpret_cast<const uint32_t *>(par + (tok * 2 * G + G + h) * 4);
        if (kv4_nan_step<T>(of_v)) param = of_v;
      }
      if (wanted) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float f[8] = {};
          if (held) dequantise8<T>(word[x], param, f);
          store_row8<T, VEC>(p + 64 * h + 16 * x, f);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tok = 2 * t + (i & 1) + 8 * (i >> 1);
    const bool held = at.tile != nullptr && row_here(at, tok);
    const bool wanted = at.row0 + tok >= 0 && at.row0 + tok < end;
    T *p = v + (at.row0 + tok) * r.vs[1] + 8 * g;
#pragma unroll
    for (int h = 0; h < G; ++h) {
      uint32_t param = held ? *reinterpret_cast<const uint32_t *>(par + (tok * 2 * G + G + h) * 4) : 0u;
      if (r.pad > 0 && kv4_nan_step<T>(param)) param = 0u;
      if (wanted) {
        float f[8] = {};
        if (held) dequantise8<T>(vw[i * G + h], param, f);
        store_row8<T, VEC>(p + 64 * h, f);
      }
    }
  }
}

// ---- few rows: a thread takes channels [8c, 8c + 8) of one row and kv head

struct RowAt {
  int b, h, c, len, tok;
  long long row;
  unsigned char *tile;  // null where no page holds the row
};
template <int D>
__device__ __forceinline__ RowAt row_at(const Kv4Args &a, const RowArgs &r) {
  RowAt t;
  t.b = blockIdx.y;
  const uint32_t idx = blockIdx.x * kRowThreads + threadIdx.x;
  t.c = (int)(idx % (D / 8));
  t.h = (int)(idx / (D / 8) % (uint32_t)a.Hkv);
  t.row = idx / (D / 8) / (uint32_t)a.Hkv;
  t.len = clamp_len(r.lens, t.b, r.S);
  t.tile = nullptr;
  t.tok = 0;
  if (t.row < t.len) {
    const long long pos = (r.start ? (long long)r.start[t.b] : 0) + t.row;
    if (pos >= 0 && pos < (long long)a.max_pages * a.page_size) {
      const int p = (int)pos / a.page_size, in = (int)pos - p * a.page_size;
      const long long off = kv4_page_offset(a, t.b, p);
      t.tok = in & 15;
      if (off >= 0) t.tile = a.data + off + t.h * a.head_stride + (long long)(in >> 4) * kv4_tile_bytes(D);
    } else {
      raise_error(a.err, kDevErrBadPage);
    }
  }
  return t;
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv4_store_few_kernel(const __grid_constant__ Kv4Args a,
                                                                    const __grid_constant__ RowArgs r) {
  constexpr int G = D / kKv4Group;
  const RowAt at = row_at<D>(a, r);
  uint4 kr[1] = {make_uint4(0u, 0u, 0u, 0u)}, vr[1] = {make_uint4(0u, 0u, 0u, 0u)};
  if (at.row < at.len) {
    kr[0] = load_row8<T, VEC>(static_cast<const T *>(r.k) + at.b * r.ks[0] + at.row * r.ks[1] + at.h * r.ks[2] + at.c * 8);
    vr[0] = load_row8<T, VEC>(static_cast<const T *>(r.v) + at.b * r.vs[0] + at.row * r.vs[1] + at.h * r.vs[2] + at.c * 8);
  }
  // The 8 threads of a group are in one warp and all of them come here.
  uint32_t kp[1], vp[1], x[1] = {low_high<T, 1>(kr)}, y[1] = {low_high<T, 1>(vr)};
  float ki[1], vi[1];
  const int lane = threadIdx.x % 32;
  finish_groups<T, 1, 8, 1>(x, kp, ki, lane, [](int, uint32_t) {});
  finish_groups<T, 1, 8, 1>(y, vp, vi, lane, [](int, uint32_t) {});
  if (at.tile == nullptr) return;
  *reinterpret_cast<uint32_t *>(at.tile + kv4_k_word(at.tok, at.c, G)) = codes_any<T>(kr[0], kp[0], ki[0]);
  *reinterpret_cast<uint32_t *>(at.tile + kv4_v_word(at.tok, at.c, G)) = codes_any<T>(vr[0], vp[0], vi[0]);
  if ((at.c & 7) == 0) {
    *reinterpret_cast<uint32_t *>(at.tile + kv4_param(at.tok, 0, at.c >> 3, G)) = kp[0];
    *reinterpret_cast<uint32_t *>(at.tile + kv4_param(at.tok, 1, at.c >> 3, G)) = vp[0];
  }
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv4_load_few_kernel(const __grid_constant__ Kv4Args a,
                                                                   const __grid_constant__ RowArgs r) {
  constexpr int G = D / kKv4Group;
  const RowAt at = row_at<D>(a, r);
  const long long end = r.pad > 0 ? min((long long)r.S, ((long long)at.len + r.pad - 1) / r.pad * r.pad) : r.S;
  if (at.row >= end) return;
  float kf[8] = {}, vf[8] = {};
  if (at.tile != nullptr) {
    const uint32_t kc = *reinterpret_cast<const uint32_t *>(at.tile + kv4_k_word(at.tok, at.c, G));
    const uint32_t vc = *reinterpret_cast<const uint32_t *>(at.tile + kv4_v_word(at.tok, at.c, G));
    uint32_t kp = *reinterpret_cast<const uint32_t *>(at.tile + kv4_param(at.tok, 0, at.c >> 3, G));
    uint32_t vp = *reinterpret_cast<const uint32_t *>(at.tile + kv4_param(at.tok, 1, at.c >> 3, G));
    if (r.pad > 0 && kv4_nan_step<T>(vp)) {
      kp = vp;
      vp = 0u;
    }
    dequantise8<T>(kc, kp, kf);
    dequantise8<T>(vc, vp, vf);
  }
  store_row8<T, VEC>(static_cast<T *>(const_cast<void *>(r.k)) + at.b * r.ks[0] + at.row * r.ks[1] + at.h * r.ks[2] + at.c * 8, kf);
  store_row8<T, VEC>(static_cast<T *>(const_cast<void *>(r.v)) + at.b * r.vs[0] + at.row * r.vs[1] + at.h * r.vs[2] + at.c * 8, vf);
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

llmx_status bad(const char *msg) { return record_error(LLMX_ERR_INVALID_ARGUMENT, msg); }

// What the kernels number in 32 bits: the tiles of a sequence's rows, all heads.
bool rows_fit(const llmx_kv4_rows &r, int heads) {
  return ((long long)r.max_rows / 16 + 2) * heads < (1LL << 31);
}

llmx_status validate_rows(const llmx_kv4_rows *r) {
  if (r == nullptr) return bad("kv4: rows is NULL");
  if (r->batch < 0 || r->batch > 65535 || r->max_rows < 0) return bad("kv4: batch must be in [0, 65535] and max_rows >= 0");
  if (r->batch == 0 || r->max_rows == 0) return LLMX_OK;  // nothing to do: the pointers may be NULL
  if (r->k == nullptr || r->v == nullptr) return bad("kv4: k and v must be non-NULL");
  if (((reinterpret_cast<uintptr_t>(r->k) | reinterpret_cast<uintptr_t>(r->v)) & 1u) != 0)
    return bad("kv4: k and v must be aligned to their elements");
  for (int i = 0; i < 3; ++i)
    if (r->k_stride[i] < 0 || r->v_stride[i] < 0) return bad("kv4: strides must be >= 0");
  return LLMX_OK;
}

RowArgs row_args(const llmx_kv4_rows &r, int pad, bool *vec) {
  RowArgs a{};
  a.k = r.k;
  a.v = r.v;
  *vec = al16(r.k) && al16(r.v);
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = r.k_stride[i];
    a.vs[i] = r.v_stride[i];
    *vec = *vec && a.ks[i] % 8 == 0 && a.vs[i] % 8 == 0;
  }
  a.start = r.start;
  a.lens = r.lens;
  a.B = r.batch;
  a.S = r.max_rows;
  a.pad = pad;
  return a;
}

template <typename T, int D, bool VEC>
cudaError_t launch_rows_v(bool store, const Kv4Args &k, const RowArgs &r, cudaStream_t s) {
  // A warp for each tile that a sequence's rows can touch, heads fastest.
  const long long tiles = (((long long)r.S + 14) / 16 + 1) * k.Hkv;
  if (r.S >= kKv4TileTokens && tiles * r.B >= kManyTiles) {
    const dim3 grid((unsigned)((tiles + kRowThreads / 32 - 1) / (kRowThreads / 32)), (unsigned)r.B);
    if (store) kv4_store_kernel<T, D, VEC><<<grid, kRowThreads, 0, s>>>(k, r);
    else kv4_load_kernel<T, D, VEC><<<grid, kRowThreads, 0, s>>>(k, r);
  } else {
    const long long n = (long long)r.S * k.Hkv * (D / 8);
    const dim3 grid((unsigned)((n + kRowThreads - 1) / kRowThreads), (unsigned)r.B);
    if (store) kv4_store_few_kernel<T, D, VEC><<<grid, kRowThreads, 0, s>>>(k, r);
    else kv4_load_few_kernel<T, D, VEC><<<grid, kRowThreads, 0, s>>>(k, r);
  }
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_rows_d(bool store, const Kv4Args &k, const RowArgs &r, bool vec, cudaStream_t s) {
  return vec ? launch_rows_v<T, D, true>(store, k, r, s) : launch_rows_v<T, D, false>(store, k, r, s);
}

template <typename T>
cudaError_t launch_rows_t(bool store, const Kv4Args &k, const RowArgs &r, bool vec, cudaStream_t s) {
  switch (k.D) {
    case 64: return launch_rows_d<T, 64>(store, k, r, vec, s);
    case 128: return launch_rows_d<T, 128>(store, k, r, vec, s);
    case 256: return launch_rows_d<T, 256>(store, k, r, vec, s);
  }
  return cudaErrorNotSupported;
}

cudaError_t launch_rows(bool store, const Kv4Args &k, const llmx_kv4_rows &rows, int dtype, int pad, cudaStream_t s) {
  bool vec = false;
  const RowArgs r = row_args(rows, pad, &vec);
  return dtype == LLMX_FP16 ? launch_rows_t<__half>(store, k, r, vec, s)
                            : launch_rows_t<__nv_bfloat16>(store, k, r, vec, s);
}

}  // namespace

llmx_status validate_kv4(const llmx_kv4_cache *c, int batch, Kv4Args *k) {
  if (c == nullptr) return bad("kv4: cache is NULL");
  if (c->dtype != LLMX_FP16 && c->dtype != LLMX_BF16)
    return record_error(LLMX_ERR_UNSUPPORTED, "kv4: dtype must be fp16 or bf16");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return record_error(LLMX_ERR_UNSUPPORTED, "kv4: head_dim must be 64, 128 or 256");
  if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return bad("kv4: n_kv_heads must be in [1, 65535]");
  if (c->page_size < 16 || c->page_size % 16) return bad("kv4: page_size must be a multiple of 16");
  if (c->n_pages < 1 || c->max_pages < 1) return bad("kv4: n_pages and max_pages must be >= 1");
  if ((long long)c->max_pages * c->page_size > (1LL << 30))
    return bad("kv4: max_pages * page_size must be at most 2^30");
  if (c->data == nullptr || !al16(c->data)) return bad("kv4: data must be non-NULL and 16-byte aligned");
  const long long page = (long long)c->page_size / 16 * kv4_tile_bytes(c->head_dim);
  if (c->page_stride < 0 || c->page_stride % 16 || c->head_stride < 0 || c->head_stride % 16)
    return bad("kv4: page_stride and head_stride must be >= 0 and multiples of 16");
  if ((c->n_kv_heads > 1 && c->head_stride < page) || (c->n_pages > 1 && c->page_stride < page))
    return bad("kv4: page_stride and head_stride must hold a page of one kv head");
  if (c->block_table != nullptr && c->table_stride < 0) return bad("kv4: table_stride must be >= 0");
  if (c->block_table == nullptr && (long long)batch * c->max_pages > c->n_pages)
    return bad("kv4: without a block table the cache must hold batch * max_pages pages");
  k->data = static_cast<unsigned char *>(c->data);
  k->table = c->block_table;
  k->page_stride = c->page_stride;
  k->head_stride = c->head_stride;
  k->table_stride = c->table_stride;
  k->n_pages = c->n_pages;
  k->max_pages = c->max_pages;
  k->page_size = c->page_size;
  k->Hkv = c->n_kv_heads;
  k->D = c->head_dim;
  k->vec = 0;
  k->err = nullptr;
  return LLMX_OK;
}

llmx_status prepare_kv4(const llmx_kv4_cache *c, const llmx_kv4_rows &rows, Kv4Args *k) {
  const llmx_status s = validate_kv4(c, rows.batch, k);
  if (s != LLMX_OK) return s;
  if (!rows_fit(rows, c->n_kv_heads)) return bad("kv4: max_rows / 16 * n_kv_heads must stay below 2^31");
  int sms = 0;
  return current_device_info(&k->err, &sms);
}

cudaError_t launch_kv4_load(const Kv4Args &k, const llmx_kv4_rows &rows, int dtype, int pad, cudaStream_t s) {
  return launch_rows(false, k, rows, dtype, pad, s);
}

}  // namespace llmx_b200

using namespace llmx_b200;

extern "C" llmx_status llmx_kv4_page_bytes(int32_t head_dim, int32_t page_size, int64_t *bytes) {
  if (bytes == nullptr) return bad("kv4: bytes is NULL");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return record_error(LLMX_ERR_UNSUPPORTED, "kv4: head_dim must be 64, 128 or 256");
  if (page_size < 16 || page_size % 16) return bad("kv4: page_size must be a multiple of 16");
  *bytes = (int64_t)page_size / 16 * kv4_tile_bytes(head_dim);
  return LLMX_OK;
}

extern "C" llmx_status llmx_kv4_store(const llmx_kv4_cache *c, const llmx_kv4_rows *rows, void *stream) {
  llmx_status st = validate_rows(rows);
  if (st != LLMX_OK) return st;
  Kv4Args k;
  st = prepare_kv4(c, *rows, &k);
  if (st != LLMX_OK || rows->batch == 0 || rows->max_rows == 0) return st;
  const cudaError_t e = launch_rows(true, k, *rows, c->dtype, 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? LLMX_OK : record_error(LLMX_ERR_CUDA, cudaGetErrorString(e));
}

extern "C" llmx_status llmx_kv4_load(const llmx_kv4_cache *c, const llmx_kv4_rows *rows, void *stream) {
  llmx_status st = validate_rows(rows);
  if (st != LLMX_OK) return st;
  Kv4Args k;
  st = prepare_kv4(c, *rows, &k);
  if (st != LLMX_OK || rows->batch == 0 || rows->max_rows == 0) return st;
  const int64_t extent[3] = {rows->batch, rows->max_rows, c->n_kv_heads};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (rows->k_stride[i] == 0 || rows->v_stride[i] == 0))
      return bad("kv4: rows that are written must not overlap (stride 0)");
  const cudaError_t e = launch_kv4_load(k, *rows, c->dtype, 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? LLMX_OK : record_error(LLMX_ERR_CUDA, cudaGetErrorString(e));
}
