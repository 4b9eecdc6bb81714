// The 4-bit key/value cache: its layout (include/llmx_attn.h) as the kernels
// address it, shared by the store / load kernels (kv4_cache.cu) and the
// attention over it (attn_kv4.cu).
#pragma once

#include "common.cuh"

namespace llmx_b200 {

// A validated cache and the lengths that bound its use.
struct Kv4Args {
  unsigned char *data;
  const int *table;  // nullable
  long long page_stride, head_stride, table_stride;
  int n_pages, max_pages, page_size, Hkv, D;
  int vec;  // attention: q and o rows can be read and written 16 bytes at a time
  unsigned int *err;
};

// Checks *c for `rows` and the current device; fills *k.
llmx_status prepare_kv4(const llmx_kv4_cache *c, const llmx_kv4_rows &rows, Kv4Args *k);
// The checks alone, without a device.
llmx_status validate_kv4(const llmx_kv4_cache *c, int batch, Kv4Args *k);
// The load without its checks, for the attention's expanded form: rows
// [lens[b], lens[b] rounded up to `pad`) are written as 0 and the ones behind
// them are left alone (pad 0: all of them are written as 0).  With a pad a V
// group that holds a NaN is written as 0, and K's group of its token as NaN: the
// prefill multiplies V by weights that are 0 for the rows that do not see the
// token, and 0 times NaN would reach them; a score is of one token alone, and
// masked ones are replaced.
cudaError_t launch_kv4_load(const Kv4Args &k, const llmx_kv4_rows &r, int dtype, int pad, cudaStream_t s);

constexpr int kKv4Group = LLMX_KV4_GROUP;
constexpr int kKv4TileTokens = LLMX_KV4_TILE_TOKENS;

__host__ __device__ inline int kv4_tile_bytes(int D) { return 18 * D; }

// Byte offset of the page that holds token `j` of sequence b, for j in
// [0, max_pages * page_size), or -1 (and the error word set) where the table
// points outside the cache.
__device__ __forceinline__ long long kv4_page_offset(const Kv4Args &a, int b, int page) {
  const long long id = a.table != nullptr ? (long long)a.table[b * a.table_stride + page]
                                          : (long long)b * a.max_pages + page;
  if (id < 0 || id >= a.n_pages) {
    raise_error(a.err, kDevErrBadPage);
    return -1;
  }
  return id * a.page_stride;
}

// Byte offset inside a tile of the code word of channels [8c, 8c + 8) of
// token `tok` (0..15), and of the token's parameters of channel group h.
__device__ __forceinline__ int kv4_k_word(int tok, int c, int G) {
  const int h = c >> 3, t = (c >> 1) & 3, w = c & 1;
  const int x = ((tok >> 3) * G + h) * 2 + w;
  return (x >> 2) * 512 + (4 * (tok & 7) + t) * 16 + (x & 3) * 4;
}
__device__ __forceinline__ int kv4_v_word(int tok, int c, int G) {
  const int h = c >> 3, g = c & 7;
  const int x = (2 * (tok >> 3) + (tok & 1)) * G + h;
  return 8 * 64 * G + (x >> 2) * 512 + (4 * g + ((tok & 7) >> 1)) * 16 + (x & 3) * 4;
}
__device__ __forceinline__ int kv4_param(int tok, int is_v, int h, int G) {
  return 16 * 64 * G + ((tok * 2 + is_v) * G + h) * 4;
}

// The two halves of a parameter word (s, m) as fp32.
template <typename T>
__device__ __forceinline__ float2 kv4_unpack_param(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}

// Whether the group of a parameter word reads back as NaN.
template <typename T>
__device__ __forceinline__ bool kv4_nan_step(uint32_t w) {
  return (w & 0x7fffu) > (std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u);
}

}  // namespace llmx_b200
