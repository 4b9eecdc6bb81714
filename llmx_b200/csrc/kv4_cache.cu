// Writing rows of K and V into the 4-bit cache and reading them back.
//
// One thread takes 8 consecutive channels of one (token, kv head) of K and of
// V, which is one 32-bit code word of each; the 8 threads of a 64-channel
// group reduce its minimum and maximum with shuffles.
#include <string>

#include "kv4.cuh"

namespace llmx_b200 {
namespace {

constexpr int kRowThreads = 256;

struct RowArgs {
  const void *k, *v;
  long long ks[3], vs[3];
  const int *start, *lens;
  int B, S, pad;
};

template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T *p, float (&f)[8]) {
  if constexpr (VEC) {
    unpack8<T>(*reinterpret_cast<const uint4 *>(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to_f(p[i]);
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

// min / max that hand a NaN on.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ T round_up_to(float r);
template <>
__device__ __forceinline__ __half round_up_to<__half>(float r) { return __float2half_ru(r); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_up_to<__nv_bfloat16>(float r) { return __float2bfloat16_ru(r); }

// The code word of this thread's 8 channels and the group's parameter word.
// All 8 threads of the group call it.
template <typename T>
__device__ __forceinline__ void quantise8(const float (&f)[8], uint32_t &codes, uint32_t &param) {
  float lo = f[0], hi = f[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, f[i]);
    hi = max_nan(hi, f[i]);
  }
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  const T st = round_up_to<T>(__fdiv_rn(hi - lo, 15.f));
  const T mt = Elem<T>::from_f(lo);  // exact: lo is one of the inputs
  const float s = Elem<T>::to_f(st);
  codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // s > 0 fails for a NaN too; inf / inf converts to 0.  The group reads
    // back as NaN then, through s or m.
    const float q = s > 0.f ? __fdiv_rn(f[i] - lo, s) : 0.f;
    codes |= (uint32_t)min(15, __float2int_rn(q)) << (4 * i);
  }
  const unsigned short sb = *reinterpret_cast<const unsigned short *>(&st);
  const unsigned short mb = *reinterpret_cast<const unsigned short *>(&mt);
  param = (uint32_t)sb | ((uint32_t)mb << 16);
}

template <typename T>
__device__ __forceinline__ void dequantise8(uint32_t codes, uint32_t param, float (&f)[8]) {
  const float2 p = kv4_unpack_param<T>(param);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = fmaf((float)((codes >> (4 * i)) & 15u), p.x, p.y);
}

// Where token `row` of sequence b lies (byte offset of the tile of kv head h)
// and its place in the tile, or -1.
__device__ __forceinline__ long long locate(const Kv4Args &a, int b, long long pos, int h, int &tok) {
  if (pos < 0 || pos >= (long long)a.max_pages * a.page_size) {
    raise_error(a.err, kDevErrBadPage);
    return -1;
  }
  const int p = (int)(pos / a.page_size), in = (int)(pos - (long long)p * a.page_size);
  const long long off = kv4_page_offset(a, b, p);
  if (off < 0) return -1;
  tok = in & 15;
  return off + h * a.head_stride + (long long)(in >> 4) * kv4_tile_bytes(a.D);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv4_store_kernel(Kv4Args a, RowArgs r) {
  const int C = a.D / 8, G = a.D / kKv4Group;
  const int b = blockIdx.y;
  const long long idx = (long long)blockIdx.x * kRowThreads + threadIdx.x;
  const int c = (int)(idx % C);
  const int h = (int)(idx / C % a.Hkv);
  const long long row = idx / C / a.Hkv;
  const bool live = row < clamp_len(r.lens, b, r.S);
  float kf[8] = {}, vf[8] = {};
  if (live) {
    load_row8<T, VEC>(static_cast<const T *>(r.k) + b * r.ks[0] + row * r.ks[1] + h * r.ks[2] + c * 8, kf);
    load_row8<T, VEC>(static_cast<const T *>(r.v) + b * r.vs[0] + row * r.vs[1] + h * r.vs[2] + c * 8, vf);
  }
  uint32_t kc, kp, vc, vp;
  quantise8<T>(kf, kc, kp);
  quantise8<T>(vf, vc, vp);
  if (!live) return;
  int tok = 0;
  const long long off = locate(a, b, (r.start ? (long long)r.start[b] : 0) + row, h, tok);
  if (off < 0) return;
  unsigned char *tile = a.data + off;
  *reinterpret_cast<uint32_t *>(tile + kv4_k_word(tok, c, G)) = kc;
  *reinterpret_cast<uint32_t *>(tile + kv4_v_word(tok, c, G)) = vc;
  if ((c & 7) == 0) {
    *reinterpret_cast<uint32_t *>(tile + kv4_param(tok, 0, c >> 3, G)) = kp;
    *reinterpret_cast<uint32_t *>(tile + kv4_param(tok, 1, c >> 3, G)) = vp;
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv4_load_kernel(Kv4Args a, RowArgs r) {
  const int C = a.D / 8, G = a.D / kKv4Group;
  const int b = blockIdx.y;
  const long long idx = (long long)blockIdx.x * kRowThreads + threadIdx.x;
  const int c = (int)(idx % C);
  const int h = (int)(idx / C % a.Hkv);
  const long long row = idx / C / a.Hkv;
  const int len = clamp_len(r.lens, b, r.S);
  const int end = r.pad > 0 ? min(r.S, (len + r.pad - 1) / r.pad * r.pad) : r.S;
  if (row >= end) return;
  float kf[8] = {}, vf[8] = {};
  if (row < len) {
    int tok = 0;
    const long long off = locate(a, b, (r.start ? (long long)r.start[b] : 0) + row, h, tok);
    if (off >= 0) {
      const unsigned char *tile = a.data + off;
      const uint32_t kc = *reinterpret_cast<const uint32_t *>(tile + kv4_k_word(tok, c, G));
      const uint32_t vc = *reinterpret_cast<const uint32_t *>(tile + kv4_v_word(tok, c, G));
      const uint32_t kp = *reinterpret_cast<const uint32_t *>(tile + kv4_param(tok, 0, c >> 3, G));
      const uint32_t vp = *reinterpret_cast<const uint32_t *>(tile + kv4_param(tok, 1, c >> 3, G));
      dequantise8<T>(kc, kp, kf);
      dequantise8<T>(vc, vp, vf);
    }
  }
  store_row8<T, VEC>(static_cast<T *>(const_cast<void *>(r.k)) + b * r.ks[0] + row * r.ks[1] + h * r.ks[2] + c * 8, kf);
  store_row8<T, VEC>(static_cast<T *>(const_cast<void *>(r.v)) + b * r.vs[0] + row * r.vs[1] + h * r.vs[2] + c * 8, vf);
}

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

llmx_status bad(const char *msg) { return record_error(LLMX_ERR_INVALID_ARGUMENT, msg); }

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

dim3 row_grid(const Kv4Args &k, const RowArgs &r) {
  const long long n = (long long)r.S * k.Hkv * (k.D / 8);
  return dim3((unsigned)((n + kRowThreads - 1) / kRowThreads), (unsigned)r.B);
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
  k->err = nullptr;
  return LLMX_OK;
}

llmx_status prepare_kv4(const llmx_kv4_cache *c, int batch, Kv4Args *k) {
  const llmx_status s = validate_kv4(c, batch, k);
  if (s != LLMX_OK) return s;
  int sms = 0;
  return current_device_info(&k->err, &sms);
}

cudaError_t launch_kv4_load(const Kv4Args &k, const llmx_kv4_rows &rows, int dtype, int pad, cudaStream_t s) {
  bool vec = false;
  const RowArgs r = row_args(rows, pad, &vec);
  const dim3 grid = row_grid(k, r);
  if (dtype == LLMX_FP16) {
    if (vec) kv4_load_kernel<__half, true><<<grid, kRowThreads, 0, s>>>(k, r);
    else kv4_load_kernel<__half, false><<<grid, kRowThreads, 0, s>>>(k, r);
  } else {
    if (vec) kv4_load_kernel<__nv_bfloat16, true><<<grid, kRowThreads, 0, s>>>(k, r);
    else kv4_load_kernel<__nv_bfloat16, false><<<grid, kRowThreads, 0, s>>>(k, r);
  }
  return cudaGetLastError();
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
  st = prepare_kv4(c, rows->batch, &k);
  if (st != LLMX_OK || rows->batch == 0 || rows->max_rows == 0) return st;
  bool vec = false;
  const RowArgs r = row_args(*rows, 0, &vec);
  const dim3 grid = row_grid(k, r);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->dtype == LLMX_FP16) {
    if (vec) kv4_store_kernel<__half, true><<<grid, kRowThreads, 0, s>>>(k, r);
    else kv4_store_kernel<__half, false><<<grid, kRowThreads, 0, s>>>(k, r);
  } else {
    if (vec) kv4_store_kernel<__nv_bfloat16, true><<<grid, kRowThreads, 0, s>>>(k, r);
    else kv4_store_kernel<__nv_bfloat16, false><<<grid, kRowThreads, 0, s>>>(k, r);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LLMX_OK : record_error(LLMX_ERR_CUDA, cudaGetErrorString(e));
}

extern "C" llmx_status llmx_kv4_load(const llmx_kv4_cache *c, const llmx_kv4_rows *rows, void *stream) {
  llmx_status st = validate_rows(rows);
  if (st != LLMX_OK) return st;
  Kv4Args k;
  st = prepare_kv4(c, rows->batch, &k);
  if (st != LLMX_OK || rows->batch == 0 || rows->max_rows == 0) return st;
  const cudaError_t e = launch_kv4_load(k, *rows, c->dtype, 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? LLMX_OK : record_error(LLMX_ERR_CUDA, cudaGetErrorString(e));
}
