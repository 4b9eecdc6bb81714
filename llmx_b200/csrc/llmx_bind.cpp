// Torch binding of llmx's attention op: the Python function the reference
// exposes from csrc/llmx_bind.cpp:35-78,
//
//   single_mha_attention_half(output, q, k, v, sm_scale,
//                             sliding_window=-1, logits_soft_cap=0.0)
//
// with the same name, argument order, defaults and TORCH_CHECK conditions
// (3-D tensors, one dtype, CUDA tensors on one device, n_heads divisible by
// n_kv_heads, matching head_dim; llmx_bind.cpp:41-58), built as a torch
// extension over the C ABI in llmx_attn.h.  Differences, all additive:
//  * keyword arguments alibi_slopes, causal, q_lens, kv_lens, lse (the
//    reference always passes no slopes and runs causal only,
//    llmx_bind.cpp:69-71);
//  * 4-D [batch, seq, heads, head_dim] tensors and fp32;
//  * strided q / k / v / output (unit stride on head_dim) are passed as they
//    are instead of being made contiguous;
//  * the work runs on torch's current CUDA stream, not stream 0;
//  * split-KV decode scratch comes from torch's caching allocator;
//  * algo (force one kernel family) and kv_offset / kv_total (a shard of a
//    sequence's keys at its global positions) as in llmx_attn_params.
// Library failures raise llmx_b200.LlmxError (a RuntimeError) carrying the
// llmx_status and the library's message.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <string>

#include "llmx_attn.h"

namespace py = pybind11;

namespace {

int32_t llmx_dtype_of(const torch::Tensor &t) {
  switch (t.scalar_type()) {
    case torch::kFloat: return LLMX_FP32;
    case torch::kHalf: return LLMX_FP16;
    case torch::kBFloat16: return LLMX_BF16;
    default:
      TORCH_CHECK(false, "llmx: unsupported dtype ", t.scalar_type(),
                  ". Only float16, bfloat16, float32 are supported.");
  }
  return -1;
}

void set_strides(int64_t (&dst)[3], const torch::Tensor &t, bool four) {
  dst[0] = four ? t.stride(0) : 0;
  dst[1] = t.stride(four ? 1 : 0);
  dst[2] = t.stride(four ? 2 : 1);
}

// A failing llmx_status, raised to Python as llmx_b200.LlmxError(status, message).
struct StatusError {
  int status;
  std::string message;
};

void check_status(llmx_status s) {
  if (s != LLMX_OK) throw StatusError{(int)s, llmx_attn_last_error()};
}

int32_t algo_code(const std::string &name) {
  if (name == "auto") return LLMX_ALGO_AUTO;
  if (name == "simt") return LLMX_ALGO_SIMT;
  if (name == "decode") return LLMX_ALGO_DECODE;
  if (name == "tcgen05") return LLMX_ALGO_TCGEN05;
  TORCH_CHECK(false, "algo must be one of auto, simt, decode, tcgen05");
  return 0;
}

}  // namespace

void single_mha_attention_half(torch::Tensor output, torch::Tensor q, torch::Tensor k, torch::Tensor v,
                               double sm_scale, int64_t sliding_window, double logits_soft_cap,
                               std::optional<torch::Tensor> alibi_slopes, bool causal,
                               std::optional<torch::Tensor> q_lens, std::optional<torch::Tensor> kv_lens,
                               std::optional<torch::Tensor> lse, const std::string &algo, int64_t kv_offset,
                               int64_t kv_total) {
  const int64_t nd = q.dim();
  TORCH_CHECK((nd == 3 || nd == 4) && k.dim() == nd && v.dim() == nd && output.dim() == nd,
              "q, k, v must be 3-D: [seq, heads, head_dim] (or all 4-D: [batch, seq, heads, head_dim])");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
              "q, k, v must have the same dtype");
  TORCH_CHECK(output.scalar_type() == q.scalar_type(), "output must have the dtype of q");
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda() && output.is_cuda(), "q, k, v must be CUDA tensors");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device() && q.device() == output.device(),
              "q, k, v must be on the same device");
  const bool four = nd == 4;
  const int64_t B = four ? q.size(0) : 1;
  const int64_t Sq = q.size(nd - 3), H = q.size(nd - 2), D = q.size(nd - 1);
  const int64_t Skv = k.size(nd - 3), Hkv = k.size(nd - 2);
  TORCH_CHECK(H % Hkv == 0, "n_heads (", H, ") must be divisible by n_kv_heads (", Hkv, ")");
  TORCH_CHECK(q.size(nd - 1) == k.size(nd - 1) && q.size(nd - 1) == v.size(nd - 1),
              "head_dim must match across q, k, v");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
  TORCH_CHECK(output.sizes() == q.sizes(), "output must have the shape of q");
  TORCH_CHECK(!four || (k.size(0) == B && v.size(0) == B), "batch sizes must match");
  // Rows with a unit head_dim stride are taken as they are (the reference
  // makes every input contiguous, llmx_bind.cpp:60-62).
  if (q.stride(-1) != 1) q = q.contiguous();
  if (k.stride(-1) != 1) k = k.contiguous();
  if (v.stride(-1) != 1) v = v.contiguous();
  TORCH_CHECK(output.stride(-1) == 1, "output must have a unit stride on head_dim");

  const c10::cuda::CUDAGuard guard(q.device());
  llmx_attn_params p;
  check_status(llmx_attn_params_init(&p));
  p.dtype = llmx_dtype_of(q);
  p.batch = (int32_t)B;
  p.n_heads = (int32_t)H;
  p.n_kv_heads = (int32_t)Hkv;
  p.head_dim = (int32_t)D;
  p.max_q_len = (int32_t)Sq;
  p.max_kv_len = (int32_t)Skv;
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.o = output.data_ptr();
  set_strides(p.q_stride, q, four);
  set_strides(p.k_stride, k, four);
  set_strides(p.v_stride, v, four);
  set_strides(p.o_stride, output, four);
  torch::Tensor slopes, ql, kl;
  if (alibi_slopes.has_value()) {
    TORCH_CHECK(alibi_slopes->is_cuda() && alibi_slopes->device() == q.device(), "alibi_slopes must be on q's device");
    slopes = alibi_slopes->to(torch::kFloat).contiguous();
    TORCH_CHECK(slopes.numel() == H, "alibi_slopes must have n_heads elements");
    p.alibi_slopes = slopes.data_ptr<float>();
  }
  if (q_lens.has_value()) {
    TORCH_CHECK(q_lens->is_cuda() && q_lens->device() == q.device(), "q_lens must be on q's device");
    ql = q_lens->to(torch::kInt).contiguous();
    TORCH_CHECK(ql.numel() == B, "q_lens must have batch elements");
    p.q_lens = ql.data_ptr<int32_t>();
  }
  if (kv_lens.has_value()) {
    TORCH_CHECK(kv_lens->is_cuda() && kv_lens->device() == q.device(), "kv_lens must be on q's device");
    kl = kv_lens->to(torch::kInt).contiguous();
    TORCH_CHECK(kl.numel() == B, "kv_lens must have batch elements");
    p.kv_lens = kl.data_ptr<int32_t>();
  }
  if (lse.has_value()) {
    TORCH_CHECK(lse->scalar_type() == torch::kFloat && lse->is_contiguous() && lse->device() == q.device() &&
                    lse->dim() == 3 && lse->size(0) == B && lse->size(1) == H && lse->size(2) == Sq,
                "lse must be contiguous fp32 [batch, n_heads, max_q_len] on q's device");
    p.lse = lse->data_ptr<float>();
  }
  p.sm_scale = (float)sm_scale;
  p.causal = causal ? 1 : 0;
  p.sliding_window = (int32_t)sliding_window;
  p.logits_soft_cap = (float)logits_soft_cap;
  p.algo = algo_code(algo);
  p.kv_offset = (int32_t)kv_offset;
  p.kv_total = (int32_t)kv_total;
  size_t ws_bytes = 0;
  check_status(llmx_attn_workspace_size(&p, &ws_bytes));
  torch::Tensor ws;
  if (ws_bytes > 0) {
    ws = torch::empty({(int64_t)ws_bytes}, q.options().dtype(torch::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = ws_bytes;
  }
  check_status(llmx_attn_fwd(&p, at::cuda::getCurrentCUDAStream(q.device().index()).stream()));
}

// ---- 4-bit key/value cache (llmx_b200/kv4.py documents the arguments) -----

namespace {

// An optional per-sequence int32 argument on `dev`; the tensor is kept in `keep`.
const int32_t *int_arg(const char *name, const std::optional<torch::Tensor> &t, int64_t batch, torch::Device dev,
                       torch::Tensor &keep) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->is_cuda() && t->device() == dev, name, " must be on the cache's device");
  // The usual tensor is taken as it is: each conversion call costs a microsecond even when it has nothing to do.
  // Of 64 bits, what 32 do not hold becomes the nearest number that they do, not its low half.
  if (t->scalar_type() == torch::kInt) keep = t->is_contiguous() ? *t : t->contiguous();
  else if (t->scalar_type() == torch::kLong) keep = t->clamp((int64_t)INT32_MIN, (int64_t)INT32_MAX).to(torch::kInt).contiguous();
  else keep = t->to(torch::kInt).contiguous();
  TORCH_CHECK(keep.numel() == batch, name, " must have batch elements");
  return keep.data_ptr<int32_t>();
}

llmx_kv4_cache cache_arg(const torch::Tensor &cache, int64_t batch, const torch::Tensor &like, int64_t head_dim,
                         const std::optional<torch::Tensor> &block_table, torch::Tensor &keep) {
  TORCH_CHECK(cache.scalar_type() == torch::kByte && cache.dim() == 4,
              "kv4: cache must be uint8 [n_pages, n_kv_heads, page_size / 16, 18 * head_dim]");
  TORCH_CHECK(cache.is_cuda(), "kv4: cache must be a CUDA tensor");
  TORCH_CHECK(like.scalar_type() == torch::kHalf || like.scalar_type() == torch::kBFloat16,
              "kv4: only float16 and bfloat16 are supported");
  TORCH_CHECK(cache.size(3) == 18 * head_dim, "kv4: cache tiles must have 18 * head_dim = ", 18 * head_dim, " bytes");
  TORCH_CHECK(cache.stride(3) == 1 && (cache.size(2) == 1 || cache.stride(2) == cache.size(3)),
              "kv4: the tiles of a page must be contiguous");
  TORCH_CHECK(cache.size(0) <= INT32_MAX && cache.size(1) <= INT32_MAX && cache.size(2) <= INT32_MAX / 16,
              "kv4: cache dimensions must fit 31 bits");
  llmx_kv4_cache c{};
  c.dtype = llmx_dtype_of(like);
  c.n_kv_heads = (int32_t)cache.size(1);
  c.head_dim = (int32_t)head_dim;
  c.page_size = (int32_t)cache.size(2) * LLMX_KV4_TILE_TOKENS;
  c.n_pages = (int32_t)cache.size(0);
  c.data = cache.data_ptr();
  c.page_stride = cache.stride(0);
  c.head_stride = cache.stride(1);
  if (block_table.has_value()) {
    TORCH_CHECK(block_table->is_cuda() && block_table->device() == cache.device(),
                "kv4: block_table must be on the cache's device");
    TORCH_CHECK(block_table->scalar_type() == torch::kInt && block_table->dim() == 2 && block_table->size(0) == batch &&
                    block_table->size(1) >= 1 && block_table->size(1) <= INT32_MAX,
                "kv4: block_table must be int32 [batch, max_pages]");
    keep = block_table->stride(1) == 1 ? *block_table : block_table->contiguous();
    c.max_pages = (int32_t)keep.size(1);
    c.block_table = keep.data_ptr<int32_t>();
    c.table_stride = keep.stride(0);
  } else {
    TORCH_CHECK(batch == 0 || cache.size(0) >= batch, "kv4: without a block_table the cache needs a page per sequence");
    c.max_pages = (int32_t)(cache.size(0) / std::max<int64_t>(batch, 1));
  }
  return c;
}

void kv4_rows(bool store, const torch::Tensor &cache, torch::Tensor k, torch::Tensor v,
              const std::optional<torch::Tensor> &start, const std::optional<torch::Tensor> &lens,
              const std::optional<torch::Tensor> &block_table) {
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4, "kv4: k and v must be [batch, rows, n_kv_heads, head_dim]");
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
              "kv4: k and v must have the same shape and dtype");
  TORCH_CHECK(k.is_cuda() && v.is_cuda() && k.device() == v.device() && k.device() == cache.device(),
              "kv4: k, v and cache must be on one CUDA device");
  TORCH_CHECK(cache.dim() == 4 && k.size(2) == cache.size(1), "kv4: k and v must have the cache's n_kv_heads");
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX, "kv4: batch and rows must fit 31 bits");
  if (store) {
    if (k.stride(-1) != 1) k = k.contiguous();
    if (v.stride(-1) != 1) v = v.contiguous();
  }
  TORCH_CHECK(k.stride(-1) == 1 && v.stride(-1) == 1, "kv4: k and v must have a unit stride on head_dim");
  const c10::cuda::CUDAGuard guard(k.device());
  torch::Tensor keep_table, keep_start, keep_lens;
  const llmx_kv4_cache c = cache_arg(cache, k.size(0), k, k.size(3), block_table, keep_table);
  llmx_kv4_rows r{};
  r.batch = (int32_t)k.size(0);
  r.max_rows = (int32_t)k.size(1);
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  set_strides(r.k_stride, k, true);
  set_strides(r.v_stride, v, true);
  r.start = int_arg("start", start, k.size(0), k.device(), keep_start);
  r.lens = int_arg("lens", lens, k.size(0), k.device(), keep_lens);
  void *stream = at::cuda::getCurrentCUDAStream(k.device().index()).stream();
  check_status(store ? llmx_kv4_store(&c, &r, stream) : llmx_kv4_load(&c, &r, stream));
}

}  // namespace

void kv4_store(torch::Tensor cache, torch::Tensor k, torch::Tensor v, std::optional<torch::Tensor> start,
               std::optional<torch::Tensor> lens, std::optional<torch::Tensor> block_table) {
  kv4_rows(true, cache, k, v, start, lens, block_table);
}

void kv4_load(torch::Tensor cache, torch::Tensor k, torch::Tensor v, std::optional<torch::Tensor> start,
              std::optional<torch::Tensor> lens, std::optional<torch::Tensor> block_table) {
  kv4_rows(false, cache, k, v, start, lens, block_table);
}

void kv4_attention(torch::Tensor output, torch::Tensor q, torch::Tensor cache, double sm_scale, int64_t sliding_window,
                   double logits_soft_cap, std::optional<torch::Tensor> kv_lens,
                   std::optional<torch::Tensor> block_table, std::optional<torch::Tensor> q_lens,
                   std::optional<torch::Tensor> alibi_slopes, bool causal, std::optional<torch::Tensor> lse,
                   const std::string &algo, int64_t max_kv_len) {
  TORCH_CHECK(q.dim() == 4 && output.dim() == 4, "kv4: q must be [batch, q_len, n_heads, head_dim]");
  TORCH_CHECK(output.scalar_type() == q.scalar_type() && output.sizes() == q.sizes(),
              "output must have the shape and dtype of q");
  TORCH_CHECK(q.is_cuda() && output.is_cuda() && q.device() == output.device() && q.device() == cache.device(),
              "q, output and cache must be on one CUDA device");
  TORCH_CHECK(output.stride(-1) == 1, "output must have a unit stride on head_dim");
  if (q.stride(-1) != 1) q = q.contiguous();
  const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2), D = q.size(3);
  if (q.numel() == 0) return;
  TORCH_CHECK(B <= INT32_MAX && Sq <= INT32_MAX && H <= INT32_MAX, "kv4: the sizes of q must fit 31 bits");
  const c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor keep_table, ql, kl, slopes;
  const llmx_kv4_cache c = cache_arg(cache, B, q, D, block_table, keep_table);
  llmx_attn_params p;
  check_status(llmx_attn_params_init(&p));
  p.dtype = c.dtype;
  p.batch = (int32_t)B;
  p.n_heads = (int32_t)H;
  p.n_kv_heads = c.n_kv_heads;
  p.head_dim = (int32_t)D;
  p.max_q_len = (int32_t)Sq;
  const int64_t room = (int64_t)c.max_pages * c.page_size;
  TORCH_CHECK(max_kv_len <= room, "max_kv_len must be at most max_pages * page_size");
  p.max_kv_len = (int32_t)std::min<int64_t>(max_kv_len > 0 ? max_kv_len : room, INT32_MAX);
  p.q = q.data_ptr();
  p.o = output.data_ptr();
  set_strides(p.q_stride, q, true);
  set_strides(p.o_stride, output, true);
  p.q_lens = int_arg("q_lens", q_lens, B, q.device(), ql);
  p.kv_lens = int_arg("kv_lens", kv_lens, B, q.device(), kl);
  if (alibi_slopes.has_value()) {
    TORCH_CHECK(alibi_slopes->is_cuda() && alibi_slopes->device() == q.device(), "alibi_slopes must be on q's device");
    slopes = alibi_slopes->to(torch::kFloat).contiguous();
    TORCH_CHECK(slopes.numel() == H, "alibi_slopes must have n_heads elements");
    p.alibi_slopes = slopes.data_ptr<float>();
  }
  if (lse.has_value()) {
    TORCH_CHECK(lse->scalar_type() == torch::kFloat && lse->is_contiguous() && lse->device() == q.device() &&
                    lse->dim() == 3 && lse->size(0) == B && lse->size(1) == H && lse->size(2) == Sq,
                "lse must be contiguous fp32 [batch, n_heads, max_q_len] on q's device");
    p.lse = lse->data_ptr<float>();
  }
  p.sm_scale = (float)sm_scale;
  p.causal = causal ? 1 : 0;
  p.sliding_window = (int32_t)std::min<int64_t>(std::max<int64_t>(sliding_window, -1), INT32_MAX / 2);
  p.logits_soft_cap = (float)logits_soft_cap;
  p.algo = algo_code(algo);
  size_t ws_bytes = 0;
  check_status(llmx_kv4_attn_workspace_size(&p, &c, &ws_bytes));
  torch::Tensor ws;
  if (ws_bytes > 0) {
    ws = torch::empty({(int64_t)ws_bytes}, q.options().dtype(torch::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = ws_bytes;
  }
  check_status(llmx_kv4_attn_fwd(&p, &c, at::cuda::getCurrentCUDAStream(q.device().index()).stream()));
}

// ---- paged 16-bit key/value cache (llmx_b200/paged.py documents the arguments) -----

namespace {

const int32_t *paged_table(const char *name, const torch::Tensor &t, int64_t batch, torch::Device dev, torch::Tensor &keep) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, "paged: ", name, " must be on the cache's device");
  TORCH_CHECK(t.scalar_type() == torch::kInt && t.dim() == 2 && t.size(0) == batch && t.size(1) >= 1 && t.size(1) <= INT32_MAX,
              "paged: ", name, " must be int32 [batch, max_pages]");
  keep = t.stride(1) == 1 ? t : t.contiguous();
  return keep.data_ptr<int32_t>();
}

llmx_paged_cache paged_cache(const torch::Tensor &k, const torch::Tensor &v, int64_t batch,
                             const std::optional<torch::Tensor> &block_table,
                             const std::optional<torch::Tensor> &key_weights, torch::Tensor &keep) {
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes(),
              "paged: the cache must be two tensors [n_pages, n_kv_heads, page_size, head_dim]");
  TORCH_CHECK(k.is_cuda() && k.device() == v.device(), "paged: the cache must be on one CUDA device");
  TORCH_CHECK(k.scalar_type() == v.scalar_type() && (k.scalar_type() == torch::kHalf || k.scalar_type() == torch::kBFloat16),
              "paged: only float16 and bfloat16 are supported");
  TORCH_CHECK(k.stride(3) == 1 && v.stride(3) == 1, "paged: the cache must have a unit stride on head_dim");
  TORCH_CHECK(batch <= INT32_MAX, "paged: batch must fit 31 bits");
  for (int i = 0; i < 4; ++i) TORCH_CHECK(k.size(i) <= INT32_MAX, "paged: cache dimensions must fit 31 bits");
  llmx_paged_cache c{};
  c.dtype = llmx_dtype_of(k);
  c.n_pages = (int32_t)k.size(0);
  c.n_kv_heads = (int32_t)k.size(1);
  c.page_size = (int32_t)k.size(2);
  c.head_dim = (int32_t)k.size(3);
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  set_strides(c.k_stride, k, true);
  set_strides(c.v_stride, v, true);
  if (block_table.has_value()) {
    c.block_table = paged_table("block_table", *block_table, batch, k.device(), keep);
    c.max_pages = (int32_t)keep.size(1);
    c.table_stride = keep.stride(0);
  } else {
    TORCH_CHECK(batch == 0 || k.size(0) >= batch, "paged: without a block_table the cache needs a page per sequence");
    c.max_pages = (int32_t)(k.size(0) / std::max<int64_t>(batch, 1));
  }
  if (key_weights.has_value()) {
    const torch::Tensor &w = *key_weights;
    TORCH_CHECK(w.scalar_type() == torch::kFloat && w.dim() == 3 && w.size(0) == k.size(0) && w.size(1) == k.size(1) &&
                    w.size(2) == k.size(2) && w.device() == k.device() && w.stride(2) == 1,
                "paged: key_weights must be fp32 [n_pages, n_kv_heads, page_size] on the cache's device, unit stride on tokens");
    c.key_weights = w.data_ptr<float>();
    c.w_stride[0] = w.stride(0);
    c.w_stride[1] = w.stride(1);
  }
  return c;
}

}  // namespace

void paged_store(torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor k, torch::Tensor v,
                 std::optional<torch::Tensor> start, std::optional<torch::Tensor> lens,
                 std::optional<torch::Tensor> block_table) {
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(), "paged: k and v must be [batch, rows, n_kv_heads, head_dim]");
  TORCH_CHECK(k.scalar_type() == v.scalar_type() && k.scalar_type() == k_cache.scalar_type(),
              "paged: k and v must have the cache's dtype");
  TORCH_CHECK(k.device() == v.device() && k.device() == k_cache.device(), "paged: k, v and the cache must be on one CUDA device");
  TORCH_CHECK(k_cache.dim() == 4 && k.size(2) == k_cache.size(1) && k.size(3) == k_cache.size(3),
              "paged: k and v must have the cache's n_kv_heads and head_dim");
  TORCH_CHECK(k.size(1) <= INT32_MAX, "paged: rows must fit 31 bits");
  if (k.stride(-1) != 1) k = k.contiguous();
  if (v.stride(-1) != 1) v = v.contiguous();
  torch::Tensor keep_table, keep_start, keep_lens;
  const llmx_paged_cache c = paged_cache(k_cache, v_cache, k.size(0), block_table, std::nullopt, keep_table);
  const c10::cuda::CUDAGuard guard(k.device());
  llmx_kv4_rows r{};
  r.batch = (int32_t)k.size(0);
  r.max_rows = (int32_t)k.size(1);
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  set_strides(r.k_stride, k, true);
  set_strides(r.v_stride, v, true);
  r.start = int_arg("start", start, k.size(0), k.device(), keep_start);
  r.lens = int_arg("lens", lens, k.size(0), k.device(), keep_lens);
  check_status(llmx_paged_store(&c, &r, at::cuda::getCurrentCUDAStream(k.device().index()).stream()));
}

void paged_attention(torch::Tensor output, torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache, double sm_scale,
                     int64_t sliding_window, double logits_soft_cap, std::optional<torch::Tensor> kv_lens,
                     std::optional<torch::Tensor> block_table, std::optional<torch::Tensor> q_lens,
                     std::optional<torch::Tensor> alibi_slopes, bool causal, std::optional<torch::Tensor> lse,
                     std::optional<torch::Tensor> key_weights, double decay, const std::string &algo, int64_t max_kv_len) {
  TORCH_CHECK(q.dim() == 4 && output.dim() == 4, "paged: q must be [batch, q_len, n_heads, head_dim]");
  TORCH_CHECK(output.scalar_type() == q.scalar_type() && output.sizes() == q.sizes(),
              "output must have the shape and dtype of q");
  TORCH_CHECK(q.is_cuda() && output.is_cuda() && q.device() == output.device() && q.device() == k_cache.device(),
              "q, output and the cache must be on one CUDA device");
  TORCH_CHECK(output.stride(-1) == 1, "output must have a unit stride on head_dim");
  TORCH_CHECK(k_cache.dim() == 4 && q.scalar_type() == k_cache.scalar_type() && q.size(3) == k_cache.size(3),
              "paged: q must have the cache's dtype and head_dim");
  if (q.stride(-1) != 1) q = q.contiguous();
  const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2), D = q.size(3);
  if (q.numel() == 0) {
    TORCH_CHECK(!key_weights.has_value(), "paged: key_weights need query rows");
    return;
  }
  TORCH_CHECK(B <= INT32_MAX && Sq <= INT32_MAX && H <= INT32_MAX, "paged: the sizes of q must fit 31 bits");
  const c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor keep_table, ql, kl, slopes;
  const llmx_paged_cache c = paged_cache(k_cache, v_cache, B, block_table, key_weights, keep_table);
  llmx_attn_params p;
  check_status(llmx_attn_params_init(&p));
  p.dtype = c.dtype;
  p.batch = (int32_t)B;
  p.n_heads = (int32_t)H;
  p.n_kv_heads = c.n_kv_heads;
  p.head_dim = (int32_t)D;
  p.max_q_len = (int32_t)Sq;
  const int64_t room = (int64_t)c.max_pages * c.page_size;
  TORCH_CHECK(max_kv_len <= room, "max_kv_len must be at most max_pages * page_size");
  p.max_kv_len = (int32_t)std::min<int64_t>(max_kv_len > 0 ? max_kv_len : room, INT32_MAX);
  p.q = q.data_ptr();
  p.o = output.data_ptr();
  set_strides(p.q_stride, q, true);
  set_strides(p.o_stride, output, true);
  p.q_lens = int_arg("q_lens", q_lens, B, q.device(), ql);
  p.kv_lens = int_arg("kv_lens", kv_lens, B, q.device(), kl);
  if (alibi_slopes.has_value()) {
    TORCH_CHECK(alibi_slopes->is_cuda() && alibi_slopes->device() == q.device(), "alibi_slopes must be on q's device");
    slopes = alibi_slopes->to(torch::kFloat).contiguous();
    TORCH_CHECK(slopes.numel() == H, "alibi_slopes must have n_heads elements");
    p.alibi_slopes = slopes.data_ptr<float>();
  }
  if (lse.has_value()) {
    TORCH_CHECK(lse->scalar_type() == torch::kFloat && lse->is_contiguous() && lse->device() == q.device() &&
                    lse->dim() == 3 && lse->size(0) == B && lse->size(1) == H && lse->size(2) == Sq,
                "lse must be contiguous fp32 [batch, n_heads, max_q_len] on q's device");
    p.lse = lse->data_ptr<float>();
  }
  p.sm_scale = (float)sm_scale;
  p.causal = causal ? 1 : 0;
  p.sliding_window = (int32_t)std::min<int64_t>(std::max<int64_t>(sliding_window, -1), 1 << 30);
  p.logits_soft_cap = (float)logits_soft_cap;
  TORCH_CHECK(algo == "auto" || algo == "decode" || algo == "tcgen05", "paged: algo must be one of auto, decode, tcgen05");
  p.algo = algo_code(algo);
  size_t ws_bytes = 0;
  check_status(llmx_paged_attn_workspace_size(&p, &c, &ws_bytes));
  torch::Tensor ws;
  if (ws_bytes > 0) {
    ws = torch::empty({(int64_t)ws_bytes}, q.options().dtype(torch::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = ws_bytes;
  }
  check_status(llmx_paged_attn_fwd(&p, &c, (float)decay, at::cuda::getCurrentCUDAStream(q.device().index()).stream()));
}

std::tuple<torch::Tensor, torch::Tensor> paged_evict(torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor key_weights,
                                                     int64_t budget, torch::Tensor kv_lens,
                                                     std::optional<torch::Tensor> block_table, int64_t recent, int64_t sinks,
                                                     std::optional<torch::Tensor> out_table, std::optional<torch::Tensor> kept,
                                                     std::optional<torch::Tensor> new_lens, int64_t max_kv_len) {
  TORCH_CHECK(budget >= 1 && budget <= INT32_MAX && recent >= 0 && recent <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX,
              "paged: budget must be >= 1, recent and sinks >= 0");
  TORCH_CHECK(kv_lens.dim() == 1, "kv_lens must be [batch]");
  const int64_t B = kv_lens.size(0);
  torch::Tensor keep_table, keep_out, keep_lens;
  const llmx_paged_cache c = paged_cache(k_cache, v_cache, B, block_table, key_weights, keep_table);
  const torch::Device dev = k_cache.device();
  const c10::cuda::CUDAGuard guard(dev);
  const auto ints = torch::TensorOptions().dtype(torch::kInt).device(dev);
  const torch::Tensor out_kept = kept.has_value() ? *kept : torch::empty({B, k_cache.size(1), budget}, ints);
  const torch::Tensor out_lens = new_lens.has_value() ? *new_lens : torch::empty({B}, ints);
  TORCH_CHECK(out_kept.scalar_type() == torch::kInt && out_kept.dim() == 3 && out_kept.size(0) == B &&
                  out_kept.size(1) == k_cache.size(1) && out_kept.size(2) == budget && out_kept.is_contiguous() &&
                  out_kept.device() == dev,
              "paged: kept must be contiguous int32 [batch, n_kv_heads, budget] on the cache's device");
  TORCH_CHECK(out_lens.scalar_type() == torch::kInt && out_lens.dim() == 1 && out_lens.size(0) == B && out_lens.is_contiguous() &&
                  out_lens.device() == dev,
              "paged: new_lens must be contiguous int32 [batch] on the cache's device");
  llmx_paged_evict_params e{};
  const int64_t room = (int64_t)c.max_pages * c.page_size;
  TORCH_CHECK(max_kv_len <= room, "max_kv_len must be at most max_pages * page_size");
  e.batch = (int32_t)B;
  e.budget = (int32_t)budget;
  e.recent = (int32_t)recent;
  e.sinks = (int32_t)sinks;
  e.max_kv_len = (int32_t)std::min<int64_t>(max_kv_len > 0 ? max_kv_len : room, INT32_MAX);
  e.kv_lens = int_arg("kv_lens", kv_lens, B, dev, keep_lens);
  if (out_table.has_value()) {
    e.out_table = paged_table("out_table", *out_table, B, dev, keep_out);
    e.out_table_stride = keep_out.stride(0);
    e.out_pages = (int32_t)keep_out.size(1);
  }
  e.kept = out_kept.data_ptr<int32_t>();
  e.new_lens = out_lens.data_ptr<int32_t>();
  check_status(llmx_paged_evict(&c, &e, at::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {out_kept, out_lens};
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "llmx attention op on B200 (sm_100a): torch binding over libllmx_attn.so";
  static py::object error_cls = py::module_::import("llmx_b200._lib").attr("LlmxError");
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const StatusError &e) {
      py::object err = error_cls(e.status, e.message);
      PyErr_SetObject(error_cls.ptr(), err.ptr());
    }
  });
  m.def("single_mha_attention_half", &single_mha_attention_half, py::arg("output"), py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("sm_scale"), py::arg("sliding_window") = -1, py::arg("logits_soft_cap") = 0.0,
        py::kw_only(), py::arg("alibi_slopes") = py::none(), py::arg("causal") = true,
        py::arg("q_lens") = py::none(), py::arg("kv_lens") = py::none(), py::arg("lse") = py::none(),
        py::arg("algo") = "auto", py::arg("kv_offset") = 0, py::arg("kv_total") = 0);
  m.def("kv4_store", &kv4_store, py::arg("cache"), py::arg("k"), py::arg("v"), py::kw_only(),
        py::arg("start") = py::none(), py::arg("lens") = py::none(), py::arg("block_table") = py::none());
  m.def("kv4_load", &kv4_load, py::arg("cache"), py::arg("k"), py::arg("v"), py::kw_only(),
        py::arg("start") = py::none(), py::arg("lens") = py::none(), py::arg("block_table") = py::none());
  m.def("kv4_attention", &kv4_attention, py::arg("output"), py::arg("q"), py::arg("cache"), py::arg("sm_scale"),
        py::arg("sliding_window") = -1, py::arg("logits_soft_cap") = 0.0, py::kw_only(),
        py::arg("kv_lens") = py::none(), py::arg("block_table") = py::none(), py::arg("q_lens") = py::none(),
        py::arg("alibi_slopes") = py::none(), py::arg("causal") = true, py::arg("lse") = py::none(),
        py::arg("algo") = "auto", py::arg("max_kv_len") = 0);
  m.def("paged_store", &paged_store, py::arg("k_cache"), py::arg("v_cache"), py::arg("k"), py::arg("v"), py::kw_only(),
        py::arg("start") = py::none(), py::arg("lens") = py::none(), py::arg("block_table") = py::none());
  m.def("paged_attention", &paged_attention, py::arg("output"), py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("sm_scale"), py::arg("sliding_window") = -1, py::arg("logits_soft_cap") = 0.0, py::kw_only(),
        py::arg("kv_lens") = py::none(), py::arg("block_table") = py::none(), py::arg("q_lens") = py::none(),
        py::arg("alibi_slopes") = py::none(), py::arg("causal") = true, py::arg("lse") = py::none(),
        py::arg("key_weights") = py::none(), py::arg("decay") = 1.0, py::arg("algo") = "auto", py::arg("max_kv_len") = 0);
  m.def("paged_evict", &paged_evict, py::arg("k_cache"), py::arg("v_cache"), py::arg("key_weights"), py::arg("budget"),
        py::kw_only(), py::arg("kv_lens"), py::arg("block_table") = py::none(), py::arg("recent") = 0, py::arg("sinks") = 0,
        py::arg("out_table") = py::none(), py::arg("kept") = py::none(), py::arg("new_lens") = py::none(),
        py::arg("max_kv_len") = 0);
  m.def("abi_version", [] { return llmx_attn_abi_version(); });
}
