/*
 * llmx_attn.h -- C ABI of the B200 (sm_100a) attention forward engine.
 *
 * Plain pointers and sizes only; every entry point returns an llmx_status and
 * allocates nothing.  All device pointers must live on the CUDA device that is
 * current on the calling thread; work is enqueued on the caller's stream.
 *
 * Reference interfaces this ABI replaces (paths inside DucHUNG312/llmx):
 *   llmx_single_mha_attention   include/llmx/cuda/attention/attention_api.h:8-14
 *                               src/cuda/attention/attention_api.cpp:14-72
 *   MHAParams (+ normalize)     include/llmx/cuda/attention/params.h:7-51
 *   single_mha_attention_launcher
 *                               include/llmx/cuda/attention/device/single_mha_kernel.cuh:595-635
 * The reference signature is one causal sequence on stream 0; llmx_attn_fwd
 * adds the batch axis, a non-causal mode, per-sequence lengths (padding),
 * fp32, a caller stream, an optional log-sum-exp output and a caller-owned
 * workspace for split-KV decoding.
 */
#ifndef LLMX_ATTN_H
#define LLMX_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LLMX_ATTN_ABI_VERSION 3

#if defined(__GNUC__)
#define LLMX_API __attribute__((visibility("default")))
#else
#define LLMX_API
#endif

typedef enum llmx_status {
  LLMX_OK = 0,
  LLMX_ERR_INVALID_ARGUMENT = 1, /* bad shape, stride, pointer or value      */
  LLMX_ERR_UNSUPPORTED = 2,      /* valid request no kernel here implements  */
  LLMX_ERR_WORKSPACE_TOO_SMALL = 3,
  LLMX_ERR_CUDA = 4,             /* a CUDA runtime call or launch failed     */
  LLMX_ERR_TIMEOUT = 5,          /* a bounded device-side wait expired       */
  LLMX_ERR_NO_DEVICE = 6
} llmx_status;

/* Element types, numbered as llmx::ScalarType (include/llmx/tensor.h:19). */
typedef enum llmx_dtype { LLMX_FP32 = 0, LLMX_FP16 = 1, LLMX_BF16 = 2 } llmx_dtype;

/* Kernel selection.  AUTO picks per request; the others force one family and
 * fail with LLMX_ERR_UNSUPPORTED when it cannot run the request. */
typedef enum llmx_attn_algo {
  LLMX_ALGO_AUTO = 0,
  LLMX_ALGO_SIMT = 1,    /* fp32-accumulating CUDA-core kernel, every shape  */
  LLMX_ALGO_DECODE = 2,  /* split-KV decode, max_q_len == 1, fp16/bf16       */
  LLMX_ALGO_TCGEN05 = 3  /* TMA + tcgen05/TMEM prefill, fp16/bf16, D 64/128/256 */
} llmx_attn_algo;

/*
 * One attention forward over a padded batch.
 *   q, o : [batch, max_q_len,  n_heads,    head_dim]
 *   k, v : [batch, max_kv_len, n_kv_heads, head_dim]
 * given by element strides {batch, seq, head}; the head_dim stride is 1.
 * Sequence b uses its first q_lens[b] query rows and kv_lens[b] keys (NULL
 * means the max extent; device int32 arrays, values are clamped to
 * [0, max]).  Query row i of sequence b attends to key j when
 *   j < kv_len_b,
 *   causal:  j <= i + (kv_len_b - q_len_b)        (bottom-right, mask.h:54-63)
 *   window:  (i + kv_len_b - q_len_b) - j <= sliding_window  (mask.h:60,66)
 * Score = q.k * sm_scale, then tanh(s/cap)*cap if logits_soft_cap > 0
 * (params.h:35-50), then + alibi_slopes[h] * j (mask.h:75-77).
 * Query rows past q_len_b and rows that see no key are written as 0 (their
 * lse as -inf).  GQA: head h reads kv head h / (n_heads / n_kv_heads).
 * With kv_offset / kv_total (below) j is the key's global position.
 */
typedef struct llmx_attn_params {
  int32_t dtype;      /* llmx_dtype of q, k, v and o                    */
  int32_t batch;      /* >= 1                                            */
  int32_t n_heads;    /* >= 1                                            */
  int32_t n_kv_heads; /* >= 1, divides n_heads                           */
  int32_t head_dim;   /* 1..256                                          */
  int32_t max_q_len;  /* >= 1                                            */
  int32_t max_kv_len; /* >= 1                                            */
  int32_t algo;       /* llmx_attn_algo                                  */
  const void *q;
  const void *k;
  const void *v;
  void *o;
  int64_t q_stride[3]; /* elements: batch, seq, head                     */
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t o_stride[3];
  const int32_t *q_lens;      /* device [batch] or NULL                  */
  const int32_t *kv_lens;     /* device [batch] or NULL                  */
  const float *alibi_slopes;  /* device [n_heads] fp32 or NULL           */
  float sm_scale;
  int32_t causal;             /* 1 = causal (the reference's only mode)  */
  int32_t sliding_window;     /* < 0 disables                            */
  float logits_soft_cap;      /* <= 0 disables                           */
  float *lse;                 /* NULL or device [batch, n_heads, max_q_len] fp32 */
  void *workspace;            /* device scratch for split-KV partials    */
  size_t workspace_bytes;
  /* Key shards (a sequence's keys split across calls or GPUs): local key j
   * sits at global position kv_offset + j, and the causal / window diagonal
   * of query row i is i + (kv_total - q_len_b) (kv_total <= 0: the local
   * kv_len_b).  ALiBi uses the global position.  Both 0 for unsharded keys. */
  int32_t kv_offset;
  int32_t kv_total;
} llmx_attn_params;

/* Fills *p with defaults: contiguous-stride fields zero, causal = 1,
 * sliding_window = -1, logits_soft_cap = 0, algo = AUTO. */
LLMX_API llmx_status llmx_attn_params_init(llmx_attn_params *p);

/* Sets the four stride triples for contiguous [B, S, H, D] tensors. */
LLMX_API llmx_status llmx_attn_set_contiguous_strides(llmx_attn_params *p);

/* Workspace bytes llmx_attn_fwd wants for *p (0 when none).  A call given
 * less (or NULL) still runs, without splitting the KV axis. */
LLMX_API llmx_status llmx_attn_workspace_size(const llmx_attn_params *p, size_t *bytes);

/* Enqueues the forward on `stream` (a cudaStream_t; NULL = legacy stream).
 * Replaces llmx_single_mha_attention (attention_api.cpp:14-72) for batched,
 * padded and non-causal requests. */
LLMX_API llmx_status llmx_attn_fwd(const llmx_attn_params *p, void *stream);

/* The reference's entry point with plain pointers: one causal sequence,
 * q/o [q_len, n_heads, head_dim], k/v [kv_len, n_kv_heads, head_dim],
 * contiguous.  Same arguments and meaning as
 * llmx::llmx_single_mha_attention (attention_api.h:8-14) plus dtype, the
 * sizes the Tensor carried, and a stream. */
LLMX_API llmx_status llmx_single_mha_attention_c(void *output, const void *q, const void *k, const void *v,
                                        const float *alibi_slopes, int32_t dtype, int32_t q_len,
                                        int32_t kv_len, int32_t n_heads, int32_t n_kv_heads,
                                        int32_t head_dim, float sm_scale, int32_t sliding_window,
                                        float logits_soft_cap, void *stream);

/* Split-KV decode that allocates nothing, for callers that cannot allocate
 * device memory after start-up (a fixed memory budget reserved up front, or a
 * latency-critical loop that must not hit cudaMalloc's implicit device-wide
 * synchronisation) and so cannot pass a workspace.  No counterpart in the
 * reference.  Same request and results as llmx_attn_fwd on the decode path
 * (fp16/bf16, max_q_len == 1, head_dim 64/128/256); the split partials live
 * in one static device array of LLMX_DECODE_NOALLOC_SCRATCH_BYTES per GPU,
 * held by every GPU that loads the library until the process exits.
 *  - Requests needing more scratch than that are refused with
 *    LLMX_ERR_WORKSPACE_TOO_SMALL.  The need is n_splits * batch * n_heads *
 *    (head_dim + 1) * 4 bytes, where a split holds between 64 and 256 keys:
 *    256, halved (down to 64) while batch x kv-head units alone cannot give
 *    the GPU four waves of work, so small batches need up to four times the
 *    256-key figure.  llmx_attn_workspace_size returns the exact need for a
 *    request (the same plan); compare it with the constant below.
 *  - The first call on a device looks up the array's device address
 *    (cudaGetSymbolAddress, with that device current) and keeps it once the
 *    lookup succeeds; a failed lookup is retried on the next call.  Make
 *    that first call before any stream capture.  After cudaDeviceReset the
 *    kept address is stale: do not call this entry point again in that
 *    process.
 *  - All calls on a device share the array: calls that overlap on the GPU
 *    (different streams, or concurrent host threads) race and corrupt each
 *    other's results.  p->workspace is ignored.
 *  - Calls no cudaMalloc, cudaFree or other allocating routine. */
#define LLMX_DECODE_NOALLOC_SCRATCH_BYTES (32u << 20)
LLMX_API llmx_status llmx_attn_decode_noalloc(const llmx_attn_params *p, void *stream);

/* Log-sum-exp merge of attention partials over disjoint key sets (a
 * sequence's keys split across calls or GPUs).  No counterpart in the
 * reference (it has no key splitting); the algebra is its online-softmax
 * rescale (softmax.h:53-110) applied across shards:
 *   m = max_c lse_c,  w_c = exp(lse_c - m),  O = sum_c w_c O_c / sum_c w_c,
 *   lse = m + log(sum_c w_c).
 * Part c covers output rows [row_lo, row_hi) of every (batch, head); for
 * output row s in that range its O element (b, s, h, d) is at
 *   o[b*o_stride[0] + (s - row_lo)*o_stride[1] + h*o_stride[2] + d]
 * and its natural-log lse (-inf: the part saw no key) at
 *   lse[b*lse_stride[0] + h*lse_stride[1] + (s - row_lo)].
 * Rows outside a part's range get no term from it, and a part's O is not
 * read where its lse is -inf, so those rows may hold anything.  Output:
 * out [batch, seq, n_heads, head_dim] with element strides out_stride
 * (batch, seq, head; multiples of 8), in the partials' dtype (fp16/bf16),
 * 0 where no part saw a key; lse_out (NULL or contiguous fp32
 * [batch, n_heads, seq]) = -inf there.  n_parts <= 16; head_dim a
 * multiple of 8; O pointers and strides 16-byte aligned. */
typedef struct llmx_merge_part {
  const void *o;
  const float *lse;
  int64_t o_stride[3];   /* elements: batch, row, head */
  int64_t lse_stride[2]; /* elements: batch, head      */
  int32_t row_lo, row_hi;
} llmx_merge_part;

LLMX_API llmx_status llmx_attn_lse_merge(int32_t n_parts, const llmx_merge_part *parts, int32_t dtype,
                                         int32_t batch, int32_t seq, int32_t n_heads, int32_t head_dim, void *out,
                                         const int64_t *out_stride, float *lse_out, void *stream);

/* Row-scattered partial output: the tensor-core prefill writes query row R
 * (global row row_base + local row) of its partial O and lse into
 * destination p = R / slice_rows, at row R - p * slice_rows of
 *   o[p]   : [batch, slice_rows, n_heads, head_dim] in the input dtype
 *   lse[p] : [batch, n_heads, slice_rows] fp32 (natural log)
 * instead of p->o / p->lse.  The pointers may be another GPU's memory mapped
 * into this process (llmx_ipc_open): a rank of a KV split then delivers each
 * row of its partial straight to the rank that merges that row, while the
 * kernel runs, and every thread fences its writes system-wide before it
 * exits, so a cross-GPU barrier after the launch (an NCCL all-reduce on the
 * same stream) orders them before the owner's merge.  No counterpart in the
 * reference (it has no key splitting).  n_dst <= 8; slice_rows and row_base
 * multiples of 16; every row the launch computes (row_base .. row_base +
 * max_q_len - 1) must fall in a destination; pointers 16-byte aligned. */
#define LLMX_SCATTER_MAX_DST 8
typedef struct llmx_row_scatter {
  int32_t n_dst;
  int32_t slice_rows;
  int32_t row_base;
  int32_t reserved;
  void *o[LLMX_SCATTER_MAX_DST];
  float *lse[LLMX_SCATTER_MAX_DST];
} llmx_row_scatter;

/* llmx_attn_fwd with the output rows scattered as *x describes (p->o and
 * p->lse are ignored).  Runs only on the tensor-core prefill (fp16/bf16,
 * head_dim 64/128); LLMX_ERR_UNSUPPORTED otherwise. */
LLMX_API llmx_status llmx_attn_fwd_scatter(const llmx_attn_params *p, const llmx_row_scatter *x, void *stream);

/* Device buffers shared between the GPUs of one node (one process per GPU)
 * through CUDA IPC, for llmx_attn_fwd_scatter's destinations.  Set-up only,
 * not for the per-call path: llmx_ipc_alloc allocates `bytes` of device
 * memory on the current device (zeroed) and writes its 64-byte IPC handle;
 * another process opens it with llmx_ipc_open (on its own current device, with
 * peer access enabled as needed) and gets a pointer it can store to;
 * llmx_ipc_close unmaps an opened pointer; llmx_ipc_free frees a buffer this
 * process allocated (after every peer has closed it).  Both accept NULL and
 * then do nothing. */
#define LLMX_IPC_HANDLE_BYTES 64
LLMX_API llmx_status llmx_ipc_alloc(size_t bytes, void **ptr, void *handle);
LLMX_API llmx_status llmx_ipc_open(const void *handle, void **ptr);
LLMX_API llmx_status llmx_ipc_close(void *ptr);
LLMX_API llmx_status llmx_ipc_free(void *ptr);

/* Element-type conversion of n contiguous elements between fp32, fp16 and
 * bf16 (round to nearest even), enqueued on `stream`.  Replaces the
 * reference's llmx_copy(ScalarType, ScalarType, ...) (src/tensor.cpp:108-118)
 * and the launch_scalar_convert kernels behind it (src/scalar.cu:33-62),
 * which back the to_fp32 / to_fp16 / to_bf16 ops (include/llmx/ops.h:25-74,
 * 215-229).  fp16 <-> bf16 goes through fp32 as in scalar.cu:6-31.  When the
 * two types match the elements are copied (the reference's same-type
 * converter leaves the output unwritten, include/llmx/scalar.h:13-15).
 * Any pointer alignment is accepted; 16-byte aligned buffers take the
 * vector path. */
LLMX_API llmx_status llmx_convert(const void *src, int32_t src_dtype, void *dst, int32_t dst_dtype, size_t n,
                                  void *stream);

/* ------------------------------------------------------------------------
 * Key/value cache held in 4 bits.  No counterpart in the reference (it has
 * no cache).  K and V (fp16 / bf16, head_dim 64, 128 or 256) are quantised
 * in groups of LLMX_KV4_GROUP channels of one (token, kv head), each with a
 * step s and a minimum m held in the type T of K and V:
 *   m = min x,  r = fl32(fl32(max x - m) / 15),  s = the smallest T >= r
 *   (the next one below where 15 s + m would round to infinity in T),
 *   n = min(15, rint(fl32(fl32(x - m) / s)))  (0 where s = 0),
 *   value = n s + m, within s / 2 of x; finite x read back finite.
 * A group with a NaN or an infinity in it (or, for bf16, a range max x - m
 * past fp32) has s = NaN and reads back as NaN.  4.5 bits a value:
 * 18 * head_dim bytes per 16 tokens of K and V of one kv head.
 *
 * The cache is made of pages of page_size tokens (a multiple of 16).  Page p,
 * kv head h starts at data + p * page_stride + h * head_stride and holds
 * page_size / 16 tiles of 18 * head_dim bytes, one after the other.  A tile is
 * [K codes, 8 * head_dim][V codes, 8 * head_dim][parameters, 2 * head_dim].
 * Codes are 32-bit words of 8 consecutive channels, channel c of the word in
 * bits 4c .. 4c + 3.  Word x of lane (g, t) (g < 8, t < 4) lies at byte
 * (x / 4) * 512 + (4 g + t) * 16 + (x % 4) * 4 of its section, where with
 * G = head_dim / 64
 *   K: x = (r * G + h) * 2 + w     token 8 r + g, channels 64 h + 16 t + 8 w ..
 *   V: x = (2 a + c) * G + h       token 8 a + 2 t + c, channels 64 h + 8 g ..
 * which is the order of the matrix fragments that the attention kernel feeds
 * to the tensor cores, so a tile is read with whole 16-byte loads.  The
 * parameters are [16 tokens][K, V][G][s, m] in T.
 *
 * Token j of sequence b lies in page block_table[b * table_stride + j /
 * page_size] (NULL: page b * max_pages + j / page_size).  Entries that hold
 * no token of the sequence are not read.  An entry outside [0, n_pages), or a
 * position outside [0, max_pages * page_size), is skipped, never followed: a
 * store drops those rows, a load writes 0 for them, the attention does not
 * see them (its expanded form takes them as the load's zeros), and
 * llmx_attn_device_status then returns LLMX_ERR_INVALID_ARGUMENT.  Two rows stored to the same place by one call
 * leave an undefined mix of both there. */
#define LLMX_KV4_GROUP 64
#define LLMX_KV4_TILE_TOKENS 16
typedef struct llmx_kv4_cache {
  int32_t dtype;      /* llmx_dtype of K and V: fp16 or bf16              */
  int32_t n_kv_heads; /* >= 1                                             */
  int32_t head_dim;   /* 64, 128 or 256                                   */
  int32_t page_size;  /* tokens, a multiple of 16                         */
  int32_t n_pages;    /* >= 1                                             */
  int32_t max_pages;  /* pages of one sequence (columns of block_table);
                         max_pages * page_size <= 2^30                    */
  void *data;         /* device, 16-byte aligned                          */
  int64_t page_stride; /* bytes, multiples of 16                          */
  int64_t head_stride;
  const int32_t *block_table; /* device [batch, max_pages] or NULL        */
  int64_t table_stride;       /* elements between its rows                */
} llmx_kv4_cache;

/* Rows of K and V outside the cache: [batch, max_rows, n_kv_heads, head_dim]
 * by element strides {batch, row, head}, unit stride on head_dim.  Row i <
 * lens[b] (NULL: max_rows; clamped to [0, max_rows]) is token start[b] + i
 * (NULL: i) of sequence b. */
typedef struct llmx_kv4_rows {
  int32_t batch;
  int32_t max_rows;
  void *k;
  void *v;
  int64_t k_stride[3];
  int64_t v_stride[3];
  const int32_t *start; /* device [batch] or NULL                         */
  const int32_t *lens;  /* device [batch] or NULL                         */
} llmx_kv4_rows;

/* Bytes of one page of one kv head (the least head_stride). */
LLMX_API llmx_status llmx_kv4_page_bytes(int32_t head_dim, int32_t page_size, int64_t *bytes);

/* Quantises the rows of K and V into the cache (a prompt's, or one new token's
 * per sequence).  Nothing else of the cache changes. */
LLMX_API llmx_status llmx_kv4_store(const llmx_kv4_cache *c, const llmx_kv4_rows *rows, void *stream);

/* Reads rows of the cache back (n s + m in fp32, rounded to T) into k and v;
 * rows at or past lens[b] are written as 0. */
LLMX_API llmx_status llmx_kv4_load(const llmx_kv4_cache *c, const llmx_kv4_rows *rows, void *stream);

/* llmx_attn_fwd over the cache instead of dense K / V: same request, masks
 * and results (p->k, p->v and their strides are ignored; p->dtype, n_kv_heads
 * and head_dim must match the cache; p->max_kv_len <= max_pages * page_size
 * bounds kv_lens; kv_offset / kv_total must be 0).  p->algo:
 *   DECODE  reads the 4-bit tiles directly, in one pass per 8 (head, query
 *           row) pairs of a kv head; any max_q_len, any q / o alignment.  The
 *           values n s + m are used unrounded; q is used in 16 bits of its
 *           row's largest element (steps of 1/32512), p s in fp16.
 *   TCGEN05 expands the sequences into the workspace (values rounded to T)
 *           and runs the tensor-core prefill on them; needs its workspace.
 *           ALiBi adds slope * position in fp32, as llmx_attn_fwd does (DECODE:
 *           the distance from the row's largest bias).
 *   AUTO    DECODE, or for long query blocks TCGEN05 where it can run, is
 *           expected to be faster, takes at most 4 GiB and has its workspace.
 *           (Query blocks that DECODE cannot count take TCGEN05 in any case,
 *           and fail without its workspace.)
 * A call on the DECODE path given too little workspace runs without
 * splitting a sequence's keys.  Calls that share a workspace must not overlap
 * on the GPU.  A NaN reaches the rows that see it and no others: one in K makes
 * the row NaN, one in V the channels of its group (TCGEN05: the row and its lse
 * as well), and an infinity or NaN in q its row (TCGEN05 with a soft-cap takes
 * the infinite scores as +- the cap).  A row's p s keeps
 * 11 bits down to 2^-21 of its largest, by the largest p and the largest V step
 * that the row sees, and p itself in sums and lse down to 2^-48; a bf16 K is
 * taken up to 2^96 in size. */
LLMX_API llmx_status llmx_kv4_attn_workspace_size(const llmx_attn_params *p, const llmx_kv4_cache *c, size_t *bytes);
LLMX_API llmx_status llmx_kv4_attn_fwd(const llmx_attn_params *p, const llmx_kv4_cache *c, void *stream);

/* ------------------------------------------------------------------------
 * Paged key/value cache in 16 bits.  No counterpart in the reference (it has
 * no cache).  K and V (fp16 / bf16, head_dim 64, 128 or 256) lie in pages of
 * page_size tokens (a multiple of 16), each with its own element strides
 * {page, kv head, token} and unit stride on head_dim; strides are multiples
 * of 8 and pointers 16-byte aligned, and no two elements may share a place.
 * Token j of sequence b lies in page block_table[b * table_stride + j /
 * page_size] (NULL: page b * max_pages + j / page_size).  Entries that hold
 * no token of a sequence are not read, and neither is what a page holds
 * behind a sequence's length.  An entry outside [0, n_pages), or a position
 * outside [0, max_pages * page_size), is never followed: rows there are not
 * written and read as zeros, and llmx_attn_device_status then returns
 * LLMX_ERR_INVALID_ARGUMENT.
 *   key_weights (NULL or device fp32, element strides {page, kv head}, unit
 * stride on the token; 16-byte aligned, strides multiples of 4) has a weight
 * for every cached (token, kv head), in the same pages. */
typedef struct llmx_paged_cache {
  int32_t dtype;      /* llmx_dtype of K and V: fp16 or bf16              */
  int32_t n_kv_heads; /* >= 1                                             */
  int32_t head_dim;   /* 64, 128 or 256                                   */
  int32_t page_size;  /* tokens, a multiple of 16                         */
  int32_t n_pages;    /* >= 1                                             */
  int32_t max_pages;  /* pages of one sequence (columns of block_table);
                         max_pages * page_size <= 2^30                    */
  void *k;
  void *v;
  int64_t k_stride[3]; /* elements: page, kv head, token                  */
  int64_t v_stride[3];
  const int32_t *block_table; /* device [batch, max_pages] or NULL        */
  int64_t table_stride;       /* elements between its rows                */
  float *key_weights;
  int64_t w_stride[2]; /* elements: page, kv head                         */
} llmx_paged_cache;

/* Copies the rows of K and V (the same description of rows as the 4-bit
 * cache's) into the cache: row i < lens[b] becomes token start[b] + i of
 * sequence b.  Nothing else of the cache changes.  Two rows stored to the
 * same place by one call leave an undefined mix of both there. */
LLMX_API llmx_status llmx_paged_store(const llmx_paged_cache *c, const llmx_kv4_rows *rows, void *stream);

/* llmx_attn_fwd over the cache instead of dense K / V: same request, masks
 * and results (p->k, p->v and their strides are ignored; p->dtype, n_kv_heads
 * and head_dim must match the cache; p->max_kv_len <= max_pages * page_size
 * bounds kv_lens; kv_offset / kv_total must be 0; q and o rows 16-byte
 * aligned).  Any max_q_len: one new token a sequence, a few, or a chunk of a
 * prompt; a sequence's query rows are its last q_len tokens under the causal
 * mask.  p->algo:
 *   DECODE  streams K and V once for every 16 or 32 (head_dim 256: or 64)
 *           (query row, head) pairs of a kv head, split over the machine.
 *   TCGEN05 tiles of 128 such pairs; sm_scale > 0, at most 128 query heads a
 *           kv head.
 *   AUTO    DECODE up to 32 pairs, TCGEN05 above where it can run.
 * ALiBi's biases count from each row's largest one, so that they keep their
 * bits far into a sequence; lse is that of slope * position.  A NaN or an
 * infinity in a cached token reaches the rows that see the token and no
 * others; one in V may make such a row of o NaN as a whole, and shows in
 * neither lse nor key weights.  bf16 values of V are to stay below
 * 2^64 / kv_len: their weighted sums are kept in fp32, before the division,
 * with weights of up to 2^64.  A soft-capped score is right to 2^-20 of itself.
 *   With c->key_weights, the weight of every token j < kv_lens[b] of every kv
 * head becomes
 *   decay * (what was there) + sum of softmax(row)[j] over the query rows and
 *                              the query heads of the kv head,
 * where what was there counts as 0 for the call's own tokens (causal: the
 * last q_lens[b] ones), and for all where decay is 0 (it is not read then).
 * decay must be finite and >= 0.  o must then not overlap q, and sequences that
 * share a page leave either's weights there.
 *   A call given too little workspace for its partial results runs without
 * splitting sequences; with key_weights it is refused
 * (LLMX_ERR_WORKSPACE_TOO_SMALL).  The workspace then also holds the scores of
 * calls with up to 32 (row, head) pairs a kv head, up to 1 GiB, and of calls
 * with more than 128 query heads a kv head or a q of stride 0, where more than
 * 16 GiB are refused (LLMX_ERR_UNSUPPORTED).  Calls that share a workspace must
 * not overlap on the GPU. */
LLMX_API llmx_status llmx_paged_attn_workspace_size(const llmx_attn_params *p, const llmx_paged_cache *c,
                                                    size_t *bytes);
LLMX_API llmx_status llmx_paged_attn_fwd(const llmx_attn_params *p, const llmx_paged_cache *c, float decay,
                                         void *stream);

/* Eviction by weight.  Of each sequence b and kv head the n = min(kv_lens[b],
 * budget) tokens are kept that are
 *   the first `sinks`, the last `recent`, and of the others those of the
 *   largest key_weights (of equal ones the earliest; a NaN counts as -inf),
 * in their order.  (A token whose page lies outside the cache ranks as -inf
 * and, if kept, becomes zeros with weight 0.)  Their rows of K, V and
 * key_weights become tokens 0 .. n - 1 of the pages of out_table[b] (NULL: of
 * the sequence's own pages, in place; sequences must then share no page).  With
 * an out_table its pages must hold no token that the call reads, and share none
 * with one another.  kept [batch, n_kv_heads, budget] gets their former
 * positions (-1 behind n), new_lens[b] = n; it may be kv_lens itself.  Nothing
 * else of the cache changes.  No workspace. */
typedef struct llmx_paged_evict_params {
  int32_t batch;
  int32_t budget;            /* >= 1, >= sinks + recent                   */
  int32_t recent;            /* >= 0                                      */
  int32_t sinks;             /* >= 0                                      */
  int32_t max_kv_len;        /* bounds kv_lens; <= max_pages * page_size  */
  int32_t out_pages;         /* columns of out_table                      */
  const int32_t *kv_lens;    /* device [batch]                            */
  const int32_t *out_table;  /* device [batch, out_pages] or NULL         */
  int64_t out_table_stride;  /* elements between its rows                 */
  int32_t *kept;             /* device [batch, n_kv_heads, budget]        */
  int32_t *new_lens;         /* device [batch]                            */
} llmx_paged_evict_params;

LLMX_API llmx_status llmx_paged_evict(const llmx_paged_cache *c, const llmx_paged_evict_params *e, void *stream);

/* Which kernel family llmx_attn_fwd would run for *p (an llmx_attn_algo). */
LLMX_API llmx_status llmx_attn_select_algo(const llmx_attn_params *p, int32_t *algo);

/* Synchronises `device` and reads (and optionally clears) its device-side
 * error word: LLMX_ERR_TIMEOUT if any kernel gave up on a bounded wait,
 * LLMX_ERR_INVALID_ARGUMENT if a cache was given a page or position outside
 * it. */
LLMX_API llmx_status llmx_attn_device_status(int32_t device, int32_t clear);

LLMX_API const char *llmx_status_string(llmx_status s);
/* Message of the last failing call on this thread ("" if none). */
LLMX_API const char *llmx_attn_last_error(void);
LLMX_API int32_t llmx_attn_abi_version(void);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* LLMX_ATTN_H */
