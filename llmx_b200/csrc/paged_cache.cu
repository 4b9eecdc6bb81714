// Paged 16-bit key/value cache: storing rows, and eviction of the tokens with
// the least weight.  No counterpart in the reference (it has no cache); the
// layout and the rules are in include/llmx_attn.h.
//
// Store: a copy, bound by HBM on prompts (8 x 2048 rows, 32 heads of 128: 86 us,
// 6.2 TB/s) and by its launch on single tokens (64 rows: 4.6 us).
//
// Eviction, two launches:
//   select   a cluster of CTAs per (sequence, kv head) finds the k-th largest
//            weight by radix (four rounds of 8 bits over the order-preserving
//            image of the fp32 weights, held in shared memory after one read)
//            and writes the kept positions in ascending order;
//   compact  moves the kept rows of K, V and the weights to the front.
// 32 sequences of 2500-4096 tokens to 1024, 8 heads of 128: 65 us, 0.64 of the copy
// rate (in place 102); one of 131071 to 16384: 53 us (in place 121), 24 of it the
// selection's rounds.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "paged_attn.cuh"

namespace llmx_b200 {
namespace {

namespace cg = cooperative_groups;

llmx_status bad(const char *msg) { return record_error(LLMX_ERR_INVALID_ARGUMENT, msg); }
bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether elements at i * s[0] + j * s[1] + k * s[2] + l (l < inner) are all
// different, for strides that nest (each one spans what lies inside it).
bool nested(const long long *s, const long long *n, int dims, long long inner) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + dims, [&](int x, int y) { return s[x] < s[y]; });
  long long span = inner;
  for (int i = 0; i < dims; ++i) {
    const int d = order[i];
    if (n[d] <= 1) continue;
    if (s[d] < span) return false;
    span = s[d] * (n[d] - 1) + span;
  }
  return true;
}

// ------------------------------------------------------------------- store
struct StoreArgs {
  const void *k, *v;
  long long ks[3], vs[3];  // batch, row, head
  const int *start, *lens;
  int B, rows;
};

constexpr int kStoreThreads = 256;

// A CTA copies `tokens` rows of one sequence, K and V: their places are looked up
// once, then a thread moves 16-byte pieces (VEC; single elements where rows are
// not 16-byte aligned) of the rows' [head][channel] order, so that dense rows are
// read and pages written in whole lines; kUnroll of K and of V in flight a thread.
constexpr int kStoreTokens = 64;  // of a CTA, at most
template <bool VEC>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const PagedArgs a, const StoreArgs r, int tokens) {
  constexpr int kUnroll = 4;
  using Piece = typename std::conditional<VEC, uint4, uint16_t>::type;
  constexpr int kPer = sizeof(Piece) / 2;
  __shared__ int2 place[kStoreTokens];  // page (-1: none) and row
  const int per_head = a.D / kPer;
  const int log_per_head = 31 - __clz(per_head);  // D is a power of two
  const int pieces = a.Hkv * per_head;
  for (int b = blockIdx.y; b < r.B; b += gridDim.y) {
    const int n = clamp_len(r.lens, b, r.rows);
    const long long from = (long long)blockIdx.x * tokens;  // rows may end at 2^31 - 1
    if (from >= n) continue;
    const int lo = (int)from, hi = lo + min(n - lo, tokens);
    const long long first = r.start != nullptr ? r.start[b] : 0;
    __syncthreads();  // the places of the sequence before have been read
    if (threadIdx.x < hi - lo) {
      const long long j = first + lo + (int)threadIdx.x;
      int2 p = make_int2(-1, 0);
      if (j >= 0 && j <= INT_MAX) {
        const int slot = (int)j / a.page_size;
        p = make_int2(paged_page(a, b, slot), (int)j - slot * a.page_size);
      } else {
        raise_error(a.err, kDevErrBadPage);
      }
      place[threadIdx.x] = p;
    }
    __syncthreads();
    // Pieces of the CTA's tokens in the order token, head, chunk; tokens * pieces
    // is at most 2^31 - 1 (launch_store).
    const int total = (hi - lo) * pieces;
    int t = threadIdx.x / pieces, p = threadIdx.x - t * pieces;  // of this thread's next piece
    const int dt = kStoreThreads / pieces, dp = kStoreThreads - dt * pieces;  // and how far the one after it is
    for (int base = threadIdx.x; base < total; base += kStoreThreads * kUnroll) {
      Piece x[kUnroll], y[kUnroll];
      long long kd[kUnroll], vd[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        kd[u] = -1;
        if (base + u * kStoreThreads < total) {
          const int h = p >> log_per_head, c = (p & (per_head - 1)) * kPer;
          const int2 at = place[t];
          if (at.x >= 0) {
            kd[u] = at.x * a.ks[0] + h * a.ks[1] + at.y * a.ks[2] + c;
            vd[u] = at.x * a.vs[0] + h * a.vs[1] + at.y * a.vs[2] + c;
            const long long row = (long long)lo + t;
            x[u] = *reinterpret_cast<const Piece *>(static_cast<const uint16_t *>(r.k) + b * r.ks[0] + row * r.ks[1] +
                                                    h * r.ks[2] + c);
            y[u] = *reinterpret_cast<const Piece *>(static_cast<const uint16_t *>(r.v) + b * r.vs[0] + row * r.vs[1] +
                                                    h * r.vs[2] + c);
          }
        }
        t += dt;
        p += dp;
        if (p >= pieces) {
          p -= pieces;
          ++t;
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (kd[u] >= 0) {
          *reinterpret_cast<Piece *>(static_cast<uint16_t *>(a.k) + kd[u]) = x[u];
          *reinterpret_cast<Piece *>(static_cast<uint16_t *>(a.v) + vd[u]) = y[u];
        }
    }
  }
}

cudaError_t launch_store(const PagedArgs &a, const StoreArgs &r, bool vec, cudaStream_t s) {
  const long long pieces = (long long)a.Hkv * a.D / (vec ? 8 : 1);
  // One round of kUnroll pieces a thread, and at least one token.
  const int tokens = (int)std::max<long long>(1, std::min<long long>(std::min(r.rows, kStoreTokens), kStoreThreads * 4 / pieces));
  const dim3 grid((unsigned)(((long long)r.rows + tokens - 1) / tokens), std::min(r.B, 65535));
  if (vec)
    paged_store_kernel<true><<<grid, kStoreThreads, 0, s>>>(a, r, tokens);
  else
    paged_store_kernel<false><<<grid, kStoreThreads, 0, s>>>(a, r, tokens);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- eviction
struct EvictArgs {
  int B, budget, recent, sinks, max_kv;
  const int *kv_lens;
  const int *out_table;  // nullable: in place
  long long out_stride;
  int out_pages;
  int *kept, *new_lens;
};

// Weights of a CTA held in shared memory; more are read again in each round (one sequence
// of 131072 tokens, all held by its eight CTAs, to 16384: 57 us; of 262144, half held: 117 us).
constexpr int kSelHeld = 16384;

// The image of a weight under which unsigned order is the order of the
// weights: the sign bit flipped, or all bits of negative ones.  -0 counts as 0
// and a NaN as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -CUDART_INF_F;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct alignas(16) SelShared {
  uint4 hist[2][256];  // four copies, a lane's is lane % 4: few digits are hot
  uint32_t sum[2][256];  // of the copies, read by the cluster's other CTAs
  uint32_t warp_gt[32], warp_eq[32];
  uint32_t gt, eq;              // this CTA's counts, read by the others
  uint32_t digit, need, taken;  // a round's result
};

// Cluster `g` of CTAs handles (sequence, kv head) g; CTA `rank` of it an equal
// part of the positions, of which sinks .. L - recent - 1 are candidates.
// 1024 threads where a unit has several CTAs (few units), else 512.
template <int kSelThreads>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const PagedArgs a, const EvictArgs e) {
  constexpr int kSelWarps = kSelThreads / 32;
  extern __shared__ __align__(16) uint32_t held[];
  __shared__ SelShared sh;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  const int unit = blockIdx.x / ranks;
  const int b = unit / a.Hkv, h = unit % a.Hkv;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int L = clamp_len(e.kv_lens, b, e.max_kv);
  const int n = min(L, e.budget);
  int *kept = e.kept + ((long long)b * a.Hkv + h) * e.budget;
  const int at = rank * kSelThreads + tid, all = ranks * kSelThreads;
  for (unsigned i = n + at; i < (unsigned)e.budget; i += all) kept[i] = -1;  // budget may be 2^31 - 1: i does not wrap
  if (L <= e.budget) {  // the same in all CTAs of the cluster
    for (int i = at; i < n; i += all) kept[i] = i;
    return;
  }
  for (int i = at; i < e.sinks; i += all) kept[i] = i;
  for (int i = at; i < e.recent; i += all) kept[n - e.recent + i] = L - e.recent + i;
  const uint32_t want = n - e.sinks - e.recent;  // of the candidates; fewer than there are
  if (want == 0) return;

  // This CTA's positions [j0, j0 + mine); what is no candidate has the image 0,
  // below that of every weight, and is never needed.
  const int per = ((L + ranks - 1) / ranks + 3) & ~3;
  const int j0 = min(L, rank * per), mine = min(L, j0 + per) - j0;
  const int first = e.sinks - j0, last = L - e.recent - j0;  // candidates, from j0
  auto read = [&](int i) {
    if (i < first || i >= last) return 0u;
    const int j = j0 + i;
    const int page = paged_page(a, b, j / a.page_size);
    return weight_key(page < 0 ? CUDART_NAN_F : a.w[page * a.ws[0] + h * a.ws[1] + j % a.page_size]);
  };
  {
    // Four weights a load (pages hold a multiple of 16), four loads in flight.
    const int n_held = min(mine, kSelHeld);
    for (int base = tid * 4; base < n_held; base += kSelThreads * 16) {
      float4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + base + u * kSelThreads * 4;
        w[u] = make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F);
        if (j - j0 < n_held) {
          const int slot = j / a.page_size;
          const int page = paged_page(a, b, slot);
          if (page >= 0)
            w[u] = *reinterpret_cast<const float4 *>(a.w + page * a.ws[0] + h * a.ws[1] + (j - slot * a.page_size));
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = base + u * kSelThreads * 4;
        if (at < n_held) {
          const float x[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
          uint32_t k[4];
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4) k[e4] = at + e4 >= first && at + e4 < last ? weight_key(x[e4]) : 0u;
          *reinterpret_cast<uint4 *>(held + at) = make_uint4(k[0], k[1], k[2], k[3]);
        }
      }
    }
  }
  // The images of positions i .. i + 3 (i a multiple of 4; 0 behind the last).
  auto keys = [&](int i) {
    return i < kSelHeld ? *reinterpret_cast<const uint4 *>(held + i) : make_uint4(read(i), read(i + 1), read(i + 2), read(i + 3));
  };
  auto sync_all = [&] {
    if (ranks > 1)
      cluster.sync();
    else
      __syncthreads();
  };

  // After round r the top 8 (r + 1) bits of the threshold are `prefix`; `need`
  // of the candidates with exactly these bits are still to be taken, all with
  // more are.  Once all with these bits are needed the rest decides nothing.
  uint32_t prefix = 0, need = want;
  int shift = 32;
  bool whole = false;  // all candidates with the prefix are taken
  for (int round = 0; round < 4 && !whole; ++round) {
    uint4 *const hist = sh.hist[round & 1];
    uint32_t *const mine_hist = reinterpret_cast<uint32_t *>(hist) + lane % 4;
    if (tid < 256) hist[tid] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    const int below = shift - 8;
    for (int i = tid * 4; i < mine; i += kSelThreads * 4) {
      const uint4 k4 = keys(i);
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
      if (round == 0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) atomicAdd(&mine_hist[(k[u] >> 24) * 4], 1u);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if ((k[u] >> shift) == prefix) atomicAdd(&mine_hist[((k[u] >> below) & 255u) * 4], 1u);
      }
    }
    __syncthreads();
    uint32_t *const local = sh.sum[round & 1];
    uint32_t count = 0;  // thread t has digit 255 - t
    if (tid < 256) {
      const uint4 v = hist[255 - tid];
      count = (v.x + v.y) + (v.z + v.w);
      if (ranks > 1) local[tid] = count;
    }
    if (ranks > 1) {
      cluster.sync();
      if (tid < 256) {
        uint32_t v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = r < ranks ? cluster.map_shared_rank(local, r)[tid] : 0u;
        count = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      }
    }
    uint32_t upto = count;  // with the digits above, within the warp
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    if (tid < 256 && lane == 31) sh.warp_gt[warp] = upto;
    __syncthreads();
    if (tid < 256) {
      for (int w = 0; w < warp; ++w) upto += sh.warp_gt[w];
      if (upto - count < need && need <= upto) {  // one thread
        sh.digit = 255 - tid;
        sh.need = need - (upto - count);
        sh.taken = count == need - (upto - count);
      }
    }
    __syncthreads();
    prefix = (prefix << 8) | sh.digit;
    need = sh.need;
    whole = sh.taken != 0;
    shift = below;
    // The other histogram is cleared next; this one only after every CTA has
    // passed the next round's cluster barrier, and so has read it.
  }

  // Positions: a candidate above the threshold is taken, and of those with the
  // threshold's bits the first `need` ones.  Warp w has a contiguous part of the
  // CTA's positions, four a lane, so one pass counts and a second one writes.
  const int part = ((mine + kSelThreads * 4 - 1) / (kSelThreads * 4)) * 128;
  const int w0 = min(mine, warp * part), w1 = min(mine, w0 + part);
  // How many of the four are above, and (times 2^16) have the threshold's bits.
  auto classify = [&](int i, uint32_t (&c)[4]) {
    const uint4 k4 = i < w1 ? keys(i) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t top = k[u] >> shift;  // shift is 24 at most
      c[u] = (top > prefix ? 1u : 0u) + (k[u] != 0u && top == prefix ? 65536u : 0u);
    }
    return (c[0] + c[1]) + (c[2] + c[3]);
  };
  uint32_t gt_n = 0, eq_n = 0;
  for (int i = w0 + lane * 4; i < w1; i += 128) {
    uint32_t c[4];
    const uint32_t n4 = classify(i, c);
    gt_n += n4 & 65535u;
    eq_n += n4 >> 16;
  }
  gt_n = __reduce_add_sync(0xffffffffu, gt_n);
  eq_n = __reduce_add_sync(0xffffffffu, eq_n);
  if (lane == 0) {
    sh.warp_gt[warp] = gt_n;
    sh.warp_eq[warp] = eq_n;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t g = 0, q = 0;
    for (int w = 0; w < kSelWarps; ++w) {
      const uint32_t gw = sh.warp_gt[w], qw = sh.warp_eq[w];
      sh.warp_gt[w] = g;
      sh.warp_eq[w] = q;
      g += gw;
      q += qw;
    }
    sh.gt = g;
    sh.eq = q;
  }
  sync_all();
  uint32_t g0 = sh.warp_gt[warp], q0 = sh.warp_eq[warp];
  for (int r = 0; r < rank; ++r) {
    const SelShared *o = cluster.map_shared_rank(&sh, r);
    g0 += o->gt;
    q0 += o->eq;
  }
  for (int i = w0; i < w1; i += 128) {
    uint32_t c[4];
    const uint32_t n4 = classify(i + lane * 4, c);
    uint32_t upto = n4;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    uint32_t g = g0 + ((upto - n4) & 65535u), q = q0 + ((upto - n4) >> 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if ((c[u] & 1u) || (c[u] != 0u && q < need)) kept[e.sinks + g + min(q, need)] = j0 + i + lane * 4 + u;
      g += c[u] & 65535u;
      q += c[u] >> 16;
    }
    const uint32_t all4 = __shfl_sync(0xffffffffu, upto, 31);
    g0 += all4 & 65535u;
    q0 += all4 >> 16;
  }
  if (ranks > 1) cluster.sync();  // no CTA leaves while another reads its counts
}

constexpr int kMoveThreads = 256;

// Moves the kept rows of K, V and the weights of a (sequence, kv head).  In
// place row r's source kept[r] >= r, so a CTA that handles all rows of its
// columns in ascending order may write a batch once it has read that batch: what
// later batches read lies behind it.  Different columns never meet, which is
// what spreads a unit over CTAs.  To other pages there is no order to keep, and
// the rows are spread over CTAs instead.  Bound by HBM: 16-byte pieces, eight in
// flight a thread, whose places are looked up once a row, a batch ahead.
struct MoveArgs {
  int pieces;    // 16-byte pieces of a K and of a V row that one CTA moves
  int batch;     // rows at a time
  int chunks;    // CTAs along the rows
  int col_ctas;  // CTAs along the columns of K and V; the first has the weights too
};

// Where a row comes from and goes to: pages; from kStays: nothing is written, from
// kZeros: it lay outside the cache, where rows read as zeros.
constexpr int kStays = -1, kZeros = -2;
struct MovePlace {
  int from, from_row, to, to_row;
};
__device__ __forceinline__ MovePlace move_place(const PagedArgs &a, const EvictArgs &e, int b, const int *kept, int r, int hi) {
  MovePlace p{kStays, 0, -1, 0};
  if (r >= hi) return p;
  const int j = kept[r];
  if (j < 0 || (e.out_table == nullptr && j == r)) return p;
  const int from_slot = j / a.page_size, to_slot = r / a.page_size;
  p.from = paged_page(a, b, from_slot);
  if (p.from < 0) p.from = kZeros;
  p.from_row = j - from_slot * a.page_size;
  p.to = e.out_table == nullptr ? paged_page(a, b, to_slot)
                                : paged_page(a, e.out_table, e.out_stride, e.out_pages, b, to_slot);
  p.to_row = r - to_slot * a.page_size;
  if (p.to < 0) p.from = kStays;
  return p;
}

// One batch of a thread: its pieces of K and V and a weight, and where they go.
template <int kThreads, int kItems>
struct MoveBatch {
  uint4 x[kItems];
  uint4 *to[kItems];
  float wx;
  float *w_to;
  __device__ __forceinline__ void load(const PagedArgs &a, const MoveArgs &m, const MovePlace *places, int h, int col, int i0) {
    const int tid = threadIdx.x, log_p = 31 - __clz(m.pieces);  // a power of two
    const int items = m.batch * m.pieces * 2;
    w_to = nullptr;
    if (col == 0 && i0 == 0 && tid < m.batch) {
      const MovePlace p = places[tid];
      if (p.from != kStays) {
        float *const w = a.w + h * a.ws[1];
        wx = p.from >= 0 ? w[p.from * a.ws[0] + p.from_row] : 0.f;
        w_to = w + p.to * a.ws[0] + p.to_row;
      }
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int i = i0 + u * kThreads + tid;
      to[u] = nullptr;
      if (i >= items) continue;
      const int c = col * m.pieces + (i & (m.pieces - 1));
      const bool is_v = (i >> log_p) & 1;
      const MovePlace p = places[i >> (log_p + 1)];
      if (p.from == kStays) continue;
      const long long *st = is_v ? a.vs : a.ks;
      uint4 *const head = static_cast<uint4 *>(is_v ? a.v : a.k) + h * (st[1] / 8) + c;
      x[u] = p.from >= 0 ? head[p.from * (st[0] / 8) + p.from_row * (st[2] / 8)] : make_uint4(0u, 0u, 0u, 0u);
      to[u] = head + p.to * (st[0] / 8) + p.to_row * (st[2] / 8);
    }
  }
  __device__ __forceinline__ void store() {
#pragma unroll
    for (int u = 0; u < kItems; ++u)
      if (to[u] != nullptr) *to[u] = x[u];
    if (w_to != nullptr) *w_to = wx;
  }
};

constexpr int kInPlaceItems = 4;

// In place: two pieces of K and of V of 512 rows at a time, or with many units
// four of 128 (64 bytes, which HBM likes better, and two CTAs an SM).
template <int kInPlaceThreads>
__global__ void __launch_bounds__(kInPlaceThreads) evict_in_place_kernel(const PagedArgs a, const EvictArgs e, const MoveArgs m) {
  __shared__ MovePlace places[3][kInPlaceThreads];
  const int tid = threadIdx.x;
  const int col = blockIdx.x % m.col_ctas, unit = blockIdx.x / m.col_ctas;
  const int b = unit / a.Hkv, h = unit % a.Hkv;
  // new_lens may be kv_lens: the minimum is the same before and after its write.
  const int n = min(clamp_len(e.kv_lens, b, e.max_kv), e.budget);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // kept is there
  if (col == 0 && h == 0 && tid == 0) e.new_lens[b] = n;
  const int *kept = e.kept + ((long long)b * a.Hkv + h) * e.budget;
  auto look_up = [&](int batch) {
    if (tid < m.batch) places[batch % 3][tid] = move_place(a, e, b, kept, batch * m.batch + tid, n);
  };
  // A batch is read before the one before it is written; its places are looked up
  // a batch earlier still.
  const int batches = (n + m.batch - 1) / m.batch;
  MoveBatch<kInPlaceThreads, kInPlaceItems> cur, next;
  if (batches == 0) return;
  look_up(0);
  look_up(1);
  __syncthreads();
  cur.load(a, m, places[0], h, col, 0);
  for (int i = 0; i < batches; ++i) {
    if (i + 1 < batches) next.load(a, m, places[(i + 1) % 3], h, col, 0);
    look_up(i + 2);
    __syncthreads();  // all have read batch i (and what it overwrites lies in batches up to i)
    cur.store();
    cur = next;
  }
}

// To other pages: a batch of 128 rows a CTA, whole rows.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const PagedArgs a, const EvictArgs e, const MoveArgs m) {
  __shared__ MovePlace places[kMoveThreads];
  const int tid = threadIdx.x;
  const int chunk = blockIdx.x % m.chunks, unit = blockIdx.x / m.chunks;
  const int b = unit / a.Hkv, h = unit % a.Hkv;
  const int n = min(clamp_len(e.kv_lens, b, e.max_kv), e.budget);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (chunk == 0 && h == 0 && tid == 0) e.new_lens[b] = n;
  const int lo = chunk * m.batch;
  if (lo >= n) return;
  const int *kept = e.kept + ((long long)b * a.Hkv + h) * e.budget;
  if (tid < m.batch) places[tid] = move_place(a, e, b, kept, lo + tid, n);
  __syncthreads();
  constexpr int kItems = 8;
  for (int i0 = 0; i0 < m.batch * m.pieces * 2; i0 += kMoveThreads * kItems) {
    MoveBatch<kMoveThreads, kItems> x;
    x.load(a, m, places, h, 0, i0);
    x.store();
  }
}

cudaError_t launch_evict(const PagedArgs &a, const EvictArgs &e, int num_sms, cudaStream_t s) {
  const long long units = (long long)e.B * a.Hkv;
  // CTAs of a cluster: enough that the weights stay in shared memory, and as
  // many as keep the machine busy when there are few units, with 4096 weights each or more
  // (eight heads, with 1024 or more / 4096 or more / one CTA where it holds all, us: 4096
  // tokens 22 / 20 / 20, 16384 29 / 27 / 37; 32 heads of 2048 25 / 20 / 20).
  int ranks = 1;
  while (ranks < 8 && (e.max_kv > ranks * kSelHeld || (units * ranks * 2 <= num_sms && e.max_kv > ranks * 4096)))
    ranks *= 2;
  const int per = ((e.max_kv + ranks - 1) / ranks + 3) & ~3;
  const size_t smem = (size_t)std::min(per, kSelHeld) * 4;
  if (units * ranks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const cudaError_t attr = ranks > 1 ? allow_smem<evict_select_kernel<1024>>(kSelHeld * 4) : allow_smem<evict_select_kernel<512>>(kSelHeld * 4);
  if (attr != cudaSuccess) return attr;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * ranks));
  cfg.blockDim = dim3(ranks > 1 ? 1024 : 512);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t err = cudaLaunchKernelEx(&cfg, ranks > 1 ? evict_select_kernel<1024> : evict_select_kernel<512>, a, e);
  if (err != cudaSuccess) return err;

  MoveArgs m;
  const int row_pieces = a.D / 8;
  const int most = std::min(e.budget, e.max_kv);
  if (e.out_table != nullptr) {
    m.pieces = row_pieces;
    m.batch = 128;
    m.col_ctas = 1;
    m.chunks = (most + m.batch - 1) / m.batch;
  } else {
    // Both ways measured, us, with the selection: 256 units of 1024 rows of head_dim 128 in
    // 32 bytes 119, in 64 bytes 102; 8 units of 16384 rows 121 and 289.
    m.pieces = units * (row_pieces / 4) >= 2LL * num_sms ? 4 : 2;
    m.batch = (m.pieces == 4 ? 256 : 512) * kInPlaceItems / (2 * m.pieces);
    m.col_ctas = row_pieces / m.pieces;
    m.chunks = 1;
  }
  const long long grid = units * m.chunks * m.col_ctas;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t mc = {};
  mc.gridDim = dim3((unsigned)grid);
  mc.blockDim = dim3(e.out_table != nullptr ? kMoveThreads : (m.pieces == 4 ? 256 : 512));
  mc.stream = s;
  cudaLaunchAttribute ma[1];
  ma[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  ma[0].val.programmaticStreamSerializationAllowed = 1;
  mc.attrs = ma;
  mc.numAttrs = 1;
  if (e.out_table != nullptr) return cudaLaunchKernelEx(&mc, evict_move_kernel, a, e, m);
  return m.pieces == 4 ? cudaLaunchKernelEx(&mc, evict_in_place_kernel<256>, a, e, m)
                       : cudaLaunchKernelEx(&mc, evict_in_place_kernel<512>, a, e, m);
}

}  // namespace

llmx_status validate_paged(const llmx_paged_cache *c, int batch, PagedArgs *k) {
  if (c == nullptr) return bad("paged: cache is NULL");
  if (c->dtype != LLMX_FP16 && c->dtype != LLMX_BF16)
    return record_error(LLMX_ERR_UNSUPPORTED, "paged: dtype must be fp16 or bf16");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return record_error(LLMX_ERR_UNSUPPORTED, "paged: head_dim must be 64, 128 or 256");
  if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return bad("paged: n_kv_heads must be in [1, 65535]");
  if (c->page_size < 16 || c->page_size % 16) return bad("paged: page_size must be a multiple of 16");
  if (c->n_pages < 1 || c->max_pages < 1) return bad("paged: n_pages and max_pages must be >= 1");
  if ((long long)c->max_pages * c->page_size > (1LL << 30))
    return bad("paged: max_pages * page_size must be at most 2^30");
  if (c->k == nullptr || c->v == nullptr || !al16(c->k) || !al16(c->v))
    return bad("paged: k and v must be non-NULL and 16-byte aligned");
  const long long extent[3] = {c->n_pages, c->n_kv_heads, c->page_size};
  long long ks[3], vs[3];
  for (int i = 0; i < 3; ++i) {
    ks[i] = extent[i] > 1 ? c->k_stride[i] : 0;  // an extent of 1 is never stepped along
    vs[i] = extent[i] > 1 ? c->v_stride[i] : 0;
    // Every offset stays below 2^60 elements.
    const long long most = (1LL << 58) / extent[i];
    if (ks[i] < 0 || ks[i] % 8 || ks[i] > most || vs[i] < 0 || vs[i] % 8 || vs[i] > most)
      return bad("paged: strides of k and v must be >= 0 and multiples of 8");
  }
  if (!nested(ks, extent, 3, c->head_dim) || !nested(vs, extent, 3, c->head_dim))
    return bad("paged: pages, heads and tokens of k and v must not overlap");
  if (c->block_table != nullptr && c->table_stride < 0) return bad("paged: table_stride must be >= 0");
  if (c->block_table == nullptr && (long long)batch * c->max_pages > c->n_pages)
    return bad("paged: without a block table the cache must hold batch * max_pages pages");
  if (c->key_weights != nullptr) {
    const long long ws[2] = {extent[0] > 1 ? c->w_stride[0] : 0, extent[1] > 1 ? c->w_stride[1] : 0};
    if (!al16(c->key_weights)) return bad("paged: key_weights must be 16-byte aligned");
    for (int i = 0; i < 2; ++i)
      if (ws[i] < 0 || ws[i] % 4 || ws[i] > (1LL << 58) / extent[i])
        return bad("paged: strides of key_weights must be >= 0 and multiples of 4");
    if (!nested(ws, extent, 2, c->page_size)) return bad("paged: pages and heads of key_weights must not overlap");
  }
  k->k = c->k;
  k->v = c->v;
  for (int i = 0; i < 3; ++i) {
    k->ks[i] = ks[i];
    k->vs[i] = vs[i];
  }
  k->table = c->block_table;
  k->table_stride = c->table_stride;
  k->w = c->key_weights;
  k->ws[0] = extent[0] > 1 ? c->w_stride[0] : 0;
  k->ws[1] = extent[1] > 1 ? c->w_stride[1] : 0;
  k->n_pages = c->n_pages;
  k->max_pages = c->max_pages;
  k->page_size = c->page_size;
  k->Hkv = c->n_kv_heads;
  k->D = c->head_dim;
  k->err = nullptr;
  return LLMX_OK;
}

}  // namespace llmx_b200

using namespace llmx_b200;

extern "C" llmx_status llmx_paged_store(const llmx_paged_cache *c, const llmx_kv4_rows *rows, void *stream) {
  if (rows == nullptr) return bad("paged: rows is NULL");
  if (rows->batch < 0 || rows->max_rows < 0) return bad("paged: batch and max_rows must be >= 0");
  PagedArgs k;
  llmx_status st = validate_paged(c, rows->batch, &k);
  if (st != LLMX_OK) return st;
  if (rows->batch == 0 || rows->max_rows == 0) return LLMX_OK;
  if (rows->k == nullptr || rows->v == nullptr) return bad("paged: the rows' k and v must be non-NULL");
  StoreArgs r;
  bool vec = al16(rows->k) && al16(rows->v);
  for (int i = 0; i < 3; ++i) {
    const long long extent = i == 0 ? rows->batch : (i == 1 ? rows->max_rows : k.Hkv);
    r.ks[i] = extent > 1 ? rows->k_stride[i] : 0;
    r.vs[i] = extent > 1 ? rows->v_stride[i] : 0;
    if (r.ks[i] < 0 || r.vs[i] < 0) return bad("paged: strides must be >= 0");
    vec = vec && r.ks[i] % 8 == 0 && r.vs[i] % 8 == 0;
  }
  r.k = rows->k;
  r.v = rows->v;
  r.start = rows->start;
  r.lens = rows->lens;
  r.B = rows->batch;
  r.rows = rows->max_rows;
  int sms = 0;
  st = current_device_info(&k.err, &sms);
  if (st != LLMX_OK) return st;
  const cudaError_t e = launch_store(k, r, vec, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? LLMX_OK : record_error(LLMX_ERR_CUDA, cudaGetErrorString(e));
}

extern "C" llmx_status llmx_paged_evict(const llmx_paged_cache *c, const llmx_paged_evict_params *e, void *stream) {
  if (e == nullptr) return bad("paged evict: params is NULL");
  if (e->batch < 0) return bad("paged evict: batch must be >= 0");
  PagedArgs k;
  llmx_status st = validate_paged(c, e->batch, &k);
  if (st != LLMX_OK) return st;
  if (k.w == nullptr) return bad("paged evict: the cache has no key_weights");
  if (e->budget < 1 || e->recent < 0 || e->sinks < 0 || (long long)e->recent + e->sinks > e->budget)
    return bad("paged evict: budget must be >= 1 and hold sinks + recent, both >= 0");
  const long long room = (long long)k.max_pages * k.page_size;
  if (e->max_kv_len < 1 || e->max_kv_len > room)
    return bad("paged evict: max_kv_len must be in [1, max_pages * page_size]");
  if (e->batch == 0) return LLMX_OK;
  if (e->kv_lens == nullptr || e->kept == nullptr || e->new_lens == nullptr)
    return bad("paged evict: kv_lens, kept and new_lens must be non-NULL");
  EvictArgs a;
  a.B = e->batch;
  a.budget = e->budget;
  a.recent = e->recent;
  a.sinks = e->sinks;
  a.max_kv = e->max_kv_len;
  a.kv_lens = e->kv_lens;
  a.out_table = e->out_table;
  a.out_stride = e->out_table_stride;
  a.out_pages = e->out_pages;
  a.kept = e->kept;
  a.new_lens = e->new_lens;
  if (a.out_table != nullptr) {
    if (a.out_pages < 1 || a.out_stride < 0) return bad("paged evict: out_pages must be >= 1 and its stride >= 0");
    if ((long long)a.out_pages * k.page_size < std::min(a.budget, a.max_kv))
      return bad("paged evict: out_table must hold min(budget, max_kv_len) tokens a sequence");
  }
  int sms = 0;
  st = current_device_info(&k.err, &sms);
  if (st != LLMX_OK) return st;
  const cudaError_t err = launch_evict(k, a, sms, static_cast<cudaStream_t>(stream));
  return err == cudaSuccess ? LLMX_OK : record_error(LLMX_ERR_CUDA, cudaGetErrorString(err));
}
