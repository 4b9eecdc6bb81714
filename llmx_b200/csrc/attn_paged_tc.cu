// Attention over a paged 16-bit key/value cache on the tensor cores: chunks of
// query rows (more than 32 rows of a kv head).
//
// The scheme is the dense prefill's (attn_sm100.cu): a CTA has two tiles of up
// to 128 rows, S = Q K^T and O += P V on tcgen05.mma with both accumulators in
// tensor memory, a softmax warpgroup for each tile, lazy rescaling; at head_dim
// 256 one tile with two score accumulators.  What is different:
//
//  * Rows are packed: a tile has M = (128 / group) * group rows, all query heads
//    of a kv head for 128 / group query rows (one TMA box over [head][row]), so
//    that K and V go through shared memory once for the whole group.
//  * K and V come by pages: a 128-key block is made of boxes of
//    gcd(page_size, 128) rows, one lane of the TMA warp each, whose pages are
//    looked up a block ahead.  Boxes behind the sequence (and pages outside the
//    cache) are loaded from a page index outside the tensor map, which fills
//    zeros: nothing there is read, and the byte count stays the same.
//  * One warp passes V blocks on to the MMA thread.  In blocks that not every
//    row sees whole it first writes zeros over the rows behind the sequence's
//    length and over infinities and NaN (0 * NaN would reach the rows that do
//    not see the token); a bit for each token that lost a value goes to the
//    softmax threads, and the output of rows that see such a token becomes NaN.
//  * ALiBi: the folded slope (x_offset) is a row's own, and biases count from
//    the row's largest one (alibi_ref).
//  * Work: items (a unit's pair of tiles) longest first over one CTA an SM; the
//    items of the last, part-filled wave are cut along the keys into pieces, whose
//    partial results a second launch merges.  Of a batch with lengths of its own
//    all items may be cut, into as many pieces as suits those lengths (cut_items).
//
// Bound by the tensor pipe and the exponentials together: 2048 rows over 34816
// tokens, 32 heads on 8 of 128, take 1.09 ms, 1.04 PFLOP/s (0.64 of the measured
// peak).
#include <algorithm>
#include <climits>
#include <numeric>

#include "paged_tc.cuh"

namespace llmx_b200 {
namespace {

// What differs between head_dim 64, 128 (two tiles; warps 0-7 softmax) and 256 (one
// tile; warps 0-3).
template <int D>
struct PCfg : Cfg<D> {
  static constexpr bool kOne = false;
  static constexpr int kItemRows = kTiles * kBM;
  static constexpr int kThreads = llmx_b200::kThreads;
  static constexpr int kMma = kMmaWarp, kLoad = kTmaWarp;
  static constexpr int kV = 10;  // passes V blocks on; the last warp writes A' (ALiBi)
  static constexpr int kConsumers = 1 + 8 + 2;
};
template <>
struct PCfg<256> : Cfg256 {
  static constexpr bool kOne = true;
  static constexpr int kItemRows = kBM;
  static constexpr int kStages = 1;
  static constexpr uint32_t kTmemO0 = kTmemO, kTmemO1 = kTmemO;
  static constexpr int kThreads = 256;
  static constexpr int kMma = 4, kLoad = 5;  // 6: V
  static constexpr int kV = 7;  // writes A', then passes V blocks on
  static constexpr int kConsumers = 1 + 4 + 2;
};

template <typename T>
constexpr int tc_shift() {
  return std::is_same<T, __half>::value ? 10 : 0;
}

// A launch's items.
struct TcWork {
  PagedArgs c;
  int R;            // packed rows of a kv head
  int M;            // rows of a tile
  int tiles;        // of an item
  int n_mblocks;    // items of a unit
  int group_units;  // units whose K / V fit in L2 together
  int n_whole;      // items [0, n_whole) are whole,
  int piece;        // the others in pieces of so many blocks (the last: the rest),
  int parts;        // at most so many (cut_items may take fewer)
  int n_work;
  int cut;          // items that are cut
  int *how;         // nullable: the device cuts; piece and parts that it took
  float per_query, per_sm;  // for it: items of a query, 1 / SMs,
  int most_keys;            // and what an item sees of a window at most
  int box;         // tokens of a TMA box
  float *part_o;   // [pieces][128 tiles][D]
  float *part_ml;  // [pieces][128 tiles][2]
  float *stat;     // nullable [units][R]: log2 of the sum of 2^score
};

struct Item {
  int b, kvh, ql, kl, m0;
  BlockRange br;
  int nb0;   // blocks that tile 0 takes part in, >= 1
  int slot;  // of its partial result, or -1: whole
  int pieces;  // of the item
  bool none;
};

struct PBars {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3];
  uint64_t s_full[2], p_full[2], o_done[2];
  uint64_t v_landed[3];  // V's copy has arrived; v_full: the V warp has passed it on
  uint64_t drain;
  uint64_t sched_full[kSchedSlots], sched_empty[kSchedSlots];
  int sched_w[kSchedSlots];
  Item sched_item[kSchedSlots];
  uint32_t lost[3][4];  // tokens of the stage's V block that lost a value
  uint32_t tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(PBars) <= 1024, "barriers");

// What a cut of the longest item, of nb blocks, into s pieces costs, in blocks of
// 128 keys on an SM.  A piece costs its blocks and about 3 for its start and end, and
// 1.5 for the merge, as it writes and reads 128 KB of it.  `share` is the items' mean
// length over the longest's.  The launch ends with its last wave, or, as the pieces
// are dealt as CTAs come free, a part of a piece after its mean.
//   What the choice by this cost is worth, us, 32 heads on 8 of 128, against the best of 1 to
// 64 pieces for each shape / uncut: 64 queries on each of 16 x 4,096 tokens 87, 82 / 80; 16 x
// 8,192 151, 143 / 148; 32,768 among fifteen of 300 113, 99 / 490; 8 of 1,000-9,000 83, 75 /
// 133; 32 of those 226, 214 / 252; one sequence of 32,768 with 10 queries 51, 51 / 476, with
// 512 276, 276 / 493; of 131,072 with 16 130, 139 / 1,820; 400 queries on 700, 2,000 and 5,000,
// 16 heads on 4 of 64, 74, 63 / 82; 128 on 300-4,000, 16 heads on 8 of 256, 58, 52 / 76.
__host__ __device__ __forceinline__ float cut_cost(float nb, float s, float items, float share, float per_sm) {
  const float n = items * (1.f - share + share * s) * per_sm;  // pieces of an SM
  const float piece = ceilf(nb / s) + 3.f;
  const float mean = items * share * nb * per_sm + 3.f * n;
  return (s > 1.f ? 2.f + 1.5f * n : 0.f) +
         fminf(ceilf(items * s * per_sm) * piece, fmaxf(piece, mean + (0.2f + 0.8f * share) * piece));
}

// The cut that suits the lengths that the device has, at most as many pieces as the
// workspace was laid out for: 16 sequences of 4,096 tokens with 64 queries, 32 heads
// over 8 of 128, took 115 us cut for ragged lengths, of 0.6 of the longest one's in
// the mean, and take 82 us; of 8,192 tokens 184 and 144 us.
struct Cut {
  int piece, parts, n_work;
};
__device__ __forceinline__ int seen_blocks(const RowsSee &s) {
  return s.hi > s.lo ? (s.hi - s.lo / kBN * kBN + kBN - 1) / kBN : 0;
}
__device__ __forceinline__ Cut cut_items(const AttnArgs &a, const TcWork &wk) {  // by the load warp
  Cut c{wk.piece, wk.parts, wk.n_work};
  if (wk.how == nullptr) return c;
  // Few instructions: the first item waits for them, and they come from L2.  An
  // item sees about as much as the middle row of its sequence.
  const int lane = threadIdx.x % 32;
  const bool windowed = a.causal && a.window >= 0;
  float items = 0.f, total = 0.f, longest = 1.f;
#pragma unroll 1
  for (int b = lane; b < a.B; b += 32) {
    const int ql = clamp_len(a.q_lens, b, a.Sq), kl = clamp_len(a.kv_lens, b, a.Skv);
    const float n = kl > 0 ? ceilf((float)ql * wk.per_query) : 0.f;
    const float most = (float)(windowed ? min(kl, wk.most_keys) : kl) * (1.f / kBN);
    items += n;
    total += n * (a.causal && !windowed ? fmaxf(most - (float)ql * (0.5f / kBN), 0.f) : most);
    if (n > 0.f) longest = fmaxf(longest, ceilf(most));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    items += __shfl_xor_sync(0xffffffffu, items, off);
    total += __shfl_xor_sync(0xffffffffu, total, off);
    longest = fmaxf(longest, __shfl_xor_sync(0xffffffffu, longest, off));
  }
  const float share = items > 0.f ? fminf(1.f, __fdividef(total, items * longest)) : 1.f;
  items = fminf(items * (float)a.Hkv, (float)wk.cut);
  float best = CUDART_INF_F;
  int s = 1;
#pragma unroll 1
  for (int t = lane + 1; t <= min(wk.parts, (int)longest / 4); t += 32) {
    const float cost = cut_cost(longest, (float)t, items, share, wk.per_sm);
    if (cost < best) best = cost, s = t;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float cost = __shfl_xor_sync(0xffffffffu, best, off);
    const int t = __shfl_xor_sync(0xffffffffu, s, off);
    if (cost < best || (cost == best && t < s)) best = cost, s = t;
  }
  c.piece = (int)ceilf(__fdividef(longest, (float)s));
  c.parts = s;
  c.n_work = wk.n_whole + wk.cut * s;
  if (blockIdx.x == 0 && lane == 0) wk.how[0] = c.piece, wk.how[1] = c.parts;  // for the merge
  return c;
}

// Work item w: units in groups whose K / V fit in L2 together, inside a group the
// last rows (which see the most keys) first, as in the dense prefill.
__device__ __forceinline__ Item decode_item(const AttnArgs &a, const TcWork &wk, const Cut &c, int w) {
  Item t;
  int idx = w, part = 0;
  t.slot = -1;
  const bool cut = w >= wk.n_whole && c.parts > 1;
  if (cut) {
    idx = wk.n_whole + (w - wk.n_whole) / c.parts;
    part = (w - wk.n_whole) % c.parts;
  }
  const int units = a.B * a.Hkv;
  const int per_group = wk.group_units * wk.n_mblocks;
  const int g = idx / per_group, within = idx - g * per_group;
  const int gu = min(wk.group_units, units - g * wk.group_units);
  const int rank = within / gu, unit = g * wk.group_units + within % gu;
  const int mblk = a.causal ? wk.n_mblocks - 1 - rank : rank;
  t.kvh = unit % a.Hkv;
  t.b = unit / a.Hkv;
  t.ql = clamp_len(a.q_lens, t.b, a.Sq);
  t.kl = clamp_len(a.kv_lens, t.b, a.Skv);
  t.m0 = mblk * wk.tiles * wk.M;
  const RowsSee s = rows_see(a, t.m0, wk.tiles * wk.M, t.ql, t.kl);
  const int lo = s.lo / kBN * kBN;
  const int nb = seen_blocks(s);
  int nb0 = nb;
  if (nb > 0 && wk.tiles == 2) {
    const RowsSee s0 = rows_see(a, t.m0, wk.M, t.ql, t.kl);
    nb0 = (max(s0.hi, lo) - lo + kBN - 1) / kBN;
  }
  int p0 = 0, p1 = nb;
  if (cut) {
    t.pieces = min(c.parts, (nb + c.piece - 1) / c.piece);
    p0 = min(nb, part * c.piece);
    p1 = part == c.parts - 1 ? nb : min(nb, p0 + c.piece);
    if (t.pieces > 1) t.slot = w - wk.n_whole;
  } else {
    t.pieces = 1;
  }
  t.none = part > 0 && p0 == p1;  // the item has fewer pieces
  t.br.n_start = lo + p0 * kBN;
  t.br.nb = p1 - p0;
  t.nb0 = min(t.br.nb, max(min(1, t.br.nb), nb0 - p0));
  return t;
}

__device__ __forceinline__ bool publish(PBars *bars, int n, int w, const Item &t) {
  const int slot = n % kSchedSlots;
  if (n >= kSchedSlots &&
      !mbar_wait_or_abort(&bars->sched_empty[slot], ((n / kSchedSlots) - 1) & 1, kTimeoutNs, &bars->abort_flag))
    return false;
  bars->sched_w[slot] = w;
  bars->sched_item[slot] = t;
  mbar_arrive(&bars->sched_full[slot]);  // release: orders the stores above
  return true;
}

// The n-th item for a consumer role (w >= n_work: the end), or -1 on abort.
__device__ __forceinline__ int take(PBars *bars, int n, bool warp_wide, Item &t) {
  const int slot = n % kSchedSlots;
  bool ok = mbar_wait_or_abort(&bars->sched_full[slot], (n / kSchedSlots) & 1, kTimeoutNs, &bars->abort_flag);
  if (warp_wide) ok = __all_sync(0xffffffffu, ok);
  if (!ok) return -1;
  const int w = *reinterpret_cast<volatile int *>(&bars->sched_w[slot]);
  t = bars->sched_item[slot];
  if (warp_wide) __syncwarp();
  if (!warp_wide || (threadIdx.x % 32) == 0) mbar_arrive(&bars->sched_empty[slot]);
  return w;
}

// ---------------------------------------------------------------- TMA warp
// Loads of one item: Q tile 0, then per key block K (and after the first K, Q
// tile 1) and V.  Lane i < 128 / box has box i of a block.
struct Loads {
  int k = 0, v = 0, q[2] = {0, 0};
};

// kWhat: 3 all, 1 Q and K, 2 V.
// `first` is where the lane's box of the first block lies; after() runs once that
// block's loads are issued.
template <int D, bool kReverse, int kWhat, typename F>
__device__ bool load_item(const CUtensorMap *tm_q, const CUtensorMap *tm_k, const CUtensorMap *tm_v, uint8_t *smem, PBars *bars,
                          const AttnArgs &a, const TcWork &wk, const Item &t, const BoxPlace &first, int tile_it, int kv_base, Loads &n, F after) {
  using C = PCfg<D>;
  const int lane = threadIdx.x % 32;
  auto wait = [&](uint64_t *bar, uint32_t par) {
    const bool ok = mbar_wait_or_abort(bar, par, kTimeoutNs, &bars->abort_flag);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  auto load_q = [&](int q) {
    if (tile_it > 0 && !wait(&bars->q_empty[q], (tile_it - 1) & 1)) return false;
    if (lane == 0) {
      mbar_arrive_expect_tx(&bars->q_full[q], C::kChunks * wk.M * 128);
      for (int c = 0; c < C::kChunks; ++c)
        tma_load_4d(smem + C::kQOff + q * C::kTileBytes + c * C::kChunkBytes, tm_q, &bars->q_full[q], c * 64, t.kvh * a.group,
                    (t.m0 + q * wk.M) / a.group, t.b);
    }
    n.q[q] = tile_it + 1;
    return true;
  };
  BoxPlace next = first;
  if ((kWhat & 1) && !load_q(0)) return false;
  for (int j = 0; j < t.br.nb; ++j) {
    const int g = kv_base + j;
    const int s = g % C::kStages;
    const uint32_t par = ((g / C::kStages) & 1) ^ 1;
    const BoxPlace p = next;
    if (j + 1 < t.br.nb) next = box_place(wk.c, wk.box, t.b, t.kl, block_n0<kReverse>(t.br, j + 1));
    if (kWhat & 1) {
      if (!wait(&bars->k_empty[s], par)) return false;
      load_boxes<D>(smem + C::kKOff + s * C::kTileBytes, tm_k, &bars->k_full[s], wk.box, t.kvh, p);
      n.k = g + 1;
      if (!C::kOne && j == 0 && !load_q(1)) return false;
    }
    if (kWhat & 2) {
      if (!wait(&bars->v_empty[s], par)) return false;
      load_boxes<D>(smem + C::kVOff + s * C::kTileBytes, tm_v, &bars->v_landed[s], wk.box, t.kvh, p);
      n.v = g + 1;
    }
    if (j == 0) after();
  }
  return true;
}

// Every load issued must have landed before the CTA may exit.
template <int D>
__device__ void drain_loads(PBars *bars, const Loads &n) {
  using C = PCfg<D>;
  for (int q = 0; q < 2; ++q)
    if (n.q[q] > 0) mbar_wait(&bars->q_full[q], (n.q[q] - 1) & 1, kTimeoutNs);
  for (int g = max(0, n.k - C::kStages); g < n.k; ++g)
    mbar_wait(&bars->k_full[g % C::kStages], (g / C::kStages) & 1, kTimeoutNs);
  for (int g = max(0, n.v - C::kStages); g < n.v; ++g)
    mbar_wait(&bars->v_landed[g % C::kStages], (g / C::kStages) & 1, kTimeoutNs);
}

// ------------------------------------------------------------------ V warp
// Lane l has rows l, l + 32, .. of the block at n0.  16-byte chunk c of row r
// lies at chunk c ^ (r % 8) of its 128 bytes, so lanes that take the same c do
// not meet in a bank.  Tokens that no row of the item sees become zeros; of
// those that only some see, infinities and NaN do; the others stay.
template <typename T>
__device__ __forceinline__ uint32_t fma_zero(uint32_t x, uint32_t acc) {  // acc + 0 * x: NaN from an infinity or NaN on
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&x), __float2half2_rn(0.f), *reinterpret_cast<const __half2 *>(&acc));
    return *reinterpret_cast<const uint32_t *>(&r);
  } else {
    const __nv_bfloat162 r =
        __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&x), __float2bfloat162_rn(0.f), *reinterpret_cast<const __nv_bfloat162 *>(&acc));
    return *reinterpret_cast<const uint32_t *>(&r);
  }
}
template <typename T, int D>
__device__ void clean_block(uint8_t *v, uint32_t (&lost)[4], const RowsSee &see, int n0) {
  using C = PCfg<D>;
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const int lane = threadIdx.x % 32;
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int r = i * 32 + lane, j = n0 + r;
    bool bad = false;
    uint8_t *const row = v + r * 128;
    auto at = [&](int p) { return reinterpret_cast<uint4 *>(row + p / 8 * C::kChunkBytes + (((p % 8) ^ (r & 7)) << 4)); };
    if (j < see.lo || j >= see.hi) {
#pragma unroll 8
      for (int p = 0; p < D / 8; ++p) *at(p) = make_uint4(0u, 0u, 0u, 0u);
    } else if (j < see.all_lo || j >= see.all_hi) {
      uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll 8
      for (int p = 0; p < D / 8; ++p) {
        const uint4 x = *at(p);
        acc[0] = fma_zero<T>(x.x, acc[0]);
        acc[1] = fma_zero<T>(x.y, acc[1]);
        acc[2] = fma_zero<T>(x.z, acc[2]);
        acc[3] = fma_zero<T>(x.w, acc[3]);
      }
      const uint32_t any = acc[0] | acc[1] | acc[2] | acc[3];  // NaN in one of them sets all exponent bits
      bad = (any & kExp) == kExp || ((any >> 16) & kExp) == kExp;
      if (bad) {
#pragma unroll 1
        for (int p = 0; p < D / 8; ++p) {
          const uint4 x = *at(p);
          uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if ((w[e] & kExp) == kExp) w[e] &= 0xffff0000u;
            if (((w[e] >> 16) & kExp) == kExp) w[e] &= 0x0000ffffu;
          }
          *at(p) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, bad);
    if (lane == 0) lost[i] = bits;
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// ------------------------------------------------------------ softmax role
// As softmax_tile of the dense prefill; thread r of warpgroup t has packed row
// m0 + t M + r.  blk_base: blocks of this tile in earlier items, kv_base: blocks
// of earlier items.
template <typename T, int D, bool kAlibi, bool kSoftcap>
__device__ bool softmax_rows(const AttnArgs &a, const TcWork &wk, PBars *bars, uint32_t tmem, int warp, const Item &w, int blk_base,
                             int kv_base) {
  using C = PCfg<D>;
  constexpr int kShift = tc_shift<T>();
  const float kNegInf = -CUDART_INF_F;
  const int t = C::kOne ? 0 : warp / 4;
  BlockRange br = w.br;
  if (!C::kOne && t == 0) br.nb = w.nb0;
  const int r = threadIdx.x % kBM;
  const int row0 = w.m0 + t * wk.M;
  const int pr = row0 + r;
  const bool real = r < wk.M && pr < wk.R;
  const int qi = real ? pr / a.group : 0;
  const int h = w.kvh * a.group + (real ? pr - qi * a.group : 0);
  const Visible vis = real ? row_visible(a, qi, w.ql, w.kl) : Visible{0, 0};
  const RowsSee tile = rows_see(a, row0, wk.M, w.ql, w.kl);
  const RowsSee both = rows_see(a, w.m0, wk.tiles * wk.M, w.ql, w.kl);
  const uint32_t lane_off = (uint32_t)((warp % 4) * 32) << 16;
  const uint32_t tO = tmem + lane_off + (t ? C::kTmemO1 : C::kTmemO0);
  const float scale2 = a.sm_scale * kLog2e;
  const float slope = kAlibi ? a.alibi[h] : 0.f;
  const float slope2 = slope * kLog2e;
  const int ref = kAlibi ? alibi_ref(vis, slope) : 0;
  const float cap_in = kSoftcap ? a.sm_scale / a.softcap : 0.f;
  const float cap_out = kSoftcap ? a.softcap * kLog2e : 0.f;
  float m_used = kNegInf, l = 0.f;
  bool aborted = false;
  bool lost = false;  // sees a token that lost a value of V: its output is NaN, not its sum
  // The barrier of block i of the launch and its phase: a tile's own, or with one
  // tile by the block's parity, as the score accumulators.
  auto which = [&](int i) { return C::kOne ? i & 1 : t; };
  auto phase = [&](int i) { return (uint32_t)(C::kOne ? (i >> 1) & 1 : i & 1); };

  for (int j = 0; j < br.nb; ++j) {
    const int n0 = block_n0<kAlibi>(br, j), i = blk_base + j;
    const uint32_t tS = tmem + lane_off + (which(i) ? C::kTmemS1 : C::kTmemS0);
    bool ok = mbar_wait_or_abort(&bars->s_full[which(i)], phase(i), kTimeoutNs, &bars->abort_flag);
    if (!__all_sync(0xffffffffu, ok)) {
      set_abort(bars, a.err);
      aborted = true;
      break;
    }
    tc_fence_after();
    const int lo = max(0, vis.lo - n0), hi = min(kBN, vis.hi - n0);
    const bool need_mask = partly(tile, n0);
    float alpha = 1.f;
    bool rescale = false;
    if (need_mask && __all_sync(0xffffffffu, hi <= lo)) {
      uint32_t z[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) z[c] = 0u;
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_st16(tS + q * 16, z);
    } else if (need_mask) {
      softmax_block<T, kAlibi, kSoftcap, true, kShift, true>(tS, n0 - ref, 0, lo, hi, scale2, slope2, cap_in, cap_out, m_used, l, alpha,
                                                       rescale);
    } else {
      softmax_block<T, kAlibi, kSoftcap, false, kShift, true>(tS, n0 - ref, 0, lo, hi, scale2, slope2, cap_in, cap_out, m_used, l, alpha,
                                                        rescale);
    }
    if (partly(both, n0)) {
      // The V warp has looked at this block: a row that sees a token whose
      // infinity or NaN was taken as 0 is NaN.  (Block index in the item: tile
      // 0's blocks are the last ones in reverse order.)
      const int g = kv_base + (kAlibi && t == 0 ? w.br.nb - w.nb0 : 0) + j;
      const int s = g % C::kStages;
      // A wait by parity needs the stage's block before this one to have been passed
      // on, else it returns a phase early.  With two tiles the MMA thread has waited
      // for that before it issued these scores.  With one stage it is block g - 1,
      // which the products may still be waiting for when these scores are there: its
      // product is waited for first (the next one on that barrier needs this thread's
      // P of a later block, so this phase cannot be passed over; before an item's first
      // block the epilogue has waited for it).
      ok = true;
      if (C::kOne && j > 0) ok = mbar_wait_or_abort(&bars->o_done[which(i - 1)], phase(i - 1), kTimeoutNs, &bars->abort_flag);
      ok = ok && mbar_wait_or_abort(&bars->v_full[s], (g / C::kStages) & 1, kTimeoutNs, &bars->abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        set_abort(bars, a.err);
        aborted = true;
        break;
      }
#pragma unroll
      for (int word = 0; word < 4; ++word) {
        const uint32_t bits = *reinterpret_cast<volatile uint32_t *>(&bars->lost[s][word]);
        if (bits != 0u) {
          const int b0 = min(max(lo - word * 32, 0), 32), b1 = min(max(hi - word * 32, 0), 32);
          const uint32_t below1 = b1 >= 32 ? 0xffffffffu : ((1u << b1) - 1u);
          const uint32_t below0 = b0 >= 32 ? 0xffffffffu : ((1u << b0) - 1u);
          if (bits & below1 & ~below0) lost = true;
        }
      }
    }
    if (__any_sync(0xffffffffu, rescale)) {
      ok = mbar_wait_or_abort(&bars->o_done[which(i - 1)], phase(i - 1), kTimeoutNs, &bars->abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        set_abort(bars, a.err);
        aborted = true;
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int ch = 0; ch < D / 32; ++ch) {
        uint32_t o[32];
        tmem_ld32(tO + ch * 32, o);
        tmem_wait_ld();
        reg_fence32(o);
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
        tmem_st32(tO + ch * 32, o);
      }
    }
    tmem_wait_st();
    tc_fence_before();
    mbar_arrive(&bars->p_full[which(i)]);
  }

  if (!aborted && br.nb > 0) {
    const int i = blk_base + br.nb - 1;
    bool ok = mbar_wait_or_abort(&bars->o_done[which(i)], phase(i), kTimeoutNs, &bars->abort_flag);
    if (!__all_sync(0xffffffffu, ok)) {
      set_abort(bars, a.err);
      aborted = true;
    } else {
      tc_fence_after();
    }
  }
  const bool have = !aborted && br.nb > 0;
  if (w.slot >= 0) {
    // A piece: O and l as they are (P of the row's maximum is 2^kShift).
    const long long prow = (long long)w.slot * C::kItemRows + t * kBM + r;
    float *po = wk.part_o + prow * D;
#pragma unroll 1
    for (int ch = 0; ch < D / 32; ++ch) {
      uint32_t o[32];
      if (have) {
        tmem_ld32(tO + ch * 32, o);
        tmem_wait_ld();
        reg_fence32(o);
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = 0u;
      }
      if (real) {
        if (lost) {
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(CUDART_NAN_F);
        }
#pragma unroll
        for (int c = 0; c < 32; c += 4)
          *reinterpret_cast<uint4 *>(po + ch * 32 + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
      }
    }
    if (real) *reinterpret_cast<float2 *>(wk.part_ml + prow * 2) = make_float2(m_used, l);
    return !aborted;
  }
  const bool sees = vis.hi > vis.lo && have;
  const float inv = sees ? (lost ? CUDART_NAN_F : 1.f / l) : 0.f;
  // As in the dense prefill, groups of four lanes swap pieces so that a store
  // writes 64 contiguous bytes of 8 rows.
  const int gi = threadIdx.x & 3;
  T *to[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int rk = r - gi + k, pk = row0 + rk;
    to[k] = nullptr;
    if (rk < wk.M && pk < wk.R) {
      const int i = pk / a.group;
      to[k] = static_cast<T *>(a.o) + w.b * a.os[0] + i * a.os[1] + (w.kvh * a.group + pk - i * a.group) * a.os[2] + gi * 8;
    }
  }
#pragma unroll 1
  for (int ch = 0; ch < D / 32; ++ch) {
    uint32_t o[32];
    if (have) {
      tmem_ld32(tO + ch * 32, o);
      tmem_wait_ld();
      reg_fence32(o);
    } else {
#pragma unroll
      for (int c = 0; c < 32; ++c) o[c] = 0u;
    }
    uint32_t x[16];
#pragma unroll
    for (int c = 0; c < 16; ++c)
      x[c] = sees ? pack2<T>(__uint_as_float(o[2 * c]) * inv, __uint_as_float(o[2 * c + 1]) * inv) : 0u;
    uint4 u[4];
#pragma unroll
    for (int v4 = 0; v4 < 4; ++v4) u[v4] = make_uint4(x[4 * v4], x[4 * v4 + 1], x[4 * v4 + 2], x[4 * v4 + 3]);
    transpose_units4(u);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (to[k] != nullptr) *reinterpret_cast<uint4 *>(to[k] + ch * 32) = u[k];
  }
  if (real) {
    const float lse2 = m_used - (float)kShift + log2f(l);
    if (a.lse != nullptr)
      a.lse[((long long)w.b * a.H + h) * a.Sq + qi] = sees ? lse2 * kLn2 + (kAlibi ? slope * (float)ref : 0.f) : kNegInf;
    if (wk.stat != nullptr) wk.stat[((long long)w.b * a.Hkv + w.kvh) * wk.R + pr] = lse2;
  }
  return !aborted;
}

// ------------------------------------------------------------------ kernel
template <typename T, int D, bool kAlibi, bool kSoftcap>
__global__ void __launch_bounds__(PCfg<D>::kThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnArgs a,
                    const __grid_constant__ TcWork wk, int *work_ctr) {
  using C = PCfg<D>;
  constexpr bool kFold = kAlibi && !kSoftcap;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  PBars *bars = reinterpret_cast<PBars *>(smem + C::kBarOff);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (threadIdx.x == 0) {
    for (int q = 0; q < kTiles; ++q) {
      mbar_init(&bars->q_full[q], kFold ? 2 : 1);
      mbar_init(&bars->q_empty[q], 1);
      mbar_init(&bars->s_full[q], 1);
      mbar_init(&bars->p_full[q], kBM);
      mbar_init(&bars->o_done[q], 1);
    }
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_landed[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int i = 0; i < kSchedSlots; ++i) {
      mbar_init(&bars->sched_full[i], 1);
      mbar_init(&bars->sched_empty[i], C::kConsumers);
    }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if constexpr (kFold) {
    // B' row c = [c, c, c, 0, ...]; A' zero (its columns 0-2 are written per item).
    constexpr int kA = C::kOne ? 1 : 2;  // of A'
    for (int u = threadIdx.x; u < (kA + 1) * 256; u += C::kThreads) {
      const int op = u >> 8, e = u & 255;
      const int r = (e >> 4) * 8 + (e & 7), khalf = (e >> 3) & 1;
      const float c = (op == kA && khalf == 0) ? (float)r : 0.f;
      const float f[8] = {c, c, c, 0.f, 0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<uint4 *>(smem + C::kXOff + op * C::kXBytes + x_offset(r, khalf * 8)) = pack8<T>(f);
    }
    fence_proxy_async_smem();
  }
  if (warp == C::kLoad && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (warp == C::kMma) {
    tmem_alloc(&bars->tmem_base, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  // Each role runs through the items; what it does with one returns false when the
  // kernel is aborting.
  auto each_item = [&](bool warp_wide, auto role) {
    for (int seq = 0;; ++seq) {
      Item t;
      const int w = take(bars, seq, warp_wide, t);
      if (w >= wk.n_work) break;
      if (w < 0 || !role(t)) {
        set_abort(bars, a.err);
        break;
      }
    }
  };
  // A' of an item (ALiBi): beta = slope / sm_scale as three 16-bit parts (each the
  // rounding of what the ones before it leave), in columns 0-2 of the rows.
  auto write_slopes = [&](const Item &t, int it) {
    for (int q = 0; q < wk.tiles; ++q) {
      bool ok = true;
      if (it > 0) ok = mbar_wait_or_abort(&bars->q_empty[q], (it - 1) & 1, kTimeoutNs, &bars->abort_flag);
      if (!__all_sync(0xffffffffu, ok)) return false;
#pragma unroll 1
      for (int r = lane; r < kBM; r += 32) {
        const float b = a.alibi[t.kvh * a.group + (t.m0 + q * wk.M + r) % a.group] / a.sm_scale;
        const float r1 = b - Elem<T>::to_f(Elem<T>::from_f(b));
        const float r2 = r1 - Elem<T>::to_f(Elem<T>::from_f(r1));
        const float f[8] = {b, r1, r2, 0.f, 0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<uint4 *>(smem + C::kXOff + q * C::kXBytes + x_offset(r, 0)) = pack8<T>(f);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full[q]);
    }
    return true;
  };
  auto pass_v = [&](const Item &t, int kv) {
    const RowsSee both = rows_see(a, t.m0, wk.tiles * wk.M, t.ql, t.kl);
    for (int j = 0; j < t.br.nb; ++j) {
      const int g = kv + j, s = g % C::kStages;
      const bool ok = mbar_wait_or_abort(&bars->v_landed[s], (g / C::kStages) & 1, kTimeoutNs, &bars->abort_flag);
      if (!__all_sync(0xffffffffu, ok)) return false;
      const int n0 = block_n0<kAlibi>(t.br, j);
      if (partly(both, n0)) clean_block<T, D>(smem + C::kVOff + s * C::kTileBytes, bars->lost[s], both, n0);
      if (lane == 0) mbar_arrive(&bars->v_full[s]);
    }
    return true;
  };
  constexpr int kSoftmaxWarps = C::kOne ? 4 : 8;
  if (warp >= kSoftmaxWarps) {
    if constexpr (!C::kOne) regs_decrease<kRegsControl>();
    if (warp == C::kLoad) {
      // The item after the one that is loaded is fetched, published and its first
      // pages looked up while that one's loads run.
      Loads n;
      int kv = 0, it = 0, seq = 0, w = 0;
      Item t{};
      BoxPlace first{0, 0};
      bool ok = true;
      const Cut cut = cut_items(a, wk);
      auto fetch = [&](int from) {  // the item of ticket `from`, or of the first one after it that has work
        for (w = from; w < cut.n_work;) {
          t = decode_item(a, wk, cut, w);
          if (!t.none) break;
          w = wk.n_work;
          if (work_ctr != nullptr) {
            if (lane == 0) w = (int)gridDim.x + atomicAdd(work_ctr, 1);
            w = __shfl_sync(0xffffffffu, w, 0);
          }
        }
        if (w >= cut.n_work) w = wk.n_work;
        bool done = true;
        if (lane == 0) done = publish(bars, seq, w, t);
        ok = __all_sync(0xffffffffu, done) != 0;
        ++seq;
        if (w < wk.n_work && t.br.nb > 0) first = box_place(wk.c, wk.box, t.b, t.kl, block_n0<kAlibi>(t.br, 0));
      };
      auto ticket = [&] {
        int x = wk.n_work;
        if (work_ctr != nullptr) {
          if (lane == 0) x = (int)gridDim.x + atomicAdd(work_ctr, 1);
          x = __shfl_sync(0xffffffffu, x, 0);
        }
        return x;
      };
      fetch((int)blockIdx.x);
      while (ok && w < wk.n_work) {
        const Item now = t;
        const BoxPlace now_first = first;
        if (now.br.nb == 0) {
          fetch(ticket());
          continue;
        }
        bool fetched = true;
        const bool done = load_item<D, kAlibi, C::kOne ? 1 : 3>(&tm_q, &tm_k, &tm_v, smem, bars, a, wk, now, now_first, it, kv, n, [&] {
          fetch(ticket());
          fetched = ok;
        });
        kv += now.br.nb;
        ++it;
        ok = done && fetched;
      }
      if (!ok) set_abort(bars, a.err);
      drain_loads<D>(bars, n);
    } else if (warp == C::kMma) {
      if (lane == 0) {
        int kv = 0, it = 0, blk0 = 0;
        each_item(false, [&](const Item &t) {
          if (t.br.nb == 0) return true;
          bool ok;
          if constexpr (C::kOne) {
            const Mma256Bars mb = {bars->q_full, bars->q_empty, bars->k_full, bars->k_empty, bars->v_full, bars->v_empty,
                                   bars->s_full, bars->p_full,  bars->o_done, &bars->abort_flag};
            ok = mma_256<kBF16, kFold>(smem, mb, tmem, t.br.nb, it, kv);
          } else {
            ok = mma_tile<D, kBF16, kFold, kAlibi>(smem, bars, tmem, t.br.nb, t.nb0, it, kv, blk0, kv);
          }
          kv += t.br.nb;
          blk0 += t.nb0;
          ++it;
          return ok;
        });
        tc_commit(&bars->drain);
        mbar_wait(&bars->drain, 0, kTimeoutNs);
      }
    } else if (warp == C::kV) {
      int kv = 0, it = 0;
      each_item(true, [&](const Item &t) {
        if (t.br.nb == 0) return true;
        if constexpr (C::kOne && kFold)
          if (!write_slopes(t, it)) return false;
        const bool ok = pass_v(t, kv);
        kv += t.br.nb;
        ++it;
        return ok;
      });
    } else {
      if constexpr (C::kOne) {
        // V's loads.
        Loads n;
        int kv = 0;
        each_item(true, [&](const Item &t) {
          if (t.br.nb == 0) return true;
          const BoxPlace first = box_place(wk.c, wk.box, t.b, t.kl, block_n0<kAlibi>(t.br, 0));
          const bool ok = load_item<D, kAlibi, 2>(&tm_q, &tm_k, &tm_v, smem, bars, a, wk, t, first, 0, kv, n, [] {});
          kv += t.br.nb;
          return ok;
        });
        drain_loads<D>(bars, n);
      } else {
        int it = 0;
        each_item(true, [&](const Item &t) {
          if (!kFold || t.br.nb == 0) return true;
          return write_slopes(t, it++);
        });
      }
    }
  } else {
    if constexpr (!C::kOne) regs_increase<kRegsSoftmax>();
    int blk = 0, kv = 0;
    each_item(true, [&](const Item &t) {
      const bool ok = softmax_rows<T, D, kAlibi, kSoftcap>(a, wk, bars, tmem, warp, t, blk, kv);
      blk += !C::kOne && warp < 4 ? t.nb0 : t.br.nb;
      kv += t.br.nb;
      return ok;
    });
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kMma) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Merges the pieces of the items that were cut: a warp a row, four rows a CTA (16
// rows a CTA took 43 -> 57 us for one sequence of 32,768 tokens and 10 queries of 32
// heads over 8 of 128, and gained nothing with many items), four pieces at a time.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_tc_merge_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ TcWork wk) {
  constexpr int E = D / 32, kItemRows = PCfg<D>::kItemRows;
  constexpr float kShift = (float)tc_shift<T>();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  constexpr int kPerItem = kItemRows / 4;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Cut how{wk.piece, wk.parts, wk.n_work};
  Item t;
  if (wk.how == nullptr) t = decode_item(a, wk, how, wk.n_whole + blockIdx.x / kPerItem * how.parts);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (wk.how != nullptr) {
    how = {wk.how[0], wk.how[1], 0};
    if (how.parts == 1) return;
  }
  for (int x = blockIdx.x; x < wk.cut * kPerItem; x += gridDim.x) {
    const int cut = x / kPerItem, in_item = x % kPerItem * 4 + warp;
    if (wk.how != nullptr) t = decode_item(a, wk, how, wk.n_whole + cut * how.parts);
    if (t.slot < 0) continue;
    const int tile = in_item / kBM, r = in_item % kBM;
    const int pr = t.m0 + tile * wk.M + r;
    if (r >= wk.M || pr >= wk.R) continue;
    auto at = [&](int s) { return ((long long)cut * how.parts + s) * kItemRows + in_item; };
    float m = -CUDART_INF_F;
    for (int s = lane; s < t.pieces; s += 32) m = fmaxf(m, wk.part_ml[at(s) * 2]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    constexpr int kAtOnce = 4;
    for (int s0 = 0; s0 < t.pieces; s0 += kAtOnce) {
      float2 ml[kAtOnce], v[kAtOnce][E / 2];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        ml[u] = make_float2(-CUDART_INF_F, 0.f);
        const bool in = s0 + u < t.pieces;
        if (in) ml[u] = *reinterpret_cast<const float2 *>(wk.part_ml + at(s0 + u) * 2);
#pragma unroll
        for (int e = 0; e < E / 2; ++e)
          v[u][e] = in ? *reinterpret_cast<const float2 *>(wk.part_o + at(s0 + u) * D + lane * E + 2 * e) : make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const float w = ex2_approx(ml[u].x - base);
        l = fmaf(w, ml[u].y, l);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          o[2 * e] = fmaf(w, v[u][e].x, o[2 * e]);
          o[2 * e + 1] = fmaf(w, v[u][e].y, o[2 * e + 1]);
        }
      }
    }
    const int i = pr / a.group, h = t.kvh * a.group + pr % a.group;
    const Visible v = row_visible(a, i, t.ql, t.kl);
    const bool sees = v.hi > v.lo;
    const float inv = sees ? 1.f / l : 0.f;
    T *op = static_cast<T *>(a.o) + t.b * a.os[0] + i * a.os[1] + h * a.os[2] + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(op + e) = sees ? pack2<T>(o[e] * inv, o[e + 1] * inv) : 0u;
    if (lane == 0) {
      const float lse2 = m - kShift + log2f(l);
      if (a.lse != nullptr) {
        const float slope = a.alibi != nullptr ? a.alibi[h] : 0.f;
        a.lse[((long long)t.b * a.H + h) * a.Sq + i] =
            sees ? lse2 * kLn2 + (a.alibi != nullptr ? slope * (float)alibi_ref(v, slope) : 0.f) : -CUDART_INF_F;
      }
      if (wk.stat != nullptr) wk.stat[((long long)t.b * a.Hkv + t.kvh) * wk.R + pr] = lse2;
    }
  }
}

// -------------------------------------------------------------------- host
template <typename T, int D, bool kAlibi, bool kSoftcap>
cudaError_t launch_tc_t(const AttnArgs &a, const TcWork &wk, int grid, int *ctr, cudaStream_t s) {
  using C = PCfg<D>;
  CUtensorMap tq, tk, tv;
  if (!make_q_map(&tq, a, wk.M) || !make_page_map(&tk, wk.c, wk.c.k, wk.c.ks, a.dtype, wk.box) ||
      !make_page_map(&tv, wk.c, wk.c.v, wk.c.vs, a.dtype, wk.box))
    return cudaErrorInvalidValue;
  constexpr auto kern = paged_tc_kernel<T, D, kAlibi, kSoftcap>;
  const cudaError_t attr = allow_smem<kern>(C::kSmemBytes);
  if (attr != cudaSuccess) return attr;
  kern<<<grid, C::kThreads, C::kSmemBytes, s>>>(tq, tk, tv, a, wk, ctr);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || wk.parts == 1) return e;
  const int groups = wk.cut * (C::kItemRows / 4);
  return launch_paged_after(paged_tc_merge_kernel<T, D>, dim3(wk.how != nullptr ? std::min(groups, 16 * a.num_sms) : groups),
                            128, 0, s, a, wk);
}

template <typename T, int D>
cudaError_t launch_tc_d(const AttnArgs &a, const TcWork &wk, int grid, int *ctr, cudaStream_t s) {
  const bool alibi = a.alibi != nullptr, cap = a.softcap > 0.f;
  if (alibi) return cap ? launch_tc_t<T, D, true, true>(a, wk, grid, ctr, s) : launch_tc_t<T, D, true, false>(a, wk, grid, ctr, s);
  return cap ? launch_tc_t<T, D, false, true>(a, wk, grid, ctr, s) : launch_tc_t<T, D, false, false>(a, wk, grid, ctr, s);
}

template <typename T>
cudaError_t launch_tc(const AttnArgs &a, const TcWork &wk, int grid, int *ctr, cudaStream_t s) {
  switch (a.D) {
    case 64: return launch_tc_d<T, 64>(a, wk, grid, ctr, s);
    case 128: return launch_tc_d<T, 128>(a, wk, grid, ctr, s);
    default: return launch_tc_d<T, 256>(a, wk, grid, ctr, s);
  }
}

}  // namespace

bool paged_tc_supports(const AttnArgs &a) {
  // The softmax takes the row max on raw scores (sm_scale > 0).
  if (!(a.sm_scale > 0.f) || a.group > kBM) return false;
  const long long units = (long long)a.B * a.Hkv;
  const long long M = kBM / a.group * a.group;
  if (units * (((long long)a.Sq * a.group + M - 1) / M) > INT_MAX / 128) return false;
  return paged_weights_supports(a);
}

PagedTcPlan plan_paged_tc(const AttnArgs &a, bool have_ws) {
  PagedTcPlan p{};
  p.M = kBM / a.group * a.group;
  const int tiles = a.D == 256 ? 1 : kTiles;
  p.n_mblocks = (int)(((long long)a.Sq * a.group + tiles * p.M - 1) / (tiles * p.M));
  const int items = a.B * a.Hkv * p.n_mblocks;
  const int sms = std::max(1, a.num_sms);
  p.parts = 1;
  p.n_whole = items;
  // Blocks of the longest item.
  long long keys = a.Skv;
  if (a.window >= 0 && a.causal) keys = std::min<long long>(keys, (long long)a.window + tiles * p.M / a.group + kBN);
  const int nb = (int)((keys + kBN - 1) / kBN);
  p.piece = nb;
  if (have_ws) {
    // Of equal lengths only the items of the last, part-filled wave are cut; with
    // lengths that only the device knows all of them, where they are few: below four waves.
    // Above, us, uncut / cut: 64 queries on each of 80 sequences of 1,000-9,000 tokens 537 /
    // 605, on 160 of 500-5,000 543 / 539, but one of 32,768 among 99 of 300 519 / 236, which
    // a host that does not know the lengths cannot tell from the first.
    const bool ragged = a.B > 1 && (a.kv_lens != nullptr || a.q_lens != nullptr);
    const int cut = ragged ? (items < 4 * sms ? items : 0) : items % sms;
    const int most = std::min(64, std::max(1, nb / 4));
    auto best = [&](float share) {
      int at = 1;
      for (int s = 2; s <= most; ++s)
        if (cut_cost((float)nb, (float)s, (float)cut, share, 1.f / sms) < cut_cost((float)nb, (float)at, (float)cut, share, 1.f / sms)) at = s;
      return at;
    };
    if (cut > 0) {
      int s = best(1.f);
      if (ragged) {
        // The device may cut a few long ones among short ones into more pieces.  Short
        // ones are left whole: its choice and the merge's launch cost about 8 us.
        s = std::max(s, best(0.6f));
        if (nb >= 32) s = std::max(s, std::min(most, 2 * sms / cut));
        p.on_device = s > 1;
      }
      p.piece = (nb + s - 1) / s;
    }
    p.parts = (nb + p.piece - 1) / p.piece;
    if (p.parts > 1) p.n_whole = items - cut;
    p.part_bytes = p.parts > 1 ? (size_t)cut * p.parts * tiles * kBM * (a.D + 2) * sizeof(float) : 0;
  }
  p.n_work = p.n_whole + (items - p.n_whole) * p.parts;
  return p;
}

cudaError_t launch_paged_tc(const AttnArgs &a, const PagedArgs &c, const PagedTcPlan &p, int *ctr, float *part, float *stat,
                            cudaStream_t s) {
  TcWork wk{};
  wk.c = c;
  wk.R = a.Sq * a.group;
  wk.M = p.M;
  wk.tiles = a.D == 256 ? 1 : kTiles;
  wk.n_mblocks = p.n_mblocks;
  const long long kv_unit = std::max<long long>(1, (long long)a.Skv * a.D * 4);
  wk.group_units = (int)std::max<long long>(1, std::min<long long>((long long)a.B * a.Hkv, (64ll << 20) / kv_unit));
  wk.n_whole = p.n_whole;
  wk.piece = p.piece;
  wk.parts = p.parts;
  wk.n_work = p.n_work;
  wk.cut = (p.n_work - p.n_whole) / p.parts;
  wk.how = p.on_device && p.parts > 1 ? ctr + 1 : nullptr;
  wk.per_query = (float)a.group / (float)(wk.tiles * p.M);
  wk.per_sm = 1.f / (float)std::max(1, a.num_sms);
  wk.most_keys = std::min(std::max(0, a.window), 1 << 30) + wk.tiles * p.M / a.group + kBN;
  wk.box = std::gcd(c.page_size, kBN);
  wk.part_o = part;
  wk.part_ml = p.parts > 1 ? part + (size_t)(p.n_work - p.n_whole) * wk.tiles * kBM * a.D : nullptr;
  wk.stat = stat;
  int grid = p.n_work;
  if (ctr != nullptr && p.n_work > a.num_sms) {
    const cudaError_t e = cudaMemsetAsync(ctr, 0, sizeof(int), s);
    if (e != cudaSuccess) return e;
    grid = a.num_sms;
  } else {
    ctr = nullptr;
  }
  return a.dtype == LLMX_FP16 ? launch_tc<__half>(a, wk, grid, ctr, s) : launch_tc<__nv_bfloat16>(a, wk, grid, ctr, s);
}

}  // namespace llmx_b200
