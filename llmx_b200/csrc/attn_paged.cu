// Attention over a paged 16-bit key/value cache (include/llmx_attn.h): the
// request's checks and the choice between its two forms, and the form for few
// query rows, which streams K and V once past all rows of a kv head.
//
// Products.  A unit is one (sequence, kv head) and a block of up to N packed rows
// (16 or 32; 64 at head_dim 256).  Both products are transposed, so that the 128 rows of the
// tensor core's tile are tokens or channels, which there are enough of, and the
// few query rows are its columns:
//   S^T [128 tokens x N] = K Q^T,   O^T [channels x N] += V^T P^T
// on tcgen05.mma with both accumulators in tensor memory.  A softmax thread has
// one token and N scores: no work is done for rows that are not there, and the
// sum over tokens stays in its registers until the unit's end.  A row's
// reference for the exponentials is common to all threads and moves (and O^T is
// rescaled) only when some score passes it by more than a limit, which one
// barrier with a vote finds out; the first block sets it.
//
// Work.  The blocks of 128 tokens of all units, end to end, are dealt to the
// resident CTAs in equal shares, so that sequences of any lengths finish
// together; a CTA writes the result of a unit that it has whole and a partial
// result (unnormalised O, reference and sum; at most two a CTA) of one that it
// shares, which a second, overlapped launch merges.
//
// A CTA: one warpgroup for the softmax (two, each with half of the rows, from 32
// rows on: the code that a cold instruction cache has to fetch stays small), a
// warp that issues the products, and one for the copies: K and V by TMA boxes
// from the pages into one ring of slots, in the order in which they are used (K
// of a block comes before V of the block before it).
//
// Bound by HBM: 32 sequences of 1001-8191 tokens, 32 heads on 8 of 128, take 102 us
// (5.9 TB/s, 0.90 of the measured copy rate), one of 131071 tokens 94 us (5.7 TB/s);
// what is missing is the start and the merge.  Short calls are their launch (8 us).
//
// Masked tokens.  A NaN or an infinity in K only reaches scores that are
// replaced.  One in V would reach every row through 0 * V, so in blocks that not
// every row sees whole, the thread of a token first writes zeros over such
// values (and over all of a token that no row sees: nothing behind a sequence's
// length counts), and the output of the rows that see it becomes NaN (their sums,
// lse and key weights do not: V has no part in them).
#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstring>
#include <numeric>

#include "paged_tc.cuh"

namespace llmx_b200 {
namespace {

// AUTO: packed rows of a kv head up to which this form is taken.  Both forms, us, at
// 16 / 32 / 48 / 64 / 128 rows (L2 flushed): 16 sequences of 4096 tokens, 8 kv heads of
// 128: this 69 / 75 / 118 / 120 / 202, tiles 84 at all; one of 32768: 48 / 48 / 58 / 56 /
// 93, 50 / 52 / 52 / 54 / 56; 4 of 4096 at head_dim 256: 50 / 50 / 54 / 54 / 75, 51 / 53 /
// 55 / 55 / 59; 16 of 2048 at 256: 77 / 81 / 89 / 93 / 142, 69 at all.
//   Above that this form is taken where it is asked for and where tiles cannot be (a scale
// that is not positive, an expanded q, more than 128 heads a kv head).  At head_dim 256 a
// block then has 64 rows, else 32 (whose code and ring suit 64 and 128 better): one of 32768
// tokens, 64 rows, 61 us against 70 in two blocks of 32, 16 of 2048 58 against 65.
constexpr int kStepRows = 32;
constexpr size_t kCounterBytes = 256;

// A launch's units and shares.
struct StepWork {
  PagedArgs c;
  int R;          // packed rows of a kv head
  int nrb;        // row blocks
  int workers;    // CTAs that take a share, at most
  int min_steps;  // a share is at least this long
  int split;      // 0: CTA i has unit i whole
  int reverse;    // a unit's blocks go last to first (ALiBi: the largest biases come first)
  int box;        // tokens of a TMA box
  float *part_o;   // [2 workers][N][D]
  float *part_ml;  // [2 workers][N][2]
  float *stat;     // nullable [B * Hkv][R]: log2 of the sum of 2^score
  float *score;    // nullable [B * Hkv][R][pitch], log2 units
  long long pitch;
  float decay;
};

// Row block rb of sequence b: blocks of 128 tokens lo128 + 128 i .., tokens in
// [lo, hi) are visible to some row.  A unit's steps are its blocks and, before
// them, kUnitSteps that stand for what starting and ending a unit costs (us for 0 / 1 / 2 /
// 4 of them: 128 sequences of 1-600 tokens 74 / 63 / 61 / 61, three of 9000 among 21 of 100
// 57 / 47 / 43 / 41; sequences of equal lengths take the same time with any).
constexpr int kUnitSteps = 2;
struct Span {
  int ql, kl, lo, hi, all_lo, all_hi;
  __device__ __forceinline__ int lo128() const { return lo & ~(kBN - 1); }
  __device__ __forceinline__ int blocks() const { return hi > lo ? (hi - lo128() + kBN - 1) / kBN : 0; }
  __device__ __forceinline__ int steps() const { return kUnitSteps + blocks(); }
  // First token of the unit's i-th block.
  __device__ __forceinline__ int token(int i, int reverse) const { return lo128() + (reverse ? blocks() - 1 - i : i) * kBN; }
};
__device__ __forceinline__ Span span_of(const AttnArgs &a, int R, int rows, int b, int rb) {
  Span s;
  s.ql = clamp_len(a.q_lens, b, a.Sq);
  s.kl = clamp_len(a.kv_lens, b, a.Skv);
  const RowsSee v = rows_see(a, rb * rows, min(rows, R - rb * rows), s.ql, s.kl);
  s.lo = v.lo;
  s.hi = v.hi;
  s.all_lo = v.all_lo;
  s.all_hi = v.all_hi;
  if (s.hi <= s.lo) s.lo = s.hi = 0;
  return s;
}

// Steps of all units of sequence b.  (All steps of a launch stay below 2^31:
// plan_step.)
__device__ __forceinline__ int steps_of(const AttnArgs &a, const StepWork &wk, int rows, int b) {
  int n = 0;
  for (int rb = 0; rb < wk.nrb; ++rb) n += span_of(a, wk.R, rows, b, rb).steps();
  return n * a.Hkv;
}

// Shares: worker w of n has the steps [total * w / n, total * (w + 1) / n).
__device__ __forceinline__ int share_count(const StepWork &wk, int total) { return max(1, min(wk.workers, total / wk.min_steps)); }
__device__ __forceinline__ int share_begin(int total, int w, int n) {
  const int q = total / n, r = total - q * n;  // r, w <= n, a few per SM
  return q * w + r * w / n;
}
__device__ __forceinline__ int share_of(int total, int step, int n) {
  int w = min(n - 1, (int)((float)step * (float)n / (float)total));  // within a few of it, put right
  while (w > 0 && share_begin(total, w, n) > step) --w;
  while (w < n - 1 && share_begin(total, w + 1, n) <= step) ++w;
  return w;
}

// A scan over the sequences by the whole CTA: the steps of all, then of the
// sequence b that pick(b, before, steps, total) names, and the steps before it.
struct ScanShared {
  int warp_sum[12];
  int before, steps, total;
  int b;
};
template <typename F>
__device__ void scan_steps(const AttnArgs &a, const StepWork &wk, int rows, ScanShared &sh, F pick) {
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, threads = blockDim.x;
  const int rounds = (a.B + threads - 1) / threads;
  int total = 0;
  // With one round of threads the second pass has its numbers already.
  for (int pass = 0; pass < 2; ++pass) {
    int base = 0;
    for (int round = 0; round < rounds; ++round) {
      const int b = round * threads + tid;
      const int mine = b < a.B ? steps_of(a, wk, rows, b) : 0;
      int x = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += o;
      }
      if (lane == 31) sh.warp_sum[warp] = x;
      __syncthreads();
      int before = base + x - mine;
      for (int w = 0; w < threads / 32; ++w) {
        if (w < warp) before += sh.warp_sum[w];
        base += sh.warp_sum[w];
      }
      if (pass == 0) total = base;
      if ((pass == 1 || rounds == 1) && b < a.B && pick(b, before, mine, total)) {
        sh.b = b;
        sh.before = before;
        sh.steps = mine;
      }
      __syncthreads();
    }
    if (rounds == 1) break;
  }
  if (tid == 0) sh.total = total;
  __syncthreads();
}

// A share's position: `left` steps from step `at` of unit (b, kvh, rb) on.
struct Cursor {
  int b, kvh, rb, at, left;
  Span sp;
  __device__ __forceinline__ int end() const { return min(sp.steps(), at + left); }
  // The part's blocks [first(), last()).  A part without any is not the unit's,
  // but of a unit that has none the one with its first step is.
  __device__ __forceinline__ int first() const { return max(0, at - kUnitSteps); }
  __device__ __forceinline__ int last() const { return max(0, end() - kUnitSteps); }
  __device__ __forceinline__ bool none() const { return sp.hi > sp.lo ? first() == last() : at > 0; }
  // Past this unit's part, to the next unit.  False at the share's end.
  __device__ __forceinline__ bool next(const AttnArgs &a, const StepWork &wk, int rows) {
    left -= end() - at;
    if (left <= 0) return false;
    at = 0;
    if (++rb == wk.nrb) {
      rb = 0;
      if (++kvh == a.Hkv) {
        kvh = 0;
        ++b;
      }
    }
    sp = span_of(a, wk.R, rows, b, rb);
    return true;
  }
};

// ------------------------------------------------------------------ kernel
// A slot of the ring holds 128 tokens x up to 128 channels of K or V.  Two CTAs
// an SM where their rings are deep enough (a CTA's start and end are then
// covered by the other), else one; about 200 KB of copies an SM either way.
template <int D, int N>
struct StepCfg {
  static constexpr int kGroups = N == 16 ? 1 : 2;  // softmax warpgroups
  static constexpr int kCols = N / kGroups;        // rows of one of them
  static constexpr int kSoftmax = 128 * kGroups, kThreads = kSoftmax + 64;
  static constexpr int kMmaWarp = 4 * kGroups, kTmaWarp = kMmaWarp + 1;
  static constexpr int kDH = D < 128 ? D : 128;  // channels of a slot
  static constexpr int kHalves = D / kDH;        // slots of a block of K or V
  static constexpr int kSlot = kBN * kDH * 2;
  static constexpr int kCtas = D == 256 || N > 16 ? 1 : 2;
  static constexpr int kQ = N * D * 2, kP = N * kBN * 2;
  static constexpr int kInfo = N == 16 ? 1792 : (N == 32 ? 2816 : 4864);  // RowInfo, barriers
  static constexpr int kBudget = (kCtas == 2 ? 113 : 227) * 1024 - 1024 - 256;  // less alignment and static arrays
  static constexpr int kFit = (kBudget - kQ - 2 * kP - kInfo) / kSlot;
  static constexpr int kSlots = kFit < 12 ? kFit : 12;
  // What the products need, and what the softmax's wait for V does (where it looks at V).
  static_assert(kSlots >= 3 || kHalves > 1, "ring");
  static_assert(kSlots >= 2 * kHalves, "ring");
  static constexpr int kQOff = kSlots * kSlot, kPOff = kQOff + kQ, kInfoOff = kPOff + 2 * kP;
  static constexpr int kSmem = kInfoOff + kInfo + 1024;
  // Tensor memory: two score accumulators, then O^T (one for each 128 channels).
  static constexpr uint32_t kO = 2 * N;
  static constexpr uint32_t kTmem = N == 16 ? 64 : (N == 32 ? 128 : 256);
  static_assert(2 * N + kHalves * N <= (int)kTmem, "tensor memory");
};

template <int N>
struct RowInfo {
  long long out[N];  // where the row's output begins
  float base[N];   // what is subtracted from a score: the reference less the weights' shift
  float limit[N];  // scores above it move the reference; -inf before the first
  float ref[N];    // the reference
  float alpha[N];
  float slope2[N];
  int bias0[N];  // the token whose ALiBi bias counts as 0
  int lo[N], hi[N];
  float wmax[4][N];  // by warp: maxima, then sums
  float scale[N];    // 1, or NaN: the row sees a token that lost a value of V; of a whole unit then over the sum
};
struct SBars {
  uint64_t full[12], empty[12];
  uint64_t q_full, s_full[2], p_full[2], o_done[2], drain;  // [2]: by the block's parity
  uint8_t lost[2][2][128];  // by the block's parity and the warpgroup: the token lost a value of V
  uint32_t tmem_base;
  volatile int abort_flag;
};

// fp16 weights are taken 2^10 times as large, so that small ones keep their
// bits, and pass the reference by 2^5 at most; bf16 has the exponents of fp32.
template <typename T>
constexpr float weight_shift() {
  return std::is_same<T, __half>::value ? 10.f : 0.f;
}
template <typename T>
constexpr float weight_room() {
  return std::is_same<T, __half>::value ? 5.f : 64.f;
}

template <int N>
__device__ __forceinline__ void tmem_ld_n(uint32_t at, float (&x)[N]) {
  if constexpr (N == 16) {
    uint32_t v[16];
    tmem_ld16(at, v);
    tmem_wait_ld();
    reg_fence16(v);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(v[i]);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 32) {
      uint32_t v[32];
      tmem_ld32(at + c, v);
      tmem_wait_ld();
      reg_fence32(v);
#pragma unroll
      for (int i = 0; i < 32; ++i) x[c + i] = __uint_as_float(v[i]);
    }
  }
}
template <int N>
__device__ __forceinline__ void tmem_st_n(uint32_t at, const float (&x)[N]) {
  if constexpr (N == 16) {
    uint32_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(x[i]);
    tmem_st16(at, v);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 32) {
      uint32_t v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(x[c + i]);
      tmem_st32(at + c, v);
    }
  }
}

// The four warps of softmax warpgroup g: a barrier, and one with a vote.  These
// are not bounded: every warp runs through all blocks of the share, also after
// an abort.
__device__ __forceinline__ void wg_sync(int g) { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); }
__device__ __forceinline__ bool wg_any(int g, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)p), "r"(1 + g)
      : "memory");
  return r != 0;
}

// Reduces v[0 .. N) over a warp's lanes, each exchange handing over half of what
// is left: N - 1 to N + 1 shuffles instead of 5 N.  Lane l gets row l (N = 32),
// rows l and l + 32 in v[0], v[32] (64), or row l / 2 (16).
template <int N, typename Op>
__device__ __forceinline__ void reduce_rows(float (&v)[N], Op op) {
  const int lane = threadIdx.x % 32;
  constexpr int M = N < 32 ? N : 32;
#pragma unroll
  for (int base = 0; base < N; base += M) {
#pragma unroll
    for (int h = M / 2, bit = 16; h >= 1; h /= 2, bit /= 2) {
      const bool up = lane & bit;
#pragma unroll
      for (int i = 0; i < h; ++i) {
        const float lo = v[base + i], hi = v[base + i + h];
        v[base + i] = op(up ? hi : lo, __shfl_xor_sync(0xffffffffu, up ? lo : hi, bit));
      }
    }
    if constexpr (M == 16) v[base] = op(v[base], __shfl_xor_sync(0xffffffffu, v[base], 1));
  }
}
template <int N>
__device__ __forceinline__ void put_rows(float *to, const float (&v)[N]) {
  const int lane = threadIdx.x % 32;
  if constexpr (N == 16) {
    if (!(lane & 1)) to[lane / 2] = v[0];
  } else {
#pragma unroll
    for (int base = 0; base < N; base += 32) to[base + lane] = v[base];
  }
}

// A token's channels of V in a slot (its row `r`), `n` 16-byte pieces from piece
// `first` on: infinities and NaN become 0 (true if there was one), or everything
// does.  Piece p lies in 64-channel chunk p / 8 at (p % 8) ^ (r % 8).
template <typename T>
__device__ __forceinline__ bool clean_row(uint8_t *slot, int r, int first, int n, bool all) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  bool lost = false;
#pragma unroll 2
  for (int p = first; p < first + n; ++p) {
    uint4 *const at = reinterpret_cast<uint4 *>(slot + (p / 8) * 128 * 128 + r * 128 + (((p % 8) ^ (r & 7)) << 4));
    if (all) {
      *at = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    const uint4 x = *at;
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool any = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t m = (w[e] & kExp) ^ kExp;  // a half that is 0: all exponent bits set
      if ((m & 0xffffu) == 0u) {
        w[e] &= 0xffff0000u;
        any = true;
      }
      if ((m >> 16) == 0u) {
        w[e] &= 0x0000ffffu;
        any = true;
      }
    }
    if (any) {
      *at = make_uint4(w[0], w[1], w[2], w[3]);
      lost = true;
    }
  }
  return lost;
}

// kMode: 1 ALiBi, 2 a soft-cap (with ALiBi or without), 0 neither.
template <typename T, int D, int N, int kMode>
__global__ void __launch_bounds__(StepCfg<D, N>::kThreads, StepCfg<D, N>::kCtas)
    paged_step_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ AttnArgs a, const __grid_constant__ StepWork wk) {
  using C = StepCfg<D, N>;
  constexpr int H = C::kHalves;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  RowInfo<N> *const info = reinterpret_cast<RowInfo<N> *>(smem + C::kInfoOff);
  SBars *const bars = reinterpret_cast<SBars *>(smem + C::kInfoOff + sizeof(RowInfo<N>));
  static_assert(sizeof(RowInfo<N>) % 16 == 0 && sizeof(RowInfo<N>) + sizeof(SBars) <= C::kInfo, "row info");
  __shared__ ScanShared sh;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == C::kTmaWarp && lane == 0) {  // which then needs no one to start copying
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->empty[i], 1);
    }
    mbar_init(&bars->q_full, C::kSoftmax);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], C::kSoftmax);
      mbar_init(&bars->o_done[i], 1);
    }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }

  // ---- this CTA's share
  Cursor cur;
  const int worker = blockIdx.x;
  if (wk.split) {
    scan_steps(a, wk, N, sh, [&](int, int before, int steps, int total) {
      const int n = share_count(wk, total);
      if (worker >= n) return false;
      const int begin = share_begin(total, worker, n);
      return before <= begin && begin < before + steps;
    });
    const int total = sh.total;
    const int n = share_count(wk, total);
    if (worker >= n) return;
    const int begin = share_begin(total, worker, n);
    cur.left = share_begin(total, worker + 1, n) - begin;
    if (cur.left <= 0) return;
    cur.b = sh.b;
    int within = begin - sh.before;
    const int per_head = sh.steps / a.Hkv;
    cur.kvh = (int)(within / per_head);
    within -= cur.kvh * per_head;
    for (cur.rb = 0;; ++cur.rb) {
      cur.sp = span_of(a, wk.R, N, cur.b, cur.rb);
      if (within < cur.sp.steps()) break;
      within -= cur.sp.steps();
    }
    cur.at = (int)within;
  } else {
    cur.rb = worker % wk.nrb;
    const int u = worker / wk.nrb;
    cur.kvh = u % a.Hkv;
    cur.b = u / a.Hkv;
    cur.sp = span_of(a, wk.R, N, cur.b, cur.rb);
    cur.at = 0;
    cur.left = cur.sp.steps();
  }
  // Each role meets the others when it has its first loads under way.
  uint32_t tmem = 0;
  auto meet = [&] {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    tmem = bars->tmem_base;
  };
  auto wait = [&](uint64_t *bar, uint32_t par) { return mbar_wait_or_abort(bar, par, kTimeoutNs, &bars->abort_flag); };

  if (warp == C::kTmaWarp) {
    // ---- copies, in the order K 0, K 1, V 0, K 2, V 1, ..
    int g = 0;  // slots filled
    bool ok = true;
    __syncwarp();  // the barriers are set up
    auto copy = [&](const CUtensorMap *tm, const BoxPlace &p) {
      for (int half = 0; half < H && ok; ++half, ++g) {
        const int s = g % C::kSlots;
        ok = __all_sync(0xffffffffu, wait(&bars->empty[s], ((g / C::kSlots) & 1) ^ 1)) != 0;
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars->full[s], C::kSlot);
        __syncwarp();
        if (lane < kBN / wk.box)
          for (int c = 0; c < C::kDH / 64; ++c)
            tma_load_4d(smem + s * C::kSlot + c * 128 * 128 + lane * wk.box * 128, tm, &bars->full[s], half * 128 + c * 64, p.row,
                        cur.kvh, p.page);
      }
    };
    bool met = false;
    do {
      const int b0 = cur.first(), b1 = cur.last();
      BoxPlace kp, vp;
      if (b0 < b1) {
        kp = box_place(wk.c, wk.box, cur.b, cur.sp.kl, cur.sp.token(b0, wk.reverse));
        vp = kp;
        copy(&tm_k, kp);
      }
      if (!met) meet();
      met = true;
      for (int j = b0; j < b1 && ok; ++j) {
        if (j + 1 < b1) {
          kp = box_place(wk.c, wk.box, cur.b, cur.sp.kl, cur.sp.token(j + 1, wk.reverse));
          copy(&tm_k, kp);
        }
        if (ok) copy(&tm_v, vp);
        vp = kp;
      }
    } while (ok && cur.next(a, wk, N));
    if (!ok) set_abort(bars, a.err);
    // Every copy issued lands before the CTA may exit.
    for (int i = max(0, g - C::kSlots); i < g; ++i) mbar_wait(&bars->full[i % C::kSlots], (i / C::kSlots) & 1, kTimeoutNs);
  } else if (warp == C::kMmaWarp) {
    tmem_alloc(&bars->tmem_base, C::kTmem);
    tmem_relinquish();
    meet();
    if (lane == 0) {
      // ---- products: S^T(j + 1) is issued before O^T += .. (j)
      constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
      constexpr uint32_t idesc_s = idesc_f16(128, N, kBF16, false);
      constexpr uint32_t idesc_o = idesc_f16(128, N, kBF16, true) | (1u << 15);  // V^T: M-major
      int g = 0, blk = 0, parts = 0;  // slots used, blocks, parts with blocks
      bool ok = true;
      const uint32_t q_base = smem_u32(smem + C::kQOff), p_base = smem_u32(smem + C::kPOff), ring = smem_u32(smem);
      auto scores = [&](int at) {
        for (int half = 0; half < H && ok; ++half, ++g) {
          const int s = g % C::kSlots;
          ok = wait(&bars->full[s], (g / C::kSlots) & 1);
          if (!ok) return;
          tc_fence_after();
          uint64_t da = smem_desc_sw128(ring + s * C::kSlot, 16, 1024);
          uint64_t db = smem_desc_sw128(q_base + half * 2 * N * 128, 16, 1024);
          asm volatile("" : "+l"(da), "+l"(db));
#pragma unroll
          for (int kk = 0; kk < C::kDH / 16; ++kk)
            mma_ss(tmem + (at & 1) * N, da + (uint64_t)(((kk / 4) * 128 * 128 + (kk % 4) * 32) >> 4),
                   db + (uint64_t)(((kk / 4) * N * 128 + (kk % 4) * 32) >> 4), idesc_s, (half > 0 || kk > 0) ? 1u : 0u);
          tc_commit(&bars->empty[s]);
        }
        if (ok) tc_commit(&bars->s_full[at & 1]);
      };
      do {
        const int b0 = cur.first(), b1 = cur.last();
        if (b0 == b1) continue;
        ok = wait(&bars->q_full, parts & 1);
        ++parts;
        if (!ok) break;
        scores(blk);
        for (int j = b0; j < b1 && ok; ++j, ++blk) {
          if (j + 1 < b1) scores(blk + 1);
          if (!ok) break;
          ok = wait(&bars->p_full[blk & 1], (blk >> 1) & 1);
          for (int half = 0; half < H && ok; ++half, ++g) {
            const int s = g % C::kSlots;
            ok = wait(&bars->full[s], (g / C::kSlots) & 1);
            if (!ok) break;
            tc_fence_after();
            // V^T by 64-channel chunks; at head_dim 64 the second 64 rows of the
            // tile repeat the first and are not used.
            uint64_t da = smem_desc_sw128(ring + s * C::kSlot, D == 64 ? 0 : 128 * 128, 1024);
            // P^T: 8 tokens x 8 rows of 128 bytes, 128 bytes apart along the
            // tokens and 2048 along the rows.
            uint64_t db = smem_desc_noswz(p_base + (blk & 1) * C::kP, 128, 2048);
            asm volatile("" : "+l"(da), "+l"(db));
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              mma_ss(tmem + C::kO + half * N, da + (uint64_t)((kk * 16 * 128) >> 4), db + (uint64_t)((kk * 256) >> 4), idesc_o,
                     (j > b0 || kk > 0) ? 1u : 0u);
            tc_commit(&bars->empty[s]);
          }
          if (ok) tc_commit(&bars->o_done[blk & 1]);
        }
      } while (ok && cur.next(a, wk, N));
      if (!ok) set_abort(bars, a.err);
      tc_commit(&bars->drain);
      mbar_wait(&bars->drain, 0, kTimeoutNs);
    }
  } else {
    // ---- softmax: a thread has a token of each block and a channel (or two) of
    // O^T, and its warpgroup's rows c0 .. of them
    constexpr int W = C::kCols;
    const int wg = warp / 4, tok = tid % 128, c0 = wg * W;
    const uint32_t lane_off = (uint32_t)(warp % 4 * 32) << 16;
    const float scale2 = a.sm_scale * kLog2e;
    const SoftCap cap(kMode == 2 ? a.sm_scale / a.softcap : 0.f, a.softcap * kLog2e);
    constexpr float kShift = weight_shift<T>();
    int g = 0, blk = 0;
    bool ok = true;
    auto wait_all = [&](uint64_t *bar, uint32_t par) {
      const bool w = __all_sync(0xffffffffu, wait(bar, par)) != 0;
      if (!w && ok) set_abort(bars, a.err);
      ok = ok && w;
    };
    // Q [row][64 channels] in 128 bytes a row, chunk c at c ^ (row % 8).  The next
    // part's rows are read while this one's blocks pass (where they are few).
    constexpr int kPieces = N * D / 8 / C::kSoftmax;  // of a thread
    constexpr bool kAhead = kPieces <= 4;
    uint4 qx[kPieces];
    auto read_q = [&](const Cursor &c) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        const int r = (u * C::kSoftmax + tid) / (D / 8), ch = (u * C::kSoftmax + tid) % (D / 8);
        const int pr = c.rb * N + r, i = pr / a.group;
        qx[u] = make_uint4(0u, 0u, 0u, 0u);
        if (pr < wk.R && i < c.sp.ql && c.first() < c.last())
          qx[u] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + c.b * a.qs[0] + i * a.qs[1] +
                                                   (c.kvh * a.group + pr - i * a.group) * a.qs[2] + ch * 8);
      }
    };
    if (kAhead) read_q(cur);
    meet();
    for (bool more = true; more;) {
      Cursor nx = cur;
      const bool none = cur.none();
      more = nx.next(a, wk, N);
      if (none) {
        cur = nx;
        if (kAhead && more) read_q(cur);
        continue;
      }
      const Span sp = cur.sp;
      const int b0 = cur.first(), b1 = cur.last();
      const int row0 = cur.rb * N, rows = min(N, wk.R - row0);
      if (!kAhead) read_q(cur);
      // Everything of the last part has been read (the barrier at its end).
      if (tok < W) {
        const int row = c0 + tok, r = row0 + row, i = r / a.group, h = cur.kvh * a.group + r - i * a.group;
        const bool real = row < rows && i < sp.ql;
        const Visible v = real ? row_visible(a, i, sp.ql, sp.kl) : Visible{0, 0};
        const float slope = kMode != 0 && a.alibi != nullptr && real ? a.alibi[h] : 0.f;
        info->lo[row] = v.lo;
        info->hi[row] = v.hi;
        info->slope2[row] = slope * kLog2e;
        info->bias0[row] = alibi_ref(v, slope);
        info->ref[row] = info->limit[row] = -CUDART_INF_F;
        info->base[row] = -kShift;
        info->scale[row] = 1.f;
        info->out[row] = cur.b * a.os[0] + i * a.os[1] + h * a.os[2];
      }
      if (b0 < b1) {
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
          const int r = (u * C::kSoftmax + tid) / (D / 8), c = (u * C::kSoftmax + tid) % (D / 8);
          *reinterpret_cast<uint4 *>(smem + C::kQOff + (c / 8) * N * 128 + r * 128 + (((c % 8) ^ (r & 7)) << 4)) = qx[u];
        }
        fence_proxy_async_smem();
        mbar_arrive(&bars->q_full);
      }
      if (kAhead && more) read_q(nx);
      wg_sync(wg);  // the rows' values
      float l[W];
#pragma unroll
      for (int r = 0; r < W; ++r) l[r] = 0.f;

      for (int at = b0; at < b1; ++at, ++blk) {
        const int buf = blk & 1;
        wait_all(&bars->s_full[buf], (blk >> 1) & 1);
        tc_fence_after();
        float x[W];
        tmem_ld_n<W>(tmem + lane_off + buf * N + c0, x);
        const int n0 = sp.token(at, wk.reverse), j = n0 + tok;
        const bool part = n0 < sp.all_lo || n0 + kBN > sp.all_hi;
#pragma unroll
        for (int r = 0; r < W; r += 4) {
          if constexpr (kMode != 0) {
            const float4 sl = *reinterpret_cast<const float4 *>(&info->slope2[c0 + r]);
            const int4 b = *reinterpret_cast<const int4 *>(&info->bias0[c0 + r]);
            const float s4[4] = {sl.x, sl.y, sl.z, sl.w};
            const int b4[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[r + e] = kMode == 2 ? cap(x[r + e], 0.f) : x[r + e] * scale2;
              x[r + e] = fmaf(s4[e], (float)(j - b4[e]), x[r + e]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[r + e] *= scale2;
          }
        }
        if (part) {
          // Tokens that no row sees are zeros in V; ones that only some rows see must
          // not hand an infinity or NaN to the others.  Each warpgroup does its share
          // of the channels.
          const bool none = j < sp.lo || j >= sp.hi, some = j < sp.all_lo || j >= sp.all_hi;
          bool lost = false;
          // A wait by parity needs the slot's filling before V's to be over, else it
          // returns a phase early.  The scores show that K of this block and V of two
          // blocks back have come; in a ring of fewer than three blocks the filling
          // before may be V of the last block, whose product is waited for (the next
          // one on that barrier needs this thread's weights of the block after this
          // one, so the phase cannot be passed over; another part's slots have all
          // been used up).
          if (C::kSlots < 3 * H && at > b0) wait_all(&bars->o_done[(blk - 1) & 1], ((blk - 1) >> 1) & 1);
          const int v0 = g + H * (min(at - b0 + 2, b1 - b0) + at - b0);  // V's first slot of the block
#pragma unroll 1
          for (int half = 0; half < H; ++half) {
            const int s = (v0 + half) % C::kSlots;
            wait_all(&bars->full[s], ((v0 + half) / C::kSlots) & 1);
            constexpr int kShare = C::kDH / 8 / C::kGroups;
            if (some && ok) lost |= clean_row<T>(smem + s * C::kSlot, tok, wg * kShare, kShare, none);
          }
          if constexpr (C::kGroups > 1) {
            // Where some rows see a token that others do not, the shares' findings meet.
            if (max(n0, sp.lo) < sp.all_lo || min(n0 + kBN, sp.hi) > sp.all_hi) {
              bars->lost[buf][wg][tok] = lost;
              asm volatile("bar.sync 3, 256;" ::: "memory");
              lost = bars->lost[buf][0][tok] | bars->lost[buf][1][tok];
            }
          }
#pragma unroll
          for (int r = 0; r < W; r += 4) {
            const int4 lo = *reinterpret_cast<const int4 *>(&info->lo[c0 + r]), hi = *reinterpret_cast<const int4 *>(&info->hi[c0 + r]);
            const int l4[4] = {lo.x, lo.y, lo.z, lo.w}, h4[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[r + e] = j >= l4[e] && j < h4[e] ? x[r + e] : -CUDART_INF_F;
          }
          if (lost) {  // the rows that see the token; scores and sums have nothing to do with V
#pragma unroll 1
            for (int r = c0; r < c0 + W; ++r)
              if (j >= info->lo[r] && j < info->hi[r]) info->scale[r] = CUDART_NAN_F;
          }
        }
        if (wk.score != nullptr && j < wk.pitch) {
          float *sc = wk.score + (((long long)cur.b * a.Hkv + cur.kvh) * wk.R + row0 + c0) * wk.pitch + j;
#pragma unroll
          for (int r = 0; r < W; ++r)
            if (c0 + r < rows) sc[r * wk.pitch] = x[r];
        }
        bool over = false;
#pragma unroll
        for (int r = 0; r < W; r += 4) {
          const float4 lim = *reinterpret_cast<const float4 *>(&info->limit[c0 + r]);
          over |= x[r] > lim.x || x[r + 1] > lim.y || x[r + 2] > lim.z || x[r + 3] > lim.w;
        }
        if (wg_any(wg, over)) {
          // Some score passes its row's limit: new references.
          {
            float mx[W];
#pragma unroll
            for (int r = 0; r < W; ++r) mx[r] = x[r];
            reduce_rows<W>(mx, [](float p, float q) { return fmaxf(p, q); });
            put_rows<W>(info->wmax[warp % 4] + c0, mx);
          }
          wg_sync(wg);
          if (tok < W) {
            const int row = c0 + tok;
            const float mx = fmaxf(fmaxf(info->wmax[0][row], info->wmax[1][row]), fmaxf(info->wmax[2][row], info->wmax[3][row]));
            const float old = info->ref[row];
            float alpha = 1.f;
            if (mx > info->limit[row]) {
              alpha = old == -CUDART_INF_F ? 1.f : ex2_approx(old - mx);
              info->ref[row] = mx;
              info->base[row] = mx - kShift;
              info->limit[row] = mx + weight_room<T>();
            }
            info->alpha[row] = alpha;
          }
          wg_sync(wg);
#pragma unroll
          for (int r = 0; r < W; r += 4) {
            const float4 al = *reinterpret_cast<const float4 *>(&info->alpha[c0 + r]);
            l[r] *= al.x;
            l[r + 1] *= al.y;
            l[r + 2] *= al.z;
            l[r + 3] *= al.w;
          }
          if (at > b0) {
            // O^T holds the blocks before once their products are done.
            wait_all(&bars->o_done[(blk - 1) & 1], ((blk - 1) >> 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int half = 0; half < H; ++half) {
              float o[W];
              tmem_ld_n<W>(tmem + lane_off + C::kO + half * N + c0, o);
#pragma unroll
              for (int r = 0; r < W; r += 4) {
                const float4 al = *reinterpret_cast<const float4 *>(&info->alpha[c0 + r]);
                o[r] *= al.x;
                o[r + 1] *= al.y;
                o[r + 2] *= al.z;
                o[r + 3] *= al.w;
              }
              tmem_st_n<W>(tmem + lane_off + C::kO + half * N + c0, o);
            }
            tmem_wait_st();
          }
        }
        uint8_t *const pt = smem + C::kPOff + buf * C::kP + c0 / 8 * 2048 + tok * 16;
#pragma unroll
        for (int r = 0; r < W; r += 8) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const float4 bs = *reinterpret_cast<const float4 *>(&info->base[c0 + r + e]);
            const float p0 = ex2_approx(x[r + e] - bs.x), p1 = ex2_approx(x[r + e + 1] - bs.y);
            const float p2 = ex2_approx(x[r + e + 2] - bs.z), p3 = ex2_approx(x[r + e + 3] - bs.w);
            l[r + e] += p0;
            l[r + e + 1] += p1;
            l[r + e + 2] += p2;
            l[r + e + 3] += p3;
            w[e / 2] = pack2<T>(p0, p1);
            w[e / 2 + 1] = pack2<T>(p2, p3);
          }
          *reinterpret_cast<uint4 *>(pt + (r / 8) * 2048) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&bars->p_full[buf]);
      }
      g += 2 * H * (b1 - b0);

      // ---- the part's end
      reduce_rows<W>(l, [](float p, float q) { return p + q; });
      put_rows<W>(info->wmax[warp % 4] + c0, l);
      if (b0 < b1) {
        // (The products complete in order, and those two blocks back are done, since
        // the last block's scores were issued after them: no phase is passed over.)
        wait_all(&bars->o_done[(blk - 1) & 1], ((blk - 1) >> 1) & 1);
        tc_fence_after();
      }
      wg_sync(wg);
      const bool whole = b0 == 0 && b1 == sp.blocks();
      const long long slot = 2LL * worker + (cur.at == 0 ? 1 : 0);
      if (tok < W && c0 + tok < rows) {
        const int row = c0 + tok;
        const float sum = (info->wmax[0][row] + info->wmax[1][row]) + (info->wmax[2][row] + info->wmax[3][row]);
        const int r = row0 + row;
        if (whole) {
          const int i = r / a.group, h = cur.kvh * a.group + r % a.group;
          const bool sees = info->hi[row] > info->lo[row];
          const float lse2 = info->ref[row] - kShift + log2f(sum);
          info->scale[row] = sees ? info->scale[row] / sum : 0.f;
          if (a.lse != nullptr)
            a.lse[((long long)cur.b * a.H + h) * a.Sq + i] =
                sees ? lse2 * kLn2 + (kMode != 0 && a.alibi != nullptr ? a.alibi[h] * (float)info->bias0[row] : 0.f) : -CUDART_INF_F;
          if (wk.stat != nullptr) wk.stat[((long long)cur.b * a.Hkv + cur.kvh) * wk.R + r] = lse2;
        } else {
          *reinterpret_cast<float2 *>(wk.part_ml + (slot * N + row) * 2) = make_float2(info->ref[row], sum);
        }
      }
      wg_sync(wg);
#pragma unroll 1
      for (int half = 0; half < H; ++half) {
        float o[W];
        if (b0 < b1) {
          tmem_ld_n<W>(tmem + lane_off + C::kO + half * N + c0, o);
        } else {
#pragma unroll
          for (int r = 0; r < W; ++r) o[r] = 0.f;
        }
        if (tok >= C::kDH) continue;
        const int ch = half * 128 + tok;
        if (whole) {
#pragma unroll
          for (int r = 0; r < W; ++r)
            if (c0 + r < rows) {
              // 0 for a row that sees nothing, and chosen so: the sums of a padded row,
              // which is not masked where all others see a block, may be anything.
              const float scale = info->scale[c0 + r];
              static_cast<T *>(a.o)[info->out[c0 + r] + ch] = Elem<T>::from_f(scale != 0.f ? o[r] * scale : 0.f);
            }
        } else {
          float *po = wk.part_o + (slot * N + c0) * D + ch;
#pragma unroll
          for (int r = 0; r < W; ++r)
            if (c0 + r < rows) po[r * D] = o[r] * info->scale[c0 + r];
        }
      }
      tc_fence_before();  // O^T is read before the next part's products write it
      wg_sync(wg);          // and the rows' values before they are set anew
      cur = nx;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over the shares of a unit
// that several CTAs have: a warp a row, a lane D / 32 channels, four rows a CTA.
constexpr int kMergeThreads = 128;
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const __grid_constant__ AttnArgs a,
                                                                     const __grid_constant__ StepWork wk, int rows) {
  constexpr int E = D / 32;
  __shared__ ScanShared sh;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int unit = blockIdx.x;
  const int rb = unit % wk.nrb, kvh = unit / wk.nrb % a.Hkv, b = unit / wk.nrb / a.Hkv;
  const int in_block = blockIdx.y * (kMergeThreads / 32) + warp;
  scan_steps(a, wk, rows, sh, [b](int x, int, int, int) { return x == b; });
  const int total = sh.total;
  int first = sh.before + sh.steps / a.Hkv * kvh;
  for (int i = 0; i < rb; ++i) first += span_of(a, wk.R, rows, b, i).steps();
  const Span sp = span_of(a, wk.R, rows, b, rb);
  const int n = share_count(wk, total);
  // The shares from the one that has the unit's first block on.
  const int w0 = share_of(total, first + min(kUnitSteps, sp.steps() - 1), n);
  const int used = share_of(total, first + sp.steps() - 1, n) - w0 + 1;
  const int slot0 = share_begin(total, w0, n) <= first ? 1 : 0;
  // Every thread waits for the shares, also where there is nothing to do, so
  // that this kernel ends after them.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (used <= 1) return;
  constexpr float kShift = weight_shift<T>();
  {
    const int r = rb * rows + in_block;
    if (in_block >= rows || r >= wk.R) return;
    auto slot = [&](int s) { return (2LL * (w0 + s) + (s == 0 ? slot0 : 0)) * rows + in_block; };
    // The maximum first (a lane a share), then the weighted sums.
    float m = -CUDART_INF_F;
    for (int s = lane; s < used; s += 32) m = fmaxf(m, wk.part_ml[slot(s) * 2]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    constexpr int kAtOnce = 8;
    for (int s0 = 0; s0 < used; s0 += kAtOnce) {
      float2 ml[kAtOnce];
      float x[kAtOnce][E];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        ml[u] = make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = 0.f;
        if (s0 + u < used) {
          const long long at = slot(s0 + u);
          ml[u] = *reinterpret_cast<const float2 *>(wk.part_ml + at * 2);
          const float *po = wk.part_o + at * D + lane * E;
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const float2 v = *reinterpret_cast<const float2 *>(po + e);
            x[u][e] = v.x;
            x[u][e + 1] = v.y;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const float w = ex2_approx(ml[u].x - base);
        l = fmaf(w, ml[u].y, l);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(w, x[u][e], o[e]);
      }
    }
    const int i = r / a.group, h = kvh * a.group + r % a.group;
    const Visible v = row_visible(a, i, sp.ql, sp.kl);
    const bool sees = v.hi > v.lo;
    const float inv = sees ? 1.f / l : 0.f;
    const float lse2 = m - kShift + log2f(l);
    T *op = static_cast<T *>(a.o) + b * a.os[0] + i * a.os[1] + h * a.os[2] + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(op + e) = sees ? pack2<T>(o[e] * inv, o[e + 1] * inv) : 0u;
    if (lane == 0) {
      if (a.lse != nullptr) {
        const float slope = a.alibi != nullptr ? a.alibi[h] : 0.f;
        a.lse[((long long)b * a.H + h) * a.Sq + i] =
            sees ? lse2 * kLn2 + (a.alibi != nullptr ? slope * (float)alibi_ref(v, slope) : 0.f) : -CUDART_INF_F;
      }
      if (wk.stat != nullptr) wk.stat[((long long)b * a.Hkv + kvh) * wk.R + r] = lse2;
    }
  }
}

// The weight of each cached token from the scores that the attention left:
// sum over rows of 2^(score - lse2).  A thread has four tokens.
constexpr int kWeightRows = 64;  // rows whose sums lie in shared memory at a time
constexpr int kWeightThreads = 128;
__global__ void __launch_bounds__(kWeightThreads) paged_weights_kernel(const __grid_constant__ AttnArgs a,
                                                                  const __grid_constant__ StepWork wk) {
  __shared__ float lse2[kWeightRows];
  __shared__ Visible vis[kWeightRows];
  const int unit = blockIdx.y;
  const int b = unit / a.Hkv, kvh = unit % a.Hkv;
  const int ql = clamp_len(a.q_lens, b, a.Sq), kl = clamp_len(a.kv_lens, b, a.Skv);
  const int j0 = (blockIdx.x * kWeightThreads + threadIdx.x) * 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)blockIdx.x * kWeightThreads * 4 >= kl) return;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  const int R = min(wk.R, ql * a.group);
  for (int r0 = 0; r0 < R; r0 += kWeightRows) {
    __syncthreads();
    const int n = min(kWeightRows, R - r0);
    for (int i = threadIdx.x; i < n; i += kWeightThreads) {
      const int r = r0 + i;
      lse2[i] = wk.stat[(long long)unit * wk.R + r];
      vis[i] = row_visible(a, r / a.group, ql, kl);
    }
    __syncthreads();
    if (j0 >= kl) continue;
    const float *sc = wk.score + ((long long)unit * wk.R + r0) * wk.pitch + j0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const Visible v = vis[i];
      if (v.lo >= v.hi || j0 + 3 < v.lo || j0 >= v.hi) continue;  // nothing was written where no row sees a token
      const float4 x = *reinterpret_cast<const float4 *>(sc + i * wk.pitch);
      const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j0 + e >= v.lo && j0 + e < v.hi) w[e] += ex2_approx(xs[e] - lse2[i]);
    }
  }
  if (j0 >= kl) return;
  const int page = paged_page(wk.c, b, j0 / wk.c.page_size);
  if (page < 0) return;
  float *to = wk.c.w + page * wk.c.ws[0] + kvh * wk.c.ws[1] + j0 % wk.c.page_size;
  const int old = wk.decay == 0.f ? 0 : (a.causal ? kl - ql : kl);  // tokens that had a weight before
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (j0 + e >= kl) break;
    to[e] = j0 + e < old ? fmaf(wk.decay, to[e], w[e]) : w[e];
  }
}

// -------------------------------------------------------------------- host
struct StepPlan {
  int rows;  // of a block: 16, 32 or 64
  int workers;
  bool split;
  size_t part_bytes, stat_bytes, score_bytes;
  long long pitch;
};

template <int N>
constexpr int ctas_of(int D) {
  return D == 64 ? StepCfg<64, N>::kCtas : (D == 128 ? StepCfg<128, N>::kCtas : StepCfg<256, N>::kCtas);
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// `weights`: the rows' sums are wanted; `scores`: and their scores kept.
StepPlan plan_step(const AttnArgs &a, bool weights, bool scores) {
  StepPlan p{};
  const long long R = (long long)a.Sq * a.group;
  p.rows = R <= 16 ? 16 : (R <= 32 || a.D != 256 ? 32 : 64);
  p.workers = a.num_sms * (p.rows == 16 ? ctas_of<16>(a.D) : (p.rows == 32 ? ctas_of<32>(a.D) : StepCfg<256, 64>::kCtas));
  // Up to two blocks a unit there is too little to share.  Steps are counted in 32 bits.
  const double steps = (double)a.B * a.Hkv * ((R + p.rows - 1) / p.rows) * (a.Skv / kBN + 2 + kUnitSteps);
  p.split = a.Skv > 2 * kBN && steps < 2147483647.0;
  p.part_bytes = p.split ? up256((size_t)2 * p.workers * p.rows * (a.D + 2) * sizeof(float)) : 0;
  p.stat_bytes = weights ? up256((size_t)a.B * a.Hkv * R * sizeof(float)) : 0;
  p.pitch = ((long long)a.Skv + 15) / 16 * 16;
  p.score_bytes = scores ? up256((size_t)a.B * a.Hkv * R * p.pitch * sizeof(float)) : 0;
  return p;
}

template <typename T, int D, int N, int kMode>
cudaError_t launch_step_t(const AttnArgs &a, const StepWork &wk, long long units, cudaStream_t s) {
  using C = StepCfg<D, N>;
  CUtensorMap tk, tv;
  if (!make_page_map(&tk, wk.c, wk.c.k, wk.c.ks, a.dtype, wk.box) || !make_page_map(&tv, wk.c, wk.c.v, wk.c.vs, a.dtype, wk.box))
    return cudaErrorInvalidValue;
  constexpr auto kern = paged_step_kernel<T, D, N, kMode>;
  const cudaError_t attr = allow_smem<kern>(C::kSmem);
  if (attr != cudaSuccess) return attr;
  const unsigned grid = (unsigned)(wk.split ? wk.workers : units);
  kern<<<grid, C::kThreads, C::kSmem, s>>>(tk, tv, a, wk);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (wk.split) {
    const dim3 grid_m((unsigned)units, (unsigned)((std::min(wk.R, N) + 3) / 4));
    e = launch_paged_after(paged_merge_kernel<T, D>, grid_m, kMergeThreads, 0, s, a, wk, N);
  }
  if (e != cudaSuccess || wk.score == nullptr) return e;
  const dim3 grid_w((unsigned)((a.Skv + kWeightThreads * 4 - 1) / (kWeightThreads * 4)), (unsigned)(a.B * a.Hkv));
  return launch_paged_after(paged_weights_kernel, grid_w, kWeightThreads, 0, s, a, wk);
}

template <typename T, int D, int N>
cudaError_t launch_step_m(const AttnArgs &a, const StepWork &wk, long long units, cudaStream_t s) {
  if (a.softcap > 0.f) return launch_step_t<T, D, N, 2>(a, wk, units, s);
  return a.alibi != nullptr ? launch_step_t<T, D, N, 1>(a, wk, units, s) : launch_step_t<T, D, N, 0>(a, wk, units, s);
}
template <typename T, int D>
cudaError_t launch_step_r(const AttnArgs &a, const StepWork &wk, int rows, long long units, cudaStream_t s) {
  if (rows == 16) return launch_step_m<T, D, 16>(a, wk, units, s);
  if constexpr (D == 256)
    if (rows == 64) return launch_step_m<T, D, 64>(a, wk, units, s);
  return launch_step_m<T, D, 32>(a, wk, units, s);
}

template <typename T>
cudaError_t launch_step_d(const AttnArgs &a, const StepWork &wk, int rows, long long units, cudaStream_t s) {
  switch (a.D) {
    case 64: return launch_step_r<T, 64>(a, wk, rows, units, s);
    case 128: return launch_step_r<T, 128>(a, wk, rows, units, s);
    case 256: return launch_step_r<T, 256>(a, wk, rows, units, s);
  }
  return cudaErrorNotSupported;
}

cudaError_t launch_step(const AttnArgs &a, const PagedArgs &c, const StepPlan &p, float decay, void *ws, cudaStream_t s) {
  StepWork wk{};
  wk.c = c;
  wk.R = a.Sq * a.group;
  wk.nrb = (wk.R + p.rows - 1) / p.rows;
  wk.workers = p.workers;
  // A share's least length: of 2 / 4 / 8 / 16 steps one sequence of 300 tokens takes 16 / 18 /
  // 25 / 35 us, one of 8192 25 / 23 / 27 / 33; 64 of 300 and longer batches take the same time.
  wk.min_steps = 2 + kUnitSteps;
  wk.split = p.split;
  wk.reverse = a.alibi != nullptr;
  wk.box = std::gcd(c.page_size, kBN);
  unsigned char *at = static_cast<unsigned char *>(ws);
  if (p.split) {
    wk.part_o = reinterpret_cast<float *>(at);
    wk.part_ml = wk.part_o + (size_t)2 * p.workers * p.rows * a.D;
    at += p.part_bytes;
  }
  if (p.stat_bytes != 0) wk.stat = reinterpret_cast<float *>(at);
  if (p.score_bytes != 0) wk.score = reinterpret_cast<float *>(at + p.stat_bytes);
  wk.pitch = p.pitch;
  wk.decay = decay;
  const long long units = (long long)a.B * a.Hkv * wk.nrb;
  return a.dtype == LLMX_FP16 ? launch_step_d<__half>(a, wk, p.rows, units, s)
                              : launch_step_d<__nv_bfloat16>(a, wk, p.rows, units, s);
}

llmx_status bad(const char *msg) { return record_error(LLMX_ERR_INVALID_ARGUMENT, msg); }

llmx_status prepare(const llmx_attn_params *p, const llmx_paged_cache *c, AttnArgs *a, PagedArgs *k) {
  llmx_status s = validate_without_kv(p, a);
  if (s != LLMX_OK) return s;
  s = validate_paged(c, p->batch, k);
  if (s != LLMX_OK) return s;
  if (p->dtype != c->dtype || p->n_kv_heads != c->n_kv_heads || p->head_dim != c->head_dim)
    return bad("paged attention: dtype, n_kv_heads and head_dim must be the cache's");
  if (p->kv_offset != 0 || p->kv_total != 0) return bad("paged attention: kv_offset and kv_total must be 0");
  if (p->max_kv_len > (long long)c->max_pages * c->page_size)
    return bad("paged attention: max_kv_len must be at most max_pages * page_size");
  if ((long long)a->Sq * a->group > (1LL << 30)) return bad("paged attention: max_q_len * group must be at most 2^30");
  if (p->algo == LLMX_ALGO_SIMT) return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: algo must be AUTO, DECODE or TCGEN05");
  if ((reinterpret_cast<uintptr_t>(a->q) & 15u) || (reinterpret_cast<uintptr_t>(a->o) & 15u))
    return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: q and o must be 16-byte aligned");
  const int extent[3] = {a->B, a->Sq, a->H};
  for (int i = 0; i < 3; ++i) {
    if (extent[i] == 1) a->qs[i] = a->os[i] = 0;  // never stepped along
    if (a->qs[i] % 8 || a->os[i] % 8)
      return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: strides of q and o must be multiples of 8");
    if (extent[i] > 1 && a->os[i] == 0) return bad("paged attention: rows of o must not overlap (stride 0)");
  }
  // Bytes of a stride of a tensor map stay below 2^40.
  const int kv_extent[3] = {k->n_pages, k->Hkv, k->page_size};
  for (int i = 0; i < 3; ++i)
    if (kv_extent[i] > 1 && (k->ks[i] >= (1LL << 39) || k->vs[i] >= (1LL << 39)))
      return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: strides of the cache must stay below 2^39 elements");
  const long long blocks = (long long)a->B * a->Hkv * (((long long)a->Sq * a->group + 15) / 16);
  if (blocks > INT_MAX / 2 || (k->w != nullptr && (long long)a->B * a->Hkv > 65535))
    return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: too many sequences, heads and rows for one call");
  a->window = std::min(a->window, 1 << 30);
  return LLMX_OK;
}

// A request's form and its workspace: [work counter][partial results][the
// rows' sums][scores].
struct Plan {
  bool tc;
  bool again;  // key weights by computing the scores again
  StepPlan step;
  PagedTcPlan tcp;
  size_t stat_at, bytes;
};

// Key weights: the scores of a few rows are kept, 8 bytes written and read a row
// and token (at 32 rows as much as K itself at head_dim 128), if that takes at
// most 1 GiB; otherwise they are computed again.  Kept / again, us, 32 heads on 8 of 128: 16
// sequences of 4096 tokens, 4 rows 75 / 118, 32 rows 103 / 129, 64 rows 180 / 170; one of
// 32768, 4 rows 51 / 76, 32 rows 72 / 78, 48 rows 97 / 87; three of 300-900, 16 rows 29 / 31,
// 32 rows 37 / 31.  The 1 GiB is for the memory's sake: 256 of 16384, 32 rows, 4 GiB of
// scores, take 4.42 ms kept and 5.70 again.
constexpr int kScoreRows = 32;
constexpr double kScoreBytes = double(1 << 30);
// Where they cannot be (more than 128 query heads a kv head, a q that is expanded) all are
// kept, as long as a tenth of the device's memory holds them.
constexpr double kMostScoreBytes = 16 * kScoreBytes;

llmx_status choose(const llmx_attn_params *p, const AttnArgs &a, const PagedArgs &k, Plan *plan) {
  const bool can = paged_tc_supports(a);
  if (p->algo == LLMX_ALGO_TCGEN05 && !can)
    return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: TCGEN05 needs sm_scale > 0 and at most 128 query heads a kv head");
  plan->tc = can && (p->algo == LLMX_ALGO_TCGEN05 || (p->algo == LLMX_ALGO_AUTO && (long long)a.Sq * a.group > kStepRows));
  const bool weights = k.w != nullptr;
  const long long R = (long long)a.Sq * a.group;
  if (plan->tc) {
    plan->again = weights;
    plan->tcp = plan_paged_tc(a, true);
    plan->stat_at = kCounterBytes + plan->tcp.part_bytes;
    plan->bytes = plan->stat_at + (weights ? (size_t)a.B * a.Hkv * R * sizeof(float) : 0);
  } else {
    // (In floating point: the number of scores may pass 64 bits.)
    const double kept = 4.0 * a.B * a.Hkv * (double)R * (((double)a.Skv + 15) / 16 * 16);
    plan->again = weights && (R > kScoreRows || kept > kScoreBytes) && paged_weights_supports(a);
    if (weights && !plan->again && kept > kMostScoreBytes)
      return record_error(LLMX_ERR_UNSUPPORTED,
                          "paged attention: key weights with more than 128 query heads a kv head, or of an expanded q, keep "
                          "every score, and this call's would pass 16 GiB");
    plan->step = plan_step(a, weights, weights && !plan->again);
    plan->stat_at = plan->step.part_bytes;
    plan->bytes = plan->step.part_bytes + plan->step.stat_bytes + plan->step.score_bytes;
  }
  return LLMX_OK;
}

}  // namespace
}  // namespace llmx_b200

using namespace llmx_b200;

extern "C" llmx_status llmx_paged_attn_workspace_size(const llmx_attn_params *p, const llmx_paged_cache *c, size_t *bytes) {
  if (bytes == nullptr) return bad("paged attention: bytes is NULL");
  AttnArgs a;
  PagedArgs k;
  const llmx_status s = prepare(p, c, &a, &k);
  if (s != LLMX_OK) return s;
  unsigned int *err = nullptr;
  int sms = 0;
  if (current_device_info(&err, &sms) == LLMX_OK) a.num_sms = sms;
  Plan plan;
  const llmx_status st = choose(p, a, k, &plan);
  if (st == LLMX_OK) *bytes = plan.bytes;
  return st;
}

extern "C" llmx_status llmx_paged_attn_fwd(const llmx_attn_params *p, const llmx_paged_cache *c, float decay, void *stream) {
  AttnArgs a;
  PagedArgs k;
  llmx_status s = prepare(p, c, &a, &k);
  if (s != LLMX_OK) return s;
  if (k.w != nullptr && !(decay >= 0.f && decay <= 3.4e38f)) return bad("paged attention: decay must be finite and >= 0");
  if (k.w != nullptr && p->q == p->o) return bad("paged attention: with key_weights o must not be q, which is read again");
  if (reinterpret_cast<uintptr_t>(p->workspace) & 15u) return bad("paged attention: workspace must be 16-byte aligned");
  Plan plan;
  s = choose(p, a, k, &plan);
  if (s != LLMX_OK) return s;
  s = current_device_info(&a.err, &a.num_sms);
  if (s != LLMX_OK) return s;
  k.err = a.err;
  s = choose(p, a, k, &plan);  // with the device's SM count
  if (s != LLMX_OK) return s;
  const size_t have = p->workspace != nullptr ? p->workspace_bytes : 0;
  if (have < plan.bytes) {
    if (k.w != nullptr)
      return record_error(LLMX_ERR_WORKSPACE_TOO_SMALL, "paged attention: key_weights need the workspace");
    plan.step.split = false;
    plan.step.part_bytes = 0;
    if (plan.tc) plan.tcp = plan_paged_tc(a, false);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  unsigned char *ws = static_cast<unsigned char *>(p->workspace);
  float *const stat = k.w != nullptr ? reinterpret_cast<float *>(ws + plan.stat_at) : nullptr;
  if (plan.tc) {
    int *const ctr = have >= kCounterBytes ? reinterpret_cast<int *>(ws) : nullptr;
    float *const part = plan.tcp.part_bytes > 0 ? reinterpret_cast<float *>(ws + kCounterBytes) : nullptr;
    e = launch_paged_tc(a, k, plan.tcp, ctr, part, stat, st);
  } else {
    e = launch_step(a, k, plan.step, decay, ws, st);
  }
  if (e == cudaSuccess && plan.again) e = launch_paged_weights(a, k, stat, decay, st);
  return e == cudaSuccess ? LLMX_OK : record_error(LLMX_ERR_CUDA, cudaGetErrorString(e));
}
