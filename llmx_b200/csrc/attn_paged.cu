// Attention over a paged 16-bit key/value cache (include/llmx_attn.h): the
// request's checks and the choice between its two forms, and the form for few
// query rows, which streams K and V once past all rows of a kv head.
//
// Work.  A unit is one (sequence, kv head) and a block of up to 16 * RT packed
// rows.  Its visible tokens are taken in steps of 64, 16 of which belong to one
// page, whatever the page size.  The steps of all units, end to end, are dealt
// to the resident CTAs in equal shares, so that sequences of any lengths finish
// together; a CTA writes the result of a unit that it has whole and a partial
// result (unnormalised O, maximum and sum; at most two a CTA) of one that it
// shares, which a second, overlapped launch merges.
//
// A CTA's four warps hold RT row tiles of 16 rows, and 4 / RT warps of a row
// tile take different 16 tokens of a step and are merged in shared memory at
// the unit's end.  K and V go through a ring of steps in shared memory by
// 16-byte asynchronous copies, which write zeros for tokens that no row sees
// (nothing behind a sequence's length is read), swizzled so that the matrix
// loads of the fragments are free of conflicts; the next step's page is looked
// up one step ahead.  Products are m16n8k16 with fp32 sums.  At 16 rows a step
// of head_dim 128 costs a warp about 700 cycles against 2800 that its 32 KB
// cost an SM at the HBM rate, which is why the legacy matrix instruction is
// enough here and tiles of 128 rows (attn_paged_tc.cu) start above 64 rows.
//
// Masked tokens.  A NaN or an infinity in K only reaches scores that are
// replaced.  One in V would reach every row of the tile through 0 * V, so in
// steps that some rows see and others do not such values are taken as 0 and
// the rows that see their token become NaN.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "paged_attn.cuh"
#include "sm100_ptx.cuh"

namespace llmx_b200 {
namespace {

using sm100::smem_u32;

constexpr int kThreads = 128;
constexpr int kWarps = 4;
constexpr int kStep = 64;  // tokens of a step
constexpr int kStepRows = 64;  // AUTO: packed rows of a kv head up to which this form is taken
constexpr size_t kCounterBytes = 256;

// fp16 weights are taken 2^10 times as large: a weight 2^-24 of the largest
// still has 10 bits then; bf16 has the exponents of fp32.
template <typename T>
constexpr float weight_shift() {
  return std::is_same<T, __half>::value ? 10.f : 0.f;
}

// A launch's units and shares.
struct StepWork {
  PagedArgs c;
  int R;          // packed rows of a kv head
  int nrb;        // row blocks
  int workers;    // CTAs that take a share, at most
  int min_steps;  // a share is at least this long
  int split;      // 0: CTA i has unit i whole
  float *part_o;  // [2 workers][rows of a block][D]
  float *part_ml;  // [2 workers][rows of a block][2]
  float *stat;     // nullable [B * Hkv][R]: log2 of the sum of 2^score
  float *score;    // nullable [B * Hkv][R][pitch], log2 units
  long long pitch;
  float decay;
};

// Steps of row block rb of sequence b: tokens lo16 + 64 i .., those in [lo, hi)
// are visible to some row.  At least one step, which may have no token.
struct Span {
  int ql, kl, lo, hi, q0, q1;  // q0 .. q1: query rows of the block
  __device__ __forceinline__ int lo16() const { return lo & ~15; }
  __device__ __forceinline__ int steps() const { return max(1, (hi - lo16() + kStep - 1) / kStep); }
};
__device__ __forceinline__ Span span_of(const AttnArgs &a, int R, int rows, int b, int rb) {
  Span s;
  s.ql = clamp_len(a.q_lens, b, a.Sq);
  s.kl = clamp_len(a.kv_lens, b, a.Skv);
  s.q0 = rb * rows / a.group;
  s.q1 = min(s.ql, (min(R, (rb + 1) * rows) - 1) / a.group + 1);
  s.lo = s.hi = 0;
  if (s.q0 < s.q1) {
    const Visible first = row_visible(a, s.q0, s.ql, s.kl), last = row_visible(a, s.q1 - 1, s.ql, s.kl);
    s.lo = first.lo;
    s.hi = last.hi;
    if (s.hi <= s.lo) s.lo = s.hi = 0;
  }
  return s;
}

// Steps of all units of sequence b.
__device__ __forceinline__ long long steps_of(const AttnArgs &a, const StepWork &wk, int rows, int b) {
  long long n = 0;
  for (int rb = 0; rb < wk.nrb; ++rb) n += span_of(a, wk.R, rows, b, rb).steps();
  return n * a.Hkv;
}

// Shares: worker w of n has the steps [total * w / n, total * (w + 1) / n).
__device__ __forceinline__ int share_count(const StepWork &wk, long long total) {
  return (int)max(1LL, min((long long)wk.workers, total / wk.min_steps));
}
__device__ __forceinline__ long long share_begin(long long total, int w, int n) { return total * w / n; }
__device__ __forceinline__ int share_of(long long total, long long step, int n) {
  int w = (int)(step * n / total);
  while (w > 0 && share_begin(total, w, n) > step) --w;
  while (w < n - 1 && share_begin(total, w + 1, n) <= step) ++w;
  return w;
}

// A scan over the sequences by the whole CTA: the steps before sequence b, of
// sequence b, and of all.  pick(b, before, steps) says which b is meant.
struct ScanShared {
  long long warp_sum[kWarps];
  long long before, total;
  int b;
};
template <typename F>
__device__ void scan_steps(const AttnArgs &a, const StepWork &wk, int rows, ScanShared &sh, F pick) {
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  long long base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid;
    const long long mine = b < a.B ? steps_of(a, wk, rows, b) : 0;
    long long x = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += o;
    }
    if (lane == 31) sh.warp_sum[warp] = x;
    __syncthreads();
    long long before = base;
    for (int w = 0; w < warp; ++w) before += sh.warp_sum[w];
    before += x - mine;
    if (b < a.B && pick(b, before, mine)) {
      sh.b = b;
      sh.before = before;
    }
    for (int w = 0; w < kWarps; ++w) base += sh.warp_sum[w];
    __syncthreads();
  }
  if (tid == 0) sh.total = base;
  __syncthreads();
}

// ------------------------------------------------------------- instructions
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}
// The halves of w that are infinite or NaN become 0; bits says which.
template <typename T>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w, int &bits) {
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  bits = 0;
  if ((w & kExp) == kExp) {
    bits |= 1;
    w &= 0xffff0000u;
  }
  if ((w & (kExp << 16)) == (kExp << 16)) {
    bits |= 2;
    w &= 0x0000ffffu;
  }
  return w;
}

// ------------------------------------------------------------------ kernel
// Steps in the ring and CTAs an SM: 64 KB and more of copies in flight an SM.
template <int D>
struct StepCfg {
  static constexpr int kStepBytes = 2 * kStep * D * 2;  // K and V
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kCtas = D == 64 ? 3 : (D == 128 ? 2 : 1);
  // A row tile's O in fragments (and m, l) for the merge of a row tile's warps:
  // at most two are handed over at a time.
  static constexpr int kTileFloats = 16 * D + 8 * 4;
  static constexpr int kSmem = kStages * kStepBytes + 2 * kTileFloats * 4;
  static_assert(kCtas * (kSmem + 1024 + 256) <= 228 * 1024, "shared memory of an SM");
};

// The result of a part of a unit, or of the whole: rows of one warp.
template <typename T, int D, int RT>
__global__ void __launch_bounds__(kThreads, StepCfg<D>::kCtas)
    paged_step_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ StepWork wk) {
  using C = StepCfg<D>;
  constexpr int kRows = 16 * RT;
  constexpr int kKG = kWarps / RT;  // warps of a row tile
  constexpr int kKS = D / 16;       // products of a score
  constexpr int kNT = D / 8;        // column tiles of O
  constexpr int kChunks = D / 8;    // 16-byte chunks of a token
  constexpr int kRowBytes = D * 2;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ ScanShared sh;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int g = lane / 4, t = lane % 4;
  const int rt = warp % RT, kg = warp / RT;
  const uint32_t ring = smem_u32(smem);
  float *const hand = reinterpret_cast<float *>(smem + C::kStages * C::kStepBytes);

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's share: `left` steps from step `at` of unit (b, kvh, rb) on
  struct Cursor {
    int b, kvh, rb, at;
    Span sp;
  };
  Cursor cur;
  long long left;
  const int worker = blockIdx.x;
  if (wk.split) {
    scan_steps(a, wk, kRows, sh, [](int, long long, long long) { return false; });
    const long long total = sh.total;
    const int n = share_count(wk, total);
    if (worker >= n) return;
    const long long begin = share_begin(total, worker, n);
    left = share_begin(total, worker + 1, n) - begin;
    if (left <= 0) return;
    __syncthreads();
    scan_steps(a, wk, kRows, sh, [begin](int, long long before, long long steps) { return before <= begin && begin < before + steps; });
    cur.b = sh.b;
    long long within = begin - sh.before;
    const long long per_head = steps_of(a, wk, kRows, cur.b) / a.Hkv;
    cur.kvh = (int)(within / per_head);
    within -= cur.kvh * per_head;
    for (cur.rb = 0;; ++cur.rb) {
      cur.sp = span_of(a, wk.R, kRows, cur.b, cur.rb);
      if (within < cur.sp.steps()) break;
      within -= cur.sp.steps();
    }
    cur.at = (int)within;
  } else {
    cur.rb = worker % wk.nrb;
    const int u = worker / wk.nrb;
    cur.kvh = u % a.Hkv;
    cur.b = u / a.Hkv;
    cur.sp = span_of(a, wk.R, kRows, cur.b, cur.rb);
    cur.at = 0;
    left = cur.sp.steps();
  }
  auto next_unit = [&](Cursor &c) {
    c.at = 0;
    if (++c.rb == wk.nrb) {
      c.rb = 0;
      if (++c.kvh == a.Hkv) {
        c.kvh = 0;
        ++c.b;
      }
    }
    c.sp = span_of(a, wk.R, kRows, c.b, c.rb);
  };

  // ---- copies.  Warp w copies tokens 16 w .. of each step.
  Cursor pre = cur;  // the next step to be copied
  long long pre_left = left;
  auto first_token = [&](const Cursor &c) { return c.sp.lo16() + c.at * kStep + warp * 16; };
  // The page of the warp's tokens of the step, or -1 where there is nothing to read.
  auto look_up = [&](const Cursor &c) {
    const int j = first_token(c);
    return j < c.sp.hi ? paged_page(wk.c, c.b, j / wk.c.page_size) : -1;
  };
  int page = look_up(pre);
  auto copy_step = [&](int stage) {
    if (pre_left > 0) {
      const int j = first_token(pre);
      const int in_page = j % wk.c.page_size;
      constexpr int kPerPass = 32 / kChunks;  // tokens of one instruction
      const int row0 = lane / kChunks, chunk = lane % kChunks;
      const long long pg = max(page, 0);
      const T *const kp = static_cast<const T *>(wk.c.k) + pg * wk.c.ks[0] + pre.kvh * wk.c.ks[1] + chunk * 8;
      const T *const vp = static_cast<const T *>(wk.c.v) + pg * wk.c.vs[0] + pre.kvh * wk.c.vs[1] + chunk * 8;
      const uint32_t dst = ring + stage * C::kStepBytes;
#pragma unroll
      for (int i = 0; i < 16 / kPerPass; ++i) {
        const int row = i * kPerPass + row0;
        const bool valid = page >= 0 && j + row >= pre.sp.lo && j + row < pre.sp.hi;
        const long long tok = valid ? in_page + row : 0;
        const uint32_t at = (warp * 16 + row) * kRowBytes + ((chunk ^ (row & 7)) << 4);
        cp_async16(dst + at, kp + tok * wk.c.ks[2], valid);
        cp_async16(dst + kStep * kRowBytes + at, vp + tok * wk.c.vs[2], valid);
      }
      if (--pre_left > 0) {
        if (++pre.at == pre.sp.steps()) next_unit(pre);
        page = look_up(pre);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) copy_step(i);

  const float scale2 = a.sm_scale * kPagedLog2e;
  const float cap_in = a.softcap > 0.f ? a.sm_scale / a.softcap : 0.f, cap_out = a.softcap * kPagedLog2e;
  constexpr float kShift = weight_shift<T>();
  int stage = 0;

  while (left > 0) {
    // ---- a unit, or the share's part of it
    const Span sp = cur.sp;
    const int part0 = cur.at, part1 = (int)min((long long)sp.steps(), part0 + left);
    uint32_t qf[kKS][4];
    float slope2[2];
    Visible vis[2];
    int ref[2];
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
      const int r = cur.rb * kRows + rt * 16 + g + 8 * rr;
      const int i = r / a.group, h = cur.kvh * a.group + r % a.group;
      const bool real = r < wk.R && i < sp.ql;
      vis[rr] = real ? row_visible(a, i, sp.ql, sp.kl) : Visible{0, 0};
      const float slope = a.alibi != nullptr && real ? a.alibi[h] : 0.f;
      slope2[rr] = slope * kPagedLog2e;
      ref[rr] = alibi_ref(vis[rr], slope);
      const T *qp = static_cast<const T *>(a.q) + (real ? cur.b * a.qs[0] + i * a.qs[1] + h * a.qs[2] : 0) + 2 * t;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        qf[ks][rr] = real ? *reinterpret_cast<const uint32_t *>(qp + ks * 16) : 0u;
        qf[ks][2 + rr] = real ? *reinterpret_cast<const uint32_t *>(qp + ks * 16 + 8) : 0u;
      }
    }
    // Every row of the block sees the tokens [all_lo, all_hi).
    const int all_lo = sp.q0 < sp.q1 ? row_visible(a, sp.q1 - 1, sp.ql, sp.kl).lo : 0;
    const int all_hi = sp.q0 < sp.q1 ? row_visible(a, sp.q0, sp.ql, sp.kl).hi : 0;
    const bool mixed = sp.q1 - sp.q0 > 1;  // rows that see different tokens
    float o[kNT][4], m[2], l[2];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;

    for (int at = part0; at < part1; ++at) {
      cp_async_wait<C::kStages - 2>();
      __syncthreads();
      copy_step(stage == 0 ? C::kStages - 1 : stage - 1);
      const uint32_t kbase = ring + stage * C::kStepBytes, vbase = kbase + kStep * kRowBytes;
      stage = stage == C::kStages - 1 ? 0 : stage + 1;
#pragma unroll 1
      for (int sub = kg; sub < 4; sub += kKG) {
        const int j0 = sp.lo16() + at * kStep + sub * 16;
        if (j0 >= sp.hi) break;
        // ---- scores of 16 rows and 16 tokens
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
        {
          const int key = ((lane >> 4) << 3) + (lane & 7);
          const uint32_t row = kbase + (sub * 16 + key) * kRowBytes;
          const int half = (lane >> 3) & 1;
#pragma unroll
          for (int ks = 0; ks < kKS; ++ks) {
            uint32_t kf[4];
            ldmatrix4(row + (((2 * ks + half) ^ (key & 7)) << 4), kf);
            mma16816<T>(s[0], qf[ks], kf[0], kf[1]);
            mma16816<T>(s[1], qf[ks], kf[2], kf[3]);
          }
        }
        const bool need_mask = j0 < all_lo || j0 + 16 > all_hi;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rr = i >> 1, j = j0 + n * 8 + 2 * t + (i & 1);
            float x = a.softcap > 0.f ? tanhf(s[n][i] * cap_in) * cap_out : s[n][i] * scale2;
            if (a.alibi != nullptr) x = fmaf(slope2[rr], (float)(j - ref[rr]), x);
            if (need_mask && (j < vis[rr].lo || j >= vis[rr].hi)) x = -CUDART_INF_F;
            s[n][i] = x;
          }
        if (wk.score != nullptr) {
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) {
            const int r = cur.rb * kRows + rt * 16 + g + 8 * rr;
            if (r < wk.R) {
              float *sc = wk.score + (((long long)cur.b * a.Hkv + cur.kvh) * wk.R + r) * wk.pitch + j0 + 2 * t;
              *reinterpret_cast<float2 *>(sc) = make_float2(s[0][2 * rr], s[0][2 * rr + 1]);
              *reinterpret_cast<float2 *>(sc + 8) = make_float2(s[1][2 * rr], s[1][2 * rr + 1]);
            }
          }
        }
        // ---- running maximum and sum
        float alpha[2];
        bool moved = false;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          float mx = fmaxf(fmaxf(s[0][2 * rr], s[0][2 * rr + 1]), fmaxf(s[1][2 * rr], s[1][2 * rr + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          alpha[rr] = 1.f;
          if (mx > m[rr]) {
            alpha[rr] = ex2(m[rr] - mx);
            m[rr] = mx;
            moved = true;
          }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) l[rr] *= alpha[rr];
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= alpha[i >> 1];
        }
        uint32_t pf[4];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const float base = (m[rr] == -CUDART_INF_F ? 0.f : m[rr]) - kShift;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float p0 = ex2(s[n][2 * rr] - base), p1 = ex2(s[n][2 * rr + 1] - base);
            l[rr] += p0 + p1;
            pf[2 * n + rr] = pack2<T>(p0, p1);
          }
        }
        // ---- O += P V
        {
          const int key = (((lane >> 3) & 1) << 3) + (lane & 7);
          const uint32_t row = vbase + (sub * 16 + key) * kRowBytes;
          const int half = lane >> 4;
          if (!(need_mask && mixed)) {
#pragma unroll
            for (int n = 0; n < kNT; n += 2) {
              uint32_t vf[4];
              ldmatrix4_trans(row + (((n + half) ^ (key & 7)) << 4), vf);
              mma16816<T>(o[n], pf, vf[0], vf[1]);
              mma16816<T>(o[n + 1], pf, vf[2], vf[3]);
            }
          } else {
            uint32_t lost = 0;  // tokens of the 16 with an infinity or NaN in V
#pragma unroll
            for (int n = 0; n < kNT; n += 2) {
              uint32_t vf[4];
              ldmatrix4_trans(row + (((n + half) ^ (key & 7)) << 4), vf);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                int bits;
                vf[i] = finite_or_zero<T>(vf[i], bits);
                lost |= (uint32_t)bits << (2 * t + 8 * (i & 1));
              }
              mma16816<T>(o[n], pf, vf[0], vf[1]);
              mma16816<T>(o[n + 1], pf, vf[2], vf[3]);
            }
            lost = __reduce_or_sync(0xffffffffu, lost);
            if (lost != 0) {
#pragma unroll
              for (int rr = 0; rr < 2; ++rr) {
                const int lo = min(max(vis[rr].lo - j0, 0), 16), hi = min(max(vis[rr].hi - j0, 0), 16);
                if (hi > lo && (lost & ((1u << hi) - (1u << lo))) != 0) l[rr] = CUDART_NAN_F;
              }
            }
          }
        }
      }
    }

    // ---- the unit's end: the sums of a row's four lanes, then its warps
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 1);
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 2);
    }
#pragma unroll
    for (int half = kKG / 2; half >= 1; half /= 2) {
      if (kg >= half && kg < 2 * half) {
        float *const buf = hand + ((kg - half) * RT + rt) * C::kTileFloats;
#pragma unroll
        for (int n = 0; n < kNT; ++n)
          *reinterpret_cast<float4 *>(buf + (n * 32 + lane) * 4) = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
        if (t == 0) *reinterpret_cast<float4 *>(buf + 16 * D + g * 4) = make_float4(m[0], m[1], l[0], l[1]);
      }
      __syncthreads();
      if (kg < half) {
        const float *const buf = hand + (kg * RT + rt) * C::kTileFloats;
        const float4 ml = *reinterpret_cast<const float4 *>(buf + 16 * D + g * 4);
        const float om[2] = {ml.x, ml.y}, ol[2] = {ml.z, ml.w};
        float w0[2], w1[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const float mn = fmaxf(m[rr], om[rr]);
          const float base = mn == -CUDART_INF_F ? 0.f : mn;
          w0[rr] = ex2(m[rr] - base);
          w1[rr] = ex2(om[rr] - base);
          m[rr] = mn;
          l[rr] = l[rr] * w0[rr] + ol[rr] * w1[rr];
        }
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          const float4 x = *reinterpret_cast<const float4 *>(buf + (n * 32 + lane) * 4);
          o[n][0] = o[n][0] * w0[0] + x.x * w1[0];
          o[n][1] = o[n][1] * w0[0] + x.y * w1[0];
          o[n][2] = o[n][2] * w0[1] + x.z * w1[1];
          o[n][3] = o[n][3] * w0[1] + x.w * w1[1];
        }
      }
      __syncthreads();
    }
    if (kg == 0) {
      const bool whole = part0 == 0 && part1 == sp.steps();
      const long long slot = 2LL * worker + (part0 == 0 ? 1 : 0);
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const int in_block = rt * 16 + g + 8 * rr, r = cur.rb * kRows + in_block;
        if (r >= wk.R) continue;
        if (whole) {
          const int i = r / a.group, h = cur.kvh * a.group + r % a.group;
          const bool sees = vis[rr].hi > vis[rr].lo;
          const float inv = sees ? 1.f / l[rr] : 0.f;
          const float lse2 = m[rr] - kShift + log2f(l[rr]);
          T *op = static_cast<T *>(a.o) + cur.b * a.os[0] + i * a.os[1] + h * a.os[2] + 2 * t;
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            *reinterpret_cast<uint32_t *>(op + n * 8) = sees ? pack2<T>(o[n][2 * rr] * inv, o[n][2 * rr + 1] * inv) : 0u;
          if (t == 0) {
            if (a.lse != nullptr)
              a.lse[((long long)cur.b * a.H + h) * a.Sq + i] =
                  sees ? lse2 * kPagedLn2 + (a.alibi != nullptr ? a.alibi[h] * (float)ref[rr] : 0.f) : -CUDART_INF_F;
            if (wk.stat != nullptr) wk.stat[((long long)cur.b * a.Hkv + cur.kvh) * wk.R + r] = lse2;
          }
        } else {
          float *po = wk.part_o + (slot * kRows + in_block) * D + 2 * t;
#pragma unroll
          for (int n = 0; n < kNT; ++n) *reinterpret_cast<float2 *>(po + n * 8) = make_float2(o[n][2 * rr], o[n][2 * rr + 1]);
          if (t == 0) *reinterpret_cast<float2 *>(wk.part_ml + (slot * kRows + in_block) * 2) = make_float2(m[rr], l[rr]);
        }
      }
    }
    left -= part1 - part0;
    if (left > 0) next_unit(cur);
  }
  cp_async_wait<0>();
}

// O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over the shares of a unit
// that several CTAs have: a CTA a unit, a warp a row, a lane D / 32 channels.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_merge_kernel(const __grid_constant__ AttnArgs a,
                                                                const __grid_constant__ StepWork wk, int rows) {
  constexpr int E = D / 32;
  __shared__ ScanShared sh;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int unit = blockIdx.x;
  const int rb = unit % wk.nrb, kvh = unit / wk.nrb % a.Hkv, b = unit / wk.nrb / a.Hkv;
  scan_steps(a, wk, rows, sh, [b](int x, long long, long long) { return x == b; });
  const long long total = sh.total;
  long long first = sh.before + steps_of(a, wk, rows, b) / a.Hkv * kvh;
  for (int i = 0; i < rb; ++i) first += span_of(a, wk.R, rows, b, i).steps();
  const Span sp = span_of(a, wk.R, rows, b, rb);
  const int n = share_count(wk, total);
  const int w0 = share_of(total, first, n), used = share_of(total, first + sp.steps() - 1, n) - w0 + 1;
  // Every thread waits for the shares, also where there is nothing to do, so
  // that this kernel ends after them.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (used <= 1) return;
  constexpr float kShift = weight_shift<T>();
  for (int in_block = warp; in_block < rows; in_block += kWarps) {
    const int r = rb * rows + in_block;
    if (r >= wk.R) break;
    auto slot = [&](int s) { return (2LL * (w0 + s) + (s == 0 ? 1 : 0)) * rows + in_block; };
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
        const float w = ex2(ml[u].x - base);
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
            sees ? lse2 * kPagedLn2 + (a.alibi != nullptr ? slope * (float)alibi_ref(v, slope) : 0.f) : -CUDART_INF_F;
      }
      if (wk.stat != nullptr) wk.stat[((long long)b * a.Hkv + kvh) * wk.R + r] = lse2;
    }
  }
}

// The weight of each cached token from the scores that the attention left:
// sum over rows of 2^(score - lse2).  A thread has four tokens.
constexpr int kWeightRows = 64;  // rows whose sums lie in shared memory at a time
__global__ void __launch_bounds__(kThreads) paged_weights_kernel(const __grid_constant__ AttnArgs a,
                                                                  const __grid_constant__ StepWork wk) {
  __shared__ float lse2[kWeightRows];
  __shared__ Visible vis[kWeightRows];
  const int unit = blockIdx.y;
  const int b = unit / a.Hkv, kvh = unit % a.Hkv;
  const int ql = clamp_len(a.q_lens, b, a.Sq), kl = clamp_len(a.kv_lens, b, a.Skv);
  const int j0 = (blockIdx.x * kThreads + threadIdx.x) * 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)blockIdx.x * kThreads * 4 >= kl) return;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  const int R = min(wk.R, ql * a.group);
  for (int r0 = 0; r0 < R; r0 += kWeightRows) {
    __syncthreads();
    const int n = min(kWeightRows, R - r0);
    for (int i = threadIdx.x; i < n; i += kThreads) {
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
        if (j0 + e >= v.lo && j0 + e < v.hi) w[e] += ex2(xs[e] - lse2[i]);
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
  int rt;  // row tiles: 1, 2 or 4
  int workers;
  bool split;
  size_t part_bytes, stat_bytes, score_bytes;
  long long pitch;
};

int ctas_of(int D) { return D == 64 ? StepCfg<64>::kCtas : (D == 128 ? StepCfg<128>::kCtas : StepCfg<256>::kCtas); }

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// `weights`: the rows' sums are wanted; `scores`: and their scores kept.
StepPlan plan_step(const AttnArgs &a, bool weights, bool scores) {
  StepPlan p{};
  const long long R = (long long)a.Sq * a.group;
  p.rt = R <= 16 ? 1 : (R <= 32 ? 2 : 4);
  const int rows = 16 * p.rt;
  p.workers = a.num_sms * ctas_of(a.D);
  // Up to four steps a unit there is too little to share.
  p.split = a.Skv > 4 * kStep;
  p.part_bytes = p.split ? up256((size_t)2 * p.workers * rows * (a.D + 2) * sizeof(float)) : 0;
  p.stat_bytes = weights ? up256((size_t)a.B * a.Hkv * R * sizeof(float)) : 0;
  p.pitch = ((long long)a.Skv + 15) / 16 * 16;
  p.score_bytes = scores ? up256((size_t)a.B * a.Hkv * R * p.pitch * sizeof(float)) : 0;
  return p;
}

template <typename T, int D, int RT>
cudaError_t launch_step_t(const AttnArgs &a, const StepWork &wk, long long units, cudaStream_t s) {
  auto kern = paged_step_kernel<T, D, RT>;
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  std::call_once(once, [&] {
    attr = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, StepCfg<D>::kSmem);
  });
  if (attr != cudaSuccess) return attr;
  const unsigned grid = (unsigned)(wk.split ? wk.workers : units);
  kern<<<grid, kThreads, StepCfg<D>::kSmem, s>>>(a, wk);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (wk.split) e = launch_paged_after(paged_merge_kernel<T, D>, dim3((unsigned)units), kThreads, 0, s, a, wk, 16 * RT);
  if (e != cudaSuccess || wk.score == nullptr) return e;
  const dim3 grid_w((unsigned)((a.Skv + kThreads * 4 - 1) / (kThreads * 4)), (unsigned)(a.B * a.Hkv));
  return launch_paged_after(paged_weights_kernel, grid_w, kThreads, 0, s, a, wk);
}

template <typename T, int D>
cudaError_t launch_step_r(const AttnArgs &a, const StepWork &wk, int rt, long long units, cudaStream_t s) {
  switch (rt) {
    case 1: return launch_step_t<T, D, 1>(a, wk, units, s);
    case 2: return launch_step_t<T, D, 2>(a, wk, units, s);
    default: return launch_step_t<T, D, 4>(a, wk, units, s);
  }
}

template <typename T>
cudaError_t launch_step_d(const AttnArgs &a, const StepWork &wk, int rt, long long units, cudaStream_t s) {
  switch (a.D) {
    case 64: return launch_step_r<T, 64>(a, wk, rt, units, s);
    case 128: return launch_step_r<T, 128>(a, wk, rt, units, s);
    case 256: return launch_step_r<T, 256>(a, wk, rt, units, s);
  }
  return cudaErrorNotSupported;
}

cudaError_t launch_step(const AttnArgs &a, const PagedArgs &c, const StepPlan &p, float decay, void *ws, cudaStream_t s) {
  StepWork wk{};
  wk.c = c;
  wk.R = a.Sq * a.group;
  wk.nrb = (wk.R + 16 * p.rt - 1) / (16 * p.rt);
  wk.workers = p.workers;
  wk.min_steps = 4;
  wk.split = p.split;
  unsigned char *at = static_cast<unsigned char *>(ws);
  if (p.split) {
    wk.part_o = reinterpret_cast<float *>(at);
    wk.part_ml = wk.part_o + (size_t)2 * p.workers * 16 * p.rt * a.D;
    at += p.part_bytes;
  }
  if (p.stat_bytes != 0) wk.stat = reinterpret_cast<float *>(at);
  if (p.score_bytes != 0) wk.score = reinterpret_cast<float *>(at + p.stat_bytes);
  wk.pitch = p.pitch;
  wk.decay = decay;
  const long long units = (long long)a.B * a.Hkv * wk.nrb;
  return a.dtype == LLMX_FP16 ? launch_step_d<__half>(a, wk, p.rt, units, s)
                              : launch_step_d<__nv_bfloat16>(a, wk, p.rt, units, s);
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
    if (a->qs[i] % 8 || a->os[i] % 8)
      return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: strides of q and o must be multiples of 8");
    if (extent[i] > 1 && a->os[i] == 0) return bad("paged attention: rows of o must not overlap (stride 0)");
  }
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
// most 1 GiB; otherwise they are computed again.
constexpr int kScoreRows = 32;
constexpr size_t kScoreBytes = size_t(1) << 30;

llmx_status choose(const llmx_attn_params *p, const AttnArgs &a, const PagedArgs &k, Plan *plan) {
  const bool can = paged_tc_supports(a, k);
  if (p->algo == LLMX_ALGO_TCGEN05 && !can)
    return record_error(LLMX_ERR_UNSUPPORTED, "paged attention: TCGEN05 needs head_dim 64 or 128, sm_scale > 0 and at most 128 "
                                              "query heads a kv head");
  plan->tc = can && (p->algo == LLMX_ALGO_TCGEN05 || (p->algo == LLMX_ALGO_AUTO && (long long)a.Sq * a.group > kStepRows));
  const bool weights = k.w != nullptr;
  const long long R = (long long)a.Sq * a.group;
  if (plan->tc) {
    plan->again = weights;
    plan->tcp = plan_paged_tc(a, true);
    plan->stat_at = kCounterBytes + plan->tcp.part_bytes;
    plan->bytes = plan->stat_at + (weights ? (size_t)a.B * a.Hkv * R * sizeof(float) : 0);
  } else {
    plan->step = plan_step(a, weights, weights);
    plan->again = weights && (R > kScoreRows || plan->step.score_bytes > kScoreBytes) && a.sm_scale > 0.f && paged_weights_supports(a, k);
    if (plan->again) plan->step.score_bytes = 0;
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
