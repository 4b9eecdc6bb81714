// Key weights of a chunk of query rows: for every cached token j of a kv head
//   w[j] = sum over packed rows r of 2^(score[r, j] - stat[r]),
// with the scores computed once more on the tensor cores, since a chunk's are
// too many to keep (few rows' scores are kept: attn_paged.cu).
//
// The product is transposed, S^T = K Q^T: a thread has one token (a row of the
// accumulator) and sums along its row in registers, so there is no exchange
// between threads and the sum's order is fixed.  A CTA keeps NT tiles of 128
// tokens in shared memory and streams the query rows that see them past in
// blocks of up to 128 packed rows.  Four warpgroups, each with an accumulator in
// tensor memory, share a tile's row blocks by turns (two for each of two tiles;
// at head_dim 256, where two tiles and the ring do not fit, four for one), so
// that products and exponentials overlap and the special-function units have
// four warps each to draw on (two left them idle half of the time).
//
// Bound by the exponentials: 128 x 128 of them take an SM 1024 cycles (16 a
// cycle) beside 512 cycles of products at head_dim 128.  2048 rows over 34816 tokens,
// 32 heads on 8 of 128: 0.74 ms (two warpgroups: 1.0 ms).
#include <algorithm>
#include <climits>
#include <numeric>

#include "paged_tc.cuh"

namespace llmx_b200 {
namespace {

constexpr int kGroups = 4;  // softmax warpgroups
constexpr int kWThreads = 128 * kGroups + 64;
constexpr int kWMmaWarp = 4 * kGroups, kWTmaWarp = kWMmaWarp + 1;

template <int D>
struct WCfg {
  static constexpr int kNT = D == 256 ? 1 : 2;      // token tiles
  static constexpr int kEvery = kGroups / kNT;      // warpgroups of a tile
  static constexpr int kTile = 128 * D * 2;                        // bytes of a tile
  static constexpr int kKBufs = D == 256 ? 1 : 2;  // an item's tokens are loaded while the one before is worked on
  static constexpr int kStages = D == 64 ? 4 : 2;  // blocks of rows in the ring
  static constexpr int kKOff = 0;
  static constexpr int kQOff = kKBufs * kNT * kTile;
  static constexpr int kConstOff = kQOff + kStages * kTile;  // [warpgroup][2][128] offsets, then slopes
  static constexpr int kOtherOff = kConstOff + kGroups * 2 * 2 * 128 * 4;  // [warpgroup][128] sums handed over
  static constexpr int kBarOff = kOtherOff + kGroups * 128 * 4;
  static constexpr int kSmem = kBarOff + 1024 + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory per CTA");
};

struct WBars {
  uint64_t k_full[2], k_empty[2];
  uint64_t q_full[4], q_empty[4];
  uint64_t s_full[kGroups], s_empty[kGroups];
  uint64_t c_full[kGroups][2];                       // offsets of a block's columns are written
  uint64_t other_full[kGroups], other_empty[kGroups];  // sums handed over to a tile's first warpgroup
  uint64_t drain;
  uint32_t tmem_base;
  volatile int abort_flag;
};

struct WeightWork {
  PagedArgs c;
  int R, M;
  int units;
  int n_work;
  int box;
  const float *stat;  // [units][R]
  float decay;
};

// An item: tokens [n0, n0 + 128 NT) of a unit, and the blocks of M packed rows
// [q0, q1) that may see one of them.
struct WItem {
  int b, kvh, ql, kl, n0, q0, q1;
};
template <int NT>
__device__ __forceinline__ WItem weight_item(const AttnArgs &a, const WeightWork &wk, int w) {
  WItem t;
  // Tiles outside, units inside: CTAs that take every grid-th item get some of each length.
  const int tile = w / wk.units, unit = w - tile * wk.units;
  t.kvh = unit % a.Hkv;
  t.b = unit / a.Hkv;
  t.ql = clamp_len(a.q_lens, t.b, a.Sq);
  t.kl = clamp_len(a.kv_lens, t.b, a.Skv);
  t.n0 = tile * kBN * NT;
  t.q0 = t.q1 = 0;
  if (t.n0 < t.kl && t.ql > 0) {
    // Row i sees token j where j <= i + off (causal) and i + off - j <= window.
    const int off = t.kl - t.ql, last = min(t.kl, t.n0 + kBN * NT) - 1;
    const int lo = a.causal ? max(0, t.n0 - off) : 0;
    const int hi = a.window >= 0 ? (int)max(0LL, min((long long)t.ql, (long long)last + a.window - off + 1)) : t.ql;
    if (hi > lo) {
      const int rows = wk.M / a.group;
      t.q0 = lo / rows;
      t.q1 = (hi + rows - 1) / rows;
    }
  }
  return t;
}

template <typename T, int D, bool kAlibi, bool kSoftcap>
__global__ void __launch_bounds__(kWThreads, 1)
    paged_weight_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ AttnArgs a, const __grid_constant__ WeightWork wk) {
  using C = WCfg<D>;
  constexpr int NT = C::kNT;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  WBars *bars = reinterpret_cast<WBars *>(smem + C::kBarOff);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kKBufs; ++i) {
      mbar_init(&bars->k_full[i], NT);
      mbar_init(&bars->k_empty[i], 1);
    }
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars->q_full[s], 1);
      mbar_init(&bars->q_empty[s], 1);
    }
    for (int g = 0; g < kGroups; ++g) {
      mbar_init(&bars->s_full[g], 1);
      mbar_init(&bars->s_empty[g], 128);
      mbar_init(&bars->c_full[g][0], 128);
      mbar_init(&bars->c_full[g][1], 128);
      mbar_init(&bars->other_full[g], 128);
      mbar_init(&bars->other_empty[g], 128);
    }
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWTmaWarp && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
  }
  if (warp == kWMmaWarp) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  // The attention's sums (stat) come from the launch before.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  auto wait1 = [&](uint64_t *bar, uint32_t par) { return mbar_wait_or_abort(bar, par, kTimeoutNs, &bars->abort_flag); };
  auto wait_all = [&](uint64_t *bar, uint32_t par) { return __all_sync(0xffffffffu, wait1(bar, par)) != 0; };
  // `block` counts the row blocks of all items, `item` the items that have any.
  if (warp >= 4 * kGroups) {
    if (warp == kWTmaWarp) {
      int block = 0, item = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < wk.n_work && ok; w += gridDim.x) {
        const WItem t = weight_item<NT>(a, wk, w);
        if (t.q1 <= t.q0) continue;
        BoxPlace p[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) p[i] = box_place(wk.c, wk.box, t.b, t.kl, t.n0 + i * kBN);
        const int kb = item % C::kKBufs;
        ok = wait_all(&bars->k_empty[kb], ((item / C::kKBufs) & 1) ^ 1);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          load_boxes<D>(smem + C::kKOff + (kb * NT + i) * C::kTile, &tm_k, &bars->k_full[kb], wk.box, t.kvh, p[i]);
        ++item;
        for (int q = t.q0; q < t.q1 && ok; ++q, ++block) {
          const int s = block % C::kStages;
          ok = wait_all(&bars->q_empty[s], ((block / C::kStages) & 1) ^ 1);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&bars->q_full[s], D / 64 * wk.M * 128);
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(smem + C::kQOff + s * C::kTile + c * 128 * 128, &tm_q, &bars->q_full[s], c * 64, t.kvh * a.group,
                          q * (wk.M / a.group), t.b);
          }
          __syncwarp();
        }
      }
      if (!ok) set_abort(bars, a.err);
      // Every load issued lands before the CTA may exit.
      for (int i = max(0, item - C::kKBufs); i < item; ++i)
        mbar_wait(&bars->k_full[i % C::kKBufs], (i / C::kKBufs) & 1, kTimeoutNs);
      for (int g = max(0, block - C::kStages); g < block; ++g)
        mbar_wait(&bars->q_full[g % C::kStages], (g / C::kStages) & 1, kTimeoutNs);
    } else if (warp == kWMmaWarp && lane == 0) {
      constexpr uint32_t idesc = idesc_f16(128, 128, kBF16, false);
      int block = 0, item = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < wk.n_work && ok; w += gridDim.x) {
        const WItem t = weight_item<NT>(a, wk, w);
        if (t.q1 <= t.q0) continue;
        const int kb = item % C::kKBufs;
        ok = wait1(&bars->k_full[kb], (item / C::kKBufs) & 1);
        for (int q = t.q0; q < t.q1 && ok; ++q, ++block) {
          const int s = block % C::kStages;
          ok = wait1(&bars->q_full[s], (block / C::kStages) & 1);
          for (int i = 0; i < NT && ok; ++i) {
            const int g = i * C::kEvery + block % C::kEvery, use = block / C::kEvery;
            ok = wait1(&bars->s_empty[g], (use & 1) ^ 1);
            if (!ok) break;
            tc_fence_after();
            uint64_t da = smem_desc_sw128(smem_u32(smem + C::kKOff + (kb * NT + i) * C::kTile), 16, 1024);
            uint64_t db = smem_desc_sw128(smem_u32(smem + C::kQOff + s * C::kTile), 16, 1024);
            asm volatile("" : "+l"(da), "+l"(db));
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint64_t o = (uint64_t)(((kk / 4) * 128 * 128 + (kk % 4) * 32) >> 4);
              mma_ss(tmem + g * 128, da + o, db + o, idesc, kk > 0 ? 1u : 0u);
            }
            tc_commit(&bars->s_full[g]);
          }
          if (ok) tc_commit(&bars->q_empty[s]);
        }
        if (ok) tc_commit(&bars->k_empty[kb]);
        ++item;
      }
      if (!ok) set_abort(bars, a.err);
      tc_commit(&bars->drain);
      mbar_wait(&bars->drain, 0, kTimeoutNs);
    }
  } else {
    const int g = warp / 4, tid = threadIdx.x % 128;
    constexpr int kEvery = C::kEvery;
    const int tile = g / kEvery, turn = g % kEvery;
    float *const cst = reinterpret_cast<float *>(smem + C::kConstOff) + g * 2 * 256;  // [2][offsets 128, slopes 128]
    const uint32_t lane_off = (uint32_t)((warp % 4) * 32) << 16;
    const float scale2 = a.sm_scale * kLog2e;
    const float cap_in = kSoftcap ? a.sm_scale / a.softcap : 0.f, cap_out = kSoftcap ? a.softcap * kLog2e : 0.f;
    int block = 0, handed = 0;
    bool ok = true;
    // What is added to column tid's score in row block q of item t: -stat, and with
    // ALiBi slope * (n0 - ref).
    auto column = [&](const WItem &t, int q, float &add, float &slope2) {
      const int pr = q * wk.M + tid;
      add = -CUDART_INF_F;
      slope2 = 0.f;
      if (tid < wk.M && pr < t.ql * a.group) {
        add = -wk.stat[((long long)t.b * a.Hkv + t.kvh) * wk.R + pr];
        if constexpr (kAlibi) {
          const int i = pr / a.group;
          const Visible v = row_visible(a, i, t.ql, t.kl);
          const float slope = a.alibi[t.kvh * a.group + pr - i * a.group];
          slope2 = slope * kLog2e;
          add = fmaf(slope2, (float)(t.n0 + tile * kBN - alibi_ref(v, slope)), add);
        }
      }
    };
    // This warpgroup's first block of an item that begins with the launch's block
    // number `at`: every kEvery-th is its.
    auto first_of = [&](int at) { return (turn + kEvery - at % kEvery) % kEvery; };
    // The first column of an item is read while the item before it is worked on.
    float next_add = 0.f, next_slope = 0.f;
    auto first_column = [&](int w, int at) {
      if (w >= wk.n_work) return;
      const WItem t = weight_item<NT>(a, wk, w);
      const int q = t.q0 + first_of(at);
      if (q < t.q1) column(t, q, next_add, next_slope);
    };
    first_column(blockIdx.x, 0);
    for (int w = blockIdx.x; w < wk.n_work && ok; w += gridDim.x) {
      const WItem t = weight_item<NT>(a, wk, w);
      float add = next_add, slope2 = next_slope;
      const int blocks = t.q1 - t.q0, first = first_of(block);
      first_column(w + gridDim.x, block + blocks);
      if (t.n0 >= t.kl) continue;
      const int n0 = t.n0 + tile * kBN;
      const int j = n0 + tid;
      const int off = t.kl - t.ql;
      // The query rows [see0, see1) that see token j, and those that see every token of the tile.
      auto sees = [&](int tok, int &r0, int &r1) {
        r0 = a.causal ? max(0, tok - off) : 0;
        r1 = a.window >= 0 ? (int)max(0LL, min((long long)t.ql, (long long)tok + a.window - off + 1)) : t.ql;
      };
      int see0, see1, first0, first1, last0, last1;
      sees(j, see0, see1);
      sees(n0, first0, first1);
      sees(n0 + kBN - 1, last0, last1);
      const int row_lo = see0 * a.group, row_hi = max(see0, see1) * a.group;  // as packed rows
      const int all_lo = last0 * a.group, all_hi = first1 * a.group;
      uint64_t acc0 = f2(0.f, 0.f), acc1 = f2(0.f, 0.f);
      for (int i = first; i < blocks; i += kEvery) {
        const int q = t.q0 + i, use = (block + i) / kEvery, buf = use & 1;
        cst[buf * 256 + tid] = add;
        if constexpr (kAlibi) cst[buf * 256 + 128 + tid] = slope2;
        if (i + kEvery < blocks) column(t, q + kEvery, add, slope2);
        mbar_arrive(&bars->c_full[g][buf]);
        ok = wait_all(&bars->c_full[g][buf], (use >> 1) & 1) && wait_all(&bars->s_full[g], use & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tS = tmem + lane_off + g * 128;
        const int base = q * wk.M;
        const int lo = min(max(row_lo - base, 0), 128), hi = min(max(row_hi - base, 0), wk.M);
        const bool need_mask = base < all_lo || base + 128 > all_hi || wk.M < 128;
        const float4 *const ca = reinterpret_cast<const float4 *>(cst + buf * 256);
        const float4 *const cs = ca + 32;
        const float kf = (float)tid;
#pragma unroll 1
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t vc[32];
          tmem_ld32(tS + ch * 32, vc);
          tmem_wait_ld();
          reg_fence32(vc);
          if (ch == 3) {
            tc_fence_before();
            mbar_arrive(&bars->s_empty[g]);
          }
          uint32_t seen = 0xffffffffu;
          if (need_mask) {
            const int b0 = min(max(lo - ch * 32, 0), 32), b1 = min(max(hi - ch * 32, 0), 32);
            seen = (b1 >= 32 ? 0xffffffffu : (1u << b1) - 1u) & ~(b0 >= 32 ? 0xffffffffu : (1u << b0) - 1u);
          }
          // Adds the 32 columns up; kSmall: all scores are small for the soft-cap.
          auto add_up = [&](auto kSmall) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              const float4 ad = ca[ch * 8 + c / 4];
              float x[4] = {ad.x, ad.y, ad.z, ad.w};
              if constexpr (kAlibi) {
                const float4 sl = cs[ch * 8 + c / 4];
                x[0] = fmaf(sl.x, kf, x[0]);
                x[1] = fmaf(sl.y, kf, x[1]);
                x[2] = fmaf(sl.z, kf, x[2]);
                x[3] = fmaf(sl.w, kf, x[3]);
              }
              const uint64_t v0 = f2(__uint_as_float(vc[c]), __uint_as_float(vc[c + 1]));
              const uint64_t v1 = f2(__uint_as_float(vc[c + 2]), __uint_as_float(vc[c + 3]));
              if constexpr (kSoftcap) {
                const SoftCap cap(cap_in, cap_out);
                f2_split(cap.template pair<decltype(kSmall)::value>(v0, f2(x[0], x[1])), x[0], x[1]);
                f2_split(cap.template pair<decltype(kSmall)::value>(v1, f2(x[2], x[3])), x[2], x[3]);
              } else {
                const uint64_t sc = f2(scale2, scale2);
                f2_split(fma2(v0, sc, f2(x[0], x[1])), x[0], x[1]);
                f2_split(fma2(v1, sc, f2(x[2], x[3])), x[2], x[3]);
              }
              if (need_mask) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (seen & (1u << (c + e))) ? x[e] : -CUDART_INF_F;
              }
              acc0 = add2(acc0, f2(ex2_approx(x[0]), ex2_approx(x[1])));
              acc1 = add2(acc1, f2(ex2_approx(x[2]), ex2_approx(x[3])));
            }
          };
          // (By size: the scale may be negative.)
          if (kSoftcap && !__all_sync(0xffffffffu, chunk_size(vc) * fabsf(cap_in) <= kCapSmall))
            add_up(std::false_type{});
          else
            add_up(std::true_type{});
        }
      }
      block += blocks;
      if (!ok) break;
      float s0, s1, s2, s3;
      f2_split(acc0, s0, s1);
      f2_split(acc1, s2, s3);
      float sum = (s0 + s1) + (s2 + s3);
      {
        // The sums of a tile's other warpgroups are handed to its first one.
        float *const other = reinterpret_cast<float *>(smem + C::kOtherOff);
        const int turn_no = handed++;
        if (turn != 0) {
          ok = wait_all(&bars->other_empty[g], (turn_no & 1) ^ 1);
          if (!ok) break;
          other[g * 128 + tid] = sum;
          mbar_arrive(&bars->other_full[g]);
          continue;
        }
#pragma unroll
        for (int o = 1; o < kEvery; ++o) {
          ok = ok && wait_all(&bars->other_full[g + o], turn_no & 1);
          if (!ok) break;
          sum += other[(g + o) * 128 + tid];
          mbar_arrive(&bars->other_empty[g + o]);
        }
        if (!ok) break;
      }
      if (j < t.kl) {
        const int page = paged_page(wk.c, t.b, j / wk.c.page_size);
        if (page >= 0) {
          float *to = wk.c.w + page * wk.c.ws[0] + t.kvh * wk.c.ws[1] + j % wk.c.page_size;
          const int old = wk.decay == 0.f ? 0 : (a.causal ? t.kl - t.ql : t.kl);
          *to = j < old ? fmaf(wk.decay, *to, sum) : sum;
        }
      }
    }
    if (!ok) set_abort(bars, a.err);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kWMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------------------- host
template <typename T, int D, bool kAlibi, bool kSoftcap>
cudaError_t launch_weight_t(const AttnArgs &a, WeightWork wk, cudaStream_t s) {
  using C = WCfg<D>;
  CUtensorMap tq, tk;
  if (!make_q_map(&tq, a, wk.M) || !make_page_map(&tk, wk.c, wk.c.k, wk.c.ks, a.dtype, wk.box)) return cudaErrorInvalidValue;
  wk.units = a.B * a.Hkv;
  const long long work = (long long)wk.units * ((a.Skv + kBN * C::kNT - 1) / (kBN * C::kNT));
  if (work > INT_MAX / 2) return cudaErrorInvalidValue;
  wk.n_work = (int)work;
  constexpr auto kern = paged_weight_kernel<T, D, kAlibi, kSoftcap>;
  const cudaError_t attr = allow_smem<kern>(C::kSmem);
  if (attr != cudaSuccess) return attr;
  return launch_paged_after(kern, dim3(std::min(wk.n_work, std::max(1, a.num_sms))), kWThreads, C::kSmem, s, tq, tk, a, wk);
}

template <typename T, int D>
cudaError_t launch_weight_d(const AttnArgs &a, const WeightWork &wk, cudaStream_t s) {
  const bool alibi = a.alibi != nullptr, cap = a.softcap > 0.f;
  if (alibi) return cap ? launch_weight_t<T, D, true, true>(a, wk, s) : launch_weight_t<T, D, true, false>(a, wk, s);
  return cap ? launch_weight_t<T, D, false, true>(a, wk, s) : launch_weight_t<T, D, false, false>(a, wk, s);
}
template <typename T>
cudaError_t launch_weight(const AttnArgs &a, const WeightWork &wk, cudaStream_t s) {
  switch (a.D) {
    case 64: return launch_weight_d<T, 64>(a, wk, s);
    case 128: return launch_weight_d<T, 128>(a, wk, s);
    default: return launch_weight_d<T, 256>(a, wk, s);
  }
}

}  // namespace

bool paged_weights_supports(const AttnArgs &a) {
  // A block holds whole groups.  Bytes of a stride of q's tensor map stay below 2^40.
  if (a.group > kBM) return false;
  if ((long long)a.B * a.Hkv * ((a.Skv + kBN - 1) / kBN) > INT_MAX / 2) return false;
  const int extent[3] = {a.B, a.Sq, a.H};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (a.qs[i] == 0 || a.qs[i] >= (1LL << 39))) return false;
  return true;
}

cudaError_t launch_paged_weights(const AttnArgs &a, const PagedArgs &c, const float *stat, float decay, cudaStream_t s) {
  WeightWork wk{};
  wk.c = c;
  wk.R = a.Sq * a.group;
  wk.M = kBM / a.group * a.group;
  wk.box = std::gcd(c.page_size, kBN);
  wk.stat = stat;
  wk.decay = decay;
  return a.dtype == LLMX_FP16 ? launch_weight<__half>(a, wk, s) : launch_weight<__nv_bfloat16>(a, wk, s);
}

}  // namespace llmx_b200
