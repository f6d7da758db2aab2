// Cross attention forward on the tensor cores, for several queries.
//
// A CTA holds two tiles of 128 query rows of one head and walks over tiles of 128 keys. For each
// pair of tiles S = q k^T is a product into tensor memory; a warpgroup with one thread for each
// query row reads its row of S, keeps the running maximum and sum, writes P = exp(S - max) back
// into tensor memory in 16 bits, and P v is added to the row's accumulator, also there. Four warps
// serve the first query tile, four the second; two issue their products, on schedulers of their own
// (one for both held the tensor pipe up: 204 -> 293 us in the first case below), one the copies, one
// clears v's rows past the keys' end and at keys that no query keeps. While one tile's softmax runs, the other tile's products do.
//
// What bounds it, at D 64, is the exponentials: 1,024 clocks of the special-function unit for a pair
// of tiles whose two products take 512 (measured: that unit 69% busy, the tensor pipe 34%); at D 128
// both take 1,024. One item of 4,096 queries, bfloat16: 16 heads of 64 x 8,160 keys 193 us, 710
// TFLOP/s; 16 heads of 128 x 4,096 keys 147 us, 940 TFLOP/s.
//
// The maximum that P is formed with may lag behind the true one by up to kLag powers of two: the
// accumulator (128 rows x D numbers through registers) is rescaled only when a row's maximum has
// grown by more, which after the first tiles is rare. P is rounded to 16 bits, the products' operand
// type, while the row sum adds it before that, in 32 bits. For bfloat16 the rounding is relative
// all the way down. Half has few exponents, so P is formed with what the lag leaves of them, 2^(15 -
// kLag) times larger: relative down to 2^-21 of the (lagging) maximum, and 65,000 keys below that
// are still off by less than 2^-16 of it together.
//
// With few query tiles the keys are split over CTAs: each has its normalised output in 32 bits and
// its lse, and the splits of a block, as a cluster through shared memory, or combine_kernel join them
// with weights exp(lse_split - lse). With few queries,
// heads that share a key head share a tile of rows too, so that k and v are read and multiplied once
// for all of them (2 x 1 query x 65,280 keys, 24 heads on each of 8 of 128: 2,533 -> 106 us; 4 x 40 x
// 3,600, 4 on each of 4 of 64: 24.3 -> 17.3).
#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "capi_internal.h"
#include "tensor_core.cuh"

namespace gs {

constexpr int kTileQ = 128;   // query rows of one warpgroup
constexpr int kTileK = 128;   // keys of one tile
constexpr float kLag = 8.0f;  // powers of two
constexpr int kFwdThreads = 384;
// P is formed 2^kUp times larger.
template <typename T>
constexpr float kUp = 0.0f;
template <>
constexpr float kUp<__half> = kHalfLog2 - kLag;
// Registers of a softmax thread and of the others: 2 x 128 x 200 + 128 x 104 = 384 x 168, what the
// CTA is launched with.
constexpr int kSoftmaxRegs = 200, kOtherRegs = 104;

struct ForwardParams {
  AttentionParams a;
  unsigned* errors;  // the device's error word
  float scale_log2;  // |scale| log2 e, above 0
  float lag;         // kLag in units of unscaled scores
  int negate;        // scale < 0: scores change sign first
  int tiles;   // query tiles a CTA holds, 1 or 2
  int pack;    // query heads a tile holds: above 1 it holds all queries of each
  int groups, shared, q_blocks;  // Hq / pack, Hq / Hkv, CTAs a group of heads
  int splits;
  int cluster;  // the splits of a block are a cluster, which joins them itself
  int kb, kh, vb, vh, qb, qh;  // 0 where all batch items (heads) share the tensor, else 1
  float* part_out;  // [splits, B, Hq, Lq, D] where splits > 1
  float* part_lse;  // [splits, B, Hq, Lq]
};

template <int DP>
struct ForwardShared {
  static constexpr int kBoxes = DP / 64;
  static constexpr int kTileBytes = kBoxes * 128 * 128;
  static constexpr int kStages = DP == 128 ? 2 : 4;
  static constexpr int kBytes = 1024 + 2 * kTileBytes + 2 * kStages * kTileBytes + 256;
};

// MASK: with a mask; calls without one have a kernel without its code and registers (4,096 x 8,160, 16 heads of
// 64, half: 198 us in one kernel for both, 192 so; 3 x 1,111 x 777 with a mask 43.6 and 42.3).
template <typename T, int DP, bool MASK>
__global__ void __launch_bounds__(kFwdThreads, 1)
    attention_forward_kernel(const __grid_constant__ ForwardParams p,
                             const __grid_constant__ CUtensorMap map_q,
                             const __grid_constant__ CUtensorMap map_k,
                             const __grid_constant__ CUtensorMap map_v) {
  using S = ForwardShared<DP>;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t q_full, k_full[S::kStages], k_free[S::kStages], v_full[S::kStages],
      v_clean[S::kStages], v_free[S::kStages], s_full[2], s_read[2], p_ready[2], o_done[2], o_full[2], turn[2];
  __shared__ float lse_part[2 * kTileQ];
  __shared__ unsigned tmem_slot;
  __shared__ volatile int gave_up;
  const unsigned base = (smem_u32(raw) + 1023u) & ~1023u;
  const unsigned sm_q = base, sm_k = base + 2 * S::kTileBytes,
                 sm_v = sm_k + S::kStages * S::kTileBytes;
  const int warp = warp_uniform(threadIdx.x / 32);
  const AttentionParams& a = p.a;
  const int queries = p.pack * a.Lq;
  const unsigned bh = blockIdx.x / (unsigned)p.q_blocks, block = blockIdx.x - bh * p.q_blocks;
  const int q0 = block * p.tiles * kTileQ, b = bh / (unsigned)p.groups,
            h0 = (bh - b * p.groups) * p.pack, hk = (unsigned)h0 / (unsigned)p.shared;
  const bool both = p.tiles == 2 && q0 + kTileQ < queries;
  if (threadIdx.x == 288) {  // of warp 9
    prefetch_map(&map_q);
    prefetch_map(&map_k);
    prefetch_map(&map_v);
    gave_up = 0;
    mbar_set(&q_full, 1);
    for (int i = 0; i < S::kStages; ++i) {
      mbar_set(&k_full[i], 1);
      mbar_set(&k_free[i], both ? 2 : 1);
      mbar_set(&v_full[i], 1);
      mbar_set(&v_clean[i], 1);
      mbar_set(&v_free[i], both ? 2 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_set(&s_full[i], 1);
      mbar_set(&s_read[i], 4);
      mbar_set(&p_ready[i], 4);
      mbar_set(&o_done[i], 1);
      mbar_set(&o_full[i], 1);
      mbar_set(&turn[i], 4);
    }
    mbar_ready();
  }
  __syncwarp();
  // With a mask this kernel may run beside the one that packs it, which has itself waited for what
  // came before; only the mask's bits are waited for then.
  if (!MASK) wait_for_previous();
  const int n = warp_uniform(key_count(a, b));
  const int tiles = (n + kTileK - 1) / kTileK;
  // fewer than 2^24 tiles times at most kSms splits fit 32 bits, which divide faster than 64
  const unsigned splits = (unsigned)p.splits;
  const int t0 = (int)((unsigned)tiles * blockIdx.y / splits);
  const int count = (int)((unsigned)tiles * (blockIdx.y + 1) / splits) - t0;

  const auto load_k = [&](int j) {
    const int st = j % S::kStages;
    mbar_arrive_expect_tx(&k_full[st], S::kTileBytes);
    for (int x = 0; x < S::kBoxes; ++x)
      tma_load_4d(sm_k + st * S::kTileBytes + x * 16384, &map_k, x * 64, (t0 + j) * kTileK,
                  hk * p.kh, b * p.kb, &k_full[st]);
  };
  const auto load_v = [&](int j) {
    const int st = j % S::kStages;
    mbar_arrive_expect_tx(&v_full[st], S::kTileBytes);
    for (int x = 0; x < S::kBoxes; ++x)
      tma_load_4d(sm_v + st * S::kTileBytes + x * 16384, &map_v, x * 64, (t0 + j) * kTileK,
                  hk * p.vh, b * p.vb, &v_full[st]);
  };
  let_next_start();
  if (warp == 9) {  // goes on to the first copies while the others get ready
    ready_arrive<kFwdThreads>();
    if (threadIdx.x % 32 == 0 && count > 0) {
      const int bq = b * p.qb, hq = h0 * p.qh;
      mbar_arrive_expect_tx(&q_full, p.pack > 1 ? queries * S::kBoxes * 128
                                                : (both ? 2 : 1) * S::kTileBytes);
      for (int t = 0; t < (both ? 2 : 1); ++t)
        for (int x = 0; x < S::kBoxes; ++x)
          tma_load_4d(sm_q + t * S::kTileBytes + x * 16384, &map_q, x * 64, q0 + t * kTileQ, hq, bq,
                      &q_full);
      for (int j = 0; j < S::kStages && j < count; ++j) {
        load_k(j);
        load_v(j);
      }
    }
  } else {
    if (warp == 8) tc_alloc(&tmem_slot, 512);
    // rows that no query is copied to: as good as a query of zeros
    if (warp == 11 && p.pack > 1)
      clear_rows<S::kBoxes>(sm_q, queries, make_uint4(~0u, ~0u, ~0u, ~0u));
    tc_fence_before();
    ready_wait<kFwdThreads>();
    tc_fence_after();
  }
  const unsigned tmem = warp == 9 ? 0u : (unsigned)warp_uniform((int)tmem_slot);
  // Tensor memory, 512 columns: S of both tiles 256, O of both 2 DP. Up to D = 64 there is room
  // for P beside S; above, P takes the first half of S's own columns.
  constexpr bool kAhead = DP == 64;
  const unsigned tm_s = tmem, tm_o = tmem + (kAhead ? 384 : 256);
  const unsigned tm_p = kAhead ? tmem + 256 : tmem;
  constexpr unsigned kStepP = kAhead ? 64 : 128, kStepO = kAhead ? 64 : 128;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---- softmax: one thread for each query row ----
    const int t = warp / 4;
    // the thread's row, one of `queries`, and what it is of: query i of head h0 + s
    const int row_q = q0 + t * kTileQ + threadIdx.x % 128;
    const bool live = row_q < queries;
    int i = min(row_q, queries - 1), h = h0;
    if (p.pack > 1) {
      const int s = (unsigned)i / (unsigned)a.Lq;
      h += s;
      i -= s * a.Lq;
    }
    if (t == 0 || both) {
      const unsigned lanes = (unsigned)(warp % 4 * 32) << 16;
      const unsigned my_s = tm_s + t * 128 + lanes, my_o = tm_o + t * kStepO + lanes,
                     my_p = tm_p + t * kStepP + lanes;
      const uint4* keep_row =
          MASK ? reinterpret_cast<const uint4*>(a.bits + b * a.bits_b + h * a.bits_h +
                                                  (long long)i * a.bits_q)
                 : nullptr;
      float m = -INFINITY, l = 0.0f;
      bool ok = true;
      if (MASK) wait_for_previous();
      uint4 keep_next = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (MASK && count > 0) keep_next = keep_row[t0];
      for (int j = 0; j < count; ++j) {
        const int key = (t0 + j) * kTileK;
        const uint4 keep = keep_next;
        if (MASK && j + 1 < count) keep_next = keep_row[t0 + j + 1];
        ok = tc_wait_warp(&s_full[t], j & 1);
        if (!ok) break;
        tc_fence_after();
        unsigned s[kTileK];
#pragma unroll
        for (int c = 0; c < kTileK; c += 32) tc_ld32(my_s + c, s + c);
        tc_wait_ld();
        if (kAhead) {
          tc_fence_before();
          mbar_arrive_warp(&s_read[t]);
        }
        if (p.negate) {
#pragma unroll
          for (int k = 0; k < kTileK; ++k) s[k] ^= 0x80000000u;
        }
        if (MASK || key + kTileK > n) {
          hide32(keep.x & below(n - key, 0), s);
          hide32(keep.y & below(n - key, 1), s + 32);
          hide32(keep.z & below(n - key, 2), s + 64);
          hide32(keep.w & below(n - key, 3), s + 96);
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < kTileK; k += 2)
          top[k / 2 % 4] = max_nan(max_nan(top[k / 2 % 4], __uint_as_float(s[k])),
                                   __uint_as_float(s[k + 1]));
        const float mx = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3]));
        const bool grew = !(mx <= m + p.lag);  // NaN too: then the row is NaN from here on
        if (kAhead && j > 0) {  // the product that read the P before, and added to O, is over
          ok = tc_wait_warp(&o_done[t], (j - 1) & 1);
          if (!ok) break;
          tc_fence_after();
        }
        if (__any_sync(~0u, grew)) {
          const float f = grew ? fast_exp2((m - mx) * p.scale_log2) : 1.0f;
          if (grew) m = mx;
          l *= f;
          if (j > 0) {
            for (int c = 0; c < DP; c += 16) {
              unsigned o[16];
              tc_ld16(my_o + c, o);
              tc_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tc_st16(my_o + c, o);
            }
          }
        }
        // Where S waits for P v, the two query tiles do best half a period apart, one's products
        // beside the other's exponentials; started together they may stay together. So they take
        // turns for the first two tiles and keep the distance after that (4,096 x 8,192, 16 heads:
        // 458 -> 331 us at D 80, 437 -> 345 at D 96, 383 -> 364 at D 128).
        const bool turns = !kAhead && both && j < 2;
        if (turns && (t == 1 || j > 0)) {
          ok = tc_wait_warp(&turn[t], (t == 1 ? j : j - 1) & 1);
          if (!ok) break;
        }
        // m - m is 0, or NaN where the row holds an infinite score
        const float off = m == -INFINITY ? 0.0f : fmaf(m, p.scale_log2, (m - m) - kUp<T>);
        const Two scale2 = two(p.scale_log2, p.scale_log2), off2 = two(-off, -off);
        Two sum[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
#pragma unroll
        for (int c = 0; c < kTileK; c += 32) {
          unsigned packed[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const Two x = fma2(two(__uint_as_float(s[c + 2 * k]), __uint_as_float(s[c + 2 * k + 1])),
                               scale2, off2);
            float e0, e1;
            split(x, e0, e1);
            e0 = fast_exp2(e0);
            e1 = fast_exp2(e1);
            sum[k % 2] = add2(sum[k % 2], two(e0, e1));
            packed[k] = pack2<T>(e0, e1);
          }
          tc_st16(my_p + c / 2, packed);
        }
        if (turns) mbar_arrive_warp(&turn[1 - t]);
        float sum0, sum1;
        split(add2(sum[0], sum[1]), sum0, sum1);
        l += sum0 + sum1;
        tc_wait_st();
        tc_fence_before();
        mbar_arrive_warp(&p_ready[t]);
      }
      if (ok && count > 0) ok = tc_wait_warp(&o_full[t], 0);
      if (!ok) gave_up = 1;
      tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const float lse = l == 0.0f ? -INFINITY
                                  : m * p.scale_log2 * 0.6931471805599453f +
                                        logf(l * (1.0f / (1 << (int)kUp<T>)));
      const long long row = ((long long)b * a.Hq + h0) * a.Lq + row_q;
      const long long rows = (long long)a.B * a.Hq * a.Lq;
      const bool wide = p.splits > 1;
      // rows of several heads follow one another in the parts, but not in `out`
      const int lane = threadIdx.x % 32;
      char* to;
      if (wide)
        to = reinterpret_cast<char*>(p.part_out + (blockIdx.y * rows + row - lane) * a.D);
      else if (p.pack > 1)
        to = reinterpret_cast<char*>(a.out.at<T>(b, i, h));
      else
        to = reinterpret_cast<char*>(a.out.at<T>(b, row_q - lane, h0));
      if (p.cluster) {
        // the keys and values have done their work once both query tiles are through: the parts of the
        // block take their place, rows of DP numbers in 16-byte pieces, swizzled
        if (both)
          asm volatile("bar.sync 2, 256;" ::: "memory");
        else
          asm volatile("bar.sync 2, 128;" ::: "memory");
        const int r = t * kTileQ + threadIdx.x % 128;
        for (int c = 0; c < DP; c += 32) {
          unsigned o[32];
          if (ok && count > 0) tc_ld32(my_o + c, o);
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            float f[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) f[d] = l != 0.0f ? __uint_as_float(o[k + d]) * inv : 0.0f;
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                             sm_k + r * (DP * 4) + (((c + k) / 4 ^ (r & 7)) << 4)),
                         "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3])
                         : "memory");
          }
        }
        lse_part[r] = lse;
      } else {
        // the tile's queries in shared memory have done their work
        store_rows<T, DP>(my_o, ok && count > 0, l != 0.0f, inv, a.D, wide,
                          sm_q + t * S::kTileBytes + warp % 4 * (DP * 64), to,
                          wide ? a.D * 4ll : p.pack > 1 ? 0 : a.out.l * 2,
                          queries - row_q + lane);
        if (live) {
          if (p.splits > 1)
            p.part_lse[blockIdx.y * rows + row] = lse;
          else if (a.lse)
            a.lse[row] = lse;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
      // ---- copies: the first tiles are on their way ----
      if (threadIdx.x % 32 == 0)
        for (int j = S::kStages; j < count; ++j) {
          const int st = j % S::kStages;
          const unsigned phase = (j / S::kStages & 1) ^ 1;
          if (!tc_wait(&k_free[st], phase)) { gave_up = 1; break; }
          load_k(j);
          if (!tc_wait(&v_free[st], phase)) { gave_up = 1; break; }
          load_v(j);
        }
    } else if (warp == 11) {
      // ---- what v holds at keys that no query of the item's key head keeps must not reach the
      // product, which would make 0 times NaN of it: those rows are set to zero before the product may
      // read them
      if (MASK) wait_for_previous();
      for (int j = 0; j < count; ++j) {
        const int st = j % S::kStages, key = (t0 + j) * kTileK;
        uint4 keep = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (MASK) keep = kept_begin(a, b, hk, t0 + j);
        if (!tc_wait_warp(&v_full[st], j / S::kStages & 1)) { gave_up = 1; break; }
        if (MASK) keep = kept_end(keep);
        if (has_hidden_rows(n - key, keep))
          clear_rows<S::kBoxes>(sm_v + st * S::kTileBytes, n - key, keep);
        mbar_arrive_warp(&v_clean[st]);
      }
    } else if (warp == 8 || (warp == 10 && both)) {
      // ---- products: a warp for each query tile, on different schedulers ----
      const int t = warp == 10;
      const int steps = (a.D + 15) / 16;
      const unsigned idesc_s = tc_idesc<T>(kTileK, false);
      const unsigned idesc_o = tc_idesc<T>(steps * 16, true);
      // descriptor units are 16 bytes
      const uint64_t desc_q = tc_desc(sm_q + t * S::kTileBytes, 16), desc_k = tc_desc(sm_k, 16),
                     desc_v = tc_desc(sm_v, 16384);
      const unsigned tm_st = tm_s + t * 128, tm_pt = tm_p + t * kStepP, tm_ot = tm_o + t * kStepO;
      // S = q k^T of tile j, once k is there and (where P has its own columns) the softmax has read
      // the S before
      const auto next_scores = [&](int j) {
        const int st = j % S::kStages;
        if (!tc_wait_warp(&k_full[st], j / S::kStages & 1)) return false;
        if (kAhead && j > 0) {
          if (!tc_wait_warp(&s_read[t], (j - 1) & 1)) return false;
          tc_fence_after();
        }
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const unsigned off = ((k / 4) * 16384 + (k % 4) * 32) / 16;
            if (k < steps)
              tc_mma_ss(tm_st, desc_q + off, desc_k + st * (S::kTileBytes / 16) + off, idesc_s, k > 0);
          }
          tc_commit(&s_full[t]);
          tc_commit(&k_free[st]);
        }
        __syncwarp();
        return true;
      };
      const auto values = [&](int st, bool add) {  // O += P v
#pragma unroll
        for (int k = 0; k < kTileK / 16; ++k)
          tc_mma_ts(tm_ot, tm_pt + k * 8, desc_v + st * (S::kTileBytes / 16) + k * 128, idesc_o,
                    add || k > 0);
      };
      constexpr int kLead = kAhead ? 2 : 1;  // tiles that S is ahead of P
      bool ok = count > 0 && tc_wait_warp(&q_full, 0);
      for (int j = 0; j < kLead; ++j) ok = ok && (j >= count || next_scores(j));
      for (int j = 0; ok && j < count; ++j) {
        const int st = j % S::kStages;
        ok = tc_wait_warp(&v_clean[st], j / S::kStages & 1);
        if (!ok) break;
        ok = tc_wait_warp(&p_ready[t], j & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          values(st, j > 0);
          if (kAhead) tc_commit(&o_done[t]);
          tc_commit(&v_free[st]);
          if (j + 1 == count) tc_commit(&o_full[t]);
        }
        __syncwarp();
        if (j + kLead < count) ok = next_scores(j + kLead);
      }
      if (!ok && count > 0) gave_up = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (gave_up) {
    // A wait ran out. Copies still in flight end before the CTA's memory is given up.
    if (threadIdx.x == 0) {
      atomicOr(p.errors, kErrMmaTimeout);
      const unsigned long long t = tma_global_ns();
      for (int k = 0; k < (1 << 20) && tma_global_ns() - t < 10000000ull; ++k) __nanosleep(1000);
    }
    __syncthreads();
  }
  if (warp == 8) {
    tc_fence_after();
    tc_free(tmem, 512);
  }
  if (!p.cluster) return;
  // out = sum over splits of exp(lse_s - lse) out_s from the shared memory of the cluster's CTAs, each
  // of which takes every splits-th row
  cluster_arrive();
  cluster_wait();
  const int rows = min(queries - q0, both ? 2 * kTileQ : kTileQ);
  for (int at = threadIdx.x;; at += kFwdThreads) {
    const int r = at / (DP / 4) * p.splits + blockIdx.y, c = at % (DP / 4);
    if (r >= rows) break;
    if (c * 4 >= a.D) continue;
    float top = -INFINITY, total = 0.0f, acc[4] = {};
    for (int s = 0; s < p.splits; ++s) top = max_nan(top, cluster_load(&lse_part[r], s));
    for (int s = 0; s < p.splits; ++s) {
      const float f = top == -INFINITY ? 0.0f : expf(cluster_load(&lse_part[r], s) - top);
      const float4 v = cluster_load4(sm_k + r * (DP * 4) + ((c ^ (r & 7)) << 4), s);
      total += f;
      acc[0] = fmaf(f, v.x, acc[0]), acc[1] = fmaf(f, v.y, acc[1]);
      acc[2] = fmaf(f, v.z, acc[2]), acc[3] = fmaf(f, v.w, acc[3]);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    int i = q0 + r, h = h0;
    if (p.pack > 1) {
      const int s = (unsigned)i / (unsigned)a.Lq;
      h += s;
      i -= s * a.Lq;
    }
    *reinterpret_cast<uint2*>(a.out.at<T>(b, i, h) + c * 4) =
        make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
    if (c == 0 && a.lse)
      a.lse[((long long)b * a.Hq + h0) * a.Lq + q0 + r] =
          total == 0.0f ? -INFINITY : top + logf(total);
  }
  cluster_arrive();  // the others may still be reading this CTA's memory
  cluster_wait();
}

// out = sum over splits of exp(lse_s - lse) out_s: WARPS warps for each row, each with every
// WARPS-th split, a lane for 4 of the row's numbers. 4 warps where there are more than 8 splits:
// with the forward before it 256 x 30,000 of 2 heads of 64 then takes 19.8 us instead of 25.0 with
// one warp, but 1,000 x 8,160 (up to 8 splits) 17.7 with one and 19.2 with four.
template <typename T, int WARPS>
__global__ void __launch_bounds__(128) combine_kernel(AttentionParams a, int splits,
                                                      const float* part_out,
                                                      const float* part_lse) {
  __shared__ float s_top[4], s_total[4], s_acc[4][128];
  wait_for_previous();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, first = warp % WARPS;
  const unsigned rows = (unsigned)a.B * a.Hq * a.Lq;
  const unsigned row = blockIdx.x * (4 / WARPS) + warp / WARPS;
  if (row >= rows) return;  // whole CTAs where WARPS is 4
  const int d = lane * 4;
  float top = -INFINITY, total = 0.0f, acc[4] = {};
  // chunks of 32 splits of this warp, a lane each; the maximum may grow from chunk to chunk
  for (int s0 = 0; s0 * WARPS + first < splits; s0 += 32) {
    const int own = (s0 + lane) * WARPS + first;
    const float lse = own < splits ? part_lse[(long long)own * rows + row] : -INFINITY;
    float most = lse;
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
    most = fmaxf(most, top);
    if (most > top) {
      const float f = expf(top - most);
      total *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] *= f;
      top = most;
    }
    const float w = expf(lse - (top == -INFINITY ? 0.0f : top));
    total += w;
    const int n = min(32, (splits - first - s0 * WARPS + WARPS - 1) / WARPS);
    const float* part = part_out + ((long long)(s0 * WARPS + first) * rows + row) * a.D + d;
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float ws = __shfl_sync(~0u, w, s);
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (d < a.D) o = *reinterpret_cast<const float4*>(part + (long long)s * WARPS * rows * a.D);
      acc[0] = fmaf(ws, o.x, acc[0]), acc[1] = fmaf(ws, o.y, acc[1]);
      acc[2] = fmaf(ws, o.z, acc[2]), acc[3] = fmaf(ws, o.w, acc[3]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
  if constexpr (WARPS > 1) {
    if (lane == 0) s_top[warp] = top, s_total[warp] = total;
#pragma unroll
    for (int i = 0; i < 4; ++i) s_acc[warp][d + i] = acc[i];
    __syncthreads();
    if (warp) return;
    top = s_top[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, s_top[w]);
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = top == -INFINITY ? 0.0f : expf(s_top[w] - top);
      total = fmaf(f, s_total[w], total);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(f, s_acc[w][d + i], acc[i]);
    }
  }
  // a NaN among the parts is in `total`, whatever the maximum
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (d < a.D) {
    const unsigned bh = row / (unsigned)a.Lq, i = row - bh * (unsigned)a.Lq;
    const unsigned b = bh / (unsigned)a.Hq, h = bh - b * (unsigned)a.Hq;
    *reinterpret_cast<uint2*>(a.out.at<T>(b, i, h) + d) = make_uint2(
        pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
  }
  if (a.lse && lane == 0) a.lse[row] = total == 0.0f ? -INFINITY : top + logf(total);
}

struct ForwardPlan {
  int pack, tiles, splits;
};

// How many query heads that share a key head go into one tile (1, or as many as fit with all their
// queries), query tiles a CTA and splits of the keys (each with at least two tiles of keys, and all in
// one wave of CTAs), by the time they should take in us: waves of CTAs, each with some 4 us to begin
// and end and, for a tile of keys, what one and two query tiles take together (measured: 1.35 and
// 1.65 at D 64, 1.7 and 2.2 at D 128); joining splits takes another launch and the parts' way
// through memory.
static ForwardPlan forward_plan(const gs_attention_args& a) {
  const int shared = a.Hq / a.Hkv, key_tiles = (a.Lk + kTileK - 1) / kTileK;
  const double part_us = (double)a.B * a.Hq * a.Lq * a.D * 8.0 / 3e6;
  int most = shared;
  while (most > 1 && (shared % most || (long long)most * a.Lq > kTileQ)) --most;
  ForwardPlan best{1, 2, 1};
  double least = 1e30;
  for (int tiles = 2; tiles >= 1; --tiles)
    for (int pack = 1;; pack = most) {
      const int q_tiles = (int)(((long long)pack * a.Lq + kTileQ - 1) / kTileQ);
      const double ctas = (double)a.B * (a.Hq / pack) * ((q_tiles + tiles - 1) / tiles);
      const double step = a.D <= 64 ? (tiles == 2 ? 1.65 : 1.35) : (tiles == 2 ? 2.2 : 1.7);
      const auto consider = [&](int splits) {
        const double us = std::ceil(ctas * splits / kSms) *
                              (4.0 + step * ((key_tiles + splits - 1) / splits)) +
                          (splits > 1 ? 4.0 + part_us * splits : 0.0);
        if (us < least) {
          least = us;
          best = {pack, tiles, splits};
        }
      };
      consider(1);
      // more splits than that take longer to join than they save
      const double enough = std::sqrt(step * key_tiles / part_us);
      const int splits = (int)std::min({enough + 1.0, (double)(key_tiles / 2), kSms / ctas});
      if (splits > 1) {
        const int longest = (key_tiles + splits - 1) / splits;
        consider((key_tiles + longest - 1) / longest);  // the fewest with tiles that long
      }
      if (pack == most) break;
    }
  return best;
}

// Whether a cluster joins the splits, rather than a second kernel: up to 4 of them, and where all
// clusters still run at once, a cluster's CTAs having to lie in one part of the chip (pairs always find
// their SMs; with 144 CTAs in threes some waited for a second round, 39 us instead of 25 at 3 x 128 x
// 3,600, 16 heads of 64). It saves 1 to 4 us: 2 x 999 x 3,600, 8 heads of 64 in pairs 41 -> 37,
// 2 x 128 x 3,600, 16 heads of 64 in fours 20.7 -> 19.4.
static bool in_clusters(const gs_attention_args& a, const ForwardPlan& plan) {
  const long long rows = plan.tiles * kTileQ;
  const long long ctas = ((long long)plan.pack * a.Lq + rows - 1) / rows * a.B * (a.Hq / plan.pack);
  return plan.splits == 2 ||
         (plan.splits > 2 && plan.splits <= 4 && ctas * plan.splits <= 128);
}

size_t attention_forward_workspace(const gs_attention_args& a) {
  const ForwardPlan plan = forward_plan(a);
  const long long rows = (long long)a.B * a.Hq * a.Lq;
  return attention_mask_bytes(a) + (plan.splits > 1 && !in_clusters(a, plan)
                                        ? (size_t)(plan.splits * rows) * (a.D + 1) * sizeof(float)
                                        : 0);
}

template <typename T, int DP, bool MASK>
static cudaError_t launch_forward(const ForwardParams& p, const CUtensorMap& q,
                                  const CUtensorMap& k, const CUtensorMap& v,
                                  cudaStream_t stream) {
  const auto kernel = attention_forward_kernel<T, DP, MASK>;
  const cudaError_t err =
      allow_shared<attention_forward_kernel<T, DP, MASK>>(ForwardShared<DP>::kBytes);
  if (err != cudaSuccess) return err;
  const dim3 grid(p.q_blocks * p.a.B * p.groups, p.splits);
  return launch_overlapped_clusters(kernel, grid, dim3(1, p.cluster ? p.splits : 1), kFwdThreads,
                                    ForwardShared<DP>::kBytes, stream, p, q, k, v);
}

template <typename T>
static cudaError_t launch_forward(const ForwardParams& p, const CUtensorMap& q,
                                  const CUtensorMap& k, const CUtensorMap& v,
                                  cudaStream_t stream) {
  if (p.a.bits)
    return p.a.D <= 64 ? launch_forward<T, 64, true>(p, q, k, v, stream)
                       : launch_forward<T, 128, true>(p, q, k, v, stream);
  return p.a.D <= 64 ? launch_forward<T, 64, false>(p, q, k, v, stream)
                     : launch_forward<T, 128, false>(p, q, k, v, stream);
}

template <typename T>
static cudaError_t launch_combine(const AttentionParams& a, int splits, const float* out,
                                  const float* lse, cudaStream_t stream) {
  const long long rows = (long long)a.B * a.Hq * a.Lq;
  if (splits > 8)
    return launch_overlapped(combine_kernel<T, 4>, dim3((unsigned)rows), 128, 0, stream, a, splits,
                             out, lse);
  return launch_overlapped(combine_kernel<T, 1>, dim3((unsigned)((rows + 3) / 4)), 128, 0, stream,
                           a, splits, out, lse);
}

cudaError_t attention_combine(const gs_attention_args& args, int splits, const float* out,
                              const float* lse, cudaStream_t stream) {
  const AttentionParams a = attention_params(args);
  return args.dtype == GS_FP16 ? launch_combine<__half>(a, splits, out, lse, stream)
                               : launch_combine<__nv_bfloat16>(a, splits, out, lse, stream);
}

int attention_forward(const gs_attention_args& a, void* workspace, cudaStream_t stream) {
  ForwardParams p{};
  p.a = attention_params(a);
  GS_CUDA(device_error_word(&p.errors));
  const float magnitude = std::max(std::fabs(a.scale), 1e-30f);  // a scale of 0 weighs all alike
  p.scale_log2 = magnitude * 1.4426950408889634f;
  p.lag = std::min(kLag / p.scale_log2, 1e30f);
  p.negate = a.scale < 0.0f;
  const ForwardPlan plan = forward_plan(a);
  p.pack = plan.pack;
  p.tiles = plan.tiles;
  p.splits = plan.splits;
  p.cluster = in_clusters(a, plan);
  p.groups = a.Hq / p.pack, p.shared = a.Hq / a.Hkv;
  p.q_blocks = (int)(((long long)p.pack * a.Lq + p.tiles * kTileQ - 1) / (p.tiles * kTileQ));
  const size_t mask_bytes = attention_mask_bytes(a);
  if (const int status = attention_pack_mask(a, p.a, workspace, stream)) return status;
  p.part_out = reinterpret_cast<float*>(static_cast<char*>(workspace) + mask_bytes);
  const long long rows = (long long)a.B * a.Hq * a.Lq;
  p.part_lse = p.part_out + p.splits * rows * a.D;
  p.qb = a.B > 1 && a.q.batch_stride != 0, p.qh = a.Hq > 1;
  p.kb = a.B > 1 && a.k.batch_stride != 0, p.kh = a.Hkv > 1;
  p.vb = a.B > 1 && a.v.batch_stride != 0, p.vh = a.Hkv > 1;
  CUtensorMap q, k, v;
  GS_REQUIRE(encode_tokens(&q, a.dtype, a.q.data, a.D, a.Lq, a.Hq, a.B, a.q.token_stride,
                           a.q.head_stride, a.q.batch_stride, plan.pack > 1 ? a.Lq : kTileQ, plan.pack),
             "the driver refused to describe q");
  k = v = q;  // without keys nothing is copied
  if (a.Lk > 0) {
    GS_REQUIRE(encode_tokens(&k, a.dtype, a.k.data, a.D, a.Lk, a.Hkv, a.B, a.k.token_stride,
                             a.k.head_stride, a.k.batch_stride, kTileK),
               "the driver refused to describe k");
    GS_REQUIRE(encode_tokens(&v, a.dtype, a.v.data, a.D, a.Lk, a.Hkv, a.B, a.v.token_stride,
                             a.v.head_stride, a.v.batch_stride, kTileK),
               "the driver refused to describe v");
  }
  GS_CUDA(a.dtype == GS_FP16 ? launch_forward<__half>(p, q, k, v, stream)
                             : launch_forward<__nv_bfloat16>(p, q, k, v, stream));
  count_launches(1u);
  if (p.splits > 1 && !p.cluster) {
    GS_CUDA(attention_combine(a, p.splits, p.part_out, p.part_lse, stream));
    count_launches(1u);
  }
  return GS_OK;
}

}  // namespace gs
