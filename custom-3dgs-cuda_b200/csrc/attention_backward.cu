// Cross attention backward on the tensor cores.
//
//   P = exp(scale q k^T - lse),  dP = dO v^T,  dS = P o (dP - delta),  delta = rowsum(dO o O),
//   dv = P^T dO,  dk = scale dS^T q,  dq = scale dS k.
// Three kernels, none of which adds to memory that another CTA adds to, so that the sums have a
// fixed order: delta and lse of every row (prepare_kernel), then one kernel that owns tiles of
// 128 keys and walks over the queries of every head that shares them (dk, dv), and one that owns
// tiles of 128 queries and walks over the keys (dq). Both recompute S and dP: 7 products for
// each pair of tiles instead of the 5 that one kernel with shared sums would need.
//
// Both are the same kernel, with KEYS telling which side is owned. The owned ("outer") tile of 128
// rows stays in shared memory, the others ("inner", 128 rows) stream through. S and dP, outer rows
// x inner rows, are products into tensor memory; two warpgroups, each with a thread for each outer
// row and half of the inner columns, turn S into P and then dP into dS, both in 16 bits and back in
// tensor memory, where they are the left operands of the sums, with the same inner tile read
// across as the right operand.
//
// What bounds it: at D = 128 a pair of tiles takes 512 clocks of the tensor pipe for each product
// (2,048 for dk and dv, 1,536 for dq), and the exponentials 1,024 clocks of the special-function
// unit; at D = 64 the products take half of that. So S of the next tile has to be formed while
// this one's P and dS are: where tensor memory has room (512 columns: S 128, dP 128, a sum D, P and
// dS 64 each) P and dS have their own columns, S and dP are free again as soon as they have been
// read, and one warp issues S and dP, another the sums. For dk and dv at D above 64 there is no
// room: P takes S's columns and dS dP's, and one warp issues dv, the next S, dk, the next dP, each
// as its operand arrives, so that S is formed beside the dS of the tile before.
//
// Measured, 4,096 queries x 4,096 keys, 16 heads, bfloat16: at D 128 14.5 us for delta, 237 to 255 for dk
// and dv (1,080 to 1,160 TFLOP/s executed, tensor pipe 62% busy) and 159 to 178 for dq (1,160 to 1,300,
// 72%); at D 64 10, 163 to 174 and 138 to 151. 8,192 x 16,320, 16 heads of 128, forward included: 4.2 to
// 4.3 ms, 18 units of executed products of 2.7e11 operations, 1,150 to 1,170 TFLOP/s, 84 to 86% of what a
// library product sustains under the power cap (1,357).
//
// The rounding of P and dS makes a gradient about 1.4 roundings off instead of one (in norm, random inputs:
// 2.33e-3 for bfloat16, 1.66e-3 for the exact gradient rounded once). delta is formed from the output as it was
// written, in 16 bits, which adds little to that: 2.33e-3 -> 2.37e-3 with 1,200 keys of 64 numbers, 2.45e-3 ->
// 2.52e-3 with 64 keys of 80. A 32-bit copy of the output, written by the forward and read here, would
// take twice the output's memory between the two.
//
// P and dS are rounded to the products' 16-bit type, a relative error for bfloat16 down to 2^-126,
// where the exponential's results and the products' operands end. Both are formed 2^32 times
// larger and the sums scaled back, so that probabilities down to 2^-158 still count. Half has few
// exponents: P is formed 2^15 times larger there, and dS by a power of two for each (item, key head),
// whose query heads dk adds up: |dS| = P |dP - delta| is at most |dO| |v| / 2, so with the largest
// norms of a row of dO and of a kept row of v the largest dS ends up below 2^15, and those down to
// 2^-29 of it keep all their bits. (As it is, dS of 999 x 3,600 lies among half's subnormals
// from a dO of deviation 1e-3 down: 6 times the error of the results' own rounding.) Reading v once more
// for its norms takes attention_prepare_kernel from 9 to 16 us at 4,096 x 4,096, 16 heads of 64, of 393 with
// the forward. The power is at least 1: where dO is so large that dS may pass 65,504, the loss is scaled too far up, as with any
// half gradient.
#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "capi_internal.h"
#include "tensor_core.cuh"

namespace gs {

constexpr int kOuter = 128, kInner = 128;
constexpr int kBwdThreads = 384;
// Registers of a thread of the P and dS warps and of the others: 2 x 128 x 200 + 128 x 104 =
// 384 x 168, what the CTA is launched with.
constexpr int kMathRegs = 200, kRestRegs = 104;

struct BackwardParams {
  AttentionParams a;
  unsigned* errors;  // the device's error word
  float scale_log2;
  // [B, Hq, lq_pad / kInner, 2, kInner]: lse log2 e - kLog2 (+inf: no probability), delta
  const float* stats;
  int lq_pad;           // Lq rounded up to kInner
  int splits;           // of the inner tiles
  int x1b, x1h, x2b, x2h, y1b, y1h, y2b, y2h;  // 0 where items or heads share the tensor, else 1
  const float* norms;   // half only: see attention_prepare_kernel
  float* part1;  // [splits, outer rows, D] where splits > 1: dq or dk
  float* part2;  // dv
};

template <int DP, bool KEYS>
struct BackwardShared {
  static constexpr int kBoxes = DP / 64;
  static constexpr int kOuterBytes = kBoxes * kOuter * 128;
  static constexpr int kInnerBytes = kBoxes * kInner * 128;
  static constexpr bool kOwnP = !(KEYS && DP == 128);  // P and dS have their own columns
  // Tiles of y1 and of y2 in shared memory: what 227 KB hold. dq needs y2 (v) for dP alone and
  // gives it up a tile earlier than y1 (k).
  static constexpr int kStages1 = DP == 64 ? 4 : KEYS ? 2 : 3;
  static constexpr int kStages2 = DP == 64 ? 4 : 2;
  static constexpr int kStatBytes = KEYS ? kInner * 8 : 0;  // beside each y1
  static constexpr int kBytes = 1024 + 2 * kOuterBytes + (kStages1 + kStages2) * kInnerBytes +
                                kStages1 * kStatBytes;
};

// P is formed 2^kLog2 times larger, kAcc brings its sums back. kOwnDs: dS has a scale of its own
// (ds_log2), else it is P's.
template <typename T>
struct ProbabilityScale {
  static constexpr float kLog2 = 32.0f, kAcc = 1.0f / 4294967296.0f;
  static constexpr bool kOwnDs = false;
};
template <>
struct ProbabilityScale<__half> {
  static constexpr float kLog2 = 15.0f, kAcc = 1.0f / 32768.0f;
  static constexpr bool kOwnDs = true;
};

// How many powers of two dS of a key head is formed larger, from the squares of the largest norms of its
// rows of dO and v: the largest |dO| |v| / 2 comes to lie in [2^14, 2^15], where that is up.
__device__ __forceinline__ int ds_log2(const float* norms) {
  const float bound = 0.5f * sqrtf(norms[0]) * sqrtf(norms[1]);
  const int exponent = (int)(__float_as_uint(bound) >> 23) - 126;  // bound < 2^exponent
  return bound > 0.0f ? min(max(15 - exponent, 0), 60) : 0;
}

// Raises norms[0] to the largest of the CTA's values, whose 8 lanes a row agree; rows that hold a NaN or
// an infinity do not count: either no result sees them or all that do are NaN. Not negative, so
// the largest integer is the largest number, and the order of the CTAs does not matter.
__device__ __forceinline__ void raise_norm(float square, float* norm) {
  __shared__ float shared[8];
  square = square < INFINITY ? square : 0.0f;
#pragma unroll
  for (int w = 8; w < 32; w <<= 1) square = fmaxf(square, __shfl_xor_sync(~0u, square, w));
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = square;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 1; k < 8; ++k) square = fmaxf(square, shared[k]);
    atomicMax(reinterpret_cast<int*>(norm), __float_as_int(square));
  }
}

// delta and lse in powers of two of every query row, 8 lanes a row; the rows, padded to a multiple
// of kInner for each head, fill the first `query_blocks` of the grid exactly. For half also the squares
// of the largest norms of the rows of dO and of v, [B, Hkv, 2], zero before; the CTAs past the queries'
// read v, 32 keys each.
template <typename T>
__global__ void __launch_bounds__(256) attention_prepare_kernel(AttentionParams a, int lq_pad,
                                                                unsigned query_blocks, float* stats,
                                                                float* norms) {
  constexpr bool kNorms = ProbabilityScale<T>::kOwnDs;
  wait_for_previous();
  let_next_start();
  const int sub = threadIdx.x % 8;
  float square = 0.0f;
  if (kNorms && blockIdx.x >= query_blocks) {
    const unsigned key_blocks = (unsigned)(a.Lk + 31) / 32, at = blockIdx.x - query_blocks;
    const unsigned bh = at / key_blocks;
    const int j = (int)(at - bh * key_blocks) * 32 + threadIdx.x / 8;
    const int b = bh / (unsigned)a.Hkv, h = bh - b * (unsigned)a.Hkv;
    unsigned keep = ~0u;  // the CTA's 32 keys that any query keeps
    if (a.bits) {
      keep = 0;
      const unsigned* rows = a.kept + b * a.kept_b + h * a.kept_h +
                             (long long)(j / 128) * a.kept_tile + j / 32 % 4;
      for (int r = threadIdx.x % 32; r < a.kept_rows; r += 32) keep |= rows[(long long)r * a.kept_row];
      keep = __reduce_or_sync(~0u, keep);
    }
    if (j < key_count(a, b) && (keep >> (j % 32) & 1u)) {
      const T* v = a.v.at<T>(b, j, h);
      for (int d = sub * 8; d < a.D; d += 64) {
        float x[8];
        load_pack<T, 8>(v + d, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) square = fmaf(x[k], x[k], square);
      }
    }
#pragma unroll
    for (int w = 4; w; w >>= 1) square += __shfl_xor_sync(~0u, square, w);
    raise_norm(square, norms + 2ll * bh + 1);
    return;
  }
  const long long at = (long long)blockIdx.x * 32 + threadIdx.x / 8;
  const int i = (int)(at % lq_pad), h = (int)(at / lq_pad % a.Hq), b = (int)(at / lq_pad / a.Hq);
  float delta = 0.0f, lse = INFINITY;
  if (i < a.Lq) {
    const T* o = a.out.at<T>(b, i, h);
    const T* g = a.dout.at<T>(b, i, h);
    for (int d = sub * 8; d < a.D; d += 64) {
      float x[8], y[8];
      load_pack<T, 8>(o + d, x);
      load_pack<T, 8>(g + d, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) delta = fmaf(x[k], y[k], delta);
      if (kNorms)
#pragma unroll
        for (int k = 0; k < 8; ++k) square = fmaf(y[k], y[k], square);
    }
    lse = a.lse[((long long)b * a.Hq + h) * a.Lq + i];
    lse = lse == -INFINITY ? INFINITY
                           : fmaf(lse, 1.4426950408889634f, -ProbabilityScale<T>::kLog2);
  }
#pragma unroll
  for (int w = 4; w; w >>= 1) delta += __shfl_xor_sync(~0u, delta, w);
  if (lse == INFINITY) delta = 0.0f;  // keeps no key, whatever dO holds
  if (sub == 0) {
    float* tile = stats + at / kInner * (2 * kInner) + at % kInner;
    tile[0] = lse;
    tile[kInner] = delta;
  }
  if constexpr (kNorms) {
    if (lse == INFINITY) square = 0.0f;  // keeps no key
#pragma unroll
    for (int w = 4; w; w >>= 1) square += __shfl_xor_sync(~0u, square, w);
    raise_norm(square, norms + 2 * ((long long)b * a.Hkv + h / (a.Hq / a.Hkv)));
  }
}

__device__ __forceinline__ float4 ld_shared4(unsigned at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at));
  return v;
}

__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Where a column's bit in `keep` is 0: no probability (s to the side of the exponent's sign that
// gives 0), and 0 times what the value product holds there, NaN included, is 0.
__device__ __forceinline__ void hide(const unsigned (&keep)[2], bool negative, unsigned* s,
                                     unsigned* dp) {
  const unsigned none = negative ? 0x7f800000u : kMinusInf;
#pragma unroll
  for (int k = 0; k < 64; ++k)
    if (!(keep[k / 32] >> (k % 32) & 1u)) {
      if (s) s[k] = none;
      if (dp) dp[k] = 0u;
    }
}

// P = 2^(S c - lse) of 32 columns, in place. lse is the columns' in shared memory (KEYS) or the
// row's own.
template <bool KEYS>
__device__ __forceinline__ void probabilities(unsigned* s, float c, unsigned at, float own) {
#pragma unroll
  for (int k = 0; k < 32; k += 4) {
    float4 l = make_float4(own, own, own, own);
    if (KEYS) l = ld_shared4(at + k * 4);
    s[k] = __float_as_uint(fast_exp2(fmaf(__uint_as_float(s[k]), c, -l.x)));
    s[k + 1] = __float_as_uint(fast_exp2(fmaf(__uint_as_float(s[k + 1]), c, -l.y)));
    s[k + 2] = __float_as_uint(fast_exp2(fmaf(__uint_as_float(s[k + 2]), c, -l.z)));
    s[k + 3] = __float_as_uint(fast_exp2(fmaf(__uint_as_float(s[k + 3]), c, -l.w)));
  }
}

// dS = P (dP - delta) scale of 32 columns, in P's place.
template <bool KEYS>
__device__ __forceinline__ void differences(unsigned* p, const unsigned* dp, unsigned at,
                                            float own, float scale) {
#pragma unroll
  for (int k = 0; k < 32; k += 4) {
    float4 d = make_float4(own, own, own, own);
    if (KEYS) d = ld_shared4(at + k * 4);
    const auto ds = [&](int i, float delta) {
      return __float_as_uint(__uint_as_float(p[i]) * ((__uint_as_float(dp[i]) - delta) * scale));
    };
    p[k] = ds(k, d.x), p[k + 1] = ds(k + 1, d.y);
    p[k + 2] = ds(k + 2, d.z), p[k + 3] = ds(k + 3, d.w);
  }
}

// 32 columns rounded to 16 bits, into 16 columns of tensor memory.
template <typename T>
__device__ __forceinline__ void store_packed(unsigned at, const unsigned* v) {
  unsigned packed[16];
#pragma unroll
  for (int k = 0; k < 16; ++k)
    packed[k] = pack2<T>(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]));
  tc_st16(at, packed);
}

// MASK: with a mask. Without one its code and the barriers of the warp that looks the tiles over for it
// are not there (dk and dv of 2 x 999 x 3,600, 8 heads of 64: 57 us with them, 47 so).
template <typename T, int DP, bool KEYS, bool MASK>
__global__ void __launch_bounds__(kBwdThreads, 1)
    attention_backward_kernel(const __grid_constant__ BackwardParams p,
                              const __grid_constant__ CUtensorMap map_x1,
                              const __grid_constant__ CUtensorMap map_x2,
                              const __grid_constant__ CUtensorMap map_y1,
                              const __grid_constant__ CUtensorMap map_y2) {
  using S = BackwardShared<DP, KEYS>;
  using PS = ProbabilityScale<T>;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t x_full, y1_full[S::kStages1], y1_free[S::kStages1], y2_full[S::kStages2],
      y2_free[S::kStages2], y1_clean[S::kStages1], y2_clean[S::kStages2], s_full, s_read, dp_full,
      p_ready, ds_ready, acc_done, acc_full;
  __shared__ unsigned tmem_slot;
  __shared__ volatile int gave_up;
  const unsigned base = (smem_u32(raw) + 1023u) & ~1023u;
  const unsigned sm_x1 = base, sm_x2 = sm_x1 + S::kOuterBytes, sm_y1 = sm_x2 + S::kOuterBytes,
                 sm_y2 = sm_y1 + S::kStages1 * S::kInnerBytes,
                 sm_stats = sm_y2 + S::kStages2 * S::kInnerBytes;
  const int warp = warp_uniform(threadIdx.x / 32), lane = threadIdx.x % 32;
  if (threadIdx.x == 288) {  // of warp 9
    prefetch_map(&map_x1);
    prefetch_map(&map_x2);
    prefetch_map(&map_y1);
    prefetch_map(&map_y2);
    gave_up = 0;
    mbar_set(&x_full, 1);
    mbar_set(&acc_full, 1);
    for (int i = 0; i < S::kStages1; ++i) {
      mbar_set(&y1_full[i], 1);
      if (MASK) mbar_set(&y1_clean[i], 1);
      mbar_set(&y1_free[i], 1);
    }
    for (int i = 0; i < S::kStages2; ++i) {
      mbar_set(&y2_full[i], 1);
      if (MASK && KEYS) mbar_set(&y2_clean[i], 1);
      mbar_set(&y2_free[i], 1);
    }
    for (uint64_t* bar : {&s_full, &dp_full, &acc_done}) mbar_set(bar, 1);
    for (uint64_t* bar : {&s_read, &p_ready, &ds_ready}) mbar_set(bar, 8);
    mbar_ready();
  }
  __syncwarp();
  const AttentionParams& a = p.a;
  const int shared_heads = a.Hq / a.Hkv;
  const int outer_rows = KEYS ? a.Lk : a.Lq, outer_heads = KEYS ? a.Hkv : a.Hq;
  const int outer_tiles = (outer_rows + kOuter - 1) / kOuter;
  const int x0 = blockIdx.x % outer_tiles * kOuter, bh = blockIdx.x / outer_tiles;
  const int b = bh / outer_heads, ho = bh % outer_heads, hk = KEYS ? ho : ho / shared_heads;
  const int n = warp_uniform(key_count(a, b));
  const int q_tiles = p.lq_pad / kInner;
  const int tiles = KEYS ? (x0 < n ? q_tiles * shared_heads : 0) : (n + kInner - 1) / kInner;
  // dq's tiles of keys, fewer than 2^24, times at most kSms splits fit 32 bits, which divide faster
  const auto begin = [&](unsigned piece) {
    return KEYS ? piece_begin(tiles, piece, p.splits)
                : (int)((unsigned)tiles * piece / (unsigned)p.splits);
  };
  const int t0 = begin(blockIdx.y), count = begin(blockIdx.y + 1) - t0;
  const bool key_mask = MASK && a.bits_h == 0 && a.bits_q == 0;

  // dk and dv need the rows' statistics and with them the packed mask; the CTAs of dq that start
  // beside the last of dk's and dv's then find both, and only end after them
  if (KEYS) wait_for_previous();
  let_next_start();
  if (warp == 9) {  // goes on to the first copies while the others get ready
    ready_arrive<kBwdThreads>();
  } else {
    if (warp == 8) tc_alloc(&tmem_slot, 512);
    tc_fence_before();
    ready_wait<kBwdThreads>();
    tc_fence_after();
  }
  const unsigned tmem = warp == 9 ? 0u : (unsigned)warp_uniform((int)tmem_slot);
  // Tensor memory: S, dP, the sums, P and dS (in S's and dP's columns unless kOwnP). The 16-bit
  // numbers of warpgroup w's 64 inner columns take 32 columns from w * kHalf on.
  constexpr unsigned kHalf = S::kOwnP ? 32 : 64;
  const unsigned tm_s = tmem, tm_dp = tmem + 128, tm_acc1 = tmem + 256,
                 tm_acc2 = tmem + 256 + DP;
  const unsigned tm_p = S::kOwnP ? tmem + 384 : tm_s, tm_ds = S::kOwnP ? tmem + 448 : tm_dp;
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMathRegs));
    // ---- P and dS: one thread for each outer row ----
    const int wg = warp / 4, row = threadIdx.x % 128, x = x0 + row;
    const unsigned lanes = (unsigned)(warp % 4 * 32) << 16;
    const float c = p.scale_log2;
    // dS's scale over P's, and dS's back to 1; dq, which needs P for dS alone, forms P with dS's scale
    float ds_up = 1.0f, ds_back = PS::kAcc, p_log2 = 0.0f;
    if (PS::kOwnDs && count > 0) {
      const int k = ds_log2(p.norms + 2 * ((long long)b * a.Hkv + hk));
      ds_back = __uint_as_float((unsigned)(127 - k) << 23);
      if (KEYS)
        ds_up = PS::kAcc / ds_back;
      else
        p_log2 = (float)k - PS::kLog2;
    }
    float2 mine = make_float2(INFINITY, 0.0f);
    const unsigned* keep_row = nullptr;
    // KEYS: the warp's 32 keys that are below the length, and that a key mask leaves
    unsigned alive = 0;
    if (KEYS) {
      alive = below(n - x0, warp % 4);
      if (key_mask) alive &= a.bits[b * a.bits_b + x0 / 32 + warp % 4];
    } else {
      if (x < a.Lq) {
        const float* tile = p.stats + (((long long)b * a.Hq + ho) * p.lq_pad + x0) * 2 + row;
        mine = make_float2(tile[0] - p_log2, tile[kInner]);
      }
      if (MASK)
        keep_row = a.bits + b * a.bits_b + ho * a.bits_h + (long long)min(x, a.Lq - 1) * a.bits_q;
    }
    const unsigned my_s = tm_s + lanes + wg * 64, my_dp = tm_dp + lanes + wg * 64,
                   my_p = tm_p + lanes + wg * kHalf, my_ds = tm_ds + lanes + wg * kHalf;
    bool ok = true;
    for (int j = 0; j < count; ++j) {
      const int st = j % S::kStages1, t = t0 + j;
      const int y0 = (KEYS ? t % q_tiles : t) * kInner + wg * 64;  // first of this thread's columns
      const bool hidden = MASK || (KEYS ? x0 + kOuter > n : y0 + 64 > n);
      unsigned keep[2] = {~0u, ~0u};
      if (hidden) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (KEYS) {
            keep[w] = alive >> lane & 1u ? ~0u : 0u;
            if (MASK && !key_mask) {
              // lane k has the word of query y0 + 32 w + k for the warp's 32 keys; each lane
              // gathers its own key's bit of all 32
              const int head = ho * shared_heads + t / q_tiles;
              const unsigned word =
                  a.bits[b * a.bits_b + head * a.bits_h +
                         (long long)min(y0 + 32 * w + lane, a.Lq - 1) * a.bits_q + x0 / 32 +
                         warp % 4];
              unsigned column = 0;
#pragma unroll
              for (int k = 0; k < 32; ++k)
                column |= (__shfl_sync(~0u, word, k) >> lane & 1u) << k;
              keep[w] &= column;
            }
          } else {
            keep[w] = below(n - y0, w);
            if (keep_row) keep[w] &= keep_row[y0 / 32 + w];
          }
        }
      }
      ok = tc_wait_warp(&s_full, j & 1);
      // the statistics came by the copy engine: their own barrier makes them visible
      if (KEYS && ok) ok = tc_wait_warp(&y1_full[st], j / S::kStages1 & 1);
      if (!ok) break;
      tc_fence_after();
      const unsigned stat = sm_stats + st * S::kStatBytes + wg * 64 * 4;
      unsigned pr[64], dp[64];  // S, then P in 32 bits; dP
      tc_ld32(my_s, pr);
      tc_ld32(my_s + 32, pr + 32);
      if constexpr (S::kOwnP) {
        tc_ld32(my_dp, dp);
        tc_ld32(my_dp + 32, dp + 32);
        tc_wait_ld();
        tc_fence_before();
        mbar_arrive_warp(&s_read);  // the next scores may overwrite these
        if (hidden) hide(keep, c < 0.0f, pr, dp);
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
          probabilities<KEYS>(pr + h, c, stat + h * 4, mine.x);
          if (h == 0 && j > 0) {  // the products that read the P and dS before are over
            ok = tc_wait_warp(&acc_done, (j - 1) & 1);
            tc_fence_after();
          }
          if (KEYS) store_packed<T>(my_p + h / 2, pr + h);
          differences<KEYS>(pr + h, dp + h, stat + kInner * 4 + h * 4, mine.y, ds_up);
          store_packed<T>(my_ds + h / 2, pr + h);
        }
        if (!ok) break;
      } else {
        tc_wait_ld();
        if (hidden) hide(keep, c < 0.0f, pr, nullptr);
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
          probabilities<KEYS>(pr + h, c, stat + h * 4, mine.x);
          store_packed<T>(my_p + h / 2, pr + h);
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive_warp(&p_ready);
        ok = tc_wait_warp(&dp_full, j & 1);
        if (!ok) break;
        tc_fence_after();
        tc_ld32(my_dp, dp);
        tc_ld32(my_dp + 32, dp + 32);
        tc_wait_ld();
        if (hidden) hide(keep, c < 0.0f, nullptr, dp);
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
          differences<KEYS>(pr + h, dp + h, stat + kInner * 4 + h * 4, mine.y, ds_up);
          store_packed<T>(my_ds + h / 2, pr + h);
        }
      }
      tc_wait_st();
      tc_fence_before();
      mbar_arrive_warp(&ds_ready);
    }
    if (ok && count > 0) ok = tc_wait_warp(&acc_full, 0);
    if (!ok) gave_up = 1;
    tc_fence_after();
    // KEYS: the first warpgroup writes dk, the second dv; else they take half of dq's columns each
    const bool first = !KEYS || wg == 0;
    const float factor = first ? a.scale * ds_back : PS::kAcc;
    const TokenView& view = KEYS ? (first ? a.dk : a.dv) : a.dq;
    const long long rows = (long long)a.B * outer_heads * outer_rows;
    float* part = first ? p.part1 : p.part2;
    const int d = KEYS ? 0 : wg * (DP / 2), r0 = x - lane;
    // the outer tiles in shared memory have done their work
    constexpr int kCols = KEYS ? DP : DP / 2;
    const bool wide = p.splits > 1;
    char* to = wide ? reinterpret_cast<char*>(
                          part +
                          (blockIdx.y * rows + (long long)bh * outer_rows + r0) * a.D + d)
                    : reinterpret_cast<char*>(view.at<T>(b, r0, ho) + d);
    store_rows<T, kCols>((first ? tm_acc1 : tm_acc2) + lanes + d, ok && count > 0, true, factor,
                         a.D - d, wide, (wg ? sm_x2 : sm_x1) + warp % 4 * (kCols * 64), to,
                         wide ? a.D * 4ll : view.l * 2, outer_rows - r0);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRestRegs));
    if (warp == 9) {
      // ---- copies ----
      if (lane == 0 && count > 0) {
        mbar_arrive_expect_tx(&x_full, 2 * S::kOuterBytes);
        for (int x = 0; x < S::kBoxes; ++x) {
          tma_load_4d(sm_x1 + x * kOuter * 128, &map_x1, x * 64, x0, ho * p.x1h, b * p.x1b, &x_full);
          tma_load_4d(sm_x2 + x * kOuter * 128, &map_x2, x * 64, x0, ho * p.x2h, b * p.x2b, &x_full);
        }
        for (int j = 0; j < count; ++j) {
          const int t = t0 + j;
          const int head = KEYS ? ho * shared_heads + t / q_tiles : hk;
          const int y = (KEYS ? t % q_tiles : t) * kInner;
          const int st1 = j % S::kStages1, st2 = j % S::kStages2;
          if (!tc_wait(&y1_free[st1], (j / S::kStages1 & 1) ^ 1)) { gave_up = 1; break; }
          mbar_arrive_expect_tx(&y1_full[st1], S::kInnerBytes + S::kStatBytes);
          for (int x = 0; x < S::kBoxes; ++x)
            tma_load_4d(sm_y1 + st1 * S::kInnerBytes + x * kInner * 128, &map_y1, x * 64, y,
                        head * p.y1h, b * p.y1b, &y1_full[st1]);
          if (KEYS)
            bulk_load(sm_stats + st1 * S::kStatBytes,
                      p.stats + (((long long)b * a.Hq + head) * p.lq_pad + y) * 2, S::kStatBytes,
                      &y1_full[st1]);
          if (!tc_wait(&y2_free[st2], (j / S::kStages2 & 1) ^ 1)) { gave_up = 1; break; }
          mbar_arrive_expect_tx(&y2_full[st2], S::kInnerBytes);
          for (int x = 0; x < S::kBoxes; ++x)
            tma_load_4d(sm_y2 + st2 * S::kInnerBytes + x * kInner * 128, &map_y2, x * 64, y,
                        head * p.y2h, b * p.y2b, &y2_full[st2]);
        }
      }
    } else if (warp == 8 || (warp == 10 && S::kOwnP)) {
      // ---- products ----
      const int steps = (a.D + 15) / 16;
      const unsigned idesc_s = tc_idesc<T>(kInner, false);
      const unsigned idesc_acc = tc_idesc<T>(steps * 16, true);
      // descriptor units are 16 bytes; y is read along its rows and across them
      const uint64_t desc_x1 = tc_desc(sm_x1, 16), desc_x2 = tc_desc(sm_x2, 16),
                     desc_y1 = tc_desc(sm_y1, 16), desc_y2 = tc_desc(sm_y2, 16),
                     desc_y1t = tc_desc(sm_y1, kInner * 128),
                     desc_y2t = tc_desc(sm_y2, kInner * 128);
      const auto in1 = [](int j) { return j % S::kStages1 * (S::kInnerBytes / 16); };
      const auto in2 = [](int j) { return j % S::kStages2 * (S::kInnerBytes / 16); };
      // S (second = 0) or dP (1) of inner tile j
      const auto scores = [&](int j, int second) {
        const uint64_t in = second ? desc_y2 + in2(j) : desc_y1 + in1(j);
        const uint64_t out = second ? desc_x2 : desc_x1;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          if (k < steps)
            tc_mma_ss(second ? tm_dp : tm_s, out + (k / 4) * (kOuter * 8) + (k % 4) * 2,
                      in + (k / 4) * (kInner * 8) + (k % 4) * 2, idesc_s, k > 0);
      };
      // acc2 += P y2 (second = 1) or acc1 += dS y1 (0)
      const auto sums = [&](int j, int second) {
        const uint64_t in = second ? desc_y2t + in2(j) : desc_y1t + in1(j);
#pragma unroll
        for (int k = 0; k < kInner / 16; ++k)
          tc_mma_ts(second ? tm_acc2 : tm_acc1,
                    (second ? tm_p : tm_ds) + (k / 4) * kHalf + (k % 4) * 8, in + k * 128,
                    idesc_acc, j > 0 || k > 0);
      };
      // with a mask, another warp has looked the tiles over
      const auto arrived1 = [&](int j) {
        const int st = j % S::kStages1, left = n - (t0 + j) * kInner;
        if (!tc_wait_warp(MASK ? &y1_clean[st] : &y1_full[st], j / S::kStages1 & 1)) return false;
        if (!KEYS && !MASK && warp == 8 && left < kInner)  // k past the length
          clear_rows<S::kBoxes>(sm_y1 + st * S::kInnerBytes, left, make_uint4(~0u, ~0u, ~0u, ~0u));
        return true;
      };
      const auto arrived2 = [&](int j) {
        const int st = j % S::kStages2;
        return tc_wait_warp(KEYS && MASK ? &y2_clean[st] : &y2_full[st], j / S::kStages2 & 1);
      };
      const auto when = [&](uint64_t* bar, int j) {
        const bool done = tc_wait_warp(bar, j & 1);
        tc_fence_after();
        return done;
      };
      bool ok = count > 0;
      if (warp == 8) ok = ok && tc_wait_warp(&x_full, 0);
      if (S::kOwnP && warp == 8) {
        for (int j = 0; ok && j < count; ++j) {
          ok = arrived1(j) && (j == 0 || when(&s_read, j - 1));
          if (ok && elect_one()) scores(j, 0);
          __syncwarp();
          ok = ok && arrived2(j);
          if (ok && elect_one()) {
            scores(j, 1);
            tc_commit(&s_full);
            if (!KEYS) tc_commit(&y2_free[j % S::kStages2]);
          }
          __syncwarp();
        }
      } else if (S::kOwnP) {
        for (int j = 0; ok && j < count; ++j) {
          ok = arrived1(j) && (!KEYS || arrived2(j)) && when(&ds_ready, j);
          if (ok && elect_one()) {
            if (KEYS) sums(j, 1);
            sums(j, 0);
            tc_commit(&acc_done);
            if (KEYS) tc_commit(&y2_free[j % S::kStages2]);
            tc_commit(&y1_free[j % S::kStages1]);
            if (j + 1 == count) tc_commit(&acc_full);
          }
          __syncwarp();
        }
      } else {
        ok = ok && arrived1(0) && arrived2(0);
        if (ok && elect_one()) {
          scores(0, 0);
          tc_commit(&s_full);
          scores(0, 1);
          tc_commit(&dp_full);
        }
        __syncwarp();
        for (int j = 0; ok && j < count; ++j) {
          ok = when(&p_ready, j);
          if (ok && elect_one()) {
            sums(j, 1);  // dP of this tile was issued before: y2 is free after both
            tc_commit(&y2_free[j % S::kStages2]);
          }
          __syncwarp();
          if (j + 1 < count) {
            ok = ok && arrived1(j + 1);
            if (ok && elect_one()) {
              scores(j + 1, 0);
              tc_commit(&s_full);
            }
            __syncwarp();
            ok = ok && arrived2(j + 1);
          }
          ok = ok && when(&ds_ready, j);
          if (ok && elect_one()) {
            sums(j, 0);
            tc_commit(&y1_free[j % S::kStages1]);
            if (j + 1 < count) {
              scores(j + 1, 1);
              tc_commit(&dp_full);
            } else {
              tc_commit(&acc_full);
            }
          }
          __syncwarp();
        }
      }
      if (!ok && count > 0) gave_up = 1;
    } else if (warp == 11 && KEYS && MASK) {
      // ---- nor must what q and dO hold at queries that keep no key reach dk and dv
      for (int j = 0; j < count; ++j) {
        const int st1 = j % S::kStages1, st2 = j % S::kStages2;
        if (!tc_wait_warp(&y1_full[st1], j / S::kStages1 & 1)) { gave_up = 1; break; }
        unsigned keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {  // the rows past the last query are zero as it is
          float lse;
          asm volatile("ld.shared.f32 %0, [%1];"
                       : "=f"(lse)
                       : "r"(sm_stats + st1 * S::kStatBytes + (32 * w + lane) * 4));
          keep[w] = __ballot_sync(~0u, lse != INFINITY) |
                    ~below(a.Lq - (t0 + j) % q_tiles * kInner, w);
        }
        const uint4 rows = make_uint4(keep[0], keep[1], keep[2], keep[3]);
        const bool some = has_hidden_rows(kInner, rows);
        if (some) clear_rows<S::kBoxes>(sm_y1 + st1 * S::kInnerBytes, kInner, rows);
        mbar_arrive_warp(&y1_clean[st1]);
        if (!tc_wait_warp(&y2_full[st2], j / S::kStages2 & 1)) { gave_up = 1; break; }
        if (some) clear_rows<S::kBoxes>(sm_y2 + st2 * S::kInnerBytes, kInner, rows);
        mbar_arrive_warp(&y2_clean[st2]);
      }
    } else if (warp == 11 && !KEYS && MASK) {
      // ---- what k holds at keys that no query of the item's key head keeps must not reach dq, where
      // 0 times NaN would be added: those rows are set to zero before the products may read them
      for (int j = 0; j < count; ++j) {
        const int st = j % S::kStages1, key = (t0 + j) * kInner;
        uint4 keep = kept_begin(a, b, hk, t0 + j);
        if (!tc_wait_warp(&y1_full[st], j / S::kStages1 & 1)) { gave_up = 1; break; }
        keep = kept_end(keep);
        if (has_hidden_rows(n - key, keep))
          clear_rows<S::kBoxes>(sm_y1 + st * S::kInnerBytes, n - key, keep);
        mbar_arrive_warp(&y1_clean[st]);
      }
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
  if (!KEYS) wait_for_previous();
}

// out[b, row, h] = the sum of the splits' parts, in order.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float* part, int splits,
                                                        TokenView out, int rows_a_head, int heads,
                                                        long long rows, int D) {
  const int per_row = D / 4;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= rows * per_row) return;
  const long long row = at / per_row;
  const int d = (int)(at % per_row) * 4;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int k = 0; k < splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(part + (k * rows + row) * D + d);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const int x = (int)(row % rows_a_head), bh = (int)(row / rows_a_head);
  T* o = out.at<T>(bh / heads, x, bh % heads) + d;
  *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

struct BackwardPlan {
  int key_splits = 1, query_splits = 1;
  long long lq_pad = 0, norm_floats = 0, key_floats = 0, query_floats = 0;
  size_t bytes = 0;
};

// The inner tiles are split where the outer tiles leave SMs idle, each split with at least two.
static BackwardPlan backward_plan(const gs_attention_args& a) {
  BackwardPlan plan;
  const auto tiles = [](long long rows, long long tile) { return (rows + tile - 1) / tile; };
  const auto splits = [](long long ctas, long long inner) {
    return (int)std::max(1ll, std::min(kSms / std::max(1ll, ctas), inner / 2));
  };
  plan.lq_pad = tiles(a.Lq, kInner) * kInner;
  if (a.Hkv > 0)
    plan.key_splits = splits((long long)a.B * a.Hkv * tiles(a.Lk, kOuter),
                             tiles(a.Lq, kInner) * (a.Hq / a.Hkv));
  plan.query_splits = splits((long long)a.B * a.Hq * tiles(a.Lq, kOuter), tiles(a.Lk, kInner));
  if (plan.key_splits > 1)
    plan.key_floats = (long long)plan.key_splits * a.B * a.Hkv * a.Lk * a.D;
  if (plan.query_splits > 1)
    plan.query_floats = (long long)plan.query_splits * a.B * a.Hq * a.Lq * a.D;
  if (a.dtype == GS_FP16 && plan.lq_pad && a.Hq > 0)
    plan.norm_floats = ((long long)a.B * a.Hkv * 2 + 3) / 4 * 4;
  // dk, dv and dq in turn use the same parts
  plan.bytes = (size_t)((long long)a.B * a.Hq * plan.lq_pad * 2 + plan.norm_floats) * sizeof(float) +
               (size_t)std::max(2 * plan.key_floats, plan.query_floats) * sizeof(float);
  return plan;
}

size_t attention_backward_workspace(const gs_attention_args& a) {
  return attention_mask_bytes(a) + backward_plan(a).bytes;
}

template <typename T, int DP, bool KEYS, bool MASK>
static cudaError_t launch_backward(const BackwardParams& p, const CUtensorMap (&m)[4],
                                   bool overlapped, cudaStream_t stream) {
  const auto kernel = attention_backward_kernel<T, DP, KEYS, MASK>;
  const cudaError_t err =
      allow_shared<attention_backward_kernel<T, DP, KEYS, MASK>>(BackwardShared<DP, KEYS>::kBytes);
  if (err != cudaSuccess) return err;
  const int rows = KEYS ? p.a.Lk : p.a.Lq, heads = KEYS ? p.a.Hkv : p.a.Hq;
  const dim3 grid((rows + kOuter - 1) / kOuter * p.a.B * heads, p.splits);
  if (overlapped)
    return launch_overlapped(kernel, grid, kBwdThreads, BackwardShared<DP, KEYS>::kBytes, stream, p,
                             m[0], m[1], m[2], m[3]);
  kernel<<<grid, kBwdThreads, BackwardShared<DP, KEYS>::kBytes, stream>>>(p, m[0], m[1], m[2], m[3]);
  return cudaGetLastError();
}

template <typename T, bool KEYS>
static cudaError_t launch_backward(const BackwardParams& p, const CUtensorMap (&m)[4],
                                   bool overlapped, cudaStream_t stream) {
  if (p.a.bits)
    return p.a.D <= 64 ? launch_backward<T, 64, KEYS, true>(p, m, overlapped, stream)
                       : launch_backward<T, 128, KEYS, true>(p, m, overlapped, stream);
  return p.a.D <= 64 ? launch_backward<T, 64, KEYS, false>(p, m, overlapped, stream)
                     : launch_backward<T, 128, KEYS, false>(p, m, overlapped, stream);
}

template <typename T>
static cudaError_t launch_add(const float* part, int splits, const TokenView& out, int rows_a_head,
                              int heads, int B, int D, cudaStream_t stream) {
  const long long rows = (long long)B * heads * rows_a_head;
  add_parts_kernel<T><<<(unsigned)((rows * (D / 4) + 255) / 256), 256, 0, stream>>>(
      part, splits, out, rows_a_head, heads, rows, D);
  return cudaGetLastError();
}

template <typename T>
static int run_backward(const gs_attention_args& a, const gs_token_view& dout,
                        const gs_token_view& dq, const gs_token_view& dk, const gs_token_view& dv,
                        void* workspace, cudaStream_t stream) {
  const BackwardPlan plan = backward_plan(a);
  BackwardParams p{};
  p.a = attention_params(a);
  GS_CUDA(device_error_word(&p.errors));
  p.a.dout = TokenView(dout), p.a.dq = TokenView(dq), p.a.dk = TokenView(dk),
  p.a.dv = TokenView(dv);
  // a scale of 0 weighs all keys alike; -inf, where a key is left out, has to stay what it is
  p.scale_log2 = (a.scale == 0.0f ? 1e-30f : a.scale) * 1.4426950408889634f;
  p.lq_pad = (int)plan.lq_pad;
  const size_t mask_bytes = attention_mask_bytes(a);
  float* stats = reinterpret_cast<float*>(static_cast<char*>(workspace) + mask_bytes);
  p.stats = stats;
  const long long stat_rows = (long long)a.B * a.Hq * plan.lq_pad;
  float* norms = stats + 2 * stat_rows;
  p.norms = norms;
  float* parts = norms + plan.norm_floats;
  // before the mask's kernel, beside whose end the next one may then start
  if (plan.norm_floats)
    GS_CUDA(cudaMemsetAsync(norms, 0, plan.norm_floats * sizeof(float), stream));
  if (const int status = attention_pack_mask(a, p.a, workspace, stream)) return status;
  if (stat_rows) {
    const unsigned query_blocks = (unsigned)(stat_rows / 32);
    const long long key_blocks = plan.norm_floats ? (long long)a.B * a.Hkv * ((a.Lk + 31) / 32) : 0;
    GS_CUDA(launch_overlapped(attention_prepare_kernel<T>, dim3((unsigned)(query_blocks + key_blocks)),
                              256, 0, stream, p.a, p.lq_pad, query_blocks, stats, norms));
    count_launches(1u);
  }
  // Outer and inner tiles have the same box, so one map of each tensor serves both kernels. A map
  // whose tensor has no rows is never used and stands for any other.
  static_assert(kOuter == kInner, "one box for both");
  const auto describe = [&](CUtensorMap* map, const gs_token_view& v, int L, int H) {
    return encode_tokens(map, a.dtype, v.data, a.D, L, H, a.B, v.token_stride, v.head_stride,
                         v.batch_stride, kOuter);
  };
  const auto items = [&](const gs_token_view& v) { return a.B > 1 && v.batch_stride != 0; };
  CUtensorMap map_q{}, map_g{}, map_k{}, map_v{};
  GS_REQUIRE((a.Lk == 0 || (describe(&map_k, a.k, a.Lk, a.Hkv) && describe(&map_v, a.v, a.Lk, a.Hkv))) &&
                 (stat_rows == 0 ||
                  (describe(&map_q, a.q, a.Lq, a.Hq) && describe(&map_g, dout, a.Lq, a.Hq))),
             "the driver refused to describe a tensor");
  if (stat_rows == 0) map_q = map_g = map_k;
  if (a.Lk == 0) map_k = map_v = map_q;
  if (a.Lk > 0) {
    p.x1b = items(a.k), p.x2b = items(a.v), p.y1b = items(a.q), p.y2b = items(dout);
    p.x1h = p.x2h = a.Hkv > 1, p.y1h = p.y2h = a.Hq > 1;
    p.splits = plan.key_splits;
    p.part1 = parts, p.part2 = parts + plan.key_floats;
    const CUtensorMap m[4] = {map_k, map_v, map_q, map_g};
    GS_CUDA((launch_backward<T, true>(p, m, stat_rows > 0, stream)));
    count_launches(1u);
    if (p.splits > 1) {
      GS_CUDA(launch_add<T>(p.part1, p.splits, p.a.dk, a.Lk, a.Hkv, a.B, a.D, stream));
      GS_CUDA(launch_add<T>(p.part2, p.splits, p.a.dv, a.Lk, a.Hkv, a.B, a.D, stream));
      count_launches(2u);
    }
  }
  if (!stat_rows) return GS_OK;
  p.x1b = items(a.q), p.x2b = items(dout), p.y1b = items(a.k), p.y2b = items(a.v);
  p.x1h = p.x2h = a.Hq > 1, p.y1h = p.y2h = a.Hkv > 1;
  p.splits = plan.query_splits;
  p.part1 = parts, p.part2 = nullptr;
  const CUtensorMap m[4] = {map_q, map_g, map_k, map_v};
  // dq starts beside the end of dk and dv, unless both use the parts in turn
  const bool beside = a.Lk > 0 && (plan.key_splits == 1 || plan.query_splits == 1);
  GS_CUDA((launch_backward<T, false>(p, m, beside, stream)));
  count_launches(1u);
  if (p.splits > 1) {
    GS_CUDA(launch_add<T>(p.part1, p.splits, p.a.dq, a.Lq, a.Hq, a.B, a.D, stream));
    count_launches(1u);
  }
  return GS_OK;
}

int attention_backward(const gs_attention_args& a, const gs_token_view& dout,
                       const gs_token_view& dq, const gs_token_view& dk, const gs_token_view& dv,
                       void* workspace, cudaStream_t stream) {
  return a.dtype == GS_FP16
             ? run_backward<__half>(a, dout, dq, dk, dv, workspace, stream)
             : run_backward<__nv_bfloat16>(a, dout, dq, dk, dv, workspace, stream);
}

}  // namespace gs
