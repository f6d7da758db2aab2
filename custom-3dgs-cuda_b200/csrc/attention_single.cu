// Cross attention forward for single queries: up to 16 rows (D above 64: 8) share the keys of a
// (batch item, key head), counting the query heads that share the key head and the queries of each.
//
// Bound by HBM: every key and value is read once, for a few rows of work on it. 2 x 65,280 keys, 32
// query heads on 8 of 128, half: 82 us back to back, 6.5 TB/s; 4 x 3,600 keys of 16 heads of 64: 12.5 us,
// of which the loads' latency is the larger part (five rounds of them a warp). So nothing is
// staged: each lane loads 16 bytes of a row of k or v straight into the registers in which the
// warp-wide product (16 x 8 x 16) takes them. The product's contraction index may be numbered
// freely as long as both operands agree, which turns a lane's 8 consecutive numbers into the
// fragments of two steps:
//   S^T[16 keys, 8 rows] = k q^T: A from k, lane (g = lane / 4, t = lane % 4) holds keys g, g + 8;
//   O^T[16 numbers, 8 rows] += v^T P^T: A from v, the lane holds keys 2t, 2t + 1, 2t + 8, 2t + 9
//   and interleaves pairs of them by byte permutes; P^T is S^T's fragment transposed in 8 x 8.
// Rows are columns of both results, so the running maximum of a row is rescaled in place. P is rounded
// to 16 bits for the second product; half, which has few exponents, takes it 2^15 times larger, so
// that weights down to 2^-29 of the largest keep all their bits.
// A warp walks over chunks of 16 keys (D above 64) or 32, the next chunk's loads in flight while
// it works on this one; CTAs of 4 warps split the keys, and a cluster joins its CTAs' parts or, where
// there are more than 8, combine_kernel.
#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "capi_internal.h"
#include "tensor_core.cuh"

namespace gs {

constexpr int kSingleWarps = 4;
// P is formed 2^kUp times larger.
template <typename T>
constexpr float kUp = 0.0f;
template <>
constexpr float kUp<__half> = kHalfLog2;
constexpr int kClusterSplits = 8;  // at most, of those that a cluster joins
// resident CTAs an SM, by groups of 8 rows: 168 registers a thread hold one, 255 two
constexpr int single_ctas(int groups) { return groups == 1 ? 3 : 2; }

struct SingleParams {
  AttentionParams a;
  float scale_log2;  // scale * log2 e
  int splits, rows;  // rows = Lq * Hq / Hkv
  int cluster;       // the splits of a key head are a cluster, which joins them itself
  float* part_out;
  float* part_lse;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2,
                                         unsigned a3, unsigned b0, unsigned b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], unsigned a0, unsigned a1,
                                                 unsigned a2, unsigned a3, unsigned b0,
                                                 unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], unsigned a0, unsigned a1,
                                                        unsigned a2, unsigned a3, unsigned b0,
                                                        unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Not the read-only path: this kernel may start while the one that makes q, k or v still runs.
__device__ __forceinline__ uint4 load16(const void* p, bool in) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (in)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

__device__ __forceinline__ unsigned part(const uint4& v, int u) {
  return u == 0 ? v.x : u == 1 ? v.y : u == 2 ? v.z : v.w;
}

// DP: head size rounded up to 64 or 128. NT: groups of 8 rows. Calls without a mask have
// a kernel of their own (2 x 65,280 keys, 8 heads of 128: 94 -> 82 us, 4 x 3,600 of 16 of 64: 14.7 -> 12.5).
template <typename T, int DP, int NT, bool MASK>
__global__ void __launch_bounds__(kSingleWarps * 32, single_ctas(NT))
    attention_single_kernel(const __grid_constant__ SingleParams p) {
  constexpr int MT = 128 / DP;        // blocks of 16 keys in a chunk
  constexpr int kChunk = 16 * MT;
  constexpr int KL = DP / 32;         // 16-byte loads a lane makes of a row of k
  constexpr int VB = DP / 64;         // blocks of 64 numbers of v
  wait_for_previous();
  let_next_start();
  const AttentionParams& a = p.a;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int shared_heads = a.Hq / a.Hkv;
  const int b = blockIdx.x / a.Hkv, hk = blockIdx.x % a.Hkv;
  const int n = key_count(a, b);
  const int chunks = (n + kChunk - 1) / kChunk;
  const int c0 = piece_begin(chunks, blockIdx.y, p.splits);
  const int c1 = piece_begin(chunks, blockIdx.y + 1, p.splits);
  const unsigned char* mask_b = a.mask + b * a.mask_b;

  const auto head_of = [&](int r) { return hk * shared_heads + r % shared_heads; };
  uint4 q[NT][KL];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g;
    const bool in = r < p.rows;
    const T* row = in ? a.q.at<T>(b, r / shared_heads, head_of(r)) : nullptr;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int d = (i * 4 + t) * 8;
      q[nt][i] = load16(row + d, in && d < a.D);
    }
  }
  // the mask rows of the two query rows whose scores this lane holds in each group of 8
  const unsigned char* mask_row[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = min(nt * 8 + 2 * t + e, p.rows - 1);
      mask_row[nt][e] = mask_b + (long long)head_of(r) * a.mask_h +
                        (long long)(r / shared_heads) * a.mask_q;
    }

  const T* kp = a.k.at<T>(b, 0, hk);
  const T* vp = a.v.at<T>(b, 0, hk);
  uint4 kr[MT][2][KL], vr[MT][VB][4];
  const auto load_k = [&](int c) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = c * kChunk + m * 16 + g + 8 * e;
        const bool in = c < c1 && j < n;
        const T* row = kp + (long long)j * a.k.l;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const int d = (i * 4 + t) * 8;
          kr[m][e][i] = load16(row + d, in && d < a.D);
        }
      }
  };
  const auto load_v = [&](int c) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = c * kChunk + m * 16 + 2 * t + (e & 1) + 8 * (e >> 1);
        const bool in = c < c1 && j < n;
        const T* row = vp + (long long)j * a.v.l;
#pragma unroll
        for (int x = 0; x < VB; ++x) {
          const int d = x * 64 + g * 8;
          vr[m][x][e] = load16(row + d, in && d < a.D);
        }
      }
  };

  float o[NT][VB][4][4] = {};
  float m_row[NT][2], l_row[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) m_row[nt][e] = -INFINITY, l_row[nt][e] = 0.0f;

  int c = c0 + warp;
  load_k(c);
  load_v(c);
  for (; c < c1; c += kSingleWarps) {
    float s[NT][MT][4] = {};
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const uint4 x = kr[m][0][i], y = kr[m][1][i];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816<T>(s[nt][m], x.x, y.x, x.y, y.y, q[nt][i].x, q[nt][i].y);
          mma16816<T>(s[nt][m], x.z, y.z, x.w, y.w, q[nt][i].z, q[nt][i].w);
        }
      }
    load_k(c + kSingleWarps);
    unsigned pt[NT][MT][2];
    unsigned kept = 0;  // bit 2 m + e: key g + 8 e of block m, by one of this lane's rows
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // key g + 8 (e / 2), row 2t + e % 2
          const int j = c * kChunk + m * 16 + g + 8 * (e >> 1);
          float v = s[nt][m][e] * p.scale_log2;
          if (j >= n || (MASK && !mask_row[nt][e & 1][j]))
            v = -INFINITY;
          else if (MASK)
            kept |= 1u << (2 * m + (e >> 1));
          s[nt][m][e] = v;
          top[e & 1] = fmaxf(top[e & 1], v);
        }
#pragma unroll
      for (int w = 4; w < 32; w <<= 1)
#pragma unroll
        for (int e = 0; e < 2; ++e) top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], w));
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float m_new = fmaxf(m_row[nt][e], top[e]);
        f[e] = m_new == m_row[nt][e] ? 1.0f : fast_exp2(m_row[nt][e] - m_new);
        m_row[nt][e] = m_new;
      }
      if (__any_sync(~0u, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
        for (int x = 0; x < VB; ++x)
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][x][u][e] *= f[e & 1];
        l_row[nt][0] *= f[0];
        l_row[nt][1] *= f[1];
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float top_e = m_row[nt][e & 1];
          s[nt][m][e] = fast_exp2(s[nt][m][e] - (top_e == -INFINITY ? 0.0f : top_e) + kUp<T>);
          l_row[nt][e & 1] += s[nt][m][e];
        }
        pt[nt][m][0] = transpose8x8(pack2<T>(s[nt][m][0], s[nt][m][1]));
        pt[nt][m][1] = transpose8x8(pack2<T>(s[nt][m][2], s[nt][m][3]));
      }
    }
    if (MASK) {
      // what v holds at a key that none of the rows keeps must not be multiplied with its weight of 0:
      // lanes 4 g .. 4 g + 3 know of key g + 8 e, this one holds keys 2 t, 2 t + 1 + 8 e of v
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned all = __ballot_sync(~0u, kept >> (2 * m + (e >> 1)) & 1u);
          if (!(all >> (4 * (2 * t + (e & 1))) & 0xfu))
#pragma unroll
            for (int x = 0; x < VB; ++x) vr[m][x][e] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < VB; ++x)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const unsigned k0 = part(vr[m][x][0], u), k1 = part(vr[m][x][1], u),
                         k8 = part(vr[m][x][2], u), k9 = part(vr[m][x][3], u);
          const unsigned a0 = __byte_perm(k0, k1, 0x5410), a1 = __byte_perm(k0, k1, 0x7632),
                         a2 = __byte_perm(k8, k9, 0x5410), a3 = __byte_perm(k8, k9, 0x7632);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<T>(o[nt][x][u], a0, a1, a2, a3, pt[nt][m][0], pt[nt][m][1]);
        }
    load_v(c + kSingleWarps);
  }

  // the warps' results meet: M = max m, weights 2^(m - M)
  __shared__ float s_m[kSingleWarps][8], s_l[kSingleWarps][8];
  __shared__ __align__(16) float s_o[kSingleWarps][8][DP], s_part[NT * 8][DP];
  __shared__ float s_lse[NT * 8];  // to base 2
  const long long all_rows = (long long)a.B * a.Hq * a.Lq;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (nt) __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_row[nt][e];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(~0u, l, w);
      if (g == 0) s_m[warp][2 * t + e] = m_row[nt][e], s_l[warp][2 * t + e] = l;
    }
#pragma unroll
    for (int x = 0; x < VB; ++x)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)  // number x 64 + g 8 + 2 u + e / 2, row 2 t + e % 2
          s_o[warp][2 * t + (e & 1)][x * 64 + g * 8 + 2 * u + (e >> 1)] = o[nt][x][u][e];
    __syncthreads();
    for (int k = threadIdx.x; k < 8 * (DP / 4); k += kSingleWarps * 32) {
      const int r8 = k / (DP / 4), d = k % (DP / 4) * 4, r = nt * 8 + r8;
      if (r >= p.rows || d >= a.D) continue;
      float top = -INFINITY, l = 0.0f, acc[4] = {};
#pragma unroll
      for (int w = 0; w < kSingleWarps; ++w) top = fmaxf(top, s_m[w][r8]);
#pragma unroll
      for (int w = 0; w < kSingleWarps; ++w) {
        const float f = top == -INFINITY ? 0.0f : fast_exp2(s_m[w][r8] - top);
        l = fmaf(f, s_l[w][r8], l);
        const float4 v = *reinterpret_cast<const float4*>(&s_o[w][r8][d]);
        acc[0] = fmaf(f, v.x, acc[0]), acc[1] = fmaf(f, v.y, acc[1]);
        acc[2] = fmaf(f, v.z, acc[2]), acc[3] = fmaf(f, v.w, acc[3]);
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = l == 0.0f ? 0.0f : acc[i] * inv;
      const float lse2 = l == 0.0f ? -INFINITY : top + log2f(l * (1.0f / (1 << (int)kUp<T>))),
                  lse = lse2 * 0.6931471805599453f;
      if (p.cluster) {
        *reinterpret_cast<float4*>(&s_part[r][d]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) s_lse[r] = lse2;
        continue;
      }
      const int i = r / shared_heads, h = head_of(r);
      const long long row = ((long long)b * a.Hq + h) * a.Lq + i;
      if (p.splits > 1) {
        *reinterpret_cast<float4*>(p.part_out + (blockIdx.y * all_rows + row) * a.D + d) =
            make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) p.part_lse[blockIdx.y * all_rows + row] = lse;
      } else {
        *reinterpret_cast<uint2*>(a.out.at<T>(b, i, h) + d) =
            make_uint2(pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3]));
        if (d == 0 && a.lse) a.lse[row] = lse;
      }
    }
  }
  if (!p.cluster) return;
  // out = sum over splits of 2^(lse_s - lse) out_s, from the shared memory of the cluster's CTAs, each
  // of which takes its share of the numbers
  cluster_arrive();
  cluster_wait();
  for (int k = threadIdx.x * p.splits + blockIdx.y; k < p.rows * (DP / 4);
       k += kSingleWarps * 32 * p.splits) {
    const int r = k / (DP / 4), d = k % (DP / 4) * 4;
    if (d >= a.D) continue;
    float top = -INFINITY, total = 0.0f, acc[4] = {}, w[kClusterSplits];
    float4 v[kClusterSplits];
#pragma unroll
    for (int s = 0; s < kClusterSplits; ++s) {
      w[s] = s < p.splits ? cluster_load(&s_lse[r], s) : -INFINITY;
      v[s] = s < p.splits ? cluster_load4(smem_u32(&s_part[r][d]), s) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      top = max_nan(top, w[s]);
    }
#pragma unroll
    for (int s = 0; s < kClusterSplits; ++s) {
      const float f = top == -INFINITY ? 0.0f : fast_exp2(w[s] - top);
      total += f;
      acc[0] = fmaf(f, v[s].x, acc[0]), acc[1] = fmaf(f, v[s].y, acc[1]);
      acc[2] = fmaf(f, v[s].z, acc[2]), acc[3] = fmaf(f, v[s].w, acc[3]);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int i = r / shared_heads, h = head_of(r);
    *reinterpret_cast<uint2*>(a.out.at<T>(b, i, h) + d) =
        make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
    if (d == 0 && a.lse)
      a.lse[((long long)b * a.Hq + h) * a.Lq + i] =
          total == 0.0f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
  }
  cluster_arrive();  // the others may still be reading this CTA's memory
  cluster_wait();
}

// Against the kernel with tiles of 128 rows, in us with the joining of the splits: up to 8 rows 84
// against 105 (2 x 65,280 keys, 8 heads of 128) and 15 against 25 (4 x 3,600, 16 of 64), 9 to 16 rows
// at D up to 64 58 against 81 (2 x 65,280, 8 heads) and 20 against 25 (4 x 3,600, 16 heads); above,
// where two groups of rows leave 2 CTAs an SM, it lost: 126 against 106, 40 against 35.
bool attention_is_single(const gs_attention_args& a) {
  return a.Hkv > 0 && (long long)a.Lq * (a.Hq / a.Hkv) <= (a.D <= 64 ? 16 : 8);
}

// Splits of the keys: one wave of CTAs, each with at least two chunks for every warp. Up to 8 of them
// are a cluster, which joins its parts through shared memory (2 to 3 us less than a second kernel), so
// there are 8 rather than a few more, and where a warp has at most 4 chunks with 8 (2 x 3,600, 16
// heads of 64: 11.5 us with 8, 13.1 with 13; 3 x 8,160: 21.0 with 8, 22.5 with 9; but 2 x 16,320 took
// 3 us more with 8 than with 13).
static int single_splits(const gs_attention_args& a) {
  const long long pairs = (long long)a.B * a.Hkv;
  const long long chunk = a.D <= 64 ? 32 : 16;
  const long long most = a.Lk / (2 * kSingleWarps * chunk);
  const long long wave = kSms * single_ctas((long long)a.Lq * (a.Hq / a.Hkv) <= 8 ? 1 : 2);
  const long long splits = std::max(1ll, std::min(wave / std::max(1ll, pairs), most));
  const bool short_enough = a.Lk <= 4 * kClusterSplits * kSingleWarps * chunk;
  return (int)(splits > kClusterSplits && (splits <= 10 || short_enough) ? kClusterSplits : splits);
}

size_t attention_single_workspace(const gs_attention_args& a) {
  const long long splits = single_splits(a), rows = (long long)a.B * a.Hq * a.Lq;
  return splits > kClusterSplits ? (size_t)(splits * rows) * (a.D + 1) * sizeof(float) : 0;
}

template <typename T, int DP, int NT>
static cudaError_t launch_single(const SingleParams& p, cudaStream_t stream) {
  const dim3 grid((unsigned)p.a.B * p.a.Hkv, p.splits), cluster(1, p.cluster ? p.splits : 1);
  return launch_overlapped_clusters(p.a.mask ? attention_single_kernel<T, DP, NT, true>
                                             : attention_single_kernel<T, DP, NT, false>,
                                    grid, cluster, kSingleWarps * 32, 0, stream, p);
}

template <typename T>
static cudaError_t launch_single(const SingleParams& p, cudaStream_t stream) {
  return p.a.D > 64   ? launch_single<T, 128, 1>(p, stream)
         : p.rows > 8 ? launch_single<T, 64, 2>(p, stream)
                      : launch_single<T, 64, 1>(p, stream);
}

int attention_single(const gs_attention_args& a, void* workspace, cudaStream_t stream) {
  SingleParams p{};
  p.a = attention_params(a);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.rows = a.Lq * (a.Hq / a.Hkv);
  p.splits = single_splits(a);
  p.cluster = p.splits > 1 && p.splits <= kClusterSplits;
  const long long rows = (long long)a.B * a.Hq * a.Lq;
  p.part_out = static_cast<float*>(workspace);
  p.part_lse = p.part_out + p.splits * rows * a.D;
  GS_CUDA(a.dtype == GS_FP16 ? launch_single<__half>(p, stream)
                             : launch_single<__nv_bfloat16>(p, stream));
  count_launches(1u);
  if (p.splits > kClusterSplits) {
    GS_CUDA(attention_combine(a, p.splits, p.part_out, p.part_lse, stream));
    count_launches(1u);
  }
  return GS_OK;
}

}  // namespace gs
