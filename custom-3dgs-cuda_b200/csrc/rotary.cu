// Rotary positions with several axes.
//
// Axis a owns d_a consecutive numbers of every head (d_a even); pair j < d_a / 2 of that block is
// turned by the angle p_a * base_a^(-2 j / d_a):
//   (u, v) -> (u cos - v sin, u sin + v cos),
// with (u, v) at (j, j + d_a / 2) of the block, or at (2 j, 2 j + 1) when interleaved. Numbers
// past the last block are copied. The gradient is the rotation by the negative angle (inverse).
//
// The angle is formed in turns, not radians: p * (f / 2 pi) with the frequency split into two
// floats (made in double on the host) and the product's rounding error recovered by one fused
// multiply-add, so the whole turns drop out exactly and a coordinate of a few thousand costs no
// accuracy. Coordinates are float32, or int32 converted to float32 (exact up to 2^24).
//
// Bound by HBM: every element is read once and written once. The angles depend on the token and
// the pair but not on the head, so a thread keeps VEC pairs' sines and cosines and walks over
// heads, the loads of FLIGHT heads in flight at once. 65,280 tokens of 16 heads of 64 bfloat16 take
// 54 us (5.0 TB/s) with neighbouring pairs and 59 with pairs half a block apart, 55 in the kernel
// below that reads and writes those in whole lines. (Staging whole rows in shared memory took 115.)
#include <algorithm>
#include <cmath>

#include "capi_internal.h"
#include "gs_common.cuh"
#include "overlap.cuh"
#include "token_types.cuh"

namespace gs {

constexpr int kRotaryMaxAxes = 4;
constexpr int kRotaryMaxPairs = 128;
constexpr int kRotaryThreads = 256;  // at most, a CTA
constexpr long long kWave = 148 * 1024;

struct RotaryParams {
  const void* x;
  void* y;
  long long xb, xl, xh, yb, yl, yh;  // strides in elements
  const void* pos;
  long long pos_b, pos_l;
  unsigned tokens;  // B * L
  int L, H;
  int n_axes;
  int pairs, turned;      // pairs a head, and how many of them are turned
  int items;              // pairs / VEC
  int head_lanes;         // threads that share a token's item, each walking over its own heads
  int threads, tokens_per_block;
  int flight;             // heads whose loads a thread issues at once
  int interleaved;
  float sign;
  int axis_start[kRotaryMaxAxes + 1];  // first pair of each axis; [n_axes] = turned
  float freq_hi[kRotaryMaxPairs], freq_lo[kRotaryMaxPairs];  // turns per unit of position
};

template <typename T>
__device__ __forceinline__ float2 unpack2(unsigned v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(unsigned v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ unsigned pack_pair(float lo, float hi) {
  return (unsigned)__builtin_bit_cast(unsigned short, from_f32<T>(lo)) |
         (unsigned)__builtin_bit_cast(unsigned short, from_f32<T>(hi)) << 16;
}

template <typename T, int VEC, bool INTERLEAVED, typename P, int FLIGHT>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__
                                                                RotaryParams p) {
  __shared__ float s_hi[kRotaryMaxPairs], s_lo[kRotaryMaxPairs];
  for (int i = threadIdx.x; i < p.turned; i += blockDim.x) {
    s_hi[i] = p.freq_hi[i];
    s_lo[i] = p.freq_lo[i];
  }
  __syncthreads();
  const int per_token = p.items * p.head_lanes;
  const int slot = threadIdx.x / per_token;
  if (slot >= p.tokens_per_block) return;
  const int in_token = threadIdx.x - slot * per_token;
  const int lane_h = in_token / p.items;
  const int pair = (in_token - lane_h * p.items) * VEC;
  const unsigned token = blockIdx.x * (unsigned)p.tokens_per_block + slot;
  if (token >= p.tokens) return;
  const unsigned b = token / (unsigned)p.L, l = token - b * p.L;

  const bool turned = pair < p.turned;
  int axis = 0;
#pragma unroll
  for (int a = 1; a < kRotaryMaxAxes; ++a)
    if (a < p.n_axes && pair >= p.axis_start[a]) axis = a;
  const int first = turned ? p.axis_start[axis] : p.turned;
  const int end = turned ? p.axis_start[axis + 1] : p.pairs;
  // the block starts at 2 * first and its pair k is (k, k + half), or (2 k, 2 k + 1), whose second
  // VEC numbers follow the first
  const int off_u = INTERLEAVED ? 2 * pair : first + pair;
  const int off_v = INTERLEAVED ? off_u + VEC : off_u + (end - first);
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.xb + l * p.xl;
  T* y = reinterpret_cast<T*>(p.y) + b * p.yb + l * p.yl;
  Pack<T, VEC> u[FLIGHT], v[FLIGHT];
  const auto load = [&](int h0) {
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) {
      const int h = h0 + k * p.head_lanes;
      if (h < p.H) {
        u[k] = *reinterpret_cast<const Pack<T, VEC>*>(x + h * p.xh + off_u);
        v[k] = *reinterpret_cast<const Pack<T, VEC>*>(x + h * p.xh + off_v);
      }
    }
  };
  wait_for_previous();
  let_next_start();
  load(lane_h);  // in flight while the angles are formed

  float c[VEC], s[VEC];
  if (turned) {
    const P raw = reinterpret_cast<const P*>(p.pos)[b * p.pos_b + l * p.pos_l + axis];
    const float at = p.sign * (float)raw;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float hi = s_hi[pair + i];
      const float r = at * hi;
      const float err = fmaf(at, hi, -r) + at * s_lo[pair + i];
      sincospif(2.0f * ((r - rintf(r)) + err), &s[i], &c[i]);
    }
  }
  for (int h0 = lane_h; h0 < p.H; h0 += FLIGHT * p.head_lanes) {
    if (h0 != lane_h) load(h0);
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) {
      const int h = h0 + k * p.head_lanes;
      if (h >= p.H) break;
      if (turned) {
        float z[2 * VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[i] = to_f32<T>(u[k].v[i]), z[VEC + i] = to_f32<T>(v[k].v[i]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int iu = INTERLEAVED ? 2 * i : i, iv = INTERLEAVED ? 2 * i + 1 : VEC + i;
          const float a = z[iu], d = z[iv];
          z[iu] = a * c[i] - d * s[i];
          z[iv] = a * s[i] + d * c[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          u[k].v[i] = from_f32<T>(z[i]), v[k].v[i] = from_f32<T>(z[VEC + i]);
      }
      *reinterpret_cast<Pack<T, VEC>*>(y + h * p.yh + off_u) = u[k];
      *reinterpret_cast<Pack<T, VEC>*>(y + h * p.yh + off_v) = v[k];
    }
  }
}

// Pairs half a block apart, 16-bit numbers, blocks of multiples of 8 numbers: a lane holds 8 numbers of
// a head that follow one another, in groups of 4, and gets their partners from the lanes that hold
// them, so that whole lines are read and written, with half as many accesses; the next heads' loads
// are in flight beside this ones' arithmetic. A lane forms the angles of 4 pairs. Against the kernel
// above at 16 heads a thread, in us: 65,280 tokens of 16 heads of 64 55 and 59, 32,640 of them 33 and 35,
// 65,280 of 8 heads of 128 58 and 59; at fewer heads a thread it loses (16,320 tokens: 19 and 17).
template <typename T, typename P>
__global__ void __launch_bounds__(kRotaryThreads) rotary_rows_kernel(const __grid_constant__
                                                                     RotaryParams p) {
  constexpr int kFlight = 4;
  __shared__ float s_hi[kRotaryMaxPairs], s_lo[kRotaryMaxPairs];
  for (int i = threadIdx.x; i < p.turned; i += blockDim.x) {
    s_hi[i] = p.freq_hi[i];
    s_lo[i] = p.freq_lo[i];
  }
  __syncthreads();
  const int lanes = p.pairs / 4, in_warp = 32 / lanes;  // of a head, and heads a warp holds
  const int lane = threadIdx.x % 32, slot = lane / lanes, i = lane - slot * lanes, lane0 = slot * lanes;
  const unsigned at = (blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) * in_warp + slot;
  const unsigned token = at / (unsigned)p.head_lanes;
  const int lane_h = at - token * p.head_lanes;
  const int H = slot < in_warp && token < p.tokens ? p.H : 0;  // no heads for the lanes left over
  const unsigned b = token / (unsigned)p.L, l = token - b * p.L;
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.xb + l * p.xl + 8 * i;
  T* y = reinterpret_cast<T*>(p.y) + b * p.yb + l * p.yl + 8 * i;
  uint4 w[kFlight], ahead[kFlight];
  const auto load = [&](uint4 (&w)[kFlight], int h0) {
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const int h = h0 + k * p.head_lanes;
      w[k] = make_uint4(0u, 0u, 0u, 0u);
      if (h < H) w[k] = *reinterpret_cast<const uint4*>(x + h * p.xh);
    }
  };
  wait_for_previous();
  let_next_start();
  load(w, lane_h);  // in flight while the angles are formed

  const auto axis_of = [&](int pair) {
    int axis = 0;
#pragma unroll
    for (int a = 1; a < kRotaryMaxAxes; ++a)
      if (a < p.n_axes && pair >= p.axis_start[a]) axis = a;
    return axis;
  };
  float c[4] = {}, s[4] = {};
  if (4 * i < p.turned && H) {
    const P raw = reinterpret_cast<const P*>(p.pos)[b * p.pos_b + l * p.pos_l + axis_of(4 * i)];
    const float pos = p.sign * (float)raw;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float hi = s_hi[4 * i + k];
      const float t = pos * hi;
      const float err = fmaf(pos, hi, -t) + pos * s_lo[4 * i + k];
      sincospif(2.0f * ((t - rintf(t)) + err), &s[k], &c[k]);
    }
  }
  // this lane's numbers are 4 q, 4 q + 4 of its axis's block, whose pairs are `half` groups apart
  const bool turned = 4 * i < p.turned;
  const int axis = axis_of(4 * i), first = turned ? p.axis_start[axis] / 4 : i;
  const int half = turned ? p.axis_start[axis + 1] / 4 - first : 1, q = 2 * (i - first);
  int from[2];
  float cs[2][4], sn[2][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool second = q + e >= half;
    const int pair = second ? q + e - half : q + e;
    from[e] = lane0 + first + (second ? pair : pair + half) / 2;
    if (!turned) from[e] = lane;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      cs[e][k] = __shfl_sync(~0u, c[k], lane0 + first + pair);
      sn[e][k] = __shfl_sync(~0u, s[k], lane0 + first + pair);
      if (!second) sn[e][k] = -sn[e][k];
    }
  }
  const bool swap = half & 1;
  for (int h0 = lane_h; __any_sync(~0u, h0 < H); h0 += kFlight * p.head_lanes) {
    load(ahead, h0 + kFlight * p.head_lanes);
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const int h = h0 + k * p.head_lanes;
      const unsigned own[2][2] = {{w[k].x, w[k].y}, {w[k].z, w[k].w}};
      unsigned out[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const unsigned partner = __shfl_sync(~0u, swap ? own[1 - e][d] : own[e][d], from[e]);
          const float2 a = unpack2<T>(own[e][d]), z = unpack2<T>(partner);
          const float lo = fmaf(a.x, cs[e][2 * d], z.x * sn[e][2 * d]);
          const float hi = fmaf(a.y, cs[e][2 * d + 1], z.y * sn[e][2 * d + 1]);
          out[e][d] = turned ? pack_pair<T>(lo, hi) : own[e][d];
        }
      if (h < H)
        *reinterpret_cast<uint4*>(y + h * p.yh) = make_uint4(out[0][0], out[0][1], out[1][0], out[1][1]);
    }
#pragma unroll
    for (int k = 0; k < kFlight; ++k) w[k] = ahead[k];
  }
}

template <typename T>
static cudaError_t launch_rotary_rows(const RotaryParams& p, int position_type,
                                      cudaStream_t stream) {
  const long long heads_a_cta = 4 * (32 / (p.pairs / 4));
  const dim3 blocks((unsigned)(((long long)p.tokens * p.head_lanes + heads_a_cta - 1) / heads_a_cta));
  return position_type == GS_FP32
             ? launch_overlapped(rotary_rows_kernel<T, float>, blocks, 128, 0, stream, p)
             : launch_overlapped(rotary_rows_kernel<T, int>, blocks, 128, 0, stream, p);
}

template <typename T, int VEC, bool INTERLEAVED, typename P>
static cudaError_t launch_rotary(const RotaryParams& p, unsigned blocks, cudaStream_t stream) {
  if (p.flight == 4)
    return launch_overlapped(rotary_kernel<T, VEC, INTERLEAVED, P, 4>, dim3(blocks), p.threads, 0,
                             stream, p);
  return launch_overlapped(rotary_kernel<T, VEC, INTERLEAVED, P, 1>, dim3(blocks), p.threads, 0, stream, p);
}

template <typename T, int VEC, bool INTERLEAVED>
static cudaError_t launch_rotary(const RotaryParams& p, int position_type, unsigned blocks,
                          cudaStream_t stream) {
  if (position_type == GS_FP32)
    return launch_rotary<T, VEC, INTERLEAVED, float>(p, blocks, stream);
  else
    return launch_rotary<T, VEC, INTERLEAVED, int>(p, blocks, stream);
}

template <typename T, int VEC>
static cudaError_t launch_rotary(const RotaryParams& p, int position_type, unsigned blocks,
                          cudaStream_t stream) {
  if (p.interleaved)
    return launch_rotary<T, VEC, true>(p, position_type, blocks, stream);
  else
    return launch_rotary<T, VEC, false>(p, position_type, blocks, stream);
}

template <typename T>
static cudaError_t launch_rotary(const RotaryParams& p, int vec, int position_type, unsigned blocks,
                          cudaStream_t stream) {
  if (vec == 4)
    return launch_rotary<T, 4>(p, position_type, blocks, stream);
  else if (vec == 2)
    return launch_rotary<T, 2>(p, position_type, blocks, stream);
  else
    return launch_rotary<T, 1>(p, position_type, blocks, stream);
}

}  // namespace gs

using namespace gs;

extern "C" int gs_rotary_axes(int dtype, int B, int L, int H, int D, const gs_token_view* x,
                              const gs_token_view* y, const void* positions, int position_type,
                              long long position_batch_stride, long long position_token_stride,
                              int n_axes, const int* axis_dims, const double* bases,
                              int interleaved, int inverse, void* stream) {
  GS_API_BEGIN();
  GS_REQUIRE(known_type(dtype), "dtype must be GS_FP32, GS_FP16 or GS_BF16");
  GS_REQUIRE(position_type == GS_FP32 || position_type == GS_INT32,
             "positions must be GS_FP32 or GS_INT32");
  GS_REQUIRE(B >= 0 && L >= 0 && H >= 0, "sizes must be non-negative");
  GS_REQUIRE(D >= 2 && D <= 2 * kRotaryMaxPairs && D % 2 == 0,
             "the head size must be even, between 2 and 256");
  GS_REQUIRE(n_axes >= 1 && n_axes <= kRotaryMaxAxes, "between 1 and 4 axes");
  GS_REQUIRE(x && y && axis_dims && bases, "null pointer");
  int sum = 0;
  RotaryParams p{};
  for (int a = 0; a < n_axes; ++a) {
    GS_REQUIRE(axis_dims[a] >= 2 && axis_dims[a] % 2 == 0 && axis_dims[a] <= D,
               "each axis must own an even number of at least 2 of the head's numbers");
    GS_REQUIRE(bases[a] > 0.0 && std::isfinite(bases[a]), "bases must be positive");
    p.axis_start[a] = sum / 2;
    for (int j = 0; j < axis_dims[a] / 2 && sum + 2 * j < D; ++j) {
      const double turns = std::pow(bases[a], -2.0 * j / axis_dims[a]) / (2.0 * M_PI);
      p.freq_hi[sum / 2 + j] = (float)turns;
      p.freq_lo[sum / 2 + j] = (float)(turns - (double)p.freq_hi[sum / 2 + j]);
    }
    sum += axis_dims[a];
    GS_REQUIRE(sum <= D, "the axes own more numbers than a head has");
  }
  p.axis_start[n_axes] = sum / 2;
  if (B == 0 || L == 0 || H == 0) return GS_OK;
  GS_REQUIRE(x->data && y->data && positions, "null pointer");
  p.x = x->data;
  p.y = y->data;
  p.xb = x->batch_stride, p.xl = x->token_stride, p.xh = x->head_stride;
  p.yb = y->batch_stride, p.yl = y->token_stride, p.yh = y->head_stride;
  p.pos = positions;
  p.pos_b = position_batch_stride, p.pos_l = position_token_stride;
  GS_REQUIRE((long long)B * L < (1ll << 31), "too many tokens");
  p.tokens = (unsigned)B * (unsigned)L;
  p.L = L, p.H = H, p.n_axes = n_axes;
  p.pairs = D / 2, p.turned = sum / 2;
  p.interleaved = interleaved != 0;
  p.sign = inverse ? -1.0f : 1.0f;
  // pairs a thread: the largest of 4, 2, 1 that divides every block of pairs, with every access
  // (VEC elements, so 16 bytes at most) aligned
  const size_t size = element_size(dtype);
  int vec = 4;
  const auto fits = [&](int n) {
    for (int a = 0; a < n_axes; ++a)
      if (axis_dims[a] / 2 % n) return false;
    if ((p.pairs - p.turned) % n) return false;
    for (const long long s : {p.xb, p.xl, p.xh, p.yb, p.yl, p.yh})
      if (s % n) return false;
    return (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y)) % (n * size) == 0;
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  p.items = p.pairs / vec;
  // Heads a thread walks over: few sines and divisions for each number once there is work for
  // kWave threads at 16 or 4 heads each (65,280 tokens, 16 heads of 64 bfloat16: 76 us at 4 heads,
  // 54 at 16; 1,000 tokens: 3.1 us at one head, 4.6 at 16).
  const long long pieces = (long long)p.tokens * p.items * H;
  const int heads = pieces >= 16 * kWave ? 16 : pieces >= 2 * kWave ? 4 : 1;
  const int cta = heads == 1 ? 256 : 128;  // one head a thread: fewer CTAs that repeat the sines
  p.threads = cta;
  p.flight = std::min(heads, 4);
  p.head_lanes = (H + heads - 1) / heads;
  const cudaStream_t st = (cudaStream_t)stream;
  // whole lines where there is work for 16 heads a thread (rotary_rows_kernel)
  bool rows = heads == 16 && size == 2 && !interleaved && D % 8 == 0;
  for (int a = 0; a < n_axes; ++a) rows = rows && axis_dims[a] % 8 == 0;
  for (const long long stride : {p.xb, p.xl, p.xh, p.yb, p.yl, p.yh}) rows = rows && stride % 8 == 0;
  rows = rows && (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y)) % 16 == 0;
  if (rows) {
    GS_CUDA(dtype == GS_FP16 ? launch_rotary_rows<__half>(p, position_type, st)
                             : launch_rotary_rows<__nv_bfloat16>(p, position_type, st));
    gs::count_launches(1u);
    return GS_OK;
  }
  while (p.head_lanes > 1 && p.items * p.head_lanes > cta)
    p.head_lanes = (p.head_lanes + 1) / 2;
  p.tokens_per_block = std::max(1, cta / (p.items * p.head_lanes));
  const unsigned blocks = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  GS_CUDA(dtype == GS_FP32   ? launch_rotary<float>(p, vec, position_type, blocks, st)
          : dtype == GS_FP16 ? launch_rotary<__half>(p, vec, position_type, blocks, st)
                             : launch_rotary<__nv_bfloat16>(p, vec, position_type, blocks, st));
  gs::count_launches(1u);
  return GS_OK;
  GS_API_END();
}
