// Root-mean-square norm with the residual's addition, its gradient, and its 8-bit output.
//
//   h = x + r (or x),  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w.
// Statistics and products are in 32 bits; h is rounded once when it is written to the residual
// stream, and y is formed from the unrounded h. With u = h rstd and g = dy w:
//   dh_total = rstd (g - u mean(g u)) + dh,  dx = dr = dh_total,  dw = sum over rows of dy u.
// The backward reads the h that the forward wrote, rounded to T, and the forward's rstd, which is of the
// unrounded one. dx hardly notices; dw is about 1.4 roundings off instead of one (in norm, 2.4e-3 for
// bfloat16 instead of 1.7e-3). Reading x and r in h's place would cost one more input (134 MB, 20 us of 103, at
// 65,280 rows of 1,024 bfloat16).
// 8 bits: for each row, or each group of `group` numbers of it, s = max|y| / 448 and
// q = e4m3(y / s), so that y ~ q s (448 is e4m3's largest number); s = 0 where y is all zero, else
// at least 2^-126, whose reciprocal is finite. y is multiplied by the reciprocal, two roundings in 32
// bits where a division has one: where y / s lies that near to the middle of two e4m3 numbers, the other may
// be taken.
//
// Bound by HBM: each input is read once and each output written once, the row staying in
// registers between the sum of squares and the scaling. ROW threads hold one row, up to CHUNKS
// packs of VEC elements each; the shape that fits the width best takes it (with_row_shape).
// 65,280 rows of 1,024 bfloat16 with residual: 83 us (6.4 TB/s), with 8-bit rows 81 (5.8 TB/s),
// gradient 103 (5.2 TB/s). Where a row does not start on 16 bytes or has an odd end, single elements are
// read: 16,384 rows of 1,001 bfloat16 take 21 us and 46 for the gradient, and above 1,024 numbers a row,
// where a CTA of 1,024 threads has 64 registers a thread and spills, 8,192 of 2,001 225 and 782. So does
// the gradient of more than 8,192 16-bit numbers (4,096 x 16,384: 242 us, 1.7 TB/s).
// dw is summed by a fixed set of CTAs over their own rows into partial rows, which a second
// kernel adds in a fixed order: the same bits on every run.
#include <cuda_fp8.h>

#include <algorithm>

#include "capi_internal.h"
#include "gs_common.cuh"
#include "overlap.cuh"
#include "token_types.cuh"

namespace gs {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: its reciprocal is finite
constexpr int kNormMaxWidth = 32768;
constexpr int kNormMaxBlocks = 148 * 2;  // CTAs (and partial rows of dw) of the backward

struct NormParams {
  const void* x;
  const void* r;
  const void* w;
  void* y;        // T, or e4m3 bytes
  void* h;        // residual stream out, or null
  float* rstd;    // [rows] or null
  float* scales;  // [rows, width / group]
  long long rows;
  int width, group;
  float eps;
};

__device__ __forceinline__ float e4m3_scale(float top) {
  return top > 0.0f ? fmaxf(top / kE4m3Max, kMinScale) : top;  // 0 and NaN stay
}

// Waits for the ROW threads of a row: the whole CTA, or the row's own part of one that holds several.
template <int ROW, int THREADS>
__device__ __forceinline__ void row_sync() {
  if constexpr (ROW == THREADS)
    __syncthreads();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.x / ROW), "n"(ROW) : "memory");
}

template <int ROW, int THREADS>
__device__ __forceinline__ float row_sum(float v, float* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if constexpr (ROW > 32) {
    constexpr int W = ROW / 32;
    float* mine = shared + threadIdx.x / ROW * W;
    row_sync<ROW, THREADS>();  // the previous use of `shared` is over
    if (threadIdx.x % 32 == 0) mine[threadIdx.x % ROW / 32] = v;
    row_sync<ROW, THREADS>();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += mine[i];
  }
  return v;
}

// NaN where the row holds one, so that its scale says so.
template <int ROW, int THREADS>
__device__ __forceinline__ float row_max(float v, float* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(~0u, v, o));
  if constexpr (ROW > 32) {
    constexpr int W = ROW / 32;
    float* mine = shared + threadIdx.x / ROW * W;
    row_sync<ROW, THREADS>();
    if (threadIdx.x % 32 == 0) mine[threadIdx.x % ROW / 32] = v;
    row_sync<ROW, THREADS>();
    v = mine[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = max_nan(v, mine[i]);
  }
  return v;
}

template <int VEC>
__device__ __forceinline__ void store_e4m3(unsigned char* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = (unsigned char)__nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    Pack<unsigned short, VEC / 2> a;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i)
      a.v[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE,
                                        __NV_E4M3);
    *reinterpret_cast<Pack<unsigned short, VEC / 2>*>(p) = a;
  }
}

// CTAs of one row, or of four rows of a warp each. Each row's threads take packs at stride ROW, so a
// warp's accesses are consecutive.
constexpr int forward_threads(int row) { return row == 32 ? 128 : row; }

template <typename T, int VEC, int CHUNKS, int ROW, bool E4M3>
__global__ void __launch_bounds__(forward_threads(ROW)) rms_norm_kernel(NormParams p) {
  constexpr int kThreads = forward_threads(ROW);
  __shared__ float shared[32];
  const int lane = threadIdx.x % ROW;
  const long long row = (long long)blockIdx.x * (kThreads / ROW) + threadIdx.x / ROW;
  if (row >= p.rows) return;  // whole warps, and whole CTAs where ROW > 32
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.width;
  const T* r = p.r ? reinterpret_cast<const T*>(p.r) + row * p.width : nullptr;
  const T* w = reinterpret_cast<const T*>(p.w);
  float h[CHUNKS][VEC];
  float sum = 0.0f;
  wait_for_previous();
  let_next_start();
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = (c * ROW + lane) * VEC;
    if (i < p.width) {
      load_pack<T, VEC>(x + i, h[c]);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) h[c][k] = 0.0f;
    }
  }
  if (r) {
    float a[CHUNKS][VEC];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = (c * ROW + lane) * VEC;
      if (i < p.width) load_pack<T, VEC>(r + i, a[c]);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = (c * ROW + lane) * VEC;
      if (i < p.width) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[c][k] += a[c][k];
        if (p.h) store_pack<T, VEC>(reinterpret_cast<T*>(p.h) + row * p.width + i, h[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum = fmaf(h[c][k], h[c][k], sum);
  sum = row_sum<ROW, kThreads>(sum, shared);
  const float rstd = rsqrtf(sum / (float)p.width + p.eps);
  if (p.rstd && lane == 0) p.rstd[row] = rstd;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = (c * ROW + lane) * VEC;
    if (i < p.width) {
      float wv[VEC];
      load_pack<T, VEC>(w + i, wv);
#pragma unroll
      for (int k = 0; k < VEC; ++k) h[c][k] = h[c][k] * rstd * wv[k];
      if constexpr (!E4M3) store_pack<T, VEC>(reinterpret_cast<T*>(p.y) + row * p.width + i, h[c]);
    }
  }
  if constexpr (E4M3) {
    unsigned char* q = reinterpret_cast<unsigned char*>(p.y) + row * p.width;
    if (p.group == p.width) {
      float top = 0.0f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int k = 0; k < VEC; ++k) top = max_nan(top, fabsf(h[c][k]));
      top = row_max<ROW, kThreads>(top, shared);
      const float s = e4m3_scale(top);
      const float inv = s > 0.0f ? 1.0f / s : 0.0f;
      if (lane == 0) p.scales[row] = s;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int i = (c * ROW + lane) * VEC;
        if (i < p.width) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) h[c][k] *= inv;
          store_e4m3<VEC>(q + i, h[c]);
        }
      }
    } else {
      // groups of 128 are 128 / VEC neighbouring lanes (VEC is 4 or 8 here): half a warp or one
      if constexpr (VEC >= 4) {
        const int groups = p.width / 128;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const int i = (c * ROW + lane) * VEC;
          float top = 0.0f;
#pragma unroll
          for (int k = 0; k < VEC; ++k) top = max_nan(top, fabsf(h[c][k]));
#pragma unroll
          for (int o = 64 / VEC; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, o));
          const float s = e4m3_scale(top);
          const float inv = s > 0.0f ? 1.0f / s : 0.0f;
          if (i < p.width) {
            if (i % 128 == 0) p.scales[row * groups + i / 128] = s;
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[c][k] *= inv;
            store_e4m3<VEC>(q + i, h[c]);
          }
        }
      }
    }
  }
}

struct NormBackwardParams {
  const void* dy;
  const void* dh;  // or null
  const void* h;
  const void* w;
  const float* rstd;
  void* dx;
  float* partial;  // [gridDim.x, width]
  long long rows;
  int width;
};

// CTAs of 512 threads, two an SM, as many rows at a time as fit: enough bytes on their way, and few
// partial rows.
constexpr int backward_threads(int row) { return row < 512 ? 512 : row; }

template <typename T, int VEC, int CHUNKS, int ROW>
__global__ void __launch_bounds__(backward_threads(ROW), ROW <= 512 && CHUNKS * VEC <= 8 ? 2 : 1)
    rms_norm_backward_kernel(NormBackwardParams p) {
  constexpr int kThreads = backward_threads(ROW);
  constexpr int kRows = kThreads / ROW;
  __shared__ float shared[32];
  // the CTA's rows of dw meet here, CHUNKS * VEC * ROW floats for each of kRows - 1 rows
  extern __shared__ float meet[];
  const int lane = threadIdx.x % ROW, slot = threadIdx.x / ROW;
  const T* w = reinterpret_cast<const T*>(p.w);
  wait_for_previous();
  let_next_start();
  float dw[CHUNKS][VEC];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int k = 0; k < VEC; ++k) dw[c][k] = 0.0f;
  for (long long row = (long long)blockIdx.x * kRows + slot; row < p.rows;
       row += (long long)gridDim.x * kRows) {
    const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.width;
    const T* h = reinterpret_cast<const T*>(p.h) + row * p.width;
    const T* dh = p.dh ? reinterpret_cast<const T*>(p.dh) + row * p.width : nullptr;
    T* dx = reinterpret_cast<T*>(p.dx) + row * p.width;
    const float rstd = p.rstd[row];
    Pack<T, VEC> g[CHUNKS], u[CHUNKS], add[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = (c * ROW + lane) * VEC;
      if (i < p.width) {
        g[c] = *reinterpret_cast<const Pack<T, VEC>*>(dy + i);
        u[c] = *reinterpret_cast<const Pack<T, VEC>*>(h + i);
        if (dh) add[c] = *reinterpret_cast<const Pack<T, VEC>*>(dh + i);
      }
    }
    float dot = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = (c * ROW + lane) * VEC;
      if (i < p.width) {
        float wv[VEC];
        load_pack<T, VEC>(w + i, wv);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float a = to_f32<T>(g[c].v[k]), b = to_f32<T>(u[c].v[k]) * rstd;
          dw[c][k] = fmaf(a, b, dw[c][k]);
          dot = fmaf(a * wv[k], b, dot);
        }
      }
    }
    dot = row_sum<ROW, kThreads>(dot, shared) / (float)p.width;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = (c * ROW + lane) * VEC;
      if (i < p.width) {
        float wv[VEC], o[VEC];
        load_pack<T, VEC>(w + i, wv);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float a = to_f32<T>(g[c].v[k]) * wv[k], b = to_f32<T>(u[c].v[k]) * rstd;
          o[k] = rstd * (a - b * dot);
          if (dh) o[k] += to_f32<T>(add[c].v[k]);
        }
        store_pack<T, VEC>(dx + i, o);
      }
    }
  }
  if constexpr (kRows > 1) {
    constexpr int kPer = CHUNKS * VEC * ROW;
    if (slot > 0) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          meet[(slot - 1) * kPer + (c * VEC + k) * ROW + lane] = dw[c][k];
    }
    __syncthreads();
    if (slot) return;
#pragma unroll
    for (int s = 0; s < kRows - 1; ++s)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dw[c][k] += meet[s * kPer + (c * VEC + k) * ROW + lane];
  }
  float* out = p.partial + (long long)blockIdx.x * p.width;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = (c * ROW + lane) * VEC;
    if (i < p.width) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) out[i + k] = dw[c][k];
    }
  }
}

// dw = the sum of the partial rows: a warp's lanes take 32 neighbouring columns, the CTA's 8 warps
// every eighth partial row, and the 8 sums meet in shared memory in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) norm_dw_kernel(const float* partial, int parts, int width,
                                                      void* dw) {
  __shared__ float meet[8][32];
  const int col = blockIdx.x * 32 + threadIdx.x % 32, first = threadIdx.x / 32;
  float s = 0.0f;
  wait_for_previous();
  let_next_start();
  if (col < width)
    for (int i = first; i < parts; i += 8) s += partial[(long long)i * width + col];
  meet[first][threadIdx.x % 32] = s;
  __syncthreads();
  if (first == 0 && col < width) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += meet[i][threadIdx.x];
    reinterpret_cast<T*>(dw)[col] = from_f32<T>(s);
  }
}

// Calls f with the (VEC, CHUNKS, ROW) that holds a row: 16-byte packs where width and pointers
// allow them, else single elements. MOST packs a thread, more only where 1,024 threads do not hold
// the row otherwise: 4 forward; backward, which keeps three inputs and its part of dw, 8 elements,
// for which 64 registers do (65,280 rows of 1,024 bfloat16: 103 us at 8 elements a thread, 143 at
// 16). Narrow rows take a warp each, whose sums need no barrier.
template <typename T, int MOST, typename F>
static void with_row_shape(int width, bool packed, F&& f) {
  constexpr int V = 16 / (int)sizeof(T);
  if (!packed) {
    if (width <= 1024)
      f.template operator()<1, 8, 128>();
    else
      f.template operator()<1, 32, 1024>();
    return;
  }
  const int n = width / V;
  if (n <= 32) return f.template operator()<V, 1, 32>();
  if (n <= 64) return f.template operator()<V, 2, 32>();
  if constexpr (MOST > 2)
    if (n <= 32 * MOST) return f.template operator()<V, MOST, 32>();
  if constexpr (MOST > 1)
    if (n <= 64 * MOST) return f.template operator()<V, MOST, 64>();
  if (n <= 128 * MOST)
    f.template operator()<V, MOST, 128>();
  else if (n <= 256 * MOST)
    f.template operator()<V, MOST, 256>();
  else if (n <= 512 * MOST)
    f.template operator()<V, MOST, 512>();
  else if (n <= 1024 * MOST)
    f.template operator()<V, MOST, 1024>();
  else
    f.template operator()<V, 32 / V, 1024>();
}

template <typename F>
static void with_type(int dtype, F&& f) {
  if (dtype == GS_FP32)
    f.template operator()<float>();
  else if (dtype == GS_FP16)
    f.template operator()<__half>();
  else
    f.template operator()<__nv_bfloat16>();
}

static bool packs(int dtype, int width, std::initializer_list<const void*> pointers) {
  const size_t size = element_size(dtype);
  if (width * size % 16) return false;
  for (const void* q : pointers)
    if (reinterpret_cast<uintptr_t>(q) % 16) return false;
  return true;
}

template <typename T, bool E4M3>
struct NormLaunch {
  const NormParams& p;
  cudaStream_t stream;
  cudaError_t* err;
  template <int VEC, int CHUNKS, int ROW>
  void operator()() const {
    constexpr int threads = forward_threads(ROW);
    const long long blocks = (p.rows + threads / ROW - 1) / (threads / ROW);
    *err = launch_overlapped(rms_norm_kernel<T, VEC, CHUNKS, ROW, E4M3>, dim3((unsigned)blocks),
                             threads, 0, stream, p);
  }
};

template <bool E4M3>
struct NormByType {
  const NormParams& p;
  bool packed;
  cudaStream_t stream;
  cudaError_t* err;
  template <typename T>
  void operator()() const {
    with_row_shape<T, 4>(p.width, packed, NormLaunch<T, E4M3>{p, stream, err});
  }
};

// CTAs of the backward: a bound that holds for every shape, since a CTA takes one row at least.
static int norm_blocks(long long rows) {
  return (int)std::max(1ll, std::min(rows, (long long)kNormMaxBlocks));
}

template <typename T>
struct NormBackwardLaunch {
  const NormBackwardParams& p;
  int blocks;
  cudaStream_t stream;
  cudaError_t* err;
  template <int VEC, int CHUNKS, int ROW>
  void operator()() const {
    constexpr int threads = backward_threads(ROW);
    constexpr size_t meet = (size_t)(threads / ROW - 1) * CHUNKS * VEC * ROW * sizeof(float);
    static_assert(meet <= 48 * 1024, "the rows of dw meet in shared memory");
    *err = launch_overlapped(rms_norm_backward_kernel<T, VEC, CHUNKS, ROW>, dim3((unsigned)blocks),
                             threads, meet, stream, p);
  }
};

struct NormBackwardByType {
  const NormBackwardParams& p;
  bool packed;
  int blocks;
  void* dw;
  cudaStream_t stream;
  cudaError_t* err;
  template <typename T>
  void operator()() const {
    with_row_shape<T, sizeof(T) == 4 ? 2 : 1>(p.width, packed, NormBackwardLaunch<T>{p, blocks, stream, err});
    if (*err != cudaSuccess) return;
    *err = launch_overlapped(norm_dw_kernel<T>, dim3((unsigned)(p.width + 31) / 32), 256, 0, stream,
                             p.partial, blocks, p.width, dw);
  }
};

}  // namespace gs

using namespace gs;

extern "C" int gs_rms_norm_forward(int dtype, long long rows, int width, const void* x,
                                   const void* residual, const void* weight, float eps, void* y,
                                   void* h, float* rstd, void* stream) {
  GS_API_BEGIN();
  GS_REQUIRE(known_type(dtype), "dtype must be GS_FP32, GS_FP16 or GS_BF16");
  GS_REQUIRE(rows >= 0 && rows < (1ll << 31), "rows must be in [0, 2^31)");
  GS_REQUIRE(width >= 1 && width <= kNormMaxWidth, "width must be in [1, 32768]");
  GS_REQUIRE(eps >= 0.0f, "eps must be non-negative");
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && weight && y, "null pointer");
  GS_REQUIRE(!h || residual, "the residual stream is written only where a residual is added");
  const NormParams p{x, residual, weight, y, h, rstd, nullptr, rows, width, width, eps};
  const bool packed = packs(dtype, width, {x, residual, weight, y, h});
  cudaError_t err = cudaSuccess;
  with_type(dtype, NormByType<false>{p, packed, (cudaStream_t)stream, &err});
  GS_CUDA(err);
  gs::count_launches(1u);
  return GS_OK;
  GS_API_END();
}

extern "C" int gs_rms_norm_e4m3(int dtype, long long rows, int width, int group, const void* x,
                                const void* residual, const void* weight, float eps, void* q,
                                float* scales, void* h, void* stream) {
  GS_API_BEGIN();
  GS_REQUIRE(known_type(dtype), "dtype must be GS_FP32, GS_FP16 or GS_BF16");
  GS_REQUIRE(rows >= 0 && rows < (1ll << 31), "rows must be in [0, 2^31)");
  GS_REQUIRE(width >= 1 && width <= kNormMaxWidth, "width must be in [1, 32768]");
  GS_REQUIRE(eps >= 0.0f, "eps must be non-negative");
  GS_REQUIRE(group == 0 || (group == 128 && width % 128 == 0),
             "group must be 0 (one scale a row) or 128, dividing the width");
  if (rows == 0) return GS_OK;
  GS_REQUIRE(x && weight && q && scales, "null pointer");
  GS_REQUIRE(!h || residual, "the residual stream is written only where a residual is added");
  const bool packed = packs(dtype, width, {x, residual, weight, q, h});
  GS_REQUIRE(group == 0 || packed, "with groups, every buffer must start on a 16-byte boundary");
  const NormParams p{x, residual, weight, q, h, nullptr, scales, rows, width,
                     group ? group : width, eps};
  // a group as wide as the row is a row
  cudaError_t err = cudaSuccess;
  with_type(dtype, NormByType<true>{p, packed, (cudaStream_t)stream, &err});
  GS_CUDA(err);
  gs::count_launches(1u);
  return GS_OK;
  GS_API_END();
}

extern "C" size_t gs_rms_norm_backward_workspace_size(long long rows, int width) {
  if (rows <= 0 || width <= 0 || width > kNormMaxWidth) return 0;
  return (size_t)norm_blocks(rows) * width * sizeof(float);
}

extern "C" int gs_rms_norm_backward(int dtype, long long rows, int width, const void* dy,
                                    const void* dh, const void* h, const void* weight,
                                    const float* rstd, void* dx, void* dw, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  GS_API_BEGIN();
  GS_REQUIRE(known_type(dtype), "dtype must be GS_FP32, GS_FP16 or GS_BF16");
  GS_REQUIRE(rows >= 0 && rows < (1ll << 31), "rows must be in [0, 2^31)");
  GS_REQUIRE(width >= 1 && width <= kNormMaxWidth, "width must be in [1, 32768]");
  GS_REQUIRE(dw, "null pointer");
  if (rows == 0) {
    GS_CUDA(cudaMemsetAsync(dw, 0, element_size(dtype) * width, (cudaStream_t)stream));
    return GS_OK;
  }
  GS_REQUIRE(dy && h && weight && rstd && dx && workspace, "null pointer");
  GS_REQUIRE(workspace_bytes >= gs_rms_norm_backward_workspace_size(rows, width),
             "workspace too small");
  GS_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "misaligned workspace");
  const NormBackwardParams p{dy, dh, h, weight, rstd, dx, static_cast<float*>(workspace), rows,
                             width};
  const bool packed = packs(dtype, width, {dy, dh, h, weight, dx});
  cudaError_t err = cudaSuccess;
  with_type(dtype, NormBackwardByType{p, packed, norm_blocks(rows), dw,
                                      (cudaStream_t)stream, &err});
  GS_CUDA(err);
  gs::count_launches(2u);
  return GS_OK;
  GS_API_END();
}
