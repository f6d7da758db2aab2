// Fifth-generation tensor-core matrix products (tcgen05) with accumulators in tensor memory, and
// the copies and barriers that feed them.
//
// Conventions of the callers: operand tiles lie in shared memory as the 128-byte-swizzled boxes
// that the copy engine writes, rows of 64 16-bit numbers (128 bytes), 8 rows to a 1,024-byte
// group, tiles starting on 1,024-byte boundaries. A tile read along its rows (contraction over
// the 64 numbers) is "K-major"; the same tile read across (contraction over the rows) is
// "MN-major". Wider rows are several such boxes one after another. Accumulator row r is lane r
// of tensor memory, column j of the product its column j.
#pragma once

#include "tma.cuh"
#include "token_types.cuh"

namespace gs {

// Limit of a wait inside the attention kernels; a wait that runs out ends the kernel with
// kErrMmaTimeout.
constexpr unsigned long long kTcWaitNs = 2000000000ull;

// Waits for phase `parity` of the barrier; false if the limit ran out. The clock is read once in
// 64 polls, each of which may suspend the thread for a time that the hardware sets.
__device__ __forceinline__ bool tc_wait(uint64_t* bar, unsigned parity) {
  const unsigned addr = smem_u32(bar);
  unsigned long long t0 = 0;
  for (unsigned k = 0; k < (1u << 28); ++k) {
    unsigned done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if (k % 64 == 63) {
      const unsigned long long t = tma_global_ns();
      if (t0 == 0) t0 = t;
      if (t - t0 > kTcWaitNs) return false;
    }
  }
  return false;
}

// The same for a whole warp: false for every lane where it is for one.
__device__ __forceinline__ bool tc_wait_warp(uint64_t* bar, unsigned parity) {
  return __all_sync(~0u, tc_wait(bar, parity));
}

// A barrier's first state, to be seen by the other threads and engines after mbar_ready and a
// __syncthreads.
__device__ __forceinline__ void mbar_set(uint64_t* bar, unsigned arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(arrivals)
               : "memory");
}
__device__ __forceinline__ void mbar_ready() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
// Named barrier 1 over THREADS threads: a warp that only arrives goes on at once, what it wrote
// before is seen by those that wait.
template <int THREADS>
__device__ __forceinline__ void ready_arrive() {
  asm volatile("bar.arrive 1, %0;" ::"n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void ready_wait() {
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// True in one lane of the (converged) warp. The products and commits below are issued under it
// rather than under `lane == 0`: the compiler then knows that one thread runs them (105 clocks to
// issue a product under `lane == 0`, under 64 so).
__device__ __forceinline__ bool elect_one() {
  unsigned is;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(is));
  return is != 0;
}

// A value that all lanes of the (converged) warp share, so that the compiler knows it: branches on
// it are not divergent and descriptors made of it live in uniform registers.
__device__ __forceinline__ int warp_uniform(int v) { return __shfl_sync(~0u, v, 0); }

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// One arrival for the warp, after what its lanes have done (32 arrivals of a warp on one barrier
// would queue up).
__device__ __forceinline__ void mbar_arrive_warp(uint64_t* bar) {
  __syncwarp();
  if (elect_one()) mbar_arrive(bar);
}

// Box at (x, y, z, w), innermost first, into swizzled shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load_4d(unsigned dst, const CUtensorMap* map, int x, int y,
                                            int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tc_alloc(unsigned* slot, unsigned columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_u32(slot)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tc_free(unsigned base, unsigned columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Arrives on `bar` when every matrix product issued by this thread so far has completed.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

// D[tmem] (+)= A[shared] B[shared]^T, one step of 16 along the contraction.
__device__ __forceinline__ void tc_mma_ss(unsigned d, uint64_t a, uint64_t b, unsigned idesc,
                                          unsigned accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A in tensor memory: 8 columns of two 16-bit numbers each.
__device__ __forceinline__ void tc_mma_ts(unsigned d, unsigned a, uint64_t b, unsigned idesc,
                                          unsigned accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor: 32-bit accumulators, A and B both half (0) or both bfloat16 (1), M = 128
// rows, N columns (a multiple of 16), B K-major or MN-major, A K-major.
template <typename T>
struct TcFormat;
template <>
struct TcFormat<__half> {
  static constexpr unsigned kId = 0;
};
template <>
struct TcFormat<__nv_bfloat16> {
  static constexpr unsigned kId = 1;
};
template <typename T>
__device__ __forceinline__ unsigned tc_idesc(unsigned n, bool b_mn_major) {
  return (1u << 4) | (TcFormat<T>::kId << 7) | (TcFormat<T>::kId << 10) |
         ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// Shared-memory operand descriptor of a 128-byte-swizzled tile. `group_bytes`: distance of
// neighbouring 64-number boxes (MN-major operands wider than 64 only).
__device__ __forceinline__ uint64_t tc_desc(unsigned addr, unsigned group_bytes) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(group_bytes >> 4) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

#define GS_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), \
                    "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define GS_I8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), \
                    "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])

// 32 consecutive columns of the thread's lane (asynchronous: tc_wait_ld before use).
__device__ __forceinline__ void tc_ld32(unsigned addr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19,"
      " %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : GS_R8(r, 0), GS_R8(r, 8), GS_R8(r, 16), GS_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tc_ld16(unsigned addr, unsigned* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : GS_R8(r, 0), GS_R8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void tc_st16(unsigned addr, const unsigned* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::GS_I8(r, 0),
      GS_I8(r, 8), "r"(addr)
      : "memory");
}

// Two floats rounded to two 16-bit numbers, `lo` in the low half.
template <typename T>
__device__ __forceinline__ unsigned pack2(float lo, float hi);
template <>
__device__ __forceinline__ unsigned pack2<__half>(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Writes COLS columns from `addr` on of the warp's 32 accumulator rows, times `factor`, as far as
// `left` columns go (a multiple of 8): rounded to T, or in 32 bits (`wide`), to rows `pitch` bytes
// apart from `to` on or, with a pitch of 0, each lane's row to its own `to`; the first `rows` rows
// exist. Where there is nothing to read (`have` false, for the whole
// warp) or the lane's row counts for nothing (`live` false) zeros are written. The rows pass through COLS * 64 bytes of shared memory at `stage`, of this warp alone, so that neighbouring
// lanes write neighbouring 16 bytes: a lane writing its own row would touch 32 lines at a time. The
// loop that writes is kept short: it runs once a CTA, from a cold instruction cache.
template <typename T, int COLS>
__device__ __forceinline__ void store_rows(unsigned addr, bool have, bool live, float factor,
                                           int left, bool wide, unsigned stage, char* to,
                                           long long pitch, int rows) {
  constexpr int kPieces = COLS / 8, kSwizzle = (kPieces < 8 ? kPieces : 8) - 1;
  const int lane = threadIdx.x % 32;
  float f[COLS];
  if (have) {
    unsigned o[COLS];
#pragma unroll
    for (int c = 0; c < COLS; c += 32) tc_ld32(addr + c, o + c);
    tc_wait_ld();
#pragma unroll
    for (int c = 0; c < COLS; ++c) f[c] = live ? __uint_as_float(o[c]) * factor : 0.0f;
  } else {
#pragma unroll
    for (int c = 0; c < COLS; ++c) f[c] = 0.0f;
  }
  const unsigned mine = stage + lane * kPieces * 16;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half && !wide) break;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      uint4 w;
      if (wide) {
        const float* x = f + half * (COLS / 2) + c * 4;
        w = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                       __float_as_uint(x[3]));
      } else {
        const float* x = f + c * 8;
        w = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                       pack2<T>(x[6], x[7]));
      }
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                       mine + ((c ^ (lane & kSwizzle)) << 4)),
                   "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                   : "memory");
    }
    __syncwarp();
    const int c = lane % kPieces, column = wide ? half * (COLS / 2) + c * 4 : c * 8;
#pragma unroll 2
    for (int r = lane / kPieces; r < 32; r += 32 / kPieces) {
      uint4 w;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                   : "r"(stage + r * kPieces * 16 + ((c ^ (r & kSwizzle)) << 4))
                   : "memory");
      char* row = to + r * pitch;
      if (!pitch)
        row = reinterpret_cast<char*>(__shfl_sync(~0u, reinterpret_cast<uintptr_t>(to), r));
      if (r < rows && column < left) *reinterpret_cast<uint4*>(row + column * (wide ? 4 : 2)) = w;
    }
    __syncwarp();
  }
}

// The barrier of a cluster's threads, and shared memory of its CTA `rank` where this CTA's p is.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ unsigned cluster_address(unsigned p, int rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(rank));
  return r;
}
__device__ __forceinline__ float cluster_load(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_address(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_load4(unsigned p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_address(p, rank))
               : "memory");
  return v;
}

// 2^x by the special-function unit: relative error below 2^-22, 0 for -inf, results below 2^-126
// are flushed to 0.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in a 64-bit register: one instruction adds or multiplies both.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float lo, float hi) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(Two v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Host: describes a [B, L, H, D] tensor of 16-bit numbers as (D, L, H, B), innermost first, copied
// in boxes of 64 numbers x `rows` tokens x `heads` heads, 128-byte-swizzled; what lies past D or L
// reads as zero. Axes of one element, and a batch stride of 0 (all items alike), are encoded as
// one element: the caller passes coordinate 0 there.
inline bool encode_tokens(CUtensorMap* map, int dtype, const void* base, int D, int L, int H,
                          int B, long long stride_l, long long stride_h, long long stride_b,
                          unsigned rows, unsigned heads = 1) {
  const EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const auto one = [](long long n, long long stride) { return n <= 1 || stride == 0; };
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)(one(L, stride_l) ? 1 : L),
                              (cuuint64_t)(one(H, stride_h) ? 1 : H),
                              (cuuint64_t)(one(B, stride_b) ? 1 : B)};
  const cuuint64_t row = (cuuint64_t)(D * 2 + 15) / 16 * 16;
  const cuuint64_t strides[3] = {one(L, stride_l) ? row : (cuuint64_t)stride_l * 2,
                                 one(H, stride_h) ? row : (cuuint64_t)stride_h * 2,
                                 one(B, stride_b) ? row : (cuuint64_t)stride_b * 2};
  const cuuint32_t box[4] = {64, rows, heads, 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  return fn(map,
            dtype == GS_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            4, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace gs
