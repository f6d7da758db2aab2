// What the cross-attention kernels share: the operands' description, lengths and masks.
#pragma once

#include <atomic>

#include "device_errors.h"
#include "overlap.cuh"
#include "pieces.h"
#include "token_types.cuh"

namespace gs {

// A [batch, token, head, D] tensor whose last axis is contiguous; strides in elements.
struct TokenView {
  void* data = nullptr;
  long long b = 0, l = 0, h = 0;

  TokenView() = default;
  explicit TokenView(const gs_token_view& v)
      : data(v.data), b(v.batch_stride), l(v.token_stride), h(v.head_stride) {}
  template <typename T>
  __device__ __forceinline__ T* at(int batch, int token, int head) const {
    return static_cast<T*>(data) + batch * b + token * l + head * h;
  }
};

struct AttentionParams {
  int B, Lq, Lk, Hq, Hkv, D;
  float scale;
  TokenView q, k, v, out, dout, dq, dk, dv;
  const int* lengths;         // [B] or null
  const unsigned char* mask;  // keys contiguous; 0 leaves a key out; or null
  long long mask_b, mask_h, mask_q;
  // the mask as bits, rows of 4 words for each 128 keys; strides in words, 0 where shared; or null
  const unsigned* bits;
  long long bits_b, bits_h, bits_q;
  // rows of such words whose OR says which keys any query and head of a key head keeps: kept_rows of
  // them for each batch item and key head, 4 words for each 128 keys; strides in words
  const unsigned* kept;
  long long kept_b, kept_h;
  int kept_rows, kept_row, kept_tile;
  float* lse;  // [B, Hq, Lq] or null
};

// Keys of batch item b: its length, held to [0, Lk].
__device__ __forceinline__ int key_count(const AttentionParams& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.Lk) : p.Lk;
}

// The bits of keys 32 w .. 32 w + 31 that lie below `left`.
__device__ __forceinline__ unsigned below(int left, int w) {
  const int k = left - 32 * w;
  return k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u;
}

// The keys of tile `tile` (of 128) that any query of key head hk keeps, in two steps so that the loads can
// be in flight meanwhile; for a whole warp, whose lanes then all have it. All loads are in flight at
// once (a loop with a trip count of each lane's own takes its odd trips one after another: 306 -> 641 us
// at 3 x 6,000 x 10,000, 4 heads of 64).
constexpr int kKeptMost = 256;  // rows, at most
__device__ __forceinline__ uint4 kept_begin(const AttentionParams& p, int b, int hk, int tile) {
  const int lane = threadIdx.x % 32;
  const long long step = 32ll * p.kept_row;
  const unsigned* at = p.kept + b * p.kept_b + hk * p.kept_h + (long long)tile * p.kept_tile +
                       (long long)lane * p.kept_row;
  uint4 w[kKeptMost / 32], any = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int k = 0; k < kKeptMost / 32; ++k) {
    w[k] = make_uint4(0u, 0u, 0u, 0u);
    if (32 * k + lane < p.kept_rows) w[k] = *reinterpret_cast<const uint4*>(at);
    at += step;
  }
#pragma unroll
  for (int k = 0; k < kKeptMost / 32; ++k)
    any.x |= w[k].x, any.y |= w[k].y, any.z |= w[k].z, any.w |= w[k].w;
  return any;
}
__device__ __forceinline__ uint4 kept_end(const uint4& any) {
  return make_uint4(__reduce_or_sync(~0u, any.x), __reduce_or_sync(~0u, any.y),
                    __reduce_or_sync(~0u, any.z), __reduce_or_sync(~0u, any.w));
}

constexpr unsigned kMinusInf = 0xff800000u;

// 2^kHalfLog2 is half's largest power of two.
constexpr float kHalfLog2 = 15.0f;

// Sets the scores s of 32 keys to -inf where their bit in `keep` is 0.
__device__ __forceinline__ void hide32(unsigned keep, unsigned* s) {
#pragma unroll
  for (int k = 0; k < 32; ++k)
    if (!(keep >> k & 1u)) s[k] = kMinusInf;
}

// Zeroes, in a swizzled tile of 128 rows (BOXES boxes of 128 bytes a row) at shared address `tile`, the
// rows from `left` on and those whose bit in `keep` is 0: whole rows, so the swizzle inside them does
// not matter. One warp; the matrix engine sees it afterwards.
template <int BOXES>
__device__ __forceinline__ void clear_rows(unsigned tile, int left, const uint4& keep) {
  constexpr int kRows = 128;
  const int lane = threadIdx.x % 32;
  for (int x = 0; x < BOXES; ++x)
#pragma unroll 4
    for (int at = left * 128 + lane * 16; at < kRows * 128; at += 512)
      asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tile + x * kRows * 128 + at),
                   "r"(0)
                   : "memory");
#pragma unroll
  for (int w = 0; w < kRows / 32; ++w) {
    const unsigned kept = w == 0 ? keep.x : w == 1 ? keep.y : w == 2 ? keep.z : keep.w;
    unsigned out = below(left, w) & ~kept;
    while (out) {
      const int k = w * 32 + __ffs(out) - 1;
      out &= out - 1;
#pragma unroll
      for (int x = 0; x < BOXES; ++x)
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(tile + (x * kRows + k) * 128 + lane * 4), "r"(0)
                     : "memory");
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}
// Whether clear_rows would find anything to clear.
__device__ __forceinline__ bool has_hidden_rows(int left, const uint4& keep) {
  return left < 128 || (keep.x & keep.y & keep.z & keep.w) != ~0u;
}

// Lets a kernel have `bytes` of dynamic shared memory on the current device; asked of the runtime
// once for each kernel and device.
template <auto KERNEL>
cudaError_t allow_shared(int bytes) {
  static std::atomic<unsigned long long> done{0};  // a bit for each device
  int dev = 0;
  if (const cudaError_t err = cudaGetDevice(&dev)) return err;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  const cudaError_t err = cudaFuncSetAttribute(
      KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_acq_rel);
  return err;
}

constexpr long long kSms = 148;  // streaming multiprocessors of a B200

// The mask's bits in `workspace` (16-byte aligned, attention_mask_bytes long).
size_t attention_mask_bytes(const gs_attention_args& a);
int attention_pack_mask(const gs_attention_args& a, AttentionParams& p, void* workspace,
                        cudaStream_t stream);
AttentionParams attention_params(const gs_attention_args& a);
size_t attention_forward_workspace(const gs_attention_args& a);
int attention_forward(const gs_attention_args& a, void* workspace, cudaStream_t stream);
cudaError_t attention_combine(const gs_attention_args& args, int splits, const float* out,
                              const float* lse, cudaStream_t stream);
// Few rows for each key head: the kernel that reads k and v straight into registers.
bool attention_is_single(const gs_attention_args& a);
size_t attention_single_workspace(const gs_attention_args& a);
int attention_single(const gs_attention_args& a, void* workspace, cudaStream_t stream);

size_t attention_backward_workspace(const gs_attention_args& a);
int attention_backward(const gs_attention_args& a, const gs_token_view& dout,
                       const gs_token_view& dq, const gs_token_view& dk, const gs_token_view& dv,
                       void* workspace, cudaStream_t stream);

}  // namespace gs
