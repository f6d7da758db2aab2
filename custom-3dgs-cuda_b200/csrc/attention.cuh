// What the cross-attention kernels share: the operands' description, lengths and masks.
#pragma once

#include "gs_common.cuh"
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
  float* lse;  // [B, Hq, Lq] or null
};

// Keys of batch item b: its length, held to [0, Lk].
__device__ __forceinline__ int key_count(const AttentionParams& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.Lk) : p.Lk;
}

// Sets s = -inf at the keys that a query leaves out: past `n`, or 0 in its row of the mask (or
// null). `j0`: the first of the N keys in s.
template <int N>
__device__ __forceinline__ void hide(int packs, const unsigned char* row, int j0, int n,
                                     unsigned* s) {
  constexpr unsigned kMinusInf = 0xff800000u;
  if (j0 + N <= n && packs && row) {
#pragma unroll
    for (int c = 0; c < N; c += 16) {
      const uint4 m = *reinterpret_cast<const uint4*>(row + j0 + c);
      const unsigned w[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (!((w[k / 4] >> (8 * (k % 4))) & 0xffu)) s[c + k] = kMinusInf;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (j0 + k >= n || (row && !row[j0 + k])) s[k] = kMinusInf;
}

// Zeroes, in a swizzled tile of `rows` keys (BOXES boxes of 128 bytes a row) at shared address
// `tile`, the rows from `left` on and those whose byte in `mask` is 0 (or null): whole rows, so
// the swizzle inside them does not matter. One warp; the matrix engine sees it afterwards.
template <int BOXES>
__device__ __forceinline__ void clear_rows(unsigned tile, int rows, int left,
                                           const unsigned char* mask) {
  const int lane = threadIdx.x % 32;
  for (int r0 = 0; r0 < rows; r0 += 32) {
    const int r = r0 + lane;
    unsigned out = __ballot_sync(~0u, r >= left || (mask && !mask[r]));
    while (out) {
      const int k = r0 + __ffs(out) - 1;
      out &= out - 1;
#pragma unroll
      for (int x = 0; x < BOXES; ++x)
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(tile + (x * rows + k) * 128 + lane * 4),
                     "r"(0)
                     : "memory");
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

constexpr long long kSms = 148;  // streaming multiprocessors of a B200

int attention_mask_packs(const gs_attention_args& a);
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
