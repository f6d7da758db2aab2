// The mask of the attention kernels, packed from a byte to a bit for each key.
//
// A thread of those kernels holds one query's scores of 128 keys: as bytes its part of the mask
// would be 128 loads that no two lanes share, in an order that no alignment helps (a mask of 777
// keys has rows of 777 bytes); as bits it is one load of 16 bytes. Heads that share a mask share
// its bits. A warp takes 256 keys of a row, its loads all in flight. Reading the bytes in the
// attention kernel instead made its 3 x 1,111 x 777 of 12 heads take 365 us; with the bits it took 67.
#include "attention.cuh"
#include "capi_internal.h"

namespace gs {

struct MaskShape {
  long long b, h, q;  // 1 where batch items, heads or queries share
  int words;          // 32-bit words a row: 4 for each 128 keys
};

static MaskShape mask_shape(const gs_attention_args& a) {
  return {a.mask_batch_stride ? a.B : 1, a.mask_head_stride ? a.Hq : 1,
          a.mask_query_stride ? a.Lq : 1, (a.Lk + 127) / 128 * 4};
}

constexpr int kMaskWords = 8;  // a warp's

// ALIGNED: rows start on 4-byte boundaries, and a lane reads 4 keys at once.
template <bool ALIGNED>
__global__ void __launch_bounds__(256) mask_bits_kernel(const unsigned char* mask, long long sb,
                                                        long long sh, long long sq, MaskShape m,
                                                        int Lk, unsigned* bits) {
  wait_for_previous();
  let_next_start();
  const int lane = threadIdx.x % 32;
  const unsigned segments = (m.words + kMaskWords - 1) / kMaskWords;
  const unsigned at = blockIdx.x * 8 + threadIdx.x / 32, row = at / segments;
  if (row >= (unsigned)(m.b * m.h * m.q)) return;
  const int w0 = (int)(at - row * segments) * kMaskWords;
  const unsigned bh = row / (unsigned)m.q, q = row - bh * (unsigned)m.q;
  const unsigned b = bh / (unsigned)m.h, h = bh - b * (unsigned)m.h;
  const unsigned char* p = mask + b * sb + h * sh + q * sq;
  unsigned mine = 0;
  if (ALIGNED) {
    unsigned v[kMaskWords / 4];
#pragma unroll
    for (int k = 0; k < kMaskWords / 4; ++k) {  // keys w0 32 + 128 k + 4 lane and the next 3
      const int j = w0 * 32 + 128 * k + 4 * lane;
      v[k] = 0;
      if (j + 4 <= Lk) {
        v[k] = *reinterpret_cast<const unsigned*>(p + j);
      } else {
        for (int i = 0; i < 4; ++i)
          if (j + i < Lk) v[k] |= (unsigned)p[j + i] << (8 * i);
      }
    }
#pragma unroll
    for (int k = 0; k < kMaskWords / 4; ++k) {
      // four bytes to four bits, then eight lanes' bits to a word
      const unsigned nz = __vcmpne4(v[k], 0u) & 0x01010101u;
      unsigned word = ((nz * 0x01020408u) >> 24 & 0xfu) << (4 * (lane % 8));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) word |= __shfl_xor_sync(~0u, word, o);
      // words 4 k .. 4 k + 3 are in lanes 0, 8, 16, 24; lane 4 k + i keeps word 4 k + i
      const unsigned got = __shfl_sync(~0u, word, lane % 4 * 8);
      if (lane / 4 == k) mine = got;
    }
  } else {
    unsigned char v[kMaskWords];
#pragma unroll
    for (int k = 0; k < kMaskWords; ++k) {
      const int j = (w0 + k) * 32 + lane;
      v[k] = j < Lk ? p[j] : 0;
    }
#pragma unroll
    for (int k = 0; k < kMaskWords; ++k) {
      const unsigned word = __ballot_sync(~0u, v[k] != 0);
      if (lane == k) mine = word;
    }
  }
  if (lane < kMaskWords && w0 + lane < m.words) bits[(long long)row * m.words + w0 + lane] = mine;
}

size_t attention_mask_bytes(const gs_attention_args& a) {
  if (!a.mask || a.Lk == 0) return 0;
  const MaskShape m = mask_shape(a);
  return (size_t)(m.b * m.h * m.q) * m.words * sizeof(unsigned);
}

int attention_pack_mask(const gs_attention_args& a, AttentionParams& p, void* workspace,
                        cudaStream_t stream) {
  if (!a.mask || a.Lk == 0) return GS_OK;
  const MaskShape m = mask_shape(a);
  unsigned* bits = static_cast<unsigned*>(workspace);
  p.bits = bits;
  p.bits_q = m.q > 1 ? m.words : 0;
  p.bits_h = m.h > 1 ? m.q * m.words : 0;
  p.bits_b = m.b > 1 ? m.h * m.q * m.words : 0;
  const long long warps = m.b * m.h * m.q * ((m.words + kMaskWords - 1) / kMaskWords);
  GS_REQUIRE(m.b * m.h * m.q < (1ll << 31) && warps < (1ll << 32) - 8, "the mask is too large");
  const unsigned blocks = (unsigned)((warps + 7) / 8);
  const bool aligned = (reinterpret_cast<uintptr_t>(a.mask) | (uintptr_t)a.mask_batch_stride |
                        (uintptr_t)a.mask_head_stride | (uintptr_t)a.mask_query_stride) % 4 == 0;
  GS_CUDA(launch_overlapped(aligned ? mask_bits_kernel<true> : mask_bits_kernel<false>, dim3(blocks),
                            256, 0, stream, a.mask, a.mask_batch_stride, a.mask_head_stride,
                            a.mask_query_stride, m, a.Lk, bits));
  count_launches(1u);
  return GS_OK;
}

}  // namespace gs
