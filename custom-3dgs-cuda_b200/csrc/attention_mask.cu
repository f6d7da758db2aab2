// The mask of the attention kernels, packed from a byte to a bit for each key.
//
// A thread of those kernels holds one query's scores of 128 keys: as bytes its part of the mask
// would be 128 loads that no two lanes share, in an order that no alignment helps (a mask of 777
// keys has rows of 777 bytes); as bits it is one load of 16 bytes. Heads that share a mask share
// its bits. A warp takes 256 keys of a row, its loads all in flight. Reading the bytes in the
// attention kernel instead made its 3 x 1,111 x 777 of 12 heads take 365 us; with the bits it took 67.
//
// A key that none of the queries and heads keeps that share it may hold anything, NaN included, which a
// weight of 0 does not hide from a product; the kernels that multiply with v (or, in the gradient, k)
// clear those rows. For that they need the OR of all rows of the mask over an item's key head. Up to
// kKeptRows of them a warp gets from the bits; where there are more, the rows are packed by warps that
// take several and leave the OR of those, kKeptMost a key head at most, in a place of its own: no memory
// that warps share, nothing to clear first. With its four rows read at once that is also the faster form
// where there are many (3 x 6,000 x 10,000: 140 us a row a warp, 73 so; 3 x 1,111 x 777: 6.0 and 7.5).
// More parts cost the kernel that reads them more (512: 389 us instead of 286 there).
#include <algorithm>

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

constexpr int kMaskWords = 8;   // a warp's
constexpr int kKeptRows = 128;  // rows of the bits that a warp ORs for itself
constexpr int kAtOnce = 4;      // rows that a warp reads at once where it ORs them

// The mask's rows that one key head's keys are kept by; they follow one another in the bits.
struct KeptShape {
  long long groups, rows;  // (batch item, key head) pairs with rows of their own, and rows of each
  unsigned parts, each;    // ORs of `each` rows, where there are more than kKeptRows; else 0
};

static KeptShape kept_shape(const gs_attention_args& a, const MaskShape& m) {
  KeptShape k{};
  k.groups = m.b * (m.h > 1 ? a.Hkv : 1);
  k.rows = (m.h > 1 ? a.Hq / a.Hkv : 1) * m.q;
  if (k.rows > kKeptRows) {
    k.each = (unsigned)(((k.rows + kKeptMost - 1) / kKeptMost + kAtOnce - 1) / kAtOnce * kAtOnce);
    k.parts = (unsigned)((k.rows + k.each - 1) / k.each);
  }
  return k;
}

// What a lane reads of kMaskWords words' keys from w0 on. ALIGNED: rows start on 4-byte boundaries, and
// a lane reads 4 keys at once.
template <bool ALIGNED>
struct MaskBytes {
  static constexpr int kLoads = ALIGNED ? kMaskWords / 4 : kMaskWords;
  unsigned v[kLoads];

  __device__ __forceinline__ void load(const unsigned char* p, int w0, int Lk) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      v[k] = 0;
      if (ALIGNED) {  // keys w0 32 + 128 k + 4 lane and the next 3
        const int j = w0 * 32 + 128 * k + 4 * lane;
        if (j + 4 <= Lk) {
          v[k] = *reinterpret_cast<const unsigned*>(p + j);
        } else {
          for (int i = 0; i < 4; ++i)
            if (j + i < Lk) v[k] |= (unsigned)p[j + i] << (8 * i);
        }
      } else {
        const int j = (w0 + k) * 32 + lane;
        if (j < Lk) v[k] = p[j];
      }
    }
  }

  // Word w0 + lane, in the first kMaskWords lanes.
  __device__ __forceinline__ unsigned word() const {
    const int lane = threadIdx.x % 32;
    unsigned mine = 0;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      if (ALIGNED) {
        // four bytes to four bits, then eight lanes' bits to a word
        const unsigned nz = __vcmpne4(v[k], 0u) & 0x01010101u;
        unsigned word = ((nz * 0x01020408u) >> 24 & 0xfu) << (4 * (lane % 8));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) word |= __shfl_xor_sync(~0u, word, o);
        // words 4 k .. 4 k + 3 are in lanes 0, 8, 16, 24; lane 4 k + i keeps word 4 k + i
        const unsigned got = __shfl_sync(~0u, word, lane % 4 * 8);
        if (lane / 4 == k) mine = got;
      } else {
        const unsigned word = __ballot_sync(~0u, v[k] != 0);
        if (lane == k) mine = word;
      }
    }
    return mine;
  }
};

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
  MaskBytes<ALIGNED> bytes;
  bytes.load(mask + b * sb + h * sh + q * sq, w0, Lk);
  const unsigned mine = bytes.word();
  if (lane < kMaskWords && w0 + lane < m.words) bits[(long long)row * m.words + w0 + lane] = mine;
}

// The same with a warp for `each` rows of a group and kMaskWords words, whose OR goes to row `part` of the
// group's, the rows of a tile of 128 keys beside one another: [groups, words / 4, parts, 4].
template <bool ALIGNED>
__global__ void __launch_bounds__(256) mask_parts_kernel(const unsigned char* mask, long long sb,
                                                         long long sh, long long sq, MaskShape m,
                                                         KeptShape g, int Lk, unsigned* bits,
                                                         unsigned* kept) {
  wait_for_previous();
  let_next_start();
  const int lane = threadIdx.x % 32;
  const unsigned segments = (m.words + kMaskWords - 1) / kMaskWords;
  const unsigned at = blockIdx.x * 8 + threadIdx.x / 32, slot = at / segments;
  const unsigned group = slot / g.parts;
  if (group >= (unsigned)g.groups) return;
  const int w0 = (int)(at - slot * segments) * kMaskWords;
  const unsigned first = group * (unsigned)g.rows, from = (slot - group * g.parts) * g.each;
  const unsigned end = min(from + g.each, (unsigned)g.rows);
  unsigned bh = (first + from) / (unsigned)m.q, q = first + from - bh * (unsigned)m.q;
  const unsigned char* p = mask + bh / (unsigned)m.h * sb + bh % (unsigned)m.h * sh + q * sq;
  const bool writes = lane < kMaskWords && w0 + lane < m.words;
  unsigned* to = bits + (long long)(first + from) * m.words + w0 + lane;
  unsigned any = 0;
  for (unsigned row = from; row < end; row += kAtOnce) {
    MaskBytes<ALIGNED> bytes[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      bytes[k].load(p, w0, Lk);
      if (row + k + 1 >= end) continue;  // the last row again
      if (++q == (unsigned)m.q) {  // the next head of the group, which is of one batch item
        p += sh - (q - 1) * sq;
        q = 0;
      } else {
        p += sq;
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const unsigned mine = bytes[k].word();
      any |= mine;
      if (writes && row + k < end) *to = mine;
      to += m.words;
    }
  }
  if (writes) {
    const int w = w0 + lane;
    const long long tile = (long long)group * (m.words / 4) + w / 4;
    kept[(tile * g.parts + (slot - group * g.parts)) * 4 + w % 4] = any;
  }
}

size_t attention_mask_bytes(const gs_attention_args& a) {
  if (!a.mask || a.Lk == 0) return 0;
  const MaskShape m = mask_shape(a);
  const KeptShape g = kept_shape(a, m);
  return (size_t)(m.b * m.h * m.q + g.groups * g.parts) * m.words * sizeof(unsigned);
}

int attention_pack_mask(const gs_attention_args& a, AttentionParams& p, void* workspace,
                        cudaStream_t stream) {
  const MaskShape m = mask_shape(a);
  if (!a.mask || a.Lk == 0 || m.b * m.h * m.q == 0) return GS_OK;
  unsigned* bits = static_cast<unsigned*>(workspace);
  p.bits = bits;
  p.bits_q = m.q > 1 ? m.words : 0;
  p.bits_h = m.h > 1 ? m.q * m.words : 0;
  p.bits_b = m.b > 1 ? m.h * m.q * m.words : 0;
  const KeptShape g = kept_shape(a, m);
  unsigned* parts = bits + m.b * m.h * m.q * m.words;
  p.kept = g.parts ? parts : bits;
  p.kept_rows = (int)(g.parts ? g.parts : g.rows);
  p.kept_row = g.parts ? 4 : m.words;
  p.kept_tile = g.parts ? (int)g.parts * 4 : 4;
  p.kept_h = m.h > 1 ? (long long)p.kept_rows * m.words : 0;
  p.kept_b = m.b > 1 ? g.groups / m.b * p.kept_rows * m.words : 0;
  const long long segments = (m.words + kMaskWords - 1) / kMaskWords;
  const long long warps = (g.parts ? g.groups * g.parts : m.b * m.h * m.q) * segments;
  GS_REQUIRE(m.b * m.h * m.q < (1ll << 31) && warps < (1ll << 32) - 8, "the mask is too large");
  const bool aligned = (reinterpret_cast<uintptr_t>(a.mask) | (uintptr_t)a.mask_batch_stride |
                        (uintptr_t)a.mask_head_stride | (uintptr_t)a.mask_query_stride) % 4 == 0;
  const dim3 grid((unsigned)((warps + 7) / 8));
  if (g.parts)
    GS_CUDA(launch_overlapped(aligned ? mask_parts_kernel<true> : mask_parts_kernel<false>, grid, 256,
                              0, stream, a.mask, a.mask_batch_stride, a.mask_head_stride,
                              a.mask_query_stride, m, g, a.Lk, bits, parts));
  else
    GS_CUDA(launch_overlapped(aligned ? mask_bits_kernel<true> : mask_bits_kernel<false>, grid, 256, 0,
                              stream, a.mask, a.mask_batch_stride, a.mask_head_stride,
                              a.mask_query_stride, m, a.Lk, bits));
  count_launches(1u);
  return GS_OK;
}

}  // namespace gs
