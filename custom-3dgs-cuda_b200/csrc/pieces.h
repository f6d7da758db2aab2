// An axis cut into pieces of nearly the same length.
#pragma once

#ifdef __CUDACC__
#define GS_HOST_DEVICE __host__ __device__
#else
#define GS_HOST_DEVICE
#endif

namespace gs {

// The first of `count` things that `piece` of `pieces` takes; the piece after it begins at its end. The
// product is formed in 64 bits: a key head shared by 2^25 query heads has that many tiles of queries.
GS_HOST_DEVICE constexpr int piece_begin(int count, int piece, int pieces) {
  return pieces == 1 ? piece * count : (int)((long long)count * piece / pieces);
}

}  // namespace gs
