// simple.hpp -- a plain tiled product for any layout of its operands: 64 x 64 tiles, elements one by one through LDS.
#pragma once
#include "act.hpp"
#include "mx4.hpp"

namespace ggemm {

// Tile t of the groups in order (64 rows, nt of them along n): its group, rows [lo, hi) from the tile's first on.
__device__ __forceinline__ bool simple_rows(const int32_t* offsets, int groups, int m, int nt, int t, int& g, int& lo, int& hi, int& tn) {
  for (g = 0; g < groups; ++g) {
    lo = offsets ? min(max(offsets[g], 0), m) : 0;
    hi = offsets ? min(max(offsets[g + 1], 0), m) : m;
    const int tiles = ceil_div(max(hi - lo, 0), 64) * nt;
    if (t < tiles) {
      lo += t / nt * 64;
      tn = t % nt;
      return true;
    }
    t -= tiles;
  }
  return false;
}

// P: Acc, kPairs (products of a pass), place(tile), depth(), a(pair, i, k), b(pair, j, k), emit(i, j, sums)
template <class P>
__global__ void __launch_bounds__(256) simple_kernel(P p) {
  using Acc = typename P::Acc;
  constexpr int K = 16;
  __shared__ Acc la[K][65], lb[P::kPairs][K][65];
  if (!p.place(blockIdx.x)) return;
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  Acc acc[P::kPairs][4][4] = {};
  for (int k0 = 0; k0 < p.depth(); k0 += K) {
    for (int e = threadIdx.x; e < 64 * K; e += 256) {
      const int i = e / K, k = e % K;
      la[k][i] = p.a(i, k0 + k);
      for (int z = 0; z < P::kPairs; ++z) lb[z][k][i] = p.b(z, i, k0 + k);
    }
    __syncthreads();
    for (int k = 0; k < K; ++k)
      for (int z = 0; z < P::kPairs; ++z)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) acc[z][i][j] += la[k][ti + i] * lb[z][k][tj + j];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      Acc s[P::kPairs];
      for (int z = 0; z < P::kPairs; ++z) s[z] = acc[z][i][j];
      p.emit(ti + i, tj + j, s);
    }
}

}  // namespace ggemm
