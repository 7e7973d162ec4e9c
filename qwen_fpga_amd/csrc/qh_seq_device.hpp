// Device helpers of the operators over packed sequences.
#pragma once
#include "qh_device.hpp"
#include "qh_seq.hpp"

namespace qh {

// The sequence and the tile in it of row tile b (tiles of `tile` rows; a token is `mult` rows).
struct TileAt {
  int seq, tile;
  SeqSpan sp;
};
__device__ __forceinline__ bool find_tile(const int32_t* cu, int n_seq, int rows, int mult, int tile, int b, TileAt& o) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < n_seq; s0 += 64) {
    const int i = s0 + lane;
    SeqSpan sp = {0, 0};
    if (i < n_seq) sp = seq_span(as_global(cu)[i], as_global(cu)[i + 1], rows);
    const int n = seq_tiles(sp.len * mult, tile);
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int t = __shfl_up(inc, d);
      if (lane >= d) inc += t;
    }
    const uint64_t past = __ballot(base + inc > b);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      o.seq = s0 + l;
      o.tile = b - base - (__builtin_amdgcn_readlane(inc, l) - __builtin_amdgcn_readlane(n, l));
      o.sp = {__builtin_amdgcn_readlane(sp.start, l), __builtin_amdgcn_readlane(sp.len, l)};
      return o.tile >= 0 && o.tile < __builtin_amdgcn_readlane(n, l);   // (overlapping bounds can overflow the count)
    }
    base += __builtin_amdgcn_readlane(inc, 63);
  }
  return false;
}

}  // namespace qh
