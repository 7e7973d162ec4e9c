// Device helpers of the operators over packed sequences.
#pragma once
#include "qh_device.hpp"
#include "qh_seq.hpp"

namespace qh {

// The sum over this lane and those before it, by DPP (within rows of 16 lanes, then the row before and the half before).
__device__ __forceinline__ int sum_up_to(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15, rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31, rows 2 and 3
  return v;
}
// The sum over all lanes of values from 0 to 2^48 (larger ones count as that).
__device__ __forceinline__ int64_t sum_all(int64_t v) {
  v = min(v, (int64_t)1 << 48);
  const uint32_t lo = __builtin_amdgcn_readlane(sum_up_to((int)(v & 0xffffff)), 63), hi = __builtin_amdgcn_readlane(sum_up_to((int)(v >> 24)), 63);
  return ((int64_t)hi << 24) + lo;
}

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
    const int inc = sum_up_to(n);
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

// The sequence in place i when each 64 sequences stand with the longest first (the earlier of equal ones): the
// workgroups that have most to do are then not the last to start.
__device__ __forceinline__ int longest_first(const int32_t* cu, int n_seq, int rows, int i) {
  const int lane = threadIdx.x & 63, s0 = i & ~63, n = min(n_seq - s0, 64);
  int len = -1;
  if (lane < n) len = seq_span(as_global(cu)[s0 + lane], as_global(cu)[s0 + lane + 1], rows).len;
  int rank = 0;
  for (int l = 0; l < n; ++l) {
    const int o = __builtin_amdgcn_readlane(len, l);
    rank += o > len || (o == len && l < lane);
  }
  const uint64_t at = __ballot(lane < n && rank == (i & 63));
  return s0 + __builtin_ctzll(at);
}

// LDS by its 32-bit address.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
template <typename T>
__device__ __forceinline__ __attribute__((address_space(3))) T* lds_at(uint32_t p) {
  return (__attribute__((address_space(3))) T*)(uintptr_t)p;
}

// 16 bytes per lane from base + off (base the same for the wave) to LDS at `to` + 16 lane (`to` the same for the
// wave, in m0, which the compiler sets as the operand that it is).  In assembly, so that the caller counts the loads in
// flight itself (s_waitcnt vmcnt before the barrier that hands a stage over): the compiler waits for every such load
// before any transposing LDS read.  Nothing is returned to a register.
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t off, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(__builtin_amdgcn_readfirstlane(to)), "v"(off), "s"(base) : "memory");
}

}  // namespace qh
