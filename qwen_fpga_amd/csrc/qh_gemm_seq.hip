// y[t][o] = float(sum_i xq[t][i] w[o][i]) * sx[t] * scale[o] for the int8 activations of many tokens.
// The int32 sums are exact in any order, and the two products are rounded as the one-token op rounds
// them, so an fp32 y equals qh_gemv_i8_w8a8's bit for bit.
//
// In both kernels an MFMA's A operand (rows of the result) is 16 weight rows and its B operand 16 tokens,
// so that a lane ends with four consecutive outputs of one token.
#include "qh_device.hpp"
#include "qh_seq.hpp"

namespace qh {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

namespace {

// Scales of the outputs n .. n + 3 (past the last one: the last one's).
__device__ __forceinline__ f32x4 scale4(const GemmSeq& a, int n) {
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = as_global(a.scale)[min(n + r, a.out - 1)];
  return v;
}

// Outputs n .. n + 3 of token m from their sums.  wide: all four exist and their place is aligned for one store.
template <bool BF16>
__device__ __forceinline__ void put4(const GemmSeq& a, int m, int n, const i32x4& acc, float xs, const f32x4& sc, bool wide) {
  const int64_t at = (int64_t)m * a.y.ld + n;
  f32x4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = ((float)acc[r] * xs) * sc[r];
  if (wide) {
    if constexpr (BF16) {
      u32x2 p;
#pragma unroll
      for (int r = 0; r < 2; ++r)
        p[r] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * r]) |
               (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * r + 1]) << 16;
      *as_global_w(reinterpret_cast<u32x2*>(static_cast<__bf16*>(a.y.p) + at)) = p;
    } else {
      *as_global_w(reinterpret_cast<f32x4*>(static_cast<float*>(a.y.p) + at)) = v;
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < a.out) {
        if constexpr (BF16)
          as_global_w(static_cast<__bf16*>(a.y.p))[at + r] = (__bf16)v[r];
        else
          as_global_w(static_cast<float*>(a.y.p))[at + r] = v[r];
      }
  }
}

// Few tokens, or few outputs: a wave takes 16 RT rows and 16 TT tokens, operands straight from memory into the
// MFMAs' registers, PF steps of 64 in flight.  KS waves share the rows and every KS-th pair of steps (a 128-byte
// line of each row) is a wave's own; their sums meet in LDS.
template <bool BF16, int RT, int TT, int KS>
__global__ __launch_bounds__(256) void gemm_rows_kernel(const GemmSeq a) {
  constexpr int PF = 4;
  __shared__ i32x4 red[KS > 1 ? KS : 1][KS > 1 ? RT * TT : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int ks = KS > 1 ? wave : 0;
  const int n0 = (KS > 1 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave) * 16 * RT, m0 = (int)blockIdx.y * 16 * TT;
  if (n0 >= a.out) return;   // (KS == 1: a whole wave; KS > 1: never)
  const int NC = a.in >> 4;
  const int8_t *wp[RT], *xp[TT];
#pragma unroll
  for (int r = 0; r < RT; ++r) wp[r] = a.w + (size_t)min(n0 + 16 * r + j, a.out - 1) * a.in;
#pragma unroll
  for (int t = 0; t < TT; ++t) xp[t] = static_cast<const int8_t*>(a.x.p) + (int64_t)min(m0 + 16 * t + j, a.tokens - 1) * a.x.ld;
  i32x4 acc[RT][TT], wb[PF][RT], xb[PF][TT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[r][t] = i32x4{0, 0, 0, 0};
  auto chunk = [&](int i) { return 4 * ((i >> 1) * 2 * KS + 2 * ks + (i & 1)) + g; };   // of this wave's step i
  auto load = [&](int i, i32x4 (&w)[RT], i32x4 (&x)[TT]) {
    const int c = 16 * min(chunk(i), NC - 1);
#pragma unroll
    for (int r = 0; r < RT; ++r) w[r] = *as_global(reinterpret_cast<const i32x4*>(wp[r] + c));
#pragma unroll
    for (int t = 0; t < TT; ++t) x[t] = *as_global(reinterpret_cast<const i32x4*>(xp[t] + c));
  };
  const int n = ((NC + 8 * KS - 1) / (8 * KS)) * 2;   // steps of a wave
#pragma unroll
  for (int p = 0; p < PF; ++p)
    if (p < n) load(p, wb[p], xb[p]);
  for (int i0 = 0; i0 < n; i0 += PF) {
#pragma unroll
    for (int p = 0; p < PF; ++p) {
      const int i = i0 + p;
      if (i < n) {
        const bool in = chunk(i) < NC;   // past the end of the row: nothing
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const i32x4 wv = in ? wb[p][r] : i32x4{0, 0, 0, 0};
#pragma unroll
          for (int t = 0; t < TT; ++t) acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xb[p][t], acc[r][t], 0, 0, 0);
        }
        if (i + PF < n) load(i + PF, wb[p], xb[p]);
      }
    }
  }
  if constexpr (KS > 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t) red[ks][r * TT + t][lane] = acc[r][t];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < (RT * TT + KS - 1) / KS; ++u) {
      const int q = u * KS + ks;
      if (q >= RT * TT) break;
      i32x4 s = red[0][q][lane];
#pragma unroll
      for (int w = 1; w < KS; ++w) s += red[w][q][lane];
      const int m = m0 + 16 * (q % TT) + j;
      const int n = n0 + 16 * (q / TT) + 4 * g;
      if (m < a.tokens) put4<BF16>(a, m, n, s, as_global(a.sx)[m], scale4(a, n), a.wide && n + 4 <= a.out);
    }
  } else {
    f32x4 sc[RT];
    float xs[TT];
#pragma unroll
    for (int r = 0; r < RT; ++r) sc[r] = scale4(a, n0 + 16 * r + 4 * g);
#pragma unroll
    for (int t = 0; t < TT; ++t) xs[t] = as_global(a.sx)[min(m0 + 16 * t + j, a.tokens - 1)];
    const bool wide = a.wide && n0 + 16 * RT <= a.out;
#pragma unroll
    for (int t = 0; t < TT; ++t)
      if (m0 + 16 * t + j < a.tokens)
#pragma unroll
        for (int r = 0; r < RT; ++r) put4<BF16>(a, m0 + 16 * t + j, n0 + 16 * r + 4 * g, acc[r][t], xs[t], sc[r], wide);
  }
}

// Many tokens: a workgroup takes 128 rows and 128 tokens, in steps of 64 through a ring of four LDS stages that
// global -> LDS loads fill three steps ahead; a wave multiplies 64 x 64.  A row's 16-byte chunk c stands at chunk
// c ^ (row / 4 % 4) of its 64 bytes, so that the 16 rows that a fragment reads lie in 16 different bank groups.
constexpr int kBT = 128, kStages = 4, kStageBytes = 2 * kBT * 64;

template <bool BF16>
__global__ __launch_bounds__(256, 2) void gemm_tile_kernel(const GemmSeq a, int nt, int mt) {
  __shared__ __attribute__((aligned(16))) int8_t lds[kStages * kStageBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int b = blockIdx.x;
  const int n0 = (b / mt) * kBT, m0 = (b % mt) * kBT;
  const int wr = 64 * (wave & 1), wt = 64 * (wave >> 1);
  const int NC = a.in >> 4, NS = (NC + 3) >> 2;
  // a wave's loads of a step: 2 x 16 rows of w, 2 x 16 of x; lane l brings chunk (l % 4) ^ (row / 4 % 4) of row l / 4
  const int lr = lane >> 2, lc = (lane & 3) ^ ((lr >> 2) & 3);
  const int8_t* src[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * wave + 16 * i + lr;
    src[i] = a.w + (size_t)min(n0 + r, a.out - 1) * a.in;
    src[2 + i] = static_cast<const int8_t*>(a.x.p) + (int64_t)min(m0 + r, a.tokens - 1) * a.x.ld;
  }
  auto stage = [&](int s) {
    const int c = 16 * min(4 * s + lc, NC - 1);
    int8_t* base = lds + (s & (kStages - 1)) * kStageBytes + 32 * wave * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_global_load_lds(as_global(src[i] + c), as_lds_w(base + (i >> 1) * (kBT * 64) + (i & 1) * 1024), 16, 0, 0);
  };
  i32x4 acc[4][4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[r][t] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s)
    if (s < NS) stage(s);
  const int fo = j * 64 + 16 * (g ^ ((j >> 2) & 3));   // a fragment's place
  for (int s = 0; s < NS; ++s) {
    // this wave's loads of step s have landed (those of the next two stay in flight) and its reads of step s - 1 are
    // done; after the barrier every wave's
    if (s + 2 < NS)
      asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if (s + 1 < NS)
      asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + 3 < NS) stage(s + 3);
    const int8_t* base = lds + (s & (kStages - 1)) * kStageBytes;
    i32x4 wv[4], xv[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      wv[t] = *as_lds(reinterpret_cast<const i32x4*>(base + (wr + 16 * t) * 64 + fo));
      xv[t] = *as_lds(reinterpret_cast<const i32x4*>(base + kBT * 64 + (wt + 16 * t) * 64 + fo));
    }
    if (4 * s + 4 > NC) {   // past the end of the row: nothing
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (4 * s + g >= NC) wv[t] = i32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[r], xv[t], acc[r][t], 0, 0, 0);
  }
  f32x4 sc[4];
  float xs[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) sc[r] = scale4(a, n0 + wr + 16 * r + 4 * g);
#pragma unroll
  for (int t = 0; t < 4; ++t) xs[t] = as_global(a.sx)[min(m0 + wt + 16 * t + j, a.tokens - 1)];
  const bool wide = a.wide && n0 + kBT <= a.out;
#pragma unroll
  for (int t = 0; t < 4; ++t)
    if (m0 + wt + 16 * t + j < a.tokens)
#pragma unroll
      for (int r = 0; r < 4; ++r) put4<BF16>(a, m0 + wt + 16 * t + j, n0 + wr + 16 * r + 4 * g, acc[r][t], xs[t], sc[r], wide);
}

template <bool BF16, int TT>
void launch_rows(const GemmSeq& a, hipStream_t s) {
  const int nt = (a.out + 15) / 16, mt = (a.tokens + 16 * TT - 1) / (16 * TT);
  if ((int64_t)nt * mt >= 4096)
    gemm_rows_kernel<BF16, 2, TT, 1><<<dim3((nt + 7) / 8, mt), 256, 0, s>>>(a);
  else
    gemm_rows_kernel<BF16, 1, TT, 4><<<dim3(nt, mt), 256, 0, s>>>(a);
}

template <bool BF16>
hipError_t launch(const GemmSeq& a, hipStream_t s) {
  const int nt = (a.out + kBT - 1) / kBT, mt = (a.tokens + kBT - 1) / kBT;
  if (a.tokens <= 16)
    launch_rows<BF16, 1>(a, s);
  else if (a.tokens <= 32)
    launch_rows<BF16, 2>(a, s);
  else if (a.tokens <= 64 || (int64_t)nt * mt < 64)
    launch_rows<BF16, 4>(a, s);
  else
    gemm_tile_kernel<BF16><<<(unsigned)((int64_t)nt * mt), 256, 0, s>>>(a, nt, mt);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_gemm_seq(const GemmSeq& a0, hipStream_t s) {
  GemmSeq a = a0;
  const int wb = a.bf16 ? 8 : 16;   // four outputs
  a.wide = (reinterpret_cast<uintptr_t>(a.y.p) % wb) == 0 && (a.tokens == 1 || a.y.ld % 4 == 0);
  return a.bf16 ? launch<true>(a, s) : launch<false>(a, s);
}

}  // namespace qh
