// y[t][o] = float(sum_i xq[t][i] w[o][i]) * sx[t] * scale[o] for the int8 activations of many tokens.
// The int32 sums are exact in any order, and the two products are rounded as the one-token op rounds
// them, so an fp32 y equals qh_gemv_i8_w8a8's bit for bit.
//
// In both kernels an MFMA's A operand (rows of the result) is 16 weight rows and its B operand 16 tokens,
// so that a lane ends with four consecutive outputs of one token.
#include "qh_seq_device.hpp"

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

// Few tokens, or few outputs: a workgroup takes 16 rows and 16 TT tokens, operands straight from memory into the MFMAs'
// registers, PF steps of 64 in flight.  Every fourth pair of steps (a 128-byte line of each row) is one wave's; the four
// waves' sums meet in LDS.  Bound by the rows' way from memory: 151936 x 1024 weights and 4 tokens 27 us, 5.7 TB/s.
template <bool BF16, int TT>
__global__ __launch_bounds__(256) void gemm_rows_kernel(const GemmSeq a) {
  constexpr int PF = 4, KS = 4;
  __shared__ i32x4 red[KS][TT][64];
  const int lane = threadIdx.x & 63, ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * TT;
  const int NC = a.in >> 4;
  const int8_t *wp = a.w + (size_t)min(n0 + j, a.out - 1) * a.in, *xp[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) xp[t] = static_cast<const int8_t*>(a.x.p) + (int64_t)min(m0 + 16 * t + j, a.tokens - 1) * a.x.ld;
  i32x4 acc[TT], wb[PF], xb[PF][TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[t] = i32x4{0, 0, 0, 0};
  auto chunk = [&](int i) { return 4 * ((i >> 1) * 2 * KS + 2 * ks + (i & 1)) + g; };   // of this wave's step i
  auto load = [&](int i, i32x4& w, i32x4 (&x)[TT]) {
    const int c = 16 * min(chunk(i), NC - 1);
    w = *as_global(reinterpret_cast<const i32x4*>(wp + c));
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
        const i32x4 wv = chunk(i) < NC ? wb[p] : i32x4{0, 0, 0, 0};   // past the end of the row: nothing
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xb[p][t], acc[t], 0, 0, 0);
        if (i + PF < n) load(i + PF, wb[p], xb[p]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) red[ks][t][lane] = acc[t];
  __syncthreads();
  if (ks >= TT) return;
  i32x4 s = red[0][ks][lane];
#pragma unroll
  for (int w = 1; w < KS; ++w) s += red[w][ks][lane];
  const int m = m0 + 16 * ks + j, o = n0 + 4 * g;
  if (m < a.tokens) put4<BF16>(a, m, o, s, as_global(a.sx)[m], scale4(a, o), a.wide && o + 4 <= a.out);
}

// Many tokens: a workgroup takes kBT (128 or 64) rows and kBT tokens, in steps of 64 through a ring of four LDS stages
// that global -> LDS loads fill three steps ahead; a wave multiplies a quarter, and reads the fragments of a step beside
// the products of the one before.  A row's 16-byte chunk c stands at chunk c ^ (row / 2 % 4) of its 64 bytes, so that
// eight rows of a fragment, which are read at once, lie in all banks.  4096 tokens of 3584 -> 1024: 23 us, the loop 16.8
// of them (1.8 POP/s at 1.95 GHz; LDS and MFMA pipes are busy for 65 and 45% of it); 1500 tokens of 1024 -> 7168: 26 us,
// two rounds of workgroups, each 8 us of loop and 5 of start and of writing 43 MB of fp32 outputs.  Tiles of 64 are for
// products with fewer tiles than CUs, which the way of one tile bounds: 1024 tokens of 3584 -> 1024 11 us, not 18.
constexpr int kStages = 4;

template <bool BF16, int kBT>
__global__ __launch_bounds__(256, 2) void gemm_tile_kernel(const GemmSeq a, int mt) {
  constexpr int F = kBT / 32, NL = kBT / 64, kStageBytes = 2 * kBT * 64;   // fragments of a wave; loads of w's and of x's rows
  __shared__ __attribute__((aligned(16))) int8_t lds[kStages * kStageBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int b = blockIdx.x;
  const int n0 = (b / mt) * kBT, m0 = (b % mt) * kBT;
  const int wr = 16 * F * (wave & 1), wt = 16 * F * (wave >> 1);
  const int NC = a.in >> 4, NS = (NC + 3) >> 2;
  // a wave's loads of a step: NL x 16 rows of w, NL x 16 of x; lane l brings chunk (l % 4) ^ (row / 2 % 4) of row l / 4
  const int lr = lane >> 2, lc = (lane & 3) ^ ((lr >> 1) & 3);
  const char* src[2] = {reinterpret_cast<const char*>(a.w) + (size_t)n0 * a.in, static_cast<const char*>(a.x.p) + (int64_t)m0 * a.x.ld};
  uint32_t off[2 * NL];   // (below 128 rows of less than 2^24 bytes: the launch's rule)
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = 16 * (NL * wave + i) + lr;
    off[i] = (uint32_t)min(r, a.out - 1 - n0) * (uint32_t)a.in;
    off[NL + i] = (uint32_t)min(r, a.tokens - 1 - m0) * (uint32_t)a.x.ld;
  }
  auto stage = [&](int s) {
    const int c = 16 * min(4 * s + lc, NC - 1);
    const uint32_t base = lds_address(lds) + (s & (kStages - 1)) * kStageBytes + 16 * NL * wave * 64;
#pragma unroll
    for (int i = 0; i < 2 * NL; ++i) load_to_lds(src[i / NL], off[i] + c, base + i / NL * (kBT * 64) + i % NL * 1024);
  };
  i32x4 acc[F][F];
#pragma unroll
  for (int r = 0; r < F; ++r)
#pragma unroll
    for (int t = 0; t < F; ++t) acc[r][t] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < kStages; ++s)
    if (s < NS) stage(s);
  const int fo = j * 64 + 16 * (g ^ ((j >> 1) & 3));   // a fragment's place
  i32x4 wv[2][F], xv[2][F];   // fragments of the steps s and s + 1
  // this wave's loads of step s have landed (those of the `ahead` next stay in flight) and its reads of step s - 1 are
  // done; after the barrier every wave's
  auto wait = [&](int ahead) {
    static_assert(kStages == 4, "a case for each number of stages ahead");
    switch (ahead) {
#define QH_WAIT(n) case n: asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NL * n) : "memory"); break;
      QH_WAIT(1) QH_WAIT(2) QH_WAIT(3)
#undef QH_WAIT
      default: asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
  };
  auto read = [&](int s, i32x4 (&w)[F], i32x4 (&x)[F]) {
    const int8_t* base = lds + (s & (kStages - 1)) * kStageBytes;
#pragma unroll
    for (int t = 0; t < F; ++t) {
      w[t] = *as_lds(reinterpret_cast<const i32x4*>(base + (wr + 16 * t) * 64 + fo));
      x[t] = *as_lds(reinterpret_cast<const i32x4*>(base + kBT * 64 + (wt + 16 * t) * 64 + fo));
    }
  };
  wait(min(NS - 1, kStages - 1));
  read(0, wv[0], xv[0]);
  auto mul = [&](const i32x4 (&w)[F], const i32x4 (&x)[F]) {
#pragma unroll
    for (int r = 0; r < F; ++r)
#pragma unroll
      for (int t = 0; t < F; ++t) acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[r], x[t], acc[r][t], 0, 0, 0);
  };
  int s = 0;
  for (; s + 1 + kStages < NS; s += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      wait(kStages - 2);
      stage(s + u + kStages);   // (into the place of step s + u, whose fragments every wave holds)
      read(s + u + 1, wv[1 - u], xv[1 - u]);
      mul(wv[u], xv[u]);
    }
  }
  for (; s < NS; ++s) {
    if (4 * s + 4 > NC) {   // past the end of the row: nothing
#pragma unroll
      for (int t = 0; t < F; ++t)
        if (4 * s + g >= NC) wv[0][t] = i32x4{0, 0, 0, 0};
    }
    mul(wv[0], xv[0]);
    if (s + 1 < NS) {
      wait(min(NS - 2 - s, kStages - 2));
      if (s + kStages < NS) stage(s + kStages);
      read(s + 1, wv[0], xv[0]);
    }
  }
  f32x4 sc[F];
  float xs[F];
#pragma unroll
  for (int r = 0; r < F; ++r) sc[r] = scale4(a, n0 + wr + 16 * r + 4 * g);
#pragma unroll
  for (int t = 0; t < F; ++t) xs[t] = as_global(a.sx)[min(m0 + wt + 16 * t + j, a.tokens - 1)];
  const bool wide = a.wide && n0 + kBT <= a.out;
#pragma unroll
  for (int t = 0; t < F; ++t)
    if (m0 + wt + 16 * t + j < a.tokens)
#pragma unroll
      for (int r = 0; r < F; ++r) put4<BF16>(a, m0 + wt + 16 * t + j, n0 + wr + 16 * r + 4 * g, acc[r][t], xs[t], sc[r], wide);
}

template <bool BF16>
hipError_t launch(const GemmSeq& a, hipStream_t s) {
  const GemmForm f = gemm_form(a.tokens, a.out, a.x.ld);
  const unsigned rt = (a.out + 15) / 16;
  auto tiles = [&]() { return (unsigned)((a.out + f.tile - 1) / f.tile) * ((a.tokens + f.tile - 1) / f.tile); };
  if (f.unit == 16)
    gemm_rows_kernel<BF16, 1><<<dim3(rt, (a.tokens + 15) / 16), 256, 0, s>>>(a);
  else if (f.unit == 32)
    gemm_rows_kernel<BF16, 2><<<dim3(rt, (a.tokens + 31) / 32), 256, 0, s>>>(a);
  else if (f.tile == 64)
    gemm_tile_kernel<BF16, 64><<<tiles(), 256, 0, s>>>(a, (a.tokens + 63) / 64);
  else
    gemm_tile_kernel<BF16, 128><<<tiles(), 256, 0, s>>>(a, (a.tokens + 127) / 128);
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
