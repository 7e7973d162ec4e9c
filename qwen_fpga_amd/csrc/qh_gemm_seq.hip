// y[t][o] = float(sum_i xq[t][i] w[o][i]) * sx[t] * scale[o] for the int8 activations of many tokens.
// The int32 sums are exact in any order, and the two products are rounded as the one-token op rounds
// them, so an fp32 y equals qh_gemv_i8_w8a8's bit for bit.
#include "qh_device.hpp"
#include "qh_seq.hpp"

namespace qh {

typedef int i32x4 __attribute__((ext_vector_type(4)));

namespace {

template <bool BF16>
__device__ __forceinline__ void put(void* y, int64_t at, float v) {
  if constexpr (BF16)
    as_global_w(static_cast<__bf16*>(y))[at] = (__bf16)v;
  else
    as_global_w(static_cast<float*>(y))[at] = v;
}

// A wave per tile of 16 weight rows x 16 tokens, operands straight from memory.
template <bool BF16>
__global__ __launch_bounds__(256) void gemm_seq_kernel(const GemmSeq a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int n0 = ((int)blockIdx.x * 4 + wave) * 16, m0 = (int)blockIdx.y * 16;
  if (n0 >= a.out) return;
  const int nr = min(n0 + j, a.out - 1), mr = min(m0 + j, a.tokens - 1);
  const int8_t* wp = a.w + (size_t)nr * a.in;
  const int8_t* xp = static_cast<const int8_t*>(a.x.p) + (int64_t)mr * a.x.ld;
  i32x4 acc = {0, 0, 0, 0};
  for (int k = 16 * g; k < a.in + 16 * g; k += 64) {
    i32x4 wv = {0, 0, 0, 0}, xv = {0, 0, 0, 0};
    if (k < a.in) {
      wv = *as_global(reinterpret_cast<const i32x4*>(wp + k));
      xv = *as_global(reinterpret_cast<const i32x4*>(xp + k));
    }
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, xv, acc, 0, 0, 0);
  }
  const int m = m0 + j;
  if (m >= a.tokens) return;
  const float xs = as_global(a.sx)[m];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int n = n0 + 4 * g + r;
    if (n < a.out) put<BF16>(a.y.p, (int64_t)m * a.y.ld + n, ((float)acc[r] * xs) * as_global(a.scale)[n]);
  }
}

}  // namespace

hipError_t launch_gemm_seq(const GemmSeq& a, hipStream_t s) {
  const dim3 grid((a.out + 63) / 64, (a.tokens + 15) / 16);
  if (a.bf16)
    gemm_seq_kernel<true><<<grid, 256, 0, s>>>(a);
  else
    gemm_seq_kernel<false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace qh
