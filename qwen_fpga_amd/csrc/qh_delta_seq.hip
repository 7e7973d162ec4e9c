// The gated delta rule over packed sequences.  A token of one head, with S [128][128] (k-major), does
//   S = exp(g) S;  d = beta (v - S^T k);  S = S + k d^T;  out = S^T q
#include "qh_device.hpp"
#include "qh_seq.hpp"

namespace qh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr int kD = 128;

template <bool BF16>
__device__ __forceinline__ void load8(const void* p, int64_t at, float (&v)[8]) {
  if constexpr (BF16) {
    const bf16x8 t = *as_global(reinterpret_cast<const bf16x8*>(static_cast<const __bf16*>(p) + at));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
  } else {
    const f32x4* f = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const f32x4 a = *as_global(f), b = *as_global(f + 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  }
}
template <bool BF16>
__device__ __forceinline__ float load1(const void* p, int64_t at) {
  if constexpr (BF16)
    return (float)as_global(static_cast<const __bf16*>(p))[at];
  else
    return as_global(static_cast<const float*>(p))[at];
}
template <bool BF16>
__device__ __forceinline__ void store1(void* p, int64_t at, float v) {
  if constexpr (BF16)
    as_global_w(static_cast<__bf16*>(p))[at] = (__bf16)v;
  else
    as_global_w(static_cast<float*>(p))[at] = v;
}

// Sums of four values over the 16 lanes of equal lane % 4, scattered: the lane ends with value
// 2 (lane / 32) + lane / 16 % 2.
__device__ __forceinline__ float sum16(const float (&p)[4]) {
  float x = swap_add<16>(swap_add<32>(p[0], p[2]), swap_add<32>(p[1], p[3]));
  x = x + xor_perm<8>(x);
  return x + xor_perm<4>(x);
}
// All four of the values that sum16 scattered.
__device__ __forceinline__ void gather4(float x, float (&v)[4]) {
  unsigned a = __float_as_uint(x), b = a;
  permlane16_swap(a, b);
  unsigned a2 = a, b2 = b;
  permlane32_swap(a, a2);
  permlane32_swap(b, b2);
  v[0] = __uint_as_float(a);
  v[1] = __uint_as_float(b);
  v[2] = __uint_as_float(a2);
  v[3] = __uint_as_float(b2);
}

// Token by token: a wave keeps 16 columns of one head's state in registers (lane: 8 k of 4 columns).
template <bool BF16>
__global__ __launch_bounds__(256) void delta_step_kernel(const DeltaSeq a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u = (int)blockIdx.x * 4 + wave;   // unit: sequence, head, 16 columns
  const int sl = u & 7, h = (u >> 3) % a.heads, i = (u >> 3) / a.heads;
  if (i >= a.n_seq) return;
  const SeqSpan sp = seq_span(as_global(a.cu)[i], as_global(a.cu)[i + 1], a.tokens);
  if (sp.len == 0) return;
  const int hk = h / (a.heads / a.k_heads);
  const int cq = lane & 3, kg = lane >> 2, col = 16 * sl + 4 * cq;
  const int mine = ((lane >> 5) << 1) + ((lane >> 4) & 1);   // the column sum16 leaves here
  f32x4* Sp = reinterpret_cast<f32x4*>(a.S + (((size_t)i * a.heads + h) * kD + 8 * kg) * kD + col);
  f32x4 s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = *as_global(Sp + e * (kD / 4));
  for (int t = sp.start; t < sp.start + sp.len; ++t) {
    float kk[8], qq[8];
    load8<BF16>(a.k.p, t * a.k.ld + hk * a.k.hs + 8 * kg, kk);
    load8<BF16>(a.q.p, t * a.q.ld + hk * a.q.hs + 8 * kg, qq);
    const float vv = load1<BF16>(a.v.p, t * a.v.ld + h * a.v.hs + col + mine);
    const float dec = dev_expf(as_global(a.g)[t * a.ldg + h]), be = as_global(a.beta)[t * a.ldb + h];
    float p[4] = {0.0f, 0.0f, 0.0f, 0.0f}, d[4];
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[e][c] *= dec;
        p[c] = __builtin_fmaf(s[e][c], kk[e], p[c]);
      }
    gather4((vv - sum16(p)) * be, d);
#pragma unroll
    for (int c = 0; c < 4; ++c) p[c] = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[e][c] = __builtin_fmaf(kk[e], d[c], s[e][c]);
        p[c] = __builtin_fmaf(s[e][c], qq[e], p[c]);
      }
    const float o = sum16(p);
    if ((kg & 3) == 0) store1<BF16>(a.out.p, t * a.out.ld + h * a.out.hs + col + mine, o);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) *as_global_w(Sp + e * (kD / 4)) = s[e];
}

}  // namespace

hipError_t launch_delta_seq(const DeltaSeq& a, hipStream_t s) {
  const unsigned grid = (unsigned)(((int64_t)a.n_seq * a.heads * 8 + 3) / 4);
  if (a.bf16)
    delta_step_kernel<true><<<grid, 256, 0, s>>>(a);
  else
    delta_step_kernel<false><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace qh
