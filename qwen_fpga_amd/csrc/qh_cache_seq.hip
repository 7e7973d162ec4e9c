// What stands between the projections and the attention over an int8 cache, for the rows of many tokens: the norms of
// queries and keys with their position rotation, keys and values quantised into rows of the cache, and rows of the
// cache as the values that they stand for.  All three are bound by memory (few tokens: by a launch).
#include "qh_seq_device.hpp"

namespace qh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace {

// Eight neighbours of a row, widened.
template <bool BF16>
__device__ __forceinline__ void load8(const char* p, float (&x)[8]) {
  if constexpr (BF16) {
    const u32x4 v = *as_global(reinterpret_cast<const u32x4*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  } else {
    const f32x4 a = *as_global(reinterpret_cast<const f32x4*>(p)), b = *as_global(reinterpret_cast<const f32x4*>(p) + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  }
}
template <bool BF16>
__device__ __forceinline__ void store8(char* p, const float (&x)[8]) {
  if constexpr (BF16) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (__bf16)x[i];
    *as_global_w(reinterpret_cast<bf16x8*>(p)) = v;
  } else {
    *as_global_w(reinterpret_cast<f32x4*>(p)) = f32x4{x[0], x[1], x[2], x[3]};
    *as_global_w(reinterpret_cast<f32x4*>(p) + 1) = f32x4{x[4], x[5], x[6], x[7]};
  }
}

// y = x / sqrt(mean(x^2) + eps) * (1 + w) of each head, then elements i and i + rot / 2 (i < rot / 2) turned by the
// angle pos * theta^(-2 i / rot).  A workgroup takes one token: its first threads form the angles, counted in turns in
// 64 bits (a float holds an angle of 131071 to 2^-7), the others' loads on their way meanwhile; then D / 8 lanes take a
// head's row at a time, and read the other element of a pair from the lane that holds it.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void norm_rope_kernel(const NormRope a) {
  constexpr int L = D / 8, E = BF16 ? 2 : 4, NG = 256 / L;
  __shared__ __attribute__((aligned(16))) float cs[2][D / 2];
  const int tok = blockIdx.x, c = threadIdx.x % L, grp = threadIdx.x / L, n = a.heads + a.kv_heads, half = a.rot / 2;
  auto load = [&](int r, float (&x)[8]) {
    const bool q = r < a.heads;
    const SeqIn& s = q ? a.q : a.k;
    load8<BF16>(static_cast<const char*>(s.p) + (tok * s.ld + (q ? r : r - a.heads) * s.hs + 8 * c) * E, x);
  };
  float x[8];
  load(min(grp, n - 1), x);
  if ((int)threadIdx.x < half) {
    const double t = (double)as_global(a.pos)[tok] * a.turns[threadIdx.x];
    float si, co;
    sincospif(2.0f * (float)(t - __builtin_rint(t)), &si, &co);
    cs[0][threadIdx.x] = co;
    cs[1][threadIdx.x] = si;
  }
  __syncthreads();
  const int hc = half / 8;                        // pieces of eight in half a rotated part
  const bool lower = c < hc, turned = c < 2 * hc;
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) co[i] = 1.0f, si[i] = 0.0f;
  if (turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      co[i] = cs[0][8 * (lower ? c : c - hc) + i];
      si[i] = cs[1][8 * (lower ? c : c - hc) + i];
      si[i] = lower ? -si[i] : si[i];
    }
  }
  const int lane = threadIdx.x & 63, other = turned ? (lower ? lane + hc : lane - hc) : lane;
  for (int r0 = 0; r0 < n; r0 += NG) {
    const int r = r0 + grp;
    float y[8], next[8];
    if (r0 + NG < n) load(min(r + NG, n - 1), next);
    const bool q = r < a.heads;
    load8<false>(reinterpret_cast<const char*>((q ? a.qw : a.kw) + 8 * c), y);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
    ss = xor_sum<L>(ss);
    const float inv = 1.0f / __builtin_sqrtf(ss / (float)D + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] * inv * (1.0f + y[i]);
    if (hc > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float o = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * other, __float_as_int(y[i])));
        y[i] = turned ? __builtin_fmaf(o, si[i], y[i] * co[i]) : y[i];
      }
    }
    if (r < n) {
      const SeqOut& s = q ? a.qo : a.ko;
      store8<BF16>(static_cast<char*>(s.p) + (tok * s.ld + (q ? r : r - a.heads) * s.hs + 8 * c) * E, y);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = next[i];
  }
}

// The largest of L lanes' values.
template <int L>
__device__ __forceinline__ uint32_t max_of(uint32_t v) {
  if constexpr (L >= 32) v = max(v, (uint32_t)xor_perm_i<16>((int)v));
  v = max(v, (uint32_t)xor_perm_i<8>((int)v));
  v = max(v, (uint32_t)xor_perm_i<4>((int)v));
  v = max(v, (uint32_t)xor_perm_i<2>((int)v));
  return max(v, (uint32_t)xor_perm_i<1>((int)v));
}

// A token's place in a call over the cache: D / 8 lanes take one row (a token, a head, keys or values).
template <int D>
struct RowAt {
  int tok, head, side, c;
  bool there;
  __device__ __forceinline__ explicit RowAt(const CacheSeq& a) {
    constexpr int L = D / 8;
    const int64_t u = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int per = 2 * a.heads;
    c = threadIdx.x % L;
    there = u < (int64_t)a.tokens * per;
    tok = there ? (int)(u / per) : 0;
    const int r = there ? (int)(u - (int64_t)tok * per) : 0;
    side = r >= a.heads;
    head = r - side * a.heads;
  }
};

// The scale is the row's largest magnitude over 127 and a code rint(x / scale), half to even, as quant_rows has them, bit
// for bit; a row that is not finite gets scale NaN and codes 0.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheSeq a) {
  constexpr int L = D / 8, E = BF16 ? 2 : 4;
  const RowAt<D> at(a);
  const int64_t slot = as_global(a.slot)[at.tok];
  float x[8];
  load8<BF16>(static_cast<const char*>(a.x[at.side]) + (at.tok * a.ld[at.side] + at.head * a.hs[at.side] + 8 * at.c) * E, x);
  uint32_t top = 0;                               // of the magnitudes' bits: infinities and NaN are the largest
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max_of<L>(top);
  const bool bad = top >= 0x7f800000u;
  const float s = bad ? __builtin_nanf("") : code_scale(__uint_as_float(top));
  int q[8];
  if (s >= 0x1p-100f) {
    const float rs = 1.0f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = quant_one_r(x[i], s, rs);
  } else {                                        // (1 / s may be infinite)
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = bad ? 0 : quant_one(x[i], s);
  }
  if (!at.there || !has_slot(slot, a.rows)) return;
  const CacheSide& o = a.c[at.side];
  *as_global_w(reinterpret_cast<u32x2*>(o.q + slot * o.ld + at.head * o.hs + 8 * at.c)) =
      u32x2{pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7])};
  if (at.c == 0) as_global_w(o.s)[slot * o.lds + at.head * o.hss] = s;
}

template <bool BF16, int D>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheSeq a) {
  constexpr int E = BF16 ? 2 : 4;
  const RowAt<D> at(a);
  if (!at.there) return;
  const int64_t slot = as_global(a.slot)[at.tok];
  if (!has_slot(slot, a.rows)) return;
  const CacheSide& o = a.c[at.side];
  const u32x2 q = *as_global(reinterpret_cast<const u32x2*>(o.q + slot * o.ld + at.head * o.hs + 8 * at.c));
  const float s = as_global(o.s)[slot * o.lds + at.head * o.hss];
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(q[i >> 2] >> (8 * (i & 3))) * s;
  store8<BF16>(const_cast<char*>(static_cast<const char*>(a.x[at.side])) + (at.tok * a.ld[at.side] + at.head * a.hs[at.side] + 8 * at.c) * E, x);
}

unsigned row_blocks(const CacheSeq& a) {
  const int64_t rows = 2ll * a.tokens * a.heads, per = 256 / (a.dim / 8);
  return (unsigned)((rows + per - 1) / per);
}

}  // namespace

hipError_t launch_norm_rope(const NormRope& a, hipStream_t s) {
  auto go = [&](auto kernel) { kernel<<<(unsigned)a.tokens, 256, 0, s>>>(a); };
  if (a.dim == 256)
    a.bf16 ? go(norm_rope_kernel<true, 256>) : go(norm_rope_kernel<false, 256>);
  else
    a.bf16 ? go(norm_rope_kernel<true, 128>) : go(norm_rope_kernel<false, 128>);
  return hipGetLastError();
}

hipError_t launch_cache_write(const CacheSeq& a, hipStream_t s) {
  auto go = [&](auto kernel) { kernel<<<row_blocks(a), 256, 0, s>>>(a); };
  if (a.dim == 256)
    a.bf16 ? go(cache_write_kernel<true, 256>) : go(cache_write_kernel<false, 256>);
  else
    a.bf16 ? go(cache_write_kernel<true, 128>) : go(cache_write_kernel<false, 128>);
  return hipGetLastError();
}

hipError_t launch_cache_read(const CacheSeq& a, hipStream_t s) {
  auto go = [&](auto kernel) { kernel<<<row_blocks(a), 256, 0, s>>>(a); };
  if (a.dim == 256)
    a.bf16 ? go(cache_read_kernel<true, 256>) : go(cache_read_kernel<false, 256>);
  else
    a.bf16 ? go(cache_read_kernel<true, 128>) : go(cache_read_kernel<false, 128>);
  return hipGetLastError();
}

}  // namespace qh
