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
// angle pos * theta^(-2 i / rot).  WPT waves take a token, D / 8 lanes a head's row; the first rows are on their way while
// a wave forms the token's angles, counted in turns in 64 bits (a float holds an angle of 131071 to 2^-7), and a lane reads
// the other element of a pair from the lane that holds it.  Bound by memory: 16345 tokens of 8 and 2 heads of 256 in bfloat16
// (168 MB) 36.7 us, 4.6 TB/s; with two rows of a wave on their way at once 39.9, with five (fewer waves) 45; 1500 in fp32
// (31 MB) 9.1 us; one token 3.3, a launch.
template <bool BF16, int D, int WPT>
__global__ __launch_bounds__(256) void norm_rope_kernel(const NormRope a) {
  constexpr int L = D / 8, E = BF16 ? 2 : 4, NG = 64 / L;   // rows of a wave at a time
  __shared__ __attribute__((aligned(16))) float cs[4][2][D / 2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int tok = ((int)blockIdx.x * 4 + wave) / WPT, part = ((int)blockIdx.x * 4 + wave) % WPT;
  if (tok >= a.tokens) return;
  const int c = lane % L, grp = lane / L, n = a.heads + a.kv_heads, half = a.rot / 2;
  const char* qp = static_cast<const char*>(a.q.p) + (tok * a.q.ld + 8 * c) * E;
  const char* kp = static_cast<const char*>(a.k.p) + (tok * a.k.ld + 8 * c) * E;
  char* qo = static_cast<char*>(a.qo.p) + (tok * a.qo.ld + 8 * c) * E;
  char* ko = static_cast<char*>(a.ko.p) + (tok * a.ko.ld + 8 * c) * E;
  float x[8];
  auto load = [&](int r) {
    if (r < n) load8<BF16>(r < a.heads ? qp + r * a.q.hs * E : kp + (r - a.heads) * a.k.hs * E, x);
  };
  load(part * NG + grp);
  for (int i = lane; i < half; i += 64) {
    const double t = (double)as_global(a.pos)[tok] * a.turns[i];
    float si, co;
    sincospif(2.0f * (float)(t - __builtin_rint(t)), &si, &co);
    cs[wave][0][i] = co;
    cs[wave][1][i] = si;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  const int hc = half / 8;                        // pieces of eight in half a rotated part
  const bool lower = c < hc, turned = c < 2 * hc;
  float co[8] = {}, si[8] = {};
  if (turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      co[i] = cs[wave][0][8 * (lower ? c : c - hc) + i];
      si[i] = cs[wave][1][8 * (lower ? c : c - hc) + i];
      si[i] = lower ? -si[i] : si[i];
    }
  }
  const int other = turned ? (lower ? lane + hc : lane - hc) : lane;
  float qw[8], kw[8];
  load8<false>(reinterpret_cast<const char*>(a.qw + 8 * c), qw);
  load8<false>(reinterpret_cast<const char*>(a.kw + 8 * c), kw);
  for (int r0 = part * NG; r0 < n; r0 += WPT * NG) {
    const int r = r0 + grp;
    const bool q = r < a.heads;
    float ss = 0.0f, y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
    ss = xor_sum<L>(ss);
    const float inv = 1.0f / __builtin_sqrtf(ss / (float)D + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] * inv * (1.0f + (q ? qw[i] : kw[i]));
    load(r + WPT * NG);
    if (hc > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float o = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * other, __float_as_int(y[i])));
        y[i] = turned ? __builtin_fmaf(o, si[i], y[i] * co[i]) : y[i];
      }
    }
    if (r < n) store8<BF16>(q ? qo + r * a.qo.hs * E : ko + (r - a.heads) * a.ko.hs * E, y);
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

// A call over the cache: D / 8 lanes take R of a token's rows (heads of keys, then of values), all of them on their
// way at once, for one look at the token's slot: four where there are many rows, one where there are few.
template <int D, int R>
struct RowsAt {
  int tok, r0, n, c;     // rows r0 .. n - 1 of 2 * heads
  bool there;
  __device__ __forceinline__ explicit RowsAt(const CacheSeq& a) {
    constexpr int L = D / 8;
    const int64_t u = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int per = (2 * a.heads + R - 1) / R;
    there = u < (int64_t)a.tokens * per;
    tok = there ? (int)(u / per) : 0;
    r0 = there ? (int)(u - (int64_t)tok * per) * R : 0;
    n = min(2 * a.heads, r0 + R);
    c = threadIdx.x % L;
  }
};

// The scale is the row's largest magnitude over 127 and a code rint(x / scale), half to even, as quant_rows has them, bit
// for bit; a row that is not finite gets scale NaN and codes 0.  Bound by memory: 16345 bfloat16 tokens of 2 heads of 256
// (51 MB) 15.1 us, 3.4 TB/s; 35 tokens 3.1, a launch.
template <bool BF16, int D, int R>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheSeq a) {
  constexpr int L = D / 8, E = BF16 ? 2 : 4;
  const RowsAt<D, R> at(a);
  const int64_t slot = as_global(a.slot)[at.tok];
  float x[R][8];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int r = min(at.r0 + u, at.n - 1), side = r >= a.heads;
    load8<BF16>(static_cast<const char*>(a.x[side]) + (at.tok * a.ld[side] + (r - side * a.heads) * a.hs[side] + 8 * at.c) * E, x[u]);
  }
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int r = at.r0 + u, side = r >= a.heads, head = r - side * a.heads;
    uint32_t top = 0;                             // of the magnitudes' bits: infinities and NaN are the largest
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[u][i]) & 0x7fffffffu);
    top = max_of<L>(top);
    const bool bad = top >= 0x7f800000u;
    const float s = bad ? __builtin_nanf("") : code_scale(__uint_as_float(top));
    int q[8];
    if (s >= 0x1p-100f) {
      const float rs = 1.0f / s;
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = quant_one_r(x[u][i], s, rs);
    } else {                                      // (1 / s may be infinite)
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = bad ? 0 : quant_one(x[u][i], s);
    }
    if (!at.there || r >= at.n || !has_slot(slot, a.rows)) continue;
    const CacheSide& o = a.c[side];
    *as_global_w(reinterpret_cast<u32x2*>(o.q + slot * o.ld + head * o.hs + 8 * at.c)) =
        u32x2{pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7])};
    if (at.c == 0) as_global_w(o.s)[slot * o.lds + head * o.hss] = s;
  }
}

// Code times scale in fp32, rounded once more to bfloat16.  Bound by memory: 60001 bfloat16 tokens of 2 heads of 256 (185
// MB) 35.2 us, 5.2 TB/s; 641 fp32 ones 3.8, a launch.
template <bool BF16, int D, int R>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheSeq a) {
  constexpr int E = BF16 ? 2 : 4;
  const RowsAt<D, R> at(a);
  if (!at.there) return;
  const int64_t slot = as_global(a.slot)[at.tok];
  if (!has_slot(slot, a.rows)) return;
  u32x2 q[R];
  float s[R];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int r = min(at.r0 + u, at.n - 1), side = r >= a.heads, head = r - side * a.heads;
    const CacheSide& o = a.c[side];
    q[u] = *as_global(reinterpret_cast<const u32x2*>(o.q + slot * o.ld + head * o.hs + 8 * at.c));
    s[u] = as_global(o.s)[slot * o.lds + head * o.hss];
  }
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int r = at.r0 + u, side = r >= a.heads;
    if (r >= at.n) return;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(q[u][i >> 2] >> (8 * (i & 3))) * s[u];
    char* to = const_cast<char*>(static_cast<const char*>(a.x[side]));
    store8<BF16>(to + (at.tok * a.ld[side] + (r - side * a.heads) * a.hs[side] + 8 * at.c) * E, x);
  }
}

// One row at a time up to 16384 of them (2048 workgroups of heads of 256): 35 tokens of 2 heads written in 3.1 us and in
// 4.0 four at a time, 641 read in 3.3 and 3.9; 16345 written in 16.6 and 15.2, 60001 read in 62 and 35.
template <typename One, typename Four>
hipError_t launch_rows(const CacheSeq& a, One one, Four four, hipStream_t s) {
  const bool few = 2ll * a.tokens * a.heads <= 16384;
  const int64_t units = (int64_t)a.tokens * (few ? 2 * a.heads : (2 * a.heads + 3) / 4), per = 256 / (a.dim / 8);
  const unsigned n = (unsigned)((units + per - 1) / per);
  if (few)
    one<<<n, 256, 0, s>>>(a);
  else
    four<<<n, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm_rope(const NormRope& a, hipStream_t s) {
  const bool single = norm_rope_waves(a.tokens, (int64_t)a.heads + a.kv_heads, a.dim, a.bf16) == 1;
  auto go = [&](auto one, auto four) {
    if (single)
      one<<<(unsigned)((a.tokens + 3) / 4), 256, 0, s>>>(a);
    else
      four<<<(unsigned)a.tokens, 256, 0, s>>>(a);
  };
  if (a.dim == 256)
    a.bf16 ? go(norm_rope_kernel<true, 256, 1>, norm_rope_kernel<true, 256, 4>)
           : go(norm_rope_kernel<false, 256, 1>, norm_rope_kernel<false, 256, 4>);
  else
    a.bf16 ? go(norm_rope_kernel<true, 128, 1>, norm_rope_kernel<true, 128, 4>)
           : go(norm_rope_kernel<false, 128, 1>, norm_rope_kernel<false, 128, 4>);
  return hipGetLastError();
}

hipError_t launch_cache_write(const CacheSeq& a, hipStream_t s) {
  auto go = [&](auto one, auto four) { return launch_rows(a, one, four, s); };
  if (a.dim == 256)
    return a.bf16 ? go(cache_write_kernel<true, 256, 1>, cache_write_kernel<true, 256, 4>)
                  : go(cache_write_kernel<false, 256, 1>, cache_write_kernel<false, 256, 4>);
  return a.bf16 ? go(cache_write_kernel<true, 128, 1>, cache_write_kernel<true, 128, 4>)
                : go(cache_write_kernel<false, 128, 1>, cache_write_kernel<false, 128, 4>);
}

hipError_t launch_cache_read(const CacheSeq& a, hipStream_t s) {
  auto go = [&](auto one, auto four) { return launch_rows(a, one, four, s); };
  if (a.dim == 256)
    return a.bf16 ? go(cache_read_kernel<true, 256, 1>, cache_read_kernel<true, 256, 4>)
                  : go(cache_read_kernel<false, 256, 1>, cache_read_kernel<false, 256, 4>);
  return a.bf16 ? go(cache_read_kernel<true, 128, 1>, cache_read_kernel<true, 128, 4>)
                : go(cache_read_kernel<false, 128, 1>, cache_read_kernel<false, 128, 4>);
}

}  // namespace qh
