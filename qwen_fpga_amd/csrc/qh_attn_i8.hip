// Causal attention with grouped heads over packed sequences whose keys and values are rows of an int8 cache, a scale for
// each row and head:  out = softmax(scale q (s_k K)^T) (s_v V)  over the keys a row sees; 0 without any.
#include <algorithm>
#include <type_traits>

#include "qh_attn_device.hpp"

namespace qh {

typedef int i32x4 __attribute__((ext_vector_type(4)));

namespace {

// A query row as whole numbers: the row's largest magnitude becomes `top` = 2 or 3 digits of eight bits (the upper one
// 127), an element the nearest whole number, so that  q k = (sum_i digits_i 256^i k) * unit  and the sums of digit times
// code are exact in 32 bits.  Two digits leave out 2^-16 of the row's largest element at most, three 2^-24.
constexpr int kTop2 = 127 * 256 + 127, kTop3 = kTop2 * 256 + 127;
// digit i of four whole numbers, as bytes
__device__ __forceinline__ uint32_t bytes4(int a, int b, int c, int d) {
  const uint32_t lo = __builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x0c0c0400u), hi = __builtin_amdgcn_perm((uint32_t)d, (uint32_t)c, 0x04000c0cu);
  return lo | hi;
}

// Byte B of x, signed, as a float, in one instruction (the compiler takes three).
template <int B>
__device__ __forceinline__ uint32_t code_float(uint32_t x) {
  uint32_t f;
  if constexpr (B == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(x));
  if constexpr (B == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(x));
  if constexpr (B == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(x));
  if constexpr (B == 3) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(x));
  return f;
}
// Byte C of eight rows as bfloat16, rows 2 i and 2 i + 1 in dword i.  A code has eight bits, a bfloat16 as well: the upper half of
// the float is all of it.
template <int C, typename V>
__device__ __forceinline__ u32x4 widen(const V (&rows)[8]) {
  u32x4 t;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    t[i] = __builtin_amdgcn_perm(code_float<C & 3>(rows[2 * i + 1][C >> 2]), code_float<C & 3>(rows[2 * i][C >> 2]), 0x07060302u);
  return t;
}
// f(0), f(1) .. f(N - 1) with constants
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// Few query rows: a workgroup takes 16 rows (tokens x query heads of one kv head) and one chunk of the keys, its four
// waves every fourth step of 32 keys.  S^T = K Q^T runs on the int8 MFMAs, a product for each digit of Q, so that K goes
// from memory into them as it is; O^T = V^T P^T on the bfloat16 ones, P (times V's scales) cut into two bfloat16 parts, which leave
// out 2^-16 of it at most (bfloat16), or three, which leave out nothing (fp32).  V's codes are widened in registers, 1.5 instructions an element.
template <bool BF16, int D>
__global__ __launch_bounds__(256, 2) void attn_i8_split_kernel(const AttnI8 a) {
  constexpr int NP = BF16 ? 2 : 3;        // digits of Q, parts of P
  constexpr int NS = D / 64;              // 16-byte pieces of a K row in a lane
  constexpr int VB = D / 16;              // bytes of a V row in a lane
  constexpr int NT = D / 16, E = BF16 ? 2 : 4;
  typedef uint32_t vrow __attribute__((ext_vector_type(VB / 4)));
  __shared__ __attribute__((aligned(16))) float lacc[2][64][NT * 4 + 4];
  __shared__ u32x4 lq[NS][NP][64];
  __shared__ uint32_t ltop[4][16];
  __shared__ __attribute__((aligned(16))) float lsc[4][64];
  __shared__ float lm[2][16], ll[2][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int G = a.heads / a.kv_heads;
  const int kvh = (int)blockIdx.x % a.kv_heads;
  Unit at;
  if (!find_unit<false>(a, (int)blockIdx.x / a.kv_heads, at)) return;
  const int64_t ks = at.ks;
  const int kl = at.kl;
  const int rows = at.sp.len * G, r0 = 16 * at.tile;
  const int row = min(r0 + j, rows - 1), tok = row / G, hq = kvh * G + row % G;
  const int seen = keys_seen(tok, at.sp.len, kl);                                    // this lane's row
  const int end = keys_seen(min(r0 + 15, rows - 1) / G, at.sp.len, kl);              // the tile's last row
  const int k0 = at.split * at.chunk, k1 = min(end, at.split + 1 == at.nsplit ? end : k0 + at.chunk);
  if (at.split > 0 && k0 >= end) return;   // (no row of the tile sees it)

  // A step's rows by 32-bit offsets from its first key (the strides are below 2^24: the entry point's rule); the next
  // step's are loaded as soon as these are used.
  const uint32_t kld = (uint32_t)a.k.ld, vld = (uint32_t)a.v.ld, sld = (uint32_t)(lane < 32 ? a.ldks : a.ldvs);
  const char* kp = static_cast<const char*>(a.k.p) + ks * a.k.ld + kvh * a.k.hs;
  const char* vp = static_cast<const char*>(a.v.p) + ks * a.v.ld + kvh * a.v.hs;
  const float *ksp = a.ks + ks * a.ldks + kvh * a.hsks, *vsp = a.vs + ks * a.ldvs + kvh * a.hsvs;
  u32x4 kv[2][NS];
  vrow vv[8];
  float sc = 0.0f;   // of key lane % 32 of the step: K's scale, in the upper half V's
  auto load_k = [&](int kb) {   // kb: the same for the wave, below k1
    const int last = k1 - 1 - kb;
    const float* sp = lane < 32 ? ksp + kb * a.ldks : vsp + kb * a.ldvs;
    sc = as_global(sp)[__umul24(min(lane & 31, last), sld)];
    const char* p = kp + kb * a.k.ld;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t o = __umul24(min(16 * t + j, last), kld) + 16 * g;
#pragma unroll
      for (int s = 0; s < NS; ++s) kv[t][s] = *as_global(reinterpret_cast<const u32x4*>(p + o + 64 * s));
    }
  };
  auto load_v = [&](int kb) {
    const int last = k1 - 1 - kb;
    const char* p = vp + kb * a.v.ld;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      vv[i] = *as_global(reinterpret_cast<const vrow*>(p + (uint32_t)(__umul24(min(16 * (i >> 2) + 4 * g + (i & 3), last), vld) + VB * j)));
  };
  int kb = k0 + 32 * wave;
  if (kb < k1) load_k(kb), load_v(kb);

  // Q's digits: wave s forms those of elements 64 s + 16 g .. of row j
  float qv[16];
  uint32_t top = 0;   // of the magnitudes' bits: infinities and NaN are the largest
  if (wave < NS) {
    const char* qp = static_cast<const char*>(a.q.p) + ((at.sp.start + tok) * a.q.ld + hq * a.q.hs + 64 * wave + 16 * g) * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const u32x4 v = *as_global(reinterpret_cast<const u32x4*>(qp) + i);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (BF16)
          qv[8 * i + 2 * c] = __uint_as_float(v[c] << 16), qv[8 * i + 2 * c + 1] = __uint_as_float(v[c] & 0xffff0000u);
        else
          qv[4 * i + c] = __uint_as_float(v[c]);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(qv[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)xor_perm_i<16>((int)top));
    top = max(top, (uint32_t)xor_perm_i<32>((int)top));
    if (g == 0) ltop[wave][j] = top;
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < NS; ++s) top = max(top, ltop[s][j]);
  constexpr int kTop = BF16 ? kTop2 : kTop3;
  // (a row of very small elements is moved up first: kTop / its largest would overflow)
  const float up = top < 0x20000000u ? 0x1p64f : 1.0f, big = __uint_as_float(top) * up;   // 0x20000000: 2^-63
  const float unit = top >= 0x7f800000u ? __builtin_nanf("") : big / (float)kTop / up, to = big > 0.0f ? (float)kTop / big : 0.0f;
  if (wave < NS) {
    int x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = (int)__builtin_rintf(fminf(fmaxf(qv[i] * up * to, -(float)kTop), (float)kTop));
#pragma unroll
    for (int p = NP - 1; p >= 0; --p) {   // the lowest digit first; what is left is a multiple of 256
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = bytes4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      lq[wave][p][lane] = v;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = (x[i] + 128) >> 8;
    }
  }
  __syncthreads();

  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNegInf, l = 0.0f;
  const float fac = unit * (a.scale * kLog2e);
  const int lim = min(seen, k1);
  for (; kb < k1; kb += 128) {
    lsc[wave][lane] = sc;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    i32x4 dg[NP][2] = {};
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const u32x4 qs = lq[s][p][lane];
#pragma unroll
        for (int t = 0; t < 2; ++t)
          dg[p][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, kv[t][s]), __builtin_bit_cast(i32x4, qs), dg[p][t], 0, 0, 0);
      }
    load_k(min(kb + 128, k1 - 1));
    float p[8], mx = kNegInf;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 ksc = *as_lds(reinterpret_cast<const f32x4*>(&lsc[wave][16 * t + 4 * g]));
      settle(ksc);   // (read by all lanes, not under the condition below)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = kb + 16 * t + 4 * g + r;
        float x = (float)(dg[0][t][r] * 256 + dg[1][t][r]);   // below 2^30
        if constexpr (!BF16) x = __builtin_fmaf(x, 256.0f, (float)dg[NP - 1][t][r]);
        p[4 * t + r] = key < lim ? x * fac * ksc[r] : kNegInf;
        mx = fmaxf(mx, p[4 * t + r]);
      }
    }
    mx = fmaxf(mx, xor_perm<16>(mx));
    mx = fmaxf(mx, xor_perm<32>(mx));
    // the running maximum moves only when a score passes it by more than 8 (a factor of 256, exact in the sums); a row's
    // own scores decide, so that other rows have no influence on it
    const bool up = mx > m + 8.0f;
    if (__ballot(up) != 0) {
      const float mn = up ? mx : m, al = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.0f : mn));
      m = mn;
      l *= al;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[t][c] *= al;
    }
    const float mu = m == kNegInf ? 0.0f : m;
    float ps = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 vsc = *as_lds(reinterpret_cast<const f32x4*>(&lsc[wave][32 + 16 * t + 4 * g]));
      settle(vsc);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(p[4 * t + r] - mu);
        ps += e;
        p[4 * t + r] = kb + 16 * t + 4 * g + r < lim ? e * vsc[r] : 0.0f;   // (a hidden row's scale may be anything)
      }
    }
    l += ps;
    u32x4 pb[NP];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      float x = p[2 * d], y = p[2 * d + 1];
#pragma unroll
      for (int i = 0; i < NP - 1; ++i) {   // cut: what is left is exact
        const uint32_t u = __float_as_uint(x), w = __float_as_uint(y);
        pb[i][d] = __builtin_amdgcn_perm(w, u, 0x07060302u);
        x -= __uint_as_float(u & 0xffff0000u);
        y -= __uint_as_float(w & 0xffff0000u);
      }
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      const bf16x2 last = {(__bf16)x, (__bf16)y};
      pb[NP - 1][d] = __builtin_bit_cast(uint32_t, last);
    }
    __builtin_amdgcn_sched_barrier(0);   // (the codes are widened where they are used: all at once they would not fit the registers)
    each<VB>([&](auto C) {
      const u32x4 t = widen<C>(vv);
#pragma unroll
      for (int i = NP - 1; i >= 0; --i)
        acc[C] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t), __builtin_bit_cast(bf16x8, pb[i]), acc[C], 0, 0, 0);
    });
    __builtin_amdgcn_sched_group_barrier(0x2, 24, 0);
#pragma unroll
    for (int c = 0; c < VB - 2; ++c) {
      __builtin_amdgcn_sched_group_barrier(0x8, NP, 0);
      __builtin_amdgcn_sched_group_barrier(0x2, 12, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, 2 * NP, 0);
    __builtin_amdgcn_sched_barrier(0);
    load_v(min(kb + 128, k1 - 1));
  }
  l = l + xor_perm<16>(l);
  l = l + xor_perm<32>(l);
  // the four waves' sums meet in pairs: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    __syncthreads();
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < NT; ++t) *as_lds_w(reinterpret_cast<f32x4*>(&lacc[wave - half][lane][4 * t])) = acc[t];
      if (g == 0) lm[wave - half][j] = m, ll[wave - half][j] = l;
    }
    __syncthreads();
    if (wave < half) {
      const float mo = lm[wave][j], lo = ll[wave][j], M = fmaxf(m, mo), mu = M == kNegInf ? 0.0f : M;
      const float e0 = __builtin_amdgcn_exp2f(m - mu), e1 = __builtin_amdgcn_exp2f(mo - mu);
      m = M;
      l = l * e0 + lo * e1;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4 o = *as_lds(reinterpret_cast<const f32x4*>(&lacc[wave][lane][4 * t]));
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[t][c] = acc[t][c] * e0 + o[c] * e1;
      }
    }
  }
  if (wave != 0 || r0 + j >= rows) return;
  // element VB (4 g + r) + c of the row is acc[c][r]
  if (at.nsplit == 1) {
    const float inv = kl < 0 ? __builtin_nanf("") : seen == 0 ? 0.0f : 1.0f / l;
    char* op = static_cast<char*>(a.out.p) + ((at.sp.start + tok) * a.out.ld + hq * a.out.hs) * E;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < VB; c += 16 / E) {
        char* q = op + (VB * (4 * g + r) + c) * E;
        if constexpr (BF16) {
          bf16x8 o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = (__bf16)(acc[c + i][r] * inv);
          *as_global_w(reinterpret_cast<bf16x8*>(q)) = o;
        } else {
          *as_global_w(reinterpret_cast<f32x4*>(q)) = f32x4{acc[c][r], acc[c + 1][r], acc[c + 2][r], acc[c + 3][r]} * inv;
        }
      }
  } else {
    float* pp = a.part + (size_t)blockIdx.x * part_floats(D);   // (unit first + split, kv head)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < VB; c += 4)
        *as_global_w(reinterpret_cast<f32x4*>(pp + j * D + VB * (4 * g + r) + c)) =
            f32x4{acc[c][r], acc[c + 1][r], acc[c + 2][r], acc[c + 3][r]};
    if (g == 0) pp[16 * D + j] = m, pp[16 * D + 16 + j] = l;
  }
}

template <bool BF16, int D>
hipError_t launch(const AttnI8& a, hipStream_t s) {
  const unsigned tiles = (unsigned)(seq_tiles_max((int64_t)a.q_rows * (a.heads / a.kv_heads), a.n_seq, 16) * a.kv_heads);
  attn_i8_split_kernel<BF16, D><<<a.limit > 0 ? tiles + kFill : tiles, 256, 0, s>>>(a);
  if (a.limit > 0) attn_join_kernel<BF16, D><<<dim3(tiles, 4), 1024, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

AttnForm attn_i8_form(int64_t q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int dim, bool bf16) {
  AttnForm f = {0, 0, 0};
  if (max_k > kMinChunk) {
    f.limit = 1;
    f.bytes = (size_t)(seq_tiles_max(q_rows * (heads / kv_heads), n_seq, 16) * kv_heads + kFill) * part_floats(dim) * sizeof(float);
  }
  return f;
}

hipError_t launch_attn_i8(const AttnI8& a, hipStream_t s) {
  if (a.dim == 256) return a.bf16 ? launch<true, 256>(a, s) : launch<false, 256>(a, s);
  return a.bf16 ? launch<true, 128>(a, s) : launch<false, 128>(a, s);
}

}  // namespace qh
