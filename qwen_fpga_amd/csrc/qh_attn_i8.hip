// Causal attention with grouped heads over packed sequences whose keys and values are rows of an int8 cache, a scale for
// each row and head:  out = softmax(scale q (s_k K)^T) (s_v V)  over the keys a row sees; 0 without any.
#include <algorithm>
#include <type_traits>

#include "qh_attn_device.hpp"

namespace qh {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

namespace {

// A query row as whole numbers of two or three digits in base 256, from -128 to 127 each: its largest magnitude becomes
// `top`, an element the nearest whole number, so that  q k = (sum_i digit_i 256^i k) * unit  and the sums of digit times
// code are exact in 32 bits.  Two digits leave out 2^-16 of the row's largest element at most, three 2^-24.
template <bool BF16>
struct Row {
  static constexpr int NP = BF16 ? 2 : 3;
  static constexpr float kTop = BF16 ? 127 * 256 + 127 : 127 * 65536 + 127 * 256 + 120;   // (a rounding above it has the same digits)
  float unit, up, to;   // (to * up may overflow: a row of very small elements is moved up first)
  // top: the largest of the magnitudes' bits (infinities and NaN are above all numbers; the row is NaN then)
  __device__ __forceinline__ explicit Row(uint32_t top) {
    up = top < 0x20000000u ? 0x1p64f : 1.0f;   // below 2^-63
    const float big = __uint_as_float(top) * up;
    unit = top >= 0x7f800000u ? __builtin_nanf("") : big / kTop / up;
    to = big > 0.0f ? kTop / big : 0.0f;
  }
  // The digits of 16 elements as they were loaded, the highest first: bytes of x + 0x80 (0x8080), of which all but the
  // highest are 0x80 off.
  template <bool UP>
  __device__ __forceinline__ void digits(const u32x4 (&q)[BF16 ? 2 : 4], u32x4 (&o)[NP]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v;
        if constexpr (BF16) {
          const uint32_t two = q[i / 2][2 * (i % 2) + e / 2];
          v = __uint_as_float(e % 2 ? two & 0xffff0000u : two << 16);
        } else {
          v = __uint_as_float(q[i][e]);
        }
        if constexpr (UP) v *= up;
        if constexpr (BF16)
          y[e] = __float_as_uint(__builtin_fmaf(v, to, 12582912.0f + 128.0f));   // 1.5 * 2^23: the whole number stands in the lowest bits
        else
          y[e] = (uint32_t)((int)__builtin_rintf(v * to) + 0x8080);
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const uint32_t sel = NP - 1 - p, two = 0x0c0c0000u | (sel + 4) << 8 | sel;
        const uint32_t t = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], two), __builtin_amdgcn_perm(y[1], y[0], two), 0x05040100u);
        o[p][i] = p == 0 ? t : t ^ 0x80808080u;
      }
    }
  }
};
// 16 neighbours of a row of queries, and the largest of `top` and their magnitudes' bits (bfloat16: in each half of `top`)
template <bool BF16>
__device__ __forceinline__ void load16(const char* p, u32x4 (&q)[BF16 ? 2 : 4]) {
#pragma unroll
  for (int i = 0; i < (BF16 ? 2 : 4); ++i) q[i] = *as_global(reinterpret_cast<const u32x4*>(p) + i);
}
template <bool BF16>
__device__ __forceinline__ uint32_t larger_of(uint32_t top, const u32x4 (&q)[BF16 ? 2 : 4]) {
#pragma unroll
  for (int i = 0; i < (BF16 ? 2 : 4); ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if constexpr (BF16) {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        const u16x2 two = __builtin_bit_cast(u16x2, q[i][c] & 0x7fff7fffu);
        top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), two));
      } else {
        top = max(top, q[i][c] & 0x7fffffffu);
      }
    }
  return top;
}
// that as the bits of one float
template <bool BF16>
__device__ __forceinline__ uint32_t largest(uint32_t top) {
  return BF16 ? max(top & 0xffff0000u, top << 16) : top;
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
// Byte C of eight rows as bfloat16, rows 2 i and 2 i + 1 in dword i.  A code has eight bits, a bfloat16 as well: the upper
// half of the float is all of it.
template <int C, typename V>
__device__ __forceinline__ u32x4 widen(const V (&rows)[8]) {
  u32x4 t;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    t[i] = __builtin_amdgcn_perm(code_float<C & 3>(rows[2 * i + 1][C >> 2]), code_float<C & 3>(rows[2 * i][C >> 2]), 0x07060302u);
  return t;
}
// Lane C's value of each 16 lanes (a modifier of the instruction that takes it).
template <int C>
__device__ __forceinline__ float lane_of_16(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + C, 0xf, 0xf, true));   // row_newbcast
}
// f(0), f(1) .. f(N - 1) with constants
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// Few query rows: a workgroup takes 16 rows (tokens x query heads of one kv head) and one chunk of the keys, its four
// waves every fourth step of 32 keys.  S^T = K Q^T runs on the int8 MFMAs, a product for each digit of Q, so that K goes
// from memory into them as it is; O^T = V^T P^T on the bfloat16 ones, P (times V's scales) cut into two bfloat16 parts,
// which leave out 2^-16 of it at most (bfloat16), or three, which leave out nothing (fp32).  V's codes are widened in
// registers, 1.5 instructions an element.
// Bound by memory where there are keys for all CUs: one token behind 131070 keys, 8 / 2 heads of 256 (135 MB), 28.3 us, 4.8
// TB/s (and 8 to join).  With fewer keys by what follows one after the other: one key 7 us, 128 more for each workgroup 1.7
// us more; 16 tokens of 42000 keys together (43 MB) 16.5, 2.6 TB/s.  With many rows by the vector instructions that widen V,
// which every 16 rows do again: 1500 tokens 39 us (fp32 42).  The tiles that see the most keys start first (2000 tokens in
// fp32 68 -> 61 us).  Three instructions a code instead of 1.5 and spilled registers took twice as long; Q asked for before K,
// no loads behind the last step, chunks of a multiple of 128 keys and 384, 768 or 1024 units instead of 512 made no difference
// or took longer.
template <bool BF16, int D>
__global__ __launch_bounds__(256, 2) void attn_i8_split_kernel(const AttnI8 a) {
  constexpr int NP = Row<BF16>::NP;       // digits of Q, parts of P
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
  if (!find_unit<false, true>(a, (int)blockIdx.x / a.kv_heads, at)) return;
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
  u32x4 qv[BF16 ? 2 : 4];
  uint32_t top = 0;
  if (wave < NS) {
    load16<BF16>(static_cast<const char*>(a.q.p) + ((at.sp.start + tok) * a.q.ld + hq * a.q.hs + 64 * wave + 16 * g) * E, qv);
    top = largest<BF16>(larger_of<BF16>(0, qv));
    top = max(top, (uint32_t)xor_perm_i<16>((int)top));
    top = max(top, (uint32_t)xor_perm_i<32>((int)top));
    if (g == 0) ltop[wave][j] = top;
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < NS; ++s) top = max(top, ltop[s][j]);
  const Row<BF16> qr(top);
  if (wave < NS) {
    u32x4 v[NP];
    qr.template digits<true>(qv, v);
#pragma unroll
    for (int p = 0; p < NP; ++p) lq[wave][p][lane] = v[p];
  }
  __syncthreads();

  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNegInf, l = 0.0f;
  const float fac = qr.unit * (a.scale * kLog2e);
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
    const int64_t place = ((int64_t)at.first + at.split) * a.kv_heads + kvh;
    if (at.first < 0 || place >= (int64_t)gridDim.x) return;   // (bounds that overlap can make more units than there is place for)
    float* pp = a.part + place * part_floats(D);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < VB; c += 4)
        *as_global_w(reinterpret_cast<f32x4*>(pp + j * D + VB * (4 * g + r) + c)) =
            f32x4{acc[c][r], acc[c + 1][r], acc[c + 2][r], acc[c + 3][r]};
    if (g == 0) pp[16 * D + j] = m, pp[16 * D + 16 + j] = l;
  }
}

// Prompts: a workgroup takes 256 rows (fp32: 128; tokens x query heads of one kv head) over all the keys they see, 32
// (16) rows a wave, with the products of the form for few rows.  Keys come 8 KB of codes at a time (a stage: 32 keys of 256
// elements, 64 of 128) by global -> LDS loads, three stages ahead.  K's codes stay codes; V's are widened to bfloat16 once a
// workgroup, one stage ahead, by the wave that loaded them.  16-byte chunk c of K's row r stands at chunk c ^ (r % 16) (128
// elements: c ^ (r / 2 % 8)), so that 16 keys of one chunk lie in all banks, and chunk c of V's widened row r at
// c ^ (4 (r % 4) + 2 (r / 4 % 2)), as the transposing reads take four keys of 32 elements or eight of 16.  P (times V's scales)
// is rounded to bfloat16 once for bfloat16 (2^-8 of sum p |v|: a second part would double the products with V) and taken in
// three parts for fp32 (exact).
// A stage takes 2.1 us (bfloat16, 256 elements): its products would take 0.85 at the pipe's peak and 1.9 at the rates that
// large products of the two types reach here (2107 and 1205 T/s).  A product comes every 46 cycles of a wave's turn, not
// 32, as each fragment is read from LDS by all eight waves, and the vector instructions of the SIMD's other wave take 5
// to 7 cycles each beside them.  16345 packed tokens, 8 / 2 heads of 256: 437 us, 840 TFLOP/s (fp32 725 us).  Without turns,
// the waves of a SIMD took 5 to 8% longer; with V widened in the probabilities' turn, or the loads sent for there, longer as well.
template <bool BF16, int D>
__global__ __launch_bounds__(512, 2) void attn_i8_tile_kernel(const AttnI8 a) {
  constexpr int E = BF16 ? 2 : 4, kTile = tile_rows(BF16), NR = kTile / 8, NP = Row<BF16>::NP;
  constexpr int SK = 8192 / D, CH = D / 16, kRing = 4;    // keys of a stage; 16-byte chunks of a row of codes
  constexpr int kWide = 16384, kScales = 512;             // bytes of a stage's widened V, of its scales (K's, V's 256 bytes on)
  constexpr int LR = 64 / NR, FB = 16 * LR;               // lanes of a row; its elements in a fragment of K and Q
  constexpr int NF = D / FB, NT = D / NR, VW = BF16 ? 16 : 4;   // fragments; accumulators, their elements
  constexpr int NM = SK / NR, NK = SK / (2 * LR) / 2;     // tiles of a stage's scores; quads of scores of a lane
  constexpr int NQ = NT * VW / 4, PP = BF16 ? 1 : 3;      // quads of a lane's output; parts of P
  typedef std::conditional_t<BF16, f32x16, f32x4> fvec;
  typedef std::conditional_t<BF16, i32x16, i32x4> ivec;
  __shared__ __attribute__((aligned(256))) char lds[kRing * 16384 + 2 * kWide + 2 * kRing * kScales];
  constexpr int kRaw = kRing * 8192, kV = 2 * kRaw, kS = kV + 2 * kWide;      // V's codes, widened V, scales
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane / NR, j = lane % NR;
  const int G = a.heads / a.kv_heads;
  const int kvh = (int)blockIdx.x % a.kv_heads;
  TileUnit at;
  if (!find_tile_unit<false, kTile>(a, (int)blockIdx.x / a.kv_heads, at)) return;
  const int rows = at.sp.len * G, r0 = kTile * at.tile, w0 = r0 + NR * wave;
  auto all = [&](int row) { return keys_seen(min(row, rows - 1) / G, at.sp.len, at.kl); };
  const int piece = unit_keys(all(r0 + kTile - 1), at.nsplit), k0 = at.split * piece;   // keys are counted from here
  auto sees = [&](int row) { return all(row) - k0; };
  const int end = min(sees(r0 + kTile - 1), piece);
  if (at.split > 0 && end <= 0) return;   // (a unit of no key that the tile sees)

  // A thread's place in a stage is row tid / CH, chunk tid % CH.  (What follows from the thread's number alone is formed
  // where it is used, by tid_here: held over the loop it would not fit the registers.)
  const char* kp = static_cast<const char*>(a.k.p) + (at.ks + k0) * a.k.ld + kvh * a.k.hs;
  const char* vp = static_cast<const char*>(a.v.p) + (at.ks + k0) * a.v.ld + kvh * a.v.hs;
  const uint32_t kld = (uint32_t)a.k.ld, vld = (uint32_t)a.v.ld;   // (below 2^24: the entry point's rule)
  const uint32_t lds0 = lds_address(lds);
  const bool scales = wave < 2;   // wave 0 brings K's scales, wave 1 V's
  const float* sp = wave == 0 ? a.ks + (at.ks + k0) * a.ldks + kvh * a.hsks : a.vs + (at.ks + k0) * a.ldvs + kvh * a.hsvs;
  const int64_t sld = wave == 0 ? a.ldks : a.ldvs;
  auto stage = [&](int it) __attribute__((always_inline)) {
    const int last = end - 1 - SK * it, slot = it & (kRing - 1);   // last: the last row that is there
    const uint32_t t = tid_here(), pr = t / CH, pc = t % CH, r = min(pr, (uint32_t)last);
    const uint32_t kc = 16 * (pc ^ (D == 256 ? pr & 15 : (pr >> 1) & 7)), vc = 16 * pc;
    load_to_lds<5>(kp + (int64_t)it * SK * a.k.ld, __umul24(r, kld) + kc, lds0 + slot * 8192 + 1024 * wave);
    load_to_lds<5>(vp + (int64_t)it * SK * a.v.ld, __umul24(r, vld) + vc, lds0 + kRaw + slot * 8192 + 1024 * wave);
    if (scales)
      load_word_to_lds<5>(sp + it * SK * sld, 4 * __umul24(min(t % SK, (uint32_t)last), (uint32_t)sld),
                          lds0 + kS + (it & (2 * kRing - 1)) * kScales + 256 * wave);
  };
  const int n = seq_tiles(end, SK);
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i)
    if (i < n) stage(i);

  // Q's digits: a lane has elements FB s + 16 h .. of row j
  const int row = min(w0 + j, rows - 1), tok = row / G, hq = kvh * G + row % G;
  const int seen = min(sees(row), end);   // (a unit may end inside a stage)
  u32x4 qf[NF][NP];
  float fac;
  {
    const char* qp = static_cast<const char*>(a.q.p) + ((at.sp.start + tok) * a.q.ld + hq * a.q.hs + 16 * h) * E;
    u32x4 x[NF][BF16 ? 2 : 4];
#pragma unroll
    for (int s = 0; s < NF; ++s) load16<BF16>(qp + FB * E * s, x[s]);
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < NF; ++s) top = larger_of<BF16>(top, x[s]);
    top = largest<BF16>(top);
    if constexpr (!BF16) top = max(top, (uint32_t)xor_perm_i<16>((int)top));
    top = max(top, (uint32_t)xor_perm_i<32>((int)top));
    Row<BF16> qr(top);
    fac = qr.unit * (fabsf(a.scale) * kLog2e);
    if (a.scale < 0.0f) qr.to = -qr.to;   // (-q) k |scale|: a maximum stays one
    if (__ballot(qr.up != 1.0f) == 0) {
#pragma unroll
      for (int s = 0; s < NF; ++s) qr.template digits<false>(x[s], qf[s]);
    } else {
#pragma unroll
      for (int s = 0; s < NF; ++s) qr.template digits<true>(x[s], qf[s]);
    }
  }

  fvec acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = fvec{};
  float m = kNegInf, l = 0.0f;
  // this wave's loads of stage `it` have landed (those of the next `after` stages stay in flight)
  auto landed = [&](int after) __attribute__((always_inline)) {
    if (after >= 2) {
      if (scales) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    } else if (after == 1) {
      if (scales) asm volatile("s_waitcnt vmcnt(3)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
  };
  auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  // a lane holds four neighbours of its row from place(i) on, i below NQ
  auto place = [&](int i) { return BF16 ? 32 * (i >> 2) + 8 * (i & 3) + 4 * h : 16 * i + 4 * h; };
  constexpr int KS = 4 * LR;   // a lane's quad i of scores is of the keys KS i + 4 h ..
  // A turn at the matrix pipe: O^T += V^T P^T of stage it - 1 (not in the FIRST turn), and S^T of stage it, digit by
  // digit, if there is one (not in the LAST); between the products the thread's 16 codes of stage it of V are widened.  The
  // fragments of V and K come from LDS kAhead products before they are used: the order is the program's, which the
  // compiler left to itself does not keep (it waited for each fragment right after asking for it).
  constexpr int kAhead = 3, NV = NT * NK / 2, NKF = NF * NM;
  ivec dg[NP][NM];
  u32x4 pf[PP][NK / 2];
  auto matrix = [&](int it, auto FIRST, auto LAST) __attribute__((always_inline)) {
    constexpr bool first = decltype(FIRST)::value, last = decltype(LAST)::value;
    constexpr int i0 = first ? NV : 0, i1 = last ? NV : NV + NKF;
    const uint32_t tid = tid_here(), ln = tid & 63, h = ln / NR, j = ln % NR;
    const uint32_t vx = (ln & 15) >> 2;   // the key of four that this lane's transposing read brings
    const uint32_t kl = lds0 + (it & (kRing - 1)) * 8192 + j * D + 16 * (h ^ (D == 256 ? j & 15 : (j >> 1) & 7));
    const uint32_t vl = lds0 + kV + ((it - 1) & 1) * kWide + (4 * h + vx) * D * 2 +
                        ((BF16 ? 32 * ((ln >> 4) & 1) : 0) ^ (64 * vx + 32 * (h & 1))) + 16 * ((ln & 3) >> 1) + 8 * (ln & 1);
    u32x4 f[kAhead], codes, o;
    auto ask = [&](auto I, u32x4& to) __attribute__((always_inline)) {
      constexpr int i = I;
      if constexpr (i < NV) {
        // tile t of the elements, keys 16 kk + 4 h .., + 8 of element 32 t + lane % 32 (fp32: 32 kk + 4 h .., + 16 of
        // 16 t + lane % 16)
        constexpr int t = i / (NK / 2), kk = i % (NK / 2);
        const uint32_t p = (BF16 ? (vl ^ (64 * (t & 3))) + 256 * (t >> 2) : (vl ^ (32 * (t & 7))) + 256 * (t >> 3)) + 4 * KS * D * kk;
        union {
          i16x4 q[2];
          u32x4 v;
        } w;
        w.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<i16x4>(p));
        w.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<i16x4>(p + 2 * KS * D));
        to = w.v;
      } else {
        constexpr int s = (i - NV) / NM, t = (i - NV) % NM;
        to = *lds_at<u32x4>((kl ^ (FB * s)) + NR * D * t);
      }
    };
    if constexpr (!last) codes = *lds_at<u32x4>(lds0 + kRaw + (it & (kRing - 1)) * 8192 + 16 * tid);
    each<kAhead>([&](auto I) { ask(std::integral_constant<int, i0 + I>{}, f[(i0 + I) % kAhead]); });
    const uint32_t pr = tid / CH, pc = tid % CH;
    const uint32_t vw = lds0 + kV + (it & 1) * kWide + pr * D * 2 + ((32 * pc) ^ (64 * (pr & 3) + 32 * ((pr >> 2) & 1)));
    __builtin_amdgcn_sched_barrier(0);
    each<i1 - i0>([&](auto I) {
      constexpr int i = i0 + I;
      u32x4& x = f[i % kAhead];
      if constexpr (i < NV) {
        constexpr int t = i / (NK / 2), kk = i % (NK / 2);
#pragma unroll
        for (int p = PP - 1; p >= 0; --p) {
          if constexpr (BF16)
            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, pf[p][kk]), acc[t], 0, 0, 0);
          else
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, pf[p][kk]), acc[t], 0, 0, 0);
        }
      } else {
        constexpr int s = (i - NV) / NM, t = (i - NV) % NM;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const ivec c = s == 0 ? ivec{} : dg[p][t];
          if constexpr (BF16)
            dg[p][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, x), __builtin_bit_cast(i32x4, qf[s][p]), c, 0, 0, 0);
          else
            dg[p][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x), __builtin_bit_cast(i32x4, qf[s][p]), c, 0, 0, 0);
        }
      }
      if constexpr (i + kAhead < i1) ask(std::integral_constant<int, i + kAhead>{}, x);
      // a dword of widened codes after a product, four to a store
      constexpr int d = I - (first ? 0 : 3);
      static_assert(last || i1 - i0 >= (first ? 8 : 11), "a product for each dword");
      if constexpr (!last && d >= 0 && d < 8) {
        constexpr int b = 2 * (d % 2);
        o[d % 4] = __builtin_amdgcn_perm(code_float<b + 1>(codes[d / 2]), code_float<b>(codes[d / 2]), 0x07060302u);
        if constexpr (d % 4 == 3) *lds_at<u32x4>(vw + 16 * (d / 4)) = o;
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // The scales of a stage: each 16 lanes hold those of their scores, lane c of them score 16 q + c's in register q.
  constexpr int NSC = (NK + 3) / 4;
  float ksc[NSC], vsc[NSC];
  auto scales_of = [&](int it) __attribute__((always_inline)) {
    const uint32_t t8 = tid_here() & 63, c = t8 & 15;
    const uint32_t sl = lds0 + kS + (it & (2 * kRing - 1)) * kScales + 16 * (t8 / NR) + 4 * (KS * ((c >> 2) % NK) + (c & 3));
#pragma unroll
    for (int q = 0; q < NSC; ++q) ksc[q] = *lds_at<float>(sl + 16 * KS * q), vsc[q] = *lds_at<float>(sl + 256 + 16 * KS * q);
  };
  // P^T of a stage's keys from its scores.  PART: some row may see them only in part.
  auto softmax = [&](int it, auto PART) __attribute__((always_inline)) {
    constexpr bool part = decltype(PART)::value;
    const int h = (uint32_t)(tid_here() & 63) / NR, kb = SK * it + 4 * h;
    float st[4 * NK];
    // bfloat16: the scores without the row's unit, which the exponent's multiplication brings.  A scale of K that could take a
    // whole number beyond a float's range is taken 2^32 smaller; the rows that see its key then put unit and 2^32 to their
    // scores below.  A row's own keys decide, so that others have no influence; hardly any stage takes the branch.
    float unit = fac;
    uint64_t far[NSC] = {}, any = 0;   // the lanes that hold such a scale
    if constexpr (BF16) {
#pragma unroll
      for (int q = 0; q < NSC; ++q) {
        const bool large = !(fabsf(ksc[q]) < 0x1p96f);
        any |= far[q] = __ballot(large);
        ksc[q] = large ? ksc[q] * 0x1p-32f : ksc[q];
      }
    }
    each<NK>([&](auto I) {
      each<4>([&](auto R) {
        constexpr int i = I, r = R;
        auto d = [&](int p) { return BF16 ? dg[p][i / 4][4 * (i % 4) + r] : dg[p][i % NM][r]; };
        float x = (float)(d(0) * 256 + d(1));   // a whole number below 2^30
        // (fp32: the row's unit first, a sum of three digits times a large scale could overflow)
        if constexpr (!BF16) x = __builtin_fmaf(x, 256.0f * fac, (float)d(NP - 1) * fac);
        st[4 * i + r] = x * lane_of_16<(4 * i + r) % 16>(ksc[(4 * i + r) / 16]);
        if (part && kb + KS * i + r >= seen) st[4 * i + r] = kNegInf;
      });
    });
    if (BF16 && any != 0) {
      float by[NSC], most = 1.0f;
#pragma unroll
      for (int q = 0; q < NSC; ++q) by[q] = far[q] >> (tid_here() & 63) & 1 ? 0x1p32f : 1.0f;
      auto of = [&](auto I) { return lane_of_16<I % 16>(by[I / 16]); };
      int to = seen - kb;
      asm volatile("" : "+v"(to));   // (masks kept from the loop above would not fit the scalar registers)
      each<4 * NK>([&](auto I) { most = fmaxf(most, part && KS * (I / 4) + I % 4 >= to ? 1.0f : of(I)); });
      most = fmaxf(most, xor_perm<32>(most));
      const bool sees = most != 1.0f;
      const float first = sees ? fac : 1.0f;
      unit = sees ? 1.0f : fac;
      each<4 * NK>([&](auto I) {   // (all lanes take part in reading another's)
        const float f = of(I);
        st[I] = st[I] * first * (sees ? f : 1.0f);
      });
    }
    float mt = st[0];
#pragma unroll
    for (int r = 1; r < 4 * NK; ++r) mt = fmaxf(mt, st[r]);
    if constexpr (!BF16) mt = fmaxf(mt, xor_perm<16>(mt));
    mt = fmaxf(mt, xor_perm<32>(mt));
    if constexpr (BF16) mt = mt == kNegInf ? kNegInf : mt * unit;   // (0 times it is not it)
    const bool up = mt > m + 8.0f;                       // (as in the form for few rows)
    if (__ballot(up) != 0) {
      const float mn = up ? mt : m, al = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.0f : mn));
      m = mn;
      l *= al;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < VW; ++r) acc[t][r] *= al;
    }
    const float mu = m == kNegInf ? 0.0f : m;
    // (bfloat16: the exponent's product is not rounded, the maximum was: 2^-24 of a score of 2^31 would be too large a power.
    // A row's own maximum decides: the other rows of the wave have no influence on it)
    const bool large = fabsf(mu) >= 0x1p20f;
    if (BF16 && __ballot(large) != 0) {
      const float by = large ? unit : 1.0f;
#pragma unroll
      for (int i = 0; i < 4 * NK; ++i) st[i] *= by;
      unit = large ? 1.0f : unit;
    }
    float ps = 0.0f;
    each<NK>([&](auto I) {
      each<4>([&](auto R) {
        constexpr int i = I, r = R;
        const bool hidden = part && kb + KS * i + r >= seen;
        float p = __builtin_amdgcn_exp2f(BF16 ? __builtin_fmaf(st[4 * i + r], unit, -mu) : st[4 * i + r] - mu);
        if (BF16 && hidden) p = 0.0f;   // (a unit of 0)
        ps += p;
        const float v = p * lane_of_16<(4 * i + r) % 16>(vsc[(4 * i + r) / 16]);
        st[4 * i + r] = hidden ? 0.0f : v;   // (a hidden row's scale may be anything)
      });
    });
    l += ps;
#pragma unroll
    for (int d = 0; d < 2 * NK; ++d) {
      float x = st[2 * d], y = st[2 * d + 1];
#pragma unroll
      for (int p = 0; p < PP - 1; ++p) {   // cut: what is left is exact
        const uint32_t u0 = __float_as_uint(x), u1 = __float_as_uint(y);
        pf[p][d >> 2][d & 3] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        x -= __uint_as_float(u0 & 0xffff0000u);
        y -= __uint_as_float(u1 & 0xffff0000u);
      }
      const bf16x2 last = {(__bf16)x, (__bf16)y};
      pf[PP - 1][d >> 2][d & 3] = __builtin_bit_cast(uint32_t, last);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // The two waves of a SIMD (w and w + 4) take turns at the matrix pipe: while the one forms stage it - 1's outputs and
  // stage it's scores, the other turns its scores into probabilities, and a barrier ends each turn.  In turn t = 0, 1 .. the
  // first four waves are at the matrix pipe when t is even, with it = t / 2, and at the probabilities of stage (t - 1) / 2
  // when t is odd; the last four are one turn behind.  In its turn at the matrix pipe a wave also widens its part of stage it
  // (in turn 2 it or 2 it + 1; read from turn 2 it + 2 on; the place held stage it - 2, last read in turn 2 it - 1), sends for
  // its part of stage it + 3 (in the place of stage it - 1, whose K was last read in turn 2 it - 1; the scales, read until
  // turn 2 it, have places of their own) and waits for its part of stage it + 1 (read from turn 2 it + 2 on).
  const int second = wave >> 2;
  if (n > 0) {
    landed(min(n - 1, 2));
    barrier();
    if (second) barrier();
    const int full = max(min(sees(r0), end), 0) / SK;  // stages that every row sees whole
    auto turns = [&](int it, auto FIRST, auto PART) __attribute__((always_inline)) {
      __builtin_amdgcn_s_setprio(2);   // (before the other wave's vector instructions: 8% of a stage)
      if (it + kRing - 1 < n) stage(it + kRing - 1);
      matrix(it, FIRST, std::false_type{});
      __builtin_amdgcn_s_setprio(0);
      if (it + 1 < n) landed(min(n - 2 - it, 2));
      barrier();
      scales_of(it);
      softmax(it, PART);
      barrier();
    };
    turns(0, std::true_type{}, std::true_type{});
    int it = 1;
    for (; it < full; ++it) turns(it, std::false_type{}, std::false_type{});
    for (; it < n; ++it) turns(it, std::false_type{}, std::true_type{});
    matrix(n, std::false_type{}, std::true_type{});
    if (!second) barrier();
  }
  if constexpr (!BF16) l = l + xor_perm<16>(l);
  l = l + xor_perm<32>(l);
  if (w0 + j >= rows) return;
  auto quad = [&](int i) {
    if constexpr (BF16)
      return f32x4{acc[i >> 2][4 * (i & 3)], acc[i >> 2][4 * (i & 3) + 1], acc[i >> 2][4 * (i & 3) + 2], acc[i >> 2][4 * (i & 3) + 3]};
    else
      return acc[i];
  };
  if (at.nsplit > 1) {
    float* pp = a.part + ((size_t)at.slot * a.kv_heads + kvh) * tile_part_floats(kTile, D);
    const int rr = row - r0;
#pragma unroll
    for (int i = 0; i < NQ; ++i) *as_global_w(reinterpret_cast<f32x4*>(pp + rr * D + place(i))) = quad(i);
    if (h == 0) pp[kTile * D + rr] = m, pp[kTile * D + kTile + rr] = l;
    return;
  }
  const float inv = at.kl < 0 ? __builtin_nanf("") : seen <= 0 ? 0.0f : 1.0f / l;
  char* op = static_cast<char*>(a.out.p) + ((at.sp.start + tok) * a.out.ld + hq * a.out.hs) * E;
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const f32x4 o = quad(i) * inv;
    if constexpr (BF16)
      *as_global_w(reinterpret_cast<bf16x4*>(op + place(i) * 2)) = bf16x4{(__bf16)o[0], (__bf16)o[1], (__bf16)o[2], (__bf16)o[3]};
    else
      *as_global_w(reinterpret_cast<f32x4*>(op + place(i) * 4)) = o;
  }
}

template <bool BF16, int D>
hipError_t launch(const AttnI8& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.q_rows * (a.heads / a.kv_heads);
  if (a.tile > 0) {
    const int64_t t = seq_tiles_max(rows, a.n_seq, a.tile) * a.kv_heads;
    attn_i8_tile_kernel<BF16, D><<<(unsigned)(t + a.limit), 512, 0, s>>>(a);
    if (a.limit > 0) {
      const int64_t split = std::min<int64_t>(t, a.limit / 2);
      attn_tile_join_kernel<BF16, D><<<dim3((unsigned)split, (unsigned)std::clamp<int64_t>(1024 / split, 8, a.tile / 4)), 256, 0, s>>>(a);
    }
    return hipGetLastError();
  }
  const unsigned tiles = (unsigned)(seq_tiles_max(rows, a.n_seq, 16) * a.kv_heads);
  attn_i8_split_kernel<BF16, D><<<a.limit > 0 ? tiles + kFill : tiles, 256, 0, s>>>(a);
  // rows of a tile side by side where there are few tiles (4 tokens behind 29996 keys: 16 workgroups 23 us, 4 36), few
  // workgroups where there are many, most of which find nothing to join (16 x 128 behind 1872: 4 106 us, 1 97), and none for
  // rows that max_q does not promise
  const int64_t there = std::max<int64_t>((int64_t)a.max_q * (a.heads / a.kv_heads), 1);
  const unsigned side = (unsigned)std::min<int64_t>(there, tiles >= 256 ? 1 : tiles >= 64 ? 4 : 16);
  if (a.limit > 0) attn_join_kernel<BF16, D, true><<<dim3(tiles, side), 1024, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

AttnForm attn_i8_form(int64_t q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int dim, bool bf16) {
  const int G = heads / kv_heads;
  AttnForm f = {0, 0, 0};
  if (attn_i8_prompts(q_rows, n_seq, max_q, max_k, heads, kv_heads, dim, tile_rows(bf16), bf16)) {
    f.tile = tile_rows(bf16);
    const int64_t tiles = seq_tiles_max(q_rows * G, n_seq, f.tile) * kv_heads;
    // two workspace places a CU: the chunks are such that more are hardly ever taken
    if (max_k > min_tile_chunk(bf16)) {
      const int64_t splits = max_k / min_tile_chunk(bf16) + 1;
      f.limit = (int)std::min<int64_t>(2 * kCUs, tiles * std::min<int64_t>(splits, kMaxTileSplits));
    }
    f.bytes = (size_t)f.limit * tile_part_floats(f.tile, dim) * sizeof(float);
  } else if (max_k > kMinChunk + few_whole((q_rows * G + 15) / 16 * kv_heads)) {
    // (splitting may pay, with a second kernel: the workgroups, which know the lengths, decide)
    f.limit = 1;
    f.bytes = (size_t)(seq_tiles_max(q_rows * G, n_seq, 16) * kv_heads + kFill) * part_floats(dim) * sizeof(float);
  }
  return f;
}

hipError_t launch_attn_i8(const AttnI8& a, hipStream_t s) {
  if (a.dim == 256) return a.bf16 ? launch<true, 256>(a, s) : launch<false, 256>(a, s);
  return a.bf16 ? launch<true, 128>(a, s) : launch<false, 128>(a, s);
}

}  // namespace qh
