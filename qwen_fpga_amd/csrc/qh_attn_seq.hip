// Causal attention with grouped heads over packed sequences.  Row r of a sequence with q_len rows and k_len
// keys sees the first r + 1 + k_len - q_len keys:  out = softmax(scale q K^T) V  over those; 0 without any.
#include <algorithm>
#include <type_traits>

#include "qh_attn_device.hpp"

namespace qh {

namespace {

__device__ __forceinline__ bool non_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }

// Sets the non-finite elements of 16 bytes to zero; true if there was one.
template <bool BF16>
__device__ __forceinline__ bool zero_non_finite(u32x4& v) {
  bool bad = false;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t x = v[d];
    if constexpr (BF16) {
      const bool lo = (x & 0x7f80u) == 0x7f80u, hi = (x & 0x7f800000u) == 0x7f800000u;
      v[d] = (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
      bad |= lo || hi;
    } else {
      const bool b = (x & 0x7f800000u) == 0x7f800000u;
      v[d] = b ? 0u : x;
      bad |= b;
    }
  }
  return bad;
}

template <bool BF16>
__device__ __forceinline__ float elem(const u32x4& v, int e) {
  if constexpr (BF16)
    return __uint_as_float((e & 1) ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
  else
    return __uint_as_float(v[e]);
}

// Few query rows: a workgroup takes 16 rows (tokens x query heads of one kv head) and one chunk of the keys,
// its four waves every fourth step of KT keys.  Per step a wave forms S^T = K Q^T, so that a lane holds the
// scores of one row, and O^T = V^T P^T, whose operand P^T those registers are (the keys of a step stand in the
// order in which the lanes hold them).  Bound by K and V's way from memory: 16 sequences of 1 to 8191 keys in fp32 40 us,
// 4.2 TB/s; one of 131071 in bfloat16 51 us, 5.2 TB/s; a join 6 and 9.
template <bool BF16, int D>
__global__ __launch_bounds__(256, 2) void attn_split_kernel(const AttnSeq a) {
  constexpr int EV = BF16 ? 8 : 4;        // elements of 16 bytes
  constexpr int KT = BF16 ? 32 : 16;      // keys of a step
  constexpr int NQ = D / (4 * EV);        // 16-byte pieces of a row in a lane
  constexpr int NG = D / (16 * EV);
  constexpr int NK = BF16 ? 8 : 4;        // V rows of a lane in a step
  constexpr int NT = D / 16;
  constexpr bool kQLds = D == 256;   // the query rows in LDS where two waves a SIMD would not hold them
  __shared__ __attribute__((aligned(16))) float lacc[2][64][NT * 4 + 4];
  __shared__ u32x4 lq[kQLds ? NQ : 1][64];
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
  const int all = keys_seen(r0 / G, at.sp.len, kl);                                  // its first
  const int k0 = at.split * at.chunk, k1 = min(end, at.split + 1 == at.nsplit ? end : k0 + at.chunk);
  if (at.split > 0 && k0 >= end) return;   // (no row of the tile sees it)

  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNegInf, l = 0.0f;
  const float sc = a.scale * kLog2e;
  const int64_t kld = a.k.ld * (BF16 ? 2 : 4), vld = a.v.ld * (BF16 ? 2 : 4);
  const char* kp = static_cast<const char*>(a.k.p) + (ks * a.k.ld + kvh * a.k.hs) * (BF16 ? 2 : 4) + 16 * g;
  const char* vp = static_cast<const char*>(a.v.p) + (ks * a.v.ld + kvh * a.v.hs) * (BF16 ? 2 : 4) + 16 * j;
  u32x4 kv[KT / 16][NQ], vv[NK][NG];   // a step's rows; the next step's are loaded as soon as these are used
  auto load_k = [&](int kb) {
#pragma unroll
    for (int t = 0; t < KT / 16; ++t) {
      const char* p = kp + min(kb + 16 * t + j, k1 - 1) * kld;
#pragma unroll
      for (int s = 0; s < NQ; ++s) kv[t][s] = *as_global(reinterpret_cast<const u32x4*>(p + 64 * s));
    }
  };
  auto load_v = [&](int kb) {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const char* p = vp + min(kb + 16 * (i >> 2) + 4 * g + (i & 3), k1 - 1) * vld;
#pragma unroll
      for (int s = 0; s < NG; ++s) vv[i][s] = *as_global(reinterpret_cast<const u32x4*>(p + 256 * s));
    }
  };
  int kb = k0 + KT * wave;
  if (kb < k1) load_k(kb), load_v(kb);
  u32x4 qv[kQLds ? 1 : NQ];
  const char* qp = static_cast<const char*>(a.q.p) + ((at.sp.start + tok) * a.q.ld + hq * a.q.hs) * (BF16 ? 2 : 4) + 16 * g;
  if constexpr (kQLds) {
#pragma unroll
    for (int s = 0; s < NQ / 4; ++s)
      lq[4 * s + wave][lane] = *as_global(reinterpret_cast<const u32x4*>(qp + 64 * (4 * s + wave)));
    __syncthreads();
  } else {
#pragma unroll
    for (int s = 0; s < NQ; ++s) qv[s] = *as_global(reinterpret_cast<const u32x4*>(qp + 64 * s));
  }
  for (; kb < k1; kb += 4 * KT) {
    f32x4 st[KT / 16];
#pragma unroll
    for (int t = 0; t < KT / 16; ++t) st[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < NQ; ++s) {
      const u32x4 qs = kQLds ? lq[kQLds ? s : 0][lane] : qv[kQLds ? 0 : s];
#pragma unroll
      for (int t = 0; t < KT / 16; ++t) {
        if constexpr (BF16) {
          st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kv[t][s]), __builtin_bit_cast(bf16x8, qs),
                                                          st[t], 0, 0, 0);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kv[t][s][c]), __uint_as_float(qs[c]), st[t], 0, 0, 0);
        }
      }
    }
    load_k(min(kb + 4 * KT, k1 - 1));
    float p[NK], mx = kNegInf;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int key = kb + 16 * (i >> 2) + 4 * g + (i & 3);
      p[i] = key < min(seen, k1) ? st[i >> 2][i & 3] * sc : kNegInf;
      mx = fmaxf(mx, p[i]);
    }
    mx = fmaxf(mx, xor_perm<16>(mx));
    mx = fmaxf(mx, xor_perm<32>(mx));
    const float mn = fmaxf(m, mx), mu = mn == kNegInf ? 0.0f : mn;
    const float al = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    float ps = 0.0f;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      p[i] = __builtin_amdgcn_exp2f(p[i] - mu);
      ps += p[i];
    }
    l = l * al + ps;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[t][c] *= al;
    // A step that some row sees only in part: P is 0 in the hidden places, but 0 times an infinity or a NaN
    // is not, so those elements of V stay out of the product and go to the rows that see them afterwards.
    bool bad = false;
    if (kb + KT > min(all, k1)) {
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int s = 0; s < NG; ++s) bad |= zero_non_finite<BF16>(vv[i][s]);
    }
    if constexpr (BF16) {
      // P in two bfloat16 parts, which leave out 2^-14 of a probability at most: one part would cost 2^-8 of
      // sum p |V|, often more than the output's own rounding, and the second product's time is hidden by the loads.  The
      // first is cut, and the second moved up by p 2^-18, so that both are positive where p is: an infinity in V stays one.
      u32x4 pb, pl;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t x = __float_as_uint(p[2 * d]), y = __float_as_uint(p[2 * d + 1]);
        const bf16x2 lo = {(__bf16)__builtin_fmaf(p[2 * d], 0x1p-18f, p[2 * d] - __uint_as_float(x & 0xffff0000u)),
                           (__bf16)__builtin_fmaf(p[2 * d + 1], 0x1p-18f, p[2 * d + 1] - __uint_as_float(y & 0xffff0000u))};
        pb[d] = __builtin_amdgcn_perm(y, x, 0x07060302u);
        pl[d] = __builtin_bit_cast(uint32_t, lo);
      }
#pragma unroll
      for (int s = 0; s < NG; ++s)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          u32x4 t;   // element c of the lane's eight V rows
#pragma unroll
          for (int d = 0; d < 4; ++d)
            t[d] = __builtin_amdgcn_perm(vv[2 * d + 1][s][c >> 1], vv[2 * d][s][c >> 1], (c & 1) ? 0x07060302u : 0x05040100u);
          f32x4& o = acc[8 * s + c];
          o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t), __builtin_bit_cast(bf16x8, pl), o, 0, 0, 0);
          o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t), __builtin_bit_cast(bf16x8, pb), o, 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int s = 0; s < NG; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[4 * s + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vv[i][s][c]), p[i], acc[4 * s + c], 0, 0, 0);
    }
    load_v(min(kb + 4 * KT, k1 - 1));
    if (__ballot(bad) != 0) {
      for (int key = kb; key < min(kb + KT, k1); ++key) {
        const char* q = static_cast<const char*>(a.v.p) + ((ks + key) * a.v.ld + kvh * a.v.hs) * (BF16 ? 2 : 4);
#pragma unroll
        for (int s = 0; s < NG; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const u32x4 x = *as_global(reinterpret_cast<const u32x4*>(q + 256 * s + 16 * (4 * g + r)));
#pragma unroll
            for (int c = 0; c < EV; ++c) {
              const float e = elem<BF16>(x, c);
              if (key < seen && non_finite(e)) acc[EV * s + c][r] += e;
            }
          }
      }
    }
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
  if (at.nsplit == 1) {
    const float inv = kl < 0 ? __builtin_nanf("") : seen == 0 ? 0.0f : 1.0f / l;
    char* op = static_cast<char*>(a.out.p) + ((at.sp.start + tok) * a.out.ld + hq * a.out.hs) * (BF16 ? 2 : 4);
#pragma unroll
    for (int s = 0; s < NG; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        u32x4 o;
#pragma unroll
        for (int c = 0; c < EV; ++c) {
          const float v = acc[EV * s + c][r] * inv;
          if constexpr (BF16) {
            const uint32_t b = __builtin_bit_cast(uint16_t, (__bf16)v);
            o[c >> 1] = (c & 1) ? o[c >> 1] | b << 16 : b;
          } else {
            o[c] = __float_as_uint(v);
          }
        }
        *as_global_w(reinterpret_cast<u32x4*>(op + 256 * s + 16 * (4 * g + r))) = o;
      }
  } else {
    float* pp = a.part + (size_t)blockIdx.x * part_floats(D);   // (unit first + split, kv head)
#pragma unroll
    for (int s = 0; s < NG; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < EV; c += 4)
          *as_global_w(reinterpret_cast<f32x4*>(pp + j * D + 16 * EV * s + EV * (4 * g + r) + c)) =
              f32x4{acc[EV * s + c][r], acc[EV * s + c + 1][r], acc[EV * s + c + 2][r], acc[EV * s + c + 3][r]};
    if (g == 0) pp[16 * D + j] = m, pp[16 * D + 16 + j] = l;
  }
}

// Prompts: a workgroup takes 256 rows (fp32: 128; tokens x query heads of one kv head) over all the keys they see, 32
// (16) rows a wave.  As in the split form the products are S^T = K Q^T and O^T = V^T P^T, and P never leaves the
// registers.  K and V come 32 (16) keys at a time through a ring of LDS stages that global -> LDS loads fill three
// ahead.  16-byte chunk c of key r stands at chunk c ^ (r % 16) of K's rows (the keys of one chunk lie in all banks)
// and c ^ 4 (r % 4) of V's in bfloat16 (four keys of 32 elements do, as the transposing read takes them).  The running
// maximum moves only when a score passes it by more than 8 (a factor of 256, exact in the sums), so that the sums are
// rarely rescaled.
// bfloat16: at full load the card's power bounds it (1.85 GHz): one and two sequences of 8000 tokens and 8 heads of 256
// elements 900 and 1150 TFLOP/s, of 128 elements (the same softmax for half the products) 680 and 910.  With 64 rows a
// wave, 128 elements took 301 us for 8000 tokens, and 32 rows take 190.
// fp32: the fp32 MFMAs bound it, 89% of their cycles at 2.15 GHz; 1500 tokens 163 us in the form for few rows, 119 in
// this, of which the join takes 10 and a CU has work for 84; 512 tokens behind 7488 keys 116 TFLOP/s.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <bool BF16, int D>
__global__ __launch_bounds__(512, 2) void attn_tile_kernel(const AttnSeq a) {
  constexpr int E = BF16 ? 2 : 4, kTile = tile_rows(BF16), NR = kTile / 8;   // bytes of an element; a wave's rows
  constexpr int kKeys = BF16 ? 32 : 16, kRing = 4, CH = D * E / 16, kHalf = kKeys * D * E, kStage = 2 * kHalf;
  constexpr int NI = kHalf / 8192;               // loads of a wave for K's part of a stage (and for V's)
  constexpr int NS = D / 16, NT = D / NR;        // K fragments; accumulators, of VW elements of a lane
  constexpr int VW = BF16 ? 16 : 4, NQ = NT * VW / 4;
  typedef std::conditional_t<BF16, f32x16, f32x4> fvec;
  __shared__ __attribute__((aligned(256))) char lds[kRing * kStage];
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
  const int end = min(sees(r0 + kTile - 1), piece), wend = w0 < rows ? min(sees(w0 + NR - 1), end) : 0;
  if (at.split > 0 && end <= 0) return;   // (a unit of no key that the tile sees)
  u32x4 qf[NS];
  const uint32_t flip = a.scale < 0.0f ? (BF16 ? 0x80008000u : 0x80000000u) : 0u;   // (-q) k |scale|: a maximum stays one
  const float sc = fabsf(a.scale) * kLog2e;
  const int row = min(w0 + j, rows - 1), tok = row / G, hq = kvh * G + row % G;
  const int seen = sees(row);
  const char* qp = static_cast<const char*>(a.q.p) + ((at.sp.start + tok) * a.q.ld + hq * a.q.hs) * E + 16 * h;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    qf[s] = *as_global(reinterpret_cast<const u32x4*>(qp + 16 * (64 / NR) * s));
#pragma unroll
    for (int e = 0; e < 4; ++e) qf[s][e] ^= flip;
  }
  // a wave's loads: LDS places 64 (NI wave + i) + lane of a stage's K (V) rows
  const char* kp = static_cast<const char*>(a.k.p) + ((at.ks + k0) * a.k.ld + kvh * a.k.hs) * E;
  const char* vp = static_cast<const char*>(a.v.p) + ((at.ks + k0) * a.v.ld + kvh * a.v.hs) * E;
  const uint32_t kld = (uint32_t)a.k.ld * E, vld = (uint32_t)a.v.ld * E;   // (below 2^26: the launch's rule)
  auto k_off = [&](int i, int last) {   // last: the last row of the stage that is there
    const int place = 64 * (NI * wave + i) + lane, r = place / CH;
    return min(r, last) * kld + 16 * ((place % CH) ^ (r & 15));
  };
  auto v_off = [&](int i, int last) {
    const int place = 64 * (NI * wave + i) + lane, r = place / CH;
    return min(r, last) * vld + 16 * ((place % CH) ^ (BF16 ? (r & 3) << 2 : 0));
  };
  uint32_t ko[NI], vo[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) ko[i] = k_off(i, kKeys), vo[i] = v_off(i, kKeys);
  const uint32_t lds0 = lds_address(lds);
  auto put = [&](int it, int i, uint32_t k, uint32_t v) {
    const uint32_t base = lds0 + (it & (kRing - 1)) * kStage + (NI * wave + i) * 1024;
    load_to_lds(kp + (size_t)it * kKeys * kld, k, base);
    load_to_lds(vp + (size_t)it * kKeys * vld, v, base + kHalf);
  };
  auto stage = [&](int it) {
    const int last = end - 1 - kKeys * it;
    if (last >= kKeys - 1) {
#pragma unroll
      for (int i = 0; i < NI; ++i) put(it, i, ko[i], vo[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) put(it, i, k_off(i, last), v_off(i, last));
    }
  };
  fvec acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = fvec{};
  float m = kNegInf, l = 0.0f;
  const int n = seq_tiles(end, kKeys);
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i)
    if (i < n) stage(i);
  // places of a lane's first fragments; those of the others are these, xor-ed by the chunk and moved by whole 256 bytes
  const int vx = (lane & 15) >> 2;   // the key of four that this lane's transposing read brings
  const uint32_t kl0 = lds0 + j * D * E + 16 * (h ^ (j & 15));
  const uint32_t vl0 = lds0 + kHalf + (BF16 ? (4 * h + vx) * D * 2 + 32 * ((lane >> 4) & 1) + 16 * ((lane & 3) >> 1) + 8 * (lane & 1) + 64 * vx
                                            : 4 * h * D * 4 + 16 * j);
  // a lane holds four neighbours of its row from place(i) on, i below NQ
  auto place = [&](int i) { return BF16 ? 32 * (i >> 2) + 8 * (i & 3) + 4 * h : 64 * (i >> 2) + 16 * h + 4 * (i & 3); };
  auto wait = [&](int it) {
    // this wave's loads of the stage have landed (those of the next two stay in flight) and its reads of the stage
    // before are done; after the barrier every wave's
    if (it + 2 < n)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(4 * NI) : "memory");
    else if (it + 1 < n)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NI) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (it + kRing - 1 < n) stage(it + kRing - 1);
  };
  // kKeys keys.  PART: some row may see them only in part.
  auto step = [&](int it, auto PART) {
    constexpr bool part = decltype(PART)::value;
    const int kb = kKeys * it;
    // (opaque, so that the places are formed where they are used: held over the loop they would not fit the registers)
    uint32_t kl = kl0 + (it & (kRing - 1)) * kStage, vl = vl0 + (it & (kRing - 1)) * kStage;
    asm volatile("" : "+v"(kl), "+v"(vl));
    fvec st = {};
    if constexpr (BF16) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const u32x4 kf = *lds_at<u32x4>((kl ^ (32 * (s & 7))) + 256 * (s >> 3));
        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[s]), st, 0, 0, 0);
      }
    } else {
      fvec s2[2] = {};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const f32x4 kf = *lds_at<f32x4>((kl ^ (64 * (s & 3))) + 256 * (s >> 2));
#pragma unroll
        for (int c = 0; c < 4; ++c)
          s2[c & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[c], __uint_as_float(qf[s][c]), s2[c & 1], 0, 0, 0);
      }
      st = s2[0] + s2[1];
    }
    if constexpr (!part) {
      __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
      for (int i = 0; i < NS - 3; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, BF16 ? 1 : 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, BF16 ? 3 : 12, 0);
    }
    auto key_of = [&](int r) { return kb + 8 * (r >> 2) + 4 * h + (r & 3); };   // (fp32: four in all)
    if constexpr (part) {
#pragma unroll
      for (int r = 0; r < VW; ++r)
        if (key_of(r) >= seen) st[r] = kNegInf;
    }
    float x = st[0];
#pragma unroll
    for (int r = 1; r < VW; ++r) x = fmaxf(x, st[r]);
    if constexpr (!BF16) x = fmaxf(x, xor_perm<16>(x));
    x = fmaxf(x, xor_perm<32>(x));
    const float mt = x == kNegInf ? kNegInf : x * sc;   // (0 times it is not it)
    const bool up = mt > m + 8.0f;
    if (__ballot(up) != 0) {
      // (a row's own scores decide, so that other rows have no influence on it)
      const float mn = up ? mt : m, al = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.0f : mn));
      m = mn;
      l *= al;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < VW; ++r) acc[t][r] *= al;
    }
    const float mu = m == kNegInf ? 0.0f : m;
    float ps = 0.0f;
#pragma unroll
    for (int r = 0; r < VW; ++r) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], sc, -mu));
      st[r] = part && st[r] == kNegInf ? 0.0f : p;   // (a scale of 0)
      ps += st[r];
    }
    l += ps;
    bool bad = false;   // (see attn_split_kernel: what is not finite in V goes only to the rows that see it)
    if constexpr (BF16) {
      // P rounded to bfloat16 once, 2^-8 of sum p |V|.  Two parts, as in the form for few rows, would be half as many
      // products again: 8000 tokens 304 -> 427 us, 1024 44 -> 50.
      u32x4 pf[2];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const bf16x2 pk = {(__bf16)st[r], (__bf16)st[r + 1]};
        pf[r >> 3][(r >> 1) & 3] = __builtin_bit_cast(uint32_t, pk);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {   // keys 16 kk + 4 h .., + 8 of d = 32 t + lane % 32
          const uint32_t p = (vl ^ (64 * (t & 3))) + 256 * (t >> 2) + 16 * kk * D * 2;
          union {
            i16x4 h[2];
            u32x4 v;
          } u;
#pragma unroll
          for (int q = 0; q < 2; ++q)
            u.h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<i16x4>(p + 8 * q * D * 2));
          if constexpr (part) bad |= zero_non_finite<true>(u.v);
          acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, u.v), __builtin_bit_cast(bf16x8, pf[kk]),
                                                           acc[t], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)   // key 4 h + r
#pragma unroll
        for (int t = 0; t < NT / 4; ++t) {   // d = 64 t + 4 (lane % 16) + c
          u32x4 v = *lds_at<u32x4>(vl + r * D * 4 + 256 * t);
          if constexpr (part) bad |= zero_non_finite<false>(v);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            acc[4 * t + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[c]), st[r], acc[4 * t + c], 0, 0, 0);
        }
    }
    if constexpr (!part) {   // fragments on their way ahead of the product they are for
      constexpr int kReads = BF16 ? 2 : 1, kProducts = BF16 ? 1 : 4, kSteps = BF16 ? 2 * NT : NT;
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * kReads, 0);
#pragma unroll
      for (int i = 0; i < kSteps - 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, kProducts, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, 2 * kProducts, 0);
    }
    if constexpr (part) {
      if (__ballot(bad) != 0) {
        for (int key = kb; key < min(kb + kKeys, end); ++key) {
          const char* q = vp + (int64_t)key * a.v.ld * E;
#pragma unroll
          for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float e;
              if constexpr (BF16)
                e = (float)as_global(reinterpret_cast<const __bf16*>(q))[place(i) + c];
              else
                e = as_global(reinterpret_cast<const float*>(q))[place(i) + c];
              if (non_finite(e) && key < seen) {
                if constexpr (BF16)
                  acc[i >> 2][4 * (i & 3) + c] += e;
                else
                  acc[4 * (i >> 2) + c][i & 3] += e;
              }
            }
        }
      }
    }
  };
  const int full = max(min(sees(r0), end), 0) / kKeys;   // steps that every row sees whole
  int it = 0;
  for (; it < full; ++it) {
    wait(it);
    step(it, std::false_type{});
  }
  for (; it < n; ++it) {
    wait(it);
    if (kKeys * it < wend) step(it, std::true_type{});
  }
  if constexpr (!BF16) l = l + xor_perm<16>(l);
  l = l + xor_perm<32>(l);
  if (w0 + j >= rows) return;
  auto quad = [&](int i) {
    if constexpr (BF16)
      return f32x4{acc[i >> 2][4 * (i & 3)], acc[i >> 2][4 * (i & 3) + 1], acc[i >> 2][4 * (i & 3) + 2], acc[i >> 2][4 * (i & 3) + 3]};
    else
      return f32x4{acc[4 * (i >> 2)][i & 3], acc[4 * (i >> 2) + 1][i & 3], acc[4 * (i >> 2) + 2][i & 3], acc[4 * (i >> 2) + 3][i & 3]};
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
hipError_t launch(const AttnSeq& a, hipStream_t s) {
  if (a.tile > 0) {
    const int64_t t = seq_tiles_max((int64_t)a.q_rows * (a.heads / a.kv_heads), a.n_seq, a.tile) * a.kv_heads;
    attn_tile_kernel<BF16, D><<<(unsigned)(t + a.limit), 512, 0, s>>>(a);
    if (a.limit > 0) {
      const int64_t split = std::min<int64_t>(t, a.limit / 2);
      attn_tile_join_kernel<BF16, D><<<dim3((unsigned)split, (unsigned)std::clamp<int64_t>(1024 / split, 8, a.tile / 4)), 256, 0, s>>>(a);
    }
    return hipGetLastError();
  }
  const unsigned tiles = (unsigned)(seq_tiles_max((int64_t)a.q_rows * (a.heads / a.kv_heads), a.n_seq, 16) * a.kv_heads);
  attn_split_kernel<BF16, D><<<a.limit > 0 ? tiles + kFill : tiles, 256, 0, s>>>(a);
  if (a.limit > 0) attn_join_kernel<BF16, D><<<dim3(tiles, 4), 1024, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

AttnForm attn_seq_form(int64_t q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int dim, bool bf16) {
  const int G = heads / kv_heads;
  AttnForm f = {0, 0, 0};
  // Prompts, or many short ones that see many keys.  8 / 2 heads of 256, us in this form and in the one for few rows (calls
  // one behind another over the same operands):
  // fp32   one of 128 tokens 41 and 15, of 256 49 and 30, of 512 56 and 57, of 1500 119 and 163, of 4096 705 and 811; 128
  //        behind 1372 keys 55 and 41, behind 7872 108 and 119; 16 of 128 tokens 49 and 42, behind 7872 keys 1006 and 1379
  // bf16   one of 128 tokens 22 and 11, of 256 27 and 26, of 512 34 and 42, of 4096 109 and 371; 128 behind 1372 keys
  //        35 and 31, behind 7872 47 and 61; 16 of 128 tokens 25 and 27, behind 7872 keys 162 and 589
  const int64_t seen = q_rows * heads * std::max(max_k, 1);
  if ((int64_t)max_q * G >= (bf16 ? 1024 : 2048) || ((int64_t)max_q * G >= 128 && seen >= 5000000)) {
    f.tile = tile_rows(bf16);
    const int64_t tiles = seq_tiles_max(q_rows * G, n_seq, f.tile) * kv_heads;
    // two workspace places a CU: the chunks are such that more are hardly ever taken
    if (max_k > min_tile_chunk(bf16)) {
      const int64_t splits = max_k / min_tile_chunk(bf16) + 1;
      f.limit = (int)std::min<int64_t>(2 * kCUs, tiles * std::min<int64_t>(splits, kMaxTileSplits));
    }
    f.bytes = (size_t)f.limit * tile_part_floats(f.tile, dim) * sizeof(float);
  } else if (max_k > kMinChunk) {
    f.limit = 1;
    f.bytes = (size_t)(seq_tiles_max(q_rows * G, n_seq, 16) * kv_heads + kFill) * part_floats(dim) * sizeof(float);
  }
  return f;
}

hipError_t launch_attn_seq(const AttnSeq& a, hipStream_t s) {
  if (a.dim == 256) return a.bf16 ? launch<true, 256>(a, s) : launch<false, 256>(a, s);
  return a.bf16 ? launch<true, 128>(a, s) : launch<false, 128>(a, s);
}

}  // namespace qh
