// Causal attention with grouped heads over packed sequences.  Row r of a sequence with q_len rows and k_len
// keys sees the first r + 1 + k_len - q_len keys:  out = softmax(scale q K^T) V  over those; 0 without any.
#include "qh_seq_device.hpp"

namespace qh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_inff();

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

// Splits' partials: for each (row tile, kv head, split) 16 rows of D sums, 16 maxima, 16 sums of exponentials.
__device__ __forceinline__ size_t part_at(size_t unit, int split, int nsplit, int D) {
  return (unit * nsplit + split) * (size_t)(16 * D + 32);
}

// Few query rows: a workgroup takes 16 rows (tokens x query heads of one kv head) and one chunk of the keys,
// its four waves every fourth step of KT keys.  Per step a wave forms S^T = K Q^T, so that a lane holds the
// scores of one row, and O^T = V^T P^T, whose operand P^T those registers are (the keys of a step stand in the
// order in which the lanes hold them).
template <bool BF16, int D>
__global__ __launch_bounds__(256) void attn_split_kernel(const AttnSeq a) {
  constexpr int EV = BF16 ? 8 : 4;        // elements of 16 bytes
  constexpr int KT = BF16 ? 32 : 16;      // keys of a step
  constexpr int NQ = D / (4 * EV);        // 16-byte pieces of a row in a lane
  constexpr int NG = D / (16 * EV);
  constexpr int NK = BF16 ? 8 : 4;        // V rows of a lane in a step
  constexpr int NT = D / 16;
  __shared__ __attribute__((aligned(16))) float lacc[2][64][NT * 4 + 4];
  __shared__ float lm[2][16], ll[2][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  const int G = a.heads / a.kv_heads;
  const int unit = blockIdx.x, kvh = unit % a.kv_heads, split = blockIdx.y;
  TileAt at;
  if (!find_tile(a.cu_q, a.n_seq, a.q_rows, G, 16, unit / a.kv_heads, at)) return;
  const int64_t ks = as_global(a.k_start)[at.seq];
  const int kl = key_len(ks, as_global(a.k_len)[at.seq], a.k_rows);
  const int rows = at.sp.len * G, r0 = 16 * at.tile;
  const int row = min(r0 + j, rows - 1), tok = row / G, hq = kvh * G + row % G;
  const int seen = keys_seen(tok, at.sp.len, kl);                                    // this lane's row
  const int end = keys_seen(min(r0 + 15, rows - 1) / G, at.sp.len, kl);              // the tile's last row
  const int all = keys_seen(r0 / G, at.sp.len, kl);                                  // its first
  const int k0 = split * a.chunk, k1 = min(end, a.nsplit == split + 1 ? end : k0 + a.chunk);
  if (split > 0 && k0 >= end) return;

  u32x4 qv[NQ];
  const char* qp = static_cast<const char*>(a.q.p) + ((at.sp.start + tok) * a.q.ld + hq * a.q.hs) * (BF16 ? 2 : 4) + 16 * g;
#pragma unroll
  for (int s = 0; s < NQ; ++s) qv[s] = *as_global(reinterpret_cast<const u32x4*>(qp + 64 * s));
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNegInf, l = 0.0f;
  const float sc = a.scale * kLog2e;
  const int64_t kld = a.k.ld * (BF16 ? 2 : 4), vld = a.v.ld * (BF16 ? 2 : 4);
  const char* kp = static_cast<const char*>(a.k.p) + (ks * a.k.ld + kvh * a.k.hs) * (BF16 ? 2 : 4) + 16 * g;
  const char* vp = static_cast<const char*>(a.v.p) + (ks * a.v.ld + kvh * a.v.hs) * (BF16 ? 2 : 4) + 16 * j;
  for (int kb = k0 + KT * wave; kb < k1; kb += 4 * KT) {
    u32x4 kv[KT / 16][NQ], vv[NK][NG];
#pragma unroll
    for (int t = 0; t < KT / 16; ++t) {
      const char* p = kp + min(kb + 16 * t + j, k1 - 1) * kld;
#pragma unroll
      for (int s = 0; s < NQ; ++s) kv[t][s] = *as_global(reinterpret_cast<const u32x4*>(p + 64 * s));
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const char* p = vp + min(kb + 16 * (i >> 2) + 4 * g + (i & 3), k1 - 1) * vld;
#pragma unroll
      for (int s = 0; s < NG; ++s) vv[i][s] = *as_global(reinterpret_cast<const u32x4*>(p + 256 * s));
    }
    f32x4 st[KT / 16];
#pragma unroll
    for (int t = 0; t < KT / 16; ++t) {
      st[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < NQ; ++s) {
        if constexpr (BF16) {
          st[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kv[t][s]), __builtin_bit_cast(bf16x8, qv[s]),
                                                          st[t], 0, 0, 0);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kv[t][s][c]), __uint_as_float(qv[s][c]), st[t], 0, 0, 0);
        }
      }
    }
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
      bf16x8 pb;
#pragma unroll
      for (int i = 0; i < 8; ++i) pb[i] = (__bf16)p[i];
#pragma unroll
      for (int s = 0; s < NG; ++s)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          u32x4 t;   // element c of the lane's eight V rows
#pragma unroll
          for (int d = 0; d < 4; ++d)
            t[d] = __builtin_amdgcn_perm(vv[2 * d + 1][s][c >> 1], vv[2 * d][s][c >> 1], (c & 1) ? 0x07060302u : 0x05040100u);
          acc[8 * s + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t), pb, acc[8 * s + c], 0, 0, 0);
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
  if (a.nsplit == 1) {
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
    float* pp = a.part + part_at(unit, split, a.nsplit, D);
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

// Joins the splits of one row: four waves take every fourth split.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnSeq a) {
  constexpr int W = D / 64;   // elements of a lane
  __shared__ float lo[4][D], lsum[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.heads / a.kv_heads;
  const int unit = blockIdx.x, kvh = unit % a.kv_heads, j = blockIdx.y;
  TileAt at;
  if (!find_tile(a.cu_q, a.n_seq, a.q_rows, G, 16, unit / a.kv_heads, at)) return;
  const int kl = key_len(as_global(a.k_start)[at.seq], as_global(a.k_len)[at.seq], a.k_rows);
  const int rows = at.sp.len * G, row = 16 * at.tile + j;
  if (row >= rows) return;
  const int tok = row / G, hq = kvh * G + row % G;
  const int seen = keys_seen(tok, at.sp.len, kl);
  const int ns = min(seq_tiles(seen, a.chunk), a.nsplit);   // splits that this row sees (the rest hold no key of it)
  const float* pp = a.part + part_at(unit, 0, a.nsplit, D);
  constexpr size_t kStep = 16 * D + 32;
  float m = kNegInf;
  for (int s = lane; s < ns; s += 64) m = fmaxf(m, as_global(pp)[s * kStep + 16 * D + j]);
  m = xor_max<64>(m);
  const float mu = m == kNegInf ? 0.0f : m;
  float acc[W] = {}, l = 0.0f;
  for (int s = wave; s < ns; s += 4) {
    const float e = __builtin_amdgcn_exp2f(as_global(pp)[s * kStep + 16 * D + j] - mu);
    l += e * as_global(pp)[s * kStep + 16 * D + 16 + j];
#pragma unroll
    for (int w = 0; w < W; ++w) acc[w] += e * as_global(pp)[s * kStep + j * D + 64 * w + lane];
  }
#pragma unroll
  for (int w = 0; w < W; ++w) lo[wave][64 * w + lane] = acc[w];
  if (lane == 0) lsum[wave] = l;
  __syncthreads();
  if ((int)threadIdx.x >= D) return;
  l = (lsum[0] + lsum[1]) + (lsum[2] + lsum[3]);
  const float inv = kl < 0 ? __builtin_nanf("") : seen == 0 ? 0.0f : 1.0f / l;
  const int d = threadIdx.x;
  const float v = ((lo[0][d] + lo[1][d]) + (lo[2][d] + lo[3][d])) * inv;
  const int64_t o = (at.sp.start + tok) * a.out.ld + hq * a.out.hs + d;
  if constexpr (BF16)
    as_global_w(static_cast<__bf16*>(a.out.p))[o] = (__bf16)v;
  else
    as_global_w(static_cast<float*>(a.out.p))[o] = v;
}

template <bool BF16, int D>
hipError_t launch(const AttnSeq& a, hipStream_t s) {
  const unsigned units = (unsigned)(seq_tiles_max((int64_t)a.q_rows * (a.heads / a.kv_heads), a.n_seq, 16) * a.kv_heads);
  attn_split_kernel<BF16, D><<<dim3(units, a.nsplit), 256, 0, s>>>(a);
  if (a.nsplit > 1) attn_join_kernel<BF16, D><<<dim3(units, 16), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

AttnSplit attn_seq_split(int64_t q_rows, int n_seq, int max_k, int heads, int kv_heads, int dim) {
  const int64_t units = seq_tiles_max(q_rows * (heads / kv_heads), n_seq, 16) * kv_heads;
  const int64_t want = units >= 1024 ? 1 : 2048 / (units > 0 ? units : 1);   // splits that fill the chip
  int64_t chunk = (max_k + want - 1) / want;
  chunk = (chunk + 127) / 128 * 128;
  if (chunk < 128) chunk = 128;
  const int64_t n = max_k > chunk ? (max_k + chunk - 1) / chunk : 1;
  return {(int)chunk, (int)n, n > 1 ? (size_t)(units * n) * (16 * dim + 32) * sizeof(float) : 0};
}

hipError_t launch_attn_seq(const AttnSeq& a, hipStream_t s) {
  if (a.dim == 256) return a.bf16 ? launch<true, 256>(a, s) : launch<false, 256>(a, s);
  return a.bf16 ? launch<true, 128>(a, s) : launch<false, 128>(a, s);
}

}  // namespace qh
