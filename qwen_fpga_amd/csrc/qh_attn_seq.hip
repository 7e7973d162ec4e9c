// Causal attention with grouped heads over packed sequences.  Row r of a sequence with q_len rows and k_len
// keys sees the first r + 1 + k_len - q_len keys:  out = softmax(scale q K^T) V  over those; 0 without any.
#include <algorithm>
#include <type_traits>

#include "qh_seq_device.hpp"

namespace qh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_inff();

// The work of the split form.  A unit is 16 rows of a sequence (tokens x query heads of one kv head) and one chunk
// of its keys; chunks hold the same number of keys in every sequence, chosen from all sequences' keys (which only
// the device knows) so that the units come to about kFill, two workgroups for each CU: 16 sequences of 15 to 8191
// keys took 55 us with chunks cut from the longest one's length and 43 with this.
struct Unit {
  SeqSpan sp;
  int64_t ks;   // the sequence's keys: first row, number (key_len)
  int kl;
  int tile, split, nsplit, chunk;
  int first;    // unit (before kv heads) of the tile's first split
};
constexpr int kFill = 512, kMinChunk = 128;
// Unit b of the split kernel, or (JOIN) the units of row tile b.
template <bool JOIN>
__device__ __forceinline__ bool find_unit(const AttnSeq& a, int b, Unit& o) {
  const int lane = threadIdx.x & 63, G = a.heads / a.kv_heads;
  SeqSpan sp;   // of sequence s0 + lane, as of its keys and tiles
  int64_t ks;
  int kl, tiles, chunk = kMaxKeys;
  auto load = [&](int s0) {
    const int i = min(s0 + lane, a.n_seq - 1);
    ks = as_global(a.k_start)[i];
    const int n = as_global(a.k_len)[i];
    sp = seq_span(as_global(a.cu_q)[i], as_global(a.cu_q)[i + 1], a.q_rows);
    kl = key_len(ks, n, a.k_rows);
    tiles = s0 + lane < a.n_seq ? seq_tiles(sp.len * G, 16) : 0;
  };
  load(0);
  if (a.limit > 0) {
    int64_t work = (int64_t)tiles * max(kl, 0);   // keys of all row tiles
    for (int s0 = 64; s0 < a.n_seq; s0 += 64) {
      load(s0);
      work += (int64_t)tiles * max(kl, 0);
    }
    if (a.n_seq > 64) load(0);
    work = sum_all(work);
    const int64_t c = (work * a.kv_heads + kFill - 1) / kFill;
    chunk = (int)min(max((c + 63) / 64 * 64, (int64_t)kMinChunk), (int64_t)kMaxKeys);
  }
  int base = 0, first = 0;   // of the next 64 sequences: tiles (JOIN) or units, units
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    if (s0 > 0) load(s0);
    const int ns = max(seq_tiles(max(kl, 0), chunk), 1);
    const int iu = sum_up_to(tiles * ns), it = sum_up_to(tiles);
    const uint64_t past = __ballot(base + (JOIN ? it : iu) > b);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      o.sp = {of(sp.start), of(sp.len)};
      o.ks = (int64_t)((uint64_t)(uint32_t)of((int)(ks >> 32)) << 32 | (uint32_t)of((int)ks));
      o.kl = of(kl);
      o.nsplit = of(ns);
      o.chunk = chunk;
      const int in = b - base - (of(JOIN ? it : iu) - of(JOIN ? tiles : tiles * ns));
      o.tile = JOIN ? in : in / o.nsplit;
      o.split = JOIN ? 0 : in - o.tile * o.nsplit;
      o.first = first + of(iu) - of(tiles * ns) + o.tile * o.nsplit;
      return o.tile >= 0 && o.tile < of(tiles);   // (bounds that overlap can make more tiles than an int counts)
    }
    base += __builtin_amdgcn_readlane(JOIN ? it : iu, 63);
    first += __builtin_amdgcn_readlane(iu, 63);
  }
  return false;
}

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

// Partials of a unit and kv head: 16 rows of D sums, their maxima, their sums of exponentials.
constexpr size_t part_floats(int D) { return 16 * D + 32; }

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

// Joins the splits of a tile's rows, every fourth row in a workgroup: sixteen waves take every sixteenth split, four
// in flight, each with a running maximum of its own.
template <bool BF16, int D>
__global__ __launch_bounds__(1024) void attn_join_kernel(const AttnSeq a) {
  constexpr int W = D / 64, NW = 16, U = 4;   // elements of a lane; waves; splits in flight
  typedef float vec __attribute__((ext_vector_type(W)));
  __shared__ vec lo[NW][64];
  __shared__ float lsum[NW], lmax[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.heads / a.kv_heads;
  const int kvh = (int)blockIdx.x % a.kv_heads;
  Unit at;
  if (!find_unit<true>(a, (int)blockIdx.x / a.kv_heads, at)) return;
  if (at.nsplit == 1) return;   // written by the split kernel
  if (at.first < 0 || (int64_t)(at.first + at.nsplit) * a.kv_heads > (int64_t)gridDim.x + kFill) return;   // past its grid
  const int rows = at.sp.len * G;
  const size_t step = part_floats(D) * a.kv_heads;
  const float* pp = a.part + ((size_t)at.first * a.kv_heads + kvh) * part_floats(D);
  for (int j = blockIdx.y; j < 16 && 16 * at.tile + j < rows; j += 4) {
    const int row = 16 * at.tile + j, tok = row / G, hq = kvh * G + row % G;
    const int seen = keys_seen(tok, at.sp.len, at.kl);
    const int ns = min(seq_tiles(seen, at.chunk), at.nsplit);   // splits that this row sees (the rest hold no key of it)
    float m = kNegInf, l = 0.0f;
    vec acc = {};
    for (int s0 = wave; s0 < ns; s0 += NW * U) {
      float mv[U], lv[U], mn = m;
      vec av[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* p = pp + min(s0 + NW * u, ns - 1) * step;
        mv[u] = s0 + NW * u < ns ? as_global(p)[16 * D + j] : kNegInf;
        lv[u] = as_global(p)[16 * D + 16 + j];
        av[u] = *as_global(reinterpret_cast<const vec*>(p + j * D) + lane);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, mv[u]);
      const float mu = mn == kNegInf ? 0.0f : mn, al = __builtin_amdgcn_exp2f(m - mu);
      m = mn;
      l *= al;
      acc *= al;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = __builtin_amdgcn_exp2f(mv[u] - mu);
        if (s0 + NW * u < ns) l += e * lv[u], acc += e * av[u];
      }
    }
    __syncthreads();   // the row before has been read
    lo[wave][lane] = acc;
    if (lane == 0) lsum[wave] = l, lmax[wave] = m;
    __syncthreads();
    if (wave != 0) continue;
    m = kNegInf;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, lmax[w]);
    const float mu = m == kNegInf ? 0.0f : m;
    acc = vec{};
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float e = __builtin_amdgcn_exp2f(lmax[w] - mu);
      acc += e * lo[w][lane];
      l += e * lsum[w];
    }
    acc *= seen == 0 ? 0.0f : 1.0f / l;
    const int64_t to = (at.sp.start + tok) * a.out.ld + hq * a.out.hs + W * lane;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if constexpr (BF16)
        as_global_w(static_cast<__bf16*>(a.out.p))[to + w] = (__bf16)acc[w];
      else
        as_global_w(static_cast<float*>(a.out.p))[to + w] = acc[w];
    }
  }
}

// The work of the form for prompts.  A tile is TILE rows of a sequence (tokens x query heads of one kv head) over all
// the keys they see.  The keys of a tile that sees more than `chunk` of them are split into equal units of at most a
// chunk, whose sums meet in the workspace; the other tiles are a unit each.  The chunk is the keys of all tiles over 192
// CUs, in fp32 over those that half a unit a tile leaves if they are more (but at least min_tile_chunk, and a 64th of
// the sequence).  The units then come to at most about one for each CU: a few more would start when the first ones end
// and take as long again (1500 tokens of fp32: 250 units 121 us, 294 units 165).  fp32, whose units are long, over 192
// and over what is left: 512 tokens behind 7488 keys 347 and 279 us, 1500 tokens 122 and 116; bfloat16 66 and 72 for
// 512 behind 7488, 53 and 61 for 256 behind 7744 (more units to join).  Units start in order, unit b on XCD b % 8: so
// the longest come first, and neighbours are about equally long.
// The workgroups of an XCD then walk the keys of one head side by side and find them in its L2: shares cut to the same
// length anywhere in the tiles missed it for 38% of the reads and took 15% longer for 16k packed tokens (8 / 2 heads of
// 256).  (Each pair of figures here is of one run, the two timed side by side; runs differ by some per cent.)
// Split and whole, bfloat16, calls one behind another over the same operands: one sequence of 512 tokens 34 and 36 us, 1024
// 43 and 54, 1500 47 and 70, 4096 109 and 163, 8000 290 and 316; 128 tokens behind 7872 keys 47 and 298; where there are
// tiles for all CUs without it, splitting costs a little: two of 8000 tokens 454 and 435, those 16k 361 and 354.
constexpr int kCUs = 256, kMaxTileSplits = 64;
constexpr int min_tile_chunk(bool bf16) { return bf16 ? 256 : 128; }
struct TileUnit {
  SeqSpan sp;
  int64_t ks;
  int kl, tile, split, nsplit;
  int slot;   // of the unit (JOIN: of the tile's first) among the split tiles' units
  int all;    // JOIN: split tiles
};
// Unit b, or (JOIN) split tile b and the number of split tiles.
template <bool JOIN, int TILE>
__device__ __forceinline__ bool find_tile_unit(const AttnSeq& a, int b, TileUnit& o) {
  const int lane = threadIdx.x & 63, G = a.heads / a.kv_heads;
  SeqSpan sp;   // of sequence s0 + lane, as of its keys and tiles
  int64_t ks;
  int kl, nt;
  auto load = [&](int s0) {
    const int i = min(s0 + lane, a.n_seq - 1);
    ks = as_global(a.k_start)[i];
    const int n = as_global(a.k_len)[i];
    sp = seq_span(as_global(a.cu_q)[i], as_global(a.cu_q)[i + 1], a.q_rows);
    kl = key_len(ks, n, a.k_rows);
    nt = s0 + lane < a.n_seq ? seq_tiles(sp.len * G, TILE) : 0;
  };
  auto work = [&]() -> int64_t {   // keys that the sequence's tiles see, about
    const int64_t k = max(kl, 0), past = max(k - sp.len, (int64_t)0);
    return nt * past + (nt + 1) * min(k, (int64_t)sp.len) / 2;
  };
  load(0);
  int64_t all = nt > 0 ? work() : 0, tiles = nt;
  for (int s0 = 64; s0 < a.n_seq; s0 += 64) {
    load(s0);
    all += nt > 0 ? work() : 0;
    tiles += nt;
  }
  if (a.n_seq > 64) load(0);
  all = sum_all(all);
  tiles = sum_all(tiles);
  const int fill = kCUs - (a.bf16 ? kCUs / 4 : (int)min(tiles * a.kv_heads / 2, (int64_t)kCUs / 4));
  const int64_t share = max((all * a.kv_heads + fill - 1) / fill, (int64_t)min_tile_chunk(a.bf16));
  int base = 0, slots = 0;   // of the next 64 sequences: units (JOIN: split tiles), the split tiles' units
  bool found = false;
  for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
    if (s0 > 0) load(s0);
    // the longest first: place `rank` is this lane's sequence's
    const int n = min(a.n_seq - s0, 64), len = nt > 0 ? max(kl, 0) : -1;
    int rank = lane < n ? 0 : lane;
    for (int l = 0; l < n; ++l) {
      const int other = __builtin_amdgcn_readlane(len, l);
      rank += lane < n && (other > len || (other == len && l < lane));
    }
    const int64_t c64 = (max(share, (int64_t)(max(kl, 0) / kMaxTileSplits + 1)) + 31) / 32 * 32;
    const int chunk = a.limit > 0 ? (int)min(c64, (int64_t)kMaxKeys) : kMaxKeys;
    const int big = tiles_past(sp.len, kl, G, TILE, nt, chunk);
    int su = 2 * big;   // units of the split tiles
    for (int k = 2, c; __ballot((c = tiles_past(sp.len, kl, G, TILE, nt, (int64_t)k * chunk)) > 0) != 0; ++k) su += c;
    // in the order of the places
    auto place = [&](int v) { return __builtin_amdgcn_ds_permute(4 * rank, v); };
    const int who = place(lane), su_at = place(su), big_at = place(big), past = sum_up_to(su_at);
    const bool split = su_at > 0 && ((int64_t)slots + past) * a.kv_heads <= a.limit;   // (there is place for it)
    const int m = JOIN ? (split ? big_at : 0) : place(nt) + (split ? su_at - big_at : 0), upto = base + sum_up_to(m);
    const uint64_t reach = __ballot(upto > b);
    if (!found && reach != 0) {
      const int r = __builtin_ctzll(reach), l = __builtin_amdgcn_readlane(who, r);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      auto at = [&](int v) { return __builtin_amdgcn_readlane(v, r); };
      const int t = of(nt), step = of(chunk), to = at(split);
      o.sp = {of(sp.start), of(sp.len)};
      o.ks = (int64_t)((uint64_t)(uint32_t)of((int)(ks >> 32)) << 32 | (uint32_t)of((int)ks));
      o.kl = of(kl);
      int in = b - at(upto) + at(m), before = 0, first = slots + at(past) - at(su_at);   // tiles of more than k splits; the units of those
      for (int k = to ? seq_tiles(o.kl, step) : 1;; --k) {
        const int c = k > 1 ? tiles_past(o.sp.len, o.kl, G, TILE, t, (int64_t)(k - 1) * step) - before : t - before;   // of k
        const int u = JOIN ? c : c * k;
        if (in < u || k == 1) {
          o.nsplit = k;
          o.split = k > 1 && !JOIN ? in / c : 0;
          in -= o.split * c;
          o.tile = t - 1 - before - in;
          o.slot = first + in * k + o.split;
          found = o.tile >= 0 && o.tile < t;
          break;
        }
        in -= u;
        before += c;
        first += c * k;
      }
      if (!JOIN) return found;
    }
    base = __builtin_amdgcn_readlane(upto, 63);
    slots = min(slots + __builtin_amdgcn_readlane(past, 63), kMaxKeys);   // (past the limit: none has place any more)
  }
  o.all = base;
  return found;
}
// Keys of each of a tile's `nsplit` units when its last row sees `end`.
__device__ __forceinline__ int unit_keys(int end, int nsplit) { return nsplit == 1 ? kMaxKeys : (seq_tiles(end, nsplit) + 31) / 32 * 32; }
constexpr int tile_rows(bool bf16) { return bf16 ? 256 : 128; }
constexpr size_t tile_part_floats(int tile, int D) { return (size_t)tile * (D + 2); }

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

// Joins the units of the split tiles: a wave takes a row at a time, eight units in flight.  The grid is gridDim.y
// workgroups for each of the most tiles that there can be; where less than half of those are there, and few workgroups
// each, they share all of it (16k packed tokens, 36 of 256 tiles: 38 -> 23 us).
template <bool BF16, int D>
__global__ __launch_bounds__(256) void attn_tile_join_kernel(const AttnSeq a) {
  constexpr int tile = tile_rows(BF16), W = D / 64, U = 8;   // elements of a lane; units in flight
  typedef float vec __attribute__((ext_vector_type(W)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.heads / a.kv_heads;
  TileUnit at;
  int t = blockIdx.x, y = blockIdx.y, ny = gridDim.y;
  find_tile_unit<true, tile>(a, t / a.kv_heads, at);
  const int all = at.all * a.kv_heads;
  if (all > 0 && 2 * all <= (int)gridDim.x && ny <= tile / 16) {
    ny = min((int)(gridDim.x * gridDim.y) / all, tile / 4);
    const int b = blockIdx.x * gridDim.y + blockIdx.y;
    t = b / ny, y = b % ny;
    if (t < all) find_tile_unit<true, tile>(a, t / a.kv_heads, at);
  }
  if (t >= all) return;
  const int kvh = t % a.kv_heads, rows = min(at.sp.len * G - tile * at.tile, tile);
  const int piece = unit_keys(keys_seen((tile * at.tile + rows - 1) / G, at.sp.len, at.kl), at.nsplit);
  const size_t step = tile_part_floats(tile, D) * a.kv_heads;
  const float* pp = a.part + ((size_t)at.slot * a.kv_heads + kvh) * tile_part_floats(tile, D);
  for (int j = 4 * y + wave; j < rows; j += 4 * ny) {
    const int row = tile * at.tile + j, tok = row / G, hq = kvh * G + row % G;
    const int ns = min(seq_tiles(keys_seen(tok, at.sp.len, at.kl), piece), at.nsplit);   // units that this row sees
    float m = kNegInf, l = 0.0f;
    vec acc = {};
    for (int s0 = 0; s0 < ns; s0 += U) {
      float mv[U], lv[U], mn = m;
      vec av[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* p = pp + min(s0 + u, ns - 1) * step;
        mv[u] = s0 + u < ns ? as_global(p)[tile * D + j] : kNegInf;
        lv[u] = as_global(p)[tile * D + tile + j];
        av[u] = *as_global(reinterpret_cast<const vec*>(p + j * D) + lane);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) mn = fmaxf(mn, mv[u]);
      const float mu = mn == kNegInf ? 0.0f : mn, al = __builtin_amdgcn_exp2f(m - mu);
      m = mn;
      l *= al;
      acc *= al;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = __builtin_amdgcn_exp2f(mv[u] - mu);
        if (s0 + u < ns) l += e * lv[u], acc += e * av[u];
      }
    }
    acc *= ns == 0 ? 0.0f : 1.0f / l;
    const int64_t to = (at.sp.start + tok) * a.out.ld + hq * a.out.hs + W * lane;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if constexpr (BF16)
        as_global_w(static_cast<__bf16*>(a.out.p))[to + w] = (__bf16)acc[w];
      else
        as_global_w(static_cast<float*>(a.out.p))[to + w] = acc[w];
    }
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
