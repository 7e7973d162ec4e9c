// The gated delta rule over packed sequences.  A token of one head, with S [128][128] (k-major), does
//   S = exp(g) S;  d = beta (v - S^T k);  S = S + k d^T;  out = S^T q
// Short sequences run token by token (delta_step_kernel).  Long ones in chunks of 64 tokens: with c_t the sum of
// g up to token t of the chunk and S the state before it, unrolling the recursion gives
//   d_t + sum_{j<t} A_tj d_j = beta_t (v_t - e^{c_t} S^T k_t),   A_tj = beta_t e^{c_t - c_j} (k_t . k_j)
//   out_t = e^{c_t} S^T q_t + sum_{j<=t} P_tj d_j,               P_tj = e^{c_t - c_j} (q_t . k_j)
//   S'    = e^{c_63} S + sum_t e^{c_63 - c_t} k_t d_t^T
// so with T = (I + A)^-1 a chunk is five matrix products.  T and P do not depend on the state: one launch forms
// them for all chunks at once (delta_chunk_kernel), a second follows the state through them (delta_scan_kernel).
// c is summed and subtracted in 64 bits: a factor e^{c_t - c_j} near 1 may stand between sums in the thousands.
// All products are fp32 (v_mfma_f32_16x16x4_f32: row l % 16 and column l % 16 of lane l, depth l / 16; a lane ends
// with rows 4 (l / 16) .. + 3 of column l % 16).  What a lane holds of a result is what it has to bring as the
// next product's right operand, four depths in four instructions, so results chain without a shuffle.
#include "qh_seq_device.hpp"

namespace qh {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace {

constexpr int kD = 128;
constexpr int kC = 64;                       // tokens of a chunk
// A chunk's and head's part of the workspace, in floats: T and P as ten 16 x 16 tiles each (lower triangle,
// tile (i, j) at i (i + 1) / 2 + j; lane l's four values: row l % 16, columns 4 (l / 16) ..), the row factors
// {beta, beta e^c, e^c, e^{c_63 - c}}, and whether an input is not finite.
constexpr int kTiles = 10, kOffP = kTiles * 256, kOffRow = 2 * kTiles * 256, kOffFlag = kOffRow + 4 * kC,
              kChunkFloats = kOffFlag + 64;
__device__ __forceinline__ constexpr int tri(int i, int j) { return i * (i + 1) / 2 + j; }
// A chunk's slot: one per started 64 rows and sequence, so sequences need no count of those before them.
// (floor(x) + floor(y) <= floor(x + y), so a sequence's last slot lies below the next one's first.)
__device__ __forceinline__ size_t chunk_at(const DeltaSeq& a, int seq, int start, int c, int h) {
  return ((size_t)(start / kC + seq + c) * a.heads + h) * kChunkFloats;
}

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

template <bool BF16>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t at) {
  if constexpr (BF16) {
    const bf16x4 t = *as_global(reinterpret_cast<const bf16x4*>(static_cast<const __bf16*>(p) + at));
    return f32x4{(float)t[0], (float)t[1], (float)t[2], (float)t[3]};
  } else {
    return *as_global(reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at));
  }
}
template <bool BF16>
__device__ __forceinline__ f32x2 load2(const void* p, int64_t at) {
  if constexpr (BF16) {
    const bf16x2 t = *as_global(reinterpret_cast<const bf16x2*>(static_cast<const __bf16*>(p) + at));
    return f32x2{(float)t[0], (float)t[1]};
  } else {
    return *as_global(reinterpret_cast<const f32x2*>(static_cast<const float*>(p) + at));
  }
}
__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ f32x4 mfma4(f32x4 x, f32x4 y, f32x4 c) {   // four depths
#pragma unroll
  for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], y[r], c, 0, 0, 0);
  return c;
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

// T, P and the row factors of one chunk and head.
template <bool BF16>
__global__ __launch_bounds__(256) void delta_chunk_kernel(const DeltaSeq a) {
  constexpr int LD = kC + 4;
  __shared__ __attribute__((aligned(16))) float al[kC * LD], tl[kC * LD];   // A; T
  __shared__ double cs[kC];
  __shared__ float bt[kC];
  __shared__ int bad_in[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g4 = 4 * (lane >> 4), j = lane & 15;
  TileAt at;
  if (!find_tile(a.cu, a.n_seq, a.tokens, 1, kC, blockIdx.x, at)) return;
  const int h = blockIdx.y, hk = h / (a.heads / a.k_heads);
  const int t0 = at.sp.start + kC * at.tile, n = min(kC, at.sp.start + at.sp.len - t0);   // n >= 1 tokens
  float* ws = a.ws + chunk_at(a, at.seq, at.sp.start, at.tile, h);
  bool bad = false;
  if (wave == 0) {
    // a log decay below -1e5 is 0 as a factor like any below -104, and finite in the sums
    float gv = 0.0f, be = 0.0f;
    if (lane < n) {
      gv = as_global(a.g)[(t0 + lane) * a.ldg + h];
      be = as_global(a.beta)[(t0 + lane) * a.ldb + h];
      if (gv < -1e5f) gv = -1e5f;
      bad = !finite(gv) || !finite(be);
    }
    double c = gv;
#pragma unroll
    for (int d = 1; d < kC; d *= 2) {
      const double t = __shfl_up(c, d);
      if (lane >= d) c += t;
    }
    const double last = __shfl(c, kC - 1);
    cs[lane] = c;
    bt[lane] = be;
    const float ec = dev_expf((float)c);
    *as_global_w(reinterpret_cast<f32x4*>(ws + kOffRow) + lane) = f32x4{be, be * ec, ec, dev_expf((float)(last - c))};
  }
  // wave's share of the rows: all of q, k (the tiles below) and v are looked at for values that are not finite
  for (int u = threadIdx.x; u < kC * kD / 4; u += 256) {
    const int64_t r = t0 + min(u >> 5, n - 1);
    const f32x4 x = load4<BF16>(a.v.p, r * a.v.ld + h * a.v.hs + 4 * (u & 31));
    bad |= !finite(x[0]) || !finite(x[1]) || !finite(x[2]) || !finite(x[3]);
  }
  __syncthreads();
  // the ten tiles (i, jj), dealt to the waves
  constexpr int kDeal[4][3] = {{tri(3, 0), tri(3, 1), tri(3, 2)}, {tri(2, 0), tri(2, 1), tri(2, 2)}, {tri(3, 3), tri(1, 0), -1}, {tri(1, 1), tri(0, 0), -1}};
#pragma unroll
  for (int u = 0; u < 3; ++u) {
    int tile = -1;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (wave == w) tile = kDeal[w][u];
    if (tile < 0) break;
    const int i = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, jj = tile - tri(i, 0);
    const int64_t rt = t0 + min(16 * i + j, n - 1), rj = t0 + min(16 * jj + j, n - 1);
    f32x4 G = {0.0f, 0.0f, 0.0f, 0.0f}, P = G;   // row (depth of the later products): j; column: t
#pragma unroll
    for (int s = 0; s < kD / 16; ++s) {
      const f32x4 kj = load4<BF16>(a.k.p, rj * a.k.ld + hk * a.k.hs + 16 * s + g4), kt = load4<BF16>(a.k.p, rt * a.k.ld + hk * a.k.hs + 16 * s + g4),
                  qt = load4<BF16>(a.q.p, rt * a.q.ld + hk * a.q.hs + 16 * s + g4);
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= !finite(kj[e]) || !finite(kt[e]) || !finite(qt[e]);
      G = mfma4(kj, kt, G);
      P = mfma4(kj, qt, P);
    }
    const int t = 16 * i + j;
    const double ct = cs[t];
    const float be = bt[t];
    f32x4 av;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int jr = 16 * jj + g4 + r;
      const float e = jr <= t ? dev_expf((float)(ct - cs[jr])) : 0.0f;
      av[r] = jr < t ? be * e * G[r] : 0.0f;
      P[r] = jr <= t ? e * P[r] : 0.0f;
    }
    *as_lds_w(reinterpret_cast<f32x4*>(al + t * LD + 16 * jj + g4)) = av;
    *as_global_w(reinterpret_cast<f32x4*>(ws + kOffP + tile * 256) + lane) = P;
  }
  const uint64_t any = __ballot(bad);
  if (lane == 0) bad_in[wave] = any != 0;
  __syncthreads();
  if (threadIdx.x == 0) ws[kOffFlag] = (bad_in[0] | bad_in[1] | bad_in[2] | bad_in[3]) ? 1.0f : 0.0f;
  // the diagonal tiles' inverses: lane's column j of T_ii, row after row
  {
    const float* ad = al + 16 * wave * LD + 16 * wave;
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float s = r == j ? 1.0f : 0.0f;
#pragma unroll
      for (int k = 0; k < r; ++k) s = __builtin_fmaf(-as_lds(ad)[r * LD + k], x[k], s);
      x[r] = s;
    }
    if (lane < 16)
#pragma unroll
      for (int r = 0; r < 16; ++r) tl[(16 * wave + r) * LD + 16 * wave + j] = x[r];
  }
  __syncthreads();
  // the tiles below them, a column of tiles per wave: T_ij = -T_ii sum_{k=j}^{i-1} A_ik T_kj
  f32x4 tc[4];   // T_kj, rows g4 .. of column j
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    if (wave != c) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) tc[c][r] = as_lds(tl)[(16 * c + g4 + r) * LD + 16 * c + j];
#pragma unroll
    for (int i = c + 1; i < 4; ++i) {
      f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = c; k < i; ++k) z = mfma4(*as_lds(reinterpret_cast<const f32x4*>(al + (16 * i + j) * LD + 16 * k + g4)), tc[k], z);
      f32x4 m = mfma4(*as_lds(reinterpret_cast<const f32x4*>(tl + (16 * i + j) * LD + 16 * i + g4)), z, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        tc[i][r] = -m[r];
        tl[(16 * i + g4 + r) * LD + 16 * c + j] = -m[r];
      }
    }
  }
  __syncthreads();
  for (int u = wave; u < kTiles; u += 4) {
    const int i = u < 1 ? 0 : u < 3 ? 1 : u < 6 ? 2 : 3, c = u - tri(i, 0);
    *as_global_w(reinterpret_cast<f32x4*>(ws + u * 256) + lane) =
        *as_lds(reinterpret_cast<const f32x4*>(tl + (16 * i + j) * LD + 16 * c + g4));
  }
}

// The state's way through the chunks: a workgroup takes one sequence, one head and 16 of its columns.  Every wave
// holds the whole 128 x 16 slice (s[w][c], lane l: rows 32 w + 8 (l / 16) + 2 r + c of column l % 16), wave w
// works on the chunk's tokens 16 w .. + 15 and updates the rows 32 w .. + 31.
template <bool BF16>
__global__ __launch_bounds__(256) void delta_scan_kernel(const DeltaSeq a) {
  __shared__ f32x4 rl[4][64], dl[4][64], el[4][64], sl[4][2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, j = lane & 15;
  // the eight slices of a head on one of the eight XCDs, whose L2 then holds the head's q, k, T and P
  const int b = blockIdx.x, u = (b & 7) + 8 * (b >> 6), slice = (b >> 3) & 7;
  if (u >= a.n_seq * a.heads) return;
  const int h = u % a.heads, seq = u / a.heads, hk = h / (a.heads / a.k_heads);
  const SeqSpan sp = seq_span(as_global(a.cu)[seq], as_global(a.cu)[seq + 1], a.tokens);
  if (sp.len == 0) return;
  const int col = 16 * slice + j;
  float* Sp = a.S + ((size_t)seq * a.heads + h) * kD * kD + col;
  f32x4 s[4][2];
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[w][c][r] = as_global(Sp)[(32 * w + 8 * g + 2 * r + c) * kD];

  f32x4 kf[4][2], qf[4][2], tf[4], pf[4], row[4];   // operands of one chunk, each reloaded as soon as it is used
  f32x2 kt[4][4];
  float vv[4];
  const int nc = seq_tiles(sp.len, kC);
  auto token = [&](int c, int t) -> int64_t { return min(sp.start + kC * c + t, sp.start + sp.len - 1); };
  auto ws = [&](int c) { return a.ws + chunk_at(a, seq, sp.start, c, h); };
  auto load_kv = [&](int c) {
    const int64_t at = token(c, 16 * wave + j) * a.k.ld + hk * a.k.hs + 8 * g;
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e) kf[w][e] = load4<BF16>(a.k.p, at + 32 * w + 4 * e);
#pragma unroll
    for (int r = 0; r < 4; ++r) vv[r] = load1<BF16>(a.v.p, token(c, 16 * wave + 4 * g + r) * a.v.ld + h * a.v.hs + col);
  };
  auto load_q = [&](int c) {
    const int64_t at = token(c, 16 * wave + j) * a.q.ld + hk * a.q.hs + 8 * g;
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[w][e] = load4<BF16>(a.q.p, at + 32 * w + 4 * e);
  };
  auto load_tile = [&](int c, int off, f32x4 (&f)[4]) {
    const f32x4* p = reinterpret_cast<const f32x4*>(ws(c) + off) + lane;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t <= wave) f[t] = *as_global(p + tri(wave, t) * 64);
  };
  auto load_kt = [&](int c) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        kt[t][r] = load2<BF16>(a.k.p, token(c, 16 * t + 4 * g + r) * a.k.ld + hk * a.k.hs + 32 * wave + 2 * j);
  };
  auto load_row = [&](int c) {
#pragma unroll
    for (int r = 0; r < 4; ++r) row[r] = *as_global(reinterpret_cast<const f32x4*>(ws(c) + kOffRow) + 16 * wave + 4 * g + r);
  };
  load_kv(0), load_row(0), load_q(0), load_tile(0, 0, tf), load_kt(0), load_tile(0, kOffP, pf);
  float flag = as_global(ws(0))[kOffFlag], decay = as_global(ws(0))[kOffRow + 4 * (kC - 1) + 2];
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = 0; c < nc; ++c) {
    const int nx = min(c + 1, nc - 1);
    const float dec = decay;
    if (flag != 0.0f) {
      // an input that is not finite: the products below would carry it to tokens before it (0 times it is not
      // 0), so the chunk runs token by token, in every wave alike
      const int t1 = min(kC, sp.len - kC * c);
      for (int t = 0; t < t1; ++t) {
        const int64_t tk = sp.start + kC * c + t;
        const float de = dev_expf(as_global(a.g)[tk * a.ldg + h]), be = as_global(a.beta)[tk * a.ldb + h];
        const float v1 = load1<BF16>(a.v.p, tk * a.v.ld + h * a.v.hs + col);
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float sv = s[w][e & 1][e >> 1] * de;
            s[w][e & 1][e >> 1] = sv;
            x = __builtin_fmaf(sv, load1<BF16>(a.k.p, tk * a.k.ld + hk * a.k.hs + 32 * w + 8 * g + e), x);
          }
        x = x + xor_perm<16>(x);
        x = x + xor_perm<32>(x);
        const float d = (v1 - x) * be;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float sv = __builtin_fmaf(load1<BF16>(a.k.p, tk * a.k.ld + hk * a.k.hs + 32 * w + 8 * g + e), d, s[w][e & 1][e >> 1]);
            s[w][e & 1][e >> 1] = sv;
            y = __builtin_fmaf(sv, load1<BF16>(a.q.p, tk * a.q.ld + hk * a.q.hs + 32 * w + 8 * g + e), y);
          }
        y = y + xor_perm<16>(y);
        y = y + xor_perm<32>(y);
        if (wave == 0 && g == 0) store1<BF16>(a.out.p, tk * a.out.ld + h * a.out.hs + col, y);
      }
      load_kv(nx), load_row(nx), load_q(nx), load_tile(nx, 0, tf), load_kt(nx), load_tile(nx, kOffP, pf);
      flag = as_global(ws(nx))[kOffFlag], decay = as_global(ws(nx))[kOffRow + 4 * (kC - 1) + 2];
      continue;
    }
    f32x4 x = zero, y = zero, d = zero, R, ec;
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e) x = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[w][e >> 2][e & 3], s[w][e & 1][e >> 1], x, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) R[r] = row[r][0] * vv[r] - row[r][1] * x[r];
    rl[wave][lane] = R;
    load_kv(nx);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e) y = __builtin_amdgcn_mfma_f32_16x16x4f32(qf[w][e >> 2][e & 3], s[w][e & 1][e >> 1], y, 0, 0, 0);
    load_q(nx);
    lds_barrier();
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t <= wave) d = mfma4(tf[t], rl[t][lane], d);
    load_tile(nx, 0, tf);
    dl[wave][lane] = d;
#pragma unroll
    for (int r = 0; r < 4; ++r) ec[r] = d[r] * row[r][3];
    el[wave][lane] = ec;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] *= row[r][2];
    load_row(nx);
    lds_barrier();
    f32x4 n0, n1;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      f32x4 o0 = s[0][0], o1 = s[0][1];
#pragma unroll
      for (int w = 1; w < 4; ++w)
        if (wave == w) o0 = s[w][0], o1 = s[w][1];
      n0[r] = o0[r] * dec;
      n1[r] = o1[r] * dec;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 e = el[t][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        n0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kt[t][r][0], e[r], n0, 0, 0, 0);
        n1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kt[t][r][1], e[r], n1, 0, 0, 0);
      }
    }
    sl[wave][0][lane] = n0;
    sl[wave][1][lane] = n1;
    load_kt(nx);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t <= wave) y = mfma4(pf[t], dl[t][lane], y);
    load_tile(nx, kOffP, pf);
    flag = as_global(ws(nx))[kOffFlag], decay = as_global(ws(nx))[kOffRow + 4 * (kC - 1) + 2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = kC * c + 16 * wave + 4 * g + r;
      if (t < sp.len) store1<BF16>(a.out.p, (int64_t)(sp.start + t) * a.out.ld + h * a.out.hs + col, y[r]);
    }
    lds_barrier();
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e) s[w][e] = sl[w][e][lane];
  }
  if (wave == 0)
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) as_global_w(Sp)[(32 * w + 8 * g + 2 * r + c) * kD] = s[w][c][r];
}

template <bool BF16>
hipError_t launch(const DeltaSeq& a, hipStream_t s) {
  if (a.ws == nullptr) {
    delta_step_kernel<BF16><<<(unsigned)(((int64_t)a.n_seq * a.heads * 8 + 3) / 4), 256, 0, s>>>(a);
  } else {
    delta_chunk_kernel<BF16><<<dim3((unsigned)seq_tiles_max(a.tokens, a.n_seq, kC), a.heads), 256, 0, s>>>(a);
    delta_scan_kernel<BF16><<<(unsigned)(((int64_t)a.n_seq * a.heads + 7) / 8 * 64), 256, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

size_t delta_seq_workspace(int tokens, int n_seq, int heads, int max_len) {
  if (max_len <= kDeltaStepLen) return 0;
  return ((size_t)tokens / kC + n_seq) * heads * kChunkFloats * sizeof(float);
}

hipError_t launch_delta_seq(const DeltaSeq& a, hipStream_t s) { return a.bf16 ? launch<true>(a, s) : launch<false>(a, s); }

}  // namespace qh
