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
//
// The products run on the matrix cores at fp32 precision.  A float is the sum of three bfloat16 exactly (its 24 bits
// cut into three eights, by masking), so an fp32 product is the six largest of the nine partial products (what is
// left out, the second times the third part twice over, is below 2^-21 of the product), and one with a bfloat16
// operand is three: 6 and 3 MFMAs of 16 cycles do
// what takes eight of 32 in v_mfma_f32_16x16x4_f32.  That one stays for the small triangular products with T and P.
// In all of them lane l has row l % 16 of the left and column l % 16 of the right operand, at the depths of lane group
// l / 16, and ends with rows 4 (l / 16) .. + 3 of column l % 16: what a lane holds of a result is what it has to
// bring as the next product's right operand, so results chain without a shuffle.
#include "qh_seq_device.hpp"

namespace qh {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int kD = 128;
constexpr int kC = 64;                       // tokens of a chunk
// A chunk's and head's part of the workspace, in floats: T and P in parts of bfloat16, as the operands that the wave of
// the tokens 16 w .. + 15 takes (depth 32 kk: kk = 0, and 1 for the waves 2 and 3; part by part, 16 bytes a lane: row
// l % 16, columns 32 kk + 4 (l / 16) .. and + 16); the tokens' factors beta, beta e^c, e^{c_63 - c} and e^c; whether an
// input is large or not finite, e^{c_63}.  (The factors in arrays of their own: a lane that loads what it does not use reuses
// those registers at once, and waits for the load before it.)
constexpr int kOperand = 3 * 256, kOffP = 6 * kOperand, kOffRow = 2 * kOffP, kOffFlag = kOffRow + 4 * kC, kChunkFloats = kOffFlag + 64;
__device__ __forceinline__ constexpr int operand(int w, int kk) { return w + (w == 3) + kk; }
// A chunk's slot: one per started 64 rows and sequence, so sequences need no count of those before them.
// (floor(x) + floor(y) <= floor(x + y), so a sequence's last slot lies below the next one's first.)
__device__ __forceinline__ size_t chunk_at(const DeltaSeq& a, int seq, int start, int c, int h) {
  return ((size_t)(start / kC + seq + c) * a.heads + h) * kChunkFloats;
}
// Behind those, each chunk's and key head's k and q in parts: k as it stands in LDS (key_at), q as the operands
// [tokens 16 w][depth 32 s][part][lane].  (Copies of a bfloat16 input too: its rows, a fused projection's, are powers of
// two apart, and a head's then lie in one of an L2's sixteen channels, from which eight workgroups would read them.)
constexpr int kPart = kC * kD * 2;
__host__ __device__ __forceinline__ constexpr size_t chunk_slots(int tokens, int n_seq) { return (size_t)(tokens / kC) + n_seq; }
template <int NP>
__device__ __forceinline__ char* keys_at(const DeltaSeq& a, int seq, int start, int c, int hk) {
  return reinterpret_cast<char*>(a.ws + chunk_slots(a.tokens, a.n_seq) * a.heads * kChunkFloats) +
         ((size_t)(start / kC + seq + c) * a.k_heads + hk) * (2 * NP * kPart);
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

// Token by token: a wave keeps 16 columns of one head's state in registers (lane: 8 k of 4 columns), so that the state is
// read and written once and the sums over k stay in the wave.  One token each of 32 sequences of 16 heads: bound by the
// states' way from and to memory, 11.5 us, 5.9 TB/s; many tokens: by the chain, 0.65 us a token.
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

// e^x for a difference of sums (its power of two rounded once to fp32: an error of |x| 2^-24 of what is e^x small).
__device__ __forceinline__ float exp_of(double x) { return __builtin_amdgcn_exp2f((float)(x * 1.4426950408889634)); }
// Two floats as pairs of bfloat16: the top eight bits of each, the next eight, the last eight.
__device__ __forceinline__ void cut2(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const Cut a = cut_float(x), b = cut_float(y);
  hi = __builtin_amdgcn_perm(b.p[0], a.p[0], 0x07060302u);
  mid = __builtin_amdgcn_perm(b.p[1], a.p[1], 0x07060302u);
  lo = __builtin_amdgcn_perm(b.p[2], a.p[2], 0x07060302u);
}
// Eight elements as NP parts: a bfloat16 input as it is, fp32 in three.
template <bool BF16>
struct Parts {
  static constexpr int NP = BF16 ? 1 : 3;
  u32x4 p[NP];
};
template <bool BF16>
struct Raw8 {   // eight elements as they lie in memory
  u32x4 v[BF16 ? 1 : 2];
};
template <bool BF16>
__device__ __forceinline__ Raw8<BF16> raw8(const void* p, int64_t at) {
  Raw8<BF16> o;
  const u32x4* q = reinterpret_cast<const u32x4*>(static_cast<const char*>(p) + at * (BF16 ? 2 : 4));
  o.v[0] = *as_global(q);
  if constexpr (!BF16) o.v[1] = *as_global(q + 1);
  return o;
}
template <bool BF16>
__device__ __forceinline__ Parts<BF16> parts(const Raw8<BF16>& r) {
  Parts<BF16> o;
  if constexpr (BF16) {
    o.p[0] = r.v[0];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t hi, mid, lo;
      cut2(__uint_as_float(r.v[e >> 1][2 * (e & 1)]), __uint_as_float(r.v[e >> 1][2 * (e & 1) + 1]), hi, mid, lo);
      o.p[0][e] = hi, o.p[1][e] = mid, o.p[2][e] = lo;
    }
  }
  return o;
}
// Whether an element is not finite, or so large (2^56) that a sum of products of finite ones may overflow.
constexpr uint32_t kLarge = (127 + 56) << 7;
template <bool BF16>
__device__ __forceinline__ bool any_large(const Raw8<BF16>& r) {
  bool bad = false;
#pragma unroll
  for (int q = 0; q < (BF16 ? 1 : 2); ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bad |= (r.v[q][e] & 0x7f800000u) >= kLarge << 16;
      if constexpr (BF16) bad |= (r.v[q][e] & 0x7f80u) >= kLarge;
    }
  return bad;
}
__device__ __forceinline__ f32x4 mfma32(const u32x4& x, const u32x4& y, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}
// Depth 32 of a product: x in NX parts, y in NY, the smallest partial products first.
template <int NX, int NY>
__device__ __forceinline__ f32x4 mul(const u32x4 (&x)[NX], const u32x4 (&y)[NY], f32x4 c) {
#pragma unroll
  for (int o = NX + NY - 2 < 2 ? NX + NY - 2 : 2; o >= 0; --o)
#pragma unroll
    for (int i = o < NX ? o : NX - 1; i >= 0; --i)
      if (o - i < NY) c = mfma32(x[i], y[o - i], c);
  return c;
}
// A chunk's keys in LDS, a part [64][128] bfloat16 after another: 16-byte piece c of token t at piece c ^ (t % 16),
// so that 16 tokens' pieces of one place lie in all banks.
__device__ __forceinline__ int key_at(int t, int c) { return t * (kD * 2) + 16 * (c ^ (t & 15)); }

// Eight values of a lane to the workspace in parts.
__device__ __forceinline__ void put_operand(float* to, int lane, const f32x4& x, const f32x4& y) {
  u32x4 p[3];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x4& v = e < 2 ? x : y;
    uint32_t hi, mid, lo;
    cut2(v[2 * (e & 1)], v[2 * (e & 1) + 1], hi, mid, lo);
    p[0][e] = hi, p[1][e] = mid, p[2][e] = lo;
  }
#pragma unroll
  for (int q = 0; q < 3; ++q) *as_global_w(reinterpret_cast<u32x4*>(to + 256 * q) + lane) = p[q];
}

// T, P and the row factors of one chunk, for the value heads of one key head.  Wave i forms the tiles (i, j <= i) of
// K K^T and Q K^T once; every head scales them.  A head's inputs are brought while the products of the one before run.
// What bounds it is mostly its traffic: for one sequence of 1500 fp32 tokens of 16 heads (384 workgroups, all at once, 21
// us) 37 MB of inputs and 52 MB of workspace, 18 us at the rate of a large copy; for 7.2k packed bfloat16 tokens of 32
// heads (77 us, three workgroups a CU; two: 82) 120 and 210 MB, 66 us.
template <bool BF16>
__global__ __launch_bounds__(256, BF16 ? 3 : 2) void delta_chunk_kernel(const DeltaSeq a) {
  constexpr int LD = kC + 4, NP = Parts<BF16>::NP;
  __shared__ __attribute__((aligned(256))) char kl[NP * kPart < kC * LD * 4 ? kC * LD * 4 : NP * kPart];
  __shared__ __attribute__((aligned(16))) float al[kC * LD];   // A
  float* tl = reinterpret_cast<float*>(kl);                    // T, over the keys
  __shared__ double cs[kC];
  __shared__ float bt[kC];
  __shared__ int bad_in[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, g4 = 4 * g, j = lane & 15;
  TileAt at;
  if (!find_tile(a.cu, a.n_seq, a.tokens, 1, kC, blockIdx.x, at)) return;
  const int hk = blockIdx.y, rep = a.heads / a.k_heads;
  const int t0 = at.sp.start + kC * at.tile, n = min(kC, at.sp.start + at.sp.len - t0);   // n >= 1 tokens
  bool bad = false;
  // a value head's inputs, brought while the products before it run
  constexpr int NV = kC * kD / 8 / 256;
  Raw8<BF16> vr[NV];
  float gv = 0.0f, be0 = 0.0f;
  auto load_head = [&](int h) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int e = 256 * u + threadIdx.x;
      vr[u] = raw8<BF16>(a.v.p, (int64_t)(t0 + min(e >> 4, n - 1)) * a.v.ld + h * a.v.hs + 8 * (e & 15));
    }
    if (wave == 0) {
      gv = as_global(a.g)[(int64_t)(t0 + min(lane, n - 1)) * a.ldg + h];
      be0 = as_global(a.beta)[(int64_t)(t0 + min(lane, n - 1)) * a.ldb + h];
    }
  };
  f32x4 G[4], P[4];   // tile (wave, jj): lane's token t = 16 wave + l % 16, tokens j = 16 jj + 4 (l / 16) ..
  {
    const int64_t r = t0 + min(16 * wave + j, n - 1);
    Parts<BF16> kp[4], qp[4];
    Raw8<BF16> kr[4], qr[4];   // (all on their way before the first store, which no load may pass)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      kr[s] = raw8<BF16>(a.k.p, r * a.k.ld + hk * a.k.hs + 32 * s + 8 * g);
      qr[s] = raw8<BF16>(a.q.p, r * a.q.ld + hk * a.q.hs + 32 * s + 8 * g);
    }
    load_head(hk * rep);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bad |= any_large<BF16>(kr[s]) || any_large<BF16>(qr[s]);
      kp[s] = parts<BF16>(kr[s]);
      qp[s] = parts<BF16>(qr[s]);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int at_k = p * kPart + key_at(16 * wave + j, 4 * s + g);
        *as_lds_w(reinterpret_cast<u32x4*>(kl + at_k)) = kp[s].p[p];
        char* to = keys_at<NP>(a, at.seq, at.sp.start, at.tile, hk);
        *as_global_w(reinterpret_cast<u32x4*>(to + at_k)) = kp[s].p[p];
        *as_global_w(reinterpret_cast<u32x4*>(to + NP * kPart + ((4 * wave + s) * NP + p) * 1024) + lane) = qp[s].p[p];
      }
    }
    __syncthreads();
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      G[jj] = P[jj] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (jj > wave) continue;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        u32x4 x[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) x[p] = *as_lds(reinterpret_cast<const u32x4*>(kl + p * kPart + key_at(16 * jj + j, 4 * s + g)));
        G[jj] = mul(x, kp[s].p, G[jj]);
        P[jj] = mul(x, qp[s].p, P[jj]);
      }
    }
  }
  const bool bad_qk = bad;
  for (int h = hk * rep; h < (hk + 1) * rep; ++h) {
    float* ws = a.ws + chunk_at(a, at.seq, at.sp.start, at.tile, h);
    bad = bad_qk;
    if (wave == 0) {
      // a log decay below -1e5 is 0 as a factor like any below -104, and finite in the sums
      float gl = 0.0f, be = 0.0f;
      if (lane < n) {
        gl = gv < -1e5f ? -1e5f : gv;
        be = be0;
        bad |= !(gl <= 0.5f) || !(__builtin_fabsf(be) < 0x1p56f);   // (64 tokens of 1/2: e^32)
      }
      double c = gl;
#pragma unroll
      for (int d = 1; d < kC; d *= 2) {
        const double t = __shfl_up(c, d);
        if (lane >= d) c += t;
      }
      const double last = __shfl(c, kC - 1);
      cs[lane] = c;
      bt[lane] = be;
      const float ec = exp_of(c);
      ws[kOffRow + lane] = be;
      ws[kOffRow + kC + lane] = be * ec;
      ws[kOffRow + 2 * kC + lane] = exp_of(last - c);
      ws[kOffRow + 3 * kC + lane] = ec;
      if (lane == kC - 1) ws[kOffFlag + 1] = ec;
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) bad |= any_large<BF16>(vr[u]);
    if (h + 1 < (hk + 1) * rep) load_head(h + 1);
    const uint64_t any = __ballot(bad);
    if (lane == 0) bad_in[wave] = any != 0;
    __syncthreads();
    const int t = 16 * wave + j;
    const double ct = cs[t];
    const float be = bt[t];
    f32x4 pv[4];
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
      pv[jj] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (jj > wave) continue;
      f32x4 av;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int jr = 16 * jj + g4 + r;
        const float e = jr <= t ? exp_of(ct - cs[jr]) : 0.0f;
        av[r] = jr < t ? be * e * G[jj][r] : 0.0f;
        pv[jj][r] = jr <= t ? e * P[jj][r] : 0.0f;
      }
      *as_lds_w(reinterpret_cast<f32x4*>(al + t * LD + 16 * jj + g4)) = av;
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
      if (kk <= wave >> 1) put_operand(ws + kOffP + operand(wave, kk) * kOperand, lane, pv[2 * kk], pv[2 * kk + 1]);
    if (threadIdx.x == 0) ws[kOffFlag] = (bad_in[0] | bad_in[1] | bad_in[2] | bad_in[3]) ? 1.0f : 0.0f;
    __syncthreads();
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
        const f32x4 m = mfma4(*as_lds(reinterpret_cast<const f32x4*>(tl + (16 * i + j) * LD + 16 * i + g4)), z, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          tc[i][r] = -m[r];
          tl[(16 * i + g4 + r) * LD + 16 * c + j] = -m[r];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
      if (kk <= wave >> 1) {
        f32x4 x[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          x[q] = *as_lds(reinterpret_cast<const f32x4*>(tl + (16 * wave + j) * LD + 32 * kk + 16 * q + g4));
          if (2 * kk + q > wave) x[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        put_operand(ws + operand(wave, kk) * kOperand, lane, x[0], x[1]);
      }
    __syncthreads();   // T and the sums have been read
  }
}

// The state's way through the chunks: a workgroup takes one sequence, one head and 16 NB of its columns.  What bounds it
// is the chain from one chunk's state to the next, so four waves do that alone, one on each SIMD.  Wave w keeps the
// state's rows 32 w .. + 31 in registers (lane: 32 w + 8 (l / 16) .. + 7 of column l % 16), which are at once its right
// operand; per chunk it
//   forms its rows' part of K S for all 64 tokens                                  | barrier 1
//   adds the four parts for the tokens 16 w .. + 15: R = beta v - beta e^c K S      | barrier 2
//   forms those tokens' d = T R                                                     | barrier 3
//   updates its rows: e^{c_63} S + K^T (e^{c_63 - c} d).
// Four waves beside them form the outputs e^c Q S + P d, and one brings the next chunk's keys to LDS.  All operands
// come in parts, cut once for a head's workgroups: the fp32 MFMAs run on the vector units, and cutting there, in each
// workgroup, held the chain up as much.  NB = 2 halves what a head's workgroups read from L2 (72 KB a chunk each in
// bfloat16), NB = 1 makes twice as many of them: 1500 tokens of 16, 32, 64, 96, 128 and 256 heads (sequences times heads)
// in bfloat16 88, 94, 106, 190, 211 and 400 us for NB = 2 (the chunks' launch included), 65, 73, 125, 189, 247 and 485
// for NB = 1.  With fp32's three parts of the keys NB = 2 would take 188 KB of LDS.  A chunk's way is 2.6 us.
template <bool BF16, int NB>
__global__ __launch_bounds__(576, 2) void delta_scan_kernel(const DeltaSeq a) {
  constexpr int NP = Parts<BF16>::NP, NSL = 8 / NB;
  __shared__ __attribute__((aligned(256))) char kl[2][NP * kPart];   // parts of the keys, this chunk's and the next one's
  __shared__ f32x4 xl[NB][4][4][64];             // [columns][token tile][wave]: the waves' parts of K S
  __shared__ u32x4 sl[NB][4][3][64];             // parts of the state
  __shared__ u32x2 rl[NB][4][3][64], el[NB][4][3][64], dl[NB][4][3][64];   // parts of R, of e^{c_63 - c_t} d_t, of d
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  const int g = lane >> 4, j = lane & 15;
  // the slices of a head on one of the eight XCDs, whose L2 then holds the head's operands
  const int b = blockIdx.x, u = (b & 7) + 8 * (b / (8 * NSL)), slice = (b >> 3) % NSL;
  if (u >= a.n_seq * a.heads) return;
  const int h = u % a.heads, seq = longest_first(a.cu, a.n_seq, a.tokens, u / a.heads), hk = h / (a.heads / a.k_heads);
  const SeqSpan sp = seq_span(as_global(a.cu)[seq], as_global(a.cu)[seq + 1], a.tokens);
  if (sp.len == 0) return;
  const int col = 16 * NB * slice + j;   // (+ 16 for the second)
  float* Sp = a.S + ((size_t)seq * a.heads + h) * kD * kD + col;
  const int nc = seq_tiles(sp.len, kC);
  auto token = [&](int c, int t) -> int64_t { return min(sp.start + kC * c + t, sp.start + sp.len - 1); };
  auto ws = [&](int c) { return a.ws + chunk_at(a, seq, sp.start, c, h); };
  auto flagged = [&](int c) { return as_global(ws(c))[kOffFlag]; };
  auto load_row = [&](int c, int which) {   // of this lane's four tokens
    return *as_global(reinterpret_cast<const f32x4*>(ws(c) + kOffRow + kC * which) + 4 * w + g);
  };
  auto load_operand = [&](int c, int off, u32x4 (&f)[2][3]) {   // (waves 0 and 1 have one: twice, so that the loads count alike)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int p = 0; p < 3; ++p)
        f[kk][p] = *as_global(reinterpret_cast<const u32x4*>(ws(c) + off + operand(w, min(kk, w >> 1)) * kOperand + 256 * p) + lane);
  };
  auto get_parts = [&](const u32x2 (&from)[4][3][64], int kk, u32x4 (&p)[3]) {   // depths: rows 4 (l / 16) .. of two tiles
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const u32x2 x = from[2 * kk][q][lane], y = from[2 * kk + 1][q][lane];
      p[q] = u32x4{x[0], x[1], y[0], y[1]};
    }
  };
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  int c = 0;
  if (wave < 4) {
    __builtin_amdgcn_s_setprio(3);
    float s[NB][8];
    u32x4 s3[NB][3];   // its parts
    auto cut_s = [&]() {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t hi, mid, lo;
          cut2(s[n][2 * e], s[n][2 * e + 1], hi, mid, lo);
          s3[n][0][e] = hi, s3[n][1][e] = mid, s3[n][2][e] = lo;
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) sl[n][w][q][lane] = s3[n][q];
      }
    };
    auto put_parts = [&](u32x2 (&to)[4][3][64], const f32x4& v) {
      u32x2 p[3];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t hi, mid, lo;
        cut2(v[2 * e], v[2 * e + 1], hi, mid, lo);
        p[0][e] = hi, p[1][e] = mid, p[2][e] = lo;
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) to[w][q][lane] = p[q];
    };
    // this lane's place in the transposing reads of the keys: token 4 (l / 16) + l % 16 / 4 (+ 16 tile), rows
    // 32 w + 8 (l % 4) + 4 cc .. + 3
    const int kt0 = 4 * g + (j >> 2), kc0 = 4 * w + (j & 3);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[n][e] = as_global(Sp)[(32 * w + 8 * g + e) * kD + 16 * n];
    while (c < nc) {
      if (flagged(c) != 0.0f) {
        // an input that is not finite, or from which a sum may overflow: the products below would carry it to tokens
        // before it (0 times infinity is not 0), so the chunk runs token by token, in all four waves alike (lane: rows
        // 32 w + 8 (l / 16) .. + 7 of all w)
        float* x0 = reinterpret_cast<float*>(xl);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int e = 0; e < 8; ++e) x0[(32 * n + w * 8 + e) * 64 + lane] = s[n][e];
        lds_barrier();
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float st[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) st[e] = x0[(32 * n + e) * 64 + lane];
          const int t1 = min(kC, sp.len - kC * c);
          for (int t = 0; t < t1; ++t) {
            const int64_t tk = sp.start + kC * c + t;
            const float de = dev_expf(as_global(a.g)[tk * a.ldg + h]), be = as_global(a.beta)[tk * a.ldb + h];
            const float v1 = load1<BF16>(a.v.p, tk * a.v.ld + h * a.v.hs + col + 16 * n);
            float x = 0.0f, y = 0.0f;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              st[e] *= de;
              x = __builtin_fmaf(st[e], load1<BF16>(a.k.p, tk * a.k.ld + hk * a.k.hs + 32 * (e >> 3) + 8 * g + (e & 7)), x);
            }
            x = x + xor_perm<16>(x);
            x = x + xor_perm<32>(x);
            const float d = (v1 - x) * be;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              st[e] = __builtin_fmaf(load1<BF16>(a.k.p, tk * a.k.ld + hk * a.k.hs + 32 * (e >> 3) + 8 * g + (e & 7)), d, st[e]);
              y = __builtin_fmaf(st[e], load1<BF16>(a.q.p, tk * a.q.ld + hk * a.q.hs + 32 * (e >> 3) + 8 * g + (e & 7)), y);
            }
            y = y + xor_perm<16>(y);
            y = y + xor_perm<32>(y);
            if (wave == 0 && g == 0) store1<BF16>(a.out.p, tk * a.out.ld + h * a.out.hs + col + 16 * n, y);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            s[n][e] = st[e];
#pragma unroll
            for (int q = 1; q < 4; ++q)
              if (w == q) s[n][e] = st[8 * q + e];
          }
        }
        lds_barrier();   // every wave has read the state
        ++c;
        continue;
      }
      f32x4 row[3];
      float vv[NB][4];
      u32x4 tp[2][3];
      auto load_v = [&](int c) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < NB; ++n)
            vv[n][r] = load1<BF16>(a.v.p, token(c, 16 * w + 4 * g + r) * a.v.ld + h * a.v.hs + col + 16 * n);
      };
      // (in the loop's order: the waits there count what is in flight on either way in)
      f32x2 fd = *as_global(reinterpret_cast<const f32x2*>(ws(c) + kOffFlag));
      load_v(c);
      row[0] = load_row(c, 0);
      row[1] = load_row(c, 1);
      load_operand(c, 0, tp);
      row[2] = load_row(c, 2);
      cut_s();
      lds_barrier();   // 0: the keys are there
      for (;;) {
        const int nx = min(c + 1, nc - 1);
        const float dec = fd[1];
        fd = *as_global(reinterpret_cast<const f32x2*>(ws(nx) + kOffFlag));
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          u32x4 kp[NP];
#pragma unroll
          for (int p = 0; p < NP; ++p) kp[p] = *as_lds(reinterpret_cast<const u32x4*>(kl[c & 1] + p * kPart + key_at(16 * t + j, 4 * w + g)));
#pragma unroll
          for (int n = 0; n < NB; ++n) xl[n][t][w][lane] = mul(kp, s3[n], zero);
        }
        lds_barrier();   // 1
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          f32x4 x = xl[n][w][0][lane], R;
#pragma unroll
          for (int q = 1; q < 4; ++q) x += xl[n][w][q][lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) R[r] = row[0][r] * vv[n][r] - row[1][r] * x[r];
          put_parts(rl[n], R);
        }
        load_v(nx);
        row[0] = load_row(nx, 0);
        row[1] = load_row(nx, 1);
        lds_barrier();   // 2
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          f32x4 d[2] = {zero, zero};
#pragma unroll
          for (int kk = 0; kk < 2; ++kk)
            if (kk <= w >> 1) {
              u32x4 rp[3];
              get_parts(rl[n], kk, rp);
              d[kk] = mul(tp[kk], rp, d[kk]);
            }
          d[0] += d[1];
          put_parts(el[n], d[0] * row[2]);
          put_parts(dl[n], d[0]);
        }
        load_operand(nx, 0, tp);
        row[2] = load_row(nx, 2);
        u32x4 kt[2][2][NP];   // K^T: this wave's rows (two tiles), depth tokens 32 kk + 4 (l / 16) .., + 16
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              union {
                i16x4 h[2];
                u32x4 v;
              } un;
#pragma unroll
              for (int q = 0; q < 2; ++q)
                un.h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)as_lds_w(
                    kl[c & 1] + p * kPart + key_at(32 * kk + 16 * q + kt0, kc0) + 8 * cc));
              kt[kk][cc][p] = un.v;
            }
        lds_barrier();   // 3: d and the next keys are there, this chunk's have been read
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          f32x4 sn[2];
#pragma unroll
          for (int q = 0; q < 8; ++q) sn[q >> 2][q & 3] = s[n][q] * dec;
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            u32x4 ep[3];
            get_parts(el[n], kk, ep);
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) sn[cc] = mul(kt[kk][cc], ep, sn[cc]);
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) s[n][q] = sn[q >> 2][q & 3];
        }
        if (++c >= nc || fd[0] != 0.0f) break;
        cut_s();
      }
      lds_barrier();   // every wave has read what it needs of the chunk
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 8; ++e) as_global_w(Sp)[(32 * w + 8 * g + e) * kD + 16 * n] = s[n][e];
  } else if (wave < 8) {   // outputs
    while (c < nc) {
      if (flagged(c) != 0.0f) {
        lds_barrier();
        lds_barrier();
        ++c;
        continue;
      }
      u32x4 qp[4][NP], pp[2][3];
      f32x4 row;
      auto load_q = [&](int c) {
        const char* from = keys_at<NP>(a, seq, sp.start, c, hk) + NP * kPart + 4 * NP * 1024 * w;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int p = 0; p < NP; ++p) qp[q][p] = *as_global(reinterpret_cast<const u32x4*>(from + (q * NP + p) * 1024) + lane);
      };
      load_q(c);   // (in the loop's order)
      row = load_row(c, 3);
      load_operand(c, kOffP, pp);
      float flag = flagged(c);
      lds_barrier();   // 0
      for (;;) {
        const int nx = min(c + 1, nc - 1);
        flag = flagged(nx);
        lds_barrier();   // 1: the state is there
        f32x4 o[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          f32x4 y[2] = {zero, zero};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            u32x4 sp3[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) sp3[p] = sl[n][q][p][lane];
            y[q & 1] = mul(qp[q], sp3, y[q & 1]);
          }
          o[n] = (y[0] + y[1]) * row;
        }
        load_q(nx);
        row = load_row(nx, 3);
        lds_barrier();   // 2
        lds_barrier();   // 3: d is there, the state has been read
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int kk = 0; kk < 2; ++kk)
            if (kk <= w >> 1) {
              u32x4 dp[3];
              get_parts(dl[n], kk, dp);
              o[n] = mul(pp[kk], dp, o[n]);
            }
        load_operand(nx, kOffP, pp);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = kC * c + 16 * w + 4 * g + r;
          if (t < sp.len)
#pragma unroll
            for (int n = 0; n < NB; ++n) store1<BF16>(a.out.p, (int64_t)(sp.start + t) * a.out.ld + h * a.out.hs + col + 16 * n, o[n][r]);
        }
        if (++c >= nc || flag != 0.0f) break;
      }
      lds_barrier();
    }
  } else {   // keys to LDS
    const uint32_t k0 = lds_address(kl);
    auto bring = [&](int c, int half) {
      const char* from = keys_at<NP>(a, seq, sp.start, min(c, nc - 1), hk) + half * (NP * kPart / 2);
      const uint32_t to = k0 + (c & 1) * (NP * kPart) + half * (NP * kPart / 2);
#pragma unroll 4
      for (int i = 0; i < 8 * NP; ++i) load_to_lds(from + 1024 * i, 16 * lane, to + 1024 * i);
    };
    while (c < nc) {
      if (flagged(c) != 0.0f) {
        lds_barrier();
        lds_barrier();
        ++c;
        continue;
      }
      bring(c, 0);
      bring(c, 1);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();   // 0
      for (;;) {
        const float flag = flagged(min(c + 1, nc - 1));
        bring(c + 1, 0);   // (where the chunk before this one stood: read before barrier 3)
        lds_barrier();   // 1
        bring(c + 1, 1);
        lds_barrier();   // 2
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();   // 3
        if (++c >= nc || flag != 0.0f) break;
      }
      lds_barrier();
    }
  }
}

template <bool BF16>
hipError_t launch(const DeltaSeq& a, hipStream_t s) {
  if (a.ws == nullptr) {
    delta_step_kernel<BF16><<<(unsigned)(((int64_t)a.n_seq * a.heads * 8 + 3) / 4), 256, 0, s>>>(a);
  } else {
    delta_chunk_kernel<BF16><<<dim3((unsigned)seq_tiles_max(a.tokens, a.n_seq, kC), a.k_heads), 256, 0, s>>>(a);
    const int64_t heads8 = ((int64_t)a.n_seq * a.heads + 7) / 8 * 8;
    if (BF16 && heads8 * 4 >= 256)   // (32 columns a workgroup would still be one for each CU)
      delta_scan_kernel<BF16, BF16 ? 2 : 1><<<(unsigned)(heads8 * 4), 576, 0, s>>>(a);
    else
      delta_scan_kernel<BF16, 1><<<(unsigned)(heads8 * 8), 576, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

size_t delta_seq_workspace(int tokens, int n_seq, int heads, int k_heads, bool bf16, int max_len) {
  if (max_len <= delta_step_len((int64_t)n_seq * heads)) return 0;
  return chunk_slots(tokens, n_seq) * ((size_t)heads * kChunkFloats * sizeof(float) + (size_t)k_heads * (bf16 ? 2 : 6) * kPart);
}

hipError_t launch_delta_seq(const DeltaSeq& a, hipStream_t s) { return a.bf16 ? launch<true>(a, s) : launch<false>(a, s); }

}  // namespace qh
