// Op-level C ABI of the operators over packed sequences: arguments checked on the host, work enqueued on the
// caller's stream, nothing allocated.
#include <cmath>
#include <cstdint>

#include "qh_common.hpp"
#include "qh_seq.hpp"
#include "qh_seq_view.hpp"

using namespace qh;

namespace {

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr int64_t kMaxUnits = 0x7fffffff;          // rows times heads
constexpr int kMaxGridY = 65535;
// A grid's threads in one direction stay below 2^32.
constexpr int64_t kMaxStates = 900000;             // sequences times heads: 8 workgroups of 576 each
constexpr int64_t kMaxTiles = 4000000;             // tiles of 16 rows and a kv head: a workgroup of 1024 each

constexpr int64_t kMaxCacheRows = 1 << 26;         // tokens times heads of a call over the cache: 8 rows a workgroup of 256

bool type_ok(int type) { return type == QH_F32 || type == QH_BF16; }

// The checks of a call that writes rows of an int8 cache from k and v, or k and v from its rows; a.tokens stays 0 where
// there is nothing to do.
int cache_args(CacheSeq& a, const View& kq, const View& ks, const View& vq, const View& vs, const void* k, int64_t ldk, int64_t hsk,
               const void* v, int64_t ldv, int64_t hsv, int type, const int64_t* slot, int64_t rows, int tokens, int heads, int dim,
               bool write) {
  if (!type_ok(type) || tokens < 0 || rows < 0 || heads <= 0 || (dim != 128 && dim != 256)) return QH_EINVAL;
  if (tokens == 0 || rows == 0) return QH_OK;
  if ((int64_t)tokens * heads > kMaxCacheRows || rows >= kMaxStride) return QH_ERANGE;
  const int eb = type == QH_BF16 ? 2 : 4;
  const View vk{k, tokens, heads, dim, ldk, hsk, eb}, vv{v, tokens, heads, dim, ldv, hsv, eb};
  if (!kq.readable() || !vq.readable() || !ks.strided() || !vs.strided() || !vk.readable() || !vv.readable() || !slot) return QH_EINVAL;
  if (write ? !kq.distinct() || !vq.distinct() || !ks.distinct() || !vs.distinct() : !vk.distinct() || !vv.distinct())
    return QH_EINVAL;
  if (!all_countable(kq, ks, vq, vs, vk, vv)) return QH_ERANGE;
  const View vt = flat(slot, tokens, 8);
  if (write ? overlap_any(kq, ks, vq, vs, vk, vv, vt) || overlap_any(ks, vq, vs, vk, vv, vt) || overlap_any(vq, vs, vk, vv, vt) ||
                  overlap_any(vs, vk, vv, vt)
            : overlap_any(vk, vv, kq, ks, vq, vs, vt) || overlap_any(vv, kq, ks, vq, vs, vt))
    return QH_EINVAL;
  auto side = [](const View& q, const View& s) {
    return CacheSide{static_cast<int8_t*>(const_cast<void*>(q.p)), q.ld, q.hs, static_cast<float*>(const_cast<void*>(s.p)), s.ld, s.hs};
  };
  a.c[0] = side(kq, ks);
  a.c[1] = side(vq, vs);
  a.x[0] = k, a.ld[0] = ldk, a.hs[0] = hsk;
  a.x[1] = v, a.ld[1] = ldv, a.hs[1] = hsv;
  a.slot = slot;
  a.rows = rows;
  a.tokens = tokens;
  a.heads = heads;
  a.dim = dim;
  a.bf16 = type == QH_BF16;
  return QH_OK;
}

}  // namespace

extern "C" {

int qh_gemm_i8_w8a8(void* y, int64_t ldy, int type, const int8_t* w, const float* scale, const int8_t* xq, int64_t ldx,
                    const float* sx, int tokens, int out, int in, void* stream) {
  if (!type_ok(type) || tokens < 0 || out <= 0 || in <= 0 || in % 16 != 0 || in > QH_GEMM_MAX_IN) return QH_EINVAL;
  if (tokens == 0) return QH_OK;
  if (tokens > QH_GEMM_MAX_TOKENS || out > QH_GEMM_MAX_OUT) return QH_ERANGE;
  const int eb = type == QH_BF16 ? 2 : 4;
  if (!w || !scale || !sx || !aligned16(w)) return QH_EINVAL;
  const View vx{xq, tokens, 1, in, ldx, 0, 1}, vy{y, tokens, 1, out, ldy, 0, eb};
  if (!vx.readable()) return QH_EINVAL;
  // y is written element by element: any row stride of at least a row
  if (!y || (reinterpret_cast<uintptr_t>(y) % eb) != 0 || (tokens > 1 && (ldy < out || ldy >= kMaxStride))) return QH_EINVAL;
  if (!all_countable(vx, vy)) return QH_ERANGE;
  if (overlap_any(vy, vx, flat(w, (int64_t)out * in, 1), flat(scale, out, 4), flat(sx, tokens, 4))) return QH_EINVAL;
  GemmSeq a;
  a.y = {y, ldy, 0};
  a.w = w;
  a.scale = scale;
  a.x = {xq, ldx, 0};
  a.sx = sx;
  a.tokens = tokens;
  a.out = out;
  a.in = in;
  a.bf16 = type == QH_BF16;
  return hip_status(launch_gemm_seq(a, S(stream)));
}

size_t qh_delta_rule_seq_workspace(int tokens, int n_seq, int heads, int k_heads, int type, int max_len) {
  if (tokens <= 0 || n_seq <= 0 || heads <= 0 || k_heads <= 0 || !type_ok(type) || (int64_t)n_seq * heads > kMaxStates ||
      (int64_t)tokens * heads > kMaxUnits)
    return 0;
  return delta_seq_workspace(tokens, n_seq, heads, k_heads, type == QH_BF16, max_len);
}

int qh_delta_rule_seq(void* out, int64_t ldo, int64_t hso, const void* q, int64_t ldq, int64_t hsq, const void* k, int64_t ldk,
                      int64_t hsk, const void* v, int64_t ldv, int64_t hsv, int type, const float* g, int64_t ldg,
                      const float* beta, int64_t ldb, float* state, const int32_t* cu, int n_seq, int tokens, int max_len,
                      int k_heads, int heads, void* workspace, size_t workspace_bytes, void* stream) {
  if (!type_ok(type) || n_seq < 0 || tokens < 0 || max_len < 0 || k_heads <= 0 || heads <= 0 || heads % k_heads != 0)
    return QH_EINVAL;
  if (tokens == 0 || n_seq == 0) return QH_OK;
  if ((int64_t)n_seq * heads > kMaxStates || (int64_t)tokens * heads > kMaxUnits || heads > kMaxGridY) return QH_ERANGE;
  const int eb = type == QH_BF16 ? 2 : 4;
  const View vo{out, tokens, heads, QH_LV, ldo, hso, eb}, vq{q, tokens, k_heads, QH_LK, ldq, hsq, eb},
      vk{k, tokens, k_heads, QH_LK, ldk, hsk, eb}, vv{v, tokens, heads, QH_LV, ldv, hsv, eb};
  if (!vo.writable() || !vq.readable() || !vk.readable() || !vv.readable()) return QH_EINVAL;
  if (!g || !beta || !state || !cu || !aligned16(state)) return QH_EINVAL;
  if (tokens > 1 && (ldg < 0 || ldb < 0 || ldg >= kMaxStride || ldb >= kMaxStride)) return QH_EINVAL;
  const View vg{g, tokens, 1, heads, ldg, 0, 4}, vb{beta, tokens, 1, heads, ldb, 0, 4},
      vs = flat(state, (int64_t)n_seq * heads * QH_LK * QH_LV, 4), vc = flat(cu, n_seq + 1, 4);
  if (!all_countable(vo, vq, vk, vv, vg, vb)) return QH_ERANGE;
  if (overlap_any(vo, vq, vk, vv, vg, vb, vs, vc) || overlap_any(vs, vq, vk, vv, vg, vb, vc)) return QH_EINVAL;
  const size_t need = qh_delta_rule_seq_workspace(tokens, n_seq, heads, k_heads, type, max_len);
  if (need > 0) {
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)) return QH_EINVAL;
    const View vw = flat(workspace, need, 1);
    if (overlap_any(vw, vo, vq, vk, vv, vg, vb, vs, vc)) return QH_EINVAL;
  }
  DeltaSeq a;
  a.out = {out, ldo, hso};
  a.q = {q, ldq, hsq};
  a.k = {k, ldk, hsk};
  a.v = {v, ldv, hsv};
  a.g = g;
  a.beta = beta;
  a.ldg = ldg;
  a.ldb = ldb;
  a.S = state;
  a.cu = cu;
  a.n_seq = n_seq;
  a.tokens = tokens;
  a.k_heads = k_heads;
  a.heads = heads;
  a.bf16 = type == QH_BF16;
  a.ws = need > 0 ? static_cast<float*>(workspace) : nullptr;
  return hip_status(launch_delta_seq(a, S(stream)));
}

size_t qh_attention_seq_workspace(int q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int head_dim, int type) {
  if (!type_ok(type) || q_rows <= 0 || n_seq <= 0 || n_seq > QH_ATTN_MAX_SEQ || max_q < 0 || max_k < 0 || max_k > kMaxKeys || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads != 0 || (head_dim != 128 && head_dim != 256) || (int64_t)q_rows * heads > kMaxUnits)
    return 0;
  return attn_seq_form(q_rows, n_seq, max_q, max_k, heads, kv_heads, head_dim, type == QH_BF16).bytes;
}

int qh_attention_seq(void* out, int64_t ldo, int64_t hso, const void* q, int64_t ldq, int64_t hsq, const void* k, int64_t ldk,
                     int64_t hsk, const void* v, int64_t ldv, int64_t hsv, int type, const int32_t* cu_q,
                     const int64_t* k_start, const int32_t* k_len, int n_seq, int q_rows, int64_t k_rows, int max_q, int max_k,
                     int heads, int kv_heads, int head_dim, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!type_ok(type) || n_seq < 0 || q_rows < 0 || k_rows < 0 || max_q < 0 || max_k < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads != 0 || (head_dim != 128 && head_dim != 256) || !std::isfinite(scale))
    return QH_EINVAL;
  if (q_rows == 0 || n_seq == 0) return QH_OK;
  if (n_seq > QH_ATTN_MAX_SEQ || max_k > kMaxKeys || (int64_t)q_rows * heads > kMaxUnits || k_rows >= kMaxStride ||
      seq_tiles_max((int64_t)q_rows * (heads / kv_heads), n_seq, 16) * kv_heads > kMaxTiles)
    return QH_ERANGE;
  const int eb = type == QH_BF16 ? 2 : 4;
  const View vo{out, q_rows, heads, head_dim, ldo, hso, eb}, vq{q, q_rows, heads, head_dim, ldq, hsq, eb},
      vk{k, k_rows, kv_heads, head_dim, ldk, hsk, eb}, vv{v, k_rows, kv_heads, head_dim, ldv, hsv, eb};
  if (!vo.writable() || !vq.readable()) return QH_EINVAL;
  if (k_rows > 0 && (!vk.readable() || !vv.readable())) return QH_EINVAL;
  if (!all_countable(vo, vq) || (k_rows > 0 && !all_countable(vk, vv))) return QH_ERANGE;
  if (!cu_q || !k_start || !k_len) return QH_EINVAL;
  const View vc = flat(cu_q, n_seq + 1, 4), vt = flat(k_start, n_seq, 8), vl = flat(k_len, n_seq, 4);
  if (overlap_any(vo, vq, vc, vt, vl) || (k_rows > 0 && overlap_any(vo, vk, vv))) return QH_EINVAL;
  const AttnForm form = attn_seq_form(q_rows, n_seq, max_q, max_k, heads, kv_heads, head_dim, type == QH_BF16);
  const size_t need = form.bytes;
  if (need > 0) {
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)) return QH_EINVAL;
    const View vw = flat(workspace, need, 1);
    if (overlap_any(vw, vo, vq, vc, vt, vl) || (k_rows > 0 && overlap_any(vw, vk, vv))) return QH_EINVAL;
  }
  AttnSeq a;
  a.out = {out, ldo, hso};
  a.q = {q, ldq, hsq};
  a.k = {k, ldk, hsk};
  a.v = {v, ldv, hsv};
  a.cu_q = cu_q;
  a.k_start = k_start;
  a.k_len = k_len;
  a.n_seq = n_seq;
  a.q_rows = q_rows;
  a.k_rows = k_rows;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = head_dim;
  a.scale = scale;
  a.bf16 = type == QH_BF16;
  a.part = static_cast<float*>(workspace);
  a.tile = form.tile;
  a.limit = form.limit;
  if (a.tile > 0 && (ldk >= (1 << 24) || ldv >= (1 << 24))) a.tile = a.limit = 0;   // (that form's 32-bit offsets)
  return hip_status(launch_attn_seq(a, S(stream)));
}

int qh_qk_norm_rope_seq(void* q_out, int64_t ldqo, int64_t hsqo, void* k_out, int64_t ldko, int64_t hsko, const void* q,
                        int64_t ldq, int64_t hsq, const void* k, int64_t ldk, int64_t hsk, int type, const float* q_norm,
                        const float* k_norm, const int32_t* pos, int tokens, int heads, int kv_heads, int head_dim, int rope_dim,
                        double theta, float eps, void* stream) {
  if (!type_ok(type) || tokens < 0 || heads <= 0 || kv_heads <= 0 || (head_dim != 128 && head_dim != 256) || rope_dim < 0 ||
      rope_dim > head_dim || rope_dim % 16 != 0 || !std::isfinite(theta) || theta < 1.0 || !std::isfinite(eps) || eps < 0.0f)
    return QH_EINVAL;
  if (tokens == 0) return QH_OK;
  if (tokens > QH_ROPE_MAX_TOKENS || (int64_t)tokens * ((int64_t)heads + kv_heads) > kMaxUnits) return QH_ERANGE;
  const int eb = type == QH_BF16 ? 2 : 4;
  const View vqo{q_out, tokens, heads, head_dim, ldqo, hsqo, eb}, vko{k_out, tokens, kv_heads, head_dim, ldko, hsko, eb},
      vq{q, tokens, heads, head_dim, ldq, hsq, eb}, vk{k, tokens, kv_heads, head_dim, ldk, hsk, eb};
  if (!vqo.writable() || !vko.writable() || !vq.readable() || !vk.readable()) return QH_EINVAL;
  if (!q_norm || !k_norm || !pos || !aligned16(q_norm) || !aligned16(k_norm)) return QH_EINVAL;
  if (!all_countable(vqo, vko, vq, vk)) return QH_ERANGE;
  const View wq = flat(q_norm, head_dim, 4), wk = flat(k_norm, head_dim, 4), vp = flat(pos, tokens, 4);
  // in place: a row is read whole before it is written
  if ((!same(vqo, vq) && overlap(vqo, vq)) || (!same(vko, vk) && overlap(vko, vk))) return QH_EINVAL;
  if (overlap_any(vqo, vko, vk, wq, wk, vp) || overlap_any(vko, vq, wq, wk, vp)) return QH_EINVAL;
  NormRope a;
  a.qo = {q_out, ldqo, hsqo};
  a.ko = {k_out, ldko, hsko};
  a.q = {q, ldq, hsq};
  a.k = {k, ldk, hsk};
  a.qw = q_norm;
  a.kw = k_norm;
  a.pos = pos;
  a.tokens = tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = head_dim;
  a.rot = rope_dim;
  a.eps = eps;
  a.bf16 = type == QH_BF16;
  // (a product for each pair in more than 64 bits: a power each took 1.3 us of the call)
  long double turn = 0.159154943091895335768883763372514362L;   // 1 / (2 pi)
  const long double step = rope_dim > 0 ? std::pow((long double)theta, -2.0L / rope_dim) : 1.0L;
  for (int i = 0; i < rope_dim / 2; ++i, turn *= step) a.turns[i] = (double)turn;
  return hip_status(launch_norm_rope(a, S(stream)));
}

int qh_kv_cache_write_i8(int8_t* kq, int64_t ldkq, int64_t hskq, float* ks, int64_t ldks, int64_t hsks, int8_t* vq, int64_t ldvq,
                         int64_t hsvq, float* vs, int64_t ldvs, int64_t hsvs, const void* k, int64_t ldk, int64_t hsk, const void* v,
                         int64_t ldv, int64_t hsv, int type, const int64_t* slot, int64_t rows, int tokens, int kv_heads,
                         int head_dim, void* stream) {
  CacheSeq a;
  const int st = cache_args(a, {kq, rows, kv_heads, head_dim, ldkq, hskq, 1}, {ks, rows, kv_heads, 1, ldks, hsks, 4},
                            {vq, rows, kv_heads, head_dim, ldvq, hsvq, 1}, {vs, rows, kv_heads, 1, ldvs, hsvs, 4}, k, ldk, hsk, v, ldv,
                            hsv, type, slot, rows, tokens, kv_heads, head_dim, true);
  return st != QH_OK || a.tokens == 0 ? st : hip_status(launch_cache_write(a, S(stream)));
}

int qh_kv_cache_read_i8(void* k, int64_t ldk, int64_t hsk, void* v, int64_t ldv, int64_t hsv, int type, const int8_t* kq,
                        int64_t ldkq, int64_t hskq, const float* ks, int64_t ldks, int64_t hsks, const int8_t* vq, int64_t ldvq,
                        int64_t hsvq, const float* vs, int64_t ldvs, int64_t hsvs, const int64_t* slot, int64_t rows, int tokens,
                        int kv_heads, int head_dim, void* stream) {
  CacheSeq a;
  const int st = cache_args(a, {kq, rows, kv_heads, head_dim, ldkq, hskq, 1}, {ks, rows, kv_heads, 1, ldks, hsks, 4},
                            {vq, rows, kv_heads, head_dim, ldvq, hsvq, 1}, {vs, rows, kv_heads, 1, ldvs, hsvs, 4}, k, ldk, hsk, v, ldv,
                            hsv, type, slot, rows, tokens, kv_heads, head_dim, false);
  return st != QH_OK || a.tokens == 0 ? st : hip_status(launch_cache_read(a, S(stream)));
}

size_t qh_attention_seq_i8_workspace(int q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int head_dim, int type) {
  if (!type_ok(type) || q_rows <= 0 || n_seq <= 0 || n_seq > QH_ATTN_MAX_SEQ || max_q < 0 || max_k < 0 || max_k > kMaxKeys ||
      heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || (head_dim != 128 && head_dim != 256) ||
      (int64_t)q_rows * heads > kMaxUnits)
    return 0;
  return attn_i8_form(q_rows, n_seq, max_q, max_k, heads, kv_heads, head_dim, type == QH_BF16).bytes;
}

int qh_attention_seq_i8(void* out, int64_t ldo, int64_t hso, const void* q, int64_t ldq, int64_t hsq, int type, const int8_t* kq,
                        int64_t ldkq, int64_t hskq, const float* ks, int64_t ldks, int64_t hsks, const int8_t* vq, int64_t ldvq,
                        int64_t hsvq, const float* vs, int64_t ldvs, int64_t hsvs, const int32_t* cu_q, const int64_t* k_start,
                        const int32_t* k_len, int n_seq, int q_rows, int64_t k_rows, int max_q, int max_k, int heads, int kv_heads,
                        int head_dim, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!type_ok(type) || n_seq < 0 || q_rows < 0 || k_rows < 0 || max_q < 0 || max_k < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads != 0 || (head_dim != 128 && head_dim != 256) || !std::isfinite(scale))
    return QH_EINVAL;
  if (q_rows == 0 || n_seq == 0) return QH_OK;
  if (n_seq > QH_ATTN_MAX_SEQ || max_k > kMaxKeys || (int64_t)q_rows * heads > kMaxUnits || k_rows >= kMaxStride ||
      seq_tiles_max((int64_t)q_rows * (heads / kv_heads), n_seq, 16) * kv_heads > kMaxTiles)
    return QH_ERANGE;
  const int eb = type == QH_BF16 ? 2 : 4;
  const View vo{out, q_rows, heads, head_dim, ldo, hso, eb}, vq_{q, q_rows, heads, head_dim, ldq, hsq, eb},
      vk{kq, k_rows, kv_heads, head_dim, ldkq, hskq, 1}, vv{vq, k_rows, kv_heads, head_dim, ldvq, hsvq, 1},
      sk{ks, k_rows, kv_heads, 1, ldks, hsks, 4}, sv{vs, k_rows, kv_heads, 1, ldvs, hsvs, 4};
  if (!vo.writable() || !vq_.readable()) return QH_EINVAL;
  if (k_rows > 0 && (!vk.readable() || !vv.readable() || !sk.strided() || !sv.strided())) return QH_EINVAL;
  if (!all_countable(vo, vq_) || (k_rows > 0 && !all_countable(vk, vv, sk, sv))) return QH_ERANGE;
  for (const int64_t ld : {ldkq, ldvq, ldks, ldvs})   // (the kernels' 32-bit offsets)
    if (k_rows > 1 && ld >= QH_ATTN_I8_MAX_LD) return QH_ERANGE;
  if (!cu_q || !k_start || !k_len) return QH_EINVAL;
  const View vc = flat(cu_q, n_seq + 1, 4), vt = flat(k_start, n_seq, 8), vl = flat(k_len, n_seq, 4);
  if (overlap_any(vo, vq_, vc, vt, vl) || (k_rows > 0 && overlap_any(vo, vk, vv, sk, sv))) return QH_EINVAL;
  const AttnForm form = attn_i8_form(q_rows, n_seq, max_q, max_k, heads, kv_heads, head_dim, type == QH_BF16);
  const size_t need = form.bytes;
  if (need > 0) {
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)) return QH_EINVAL;
    const View vw = flat(workspace, need, 1);
    if (overlap_any(vw, vo, vq_, vc, vt, vl) || (k_rows > 0 && overlap_any(vw, vk, vv, sk, sv))) return QH_EINVAL;
  }
  AttnI8 a;
  a.out = {out, ldo, hso};
  a.q = {q, ldq, hsq};
  a.k = {kq, ldkq, hskq};
  a.v = {vq, ldvq, hsvq};
  a.ks = ks;
  a.vs = vs;
  a.ldks = ldks;
  a.hsks = hsks;
  a.ldvs = ldvs;
  a.hsvs = hsvs;
  a.max_q = max_q;
  a.cu_q = cu_q;
  a.k_start = k_start;
  a.k_len = k_len;
  a.n_seq = n_seq;
  a.q_rows = q_rows;
  a.k_rows = k_rows;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = head_dim;
  a.scale = scale;
  a.bf16 = type == QH_BF16;
  a.part = static_cast<float*>(workspace);
  a.tile = form.tile;
  a.limit = form.limit;
  return hip_status(launch_attn_i8(a, S(stream)));
}

}  // extern "C"
