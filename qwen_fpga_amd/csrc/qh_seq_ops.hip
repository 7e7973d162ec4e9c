// Op-level C ABI of the operators over packed sequences: arguments checked on the host, work enqueued on the
// caller's stream, nothing allocated.
#include <cmath>

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

bool type_ok(int type) { return type == QH_F32 || type == QH_BF16; }

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

}  // extern "C"
