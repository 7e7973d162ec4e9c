// Operators over packed sequences (qh_seq_ops.hip and the kernels beside it): an int8 matrix product for
// the activations of many tokens, the gated delta rule and causal attention.  Sequences stand one after
// another in the rows of an array; cu[i] .. cu[i + 1] are sequence i's rows.  cu, and the key ranges of
// attention, are device data that the host does not see, so the kernels bound every index themselves:
// the rules are the functions here, which the CPU tests compile too.
#pragma once
#include <stddef.h>
#include <stdint.h>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define QH_SEQ_FN __host__ __device__ __forceinline__
#else
#define QH_SEQ_FN inline
#endif

namespace qh {

// Rows of one sequence.
struct SeqSpan {
  int start, len;
};
// Sequence i's rows from its two bounds; bounds out of order or outside [0, rows] leave it without rows.
QH_SEQ_FN SeqSpan seq_span(int a, int b, int rows) {
  if (a < 0 || b < a || b > rows) return {0, 0};
  return {a, b - a};
}
// Keys of one sequence: the row its keys start at in an array of k_rows, and their number; a range that
// does not lie inside the array, or is longer than kMaxKeys, gives -1 (the sequence's outputs are then NaN).
constexpr int kMaxKeys = 1 << 30;
QH_SEQ_FN int key_len(int64_t start, int len, int64_t k_rows) {
  if (len < 0 || len > kMaxKeys || start < 0 || start > k_rows || (int64_t)len > k_rows - start) return -1;
  return len;
}
// Row tiles of a sequence of len rows.
QH_SEQ_FN int seq_tiles(int len, int tile) { return len / tile + (len % tile != 0); }
// The most tiles that n sequences of `rows` rows in all can have.
QH_SEQ_FN int64_t seq_tiles_max(int64_t rows, int n, int tile) {
  const int64_t t = rows / tile + n;
  return t < rows ? t : rows;   // (each tile holds a row)
}
// Keys that row `row` of q_len sees of k_len: the last rows stand at the last keys.  Not below 0.
QH_SEQ_FN int keys_seen(int row, int q_len, int k_len) {
  const int64_t n = (int64_t)row + 1 + k_len - q_len;
  return n < 0 ? 0 : (int)n;
}
// Of a sequence's nt tiles (`tile` rows each, G rows a token) those whose last row sees more than `keys` keys: the last.
QH_SEQ_FN int tiles_past(int q_len, int k_len, int G, int tile, int nt, int64_t keys) {
  const int64_t tok = keys - k_len + q_len;   // the first token that does
  if (nt <= 0 || tok >= q_len) return 0;
  return tok <= 0 ? nt : nt - (int)(tok * G / tile);
}

// A float as the sum of three bfloat16, eight bits of it each: the upper halves of p[0], p[1], p[2].
struct Cut {
  uint32_t p[3];
};
QH_SEQ_FN Cut cut_float(float x) {
  Cut c;
  auto next = [&]() {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    x -= __builtin_bit_cast(float, u & 0xffff0000u);
    return u;
  };
  c.p[0] = next(), c.p[1] = next(), c.p[2] = next();
  return c;
}

// The form of the int8 product: units of 16 rows and `unit` tokens straight from memory, or tiles of tile x tile.  By what
// was measured (us, weights from the L2s and the MALL).
// Units of 16 and 32 tokens and tiles of 64: 63 tokens 3584 -> 1024 5.5, 7.1 and 9.3, 1024 -> 512 3.2, 3.8 and 4.9, 1024 ->
// 2048 (512 and 256 units) 4.1, 3.8 and 4.8, 1024 -> 7168 (1792 and 896) 8.7, 8.0 and 5.2; 200 tokens 3584 -> 1024 (832 and
// 448) 14, 12 and 9.5: the smallest units that are at most a workgroup for each CU, else tiles.  Units of 16 and tiles
// for 16 tokens: 1024 -> 7168 (448 units) 4.0 and 4.5, 1024 -> 16384 (1024) 5.9 and 5.3, 1024 -> 151936 37 and 28; for 4
// tokens there 27 and 27.
// Tiles of 128 and of 64, by the number of the former: 3584 -> 1024 64 17.9 and 10.9, 96 19.3 and 16.4, 128 19.5 and 17.8;
// 4096 -> 4096 64 20.5 and 17.1, 128 22.2 and 23.9; 2048 -> 2048 128 13.7 and 11.8, 192 14.4 and 15.8; 1024 -> 7168 112
// 8.9 and 7.1, 224 10.3 and 15.0.
struct GemmForm {
  int unit, tile;   // one of them 0
};
inline GemmForm gemm_form(int tokens, int out, int64_t ldx) {
  const int64_t rt = (out + 15) / 16;
  auto units = [&](int t) { return rt * ((tokens + t - 1) / t); };
  auto tiles = [&](int t) { return (int64_t)((out + t - 1) / t) * ((tokens + t - 1) / t); };
  if (units(16) <= 256 || tokens <= 4 || (tokens <= 16 && rt <= 512)) return {16, 0};
  if (units(32) <= 256 || ldx >= 1 << 24) return {32, 0};   // (tiles: 32-bit offsets)
  return {0, tiles(128) <= 128 ? 64 : 128};
}

}  // namespace qh

#if defined(__HIPCC__)
namespace qh {

// One operand [rows][heads][dim] in place: element (r, h, d) at p + r * ld + h * hs + d.
struct SeqIn {
  const void* p = nullptr;
  int64_t ld = 0, hs = 0;
};
struct SeqOut {
  void* p = nullptr;
  int64_t ld = 0, hs = 0;
};

struct GemmSeq {
  SeqOut y;                       // [tokens][out], fp32 or bf16
  const int8_t* w = nullptr;      // [out][in]
  const float* scale = nullptr;   // [out]
  SeqIn x;                        // [tokens][in] int8
  const float* sx = nullptr;      // [tokens]
  int tokens = 0, out = 0, in = 0;
  int bf16 = 0;                   // type of y
  int wide = 0;                   // y takes four outputs in one store (set by the launch)
};

struct DeltaSeq {
  SeqOut out;                     // [tokens][heads][128]
  SeqIn q, k, v;                  // [tokens][k_heads][128], [tokens][heads][128]; the type of out
  const float* g = nullptr;       // [tokens][heads], rows ldg apart
  const float* beta = nullptr;
  int64_t ldg = 0, ldb = 0;
  float* S = nullptr;             // [n_seq][heads][128][128]
  const int32_t* cu = nullptr;
  int n_seq = 0, tokens = 0, k_heads = 0, heads = 0;
  int bf16 = 0;
  float* ws = nullptr;            // delta_seq_workspace bytes: in chunks; null: token by token
};

struct AttnSeq {
  SeqOut out;                     // [q_rows][heads][dim]
  SeqIn q, k, v;                  // [q_rows][heads][dim], [k_rows][kv_heads][dim]; the type of out
  const int32_t* cu_q = nullptr;  // [n_seq + 1]
  const int64_t* k_start = nullptr;
  const int32_t* k_len = nullptr;
  int n_seq = 0, q_rows = 0;
  int64_t k_rows = 0;
  int heads = 0, kv_heads = 0, dim = 0;
  float scale = 0.0f;
  int bf16 = 0;
  float* part = nullptr;          // partials of units whose keys are split
  int tile = 0;                   // rows of a tile of the form for prompts; 0: the form for few rows
  int limit = 0;                  // places in the workspace (few rows: 1: the keys may be split)
};

hipError_t launch_gemm_seq(const GemmSeq& a, hipStream_t s);
hipError_t launch_delta_seq(const DeltaSeq& a, hipStream_t s);
hipError_t launch_attn_seq(const AttnSeq& a, hipStream_t s);

// Sequences of up to this many tokens run token by token, which costs about 0.65 us a token for few heads (sequences
// times heads) and less for many, where chunks cost a launch more and a whole workgroup's start a sequence.  us for
// 24 / 48 tokens: 16 heads fp32 18.2 / 33.3 token by token, 19.3 / 20.2 in chunks, bfloat16 18.6 / 33.9 and 15.6 / 15.9;
// 512 heads fp32 41 / 72 and 135 / 139, bfloat16 42 / 75 and 74 / 77.
inline int delta_step_len(int64_t heads) { return heads < 256 ? 24 : 48; }
size_t delta_seq_workspace(int tokens, int n_seq, int heads, int k_heads, bool bf16, int max_len);

// The form of a call (AttnSeq's tile and limit) and the bytes of workspace it takes.
struct AttnForm {
  int tile, limit;
  size_t bytes;
};
AttnForm attn_seq_form(int64_t q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int dim, bool bf16);

}  // namespace qh
#endif
