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

// Whether a token has a place in a cache of `rows` rows; one that has none is skipped.
QH_SEQ_FN bool has_slot(int64_t slot, int64_t rows) { return slot >= 0 && slot < rows; }

// The scale of a row of int8 codes whose largest magnitude is `top`: top / 127, 1 for a row of zeros, and at least the
// smallest number, so that no value is divided by 0.
QH_SEQ_FN float code_scale(float top) {
  const float s = top / 127.0f;
  return !(top > 0.0f) ? 1.0f : s > 0.0f ? s : 0x1p-149f;
}

// Waves that take a token of `rows` heads (queries' and keys') in the norms with the rotation, one or four; a wave takes 512 / dim
// rows at a time, `groups` times in all.  One / four, us:
//   one group (1 / 1 heads of 256 or fewer): three of four would form angles for nothing; bfloat16 100 tokens 3.7 / 3.5, 1000 3.7
//     / 3.8, 4000 4.7 / 6.7, 16000 11.4 / 17.9; fp32 4000 6.4 / 7.7, 16000 14.9 / 19.0
//   3 to 5 (4 / 1 and 8 / 2 of 256, 8 / 8 and 16 / 4 of 128): four where there are few tokens for the chip's 1024 SIMDs; 8 / 2 bfloat16
//     1000 7.5 / 5.9, 1500 8.5 / 7.3, 2000 8.9 / 9.1, 4000 11.5 / 12.8, 16000 37 / 43; fp32 1500 9.9 / 9.4, 2000 10.9 / 11.3, 4000 16.0
//     / 16.8, 6000 28.8 / 27.6, 8000 39.7 / 35.7, 16000 63.9 / 63.2; 4 / 1 fp32 8000 16.5 / 17.1; 8 / 8 bfloat16 2000 7.4 / 7.3, 4000
//     9.9 / 11.4, fp32 2000 9.4 / 10.3, 8000 30.2 / 29.6
//   10 and more (32 / 8): 32 / 8 of 128 bfloat16 2000 13.3 / 12.0, 4000 17.7 / 17.6, 6000 26.7 / 28.6, 8000 40.6 / 36.6, 16000 62 / 68;
//     of 256 2000 22.1 / 17.7, 8000 74 / 57; fp32 of 128 2000 18.3 / 15.7, 8000 74 / 62
inline int norm_rope_waves(int tokens, int64_t rows, int dim, bool bf16) {
  const int64_t groups = (rows * dim + 511) / 512;
  if (groups == 1) return 1;
  if (groups >= 10 || tokens <= 1792) return 4;
  return !bf16 && groups >= 5 && tokens >= 4096 ? 4 : 1;
}

// Whether attention over an int8 cache takes the form for prompts (a workgroup for `tile` rows, 512 threads, about 2 us for
// every 32 keys however few rows there are) and not the one for few rows (16 rows), by bounds that the host knows: it does
// where a sequence has more than 256 rows a kv head, there is work for all CUs, and the tiles are full enough.
// Work: pairs of a query row and a key that it sees, about.  A prompt behind a long prefix is split in either form; one that
// begins its sequence costs the form for few rows no split, and fp32 hardly gains by the other: so 15 million pairs where there
// are twice as many keys as new tokens, else 20 (fp32: 33).  few / prompts:
//   8 / 2 heads of 256, bfloat16: 1500 tokens 40 / 52 us, 2000 (16 million) 57 / 61, 2300 (21) 75 / 66, 3000 109 / 88, 4000 174 / 126;
//     512 behind 1488 31 / 48, behind 2500 (11) 45 / 52, behind 3488 (15) 76 / 57, 300 behind 15700 162 / 85
//   fp32: 1500 tokens 43 / 53, 2000 62 / 70, 2300 82 / 84, 3000 (36) 119 / 120, 4000 192 / 197; 512 behind 3488 80 / 58
//   8 / 8 heads of 128, bfloat16: 1500 26 / 39, 2000 38 / 49, 2300 55 / 52, 3000 76 / 64, 4000 118 / 89; 512 behind 2500 35 / 38, behind
//     3488 54 / 43
//   fp32: 2000 40 / 51, 3000 78 / 89, 4000 124 / 136; 512 behind 3488 56 / 44
//   16 / 4 heads of 128, bfloat16: 1500 (18) 40 / 54, 2000 (32) 59 / 63, 2300 86 / 75; 256 behind 3840 (16) 54 / 43; fp32: 1500 42 / 60,
//     2000 62 / 85, 2300 (42) 90 / 97, 2600 110 / 107; 256 behind 3840 57 / 45
//   64 tokens behind 31936 keys (256 rows a kv head of 8 / 2) 60 / 78, 80 86 / 83
// Tiles: a sequence of max_q tokens, the others' of equal lengths, each with a tile that it does not fill.  A tile of the
// form for prompts costs as much as 9 (heads of 128: 8; fp32, whose tiles have 128 rows: 6) of 16 rows.  Single tokens and one
// prompt, whose tiles stand few / prompts as given, 8 / 2 heads of 256, bfloat16: 31 behind 30000 keys and 65 tokens 202 / 490 us
// (1.7 times as many tiles), 255 behind 8000 and 128 tokens 387 / 1089 (1.3), 31 behind 4000 and 512 behind 3488 88 / 117 (4.2), 100
// behind 4000 and 4000 tokens 244 / 372 (6.9), 31 behind 4000 and 2048 76 / 140 (8.7), 7 behind 4000 and 512 behind 3488 83 / 71
// (9.1), 31 behind 4000 and 8000 634 / 480 (13); 16 x 80 behind 4000 132 / 117 (9.6); 8 / 8 heads of 128: 31 behind 4000 and 8000
// 461 / 382 (8.5), 7 behind 4000 and 512 behind 3488 60 / 78 (4.4); fp32, 8 / 2 heads of 256: 64 x 300 216 / 170 (7.3), 7 behind 4000
// and 512 behind 3488 85 / 72 (5.9), 31 behind 4000 and 2048 81 / 144 (5.7).
inline bool attn_i8_prompts(int64_t q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int dim, int tile, bool bf16) {
  const int64_t G = heads / kv_heads, longest = max_q * G, rest = q_rows > max_q ? q_rows - max_q : 0;
  const int64_t others = n_seq - 1 < rest ? n_seq - 1 : rest;   // (the places of a batch that no token is left for are empty)
  const int64_t pairs = q_rows * heads * ((max_k > max_q ? max_k : max_q) - max_q / 2);
  auto tiles = [&](int rows) { return (longest + rest * G) / rows + others; };
  const int64_t from = max_k / 2 >= max_q ? 15000000 : bf16 ? 20000000 : 33000000;
  return longest > 256 && pairs >= from && tiles(16) >= (!bf16 ? 6 : dim == 256 ? 9 : 8) * tiles(tile);
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

// Norms of queries and keys for each head, with the position rotation.
struct NormRope {
  SeqOut qo, ko;                  // [tokens][heads][dim], [tokens][kv_heads][dim]
  SeqIn q, k;                     // of the same type; q (k) may be qo (ko) itself
  const float* qw = nullptr;      // [dim]
  const float* kw = nullptr;
  const int32_t* pos = nullptr;   // [tokens]
  int tokens = 0, heads = 0, kv_heads = 0, dim = 0, rot = 0;
  float eps = 0.0f;
  int bf16 = 0;
  double turns[128];              // of the angle i of a pair for each position: theta^(-2 i / rot) / (2 pi)
};

// A cache of int8 rows: codes [rows][heads][dim], a scale for each row and head.
struct CacheSide {
  int8_t* q = nullptr;            // codes, element (r, h, d) at q + r * ld + h * hs + d
  int64_t ld = 0, hs = 0;
  float* s = nullptr;             // scales, (r, h) at s + r * lds + h * hss
  int64_t lds = 0, hss = 0;
};
struct CacheSeq {
  CacheSide c[2];                 // keys, values
  const void* x[2] = {};          // new keys and values, or where the read ones go (written then): [tokens][heads][dim]
  int64_t ld[2] = {}, hs[2] = {};
  const int64_t* slot = nullptr;  // [tokens]
  int64_t rows = 0;
  int tokens = 0, heads = 0, dim = 0;
  int bf16 = 0;
};

// Attention over such a cache: k and v of AttnSeq are the codes.
struct AttnI8 : AttnSeq {
  const float *ks = nullptr, *vs = nullptr;   // scales, (r, h) at ks + r * ldks + h * hsks
  int64_t ldks = 0, hsks = 0, ldvs = 0, hsvs = 0;
  int max_q = 0;                  // the caller's bound
};

hipError_t launch_attn_i8(const AttnI8& a, hipStream_t s);
hipError_t launch_norm_rope(const NormRope& a, hipStream_t s);
hipError_t launch_cache_write(const CacheSeq& a, hipStream_t s);
hipError_t launch_cache_read(const CacheSeq& a, hipStream_t s);
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
AttnForm attn_i8_form(int64_t q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int dim, bool bf16);
AttnForm attn_seq_form(int64_t q_rows, int n_seq, int max_q, int max_k, int heads, int kv_heads, int dim, bool bf16);

}  // namespace qh
#endif
