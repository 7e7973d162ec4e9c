// Device code that the attentions over packed sequences share: which rows and keys a workgroup takes, and the kernels
// that join the sums of split keys.
#pragma once
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
// Keys that the longest unsplit tile may hold more than a chunk, before splitting it (writing sums, a second kernel, more
// of it with more tiles) is worth it.  attention_seq_i8, bfloat16, 8 / 2 heads of 256, whole and split: 512 tokens 13
// and 17 us, 1024 24 and 28, 512 behind 1488 29 and 32, 100 single tokens of 1500 keys each 44 and 52, one of 500 12
// and 13; where it splits, 256 tokens behind 7744 95 and 62, 16 single tokens of 900 23 and 17.
__host__ __device__ __forceinline__ int few_whole(int64_t tiles) { return 384 + (int)(tiles > 192 ? 1536 : 8 * tiles); }
// Unit b of the split kernel, or (JOIN) the units of row tile b.  WHOLE: no tile is split where that would save no more
// than joining costs (few_whole), and a sequence's last tiles come first.
template <bool JOIN, bool WHOLE = false>
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
    int64_t all = tiles;
    int longest = tiles > 0 ? kl : 0;
    for (int s0 = 64; s0 < a.n_seq; s0 += 64) {
      load(s0);
      work += (int64_t)tiles * max(kl, 0);
      all += tiles;
      if (tiles > 0) longest = max(longest, kl);
    }
    if (a.n_seq > 64) load(0);
    work = sum_all(work);
    const int64_t c = (work * a.kv_heads + kFill - 1) / kFill;
    chunk = (int)min(max((c + 63) / 64 * 64, (int64_t)kMinChunk), (int64_t)kMaxKeys);
    if (WHOLE && __ballot(longest - chunk > few_whole(sum_all(all) * a.kv_heads)) == 0) chunk = kMaxKeys;
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
      const int nth = JOIN ? in : in / o.nsplit;
      o.tile = WHOLE && !JOIN ? of(tiles) - 1 - nth : nth;   // (the last tiles see the most keys: they start first)
      o.split = JOIN ? 0 : in - nth * o.nsplit;
      o.first = first + of(iu) - of(tiles * ns) + o.tile * o.nsplit;
      return o.tile >= 0 && o.tile < of(tiles);   // (bounds that overlap can make more tiles than an int counts)
    }
    base += __builtin_amdgcn_readlane(JOIN ? it : iu, 63);
    first += __builtin_amdgcn_readlane(iu, 63);
  }
  return false;
}

// Partials of a unit and kv head: 16 rows of D sums, their maxima, their sums of exponentials.
constexpr size_t part_floats(int D) { return 16 * D + 32; }

// Joins the splits of a tile's rows, every gridDim.y-th row in a workgroup: sixteen waves take every sixteenth split,
// four in flight, each with a running maximum of its own.
template <bool BF16, int D, bool WHOLE = false>
__global__ __launch_bounds__(1024) void attn_join_kernel(const AttnSeq a) {
  constexpr int W = D / 64, NW = 16, U = 4;   // elements of a lane; waves; splits in flight
  typedef float vec __attribute__((ext_vector_type(W)));
  __shared__ vec lo[NW][64];
  __shared__ float lsum[NW], lmax[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.heads / a.kv_heads;
  const int kvh = (int)blockIdx.x % a.kv_heads;
  Unit at;
  if (!find_unit<true, WHOLE>(a, (int)blockIdx.x / a.kv_heads, at)) return;
  if (at.nsplit == 1) return;   // written by the split kernel
  if (at.first < 0 || (int64_t)(at.first + at.nsplit) * a.kv_heads > (int64_t)gridDim.x + kFill) return;   // past its grid
  const int rows = at.sp.len * G;
  const size_t step = part_floats(D) * a.kv_heads;
  const float* pp = a.part + ((size_t)at.first * a.kv_heads + kvh) * part_floats(D);
  for (int j = blockIdx.y; j < 16 && 16 * at.tile + j < rows; j += gridDim.y) {
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

}  // namespace
}  // namespace qh
