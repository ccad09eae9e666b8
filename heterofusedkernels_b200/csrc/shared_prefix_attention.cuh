// Attention of one new token of each of `seqs` sequences over a paged cache, where all sequences share a
// prefix (one list of pages) and each has pages of its own behind it:
//
//   out[s, h*G+g] = softmax(scale * q[s, h*G+g] . [Kprefix[h]; K_s[h]]^T) [Vprefix[h]; V_s[h]]
//
// A softmax over several ranges of keys is joined from partial results (m, l, o) of each range, with
// m = max score, l = sum 2^(score - m), o = sum 2^(score - m) v (scores in units of log2 e):
//   M = max m_i,  L = sum l_i 2^(m_i - M),  out = sum o_i 2^(m_i - M) / L,  lse = ln 2 (M + log2 L).
// So the prefix is read once for all sequences: its rows of queries are (sequence, query head) pairs of one
// K/V head, seqs * G of them, and only what follows the prefix is read for each sequence alone.
// A row without any key (no prefix, length 0) is 0 with lse = -inf.
//
// 16-bit cache: weights are rounded to the cache's type, because the product wants operands of one type: 2^-9 (bf16) or 2^-12
// (fp16) of each weight, with errors of either sign, while l sums them unrounded.  Measured against 64 bits, bf16, thousands of keys:
// 0.0022 of the result, 0.0017 of which is the result's own rounding.
//
// 8-bit cache: codes are exact in fp16, so the products run on codes in fp16; the scale of a key multiplies its score,
// the scale of a value its weight.  bf16 queries become fp16 numbers times a power of two of their row that brings its largest
// to 2^14: they have fewer bits than fp16, so only what is 2^29 times smaller than that loses any, 2^-39 of it.
// (Where the prefix goes to the tensor cores, rows of like magnitude share a power of two: 2^-29 there.)
// Weights, times the value's scale, are fp16 then.  fp16 has few exponents, so they are taken relative to the largest such
// product of their own row: 2^e, a whole power, brings it to about 2^kWeightHigh, and o is rescaled when it passes 2^kWeightLimit.
// What is below 2^-14 is off by 2^-25 at most, 2^-31 of the largest, whatever the scales are and whichever keys have them.  The
// sum l of the weights without the scales has the origin m, o the origin m - e, and where a part is written o is brought to m.
// (The conversion of e4m3 to fp16 is one instruction for two codes; to bf16 it is five, which made up a third of the work of a
// tile.)
#pragma once

#include <type_traits>

#include "kv_format.cuh"
#include "kv_swap.cuh"  // load_id

namespace hfk {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  const unsigned char *q;         // row (s, head): q + s * q_seq + head * q_head (bytes)
  unsigned char *out;
  int64_t q_seq, q_head, out_seq, out_head;
  float *lse;                     // [seqs][kv_heads * group] or null
  const unsigned char *k_cache, *v_cache;
  int64_t block_stride, scales_at;
  int64_t num_blocks;
  const void *prefix_table, *tables, *lens;
  int64_t table_stride;
  int ids_are_int64;
  int prefix_len;
  int64_t own_cap;                // max_blocks * block_size: longest length the tables can name
  int seqs, kv_heads, group;
  FastDiv block, per_group;       // block size; group
  int tile;                       // keys of a tile of the line
  float scale_log2;               // scale * log2 e
  // partial results (workspace)
  float2 *part_ml;                // [parts][kItemRows]  (m, l)
  float *part_o;                  // [parts][kItemRows][head_dim]
};

// e of an 8-bit cache is at most kMostShift, so that 2^(8 + e) is an fp32 number: scales below 2^-108 lose bits.
constexpr float kWeightHigh = 10.f, kWeightLimit = 15.f, kMostShift = 118.f;

// Weights of a 16-bit cache are numbers of its type; up to 2^8 (see below), so that in fp16 2^7 times them still is one, and 2^-25,
// half its least step, is 2^-32 of the largest.
template <typename M>
__device__ __forceinline__ constexpr float raw_shift() { return std::is_same<M, __half>::value ? 128.f : 1.f; }

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- warp matrix product m16n8k16, fp32 accumulators ------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 matrix of 16-bit numbers; thread 4g + t holds row g, columns 2t and 2t + 1.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ---- codes to fp16: the four codes of a word as two pairs, exact ------------------------------------------
// int8: code ^ 0x80 is code + 128; 1024 + (code + 128) is an fp16 number with the code's bits in its mantissa.
template <int kFmt>
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if constexpr (kFmt == kFmtE4m3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(l), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(h), "r"(0x64806480u));
  }
}

// Type of the products' operands.
template <typename T, int kFmt>
using Operand = typename std::conditional<kFmt == kFmtRaw, T, __half>::type;

// bf16 queries as fp16: largest magnitude of a pair (infinities and NaN left out), the power of two that takes the
// largest of all into [2^14, 2^15), and the pair times it.
__device__ __forceinline__ float largest_of_pair(uint32_t w) {
  const uint32_t lo = (w << 16) & 0x7fffffffu, hi = w & 0x7fff0000u;
  return fmaxf(lo < 0x7f800000u ? __uint_as_float(lo) : 0.f, hi < 0x7f800000u ? __uint_as_float(hi) : 0.f);
}
__device__ __forceinline__ int shift_to_half(float largest) {
  const int e = (int)(__float_as_uint(largest) >> 23);   // biased exponent
  return largest == 0.f ? 0 : max(-126, min(126, 127 + 14 - e));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ uint32_t pair_to_half(uint32_t w, float factor) {
  const float2 f = Pair<__nv_bfloat16>::unpack(w);
  return Pair<__half>::pack(f.x * factor, f.y * factor);
}

// ---- how the work is laid out -------------------------------------------------------------------------------
// An ITEM is 8 rows of queries against one range of keys: for the prefix a (K/V head, 8 of the seqs * group
// rows), for a sequence's own keys a (sequence, K/V head, 8 of the group's rows).  Keys go by tiles of 16, of an 8-bit cache by tiles of 32: 8 KB at head_dim 128.
// All tiles of all items form one line, items of the prefix first, that is cut into equal pieces, one to a
// WARP: none has more than one tile more than another, whatever the lengths are (they are known on the
// device only).  A piece may end one item and begin the next.  The part of warp w of item i has the number
// w + i: along the line either grows, so no two parts share a number and there are at most warps + items.
constexpr int kItemRows = 8;
__host__ __device__ constexpr int tile_keys(int fmt) { return fmt == HFK_KV_RAW ? 16 : 32; }

struct AttnLine {
  int row_tiles, own_tiles;       // tiles of kItemRows rows: of the prefix's rows, of a group
  int prefix_items, prefix_tiles; // tiles of keys of an item
  int per_seq;                    // items of a sequence
  int tile;                       // keys of a tile
  __host__ __device__ AttnLine(int seqs, int kv_heads, int group, int prefix_len, int tile) : tile(tile) {
    row_tiles = (seqs * group + kItemRows - 1) / kItemRows;
    own_tiles = (group + kItemRows - 1) / kItemRows;
    prefix_tiles = (prefix_len + tile - 1) / tile;
    prefix_items = prefix_tiles > 0 ? row_tiles * kv_heads : 0;
    per_seq = kv_heads * own_tiles;
  }
  __host__ __device__ int64_t items(int seqs) const { return prefix_items + (int64_t)seqs * per_seq; }
  // Most tiles the line can have; the host takes so few sequences at a time that they number less than 2^31.
  __host__ __device__ int64_t most_tiles(int seqs, int64_t own_cap) const {
    return (int64_t)prefix_items * prefix_tiles + (int64_t)seqs * per_seq * ((own_cap + tile - 1) / tile);
  }
};

// Warps that take part: with fewer tiles than warps one tile each, so none of them is without a tile.
__device__ __forceinline__ int line_warps(int warps, int total) { return min(warps, total); }
// The first tile of warp w, and the warp that has tile x: w has [total w / warps, total (w + 1) / warps).
__device__ __forceinline__ int first_tile(int w, int warps, int total) { return (int)((int64_t)total * w / warps); }
__device__ __forceinline__ int warp_of_tile(int x, int warps, int total) { return (int)(((int64_t)warps * (x + 1) - 1) / total); }

// Clamped length of sequence s.
__device__ __forceinline__ int64_t own_length(const AttnArgs &a, int s, bool report) {
  int64_t len = load_id(a.lens, a.ids_are_int64, s);
  if (len < 0 || len > a.own_cap) {
    if (report) raise_status(HFK_DEV_BAD_SEQ_LEN);
    len = len < 0 ? 0 : a.own_cap;
  }
  return len;
}

// First tiles of the sequences (per item of a sequence) in shared memory, cu[seqs] the sum; all threads of the CTA,
// each a run of sequences, so that the lengths are one round of loads.
template <int kThreads>
__device__ __forceinline__ void scan_tiles(const AttnArgs &a, int *cu, int *warp_sums) {
  constexpr int kMost = (HFK_MAX_SEQS + kThreads - 1) / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (a.seqs + kThreads - 1) / kThreads;
  const int s0 = threadIdx.x * per;
  int n[kMost], sum = 0;
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    n[k] = k < per && s0 + k < a.seqs ? (int)((own_length(a, s0 + k, blockIdx.x == 0) + a.tile - 1) / a.tile) : 0;
    sum += n[k];
  }
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += v;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int before = inc - sum;
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    if (k < per && s0 + k < a.seqs) cu[s0 + k] = before;
    before += n[k];
  }
  if (threadIdx.x == kThreads - 1) cu[a.seqs] = before;
  __syncthreads();
}

// The item at a place of the line.
struct LineItem {
  int ordinal;
  int h, row0, rows, seq;   // its rows of queries: row0 .. row0 + rows of the prefix's rows, or of the sequence's group
  int len;                  // keys
  int tile, tiles;          // the place's tile of the item's tiles
  const void *table;        // its page ids start at table[table_at]
  int64_t table_at;
};
__device__ __forceinline__ LineItem line_item(const AttnArgs &a, const AttnLine &line, const int *cu, int at) {
  const int in_prefix = line.prefix_items * line.prefix_tiles;
  LineItem x;
  if (at < in_prefix) {
    x.ordinal = at / line.prefix_tiles;
    x.tile = at - x.ordinal * line.prefix_tiles;
    x.tiles = line.prefix_tiles;
    x.h = x.ordinal / line.row_tiles;
    x.row0 = (x.ordinal - x.h * line.row_tiles) * kItemRows;
    x.rows = min(kItemRows, a.seqs * a.group - x.row0);
    x.seq = 0;
    x.len = a.prefix_len;
    x.table = a.prefix_table;
    x.table_at = 0;
  } else {
    const int u = at - in_prefix;
    int lo = 0, hi = a.seqs;
    while (lo < hi) {         // number of sequences that end at or before u
      const int mid = (lo + hi) >> 1;
      if (cu[mid + 1] * line.per_seq <= u) lo = mid + 1; else hi = mid;
    }
    x.seq = lo;
    const int v = u - cu[lo] * line.per_seq;
    x.tiles = cu[lo + 1] - cu[lo];
    const int hg = v / x.tiles;
    x.tile = v - hg * x.tiles;
    x.ordinal = line.prefix_items + lo * line.per_seq + hg;
    x.h = hg / line.own_tiles;
    x.row0 = (hg - x.h * line.own_tiles) * kItemRows;
    x.rows = min(kItemRows, a.group - x.row0);
    x.len = (int)own_length(a, lo, false);
    x.table = a.tables;
    x.table_at = (int64_t)lo * a.table_stride;
  }
  return x;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
// A kernel launched behind another one of the same call may start while that one runs; its results are there
// after launch_wait.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void launch_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

constexpr int kLineWarps = 8;     // of a CTA; one CTA an SM

// Ring of a warp: kStages tiles, K rows, V rows, and for an 8-bit cache the scales of the keys, then of the values.
template <int kFmt, int D>
struct alignas(128) LineRing {
  static constexpr int kKeys = tile_keys(kFmt);
  static constexpr int kRow = D * (kFmt == kFmtRaw ? 2 : 1);
  static constexpr int kStages = D == 128 ? 3 : 5;
  unsigned char k[kStages][kKeys * kRow], v[kStages][kKeys * kRow];
  float scales[kStages][2 * kKeys];
  uint32_t valid[kStages];
  LineItem items[kStages + 1];    // items whose tiles are in the ring or next to come, by the number of changes so far
};

// ---- the kernel ------------------------------------------------------------------------------------------------
// Every warp works for itself: it keeps (m, l, o) of its piece, and brings its keys and values into a ring of its own
// with asynchronous copies that run ahead over the ends of items; nothing in the CTA waits for anything else.
// In the ring the 16-byte chunks of a row are XORed with bits of the row's number, so that the fragments' reads
// (K: four neighbouring chunks of two rows; V: two neighbouring chunks of four rows, two apart) hit all banks.
// Both products are taken transposed, scores^T = K Q^T and o^T = V^T weights^T: keys and head_dim fill the 16 rows of the
// instruction and the queries, of which a group has few, its 8 columns.  (With the queries as the 16 rows, half or more of
// the instructions, exponentials and accumulators were of rows that do not exist.)
// The order of the products over head_dim, and of the rows of o^T, is free, so a lane takes 16 contiguous bytes of
// a row where the operand layout would have it take two, and V needs no transposition: a lane that holds the same
// columns of four rows packs its operands with byte permutations.
//
// Bound by HBM for long sequences: 8 of 16384 to 131072 tokens, 8 heads of 128, bf16 (2.4 GB) 355 to 376 us, 6.4 to 6.8 TB/s;
// for short ones by the chain from a sequence's length over its page ids to its rows (about 5 us), and of 8-bit caches by
// what eight warps an SM can hide of a tile's latencies (50 MB 18 us).
template <typename T, int kFmt, int D>
__global__ void __launch_bounds__(kLineWarps * 32, 1) shared_prefix_attention_kernel(const __grid_constant__ AttnArgs a) {
  using Ring = LineRing<kFmt, D>;
  using M = Operand<T, kFmt>;
  constexpr int kElt = kFmt == kFmtRaw ? 2 : 1;
  constexpr int kKeys = Ring::kKeys, kRow = Ring::kRow, kStages = Ring::kStages;
  constexpr int kKc = kRow / 64;                          // 16-byte chunks of a K row per lane
  constexpr int kVb = kRow / 8 < 16 ? kRow / 8 : 16;      // bytes of a V chunk
  constexpr int kVc = kRow / 8 / kVb;                     // V chunks of a row per lane
  constexpr int kVe = kVb / kElt;                         // values of a V chunk
  constexpr int kE = 16 / kElt;                           // values of a K chunk
  constexpr int kCpr = kRow / 16, kRowsPass = 32 / kCpr;  // copies: chunks of a row, rows of a warp's pass
  constexpr int kM = kKeys / 16;                          // blocks of 16 keys
  constexpr bool kCodes = kFmt != kFmtRaw;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  Ring &ring = reinterpret_cast<Ring *>(smem_raw)[warp];
  int *cu = reinterpret_cast<int *>(smem_raw + kLineWarps * sizeof(Ring));   // [seqs + 1]
  int *warp_sums = cu + a.seqs + 1;

  launch_next();
  scan_tiles<kLineWarps * 32>(a, cu, warp_sums);
  const AttnLine line(a.seqs, a.kv_heads, a.group, a.prefix_len, kKeys);
  const int total = line.prefix_items * line.prefix_tiles + cu[a.seqs] * line.per_seq;
  const int warps = line_warps((int)gridDim.x * kLineWarps, total);
  // neighbouring pieces go to different SMs: a batch of few tiles is spread over all of them
  const int me = warp * (int)gridDim.x + (int)blockIdx.x;
  const int begin = me < warps ? first_tile(me, warps, total) : total, end = me < warps ? first_tile(me + 1, warps, total) : total;

  // ---- loads: tile `load_at` of the line is the next to be brought in, in groups of 16 keys
  // (This and line_item have one place each in the code: with the loads ahead of the loop and the items of loads and
  // products found separately, warps waited for instructions more than for anything else.)
  LineItem in = {};
  in.tile = -1;               // no item yet
  int load_at = begin, loads = 0;
  // Pages of a multiple of 16 tokens: a group lies in one page, and lane j holds the id of the page of group ids_from + j
  // of the item.  Other pages: lane j holds the id of the page of key j of the tile.
  const bool whole = a.block.d % 16 == 0;
  int64_t id = -1;
  int ids_from = 0;
  auto fetch_ids = [&](int group) {
    const int64_t key = whole ? ((int64_t)group + lane) * 16 : (int64_t)group * 16 + lane % kKeys;
    id = key < in.len ? load_id(in.table, a.ids_are_int64, in.table_at + a.block.div((uint32_t)key)) : -1;
    ids_from = group;
  };
  int load_stage = 0, changes = 0;
  const int chunk = lane % kCpr, sub = lane / kCpr;
  const int step = kRowsPass * a.kv_heads * kRow;             // bytes from pass to pass of a group in one page
  // where row `sub` of a pass goes in the ring: K, V; and what the number of the pass's first row changes in V's
  const uint32_t k_to = sub * kRow + (kCpr >= 8 ? chunk ^ ((sub & 1) << 2) : chunk) * 16;
  const uint32_t v_to = sub * kRow + (kCpr >= 8 ? chunk ^ (((sub >> 1) & 3) << 1) : chunk ^ ((sub >> 1) & 3)) * 16;
  auto v_flip = [](int r) -> uint32_t { return kCpr >= 8 ? (uint32_t)((r >> 1) & 3) << 5 : (uint32_t)((r >> 1) & 3) << 4; };
  auto load_group = [&](int group, int part) -> uint32_t {     // group `part` of the tile; returns which keys count
    const int key0 = group * 16;
    const uint32_t kb = smem_addr(ring.k[load_stage]) + part * 16 * kRow, vb = smem_addr(ring.v[load_stage]) + part * 16 * kRow;
    // lanes 0-15 the scales of the keys, 16-31 those of the values
    const uint32_t sb = smem_addr(&ring.scales[load_stage][(lane < 16 ? 0 : kKeys) + part * 16 + (lane & 15)]);
    if (whole) {
      const int64_t page_id = __shfl_sync(0xffffffffu, id, group - ids_from);
      const bool ok = page_id >= 0 && page_id < a.num_blocks;
      if (!ok && lane == 0 && key0 < in.len) raise_status(HFK_DEV_BAD_DEVICE_BLOCK_ID);
      const int64_t page = ok ? page_id * a.block_stride : 0;
      const int left = ok ? in.len - key0 : 0;              // rows behind the last key are zero
      // row of the page of the group's first key
      const uint32_t b = a.block.div((uint32_t)key0);
      const uint32_t row = ((uint32_t)key0 - b * a.block.d) * a.kv_heads + in.h;
      const int64_t from = page + (int64_t)(row + sub * a.kv_heads) * kRow + chunk * 16;
      const unsigned char *kp = a.k_cache + from, *vp = a.v_cache + from;
      const unsigned char *sp = (lane < 16 ? a.k_cache : a.v_cache) + page + a.scales_at + (int64_t)(row + (lane & 15) * a.kv_heads) * 4;
      if (left >= 16) {                                     // nearly always: no lane is left out
        if (kCodes) cp_async4(sb, sp, true);
#pragma unroll
        for (int r = 0; r < 16; r += kRowsPass) {
          cp_async16(kb + k_to + r * kRow, kp, true);
          cp_async16(vb + (v_to ^ v_flip(r)) + r * kRow, vp, true);
          kp += step;
          vp += step;
        }
        return 0xffffu;
      }
      if (kCodes) {
        const bool mine = (lane & 15) < left;
        cp_async4(sb, mine ? sp : a.k_cache, mine);
      }
#pragma unroll 1
      for (int r = 0; r < 16; r += kRowsPass) {
        const bool mine = r + sub < left;
        cp_async16(kb + k_to + r * kRow, mine ? kp : a.k_cache, mine);
        cp_async16(vb + (v_to ^ v_flip(r)) + r * kRow, mine ? vp : a.v_cache, mine);
        kp += step;
        vp += step;
      }
      return (1u << max(left, 0)) - 1u;
    }
    const int key = key0 + (lane & 15);
    const bool inside = key < in.len;
    const int64_t id_of_key = __shfl_sync(0xffffffffu, id, part * 16 + (lane & 15));
    const bool ok = inside && id_of_key >= 0 && id_of_key < a.num_blocks;
    if (inside && !ok) raise_status(HFK_DEV_BAD_DEVICE_BLOCK_ID);
    const uint32_t row = ((uint32_t)key - a.block.div((uint32_t)key) * a.block.d) * a.kv_heads + in.h;
    const int64_t page = ok ? id_of_key * a.block_stride : 0;
    const int64_t off = ok ? page + (int64_t)row * kRow : -1;
    if (kCodes) cp_async4(sb, (lane < 16 ? a.k_cache : a.v_cache) + page + a.scales_at + (ok ? (int64_t)row * 4 : 0), ok);
#pragma unroll 1
    for (int r = 0; r < 16; r += kRowsPass) {
      const int64_t o = __shfl_sync(0xffffffffu, off, r + sub);
      const int64_t from = (o < 0 ? 0 : o) + chunk * 16;
      cp_async16(kb + k_to + r * kRow, a.k_cache + from, o >= 0);
      cp_async16(vb + (v_to ^ v_flip(r)) + r * kRow, a.v_cache + from, o >= 0);
    }
    return __ballot_sync(0xffffffffu, ok) & 0xffffu;
  };
  auto load_tile = [&]() {
    if (load_at < end) {
      if (loads > 0) {
        uint32_t mask = 0;
        const int group = in.tile * (kKeys / 16);
#pragma unroll 1
        for (int part = 0; part < kKeys / 16; ++part)
          mask |= load_group(group + part, part) << (16 * part);
        if (lane == 0) ring.valid[load_stage] = mask;
        load_stage = load_stage + 1 == kStages ? 0 : load_stage + 1;
        ++load_at;
      }
      if (load_at < end) {    // the next tile's page ids, a tile ahead of their use
        const bool next_item = ++in.tile == in.tiles;
        if (next_item) {
          in = line_item(a, line, cu, load_at);
          if (lane == 0) ring.items[changes % (kStages + 1)] = in;
          ++changes;
        }
        const int next = in.tile * (kKeys / 16);
        if (next_item || !whole || next - ids_from >= 32) fetch_ids(next);
      }
    }
    ++loads;
    cp_async_commit();        // one group a tile, empty before the first and behind the last one
  };
  // queries: row g, the chunks this lane also takes of K
  uint32_t qf[D / 16][2];
  auto load_queries = [&](const LineItem &x) {
    const int r = x.row0 + g;
    const bool ok = g < x.rows;
    const int s = x.seq + (ok ? (int)a.per_group.div((uint32_t)r) : 0);
    const unsigned char *qp = a.q + s * a.q_seq + (int64_t)(x.h * a.group + (ok ? r - (s - x.seq) * a.group : 0)) * a.q_head;
#pragma unroll
    for (int c = 0; c < kKc; ++c)
#pragma unroll
      for (int j = 0; j < kE / 8; ++j) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (ok) w = *reinterpret_cast<const uint4 *>(qp + ((c * 4 + t) * kE + j * 8) * 2);
        const int ks = c * (kE / 4) + j * 2;
        qf[ks][0] = w.x;
        qf[ks][1] = w.y;
        qf[ks + 1][0] = w.z;
        qf[ks + 1][1] = w.w;
      }
  };
  int stage = 0, items = 0;
  LineItem x;
  // rows of queries 2t and 2t + 1: what their products are multiplied by, maximum, sum (of this lane's keys)
  float by[2], m[2], l[2], e[2], f[2];      // of an 8-bit cache e (see kWeightHigh) and f = 2^e
  float o[D / 16][4];
#pragma unroll 1
  for (int at = begin - kStages; at < end; ++at) {
    __syncwarp();             // the stage that is loaded now has been read by every lane
    load_tile();
    if (at < begin) continue;
    const bool first = at == begin || x.tile == x.tiles;
    if (first) {              // an item begins
      x = ring.items[items % (kStages + 1)];
      ++items;
      load_queries(x);
    }
    cp_async_wait<kStages - 1>();
    __syncwarp();             // every lane's copies of this tile have arrived
    if (first) {
      by[0] = by[1] = a.scale_log2;
      if constexpr (kCodes && !std::is_same<T, __half>::value) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) top = fmaxf(top, fmaxf(largest_of_pair(qf[k][0]), largest_of_pair(qf[k][1])));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int shift = shift_to_half(top);    // of row g
        const float up = power_of_two(shift), down = power_of_two(-shift);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[k][0] = pair_to_half(qf[k][0], up);
          qf[k][1] = pair_to_half(qf[k][1], up);
        }
        by[0] *= __shfl_sync(0xffffffffu, down, 8 * t);
        by[1] *= __shfl_sync(0xffffffffu, down, 8 * t + 4);
      }
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      e[0] = e[1] = kMostShift;
      f[0] = f[1] = ex2(kMostShift);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    }
    {
      const unsigned char *ks = ring.k[stage], *vs = ring.v[stage];
      const uint32_t valid = ring.valid[stage];

      // scores of kKeys keys and 8 rows: s[n][0..1] key 16n + g, rows 2t and 2t + 1; s[n][2..3] key 16n + g + 8
      float s[kM][4];
#pragma unroll
      for (int n = 0; n < kM; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < kKc; ++c) {
        const int at16 = kCpr >= 8 ? (c * 4 + t) ^ ((g & 1) << 2) : c * 4 + t;   // rows g and g + 8 have the same parity
#pragma unroll
        for (int n = 0; n < kM; ++n) {
          const unsigned char *kr = ks + (16 * n + g) * kRow + at16 * 16;
          const uint4 k0 = *reinterpret_cast<const uint4 *>(kr), k1 = *reinterpret_cast<const uint4 *>(kr + 8 * kRow);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
          if constexpr (!kCodes) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t ka[4] = {w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1]};
              mma16816<M>(s[n], ka, qf[2 * c + i][0], qf[2 * c + i][1]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t ka[4];
              codes_to_pairs<kFmt>(w0[i], ka[0], ka[2]);
              codes_to_pairs<kFmt>(w1[i], ka[1], ka[3]);
              mma16816<M>(s[n], ka, qf[4 * c + i][0], qf[4 * c + i][1]);
            }
          }
        }
      }
      float sv[kM][2];        // scales of the values of keys 16n + g and 16n + g + 8
#pragma unroll
      for (int n = 0; n < kM; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float sk = 1.f;
          if (kCodes) {
            sk = ring.scales[stage][16 * n + 8 * y + g];
            sv[n][y] = ring.scales[stage][kKeys + 16 * n + 8 * y + g];
          }
          // (a product of its own: an fma with the maximum would be off from the maximum's own rounding)
          s[n][2 * y] = __fmul_rn(s[n][2 * y], kCodes ? by[0] * sk : by[0]);
          s[n][2 * y + 1] = __fmul_rn(s[n][2 * y + 1], kCodes ? by[1] * sk : by[1]);
        }
      constexpr uint32_t kAll = kKeys == 32 ? 0xffffffffu : 0xffffu;
      if (valid != kAll) {
#pragma unroll
        for (int n = 0; n < kM; ++n)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if (!(valid >> (16 * n + 8 * y + g) & 1)) s[n][2 * y] = s[n][2 * y + 1] = -INFINITY;
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < kM; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) top[r] = fmaxf(top[r], fmaxf(s[n][r], s[n][2 + r]));
      // m follows a row's maximum only where it is 2^8 behind: weights up to 2^8 are as exact as weights up to 1.  Of an 8-bit
      // cache also e, where a weight times its value's scale passes 2^kWeightLimit; it is at most (largest weight) * (largest scale).
      bool move = top[0] > m[0] + 8.f || top[1] > m[1] + 8.f;
      if (kCodes) {
        float big = 0.f;                          // a NaN is left out here and passed on by the product
#pragma unroll
        for (int n = 0; n < kM; ++n) big = fmaxf(big, fmaxf(fabsf(sv[n][0]), fabsf(sv[n][1])));
        big = lg2(big);
        move = move || top[0] - m[0] + big + e[0] > kWeightLimit || top[1] - m[1] + big + e[1] > kWeightLimit;
      }
      if (__any_sync(0xffffffffu, move)) {
        // the tile's maxima: over the lanes of equal t
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
        }
        float alpha[2], rise[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          rise[r] = top[r] > m[r] + 8.f ? top[r] - m[r] : 0.f;     // infinite at the first key
          alpha[r] = ex2(-rise[r]);
          m[r] = rise[r] > 0.f ? top[r] : m[r];
          l[r] *= alpha[r];
        }
        if constexpr (kCodes) {
          float reach[2] = {-INFINITY, -INFINITY};   // log2 of the largest weight times scale
#pragma unroll
          for (int n = 0; n < kM; ++n)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float log_sv = lg2(fabsf(sv[n][y]));
              reach[0] = fmaxf(reach[0], s[n][2 * y] - m[0] + log_sv);
              reach[1] = fmaxf(reach[1], s[n][2 * y + 1] - m[1] + log_sv);
            }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            reach[0] = fmaxf(reach[0], __shfl_xor_sync(0xffffffffu, reach[0], d));
            reach[1] = fmaxf(reach[1], __shfl_xor_sync(0xffffffffu, reach[1], d));
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float before = e[r] + rise[r];
            e[r] = fminf(before, kMostShift);
            if (reach[r] + e[r] > kWeightLimit) e[r] = floorf(kWeightHigh - reach[r]);
            alpha[r] = ex2(e[r] - before);
            f[r] = ex2(e[r]);
          }
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[j][0] *= alpha[0];
          o[j][1] *= alpha[1];
          o[j][2] *= alpha[0];
          o[j][3] *= alpha[1];
        }
      }
      const float safe[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
      // o^T: block j = c * kVe / 2 + i has, of chunk c * 8 + g of a row, values 2i (o[j][0..1], rows 2t and 2t + 1) and
      // 2i + 1 (o[j][2..3])
#pragma unroll
      for (int n = 0; n < kM; ++n) {
        uint32_t pw[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float p0 = ex2(s[n][2 * y] - safe[0]), p1 = ex2(s[n][2 * y + 1] - safe[1]);
          l[0] += p0;
          l[1] += p1;
          pw[y] = transpose8(kCodes ? Pair<M>::pack(p0 * f[0] * sv[n][y], p1 * f[1] * sv[n][y])
                                    : Pair<M>::pack(p0 * raw_shift<M>(), p1 * raw_shift<M>()));
        }
#pragma unroll
        for (int c = 0; c < kVc; ++c) {
          uint32_t w[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int vr = 16 * n + 2 * t + (i & 1) + 8 * (i >> 1);
            if constexpr (kVb == 16) {
              const uint4 x4 = *reinterpret_cast<const uint4 *>(vs + vr * kRow + (((c * 8 + g) ^ (((vr >> 1) & 3) << 1)) * 16));
              w[i][0] = x4.x;
              w[i][1] = x4.y;
              w[i][2] = x4.z;
              w[i][3] = x4.w;
            } else {
              const uint2 x2 = *reinterpret_cast<const uint2 *>(vs + vr * kRow + (((g >> 1) ^ ((vr >> 1) & 3)) * 16) + (g & 1) * 8);
              w[i][0] = x2.x;
              w[i][1] = x2.y;
            }
          }
#pragma unroll
          for (int i = 0; i < kVb / 4; ++i) {
            if constexpr (!kCodes) {
              const uint32_t va[4] = {__byte_perm(w[0][i], w[1][i], 0x5410), __byte_perm(w[0][i], w[1][i], 0x7632),
                                      __byte_perm(w[2][i], w[3][i], 0x5410), __byte_perm(w[2][i], w[3][i], 0x7632)};
              mma16816<M>(o[c * (kVe / 2) + i], va, pw[0], pw[1]);
            } else {
              uint32_t va[4], vb[4];
              codes_to_pairs<kFmt>(__byte_perm(w[0][i], w[1][i], 0x5140), va[0], va[1]);
              codes_to_pairs<kFmt>(__byte_perm(w[0][i], w[1][i], 0x7362), vb[0], vb[1]);
              codes_to_pairs<kFmt>(__byte_perm(w[2][i], w[3][i], 0x5140), va[2], va[3]);
              codes_to_pairs<kFmt>(__byte_perm(w[2][i], w[3][i], 0x7362), vb[2], vb[3]);
              mma16816<M>(o[c * (kVe / 2) + 2 * i], va, pw[0], pw[1]);
              mma16816<M>(o[c * (kVe / 2) + 2 * i + 1], vb, pw[0], pw[1]);
            }
          }
        }
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    ++x.tile;
    if (x.tile != x.tiles && at + 1 != end) continue;

    // this warp's part of the item: lane (g, t) has kVe neighbouring values of each chunk, of two rows
    const int64_t part = (int64_t)me + x.ordinal;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
      const int row = 2 * t + r;
      if (row < x.rows) {
        if (g == 0) a.part_ml[part * kItemRows + row] = make_float2(m[r], l[r]);
        const float back = kCodes ? ex2(-e[r]) : 1.f / raw_shift<M>();
        float *dst = a.part_o + (part * kItemRows + row) * D;
#pragma unroll
        for (int c = 0; c < kVc; ++c)
#pragma unroll
          for (int e = 0; e < kVe; e += 4) {
            const int j = c * (kVe / 2) + e / 2;
            *reinterpret_cast<float4 *>(dst + (c * 8 + g) * kVe + e) =
                make_float4(o[j][r] * back, o[j][2 + r] * back, o[j + 1][r] * back, o[j + 1][2 + r] * back);
          }
      }
    }
  }
  cp_async_wait<0>();
  launch_wait();              // the join is launched behind this kernel and also reads what was launched before it
}

// Joins the parts of every row.  Up to three lists of parts: of the prefix's item and of the sequence's item on the
// line, and of the prefix's runs from prefix_tensor_kernel.
struct JoinArgs {
  AttnArgs a;               // as the line's kernel had it: prefix_len 0 where the prefix went to the tensor kernel
  int warps;                // warps of the line, 0: no line
  int splits, rows;         // of the tensor kernel; splits 0: not used
  const float2 *prefix_ml;
  const float *prefix_o;
};

// kJoinWarps warps a row, each with every kJoinWarps-th part and up to eight loads of a part under way: the parts (some
// dozens of a row, up to a warp's share of the line each) are in L2, and the time is that of the chain of their loads, so all
// rows should be at it at once: 16 warps a row where that fits, else four, two, one (2048 rows of 20 parts: 10 us with four,
// which take two turns, 8.5 with two).
constexpr int kJoinAhead = 8;
template <typename T, int D, int kJoinWarps>
__global__ void __launch_bounds__(kJoinWarps * 32, kJoinWarps > 14 ? 1 : 28 / kJoinWarps) shared_prefix_join_kernel(const __grid_constant__ JoinArgs args) {
  __shared__ float sums[kJoinWarps][D + 1];
  const AttnArgs &a = args.a;
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_heads = a.kv_heads * a.group;
  const int s = row / q_heads, head = row - s * q_heads, h = (int)a.per_group.div((uint32_t)head), g = head - h * a.group;
  // list k: parts first[k] + step[k] i in rows of (m, l) and of o, i < count[k].  Their places follow from the lengths alone,
  // so they are worked out while the kernels that write the parts still run.
  int count[3] = {0, 0, 0};
  int64_t first[3] = {0, 0, 0};
  if (args.warps > 0) {
    const AttnLine line(a.seqs, a.kv_heads, a.group, a.prefix_len, a.tile);
    const int in_prefix = line.prefix_items * line.prefix_tiles;
    int before = 0, all = 0;                     // tiles of the sequences before s, and of all
    for (int i = lane; i < a.seqs; i += 32) {
      const int n = (int)((own_length(a, i, false) + a.tile - 1) / a.tile);
      all += n;
      before += i < s ? n : 0;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    const int total = in_prefix + __reduce_add_sync(0xffffffffu, all) * line.per_seq;
    const int tiles_s = (int)((own_length(a, s, false) + a.tile - 1) / a.tile);
    const int warps = line_warps(args.warps, total);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int item, from, tiles, place;
      if (k == 0) {
        const int r = s * a.group + g;
        item = h * line.row_tiles + r / kItemRows;
        place = r % kItemRows;
        from = item * line.prefix_tiles;
        tiles = line.prefix_tiles;
      } else {
        const int hg = h * line.own_tiles + g / kItemRows;
        place = g % kItemRows;
        tiles = tiles_s;
        from = in_prefix + before * line.per_seq + hg * tiles;
        item = line.prefix_items + s * line.per_seq + hg;
      }
      if (tiles > 0) {
        const int w0 = warp_of_tile(from, warps, total), w1 = warp_of_tile(from + tiles - 1, warps, total);
        count[k] = w1 - w0 + 1;
        first[k] = ((int64_t)w0 + item) * kItemRows + place;
      }
    }
  }
  const int64_t stride = (int64_t)a.kv_heads * args.rows;
  if (args.splits > 0) {
    count[2] = args.splits;
    first[2] = (int64_t)h * args.rows + s * a.group + g;
  }
  const int parts = count[0] + count[1] + count[2];
  auto part_of = [&](int i, const float2 *&ml, const float *&o) {
    const bool p0 = i < count[0], p1 = i < count[0] + count[1];
    const int64_t at = p0 ? first[0] + (int64_t)i * kItemRows : p1 ? first[1] + (int64_t)(i - count[0]) * kItemRows : first[2] + (i - count[0] - count[1]) * stride;
    ml = (p1 ? a.part_ml : args.prefix_ml) + at;
    o = (p1 ? a.part_o : args.prefix_o) + at * D;
  };
  constexpr int kPer = D / 32;
  float2 ml[kJoinAhead];
  float o[kJoinAhead][kPer];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const int i = i0 + u * kJoinWarps;
      ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[u][e] = 0.f;
      if (i < parts) {
        const float2 *mp;
        const float *op;
        part_of(i, mp, op);
        ml[u] = *mp;
        if constexpr (kPer == 4) {
          const float4 x = *reinterpret_cast<const float4 *>(op + lane * 4);
          o[u][0] = x.x;
          o[u][1] = x.y;
          o[u][2] = x.z;
          o[u][3] = x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2 *>(op + lane * 2);
          o[u][0] = x.x;
          o[u][1] = x.y;
        }
      }
    }
  };
  launch_wait();
  fetch(warp);                // on their way while the maximum is found
  // the largest maximum: every warp looks at all
  float big = -INFINITY;
  for (int i = lane; i < parts; i += 32) {
    const float2 *mp;
    const float *op;
    part_of(i, mp, op);
    big = fmaxf(big, mp->x);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
  float l = 0.f, sum[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) sum[e] = 0.f;
#pragma unroll 1
  for (int i0 = warp; i0 < parts;) {
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const float f = big == -INFINITY ? 1.f : ex2(ml[u].x - big);
      l += ml[u].y * f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum[e] += o[u][e] * f;
    }
    i0 += kJoinWarps * kJoinAhead;
    if (i0 < parts) fetch(i0);
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) sums[warp][lane * kPer + e] = sum[e];
  if (lane == 0) sums[warp][D] = l;
  __syncthreads();
  for (int v = threadIdx.x * 2; v < D; v += kJoinWarps * 64) {
    float2 r = make_float2(0.f, 0.f);
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
      r.x += sums[w][v];
      r.y += sums[w][v + 1];
      l += sums[w][D];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;   // a NaN stays
    *reinterpret_cast<uint32_t *>(a.out + s * a.out_seq + (int64_t)head * a.out_head + v * 2) = Pair<T>::pack(r.x * inv, r.y * inv);
    if (a.lse != nullptr && v == 0) a.lse[(int64_t)s * q_heads + head] = l == 0.f ? -INFINITY : kLn2 * (big + log2f(l));
  }
}

}  // namespace hfk
