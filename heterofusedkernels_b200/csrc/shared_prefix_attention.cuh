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
// 8-bit cache: codes are exact in both 16-bit types, so the products run on codes; the scale of a key multiplies
// its score, the scale of a value its weight.
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
  FastDiv block;
  float scale_log2;               // scale * log2 e
  // partial results (workspace)
  int64_t *cu;                    // [seqs + 1] first tile of each sequence, per (K/V head, row tile)
  float2 *part_ml;                // [parts][16]  (m, l)
  float *part_o;                  // [parts][16][head_dim]
};

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
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- codes to a 16-bit type: the four codes of a word as two pairs, exact ----------------------------------
// e4m3 to bf16: sign, exponent and mantissa moved to their places are the number times 2^-120 (the biases
// differ by 120; subnormal codes become subnormal numbers), and one multiplication by 2^120 follows.
// int8 to bf16: with u = the low seven bits, 128 + u and 128 (or 256 where the sign bit is set) differ by the
// code; both are bf16 numbers whose mantissa is the code's bits.  int8 to fp16: 1024 + (code + 128) - 1152.
template <typename T, int kFmt>
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if constexpr (kFmt == kFmtE4m3) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
      const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
      lo = a.x | ((uint32_t)a.y << 16);
      hi = b.x | ((uint32_t)b.y << 16);
    } else {
      const uint32_t l = __byte_perm(w, 0, 0x1404), h = __byte_perm(w, 0, 0x3424);
      const uint32_t lb = (l & 0x80008000u) | ((l >> 4) & 0x07f007f0u), hb = (h & 0x80008000u) | ((h >> 4) & 0x07f007f0u);
      asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(lb), "r"(0x7b807b80u));
      asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(hb), "r"(0x7b807b80u));
    }
  } else if constexpr (std::is_same<T, __half>::value) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(l), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(h), "r"(0x64806480u));
  } else {
    const uint32_t l = __byte_perm(w, 0x43434343u, 0x4140), h = __byte_perm(w, 0x43434343u, 0x4342);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(l & 0xff7fff7fu), "r"(l & 0xff80ff80u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(h & 0xff7fff7fu), "r"(h & 0xff80ff80u));
  }
}

// ---- how the work is laid out -------------------------------------------------------------------------------
// An ITEM is 16 rows of queries against one range of keys: for the prefix a (K/V head, 16 of the seqs * group
// rows), for a sequence's own keys a (sequence, K/V head, 16 of the group's rows).  Keys go by tiles of 64.
// All tiles of all items form one line, items of the prefix first, that is cut into equal pieces, one to a
// CTA: no CTA has more than one tile more than another, whatever the lengths are (they are known on the
// device only).  A piece may end one item and begin the next.  The part of CTA c of item i has the number
// c + i: along the line either grows, so no two parts share a number and there are at most CTAs + items.
constexpr int kTileKeys = 64;

struct AttnLine {
  int row_tiles, own_tiles;       // tiles of 16 rows: of the prefix's rows, of a group
  int prefix_items, prefix_tiles; // tiles of 64 keys of an item
  int per_seq;                    // items of a sequence
  __host__ __device__ AttnLine(int seqs, int kv_heads, int group, int prefix_len) {
    row_tiles = (seqs * group + 15) / 16;
    own_tiles = (group + 15) / 16;
    prefix_tiles = (prefix_len + kTileKeys - 1) / kTileKeys;
    prefix_items = prefix_tiles > 0 ? row_tiles * kv_heads : 0;
    per_seq = kv_heads * own_tiles;
  }
  __host__ __device__ int64_t items(int seqs) const { return prefix_items + (int64_t)seqs * per_seq; }
};

// CTAs that take part: with fewer tiles than CTAs one tile each, so that none of them is without a part.
__device__ __forceinline__ int64_t line_ctas(int64_t grid, int64_t total) { return min(grid, total); }

// Clamped length of sequence s.
__device__ __forceinline__ int64_t own_length(const AttnArgs &a, int s, bool report) {
  int64_t len = load_id(a.lens, a.ids_are_int64, s);
  if (len < 0 || len > a.own_cap) {
    if (report) raise_status(HFK_DEV_BAD_SEQ_LEN);
    len = len < 0 ? 0 : a.own_cap;
  }
  return len;
}

// First tiles of the sequences (per item of the sequence), by warp 0.
__device__ __forceinline__ void scan_tiles(const AttnArgs &a, int64_t *cu) {
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  int64_t carry = 0;
  for (int base = 0; base < a.seqs; base += 32) {
    const int s = base + lane;
    const int64_t n = s < a.seqs ? (own_length(a, s, blockIdx.x == 0) + kTileKeys - 1) / kTileKeys : 0;
    int64_t inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += v;
    }
    if (s < a.seqs) cu[s] = carry + inc - n;
    carry += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) cu[a.seqs] = carry;
}

// ---- the kernel ------------------------------------------------------------------------------------------------
// Four warps; each takes 16 of a tile's 64 keys and keeps (m, l, o) of its own over the whole piece, so the
// warps meet only at the end of a piece.  K and V go from global memory straight into the registers of the
// matrix product: the order of the products over head_dim, and of the columns of o, is free, so a lane takes
// 16 contiguous bytes of a row where the operand layout would have it take two.
template <typename T, int kFmt, int D>
__global__ void __launch_bounds__(128) shared_prefix_attention_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int kElt = kFmt == kFmtRaw ? 2 : 1;
  constexpr int kRow = D * kElt;
  constexpr int kKc = kRow / 64;                          // 16-byte chunks of a K row per lane
  constexpr int kVb = kRow / 8 < 16 ? kRow / 8 : 16;      // bytes of a V chunk
  constexpr int kVc = kRow / 8 / kVb;                     // V chunks of a row per lane
  constexpr int kVe = kVb / kElt;                         // values of a V chunk
  constexpr int kE = 16 / kElt;                           // values of a K chunk
  extern __shared__ __align__(128) unsigned char smem_raw[];
  float *sm_o = reinterpret_cast<float *>(smem_raw);                      // [4][16][D]
  float2 *sm_ml = reinterpret_cast<float2 *>(sm_o + 4 * 16 * D);          // [4][16]
  int64_t *cu = reinterpret_cast<int64_t *>(sm_ml + 4 * 16);              // [seqs + 1]

  scan_tiles(a, cu);
  __syncthreads();
  const AttnLine line(a.seqs, a.kv_heads, a.group, a.prefix_len);
  const int64_t in_prefix = (int64_t)line.prefix_items * line.prefix_tiles;
  const int64_t total = in_prefix + cu[a.seqs] * line.per_seq;
  if (blockIdx.x == 0)
    for (int s = threadIdx.x; s <= a.seqs; s += blockDim.x) a.cu[s] = cu[s];
  const int64_t ctas = line_ctas(gridDim.x, total);
  const int64_t begin = blockIdx.x < ctas ? total * blockIdx.x / ctas : total;
  const int64_t end = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : total;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  for (int64_t at = begin; at < end;) {
    // the item at this place of the line, and the tiles of it that are ours
    int64_t ordinal, item_begin, item_tiles;
    int h, row0, rows, seq;     // rows of queries: row0 .. row0 + rows of the item's row space
    int64_t len;
    const void *table;
    int64_t table_at;
    if (at < in_prefix) {
      ordinal = at / line.prefix_tiles;
      item_begin = ordinal * line.prefix_tiles;
      item_tiles = line.prefix_tiles;
      h = (int)(ordinal / line.row_tiles);
      row0 = (int)(ordinal - (int64_t)h * line.row_tiles) * 16;
      rows = min(16, a.seqs * a.group - row0);
      seq = 0;
      len = a.prefix_len;
      table = a.prefix_table;
      table_at = 0;
    } else {
      const int64_t u = at - in_prefix;
      int lo = 0, hi = a.seqs;
      while (lo < hi) {         // number of sequences that end at or before u
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] * line.per_seq <= u) lo = mid + 1; else hi = mid;
      }
      seq = lo;
      item_tiles = cu[seq + 1] - cu[seq];
      const int64_t v = u - cu[seq] * line.per_seq;
      const int hg = (int)(v / item_tiles);
      item_begin = in_prefix + cu[seq] * line.per_seq + hg * item_tiles;
      ordinal = line.prefix_items + (int64_t)seq * line.per_seq + hg;
      h = hg / line.own_tiles;
      row0 = (hg - h * line.own_tiles) * 16;
      rows = min(16, a.group - row0);
      len = own_length(a, seq, false);
      table = a.tables;
      table_at = (int64_t)seq * a.table_stride;
    }
    const int64_t stop = min(end, item_begin + item_tiles);
    const int64_t tile_a = at - item_begin, tile_b = stop - item_begin;

    // queries: rows g and g + 8, the chunks this lane also takes of K
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = row0 + g + 8 * half;
      const bool ok = g + 8 * half < rows;
      const int s = seq + (ok ? r / a.group : 0);
      const unsigned char *qp = a.q + s * a.q_seq + (int64_t)(h * a.group + (ok ? r % a.group : 0)) * a.q_head;
#pragma unroll
      for (int c = 0; c < kKc; ++c)
#pragma unroll
        for (int j = 0; j < kE / 8; ++j) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (ok) w = *reinterpret_cast<const uint4 *>(qp + ((c * 4 + t) * kE + j * 8) * 2);
          const int ks = c * (kE / 4) + j * 2;
          qf[ks][half] = w.x;
          qf[ks][half + 2] = w.y;
          qf[ks + 1][half] = w.z;
          qf[ks + 1][half + 2] = w.w;
        }
    }

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, ref = 0.f;
    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    for (int64_t tile = tile_a; tile < tile_b; ++tile) {
      const int64_t key0 = tile * kTileKeys + warp * 16;
      if (key0 >= len) continue;
      // where the lane's rows are: K of keys g and g + 8, V of keys 2t, 2t + 1, 2t + 8, 2t + 9
      auto locate = [&](int i, int64_t &page, uint32_t &row) -> bool {
        const int64_t key = key0 + i;
        if (key >= len) return false;
        const uint32_t b = a.block.div((uint32_t)key);
        const int64_t id = load_id(table, a.ids_are_int64, table_at + b);
        if (id < 0 || id >= a.num_blocks) {
          raise_status(HFK_DEV_BAD_DEVICE_BLOCK_ID);
          return false;
        }
        page = id * a.block_stride;
        row = ((uint32_t)key - b * a.block.d) * a.kv_heads + h;
        return true;
      };
      uint4 kr[2][kKc], vr[4][kVc];
      float sk[4], sv[4];
      bool live[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int64_t page = 0;
        uint32_t row = 0;
        const bool ok = locate(g + 8 * i, page, row);
        const unsigned char *p = a.k_cache + page + (int64_t)row * kRow;
#pragma unroll
        for (int c = 0; c < kKc; ++c) {
          kr[i][c] = make_uint4(0, 0, 0, 0);
          if (ok) kr[i][c] = *reinterpret_cast<const uint4 *>(p + (c * 4 + t) * 16);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int64_t page = 0;
        uint32_t row = 0;
        live[i] = locate(2 * t + (i & 1) + 8 * (i >> 1), page, row);
        const unsigned char *p = a.v_cache + page + (int64_t)row * kRow;
        sk[i] = sv[i] = 0.f;
        if (kFmt != kFmtRaw && live[i]) {
          sk[i] = reinterpret_cast<const float *>(a.k_cache + page + a.scales_at)[row];
          sv[i] = reinterpret_cast<const float *>(a.v_cache + page + a.scales_at)[row];
        }
#pragma unroll
        for (int c = 0; c < kVc; ++c) {
          vr[i][c] = make_uint4(0, 0, 0, 0);
          if (live[i]) {
            if constexpr (kVb == 16) {
              vr[i][c] = *reinterpret_cast<const uint4 *>(p + (c * 8 + g) * 16);
            } else {
              const uint2 w = *reinterpret_cast<const uint2 *>(p + (c * 8 + g) * 8);
              vr[i][c].x = w.x;
              vr[i][c].y = w.y;
            }
          }
        }
      }

      // scores of 16 rows and 16 keys: s[n][0..1] row g, s[n][2..3] row g + 8, keys 8n + 2t, 8n + 2t + 1
      float s[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < kKc; ++c) {
          const uint32_t w[4] = {kr[n][c].x, kr[n][c].y, kr[n][c].z, kr[n][c].w};
          if constexpr (kFmt == kFmtRaw) {
            mma16816<T>(s[n], qf[2 * c], w[0], w[1]);
            mma16816<T>(s[n], qf[2 * c + 1], w[2], w[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t b0, b1;
              codes_to_pairs<T, kFmt>(w[i], b0, b1);
              mma16816<T>(s[n], qf[4 * c + i], b0, b1);
            }
          }
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * n + e;
          const float f = kFmt == kFmtRaw ? a.scale_log2 : a.scale_log2 * sk[i];
          s[n][e] = live[i] ? s[n][e] * f : -INFINITY;
          s[n][2 + e] = live[i] ? s[n][2 + e] * f : -INFINITY;
          top[0] = fmaxf(top[0], s[n][e]);
          top[1] = fmaxf(top[1], s[n][2 + e]);
        }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      }
      // fp16 weights of an 8-bit cache: weight * scale may leave fp16's range, so o is kept in units of the
      // largest scale of a value so far
      float grow = 1.f, unit = 1.f;
      if (kFmt != kFmtRaw && std::is_same<T, __half>::value) {
        float big = max_nan(max_nan(sv[0], sv[1]), max_nan(sv[2], sv[3]));
        big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const float next = max_nan(ref, big);
        grow = next == ref || next == 0.f ? 1.f : ref / next;
        unit = next == 0.f ? 0.f : 1.f / next;
        ref = next;
      }
      float alpha[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float next = fmaxf(m[r], top[r]);
        const float safe = next == -INFINITY ? 0.f : next;
        alpha[r] = ex2(m[r] - safe);
        m[r] = next;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = ex2(s[n][2 * r + e] - safe);
            sum += p;
            s[n][2 * r + e] = kFmt == kFmtRaw ? p : p * (sv[2 * n + e] * unit);
          }
        l[r] = l[r] * alpha[r] + sum;
        alpha[r] *= grow;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][0] *= alpha[0];
          o[j][1] *= alpha[0];
          o[j][2] *= alpha[1];
          o[j][3] *= alpha[1];
        }
      }
      const uint32_t pf[4] = {Pair<T>::pack(s[0][0], s[0][1]), Pair<T>::pack(s[0][2], s[0][3]),
                              Pair<T>::pack(s[1][0], s[1][1]), Pair<T>::pack(s[1][2], s[1][3])};
      // o column q (0..7) of block j = c * kVe + e holds value (c * 8 + q) * kVe + e of the head
#pragma unroll
      for (int c = 0; c < kVc; ++c) {
        const uint32_t w0[4] = {vr[0][c].x, vr[0][c].y, vr[0][c].z, vr[0][c].w};
        const uint32_t w1[4] = {vr[1][c].x, vr[1][c].y, vr[1][c].z, vr[1][c].w};
        const uint32_t w2[4] = {vr[2][c].x, vr[2][c].y, vr[2][c].z, vr[2][c].w};
        const uint32_t w3[4] = {vr[3][c].x, vr[3][c].y, vr[3][c].z, vr[3][c].w};
#pragma unroll
        for (int i = 0; i < kVb / 4; ++i) {
          if constexpr (kFmt == kFmtRaw) {
            mma16816<T>(o[c * kVe + 2 * i], pf, __byte_perm(w0[i], w1[i], 0x5410), __byte_perm(w2[i], w3[i], 0x5410));
            mma16816<T>(o[c * kVe + 2 * i + 1], pf, __byte_perm(w0[i], w1[i], 0x7632), __byte_perm(w2[i], w3[i], 0x7632));
          } else {
            uint32_t x0, x1, x2, x3, y0, y1, y2, y3;
            codes_to_pairs<T, kFmt>(__byte_perm(w0[i], w1[i], 0x5140), x0, x1);
            codes_to_pairs<T, kFmt>(__byte_perm(w0[i], w1[i], 0x7362), x2, x3);
            codes_to_pairs<T, kFmt>(__byte_perm(w2[i], w3[i], 0x5140), y0, y1);
            codes_to_pairs<T, kFmt>(__byte_perm(w2[i], w3[i], 0x7362), y2, y3);
            mma16816<T>(o[c * kVe + 4 * i], pf, x0, y0);
            mma16816<T>(o[c * kVe + 4 * i + 1], pf, x1, y1);
            mma16816<T>(o[c * kVe + 4 * i + 2], pf, x2, y2);
            mma16816<T>(o[c * kVe + 4 * i + 3], pf, x3, y3);
          }
        }
      }
    }

    // join the four warps
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t == 0) sm_ml[warp * 16 + g + 8 * r] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    float big[2], factor[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      big[r] = -INFINITY;
      for (int w = 0; w < 4; ++w) big[r] = fmaxf(big[r], sm_ml[w * 16 + g + 8 * r].x);
      factor[r] = big[r] == -INFINITY ? 0.f : ex2(m[r] - big[r]);
      if (kFmt != kFmtRaw && std::is_same<T, __half>::value) factor[r] *= ref;
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      const int c = j / kVe, e = j % kVe;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          sm_o[(warp * 16 + g + 8 * r) * D + (c * 8 + 2 * t + x) * kVe + e] = o[j][2 * r + x] * factor[r];
    }
    __syncthreads();
    const int64_t part = blockIdx.x + ordinal;
    for (int i = threadIdx.x; i < rows * D; i += 128)
      a.part_o[part * 16 * D + i] = (sm_o[i] + sm_o[16 * D + i]) + (sm_o[32 * D + i] + sm_o[48 * D + i]);
    if (threadIdx.x < rows) {
      float mm = -INFINITY, ll = 0.f;
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm_ml[w * 16 + threadIdx.x].x);
      for (int w = 0; w < 4; ++w) {
        const float2 x = sm_ml[w * 16 + threadIdx.x];
        ll += mm == -INFINITY ? x.y : x.y * ex2(x.x - mm);
      }
      a.part_ml[part * 16 + threadIdx.x] = make_float2(mm, ll);
    }
    __syncthreads();
    at = stop;
  }
}

// Joins the parts of every row; one warp a row.  Up to three lists of parts: of the prefix's item and of the
// sequence's item on the line, and of the prefix's runs from prefix_tensor_kernel.
struct JoinArgs {
  AttnArgs a;               // as the line's kernel had it: prefix_len 0 where the prefix went to the tensor kernel
  int grid;                 // CTAs of the line, 0: no line
  int splits, rows;         // of the tensor kernel; splits 0: not used
  const float2 *prefix_ml;
  const float *prefix_o;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) shared_prefix_join_kernel(const __grid_constant__ JoinArgs args) {
  const AttnArgs &a = args.a;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int q_heads = a.kv_heads * a.group;
  if (row >= a.seqs * q_heads) return;
  const int s = row / q_heads, head = row - s * q_heads, h = head / a.group, g = head - h * a.group;
  // list k: parts at ml[k] + step_ml i, o[k] + step_o i, i < count[k]
  int64_t count[3] = {0, 0, 0};
  const float2 *ml[3] = {nullptr, nullptr, nullptr};
  const float *o_at[3] = {nullptr, nullptr, nullptr};
  if (args.grid > 0) {
    const AttnLine line(a.seqs, a.kv_heads, a.group, a.prefix_len);
    const int64_t in_prefix = (int64_t)line.prefix_items * line.prefix_tiles;
    const int64_t total = in_prefix + a.cu[a.seqs] * line.per_seq;
    const int64_t ctas = line_ctas(args.grid, total);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int64_t item, from, tiles;
      int place;
      if (k == 0) {
        const int r = s * a.group + g;
        item = (int64_t)h * line.row_tiles + r / 16;
        place = r % 16;
        from = item * line.prefix_tiles;
        tiles = line.prefix_tiles;
      } else {
        const int hg = h * line.own_tiles + g / 16;
        place = g % 16;
        tiles = a.cu[s + 1] - a.cu[s];
        from = in_prefix + a.cu[s] * line.per_seq + hg * tiles;
        item = line.prefix_items + (int64_t)s * line.per_seq + hg;
      }
      if (tiles > 0) {
        // CTA c has [total c / ctas, total (c+1) / ctas): the one with tile x is floor((ctas (x+1) - 1) / total)
        const int64_t first = (ctas * (from + 1) - 1) / total, last = (ctas * (from + tiles) - 1) / total;
        count[k] = last - first + 1;
        ml[k] = a.part_ml + (first + item) * 16 + place;
        o_at[k] = a.part_o + ((first + item) * 16 + place) * D;
      }
    }
  }
  const int64_t step[3] = {16, 16, (int64_t)a.kv_heads * args.rows};
  if (args.splits > 0) {
    const int64_t r = (int64_t)h * args.rows + s * a.group + g;
    count[2] = args.splits;
    ml[2] = args.prefix_ml + r;
    o_at[2] = args.prefix_o + r * D;
  }
  float big = -INFINITY;
#pragma unroll
  for (int k = 0; k < 3; ++k)
    for (int64_t i = lane; i < count[k]; i += 32) big = fmaxf(big, ml[k][i * step[k]].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
  constexpr int kPer = D / 32;
  float l = 0.f, o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = 0.f;
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll 4
    for (int64_t i = 0; i < count[k]; ++i) {
      const float2 x = ml[k][i * step[k]];
      const float f = big == -INFINITY ? 1.f : ex2(x.x - big);
      l += x.y * f;
      const float *src = o_at[k] + i * step[k] * D + lane * kPer;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] += src[e] * f;
    }
  const float inv = l == 0.f ? 0.f : 1.f / l;   // a NaN stays
  unsigned char *dst = a.out + s * a.out_seq + (int64_t)head * a.out_head + lane * kPer * 2;
#pragma unroll
  for (int i = 0; i < kPer; i += 2)
    *reinterpret_cast<uint32_t *>(dst + i * 2) = Pair<T>::pack(o[i] * inv, o[i + 1] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[(int64_t)s * q_heads + head] = l == 0.f ? -INFINITY : kLn2 * (big + log2f(l));
}

}  // namespace hfk
