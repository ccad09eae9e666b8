// The shared prefix on the 5th-generation tensor cores: from a few dozen rows of queries on, reading the prefix once
// for all of them is a pair of matrix products (queries x keys, weights x values) with a softmax between.
//
// A CTA takes up to 256 rows of one K/V head (two tiles of 128, one TMEM lane a row) against a run of key tiles
// of 128, and leaves a partial result (m, l, o).  Four groups of four warps:
//   0-3, 4-7  softmax of tile 0 and of tile 1, 32 rows a warp
//   8-11      bring K and V tiles into shared memory (asynchronous copies; 8-bit codes are widened on the way)
//   12        issues the matrix products (13-15 only bring their registers)
// A thread starts with 128 registers; the warps that widen codes hold two tiles of them and would spill (to L2: shared
// memory leaves no L1), so the groups split the registers 144 + 144 + 176 + 48 = 4 x 128.
// TMEM: scores of the two tiles (128 columns each), o of the two tiles (head_dim columns each).  The 16-bit weights
// take the place of the scores they came from, and the second product reads them from there.  While one tile is
// in its softmax, the tensor cores work on the other: per 128 keys and tile, at head_dim 128, both products take about
// 1024 clocks of the tensor cores and the 128 x 128 exponentials 1024 clocks of the special function units.
//
// Measured: 8 items of 256 rows against 32768 keys, e4m3 (34 GFLOP): 58 to 59 us, of which 12 pass before the first tile's
// scores and behind the last one's, 33 with the softmax left out (a tile's two products take 1450 clocks, the operands
// from shared memory being at its bandwidth), the rest is softmax that nothing hides.  Steps to there: 105 us at first;
// 92 with the queries loaded a row's worth at a time and the parts' rows leaving as bulk copies; 64 with packed fp32
// arithmetic; 57 with short loops instead of unrolled ones (warps waited for instructions) and four rows a thread; 58 with
// powers of two and origins of each row's own and one barrier earlier.
//
// o is rescaled only where a row's maximum rises by more than 2^8 above the one in use: weights up to 2^8 are as
// exact as weights up to 1, so nothing is lost.  Of an 8-bit cache also where a row's largest weight times scale rises above
// what fp16 holds (e); both are looked at in one vote, so a tile in which nothing moves pays two additions a row.
//
// Operand layouts: rows of 128 bytes (64 values), 16-byte chunks XORed with the row number mod 8 ("128-byte swizzle"),
// head_dim 128 as two such halves.  The same bytes serve K (rows = keys, read along the row) and V (rows = keys, read
// across the rows: the transposed form of the operand).
#pragma once

#include "bounded_wait.h"
#include "shared_prefix_attention.cuh"

namespace hfk {

struct PrefixTensorArgs {
  AttnArgs a;
  int rows;          // seqs * group
  int row_blocks;    // ceil(rows / 256)
  int splits;        // runs the prefix's key tiles are cut into
  int negate;        // scale < 0: queries are negated, so the maximum of the scores is that of the products
  float2 *part_ml;   // [splits][kv_heads * rows]
  float *part_o;     // [splits][kv_heads * rows][head_dim]
};

constexpr int kPtThreads = 512, kPtRows = 128, kPtKeys = 128, kPtStages = 4, kPtMeta = 4;
constexpr int kSameScale = 10, kSharedBack = 40;   // powers of two, of bf16 queries that become fp16 numbers
constexpr int kSameValues = 4;                     // ... and of the scales of a tile's values

template <int D>
struct PrefixSmem {
  // at the end the first bytes take the 256 rows of o, D * 4 + 16 bytes each
  static constexpr int kTile = kPtKeys * D * 2;  // bytes of a tile of queries, keys or values
  unsigned char q[2][kTile];
  unsigned char ring[kPtStages][kTile];          // K of tile i in stage 2 (i % 2), V in the next
  int64_t off[kPtMeta][kPtKeys];                 // byte offset of a key's row, -1: leave out
  alignas(16) float sk[kPtMeta][kPtKeys];         // scales of keys (times scale * log2 e) and of values
  alignas(16) float sv[kPtMeta][kPtKeys];
  alignas(16) uint32_t sv_high[kPtMeta][4];       // bits of the largest and least |scale of a value| of 32 keys that count
  alignas(16) uint32_t sv_low[kPtMeta][4];
  uint32_t valid[kPtMeta][4];
  uint64_t full[kPtStages], empty[kPtStages], meta[kPtMeta], s_full[2], p_full[2], o_full, q_full;
  uint32_t tmem;
  int failed;
  uint32_t q_top, q_low;                         // bits of the largest finite |query| of any row, and of the row whose is least
  float q_back;                                  // what undoes the queries' scaling, the part that all rows share
};
static_assert(256 * (128 * 4 + 16) <= 2 * PrefixSmem<128>::kTile + kPtStages * PrefixSmem<128>::kTile, "o fits");
static_assert(256 * (64 * 4 + 16) <= 2 * PrefixSmem<64>::kTile + kPtStages * PrefixSmem<64>::kTile, "o fits");

// ---- tcgen05 ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Products and commits are issued by one lane (`leader`) of a warp whose lanes all run the code around them: operands
// have to be in uniform registers, and in a branch of one lane every instruction would first move them there (more
// registers, and spills).
__device__ __forceinline__ uint32_t elect_leader() {
  uint32_t leader;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
  return leader;
}
__device__ __forceinline__ void tc_commit(uint64_t *bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_addr(bar)),
      "r"(leader)
      : "memory");
}
// Shared-memory operand, 128-byte swizzle: start, distance of 64-value blocks (only where the operand is read across
// its rows), distance of 8-row groups (1024 bytes).
__device__ __forceinline__ uint64_t tc_operand(uint32_t addr, uint32_t block_bytes) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(block_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// fp32 accumulators, M = 128; b_across: B is read across its rows.
template <typename M>
__device__ __forceinline__ constexpr uint32_t tc_instruction(int n, bool b_across) {
  const uint32_t type = std::is_same<M, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_across ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t instr, bool add, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(instr), "r"((uint32_t)add), "r"(leader)
      : "memory");
}
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tc_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr));
}
// 32 columns of 16 lanes in the layout of a matrix product's result: register 4n + 2r + x of thread 4g + t is column
// 8n + 2t + x of lane g + 8r; and the store of pairs packed to 16 columns: register 2n + r is column 4n + t of lane g + 8r.
__device__ __forceinline__ void tc_load_block(uint32_t addr, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
}
__device__ __forceinline__ void tc_store_pairs(uint32_t addr, const uint32_t *r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
               "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr));
}
// For one tc_load32, whose registers nothing may read earlier; other memory is free to move across.
__device__ __forceinline__ void tc_wait_load(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                 "+r"(r[31]));
}
__device__ __forceinline__ void tc_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte of 16-byte chunk `chunk` of row `row` in a tile (8 chunks to a 128-byte row, halves behind each other).
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
  return (uint32_t)((chunk >> 3) * (kPtKeys * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// ---- the softmax's arithmetic, two columns an instruction ---------------------------------------------------------
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 of_pair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// A sum that no multiplication before it is drawn into (mul.rn.f32x2 and add.rn.f32x2 became one fma): rounded towards zero.
__device__ __forceinline__ uint64_t add2_apart(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// o of this warp's rows times a factor of each row
template <int D>
__device__ __forceinline__ void rescale(uint32_t o_at, float factor) {
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t s[32];
    tc_load32(o_at + c * 32, s);
    tc_wait_load(s);
#pragma unroll
    for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * factor);
    tc_store32(o_at + c * 32, s);
  }
}

// Scores of keys that do not count become -inf (the last tile of the prefix, pages that are not there), and the others are
// multiplied by a factor of the row (1 but for queries of mixed magnitudes), so that what follows needs one form only:
// every copy of the code below costs instruction cache, and the kernel waited for instructions when it had four.
__device__ __forceinline__ void amend_scores(uint32_t s_at, const uint32_t *valid, float factor) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t s[32];
    tc_load32(s_at + c * 32, s);
    tc_wait_load(s);
    const uint32_t bits = valid[c];
#pragma unroll
    for (int e = 0; e < 32; ++e) s[e] = bits >> e & 1 ? __float_as_uint(__uint_as_float(s[e]) * factor) : 0xff800000u;
    tc_store32(s_at + c * 32, s);
  }
  tc_wait_store();
}

// A warp's 32 rows of scores, 32 columns at a time: thread 4g + t has columns 8n + 2t, 8n + 2t + 1 (n < 4) of the four rows
// g + 8k, s[16 (k / 2) + 4n + 2 (k % 2)] and the next.  So a thread needs a quarter of the scales and uses each for four
// rows; with a row a thread, their loads from shared memory (512 bytes to the registers each, whatever they read) took
// longer than the exponentials.
constexpr uint32_t kUpperLanes = 16u << 16;
__device__ __forceinline__ void load_scores(uint32_t at, uint32_t (&s)[32]) {
  tc_load_block(at, s);
  tc_load_block(at + kUpperLanes, s + 16);
}

// Largest score of each of the four rows over the tile (in units of log2 e), -inf without a key.  (scale is not 0.)
template <int kFmt>
__device__ __forceinline__ void tile_max(uint32_t s_at, const float *sk, float scale, float (&top)[4]) {
  const int t2 = (threadIdx.x & 3) * 2;
  top[0] = top[1] = top[2] = top[3] = -INFINITY;
  uint32_t buf[2][32];                           // the next 32 columns are on their way while these are looked at
  auto look = [&](int c, const uint32_t (&s)[32]) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float2 f = make_float2(1.f, 1.f);
      if (kFmt != kFmtRaw) f = *reinterpret_cast<const float2 *>(sk + c * 32 + n * 8 + t2);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = 16 * (k >> 1) + 4 * n + 2 * (k & 1);
        float2 x = make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        if (kFmt != kFmtRaw) x = of_pair(mul2(pair_of(x.x, x.y), pair_of(f.x, f.y)));
        top[k] = fmaxf(top[k], fmaxf(x.x, x.y));
      }
    }
  };
  load_scores(s_at, buf[0]);
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    tc_wait_load(buf[0]);
    load_scores(s_at + (c + 1) * 32, buf[1]);
    look(c, buf[0]);
    tc_wait_load(buf[1]);
    if (c == 0) load_scores(s_at + 64, buf[0]);
    look(c + 1, buf[1]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
    top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2));
    if (kFmt == kFmtRaw) top[k] *= scale;
  }
}

// log2 of the largest weight times scale of a value, of each of the four rows over the tile: for tiles whose scales differ
// much (see below), so it is written for size.
__device__ __forceinline__ void tile_reach(uint32_t s_at, const float *sk, const float *sv, const float (&origin)[4], float (&reach)[4]) {
  const int t2 = (threadIdx.x & 3) * 2;
  reach[0] = reach[1] = reach[2] = reach[3] = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t s[32];
    load_scores(s_at + c * 32, s);
    tc_wait_load(s);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f = sk[c * 32 + n * 8 + t2 + x], log_sv = lg2(fabsf(sv[c * 32 + n * 8 + t2 + x]));   // a NaN is left out
#pragma unroll
        for (int k = 0; k < 4; ++k)
          reach[k] = fmaxf(reach[k], __fmul_rn(__uint_as_float(s[16 * (k >> 1) + 4 * n + 2 * (k & 1) + x]), f) - origin[k] + log_sv);
      }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    reach[k] = fmaxf(reach[k], __shfl_xor_sync(0xffffffffu, reach[k], 1));
    reach[k] = fmaxf(reach[k], __shfl_xor_sync(0xffffffffu, reach[k], 2));
  }
}

// Weights 2^(score - origin) of the tile's 128 keys, of an 8-bit cache times 2^e of the row and the values' scales, of an fp16
// cache times raw_shift, take the place of the scores (behind what has been read); adds this thread's columns of them,
// without these factors, to l.
// The score is rounded before the origin is taken off it, as it was when the origin was found: with one rounding for both the
// largest score of 2^28 would be up to 2^4 above its own origin, and its weight no fp16 number.
template <typename M, int kFmt>
__device__ __forceinline__ void tile_weights(uint32_t s_at, const float *sk, const float *sv, float scale, const float (&origin)[4],
                                             const float (&e)[4], float (&l)[4]) {
  const int t2 = (threadIdx.x & 3) * 2;
  const uint64_t factor = pair_of(scale, scale);
  uint64_t total[4] = {0, 0, 0, 0}, minus[4], shift[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float f = ex2(e[k]);
    minus[k] = pair_of(-origin[k], -origin[k]);
    shift[k] = kFmt == kFmtRaw ? pair_of(raw_shift<M>(), raw_shift<M>()) : pair_of(f, f);
  }
  uint32_t buf[2][32];
  auto weigh = [&](int c, const uint32_t (&s)[32]) {
    uint32_t w[16];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float2 f, g;
      if (kFmt != kFmtRaw) {
        f = *reinterpret_cast<const float2 *>(sk + c * 32 + n * 8 + t2);
        g = *reinterpret_cast<const float2 *>(sv + c * 32 + n * 8 + t2);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = 16 * (k >> 1) + 4 * n + 2 * (k & 1);
        const uint64_t score = pair_of(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        const float2 x = of_pair(add2_apart(mul2(score, kFmt == kFmtRaw ? factor : pair_of(f.x, f.y)), minus[k]));
        uint64_t p = pair_of(ex2(x.x), ex2(x.y));
        total[k] = add2(total[k], p);
        if (kFmt != kFmtRaw || raw_shift<M>() != 1.f) p = mul2(p, shift[k]);
        if (kFmt != kFmtRaw) p = mul2(p, pair_of(g.x, g.y));
        const float2 y = of_pair(p);
        w[8 * (k >> 1) + 2 * n + (k & 1)] = Pair<M>::pack(y.x, y.y);
      }
    }
    tc_store_pairs(s_at + c * 16, w);
    tc_store_pairs(s_at + kUpperLanes + c * 16, w + 8);
  };
  load_scores(s_at, buf[0]);
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    tc_wait_load(buf[0]);
    load_scores(s_at + (c + 1) * 32, buf[1]);    // columns that the weights of chunk c do not reach
    weigh(c, buf[0]);
    tc_wait_load(buf[1]);
    if (c == 0) load_scores(s_at + 64, buf[0]);
    weigh(c + 1, buf[1]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 x = of_pair(total[k]);
    l[k] += x.x + x.y;
  }
}

template <typename T, int kFmt, int D>
__global__ void __launch_bounds__(kPtThreads, 1) prefix_tensor_kernel(const __grid_constant__ PrefixTensorArgs args) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  using Smem = PrefixSmem<D>;
  // operands want 1024-byte alignment
  Smem &sm = *reinterpret_cast<Smem *>(smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023));
  const AttnArgs &a = args.a;
  constexpr bool kWide = kFmt != kFmtRaw;
  using M = Operand<T, kFmt>;
  constexpr bool kScaleQ = kWide && !std::is_same<T, M>::value;  // bf16 queries become fp16
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // uniform for the compiler

  launch_next();
  const int split = blockIdx.x % args.splits;
  const int item = blockIdx.x / args.splits;
  const int h = item / args.row_blocks;
  const int row0 = (item - h * args.row_blocks) * 256;
  const int rows = min(256, args.rows - row0);
  const int tiles = rows > kPtRows ? 2 : 1;
  const int key_tiles = (a.prefix_len + kPtKeys - 1) / kPtKeys;
  const int first = (int)((int64_t)key_tiles * split / args.splits);
  const int n = (int)((int64_t)key_tiles * (split + 1) / args.splits) - first;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kPtStages; ++i) {
      mbar_init(&sm.full[i], 128);
      mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < kPtMeta; ++i) mbar_init(&sm.meta[i], 128);
    for (int j = 0; j < 2; ++j) {
      mbar_init(&sm.s_full[j], 1);
      mbar_init(&sm.p_full[j], 128);
    }
    mbar_init(&sm.o_full, 1);
    mbar_init(&sm.q_full, tiles * 128);
    sm.failed = 0;
    sm.q_top = 0;
    sm.q_low = 0xffffffffu;
    sm.q_back = 1.f;
    mbar_fence_init();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t *>(&sm.tmem), 0);
  auto give_up = [&]() {                         // and all the others with this thread
    raise_status(HFK_DEV_WAIT_TIMEOUT);
    *reinterpret_cast<volatile int *>(&sm.failed) = 1;
  };
  auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
    const WaitEnd end = bounded_wait([=] { return mbar_try_wait(bar, parity); }, [] { return global_timer_ns(); },
                                     [&] { return *reinterpret_cast<volatile int *>(&sm.failed) != 0; }, kWaitLimitNs);
    if (end == WaitEnd::kRanOut) give_up();
    return end == WaitEnd::kDone;
  };

  auto wait_warp = [&](uint64_t *bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };

  if (warp >= 8 && warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    // ---------------------------------------------------------------- loads ---
    const int p = threadIdx.x - 256;
    // key p of a tile: where its row is
    auto page_of = [&](int i) -> int64_t {
      const int64_t key = (int64_t)(first + i) * kPtKeys + p;
      return i < n && key < a.prefix_len ? load_id(a.prefix_table, a.ids_are_int64, a.block.div((uint32_t)key)) : -1;
    };
    // ... and what it is multiplied by: loaded a tile ahead of its use
    struct Key {
      int64_t off;
      float sk, sv;
      bool ok;
    };
    auto key_of = [&](int i, int64_t id) -> Key {
      const int64_t key = (int64_t)(first + i) * kPtKeys + p;
      const bool inside = i < n && key < a.prefix_len;
      Key k;
      k.ok = inside && id >= 0 && id < a.num_blocks;
      if (inside && !k.ok) raise_status(HFK_DEV_BAD_DEVICE_BLOCK_ID);
      const uint32_t row = ((uint32_t)key - a.block.div((uint32_t)key) * a.block.d) * a.kv_heads + h;
      k.off = k.ok ? id * a.block_stride + (int64_t)row * (D * (kWide ? 1 : 2)) : -1;
      k.sk = k.sv = 0.f;
      if (kWide && k.ok) {
        k.sk = reinterpret_cast<const float *>(a.k_cache + id * a.block_stride + a.scales_at)[row];
        k.sv = reinterpret_cast<const float *>(a.v_cache + id * a.block_stride + a.scales_at)[row];
      }
      return k;
    };
    float factor = a.scale_log2;                 // of the scores
    // The rows' places go out first, so that the copies can start; the scales and which keys count follow.
    auto write_places = [&](int i, const Key &k) { sm.off[i % kPtMeta][p] = k.off; };
    auto write_scales = [&](int i, const Key &k) {
      const int m = i % kPtMeta;
      if (kWide) {
        sm.sk[m][p] = k.ok ? k.sk * factor : 1.f;   // its score is -inf, and -inf * 0 would be NaN
        sm.sv[m][p] = k.sv;
      }
      const uint32_t word = __ballot_sync(0xffffffffu, k.ok);
      if (lane == 0) sm.valid[m][p >> 5] = word;
      if (kWide) {
        const uint32_t bits = __float_as_uint(k.sv) & 0x7fffffffu;
        const uint32_t high = __reduce_max_sync(0xffffffffu, bits), low = __reduce_min_sync(0xffffffffu, k.ok ? bits : 0x7f800000u);
        if (lane == 0) {
          sm.sv_high[m][p >> 5] = high;
          sm.sv_low[m][p >> 5] = low;
        }
      }
      mbar_arrive(&sm.meta[m]);
    };
    auto producers = [&]() {
      __syncwarp();
      asm volatile("bar.sync 1, 128;" ::: "memory");
    };
    Key key = key_of(0, page_of(0));
    int64_t next = page_of(1);
    if constexpr (!kWide) {
      constexpr int kChunks = D / 8;             // 16-byte chunks of a row
      constexpr int kRowsPass = 128 / kChunks;   // rows of a pass over the 128 threads
      const int chunk = p % kChunks, row_in = p / kChunks;
      int pending = -1;                          // stage whose copies are in flight and not yet announced
      auto announce = [&]() {
        fence_async_proxy();
        mbar_arrive(&sm.full[pending]);
      };
      bool ok = true;                            // after a wait that ran out the warps still meet at the barriers
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        write_places(i, key);
        write_scales(i, key);
        key = key_of(i + 1, next);
        next = page_of(i + 2);
        producers();
#pragma unroll 1
        for (int v = 0; v < 2 && ok; ++v) {
          const int stage = (i & 1) * 2 + v;
          const uint32_t parity = ((i >> 1) & 1) ^ 1;
          if (!mbar_try_wait(&sm.empty[stage], parity)) {   // nothing free: what has arrived goes out first
            if (pending >= 0) {
              cp_async_wait<0>();
              announce();
              pending = -1;
            }
            ok = wait(&sm.empty[stage], parity);
            if (!ok) break;
          }
          const unsigned char *cache = v ? a.v_cache : a.k_cache;
          const uint32_t base = smem_addr(sm.ring[stage]);
#pragma unroll
          for (int r = 0; r < kPtKeys; r += kRowsPass) {
            const int64_t off = sm.off[i % kPtMeta][r + row_in];
            cp_async16(base + tile_at(r + row_in, chunk), cache + (off < 0 ? 0 : off) + chunk * 16, off >= 0);
          }
          cp_async_commit();
          if (pending >= 0) {
            cp_async_wait<1>();
            announce();
          }
          pending = stage;
        }
      }
      cp_async_wait<0>();
      if (pending >= 0) announce();
    } else {
      // A thread holds the codes of its next K and V tiles while it widens the ones before: each has a whole tile's time to
      // arrive.  Eight lanes take four chunks of two neighbouring rows, so that what they write hits eight bank groups.
      constexpr int kChunks = D / 16;            // 16-byte chunks of codes of a row
      constexpr int kRowsPass = 128 / kChunks;
      constexpr int kPasses = kPtKeys / kRowsPass;
      const int chunk = D == 128 ? (lane & 3) + ((lane >> 3) & 1) * 4 : lane & 3;
      const int row_in = D == 128 ? (warp - 8) * 4 + ((lane >> 2) & 1) + (lane >> 4) * 2 : (warp - 8) * 8 + (lane >> 2);
      uint4 codes[2][kPasses];
      auto fetch = [&](int i, auto which) {
        constexpr int v = decltype(which)::value;
        const unsigned char *cache = v ? a.v_cache : a.k_cache;
#pragma unroll
        for (int r = 0; r < kPasses; ++r) {
          const int64_t off = sm.off[i % kPtMeta][r * kRowsPass + row_in];
          codes[v][r] = make_uint4(0, 0, 0, 0);
          if (off >= 0) codes[v][r] = *reinterpret_cast<const uint4 *>(cache + off + chunk * 16);
        }
      };
      bool ok = true;                            // after a wait that ran out the warps still meet at the barriers
      auto widen = [&](int i, auto which) {
        constexpr int v = decltype(which)::value;
        const int stage = (i & 1) * 2 + v;
        if (ok) ok = wait(&sm.empty[stage], ((i >> 1) & 1) ^ 1);
        if (!ok) return;
        unsigned char *ring = sm.ring[stage];
#pragma unroll
        for (int r = 0; r < kPasses; ++r) {
          const uint32_t w[4] = {codes[v][r].x, codes[v][r].y, codes[v][r].z, codes[v][r].w};
          uint32_t x[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) codes_to_pairs<kFmt>(w[k], x[2 * k], x[2 * k + 1]);
          const int row = r * kRowsPass + row_in;
          *reinterpret_cast<uint4 *>(ring + tile_at(row, 2 * chunk)) = make_uint4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<uint4 *>(ring + tile_at(row, 2 * chunk + 1)) = make_uint4(x[4], x[5], x[6], x[7]);
        }
        fence_async_proxy();
        mbar_arrive(&sm.full[stage]);
      };
      constexpr std::integral_constant<int, 0> kK{};
      constexpr std::integral_constant<int, 1> kV{};
      // `key` and `next` run ahead.  The places and scales of tile i + 2 take those of tile i - 2: its rows were fetched two
      // barriers ago, and a thread that found its V stage free again knows that the softmax is done with it.  They are written
      // ahead of the barrier of tile i, behind which every warp fetches the rows of all of them.
      write_places(0, key);
      producers();
      fetch(0, kK);
      fetch(0, kV);
      const Key then = key_of(1, next);
      next = page_of(2);
      if (kScaleQ && wait(&sm.q_full, 0)) factor *= *reinterpret_cast<volatile float *>(&sm.q_back);
      write_scales(0, key);
      write_places(1, then);
      write_scales(1, then);
      producers();
      key = key_of(2, next);
      next = page_of(3);
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        widen(i, kK);
        if (i + 1 < n) fetch(i + 1, kK);
        widen(i, kV);
        if (i + 1 < n) fetch(i + 1, kV);
        write_places(i + 2, key);
        write_scales(i + 2, key);
        producers();
        key = key_of(i + 3, next);
        next = page_of(i + 4);
      }
    }
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    // ------------------------------------------------------------- products ---
    if (warp == 12 && n > 0) {
      const uint32_t leader = elect_leader();
      constexpr uint32_t kScores = tc_instruction<M>(kPtKeys, false), kValues = tc_instruction<M>(D, true);
      bool ok = wait_warp(&sm.q_full, 0);
      auto values = [&](int j, int i) {          // o_j += weights_j . V_i
        const uint64_t v = tc_operand(smem_addr(sm.ring[(i & 1) * 2 + 1]), kPtKeys * 128);
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < kPtKeys / 16; ++k)   // 16 keys: 16 rows of 128 bytes
          tc_mma_ts(tmem + 256 + j * D, tmem + j * 128 + k * 8, v + k * (2048 >> 4), kValues, i > 0 || k > 0, leader);
      };
      for (int i = 0; i < n && ok; ++i) {
        const int stage = (i & 1) * 2;
        ok = wait_warp(&sm.full[stage], (i >> 1) & 1);
        if (ok && i > 0) ok = wait_warp(&sm.full[((i - 1) & 1) * 2 + 1], ((i - 1) >> 1) & 1);
        const uint64_t kk = tc_operand(smem_addr(sm.ring[stage]), 16);
        for (int j = 0; j < tiles && ok; ++j) {
          if (i > 0) {
            ok = wait_warp(&sm.p_full[j], (i - 1) & 1);
            if (!ok) break;
            values(j, i - 1);
          }
          tc_fence_after();
          const uint64_t q = tc_operand(smem_addr(sm.q[j]), 16);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {     // 16 values of each row: 32 bytes on, or the other half
            const uint32_t at = ((k >> 2) * (kPtKeys * 128) + (k & 3) * 32) >> 4;
            tc_mma_ss(tmem + j * 128, q + at, kk + at, kScores, k > 0, leader);
          }
          tc_commit(&sm.s_full[j], leader);
        }
        if (!ok) break;
        tc_commit(&sm.empty[stage], leader);
        if (i > 0) tc_commit(&sm.empty[((i - 1) & 1) * 2 + 1], leader);
      }
      if (ok) ok = wait_warp(&sm.full[((n - 1) & 1) * 2 + 1], ((n - 1) >> 1) & 1);
      for (int j = 0; j < tiles && ok; ++j) {
        ok = wait_warp(&sm.p_full[j], (n - 1) & 1);
        if (ok) values(j, n - 1);
      }
      // also after a failure: the products that were issued have read shared memory and written TMEM before the CTA gives them up
      tc_commit(&sm.o_full, leader);
      if (!drain([&] { return mbar_try_wait(&sm.o_full, 0); }, [] { return global_timer_ns(); }, kWaitLimitNs)) give_up();
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    // -------------------------------------------------------------- softmax ---
    if (warp / 4 < tiles) {
    const int j = warp / 4;
    const uint32_t lanes = (uint32_t)(warp % 4) << 21;   // first TMEM lane of this warp, in bits 16 and up
    const uint32_t s_at = tmem + j * 128 + lanes, o_at = tmem + 256 + j * D + lanes;
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, l[4] = {0.f, 0.f, 0.f, 0.f};
    float e[4] = {kMostShift, kMostShift, kMostShift, kMostShift};    // of an 8-bit cache: see kWeightHigh
    float origin[4] = {0.f, 0.f, 0.f, 0.f};      // m, 0 without a key
    const float scale = a.scale_log2 == 0.f ? kLeastScale : a.scale_log2;   // 0 times the -inf of a masked key is NaN
    bool ok = true, mixed = false;
    float row_back = 1.f;                        // of row `lane`: what undoes its own part of the queries' scaling
    {                                            // this warp's 32 rows of queries, zero behind the last one
      constexpr int kChunks = D / 8, kRowsPass = 32 / kChunks;
      const uint32_t flip = args.negate ? 0x80008000u : 0u;
      const int chunk = lane % kChunks;
      constexpr int kPasses = 32 / kRowsPass;
      uint4 w[kPasses];
#pragma unroll
      for (int k = 0; k < kPasses; ++k) {
        const int row = warp * 32 + k * kRowsPass + lane / kChunks, r = row0 + row;
        const int sq = (int)a.per_group.div((uint32_t)r);
        w[k] = make_uint4(0, 0, 0, 0);
        if (row < rows) w[k] = *reinterpret_cast<const uint4 *>(a.q + sq * a.q_seq + (int64_t)(h * a.group + r - sq * a.group) * a.q_head + chunk * 16);
      }
      if constexpr (kScaleQ) {
        // largest of each row: over its kChunks lanes, each of which ends with one row
        static_assert(kPasses == kChunks, "a row for each lane");
        float top[kPasses];
#pragma unroll
        for (int k = 0; k < kPasses; ++k)
          top[k] = fmaxf(fmaxf(largest_of_pair(w[k].x), largest_of_pair(w[k].y)), fmaxf(largest_of_pair(w[k].z), largest_of_pair(w[k].w)));
#pragma unroll
        for (int d = kChunks / 2; d > 0; d >>= 1)
#pragma unroll
          for (int k = 0; k < d; ++k) {
            const bool upper = (lane & d) != 0;
            const float theirs = __shfl_xor_sync(0xffffffffu, upper ? top[k] : top[k + d], d);
            top[k] = fmaxf(upper ? top[k + d] : top[k], theirs);
          }
        const uint32_t bits = __float_as_uint(top[0]);   // of row chunk * kRowsPass + lane / kChunks; rows of zeros do not count
        const uint32_t most = __reduce_max_sync(0xffffffffu, bits), least = __reduce_min_sync(0xffffffffu, bits == 0 ? 0xffffffffu : bits);
        if (lane == 0) {
          atomicMax(&sm.q_top, most);
          atomicMin(&sm.q_low, least);
        }
        asm volatile("bar.sync 2, %0;" ::"r"(tiles * 128) : "memory");
        const uint32_t high = *reinterpret_cast<volatile uint32_t *>(&sm.q_top), low = *reinterpret_cast<volatile uint32_t *>(&sm.q_low);
        // One power of two for all rows where the largest of each lies within 2^kSameScale of the others' (2^-25, half the least
        // fp16 step, is then 2^(kSameScale - 39) of a row's largest).  Else each row has its own, and amend_scores undoes it; up
        // to 2^kSharedBack stays in q_back, so that scores of huge queries stay finite as long as their products with the keys'
        // scales are.
        mixed = high > low && high - low > (uint32_t)kSameScale << 23;
        const int all = shift_to_half(__uint_as_float(high)), e = mixed ? shift_to_half(top[0]) : all;
        const int shared = mixed ? min(-all, kSharedBack) : -all;
        if (threadIdx.x == 0) sm.q_back = power_of_two(shared);
        // (a row 2^166 below the largest has no such factor: its scores are nothing, not 2^40 times what they are)
        const float undo = -e - shared < -126 ? 0.f : power_of_two(-e - shared);
        if (mixed) row_back = __shfl_sync(0xffffffffu, undo, (lane % kRowsPass) * kChunks + lane / kRowsPass);
        const float own = power_of_two(e);
#pragma unroll
        for (int k = 0; k < kPasses; ++k) {
          const float f = __shfl_sync(0xffffffffu, own, (lane & ~(kChunks - 1)) + k);
          w[k] = make_uint4(pair_to_half(w[k].x, f), pair_to_half(w[k].y, f), pair_to_half(w[k].z, f), pair_to_half(w[k].w, f));
        }
      }
#pragma unroll
      for (int k = 0; k < kPasses; ++k) {
        const int at = (warp % 4) * 32 + k * kRowsPass + lane / kChunks;
        *reinterpret_cast<uint4 *>(&sm.q[j][tile_at(at, chunk)]) = make_uint4(w[k].x ^ flip, w[k].y ^ flip, w[k].z ^ flip, w[k].w ^ flip);
      }
      fence_async_proxy();
      mbar_arrive(&sm.q_full);
      __syncwarp();
    }
    for (int i = 0; i < n; ++i) {
      const int mt = i % kPtMeta;
      ok = wait(&sm.meta[mt], (i / kPtMeta) & 1) && wait(&sm.s_full[j], i & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (mixed || (sm.valid[mt][0] & sm.valid[mt][1] & sm.valid[mt][2] & sm.valid[mt][3]) != 0xffffffffu) amend_scores(s_at, sm.valid[mt], row_back);
      float top[4];
      tile_max<kFmt>(s_at, sm.sk[mt], scale, top);
      // log2 of the largest weight times scale of a value is at most that of the largest weight plus that of the largest scale
      float log_sv = 0.f;
      uint32_t high = 0, low = 0;
      if constexpr (kWide) {
        const uint4 h4 = *reinterpret_cast<const uint4 *>(sm.sv_high[mt]), l4 = *reinterpret_cast<const uint4 *>(sm.sv_low[mt]);
        high = max(max(h4.x, h4.y), max(h4.z, h4.w));
        low = min(min(l4.x, l4.y), min(l4.z, l4.w));
        log_sv = lg2(__uint_as_float(high));     // a NaN is passed on by the product
      }
      bool move = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        move = move || top[k] > m[k] + 8.f;
        if (kWide) move = move || !(top[k] - origin[k] + log_sv + e[k] <= kWeightLimit);
      }
      if (__any_sync(0xffffffffu, move)) {       // the rows' maxima in use, and e; o and l follow
        float factor[4], reach[4];               // log2 of what o is multiplied by; log2 of the largest weight times scale
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          factor[k] = 0.f;
          if (top[k] > m[k] + 8.f) {
            factor[k] = m[k] - top[k];
            m[k] = top[k];
            l[k] *= ex2(factor[k]);
          }
          origin[k] = m[k] == -INFINITY ? 0.f : m[k];
          reach[k] = top[k] - origin[k] + log_sv;
        }
        if constexpr (kWide) {
          // where the scales of the tile lie within 2^kSameValues of each other that is at most so much too high
          if (high > low && high - low > (uint32_t)kSameValues << 23) tile_reach(s_at, sm.sk[mt], sm.sv[mt], origin, reach);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float before = e[k] - factor[k];
            e[k] = fminf(before, kMostShift);
            if (reach[k] + e[k] > kWeightLimit) e[k] = floorf(kWeightHigh - reach[k]);
            factor[k] = e[k] - before;
          }
        }
        if (i > 0) {
          float mine = 0.f;                      // factor of row `lane`: thread 4 (lane % 8) has it, number lane / 8
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float f = __shfl_sync(0xffffffffu, factor[k], (lane & 7) * 4);
            if (lane >> 3 == k) mine = f;
          }
          rescale<D>(o_at, ex2(mine));
        }
      }
      tile_weights<M, kFmt>(s_at, sm.sk[mt], sm.sv[mt], scale, origin, e, l);
      tc_wait_store();
      tc_fence_before();
      mbar_arrive(&sm.p_full[j]);
    }
    if (ok && n > 0) ok = wait(&sm.o_full, 0);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after();
      // The part's rows lie one behind the other, but a thread that stored its row would touch a line of its own with
      // every instruction: the row goes to shared memory (the tiles are done with; 16 bytes of skew a row, so eight
      // lanes hit eight bank groups) and from there as one copy.
      const int at = threadIdx.x, row = at;
      unsigned char *mine = sm.q[0] + at * (D * 4 + 16);
      const int64_t part = (int64_t)split * a.kv_heads * args.rows + (int64_t)h * args.rows + row0 + row;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
        const int r = warp * 32 + 8 * k + (lane >> 2);
        if ((lane & 3) == 0 && r < rows) args.part_ml[part - row + r] = make_float2(m[k], l[k]);
      }
      float back = kWide ? 1.f : 1.f / raw_shift<M>();   // brings o of row `lane` to the origin of l
      if constexpr (kWide) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float f = __shfl_sync(0xffffffffu, e[k], (lane & 7) * 4);
          if (lane >> 3 == k) back = ex2(-f);
        }
      }
      uint32_t buf[2][32];
      tc_load32(o_at, buf[0]);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t (&s)[32] = buf[c & 1];
        tc_wait_load(s);
        if (c + 1 < D / 32) tc_load32(o_at + (c + 1) * 32, buf[(c + 1) & 1]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<float4 *>(mine + c * 128 + i * 16) =
              make_float4(__uint_as_float(s[4 * i]) * back, __uint_as_float(s[4 * i + 1]) * back, __uint_as_float(s[4 * i + 2]) * back,
                          __uint_as_float(s[4 * i + 3]) * back);
      }
      fence_async_proxy();
      if (row < rows) {
        bulk_store(args.part_o + part * D, mine, D * 4);
        bulk_commit();
        bulk_wait_all();
      }
    }
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace hfk
