// The new tokens' K and V rows go to their pages (kv_write), optionally after the per-head norm and the
// position rotation of queries and keys (qk_norm_rope_write): one pass over the projections' output.
//
//   norm      y = x * rsqrt(mean(x^2) + eps) * w                       (where a weight is given)
//   rotation  (a, b) -> (a cos - b sin, b cos + a sin) of the first `rot` elements; the pair is (i, i + rot/2)
//             or, interleaved, (2i, 2i + 1); cos and sin come from a table indexed by the token's position
//   8-bit     scale = max(max|y| * (1 / top), 2^-126), code = rne(y * (1 / scale)), top = 448 (e4m3) or 127 (int8),
//             1 / top being the fp32 number: |y| * (1 / scale) ends within 2^-22 of top and rounds to it
// All in fp32 from the 16-bit input to the single rounding at the end (to 16 bits or to a code): the pair
// "round to 16 bits, then to 8" would round twice.  A row that holds an infinity or a NaN gets the scale
// NaN and reads back as NaN.
//
// Bound by HBM (each input row is read once, each output row written once), by the launch for a few tokens.
#pragma once

#include "kv_format.cuh"
#include "kv_swap.cuh"  // load_id

namespace hfk {

struct KvWriteArgs {
  const unsigned char *q, *k, *v;       // rows: base + token * token_stride + head * head_stride (bytes)
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  unsigned char *q_out;
  int64_t qo_token, qo_head;
  unsigned char *k_cache, *v_cache;
  int64_t block_stride, scales_at;      // bytes; scales_at = start of the scales inside a page
  const void *slots;                    // slot = block * block_size + place in the block
  const void *positions;
  int slots_are_int64, positions_are_int64;
  const float *cos_sin;                 // [max_positions][rot]: cosines, then sines
  const void *q_weight, *k_weight;      // [head_dim] of the inputs' type, or null
  float eps;
  int rot, interleaved;
  int64_t max_positions, num_slots;
  uint32_t rows;                        // tokens * rows per token
  int q_heads, kv_heads, head_dim;
  FastDiv per_token, block;             // rows per token; block size
};


// A row goes to kLanes lanes by units of two blocks of eight elements, kUnits to a lane (kLanes * kUnits * 16 >= head_dim).
// Where pairs (i, i + rot/2) are rotated, unit q < rot/16 is blocks q and q + rot/16, so that a lane has either partner;
// other units are neighbouring blocks.  Consecutive groups of lanes take consecutive heads of a token, so that loads, stores
// and the 4-byte scales of neighbours fall into the same lines.
//
// HBM bounds the bytes, and close behind it the instructions: those for a row's addresses and its scale are the same
// however many elements a lane has.  Measured: 65536 tokens of 8 heads of 128, fp16 to int8 (407 MB): 102 us with 8 elements a
// lane, 70 with 16, 65 with 32; 16384 tokens with rotation of 40 heads, fp16 to e4m3 (379 MB): 135, 80 and 77 to 82 us (the
// spread between processes).  Loads of the table before the row is waited for: 86 us, for the registers they take.  Two or
// four rows a thread were slower (85 and 172 us there), and so were CTAs of 256 threads (70 and 81 us with 32 elements).  Few
// rows, and copies, take one unit a lane (write_wide); without rotation that form is held to 32 registers, so that all warps fit.
template <typename T, int kFmt, bool kRope, int kLanes, int kUnits, int kThreads>
__global__ void __launch_bounds__(kThreads, kRope || kUnits > 1 ? 1 : 16) kv_write_kernel(const __grid_constant__ KvWriteArgs a) {
  constexpr int kGroups = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const uint32_t r = blockIdx.x * (uint32_t)kGroups + threadIdx.x / kLanes;
  const int pairs = kRope && !a.interleaved ? a.rot >> 4 : 0;       // units of blocks rot/2 apart
  auto unit = [&](int u) { return lane + kLanes * u; };
  auto inside = [&](int u) { return unit(u) * 16 < a.head_dim; };
  auto block = [&](int u, int b) {
    const int q = unit(u);
    return q < pairs ? q + b * pairs : 2 * q + b;
  };

  bool live = r < a.rows;
  const uint32_t token = a.per_token.div(live ? r : 0);
  const int h = (int)((live ? r : 0) - token * a.per_token.d);      // counts q heads, then k heads, then v heads
  const int64_t slot = load_id(a.slots, a.slots_are_int64, token);
  const int64_t position = kRope ? load_id(a.positions, a.positions_are_int64, token) : 0;
  const bool is_q = kRope && h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
  const int kv_head = is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
  const unsigned char *src = is_q   ? a.q + token * a.q_token + h * a.q_head
                             : is_v ? a.v + token * a.v_token + kv_head * a.v_head
                                    : a.k + token * a.k_token + kv_head * a.k_head;
  uint4 in[kUnits][2];
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      in[u][b] = make_uint4(0, 0, 0, 0);
      if (live && inside(u)) in[u][b] = *reinterpret_cast<const uint4 *>(src + block(u, b) * 16);
    }
  // a negative slot is padding: nothing of the token is written
  if (live && slot >= a.num_slots) {
    raise_status(HFK_DEV_BAD_DEVICE_BLOCK_ID);
    live = false;
  }
  live = live && slot >= 0;
  if (kRope && live && (position < 0 || position >= a.max_positions)) {
    raise_status(HFK_DEV_BAD_POSITION);
    live = false;
  }
  unsigned char *page = nullptr;
  uint32_t place = 0;
  if (live && !is_q) {
    const uint32_t b = a.block.div((uint32_t)slot);
    place = ((uint32_t)slot - b * a.block.d) * a.kv_heads + kv_head;
    page = (is_v ? a.v_cache : a.k_cache) + (int64_t)b * a.block_stride;
  }

  if constexpr (!kRope && kFmt == kFmtRaw) {
    if (!live) return;
    unsigned char *dst = page + (int64_t)place * a.head_dim * 2;
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      if (inside(u)) {
        *reinterpret_cast<uint4 *>(dst + block(u, 0) * 16) = in[u][0];
        *reinterpret_cast<uint4 *>(dst + block(u, 1) * 16) = in[u][1];
      }
  } else {
    float x[kUnits][2][8];
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t w[4] = {in[u][b].x, in[u][b].y, in[u][b].z, in[u][b].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Pair<T>::unpack(w[i]);
          x[u][b][2 * i] = f.x;
          x[u][b][2 * i + 1] = f.y;
        }
      }

    if constexpr (kRope) {
      const void *weight = is_q ? a.q_weight : (is_v ? nullptr : a.k_weight);
      if (a.q_weight != nullptr || a.k_weight != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fmaf(x[u][0][i], x[u][0][i], fmaf(x[u][1][i], x[u][1][i], sum));
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d, kLanes);
        if (weight != nullptr) {
          const float scale = rsqrtf(sum / (float)a.head_dim + a.eps);
#pragma unroll
          for (int u = 0; u < kUnits; ++u)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              if (!inside(u)) continue;
              const uint4 g = *reinterpret_cast<const uint4 *>(static_cast<const unsigned char *>(weight) + block(u, b) * 16);
              const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = Pair<T>::unpack(gw[i]);
                x[u][b][2 * i] = x[u][b][2 * i] * scale * f.x;
                x[u][b][2 * i + 1] = x[u][b][2 * i + 1] * scale * f.y;
              }
            }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (!live || is_v || unit(u) * 16 >= a.rot) continue;
        // eight pairs of the unit, of its two blocks or neighbours inside them; four at a time
        const float *cp = a.cos_sin + position * a.rot + unit(u) * 8, *sp = cp + a.rot / 2;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4 c4 = *reinterpret_cast<const float4 *>(cp + 4 * q), s4 = *reinterpret_cast<const float4 *>(sp + 4 * q);
          const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (a.interleaved) {
              const float lo = x[u][q][2 * i], hi = x[u][q][2 * i + 1];
              x[u][q][2 * i] = lo * c[i] - hi * s[i];
              x[u][q][2 * i + 1] = hi * c[i] + lo * s[i];
            } else {
              const float lo = x[u][0][4 * q + i], hi = x[u][1][4 * q + i];
              x[u][0][4 * q + i] = lo * c[i] - hi * s[i];
              x[u][1][4 * q + i] = hi * c[i] + lo * s[i];
            }
          }
        }
      }
    }

    if (kFmt == kFmtRaw || is_q) {
      if (live) {
        unsigned char *dst = is_q ? a.q_out + token * a.qo_token + h * a.qo_head : page + (int64_t)place * a.head_dim * 2;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            if (inside(u))
              *reinterpret_cast<uint4 *>(dst + block(u, b) * 16) =
                  make_uint4(Pair<T>::pack(x[u][b][0], x[u][b][1]), Pair<T>::pack(x[u][b][2], x[u][b][3]),
                             Pair<T>::pack(x[u][b][4], x[u][b][5]), Pair<T>::pack(x[u][b][6], x[u][b][7]));
      }
    }
    if constexpr (kFmt != kFmtRaw) {
      if (__all_sync(0xffffffffu, is_q)) return;   // the other lanes of a warp may hold keys or values
      float top = 0.f;
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_nan(max_nan(top, fabsf(x[u][0][i])), fabsf(x[u][1][i]));
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d, kLanes));
      float scale = __fmul_rn(top, 1.f / top_code<kFmt>());
      if (scale < kLeastScale) scale = kLeastScale;  // a NaN stays
      if (scale > 3.4e38f) scale = __uint_as_float(0x7fffffffu);  // an infinity in the row: no code stands for its parts
      const float inv = __frcp_rn(scale);
      if (live && !is_q) {
        unsigned char *dst = page + (int64_t)place * a.head_dim;
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(x[u][b][i], inv);
            if (inside(u))
              *reinterpret_cast<uint2 *>(dst + block(u, b) * 8) =
                  make_uint2(float_to_codes<kFmt>(y[0], y[1], y[2], y[3]), float_to_codes<kFmt>(y[4], y[5], y[6], y[7]));
          }
        if (lane == 0) reinterpret_cast<float *>(page + a.scales_at)[place] = scale;
      }
    }
  }
}

}  // namespace hfk
