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


// A row is handled by kLanes lanes of a warp, eight elements each (kLanes * 8 >= head_dim); a CTA handles
// kRows consecutive rows for each of its lane groups at a time, all loads first.  Consecutive groups take
// consecutive heads of a token, so that loads, stores and the 4-byte scales of neighbours fall into the same
// lines.
template <typename T, int kFmt, bool kRope, int kLanes, int kRows, int kThreads>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const __grid_constant__ KvWriteArgs a) {
  constexpr int kGroups = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int group = threadIdx.x / kLanes;
  const bool inside = lane * 8 < a.head_dim;
  const uint32_t first = blockIdx.x * (uint32_t)(kGroups * kRows) + group;

  uint4 in[kRows];
  uint32_t token[kRows], head[kRows];   // head counts q heads, then k heads, then v heads
  int64_t slot[kRows];
  int64_t position[kRows];
  bool live[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t r = first + u * kGroups;
    live[u] = r < a.rows;
    token[u] = a.per_token.div(live[u] ? r : 0);
    head[u] = (live[u] ? r : 0) - token[u] * a.per_token.d;
    slot[u] = load_id(a.slots, a.slots_are_int64, token[u]);
    position[u] = kRope ? load_id(a.positions, a.positions_are_int64, token[u]) : 0;
    const int h = (int)head[u];
    const unsigned char *src;
    if (kRope && h < a.q_heads)
      src = a.q + token[u] * a.q_token + h * a.q_head;
    else if (h < a.q_heads + a.kv_heads)
      src = a.k + token[u] * a.k_token + (h - a.q_heads) * a.k_head;
    else
      src = a.v + token[u] * a.v_token + (h - a.q_heads - a.kv_heads) * a.v_head;
    in[u] = make_uint4(0, 0, 0, 0);
    if (inside && live[u]) in[u] = *reinterpret_cast<const uint4 *>(src + lane * 16);
  }

#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    // a negative slot is padding: nothing of the token is written
    if (live[u] && slot[u] >= a.num_slots) {
      raise_status(HFK_DEV_BAD_DEVICE_BLOCK_ID);
      live[u] = false;
    }
    live[u] = live[u] && slot[u] >= 0;
    if (kRope && live[u] && (position[u] < 0 || position[u] >= a.max_positions)) {
      raise_status(HFK_DEV_BAD_POSITION);
      live[u] = false;
    }
    const int h = (int)head[u];
    const bool is_q = kRope && h < a.q_heads;
    const bool is_v = h >= a.q_heads + a.kv_heads;
    const int kv_head = is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
    unsigned char *page = nullptr;
    uint32_t place = 0;
    if (live[u] && !is_q) {
      const uint32_t b = a.block.div((uint32_t)slot[u]);
      place = ((uint32_t)slot[u] - b * a.block.d) * a.kv_heads + kv_head;
      page = (is_v ? a.v_cache : a.k_cache) + (int64_t)b * a.block_stride;
    }

    if (!kRope && kFmt == kFmtRaw) {
      if (live[u] && inside)
        *reinterpret_cast<uint4 *>(page + (int64_t)place * a.head_dim * 2 + lane * 16) = in[u];
      continue;
    }

    const uint32_t w[4] = {in[u].x, in[u].y, in[u].z, in[u].w};
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Pair<T>::unpack(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }

    if (kRope) {
      const void *weight = is_q ? a.q_weight : (is_v ? nullptr : a.k_weight);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d, kLanes);
      if (weight != nullptr && inside) {
        const float r = rsqrtf(sum / (float)a.head_dim + a.eps);
        const uint4 g = *reinterpret_cast<const uint4 *>(static_cast<const unsigned char *>(weight) + lane * 16);
        const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Pair<T>::unpack(gw[i]);
          x[2 * i] = x[2 * i] * r * f.x;
          x[2 * i + 1] = x[2 * i + 1] * r * f.y;
        }
      }
      const bool turn = live[u] && !is_v && lane * 8 < a.rot;
      const float *table = a.cos_sin + (turn ? position[u] * a.rot : 0);
      if (a.interleaved) {
        if (turn) {
          const float4 c = *reinterpret_cast<const float4 *>(table + lane * 4);
          const float4 s = *reinterpret_cast<const float4 *>(table + a.rot / 2 + lane * 4);
          const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float lo = x[2 * i], hi = x[2 * i + 1];
            x[2 * i] = lo * cs[i] - hi * sn[i];
            x[2 * i + 1] = hi * cs[i] + lo * sn[i];
          }
        }
      } else {
        const int half = a.rot >> 4;  // lanes per half: rot / 2 elements, eight to a lane
        const bool low = lane < half;
        const int partner = low ? lane + half : lane - half;
        float other[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = __shfl_sync(0xffffffffu, x[i], partner & (kLanes - 1), kLanes);
        if (turn) {
          const float *cp = table + (low ? lane : lane - half) * 8;
          const float *sp = cp + a.rot / 2;
          const float sign = low ? -1.f : 1.f;
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const float4 c = *reinterpret_cast<const float4 *>(cp + i);
            const float4 s = *reinterpret_cast<const float4 *>(sp + i);
            x[i] = x[i] * c.x + sign * other[i] * s.x;
            x[i + 1] = x[i + 1] * c.y + sign * other[i + 1] * s.y;
            x[i + 2] = x[i + 2] * c.z + sign * other[i + 2] * s.z;
            x[i + 3] = x[i + 3] * c.w + sign * other[i + 3] * s.w;
          }
        }
      }
    }

    if (kFmt == kFmtRaw || is_q) {
      if (live[u] && inside) {
        unsigned char *dst = is_q ? a.q_out + token[u] * a.qo_token + h * a.qo_head
                                  : page + (int64_t)place * a.head_dim * 2;
        *reinterpret_cast<uint4 *>(dst + lane * 16) =
            make_uint4(Pair<T>::pack(x[0], x[1]), Pair<T>::pack(x[2], x[3]), Pair<T>::pack(x[4], x[5]),
                       Pair<T>::pack(x[6], x[7]));
      }
      if (kFmt == kFmtRaw) continue;
    }

    if (kFmt != kFmtRaw) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(x[i]));
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d, kLanes));
      float scale = __fmul_rn(top, 1.f / top_code<kFmt>());
      if (scale < kLeastScale) scale = kLeastScale;  // a NaN stays
      if (scale > 3.4e38f) scale = __uint_as_float(0x7fffffffu);  // an infinity in the row: no code stands for its parts
      const float inv = __frcp_rn(scale);
      if (live[u] && !is_q) {
        if (inside) {
          uint2 codes;
          codes.x = float_to_codes<kFmt>(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv), __fmul_rn(x[2], inv), __fmul_rn(x[3], inv));
          codes.y = float_to_codes<kFmt>(__fmul_rn(x[4], inv), __fmul_rn(x[5], inv), __fmul_rn(x[6], inv), __fmul_rn(x[7], inv));
          *reinterpret_cast<uint2 *>(page + (int64_t)place * a.head_dim + lane * 8) = codes;
        }
        if (lane == 0) reinterpret_cast<float *>(page + a.scales_at)[place] = scale;
      }
    }
  }
}

}  // namespace hfk
