// Reading an 8-bit cache back: the pages a batch of sequences owns become contiguous K and V of each
// sequence, value = code * scale in fp32, rounded once to the output's type; every layer, K and V, one launch.
// The block-table walk is the one of the paged gather (build_walk_tables, locate_page).
//
// Bound by HBM: one byte and 4/head_dim bytes of a scale in, two or four bytes out per value.  Measured: 64 sequences of 512
// to 8192 tokens, 8 heads of 128, four layers, e4m3 to bf16 (6.9 GB): 1106 us, 6.25 TB/s.
#pragma once

#include "kv_format.cuh"
#include "paged_gather.cuh"

namespace hfk {

struct GatherDequantArgs {
  GatherArgs g;         // token_bytes = codes of a token, k_out / v_out / out_layer_stride in bytes of the output
  int64_t scales_at;    // bytes from a page's start to its scales
  FastDiv vec_per_row;  // head_dim / 8
};

template <typename Out>
__device__ __forceinline__ void store8(unsigned char *out, int64_t vec, const float *x) {
  if constexpr (sizeof(Out) == 4) {
    uint4 *p = reinterpret_cast<uint4 *>(out) + 2 * vec;
    st_stream16(p, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])));
    st_stream16(p + 1, make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])));
  } else {
    st_stream16(reinterpret_cast<uint4 *>(out) + vec,
                make_uint4(Pair<Out>::pack(x[0], x[1]), Pair<Out>::pack(x[2], x[3]), Pair<Out>::pack(x[4], x[5]),
                           Pair<Out>::pack(x[6], x[7])));
  }
}

// One warp per unit; a unit is a page of one layer's K or V, or a part of it where there are fewer pages than
// warps.  The lanes work out the addresses of 32 units at a time (a table walk is a chain of dependent loads),
// then the warp moves one unit after the other, kUnroll vectors of eight codes a lane in flight.
template <int kFmt, typename Out, int kThreads, int kUnroll>
__global__ void __launch_bounds__(kThreads) paged_gather_dequant_kernel(const __grid_constant__ GatherDequantArgs args) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  const GatherArgs &a = args.g;
  GatherTables *t = reinterpret_cast<GatherTables *>(smem_raw);
  build_walk_tables(a, t);
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int64_t pages = t->cu_blk[a.num_seqs];
  if (pages == 0) return;
  const int page_vecs = (int)(a.block_size * a.token_bytes >> 3);
  const int64_t whole = pages * 2 * a.layers;
  // parts of at least 32 vectors, as many as it takes to give every warp one
  const int most = (page_vecs + 31) / 32;
  const int parts = (int)max((int64_t)1, min((int64_t)most, (warps + whole - 1) / whole));
  const int part_vecs = ((page_vecs + parts - 1) / parts + 31) & ~31;
  const int64_t units = whole * parts;

  for (int64_t base = warp; base < units; base += 32 * warps) {
    const int64_t u = base + lane * warps;
    const unsigned char *page = nullptr;
    unsigned char *out = nullptr;
    int from = 0, count = 0;
    if (u < units) {
      const int64_t w = u / parts;
      const int part = (int)(u - w * parts);
      const int lk = (int)(w / pages);
      const PageCopy c = locate_page(a, t, (int32_t)(w - lk * pages));
      const unsigned char *layer = checked_layer_ptr((lk & 1) ? a.v_layer_ptrs[lk >> 1] : a.k_layer_ptrs[lk >> 1]);
      if (c.bytes != 0 && layer != nullptr) {
        page = layer + c.src_off;
        out = ((lk & 1) ? a.v_out : a.k_out) + (lk >> 1) * a.out_layer_stride + c.dst_off * (int64_t)sizeof(Out);
        from = part * part_vecs;
        count = max(0, min((int)(c.bytes >> 3) - from, part_vecs));
      }
    }
    const int64_t left = (units - base + warps - 1) / warps;
    const int here = (int)min((int64_t)32, left);
    for (int k = 0; k < here; ++k) {
      const int n = __shfl_sync(0xffffffffu, count, k);
      if (n == 0) continue;
      const int v0 = __shfl_sync(0xffffffffu, from, k);
      const unsigned char *p = reinterpret_cast<const unsigned char *>(__shfl_sync(0xffffffffu, (unsigned long long)page, k));
      unsigned char *o = reinterpret_cast<unsigned char *>(__shfl_sync(0xffffffffu, (unsigned long long)out, k));
      const float *scales = reinterpret_cast<const float *>(p + args.scales_at);
      for (int i = lane; i < n; i += 32 * kUnroll) {
        uint2 codes[kUnroll];
        float scale[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
          const int v = v0 + i + 32 * j;
          if (i + 32 * j < n) {
            codes[j] = __ldcs(reinterpret_cast<const uint2 *>(p) + v);
            scale[j] = scales[args.vec_per_row.div(v)];
          }
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
          if (i + 32 * j < n) {
            float x[8];
            codes_to_float<kFmt>(codes[j].x, x);
            codes_to_float<kFmt>(codes[j].y, x + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= scale[j];
            store8<Out>(o, v0 + i + 32 * j, x);
          }
        }
      }
    }
  }
}

}  // namespace hfk
