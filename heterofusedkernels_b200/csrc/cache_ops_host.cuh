// Host side of the operators that fill and read the cache of an attention layer: argument checks, launch
// plans and launches.  Included by hfk_capi.cu (one translation unit owns the status word).
#pragma once

#include "kv_write.cuh"
#include "paged_gather_dequant.cuh"
#include "prefix_tensor.cuh"
#include "shared_prefix_attention.cuh"

namespace hfk {

static size_t kv_block_bytes(int64_t block_size, int64_t kv_heads, int64_t head_dim, int kv_format) {
  if (block_size <= 0 || kv_heads <= 0 || head_dim <= 0 || kv_format < HFK_KV_RAW || kv_format > HFK_KV_INT8) return 0;
  const int64_t limit = (int64_t)1 << 30;  // of a page; each factor is bounded first, so nothing overflows
  if (block_size > limit || kv_heads > limit || head_dim > limit || block_size * kv_heads > limit ||
      block_size * kv_heads * head_dim > limit)
    return 0;
  const int64_t rows = block_size * kv_heads;
  if (kv_format == HFK_KV_RAW) return (size_t)(rows * head_dim * 2);
  return (size_t)((rows * (head_dim + 4) + 15) / 16 * 16);
}

// What the descriptors of all these calls share.
static int validate_cache(const char *op, const void *k_cache, const void *v_cache, int type, int kv_format, int64_t kv_heads,
                          int64_t head_dim, int64_t block_size, int64_t stride, int64_t blocks) {
  if (type != HFK_TYPE_BF16 && type != HFK_TYPE_FP16) return fail(HFK_ERR_INVALID_ARG, "%s: type must be bf16 or fp16", op);
  if (kv_format < HFK_KV_RAW || kv_format > HFK_KV_INT8) return fail(HFK_ERR_INVALID_ARG, "%s: unknown kv_format %d", op, kv_format);
  if (kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || blocks <= 0)
    return fail(HFK_ERR_INVALID_ARG, "%s: non-positive geometry", op);
  const size_t page = kv_block_bytes(block_size, kv_heads, head_dim, kv_format);
  if (page == 0) return fail(HFK_ERR_TOO_LARGE, "%s: a page is larger than 2^30 values", op);
  if (!k_cache || !v_cache) return fail(HFK_ERR_INVALID_ARG, "%s: null cache", op);
  if (!aligned16(k_cache) || !aligned16(v_cache) || (stride & 15))
    return fail(HFK_ERR_ALIGNMENT, "%s: caches and device_block_stride must be multiples of 16 bytes", op);
  if (stride < (int64_t)page)
    return fail(HFK_ERR_INVALID_ARG, "%s: device_block_stride %lld smaller than one page (%lld)", op, (long long)stride,
                (long long)page);
  return HFK_OK;
}

static int validate_rows(const char *op, const char *name, const hfk_rows &r) {
  if (!r.base) return fail(HFK_ERR_INVALID_ARG, "%s: null %s", op, name);
  if (!aligned16(r.base) || (r.token_stride & 15) || (r.head_stride & 15))
    return fail(HFK_ERR_ALIGNMENT, "%s: base and strides of %s must be multiples of 16 bytes", op, name);
  return HFK_OK;
}

// Rows that are written must not share bytes.
static int validate_written(const char *op, const char *name, const hfk_rows &r, int64_t tokens, int64_t heads, int64_t row_bytes) {
  const int rc = validate_rows(op, name, r);
  if (rc != HFK_OK) return rc;
  if (!strides_nest(row_bytes, {r.head_stride, heads}, {r.token_stride, tokens}, {0, 1}))
    return fail(HFK_ERR_INVALID_ARG, "%s: strides of %s let its rows overlap", op, name);
  return HFK_OK;
}

// ---- writing ------------------------------------------------------------------------------------------------
template <typename T, int kFmt, bool kRope, int kLanes, int kUnits>
static cudaError_t launch_kv_write(const KvWriteArgs &a, cudaStream_t stream) {
  constexpr int kThreads = 128, kGroups = kThreads / kLanes;
  kv_write_kernel<T, kFmt, kRope, kLanes, kUnits, kThreads><<<(a.rows + kGroups - 1) / kGroups, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}
template <typename T, bool kRope, int kLanes, int kUnits>
static cudaError_t launch_kv_write(const KvWriteArgs &a, int fmt, cudaStream_t s) {
  if (fmt == HFK_KV_E4M3) return launch_kv_write<T, kFmtE4m3, kRope, kLanes, kUnits>(a, s);
  if (fmt == HFK_KV_INT8) return launch_kv_write<T, kFmtInt8, kRope, kLanes, kUnits>(a, s);
  if constexpr (!kRope && kUnits > 1)
    return cudaErrorInvalidValue;   // write_wide leaves copies to one unit
  else
    return launch_kv_write<T, kFmtRaw, kRope, kLanes, kUnits>(a, s);
}
template <typename T, bool kRope, int kUnits>
static cudaError_t launch_kv_write(const KvWriteArgs &a, int fmt, cudaStream_t s) {
  if (a.head_dim <= 64) return launch_kv_write<T, kRope, 4 / kUnits, kUnits>(a, fmt, s);
  if (a.head_dim <= 128) return launch_kv_write<T, kRope, 8 / kUnits, kUnits>(a, fmt, s);
  return launch_kv_write<T, kRope, 16 / kUnits, kUnits>(a, fmt, s);
}
template <typename T, bool kRope>
static cudaError_t launch_kv_write(const KvWriteArgs &a, int fmt, cudaStream_t s) {
  return write_wide(a.rows, a.head_dim, kRope, fmt == HFK_KV_RAW) ? launch_kv_write<T, kRope, 2>(a, fmt, s) : launch_kv_write<T, kRope, 1>(a, fmt, s);
}

static int kv_write_impl(const char *op, const hfk_kv_write_desc *d, const hfk_norm_rope_desc *n, bool rope, cudaStream_t stream) {
  if (!d || (rope && !n)) return fail(HFK_ERR_INVALID_ARG, "%s: descriptor is null", op);
  int rc = validate_cache(op, d->k_cache, d->v_cache, d->type, d->kv_format, d->kv_heads, d->head_dim, d->block_size,
                          d->device_block_stride, d->num_device_blocks);
  if (rc != HFK_OK) return rc;
  if (d->tokens < 0) return fail(HFK_ERR_INVALID_ARG, "%s: negative token count", op);
  if (d->head_dim > 256 || (d->head_dim & 15))
    return fail(HFK_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 16 up to 256", op, d->head_dim);
  if (d->num_device_blocks > INT32_MAX / d->block_size)
    return fail(HFK_ERR_TOO_LARGE, "%s: more than 2^31 slots", op);
  KvWriteArgs a = {};
  a.rot = 0;
  if (rope) {
    if (n->q_heads <= 0) return fail(HFK_ERR_INVALID_ARG, "%s: non-positive q_heads", op);
    if (n->rot_dim < 0 || n->rot_dim > d->head_dim || (n->rot_dim & 15))
      return fail(HFK_ERR_UNSUPPORTED, "%s: rot_dim %d is not a multiple of 16 up to head_dim", op, n->rot_dim);
    if (n->max_positions <= 0) return fail(HFK_ERR_INVALID_ARG, "%s: non-positive max_positions", op);
    if (!(n->eps >= 0.f)) return fail(HFK_ERR_INVALID_ARG, "%s: eps must not be negative", op);
  }
  const int64_t per_token = (rope ? (int64_t)n->q_heads : 0) + 2 * (int64_t)d->kv_heads;
  if (d->tokens > INT32_MAX / per_token) return fail(HFK_ERR_TOO_LARGE, "%s: more than 2^31 rows", op);
  if (d->tokens == 0) return HFK_OK;
  if ((rc = validate_rows(op, "k", d->k)) != HFK_OK || (rc = validate_rows(op, "v", d->v)) != HFK_OK) return rc;
  if (!d->slot_ids) return fail(HFK_ERR_INVALID_ARG, "%s: null slot ids", op);
  if (rope) {
    if ((rc = validate_rows(op, "q", n->q)) != HFK_OK) return rc;
    if ((rc = validate_written(op, "q_out", n->q_out, d->tokens, n->q_heads, (int64_t)d->head_dim * 2)) != HFK_OK) return rc;
    if (!n->positions || (n->rot_dim > 0 && !n->cos_sin)) return fail(HFK_ERR_INVALID_ARG, "%s: null positions or table", op);
    if (!aligned16(n->cos_sin) || !aligned16(n->q_weight) || !aligned16(n->k_weight))
      return fail(HFK_ERR_ALIGNMENT, "%s: table and weights must be 16-byte aligned", op);
    a.q = static_cast<const unsigned char *>(n->q.base);
    a.q_token = n->q.token_stride;
    a.q_head = n->q.head_stride;
    a.q_out = static_cast<unsigned char *>(const_cast<void *>(n->q_out.base));
    a.qo_token = n->q_out.token_stride;
    a.qo_head = n->q_out.head_stride;
    a.positions = n->positions;
    a.positions_are_int64 = n->positions_are_int64;
    a.cos_sin = n->cos_sin;
    a.q_weight = n->q_weight;
    a.k_weight = n->k_weight;
    a.eps = n->eps;
    a.rot = n->rot_dim;
    a.interleaved = n->interleaved;
    a.max_positions = n->max_positions;
    a.q_heads = n->q_heads;
  }
  a.k = static_cast<const unsigned char *>(d->k.base);
  a.k_token = d->k.token_stride;
  a.k_head = d->k.head_stride;
  a.v = static_cast<const unsigned char *>(d->v.base);
  a.v_token = d->v.token_stride;
  a.v_head = d->v.head_stride;
  a.k_cache = static_cast<unsigned char *>(d->k_cache);
  a.v_cache = static_cast<unsigned char *>(d->v_cache);
  a.block_stride = d->device_block_stride;
  a.scales_at = d->block_size * d->kv_heads * d->head_dim;
  a.slots = d->slot_ids;
  a.slots_are_int64 = d->ids_are_int64;
  a.num_slots = d->num_device_blocks * d->block_size;
  a.rows = (uint32_t)(d->tokens * per_token);
  a.kv_heads = d->kv_heads;
  a.head_dim = d->head_dim;
  a.per_token = FastDiv::make((uint32_t)per_token);
  a.block = FastDiv::make((uint32_t)d->block_size);
  cudaError_t e;
  if (d->type == HFK_TYPE_BF16)
    e = rope ? launch_kv_write<__nv_bfloat16, true>(a, d->kv_format, stream) : launch_kv_write<__nv_bfloat16, false>(a, d->kv_format, stream);
  else
    e = rope ? launch_kv_write<__half, true>(a, d->kv_format, stream) : launch_kv_write<__half, false>(a, d->kv_format, stream);
  if (e != cudaSuccess) return cuda_fail(e, "kv_write_kernel launch");
  return HFK_OK;
}

// ---- reading back -----------------------------------------------------------------------------------------------
template <int kFmt, typename Out>
static cudaError_t launch_gather_dequant(const GatherDequantArgs &a, int ctas, cudaStream_t s) {
  constexpr int kThreads = 256;
  paged_gather_dequant_kernel<kFmt, Out, kThreads, 8><<<ctas, kThreads, sizeof(GatherTables), s>>>(a);
  return cudaGetLastError();
}
template <int kFmt>
static cudaError_t launch_gather_dequant(const GatherDequantArgs &a, int out_type, int ctas, cudaStream_t s) {
  if (out_type == HFK_TYPE_BF16) return launch_gather_dequant<kFmt, __nv_bfloat16>(a, ctas, s);
  if (out_type == HFK_TYPE_FP16) return launch_gather_dequant<kFmt, __half>(a, ctas, s);
  return launch_gather_dequant<kFmt, float>(a, ctas, s);
}

static int gather_dequant_impl(const hfk_paged_gather_desc *d, int kv_format, int kv_heads, int out_type, int ctas, cudaStream_t stream) {
  const char *op = "paged_gather_dequant";
  if (!d) return fail(HFK_ERR_INVALID_ARG, "%s: descriptor is null", op);
  if (kv_format != HFK_KV_E4M3 && kv_format != HFK_KV_INT8)
    return fail(HFK_ERR_INVALID_ARG, "%s: kv_format must be e4m3 or int8 (hfk_paged_gather reads a 16-bit cache)", op);
  if (out_type < HFK_TYPE_BF16 || out_type > HFK_TYPE_FP32) return fail(HFK_ERR_INVALID_ARG, "%s: unknown out_type %d", op, out_type);
  // every check of the paged gather, with the output's layer stride in codes
  const int64_t elt = out_type == HFK_TYPE_FP32 ? 4 : 2;
  if (d->out_layer_stride % (16 * elt)) return fail(HFK_ERR_ALIGNMENT, "%s: out_layer_stride must be a multiple of 16 values", op);
  hfk_paged_gather_desc codes = *d;
  codes.out_layer_stride = d->out_layer_stride / elt;
  const int rc = validate_gather(&codes);
  if (rc != HFK_OK) return rc;
  if (kv_heads <= 0 || d->token_bytes % kv_heads || (d->token_bytes / kv_heads) & 15)
    return fail(HFK_ERR_UNSUPPORTED, "%s: token_bytes must be kv_heads times a head_dim that is a multiple of 16", op);
  const int64_t head_dim = d->token_bytes / kv_heads;
  const size_t page = kv_block_bytes(d->block_size, kv_heads, head_dim, kv_format);
  if (page == 0) return fail(HFK_ERR_TOO_LARGE, "%s: a page is larger than 2^30 values", op);
  if (d->device_block_stride < (int64_t)page)
    return fail(HFK_ERR_INVALID_ARG, "%s: device_block_stride smaller than one page (%lld)", op, (long long)page);
  if (d->num_seqs == 0 || d->max_blocks_per_seq == 0) return HFK_OK;
  GatherDequantArgs a;
  a.g.k_layer_ptrs = d->k_layer_ptrs;
  a.g.v_layer_ptrs = d->v_layer_ptrs;
  a.g.k_out = static_cast<unsigned char *>(d->k_out);
  a.g.v_out = static_cast<unsigned char *>(d->v_out);
  a.g.out_layer_stride = d->out_layer_stride;
  a.g.block_tables = d->block_tables;
  a.g.seq_lens = d->seq_lens;
  a.g.ids_are_int64 = d->ids_are_int64;
  a.g.layers = d->layers;
  a.g.max_blocks_per_seq = d->max_blocks_per_seq;
  a.g.block_table_stride = d->block_table_stride;
  a.g.block_size = d->block_size;
  a.g.token_bytes = d->token_bytes;
  a.g.device_block_stride = d->device_block_stride;
  a.g.num_device_blocks = d->num_device_blocks;
  a.g.total_tokens = d->total_tokens;
  a.g.hints = a.g.blocked = 0;
  a.scales_at = d->block_size * d->token_bytes;
  a.vec_per_row = FastDiv::make((uint32_t)(head_dim / 8));
  if (ctas <= 0) ctas = sm_count() * kGatherDequantCtasPerSm;
  for (int64_t first = 0; first < d->num_seqs; first += HFK_MAX_SEQS) {
    a.g.seq_offset = (int)first;
    a.g.num_seqs = (int)std::min<int64_t>(HFK_MAX_SEQS, d->num_seqs - first);
    const cudaError_t e = kv_format == HFK_KV_E4M3 ? launch_gather_dequant<kFmtE4m3>(a, out_type, ctas, stream)
                                                   : launch_gather_dequant<kFmtInt8>(a, out_type, ctas, stream);
    if (e != cudaSuccess) return cuda_fail(e, "paged_gather_dequant_kernel launch");
  }
  return HFK_OK;
}

// ---- attention -----------------------------------------------------------------------------------------------------
// Large batches (above HFK_MAX_SEQS sequences) go out as several groups of launches, which use the workspace in turn.
struct AttnPlan {
  bool tensor;      // the prefix goes to prefix_tensor_kernel
  int splits;       // its runs of key tiles
  int ctas, warps;  // of the line
  int seqs;         // sequences a group of launches takes
  size_t ml_bytes, o_bytes, prefix_ml_bytes, prefix_o_bytes;
  size_t bytes() const { return 256 + ml_bytes + o_bytes + prefix_ml_bytes + prefix_o_bytes; }
};

static int plan_attention(const hfk_prefix_attention_desc *d, int ctas, AttnPlan *p) {
  const char *op = "shared_prefix_attention";
  if (!d) return fail(HFK_ERR_INVALID_ARG, "%s: descriptor is null", op);
  if (d->head_dim != 64 && d->head_dim != 128) return fail(HFK_ERR_UNSUPPORTED, "%s: head_dim %d is not 64 or 128", op, d->head_dim);
  if (d->group <= 0 || d->kv_heads <= 0 || d->block_size <= 0 || d->num_seqs < 0 || d->prefix_len < 0 || d->max_blocks_per_seq < 0)
    return fail(HFK_ERR_INVALID_ARG, "%s: non-positive geometry", op);
  if (d->group > 256 || d->kv_heads > 4096) return fail(HFK_ERR_TOO_LARGE, "%s: more than 256 query heads to a K/V head, or 4096 K/V heads", op);
  const int64_t most = INT32_MAX - 1024;  // keys of a row
  if (d->block_size > most || d->prefix_len > most || (d->max_blocks_per_seq > 0 && d->max_blocks_per_seq > most / d->block_size))
    return fail(HFK_ERR_TOO_LARGE, "%s: more than 2^31 keys", op);
  if (d->num_seqs >= (int64_t)1 << 30) return fail(HFK_ERR_TOO_LARGE, "%s: too many sequences", op);
  const int sms = sm_count();
  // at most HFK_MAX_SEQS at a time, and so few that the line's tiles are counted in 32 bits
  int seqs = (int)std::min<int64_t>(d->num_seqs, HFK_MAX_SEQS);
  const int64_t cap = d->max_blocks_per_seq * d->block_size;
  // (the smaller tile of a 16-bit cache, so that the workspace does not depend on the format)
  const int tile = tile_keys(HFK_KV_RAW);
  while (seqs > 1 && AttnLine(seqs, d->kv_heads, d->group, (int)d->prefix_len, tile).most_tiles(seqs, cap) > INT32_MAX / 2) seqs = (seqs + 1) / 2;
  if (AttnLine(seqs, d->kv_heads, d->group, (int)d->prefix_len, tile).most_tiles(seqs, cap) > INT32_MAX / 2)
    return fail(HFK_ERR_TOO_LARGE, "%s: K/V heads times keys of one sequence exceed 2^34", op);
  p->seqs = seqs;
  const int64_t rows = (int64_t)seqs * d->group;
  p->tensor = d->prefix_len > 0 && rows > kPrefixTensorMinRows;
  p->splits = 0;
  if (p->tensor) {
    // as many runs as give the least time, in key tiles: waves of CTAs, each its tiles and a constant for filling the
    // pipeline, and for each run its part of every row, which is written and read again
    const int64_t items = d->kv_heads * ((rows + 255) / 256), tiles = (d->prefix_len + kPtKeys - 1) / kPtKeys;
    const int64_t room = ctas > 0 ? std::min(ctas, sms) : sms;
    int64_t best = 0;
    for (int64_t s = 1; s <= std::min<int64_t>(tiles, std::max<int64_t>(1, 2 * room / items)); ++s) {
      const int64_t cost = ((items * s + room - 1) / room) * ((tiles + s - 1) / s + kPrefixTileOverhead) * 64 +
                           s * d->kv_heads * rows * d->head_dim / kPrefixPartValues;
      if (p->splits == 0 || cost < best) {
        best = cost;
        p->splits = (int)s;
      }
    }
  }
  p->ctas = d->max_blocks_per_seq == 0 && p->tensor ? 0 : ctas > 0 ? std::min(ctas, 65535) : sms * kAttnCtasPerSm;
  const AttnLine line(seqs, d->kv_heads, d->group, p->tensor ? 0 : (int)d->prefix_len, tile);
  p->warps = p->ctas * kLineWarps;
  const size_t parts = p->ctas > 0 ? (size_t)p->warps + (size_t)line.items(seqs) : 0;
  const auto round = [](size_t n) { return (n + 255) & ~(size_t)255; };
  p->ml_bytes = round(parts * kItemRows * sizeof(float2));
  p->o_bytes = round(parts * kItemRows * d->head_dim * sizeof(float));
  p->prefix_ml_bytes = round((size_t)p->splits * d->kv_heads * rows * sizeof(float2));
  p->prefix_o_bytes = round((size_t)p->splits * d->kv_heads * rows * d->head_dim * sizeof(float));
  return HFK_OK;
}

// What no call with this descriptor, or with fewer sequences, a shorter prefix or narrower block tables, needs more than.  The plan's
// own size is not monotone: more rows of queries may take fewer runs of the prefix, and what is largest is their product.
static size_t attention_workspace_bound(const hfk_prefix_attention_desc *d, int ctas) {
  const int64_t sms = sm_count(), seqs = std::min<int64_t>(d->num_seqs, HFK_MAX_SEQS), rows = seqs * d->group;
  const int64_t row_tiles = (rows + kItemRows - 1) / kItemRows, own_tiles = (d->group + kItemRows - 1) / kItemRows;
  // the line: every part of every item, the prefix's items among them up to where they go to the tensor cores
  const int64_t most_prefix = (kPrefixTensorMinRows + kItemRows - 1) / kItemRows;
  const int64_t items = seqs * d->kv_heads * own_tiles + (d->prefix_len > 0 ? std::min(row_tiles, most_prefix) * d->kv_heads : 0);
  const int64_t parts = (ctas > 0 ? std::min<int64_t>(ctas, 65535) : sms * kAttnCtasPerSm) * kLineWarps + items;
  // the prefix: s runs of r rows of every K/V head, r up to rows; one run, or s <= 2 * room / (kv_heads * ceil(r / 256)) of them
  int64_t values = 0;
  if (d->prefix_len > 0 && rows > kPrefixTensorMinRows) {
    const int64_t room = ctas > 0 ? std::min<int64_t>(ctas, sms) : sms, tiles = (d->prefix_len + kPtKeys - 1) / kPtKeys;
    const int64_t one = d->kv_heads * rows;
    values = std::max(one, std::min(2 * room * std::min<int64_t>(rows, 256), tiles * one));
  }
  const auto round = [](int64_t n) { return ((size_t)n + 255) & ~(size_t)255; };
  return 256 + round(parts * kItemRows * sizeof(float2)) + round(parts * kItemRows * d->head_dim * sizeof(float)) +
         round(values * sizeof(float2)) + round(values * d->head_dim * sizeof(float));
}

// A launch that may start while the kernel launched before it in the same stream still runs (`early`, where that
// is one of ours and says so with launch_next).
template <typename Args>
static cudaError_t launch_behind(void (*kernel)(const Args), bool early, int ctas, int threads, size_t smem, cudaStream_t s, const Args &args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, args);
}

template <typename T, int kFmt, int D>
static cudaError_t launch_attention(const AttnArgs &a, const AttnPlan &p, unsigned char *w, cudaStream_t s) {
  JoinArgs join = {};
  join.a = a;
  join.warps = p.warps;
  join.rows = a.seqs * a.group;
  join.a.part_ml = reinterpret_cast<float2 *>(w);
  join.a.part_o = reinterpret_cast<float *>(w + p.ml_bytes);
  cudaError_t e;
  if (p.tensor) {
    PrefixTensorArgs t = {};
    t.a = a;
    t.a.scale_log2 = std::abs(a.scale_log2);
    t.negate = a.scale_log2 < 0.f;
    t.rows = join.rows;
    t.row_blocks = (t.rows + 255) / 256;
    t.splits = p.splits;
    t.part_ml = reinterpret_cast<float2 *>(w + p.ml_bytes + p.o_bytes);
    t.part_o = reinterpret_cast<float *>(w + p.ml_bytes + p.o_bytes + p.prefix_ml_bytes);
    auto k = prefix_tensor_kernel<T, kFmt, D>;
    const size_t smem = sizeof(PrefixSmem<D>) + 1024;
    if ((e = allow_smem(k, smem)) != cudaSuccess) return e;
    k<<<a.kv_heads * t.row_blocks * t.splits, kPtThreads, smem, s>>>(t);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    join.a.prefix_len = 0;
    join.splits = t.splits;
    join.prefix_ml = t.part_ml;
    join.prefix_o = t.part_o;
  }
  if (p.ctas > 0) {
    const size_t smem = kLineWarps * sizeof(LineRing<kFmt, D>) + (size_t)(a.seqs + 1 + kLineWarps) * sizeof(int);
    auto k = shared_prefix_attention_kernel<T, kFmt, D>;
    if ((e = allow_smem(k, smem)) != cudaSuccess) return e;
    if ((e = launch_behind(k, p.tensor, p.ctas, kLineWarps * 32, smem, s, join.a)) != cudaSuccess) return e;
  }
  const int rows = a.seqs * a.kv_heads * a.group;
  switch (join_warps(rows, sm_count() * kJoinWarpsPerSm)) {
    case 16: return launch_behind(shared_prefix_join_kernel<T, D, 16>, true, rows, 512, 0, s, join);
    case 4: return launch_behind(shared_prefix_join_kernel<T, D, 4>, true, rows, 128, 0, s, join);
    case 2: return launch_behind(shared_prefix_join_kernel<T, D, 2>, true, rows, 64, 0, s, join);
    default: return launch_behind(shared_prefix_join_kernel<T, D, 1>, true, rows, 32, 0, s, join);
  }
}
template <typename T, int kFmt>
static cudaError_t launch_attention(const AttnArgs &a, int head_dim, const AttnPlan &p, unsigned char *w, cudaStream_t s) {
  return head_dim == 64 ? launch_attention<T, kFmt, 64>(a, p, w, s) : launch_attention<T, kFmt, 128>(a, p, w, s);
}
template <typename T>
static cudaError_t launch_attention(const AttnArgs &a, int fmt, int head_dim, const AttnPlan &p, unsigned char *w, cudaStream_t s) {
  if (fmt == HFK_KV_E4M3) return launch_attention<T, kFmtE4m3>(a, head_dim, p, w, s);
  if (fmt == HFK_KV_INT8) return launch_attention<T, kFmtInt8>(a, head_dim, p, w, s);
  return launch_attention<T, kFmtRaw>(a, head_dim, p, w, s);
}

static int attention_impl(const hfk_prefix_attention_desc *d, int ctas, cudaStream_t stream) {
  const char *op = "shared_prefix_attention";
  AttnPlan p = {};
  int rc = plan_attention(d, ctas, &p);
  if (rc != HFK_OK) return rc;
  rc = validate_cache(op, d->k_cache, d->v_cache, d->type, d->kv_format, d->kv_heads, d->head_dim, d->block_size,
                      d->device_block_stride, d->num_device_blocks);
  if (rc != HFK_OK) return rc;
  if (d->num_seqs > 1 && d->block_table_stride < d->max_blocks_per_seq)
    return fail(HFK_ERR_INVALID_ARG, "%s: block_table_stride < max_blocks_per_seq", op);
  // (what the kernels multiply by is the product)
  if (!std::isfinite(d->scale * kLog2e)) return fail(HFK_ERR_INVALID_ARG, "%s: scale is not finite, or not below 2.3e38", op);
  if (d->num_seqs == 0) return HFK_OK;
  if ((rc = validate_rows(op, "q", d->q)) != HFK_OK) return rc;
  if ((rc = validate_written(op, "out", d->out, d->num_seqs, (int64_t)d->kv_heads * d->group, (int64_t)d->head_dim * 2)) != HFK_OK) return rc;
  if (!d->seq_lens || (d->max_blocks_per_seq > 0 && !d->block_tables) || (d->prefix_len > 0 && !d->prefix_table))
    return fail(HFK_ERR_INVALID_ARG, "%s: null block table, prefix table or sequence lengths", op);
  if (!d->workspace || (reinterpret_cast<uintptr_t>(d->workspace) & 255))
    return fail(HFK_ERR_ALIGNMENT, "%s: workspace is null or not 256-byte aligned", op);
  if (d->workspace_bytes < p.bytes())
    return fail(HFK_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu needed", op, d->workspace_bytes, p.bytes());
  AttnArgs a = {};
  a.q_seq = d->q.token_stride;
  a.q_head = d->q.head_stride;
  a.out_seq = d->out.token_stride;
  a.out_head = d->out.head_stride;
  a.k_cache = static_cast<const unsigned char *>(d->k_cache);
  a.v_cache = static_cast<const unsigned char *>(d->v_cache);
  a.block_stride = d->device_block_stride;
  a.scales_at = d->block_size * d->kv_heads * d->head_dim;
  a.num_blocks = d->num_device_blocks;
  a.prefix_table = d->prefix_table;
  a.table_stride = d->block_table_stride;
  a.ids_are_int64 = d->ids_are_int64;
  a.prefix_len = (int)d->prefix_len;
  a.own_cap = d->max_blocks_per_seq * d->block_size;
  a.kv_heads = d->kv_heads;
  a.group = d->group;
  a.block = FastDiv::make((uint32_t)d->block_size);
  a.per_group = FastDiv::make((uint32_t)d->group);
  a.tile = tile_keys(d->kv_format);
  a.scale_log2 = d->scale * kLog2e;
  unsigned char *w = static_cast<unsigned char *>(d->workspace);
  const int64_t id = d->ids_are_int64 ? 8 : 4;
  for (int64_t first = 0; first < d->num_seqs; first += p.seqs) {
    a.seqs = (int)std::min<int64_t>(p.seqs, d->num_seqs - first);
    a.q = static_cast<const unsigned char *>(d->q.base) + first * a.q_seq;
    a.out = static_cast<unsigned char *>(const_cast<void *>(d->out.base)) + first * a.out_seq;
    a.lse = d->lse ? d->lse + first * a.kv_heads * a.group : nullptr;
    a.tables = static_cast<const unsigned char *>(d->block_tables) + first * d->block_table_stride * id;
    a.lens = static_cast<const unsigned char *>(d->seq_lens) + first * id;
    const cudaError_t e = d->type == HFK_TYPE_BF16 ? launch_attention<__nv_bfloat16>(a, d->kv_format, d->head_dim, p, w, stream)
                                                   : launch_attention<__half>(a, d->kv_format, d->head_dim, p, w, stream);
    if (e != cudaSuccess) return cuda_fail(e, "shared_prefix_attention launch");
  }
  return HFK_OK;
}

}  // namespace hfk
