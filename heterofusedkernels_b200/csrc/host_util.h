// Host-side helpers shared by the translation units of libhfk_b200.so.
#pragma once

#include <cuda_runtime_api.h>

namespace hfk {

// Records a printf-style message for hfk_last_error_message() and returns `code`.
int fail(int code, const char *fmt, ...);
int cuda_fail(cudaError_t e, const char *what);

// Launch defaults when the caller passes ctas <= 0 / HFK_MOVER_AUTO ("aiv=None"
// in the torch ops).  The swap defaults are sized to fill one PCIe Gen5 x16
// link while occupying a small part of the 148 SMs; the gather defaults to fill
// HBM.
//
// Measured on a B200 behind PCIe Gen5 x16 (cudaMemcpyAsync peak 55.5 GB/s h2d, 57.2 GB/s d2h):
// the bulk mover reaches the link's plateau for kernel-issued traffic (51.5 GB/s in,
// 52.7 GB/s out) from 2 single-warp CTAs with a 16 KiB x 8 ring, the vector mover needs 4-8
// CTAs of 512 threads; 4 CTAs leave a margin.  The paged gather reaches the device's copy
// bandwidth (6.67 TB/s) with one single-warp CTA per SM and a 32 KiB x 4 ring; more stages in
// flight were slower (6.2 TB/s with 6), and the best vector geometry gave 6.2 TB/s.
constexpr int kDefaultMoverOut = 2;      // HFK_MOVER_BULK
constexpr int kDefaultMoverIn = 2;       // HFK_MOVER_BULK
constexpr int kDefaultMoverGather = 2;   // HFK_MOVER_BULK
// Bulk swap launches below this many bytes use the small ring (see swap_impl): 2 KiB x 4 stages, 64
// single-warp CTAs, at most 256 ids staged at a time = 14 KB of shared memory per CTA.  Measured for
// the layer-wise fp8 pipeline (4 layers = 16.8 MB per launch, one side stream) next to a bf16 GEMM that
// fills the device: 48.3 GB/s in / 49.5 out with the GEMM 1.8 % slower; alone 48.6 / 50.1.
constexpr long long kAutoBulkMinBytes = 256ll << 20;
constexpr int kSwapSmallStageBytes = 2048, kSwapSmallStages = 4, kSwapSmallIdTile = 256;
constexpr int kDefaultSwapCtasBulkSmall = 64;
constexpr int kDefaultSwapCtasVector = 16;
constexpr int kDefaultSwapCtasBulk = 4;
constexpr int kSwapStageBytes = 16384, kSwapStages = 8, kSwapLag = 2;
constexpr int kGatherStageBytes = 32768, kGatherStages = 4, kGatherLag = 2;
constexpr int kGatherHints = 0, kGatherBlocked = 0;  // bulk gather: no L2 hints (see below), interleaved units
// L2 evict-first hints on the gather's bulk copies measured 6.70 TB/s when an un-hinted launch had run
// before in the same process and 6.50 TB/s in a fresh process (un-hinted: 6.67 TB/s either way), so
// they stay off by default.
constexpr int kGatherVectorCtasPerSm = 2;  // vector mover: 256 threads x 8 loads, 2 CTAs per SM
constexpr int kDefaultRowGatherCtas = 32;
constexpr int kDefaultTransferCtas = 32;
constexpr int kDefaultRelayoutCtas = 32;
// Staged swap: copy-engine lanes the slot copies are dealt to, and the largest single copy (a run of
// consecutive slots is cut at this size so that every lane gets work).  Measured on the Llama-3-8B
// step (512 slots of 2 MiB): 1, 2, 3 and 4 lanes all give 50.2 GB/s out / 49.0 in with random slots
// and 55.7-56.0 / 54.0-54.3 with slots in one run, so the copies stay on the caller's stream.
constexpr int kDefaultStagedLanes = 1;
constexpr long long kStagedMaxCopyBytes = 64ll << 20;
// Block migration: 512-thread CTAs per SM (peer loads over NVLink need megabytes in flight).
constexpr int kMigrateCtasPerSm = 2;
// kv_write: whether a lane takes 32 elements of a row, not 16.  16 finish sooner while every warp is resident and a call lasts as long
// as one row's chain; 32 take fewer instructions a row, so they pay where a row has much work (a scale and codes, a norm and a
// rotation) and there are many.  A plain copy has little, and heads up to 64 leave few lanes a row to hide its latency.
// us with 16 and with 32, bf16, 4 K/V heads, rotated with 16 query heads (rows = heads of all tokens):
//   head_dim, form        16384 rows    32768       65536       524288
//   128 to e4m3           2.60, 2.60  3.73, 3.20  5.42, 5.12  34.7, 33.1
//   128 rotated, e4m3     3.53, 3.80  5.43, 5.02  8.89, 8.76  62.3, 62.6
//   256 to e4m3           3.79, 3.05  5.44, 4.50  9.58, 8.78  67.4, 62.6
//   64 to e4m3            2.26, 2.33  2.60, 2.80  3.70, 3.70  18.9, 18.0
//   64 rotated, e4m3      2.95, 3.49  3.61, 4.22  5.55, 5.70  34.3, 35.3
//   16 rotated, e4m3      2.94, 3.00  3.56, 3.31  5.51, 4.33  29.1, 22.6
//   64 copied             2.26, 2.48  2.85, 3.18  4.30, 4.47  22.1, 26.7
//   128 copied            2.80, 2.92  4.36, 4.03  6.40, 6.46  41.4, 42.8
//   16 copied             1.96, 1.90  2.15, 2.01  2.78, 2.21  10.6,  6.9
constexpr bool write_wide(long long rows, int head_dim, bool rope, bool copied) {
  return (rope || !copied) && rows >= (head_dim > 64 ? 1 << 14 : 1 << 16);
}
// Reading an 8-bit cache back: 256-thread CTAs per SM, eight 8-byte loads a lane in flight.  6.9 GB (64 sequences, 4 layers):
// 1113 us with 2, 1186 with 4, 1157 with 8 and half the loads a lane.
constexpr int kGatherDequantCtasPerSm = 2;
// Attention: CTAs of eight warps per SM (their rings take its shared memory).
constexpr int kAttnCtasPerSm = 1;
// Warps of the join that an SM holds at once (about 72 registers a thread).
constexpr int kJoinWarpsPerSm = 28;
// Warps of the join for each of `rows` rows (up to 2^30), so that all of them fit in the `resident` ones.
constexpr int join_warps(long long rows, long long resident) {
  return rows * 16 <= resident ? 16 : rows * 4 <= resident ? 4 : rows * 2 <= resident ? 2 : 1;
}
// Rows of queries (sequences x query heads of a K/V head) above which the prefix goes to the tensor-core kernel.
constexpr int kPrefixTensorMinRows = 32;
// What a CTA of that kernel costs beyond its key tiles, in tiles of about 2.6 us, and how many values of parts (8 bytes to
// and from L2 each) cost a 64th of that.
constexpr int kPrefixTileOverhead = 3;
constexpr int kPrefixPartValues = 15000;

}  // namespace hfk
