// torch operator library `pcie_through` for CUDA: a thin shim that unpacks
// tensors into the C ABI of libhfk_b200.so.
//
// Group R keeps the reference's schemas verbatim
//   gather(Tensor gmEmbed, Tensor gmEmbedDst, Tensor gmIds, int? aiv=None) -> ()
//       (pcieThrough/csrc/host/gather_torch.cpp:60)
//   multi_layer_block_transfer(Tensor deviceBlockCachePtrs, Tensor hostBlockCache, int? aiv=None) -> ()
//   fused_memcpy_multi_layer_block_transfer(Tensor deviceBlockCachePtrs, Tensor hostBlockCache,
//                                           Tensor stagingBlockCache, int? aiv=None) -> ()
//       (pcieThrough/csrc/host/multi_layer_block_transfer_torch.cpp:113-114)
// registered for the CUDA dispatch key where the reference uses PrivateUse1
// (gather_torch.cpp:65-68, multi_layer_block_transfer_torch.cpp:119-122).  Ops
// mutate their destination in place, return nothing and run asynchronously on
// the current stream (pcieThrough/csrc/host/launch_utils.h:28).
//
// Differences that are deliberate: a host tensor outside every registered range
// raises instead of handing a null alias to the kernel
// (multi_layer_block_transfer_torch.cpp:77-78 passes it on unchecked); a table
// that already lives in device memory is used directly (pcieThrough/README.md:18
// promises this, gather_torch.cpp:50-51 breaks it); launch errors are reported.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/hfk_b200.h"

namespace pciethrough {

static void check_rc(int rc, const char *op) {
  TORCH_CHECK(rc == HFK_OK, op, ": ", hfk_strerror(rc), " — ", hfk_last_error_message());
}

static int cores_from(const c10::optional<int64_t> &aiv) {
  // "aiv" keeps its meaning of "how many cores to spend"
  // (multi_layer_block_transfer_torch.cpp:59-64); None selects the tuned default.
  if (!aiv.has_value()) return 0;
  TORCH_CHECK(aiv.value() > 0, "Number of AIV blocks should be positive.");
  return static_cast<int>(aiv.value());
}

// Address a kernel can dereference for `t`: device tensors as they are, host
// tensors through the registry.
static void *device_accessible(const at::Tensor &t, const char *what) {
  if (t.is_cuda()) return t.data_ptr();
  TORCH_CHECK(t.device().is_cpu(), what, ": tensor must live on CPU (registered) or CUDA");
  const uintptr_t alias = hfk_get_device_ptr(reinterpret_cast<uintptr_t>(t.data_ptr()));
  TORCH_CHECK(alias != 0, what,
              ": host tensor is not inside a range registered with heterofusedkernels.memory "
              "(alloc_numa_pinned_tensor / host_register)");
  return reinterpret_cast<void *>(alias);
}

static int ids_are_int64(const at::Tensor &ids, const char *what) {
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, what,
              ": ids must be int64 or int32, got ", c10::toString(ids.scalar_type()));
  TORCH_CHECK(ids.dim() == 1 && ids.is_contiguous(), what, ": ids must be 1-D and contiguous");
  return ids.scalar_type() == at::kLong ? 1 : 0;
}

static void check_ptr_table(const at::Tensor &t, int64_t layers, const char *what, bool on_device) {
  TORCH_CHECK(t.scalar_type() == at::kLong && t.dim() == 1 && t.is_contiguous(), what,
              ": pointer table must be a contiguous 1-D int64 tensor");
  TORCH_CHECK(t.is_cuda() == on_device, what, on_device ? ": pointer table must be on the device"
                                                        : ": pointer table must be on the CPU");
  if (layers >= 0)
    TORCH_CHECK(t.numel() == layers, what, ": pointer table has ", t.numel(), " entries, expected ",
                layers, " (one per layer)");
}

// ---------------------------------------------------------------- Group R ---
void gather(const at::Tensor &gmEmbed, const at::Tensor &gmEmbedDst, const at::Tensor &gmIds,
            c10::optional<int64_t> aiv) {
  const int ctas = cores_from(aiv);
  TORCH_CHECK(gmEmbed.dim() == 2 && gmEmbed.is_contiguous(), "gather: gmEmbed must be a contiguous 2-D tensor");
  TORCH_CHECK(gmEmbedDst.is_cuda() && gmEmbedDst.is_contiguous(), "gather: gmEmbedDst must be a contiguous device tensor");
  const int is64 = ids_are_int64(gmIds, "gather");
  const size_t numIds = static_cast<size_t>(gmIds.size(0));
  const size_t rowBytes = static_cast<size_t>(gmEmbed.element_size()) * gmEmbed.size(1);
  TORCH_CHECK(static_cast<size_t>(gmEmbedDst.nbytes()) >= numIds * rowBytes,
              "gather: gmEmbedDst holds fewer than numIds rows");
  const c10::cuda::CUDAGuard guard(gmEmbedDst.device());
  check_rc(hfk_gather(device_accessible(gmEmbed, "gather(gmEmbed)"), gmEmbedDst.data_ptr(),
                      device_accessible(gmIds, "gather(gmIds)"), is64, numIds, rowBytes,
                      static_cast<size_t>(gmEmbed.size(0)), ctas,
                      at::cuda::getCurrentCUDAStream().stream()),
           "gather");
}

struct BlockGeometry {
  int64_t B, L, H, D, elt;
};
static BlockGeometry geometry_of(const at::Tensor &hostBlockCache, const char *op) {
  // the shape comes from the HOST tensor [BlockSize, Layers, Heads, HeadDim]
  // (multi_layer_block_transfer_torch.cpp:67-71)
  TORCH_CHECK(hostBlockCache.dim() == 4 && hostBlockCache.is_contiguous(), op,
              ": hostBlockCache must be a contiguous [BlockSize, Layers, Heads, HeadDim] tensor");
  return {hostBlockCache.size(0), hostBlockCache.size(1), hostBlockCache.size(2),
          hostBlockCache.size(3), static_cast<int64_t>(hostBlockCache.element_size())};
}

void multi_layer_block_transfer(const at::Tensor &deviceBlockCachePtrs,
                                const at::Tensor &hostBlockCache, c10::optional<int64_t> aiv) {
  const int ctas = cores_from(aiv);
  const BlockGeometry g = geometry_of(hostBlockCache, "multi_layer_block_transfer");
  check_ptr_table(deviceBlockCachePtrs, g.L, "multi_layer_block_transfer(deviceBlockCachePtrs)", true);
  const c10::cuda::CUDAGuard guard(deviceBlockCachePtrs.device());
  check_rc(hfk_multi_layer_block_transfer(
               reinterpret_cast<void *const *>(deviceBlockCachePtrs.data_ptr()),
               device_accessible(hostBlockCache, "multi_layer_block_transfer(hostBlockCache)"), g.B,
               g.L, g.H, g.D, g.elt, ctas, at::cuda::getCurrentCUDAStream().stream()),
           "multi_layer_block_transfer");
}

void fused_memcpy_multi_layer_block_transfer(const at::Tensor &deviceBlockCachePtrs,
                                             const at::Tensor &hostBlockCache,
                                             const at::Tensor &stagingBlockCache,
                                             c10::optional<int64_t> aiv) {
  const int ctas = cores_from(aiv);
  const BlockGeometry g = geometry_of(hostBlockCache, "fused_memcpy_multi_layer_block_transfer");
  check_ptr_table(deviceBlockCachePtrs, g.L, "fused_memcpy_multi_layer_block_transfer(deviceBlockCachePtrs)", true);
  TORCH_CHECK(hostBlockCache.device().is_cpu(), "fused_memcpy_multi_layer_block_transfer: hostBlockCache must be a CPU tensor");
  TORCH_CHECK(stagingBlockCache.is_cuda() && stagingBlockCache.is_contiguous() &&
                  stagingBlockCache.nbytes() >= hostBlockCache.nbytes(),
              "fused_memcpy_multi_layer_block_transfer: stagingBlockCache must be a contiguous device "
              "tensor at least as large as hostBlockCache");
  const c10::cuda::CUDAGuard guard(stagingBlockCache.device());
  check_rc(hfk_fused_memcpy_multi_layer_block_transfer(
               reinterpret_cast<void *const *>(deviceBlockCachePtrs.data_ptr()),
               hostBlockCache.data_ptr(), stagingBlockCache.data_ptr(), g.B, g.L, g.H, g.D, g.elt,
               ctas, at::cuda::getCurrentCUDAStream().stream()),
           "fused_memcpy_multi_layer_block_transfer");
}

// ---------------------------------------------------------------- Group N ---
// hostPool is a CPU tensor [slots, layers, 2, ...] whose trailing dimensions are
// contiguous and form one chunk; slot / layer / K|V strides are taken from the
// tensor, so a layer-major pool can be passed as a permuted view.
static hfk_swap_desc swap_desc(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs,
                               const at::Tensor &hostPool, const at::Tensor &deviceBlockIds,
                               const at::Tensor &hostSlotIds, int64_t numDeviceBlocks,
                               c10::optional<int64_t> deviceBlockStride, bool arrays_on_device,
                               const char *op) {
  TORCH_CHECK(hostPool.device().is_cpu() && hostPool.dim() >= 4, op,
              ": hostPool must be a CPU tensor [slots, layers, 2, ...chunk dims]");
  TORCH_CHECK(hostPool.size(2) == 2, op, ": hostPool dimension 2 must have size 2 (K, V)");
  const int64_t elt = hostPool.element_size();
  int64_t chunk_elems = 1;
  for (int64_t d = hostPool.dim() - 1; d >= 3; --d) {
    TORCH_CHECK(hostPool.stride(d) == chunk_elems, op, ": the chunk dimensions of hostPool must be contiguous");
    chunk_elems *= hostPool.size(d);
  }
  hfk_swap_desc d;
  d.layers = static_cast<int>(hostPool.size(1));
  check_ptr_table(kLayerPtrs, d.layers, op, arrays_on_device);
  check_ptr_table(vLayerPtrs, d.layers, op, arrays_on_device);
  d.ids_are_int64 = ids_are_int64(deviceBlockIds, op);
  TORCH_CHECK(ids_are_int64(hostSlotIds, op) == d.ids_are_int64, op, ": both id lists must have the same dtype");
  TORCH_CHECK(deviceBlockIds.numel() == hostSlotIds.numel(), op, ": id lists differ in length");
  TORCH_CHECK(deviceBlockIds.is_cuda() == arrays_on_device && hostSlotIds.is_cuda() == arrays_on_device,
              op, arrays_on_device ? ": id lists must be device tensors" : ": id lists must be CPU tensors");
  d.k_layer_ptrs = reinterpret_cast<void *const *>(kLayerPtrs.data_ptr());
  d.v_layer_ptrs = reinterpret_cast<void *const *>(vLayerPtrs.data_ptr());
  d.host_pool = arrays_on_device ? device_accessible(hostPool, op) : hostPool.data_ptr();
  d.device_block_ids = deviceBlockIds.data_ptr();
  d.host_slot_ids = hostSlotIds.data_ptr();
  d.n_blocks = deviceBlockIds.numel();
  d.block_bytes = chunk_elems * elt;
  d.device_block_stride = deviceBlockStride.has_value() ? deviceBlockStride.value() : d.block_bytes;
  d.host_slot_stride = hostPool.stride(0) * elt;
  d.host_layer_stride = hostPool.stride(1) * elt;
  d.host_kv_stride = hostPool.stride(2) * elt;
  d.num_device_blocks = numDeviceBlocks;
  d.num_host_slots = hostPool.size(0);
  return d;
}

static int mover_from(const c10::optional<int64_t> &mover) {
  return mover.has_value() ? static_cast<int>(mover.value()) : HFK_MOVER_AUTO;
}

void swap_out(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs, const at::Tensor &hostPool,
              const at::Tensor &deviceBlockIds, const at::Tensor &hostSlotIds,
              int64_t numDeviceBlocks, c10::optional<int64_t> deviceBlockStride,
              c10::optional<int64_t> aiv, c10::optional<int64_t> mover, c10::optional<int64_t> paceMBs) {
  const int ctas = cores_from(aiv);
  const hfk_swap_desc d = swap_desc(kLayerPtrs, vLayerPtrs, hostPool, deviceBlockIds, hostSlotIds,
                                    numDeviceBlocks, deviceBlockStride, true, "swap_out");
  const c10::cuda::CUDAGuard guard(kLayerPtrs.device());
  // paceMBs: stores paced to that many MB/s (for a swap-out that shares the link with a swap-in)
  check_rc(hfk_swap_out_paced(&d, mover_from(mover), ctas, paceMBs.has_value() ? static_cast<int>(paceMBs.value()) : 0,
                              at::cuda::getCurrentCUDAStream().stream()),
           "swap_out");
}

void swap_in(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs, const at::Tensor &hostPool,
             const at::Tensor &deviceBlockIds, const at::Tensor &hostSlotIds, int64_t numDeviceBlocks,
             c10::optional<int64_t> deviceBlockStride, c10::optional<int64_t> aiv,
             c10::optional<int64_t> mover) {
  const int ctas = cores_from(aiv);
  const hfk_swap_desc d = swap_desc(kLayerPtrs, vLayerPtrs, hostPool, deviceBlockIds, hostSlotIds,
                                    numDeviceBlocks, deviceBlockStride, true, "swap_in");
  const c10::cuda::CUDAGuard guard(kLayerPtrs.device());
  check_rc(hfk_swap_in(&d, mover_from(mover), ctas, at::cuda::getCurrentCUDAStream().stream()), "swap_in");
}

// Staged movers: a packing kernel plus one copy-engine transfer per host slot.  hostSlotIds is a
// CPU tensor here (the copies are addressed on the host); staging is a device byte buffer of at
// least one slot.
static void swap_staged(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs, const at::Tensor &hostPool,
                        const at::Tensor &deviceBlockIds, const at::Tensor &hostSlotIds, const at::Tensor &staging,
                        int64_t numDeviceBlocks, c10::optional<int64_t> deviceBlockStride,
                        c10::optional<int64_t> aiv, int to_host, const char *op) {
  const int ctas = cores_from(aiv);
  TORCH_CHECK(hostSlotIds.device().is_cpu(), op, ": hostSlotIds must be a CPU tensor");
  TORCH_CHECK(staging.is_cuda() && staging.is_contiguous(), op, ": staging must be a contiguous device tensor");
  // build the descriptor with the device id list standing in for both lists, then attach the host list
  hfk_swap_desc d = swap_desc(kLayerPtrs, vLayerPtrs, hostPool, deviceBlockIds, deviceBlockIds, numDeviceBlocks,
                              deviceBlockStride, true, op);
  TORCH_CHECK(ids_are_int64(hostSlotIds, op) == d.ids_are_int64 && hostSlotIds.numel() == deviceBlockIds.numel(),
              op, ": hostSlotIds must match deviceBlockIds in dtype and length");
  const c10::cuda::CUDAGuard guard(kLayerPtrs.device());
  check_rc(hfk_swap_staged(&d, hostSlotIds.data_ptr(), hostPool.data_ptr(), staging.data_ptr(),
                           static_cast<size_t>(staging.nbytes()), to_host, ctas,
                           at::cuda::getCurrentCUDAStream().stream()),
           op);
}

void swap_out_staged(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs, const at::Tensor &hostPool,
                     const at::Tensor &deviceBlockIds, const at::Tensor &hostSlotIds, const at::Tensor &staging,
                     int64_t numDeviceBlocks, c10::optional<int64_t> deviceBlockStride, c10::optional<int64_t> aiv) {
  swap_staged(kLayerPtrs, vLayerPtrs, hostPool, deviceBlockIds, hostSlotIds, staging, numDeviceBlocks,
              deviceBlockStride, aiv, 1, "swap_out_staged");
}

void swap_in_staged(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs, const at::Tensor &hostPool,
                    const at::Tensor &deviceBlockIds, const at::Tensor &hostSlotIds, const at::Tensor &staging,
                    int64_t numDeviceBlocks, c10::optional<int64_t> deviceBlockStride, c10::optional<int64_t> aiv) {
  swap_staged(kLayerPtrs, vLayerPtrs, hostPool, deviceBlockIds, hostSlotIds, staging, numDeviceBlocks,
              deviceBlockStride, aiv, 0, "swap_in_staged");
}

// Device that owns the memory a raw device address points into (the first entry of a CPU-resident
// pointer table); falls back to the current device when the driver does not know the address.
static c10::Device device_of_address(int64_t address) {
  cudaPointerAttributes attr;
  if (address != 0 && cudaPointerGetAttributes(&attr, reinterpret_cast<const void *>(address)) == cudaSuccess &&
      attr.type == cudaMemoryTypeDevice)
    return c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(attr.device));
  cudaGetLastError();
  return c10::Device(c10::kCUDA, c10::cuda::current_device());
}

// Copy-engine twins: every tensor argument lives on the CPU (the addresses are
// formed on the host); the copies run on the current stream of the device that
// owns the cache (taken from the first layer pointer).
void swap_out_copy_engine(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs,
                          const at::Tensor &hostPool, const at::Tensor &deviceBlockIds,
                          const at::Tensor &hostSlotIds, int64_t numDeviceBlocks,
                          c10::optional<int64_t> deviceBlockStride) {
  const hfk_swap_desc d = swap_desc(kLayerPtrs, vLayerPtrs, hostPool, deviceBlockIds, hostSlotIds,
                                    numDeviceBlocks, deviceBlockStride, false, "swap_out_copy_engine");
  const c10::cuda::CUDAGuard guard(device_of_address(kLayerPtrs.numel() ? kLayerPtrs[0].item<int64_t>() : 0));
  check_rc(hfk_swap_copy_engine(&d, 1, at::cuda::getCurrentCUDAStream().stream()), "swap_out_copy_engine");
}

void swap_in_copy_engine(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs,
                         const at::Tensor &hostPool, const at::Tensor &deviceBlockIds,
                         const at::Tensor &hostSlotIds, int64_t numDeviceBlocks,
                         c10::optional<int64_t> deviceBlockStride) {
  const hfk_swap_desc d = swap_desc(kLayerPtrs, vLayerPtrs, hostPool, deviceBlockIds, hostSlotIds,
                                    numDeviceBlocks, deviceBlockStride, false, "swap_in_copy_engine");
  const c10::cuda::CUDAGuard guard(device_of_address(kLayerPtrs.numel() ? kLayerPtrs[0].item<int64_t>() : 0));
  check_rc(hfk_swap_copy_engine(&d, 0, at::cuda::getCurrentCUDAStream().stream()), "swap_in_copy_engine");
}

// Multi-block swap in the reference's host block format.  hostPool: registered CPU tensor
// [slots, BlockSize, Layers, Heads, HeadDim] (each slot laid out like hostBlockCache of
// multi_layer_block_transfer); layerPtrs: device int64 [Layers], layer l's cache being
// [numDeviceBlocks, Heads, BlockSize, HeadDim].
static hfk_relayout_desc relayout_desc(const at::Tensor &layerPtrs, const at::Tensor &hostPool,
                                       const at::Tensor &deviceBlockIds, const at::Tensor &hostSlotIds,
                                       int64_t numDeviceBlocks, c10::optional<int64_t> deviceBlockStride,
                                       const char *op) {
  TORCH_CHECK(hostPool.device().is_cpu() && hostPool.dim() == 5, op,
              ": hostPool must be a CPU tensor [slots, BlockSize, Layers, Heads, HeadDim]");
  TORCH_CHECK(hostPool[0].is_contiguous(), op, ": every host slot must be contiguous");
  const int64_t elt = hostPool.element_size();
  hfk_relayout_desc d;
  d.layers = static_cast<int>(hostPool.size(2));
  check_ptr_table(layerPtrs, d.layers, op, true);
  d.ids_are_int64 = ids_are_int64(deviceBlockIds, op);
  TORCH_CHECK(ids_are_int64(hostSlotIds, op) == d.ids_are_int64, op, ": both id lists must have the same dtype");
  TORCH_CHECK(deviceBlockIds.numel() == hostSlotIds.numel(), op, ": id lists differ in length");
  TORCH_CHECK(deviceBlockIds.is_cuda() && hostSlotIds.is_cuda(), op, ": id lists must be device tensors");
  d.layer_ptrs = reinterpret_cast<void *const *>(layerPtrs.data_ptr());
  d.host_pool = device_accessible(hostPool, op);
  d.device_block_ids = deviceBlockIds.data_ptr();
  d.host_slot_ids = hostSlotIds.data_ptr();
  d.n_blocks = deviceBlockIds.numel();
  d.block_size = hostPool.size(1);
  d.heads = hostPool.size(3);
  d.head_bytes = hostPool.size(4) * elt;
  d.device_block_stride = deviceBlockStride.has_value() ? deviceBlockStride.value()
                                                        : d.heads * d.block_size * d.head_bytes;
  d.host_slot_stride = hostPool.stride(0) * elt;
  d.num_device_blocks = numDeviceBlocks;
  d.num_host_slots = hostPool.size(0);
  return d;
}

void swap_in_relayout(const at::Tensor &layerPtrs, const at::Tensor &hostPool, const at::Tensor &deviceBlockIds,
                      const at::Tensor &hostSlotIds, int64_t numDeviceBlocks,
                      c10::optional<int64_t> deviceBlockStride, c10::optional<int64_t> aiv) {
  const int ctas = cores_from(aiv);
  const hfk_relayout_desc d = relayout_desc(layerPtrs, hostPool, deviceBlockIds, hostSlotIds, numDeviceBlocks,
                                            deviceBlockStride, "swap_in_relayout");
  const c10::cuda::CUDAGuard guard(layerPtrs.device());
  check_rc(hfk_swap_relayout(&d, 0, ctas, at::cuda::getCurrentCUDAStream().stream()), "swap_in_relayout");
}

void swap_out_relayout(const at::Tensor &layerPtrs, const at::Tensor &hostPool, const at::Tensor &deviceBlockIds,
                       const at::Tensor &hostSlotIds, int64_t numDeviceBlocks,
                       c10::optional<int64_t> deviceBlockStride, c10::optional<int64_t> aiv) {
  const int ctas = cores_from(aiv);
  const hfk_relayout_desc d = relayout_desc(layerPtrs, hostPool, deviceBlockIds, hostSlotIds, numDeviceBlocks,
                                            deviceBlockStride, "swap_out_relayout");
  const c10::cuda::CUDAGuard guard(layerPtrs.device());
  check_rc(hfk_swap_relayout(&d, 1, ctas, at::cuda::getCurrentCUDAStream().stream()), "swap_out_relayout");
}

// kOut / vOut: [layers, total_tokens, ...token dims]; blockTables: [num_seqs, max_blocks];
// seqLens: [num_seqs].
void paged_gather(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs, const at::Tensor &kOut,
                  const at::Tensor &vOut, const at::Tensor &blockTables, const at::Tensor &seqLens,
                  int64_t blockSize, int64_t numDeviceBlocks, c10::optional<int64_t> deviceBlockStride,
                  c10::optional<int64_t> aiv, c10::optional<int64_t> mover) {
  const int ctas = cores_from(aiv);
  TORCH_CHECK(kOut.is_cuda() && vOut.is_cuda() && kOut.dim() >= 3 && kOut.sizes() == vOut.sizes() &&
                  kOut.is_contiguous() && vOut.is_contiguous(),
              "paged_gather: kOut and vOut must be contiguous device tensors [layers, total_tokens, ...] of equal shape");
  TORCH_CHECK(blockTables.is_cuda() && blockTables.dim() == 2 && blockTables.stride(1) == 1,
              "paged_gather: blockTables must be a device tensor [num_seqs, max_blocks] with unit inner stride");
  TORCH_CHECK(seqLens.is_cuda() && seqLens.dim() == 1 && seqLens.is_contiguous() &&
                  seqLens.scalar_type() == blockTables.scalar_type() &&
                  seqLens.size(0) == blockTables.size(0),
              "paged_gather: seqLens must be a device tensor [num_seqs] of the same dtype as blockTables");
  TORCH_CHECK(blockTables.scalar_type() == at::kLong || blockTables.scalar_type() == at::kInt,
              "paged_gather: blockTables must be int64 or int32");
  hfk_paged_gather_desc d;
  d.layers = static_cast<int>(kOut.size(0));
  check_ptr_table(kLayerPtrs, d.layers, "paged_gather(kLayerPtrs)", true);
  check_ptr_table(vLayerPtrs, d.layers, "paged_gather(vLayerPtrs)", true);
  d.k_layer_ptrs = reinterpret_cast<void *const *>(kLayerPtrs.data_ptr());
  d.v_layer_ptrs = reinterpret_cast<void *const *>(vLayerPtrs.data_ptr());
  d.k_out = kOut.data_ptr();
  d.v_out = vOut.data_ptr();
  d.total_tokens = kOut.size(1);
  d.token_bytes = kOut.stride(1) * kOut.element_size();
  d.out_layer_stride = kOut.stride(0) * kOut.element_size();
  d.block_tables = blockTables.data_ptr();
  d.seq_lens = seqLens.data_ptr();
  d.ids_are_int64 = blockTables.scalar_type() == at::kLong ? 1 : 0;
  d.num_seqs = blockTables.size(0);
  d.max_blocks_per_seq = blockTables.size(1);
  d.block_table_stride = blockTables.stride(0);
  d.block_size = blockSize;
  d.device_block_stride =
      deviceBlockStride.has_value() ? deviceBlockStride.value() : blockSize * d.token_bytes;
  d.num_device_blocks = numDeviceBlocks;
  const c10::cuda::CUDAGuard guard(kOut.device());
  check_rc(hfk_paged_gather(&d, mover_from(mover), ctas, at::cuda::getCurrentCUDAStream().stream()),
           "paged_gather");
}

// Block migration between two caches.  The four pointer tables and the two id lists are device
// tensors on the GPU that runs the kernel (the current device of the tables); the addresses in
// the tables may belong to a peer GPU whose access has been enabled (torch enables it on the
// first cross-device copy; hfk_enable_peer_access does it explicitly).
void migrate_blocks(const at::Tensor &srcKLayerPtrs, const at::Tensor &srcVLayerPtrs,
                    const at::Tensor &dstKLayerPtrs, const at::Tensor &dstVLayerPtrs,
                    const at::Tensor &srcBlockIds, const at::Tensor &dstBlockIds, int64_t blockBytes,
                    int64_t numSrcBlocks, int64_t numDstBlocks, c10::optional<int64_t> srcBlockStride,
                    c10::optional<int64_t> dstBlockStride, c10::optional<int64_t> aiv) {
  const int ctas = cores_from(aiv);
  hfk_migrate_desc d;
  d.layers = static_cast<int>(srcKLayerPtrs.numel());
  check_ptr_table(srcKLayerPtrs, d.layers, "migrate_blocks(srcKLayerPtrs)", true);
  check_ptr_table(srcVLayerPtrs, d.layers, "migrate_blocks(srcVLayerPtrs)", true);
  check_ptr_table(dstKLayerPtrs, d.layers, "migrate_blocks(dstKLayerPtrs)", true);
  check_ptr_table(dstVLayerPtrs, d.layers, "migrate_blocks(dstVLayerPtrs)", true);
  d.ids_are_int64 = ids_are_int64(srcBlockIds, "migrate_blocks");
  TORCH_CHECK(ids_are_int64(dstBlockIds, "migrate_blocks") == d.ids_are_int64,
              "migrate_blocks: both id lists must have the same dtype");
  TORCH_CHECK(srcBlockIds.numel() == dstBlockIds.numel(), "migrate_blocks: id lists differ in length");
  TORCH_CHECK(srcBlockIds.is_cuda() && dstBlockIds.is_cuda(), "migrate_blocks: id lists must be device tensors");
  const auto dev = srcKLayerPtrs.device();
  TORCH_CHECK(srcVLayerPtrs.device() == dev && dstKLayerPtrs.device() == dev && dstVLayerPtrs.device() == dev &&
                  srcBlockIds.device() == dev && dstBlockIds.device() == dev,
              "migrate_blocks: pointer tables and id lists must live on the GPU that runs the kernel");
  d.src_k_layer_ptrs = reinterpret_cast<void *const *>(srcKLayerPtrs.data_ptr());
  d.src_v_layer_ptrs = reinterpret_cast<void *const *>(srcVLayerPtrs.data_ptr());
  d.dst_k_layer_ptrs = reinterpret_cast<void *const *>(dstKLayerPtrs.data_ptr());
  d.dst_v_layer_ptrs = reinterpret_cast<void *const *>(dstVLayerPtrs.data_ptr());
  d.src_block_ids = srcBlockIds.data_ptr();
  d.dst_block_ids = dstBlockIds.data_ptr();
  d.n_blocks = srcBlockIds.numel();
  d.block_bytes = blockBytes;
  d.src_block_stride = srcBlockStride.has_value() ? srcBlockStride.value() : blockBytes;
  d.dst_block_stride = dstBlockStride.has_value() ? dstBlockStride.value() : blockBytes;
  d.num_src_blocks = numSrcBlocks;
  d.num_dst_blocks = numDstBlocks;
  const c10::cuda::CUDAGuard guard(dev);
  check_rc(hfk_migrate_blocks(&d, ctas, at::cuda::getCurrentCUDAStream().stream()), "migrate_blocks");
}

// ---------------------------------------------------------------- Group A ---
// One layer's cache of an attention layer.  A 16-bit cache is [numDeviceBlocks, blockSize, kvHeads, headDim]; an
// 8-bit cache is uint8 [numDeviceBlocks, at least hfk_kv_block_bytes].  Only the stride between pages is free.
static int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? HFK_TYPE_BF16 : t == at::kHalf ? HFK_TYPE_FP16 : t == at::kFloat ? HFK_TYPE_FP32 : -1;
}

static void check_cache(const at::Tensor &kCache, const at::Tensor &vCache, at::ScalarType type, int64_t blockSize,
                        int64_t kvHeads, int64_t headDim, int64_t kvFormat, const char *op) {
  TORCH_CHECK(kvFormat >= HFK_KV_RAW && kvFormat <= HFK_KV_INT8, op, ": kvFormat must be 0 (16-bit), 1 (e4m3) or 2 (int8)");
  TORCH_CHECK(kCache.is_cuda() && kCache.device() == vCache.device(), op, ": kCache and vCache must be on one CUDA device");
  TORCH_CHECK(kCache.sizes() == vCache.sizes() && kCache.strides() == vCache.strides() && kCache.scalar_type() == vCache.scalar_type(),
              op, ": kCache and vCache must have the same shape, strides and dtype");
  if (kvFormat == HFK_KV_RAW) {
    TORCH_CHECK(kCache.scalar_type() == type, op, ": a 16-bit cache must have the dtype of the call, ", c10::toString(type));
    TORCH_CHECK(kCache.dim() == 4 && kCache.size(1) == blockSize && kCache.size(2) == kvHeads && kCache.size(3) == headDim, op,
                ": a 16-bit cache must be [numDeviceBlocks, blockSize, kvHeads, headDim]");
    TORCH_CHECK(kCache.stride(3) == 1 && kCache.stride(2) == headDim && kCache.stride(1) == headDim * kvHeads, op,
                ": the pages of a 16-bit cache must be contiguous");
  } else {
    TORCH_CHECK(kCache.scalar_type() == at::kByte && kCache.dim() == 2 && kCache.stride(1) == 1, op,
                ": an 8-bit cache must be uint8 [numDeviceBlocks, page bytes] with contiguous pages");
    const size_t page = hfk_kv_block_bytes(blockSize, kvHeads, headDim, static_cast<int>(kvFormat));
    TORCH_CHECK(page > 0 && static_cast<size_t>(kCache.size(1)) >= page, op, ": a page of this cache has ", page, " bytes, the tensor's has ",
                kCache.size(1));
  }
}

static hfk_rows rows_of(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK(t.dim() == 3 && (t.stride(2) == 1 || t.size(2) <= 1), op, ": ", name, " must be [tokens, heads, headDim] with contiguous rows");
  hfk_rows r;
  r.base = t.data_ptr();
  // a dimension of size 1 has no stride that matters
  r.token_stride = t.size(0) > 1 ? t.stride(0) * t.element_size() : 0;
  r.head_stride = t.size(1) > 1 ? t.stride(1) * t.element_size() : 0;
  return r;
}

static hfk_kv_write_desc write_desc(const at::Tensor &k, const at::Tensor &v, const at::Tensor &kCache, const at::Tensor &vCache,
                                    const at::Tensor &slotIds, int64_t blockSize, int64_t kvFormat, const char *op) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), op,
              ": k and v must be device tensors [tokens, kvHeads, headDim] of the same shape and dtype");
  TORCH_CHECK(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf, op, ": k and v must be bfloat16 or float16");
  check_cache(kCache, vCache, k.scalar_type(), blockSize, k.size(1), k.size(2), kvFormat, op);
  hfk_kv_write_desc d;
  d.ids_are_int64 = ids_are_int64(slotIds, op);
  TORCH_CHECK(slotIds.numel() == k.size(0), op, ": ", slotIds.numel(), " slot ids for ", k.size(0), " tokens");
  TORCH_CHECK(v.device() == k.device() && kCache.device() == k.device() && slotIds.device() == k.device(), op,
              ": all tensors must be on one device");
  TORCH_CHECK(k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX, op, ": too many heads");
  d.k = rows_of(k, op, "k");
  d.v = rows_of(v, op, "v");
  d.k_cache = kCache.data_ptr();
  d.v_cache = vCache.data_ptr();
  d.slot_ids = slotIds.data_ptr();
  d.type = type_code(k.scalar_type());
  d.kv_format = static_cast<int>(kvFormat);
  d.kv_heads = static_cast<int>(k.size(1));
  d.head_dim = static_cast<int>(k.size(2));
  d.tokens = k.size(0);
  d.block_size = blockSize;
  d.device_block_stride = kCache.stride(0) * kCache.element_size();
  d.num_device_blocks = kCache.size(0);
  return d;
}

void kv_write(const at::Tensor &k, const at::Tensor &v, const at::Tensor &kCache, const at::Tensor &vCache, const at::Tensor &slotIds,
              int64_t blockSize, int64_t kvFormat) {
  const hfk_kv_write_desc d = write_desc(k, v, kCache, vCache, slotIds, blockSize, kvFormat, "kv_write");
  const c10::cuda::CUDAGuard guard(k.device());
  check_rc(hfk_kv_write(&d, at::cuda::getCurrentCUDAStream().stream()), "kv_write");
}

static const void *weight_of(const c10::optional<at::Tensor> &w, const at::Tensor &k, const char *name) {
  if (!w.has_value() || !w->defined()) return nullptr;
  TORCH_CHECK(w->device() == k.device() && w->scalar_type() == k.scalar_type() && w->is_contiguous() && w->dim() == 1 && w->numel() == k.size(2),
              "qk_norm_rope_write: ", name, " must be a contiguous [headDim] tensor of k's dtype and device");
  return w->data_ptr();
}

void qk_norm_rope_write(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &qOut, const at::Tensor &kCache,
                        const at::Tensor &vCache, const at::Tensor &slotIds, const at::Tensor &positions, const at::Tensor &cosSin,
                        int64_t blockSize, int64_t kvFormat, const c10::optional<at::Tensor> &qWeight,
                        const c10::optional<at::Tensor> &kWeight, double eps, bool interleaved) {
  const char *op = "qk_norm_rope_write";
  const hfk_kv_write_desc d = write_desc(k, v, kCache, vCache, slotIds, blockSize, kvFormat, op);
  TORCH_CHECK(q.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.scalar_type() == k.scalar_type(), op,
              ": q must be [tokens, qHeads, headDim] of k's dtype");
  TORCH_CHECK(qOut.sizes() == q.sizes() && qOut.scalar_type() == q.scalar_type(), op, ": qOut must have q's shape and dtype");
  TORCH_CHECK(q.size(1) <= INT32_MAX, op, ": too many heads");
  TORCH_CHECK(cosSin.scalar_type() == at::kFloat && cosSin.dim() == 2 && cosSin.is_contiguous(), op,
              ": cosSin must be a contiguous float32 [maxPositions, rotDim] tensor (cosines, then sines)");
  hfk_norm_rope_desc n;
  n.positions_are_int64 = ids_are_int64(positions, op);
  TORCH_CHECK(positions.numel() == k.size(0), op, ": ", positions.numel(), " positions for ", k.size(0), " tokens");
  TORCH_CHECK(q.device() == k.device() && qOut.device() == k.device() && positions.device() == k.device() && cosSin.device() == k.device(),
              op, ": all tensors must be on one device");
  TORCH_CHECK(cosSin.size(1) <= k.size(2), op, ": rotDim ", cosSin.size(1), " is larger than headDim");
  n.q = rows_of(q, op, "q");
  n.q_out = rows_of(qOut, op, "qOut");
  n.q_heads = static_cast<int>(q.size(1));
  n.rot_dim = static_cast<int>(cosSin.size(1));
  n.interleaved = interleaved ? 1 : 0;
  n.positions = positions.data_ptr();
  n.cos_sin = cosSin.data_ptr<float>();
  n.max_positions = cosSin.size(0);
  n.q_weight = weight_of(qWeight, k, "qWeight");
  n.k_weight = weight_of(kWeight, k, "kWeight");
  n.eps = static_cast<float>(eps);
  const c10::cuda::CUDAGuard guard(k.device());
  check_rc(hfk_qk_norm_rope_write(&d, &n, at::cuda::getCurrentCUDAStream().stream()), op);
}

// kOut / vOut: [layers, total_tokens, kvHeads, headDim] of bfloat16, float16 or float32.
void paged_gather_dequant(const at::Tensor &kLayerPtrs, const at::Tensor &vLayerPtrs, const at::Tensor &kOut, const at::Tensor &vOut,
                          const at::Tensor &blockTables, const at::Tensor &seqLens, int64_t blockSize, int64_t numDeviceBlocks,
                          int64_t kvFormat, c10::optional<int64_t> deviceBlockStride, c10::optional<int64_t> aiv) {
  const char *op = "paged_gather_dequant";
  const int ctas = cores_from(aiv);
  TORCH_CHECK(kOut.is_cuda() && kOut.dim() == 4 && kOut.sizes() == vOut.sizes() && kOut.is_contiguous() && vOut.is_contiguous() &&
                  kOut.scalar_type() == vOut.scalar_type(),
              op, ": kOut and vOut must be contiguous device tensors [layers, total_tokens, kvHeads, headDim] of equal shape and dtype");
  const int out_type = type_code(kOut.scalar_type());
  TORCH_CHECK(out_type >= 0, op, ": kOut must be bfloat16, float16 or float32");
  TORCH_CHECK(kvFormat == HFK_KV_E4M3 || kvFormat == HFK_KV_INT8, op, ": kvFormat must be 1 (e4m3) or 2 (int8); paged_gather reads a 16-bit cache");
  TORCH_CHECK(blockTables.scalar_type() == at::kLong || blockTables.scalar_type() == at::kInt, op, ": blockTables must be int64 or int32");
  TORCH_CHECK(blockTables.dim() == 2 && (blockTables.stride(1) == 1 || blockTables.size(1) <= 1), op,
              ": blockTables must be [num_seqs, max_blocks] with unit inner stride");
  TORCH_CHECK(seqLens.dim() == 1 && seqLens.is_contiguous() && seqLens.scalar_type() == blockTables.scalar_type() &&
                  seqLens.size(0) == blockTables.size(0),
              op, ": seqLens must be [num_seqs] of the same dtype as blockTables");
  const auto dev = kOut.device();
  TORCH_CHECK(vOut.device() == dev && blockTables.device() == dev && seqLens.device() == dev && kLayerPtrs.device() == dev &&
                  vLayerPtrs.device() == dev,
              op, ": all tensors must be on one device");
  hfk_paged_gather_desc d;
  d.layers = static_cast<int>(kOut.size(0));
  check_ptr_table(kLayerPtrs, d.layers, "paged_gather_dequant(kLayerPtrs)", true);
  check_ptr_table(vLayerPtrs, d.layers, "paged_gather_dequant(vLayerPtrs)", true);
  TORCH_CHECK(kOut.size(2) <= INT32_MAX, op, ": too many heads");
  d.k_layer_ptrs = reinterpret_cast<void *const *>(kLayerPtrs.data_ptr());
  d.v_layer_ptrs = reinterpret_cast<void *const *>(vLayerPtrs.data_ptr());
  d.k_out = kOut.data_ptr();
  d.v_out = vOut.data_ptr();
  d.total_tokens = kOut.size(1);
  if (d.total_tokens == 0) return;  // an empty output has no address
  d.token_bytes = kOut.size(2) * kOut.size(3);
  d.out_layer_stride = kOut.stride(0) * kOut.element_size();
  d.block_tables = blockTables.data_ptr();
  d.seq_lens = seqLens.data_ptr();
  d.ids_are_int64 = blockTables.scalar_type() == at::kLong ? 1 : 0;
  d.num_seqs = blockTables.size(0);
  d.max_blocks_per_seq = blockTables.size(1);
  d.block_table_stride = blockTables.size(0) > 1 ? blockTables.stride(0) : blockTables.size(1);  // one row has no stride that matters
  d.block_size = blockSize;
  d.device_block_stride = deviceBlockStride.has_value()
                              ? deviceBlockStride.value()
                              : static_cast<int64_t>(hfk_kv_block_bytes(blockSize, kOut.size(2), kOut.size(3), static_cast<int>(kvFormat)));
  d.num_device_blocks = numDeviceBlocks;
  const c10::cuda::CUDAGuard guard(dev);
  check_rc(hfk_paged_gather_dequant(&d, static_cast<int>(kvFormat), static_cast<int>(kOut.size(2)), out_type, ctas,
                                    at::cuda::getCurrentCUDAStream().stream()),
           op);
}

static hfk_prefix_attention_desc attention_desc(const at::Tensor &q, int64_t prefixLen, const at::Tensor &blockTables, int64_t blockSize,
                                                int64_t kvHeads, int64_t kvFormat, const char *op) {
  TORCH_CHECK(q.dim() == 3 && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf), op,
              ": q must be a bfloat16 or float16 tensor [num_seqs, qHeads, headDim]");
  TORCH_CHECK(kvHeads > 0 && q.size(1) > 0 && q.size(1) % kvHeads == 0 && q.size(1) <= INT32_MAX, op, ": ", q.size(1),
              " query heads are not a multiple of kvHeads ", kvHeads);
  TORCH_CHECK(blockTables.dim() == 2, op, ": blockTables must be [num_seqs, max_blocks]");
  hfk_prefix_attention_desc d = {};
  d.type = type_code(q.scalar_type());
  d.kv_format = static_cast<int>(kvFormat);
  d.kv_heads = static_cast<int>(kvHeads);
  d.group = static_cast<int>(q.size(1) / kvHeads);
  d.head_dim = static_cast<int>(std::min<int64_t>(q.size(2), INT32_MAX));
  d.num_seqs = q.size(0);
  d.prefix_len = prefixLen;
  d.max_blocks_per_seq = blockTables.size(1);
  d.block_table_stride = blockTables.size(0) > 1 ? blockTables.stride(0) : blockTables.size(1);
  d.block_size = blockSize;
  return d;
}

// Bytes of workspace for calls of this shape and smaller ones (a caller that keeps one workspace sizes it for its largest batch,
// longest prefix and the same aiv).
int64_t shared_prefix_attention_workspace(const at::Tensor &q, int64_t prefixLen, const at::Tensor &blockTables, int64_t blockSize,
                                          int64_t kvHeads, c10::optional<int64_t> aiv) {
  const char *op = "shared_prefix_attention_workspace";
  const hfk_prefix_attention_desc d = attention_desc(q, prefixLen, blockTables, blockSize, kvHeads, HFK_KV_RAW, op);
  const c10::cuda::OptionalCUDAGuard guard(q.is_cuda() ? c10::optional<c10::Device>(q.device()) : c10::nullopt);
  const size_t bytes = hfk_prefix_attention_workspace(&d, cores_from(aiv));
  TORCH_CHECK(bytes > 0, op, ": ", hfk_last_error_message());
  return static_cast<int64_t>(bytes);
}

void shared_prefix_attention(const at::Tensor &q, const at::Tensor &out, const at::Tensor &kCache, const at::Tensor &vCache,
                             const at::Tensor &prefixTable, int64_t prefixLen, const at::Tensor &blockTables, const at::Tensor &seqLens,
                             int64_t blockSize, int64_t kvHeads, int64_t kvFormat, c10::optional<double> scale,
                             const c10::optional<at::Tensor> &lse, const c10::optional<at::Tensor> &workspace, c10::optional<int64_t> aiv) {
  const char *op = "shared_prefix_attention";
  const int ctas = cores_from(aiv);
  hfk_prefix_attention_desc d = attention_desc(q, prefixLen, blockTables, blockSize, kvHeads, kvFormat, op);
  TORCH_CHECK(q.is_cuda() && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(), op,
              ": q must be a device tensor and out must have its shape and dtype");
  check_cache(kCache, vCache, q.scalar_type(), blockSize, kvHeads, q.size(2), kvFormat, op);
  TORCH_CHECK(blockTables.scalar_type() == at::kLong || blockTables.scalar_type() == at::kInt, op, ": blockTables must be int64 or int32");
  TORCH_CHECK(blockTables.size(0) == q.size(0) && (blockTables.stride(1) == 1 || blockTables.size(1) <= 1), op,
              ": blockTables must be [num_seqs, max_blocks] with unit inner stride");
  TORCH_CHECK(seqLens.dim() == 1 && seqLens.is_contiguous() && seqLens.size(0) == q.size(0) && prefixTable.dim() == 1 &&
                  prefixTable.is_contiguous() && seqLens.scalar_type() == blockTables.scalar_type() &&
                  prefixTable.scalar_type() == blockTables.scalar_type(),
              op, ": seqLens must be [num_seqs] and prefixTable 1-D, contiguous, of the same dtype as blockTables");
  TORCH_CHECK(prefixLen >= 0 && blockSize > 0, op, ": prefixLen must not be negative, blockSize must be positive");
  TORCH_CHECK(prefixLen == 0 || prefixTable.numel() > (prefixLen - 1) / blockSize, op, ": prefixTable has ", prefixTable.numel(),
              " pages, a prefix of ", prefixLen, " tokens needs ", prefixLen == 0 ? 0 : (prefixLen - 1) / blockSize + 1);
  const auto dev = q.device();
  TORCH_CHECK(out.device() == dev && kCache.device() == dev && prefixTable.device() == dev && blockTables.device() == dev && seqLens.device() == dev,
              op, ": all tensors must be on one device");
  d.q = rows_of(q, op, "q");
  d.out = rows_of(out, op, "out");
  if (lse.has_value() && lse->defined()) {
    TORCH_CHECK(lse->device() == dev && lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->dim() == 2 &&
                    lse->size(0) == q.size(0) && lse->size(1) == q.size(1),
                op, ": lse must be a contiguous float32 tensor [num_seqs, qHeads]");
    d.lse = lse->data_ptr<float>();
  }
  d.k_cache = kCache.data_ptr();
  d.v_cache = vCache.data_ptr();
  d.prefix_table = prefixTable.data_ptr();
  d.block_tables = blockTables.data_ptr();
  d.seq_lens = seqLens.data_ptr();
  d.ids_are_int64 = blockTables.scalar_type() == at::kLong ? 1 : 0;
  d.device_block_stride = kCache.stride(0) * kCache.element_size();
  d.num_device_blocks = kCache.size(0);
  d.scale = static_cast<float>(scale.has_value() ? scale.value() : 1.0 / std::sqrt(static_cast<double>(q.size(2))));
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor own;  // freed at return, when the work is enqueued: torch's allocator hands it on in stream order
  if (workspace.has_value() && workspace->defined()) {
    TORCH_CHECK(workspace->device() == dev && workspace->is_contiguous(), op, ": workspace must be a contiguous device tensor");
    d.workspace = workspace->data_ptr();
    d.workspace_bytes = workspace->nbytes();
  } else {
    const size_t bytes = hfk_prefix_attention_workspace(&d, ctas);
    TORCH_CHECK(bytes > 0, op, ": ", hfk_last_error_message());
    own = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    d.workspace = own.data_ptr();
    d.workspace_bytes = bytes;
  }
  check_rc(hfk_shared_prefix_attention(&d, ctas, at::cuda::getCurrentCUDAStream().stream()), op);
}

// Reads and clears the device status word of the current device (bits HFK_DEV_*).
int64_t device_status() {
  unsigned int bits = 0;
  check_rc(hfk_device_status(&bits, at::cuda::getCurrentCUDAStream().stream()), "device_status");
  return static_cast<int64_t>(bits);
}

}  // namespace pciethrough

// The library is declared once and the schemas are added as fragments, as in the
// reference (pcieThrough/csrc/host/pcie_through_torchlib.cpp:4-5).
TORCH_LIBRARY(pcie_through, m) {}

TORCH_LIBRARY_FRAGMENT(pcie_through, m) {
  m.def("gather(Tensor gmEmbed, Tensor gmEmbedDst, Tensor gmIds, int? aiv=None) -> ()");
  m.def("multi_layer_block_transfer(Tensor deviceBlockCachePtrs, Tensor hostBlockCache, int? aiv=None) -> ()");
  m.def("fused_memcpy_multi_layer_block_transfer(Tensor deviceBlockCachePtrs, Tensor hostBlockCache, Tensor stagingBlockCache, int? aiv=None) -> ()");
  m.def("swap_out(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, int numDeviceBlocks, int? deviceBlockStride=None, int? aiv=None, int? mover=None, int? paceMBs=None) -> ()");
  m.def("swap_in(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, int numDeviceBlocks, int? deviceBlockStride=None, int? aiv=None, int? mover=None) -> ()");
  m.def("swap_out_copy_engine(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, int numDeviceBlocks, int? deviceBlockStride=None) -> ()");
  m.def("swap_in_copy_engine(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, int numDeviceBlocks, int? deviceBlockStride=None) -> ()");
  m.def("paged_gather(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor kOut, Tensor vOut, Tensor blockTables, Tensor seqLens, int blockSize, int numDeviceBlocks, int? deviceBlockStride=None, int? aiv=None, int? mover=None) -> ()");
  m.def("swap_out_staged(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, Tensor staging, int numDeviceBlocks, int? deviceBlockStride=None, int? aiv=None) -> ()");
  m.def("swap_in_staged(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, Tensor staging, int numDeviceBlocks, int? deviceBlockStride=None, int? aiv=None) -> ()");
  m.def("swap_in_relayout(Tensor layerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, int numDeviceBlocks, int? deviceBlockStride=None, int? aiv=None) -> ()");
  m.def("swap_out_relayout(Tensor layerPtrs, Tensor hostPool, Tensor deviceBlockIds, Tensor hostSlotIds, int numDeviceBlocks, int? deviceBlockStride=None, int? aiv=None) -> ()");
  m.def("migrate_blocks(Tensor srcKLayerPtrs, Tensor srcVLayerPtrs, Tensor dstKLayerPtrs, Tensor dstVLayerPtrs, Tensor srcBlockIds, Tensor dstBlockIds, int blockBytes, int numSrcBlocks, int numDstBlocks, int? srcBlockStride=None, int? dstBlockStride=None, int? aiv=None) -> ()");
  m.def("kv_write(Tensor k, Tensor v, Tensor kCache, Tensor vCache, Tensor slotIds, int blockSize, int kvFormat) -> ()");
  m.def("qk_norm_rope_write(Tensor q, Tensor k, Tensor v, Tensor qOut, Tensor kCache, Tensor vCache, Tensor slotIds, Tensor positions, Tensor cosSin, int blockSize, int kvFormat, Tensor? qWeight=None, Tensor? kWeight=None, float eps=1e-6, bool interleaved=False) -> ()");
  m.def("paged_gather_dequant(Tensor kLayerPtrs, Tensor vLayerPtrs, Tensor kOut, Tensor vOut, Tensor blockTables, Tensor seqLens, int blockSize, int numDeviceBlocks, int kvFormat, int? deviceBlockStride=None, int? aiv=None) -> ()");
  m.def("shared_prefix_attention(Tensor q, Tensor out, Tensor kCache, Tensor vCache, Tensor prefixTable, int prefixLen, Tensor blockTables, Tensor seqLens, int blockSize, int kvHeads, int kvFormat, float? scale=None, Tensor? lse=None, Tensor? workspace=None, int? aiv=None) -> ()");
  m.def("shared_prefix_attention_workspace(Tensor q, int prefixLen, Tensor blockTables, int blockSize, int kvHeads, int? aiv=None) -> int");
  m.def("device_status() -> int");
}

TORCH_LIBRARY_IMPL(pcie_through, CUDA, m) {
  m.impl("gather", TORCH_FN(pciethrough::gather));
  m.impl("multi_layer_block_transfer", TORCH_FN(pciethrough::multi_layer_block_transfer));
  m.impl("fused_memcpy_multi_layer_block_transfer", TORCH_FN(pciethrough::fused_memcpy_multi_layer_block_transfer));
  m.impl("swap_out", TORCH_FN(pciethrough::swap_out));
  m.impl("swap_in", TORCH_FN(pciethrough::swap_in));
  m.impl("paged_gather", TORCH_FN(pciethrough::paged_gather));
  m.impl("swap_out_staged", TORCH_FN(pciethrough::swap_out_staged));
  m.impl("swap_in_staged", TORCH_FN(pciethrough::swap_in_staged));
  m.impl("swap_in_relayout", TORCH_FN(pciethrough::swap_in_relayout));
  m.impl("swap_out_relayout", TORCH_FN(pciethrough::swap_out_relayout));
  m.impl("migrate_blocks", TORCH_FN(pciethrough::migrate_blocks));
  m.impl("kv_write", TORCH_FN(pciethrough::kv_write));
  m.impl("qk_norm_rope_write", TORCH_FN(pciethrough::qk_norm_rope_write));
  m.impl("paged_gather_dequant", TORCH_FN(pciethrough::paged_gather_dequant));
  m.impl("shared_prefix_attention", TORCH_FN(pciethrough::shared_prefix_attention));
}

// all-CPU argument lists dispatch here; there is no CPU implementation of any
// kernel, these two only enqueue copy-engine transfers
TORCH_LIBRARY_IMPL(pcie_through, CPU, m) {
  m.impl("swap_out_copy_engine", TORCH_FN(pciethrough::swap_out_copy_engine));
  m.impl("swap_in_copy_engine", TORCH_FN(pciethrough::swap_in_copy_engine));
}

TORCH_LIBRARY_IMPL(pcie_through, CompositeExplicitAutograd, m) {
  m.impl("device_status", TORCH_FN(pciethrough::device_status));
  m.impl("shared_prefix_attention_workspace", TORCH_FN(pciethrough::shared_prefix_attention_workspace));
}
