// moe_paged.h -- host-side declarations shared by the paged-cache sources (moe_pages.cu, moe_paged_attn.cu): argument
// checks, the workspace layout and the launch helper.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/moe_paged.h"
#include "moe_common.cuh"

namespace moe {

constexpr int kPagedMaxBatch = 4096;   // list entries of one call
constexpr int kPagedMaxNew = 8;        // new tokens a sequence that the attention takes
constexpr int kPagedMaxPages = 1 << 20;
constexpr int kPagedMaxCtas = 320;     // CTAs of the attention grid at most
// ... for heads of D values: one an SM for 256, two otherwise. The partials are sized by it.
__host__ __device__ constexpr int paged_max_ctas(int D) { return D == 256 ? kPagedMaxCtas / 2 : kPagedMaxCtas; }

__host__ __device__ inline int kv_size(int kv_type) { return kv_type == MOE_KV_E4M3 ? 1 : 2; }

// Query rows of one kv head that a CTA of the attention works on: G Tq rounded up to 16, 32 or 64.
inline int paged_block_rows(int G, int Tq) {
  const int m = G * Tq;
  return m <= 16 ? 16 : (m <= 32 ? 32 : 64);
}

// Units of work that a job of the attention counts beside its units of unit_keys keys (moe_paged_attn.cu).
constexpr int setup_units(int unit_keys) { return unit_keys >= 64 ? 5 : 9; }

// The attention counts its flattened list of units in 32 bits; a unit is at least 16 keys.
inline bool paged_work_fits(const moe_paged_cache* c, int Hq, int B, int Tq) {
  const int G = Hq / c->Hkv, rows = paged_block_rows(G, Tq), blocks = (G * Tq + rows - 1) / rows;
  const int64_t units = ((int64_t)c->max_pages * c->page + 15) / 16 + setup_units(16);
  return B * units * c->Hkv * blocks < ((int64_t)1 << 31) - kPagedMaxCtas;
}

// Offsets (bytes) of the caller-owned workspace's sections, each 256-byte aligned. The error word leads; what the page
// calls and the attention keep shares the space behind it, since one workspace serves one call at a time.
struct PagedWs {
  size_t err;
  // page calls: number of page copies, their (source, destination, rows) triples, the free-page list and the page map
  size_t ncopy, copies, list, map;
  // attention: the split jobs at the borders of its CTAs, partial maxima and sums, partial accumulators
  size_t joins, ml, acc;
  size_t total;
};

inline PagedWs paged_ws(const moe_paged_cache* c, int Hq, int max_batch, int max_new) {
  PagedWs L;
  size_t o = 0;
  L.err = o;    o = ws_align(o + 4);
  const size_t base = o;
  L.ncopy = o;  o = ws_align(o + 4);
  L.copies = o; o = ws_align(o + 12 * (size_t)(c->num_pages > max_batch ? c->num_pages : max_batch));
  L.list = o;   o = ws_align(o + 4 * (size_t)c->num_pages);
  L.map = o;    o = ws_align(o + 4 * (size_t)c->num_pages);
  const size_t pages_end = o;
  o = base;
  const int rows = paged_block_rows(Hq / c->Hkv, max_new < kPagedMaxNew ? max_new : kPagedMaxNew);
  const size_t ctas = paged_max_ctas(c->D);
  L.joins = o;  o = ws_align(o + 32 * ctas);
  L.ml = o;     o = ws_align(o + sizeof(float) * 2 * ctas * 2 * rows);
  L.acc = o;    o = ws_align(o + sizeof(float) * ctas * 2 * rows * c->D);
  L.total = o > pages_end ? o : pages_end;
  return L;
}

inline bool paged_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Geometry, then pointers (moe_paged_check).
inline bool paged_shape_ok(const moe_paged_cache* c) {
  if (!c) return false;
  if (c->kv_type != MOE_KV_BF16 && c->kv_type != MOE_KV_E4M3) return false;
  if (c->D != 256 && c->D != 128 && !(c->D == 64 && c->kv_type == MOE_KV_BF16)) return false;
  if (c->page < 16 || c->page > 1024 || c->page % 16 != 0 || c->Hkv < 1 || c->Hkv > 64 || c->layers < 1) return false;
  if (c->num_pages < 1 || c->num_pages > kPagedMaxPages || c->max_seqs < 1 || c->max_seqs > 65536) return false;
  if (c->max_pages < 1 || (int64_t)c->max_pages * c->page >= ((int64_t)1 << 30)) return false;
  return true;
}
inline bool paged_ok(const moe_paged_cache* c) {
  return paged_shape_ok(c) && c->k && c->v && c->tables && c->refs && c->lens && paged_al16(c->k) && paged_al16(c->v);
}

// Bytes between a cache's layers.
inline int64_t paged_layer_bytes(const moe_paged_cache* c) {
  return (int64_t)c->num_pages * c->Hkv * c->page * c->D * kv_size(c->kv_type);
}

// Launch as a programmatic dependent of the stream's previous kernel: every kernel launched here waits for it
// (griddepcontrol.wait, in every thread) before it touches memory.
inline cudaError_t paged_launch(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t s, void** args,
                                int cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return launched(cudaLaunchKernelExC(&cfg, fn, args));
}

// SMs of the current device, asked once per device (148 where there is none: the host-side checks run without a GPU).
inline int paged_sms() {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < kDevices && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  if (dev >= 0 && dev < kDevices) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace moe
