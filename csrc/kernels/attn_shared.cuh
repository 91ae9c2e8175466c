// What the kernels of the shared-prefix attention have in common: their arguments and the table of groups.
#pragma once
#include "../include/launch.h"
#include "../include/sharing.h"
#include "../include/sm100.cuh"
#include "../include/tma_host.h"

namespace mesh {
namespace shared_attn {

constexpr int SLICE = 16;                   // keys per slice: one TMA box row block, pages hold a whole number of them
constexpr int MAX_ROWS = SHARED_MAX_ROWS;   // query rows of a sequence
constexpr int HDR = SHARED_HDR, ITEM = SHARED_ITEM;
constexpr uint64_t WAIT_NS = 2000000000ull;

struct Args : SharedAttnArgs {
  int slices_per_page;
  float scale_log2;
};

__device__ __forceinline__ int seq_prefix(const Args& a, int b) { return a.meta[HDR + b]; }
__device__ __forceinline__ int seq_base(const Args& a, int b) { return a.meta[HDR + a.B + b]; }
__device__ __forceinline__ int seq_prefix_slots(const Args& a, int b) { return a.meta[HDR + 2 * a.B + b]; }
__device__ __forceinline__ const int* members(const Args& a) { return a.meta + HDR + 3 * a.B; }
// slices of the keys behind the prefixes: those before each sequence [B + 1], then a CTA's quota; written by own_kernel
__device__ __forceinline__ int* own_before(const Args& a) { return a.meta + HDR + 4 * a.B; }
__device__ __forceinline__ const int* items(const Args& a) { return a.meta + shared_items_at(a.B); }

// Once per device: the kernel's dynamic shared memory, and that the SM keeps all its shared memory, also what the kernel
// itself does not use, so that a CTA of the other kernel can start beside it.
constexpr int MAX_DEVICES = 64;
template <typename Kern>
inline cudaError_t prepare_kernel(Kern kern, int smem, bool (&done)[MAX_DEVICES]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < MAX_DEVICES && done[dev])) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && dev < MAX_DEVICES) done[dev] = true;
  return e;
}

// rows of a prefix item against its shared keys on tcgen05 (attn_shared_tc.cu)
template <int D>
cudaError_t launch_prefix(const Args& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st);

}  // namespace shared_attn
}  // namespace mesh
