// Shared pieces of the dense attention block's operators (kv_rope_append.cu, paged_decode.cu, adapter_add.cu): 16-bit
// types, the status word, which sequence a packed row belongs to.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace wsvd {

// Positions and rows are counted in steps of up to 2048 as 32-bit numbers: what is beyond this would pass 2^31 in the last step.
constexpr int32_t kMostCounted = INT32_MAX - 4096;

// Recorded by the three operators, each in its translation unit's own word; wsvd_kernel_status reads them all.
constexpr unsigned int kOutsideTable = 5;    // a position beyond the page table's width
constexpr unsigned int kOutsideStorage = 7;  // a slot, request or adapter that does not exist
cudaError_t read_kv_append_status(unsigned int* out);
cudaError_t reset_kv_append_status();
cudaError_t read_paged_decode_status(unsigned int* out);
cudaError_t reset_paged_decode_status();
cudaError_t read_adapter_status(unsigned int* out);
cudaError_t reset_adapter_status();

__device__ __forceinline__ float wide(__half v) { return __half2float(v); }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// The sequence that packed row n belongs to: the last b with cu[b] <= n, or -1 for rows behind the last sequence
// (n >= cu[batch]) and in front of the first.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int batch, int n) {
  if (n < cu[0] || n >= cu[batch]) return -1;
  int lo = 0, hi = batch;  // cu[lo] <= n < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= n) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Kernels that are launched by launch_overlapped: everything in front of this one in the stream has finished ...
__device__ __forceinline__ void before_this() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
// ... and the blocks of the next one may be set up (once all blocks of this one have said so or ended).
__device__ __forceinline__ void let_next_in() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

// Launch of a kernel whose blocks may be set up while the kernel in front of it in the stream still ends: it calls
// before_this() before it reads or writes what another kernel may have to do with.
// `cluster`: CTAs of a cluster along y.
constexpr int kMaxDevices = 64;
template <typename K, typename... Args>
cudaError_t launch_overlapped(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, int cluster, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {1, (unsigned)cluster, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace wsvd
