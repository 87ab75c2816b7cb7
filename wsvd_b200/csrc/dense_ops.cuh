// Shared pieces of the dense attention block's operators (kv_rope_append.cu, paged_decode.cu, adapter_add.cu): 16-bit
// types and products of them, the status word, which sequence a packed row belongs to.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

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

// Two 16-bit values in a word, and back (each rounded once).
template <typename T>
__device__ __forceinline__ float2 two(uint32_t v);
template <>
__device__ __forceinline__ float2 two<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 two<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t both(float x, float y);
template <>
__device__ __forceinline__ uint32_t both<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t both<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// Asynchronous copies to shared memory, fragments from there, and the product of two: m16n8k16, sums in f32.
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {  // zeros where it is not on
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
