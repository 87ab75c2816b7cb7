// wsvd_adapter_add: low-rank adapters of many requests beside a shared projection.
//
//   out[n] = y[n] + scale[i] (x[n] A_i) B_i,   i = adapter[request of row n]
//
// Two kernels: h = x A in f32 (shrink) and out = y + scale h B (expand).
#include "dense_ops.cuh"

namespace wsvd {
namespace {

__device__ unsigned int g_status = 0;

// the adapter of row n: -1 for none, -2 for a row behind the last request
__device__ __forceinline__ int adapter_of(const WsvdAdapterAddParams& p, int n) {
  const int b = p.cu_new != nullptr ? sequence_of(p.cu_new, p.batch, n) : n;
  if (b < 0) return -2;
  const int i = p.adapter[b];
  if (i >= -1 && i < p.n_adapters) return i;
  atomicMax(&g_status, kOutsideStorage);
  return -1;
}

// h[n][r] = x[n] . A[:, r], a warp per row, lanes over the rank
template <typename T>
__global__ void __launch_bounds__(128) shrink_any_kernel(const __grid_constant__ WsvdAdapterAddParams p, float* h) {
  const int n = blockIdx.x, i = adapter_of(p, n);
  if (i < 0) return;
  const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)n * p.x_stride;
  const T* a = reinterpret_cast<const T*>(p.a) + (int64_t)i * p.a_stride_i;
  for (int r = threadIdx.x; r < p.rank; r += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < p.n_in; ++k) s = fmaf(wide(x[k]), wide(a[(int64_t)k * p.a_stride_k + r]), s);
    h[(int64_t)n * p.rank + r] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) expand_any_kernel(const __grid_constant__ WsvdAdapterAddParams p, const float* h) {
  const int n = blockIdx.x, i = adapter_of(p, n);
  if (i == -2 && !p.copy_tail) return;
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= p.n_out) return;
  float s = 0.f;
  if (i >= 0) {
    const T* b = reinterpret_cast<const T*>(p.b) + (int64_t)i * p.b_stride_i + c;
    for (int r = 0; r < p.rank; ++r) s = fmaf(h[(int64_t)n * p.rank + r], wide(b[(int64_t)r * p.b_stride_r]), s);
    if (p.scale != nullptr) s *= p.scale[i];
  }
  const float y = wide(reinterpret_cast<const T*>(p.y)[(int64_t)n * p.y_stride + c]);
  reinterpret_cast<T*>(p.out)[(int64_t)n * p.out_stride + c] = narrow<T>(y + s);
}

template <typename T>
void launch_any(const WsvdAdapterAddParams& p, float* h, cudaStream_t s) {
  shrink_any_kernel<T><<<p.rows, 128, 0, s>>>(p, h);
  expand_any_kernel<T><<<dim3(p.rows, (p.n_out + 255) / 256), 256, 0, s>>>(p, h);
}

}  // namespace

cudaError_t read_adapter_status(unsigned int* out) { return cudaMemcpyFromSymbol(out, g_status, sizeof(unsigned int)); }
cudaError_t reset_adapter_status() {
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(unsigned int));
}

}  // namespace wsvd

extern "C" {

size_t wsvd_adapter_add_workspace_bytes(const WsvdAdapterAddParams* p) {
  if (!p || p->rows <= 0 || p->rank <= 0) return 0;
  return (size_t)p->rows * p->rank * sizeof(float);
}

int wsvd_adapter_add(const WsvdAdapterAddParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (!p) return WSVD_ERR_NULL_POINTER;
  if (p->rows < 0 || p->batch < 0 || p->n_in <= 0 || p->n_out <= 0 || p->n_adapters < 0) return WSVD_ERR_BAD_SHAPE;
  if (p->rank <= 0 || p->rank > 256) return WSVD_ERR_BAD_SHAPE;
  if (p->dtype != WSVD_F16 && p->dtype != WSVD_BF16) return WSVD_ERR_BAD_DTYPE;
  if (!p->cu_new && p->rows != p->batch) return WSVD_ERR_BAD_SHAPE;
  if ((p->n_out + 255) / 256 > 65535) return WSVD_ERR_TOO_LARGE;
  if (p->rows == 0) return WSVD_OK;
  if (!p->y || !p->x || !p->out || !p->adapter) return WSVD_ERR_NULL_POINTER;
  if (p->n_adapters > 0 && (!p->a || !p->b)) return WSVD_ERR_NULL_POINTER;
  if (!workspace) return WSVD_ERR_NULL_POINTER;
  if (workspace_bytes < wsvd_adapter_add_workspace_bytes(p)) return WSVD_ERR_WORKSPACE_TOO_SMALL;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WSVD_ERR_BAD_STRIDE;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == WSVD_F16) wsvd::launch_any<__half>(*p, reinterpret_cast<float*>(workspace), s);
  else wsvd::launch_any<__nv_bfloat16>(*p, reinterpret_cast<float*>(workspace), s);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WSVD_OK : wsvd::record_cuda_error(e);
}

}  // extern "C"
