// wsvd_paged_decode: attention of one new token per sequence over a paged cache.
//
//   out = sum_s w_s v_s / sum_s w_s,  w_s = exp(c q . k_s - max),  max(0, len - window) <= s < len
//   lse = max + log(sum_s w_s);  no positions: out = 0, lse = -inf
#include "dense_ops.cuh"

namespace wsvd {
namespace {

__device__ unsigned int g_status = 0;

// The positions [first, end) of sequence b, and its row of the page table (null: the request does not exist).
struct Span {
  int first, end;
  const int32_t* page;
};
__device__ __forceinline__ Span span_of(const WsvdPagedDecodeParams& p, int b) {
  int n = p.b_seq_len[b];
  const int req = p.b_req_idx[b];
  if (n > p.max_len) {
    atomicMax(&g_status, kOutsideTable);
    n = p.max_len;
  }
  if (n <= 0) return {0, 0, nullptr};
  if (req < 0 || req >= p.n_req) {
    atomicMax(&g_status, kOutsideStorage);
    return {0, 0, nullptr};
  }
  return {p.window > 0 ? max(0, n - p.window) : 0, n, p.req_to_token + (int64_t)req * p.rtt_stride};
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Any head_dim up to 256, strides and alignment: one block per (sequence, query head), a token per warp and step, the
// dims over the lanes.
constexpr int kAnyWarps = 8;
template <typename T, typename C>
__global__ void __launch_bounds__(kAnyWarps * 32) paged_decode_any_kernel(const __grid_constant__ WsvdPagedDecodeParams p) {
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.head_dim;
  const int hk = h / (p.n_q_heads / p.n_kv_heads);
  const Span span = span_of(p, b);
  const float c = (p.sm_scale != 0.f ? p.sm_scale : rsqrtf((float)D)) * kLog2e;
  const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_stride_b + (int64_t)h * p.q_stride_h;
  float qf[8], acc[8], m = -FLT_MAX, l = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    qf[j] = lane + 32 * j < D ? wide(q[lane + 32 * j]) : 0.f;
    acc[j] = 0.f;
  }
  constexpr bool i8 = sizeof(C) == 1;
  for (int s = span.first + warp; s < span.end; s += kAnyWarps) {
    const int64_t slot = span.page[s];
    if (slot < 0 || slot >= p.n_token_slots) {
      if (lane == 0) atomicMax(&g_status, kOutsideStorage);
      continue;
    }
    const C* k = reinterpret_cast<const C*>(p.k) + slot * p.k_stride_t + (int64_t)hk * p.k_stride_h;
    const C* v = reinterpret_cast<const C*>(p.v) + slot * p.v_stride_t + (int64_t)hk * p.v_stride_h;
    float z = 0.f, vf[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      vf[j] = 0.f;
      if (d >= D) continue;
      if constexpr (i8) {
        z = fmaf(qf[j], (float)k[d], z);
        vf[j] = (float)v[d];
      } else {
        z = fmaf(qf[j], wide(k[d]), z);
        vf[j] = wide(v[d]);
      }
    }
    z = warp_sum(z) * c;
    float sv = 1.f;
    if constexpr (i8) {
      z *= __half2float(reinterpret_cast<const __half*>(p.k_scale)[slot * p.ks_stride_t + (int64_t)hk * p.ks_stride_h]);
      sv = __half2float(reinterpret_cast<const __half*>(p.v_scale)[slot * p.vs_stride_t + (int64_t)hk * p.vs_stride_h]);
    }
    const float m_new = fmaxf(m, z), keep = exp2f(m - m_new), w = exp2f(z - m_new);
    l = l * keep + w;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(w * sv, vf[j], acc[j] * keep);
    m = m_new;
  }
  __shared__ float sm_m[kAnyWarps], sm_l[kAnyWarps], sm_o[kAnyWarps][256];
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sm_o[warp][lane + 32 * j] = acc[j];
  __syncthreads();
  float top = -FLT_MAX, sum = 0.f;
  for (int w = 0; w < kAnyWarps; ++w) top = fmaxf(top, sm_m[w]);
  for (int w = 0; w < kAnyWarps; ++w) sum += sm_l[w] * exp2f(sm_m[w] - top);
  T* out = reinterpret_cast<T*>(p.out) + (int64_t)b * p.out_stride_b + (int64_t)h * p.out_stride_h;
  for (int d = threadIdx.x; d < D; d += kAnyWarps * 32) {
    float o = 0.f;
    for (int w = 0; w < kAnyWarps; ++w) o = fmaf(sm_o[w][d], exp2f(sm_m[w] - top), o);
    out[d] = narrow<T>(sum == 0.f ? 0.f : o / sum);
  }
  if (p.lse != nullptr && threadIdx.x == 0)
    p.lse[(int64_t)b * p.n_q_heads + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

template <typename T, typename C>
void launch_any(const WsvdPagedDecodeParams& p, cudaStream_t s) {
  paged_decode_any_kernel<T, C><<<dim3(p.n_q_heads, p.batch), kAnyWarps * 32, 0, s>>>(p);
}

}  // namespace

cudaError_t read_paged_decode_status(unsigned int* out) { return cudaMemcpyFromSymbol(out, g_status, sizeof(unsigned int)); }
cudaError_t reset_paged_decode_status() {
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(unsigned int));
}

}  // namespace wsvd

extern "C" {

size_t wsvd_paged_decode_workspace_bytes(const WsvdPagedDecodeParams* p) {
  (void)p;
  return 0;
}

int wsvd_paged_decode(const WsvdPagedDecodeParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (!p) return WSVD_ERR_NULL_POINTER;
  if (p->batch < 0 || p->n_q_heads <= 0 || p->n_kv_heads <= 0 || p->n_q_heads % p->n_kv_heads != 0 || p->max_len < 0 ||
      p->n_req < 0 || p->n_token_slots < 0 || p->window < 0)
    return WSVD_ERR_BAD_SHAPE;
  if (p->head_dim <= 0 || p->head_dim > 256) return WSVD_ERR_BAD_SHAPE;
  if (p->dtype != WSVD_F16 && p->dtype != WSVD_BF16) return WSVD_ERR_BAD_DTYPE;
  const bool i8 = p->cache_dtype == WSVD_I8;
  if (!i8 && p->cache_dtype != p->dtype) return WSVD_ERR_BAD_DTYPE;
  if (p->batch > 65535 || p->n_q_heads > 65535) return WSVD_ERR_TOO_LARGE;
  if (p->batch == 0) return WSVD_OK;
  if (!p->q || !p->k || !p->v || !p->out || !p->req_to_token || !p->b_req_idx || !p->b_seq_len) return WSVD_ERR_NULL_POINTER;
  if (i8 && (!p->k_scale || !p->v_scale)) return WSVD_ERR_BAD_DTYPE;
  const size_t need = wsvd_paged_decode_workspace_bytes(p);
  if (need > 0 && !workspace) return WSVD_ERR_NULL_POINTER;
  if (workspace_bytes < need) return WSVD_ERR_WORKSPACE_TOO_SMALL;
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WSVD_ERR_BAD_STRIDE;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == WSVD_F16) {
    i8 ? wsvd::launch_any<__half, int8_t>(*p, s) : wsvd::launch_any<__half, __half>(*p, s);
  } else {
    i8 ? wsvd::launch_any<__nv_bfloat16, int8_t>(*p, s) : wsvd::launch_any<__nv_bfloat16, __nv_bfloat16>(*p, s);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WSVD_OK : wsvd::record_cuda_error(e);
}

}  // extern "C"
