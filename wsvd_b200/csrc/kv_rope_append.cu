// wsvd_kv_rope_append: new rows of keys and values into the token slots of a paged cache, the keys (and the queries beside
// them) rotated to their positions on the way.
//
//   row n of sequence b, pos = b_seq_len[b] + i, angle_j = (pos + pos_offset[b]) inv_freq[j]
//   (x_j, x_j') -> (x_j cos - x_j' sin, x_j' cos + x_j sin) for the pairs of the first rot_dim dims
//   int8 caches: scale = f16(max|x| / 127), round(x / scale) of the rotated f32 row
//
// The angle of a far position needs more than f32: at position 10^5 the f32 product is off by up to 0.004 radians, a bf16
// rounding step.  It is taken in f64 (the product of an int32 and an f32 is exact there but for its last two bits), reduced
// to [-pi, pi] with a two-term 2 pi, and only then handed to sincosf in f32.
#include "dense_ops.cuh"

namespace wsvd {
namespace {

__device__ unsigned int g_status = 0;

__device__ __forceinline__ void rotation(int64_t place, float freq, float* sn, float* cs) {
  const double a = (double)place * (double)freq;
  const double turns = rint(a * 0.15915494309189535);                   // 1 / (2 pi)
  double r = fma(-turns, 6.283185307179586, a);                         // 2 pi to f64 ...
  r = fma(-turns, 2.4492935982947064e-16, r);                           // ... and what is left of it
  sincosf((float)r, sn, cs);
}

// What a row is: its sequence, its position (for the rotation) and its token slot (-1: not stored).
struct RowPlace {
  int64_t slot, place;
  bool row;  // false: padding behind the last sequence
};
__device__ __forceinline__ RowPlace place_of(const WsvdKvRopeAppendParams& p, int n) {
  RowPlace r{-1, 0, false};
  int b = n, i = 0;
  if (p.cu_new != nullptr) {
    b = sequence_of(p.cu_new, p.batch, n);
    if (b < 0) return r;
    i = n - p.cu_new[b];
  }
  r.row = true;
  const int64_t pos = (int64_t)p.b_seq_len[b] + i;
  r.place = pos + (p.pos_offset != nullptr ? p.pos_offset[b] : 0);
  if (pos < 0 || pos >= p.max_len) {
    atomicMax(&g_status, kOutsideTable);
    return r;
  }
  const int req = p.b_req_idx[b];
  if (req >= 0 && req < p.n_req) {
    const int64_t slot = p.req_to_token[(int64_t)req * p.rtt_stride + pos];
    if (slot >= 0 && slot < p.n_token_slots) r.slot = slot;
  }
  if (r.slot < 0) atomicMax(&g_status, kOutsideStorage);
  return r;
}

// Any even head_dim, strides and alignment: one warp per (row, head), pairs of dims dealt out to its lanes.
template <typename T, bool I8>
__global__ void __launch_bounds__(128) kv_append_any_kernel(const __grid_constant__ WsvdKvRopeAppendParams p) {
  const int heads = p.n_q_heads + 2 * p.n_kv_heads, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (int64_t)p.rows * heads) return;
  const int n = (int)(item / heads), head = (int)(item - (int64_t)n * heads);
  const bool is_q = head < p.n_q_heads, is_v = head >= p.n_q_heads + p.n_kv_heads;
  const int h = is_q ? head : is_v ? head - p.n_q_heads - p.n_kv_heads : head - p.n_q_heads;
  const RowPlace at = place_of(p, n);
  if (!is_q && at.slot < 0) return;
  T* q_out = reinterpret_cast<T*>(p.q_out) + (int64_t)n * p.qo_stride_n + (int64_t)h * p.qo_stride_h;
  if (!at.row) {
    if (p.clear_tail)
      for (int d = lane; d < p.head_dim; d += 32) q_out[d] = narrow<T>(0.f);
    return;
  }
  const T* src = is_q   ? reinterpret_cast<const T*>(p.q) + (int64_t)n * p.q_stride_n + (int64_t)h * p.q_stride_h
                 : is_v ? reinterpret_cast<const T*>(p.v) + (int64_t)n * p.v_stride_n + (int64_t)h * p.v_stride_h
                        : reinterpret_cast<const T*>(p.k) + (int64_t)n * p.k_stride_n + (int64_t)h * p.k_stride_h;
  const int half = is_v ? 0 : p.rot_dim / 2, apart = p.rope_layout == WSVD_ROPE_HALF ? half : 1;
  float a[4], b[4];
  int i0[4];
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pair = lane + 32 * j;
    i0[j] = -1;
    if (2 * pair >= p.head_dim) continue;
    const bool turn = pair < half;
    i0[j] = turn && apart != 1 ? pair : 2 * pair;
    const int i1 = i0[j] + (turn ? apart : 1);
    float x = wide(src[i0[j]]), y = wide(src[i1]);
    if (turn) {
      float sn, cs;
      rotation(at.place, p.inv_freq[pair], &sn, &cs);
      const float z = x * cs - y * sn;
      y = y * cs + x * sn;
      x = z;
    }
    a[j] = x;
    b[j] = y;
    amax = fmaxf(amax, fmaxf(fabsf(x), fabsf(y)));
  }
  if (is_q || !I8) {
    T* dst = is_q   ? q_out
             : is_v ? reinterpret_cast<T*>(p.cache_v) + at.slot * p.cv_stride_t + (int64_t)h * p.cv_stride_h
                    : reinterpret_cast<T*>(p.cache_k) + at.slot * p.ck_stride_t + (int64_t)h * p.ck_stride_h;
    __syncwarp();  // q_out may be q: every lane has its pairs
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0[j] < 0) continue;
      dst[i0[j]] = narrow<T>(a[j]);
      dst[i0[j] + (lane + 32 * j < half ? apart : 1)] = narrow<T>(b[j]);
    }
    return;
  }
  amax = warp_max(amax);
  // (the stored scale is f16: clamped to its range, as wsvd_latent_quant_append_i8 does)
  const __half scale = __float2half_rn(amax == 0.f ? 1.f : fminf(fmaxf(amax / 127.f, 5.9604644775390625e-8f), 65504.f));
  const float s = __half2float(scale);
  int8_t* dst = is_v ? reinterpret_cast<int8_t*>(p.cache_v) + at.slot * p.cv_stride_t + (int64_t)h * p.cv_stride_h
                     : reinterpret_cast<int8_t*>(p.cache_k) + at.slot * p.ck_stride_t + (int64_t)h * p.ck_stride_h;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (i0[j] < 0) continue;
    dst[i0[j]] = (int8_t)fminf(fmaxf(rintf(a[j] / s), -128.f), 127.f);
    dst[i0[j] + (lane + 32 * j < half ? apart : 1)] = (int8_t)fminf(fmaxf(rintf(b[j] / s), -128.f), 127.f);
  }
  if (lane == 0) {
    if (is_v) reinterpret_cast<__half*>(p.v_scale)[at.slot * p.vs_stride_t + (int64_t)h * p.vs_stride_h] = scale;
    else reinterpret_cast<__half*>(p.k_scale)[at.slot * p.ks_stride_t + (int64_t)h * p.ks_stride_h] = scale;
  }
}

template <typename T, bool I8>
void launch_any(const WsvdKvRopeAppendParams& p, cudaStream_t s) {
  const int64_t items = (int64_t)p.rows * (p.n_q_heads + 2 * p.n_kv_heads);
  kv_append_any_kernel<T, I8><<<(unsigned)((items + 3) / 4), 128, 0, s>>>(p);
}

}  // namespace

cudaError_t read_kv_append_status(unsigned int* out) { return cudaMemcpyFromSymbol(out, g_status, sizeof(unsigned int)); }
cudaError_t reset_kv_append_status() {
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(unsigned int));
}

}  // namespace wsvd

extern "C" int wsvd_kv_rope_append(const WsvdKvRopeAppendParams* p, void* stream) {
  if (!p) return WSVD_ERR_NULL_POINTER;
  if (p->rows < 0 || p->batch < 0 || p->n_q_heads < 0 || p->n_kv_heads <= 0 || p->max_len < 0 || p->n_req < 0 ||
      p->n_token_slots < 0)
    return WSVD_ERR_BAD_SHAPE;
  if (p->head_dim <= 0 || p->head_dim > 256 || p->head_dim % 2 || p->rot_dim < 0 || p->rot_dim > p->head_dim || p->rot_dim % 2)
    return WSVD_ERR_BAD_SHAPE;
  if (p->dtype != WSVD_F16 && p->dtype != WSVD_BF16) return WSVD_ERR_BAD_DTYPE;
  const bool i8 = p->cache_dtype == WSVD_I8;
  if (!i8 && p->cache_dtype != p->dtype) return WSVD_ERR_BAD_DTYPE;
  if (p->rope_layout != WSVD_ROPE_HALF && p->rope_layout != WSVD_ROPE_INTERLEAVED) return WSVD_ERR_BAD_DTYPE;
  if (!p->cu_new && p->rows != p->batch) return WSVD_ERR_BAD_SHAPE;
  if (p->rows == 0) return WSVD_OK;
  if (!p->k || !p->v || !p->cache_k || !p->cache_v || !p->req_to_token || !p->b_req_idx || !p->b_seq_len)
    return WSVD_ERR_NULL_POINTER;
  if (p->rot_dim > 0 && !p->inv_freq) return WSVD_ERR_NULL_POINTER;
  if (p->n_q_heads > 0 && (!p->q || !p->q_out)) return WSVD_ERR_NULL_POINTER;
  if (i8 && (!p->k_scale || !p->v_scale)) return WSVD_ERR_BAD_DTYPE;
  if ((int64_t)p->rows * ((int64_t)p->n_q_heads + 2 * (int64_t)p->n_kv_heads) > (int64_t)1 << 32) return WSVD_ERR_TOO_LARGE;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == WSVD_F16) {
    i8 ? wsvd::launch_any<__half, true>(*p, s) : wsvd::launch_any<__half, false>(*p, s);
  } else {
    i8 ? wsvd::launch_any<__nv_bfloat16, true>(*p, s) : wsvd::launch_any<__nv_bfloat16, false>(*p, s);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WSVD_OK : wsvd::record_cuda_error(e);
}
