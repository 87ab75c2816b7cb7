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
//
// Memory bound: 14856 rows of prompts, 40 heads of 128, f16: 139 us, 6.57 TB/s read and written (a plain copy has that rate); into
// bytes, 5665 rows of 8 KV heads and 32 queries: 34.5 us, 3.7 TB/s (two block barriers around the angles, and instructions: ncu has the
// barrier and not-selected stalls in front, DRAM at a third).  A step of up to 64 rows: 3 to 4 us, the chain length -> page -> row.
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

// A value in steps of the scale, rounded to even: the low byte of the answer.
__device__ __forceinline__ uint32_t byte_of(float x, float scale) { return (uint32_t)(int)fminf(fmaxf(rintf(x / scale), -128.f), 127.f); }

// The same from x times 1 / scale (a division a value took 43 us for 5665 rows, the product without a look at the middle 32, with it
// 34.5), for scales that are f16's own max|x| / 127, neither among its subnormals nor at its end, so that the product is between
// -128 and 128; `open` where it may not be the quotient's.  The low byte again: adding 1.5 2^23 rounds to a whole
// number, to even, and leaves it in the last bits.
// Up to 2^-15 before the middle of two steps the product rounds as the quotient does: 1 / scale and the product are each off by 2^-24,
// together by 2^-16 at 128 steps.  (The quotient itself comes to lie on the middle only if x does: the middle times an f16 scale is an
// f32 value.)  NaN is on no side.
__device__ __forceinline__ bool whole_scale(float scale) { return scale >= 6.103515625e-5f && scale < 65504.f; }
__device__ __forceinline__ uint32_t byte_by_product(float x, float to_step, bool* open) {
  const float t = x * to_step, n = t + 12582912.f;
  *open |= !(fabsf(t - (n - 12582912.f)) <= 0.5f - 1.f / 32768);
  return __float_as_uint(n);
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
  const float step = __half2float(scale);
  int8_t* dst = is_v ? reinterpret_cast<int8_t*>(p.cache_v) + at.slot * p.cv_stride_t + (int64_t)h * p.cv_stride_h
                     : reinterpret_cast<int8_t*>(p.cache_k) + at.slot * p.ck_stride_t + (int64_t)h * p.ck_stride_h;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (i0[j] < 0) continue;
    dst[i0[j]] = (int8_t)byte_of(a[j], step);
    dst[i0[j] + (lane + 32 * j < half ? apart : 1)] = (int8_t)byte_of(b[j], step);
  }
  if (lane == 0) {
    if (is_v) reinterpret_cast<__half*>(p.v_scale)[at.slot * p.vs_stride_t + (int64_t)h * p.vs_stride_h] = scale;
    else reinterpret_cast<__half*>(p.k_scale)[at.slot * p.ks_stride_t + (int64_t)h * p.ks_stride_h] = scale;
  }
}

// ---- the same for head_dim and rot_dim in whole 16s and rows of whole 16-byte vectors
//
// Bound by memory: every value is read and written once.  A thread's unit is two 8-value vectors of a row that turn into one
// another (half: dims 8 j .. and rot / 2 + 8 j ..; interleaved and what is not rotated: 16 dims in a row), so that nothing but
// the angles passes through shared memory; unit j of any head turns by the angles 8 j .. 8 j + 7 of its row.  A block takes a
// run of units of consecutive rows; the angles of those rows (f64 reduction, sine and cosine: ~100 instructions) are
// computed once for all heads.  What a row's place is (up to four dependent loads) and the angles are worked out while the
// block's vectors are on their way.
constexpr int kVecThreads = 256;
// From here on four units a thread (a block's set-up is paid for more data), below it one (more SMs at work).  (14856 rows of 40 heads:
// 139 us with four, 178 with one; the kernel alone for 64 rows of 32 + 2 x 8 heads 4.7 and 3.2, for one row 4.1 and 3.1.)
constexpr int64_t kManyUnits = 148 * 4 * kVecThreads * 4;

struct Divisor {  // n / d for n < 2^31
  uint32_t d, m, s;
  __host__ static Divisor of(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

template <typename T>
__device__ __forceinline__ void open8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = two<T>(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 close8(const float (&f)[8]) {
  return make_uint4(both<T>(f[0], f[1]), both<T>(f[2], f[3]), both<T>(f[4], f[5]), both<T>(f[6], f[7]));
}
template <typename F>
__device__ __forceinline__ uint2 bytes8(const float (&f)[8], F byte) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t low = __byte_perm(byte(f[4 * i]), byte(f[4 * i + 1]), 0x0040);
    const uint32_t high = __byte_perm(byte(f[4 * i + 2]), byte(f[4 * i + 3]), 0x0040);
    w[i] = __byte_perm(low, high, 0x5410);
  }
  return make_uint2(w[0], w[1]);
}

// lanes: log2 of the lanes of a head (D / 16 rounded up to a power of two); per_row: units of a row; U: units of a thread
// (bytes, four units: three blocks an SM, so that bf16 ones have the registers for it; with the four of 64 registers they spill: 35.2 us,
// 34.5 so; 0: as the compiler chooses)
template <typename T, bool I8, int U>
__global__ void __launch_bounds__(kVecThreads, I8 && U == 4 ? 3 : 0)
kv_append_vec_kernel(const __grid_constant__ WsvdKvRopeAppendParams p, const int lanes, const Divisor per_row, const int most_rows) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int half = p.rot_dim / 2, groups = p.rot_dim / 16;  // angles of a row, units that turn
  int64_t* row_slot = reinterpret_cast<int64_t*>(smem);     // -1: not stored, -2: padding
  int64_t* row_place = row_slot + most_rows;
  float2* turn = reinterpret_cast<float2*>(row_place + most_rows);  // [row][8][groups]: neighbouring units, neighbouring words
  before_this();
  const uint32_t total = (uint32_t)p.rows * per_row.d, first = blockIdx.x * (uint32_t)(kVecThreads * U);
  const int row0 = per_row.div(first);
  const int rows = (int)per_row.div(min(total, first + kVecThreads * U) - 1) - row0 + 1;
  const int units = p.head_dim / 16;
  const bool half_layout = p.rope_layout == WSVD_ROPE_HALF;

  // where a unit's two vectors start in its row
  auto second = [&](int j, bool turns) { return turns && half_layout ? half + 8 * j : 16 * j + 8; };
  auto start = [&](int j, bool turns) { return turns && half_layout ? 8 * j : 16 * j; };

  uint4 va[U], vb[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t idx = first + u * kVecThreads + threadIdx.x;
    if (idx >= total) continue;
    const int row = per_row.div(idx), in = idx - row * per_row.d, head = in >> lanes, j = in & ((1 << lanes) - 1);
    if (j >= units) continue;
    const int hk = head - p.n_q_heads, hv = hk - p.n_kv_heads;
    const T* src = hk < 0   ? reinterpret_cast<const T*>(p.q) + (int64_t)row * p.q_stride_n + (int64_t)head * p.q_stride_h
                   : hv < 0 ? reinterpret_cast<const T*>(p.k) + (int64_t)row * p.k_stride_n + (int64_t)hk * p.k_stride_h
                            : reinterpret_cast<const T*>(p.v) + (int64_t)row * p.v_stride_n + (int64_t)hv * p.v_stride_h;
    const bool turns = hv < 0 && j < groups;
    va[u] = *reinterpret_cast<const uint4*>(src + start(j, turns));
    vb[u] = *reinterpret_cast<const uint4*>(src + second(j, turns));
  }
  for (int r = threadIdx.x; r < rows; r += kVecThreads) {
    const RowPlace at = place_of(p, row0 + r);
    row_slot[r] = at.row ? at.slot : -2;
    row_place[r] = at.place;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * half; i += kVecThreads) {
    const int r = i / half, a = i - r * half;
    float sn, cs;
    rotation(row_place[r], p.inv_freq[a], &sn, &cs);
    turn[r * half + (a & 7) * groups + (a >> 3)] = make_float2(cs, sn);
  }
  __syncthreads();

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t idx = first + u * kVecThreads + threadIdx.x;
    const bool in_range = idx < total;
    const int row = in_range ? per_row.div(idx) : row0, in = in_range ? idx - row * per_row.d : 0;
    const int head = in >> lanes, j = in & ((1 << lanes) - 1);
    const bool active = in_range && j < units;
    const int hk = head - p.n_q_heads, hv = hk - p.n_kv_heads;
    const bool turns = active && hv < 0 && j < groups;
    const int64_t slot = row_slot[row - row0];
    float a[8], b[8];
    if (active) {
      open8<T>(va[u], a);
      open8<T>(vb[u], b);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.f;
    }
    if (turns) {
      const float2* t = turn + (row - row0) * half + j;
      if (half_layout) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 w = t[e * groups];
          const float x = a[e], y = b[e];
          a[e] = x * w.x - y * w.y;
          b[e] = y * w.x + x * w.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 w = t[e * groups];
          float* v = e < 4 ? a + 2 * e : b + 2 * (e - 4);
          const float x = v[0], y = v[1];
          v[0] = x * w.x - y * w.y;
          v[1] = y * w.x + x * w.y;
        }
      }
    }
    const int d0 = start(j, turns), d1 = second(j, turns);
    if (hk < 0) {
      if (active && (slot != -2 || p.clear_tail)) {
        T* dst = reinterpret_cast<T*>(p.q_out) + (int64_t)row * p.qo_stride_n + (int64_t)head * p.qo_stride_h;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + d0) = slot == -2 ? zero : close8<T>(a);
        *reinterpret_cast<uint4*>(dst + d1) = slot == -2 ? zero : close8<T>(b);
      }
    } else if (!I8 && active && slot >= 0) {
      T* dst = hv < 0 ? reinterpret_cast<T*>(p.cache_k) + slot * p.ck_stride_t + (int64_t)hk * p.ck_stride_h
                      : reinterpret_cast<T*>(p.cache_v) + slot * p.cv_stride_t + (int64_t)hv * p.cv_stride_h;
      *reinterpret_cast<uint4*>(dst + d0) = close8<T>(a);
      *reinterpret_cast<uint4*>(dst + d1) = close8<T>(b);
    }
    // the lanes of a head are neighbours in a warp (all lanes take part, also those without a unit); a warp of queries has none
    if (I8 && __any_sync(0xffffffffu, hk >= 0 && active)) {
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(fabsf(a[e]), fabsf(b[e])));
      for (int o = 1; o < (1 << lanes); o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (hk >= 0 && active && slot >= 0) {
        const __half scale = __float2half_rn(amax == 0.f ? 1.f : fminf(fmaxf(amax / 127.f, 5.9604644775390625e-8f), 65504.f));
        const float step = __half2float(scale), to_step = 1.f / step;
        bool open = !whole_scale(step);
        auto by_product = [&](float x) { return byte_by_product(x, to_step, &open); };
        uint2 low = bytes8(a, by_product), high = bytes8(b, by_product);
        if (open) {  // (16 values: one in a thousand)
          auto by_quotient = [&](float x) { return byte_of(x, step); };
          low = bytes8(a, by_quotient);
          high = bytes8(b, by_quotient);
        }
        int8_t* dst = hv < 0 ? reinterpret_cast<int8_t*>(p.cache_k) + slot * p.ck_stride_t + (int64_t)hk * p.ck_stride_h
                             : reinterpret_cast<int8_t*>(p.cache_v) + slot * p.cv_stride_t + (int64_t)hv * p.cv_stride_h;
        *reinterpret_cast<uint2*>(dst + d0) = low;
        *reinterpret_cast<uint2*>(dst + d1) = high;
        if (j == 0) {
          if (hv < 0) reinterpret_cast<__half*>(p.k_scale)[slot * p.ks_stride_t + (int64_t)hk * p.ks_stride_h] = scale;
          else reinterpret_cast<__half*>(p.v_scale)[slot * p.vs_stride_t + (int64_t)hv * p.vs_stride_h] = scale;
        }
      }
    }
  }
}

bool whole_vectors(const WsvdKvRopeAppendParams& p) {
  const bool i8 = p.cache_dtype == WSVD_I8;
  if (p.head_dim % 16 || p.rot_dim % 16) return false;
  const uintptr_t in = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                       (p.n_q_heads > 0 ? reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.q_out) : 0);
  const uintptr_t held = reinterpret_cast<uintptr_t>(p.cache_k) | reinterpret_cast<uintptr_t>(p.cache_v);
  int64_t strides = p.k_stride_n | p.k_stride_h | p.v_stride_n | p.v_stride_h | p.ck_stride_t | p.ck_stride_h | p.cv_stride_t |
                    p.cv_stride_h;
  if (p.n_q_heads > 0) strides |= p.q_stride_n | p.q_stride_h | p.qo_stride_n | p.qo_stride_h;
  return (in & 15) == 0 && (held & (i8 ? 7 : 15)) == 0 && strides % 8 == 0;
}

template <typename T, bool I8, int U>
cudaError_t launch_vec(const WsvdKvRopeAppendParams& p, int lanes, int per_row, cudaStream_t s) {
  const int64_t total = (int64_t)p.rows * per_row;
  const int most_rows = (kVecThreads * U - 1) / per_row + 2;
  const size_t smem = (size_t)most_rows * (2 * sizeof(int64_t) + p.rot_dim / 2 * sizeof(float2));
  return launch_overlapped(kv_append_vec_kernel<T, I8, U>, dim3((unsigned)((total + kVecThreads * U - 1) / (kVecThreads * U))),
                           kVecThreads, smem, s, 1, p, lanes, Divisor::of(per_row), most_rows);
}

template <typename T, bool I8>
cudaError_t launch_append(const WsvdKvRopeAppendParams& p, cudaStream_t s) {
  int lanes = 0;
  while (16 << lanes < p.head_dim) ++lanes;
  const int64_t heads = p.n_q_heads + 2 * (int64_t)p.n_kv_heads, per_row = heads << lanes, total = p.rows * per_row;
  if (whole_vectors(p) && total < (1ll << 31) - 4096) {
    return total >= kManyUnits ? launch_vec<T, I8, 4>(p, lanes, (int)per_row, s) : launch_vec<T, I8, 1>(p, lanes, (int)per_row, s);
  }
  const int64_t items = (int64_t)p.rows * (p.n_q_heads + 2 * p.n_kv_heads);
  kv_append_any_kernel<T, I8><<<(unsigned)((items + 3) / 4), 128, 0, s>>>(p);
  return cudaGetLastError();
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
  if (!p->k || !p->v || (p->batch > 0 && (!p->b_req_idx || !p->b_seq_len))) return WSVD_ERR_NULL_POINTER;
  const bool places = p->n_token_slots > 0 && p->n_req > 0 && p->max_len > 0;  // (else no row is stored)
  if (places && (!p->cache_k || !p->cache_v || !p->req_to_token)) return WSVD_ERR_NULL_POINTER;
  if (p->rot_dim > 0 && !p->inv_freq) return WSVD_ERR_NULL_POINTER;
  if (p->n_q_heads > 0 && (!p->q || !p->q_out)) return WSVD_ERR_NULL_POINTER;
  if (i8 && places && (!p->k_scale || !p->v_scale)) return WSVD_ERR_BAD_DTYPE;
  if ((int64_t)p->rows * ((int64_t)p->n_q_heads + 2 * (int64_t)p->n_kv_heads) > (int64_t)1 << 32) return WSVD_ERR_TOO_LARGE;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  WsvdKvRopeAppendParams call = *p;
  if (!places) call.max_len = 0;
  const cudaError_t e = p->dtype == WSVD_F16 ? (i8 ? wsvd::launch_append<__half, true>(call, s) : wsvd::launch_append<__half, false>(call, s))
                        : i8                 ? wsvd::launch_append<__nv_bfloat16, true>(call, s)
                                             : wsvd::launch_append<__nv_bfloat16, false>(call, s);
  return e == cudaSuccess ? WSVD_OK : wsvd::record_cuda_error(e);
}
