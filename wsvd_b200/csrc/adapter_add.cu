// wsvd_adapter_add: low-rank adapters of many requests beside a shared projection.
//
//   out[n] = y[n] + scale[i] (x[n] A_i) B_i,   i = adapter[request of row n]
//
// Two kernels: h = x A in f32 (shrink) and out = y + scale h B (expand).
#include <cooperative_groups.h>

#include <type_traits>

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
    const float scale = p.scale != nullptr ? p.scale[i] : 1.f;  // (on h: its products with B alone may pass f32's range)
    for (int r = 0; r < p.rank; ++r) s = fmaf(scale * h[(int64_t)n * p.rank + r], wide(b[(int64_t)r * p.b_stride_r]), s);
  }
  const float y = wide(reinterpret_cast<const T*>(p.y)[(int64_t)n * p.y_stride + c]);
  reinterpret_cast<T*>(p.out)[(int64_t)n * p.out_stride + c] = narrow<T>(y + s);
}

// ---- one row per request (a decode step): products on the CUDA cores, weights read once per four rows that share them
//
// Bound by the adapters' bytes, and by latency: a block asks for its weights as soon as it knows its row's adapter, while it
// finds out who shares it.  Every row of the batch has its blocks; those of a row that is the first, fifth, ... of its
// adapter in the batch do the work for it and the next three, so that an adapter comes from memory once and from L2 once
// per four rows, whatever the order of the requests.  The input's length is cut into slices over the blocks; the slices'
// sums are added in a fixed order by the expanding blocks, which have asked for their weights before (they are launched
// while the shrinking ones still run).  Measured, a call: four rows of 4096 to 4096, rank 16: 8 us (two launches and their chains of
// loads); 64 rows of 5120 to 15360, rank 32, 48 adapters: 24 us, 2.0 TB/s of weights: the slices' sums, half of the second
// kernel, wait for the slowest slice.
constexpr int kStepRows = 4, kStepThreads = 128, kStepCols = 8 * kStepThreads, kMaxSlices = 64, kMaxSlice = 2048;
constexpr int kStepLoads = 8;  // weights that a thread of the shrinking kernel asks for at once

// The rows (at most four) that the blocks of row n, with adapter `mine`, work for: rows[0] = n; count 0 where another row's
// blocks do, or there is no adapter.  The first warp looks the batch over; all threads get the answer.
struct Rows {
  int count;
  int row[kStepRows];
};
__device__ __forceinline__ void rows_of(const WsvdAdapterAddParams& p, int n, int mine, Rows* sm) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int before = 0, count = 1, r1 = n, r2 = n, r3 = n;
    for (int j0 = 0; j0 < p.batch && count < kStepRows; j0 += 128) {
      int a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + 32 * i + lane;
        a[i] = j < p.batch ? p.adapter[j] : -1;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + 32 * i;
        unsigned same = __ballot_sync(0xffffffffu, a[i] == mine);
        const unsigned up_to = n >= j + 31 ? 0xffffffffu : n < j ? 0u : (2u << (n - j)) - 1u;  // rows up to n
        before += __popc(same & up_to);
        same &= ~up_to;
        while (same != 0 && count < kStepRows) {
          const int row = j + __ffs(same) - 1;
          if (count == 1) r1 = row;
          else if (count == 2) r2 = row;
          else r3 = row;
          ++count;
          same &= same - 1;
        }
      }
    }
    if (lane == 0) {
      sm->count = mine < 0 || (before - 1) % kStepRows != 0 ? 0 : count;  // (`before` counts row n itself)
      sm->row[0] = n;
      sm->row[1] = r1;
      sm->row[2] = r2;
      sm->row[3] = r3;
    }
  }
  __syncthreads();
}

// acc[row][4 ranks] += x w over the `n` loaded inputs; x of the slice's input i of row j is xs[i R + j]
template <typename T, int R>
__device__ __forceinline__ void step_products(const uint2 (&w)[kStepLoads], const float* xs, int lanes, int n, float (&acc)[kStepRows][4]) {
#pragma unroll
  for (int l = 0; l < kStepLoads; ++l) {
    if (l >= n) break;
    const float2 lo = two<T>(w[l].x), hi = two<T>(w[l].y);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float x = xs[l * lanes * R + i];
      acc[i][0] = fmaf(x, lo.x, acc[i][0]);
      acc[i][1] = fmaf(x, lo.y, acc[i][1]);
      acc[i][2] = fmaf(x, hi.x, acc[i][2]);
      acc[i][3] = fmaf(x, hi.y, acc[i][3]);
    }
  }
}

// h[slice][row][r]: the sum over the slice's inputs.  A thread has four neighbouring ranks and every `lanes`-th input.
template <typename T>
__global__ void __launch_bounds__(kStepThreads)
shrink_step_kernel(const __grid_constant__ WsvdAdapterAddParams p, float* h, const int slice) {
  extern __shared__ __align__(16) float xs[];  // [inputs of the slice][rows], then [lanes][rows][rank]
  __shared__ Rows rows;
  before_this();
  let_next_in();
  const int n = blockIdx.x, mine = adapter_of(p, n);
  const int quads = p.rank / 4, lanes = kStepThreads / quads, kl = threadIdx.x / quads, quad = threadIdx.x - kl * quads;
  const int k0 = blockIdx.y * slice, k1 = min(p.n_in, k0 + slice);
  const T* a = reinterpret_cast<const T*>(p.a) + (mine >= 0 ? (int64_t)mine * p.a_stride_i : 0) + (int64_t)(k0 + kl) * p.a_stride_k + 4 * quad;
  const int64_t skip = (int64_t)lanes * p.a_stride_k;
  int left = mine >= 0 && kl < lanes && k0 + kl < k1 ? (k1 - k0 - kl + lanes - 1) / lanes : 0;  // this thread's inputs
  uint2 w[kStepLoads];
  auto load = [&]() {
#pragma unroll
    for (int l = 0; l < kStepLoads; ++l)
      if (l < left) w[l] = __ldg(reinterpret_cast<const uint2*>(a + l * skip));
  };
  load();
  rows_of(p, n, mine, &rows);
  const int count = rows.count;
  if (count == 0) return;
  const int R = count == 1 ? 1 : count == 2 ? 2 : 4;
  for (int i = 0; i < R; ++i) {
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)rows.row[i] * p.x_stride;  // (a row that is not there: row n again)
#pragma unroll 4
    for (int k = k0 + threadIdx.x; k < k1; k += kStepThreads) xs[(k - k0) * R + i] = wide(x[k]);
  }
  __syncthreads();
  float acc[kStepRows][4];
#pragma unroll
  for (int i = 0; i < kStepRows; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
  const float* x = xs + kl * R;
  while (left > 0) {
    if (R == 1) step_products<T, 1>(w, x, lanes, left, acc);
    else if (R == 2) step_products<T, 2>(w, x, lanes, left, acc);
    else step_products<T, 4>(w, x, lanes, left, acc);
    left -= kStepLoads;
    a += kStepLoads * skip;
    x += kStepLoads * lanes * R;
    load();
  }
  __syncthreads();
  if (kl < lanes) {
#pragma unroll
    for (int i = 0; i < kStepRows; ++i)
      if (i < R)
        *reinterpret_cast<float4*>(xs + (kl * R + i) * p.rank + 4 * quad) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  }
  __syncthreads();
  for (int j = threadIdx.x; j < count * p.rank; j += kStepThreads) {
    const int i = j / p.rank, r = j - i * p.rank;
    float s = 0.f;
#pragma unroll 4
    for (int l = 0; l < lanes; ++l) s += xs[(l * R + i) * p.rank + r];
    h[((int64_t)blockIdx.y * p.rows + rows.row[i]) * p.rank + r] = s;
  }
}

// out[row][8 columns a thread] of up to four rows
constexpr int kStepAhead = 8;  // ranks whose weights are asked for before the shrinking kernel has ended
template <typename T>
__global__ void __launch_bounds__(kStepThreads)
expand_step_kernel(const __grid_constant__ WsvdAdapterAddParams p, const float* h, const int slices) {
  extern __shared__ __align__(16) float hs[];  // [rank][rows], then a sum a thread
  __shared__ Rows rows;
  // What is read before the wait is nothing that the shrinking kernel writes, and that one has waited for what is in front
  // of it before it let this one in.  (Without adapters it does not run.)
  if (p.n_adapters == 0) before_this();
  const int n = blockIdx.x, mine = adapter_of(p, n), col = (blockIdx.y * kStepThreads + threadIdx.x) * 8;
  const bool on = col < p.n_out;
  if (mine < 0) {  // no adapter: y goes through
    before_this();
    if (on)
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + (int64_t)n * p.out_stride + col) =
          *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.y) + (int64_t)n * p.y_stride + col);
    return;
  }
  const T* b = reinterpret_cast<const T*>(p.b) + (int64_t)mine * p.b_stride_i + (on ? col : 0);
  uint4 ahead[kStepAhead];
#pragma unroll
  for (int r = 0; r < kStepAhead; ++r)
    if (r < p.rank) ahead[r] = __ldg(reinterpret_cast<const uint4*>(b + (int64_t)r * p.b_stride_r));
  if (on && (threadIdx.x & 7) == 0)  // (a line a thread)
    for (int r = kStepAhead; r < p.rank; ++r) asm volatile("prefetch.global.L2 [%0];\n" ::"l"(b + (int64_t)r * p.b_stride_r));
  rows_of(p, n, mine, &rows);
  const int count = rows.count;
  before_this();  // (also where another row's blocks do the work: no block ends before the shrinking kernel has)
  if (count == 0) return;
  const float scale = p.scale != nullptr ? p.scale[mine] : 1.f;
  // h: the slices' sums, dealt out to as many threads as there are, then theirs, always in the same order
  const int sums = count * p.rank, shares = sums < kStepThreads ? kStepThreads / sums : 1;
  for (int j = threadIdx.x; j < sums * shares; j += kStepThreads) {
    const int share = j / sums, i = (j - share * sums) / p.rank, r = j - share * sums - i * p.rank;
    const float* at = h + (int64_t)rows.row[i] * p.rank + r;
    const int64_t skip = (int64_t)p.rows * p.rank;
    float s = 0.f;
#pragma unroll 8
    for (int l = share; l < slices; l += shares) s += at[l * skip];
    (shares == 1 ? hs[r * kStepRows + i] : hs[kStepRows * p.rank + j]) = shares == 1 ? s * scale : s;
  }
  if (shares > 1) {
    __syncthreads();
    for (int j = threadIdx.x; j < sums; j += kStepThreads) {
      float s = 0.f;
      for (int l = 0; l < shares; ++l) s += hs[kStepRows * p.rank + l * sums + j];
      const int i = j / p.rank;
      hs[(j - i * p.rank) * kStepRows + i] = s * scale;
    }
  }
  __syncthreads();
  if (!on) return;
  float acc[kStepRows][8];
#pragma unroll
  for (int i = 0; i < kStepRows; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[i][e] = 0.f;
  auto all = [&](auto rows_at_once) {
    constexpr int R = decltype(rows_at_once)::value;
    auto add = [&](int r, const uint4& w) {
      const float4 f = *reinterpret_cast<const float4*>(hs + r * kStepRows);
      const float x[4] = {f.x, f.y, f.z, f.w};
      const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 t = two<T>(v[e]);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          acc[i][2 * e] = fmaf(x[i], t.x, acc[i][2 * e]);
          acc[i][2 * e + 1] = fmaf(x[i], t.y, acc[i][2 * e + 1]);
        }
      }
    };
#pragma unroll
    for (int r = 0; r < kStepAhead; ++r)
      if (r < p.rank) add(r, ahead[r]);
#pragma unroll 8
    for (int r = kStepAhead; r < p.rank; ++r) add(r, __ldg(reinterpret_cast<const uint4*>(b + (int64_t)r * p.b_stride_r)));
  };
  if (count == 1) all(std::integral_constant<int, 1>{});
  else if (count == 2) all(std::integral_constant<int, 2>{});
  else all(std::integral_constant<int, 4>{});
#pragma unroll
  for (int i = 0; i < kStepRows; ++i) {
    if (i >= count) continue;
    const uint4 y = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.y) + (int64_t)rows.row[i] * p.y_stride + col);
    const uint32_t v[4] = {y.x, y.y, y.z, y.w};
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 t = two<T>(v[e]);
      o[e] = both<T>(t.x + acc[i][2 * e], t.y + acc[i][2 * e + 1]);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + (int64_t)rows.row[i] * p.out_stride + col) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---- packed rows (prompts): products on the tensor cores, tiles of one request's rows (64 to shrink, 128 to expand)
//
// Bound by x, y and out.  Shrink: a warp has 16 rows and all ranks, tiles of 64 inputs come by 16-byte asynchronous copies;
// the input's length is cut into slices over the CTAs of a cluster, so that every SM has work, and their sums meet in
// shared memory in a fixed order (left to the expanding CTAs in f32 they cost those 12 us).  h is rounded once to the 16-bit
// type (PackedH, below).  Expand: tiles of 128 rows, equal shares of (tile, 64 columns) over the CTAs that the GPU holds at once; a
// warp has 32 rows and, up to 64 ranks, keeps their h in registers (less that is read from shared memory twice: 64-row tiles
// 97 us, 128 rows 92, with h in registers 89;
// 256 threads, or a third stage and a CTA less on the SM, 100 and 104).  B's columns come from L2 and y's from memory a unit ahead,
// y + product in place in shared memory, 16-byte stores.  7095 rows of 4096 to 11008, rank 64: 89 us, 4.2 TB/s of
// x, y and out (97 to 99 where the card is at its power limit): twelve warps an SM that wait for shared memory and for each other; neither
// it (60 %) nor HBM (51 %) is at its limit.
constexpr int kTileRows = 64, kTileCols = 64, kPackThreads = 128, kColPieces = kTileCols / 8;

// The row tiles of the batch, numbered through the requests in order; what is behind the last one and in front of the first
// counts as two more requests without an adapter where it is copied.  Every thread knows the tiles [before, before + mine) of its requests.
struct RowTile {
  int row, rows, adapter;  // rows 0: there is no such tile; adapter -1: none
};
template <int ROWS>
struct RowTiles {
  const WsvdAdapterAddParams& p;
  int b0, b1, before, mine, total;

  // rows [*from, result) of request b, inside [0, rows) whatever cu_new says; behind the last request (copied rows) what is behind
  // its rows, then what is in front of the first's
  __device__ __forceinline__ int span(int b, int* from) const {
    *from = b > p.batch ? 0 : min(max(p.cu_new[b], 0), p.rows);
    return b == p.batch ? p.rows : max(*from, min(p.cu_new[b > p.batch ? 0 : b + 1], p.rows));
  }
  __device__ __forceinline__ RowTiles(const WsvdAdapterAddParams& params) : p(params) {
    __shared__ int sums[kPackThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int requests = p.batch + (p.copy_tail ? 2 : 0), per = (requests + kPackThreads - 1) / kPackThreads;
    b0 = min(requests, (int)threadIdx.x * per);
    b1 = min(requests, b0 + per);
    mine = 0;
    for (int b = b0; b < b1; ++b) {
      int from;
      const int to = span(b, &from);
      mine += (to - from + ROWS - 1) / ROWS;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    before = incl - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPackThreads / 32; ++w) {
      if (w < warp) before += sums[w];
      total += sums[w];
    }
  }
  // tile number t, for all threads (between two block barriers)
  __device__ __forceinline__ RowTile find(int t) const {
    __shared__ RowTile tile;
    __syncthreads();
    if (t >= before && t < before + mine) {
      int first = before;
      for (int b = b0; b < b1; ++b) {
        int from;
        const int to = span(b, &from), n = (to - from + ROWS - 1) / ROWS;
        if (t < first + n) {
          const int row = from + (t - first) * ROWS;
          int i = b < p.batch ? p.adapter[b] : -1;
          if (i < -1 || i >= p.n_adapters) {
            atomicMax(&g_status, kOutsideStorage);
            i = -1;
          }
          tile = RowTile{row, min(ROWS, to - row), i};
          break;
        }
        first += n;
      }
    }
    __syncthreads();
    return tile;
  }
};

__device__ __forceinline__ void copy8(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(on ? 8 : 0) : "memory");
}
__device__ __forceinline__ void stmatrix4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// RP: the rank rounded up to 16, 32, 64, 128 or 256.  Pitches are an odd number of 16-byte pieces (conflict-free ldmatrix).
// Up to 64 ranks a warp takes half of the rows and every other 16 inputs, so that A is read from shared memory twice and not
// four times (its reads are what the loop waits for: 56 KB a stage with the rows alone dealt out, 40 KB so, 32 KB with the
// inputs alone, whose 128 accumulators cost a resident CTA); above, a warp takes 16 rows.
template <int RP>
struct Shrink {
  static constexpr int K = 64, STAGES = RP <= 128 ? 3 : 2;  // inputs of a stage
  static constexpr bool BY_INPUT = RP <= 64;
  static constexpr int MT = BY_INPUT ? 2 : 1;               // 16-row tiles of a warp
  static constexpr int X_PITCH = K * 2 + 16, A_PITCH = RP * 2 + 16;
  static constexpr int STAGE = kTileRows * X_PITCH + K * A_PITCH;
  static constexpr int LD = RP + 4;  // of the warps' sums (four more words a row: no bank twice)
};
// h of packed rows between the two kernels, rounded once to the rows' type.  x A has f32's range, which f16 has not, and its products with
// B may pass it where scale brings them back: rows are stored times the power of two that brings their largest to 2^14 .. 2^15
// (what is below it keeps all 11 bits of f16 down to 2^-28 of it).
// Why 16 bits: the error against 64 bits is 2.15e-4 in f16 and 1.76e-3 in bf16 (an adapter's share of a third of y, rank 64), where the
// result's own rounding is 2.08e-4 and 1.66e-3; a second 16-bit term takes that away for twice the products (7095 rows of
// 4096 to 11008: rank 64 89 us and 106 with it, rank 128 146 and 186).
template <typename T>
struct PackedH {
  T* rows;      // [rows][rp], rp: the rank rounded up to 16
  float* back;  // [rows] the inverse of the row's factor
};

// The CTAs of a cluster (along y) have one tile and a slice each.
template <typename T, int RP>
__global__ void __launch_bounds__(kPackThreads)
shrink_packed_kernel(const __grid_constant__ WsvdAdapterAddParams p, const PackedH<T> h, const int slice, const int rp) {
  using S = Shrink<RP>;
  extern __shared__ __align__(16) unsigned char smem[];
  before_this();
  let_next_in();
  const RowTiles<kTileRows> tiles(p);
  if ((int)blockIdx.x >= tiles.total) return;
  const RowTile tile = tiles.find(blockIdx.x);
  if (tile.adapter < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k0 = min(p.n_in, (int)blockIdx.y * slice), k1 = min(p.n_in, k0 + slice), steps = (k1 - k0 + S::K - 1) / S::K;
  const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)tile.row * p.x_stride;
  const T* a = reinterpret_cast<const T*>(p.a) + (int64_t)tile.adapter * p.a_stride_i;
  const uint32_t ring = smem_addr(smem);
  const bool wide_a = p.rank % 8 == 0 && p.a_stride_k % 8 == 0 && p.a_stride_i % 8 == 0 && (reinterpret_cast<uintptr_t>(p.a) & 15) == 0;
  // A thread's pieces of a stage: one column and every so many rows of x, and of A in 16- or 8-byte pieces.  (Addresses are
  // carried on: working them out took as long as the products.)
  constexpr int XP = S::K / 8, XROWS = kPackThreads / XP, XN = kTileRows / XROWS;
  const int x_row = threadIdx.x / XP, x_col = (threadIdx.x % XP) * 8;
  const T* x_at = x + (int64_t)x_row * p.x_stride + k0 + x_col;
  const int64_t x_skip = XROWS * p.x_stride;
  uint32_t x_on = 0;
#pragma unroll
  for (int i = 0; i < XN; ++i) x_on |= (uint32_t)(x_row + i * XROWS < tile.rows) << i;
  const uint32_t x_to = x_row * S::X_PITCH + x_col * 2;
  const int ap = wide_a ? RP / 8 : RP / 4, a_rows = kPackThreads / ap, a_row = threadIdx.x / ap, a_col = threadIdx.x % ap * (RP / ap);
  const bool a_on = a_col < p.rank;
  const T* a_at = a + (int64_t)(k0 + a_row) * p.a_stride_k + (a_on ? a_col : 0);
  const int64_t a_skip = a_rows * p.a_stride_k, a_step = S::K * p.a_stride_k;
  const uint32_t a_to = kTileRows * S::X_PITCH + a_row * S::A_PITCH + a_col * 2;
  int next = 0;
  uint32_t next_stage = ring;
  auto request = [&]() {
    if (next < steps) {
      const int k = k0 + next * S::K;
      const bool col_on = k + x_col < k1;
      const T* from = x_at;
#pragma unroll
      for (int i = 0; i < XN; ++i, from += x_skip) {
        const bool on = col_on && ((x_on >> i) & 1);
        copy16(next_stage + x_to + i * XROWS * S::X_PITCH, on ? from : x, on);
      }
      x_at += S::K;
      from = a_at;
      if (wide_a) {
        constexpr int ROWS = kPackThreads / (RP / 8);
#pragma unroll
        for (int i = 0; i < S::K / ROWS; ++i, from += a_skip) {
          const bool on = a_on && k + a_row + i * ROWS < k1;
          copy16(next_stage + a_to + i * ROWS * S::A_PITCH, on ? from : a, on);
        }
      } else {
        constexpr int ROWS = kPackThreads / (RP / 4);
#pragma unroll
        for (int i = 0; i < S::K / ROWS; ++i, from += a_skip) {
          const bool on = a_on && k + a_row + i * ROWS < k1;
          copy8(next_stage + a_to + i * ROWS * S::A_PITCH, on ? from : a, on);
        }
      }
      a_at += a_step;
    }
    ++next;
    next_stage = next_stage == ring + (S::STAGES - 1) * S::STAGE ? ring : next_stage + S::STAGE;
    copies_commit();
  };
  float acc[S::MT][RP / 8][4];
#pragma unroll
  for (int i = 0; i < S::MT * RP / 8 * 4; ++i) (&acc[0][0][0])[i] = 0.f;
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; ++i) request();
  uint32_t xd = ring;
  const int warp_row = S::BY_INPUT ? (warp >> 1) * 32 : warp * 16;
  for (int step = 0; step < steps; ++step) {
    copies_wait<S::STAGES - 2>();
    __syncthreads();  // this step's tiles are there for all, and all have done with the stage that is filled next
    request();
    const uint32_t ad = xd + kTileRows * S::X_PITCH;
    const uint32_t xa = xd + (warp_row + (lane & 15)) * S::X_PITCH + (lane >> 4) * 16;
    const uint32_t aa = ad + (lane & 15) * S::A_PITCH + (lane >> 4) * 16;
#pragma unroll
    for (int kk = 0; kk < S::K / 16 / (S::BY_INPUT ? 2 : 1); ++kk) {
      const int k = S::BY_INPUT ? 2 * kk + (warp & 1) : kk;
      uint32_t xr[S::MT][4];
#pragma unroll
      for (int i = 0; i < S::MT; ++i) ldmatrix4(xr[i], xa + i * 16 * S::X_PITCH + k * 32);
      constexpr int AT = RP / 16 < 4 ? RP / 16 : 4;  // loads in flight in front of their products
#pragma unroll
      for (int j0 = 0; j0 < RP / 16; j0 += AT) {
        uint32_t w[AT][4];  // ranks 16 j .. + 7: w[j][0], w[j][1] (inputs 0-7, 8-15); + 8 .. + 15: w[j][2], w[j][3]
#pragma unroll
        for (int j = 0; j < AT; ++j) ldmatrix4_trans(w[j], aa + k * 16 * S::A_PITCH + (j0 + j) * 32);
#pragma unroll
        for (int j = 0; j < AT; ++j)
#pragma unroll
          for (int i = 0; i < S::MT; ++i) {
            mma<T>(acc[i][2 * (j0 + j)], xr[i], w[j][0], w[j][1]);
            mma<T>(acc[i][2 * (j0 + j) + 1], xr[i], w[j][2], w[j][3]);
          }
      }
    }
    xd = xd == ring + (S::STAGES - 1) * S::STAGE ? ring : xd + S::STAGE;
  }
  // the sums of the warps with other inputs, then those of the slices: each CTA leaves its own in its shared memory and adds up
  // its part of the rows from all of them
  copies_wait<0>();
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
  const int g = lane >> 2, c4 = lane & 3;
#pragma unroll
  for (int pass = S::BY_INPUT ? 0 : 1; pass < 2; ++pass) {
    if (!S::BY_INPUT || (warp & 1) != pass)
#pragma unroll
      for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int j = 0; j < RP / 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float2* at = reinterpret_cast<float2*>(sums + (warp_row + 16 * i + g + 8 * e) * S::LD + 8 * j + 2 * c4);
            float2 v = make_float2(acc[i][j][2 * e], acc[i][j][2 * e + 1]);
            if (S::BY_INPUT && pass == 1) {
              const float2 w = *at;
              v.x += w.x;
              v.y += w.y;
            }
            *at = v;
          }
    if (pass == 0) __syncthreads();
  }
  const auto cluster = cooperative_groups::this_cluster();
  cluster.sync();
  const int slices = cluster.num_blocks(), part = kTileRows / slices, from = (int)cluster.block_rank() * part;
  // G lanes a row, PAIRS pairs of ranks a lane
  constexpr int G = RP / 2 < 32 ? RP / 2 : 32, PAIRS = RP / 2 / G, ROWS = kPackThreads / G;
  const int member = threadIdx.x % G;
  for (int row0 = 0; row0 < part; row0 += ROWS) {
    const int in_part = row0 + threadIdx.x / G, row = from + in_part;
    const bool on = in_part < part && row < tile.rows;
    float2 v[PAIRS];
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const int r = 2 * (member + j * G);
      float2 w[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)  // (all loads in flight)
        w[c] = on && r < rp && c < slices ? *reinterpret_cast<const float2*>(cluster.map_shared_rank(sums, c) + row * S::LD + r) : make_float2(0.f, 0.f);
      v[j] = w[0];
#pragma unroll
      for (int c = 1; c < 8; ++c) {
        v[j].x += w[c].x;
        v[j].y += w[c].y;
      }
      if (isfinite(v[j].x)) amax = fmaxf(amax, fabsf(v[j].x));
      if (isfinite(v[j].y)) amax = fmaxf(amax, fabsf(v[j].y));
    }
#pragma unroll
    for (int o = 1; o < G; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    // (rows below 2^-112 are brought up by 2^126, the largest factor whose inverse is no subnormal)
    const int e = amax > 0.f ? max(-126, (__float_as_int(amax) >> 23) - 127 - 14) : 0;
    const float up = power_of_two(-e);
    if (on && member == 0) h.back[tile.row + row] = power_of_two(e);
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const int r = 2 * (member + j * G);
      if (on && r < rp)  // (ranks up to rp: zeros)
        *reinterpret_cast<uint32_t*>(h.rows + (int64_t)(tile.row + row) * rp + r) = both<T>(v[j].x * up, v[j].y * up);
    }
  }
  cluster.sync();  // (nobody's shared memory goes while another reads it)
}

constexpr int kWideRows = 128, kWarpRows = kWideRows / (kPackThreads / 32), kMt = kWarpRows / 16;
constexpr int kColPitch = kTileCols * 2 + 16;  // bytes of a tile row of B or y
// HK: how many 16 ranks of h a warp keeps in registers (0: it reads them from shared memory again for every unit).
template <typename T, int HK>
__global__ void __launch_bounds__(kPackThreads, 3)
expand_packed_kernel(const __grid_constant__ WsvdAdapterAddParams p, const PackedH<T> h, const int rp) {
  extern __shared__ __align__(16) unsigned char smem[];  // h [128][rp], then two stages of B [rp][64] and y [128][64]
  // (What is read before the wait is nothing that the shrinking kernel writes: see expand_step_kernel.)
  if (p.n_adapters == 0) before_this();
  const RowTiles<kWideRows> tiles(p);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
  const int blocks = (p.n_out + kTileCols - 1) / kTileCols;
  const int64_t units = (int64_t)tiles.total * blocks;
  const int shares = (int)min((int64_t)gridDim.x, units);
  int64_t unit = (int)blockIdx.x < shares ? share_begin(blockIdx.x, units, shares) : 0;
  const int64_t end = (int)blockIdx.x < shares ? share_begin(blockIdx.x + 1, units, shares) : 0;
  const int h_pitch = rp * 2 + 16, b_bytes = rp * kColPitch, stage_bytes = b_bytes + kWideRows * kColPitch;
  const uint32_t hd = smem_addr(smem), ring = hd + kWideRows * h_pitch;
  bool waited = p.n_adapters == 0;
  auto wait_once = [&]() {
    if (!waited) before_this();
    waited = true;
  };
  while (unit < end) {
    // the share's columns of one tile of rows
    const int t = (int)(unit / blocks);
    const int c0 = (int)(unit - (int64_t)t * blocks) * kTileCols;
    const int steps = (int)min(end - unit, (int64_t)blocks - c0 / kTileCols), c1 = min(p.n_out, c0 + steps * kTileCols);
    unit += steps;
    const RowTile tile = tiles.find(t);
    const T* y = reinterpret_cast<const T*>(p.y) + (int64_t)tile.row * p.y_stride;
    T* out = reinterpret_cast<T*>(p.out) + (int64_t)tile.row * p.out_stride;
    if (tile.adapter < 0) {
      wait_once();
      if (p.out == p.y) continue;
      const int vecs = (c1 - c0) / 8;
      for (int i = threadIdx.x; i < tile.rows * vecs; i += kPackThreads) {
        const int row = i / vecs, col = c0 + (i - row * vecs) * 8;
        *reinterpret_cast<uint4*>(out + (int64_t)row * p.out_stride + col) =
            *reinterpret_cast<const uint4*>(y + (int64_t)row * p.y_stride + col);
      }
      continue;
    }
    const T* b = reinterpret_cast<const T*>(p.b) + (int64_t)tile.adapter * p.b_stride_i;
    // a thread's pieces of a unit: one column, every so many rows of B and of the warp's own 16 of y
    constexpr int BROWS = kPackThreads / kColPieces, YROWS = 32 / kColPieces, YN = kWarpRows / YROWS;
    const int col = (threadIdx.x % kColPieces) * 8, b_row = threadIdx.x / kColPieces, y_row = warp * kWarpRows + lane / kColPieces;
    const T* b_at = b + (int64_t)b_row * p.b_stride_r + c0 + col;
    const T* y_at = y + (int64_t)y_row * p.y_stride + c0 + col;
    T* out_at = out + (int64_t)y_row * p.out_stride + c0 + col;
    const int64_t b_skip = BROWS * p.b_stride_r, y_skip = YROWS * p.y_stride, out_skip = YROWS * p.out_stride;
    uint32_t y_on = 0;
#pragma unroll
    for (int i = 0; i < YN; ++i) y_on |= (uint32_t)(y_row + i * YROWS < tile.rows) << i;
    auto request = [&](int step) {
      if (step < steps) {
        const uint32_t bd = ring + (step & 1) * stage_bytes + b_row * kColPitch + col * 2;
        const uint32_t yd = ring + (step & 1) * stage_bytes + b_bytes + y_row * kColPitch + col * 2;
        const bool in = c0 + step * kTileCols + col < c1;
        const T* from = y_at;
#pragma unroll
        for (int i = 0; i < YN; ++i, from += y_skip) {
          const bool on = in && ((y_on >> i) & 1);
          copy16(yd + i * YROWS * kColPitch, on ? from : y, on);
        }
        y_at += kTileCols;
        from = b_at;
#pragma unroll 4
        for (int i = 0; i < rp / BROWS; ++i, from += b_skip) {
          const bool on = in && b_row + i * BROWS < p.rank;
          copy16(bd + i * BROWS * kColPitch, on ? from : b, on);
        }
        b_at += kTileCols;
      }
      copies_commit();
    };
    request(0);
    wait_once();
    const float scale = p.scale != nullptr ? p.scale[tile.adapter] : 1.f;
    for (int i = threadIdx.x; i < kWideRows * (rp / 8); i += kPackThreads) {
      const int row = i / (rp / 8), r = (i % (rp / 8)) * 8;
      const bool on = row < tile.rows;
      copy16(hd + row * h_pitch + r * 2, h.rows + (on ? (int64_t)(tile.row + row) * rp + r : 0), on);
    }
    copies_commit();
    float back[kMt][2];  // of rows g and g + 8 of every 16: the adapter's scale, and what the row's factor takes back
#pragma unroll
    for (int i = 0; i < kMt; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = warp * kWarpRows + 16 * i + 8 * e + g;
        back[i][e] = row < tile.rows ? scale * __ldcg(h.back + tile.row + row) : 0.f;
      }
    const uint32_t ha = hd + (warp * kWarpRows + (lane & 15)) * h_pitch + (lane >> 4) * 16;
    uint32_t hr[HK > 0 ? HK : 1][kMt][4];
    for (int step = 0; step < steps; ++step) {
      request(step + 1);
      copies_wait<1>();
      __syncthreads();
      if (HK > 0 && step == 0) {
#pragma unroll
        for (int k = 0; k < HK; ++k)
#pragma unroll
          for (int i = 0; i < kMt; ++i) {
            if (k < rp / 16) ldmatrix4(hr[k][i], ha + i * 16 * h_pitch + k * 32);
            else hr[k][i][0] = hr[k][i][1] = hr[k][i][2] = hr[k][i][3] = 0;
          }
      }
      const uint32_t bd = ring + (step & 1) * stage_bytes;
      const uint32_t yt = bd + b_bytes;
      float acc[kMt][kTileCols / 8][4];
#pragma unroll
      for (int i = 0; i < kMt * kTileCols / 8 * 4; ++i) (&acc[0][0][0])[i] = 0.f;
      const uint32_t ba = bd + (lane & 15) * kColPitch + (lane >> 4) * 16;
      auto products = [&](int k, const uint32_t (&h16)[kMt][4]) {
        uint32_t w[kTileCols / 16][4];
#pragma unroll
        for (int j = 0; j < kTileCols / 16; ++j) ldmatrix4_trans(w[j], ba + k * 16 * kColPitch + j * 32);
#pragma unroll
        for (int j = 0; j < kTileCols / 16; ++j)
#pragma unroll
          for (int i = 0; i < kMt; ++i) {
            mma<T>(acc[i][2 * j], h16[i], w[j][0], w[j][1]);
            mma<T>(acc[i][2 * j + 1], h16[i], w[j][2], w[j][3]);
          }
      };
      if constexpr (HK > 0) {
#pragma unroll
        for (int k = 0; k < HK; ++k)
          if (k < rp / 16) products(k, hr[k]);
      } else {
#pragma unroll 2
        for (int k = 0; k < rp / 16; ++k) {
#pragma unroll
          for (int i = 0; i < kMt; ++i) ldmatrix4(hr[0][i], ha + i * 16 * h_pitch + k * 32);
          products(k, hr[0]);
        }
      }
      // y as the accumulators hold their values, 16 rows of 16 columns at a time, and back
      const uint32_t ya = yt + (warp * kWarpRows + (lane & 15)) * kColPitch + (lane >> 4) * 16;
#pragma unroll
      for (int ij = 0; ij < kMt * kTileCols / 16; ++ij) {
        const int i = ij / (kTileCols / 16), j = ij % (kTileCols / 16);
        uint32_t v[4];  // rows 0-7 and 8-15 of columns 0-7, then of columns 8-15
        ldmatrix4(v, ya + i * 16 * kColPitch + j * 32);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = two<T>(v[e]);
          const float* d = acc[i][2 * j + (e >> 1)] + 2 * (e & 1);
          v[e] = both<T>(fmaf(back[i][e & 1], d[0], f.x), fmaf(back[i][e & 1], d[1], f.y));
        }
        stmatrix4(ya + i * 16 * kColPitch + j * 32, v);
      }
      __syncwarp();  // the warp's rows are its own
      const uint32_t from = yt + y_row * kColPitch + col * 2;
      T* to = out_at;
      const bool in = c0 + step * kTileCols + col < c1;
#pragma unroll
      for (int i = 0; i < YN; ++i, to += out_skip)
        if (in && ((y_on >> i) & 1)) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(smem + (from - hd) + i * YROWS * kColPitch);
      out_at += kTileCols;
      __syncthreads();  // the stage may be filled again
    }
    copies_wait<0>();
  }
  wait_once();  // (no block ends before the shrinking kernel has)
}

// ---- host side

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// y, out and B in whole 16-byte vectors, A in whole 8-byte ones; packed rows: x in 16-byte vectors too
bool whole_vectors(const WsvdAdapterAddParams& p) {
  if (p.rank % 4 || p.n_out % 8) return false;
  if (!aligned(p.y, 16) || !aligned(p.out, 16) || !aligned(p.b, 16) || !aligned(p.a, 8)) return false;
  if ((p.y_stride | p.out_stride | p.b_stride_i | p.b_stride_r) % 8 || (p.a_stride_i | p.a_stride_k) % 4) return false;
  if (p.cu_new == nullptr) return p.n_in <= kMaxSlices * kMaxSlice;
  return (p.n_in % 8 == 0 && aligned(p.x, 16) && p.x_stride % 8 == 0);
}
int rank_padded(int rank) {
  int r = 16;
  while (r < rank) r *= 2;
  return r;
}
int packed_tiles(const WsvdAdapterAddParams& p) { return p.rows / kTileRows + p.batch + 2; }
int rank_16(const WsvdAdapterAddParams& p) { return (p.rank + 15) / 16 * 16; }
// Steps: inputs of a slice.  A thread of the shrinking kernel asks for kStepLoads inputs at once, and a slice is so many for each
// of the block's lanes (64 rows, rank 32, 5120 inputs: 40 slices 24.9 us, 20 slices of 16 loads 26.2 us), but there are no
// more than kMaxSlices, and none is longer than kMaxSlice (four rows of it in f32: what fits shared memory).
int slice_of(const WsvdAdapterAddParams& p) {
  const int lanes = kStepThreads / (p.rank < 4 ? 1 : p.rank / 4 > kStepThreads ? kStepThreads : p.rank / 4);
  const int slice = lanes * kStepLoads, least = (p.n_in + kMaxSlices - 1) / kMaxSlices;
  return slice < least ? least : slice > kMaxSlice ? kMaxSlice : slice;
}
int slices_of(const WsvdAdapterAddParams& p) { return (p.n_in + slice_of(p) - 1) / slice_of(p); }

template <typename T>
cudaError_t launch_step(const WsvdAdapterAddParams& p, float* h, cudaStream_t s) {
  const int slice = slice_of(p), slices = slices_of(p);
  const int lanes = kStepThreads / (p.rank / 4);
  const size_t xs = (size_t)slice * kStepRows, red = (size_t)lanes * kStepRows * p.rank;
  cudaError_t e = p.n_adapters == 0 ? cudaSuccess
                                    : launch_overlapped(shrink_step_kernel<T>, dim3(p.rows, slices), kStepThreads, (xs > red ? xs : red) * sizeof(float),
                                                        s, 1, p, h, slice);
  if (e != cudaSuccess) return e;
  return launch_overlapped(expand_step_kernel<T>, dim3(p.rows, (p.n_out + kStepCols - 1) / kStepCols), kStepThreads,
                           ((size_t)kStepRows * p.rank + kStepThreads) * sizeof(float), s, 1, p, (const float*)h, slices);
}

// more than 48 KB of dynamic shared memory has to be asked for, once per kernel and device
template <typename K>
cudaError_t allow_smem(K kernel, bool (&ready)[kMaxDevices], size_t bytes) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device < 0 || device >= kMaxDevices)) e = cudaErrorInvalidDevice;
  if (e != cudaSuccess || ready[device]) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) ready[device] = true;
  return e;
}

template <typename T, int RP>
cudaError_t launch_shrink(const WsvdAdapterAddParams& p, const PackedH<T>& h, cudaStream_t s) {
  using S = Shrink<RP>;
  static bool ready[kMaxDevices];
  constexpr size_t ring = (size_t)S::STAGES * S::STAGE, sums = (size_t)kTileRows * S::LD * sizeof(float), smem = ring > sums ? ring : sums;
  const cudaError_t e = allow_smem(shrink_packed_kernel<T, RP>, ready, smem);
  if (e != cudaSuccess) return e;
  // slices: enough CTAs for every SM to have three, none shorter than 256 inputs
  int slices = 1;
  while (slices < 8 && (int64_t)(p.rows / kTileRows + 1) * slices < 148 * 3 && p.n_in / (2 * slices) >= 256) slices *= 2;
  const int slice = ((p.n_in + slices - 1) / slices + S::K - 1) / S::K * S::K;
  return launch_overlapped(shrink_packed_kernel<T, RP>, dim3(packed_tiles(p), slices), kPackThreads, smem, s, slices, p, h, slice, rank_16(p));
}

template <typename T, int HK>
cudaError_t launch_expand(const WsvdAdapterAddParams& p, const PackedH<T>& h, cudaStream_t s) {
  static bool ready[kMaxDevices];
  const int rp = rank_16(p);
  auto bytes = [](int r) { return (size_t)kWideRows * (r * 2 + 16) + 2 * ((size_t)r * kColPitch + kWideRows * kColPitch); };
  cudaError_t e = allow_smem(expand_packed_kernel<T, HK>, ready, bytes(256));
  if (e != cudaSuccess) return e;
  // CTAs that the GPU holds at once, asked once per device and rank (what is written twice is the same)
  int device = 0;
  e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  static int resident[kMaxDevices][17];
  int& fits = resident[device][rp / 16];
  if (fits == 0) {
    int per_sm = 0, sms = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, expand_packed_kernel<T, HK>, kPackThreads, bytes(rp));
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return e;
    fits = per_sm * sms > 0 ? per_sm * sms : 1;
  }
  const int64_t units = (int64_t)packed_tiles(p) * ((p.n_out + kTileCols - 1) / kTileCols);
  return launch_overlapped(expand_packed_kernel<T, HK>, dim3((unsigned)(units < fits ? units : fits)), kPackThreads, bytes(rp), s, 1, p, h, rp);
}

template <typename T>
cudaError_t launch_packed(const WsvdAdapterAddParams& p, void* workspace, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  const PackedH<T> h{reinterpret_cast<T*>(workspace), reinterpret_cast<float*>(reinterpret_cast<T*>(workspace) + (int64_t)p.rows * rank_16(p))};
  if (p.n_adapters > 0) {
    switch (rank_padded(p.rank)) {
      case 16: e = launch_shrink<T, 16>(p, h, s); break;
      case 32: e = launch_shrink<T, 32>(p, h, s); break;
      case 64: e = launch_shrink<T, 64>(p, h, s); break;
      case 128: e = launch_shrink<T, 128>(p, h, s); break;
      default: e = launch_shrink<T, 256>(p, h, s); break;
    }
    if (e != cudaSuccess) return e;
  }
  return p.rank <= 64 ? launch_expand<T, 4>(p, h, s) : launch_expand<T, 0>(p, h, s);
}

template <typename T>
cudaError_t launch_adapters(const WsvdAdapterAddParams& p, void* workspace, cudaStream_t s) {
  float* h = reinterpret_cast<float*>(workspace);
  if (whole_vectors(p)) return p.cu_new != nullptr ? launch_packed<T>(p, workspace, s) : launch_step<T>(p, h, s);
  shrink_any_kernel<T><<<p.rows, 128, 0, s>>>(p, h);
  expand_any_kernel<T><<<dim3(p.rows, (p.n_out + 255) / 256), 256, 0, s>>>(p, h);
  return cudaGetLastError();
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
  if (!p || p->rows <= 0 || p->rank <= 0 || p->n_in <= 0 || p->batch < 0) return 0;
  // packed rows: h in f32 or, its rows padded to 16s, in 16 bits with a factor a row, which is no more; one row per request: a sum per
  // slice of the input
  if (p->cu_new) return (size_t)p->rows * (p->rank < 16 ? 16 : p->rank) * sizeof(float);
  return (size_t)wsvd::slices_of(*p) * p->rows * p->rank * sizeof(float);
}

int wsvd_adapter_add(const WsvdAdapterAddParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (!p) return WSVD_ERR_NULL_POINTER;
  if (p->rows < 0 || p->batch < 0 || p->n_in <= 0 || p->n_out <= 0 || p->n_adapters < 0) return WSVD_ERR_BAD_SHAPE;
  if (p->rank <= 0 || p->rank > 256) return WSVD_ERR_BAD_SHAPE;
  if (p->dtype != WSVD_F16 && p->dtype != WSVD_BF16) return WSVD_ERR_BAD_DTYPE;
  if (!p->cu_new && p->rows != p->batch) return WSVD_ERR_BAD_SHAPE;
  if (p->rows > wsvd::kMostCounted || p->batch > wsvd::kMostCounted || p->n_in > wsvd::kMostCounted) return WSVD_ERR_TOO_LARGE;
  if ((p->n_out - 1) / 256 >= 65535) return WSVD_ERR_TOO_LARGE;
  if (p->rows == 0) return WSVD_OK;
  if (!p->y || !p->x || !p->out || (p->batch > 0 && !p->adapter)) return WSVD_ERR_NULL_POINTER;
  if (p->n_adapters > 0 && (!p->a || !p->b)) return WSVD_ERR_NULL_POINTER;
  if (!workspace) return WSVD_ERR_NULL_POINTER;
  if (workspace_bytes < wsvd_adapter_add_workspace_bytes(p)) return WSVD_ERR_WORKSPACE_TOO_SMALL;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WSVD_ERR_BAD_STRIDE;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = p->dtype == WSVD_F16 ? wsvd::launch_adapters<__half>(*p, workspace, s)
                                             : wsvd::launch_adapters<__nv_bfloat16>(*p, workspace, s);
  return e == cudaSuccess ? WSVD_OK : wsvd::record_cuda_error(e);
}

}  // extern "C"
