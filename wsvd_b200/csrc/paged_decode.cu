// wsvd_paged_decode: attention of one new token per sequence over a paged cache.
//
//   out = sum_s w_s v_s / sum_s w_s,  w_s = exp(c q . k_s - max),  max(0, len - window) <= s < len
//   lse = max + log(sum_s w_s);  no positions: out = 0, lse = -inf
#include <type_traits>

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

// ---- the tensor-core kernel: head_dim 64, 96, 128 and 256, rows of whole 16-byte pieces
//
// Memory bound: 2 D values of cache per token and KV head, once for all its query heads.  The scores of a warp's 16 tokens
// are one product S^T = K Q^T with the tokens as rows (m16n8k16: a row of 8 query heads costs nothing more than one head), and
// O^T += V^T P^T has the dims as rows, so that a query head's statistics, weights and sums sit in the same lanes and the
// accumulators are half of what 16 padded heads would take.  P^T is S^T's fragment turned by movmatrix.
//
// Every warp has a ring of its own in shared memory, filled with 16-byte asynchronous copies of its tokens' rows (zeros for
// rows that are masked: what they hold must not reach a product), waits for nothing but its own copies, and goes on from one
// sequence and head to the next without draining the ring.  The tiles of the batch are dealt out in equal shares to the CTAs
// (common.cuh), so that ragged batches load every SM alike; what several CTAs hold of one (sequence, head) they leave
// as partial sums, which paged_merge_kernel joins in a fixed order.
//
// Measured, a call: 16 sequences of 4096, 40 heads of 128, f16: 212 us, 6.3 TB/s of cache (a plain copy: 6.56); 32 of 300 to 8192,
// 32 heads on 8, bf16: 86 us, 5.7 TB/s; 48 in a window of 4096, heads of 64: 63 us, 5.3 TB/s; bytes, 8 of up to 32768: 69 to 78 us, 5.1
// to 4.5 TB/s (twelve warps an SM wait for their own instructions: seven matrix products a 16 tokens and 32 dims, values converted one by
// one); one of 2048: 14 us,
// of which the page table, the rows and the merge wait for one another 10 (at other batches 4 us are the ends of the call).
//
// Weights go into the product as two 16-bit terms (17 bits of bf16, 22 of f16): the one rounding that is left is the
// result's.  int8 keys meet their queries as bytes: a query row is taken to 24 bits below its largest value (a power of two
// times it, so that bf16 ones of any size fit) and split into three bytes, whose products with the keys' are exact.  (Two bytes
// are 9 % less time where heads are of 256, 1 % where they are of 128, and lose the small values of a row beside one large one: scores
// off by up to 0.01 where it is 200 times the others.)  int8
// values become f16 exactly (a byte under the exponent of 1024); the running maximum is that of score times v scale, so
// that the weights with the v scale in them stay at or below one.

constexpr int kWarps = 4, kThreads = kWarps * 32;
// bounds of the shares, for the workspace: CTAs of a GPU of so many SMs, CTAs of an item (one sequence of 60000 with one KV head:
// 24 us with at most 128, 48 with all of the GPU's, whose partials one block has to join)
constexpr int kMaxSms = 160, kMaxCtas = 4, kMaxParts = 128;

__device__ __forceinline__ uint32_t turned(uint32_t v) {  // an 8 x 8 fragment of 16-bit values, transposed
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma_s8_s8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_u8(int32_t (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// bytes of u (signed values + 128) at two places -> f16 pair: 0x64 on top of a byte is 1024 + byte
template <uint32_t kPlaces>
__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t u) {
  const uint32_t v = __byte_perm(u, 0x64646464u, kPlaces);
  const uint32_t k1152 = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&k1152));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Brings a line to L1 without waiting for it (the streams of rows go past L1, so it is still there when it is read).
__device__ __forceinline__ void touch(const void* p) {
  uint32_t ignored;
  asm volatile("ld.global.ca.b32 %0, [%1];\n" : "=r"(ignored) : "l"(p));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

template <typename T_, bool I8_, int D_, int NT_>
struct Cfg {
  using T = T_;                                                         // q and out
  using M = typename std::conditional<I8_, __half, T_>::type;           // the products' operands
  static constexpr bool I8 = I8_;
  static constexpr int D = D_, NT = NT_;                                // NT: eights of query heads of an item
  static constexpr int ROW = D * (I8 ? 1 : 2), PIECES = ROW / 16;       // bytes and 16-byte pieces of a cached row
  // conflict-free ldmatrix: the pieces of a row changed about by the row's number, or rows of an odd number of pieces
  static constexpr bool SWZ = PIECES == 8 || PIECES == 16 || PIECES == 32;
  static constexpr int PITCH = SWZ ? ROW : (PIECES | 1) * 16;
  static constexpr int TOK = ROW > 128 ? 16 : 32, SUBS = TOK / 16;      // tokens of a warp's step
  static constexpr int SLOT_BYTES = TOK * PITCH;                        // a ring slot: K or V rows of a step
  static constexpr int RING = kWarps * 4 * SLOT_BYTES;
  // CTAs of an SM that registers have to leave room for
  static constexpr int CTAS = NT == 2 ? 2 : D <= 128 ? 3 : 2;
  // where a row's piece is, from the row's first byte (rows start on their own size where pieces change places)
  static __device__ __forceinline__ uint32_t at(int row, int piece) {
    return row * PITCH + (SWZ ? (piece ^ (row & 7)) * 16 : piece * 16);
  }
  // the address of the piece `more` (even) behind the one at `addr`: at(row, piece) + ... for piece 0 or 1
  static __device__ __forceinline__ uint32_t skip(uint32_t addr, int more) { return SWZ ? addr ^ (more * 16) : addr + more * 16; }
  static constexpr uint32_t FULL = TOK == 32 ? 0xffffffffu : 0xffffu;
  // The reference of the weights is a past maximum until one is 2^SLACK above it: sums are rescaled once or twice instead of
  // at every new maximum.  f16 weights are lifted so far that they use all of f16's range above one: 2^7 2^8 = 2^15, and
  // what is left of them below it is 2^-31 of the reference.  bf16 ones are let down to at most one: values may be as large as f32's.
  static constexpr float SLACK = 8.f, LIFT = std::is_same<M, __half>::value ? 7.f : -SLACK;
};

// What the ring holds besides rows: which tokens count, and (read where a run begins or ends) of which item.
struct Step {
  uint32_t mask;
  int32_t flags;  // 1: first step of a run in this CTA, 2: last one
};
struct Run {
  int64_t item_first;  // the item's first tile in the batch's order
  int32_t b, it, hk, tiles, tokens;
};

// How a sequence is cut into items: `hw` neighbouring KV heads, a warp each (the CTA's other warps, where heads are few, take
// other tokens of the same ones), and a chunk of at most 16 of the `group` query heads of each, `hpi` of `chunks`.
// Four heads of a token-major cache are one run of memory per token, and no warp has to wait for another.
struct Items {
  int group, hpi, chunks, nt, hw;
};

// Partial sums of a run: [slot][head of the item][D] f32, (maximum, sum) beside them, and per item the first slot and how many.
struct Partials {
  float* o;
  float2* ml;
  int2* items;
};

template <typename C>
__global__ void __launch_bounds__(kThreads, C::CTAS)
paged_decode_kernel(const __grid_constant__ WsvdPagedDecodeParams p, const Partials part, const Items items) {
  using T = typename C::T;
  using M = typename C::M;
  constexpr int D = C::D, NT = C::NT, TOK = C::TOK, META = 4;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ Step ring[kWarps][META];
  __shared__ Run ring_run[kWarps][META];
  __shared__ __half2 sm_scale[C::I8 ? kWarps : 1][TOK];  // k and v scale of the present step's tokens
  __shared__ int64_t sm_scan[kWarps];
  __shared__ int64_t sm_before;
  __shared__ int sm_b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c4 = lane & 3;
  const int group = items.group, hpi = items.hpi, chunks = items.chunks;
  const int n_it = p.n_kv_heads / items.hw * chunks;  // items of a sequence
  const int head_of_warp = warp & (items.hw - 1), part_of_warp = warp / items.hw, tile = TOK * kWarps / items.hw;

  before_this();
  let_next_in();

  auto tiles_of = [&](int b) {
    int n = min(p.b_seq_len[b], p.max_len);
    const int req = p.b_req_idx[b];
    if (n <= 0 || req < 0 || req >= p.n_req) return 0;
    if (p.window > 0) n = min(n, p.window);
    return (n + tile - 1) / tile;
  };

  // ---- this CTA's share [lo, hi) of the tiles in the order (sequence, item, tile); a warp takes its tokens of each
  const int per = (p.batch + kThreads - 1) / kThreads, b0 = min(p.batch, (int)threadIdx.x * per), b1 = min(p.batch, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles_of(b);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sm_scan[warp] = incl;
  __syncthreads();
  int64_t total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sm_scan[w];
    total += sm_scan[w];
  }
  total *= n_it;
  before *= n_it;
  const int shares = (int)min((int64_t)gridDim.x, total), share = blockIdx.x;
  const bool busy = share < shares;
  const int64_t lo = busy ? share_begin(share, total, shares) : 0, hi = busy ? share_begin(share + 1, total, shares) : 0;
  if (busy && lo >= before && lo < before + mine * n_it) {
    int b = b0;
    int64_t first = before;
    for (;; ++b) {
      const int64_t n = (int64_t)tiles_of(b) * n_it;
      if (lo < first + n) break;
      first += n;
    }
    sm_b = b;
    sm_before = first;
  }
  __syncthreads();

  if (busy) {
    // ---- the cursor: the step whose rows are requested next
    int left = (int)(hi - lo);  // tiles not yet requested
    int cb = sm_b, cnt = tiles_of(cb), cit, ct, hk, first, end, s, tokens;
    int64_t seq_first = sm_before;
    {
      const int64_t in = lo - seq_first;
      cit = (in >> 32) == 0 ? (int)((uint32_t)in / (uint32_t)cnt) : (int)(in / cnt);
      ct = (int)(in - (int64_t)cit * cnt);
    }
    const int32_t* page;
    auto enter_sequence = [&]() {
      const Span sp = span_of(p, cb);
      first = sp.first + part_of_warp * TOK + lane;
      tokens = sp.end - sp.first;
      end = lane < TOK ? sp.end : 0;
      page = sp.page;
    };
    // A lane's pieces of a step's rows: where 32 lanes are whole rows, every lane has one column of them
    constexpr bool kColumns = 32 % C::PIECES == 0;
    constexpr int ES = C::I8 ? 1 : 2;
    const int k_row = (int)(p.k_stride_t * ES), v_row = (int)(p.v_stride_t * ES);
    const char *kb, *vb;
    auto enter_item = [&]() {
      hk = cit / chunks * items.hw + head_of_warp;
      const int col = kColumns ? (lane % C::PIECES) * 16 : 0;
      kb = reinterpret_cast<const char*>(p.k) + (int64_t)hk * p.k_stride_h * ES + col;
      vb = reinterpret_cast<const char*>(p.v) + (int64_t)hk * p.v_stride_h * ES + col;
      s = first;
    };
    enter_sequence();
    enter_item();
    s += ct * tile;
    int fresh = 1;  // the run begins with this step
    const uint32_t n_slots = (uint32_t)min((int64_t)INT32_MAX, p.n_token_slots);
    const uint32_t my_ring = smem_addr(smem) + warp * 4 * C::SLOT_BYTES;
    // lane i has token i's slot, fetched a step ahead; what the first steps and runs wait for is touched early
    int slot = s < end ? page[s] : 0;
    if (s + tile < end) touch(page + s + tile);

    // rows of one step, K or V, to a ring slot; lane i holds token i's slot, `mask` which tokens count
    auto copy_rows = [&](uint32_t dst, const char* base, int from, int stride, uint32_t mask) {
      auto copy = [&](auto all) {
#pragma unroll
        for (int i = 0; i < TOK * C::PIECES / 32; ++i) {
          const int piece = lane + 32 * i, row = piece / C::PIECES, col = kColumns ? 0 : (piece - row * C::PIECES) * 16;
          const int t = __shfl_sync(0xffffffffu, from, row);
          copy16(dst + C::at(row, piece - row * C::PIECES), base + (int64_t)t * stride + col,
                 decltype(all)::value || ((mask >> row) & 1));
        }
      };
      if (mask == C::FULL) copy(std::true_type{});
      else copy(std::false_type{});
    };
    // K of the cursor's step, and what the step is; the cursor goes on.  V of that step is requested later.
    int v_from = 0;
    uint32_t v_mask = 0;
    const char* v_base = vb;
    __half2 scales_now = __float2half2_rn(0.f), scales_next = scales_now;  // of the next step, and of the one behind it
    auto request_k = [&](uint32_t dst, int meta) {
      scales_now = scales_next;
      if (left > 0) {
        const bool ok = s < end && (uint32_t)slot < n_slots;
        const uint32_t mask = __ballot_sync(0xffffffffu, ok);
        if (mask != C::FULL && s < end && !ok) atomicMax(&g_status, kOutsideStorage);
        if (fresh) {  // the queries of a new run, a line a lane
          const int in = cit % chunks * hpi, line = lane * 64;
          if (line < min(hpi, group - in) * D)
            touch(reinterpret_cast<const T*>(p.q) + (int64_t)cb * p.q_stride_b + (int64_t)(hk * group + in + line / D) * p.q_stride_h + line % D);
        }
        v_from = ok ? slot : 0;
        v_mask = mask;
        v_base = vb;
        copy_rows(dst, kb, v_from, k_row, mask);
        if constexpr (C::I8) {  // two-byte loads, read a step later
          if (ok) {
            scales_next.x = reinterpret_cast<const __half*>(p.k_scale)[(int64_t)slot * p.ks_stride_t + (int64_t)hk * p.ks_stride_h];
            scales_next.y = reinterpret_cast<const __half*>(p.v_scale)[(int64_t)slot * p.vs_stride_t + (int64_t)hk * p.vs_stride_h];
          } else {
            scales_next = __float2half2_rn(0.f);
          }
        }
        const bool last = ct + 1 == cnt || left == 1;
        if (lane == 0) {
          ring[warp][meta] = Step{mask, fresh | (last ? 2 : 0)};
          if (fresh || last) ring_run[warp][meta] = Run{seq_first + (int64_t)cit * cnt, cb, cit, hk, cnt, tokens};
        }
        fresh = last;
        if (--left > 0) {
          s += tile;
          if (++ct == cnt) {
            ct = 0;
            if (++cit == n_it) {
              cit = 0;
              seq_first += (int64_t)cnt * n_it;
              do { cnt = tiles_of(++cb); } while (cnt == 0);
              enter_sequence();
            }
            enter_item();
          }
          slot = s < end ? page[s] : 0;
        }
      } else {
        v_mask = 0;
        v_base = nullptr;
      }
      copies_commit();
    };
    auto request_v = [&](uint32_t dst) {
      if (v_base != nullptr) copy_rows(dst, v_base, v_from, v_row, v_mask);
      copies_commit();
    };

    // Four slots: K and V of the present step and of the next one; those of the one behind it take the place of the
    // present ones as soon as the scores and the sums are there.
    request_k(my_ring, 0);
    request_v(my_ring + C::SLOT_BYTES);
    request_k(my_ring + 2 * C::SLOT_BYTES, 1);
    request_v(my_ring + 3 * C::SLOT_BYTES);

    const float c = (p.sm_scale != 0.f ? p.sm_scale : rsqrtf((float)D)) * kLog2e;
    uint32_t q[NT][D / 16][2], q_low[NT][C::I8 ? D / 32 : 1][2];
    float cq[NT][2], m[NT][2], l[NT][2], acc[D / 16][NT][4];
    const int steps = (int)(hi - lo);
    for (int step = 0; step < steps; ++step) {
      if constexpr (C::I8)
        if (lane < TOK) sm_scale[warp][lane] = scales_now;
      const uint32_t slot_k = my_ring + (step & 1) * 2 * C::SLOT_BYTES, slot_v = slot_k + C::SLOT_BYTES;
      copies_wait<3>();
      __syncwarp();
      const Step now = ring[warp][step % META];
      if (now.flags & 1) {
        const Run run = ring_run[warp][step % META];
        const int in = run.it % chunks * hpi, h0 = run.hk * group + in, heads = min(hpi, group - in);
        // queries as B operand: lane (head g, dims 2 c4, 2 c4 + 1 and + 8 of every 16; bytes: dims 4 c4 .. + 3 and + 16 of
        // every 32, high bytes in the even entries, middle ones in the odd, low ones in q_low)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const bool on = 8 * j + g < heads;
          const T* qr = reinterpret_cast<const T*>(p.q) + (int64_t)run.b * p.q_stride_b + (int64_t)(h0 + (on ? 8 * j + g : 0)) * p.q_stride_h;
          float amax = 0.f;
          bool finite = true;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = C::I8 ? 32 * (k / 2) + 2 * (k & 1) + 16 * e + 4 * c4 : 16 * k + 2 * c4 + 8 * e;
              q[j][k][e] = on ? *reinterpret_cast<const uint32_t*>(qr + d) : 0u;
              if constexpr (C::I8) {
                const float2 f = two<T>(q[j][k][e]);
                amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                finite &= fabsf(f.x) < INFINITY && fabsf(f.y) < INFINITY;
              }
            }
          }
          if constexpr (C::I8) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            finite = (__ballot_sync(0xffffffffu, finite) >> (4 * g) & 15) == 15;
            // (the exponent of the largest; below 2^-100 all is as good as 0)
            const int e = amax > 0.f && finite ? max(-100, (__float_as_int(amax) >> 23) - 127) : 0;
            const float up = power_of_two(22 - e);
#pragma unroll
            for (int k = 0; k < D / 16; k += 2)
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                const float2 f0 = two<T>(q[j][k][t]), f1 = two<T>(q[j][k + 1][t]);
                const int v[4] = {__float2int_rn(f0.x * up), __float2int_rn(f0.y * up), __float2int_rn(f1.x * up), __float2int_rn(f1.y * up)};
                uint32_t high = 0, mid = 0, low = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  high |= ((uint32_t)(v[i] >> 16) & 255u) << (8 * i);
                  mid |= ((uint32_t)(v[i] >> 8) & 255u) << (8 * i);
                  low |= ((uint32_t)v[i] & 255u) << (8 * i);
                }
                q[j][k][t] = high;
                q[j][k + 1][t] = mid;
                q_low[j][k / 2][t] = low;
              }
            // the factor of head 8 j + g; this lane's columns are heads 2 c4 and 2 c4 + 1
            const float f = finite ? c * power_of_two(e - 22) : NAN;
            cq[j][0] = __shfl_sync(0xffffffffu, f, 8 * c4);
            cq[j][1] = __shfl_sync(0xffffffffu, f, 8 * c4 + 4);
          }
          m[j][0] = m[j][1] = -FLT_MAX;
          l[j][0] = l[j][1] = 0.f;
#pragma unroll
          for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][j][i] = 0.f;
        }
      }

      // ---- scores: rows tokens, columns heads.  Two or more sums at a time: a product waits 22 cycles for the one before.
      float z[C::SUBS][NT][4];
      const uint32_t k_base = slot_k + C::at(lane & 15, lane >> 4);
      if constexpr (!C::I8) {
        constexpr int SUMS = C::SUBS == 1 ? 2 : 1;
        float part[C::SUBS][NT][SUMS][4];
#pragma unroll
        for (int i = 0; i < C::SUBS * NT * SUMS * 4; ++i) (&part[0][0][0][0])[i] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int u = 0; u < C::SUBS; ++u) {
            uint32_t a[4];
            ldmatrix4(a, C::skip(k_base + u * 16 * C::PITCH, 2 * k));
#pragma unroll
            for (int j = 0; j < NT; ++j) mma<M>(part[u][j][k % SUMS], a, q[j][k][0], q[j][k][1]);
          }
#pragma unroll
        for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) z[u][j][i] = SUMS == 1 ? part[u][j][0][i] : part[u][j][0][i] + part[u][j][SUMS - 1][i];
      } else {
        int32_t high[C::SUBS][NT][4], mid[C::SUBS][NT][4], low[C::SUBS][NT][4];
#pragma unroll
        for (int i = 0; i < C::SUBS * NT * 4; ++i) (&high[0][0][0])[i] = (&mid[0][0][0])[i] = (&low[0][0][0])[i] = 0;
        // the low bytes in a loop of their own (8 sequences of up to 32768: 69 us; in the one below, where three sums wait for one load,
        // 77), in front of the others (behind them the registers of rows of 256 do not reach)
#pragma unroll
        for (int k = 0; k < D / 16; k += 2)
#pragma unroll
          for (int u = 0; u < C::SUBS; ++u) {
            uint32_t a[4];
            ldmatrix4(a, C::skip(k_base + u * 16 * C::PITCH, k));
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_s8_u8(low[u][j], a, q_low[j][k / 2][0], q_low[j][k / 2][1]);
          }
#pragma unroll
        for (int k = 0; k < D / 16; k += 2)
#pragma unroll
          for (int u = 0; u < C::SUBS; ++u) {
            uint32_t a[4];
            ldmatrix4(a, C::skip(k_base + u * 16 * C::PITCH, k));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma_s8_s8(high[u][j], a, q[j][k][0], q[j][k][1]);
              mma_s8_u8(mid[u][j], a, q[j][k + 1][0], q[j][k + 1][1]);
            }
          }
#pragma unroll
        for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)  // (each sum is below 2^23)
              z[u][j][i] = fmaf((float)high[u][j][i], 65536.f, (float)(mid[u][j][i] * 256 + low[u][j][i]));
      }

      __syncwarp();
      request_k(slot_k, (step + 2) % META);

      // ---- weights
      float sv[C::SUBS][2], lsv[C::SUBS][2], top[NT][2];
#pragma unroll
      for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sk = 1.f;
          if constexpr (C::I8) {
            const float2 f = __half22float2(sm_scale[warp][16 * u + g + 8 * e]);
            sk = f.x;
            sv[u][e] = f.y;
            lsv[u][e] = __log2f(fmaxf(fabsf(f.y), 5.9604644775390625e-8f));  // (no less than f16's smallest: a scale of 0 is none)
          }
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) z[u][j][2 * e + i] *= C::I8 ? cq[j][i] * sk : c;
        }
      if (now.mask != C::FULL) {
#pragma unroll
        for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((now.mask >> (16 * u + g + 8 * (i >> 1))) & 1))
#pragma unroll
              for (int j = 0; j < NT; ++j) z[u][j][i] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[j][i] = m[j][i];
#pragma unroll
          for (int u = 0; u < C::SUBS; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) top[j][i] = fmaxf(top[j][i], C::I8 ? z[u][j][2 * e + i] + lsv[u][e] : z[u][j][2 * e + i]);
        }
      bool moved = false;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) top[j][i] = fmaxf(top[j][i], __shfl_xor_sync(0xffffffffu, top[j][i], o));
          moved |= top[j][i] > m[j][i] + C::SLACK;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float keep = ex2(m[j][i] - top[j][i]);
            m[j][i] = top[j][i];
            l[j][i] *= keep;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
              acc[t][j][i] *= keep;
              acc[t][j][2 + i] *= keep;
            }
          }
      }
      copies_wait<3>();
      __syncwarp();
#pragma unroll
      for (int u = 0; u < C::SUBS; ++u) {
        uint32_t hi_b[NT][2], lo_b[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              w[i] = ex2(z[u][j][2 * e + i] - (m[j][i] - C::LIFT));
              l[j][i] += w[i];
              if (C::I8) w[i] *= sv[u][e];
            }
            const uint32_t h = both<M>(w[0], w[1]);
            const float2 f = two<M>(h);
            hi_b[j][e] = turned(h);
            lo_b[j][e] = turned(both<M>(w[0] - f.x, w[1] - f.y));
          }
        // ---- values: rows dims, columns heads
        if constexpr (!C::I8) {
          const uint32_t base = slot_v + C::at(16 * u + (lane & 7) + 8 * (lane >> 4), (lane >> 3) & 1);
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            uint32_t a[4];
            ldmatrix4_trans(a, C::skip(base, 2 * t));
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma<M>(acc[t][j], a, hi_b[j][0], hi_b[j][1]);
              mma<M>(acc[t][j], a, lo_b[j][0], lo_b[j][1]);
            }
          }
        } else {
          // a transposed pair of bytes is two dims of one token: row g of the product is dim 2 g, row g + 8 dim 2 g + 1
          const uint32_t base = slot_v + C::at(16 * u + (lane & 7) + 8 * ((lane >> 3) & 1), lane >> 4);
#pragma unroll
          for (int t = 0; t < D / 16; t += 2) {
            uint32_t r[4];
            ldmatrix4_trans(r, C::skip(base, t));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t x = r[2 * e] ^ 0x80808080u, y = r[2 * e + 1] ^ 0x80808080u;
              const uint32_t a[4] = {bytes_to_f16<0x4240>(x), bytes_to_f16<0x4341>(x), bytes_to_f16<0x4240>(y), bytes_to_f16<0x4341>(y)};
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma<M>(acc[t + e][j], a, hi_b[j][0], hi_b[j][1]);
                mma<M>(acc[t + e][j], a, lo_b[j][0], lo_b[j][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      request_v(slot_v);

      if (now.flags & 2) {
        // ---- the end of a run: this warp's partial sums, or the result where no other warp has tokens
        const Run run = ring_run[warp][step % META];
        const int in = run.it % chunks * hpi, h0 = run.hk * group + in, heads = min(hpi, group - in);
        const int c0 = share_owner(run.item_first, total, shares), c1 = share_owner(run.item_first + run.tiles - 1, total, shares);
        const int64_t item = (int64_t)run.b * n_it + run.it;
        const bool alone = items.hw == kWarps ? c0 == c1 : run.tokens <= TOK;  // no other warp has tokens of these heads
        // (items and shares only grow: no two runs have the same sum)
        const int64_t at = ((item + share) * kWarps + warp) * hpi;
        if (c0 == share && threadIdx.x == 0) part.items[item] = make_int2((int)(item + c0), alone ? 0 : c1 - c0 + 1);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l[j][i] += __shfl_xor_sync(0xffffffffu, l[j][i], o);
            const int h = 8 * j + 2 * c4 + i;
            if (h >= heads || (alone && part_of_warp > 0)) continue;
            if (alone) {
              T* out = reinterpret_cast<T*>(p.out) + (int64_t)run.b * p.out_stride_b + (int64_t)(h0 + h) * p.out_stride_h;
              const float f = l[j][i] == 0.f ? 0.f : 1.f / l[j][i];
#pragma unroll
              for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  out[16 * t + (C::I8 ? 2 * g + e : g + 8 * e)] = narrow<T>(l[j][i] == 0.f ? 0.f : acc[t][j][2 * e + i] * f);
              if (g == 0 && p.lse != nullptr)
                p.lse[(int64_t)run.b * p.n_q_heads + h0 + h] = l[j][i] == 0.f ? -INFINITY : (m[j][i] - C::LIFT + log2f(l[j][i])) * kLn2;
            } else {
              float* o = part.o + (at + h) * D;  // (relative to the same maximum as the sum)
#pragma unroll
              for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) o[16 * t + (C::I8 ? 2 * g + e : g + 8 * e)] = acc[t][j][2 * e + i];
              if (g == 0) part.ml[at + h] = make_float2(m[j][i] - C::LIFT, l[j][i]);
            }
          }
      }
    }
  }

  // ---- sequences without positions
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (tiles_of(b) > 0) continue;
    if (threadIdx.x == 0) span_of(p, b);  // (records why)
    for (int i = threadIdx.x; i < p.n_q_heads * D; i += kThreads) {
      const int h = i / D, d = i - h * D;
      reinterpret_cast<T*>(p.out)[(int64_t)b * p.out_stride_b + (int64_t)h * p.out_stride_h + d] = narrow<T>(0.f);
      if (d == 0 && p.lse != nullptr) p.lse[(int64_t)b * p.n_q_heads + h] = -INFINITY;
    }
  }
}

// Joins the partial sums of one (sequence, query head): a warp takes every W-th of them, a lane D / 32 dims, four partials'
// loads in flight; the warps' sums meet in shared memory.  Always the same order.
template <typename T, int D, int W>
__global__ void __launch_bounds__(W * 32)
paged_merge_kernel(const __grid_constant__ WsvdPagedDecodeParams p, const Partials part, const Items items) {
  constexpr int E = D / 32;
  // (It does not let the next kernel in: that one's CTAs would be set up beside these, unevenly, and its shares are equal.
  // What is read before the wait has been there before the decode kernel began.)
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int req = p.b_req_idx[b], len = p.b_seq_len[b];
  before_this();
  if (len <= 0 || p.max_len <= 0 || req < 0 || req >= p.n_req) return;
  const int hk = h / items.group, in = h - hk * items.group, hw = items.hw, splits = kWarps / hw;
  const int2 info = part.items[((int64_t)b * (p.n_kv_heads / hw) + hk / hw) * items.chunks + in / items.hpi];
  const int parts = info.y * splits;
  if (parts == 0) return;
  // part k is that of CTA k / splits of the item, of its warp for this KV head and the tokens' split k % splits
  const int64_t first = ((int64_t)info.x * kWarps + hk % hw) * items.hpi + in % items.hpi;
  float m = -FLT_MAX, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int i0 = warp; i0 < parts; i0 += 4 * W) {
    float2 ml[4];
    float v[4][E];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = i0 + i * W;
      const bool on = k < parts;
      const int64_t at = first + (int64_t)(on ? k * hw : 0) * items.hpi;
      ml[i] = on ? part.ml[at] : make_float2(-FLT_MAX, 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] = on ? part.o[at * D + lane + 32 * e] : 0.f;
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);
    const float keep = ex2(m - top);
    l *= keep;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = ex2(ml[i].x - top);
      l = fmaf(ml[i].y, f, l);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(v[i][e], f, o[e]);
    }
    m = top;
  }
  __shared__ float sm_o[W][D];
  __shared__ float2 sm_ml[W];
  if (lane == 0) sm_ml[warp] = make_float2(m, l);
#pragma unroll
  for (int e = 0; e < E; ++e) sm_o[warp][lane + 32 * e] = o[e];
  __syncthreads();
  float top = sm_ml[0].x, sum = 0.f;
#pragma unroll
  for (int w = 1; w < W; ++w) top = fmaxf(top, sm_ml[w].x);
#pragma unroll
  for (int w = 0; w < W; ++w) sum = fmaf(sm_ml[w].y, ex2(sm_ml[w].x - top), sum);
  for (int d = threadIdx.x; d < D; d += W * 32) {
    float r = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) r = fmaf(sm_o[w][d], ex2(sm_ml[w].x - top), r);
    reinterpret_cast<T*>(p.out)[(int64_t)b * p.out_stride_b + (int64_t)h * p.out_stride_h + d] = narrow<T>(sum == 0.f ? 0.f : r / sum);
  }
  if (threadIdx.x == 0 && p.lse != nullptr) p.lse[(int64_t)b * p.n_q_heads + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// ---- host side

Items items_of(const WsvdPagedDecodeParams& p) {
  const int group = p.n_q_heads / p.n_kv_heads;
  const int chunks = (group + 15) / 16, hpi = (group + chunks - 1) / chunks;
  const int hw = p.n_kv_heads % 4 == 0 ? 4 : p.n_kv_heads % 2 == 0 ? 2 : 1;
  return {group, hpi, chunks, hpi <= 8 ? 1 : 2, hw};
}
size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }
struct Room {
  size_t o, ml, items, total;
};
Room room_of(const WsvdPagedDecodeParams& p) {
  const Items it = items_of(p);
  const size_t items = (size_t)p.batch * (p.n_kv_heads / it.hw) * it.chunks, ctas = (size_t)kMaxSms * kMaxCtas;
  const size_t rows = (items + (items * kMaxParts < ctas ? items * kMaxParts : ctas)) * kWarps * it.hpi;
  Room r;
  r.o = 0;
  r.ml = r.o + pad256(rows * p.head_dim * sizeof(float));
  r.items = r.ml + pad256(rows * sizeof(float2));
  r.total = r.items + pad256(items * sizeof(int2));
  return r;
}
// Whether the tensor-core kernel takes the call; the rest (other head dimensions, rows off 16 bytes) runs on the kernel for
// any shape, at about a tenth of its speed.
bool fits_tensor_cores(const WsvdPagedDecodeParams& p) {
  const int es = p.cache_dtype == WSVD_I8 ? 1 : 2, unit = 16 / es;
  if (p.head_dim != 64 && p.head_dim != 96 && p.head_dim != 128 && p.head_dim != 256) return false;
  if (((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) != 0) return false;
  if (p.k_stride_t % unit || p.k_stride_h % unit || p.v_stride_t % unit || p.v_stride_h % unit) return false;
  // token strides in bytes are multiplied as 32-bit values
  if (p.k_stride_t < 0 || p.v_stride_t < 0 || p.k_stride_t * es > INT32_MAX || p.v_stride_t * es > INT32_MAX) return false;
  return (reinterpret_cast<uintptr_t>(p.q) & 3) == 0 && p.q_stride_b % 2 == 0 && p.q_stride_h % 2 == 0;
}

template <typename C>
cudaError_t launch_fast(const WsvdPagedDecodeParams& p, const Items& it, const Partials& part, cudaStream_t s) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 0 || device >= kMaxDevices) return cudaErrorInvalidDevice;
  // how many CTAs the GPU holds at once, asked once per device (what is written twice is the same)
  static int resident[kMaxDevices];
  if (resident[device] == 0) {
    e = cudaFuncSetAttribute(paged_decode_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::RING);
    int per_sm = 0, sms = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, paged_decode_kernel<C>, kThreads, C::RING);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return e;
    resident[device] = max(1, min(kMaxSms, sms) * min(per_sm, C::CTAS));
  }
  // a share a CTA, but no more than a merge of one item can take at a time
  const int64_t items = (int64_t)p.batch * (p.n_kv_heads / it.hw) * it.chunks;
  const int tile = C::TOK * kWarps / it.hw;
  const int reach = p.window > 0 && p.window < p.max_len ? p.window : p.max_len;
  int64_t grid = resident[device];
  if (grid > items * kMaxParts) grid = items * kMaxParts;
  const int64_t tiles = items * ((reach + tile - 1) / tile);
  if (grid > tiles) grid = tiles;
  if (grid < 1) grid = 1;
  e = launch_overlapped(paged_decode_kernel<C>, dim3((unsigned)grid), kThreads, (size_t)C::RING, s, 1, p, part, it);
  if (e != cudaSuccess || reach <= C::TOK) return e;  // (one warp an item and head: no partials)
  // An item has about grid / items + 1 CTAs: one round of loads for four warps, else many warps.  (48 sequences in a window: 62 us with
  // four, 72 with sixteen; one sequence of 60000 with one KV head: 29 and 24.)
  const dim3 heads(p.n_q_heads, p.batch);
  if (grid * (kWarps / it.hw) <= 14 * items)
    return launch_overlapped(paged_merge_kernel<typename C::T, C::D, 4>, heads, 4 * 32, 0, s, 1, p, part, it);
  return launch_overlapped(paged_merge_kernel<typename C::T, C::D, 16>, heads, 16 * 32, 0, s, 1, p, part, it);
}

template <typename T, bool I8, int NT>
cudaError_t launch_dims(const WsvdPagedDecodeParams& p, const Items& it, const Partials& part, cudaStream_t s) {
  switch (p.head_dim) {
    case 64: return launch_fast<Cfg<T, I8, 64, NT>>(p, it, part, s);
    case 96: return launch_fast<Cfg<T, I8, 96, NT>>(p, it, part, s);
    case 128: return launch_fast<Cfg<T, I8, 128, NT>>(p, it, part, s);
    default: return launch_fast<Cfg<T, I8, 256, NT>>(p, it, part, s);
  }
}
template <typename T, bool I8>
cudaError_t launch_tensor_cores(const WsvdPagedDecodeParams& p, void* workspace, cudaStream_t s) {
  const Items it = items_of(p);
  const Room r = room_of(p);
  char* w = reinterpret_cast<char*>(workspace);
  const Partials part{reinterpret_cast<float*>(w + r.o), reinterpret_cast<float2*>(w + r.ml), reinterpret_cast<int2*>(w + r.items)};
  return it.nt == 1 ? launch_dims<T, I8, 1>(p, it, part, s) : launch_dims<T, I8, 2>(p, it, part, s);
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
  if (!p || p->batch <= 0 || p->n_q_heads <= 0 || p->n_kv_heads <= 0 || p->n_q_heads % p->n_kv_heads || p->head_dim <= 0) return 0;
  return wsvd::room_of(*p).total;  // (of the tensor-core kernel: whatever the strides, addresses and lengths)
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
  if (p->batch > 65535 || p->n_q_heads > 65535 || p->max_len > wsvd::kMostCounted) return WSVD_ERR_TOO_LARGE;
  if (p->batch == 0) return WSVD_OK;
  if (!p->q || !p->out || !p->b_req_idx || !p->b_seq_len) return WSVD_ERR_NULL_POINTER;
  const bool places = p->n_token_slots > 0 && p->n_req > 0 && p->max_len > 0;  // (else no sequence has positions)
  if (places && (!p->k || !p->v || !p->req_to_token)) return WSVD_ERR_NULL_POINTER;
  if (i8 && places && (!p->k_scale || !p->v_scale)) return WSVD_ERR_BAD_DTYPE;
  const size_t need = wsvd_paged_decode_workspace_bytes(p);
  if (need > 0 && !workspace) return WSVD_ERR_NULL_POINTER;
  if (workspace_bytes < need) return WSVD_ERR_WORKSPACE_TOO_SMALL;
  if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WSVD_ERR_BAD_STRIDE;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  WsvdPagedDecodeParams call = *p;
  if (!places) call.max_len = 0;
  cudaError_t e;
  if (wsvd::fits_tensor_cores(call)) {
    if (call.dtype == WSVD_F16)
      e = i8 ? wsvd::launch_tensor_cores<__half, true>(call, workspace, s) : wsvd::launch_tensor_cores<__half, false>(call, workspace, s);
    else
      e = i8 ? wsvd::launch_tensor_cores<__nv_bfloat16, true>(call, workspace, s)
             : wsvd::launch_tensor_cores<__nv_bfloat16, false>(call, workspace, s);
  } else {
    if (call.dtype == WSVD_F16) i8 ? wsvd::launch_any<__half, int8_t>(call, s) : wsvd::launch_any<__half, __half>(call, s);
    else i8 ? wsvd::launch_any<__nv_bfloat16, int8_t>(call, s) : wsvd::launch_any<__nv_bfloat16, __nv_bfloat16>(call, s);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? WSVD_OK : wsvd::record_cuda_error(e);
}

}  // extern "C"
