// Tokens sorted by expert and back, for experts that are not this library's own: the row order alone, without the
// 128-row tiles, the limit of eight distinct experts per token and the fixed workspace of the MoE block's permute.
//
//   plan      slots (t, j) of topk_idx [N,k] in the order (expert, slot): slot_row[t,j] = offsets[e] + rank of the slot
//             among the slots of e; groups start at multiples of `align`; row_slot is the inverse (-1: no slot)
//   dispatch  xs[slot_row[t,j]] = x[t], other rows zero;            its gradient  dx[t] = sum_j dxs[slot_row[t,j]]
//   combine   out[t] = sum_j w[t,j] * ys[slot_row[t,j]];            its gradients dys[slot_row[t,j]] = w[t,j] * dout[t],
//             dw[t,j] = <ys[slot_row[t,j]], dout[t]>, other rows of dys zero
// A negative index is an empty slot: it has no row, its weight is not read and its dw is 0.  An index >= E is treated
// the same way and raises the plan's status word.  Sums are fp32 in slot order: results do not depend on timing.
#include <type_traits>

#include "tc_common.cuh"

namespace bibo {

// words of the plan buffer: offsets [E+1], counts [E], status, then (16-byte aligned) slot_row [slots], row_slot [rows] and, for
// more slots than one block sorts, scratch: counts [blocks][E], then a flag of each block
__host__ __device__ inline int64_t dp_off_counts(int E) { return E + 1; }
__host__ __device__ inline int64_t dp_off_status(int E) { return 2 * (int64_t)E + 1; }
__host__ __device__ inline int64_t dp_off_slot_row(int E) { return (2 * (int64_t)E + 2 + 3) / 4 * 4; }
__host__ __device__ inline int64_t dp_off_row_slot(int E, int64_t slots) { return dp_off_slot_row(E) + (slots + 3) / 4 * 4; }
inline int64_t dp_rows_cap(int64_t slots, int E, int align) {
  const int64_t groups = slots < E ? slots : E;
  return (slots + groups * (align - 1) + align - 1) / align * align;
}
constexpr int DP_ONE_BLOCK = 8192, DP_MAX_BLOCKS = 256;     // slots that one block sorts; blocks for more
inline int64_t dp_blocks(int64_t slots) {
  if (slots <= DP_ONE_BLOCK) return 0;
  const int64_t b = (slots + 1023) / 1024;
  return b < DP_MAX_BLOCKS ? b : DP_MAX_BLOCKS;
}
inline int64_t dp_off_scratch(int64_t slots, int E, int64_t rows_cap) { return dp_off_row_slot(E, slots) + (rows_cap + 3) / 4 * 4; }
constexpr int DP_MAX_EXPERTS = 1024, DP_MAX_TOP_K = 32, DP_STATUS_INDEX = 2;

// ---- plan: a stable counting sort -------------------------------------------------------------------------------
// Each warp owns a contiguous range of slots and a histogram in shared memory.  A slot's rank among the warp's slots of its
// expert comes from one ballot per index bit; a scan over the block's warps makes it the rank in the block, which waits in
// slot_row.  Up to DP_ONE_BLOCK slots one block does everything.  Above that a first launch ranks inside blocks of >= 1024 slots and
// leaves their counts, and in a second one every block adds up the counts of the blocks below it (L2-resident), the
// offsets, and its ranks.  (One cluster of 16 blocks with the counts exchanged through distributed shared memory took 30 us for
// 196608 slots: the scattered stores of row_slot want more than 16 SMs.)
constexpr int DP_BATCH = 8;        // index loads in flight per lane

struct DpBlock {                   // shared memory of a block
  int32_t *offset, *count, *lower, *hists;      // [E+1], [E], [E], [warps][pitch]
  int pitch;
  __device__ DpBlock(int32_t* sm, int E) : offset(sm), count(sm + E + 1), lower(sm + 2 * E + 1), hists(sm + 3 * E + 1), pitch(E | 1) {}
};
static size_t dp_smem(int E, int threads) { return sizeof(int32_t) * (3 * (size_t)E + 1 + (size_t)(threads / 32) * (E | 1)); }

template <typename I> __device__ __forceinline__ int dp_expert(const I* idx, int64_t s, int64_t end, int E, int* bad) {
  if (s >= end) return -1;
  const int64_t v = (int64_t)idx[s];
  if (v >= E) *bad = 1;
  return v >= 0 && v < E ? (int)v : -1;
}
// ranks of the slots [s0, s1) of this warp inside the warp into slot_row (-1: no slot), and its histogram
template <typename I>
__device__ __forceinline__ void dp_rank(const I* __restrict__ idx, int64_t s0, int64_t s1, int E, int bits, int32_t* hist,
                                        int32_t* __restrict__ slot_row, int* bad) {
  const int lane = threadIdx.x & 31;
  for (int e = lane; e < E; e += 32) hist[e] = 0;
  __syncwarp();
  for (int64_t b0 = s0; b0 < s1; b0 += 32 * DP_BATCH) {
    int ex[DP_BATCH];
#pragma unroll
    for (int i = 0; i < DP_BATCH; ++i) ex[i] = dp_expert(idx, b0 + i * 32 + lane, s1, E, bad);
#pragma unroll
    for (int i = 0; i < DP_BATCH; ++i) {
      if (b0 + i * 32 >= s1) break;          // the whole warp
      const int e = ex[i];
      unsigned same = __ballot_sync(0xffffffffu, e >= 0);
      for (int bit = 0; bit < bits; ++bit) {
        const unsigned one = __ballot_sync(0xffffffffu, (e >> bit) & 1);
        same &= (e >> bit) & 1 ? one : ~one;
      }
      int rank = -1;
      if (e >= 0) rank = hist[e] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (e >= 0 && (same >> lane) == 1u) hist[e] = rank + 1;       // the last lane of the expert
      __syncwarp();
      if (b0 + i * 32 + lane < s1) slot_row[b0 + i * 32 + lane] = rank;
    }
  }
}
// hists: exclusive scan over the warps of the block; count: the block's slots of each expert
__device__ __forceinline__ void dp_scan_warps(const DpBlock& d, int E) {
  const int warps = blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = warp; e < E; e += warps) {
    const int c = lane < warps ? d.hists[(size_t)lane * d.pitch + e] : 0;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
    if (lane < warps) d.hists[(size_t)lane * d.pitch + e] = inc - c;
    if (lane == 31) d.count[e] = inc;
  }
}
// offsets from the counts: exclusive scan of the counts rounded up to `align`; one warp
__device__ __forceinline__ void dp_offsets(const DpBlock& d, int E, int align) {
  const int lane = threadIdx.x & 31;
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    const int c = e < E ? (d.count[e] + align - 1) / align * align : 0;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
    if (e < E) d.offset[e] = carry + inc - c;
    carry += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) d.offset[E] = carry;
}
// rows without a slot: the padding behind each group and everything behind the last group; block `b` of `n`
__device__ __forceinline__ void dp_free_rows(const DpBlock& d, int E, int align, int64_t rows_cap, int b, int n, int32_t* row_slot) {
  const int warps = blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (align > 1)
    for (int e = b * warps + warp; e < E; e += n * warps)
      for (int r = d.offset[e] + d.count[e] + lane; r < d.offset[e + 1]; r += 32) row_slot[r] = -1;
  for (int64_t r = d.offset[E] + (int64_t)b * blockDim.x + threadIdx.x; r < rows_cap; r += (int64_t)n * blockDim.x) row_slot[r] = -1;
}
__device__ __forceinline__ void dp_write_head(const DpBlock& d, int E, int bad, int32_t* plan) {
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    plan[e] = d.offset[e];
    if (e < E) plan[dp_off_counts(E) + e] = d.count[e];
  }
  if (threadIdx.x == 0) plan[dp_off_status(E)] = bad ? DP_STATUS_INDEX : 0;
}

template <typename I>
__global__ void __launch_bounds__(1024)
dispatch_plan_kernel(const I* __restrict__ idx, int64_t slots, int E, int bits, int align, int64_t rows_cap, int32_t* __restrict__ plan) {
  extern __shared__ int32_t sm[];
  __shared__ int bad_s;
  const DpBlock d(sm, E);
  const int warps = blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t* hist = d.hists + (size_t)warp * d.pitch;
  int32_t* slot_row = plan + dp_off_slot_row(E);
  int32_t* row_slot = plan + dp_off_row_slot(E, slots);
  if (threadIdx.x == 0) bad_s = 0;
  __syncthreads();
  const int64_t per = ((slots + warps - 1) / warps + 31) / 32 * 32, s0 = min(slots, warp * per), s1 = min(slots, s0 + per);
  dp_rank(idx, s0, s1, E, bits, hist, slot_row, &bad_s);
  __syncthreads();
  dp_scan_warps(d, E);
  __syncthreads();
  if (warp == 0) dp_offsets(d, E, align);
  __syncthreads();
  dp_write_head(d, E, bad_s, plan);
  dp_free_rows(d, E, align, rows_cap, 0, 1, row_slot);
  for (int64_t s = s0 + lane; s < s1; s += 32) {
    const int rank = slot_row[s];                              // written by this lane
    if (rank < 0) continue;
    const int e = (int)idx[s], row = d.offset[e] + hist[e] + rank;
    slot_row[s] = row;
    row_slot[row] = (int32_t)s;
  }
}

// more slots: ranks inside a block's slots, and its counts in scratch [blocks][E] (flags behind them)
template <typename I>
__global__ void __launch_bounds__(1024)
dispatch_count_kernel(const I* __restrict__ idx, int64_t slots, int64_t per_block, int E, int bits, int32_t* __restrict__ slot_row,
                      int32_t* __restrict__ scratch) {
  extern __shared__ int32_t sm[];
  __shared__ int bad_s;
  const DpBlock d(sm, E);
  const int warps = blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t* hist = d.hists + (size_t)warp * d.pitch;
  if (threadIdx.x == 0) bad_s = 0;
  __syncthreads();
  tc::pdl_launch_next();                     // dispatch_rows_kernel may be set up under this one
  const int64_t b0 = min(slots, blockIdx.x * per_block), b1 = min(slots, b0 + per_block);
  const int64_t per = ((b1 - b0 + warps - 1) / warps + 31) / 32 * 32, s0 = min(b1, b0 + warp * per), s1 = min(b1, s0 + per);
  dp_rank(idx, s0, s1, E, bits, hist, slot_row, &bad_s);
  __syncthreads();
  dp_scan_warps(d, E);
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) scratch[(int64_t)blockIdx.x * E + e] = d.count[e];
  if (threadIdx.x == 0) scratch[(int64_t)gridDim.x * E + blockIdx.x] = bad_s;
  for (int64_t s = s0 + lane; s < s1; s += 32) {
    const int rank = slot_row[s];
    if (rank >= 0) slot_row[s] = rank + hist[(int)idx[s]];
  }
}
// ... and the rows: every block adds up the counts of the blocks below its own
template <typename I>
__global__ void __launch_bounds__(1024)
dispatch_rows_kernel(const I* __restrict__ idx, int64_t slots, int64_t per_block, int E, int align, int64_t rows_cap,
                     const int32_t* __restrict__ scratch, int32_t* __restrict__ plan) {
  extern __shared__ int32_t sm[];
  const DpBlock d(sm, E);
  const int n = gridDim.x, b = blockIdx.x;
  for (int e = threadIdx.x; e < E; e += blockDim.x) d.count[e] = d.lower[e] = 0;
  __syncthreads();
  tc::pdl_wait();
  // a thread adds up one expert over every `groups`-th block, then once into shared memory (whole numbers: any order)
  int ep = 32;
  while (ep < E) ep *= 2;
  const int groups = blockDim.x / ep, e = threadIdx.x % ep;
  if (e < E) {
    int all = 0, low = 0;
#pragma unroll 8
    for (int at = threadIdx.x / ep; at < n; at += groups) {
      const int c = scratch[(int64_t)at * E + e];
      all += c;
      low += at < b ? c : 0;
    }
    atomicAdd(&d.count[e], all);
    atomicAdd(&d.lower[e], low);
  }
  __syncthreads();
  if (threadIdx.x < 32) dp_offsets(d, E, align);
  __syncthreads();
  int32_t* slot_row = plan + dp_off_slot_row(E);
  int32_t* row_slot = plan + dp_off_row_slot(E, slots);
  if (b == 0) {
    // n <= DP_MAX_BLOCKS flags
    dp_write_head(d, E, __syncthreads_or((int)threadIdx.x < n ? scratch[(int64_t)n * E + threadIdx.x] : 0), plan);
  }
  dp_free_rows(d, E, align, rows_cap, b, n, row_slot);
  const int64_t s0 = min(slots, b * per_block), s1 = min(slots, s0 + per_block);
  for (int64_t s = s0 + threadIdx.x; s < s1; s += blockDim.x) {
    const int rank = slot_row[s];
    if (rank < 0) continue;
    const int ex = (int)idx[s], row = d.offset[ex] + d.lower[ex] + rank;
    slot_row[s] = row;
    row_slot[row] = (int32_t)s;
  }
}

// ---- row copies and sums, by the widest access that the rows' alignment allows ------------------------------------
template <int VB> struct RowVec;
template <> struct RowVec<16> { using type = uint4; };
template <> struct RowVec<8> { using type = uint2; };
template <> struct RowVec<4> { using type = uint32_t; };
template <> struct RowVec<2> { using type = uint16_t; };

// VB bytes of T <-> fp32
template <typename T, int VB> struct RowElems;
template <int VB> struct RowElems<float, VB> {
  static constexpr int N = VB / 4;
  static __device__ __forceinline__ void unpack(const typename RowVec<VB>::type& v, float* f) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __uint_as_float(u[i]);
  }
  static __device__ __forceinline__ typename RowVec<VB>::type pack(const float* f) {
    typename RowVec<VB>::type v;
    uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = __float_as_uint(f[i]);
    return v;
  }
};
template <int VB> struct RowElems<__nv_bfloat16, VB> {
  static constexpr int N = VB / 2;
  static __device__ __forceinline__ void unpack(const typename RowVec<VB>::type& v, float* f) {
    const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&v);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __bfloat162float(h[i]);
  }
  static __device__ __forceinline__ typename RowVec<VB>::type pack(const float* f) {
    typename RowVec<VB>::type v;
    __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(&v);
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = __float2bfloat16_rn(f[i]);
    return v;
  }
};

constexpr int DW = 8;          // warps per block
constexpr int DZ_ROWS = 4;     // rows a warp looks at for zeroing (with 16 a tail of empty rows was left to a few hundred warps)

// zeroes the rows of [r0, r0 + DZ_ROWS) that have no slot
template <int VB>
__device__ __forceinline__ void zero_empty_rows(const int32_t* __restrict__ row_slot, int64_t r0, int64_t rows, int chunks,
                                                typename RowVec<VB>::type* __restrict__ dst, int lane) {
  using V = typename RowVec<VB>::type;
  const bool empty = lane < DZ_ROWS && r0 + lane < rows && row_slot[r0 + lane] < 0;
  unsigned todo = __ballot_sync(0xffffffffu, empty);
  const V zero = V{};
  while (todo) {
    const int i = __ffs(todo) - 1;
    todo &= todo - 1;
    V* d = dst + (r0 + i) * chunks;
    for (int c = lane; c < chunks; c += 32) d[c] = zero;
  }
}

// Work items: (token, part of the row) for a warp each, then blocks whose warps zero the rows without a slot.
// A part is `part` accesses of 32 lanes; few tokens are cut into many parts so that the machine is not left to a few warps.

// a token's row is read once and written to its (up to k) rows; eight loads of a lane are in flight before the first store
template <int VB>
__global__ void __launch_bounds__(DW * 32)
dispatch_kernel(const uint8_t* __restrict__ x, int64_t x_stride_bytes, const int32_t* __restrict__ slot_row,
                const int32_t* __restrict__ row_slot, int64_t n_tokens, int top_k, int64_t rows, int chunks, int parts, int part,
                uint8_t* __restrict__ xs) {
  using V = typename RowVec<VB>::type;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * DW + (threadIdx.x >> 5);
  V* dst = reinterpret_cast<V*>(xs);
  const int64_t items = n_tokens * parts;
  if (w >= items) {
    zero_empty_rows<VB>(row_slot, (w - items) * DZ_ROWS, rows, chunks, dst, lane);
    return;
  }
  const int64_t t = parts == 1 ? w : w / parts;
  const int mine = lane < top_k ? slot_row[t * top_k + lane] : -1;
  const V* src = reinterpret_cast<const V*>(x + t * x_stride_bytes);
  const int c_lo = parts == 1 ? 0 : (int)(w % parts) * part * 32, c_hi = min(chunks, c_lo + part * 32);
  const unsigned filled = __ballot_sync(0xffffffffu, mine >= 0);
  if (!filled) return;
  for (int c0 = c_lo + lane; c0 - lane < c_hi; c0 += 256) {
    V v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (c0 + u * 32 < c_hi) v[u] = src[c0 + u * 32];
    for (unsigned todo = filled; todo; todo &= todo - 1) {
      const int r = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
      V* d = dst + (int64_t)r * chunks;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c0 + u * 32 < c_hi) d[c0 + u * 32] = v[u];
    }
  }
}

// weights are fp32 or bf16, whatever the rows are
__device__ __forceinline__ float load_weight(const void* w, int is_bf16, int64_t i) {
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : static_cast<const float*>(w)[i];
}

// The rows of K slots of a token: pointers (nullptr: no row) and weights, in every lane of its warp
template <typename V, int K> struct SlotRows {
  const V* row[K];
  float w[K];
  __device__ __forceinline__ void get(const V* base, int mine, float my_w, int j0, int chunks) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int r = j0 + j < 32 ? __shfl_sync(0xffffffffu, mine, j0 + j) : -1;      // lanes beyond k hold -1
      w[j] = __shfl_sync(0xffffffffu, my_w, (j0 + j) & 31);
      row[j] = r >= 0 ? base + (int64_t)r * chunks : nullptr;
    }
  }
};

// out[t] = sum_j w[t,j] * ys[slot_row[t,j]] (weight == nullptr: 1), slots in order.  All loads of K slots and U accesses are issued
// before the first is used; ONCE: the token's slots are one such round.
template <typename T, int VB, int K, int U, bool ONCE>
__global__ void __launch_bounds__(DW * 32)
dispatch_combine_kernel(const T* __restrict__ ys, const void* __restrict__ weight, int w_bf16,
                        const int32_t* __restrict__ slot_row, int64_t n_tokens, int top_k, int chunks, int parts, int part,
                        T* __restrict__ out) {
  using V = typename RowVec<VB>::type;
  using X = RowElems<T, VB>;
  const int lane = threadIdx.x & 31;
  const int64_t wi = (int64_t)blockIdx.x * DW + (threadIdx.x >> 5);
  const int64_t t = parts == 1 ? wi : wi / parts;
  if (t >= n_tokens) return;
  const int mine = lane < top_k ? slot_row[t * top_k + lane] : -1;
  const float my_w = mine < 0 ? 0.f : weight == nullptr ? 1.f : load_weight(weight, w_bf16, t * top_k + lane);
  const V* src = reinterpret_cast<const V*>(ys);
  V* dst = reinterpret_cast<V*>(out) + t * chunks;
  const int c_lo = parts == 1 ? 0 : (int)(wi % parts) * part * 32, c_hi = min(chunks, c_lo + part * 32);
  SlotRows<V, K> rows;
  if (ONCE) rows.get(src, mine, my_w, 0, chunks);
  // N accesses from column c on: all of them exist, or (N == 1) this lane's may not
  auto block = [&](int c, auto n, bool in) {
    constexpr int N = decltype(n)::value;
    float acc[N][X::N];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < X::N; ++i) acc[u][i] = 0.f;
    for (int j0 = 0; j0 < (ONCE ? 1 : top_k); j0 += K) {
      if (!ONCE) rows.get(src, mine, my_w, j0, chunks);
      V v[N][K];
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (rows.row[j] != nullptr && in)
#pragma unroll
          for (int u = 0; u < N; ++u) v[u][j] = __ldcs(rows.row[j] + c + u * 32);
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (rows.row[j] != nullptr && in)
#pragma unroll
          for (int u = 0; u < N; ++u) {
            float f[X::N];
            X::unpack(v[u][j], f);
#pragma unroll
            for (int i = 0; i < X::N; ++i) acc[u][i] = fmaf(f[i], rows.w[j], acc[u][i]);
          }
    }
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (in) dst[c + u * 32] = X::pack(acc[u]);
  };
  int c = c_lo;
  for (; c + 32 * U <= c_hi; c += 32 * U) block(c + lane, std::integral_constant<int, U>(), true);
  if constexpr (U > 2)
    for (; c + 64 <= c_hi; c += 64) block(c + lane, std::integral_constant<int, 2>(), true);
  for (; c < c_hi; c += 32) block(c + lane, std::integral_constant<int, 1>(), c + lane < c_hi);
}

// dys rows and dw of a token's slots, WPT warps per token (more for few tokens) that share its columns; blocks behind the tokens'
// zero the rows of dys without a slot
template <typename T, int VB, int K, int WPT, int U>
__global__ void __launch_bounds__(DW * 32)
dispatch_combine_bwd_kernel(const T* __restrict__ dout, int64_t dout_stride, const T* __restrict__ ys,
                            const void* __restrict__ weight, int w_bf16, const int32_t* __restrict__ slot_row,
                            const int32_t* __restrict__ row_slot, int64_t n_tokens, int top_k, int64_t rows_, int chunks,
                            int64_t token_blocks, T* __restrict__ dys, void* __restrict__ dweight) {
  using V = typename RowVec<VB>::type;
  using X = RowElems<T, VB>;
  __shared__ float red[DW][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V* dst = reinterpret_cast<V*>(dys);
  if ((int64_t)blockIdx.x >= token_blocks) {
    zero_empty_rows<VB>(row_slot, (((int64_t)blockIdx.x - token_blocks) * DW + warp) * DZ_ROWS, rows_, chunks, dst, lane);
    return;
  }
  const int64_t t = (int64_t)blockIdx.x * (DW / WPT) + warp / WPT;
  const bool in = t < n_tokens;
  const V* g = reinterpret_cast<const V*>(dout + t * dout_stride);
  const V* src = reinterpret_cast<const V*>(ys);
  const int mine = in && lane < top_k ? slot_row[t * top_k + lane] : -1;
  const float my_w = mine < 0 ? 0.f : weight == nullptr ? 1.f : load_weight(weight, w_bf16, t * top_k + lane);
  const bool want = dweight != nullptr;
  float my_dw = 0.f;
  if (__any_sync(0xffffffffu, mine >= 0)) {
    for (int j0 = 0; j0 < top_k; j0 += K) {
      SlotRows<V, K> rows;
      rows.get(src, mine, my_w, j0, chunks);
      float dot[K];
#pragma unroll
      for (int j = 0; j < K; ++j) dot[j] = 0.f;
      // N accesses, 32 * WPT columns apart, from column c on
      auto block = [&](int c, auto n) {
        constexpr int N = decltype(n)::value;
        V gv[N], v[N][K];
#pragma unroll
        for (int u = 0; u < N; ++u) gv[u] = g[c + u * 32 * WPT];
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (want && rows.row[j] != nullptr)
#pragma unroll
            for (int u = 0; u < N; ++u) v[u][j] = __ldcs(rows.row[j] + c + u * 32 * WPT);
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (rows.row[j] != nullptr) {
            V* d = dst + (rows.row[j] - src);
            // of the N accesses, so that a lane's chain has a term per block and not per element (dw of 6000 x 8192 fp32: error 1.7e-7
            // in place of 3.0e-7, the time is the same)
            float part = 0.f;
#pragma unroll
            for (int u = 0; u < N; ++u) {
              float gf[X::N], f[X::N];
              X::unpack(gv[u], gf);
              if (want) {
                X::unpack(v[u][j], f);
#pragma unroll
                for (int i = 0; i < X::N; ++i) part = fmaf(gf[i], f[i], part);
              }
#pragma unroll
              for (int i = 0; i < X::N; ++i) f[i] = gf[i] * rows.w[j];
              d[c + u * 32 * WPT] = X::pack(f);
            }
            dot[j] += part;
          }
      };
      int c = (warp % WPT) * 32 + lane;
      for (; c + (U - 1) * 32 * WPT < chunks; c += U * 32 * WPT) block(c, std::integral_constant<int, U>());
      if (U > 1)
        for (; c < chunks; c += 32 * WPT) block(c, std::integral_constant<int, 1>());
      if (want) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
          if (lane == j0 + j) my_dw = dot[j];
        }
      }
    }
  }
  if (!want) return;
  if (WPT > 1) {
    red[warp][lane] = my_dw;
    __syncthreads();
    if (warp % WPT != 0) return;
    my_dw = 0.f;
#pragma unroll
    for (int i = 0; i < WPT; ++i) my_dw += red[warp + i][lane];
  }
  if (in && lane < top_k) {
    if (w_bf16) static_cast<__nv_bfloat16*>(dweight)[t * top_k + lane] = __float2bfloat16_rn(my_dw);
    else static_cast<float*>(dweight)[t * top_k + lane] = my_dw;
  }
}

// the widest access that all the rows allow
static int row_vec_bytes(int64_t row_bytes, int64_t stride_bytes, const void* a, const void* b, const void* c) {
  const uintptr_t all = (uintptr_t)row_bytes | (uintptr_t)stride_bytes | reinterpret_cast<uintptr_t>(a) |
                        reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c);
  return (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : (all & 3) == 0 ? 4 : 2;
}
static int dispatch_check(const char* what, int64_t n_tokens, int hidden, int n_experts, int top_k, int align, int dtype) {
  if (dtype != BIBO_F32 && dtype != BIBO_BF16) return fail(BIBO_ERR_ARG, "%s: dtype=%d", what, dtype);
  if (hidden < 1 || hidden > (1 << 24)) return fail(BIBO_ERR_UNSUPPORTED, "%s: hidden=%d", what, hidden);
  if (n_experts < 1 || n_experts > DP_MAX_EXPERTS) return fail(BIBO_ERR_UNSUPPORTED, "%s: n_experts=%d (1..%d)", what, n_experts, DP_MAX_EXPERTS);
  if (top_k < 1 || top_k > DP_MAX_TOP_K) return fail(BIBO_ERR_UNSUPPORTED, "%s: top_k=%d (1..%d)", what, top_k, DP_MAX_TOP_K);
  if (align < 1 || align > 1024) return fail(BIBO_ERR_UNSUPPORTED, "%s: align=%d (1..1024)", what, align);
  if (n_tokens < 0 || n_tokens > (1ll << 30) / top_k)
    return fail(BIBO_ERR_UNSUPPORTED, "%s: %lld tokens of %d slots", what, (long long)n_tokens, top_k);
  return BIBO_OK;
}
static unsigned dispatch_grid(int64_t warps) { return (unsigned)((warps + DW - 1) / DW); }
// parts a row is cut into, and their size in accesses of a warp: enough warps for every SM to have 64, where the row allows it
// (5003 tokens x 3 slots x 1153 fp32 combine: 24.2 us with the 34 warps an SM that the tokens make)
static int row_parts(int64_t n_tokens, int chunks, int* part) {
  const int steps = (chunks + 31) / 32;
  const int64_t want = (64 * (int64_t)sm_count() + n_tokens - 1) / n_tokens;
  const int parts = want < steps ? (int)want : steps;
  *part = (steps + parts - 1) / parts;
  return (steps + *part - 1) / *part;
}

template <typename I>
static int plan_launch(const void* idx_, int64_t slots, int E, int align, int32_t* plan, cudaStream_t st) {
  static DeviceOnce once;
  const int rc = once.get([&](int*) {
    BIBO_CUDA(cudaFuncSetAttribute(dispatch_plan_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dp_smem(DP_MAX_EXPERTS, 1024)));
    BIBO_CUDA(cudaFuncSetAttribute(dispatch_count_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dp_smem(DP_MAX_EXPERTS, 1024)));
    return (int)BIBO_OK;
  });
  if (rc) return rc;
  const I* idx = static_cast<const I*>(idx_);
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  const int64_t cap = dp_rows_cap(slots, E, align);
  const int blocks = (int)dp_blocks(slots);
  if (blocks == 0) {
    const int threads = slots <= 1024 ? 256 : 1024;
    dispatch_plan_kernel<I><<<1, threads, dp_smem(E, threads), st>>>(idx, slots, E, bits, align, cap, plan);
    BIBO_CHECK_LAUNCH("dispatch_plan_kernel");
    return BIBO_OK;
  }
  const int64_t per = (slots + blocks - 1) / blocks;
  int32_t* scratch = plan + dp_off_scratch(slots, E, cap);
  dispatch_count_kernel<I><<<blocks, 1024, dp_smem(E, 1024), st>>>(idx, slots, per, E, bits, plan + dp_off_slot_row(E), scratch);
  BIBO_CHECK_LAUNCH("dispatch_count_kernel");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(1024);
  cfg.dynamicSmemBytes = dp_smem(E, 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BIBO_CUDA(cudaLaunchKernelEx(&cfg, dispatch_rows_kernel<I>, idx, slots, per, E, align, cap, (const int32_t*)scratch, plan));
  BIBO_CHECK_LAUNCH("dispatch_rows_kernel");
  return BIBO_OK;
}

}  // namespace bibo

using namespace bibo;

extern "C" int64_t bibo_moe_dispatch_rows_cap(int64_t n_tokens, int top_k, int n_experts, int align) {
  return dispatch_check("dispatch_rows_cap", n_tokens, 1, n_experts, top_k, align, BIBO_F32) ? -1
                                                                                           : dp_rows_cap(n_tokens * top_k, n_experts, align);
}
extern "C" int64_t bibo_moe_dispatch_plan_words(int64_t n_tokens, int top_k, int n_experts, int align) {
  if (dispatch_check("dispatch_plan_words", n_tokens, 1, n_experts, top_k, align, BIBO_F32)) return -1;
  const int64_t slots = n_tokens * top_k;
  return dp_off_scratch(slots, n_experts, dp_rows_cap(slots, n_experts, align)) + dp_blocks(slots) * (n_experts + 1);
}
extern "C" int64_t bibo_moe_dispatch_off_slot_row(int n_experts) { return dp_off_slot_row(n_experts); }
extern "C" int64_t bibo_moe_dispatch_off_row_slot(int64_t n_tokens, int top_k, int n_experts) {
  return dp_off_row_slot(n_experts, n_tokens * top_k);
}

extern "C" int bibo_moe_dispatch_plan(const void* topk_idx, int idx_bytes, int64_t n_tokens, int top_k, int n_experts, int align,
                                      int32_t* plan, void* stream) {
  const int rc = dispatch_check("dispatch_plan", n_tokens, 1, n_experts, top_k, align, BIBO_F32);
  if (rc) return rc;
  if (idx_bytes != 4 && idx_bytes != 8) return fail(BIBO_ERR_ARG, "dispatch_plan: indices of %d bytes", idx_bytes);
  if (!plan || (!topk_idx && n_tokens > 0)) return fail(BIBO_ERR_ARG, "dispatch_plan: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return idx_bytes == 4 ? plan_launch<int32_t>(topk_idx, n_tokens * top_k, n_experts, align, plan, st)
                        : plan_launch<int64_t>(topk_idx, n_tokens * top_k, n_experts, align, plan, st);
}

extern "C" int bibo_moe_dispatch_fwd(const void* x, int64_t x_stride, const int32_t* plan, int64_t n_tokens, int hidden,
                                     int top_k, int n_experts, int align, int dtype, void* xs, void* stream) {
  const int rc = dispatch_check("dispatch_fwd", n_tokens, hidden, n_experts, top_k, align, dtype);
  if (rc) return rc;
  if (n_tokens == 0) return BIBO_OK;
  if (!x || !plan || !xs) return fail(BIBO_ERR_ARG, "dispatch_fwd: null pointer");
  if (n_tokens > 1 && x_stride < hidden) return fail(BIBO_ERR_ARG, "dispatch_fwd: row stride %lld below hidden=%d", (long long)x_stride, hidden);
  const int size = dtype == BIBO_F32 ? 4 : 2;
  const int64_t slots = n_tokens * top_k, rows = dp_rows_cap(slots, n_experts, align);
  const int32_t* slot_row = plan + dp_off_slot_row(n_experts);
  const int32_t* row_slot = plan + dp_off_row_slot(n_experts, slots);
  const int row_bytes = hidden * size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int vb = row_vec_bytes(row_bytes, n_tokens > 1 ? x_stride * size : 0, x, xs, nullptr);
  const int chunks = row_bytes / vb;
  int part;
  const int parts = row_parts(n_tokens, chunks, &part);
  const unsigned grid = dispatch_grid(n_tokens * parts + (rows + DZ_ROWS - 1) / DZ_ROWS);
#define BIBO_DISPATCH_CASE(VB)                                                                                              \
  case VB:                                                                                                                  \
    dispatch_kernel<VB><<<grid, DW * 32, 0, st>>>(static_cast<const uint8_t*>(x), x_stride * size, slot_row, row_slot,      \
                                                  n_tokens, top_k, rows, chunks, parts, part, static_cast<uint8_t*>(xs));   \
    break;
  switch (vb) {
    BIBO_DISPATCH_CASE(16) BIBO_DISPATCH_CASE(8) BIBO_DISPATCH_CASE(4) BIBO_DISPATCH_CASE(2)
  }
#undef BIBO_DISPATCH_CASE
  BIBO_CHECK_LAUNCH("dispatch_kernel");
  return BIBO_OK;
}

template <typename T, int VB>
static void combine_v(const void* ys, const void* weight, int w_bf16, const int32_t* slot_row, int64_t n_tokens, int top_k,
                      int hidden, void* out, cudaStream_t st) {
  const int chunks = hidden / RowElems<T, VB>::N;
  int part;
  const int parts = row_parts(n_tokens, chunks, &part);
  const unsigned grid = dispatch_grid(n_tokens * parts);
#define BIBO_COMBINE(K, U, ONCE)                                                                                            \
  dispatch_combine_kernel<T, VB, K, U, ONCE><<<grid, DW * 32, 0, st>>>(static_cast<const T*>(ys), weight, w_bf16, slot_row, n_tokens, \
                                                                 top_k, chunks, parts, part, static_cast<T*>(out))
  constexpr int M = VB == 16 ? 1 : 4;            // narrow accesses: more of them in flight
  if (top_k == 1) BIBO_COMBINE(1, 4 * M, true);
  else if (top_k == 2) BIBO_COMBINE(2, 4 * M, true);
  else if (top_k == 3) BIBO_COMBINE(3, 2 * M, true);
  else if (top_k == 4) BIBO_COMBINE(4, 2 * M, true);
  else if (top_k <= 6) BIBO_COMBINE(6, 2 * M, true);
  else if (top_k <= 8) BIBO_COMBINE(8, 2 * M, true);
  else BIBO_COMBINE(8, 2 * M, false);
#undef BIBO_COMBINE
}
template <typename T>
static int combine_t(const void* ys, const void* weight, int w_bf16, const int32_t* slot_row, int64_t n_tokens, int top_k,
                     int hidden, void* out, cudaStream_t st) {
  const int vb = row_vec_bytes((int64_t)hidden * sizeof(T), 0, ys, out, nullptr);
#define BIBO_DISPATCH_CASE(VB)                                                                                               \
  if constexpr (VB >= (int)sizeof(T))                                                                                        \
    if (vb == VB) combine_v<T, VB>(ys, weight, w_bf16, slot_row, n_tokens, top_k, hidden, out, st);
  BIBO_DISPATCH_CASE(16) BIBO_DISPATCH_CASE(8) BIBO_DISPATCH_CASE(4) BIBO_DISPATCH_CASE(2)
#undef BIBO_DISPATCH_CASE
  BIBO_CHECK_LAUNCH("dispatch_combine_kernel");
  return BIBO_OK;
}

extern "C" int bibo_moe_dispatch_combine_fwd(const void* ys, const void* topk_w, int w_dtype, const int32_t* plan,
                                             int64_t n_tokens, int hidden, int top_k, int n_experts, int align, int dtype,
                                             void* out, void* stream) {
  const int rc = dispatch_check("dispatch_combine_fwd", n_tokens, hidden, n_experts, top_k, align, dtype);
  if (rc) return rc;
  if (w_dtype != BIBO_F32 && w_dtype != BIBO_BF16) return fail(BIBO_ERR_ARG, "dispatch_combine_fwd: weight dtype=%d", w_dtype);
  if (n_tokens == 0) return BIBO_OK;
  if (!ys || !plan || !out) return fail(BIBO_ERR_ARG, "dispatch_combine_fwd: null pointer");
  const int32_t* slot_row = plan + dp_off_slot_row(n_experts);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int wb = w_dtype == BIBO_BF16;
  return dtype == BIBO_F32 ? combine_t<float>(ys, topk_w, wb, slot_row, n_tokens, top_k, hidden, out, st)
                           : combine_t<__nv_bfloat16>(ys, topk_w, wb, slot_row, n_tokens, top_k, hidden, out, st);
}

template <typename T, int VB>
static void combine_bwd_v(const void* dout, int64_t dout_stride, const void* ys, const void* weight, int w_bf16,
                          const int32_t* slot_row, const int32_t* row_slot, int64_t n_tokens, int top_k, int64_t rows, int hidden,
                          void* dys, void* dweight, cudaStream_t st) {
  const int chunks = hidden / RowElems<T, VB>::N;
  // warps per token: enough for 32 an SM
  const int64_t want = 32 * (int64_t)sm_count();
  const int wpt = n_tokens >= want ? 1 : 4 * n_tokens >= want ? 4 : DW;
  const int64_t token_blocks = (n_tokens * wpt + DW - 1) / DW;
  const unsigned grid = (unsigned)token_blocks + dispatch_grid((rows + DZ_ROWS - 1) / DZ_ROWS);
  constexpr int M = VB == 16 ? 1 : 4;            // narrow accesses: more of them in flight
#define BIBO_COMBINE_W(K, WPT)                                                                                               \
  dispatch_combine_bwd_kernel<T, VB, K, WPT, M><<<grid, DW * 32, 0, st>>>(static_cast<const T*>(dout), dout_stride,             \
                                                                       static_cast<const T*>(ys), weight, w_bf16, slot_row,  \
                                                                       row_slot, n_tokens, top_k, rows, chunks, token_blocks, \
                                                                       static_cast<T*>(dys), dweight)
#define BIBO_COMBINE(K)                      \
  do {                                       \
    if (wpt == 1) BIBO_COMBINE_W(K, 1);      \
    else if (wpt == 4) BIBO_COMBINE_W(K, 4); \
    else BIBO_COMBINE_W(K, DW);              \
  } while (0)
  if (top_k == 1) BIBO_COMBINE(1);
  else if (top_k == 2) BIBO_COMBINE(2);
  else if (top_k == 3) BIBO_COMBINE(3);
  else if (top_k == 4) BIBO_COMBINE(4);
  else if (top_k <= 6) BIBO_COMBINE(6);
  else BIBO_COMBINE(8);
#undef BIBO_COMBINE_W
#undef BIBO_COMBINE
}
template <typename T>
static int combine_bwd_t(const void* dout, int64_t dout_stride, const void* ys, const void* weight, int w_bf16,
                         const int32_t* slot_row, const int32_t* row_slot, int64_t n_tokens, int top_k, int64_t rows, int hidden,
                         void* dys, void* dweight, cudaStream_t st) {
  const int vb = row_vec_bytes((int64_t)hidden * sizeof(T), n_tokens > 1 ? dout_stride * (int64_t)sizeof(T) : 0, dout, ys, dys);
#define BIBO_DISPATCH_CASE(VB)                                                                                              \
  if constexpr (VB >= (int)sizeof(T))                                                                                       \
    if (vb == VB)                                                                                                           \
      combine_bwd_v<T, VB>(dout, dout_stride, ys, weight, w_bf16, slot_row, row_slot, n_tokens, top_k, rows, hidden, dys,   \
                           dweight, st);
  BIBO_DISPATCH_CASE(16) BIBO_DISPATCH_CASE(8) BIBO_DISPATCH_CASE(4) BIBO_DISPATCH_CASE(2)
#undef BIBO_DISPATCH_CASE
  BIBO_CHECK_LAUNCH("dispatch_combine_bwd_kernel");
  return BIBO_OK;
}

extern "C" int bibo_moe_dispatch_combine_bwd(const void* dout, int64_t dout_stride, const void* ys, const void* topk_w,
                                             int w_dtype, const int32_t* plan, int64_t n_tokens, int hidden, int top_k,
                                             int n_experts, int align, int dtype, void* dys, void* d_topk_w, void* stream) {
  const int rc = dispatch_check("dispatch_combine_bwd", n_tokens, hidden, n_experts, top_k, align, dtype);
  if (rc) return rc;
  if (w_dtype != BIBO_F32 && w_dtype != BIBO_BF16) return fail(BIBO_ERR_ARG, "dispatch_combine_bwd: weight dtype=%d", w_dtype);
  if (n_tokens == 0) return BIBO_OK;
  if (!dout || !ys || !plan || !dys) return fail(BIBO_ERR_ARG, "dispatch_combine_bwd: null pointer");
  if (n_tokens > 1 && dout_stride < hidden) return fail(BIBO_ERR_ARG, "dispatch_combine_bwd: row stride %lld below hidden=%d", (long long)dout_stride, hidden);
  const int64_t slots = n_tokens * top_k, rows = dp_rows_cap(slots, n_experts, align);
  const int32_t* slot_row = plan + dp_off_slot_row(n_experts);
  const int32_t* row_slot = plan + dp_off_row_slot(n_experts, slots);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int wb = w_dtype == BIBO_BF16;
  return dtype == BIBO_F32
             ? combine_bwd_t<float>(dout, dout_stride, ys, topk_w, wb, slot_row, row_slot, n_tokens, top_k, rows, hidden, dys, d_topk_w, st)
             : combine_bwd_t<__nv_bfloat16>(dout, dout_stride, ys, topk_w, wb, slot_row, row_slot, n_tokens, top_k, rows, hidden, dys, d_topk_w, st);
}
