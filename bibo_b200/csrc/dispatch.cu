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
#include <cooperative_groups.h>

#include "common.cuh"

namespace bibo {

namespace cg = cooperative_groups;

// words of the plan buffer: offsets [E+1], counts [E], status, then (16-byte aligned) slot_row [slots], row_slot [rows]
__host__ __device__ inline int64_t dp_off_counts(int E) { return E + 1; }
__host__ __device__ inline int64_t dp_off_status(int E) { return 2 * (int64_t)E + 1; }
__host__ __device__ inline int64_t dp_off_slot_row(int E) { return (2 * (int64_t)E + 2 + 3) / 4 * 4; }
__host__ __device__ inline int64_t dp_off_row_slot(int E, int64_t slots) { return dp_off_slot_row(E) + (slots + 3) / 4 * 4; }
inline int64_t dp_rows_cap(int64_t slots, int E, int align) {
  const int64_t groups = slots < E ? slots : E;
  return (slots + groups * (align - 1) + align - 1) / align * align;
}
constexpr int DP_MAX_EXPERTS = 1024, DP_MAX_TOP_K = 32, DP_STATUS_INDEX = 2;

// ---- plan: a stable counting sort in one launch ------------------------------------------------------------------
// One cluster.  Each warp owns a contiguous range of slots and a histogram row in shared memory; the warp totals are
// scanned per expert inside the block, the block totals across the cluster through distributed shared memory, and a
// second pass over the (L2-resident) indices hands out the rows in slot order.
template <typename I>
__global__ void __launch_bounds__(1024, 1)
dispatch_plan_kernel(const I* __restrict__ idx, int64_t slots, int E, int align, int64_t rows_cap, int32_t* __restrict__ plan) {
  extern __shared__ int32_t sm[];
  const int warps = blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  cg::cluster_group cl = cg::this_cluster();
  const int cta = (int)cl.block_rank(), n_cta = (int)cl.num_blocks();
  int32_t* total = sm;                       // [E]   this block's slots per expert (read by the other blocks)
  int32_t* base = sm + E;                    // [E+1] first row of this block's slots of an expert; before that the offsets
  int32_t* hist = sm + 2 * E + 1 + (size_t)warp * E;
  int32_t* slot_row = plan + dp_off_slot_row(E);
  int32_t* row_slot = plan + dp_off_row_slot(E, slots);
  for (int e = lane; e < E; e += 32) hist[e] = 0;
  __syncwarp();
  const int64_t n_warps = (int64_t)n_cta * warps, per = ((slots + n_warps - 1) / n_warps + 31) / 32 * 32;
  const int64_t s0 = ((int64_t)cta * warps + warp) * per, s1 = s0 + per < slots ? s0 + per : slots;
  bool bad = false;
  for (int64_t s = s0; s < s1; s += 32) {
    const int64_t v = s + lane < s1 ? (int64_t)idx[s + lane] : -1;
    const int e = v >= 0 && v < E ? (int)v : -1;
    bad |= v >= E;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) hist[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {     // exclusive scan over the warps of this block
    int run = 0;
    for (int w = 0; w < warps; ++w) {
      int32_t* h = sm + 2 * E + 1 + (size_t)w * E + e;
      const int c = *h;
      *h = run;
      run += c;
    }
    total[e] = run;
  }
  cl.sync();
  // every block: counts over the cluster and the slots of lower blocks
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int all = 0, lower = 0;
    for (int b = 0; b < n_cta; ++b) {
      const int c = cl.map_shared_rank(total, b)[e];
      all += c;
      if (b < cta) lower += c;
    }
    base[e] = all;
    if (cta == 0) plan[dp_off_counts(E) + e] = all;
    for (int w = 0; w < warps; ++w) sm[2 * E + 1 + (size_t)w * E + e] += lower;
  }
  __syncthreads();
  if (warp == 0) {                                          // offsets: exclusive scan of the padded counts
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < E ? (base[e] + align - 1) / align * align : 0;
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
      if (e < E) base[e] = carry + inc - c;
      carry += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) base[E] = carry;
  }
  __syncthreads();
  if (cta == 0) {
    for (int e = threadIdx.x; e <= E; e += blockDim.x) plan[e] = base[e];
  }
  // rows without a slot: the padding behind each group and everything behind the last group
  for (int e = cta * warps + warp; e < E; e += n_cta * warps) {
    int all = 0;
    for (int b = 0; b < n_cta; ++b) all += cl.map_shared_rank(total, b)[e];
    for (int r = base[e] + all + lane; r < base[e + 1]; r += 32) row_slot[r] = -1;
  }
  for (int64_t r = base[E] + (int64_t)cta * blockDim.x + threadIdx.x; r < rows_cap; r += (int64_t)n_cta * blockDim.x)
    row_slot[r] = -1;
  for (int64_t s = s0; s < s1; s += 32) {
    const bool in = s + lane < s1;
    const int64_t v = in ? (int64_t)idx[s + lane] : -1;
    const int e = v >= 0 && v < E ? (int)v : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    int row = -1;
    if (e >= 0) row = base[e] + hist[e] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) hist[e] += __popc(same);
    __syncwarp();
    if (in) slot_row[s + lane] = row;
    if (row >= 0) row_slot[row] = (int32_t)(s + lane);
  }
  // the status word: raised by any block, written once by block 0 after every block has looked at its slots
  __shared__ int bad_here;
  if (threadIdx.x == 0) bad_here = 0;
  __syncthreads();
  if (bad) bad_here = 1;
  cl.sync();
  if (cta == 0 && threadIdx.x == 0) {
    int any = 0;
    for (int b = 0; b < n_cta; ++b) any |= *cl.map_shared_rank(&bad_here, b);
    plan[dp_off_status(E)] = any ? DP_STATUS_INDEX : 0;
  }
  cl.sync();                                                // no block leaves while its shared memory is read
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
constexpr int DZ_ROWS = 16;    // rows a warp looks at for zeroing

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

// warps [0, N): a token's row is read once and written to its (up to k) rows; warps behind them zero empty rows
template <int VB>
__global__ void __launch_bounds__(DW * 32)
dispatch_kernel(const uint8_t* __restrict__ x, int64_t x_stride_bytes, const int32_t* __restrict__ slot_row,
                const int32_t* __restrict__ row_slot, int64_t n_tokens, int top_k, int64_t rows, int row_bytes,
                uint8_t* __restrict__ xs) {
  using V = typename RowVec<VB>::type;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * DW + (threadIdx.x >> 5);
  const int chunks = row_bytes / VB;
  V* dst = reinterpret_cast<V*>(xs);
  if (w >= n_tokens) {
    zero_empty_rows<VB>(row_slot, (w - n_tokens) * DZ_ROWS, rows, chunks, dst, lane);
    return;
  }
  const int mine = lane < top_k ? slot_row[w * top_k + lane] : -1;
  if (!__any_sync(0xffffffffu, mine >= 0)) return;
  const V* src = reinterpret_cast<const V*>(x + w * x_stride_bytes);
  for (int c0 = lane; c0 - lane < chunks; c0 += 256) {
    V v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (c0 + u * 32 < chunks) v[u] = src[c0 + u * 32];
    for (int j = 0; j < top_k; ++j) {
      const int r = __shfl_sync(0xffffffffu, mine, j);
      if (r < 0) continue;
      V* d = dst + (int64_t)r * chunks;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c0 + u * 32 < chunks) d[c0 + u * 32] = v[u];
    }
  }
}

// weights are fp32 or the rows' type
__device__ __forceinline__ float load_weight(const void* w, int is_bf16, int64_t i) {
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : static_cast<const float*>(w)[i];
}

// out[t] = sum_j w[t,j] * ys[slot_row[t,j]] (w == nullptr: 1), a warp per token, slots in order
template <typename T, int VB>
__global__ void __launch_bounds__(DW * 32)
dispatch_combine_kernel(const T* __restrict__ ys, const void* __restrict__ weight, int w_bf16,
                        const int32_t* __restrict__ slot_row, int64_t n_tokens, int top_k, int hidden, T* __restrict__ out) {
  using V = typename RowVec<VB>::type;
  using X = RowElems<T, VB>;
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * DW + (threadIdx.x >> 5);
  if (t >= n_tokens) return;
  const int chunks = hidden / X::N;
  const int mine = lane < top_k ? slot_row[t * top_k + lane] : -1;
  const float my_w = mine < 0 ? 0.f : weight == nullptr ? 1.f : load_weight(weight, w_bf16, t * top_k + lane);
  const V* src = reinterpret_cast<const V*>(ys);
  V* dst = reinterpret_cast<V*>(out) + t * chunks;
  for (int c0 = 0; c0 < chunks; c0 += 32) {
    const int c = c0 + lane;
    float acc[X::N];
#pragma unroll
    for (int i = 0; i < X::N; ++i) acc[i] = 0.f;
    for (int j = 0; j < top_k; ++j) {
      const int r = __shfl_sync(0xffffffffu, mine, j);
      const float w = __shfl_sync(0xffffffffu, my_w, j);
      if (r < 0 || c >= chunks) continue;
      float f[X::N];
      X::unpack(src[(int64_t)r * chunks + c], f);
#pragma unroll
      for (int i = 0; i < X::N; ++i) acc[i] = fmaf(f[i], w, acc[i]);
    }
    if (c < chunks) dst[c] = X::pack(acc);
  }
}

// warps [0, N): dys rows and dw of a token's slots; warps behind them zero empty rows of dys
template <typename T, int VB>
__global__ void __launch_bounds__(DW * 32)
dispatch_combine_bwd_kernel(const T* __restrict__ dout, int64_t dout_stride, const T* __restrict__ ys,
                            const void* __restrict__ weight, int w_bf16, const int32_t* __restrict__ slot_row,
                            const int32_t* __restrict__ row_slot, int64_t n_tokens, int top_k, int64_t rows, int hidden,
                            T* __restrict__ dys, void* __restrict__ dweight) {
  using V = typename RowVec<VB>::type;
  using X = RowElems<T, VB>;
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * DW + (threadIdx.x >> 5);
  const int chunks = hidden / X::N;
  V* dst = reinterpret_cast<V*>(dys);
  if (t >= n_tokens) {
    zero_empty_rows<VB>(row_slot, (t - n_tokens) * DZ_ROWS, rows, chunks, dst, lane);
    return;
  }
  const V* g = reinterpret_cast<const V*>(dout + t * dout_stride);
  const V* src = reinterpret_cast<const V*>(ys);
  const int mine = lane < top_k ? slot_row[t * top_k + lane] : -1;
  const float my_w = mine < 0 ? 0.f : weight == nullptr ? 1.f : load_weight(weight, w_bf16, t * top_k + lane);
  float my_dw = 0.f;
  for (int j = 0; j < top_k; ++j) {
    const int r = __shfl_sync(0xffffffffu, mine, j);
    const float w = __shfl_sync(0xffffffffu, my_w, j);
    if (r < 0) continue;
    float dot = 0.f;
    for (int c = lane; c < chunks; c += 32) {
      float gf[X::N], yf[X::N];
      X::unpack(g[c], gf);
      if (dweight != nullptr) {
        X::unpack(src[(int64_t)r * chunks + c], yf);
#pragma unroll
        for (int i = 0; i < X::N; ++i) dot = fmaf(gf[i], yf[i], dot);
      }
#pragma unroll
      for (int i = 0; i < X::N; ++i) gf[i] *= w;
      dst[(int64_t)r * chunks + c] = X::pack(gf);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == j) my_dw = dot;
  }
  if (dweight != nullptr && lane < top_k) {
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
  if (n_tokens < 0 || n_tokens * top_k > (1ll << 30)) return fail(BIBO_ERR_UNSUPPORTED, "%s: %lld slots", what, (long long)n_tokens * top_k);
  return BIBO_OK;
}
static unsigned dispatch_grid(int64_t warps) { return (unsigned)((warps + DW - 1) / DW); }

template <typename I>
static int plan_launch(const void* idx, int64_t slots, int E, int align, int32_t* plan, cudaStream_t st) {
  auto kern = dispatch_plan_kernel<I>;
  static DeviceOnce once;
  const int rc = once.get([&](int*) {
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(int32_t) * (34 * DP_MAX_EXPERTS + 1)));
    return (int)BIBO_OK;
  });
  if (rc) return rc;
  // one block up to 8192 slots (a cluster barrier costs more than the eighth of the work that it saves), eight above
  const int blocks = slots <= 8192 ? 1 : 8;
  const int threads = slots <= 1024 ? 256 : 1024;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = sizeof(int32_t) * (2 * (size_t)E + 1 + (size_t)(threads / 32) * E);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BIBO_CUDA(cudaLaunchKernelEx(&cfg, kern, static_cast<const I*>(idx), slots, E, align, dp_rows_cap(slots, E, align), plan));
  BIBO_CHECK_LAUNCH("dispatch_plan_kernel");
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
  return dp_off_row_slot(n_experts, n_tokens * top_k) + dp_rows_cap(n_tokens * top_k, n_experts, align);
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
  const unsigned grid = dispatch_grid(n_tokens + (rows + DZ_ROWS - 1) / DZ_ROWS);
#define BIBO_DISPATCH_CASE(VB)                                                                                              \
  case VB:                                                                                                                  \
    dispatch_kernel<VB><<<grid, DW * 32, 0, st>>>(static_cast<const uint8_t*>(x), x_stride * size, slot_row, row_slot,      \
                                                  n_tokens, top_k, rows, row_bytes, static_cast<uint8_t*>(xs));             \
    break;
  switch (row_vec_bytes(row_bytes, n_tokens > 1 ? x_stride * size : 0, x, xs, nullptr)) {
    BIBO_DISPATCH_CASE(16) BIBO_DISPATCH_CASE(8) BIBO_DISPATCH_CASE(4) BIBO_DISPATCH_CASE(2)
  }
#undef BIBO_DISPATCH_CASE
  BIBO_CHECK_LAUNCH("dispatch_kernel");
  return BIBO_OK;
}

template <typename T>
static int combine_t(const void* ys, const void* weight, int w_bf16, const int32_t* slot_row, int64_t n_tokens, int top_k,
                     int hidden, void* out, cudaStream_t st) {
  const unsigned grid = dispatch_grid(n_tokens);
  const int vb = row_vec_bytes((int64_t)hidden * sizeof(T), 0, ys, out, nullptr);
#define BIBO_DISPATCH_CASE(VB)                                                                                               \
  if constexpr (VB >= (int)sizeof(T))                                                                                        \
    if (vb == VB)                                                                                                            \
      dispatch_combine_kernel<T, VB><<<grid, DW * 32, 0, st>>>(static_cast<const T*>(ys), weight, w_bf16, slot_row, n_tokens, \
                                                               top_k, hidden, static_cast<T*>(out));
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

template <typename T>
static int combine_bwd_t(const void* dout, int64_t dout_stride, const void* ys, const void* weight, int w_bf16,
                         const int32_t* slot_row, const int32_t* row_slot, int64_t n_tokens, int top_k, int64_t rows, int hidden,
                         void* dys, void* dweight, cudaStream_t st) {
  const unsigned grid = dispatch_grid(n_tokens + (rows + DZ_ROWS - 1) / DZ_ROWS);
  const int vb = row_vec_bytes((int64_t)hidden * sizeof(T), n_tokens > 1 ? dout_stride * (int64_t)sizeof(T) : 0, dout, ys, dys);
#define BIBO_DISPATCH_CASE(VB)                                                                                          \
  if constexpr (VB >= (int)sizeof(T))                                                                                   \
    if (vb == VB)                                                                                                       \
      dispatch_combine_bwd_kernel<T, VB><<<grid, DW * 32, 0, st>>>(                                                     \
          static_cast<const T*>(dout), dout_stride, static_cast<const T*>(ys), weight, w_bf16, slot_row, row_slot,      \
          n_tokens, top_k, rows, hidden, static_cast<T*>(dys), dweight);
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
