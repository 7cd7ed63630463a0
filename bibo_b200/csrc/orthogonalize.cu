// Newton-Schulz orthogonalisation of stacked matrices, the update of an optimiser that steps along the orthogonal
// factor of the momentum of the expert stacks [E,2I,H] / [E,H,I] and the router weight:
//   x_0 = u / (|u|_F + eps);   x_{k+1} = a x_k + (b G + c G^2) x_k,  G = x_k x_k^T   (m x n with m <= n; a tall matrix is
//   transposed on the way in and out), out = bf16(x_steps)
// An odd polynomial of the singular values is applied and the singular vectors stay.
//
// Numbers.  The products run on the tensor cores with f16 operands and fp32 accumulators: bf16 operands would lose
// three bits more, tf32 would halve the rate for none, and the range is bounded (|x|_2 <= about 1.2 for the usual
// coefficients, so every entry of x, G and b G + c G^2 is below 16).  All three are kept times 2^12, which centres
// them in f16's range: an entry 2^-26 of the largest is still normal.  u enters scaled by a power of two (exact for bf16)
// and the rest of 1/(|u|_F + eps), t in [1,2), goes into the first step's epilogues in fp32, so a bf16 matrix enters
// the first step without a rounding.
//
// Cost: per step m(m+1)n + m^2(m+1) + 2 m^2 n flops, since G and G^2 are symmetric: only tiles on and below the diagonal
// are computed, and stored a second time transposed.
#include <algorithm>
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace bibo {
namespace tc {

constexpr float NS_ONE = 4096.f;                 // 1.0 as stored
constexpr int NS_MAX_PARTS = 64;                 // partial sums of squares per matrix
constexpr int NS_GRAM = 0, NS_SQUARE = 1, NS_APPLY = 2;
constexpr int NS_BN = 128, NS_STAGES = 5;
constexpr int NS_OFF_A = 0;
constexpr int NS_OFF_B = NS_OFF_A + NS_STAGES * A_BYTES;
constexpr int NS_OFF_C = NS_OFF_B + NS_STAGES * A_BYTES;     // [2] sub-tiles of 64 columns: source in, result out
constexpr int NS_OFF_T = NS_OFF_C + 2 * C_SUB;               // [2] sub-tiles of the transposed result
constexpr int NS_OFF_BAR = NS_OFF_T + 2 * C_SUB;
constexpr int NS_SMEM = NS_OFF_BAR + 256 + 1024;

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

struct NsTile { int b, i, j; };
// work item -> matrix and tile; symmetric products list the tiles of the lower triangle row by row
template <int MODE> __device__ __forceinline__ NsTile ns_decode(int64_t w, int m_tiles, int n_tiles) {
  NsTile t;
  if (MODE == NS_APPLY) {
    const int64_t per = (int64_t)m_tiles * n_tiles;
    t.b = (int)(w / per);
    const int r = (int)(w % per);
    t.i = r % m_tiles;
    t.j = r / m_tiles;
  } else {
    const int per = m_tiles * (m_tiles + 1) / 2;
    t.b = (int)(w / per);
    const int r = (int)(w % per);
    int i = (int)((sqrtf(8.f * r + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= r) ++i;
    while (i * (i + 1) / 2 > r) --i;
    t.i = i;
    t.j = r - i * (i + 1) / 2;
  }
  return t;
}

// C = alpha * (A B) + beta * S, tiles of 128 x 128
//   NS_GRAM    A = B = x (K-major), no S;   NS_SQUARE  A = B = S = G (symmetric, so K-major too)
//   NS_APPLY   A = b G + c G^2 (K-major), B = S = x with n contiguous (MN-major)
// t_scale (first step only): alpha and beta are multiplied by t^2 (NS_GRAM) or t (NS_APPLY) of the matrix.
template <int MODE>
__global__ void __launch_bounds__(NUM_THREADS, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmS, const __grid_constant__ CUtensorMap tmC, int m_tiles, int n_tiles,
                  int64_t n_work, int k_blocks, int rows, int cols, float alpha, float beta,
                  const float* __restrict__ t_scale, int* __restrict__ status) {
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + NS_OFF_BAR);
  uint64_t* empty = full + NS_STAGES;
  uint64_t* tfull = empty + NS_STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* sfull = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sfull + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 4); }
    mbar_init(sfull, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA); prefetch_tmap(&tmB); prefetch_tmap(&tmS); prefetch_tmap(&tmC);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 2 * NS_BN); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      PipeState ps;
      bool ok = true;
      for (int64_t w = blockIdx.x; w < n_work && ok; w += gridDim.x) {
        const NsTile t = ns_decode<MODE>(w, m_tiles, n_tiles);
        const bool same = MODE != NS_APPLY && t.i == t.j;          // both operands are one tile
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = mbar_wait(&empty[ps.stage], ps.phase ^ 1, abort_flag);
          if (!ok) break;
          mbar_expect_tx(&full[ps.stage], same ? A_BYTES : 2 * A_BYTES);
          unsigned char* sa = smem + NS_OFF_A + ps.stage * A_BYTES;
          unsigned char* sb = smem + NS_OFF_B + ps.stage * A_BYTES;
          tma_load_3d(sa, &tmA, &full[ps.stage], kb * BK, t.i * BM, t.b);
          if (MODE == NS_APPLY) {
            tma_load_3d(sb, &tmB, &full[ps.stage], t.j * NS_BN, kb * BK, t.b);
            tma_load_3d(sb + MN_BOX, &tmB, &full[ps.stage], t.j * NS_BN + 64, kb * BK, t.b);
          } else if (!same) {
            tma_load_3d(sb, &tmB, &full[ps.stage], kb * BK, t.j * NS_BN, t.b);
          }
          ps.next<NS_STAGES>();
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_f16(BM, NS_BN) | (MODE == NS_APPLY ? 1u << 16 : 0u);   // bit 16: B is MN-major
      PipeState ps;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int64_t w = blockIdx.x; w < n_work && ok; w += gridDim.x) {
        const NsTile t = ns_decode<MODE>(w, m_tiles, n_tiles);
        const bool same = MODE != NS_APPLY && t.i == t.j;
        ok = mbar_wait(&tempty[acc], acc_phase ^ 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = mbar_wait(&full[ps.stage], ps.phase, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + NS_OFF_A + ps.stage * A_BYTES);
          const uint32_t sb = smem_u32(smem + NS_OFF_B + ps.stage * A_BYTES);
          const uint64_t da = make_sdesc_k128(sa);
          const uint64_t db = MODE == NS_APPLY ? make_sdesc_mn128(sb) : make_sdesc_k128(same ? sa : sb);
          constexpr int b_step = MODE == NS_APPLY ? (2048 >> 4) : (32 >> 4);
#pragma unroll
          for (int k = 0; k < BK / UK; ++k)
            umma_bf16(tmem_base + acc * NS_BN, da + k * (32 >> 4), db + k * b_step, idesc, (kb | k) != 0);
          umma_commit(&empty[ps.stage]);
          ps.next<NS_STAGES>();
        }
        if (!ok) break;
        umma_commit(&tfull[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else {
    const int q = warp & 3;
    const int row = q * 32 + lane;
    const bool issuer = threadIdx.x == 64;
    int acc = 0;
    uint32_t acc_phase = 0, s_phase = 0;
    for (int64_t w = blockIdx.x; w < n_work; w += gridDim.x) {
      const NsTile t = ns_decode<MODE>(w, m_tiles, n_tiles);
      float al = alpha, be = beta;
      if (t_scale != nullptr) {
        const float ts = t_scale[t.b];
        al *= MODE == NS_GRAM ? ts * ts : ts;
        be *= ts;
      }
      const int halves = t.j * NS_BN + 64 < cols ? 2 : 1;          // a sub-tile outside the matrix is neither read nor written
      if (issuer) {
        tma_store_wait_read();                                     // the previous tile's stores have left both stagings
        if (MODE != NS_GRAM) {
          mbar_expect_tx(sfull, halves * C_SUB);
          for (int g = 0; g < halves; ++g)
            tma_load_3d(smem + NS_OFF_C + g * C_SUB, &tmS, sfull, t.j * NS_BN + g * 64, t.i * BM, t.b);
        }
      }
      const bool ok = mbar_wait(&tfull[acc], acc_phase, abort_flag) && (MODE == NS_GRAM || mbar_wait(sfull, s_phase, abort_flag));
      if (!named_bar_all(1, EPI_THREADS, ok)) break;
      s_phase ^= 1;
      tc_fence_after();
      const bool mirror = MODE != NS_APPLY && t.i != t.j;
#pragma unroll 1
      for (int g = 0; g < 2; ++g) {
        uint32_t r[2][32];
        const uint32_t ta = tmem_base + ((uint32_t)(q * 32) << 16) + acc * NS_BN + g * 64;
        tmem_ld32(ta, r[0]);
        tmem_ld32(ta + 32, r[1]);
        tmem_ld_wait();
        unsigned char* cbuf = smem + NS_OFF_C + g * C_SUB;
        unsigned char* tbuf = smem + NS_OFF_T + (row >> 6) * C_SUB;
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
          uint4* slot = reinterpret_cast<uint4*>(cbuf + swz(row, jj));
          const uint32_t* a = r[jj >> 2] + 8 * (jj & 3);
          uint4 v;
          uint32_t* pv = reinterpret_cast<uint32_t*>(&v);
          if (MODE != NS_GRAM) v = *slot;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float lo = al * __uint_as_float(a[2 * i]), hi = al * __uint_as_float(a[2 * i + 1]);
            if (MODE != NS_GRAM) {
              const float2 s = unpack_f16(pv[i]);
              lo = fmaf(be, s.x, lo);
              hi = fmaf(be, s.y, hi);
            }
            pv[i] = pack_f16(lo, hi);
          }
          *slot = v;
          if (mirror) {
            // element (row, g*64 + jj*8 + i) of the tile is element (g*64 + jj*8 + i, row) of the transposed one; for a
            // fixed column the 32 lanes write 64 consecutive bytes
            const unsigned short* h = reinterpret_cast<const unsigned short*>(&v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int tr = g * 64 + jj * 8 + i;
              *reinterpret_cast<unsigned short*>(tbuf + swz(tr, (row & 63) >> 3) + (row & 7) * 2) = h[i];
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      fence_proxy_async_smem();
      named_bar_sync(1, EPI_THREADS);
      if (issuer) {
        for (int g = 0; g < halves; ++g) tma_store_3d(&tmC, smem + NS_OFF_C + g * C_SUB, t.j * NS_BN + g * 64, t.i * BM, t.b);
        if (mirror)
          for (int g = 0; g < 2; ++g)
            if (t.i * BM + g * 64 < rows)
              tma_store_3d(&tmC, smem + NS_OFF_T + g * C_SUB, t.i * BM + g * 64, t.j * NS_BN, t.b);
        tma_store_commit();
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (issuer) tma_store_wait_all();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {                             // a wait gave up: copies may still be in flight to this shared memory
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    if (threadIdx.x == 0) atomicExch(status, 112);
  }
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, 2 * NS_BN); }
}

// ---- way in: sum of squares, then f16 with the wide side along the rows -----------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
ns_sumsq_kernel(const T* __restrict__ u, int64_t batch_stride, int64_t row_stride, int rows, int cols, float* __restrict__ partial) {
  __shared__ float red[8];
  const T* src = u + (int64_t)blockIdx.y * batch_stride;
  float s = 0.f;
  for (int r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += 256) { const float v = to_f32<T>(src[(int64_t)r * row_stride + c]); s = fmaf(v, v, s); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    for (int w = 0; w < 8; ++w) s += red[w];
    partial[(int64_t)blockIdx.y * NS_MAX_PARTS + blockIdx.x] = s;
  }
}

// x * q with q the power of two that brings the norm into (2048, 4096]; t = 4096 / ((norm + eps) q) is left in t_out
template <typename T>
__global__ void __launch_bounds__(256)
ns_enter_kernel(const T* __restrict__ u, int64_t batch_stride, int64_t row_stride, int rows, int cols, int tall, float eps,
                const float* __restrict__ partial, int n_parts, __half* __restrict__ x, int ld, float* __restrict__ t_out,
                int* __restrict__ status) {
  __shared__ float tile[32][33];
  __shared__ float q_s;
  const int64_t b = blockIdx.z;
  if (threadIdx.x == 0) {
    float s = 0.f;
    for (int p = 0; p < n_parts; ++p) s += partial[b * NS_MAX_PARTS + p];
    const float norm = sqrtf(s) + eps;
    int e = 0;
    float q = 1.f;
    if (norm > 0.f && norm < 3e38f) {
      frexpf(norm, &e);                          // norm = f * 2^e, f in [0.5, 1)
      q = ldexpf(1.f, 12 - e < 120 ? 12 - e : 120);
    }
    q_s = q;
    if (blockIdx.x == 0 && blockIdx.y == 0) {
      t_out[b] = NS_ONE / (norm * q);
      if (b == 0) *status = 0;
    }
  }
  __syncthreads();
  const float q = q_s;
  const T* src = u + b * batch_stride;
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = ty; i < 32; i += 8)
    tile[i][tx] = r0 + i < rows && c0 + tx < cols ? q * to_f32<T>(src[(int64_t)(r0 + i) * row_stride + c0 + tx]) : 0.f;
  __syncthreads();
  const int xr = tall ? cols : rows, xc = tall ? rows : cols;        // shape of x
  const int xr0 = tall ? c0 : r0, xc0 = tall ? r0 : c0;
  __half* dst = x + b * (int64_t)xr * ld;
  for (int i = ty; i < 32; i += 8)
    if (xr0 + i < xr && xc0 + tx < xc) dst[(int64_t)(xr0 + i) * ld + xc0 + tx] = __float2half_rn(tall ? tile[tx][i] : tile[i][tx]);
}

// ---- way out ---------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
ns_leave_kernel(const __half* __restrict__ x, int ld, int rows, int cols, int tall, const int* __restrict__ status,
                __nv_bfloat16* __restrict__ out) {
  __shared__ float tile[32][33];
  const int64_t b = blockIdx.z;
  const int xr = tall ? cols : rows, xc = tall ? rows : cols;
  const __half* src = x + b * (int64_t)xr * ld;
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;              // of the result
  const int xr0 = tall ? c0 : r0, xc0 = tall ? r0 : c0;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = ty; i < 32; i += 8)
    tile[i][tx] = xr0 + i < xr && xc0 + tx < xc ? __half2float(src[(int64_t)(xr0 + i) * ld + xc0 + tx]) * (1.f / NS_ONE) : 0.f;
  __syncthreads();
  const bool failed = *status != 0;                                  // a wait gave up: no number is left to stand
  for (int i = ty; i < 32; i += 8)
    if (r0 + i < rows && c0 + tx < cols)
      out[(b * rows + r0 + i) * (int64_t)cols + c0 + tx] =
          __float2bfloat16_rn(failed ? __int_as_float(0x7fffffff) : tall ? tile[tx][i] : tile[i][tx]);
}

template <int MODE>
static int ns_product(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& s, const CUtensorMap& c, int64_t batch, int rows,
                      int cols, int k_dim, float alpha, float beta, const float* t_scale, int* status, cudaStream_t st) {
  auto kern = ns_product_kernel<MODE>;
  static DeviceOnce once;
  const int rc = once.get([&](int*) {
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM));
    return (int)BIBO_OK;
  });
  if (rc) return rc;
  const int mt = (rows + BM - 1) / BM, nt = (cols + NS_BN - 1) / NS_BN;
  const int64_t work = batch * (MODE == NS_APPLY ? (int64_t)mt * nt : (int64_t)mt * (mt + 1) / 2);
  const int grid = (int)std::min<int64_t>(sm_count(), work);
  kern<<<grid, NUM_THREADS, NS_SMEM, st>>>(a, b, s, c, mt, nt, work, (k_dim + BK - 1) / BK, rows, cols, alpha, beta, t_scale, status);
  BIBO_CHECK_LAUNCH("ns_product_kernel");
  return BIBO_OK;
}

// workspace of `batch` matrices: x twice, G, b G + c G^2 (f16, rows of 16-byte multiples), partial sums, t, status
struct NsLayout {
  int m, n, ldx, ldg;
  int64_t x_bytes, g_bytes, off_g, off_f, off_x1, off_part, off_t, off_status, bytes;
  NsLayout(int64_t batch, int rows, int cols) {
    m = std::min(rows, cols);
    n = std::max(rows, cols);
    ldx = (n + 7) / 8 * 8;
    ldg = (m + 7) / 8 * 8;
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    x_bytes = up(batch * m * (int64_t)ldx * 2);
    g_bytes = up(batch * m * (int64_t)ldg * 2);
    off_x1 = x_bytes;
    off_g = 2 * x_bytes;
    off_f = off_g + g_bytes;
    off_part = off_f + g_bytes;
    off_t = off_part + up(batch * NS_MAX_PARTS * 4);
    off_status = off_t + up(batch * 4);
    bytes = off_status + 256;
  }
};
// matrices that run together: as many as a workspace of 1 GiB holds, one at least
static int64_t ns_chunk(int64_t batch, int rows, int cols) {
  const int64_t one = NsLayout(1, rows, cols).bytes;
  return std::max<int64_t>(1, std::min<int64_t>({batch, (1ll << 30) / one, 32768}));
}

}  // namespace tc
}  // namespace bibo

using namespace bibo;
using namespace bibo::tc;

extern "C" int64_t bibo_moe_orthogonalize_workspace(int64_t batch, int rows, int cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  return NsLayout(ns_chunk(batch, rows, cols), rows, cols).bytes;
}

extern "C" int bibo_moe_orthogonalize(const void* u, int64_t batch, int64_t batch_stride, int rows, int cols, int64_t row_stride,
                                      int dtype, int steps, const float* coefficients_host, float eps, void* workspace, void* out,
                                      void* stream) {
  if (dtype != BIBO_F32 && dtype != BIBO_BF16) return fail(BIBO_ERR_ARG, "orthogonalize: dtype=%d", dtype);
  if (batch < 0 || rows < 0 || cols < 0 || rows > 65535 * 32 || cols > 65535 * 32)
    return fail(BIBO_ERR_ARG, "orthogonalize: %lld matrices of %d x %d", (long long)batch, rows, cols);
  if (steps < 1 || steps > 64 || !coefficients_host) return fail(BIBO_ERR_ARG, "orthogonalize: steps=%d (1..64)", steps);
  if (batch == 0 || rows == 0 || cols == 0) return BIBO_OK;
  if (!u || !workspace || !out) return fail(BIBO_ERR_ARG, "orthogonalize: null pointer");
  if ((reinterpret_cast<uintptr_t>(workspace) & 127u) != 0) return fail(BIBO_ERR_ALIGN, "orthogonalize: workspace not 128-byte aligned");
  if ((rows > 1 && row_stride < cols) || (batch > 1 && batch_stride < (rows - 1) * row_stride + cols))
    return fail(BIBO_ERR_ARG, "orthogonalize: overlapping rows or matrices");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int tall = rows > cols, size = dtype == BIBO_F32 ? 4 : 2;
  const int64_t chunk = ns_chunk(batch, rows, cols);
  for (int64_t b0 = 0; b0 < batch; b0 += chunk) {
    const int64_t nb = std::min(chunk, batch - b0);
    const NsLayout l(nb, rows, cols);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    __half* x[2] = {reinterpret_cast<__half*>(ws), reinterpret_cast<__half*>(ws + l.off_x1)};
    float* partial = reinterpret_cast<float*>(ws + l.off_part);
    float* t = reinterpret_cast<float*>(ws + l.off_t);
    int* status = reinterpret_cast<int*>(ws + l.off_status);
    const unsigned char* src = static_cast<const unsigned char*>(u) + b0 * batch_stride * size;
    const int parts = std::min(NS_MAX_PARTS, rows);
    const dim3 sum_grid(parts, (unsigned)nb), tiles((cols + 31) / 32, (rows + 31) / 32, (unsigned)nb);
    if (dtype == BIBO_F32) {
      ns_sumsq_kernel<float><<<sum_grid, 256, 0, st>>>(reinterpret_cast<const float*>(src), batch_stride, row_stride, rows, cols, partial);
      BIBO_CHECK_LAUNCH("ns_sumsq_kernel");
      ns_enter_kernel<float><<<tiles, 256, 0, st>>>(reinterpret_cast<const float*>(src), batch_stride, row_stride, rows, cols, tall,
                                                   eps, partial, parts, x[0], l.ldx, t, status);
    } else {
      ns_sumsq_kernel<__nv_bfloat16><<<sum_grid, 256, 0, st>>>(reinterpret_cast<const __nv_bfloat16*>(src), batch_stride, row_stride,
                                                              rows, cols, partial);
      BIBO_CHECK_LAUNCH("ns_sumsq_kernel");
      ns_enter_kernel<__nv_bfloat16><<<tiles, 256, 0, st>>>(reinterpret_cast<const __nv_bfloat16*>(src), batch_stride, row_stride,
                                                           rows, cols, tall, eps, partial, parts, x[0], l.ldx, t, status);
    }
    BIBO_CHECK_LAUNCH("ns_enter_kernel");
    CUtensorMap mx[2], mxk[2], mg, mf;
    int rc;
    for (int i = 0; i < 2; ++i) {
      if ((rc = make_tmap_f16_3d(&mx[i], x[i], nb, l.m, l.n, l.ldx, BM))) return rc;
      if ((rc = make_tmap_f16_3d(&mxk[i], x[i], nb, l.m, l.n, l.ldx, 64))) return rc;
    }
    if ((rc = make_tmap_f16_3d(&mg, ws + l.off_g, nb, l.m, l.m, l.ldg, BM))) return rc;
    if ((rc = make_tmap_f16_3d(&mf, ws + l.off_f, nb, l.m, l.m, l.ldg, BM))) return rc;
    for (int s = 0; s < steps; ++s) {
      const float* co = coefficients_host + 3 * s;
      const float* ts = s == 0 ? t : nullptr;
      const int i = s & 1;
      if ((rc = ns_product<NS_GRAM>(mx[i], mx[i], mx[i], mg, nb, l.m, l.m, l.n, 1.f / NS_ONE, 0.f, ts, status, st))) return rc;
      if ((rc = ns_product<NS_SQUARE>(mg, mg, mg, mf, nb, l.m, l.m, l.m, co[2] / NS_ONE, co[1], nullptr, status, st))) return rc;
      if ((rc = ns_product<NS_APPLY>(mf, mxk[i], mx[i], mx[1 - i], nb, l.m, l.n, l.m, 1.f / NS_ONE, co[0], ts, status, st))) return rc;
    }
    ns_leave_kernel<<<tiles, 256, 0, st>>>(x[steps & 1], l.ldx, rows, cols, tall, status,
                                           static_cast<__nv_bfloat16*>(out) + b0 * rows * cols);
    BIBO_CHECK_LAUNCH("ns_leave_kernel");
  }
  return BIBO_OK;
}
