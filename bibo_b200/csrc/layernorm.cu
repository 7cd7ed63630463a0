// Layer norm over the last dimension, forward and backward, beside the RMSNorm of rmsnorm.cu:
//   mean = sum(x)/H, var = sum((x-mean)^2)/H, rstd = 1/sqrt(var+eps), xhat = (x-mean)*rstd
//   y  = xhat*w + b
//   g  = dy*w;  dx = rstd*(g - mean(g) - xhat*mean(g*xhat));  dw = sum over rows of dy*xhat;  db = sum over rows of dy
// Everything is held in fp32 and rounded once, at the store.  The variance is taken around the mean in a second
// pass over the row: E[x^2] - mean^2 loses it where the mean is large against the spread.
#include "common.cuh"

namespace bibo {

// ---- any hidden size: one block per row, the row re-read from L1 / L2 for each pass ----------------------------
constexpr int LN_T = 256;

__device__ __forceinline__ float2 ln_block_sum2(float a, float b, float2* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();                       // the previous call's readers are done with red
  if (lane == 0) red[warp] = make_float2(a, b);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int w = 0; w < (int)blockDim.x / 32; ++w) { s.x += red[w].x; s.y += red[w].y; }
  return s;
}

template <typename T, typename W>
__global__ void __launch_bounds__(LN_T)
layernorm_loop_kernel(const T* __restrict__ x, int64_t x_stride, const W* __restrict__ weight, const W* __restrict__ bias,
                      float eps, int hidden, T* __restrict__ out, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float2 red[LN_T / 32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * x_stride;
  T* yr = out + row * hidden;
  float s = 0.f;
  for (int c = threadIdx.x; c < hidden; c += LN_T) s += to_f32<T>(xr[c]);
  const float mean = ln_block_sum2(s, 0.f, red).x / (float)hidden;
  s = 0.f;
  for (int c = threadIdx.x; c < hidden; c += LN_T) { const float d = to_f32<T>(xr[c]) - mean; s = fmaf(d, d, s); }
  const float rstd = rsqrtf(ln_block_sum2(s, 0.f, red).x / (float)hidden + eps);
  if (threadIdx.x == 0 && mean_out != nullptr) { mean_out[row] = mean; rstd_out[row] = rstd; }
  for (int c = threadIdx.x; c < hidden; c += LN_T) {
    const float z = (to_f32<T>(xr[c]) - mean) * rstd;
    const float w = weight != nullptr ? to_f32<W>(weight[c]) : 1.f;
    yr[c] = from_f32<T>(fmaf(z, w, bias != nullptr ? to_f32<W>(bias[c]) : 0.f));
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(LN_T)
layernorm_bwd_dx_loop_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy, int64_t dy_stride,
                             const W* __restrict__ weight, const float* __restrict__ mean_in,
                             const float* __restrict__ rstd_in, int hidden, T* __restrict__ dx) {
  __shared__ float2 red[LN_T / 32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * x_stride;
  const T* gr = dy + row * dy_stride;
  const float mean = mean_in[row], rstd = rstd_in[row];
  float s0 = 0.f, s1 = 0.f;
  for (int c = threadIdx.x; c < hidden; c += LN_T) {
    const float g = to_f32<T>(gr[c]) * (weight != nullptr ? to_f32<W>(weight[c]) : 1.f);
    s0 += g;
    s1 = fmaf(g, (to_f32<T>(xr[c]) - mean) * rstd, s1);
  }
  const float2 s = ln_block_sum2(s0, s1, red);
  const float m0 = s.x / (float)hidden, m1 = s.y / (float)hidden;
  for (int c = threadIdx.x; c < hidden; c += LN_T) {
    const float g = to_f32<T>(gr[c]) * (weight != nullptr ? to_f32<W>(weight[c]) : 1.f);
    const float z = (to_f32<T>(xr[c]) - mean) * rstd;
    dx[row * hidden + c] = from_f32<T>(rstd * (g - m0 - z * m1));
  }
}

// dw / db of one range of rows per block row: a thread per column, rows in ascending order
template <typename T>
__global__ void __launch_bounds__(LN_T)
layernorm_bwd_cols_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy, int64_t dy_stride,
                          const float* __restrict__ mean_in, const float* __restrict__ rstd_in, int64_t n_rows, int hidden,
                          int64_t rows_per_part, float* __restrict__ partial) {
  const int c = blockIdx.y * LN_T + threadIdx.x;
  if (c >= hidden) return;
  const int64_t r0 = blockIdx.x * rows_per_part, r1 = r0 + rows_per_part < n_rows ? r0 + rows_per_part : n_rows;
  float dw = 0.f, db = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = to_f32<T>(dy[r * dy_stride + c]);
    db += g;
    dw = fmaf(g, (to_f32<T>(x[r * x_stride + c]) - mean_in[r]) * rstd_in[r], dw);
  }
  float* p = partial + (int64_t)blockIdx.x * 2 * hidden;
  p[c] = dw;
  p[hidden + c] = db;
}

// sums the partial rows of 32 columns: 32 lanes of columns x 8 warps of row ranges, joined in a fixed order
template <typename W>
__global__ void __launch_bounds__(256)
layernorm_dparam_kernel(const float* __restrict__ partial, int n_parts, int hidden, W* __restrict__ dweight,
                        W* __restrict__ dbias) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int which = blockIdx.y;                 // 0: dweight, 1: dbias
  W* dst = which == 0 ? dweight : dbias;
  if (dst == nullptr) return;                   // the whole block
  float s = 0.f;
  if (c < hidden)
    for (int p = warp; p < n_parts; p += 8) s += partial[((int64_t)p * 2 + which) * hidden + c];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < hidden) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[w][lane];
    dst[c] = from_f32<W>(s);
  }
}

constexpr int LN_MAX_PARTS = 592;
static int64_t ln_parts(int64_t n_rows) { return n_rows < LN_MAX_PARTS ? n_rows : LN_MAX_PARTS; }

template <typename T, typename W>
static int layernorm_fwd_t(const void* x, int64_t x_stride, const void* weight, const void* bias, float eps, int64_t n_rows,
                           int hidden, void* out, float* mean, float* rstd, cudaStream_t st) {
  layernorm_loop_kernel<T, W><<<(unsigned)n_rows, LN_T, 0, st>>>(
      static_cast<const T*>(x), x_stride, static_cast<const W*>(weight), static_cast<const W*>(bias), eps, hidden,
      static_cast<T*>(out), mean, rstd);
  BIBO_CHECK_LAUNCH("layernorm_loop_kernel");
  return BIBO_OK;
}

template <typename T, typename W>
static int layernorm_bwd_t(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                           const float* mean, const float* rstd, int64_t n_rows, int hidden, void* dx, float* partial,
                           void* dweight, void* dbias, cudaStream_t st) {
  layernorm_bwd_dx_loop_kernel<T, W><<<(unsigned)n_rows, LN_T, 0, st>>>(
      static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride, static_cast<const W*>(weight), mean, rstd,
      hidden, static_cast<T*>(dx));
  BIBO_CHECK_LAUNCH("layernorm_bwd_dx_loop_kernel");
  if (dweight == nullptr && dbias == nullptr) return BIBO_OK;
  const int64_t parts = ln_parts(n_rows), per = (n_rows + parts - 1) / parts;
  const int used = (int)((n_rows + per - 1) / per);
  layernorm_bwd_cols_kernel<T><<<dim3(used, (hidden + LN_T - 1) / LN_T), LN_T, 0, st>>>(
      static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride, mean, rstd, n_rows, hidden, per, partial);
  BIBO_CHECK_LAUNCH("layernorm_bwd_cols_kernel");
  layernorm_dparam_kernel<W><<<dim3((hidden + 31) / 32, 2), 256, 0, st>>>(partial, used, hidden, static_cast<W*>(dweight),
                                                                        static_cast<W*>(dbias));
  BIBO_CHECK_LAUNCH("layernorm_dparam_kernel");
  return BIBO_OK;
}

static int layernorm_check(const char* what, int64_t n_rows, int hidden, int dtype, int wdtype, int64_t stride) {
  if (dtype != BIBO_F32 && dtype != BIBO_BF16) return fail(BIBO_ERR_ARG, "%s: dtype=%d", what, dtype);
  if (wdtype != BIBO_F32 && wdtype != dtype)
    return fail(BIBO_ERR_ARG, "%s: weight dtype=%d beside activations of dtype=%d", what, wdtype, dtype);
  if (hidden < 1) return fail(BIBO_ERR_ARG, "%s: hidden=%d", what, hidden);
  if (n_rows > 0x7fffffffll) return fail(BIBO_ERR_UNSUPPORTED, "%s: %lld rows", what, (long long)n_rows);
  if (stride < hidden) return fail(BIBO_ERR_ARG, "%s: row stride %lld below hidden=%d", what, (long long)stride, hidden);
  return BIBO_OK;
}

}  // namespace bibo

using namespace bibo;

extern "C" int bibo_moe_layernorm_fwd(const void* x, int64_t x_stride, const void* weight, const void* bias, float eps,
                                      int64_t n_rows, int hidden, int dtype, int wdtype, void* out, float* mean, float* rstd,
                                      void* stream) {
  const int rc = layernorm_check("layernorm_fwd", n_rows, hidden, dtype, wdtype, n_rows > 1 ? x_stride : hidden);
  if (rc) return rc;
  if (n_rows <= 0) return BIBO_OK;
  if (!x || !out || (mean == nullptr) != (rstd == nullptr)) return fail(BIBO_ERR_ARG, "layernorm_fwd: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == BIBO_F32)
    return layernorm_fwd_t<float, float>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st);
  if (wdtype == BIBO_F32)
    return layernorm_fwd_t<__nv_bfloat16, float>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st);
  return layernorm_fwd_t<__nv_bfloat16, __nv_bfloat16>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st);
}

extern "C" int64_t bibo_moe_layernorm_bwd_parts(int64_t n_rows) { return n_rows > 0 ? ln_parts(n_rows) : 0; }

extern "C" int bibo_moe_layernorm_bwd(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                                      const float* mean, const float* rstd, int64_t n_rows, int hidden, int dtype,
                                      int wdtype, void* dx, float* partial, void* dweight, void* dbias, void* stream) {
  int rc = layernorm_check("layernorm_bwd", n_rows, hidden, dtype, wdtype, n_rows > 1 ? x_stride : hidden);
  if (!rc) rc = layernorm_check("layernorm_bwd", n_rows, hidden, dtype, wdtype, n_rows > 1 ? dy_stride : hidden);
  if (rc) return rc;
  if (n_rows <= 0) return BIBO_OK;      // the caller's dweight / dbias are sums over no rows: it zeroes them itself
  if (!x || !dy || !mean || !rstd || !dx || ((dweight || dbias) && !partial))
    return fail(BIBO_ERR_ARG, "layernorm_bwd: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == BIBO_F32)
    return layernorm_bwd_t<float, float>(x, x_stride, dy, dy_stride, weight, mean, rstd, n_rows, hidden, dx, partial, dweight,
                                         dbias, st);
  if (wdtype == BIBO_F32)
    return layernorm_bwd_t<__nv_bfloat16, float>(x, x_stride, dy, dy_stride, weight, mean, rstd, n_rows, hidden, dx, partial,
                                                 dweight, dbias, st);
  return layernorm_bwd_t<__nv_bfloat16, __nv_bfloat16>(x, x_stride, dy, dy_stride, weight, mean, rstd, n_rows, hidden, dx,
                                                       partial, dweight, dbias, st);
}
