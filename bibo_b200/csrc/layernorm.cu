// Layer norm over the last dimension, forward and backward, beside the RMSNorm of rmsnorm.cu:
//   mean = sum(x)/H, var = sum((x-mean)^2)/H, rstd = 1/sqrt(var+eps), xhat = (x-mean)*rstd
//   y  = xhat*w + b
//   g  = dy*w;  dx = rstd*(g - mean(g) - xhat*mean(g*xhat));  dw = sum over rows of dy*xhat;  db = sum over rows of dy
// Everything is held in fp32 and rounded once, at the store.  The variance is taken around the mean in a second
// pass over the row: E[x^2] - mean^2 loses it where the mean is large against the spread.
#include "tc_common.cuh"

namespace bibo {

// ---- rows held in registers ------------------------------------------------------------------------------------
// VE elements per access: 16 bytes where rows, strides and pointers allow it, else 4 (bf16 pairs) or one element.
template <typename T, int VE> struct LnVec;
template <> struct LnVec<float, 4> {
  using V = uint4;
  static __device__ __forceinline__ void unpack(const V& v, float* f) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ V pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct LnVec<float, 1> {
  using V = float;
  static __device__ __forceinline__ void unpack(const V& v, float* f) { f[0] = v; }
  static __device__ __forceinline__ V pack(const float* f) { return f[0]; }
};
template <> struct LnVec<__nv_bfloat16, 8> {
  using V = uint4;
  static __device__ __forceinline__ void unpack(const V& v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ V pack(const float* f) {
    V v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return v;
  }
};
template <> struct LnVec<__nv_bfloat16, 2> {
  using V = uint32_t;
  static __device__ __forceinline__ void unpack(const V& v, float* f) {
    f[0] = __uint_as_float(v << 16); f[1] = __uint_as_float(v & 0xffff0000u);
  }
  static __device__ __forceinline__ V pack(const float* f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const V*>(&h);
  }
};
template <> struct LnVec<__nv_bfloat16, 1> {
  using V = __nv_bfloat16;
  static __device__ __forceinline__ void unpack(const V& v, float* f) { f[0] = __bfloat162float(v); }
  static __device__ __forceinline__ V pack(const float* f) { return __float2bfloat16_rn(f[0]); }
};
// VE parameters [c * VE, (c + 1) * VE) as fp32
template <typename W, int VE> __device__ __forceinline__ void ln_param(const W* __restrict__ w, int c, float* f) {
  if constexpr (VE == 8 && sizeof(W) == 4) {
    LnVec<float, 4>::unpack(__ldg(reinterpret_cast<const uint4*>(w) + 2 * c), f);
    LnVec<float, 4>::unpack(__ldg(reinterpret_cast<const uint4*>(w) + 2 * c + 1), f + 4);
  } else if constexpr (VE == 2 && sizeof(W) == 4) {
    const float2 v = __ldg(reinterpret_cast<const float2*>(w) + c);
    f[0] = v.x; f[1] = v.y;
  } else {
    using X = LnVec<W, VE>;
    X::unpack(reinterpret_cast<const typename X::V*>(w)[c], f);
  }
}

// sum over the G threads of a row: a warp or a part of it, or the block
template <int G> __device__ __forceinline__ float ln_row_sum(float a, float* red) {
#pragma unroll
  for (int o = G > 32 ? 16 : G / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
    a = 0.f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) a += red[w];
  }
  return a;
}

// Sums of N values over a block, in every thread.  Inside a warp the values are folded onto the lanes first (N - 1 + 5 - log2 N
// shuffles instead of 5 N), so that one barrier and one shared load per thread finish the job.
template <int N, int WARPS> __device__ __forceinline__ void ln_block_sums(float (&s)[N], float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int off = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2, off /= 2) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float keep = up ? s[i + n / 2] : s[i], give = up ? s[i] : s[i + n / 2];
      s[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
    }
  }
  for (; off > 0; off /= 2) s[0] += __shfl_xor_sync(0xffffffffu, s[0], off);
  // lane's value: the bits of the lane number that were folded, the first fold being the value's highest bit
  if ((lane & (32 / N - 1)) == 0) red[warp * N + lane / (32 / N)] = s[0];
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < (WARPS * N + 31) / 32; ++i)
    if (i * 32 + lane < WARPS * N) t += red[i * 32 + lane];
#pragma unroll
  for (int o = N; o < 32; o *= 2) t += __shfl_xor_sync(0xffffffffu, t, o);
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = __shfl_sync(0xffffffffu, t, k);
}

// Forward of any alignment, and of few or short rows: G threads per row (32 and fewer: 256 / G sets of R rows a block), CH accesses per
// thread; one read and one write of a row.
template <typename T, typename W, int VE, int G, int CH, int R>
__global__ void __launch_bounds__(G > 32 ? G : 256)
layernorm_kernel(const T* __restrict__ x, int64_t x_stride, const W* __restrict__ weight, const W* __restrict__ bias, float eps,
                 int64_t n_rows, int hidden, T* __restrict__ out, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  static_assert(G <= 32 || R == 1, "a block has one row");
  using X = LnVec<T, VE>;
  using V = typename X::V;
  __shared__ float red[2][G > 32 ? G / 32 : 1];
  const int lane = threadIdx.x % G;
  const int64_t row0 = G > 32 ? blockIdx.x : ((int64_t)blockIdx.x * (256 / G) + threadIdx.x / G) * R;
  const int vecs = hidden / VE;
  const float inv = 1.f / (float)hidden;
  V v[R][CH];
  float mean[R], rstd[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const V* src = reinterpret_cast<const V*>(x + (row0 + r < n_rows ? row0 + r : 0) * x_stride);
#pragma unroll
    for (int q = 0; q < CH; ++q)
      if (q * G + lane < vecs) v[r][q] = __ldcs(src + q * G + lane);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < CH; ++q)
      if (q * G + lane < vecs) {
        float f[VE];
        X::unpack(v[r][q], f);
#pragma unroll
        for (int i = 0; i < VE; ++i) s += f[i];
      }
    mean[r] = ln_row_sum<G>(s, red[0]) * inv;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < CH; ++q)
      if (q * G + lane < vecs) {
        float f[VE];
        X::unpack(v[r][q], f);
#pragma unroll
        for (int i = 0; i < VE; ++i) { const float d = f[i] - mean[r]; s = fmaf(d, d, s); }
      }
    rstd[r] = rsqrtf(fmaf(ln_row_sum<G>(s, red[1]), inv, eps));
    if (lane == 0 && mean_out != nullptr && row0 + r < n_rows) { mean_out[row0 + r] = mean[r]; rstd_out[row0 + r] = rstd[r]; }
  }
#pragma unroll
  for (int q = 0; q < CH; ++q)
    if (q * G + lane < vecs) {
      const int c = q * G + lane;
      float w[VE], b[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) { w[i] = 1.f; b[i] = 0.f; }
      if (weight != nullptr) ln_param<W, VE>(weight, c, w);
      if (bias != nullptr) ln_param<W, VE>(bias, c, b);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row0 + r >= n_rows) continue;
        float f[VE];
        X::unpack(v[r][q], f);
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] = fmaf((f[i] - mean[r]) * rstd[r], w[i], b[i]);
        reinterpret_cast<V*>(out + (row0 + r) * hidden)[c] = X::pack(f);
      }
    }
}

// Backward: a block of NT threads walks over groups of R rows; a thread owns CH x VE columns, whose weight and bias gradients it
// carries in registers over all its rows.  The 2 R row sums of a group cross the block at once: one barrier per R rows.
// Each block leaves one row of partial sums; layernorm_dparam_kernel adds them in a fixed order.
template <typename T, typename W, int VE, int NT, int CH, int R>
__global__ void __launch_bounds__(NT)
layernorm_bwd_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy, int64_t dy_stride,
                     const W* __restrict__ weight, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                     int64_t n_rows, int hidden, T* __restrict__ dx, float* __restrict__ partial, W* __restrict__ dweight,
                     W* __restrict__ dbias) {
  using X = LnVec<T, VE>;
  using V = typename X::V;
  constexpr int WARPS = NT / 32;
  __shared__ float red[2][WARPS * 2 * R];
  const int tid = threadIdx.x;
  tc::pdl_launch_next();                   // layernorm_dparam_kernel may take its place beside this one and wait
  const int vecs = hidden / VE;
  const float inv = 1.f / (float)hidden;
  float dw[CH][VE], db[CH][VE];
#pragma unroll
  for (int q = 0; q < CH; ++q)
#pragma unroll
    for (int i = 0; i < VE; ++i) dw[q][i] = db[q][i] = 0.f;
  // the parameters of a thread's columns stay in registers where they are few
  constexpr bool KEEP = CH * VE <= 8;
  float wk[KEEP ? CH : 1][VE];
  auto param = [&](int q, float* w) {
#pragma unroll
    for (int i = 0; i < VE; ++i) w[i] = 1.f;
    if (weight != nullptr && q * NT + tid < vecs) ln_param<W, VE>(weight, q * NT + tid, w);
  };
  if (KEEP)
#pragma unroll
    for (int q = 0; q < CH; ++q) param(q, wk[KEEP ? q : 0]);
  int buf = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < n_rows; row0 += (int64_t)gridDim.x * R, buf ^= 1) {
    V xv[R][CH], gv[R][CH];
    float mean[R], rstd[R], s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = row0 + r < n_rows;
      const V* xs = reinterpret_cast<const V*>(x + (row0 + r) * x_stride);
      const V* gs = reinterpret_cast<const V*>(dy + (row0 + r) * dy_stride);
      mean[r] = in ? mean_in[row0 + r] : 0.f;
      rstd[r] = in ? rstd_in[row0 + r] : 0.f;
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int c = q * NT + tid;
        if (in && c < vecs) { xv[r][q] = __ldcs(xs + c); gv[r][q] = __ldcs(gs + c); }
        else { xv[r][q] = V{}; gv[r][q] = V{}; }          // adds nothing anywhere
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float a = 0.f, b = 0.f;
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        float f[VE], g[VE], w[VE];
        X::unpack(xv[r][q], f);
        X::unpack(gv[r][q], g);
        if (KEEP)
#pragma unroll
          for (int i = 0; i < VE; ++i) w[i] = wk[KEEP ? q : 0][i];
        else param(q, w);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float z = (f[i] - mean[r]) * rstd[r], gw = g[i] * w[i];
          a += gw;
          b = fmaf(gw, z, b);
          dw[q][i] = fmaf(g[i], z, dw[q][i]);
          db[q][i] += g[i];
        }
      }
      s[2 * r] = a;
      s[2 * r + 1] = b;
    }
    ln_block_sums<2 * R, WARPS>(s, red[buf]);    // one barrier; the other buffer's readers are a full group behind
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= n_rows) continue;
      V* ds = reinterpret_cast<V*>(dx + (row0 + r) * hidden);
      const float m0 = s[2 * r] * inv, m1 = s[2 * r + 1] * inv;
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int c = q * NT + tid;
        if (c >= vecs) continue;
        float f[VE], g[VE], w[VE];
        X::unpack(xv[r][q], f);
        X::unpack(gv[r][q], g);
        if (KEEP)
#pragma unroll
          for (int i = 0; i < VE; ++i) w[i] = wk[KEEP ? q : 0][i];
        else param(q, w);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float z = (f[i] - mean[r]) * rstd[r];
          f[i] = rstd[r] * (fmaf(g[i], w[i], -m0) - z * m1);
        }
        ds[c] = X::pack(f);
      }
    }
  }
  if (gridDim.x == 1) {                          // the only block: its sums are the gradients
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int c = q * NT + tid;
      if (c >= vecs) continue;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        if (dweight != nullptr) dweight[c * VE + i] = from_f32<W>(dw[q][i]);
        if (dbias != nullptr) dbias[c * VE + i] = from_f32<W>(db[q][i]);
      }
    }
    return;
  }
  if (partial == nullptr) return;
  float* p = partial + (int64_t)blockIdx.x * 2 * hidden;
#pragma unroll
  for (int q = 0; q < CH; ++q) {
    const int c = q * NT + tid;
    if (c >= vecs) continue;
#pragma unroll
    for (int i = 0; i < VE; ++i) { p[c * VE + i] = dw[q][i]; p[hidden + c * VE + i] = db[q][i]; }
  }
}

// Backward of short rows: G lanes per row, a block of 256 threads walks over 256 / G rows at a time and R such sets, so a row's sums cross
// lanes only.  The lanes' weight and bias gradients are joined over the block's rows at the end, in a fixed order.  (With a block per
// row group, 592 blocks of two warps were all that the partial sums allow: 400000 x 128 bf16 took 208 us, 67 this way; x 64 203 and 37.)
constexpr int LN_N = 256;
template <typename T, typename W, int VE, int G, int CH, int R>
__global__ void __launch_bounds__(LN_N)
layernorm_bwd_short_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy, int64_t dy_stride,
                           const W* __restrict__ weight, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                           int64_t n_rows, int hidden, T* __restrict__ dx, float* __restrict__ partial, W* __restrict__ dweight,
                           W* __restrict__ dbias) {
  using X = LnVec<T, VE>;
  using V = typename X::V;
  constexpr int GROUPS = LN_N / G;
  __shared__ float red[2][GROUPS][G * CH * VE];
  const int lane = threadIdx.x % G, group = threadIdx.x / G, vecs = hidden / VE;
  tc::pdl_launch_next();                   // layernorm_dparam_kernel may take its place beside this one and wait
  const float inv = 1.f / (float)hidden;
  const int64_t total = (int64_t)gridDim.x * GROUPS, first = (int64_t)blockIdx.x * GROUPS + group;
  float w[CH][VE], dw[CH][VE], db[CH][VE];
#pragma unroll
  for (int q = 0; q < CH; ++q) {
#pragma unroll
    for (int i = 0; i < VE; ++i) { w[q][i] = 1.f; dw[q][i] = db[q][i] = 0.f; }
    if (weight != nullptr && q * G + lane < vecs) ln_param<W, VE>(weight, q * G + lane, w[q]);
  }
  for (int64_t base = 0; base < n_rows; base += total * R) {     // the same number of turns for every lane
    V xv[R][CH], gv[R][CH];
    float mean[R], rstd[R], a[R], b[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * total + first;
      const bool in = row < n_rows;
      const V* xs = reinterpret_cast<const V*>(x + (in ? row : 0) * x_stride);
      const V* gs = reinterpret_cast<const V*>(dy + (in ? row : 0) * dy_stride);
      mean[r] = in ? mean_in[row] : 0.f;
      rstd[r] = in ? rstd_in[row] : 0.f;
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int c = q * G + lane;
        if (in && c < vecs) { xv[r][q] = __ldcs(xs + c); gv[r][q] = __ldcs(gs + c); }
        else { xv[r][q] = V{}; gv[r][q] = V{}; }                 // adds nothing anywhere
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      a[r] = b[r] = 0.f;
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        float f[VE], g[VE];
        X::unpack(xv[r][q], f);
        X::unpack(gv[r][q], g);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float z = (f[i] - mean[r]) * rstd[r], gw = g[i] * w[q][i];
          a[r] += gw;
          b[r] = fmaf(gw, z, b[r]);
          dw[q][i] = fmaf(g[i], z, dw[q][i]);
          db[q][i] += g[i];
        }
      }
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        a[r] += __shfl_xor_sync(0xffffffffu, a[r], o);
        b[r] += __shfl_xor_sync(0xffffffffu, b[r], o);
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * total + first;
      if (row >= n_rows) continue;
      V* ds = reinterpret_cast<V*>(dx + row * hidden);
      const float m0 = a[r] * inv, m1 = b[r] * inv;
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int c = q * G + lane;
        if (c >= vecs) continue;
        float f[VE], g[VE];
        X::unpack(xv[r][q], f);
        X::unpack(gv[r][q], g);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float z = (f[i] - mean[r]) * rstd[r];
          f[i] = rstd[r] * (fmaf(g[i], w[q][i], -m0) - z * m1);
        }
        ds[c] = X::pack(f);
      }
    }
  }
  if (partial == nullptr && (gridDim.x > 1 || (dweight == nullptr && dbias == nullptr))) return;
#pragma unroll
  for (int q = 0; q < CH; ++q)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      red[0][group][(q * G + lane) * VE + i] = dw[q][i];
      red[1][group][(q * G + lane) * VE + i] = db[q][i];
    }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * hidden; j += LN_N) {
    const int which = j >= hidden, c = j - which * hidden;
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) s += red[which][g][c];
    if (gridDim.x > 1) {
      partial[(int64_t)blockIdx.x * 2 * hidden + j] = s;
    } else {                                       // the only block: its sums are the gradients
      W* dst = which ? dbias : dweight;
      if (dst != nullptr) dst[c] = from_f32<W>(s);
    }
  }
}

// Backward of 16-byte aligned rows: the same walk, with the rows brought into shared memory by bulk copies (a ring of one to eight
// groups in the block's share of 208 KB), and z and dy*w of the group kept in registers between the sums and the result.  Where the
// share holds one group only (fp32 rows at the wide end of some classes, as 768, 1024 and 2048 columns or 1024 forward) nothing runs
// ahead inside the block, and the SM's other blocks are what has loads in flight.  Arithmetic is in pairs (two fp32 per instruction).  32768 x 2048: 104 us with loads
// into registers (57 % of the issue slots, 64 KB in flight an SM), 73 us with the ring.
__device__ __forceinline__ float2 ln_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 ln_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 ln_mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ void ln_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(tc::smem_u32(dst)), "l"(src), "r"(bytes), "r"(tc::smem_u32(bar)) : "memory");
}

constexpr int LN_MAX_STAGES = 8;
// Forward of 16-byte aligned rows, many of them: a block walks over groups of R rows that bulk copies bring into a ring in shared
// memory, up to seven groups ahead where the ring holds as many (see above); a thread owns CH x VE columns, keeps their parameters in registers and a group's values
// between the two sums.  (A warp per row re-reads the parameters from L1 for every row: with fp32 parameters beside bf16 rows
// that is twice the row's own bytes, and 32768 x 2048 took 54.7 us with L1 at 78 %; two rows a warp, 58 us, lacked loads in flight.)
template <typename T, typename W, int NT, int CH, int R>
__global__ void __launch_bounds__(NT)
layernorm_ring_kernel(const T* __restrict__ x, int64_t x_stride, const W* __restrict__ weight, const W* __restrict__ bias, float eps,
                      int64_t n_rows, int hidden, int stages, T* __restrict__ out, float* __restrict__ mean_out,
                      float* __restrict__ rstd_out) {
  constexpr int VE = 16 / sizeof(T), P = VE / 2, WARPS = NT / 32;
  using X = LnVec<T, VE>;
  extern __shared__ __align__(16) unsigned char ring[];          // [stages][R][row]
  __shared__ float red[2][WARPS * R];
  __shared__ uint64_t full[LN_MAX_STAGES];
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const int tid = threadIdx.x, vecs = hidden / VE, row_bytes = hidden * (int)sizeof(T);
  const float inv = 1.f / (float)hidden;
  const int64_t step = (int64_t)gridDim.x * R, first = (int64_t)blockIdx.x * R;
  auto load = [&](int64_t row0, int st) {                        // thread 0
    const int rows = n_rows - row0 < R ? (int)(n_rows - row0) : R;
    tc::mbar_expect_tx(&full[st], rows * row_bytes);
    for (int r = 0; r < rows; ++r)
      ln_bulk_load(ring + ((size_t)st * R + r) * row_bytes, x + (row0 + r) * x_stride, row_bytes, &full[st]);
  };
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
    abort_s = 0;
    tc::fence_barrier_init();
    for (int i = 0; i < stages; ++i)
      if (first + i * step < n_rows) load(first + i * step, i);
  }
  float2 w[CH][P], b[CH][P];
#pragma unroll
  for (int q = 0; q < CH; ++q) {
    float f[VE], g[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) { f[i] = 1.f; g[i] = 0.f; }
    if (weight != nullptr && q * NT + tid < vecs) ln_param<W, VE>(weight, q * NT + tid, f);
    if (bias != nullptr && q * NT + tid < vecs) ln_param<W, VE>(bias, q * NT + tid, g);
#pragma unroll
    for (int i = 0; i < P; ++i) { w[q][i] = make_float2(f[2 * i], f[2 * i + 1]); b[q][i] = make_float2(g[2 * i], g[2 * i + 1]); }
  }
  __syncthreads();
  int st = 0;
  uint32_t phase = 0;
  for (int64_t row0 = first; row0 < n_rows; row0 += step) {
    float poison = 0.f;
    // where the copies did not arrive no number is left to stand
    if (!tc::mbar_wait(&full[st], phase, abort_flag)) poison = __int_as_float(0x7fffffff);
    const uint4* rows = reinterpret_cast<const uint4*>(ring + (size_t)st * R * row_bytes);
    float2 v[R][CH][P];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 a = make_float2(poison, 0.f);
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        float f[VE];
        const bool in = q * NT + tid < vecs && row0 + r < n_rows;
        if (in) X::unpack(rows[r * vecs + q * NT + tid], f);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          v[r][q][i] = in ? make_float2(f[2 * i], f[2 * i + 1]) : make_float2(0.f, 0.f);
          a = ln_add2(a, v[r][q][i]);
        }
      }
      s[r] = a.x + a.y;
    }
    ln_block_sums<R, WARPS>(s, red[0]);                          // its barrier: everybody has read this stage
    if (tid == 0 && row0 + stages * step < n_rows) load(row0 + stages * step, st);
    float mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = s[r] * inv;
      const float2 nm = make_float2(-mean[r], -mean[r]);
      float2 a = make_float2(0.f, 0.f);
#pragma unroll
      for (int q = 0; q < CH; ++q)
        if (q * NT + tid < vecs) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            v[r][q][i] = ln_add2(v[r][q][i], nm);
            a = ln_fma2(v[r][q][i], v[r][q][i], a);
          }
        }
      s[r] = a.x + a.y;
    }
    ln_block_sums<R, WARPS>(s, red[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= n_rows) continue;
      const float rstd = rsqrtf(fmaf(s[r], inv, eps));
      if (tid == 0 && mean_out != nullptr) { mean_out[row0 + r] = mean[r]; rstd_out[row0 + r] = rstd; }
      const float2 rs = make_float2(rstd, rstd);
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int c = q * NT + tid;
        if (c >= vecs) continue;
        float f[VE];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 d = ln_fma2(ln_mul2(v[r][q][i], rs), w[q][i], b[q][i]);
          f[2 * i] = d.x;
          f[2 * i + 1] = d.y;
        }
        reinterpret_cast<uint4*>(out + (row0 + r) * hidden)[c] = X::pack(f);
      }
    }
    if (++st == stages) { st = 0; phase ^= 1; }
  }
  if (*abort_flag)                                               // copies may still be in flight to this shared memory
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
}

template <typename T, typename W, int NT, int CH, int R>
__global__ void __launch_bounds__(NT)
layernorm_bwd_ring_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy, int64_t dy_stride,
                          const W* __restrict__ weight, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                          int64_t n_rows, int hidden, int stages, T* __restrict__ dx, float* __restrict__ partial, W* __restrict__ dweight,
                     W* __restrict__ dbias) {
  constexpr int VE = 16 / sizeof(T), P = VE / 2, WARPS = NT / 32;
  using X = LnVec<T, VE>;
  extern __shared__ __align__(16) unsigned char ring[];          // [stages][R][x row, dy row]
  __shared__ float red[2][WARPS * 2 * R];
  __shared__ uint64_t full[LN_MAX_STAGES];
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const int tid = threadIdx.x, vecs = hidden / VE, row_bytes = hidden * (int)sizeof(T);
  const float inv = 1.f / (float)hidden;
  tc::pdl_launch_next();                   // layernorm_dparam_kernel may take its place beside this one and wait
  const int64_t step = (int64_t)gridDim.x * R, first = (int64_t)blockIdx.x * R;
  auto load = [&](int64_t row0, int st) {                        // thread 0
    const int rows = n_rows - row0 < R ? (int)(n_rows - row0) : R;
    tc::mbar_expect_tx(&full[st], 2 * rows * row_bytes);
    unsigned char* dst = ring + (size_t)st * R * 2 * row_bytes;
    for (int r = 0; r < rows; ++r) {
      ln_bulk_load(dst + (2 * r) * row_bytes, x + (row0 + r) * x_stride, row_bytes, &full[st]);
      ln_bulk_load(dst + (2 * r + 1) * row_bytes, dy + (row0 + r) * dy_stride, row_bytes, &full[st]);
    }
  };
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
    abort_s = 0;
    tc::fence_barrier_init();
    for (int i = 0; i < stages; ++i)
      if (first + i * step < n_rows) load(first + i * step, i);
  }
  float2 w[CH][P], dw[CH][P], db[CH][P];
#pragma unroll
  for (int q = 0; q < CH; ++q) {
    float f[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = 1.f;
    if (weight != nullptr && q * NT + tid < vecs) ln_param<W, VE>(weight, q * NT + tid, f);
#pragma unroll
    for (int i = 0; i < P; ++i) { w[q][i] = make_float2(f[2 * i], f[2 * i + 1]); dw[q][i] = db[q][i] = make_float2(0.f, 0.f); }
  }
  float next_mean[R], next_rstd[R];
  auto stats = [&](int64_t row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = row0 + r < n_rows;
      next_mean[r] = in ? __ldg(mean_in + row0 + r) : 0.f;
      next_rstd[r] = in ? __ldg(rstd_in + row0 + r) : 0.f;       // 0: the row adds nothing
    }
  };
  stats(first);
  __syncthreads();
  int st = 0, buf = 0;
  uint32_t phase = 0;
  for (int64_t row0 = first; row0 < n_rows; row0 += step, buf ^= 1) {
    float mean[R], rstd[R], s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) { mean[r] = next_mean[r]; rstd[r] = next_rstd[r]; }
    stats(row0 + step);                                          // a group ahead of their use
    if (!tc::mbar_wait(&full[st], phase, abort_flag)) {           // the copies did not arrive: no number is left to stand
#pragma unroll
      for (int r = 0; r < R; ++r) rstd[r] = __int_as_float(0x7fffffff);
    }
    const uint4* rows = reinterpret_cast<const uint4*>(ring + (size_t)st * R * 2 * row_bytes);
    float2 z[R][CH][P], gw[R][CH][P];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 a = make_float2(0.f, 0.f), b = a;
      const float2 rs = make_float2(rstd[r], rstd[r]), nm = make_float2(-mean[r], -mean[r]);
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int c = q * NT + tid;
        float f[VE], g[VE];
        if (c < vecs && row0 + r < n_rows) {
          X::unpack(rows[(2 * r) * vecs + c], f);
          X::unpack(rows[(2 * r + 1) * vecs + c], g);
        } else {
#pragma unroll
          for (int i = 0; i < VE; ++i) { f[i] = mean[r]; g[i] = 0.f; }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 g2 = make_float2(g[2 * i], g[2 * i + 1]);
          z[r][q][i] = ln_mul2(ln_add2(make_float2(f[2 * i], f[2 * i + 1]), nm), rs);
          gw[r][q][i] = ln_mul2(g2, w[q][i]);
          a = ln_add2(a, gw[r][q][i]);
          b = ln_fma2(gw[r][q][i], z[r][q][i], b);
          dw[q][i] = ln_fma2(g2, z[r][q][i], dw[q][i]);
          db[q][i] = ln_add2(db[q][i], g2);
        }
      }
      s[2 * r] = a.x + a.y;
      s[2 * r + 1] = b.x + b.y;
    }
    // one barrier: everybody has read this stage; the other buffer's readers are a full group behind
    ln_block_sums<2 * R, WARPS>(s, red[buf]);
    if (tid == 0 && row0 + stages * step < n_rows) load(row0 + stages * step, st);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (row0 + r >= n_rows) continue;
      const float2 rs = make_float2(rstd[r], rstd[r]);
      const float2 m0 = make_float2(-s[2 * r] * inv, -s[2 * r] * inv), m1 = make_float2(-s[2 * r + 1] * inv, -s[2 * r + 1] * inv);
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int c = q * NT + tid;
        if (c >= vecs) continue;
        float f[VE];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 d = ln_mul2(rs, ln_fma2(z[r][q][i], m1, ln_add2(gw[r][q][i], m0)));
          f[2 * i] = d.x;
          f[2 * i + 1] = d.y;
        }
        reinterpret_cast<uint4*>(dx + (row0 + r) * hidden)[c] = X::pack(f);
      }
    }
    if (++st == stages) { st = 0; phase ^= 1; }
  }
  if (gridDim.x == 1) {                          // the only block: its sums are the gradients
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int c = (q * NT + tid) * VE;
      if (c >= hidden) continue;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        if (dweight != nullptr) dweight[c + i] = from_f32<W>(i & 1 ? dw[q][i / 2].y : dw[q][i / 2].x);
        if (dbias != nullptr) dbias[c + i] = from_f32<W>(i & 1 ? db[q][i / 2].y : db[q][i / 2].x);
      }
    }
  } else if (partial != nullptr) {
    float* p = partial + (int64_t)blockIdx.x * 2 * hidden;
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int c = q * NT + tid;
      if (c >= vecs) continue;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        reinterpret_cast<float2*>(p + c * VE)[i] = dw[q][i];
        reinterpret_cast<float2*>(p + hidden + c * VE)[i] = db[q][i];
      }
    }
  }
  if (*abort_flag)                                               // copies may still be in flight to this shared memory
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
}

constexpr int LN_MAX_PARTS = 592;
constexpr int LN_ONE_BLOCK = 16;     // up to as many rows one block takes all, without partial sums and their launch
static int64_t ln_parts(int64_t n_rows) { return n_rows <= LN_ONE_BLOCK ? 0 : n_rows < LN_MAX_PARTS ? n_rows : LN_MAX_PARTS; }

// the widest access that rows of `hidden` elements of `size` bytes allow at these addresses; strides in elements (0: one row)
static int ln_access(int hidden, int size, int wsize, int64_t s0, int64_t s1, const void* a, const void* b, const void* c, const void* w,
                     const void* bias) {
  const uintptr_t all = (uintptr_t)((int64_t)hidden * size) | (uintptr_t)(s0 * size) | (uintptr_t)(s1 * size) |
                        reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c);
  const uintptr_t par = reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(bias);
  if ((all & 15) == 0 && (par & 15) == 0) return 16 / size;
  if (size == 2 && (all & 3) == 0 && (par & (2 * wsize - 1)) == 0) return 2;
  return 1;
}

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
template <typename T, typename W>
__global__ void __launch_bounds__(LN_T)
layernorm_bwd_cols_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy, int64_t dy_stride,
                          const float* __restrict__ mean_in, const float* __restrict__ rstd_in, int64_t n_rows, int hidden,
                          int64_t rows_per_part, float* __restrict__ partial, W* __restrict__ dweight, W* __restrict__ dbias) {
  const int c = blockIdx.y * LN_T + threadIdx.x;
  if (c >= hidden) return;
  const int64_t r0 = blockIdx.x * rows_per_part, r1 = r0 + rows_per_part < n_rows ? r0 + rows_per_part : n_rows;
  float dw = 0.f, db = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = to_f32<T>(dy[r * dy_stride + c]);
    db += g;
    dw = fmaf(g, (to_f32<T>(x[r * x_stride + c]) - mean_in[r]) * rstd_in[r], dw);
  }
  if (gridDim.x == 1) {
    if (dweight != nullptr) dweight[c] = from_f32<W>(dw);
    if (dbias != nullptr) dbias[c] = from_f32<W>(db);
    return;
  }
  float* p = partial + (int64_t)blockIdx.x * 2 * hidden;
  p[c] = dw;
  p[hidden + c] = db;
}

// sums the partial rows of 32 columns: 32 lanes of columns x 32 warps of rows, joined in a fixed order
template <typename W>
__global__ void __launch_bounds__(1024)
layernorm_dparam_kernel(const float* __restrict__ partial, int n_parts, int hidden, W* __restrict__ dweight,
                        W* __restrict__ dbias) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int which = blockIdx.y;                 // 0: dweight, 1: dbias
  W* dst = which == 0 ? dweight : dbias;
  if (dst == nullptr) return;                   // the whole block
  tc::pdl_wait();
  float s = 0.f;
  if (c < hidden) {
    const float* p = partial + (int64_t)which * hidden + c;
    int r = warp;
    for (; r + 96 < n_parts; r += 128) {        // four loads in flight
      const float v0 = p[(int64_t)r * 2 * hidden], v1 = p[(int64_t)(r + 32) * 2 * hidden];
      const float v2 = p[(int64_t)(r + 64) * 2 * hidden], v3 = p[(int64_t)(r + 96) * 2 * hidden];
      s += (v0 + v1) + (v2 + v3);
    }
    for (; r < n_parts; r += 32) s += p[(int64_t)r * 2 * hidden];
  }
  red[warp][lane] = s;
  __syncthreads();
  s = red[lane][warp];                          // column `warp`, parts of warp `lane`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0 && blockIdx.x * 32 + warp < hidden) dst[blockIdx.x * 32 + warp] = from_f32<W>(s);
}

template <typename T, typename W, int VE>
static int layernorm_fwd_v(const void* x, int64_t x_stride, const void* weight, const void* bias, float eps, int64_t n_rows,
                           int hidden, void* out, float* mean, float* rstd, cudaStream_t st) {
  const int vecs = hidden / VE;
#define BIBO_LN_FWD(G, CH, R)                                                                                                    \
  layernorm_kernel<T, W, VE, G, CH, R><<<(unsigned)(G > 32 ? n_rows : (n_rows + 256 / G * (R) - 1) / (256 / G * (R))), G > 32 ? G : 256, 0, st>>>( \
      static_cast<const T*>(x), x_stride, static_cast<const W*>(weight), static_cast<const W*>(bias), eps, n_rows, hidden,       \
      static_cast<T*>(out), mean, rstd)
  // Warps with rows of their own need no barrier; a block per row where the row is longer than eight accesses of a warp, or
  // where the rows are too few to fill the machine with warps (eight rows of 2048: one access a thread).
  // Short rows share a warp, two rows a thread: 400000 x 64 bf16 90 -> 20 us, x 128 93 -> 41 us (one row: 24 and 49, four: 22 and 49).
  const bool few = n_rows <= 4 * (int64_t)sm_count() && vecs > 64;
  if (vecs <= 8) BIBO_LN_FWD(8, 1, 2);
  else if (vecs <= 16) BIBO_LN_FWD(16, 1, 2);
  else if (!few && vecs <= 32) BIBO_LN_FWD(32, 1, 2);
  else if (!few && vecs <= 64) BIBO_LN_FWD(32, 2, VE * sizeof(T) == 16 ? 1 : 2);
  else if (!few && vecs <= 128) BIBO_LN_FWD(32, 4, 1);
  else if (!few && vecs <= 256) BIBO_LN_FWD(32, 8, 1);
  else if (vecs <= 256) BIBO_LN_FWD(256, 1, 1);
  else if (vecs <= 512) BIBO_LN_FWD(256, 2, 1);
  else if (vecs <= 1024) BIBO_LN_FWD(256, 4, 1);
  else if (vecs <= 2048) BIBO_LN_FWD(256, 8, 1);
  else if (vecs <= 8192) BIBO_LN_FWD(1024, 8, 1);
  else
    layernorm_loop_kernel<T, W><<<(unsigned)n_rows, LN_T, 0, st>>>(
        static_cast<const T*>(x), x_stride, static_cast<const W*>(weight), static_cast<const W*>(bias), eps, hidden,
        static_cast<T*>(out), mean, rstd);
#undef BIBO_LN_FWD
  BIBO_CHECK_LAUNCH("layernorm_kernel");
  return BIBO_OK;
}

template <typename T, typename W, int NT, int CH, int R, int CTAS>
static int layernorm_fwd_ring(const void* x, int64_t x_stride, const void* weight, const void* bias, float eps, int64_t n_rows,
                              int hidden, void* out, float* mean, float* rstd, cudaStream_t st) {
  auto kern = layernorm_ring_kernel<T, W, NT, CH, R>;
  constexpr int RING = 208 * 1024 / CTAS;        // CTAS blocks share an SM
  static DeviceOnce once;
  int per_sm = 1;                                // blocks that are resident: registers may allow fewer than CTAS
  const int rc = once.get([&](int* v) {
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING));
    BIBO_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(v, kern, NT, RING));
    return (int)BIBO_OK;
  }, &per_sm);
  if (rc) return rc;
  const int group = R * hidden * (int)sizeof(T);
  int64_t grid = (n_rows + R - 1) / R;
  if (grid > per_sm * (int64_t)sm_count()) grid = per_sm * (int64_t)sm_count();
  int stages = RING / group;
  if (stages > LN_MAX_STAGES) stages = LN_MAX_STAGES;
  kern<<<(unsigned)grid, NT, stages * group, st>>>(static_cast<const T*>(x), x_stride, static_cast<const W*>(weight),
                                                   static_cast<const W*>(bias), eps, n_rows, hidden, stages, static_cast<T*>(out),
                                                   mean, rstd);
  BIBO_CHECK_LAUNCH("layernorm_ring_kernel");
  return BIBO_OK;
}

template <typename T, typename W>
static int layernorm_fwd_t(const void* x, int64_t x_stride, const void* weight, const void* bias, float eps, int64_t n_rows,
                           int hidden, void* out, float* mean, float* rstd, cudaStream_t st) {
  const int ve = ln_access(hidden, sizeof(T), sizeof(W), n_rows > 1 ? x_stride : 0, 0, x, out, nullptr, weight, bias);
  // Threads of 16 columns, as few as cover the row in steps of 1.5 and 1.33 (idle ones cost issue slots: 2560 columns on 256 threads
  // ran at 0.67 of the copy rate, on 192 at 0.91); pieces of 16 bytes a thread, rows a group, blocks an SM.  bf16 rows with
  // fp32 parameters, 537 MB read and written, of the copy rate: 1024 0.83, 1280 0.89, 2048 0.85, 2560 0.91, 4096 0.93, 5120 0.85,
  // 7168 0.91; fp32 0.85 to 0.91.  Longer fp32 rows need no ring (0.91 to 0.95; 0.85 with it).  Below eight rows an SM a
  // ring has nothing to run ahead of.
  if (ve * sizeof(T) == 16 && n_rows > 8 * (int64_t)sm_count()) {
    constexpr int VE = 16 / sizeof(T), C16 = 16 / VE;                 // pieces of 16 bytes for 16 columns a thread
#define BIBO_LN_RING(...) return layernorm_fwd_ring<T, W, __VA_ARGS__>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st)
    if (hidden > 512 && hidden <= 64 * 16) BIBO_LN_RING(64, C16, 4, 8);
    if (hidden > 64 * 16 && hidden <= 96 * 16) BIBO_LN_RING(96, C16, 4, 4);
    if (hidden > 96 * 16 && hidden <= 128 * 16) BIBO_LN_RING(128, C16, 4, 3);
    if (hidden > 128 * 16 && hidden <= 192 * 16) BIBO_LN_RING(192, C16, 4, 3);
    if (hidden > 192 * 16 && hidden <= 256 * 16) BIBO_LN_RING(256, C16, 2, 2);
    if constexpr (sizeof(T) == 2) {
      if (hidden > 256 * 16 && hidden <= 384 * 16) BIBO_LN_RING(384, C16, 4, 1);
      if (hidden > 384 * 16 && hidden <= 512 * 16) BIBO_LN_RING(512, C16, 4, 1);
    }
#undef BIBO_LN_RING
  }
  if constexpr (sizeof(T) == 2) {
    if (ve == 8) return layernorm_fwd_v<T, W, 8>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st);
    if (ve == 2) return layernorm_fwd_v<T, W, 2>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st);
  } else {
    if (ve == 4) return layernorm_fwd_v<T, W, 4>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st);
  }
  return layernorm_fwd_v<T, W, 1>(x, x_stride, weight, bias, eps, n_rows, hidden, out, mean, rstd, st);
}

template <typename T, typename W, int VE, int NT, int CH, int R>
static int layernorm_bwd_v(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                           const float* mean, const float* rstd, int64_t n_rows, int hidden, void* dx, float* partial,
                           void* dweight, void* dbias, int* parts, cudaStream_t st) {
  auto kern = layernorm_bwd_kernel<T, W, VE, NT, CH, R>;
  static DeviceOnce once;
  int per_sm = 1;
  const int rc = once.get([&](int* v) {
    BIBO_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(v, kern, NT, 0));
    return (int)BIBO_OK;
  }, &per_sm);
  if (rc) return rc;
  int64_t grid = n_rows <= LN_ONE_BLOCK ? 1 : (n_rows + R - 1) / R;
  const int64_t fit = (int64_t)sm_count() * (per_sm > 0 ? per_sm : 1);
  if (grid > fit) grid = fit;
  if (grid > LN_MAX_PARTS) grid = LN_MAX_PARTS;
  kern<<<(unsigned)grid, NT, 0, st>>>(static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride,
                                      static_cast<const W*>(weight), mean, rstd, n_rows, hidden, static_cast<T*>(dx), partial,
                                      static_cast<W*>(dweight), static_cast<W*>(dbias));
  BIBO_CHECK_LAUNCH("layernorm_bwd_kernel");
  *parts = (int)grid;
  return BIBO_OK;
}

template <typename T, typename W, int NT, int CH, int R, int CTAS>
static int layernorm_bwd_ring(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                              const float* mean, const float* rstd, int64_t n_rows, int hidden, void* dx, float* partial,
                              void* dweight, void* dbias, int* parts, cudaStream_t st) {
  auto kern = layernorm_bwd_ring_kernel<T, W, NT, CH, R>;
  constexpr int RING = 208 * 1024 / CTAS;        // CTAS blocks share an SM
  static DeviceOnce once;
  int per_sm = 1;                                // blocks that are resident: registers may allow fewer than CTAS
  const int rc = once.get([&](int* v) {
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING));
    BIBO_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(v, kern, NT, RING));
    return (int)BIBO_OK;
  }, &per_sm);
  if (rc) return rc;
  const int group = R * 2 * hidden * (int)sizeof(T);
  int64_t grid = n_rows <= LN_ONE_BLOCK ? 1 : (n_rows + R - 1) / R;
  if (grid > per_sm * (int64_t)sm_count()) grid = per_sm * (int64_t)sm_count();
  if (grid > LN_MAX_PARTS) grid = LN_MAX_PARTS;
  int stages = RING / group;
  if (stages > LN_MAX_STAGES) stages = LN_MAX_STAGES;
  kern<<<(unsigned)grid, NT, stages * group, st>>>(static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride,
                                                   static_cast<const W*>(weight), mean, rstd, n_rows, hidden, stages,
                                                   static_cast<T*>(dx), partial, static_cast<W*>(dweight), static_cast<W*>(dbias));
  BIBO_CHECK_LAUNCH("layernorm_bwd_ring_kernel");
  *parts = (int)grid;
  return BIBO_OK;
}

template <typename T, typename W, int VE, int G, int CH, int R>
static int layernorm_bwd_short(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                               const float* mean, const float* rstd, int64_t n_rows, int hidden, void* dx, float* partial,
                               void* dweight, void* dbias, int* parts, cudaStream_t st) {
  int64_t grid = n_rows <= LN_ONE_BLOCK ? 1 : (n_rows + LN_N / G - 1) / (LN_N / G);
  if (grid > 4 * (int64_t)sm_count()) grid = 4 * (int64_t)sm_count();
  if (grid > LN_MAX_PARTS) grid = LN_MAX_PARTS;
  layernorm_bwd_short_kernel<T, W, VE, G, CH, R><<<(unsigned)grid, LN_N, 0, st>>>(
      static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride, static_cast<const W*>(weight), mean, rstd, n_rows,
      hidden, static_cast<T*>(dx), partial, static_cast<W*>(dweight), static_cast<W*>(dbias));
  BIBO_CHECK_LAUNCH("layernorm_bwd_short_kernel");
  *parts = (int)grid;
  return BIBO_OK;
}

// columns per thread and rows per group: as many loads in flight as the registers hold beside the 2 CH VE column sums
template <typename T, typename W, int VE>
static int layernorm_bwd_pick(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                              const float* mean, const float* rstd, int64_t n_rows, int hidden, void* dx, float* partial,
                              void* dweight, void* dbias, int* parts, bool* done, cudaStream_t st) {
  const int vecs = hidden / VE;
  *done = true;
  if constexpr (VE * sizeof(T) == 16) {
    constexpr int C8 = 8 / VE, C16 = 16 / VE;    // pieces of 16 bytes for 8 and 16 columns a thread
    constexpr int RB = VE / 4;                   // rows a group of the same bytes in both types
    // Threads, pieces a thread, rows a group, blocks an SM: as few threads as cover the row, as in the forward.  bf16 rows with fp32
    // weight, 805 MB read and written, of the copy rate: 768 0.82, 1024 0.91, 1280 0.81, 1536 0.89, 2048 0.85, 2560 0.88 (256 threads: 0.69),
    // 4096 0.89 (two rows a group: 0.67, registers), 5120 0.87 (512 threads: 0.69), 8192 0.87; fp32 0.85 to 0.96 (rows of 5120 and
    // more without a ring: 0.63).
#define BIBO_LN_RING(...)                                                                                                     \
  return layernorm_bwd_ring<T, W, __VA_ARGS__>(x, x_stride, dy, dy_stride, weight, mean, rstd, n_rows, hidden, dx, partial, dweight, dbias, parts, st)
    if (hidden > 512 && hidden <= 96 * 8) BIBO_LN_RING(96, C8, 4, 5);
    if (hidden > 96 * 8 && hidden <= 128 * 8) BIBO_LN_RING(128, C8, 4, 4);
    if (hidden > 128 * 8 && hidden <= 192 * 8) BIBO_LN_RING(192, C8, 2, 4);
    if (hidden > 192 * 8 && hidden <= 256 * 8) BIBO_LN_RING(256, C8, 4, 2);
    if (hidden > 128 * 16 && hidden <= 192 * 16) BIBO_LN_RING(192, C16, RB, 3);
    if (hidden > 192 * 16 && hidden <= 256 * 16) BIBO_LN_RING(256, C16, 1, 2);
    if (hidden > 256 * 16 && hidden <= 384 * 16) BIBO_LN_RING(384, C16, RB, 1);
    if (hidden > 384 * 16 && hidden <= 512 * 16) BIBO_LN_RING(512, C16, 1, 1);
#undef BIBO_LN_RING
  }
#define BIBO_LN_BWD(NT, CH, R)                                                                                              \
  return layernorm_bwd_v<T, W, VE, NT, CH, R>(x, x_stride, dy, dy_stride, weight, mean, rstd, n_rows, hidden, dx, partial, dweight, dbias, parts, st)
#define BIBO_LN_SHORT(G, CH, R)                                                                                             \
  return layernorm_bwd_short<T, W, VE, G, CH, R>(x, x_stride, dy, dy_stride, weight, mean, rstd, n_rows, hidden, dx, partial, dweight, dbias, parts, st)
  if constexpr (VE * sizeof(T) == 16) {          // what the rings leave
    // lanes a row, accesses a lane, rows a turn (bf16: two 41, four 37, eight 48 us at 400000 x 64; fp32: 53, 57, 59)
    if (vecs <= 8) BIBO_LN_SHORT(8, 1, VE / 2);
    if (vecs <= 16) BIBO_LN_SHORT(16, 1, VE / 2);
    if (vecs <= 32) BIBO_LN_SHORT(32, 1, VE / 2);
    if (vecs <= 64) BIBO_LN_SHORT(32, 2, 1);
    if constexpr (VE == 4) {
      if (vecs <= 128) BIBO_LN_SHORT(32, 4, 1);
      if (vecs <= 4096) BIBO_LN_BWD(512, 8, 1);
    } else {
      if (vecs <= 2048) BIBO_LN_BWD(512, 4, 1);
    }
  } else {
    // Narrow accesses: the issue slots bound, so few threads with many columns each (a row sum costs a thread the same whatever it
    // adds up), while the registers hold the group.  30000 rows, fp32 at odd strides / bf16 pairs, us (floor), with 256 or 512 threads
    // before: 301 columns 26 (16), 35; 777 56 (43), 77; 1531 103 (84), 130; bf16 1530 81 (42), 107; 2050 116 (56), 168.
    constexpr int R2 = VE == 2 ? 1 : 2;
    if (vecs <= 8) BIBO_LN_SHORT(8, 1, 4);
    if (vecs <= 32) BIBO_LN_SHORT(32, 1, 2);
    if (vecs <= 64) BIBO_LN_SHORT(32, 2, 2);
    if (vecs <= 128) BIBO_LN_SHORT(32, 4, 2);
    if (vecs <= 256) BIBO_LN_SHORT(32, 8, 1);
    if (vecs <= 512) BIBO_LN_BWD(128, 4, 4);
    if (vecs <= 768) BIBO_LN_BWD(192, 4, R2);
    if (vecs <= 1024) BIBO_LN_BWD(256, 4, R2);
    if (vecs <= 1536) BIBO_LN_BWD(384, 4, 1);
    if (vecs <= 2048) BIBO_LN_BWD(512, 4, 1);
    if constexpr (VE == 2) {
      if (vecs <= 384 * 8) BIBO_LN_BWD(384, 8, 1);
    }
    if (vecs <= 4096) BIBO_LN_BWD(512, 8, 1);
  }
#undef BIBO_LN_BWD
#undef BIBO_LN_SHORT
  *done = false;
  return BIBO_OK;
}

template <typename T, typename W>
static int layernorm_bwd_t(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                           const float* mean, const float* rstd, int64_t n_rows, int hidden, void* dx, float* partial,
                           void* dweight, void* dbias, cudaStream_t st) {
  const bool params = dweight != nullptr || dbias != nullptr;
  const int ve = ln_access(hidden, sizeof(T), sizeof(W), n_rows > 1 ? x_stride : 0, n_rows > 1 ? dy_stride : 0, x, dy, dx, weight,
                           nullptr);
  int used = 0, rc = BIBO_OK;
  bool done = false;
  float* part = params ? partial : nullptr;
#define BIBO_LN_PICK(VE) layernorm_bwd_pick<T, W, VE>(x, x_stride, dy, dy_stride, weight, mean, rstd, n_rows, hidden, dx, part, dweight, dbias, &used, &done, st)
  if constexpr (sizeof(T) == 2) rc = ve == 8 ? BIBO_LN_PICK(8) : ve == 2 ? BIBO_LN_PICK(2) : BIBO_LN_PICK(1);
  else rc = ve == 4 ? BIBO_LN_PICK(4) : BIBO_LN_PICK(1);
#undef BIBO_LN_PICK
  if (rc) return rc;
  if (!done) {                                   // rows too long for the registers of a block
    layernorm_bwd_dx_loop_kernel<T, W><<<(unsigned)n_rows, LN_T, 0, st>>>(
        static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride, static_cast<const W*>(weight), mean, rstd,
        hidden, static_cast<T*>(dx));
    BIBO_CHECK_LAUNCH("layernorm_bwd_dx_loop_kernel");
    if (!params) return BIBO_OK;
    const int64_t parts = n_rows <= LN_ONE_BLOCK ? 1 : ln_parts(n_rows), per = (n_rows + parts - 1) / parts;
    used = (int)((n_rows + per - 1) / per);
    layernorm_bwd_cols_kernel<T, W><<<dim3(used, (hidden + LN_T - 1) / LN_T), LN_T, 0, st>>>(
        static_cast<const T*>(x), x_stride, static_cast<const T*>(dy), dy_stride, mean, rstd, n_rows, hidden, per, partial,
        static_cast<W*>(dweight), static_cast<W*>(dbias));
    BIBO_CHECK_LAUNCH("layernorm_bwd_cols_kernel");
  }
  if (!params || used == 1) return BIBO_OK;      // one block has written the gradients itself
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((hidden + 31) / 32, 2);
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BIBO_CUDA(cudaLaunchKernelEx(&cfg, layernorm_dparam_kernel<W>, (const float*)partial, used, hidden, static_cast<W*>(dweight),
                               static_cast<W*>(dbias)));
  BIBO_CHECK_LAUNCH("layernorm_dparam_kernel");
  return BIBO_OK;
}

static int layernorm_check(const char* what, int64_t n_rows, int hidden, int dtype, int wdtype, int64_t stride) {
  if (dtype != BIBO_F32 && dtype != BIBO_BF16) return fail(BIBO_ERR_ARG, "%s: dtype=%d", what, dtype);
  if (wdtype != BIBO_F32 && wdtype != dtype)
    return fail(BIBO_ERR_ARG, "%s: weight dtype=%d beside activations of dtype=%d", what, wdtype, dtype);
  if (hidden < 1) return fail(BIBO_ERR_ARG, "%s: hidden=%d", what, hidden);
  if (hidden > 1 << 30) return fail(BIBO_ERR_UNSUPPORTED, "%s: hidden=%d", what, hidden);   // column counters pass it by a block
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
  if ((dweight || dbias) && hidden > 65535 * LN_T)      // the grid of layernorm_bwd_cols_kernel
    return fail(BIBO_ERR_UNSUPPORTED, "layernorm_bwd: parameter gradients of hidden=%d (%d at most)", hidden, 65535 * LN_T);
  if (n_rows <= 0) return BIBO_OK;      // the caller's dweight / dbias are sums over no rows: it zeroes them itself
  if (!x || !dy || !mean || !rstd || !dx || ((dweight || dbias) && !partial && ln_parts(n_rows) > 0))
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
