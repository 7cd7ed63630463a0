// Newton-Schulz orthogonalisation (see orthogonalize.cu) of matrices with a side of at most 128: everything in one launch.
// A cluster of 1-8 CTAs per matrix, each with a slice of up to 384 columns of x (m x n, m <= 128) for all the steps: x lives in
// tensor memory in fp32, times 2^24 and the next step's a, so that "a x + F x" is an accumulation onto it; its upper half in
// f16 is the operand of both products, in one shared-memory layout that is K-major for x x^T and MN-major for F x.  The Gram
// matrices of the slices are summed through distributed shared memory (each CTA reduces every C-th row and hands the rounded
// result to all); the m x m products are done by every CTA for itself, for m <= 64 on matrices in two halves (22 bits: with n
// much larger than m the singular values are alike and close to where the polynomial is steep, and the roundings of the m x m
// matrices were most of the error, 0.0026 against 0.0017 at 19 x 1794).  The launches, not the flops, are what a small matrix
// costs: 64 x 2048 fp32 took 18 launches and 211 us.
#include <algorithm>

#include "orthogonalize_common.cuh"

namespace bibo {
namespace tc {

constexpr int NS_SM_THREADS = 256, NS_SM_COLS = 384, NS_SM_MAX_CLUSTER = 8;
constexpr int NS_MAT = 2 * C_SUB;                               // a 128 x 128 f16 matrix: two sub-tiles of 64 columns
constexpr int NS_SM_OFF_M = 0;                                  // four of them; the last two double as the fp32 exchange buffer
constexpr int NS_SM_OFF_X = NS_SM_OFF_M + 4 * NS_MAT;
constexpr int NS_SM_OFF_BAR = NS_SM_OFF_X + NS_SM_COLS / 64 * C_SUB;
constexpr int NS_SM_BYTES = NS_SM_OFF_BAR + 256 + 1024;
constexpr float NS_ACC = NS_ONE * NS_ONE;                       // 1.0 in an accumulator
__device__ __forceinline__ bool aligned16_dev(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float4 ld_remote_f4(const void* local, uint32_t cta) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(map_to_cta(local, cta)) : "memory");
  return v;
}
__device__ __forceinline__ float ld_remote_f1(const void* local, uint32_t cta) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(local, cta)) : "memory");
  return v;
}
__device__ __forceinline__ void st_remote_u2(void* local, uint32_t cta, uint2 v) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1,%2};" ::"r"(map_to_cta(local, cta)), "r"(v.x), "r"(v.y) : "memory");
}

struct NsSmallArgs {
  const void* u;
  int64_t batch_stride, row_stride;
  int rows, cols, m, n, tall;
  int slice;                 // columns of x per CTA, a multiple of 64
  int steps, joint;
  float eps;
  __nv_bfloat16* out;
  float coefficients[64 * 3];
};

template <typename T, int CLUSTER>
__global__ void __launch_bounds__(NS_SM_THREADS, 1)
ns_small_kernel(const __grid_constant__ NsSmallArgs p) {
  constexpr int cluster = CLUSTER;
  extern __shared__ unsigned char smem_dyn[];
  // the same offset in every CTA of the cluster: the dynamic shared memory starts at one address in all of them
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint64_t* done = reinterpret_cast<uint64_t*>(smem + NS_SM_OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* red = reinterpret_cast<float*>(tmem_slot + 2);          // [8] warps, then [1] the block's sum of squares
  unsigned char* mat = smem + NS_SM_OFF_M;
  unsigned char* xs = smem + NS_SM_OFF_X;
  float* exch = reinterpret_cast<float*>(mat + 2 * NS_MAT);     // [128][128] fp32, 16-byte pieces swizzled by the row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
  const int row = (warp & 3) * 32 + lane;
  const uint32_t cta = cluster > 1 ? cluster_ctarank() : 0;
  const int64_t b = blockIdx.x / cluster;
  if (threadIdx.x == 0) { mbar_init(done, 1); *abort_flag = 0; fence_barrier_init(); }
  if (warp == 0) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tx = *tmem_slot, tm = tx + NS_SM_COLS;         // x, and the m x m accumulator
  const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
  const int m = p.m, mp = (m + 31) / 32 * 32, c0 = (int)cta * p.slice;
  const int cols = min(p.slice, max(0, p.n - c0));               // of this slice that exist
  const int groups = (cols + 63) / 64 * 2;                       // pieces of 32 columns, zero-filled up to 64
  // Rows m .. mp are zeros throughout; what the tiles hold in rows beyond mp takes part in nothing (a product's row depends on
  // that row of its first operand only, and the second's rows end at mp), so the warps of those rows leave them alone.
  const bool mine = (warp & 3) * 32 < mp;
  uint32_t phase = 0;

  const T* u = static_cast<const T*>(p.u) + b * p.batch_stride;
  const bool vec = !p.tall && ((reinterpret_cast<uintptr_t>(u) | (uintptr_t)(p.row_stride * sizeof(T))) & 15) == 0;
  // 32 columns of this thread's row, as they are
  auto load = [&](int col, float* v) {
    if (row >= m) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
    } else if (vec && col + 32 <= cols) {
      const uint4* s = reinterpret_cast<const uint4*>(u + (int64_t)row * p.row_stride + c0 + col);
#pragma unroll
      for (int i = 0; i < 32 * (int)sizeof(T) / 16; ++i) {
        const uint4 w = __ldg(s + i);
        const uint32_t x4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (sizeof(T) == 4) v[4 * i + k] = __uint_as_float(x4[k]);
          else { v[8 * i + 2 * k] = bf16_lo(x4[k]); v[8 * i + 2 * k + 1] = bf16_hi(x4[k]); }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int64_t c = c0 + col + i;
        v[i] = col + i < cols ? to_f32<T>(u[(int64_t)row * p.row_stride + c]) : 0.f;
      }
    }
  };
  // 32 values of this row, columns col.., times `scale` as f16 into a matrix of sub-tiles
  auto put = [&](unsigned char* base, int col, const float* v, float scale) {
    unsigned char* sub = base + (col >> 6) * C_SUB;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 o;
      o.x = pack_f16(v[8 * k] * scale, v[8 * k + 1] * scale);
      o.y = pack_f16(v[8 * k + 2] * scale, v[8 * k + 3] * scale);
      o.z = pack_f16(v[8 * k + 4] * scale, v[8 * k + 5] * scale);
      o.w = pack_f16(v[8 * k + 6] * scale, v[8 * k + 7] * scale);
      *reinterpret_cast<uint4*>(sub + swz(row, ((col & 63) >> 3) + k)) = o;
    }
  };
  // ... and with what the rounding left behind it, for the m x m matrices of m <= 64 (their second sub-tile is free)
  const bool fine = mp <= 64;
  auto put_mat = [&](unsigned char* base, int col, float* v, float scale) {
    put(base, col, v, scale);
    if (!fine) return;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = v[i] * scale - __half2float(__float2half_rn(v[i] * scale));
    put(base + C_SUB, col, v, 1.f);
  };
  // v += scale * the row's values in a matrix
  auto add = [&](const unsigned char* base, int col, float* v, float scale) {
    const unsigned char* sub = base + (col >> 6) * C_SUB;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 o = *reinterpret_cast<const uint4*>(sub + swz(row, ((col & 63) >> 3) + k));
      const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_f16(w[i]);
        v[8 * k + 2 * i] = fmaf(scale, f.x, v[8 * k + 2 * i]);
        v[8 * k + 2 * i + 1] = fmaf(scale, f.y, v[8 * k + 2 * i + 1]);
      }
    }
  };
  auto get = [&](uint32_t taddr, float* v) {
    tmem_ld32(taddr + lane_off, reinterpret_cast<uint32_t*>(v));
    tmem_ld_wait();
  };
  // everybody's shared-memory and tensor-memory accesses before, the products that follow after
  auto ready = [&]() {
    fence_proxy_async_all();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  auto wait_products = [&]() {
    mbar_wait(done, phase, abort_flag);          // where it gives up the values are poisoned below
    __syncwarp();
    phase ^= 1;
    tc_fence_after();
  };

  // ---- x_0: raw values into tensor memory, their squares over the cluster, then scaled
  float ss = 0.f;
  // u without 16-byte alignment, or tall: read in its own order into shared memory (the matrices' place, free until the first
  // Gram matrix), 192 columns at a time, and the threads take their rows from there
  constexpr int PITCH = 193;
  float* stage = reinterpret_cast<float*>(mat);
  const bool staged = !vec;
  for (int g0 = 0; g0 < groups; g0 += 6) {
  const int g1 = staged ? min(groups, g0 + 6) : groups;
  if (staged) {
    __syncthreads();                             // the last round has been read
    if (p.tall) {
      const int total = (min(cols, g1 * 32) - g0 * 32) * m;
      const T* src = u + (int64_t)(c0 + g0 * 32) * p.row_stride;
#pragma unroll 8
      for (int i = threadIdx.x; i < total; i += NS_SM_THREADS) {
        const int c = i / m, r = i - c * m;
        stage[r * PITCH + c] = to_f32<T>(src[c * p.row_stride + r]);
      }
    } else {
      for (int r = warp; r < m; r += 8) {
        const T* src = u + (int64_t)r * p.row_stride + c0 + g0 * 32;
#pragma unroll
        for (int i = 0; i < 6; ++i)
          if ((g0 + i) * 32 + lane < cols) stage[r * PITCH + i * 32 + lane] = to_f32<T>(src[i * 32 + lane]);
      }
    }
    __syncthreads();
  }
  auto take = [&](int g, float* v) {
    if (!staged || row >= m) { load(g * 32, v); return; }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = g * 32 + i < cols ? stage[row * PITCH + (g - g0) * 32 + i] : 0.f;
  };
  for (int g = g0 + half; g < g1; g += 4) {      // two pieces of a thread's row in flight
    float v[2][32];
    take(g, v[0]);
    if (g + 2 < g1) take(g + 2, v[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (g + 2 * k >= g1) break;
#pragma unroll
      for (int i = 0; i < 32; ++i) ss = fmaf(v[k][i], v[k][i], ss);
      tmem_st32(tx + lane_off + (g + 2 * k) * 32, reinterpret_cast<const uint32_t*>(v[k]));
    }
  }
  if (!staged) break;
  }
  tmem_st_wait();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  ss = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) ss += red[w];
  if (cluster > 1) {
    if (threadIdx.x == 0) red[8] = ss;
    cluster_sync_all();
    float part[cluster];
#pragma unroll
    for (int c = 0; c < cluster; ++c) part[c] = ld_remote_f1(red + 8, c);
    ss = 0.f;
#pragma unroll
    for (int c = 0; c < cluster; ++c) ss += part[c];
  }
  const float inv = 1.f / (sqrtf(ss) + p.eps);
  const float* co = p.coefficients;
  float a = p.joint ? co[0] * co[3] : co[0];
  for (int g = half; g < (mine ? groups : 0); g += 2) {
    float v[32];
    get(tx + g * 32, v);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= inv;
    put(xs, g * 32, v, NS_ONE);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= NS_ACC * a;
    tmem_st32(tx + lane_off + g * 32, reinterpret_cast<const uint32_t*>(v));
  }
  tmem_st_wait();

  // ---- mat[0] = G = x x^T over the cluster
  auto gram = [&]() {
    ready();
    if (warp == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_f16(BM, mp);
      for (int k = 0; k < groups * 2; ++k) {                     // 16 columns each
        const uint64_t d = make_sdesc_k128(smem_u32(xs + (k >> 2) * C_SUB)) + (k & 3) * (32 >> 4);
        umma_bf16(tm, d, d, idesc, k != 0);
      }
      umma_commit(done);
    }
    wait_products();
    const float poison = *abort_flag ? __int_as_float(0x7fffffff) : 0.f;
    for (int g = half; g < (mine ? mp / 32 : 0); g += 2) {
      float v[32];
      get(tm + g * 32, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = groups > 0 ? v[i] + poison : 0.f;   // an empty slice has multiplied nothing
      if (cluster == 1) {
        put_mat(mat, g * 32, v, 1.f / NS_ONE);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          reinterpret_cast<float4*>(exch)[row * 32 + ((g * 8 + k) ^ (row & 7))] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
      }
    }
    if (cluster > 1) {
      tc_fence_before();
      cluster_sync_all();
      tc_fence_after();
      const int quads = mp / 4;
      const int my_rows = (mp - (int)cta + cluster - 1) / cluster;   // rows cta, cta + cluster, ...
      for (int i = threadIdx.x; i < my_rows * quads; i += NS_SM_THREADS) {
        const int r = (int)cta + i / quads * cluster, k = i % quads;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4* at = reinterpret_cast<const float4*>(exch) + r * 32 + (k ^ (r & 7));
        float4 v[cluster];
#pragma unroll
        for (int c = 0; c < cluster; ++c) v[c] = ld_remote_f4(at, c);
#pragma unroll
        for (int c = 0; c < cluster; ++c) { s.x += v[c].x; s.y += v[c].y; s.z += v[c].z; s.w += v[c].w; }
        const float z = 1.f / NS_ONE;
        const uint2 o = make_uint2(pack_f16(s.x * z, s.y * z), pack_f16(s.z * z, s.w * z));
        const float2 o0 = unpack_f16(o.x), o1 = unpack_f16(o.y);
        const uint2 rest = make_uint2(pack_f16(s.x * z - o0.x, s.y * z - o0.y), pack_f16(s.z * z - o1.x, s.w * z - o1.y));
        unsigned char* dst = mat + (k >> 4) * C_SUB + swz(r, (k & 15) >> 1) + (k & 1) * 8;
#pragma unroll
        for (int c = 0; c < cluster; ++c) {
          st_remote_u2(dst, c, o);
          if (fine) st_remote_u2(dst + C_SUB, c, rest);
        }
      }
      fence_proxy_async_all();
      tc_fence_before();
      cluster_sync_all();
      tc_fence_after();
    }
  };
  // mat[to] = alpha mat[x] mat[y] + beta mat[s] + beta2 mat[s2]
  auto sym = [&](int x, int y, float alpha, int s, float beta, int s2, float beta2, int to) {
    ready();
    if (warp == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_f16(BM, mp);
      for (int k = 0; k < mp / 16; ++k) {
        const uint64_t dx = make_sdesc_k128(smem_u32(mat + x * NS_MAT + (k >> 2) * C_SUB)) + (k & 3) * (32 >> 4);
        const uint64_t dy = make_sdesc_k128(smem_u32(mat + y * NS_MAT + (k >> 2) * C_SUB)) + (k & 3) * (32 >> 4);
        umma_bf16(tm, dx, dy, idesc, k != 0);
        if (fine) {
          umma_bf16(tm, dx, dy + (C_SUB >> 4), idesc, 1);
          umma_bf16(tm, dx + (C_SUB >> 4), dy, idesc, 1);
        }
      }
      umma_commit(done);
    }
    wait_products();
    for (int g = half; g < (mine ? mp / 32 : 0); g += 2) {
      float v[32];
      get(tm + g * 32, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha / NS_ONE;
      add(mat + s * NS_MAT, g * 32, v, beta);
      if (fine) add(mat + s * NS_MAT + C_SUB, g * 32, v, beta);
      if (s2 >= 0) add(mat + s2 * NS_MAT, g * 32, v, beta2);
      if (s2 >= 0 && fine) add(mat + s2 * NS_MAT + C_SUB, g * 32, v, beta2);
      put_mat(mat + to * NS_MAT, g * 32, v, 1.f);
    }
  };
  // Results whose rows cannot be written in 16-byte pieces (all of a slice's columns) cross the matrices' place, all products being done
  constexpr int OUT_PITCH = NS_SM_COLS + 2;
  static_assert(BM * OUT_PITCH * 2 <= 4 * NS_MAT && BM * PITCH * 4 <= 4 * NS_MAT, "staging fits");
  __nv_bfloat16* out_stage = reinterpret_cast<__nv_bfloat16*>(mat);
  const bool out_vec = !p.tall && p.cols % 8 == 0 && aligned16_dev(p.out) && cols % 32 == 0;
  // x (already times a) += mat[f] x; then the next step's operand and factor, or the result
  auto apply = [&](int f, bool last, float next_a) {
    ready();
    if (warp == 0 && elect_one()) {
      for (int c = 0; c < groups * 32; c += 128) {
        const int width = min(128, groups * 32 - c);
        const uint32_t idesc = make_idesc_f16(BM, width) | 1u << 16;   // B is MN-major: 64-column sub-tiles C_SUB apart
        for (int k = 0; k < mp / 16; ++k) {
          const uint64_t df = make_sdesc_k128(smem_u32(mat + f * NS_MAT + (k >> 2) * C_SUB)) + (k & 3) * (32 >> 4);
          const uint64_t dx = make_sdesc_mn128(smem_u32(xs + (c >> 6) * C_SUB), C_SUB) + k * (2048 >> 4);
          umma_bf16(tx + c, df, dx, idesc, 1);
          if (fine) umma_bf16(tx + c, df + (C_SUB >> 4), dx, idesc, 1);
        }
      }
      umma_commit(done);
    }
    wait_products();
    const bool failed = *abort_flag != 0;
    for (int g = half; g < (mine ? groups : 0); g += 2) {
      float v[32];
      get(tx + g * 32, v);
      if (!last) {
        put(xs, g * 32, v, 1.f / NS_ONE);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= next_a;
        tmem_st32(tx + lane_off + g * 32, reinterpret_cast<const uint32_t*>(v));
        continue;
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = failed ? __int_as_float(0x7fffffff) : v[i] * (1.f / NS_ACC);
      if (row >= m) continue;
      __nv_bfloat16* o = p.out + b * p.rows * p.cols;
      const int64_t c = c0 + g * 32;
      if (out_vec && g * 32 + 32 <= cols) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          reinterpret_cast<uint4*>(o + (int64_t)row * p.cols + c)[k] =
              make_uint4(pack_bf16(v[8 * k], v[8 * k + 1]), pack_bf16(v[8 * k + 2], v[8 * k + 3]),
                         pack_bf16(v[8 * k + 4], v[8 * k + 5]), pack_bf16(v[8 * k + 6], v[8 * k + 7]));
      } else {                                   // in the result's order below
#pragma unroll
        for (int i = 0; i < 32; ++i) out_stage[row * OUT_PITCH + g * 32 + i] = __float2bfloat16_rn(v[i]);
      }
    }
    if (!last) tmem_st_wait();
    if (last && !out_vec) {
      __syncthreads();
      __nv_bfloat16* o = p.out + b * p.rows * p.cols;
      if (p.tall) {
#pragma unroll 4
        for (int i = threadIdx.x; i < cols * m; i += NS_SM_THREADS) {
          const int c = i / m, r = i - c * m;
          o[(int64_t)c0 * m + i] = out_stage[r * OUT_PITCH + c];
        }
      } else {
        for (int r = warp; r < m; r += 8)
          for (int c = lane; c < cols; c += 32) o[(int64_t)r * p.cols + c0 + c] = out_stage[r * OUT_PITCH + c];
      }
    }
  };

  int s = 0;
  if (p.joint) {                                                 // the first two steps as one, see orthogonalize.cu
    gram();
    sym(0, 0, co[2], 0, co[1], -1, 0.f, 1);
    sym(1, 1, 1.f, 1, 2.f * co[0], -1, 0.f, 2);
    sym(2, 0, 1.f, 0, co[0] * co[0], -1, 0.f, 3);
    sym(3, 3, co[5], 3, co[4], -1, 0.f, 0);
    sym(0, 1, 1.f, 0, co[0], 1, co[3], 2);
    apply(2, p.steps == 2, co[6]);
    s = 2;
  }
  for (; s < p.steps; ++s) {
    gram();
    sym(0, 0, co[3 * s + 2], 0, co[3 * s + 1], -1, 0.f, 1);
    apply(1, s == p.steps - 1, s + 1 < p.steps ? co[3 * s + 3] : 0.f);
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag)                               // products may still be running on this shared and tensor memory
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  if (cluster > 1) cluster_sync_all();           // nobody leaves while its shared memory is read or written
  if (warp == 0) { tc_fence_after(); tmem_dealloc(tx, 512); }
}

// CTAs per matrix of the one-launch kernel, 0: it does not take these sizes.  Slices of at most NS_SM_COLS columns; beyond that as
// many CTAs as the machine has for the batch, while a slice keeps 128 columns.
int ns_small_cluster(int64_t batch, int rows, int cols) {
  const int m = std::min(rows, cols), n = std::max(rows, cols);
  if (m > BM || n > NS_SM_COLS * NS_SM_MAX_CLUSTER) return 0;
  int c = (n + NS_SM_COLS - 1) / NS_SM_COLS;
  while (c < NS_SM_MAX_CLUSTER && n >= 128 * (c + 1) && batch * (c + 1) <= sm_count()) ++c;
  return c;
}
template <typename T, int CLUSTER>
static int ns_small(const void* u, int64_t batch, int64_t batch_stride, int rows, int cols, int64_t row_stride, int steps, bool joint,
                    const float* co, float eps, void* out, cudaStream_t st) {
  constexpr int cluster = CLUSTER;
  auto kern = ns_small_kernel<T, CLUSTER>;
  static DeviceOnce once;
  const int rc = once.get([&](int*) {
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SM_BYTES));
    return (int)BIBO_OK;
  });
  if (rc) return rc;
  NsSmallArgs p = {};
  p.batch_stride = batch_stride;
  p.row_stride = row_stride;
  p.rows = rows;
  p.cols = cols;
  p.m = std::min(rows, cols);
  p.n = std::max(rows, cols);
  p.tall = rows > cols;
  p.slice = ((p.n + cluster - 1) / cluster + 63) / 64 * 64;
  p.steps = steps;
  p.joint = joint;
  p.eps = eps;
  for (int i = 0; i < 3 * steps; ++i) p.coefficients[i] = co[i];
  const int64_t most = (1 << 30) / cluster;      // matrices of a launch
  for (int64_t b0 = 0; b0 < batch; b0 += most) {
    p.u = static_cast<const T*>(u) + b0 * batch_stride;
    p.out = static_cast<__nv_bfloat16*>(out) + b0 * rows * cols;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min(most, batch - b0) * cluster));
    cfg.blockDim = dim3(NS_SM_THREADS);
    cfg.dynamicSmemBytes = NS_SM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BIBO_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
    BIBO_CHECK_LAUNCH("ns_small_kernel");
  }
  return BIBO_OK;
}

int ns_small_launch(const void* u, int dtype, int64_t batch, int64_t batch_stride, int rows, int cols, int64_t row_stride, int steps,
                    bool joint, const float* coefficients, float eps, int cluster, void* out, cudaStream_t st) {
#define BIBO_NS_SMALL(C)                                                                                                          \
  case C:                                                                                                                         \
    return dtype == BIBO_F32                                                                                                      \
               ? ns_small<float, C>(u, batch, batch_stride, rows, cols, row_stride, steps, joint, coefficients, eps, out, st)      \
               : ns_small<__nv_bfloat16, C>(u, batch, batch_stride, rows, cols, row_stride, steps, joint, coefficients, eps, out, st);
  switch (cluster) {
    BIBO_NS_SMALL(1) BIBO_NS_SMALL(2) BIBO_NS_SMALL(3) BIBO_NS_SMALL(4)
    BIBO_NS_SMALL(5) BIBO_NS_SMALL(6) BIBO_NS_SMALL(7) BIBO_NS_SMALL(8)
    default: return fail(BIBO_ERR_UNSUPPORTED, "orthogonalize: %d CTAs per matrix", cluster);
  }
#undef BIBO_NS_SMALL
}

}  // namespace tc
}  // namespace bibo
