// Newton-Schulz orthogonalisation of stacked matrices, the update of an optimiser that steps along the orthogonal
// factor of the momentum of the expert stacks [E,2I,H] / [E,H,I] and the router weight:
//   x_0 = u / (|u|_F + eps);   x_{k+1} = a x_k + (b G + c G^2) x_k,  G = x_k x_k^T   (m x n with m <= n; a tall u is used
//   as it lies, with G = x^T x and the products' sides swapped), out = bf16(x_steps)
// An odd polynomial of the singular values is applied and the singular vectors stay.
//
// Numbers.  The products run on the tensor cores with f16 operands and fp32 accumulators: bf16 operands would lose
// three bits more, tf32 would halve the rate for none, and the range is bounded (|x|_2 <= about 1.2 for the usual
// coefficients, so every entry of x, G and b G + c G^2 is below 16).  All three are kept times 2^12, which centres
// them in f16's range: an entry 2^-26 of the largest is still normal.  u enters scaled by a power of two (exact for bf16)
// and the rest of 1/(|u|_F + eps), t in [1,2), goes into the first products' epilogues in fp32.
// A rounding of x spreads over all singular directions, and a direction of a small singular value is stretched by
// a ~ 3.4 in every step that follows, so the early x are what has to be exact:
//   - the term "a x" of a step is taken from x in two f16 halves (22 bits) where x is u (fp32) or the result of the first
//     two steps; the other factor F = b G + c G^2 is small in the weak directions and multiplies the upper half;
//   - the first two steps are one: with F1, F2 their polynomials, x_2 = a1 a2 x_0 + R x_0, R = F2 F1 + a1 F2 + a2 F1, and the
//     second Gram matrix is (a1 + F1)^2 G = a1^2 G + T G, T = F1^2 + 2 a1 F1 (all symmetric, all commute).  x_1 is never
//     formed, hence never rounded, and the two steps cost 3 m^2 n + 5 m^3 flops where two single ones cost
//     6 m^2 n + 2 m^3.  Later steps are single: there the polynomial maps values near 1 to values near 1, a Gram matrix carried
//     along instead of formed anew collects errors that three or more steps do not contract.
// On spectra from Gaussian to rank one plus 1e-3 noise the error is within a few 1e-4 of that of the bf16 rounding alone.
//
// Symmetric products (G, F, T, R, the second G) are computed and stored on and below the diagonal's 256 x 256 tiles only; an
// operand tile above it is read as the transposed tile below it, as an MN-major operand.
#include <algorithm>
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace bibo {
namespace tc {

constexpr float NS_ONE = 4096.f;                 // 1.0 as stored
constexpr float NS_LO = 2048.f;                  // scale of the lower half of a value beside the upper one
constexpr int NS_MAX_PARTS = 64;                 // partial sums of squares per matrix

// ---- products ----------------------------------------------------------------------------------------------------
// One persistent kernel on 256 x 256 tiles: a CTA pair runs tcgen05.mma.cta_group::2 (256 x 256 x 16), each CTA staging its 128
// rows of A and its half of B's rows, five stages of 32 KB; 2 x 256 TMEM columns, so the drain of a tile runs under the next
// one's products.  Warps: 0 loads, 1 products (pair leader), 2 loads the sources of the drain and stores its results,
// 4-7 drain.  Sub-tiles of 64 columns go through two 32 KB slots: source halves in, result halves out, in place.
constexpr int NS_GRAM = 0, NS_SYM = 1, NS_APPLY = 2;
constexpr int NS_T = 256, NS_STAGES = 5, NS_THREADS = 256;
constexpr int NS_OFF_A = 0;
constexpr int NS_OFF_B = NS_OFF_A + NS_STAGES * A_BYTES;
constexpr int NS_OFF_SLOT = NS_OFF_B + NS_STAGES * A_BYTES;      // [2] slots of {upper [128 x 64], lower [128 x 64]}
constexpr int NS_OFF_BAR = NS_OFF_SLOT + 4 * C_SUB;
constexpr int NS_SMEM = NS_OFF_BAR + 256 + 1024;

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

struct NsMaps {            // a matrix of a batch with boxes of 128 rows (K-major operands, sources, results) and 64 rows (MN-major)
  CUtensorMap r128, r64;
};
struct NsArgs {
  NsMaps a, b;
  CUtensorMap s_hi, s_lo, c_hi, c_lo;
  int64_t n_work;
  int m_tiles, n_tiles, k_blocks;
  int rows, cols;            // of the result
  int has_s, has_lo, out_lo; // source; source's or second source's map s_lo; result in two halves
  int out_bf16;              // the last product: c_hi is the caller's bf16 result
  float alpha, beta, beta_lo;   // C = alpha A B + beta S_hi + beta_lo S_lo
  const float* t_scale;      // first products: t of each matrix
  int* status;
  __nv_bfloat16* out;        // with out_bf16: the result itself, for a run that gave up
};

struct NsTile { int b, i, j; };
template <int MODE> __device__ __forceinline__ NsTile ns_decode(int64_t w, int m_tiles, int n_tiles) {
  NsTile t;
  if (MODE == NS_APPLY) {
    const int64_t per = (int64_t)m_tiles * n_tiles;
    t.b = (int)(w / per);
    const int r = (int)(w % per);
    t.i = r % m_tiles;
    t.j = r / m_tiles;
  } else {                                        // the lower triangle row by row
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

// How an operand's k-block is read.  OP_K: rows of the tile with k contiguous; OP_MN: k-rows with the tile's rows contiguous;
// OP_SYM: a symmetric matrix of which tiles on and below the diagonal exist: OP_K there, OP_MN from the mirrored tile above.
enum { OP_K, OP_MN, OP_SYM };
template <int OP> __device__ __forceinline__ bool ns_mn_major(int tile, int kb) {
  return OP == OP_MN || (OP == OP_SYM && kb / (NS_T / BK) > tile);
}
template <int OP>
__device__ __forceinline__ void ns_load(unsigned char* dst, const NsMaps& m, uint32_t bar, int tile, int pr, int kb, int b) {
  const int r0 = tile * NS_T + pr * BM;
  if (ns_mn_major<OP>(tile, kb)) {
    tma_load_3d_cg2(dst, &m.r64, bar, r0, kb * BK, b);
    tma_load_3d_cg2(dst + MN_BOX, &m.r64, bar, r0 + 64, kb * BK, b);
  } else {
    tma_load_3d_cg2(dst, &m.r128, bar, kb * BK, r0, b);
  }
}

template <int MODE, bool TALL>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_product_kernel(const __grid_constant__ NsArgs p) {
  constexpr int OP_A = MODE == NS_GRAM ? (TALL ? OP_MN : OP_K) : MODE == NS_SYM ? OP_SYM : TALL ? OP_K : OP_SYM;
  constexpr int OP_B = MODE == NS_GRAM ? (TALL ? OP_MN : OP_K) : MODE == NS_SYM ? OP_SYM : TALL ? OP_SYM : OP_MN;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + NS_OFF_BAR);   // pair leader
  uint64_t* empty = full + NS_STAGES;
  uint64_t* tfull = empty + NS_STAGES;
  uint64_t* tempty = tfull + 2;                                      // pair leader: 4 drain warps of each CTA
  uint64_t* sfull = tempty + 2;                                      // a slot's sources have landed (and its last store has left)
  uint64_t* cfull = sfull + 2;                                       // a slot's results are written
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(cfull + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pr = (int)(cluster_ctarank() & 1u);
  const int64_t w0 = blockIdx.x / 2, dw = gridDim.x / 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 8);
      mbar_init(&sfull[b], 1); mbar_init(&cfull[b], EPI_THREADS);
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&p.a.r128); prefetch_tmap(&p.a.r64); prefetch_tmap(&p.b.r128); prefetch_tmap(&p.b.r64);
    prefetch_tmap(&p.s_hi); prefetch_tmap(&p.c_hi);
  }
  if (warp == 1) { tmem_alloc_cg2(tmem_slot, 2 * NS_T); tmem_relinquish_cg2(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      PipeState ps;
      bool ok = true;
      for (int64_t w = w0; w < p.n_work && ok; w += dw) {
        const NsTile t = ns_decode<MODE>(w, p.m_tiles, p.n_tiles);
        const bool same = MODE == NS_GRAM && t.i == t.j;             // both operands of a CTA are the same rows
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          ok = mbar_wait<true>(&empty[ps.stage], ps.phase ^ 1, abort_flag);
          if (!ok) break;
          if (pr == 0) mbar_expect_tx(&full[ps.stage], same ? 2 * A_BYTES : 4 * A_BYTES);
          const uint32_t bar = map_to_cta(&full[ps.stage], 0);
          ns_load<OP_A>(smem + NS_OFF_A + ps.stage * A_BYTES, p.a, bar, t.i, pr, kb, t.b);
          if (!same) ns_load<OP_B>(smem + NS_OFF_B + ps.stage * A_BYTES, p.b, bar, t.j, pr, kb, t.b);
          ps.next<NS_STAGES>();
        }
      }
    }
  } else if (warp == 1) {
    if (pr == 0 && elect_one()) {
      PipeState ps;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int64_t w = w0; w < p.n_work && ok; w += dw) {
        const NsTile t = ns_decode<MODE>(w, p.m_tiles, p.n_tiles);
        const bool same = MODE == NS_GRAM && t.i == t.j;
        ok = mbar_wait<true>(&tempty[acc], acc_phase ^ 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          ok = mbar_wait<true>(&full[ps.stage], ps.phase, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + NS_OFF_A + ps.stage * A_BYTES);
          const uint32_t sb = same ? sa : smem_u32(smem + NS_OFF_B + ps.stage * A_BYTES);
          const bool amn = ns_mn_major<OP_A>(t.i, kb), bmn = ns_mn_major<OP_B>(t.j, kb);
          const uint64_t da = amn ? make_sdesc_mn128(sa) : make_sdesc_k128(sa);
          const uint64_t db = bmn ? make_sdesc_mn128(sb) : make_sdesc_k128(sb);
          const int a_step = amn ? (2048 >> 4) : (32 >> 4), b_step = bmn ? (2048 >> 4) : (32 >> 4);
          // bit 15: A is MN-major, bit 16: B is MN-major
          const uint32_t idesc = make_idesc_f16(2 * BM, NS_T) | (amn ? 1u << 15 : 0u) | (bmn ? 1u << 16 : 0u);
#pragma unroll
          for (int k = 0; k < BK / UK; ++k)
            umma_bf16_cg2(tmem_base + acc * NS_T, da + k * a_step, db + k * b_step, idesc, (kb | k) != 0);
          umma_commit_cg2_mc(&empty[ps.stage], 3);
          ps.next<NS_STAGES>();
        }
        if (!ok) break;
        umma_commit_cg2_mc(&tfull[acc], 3);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else if (warp == 2) {
    if (elect_one()) {
      // sub-tile u of this CTA: tile w0 + (u / 4) * dw, columns (u % 4) * 64; a sub-tile outside the result is passed through
      const int64_t n_sub = w0 < p.n_work ? ((p.n_work - 1 - w0) / dw + 1) * 4 : 0;
      auto place = [&](int64_t u, NsTile& t, int& x, int& y) {
        t = ns_decode<MODE>(w0 + (u >> 2) * dw, p.m_tiles, p.n_tiles);
        x = t.j * NS_T + (int)(u & 3) * 64;
        y = t.i * NS_T + pr * BM;
        return x < p.cols && y < p.rows;
      };
      auto source = [&](int64_t u) {
        if (u >= n_sub) return;
        uint64_t* bar = &sfull[u & 1];
        NsTile t;
        int x, y;
        if (!place(u, t, x, y) || !p.has_s) { mbar_arrive(bar); return; }
        unsigned char* slot = smem + NS_OFF_SLOT + (u & 1) * 2 * C_SUB;
        mbar_expect_tx(bar, p.has_lo ? 2 * C_SUB : C_SUB);
        tma_load_3d(slot, &p.s_hi, bar, x, y, t.b);
        if (p.has_lo) tma_load_3d(slot + C_SUB, &p.s_lo, bar, x, y, t.b);
      };
      source(0);
      source(1);
      for (int64_t u = 0; u < n_sub; ++u) {
        if (!mbar_wait(&cfull[u & 1], (uint32_t)(u >> 1) & 1u, abort_flag)) break;
        NsTile t;
        int x, y;
        if (place(u, t, x, y)) {
          unsigned char* slot = smem + NS_OFF_SLOT + (u & 1) * 2 * C_SUB;
          tma_store_3d(&p.c_hi, slot, x, y, t.b);
          if (p.out_lo) tma_store_3d(&p.c_lo, slot + C_SUB, x, y, t.b);
          tma_store_commit();
        }
        if (u + 2 < n_sub) {
          tma_store_wait_read();
          source(u + 2);
        }
      }
      tma_store_wait_all();
    }
  } else if (warp >= 4) {
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const bool poison = p.out_bf16 && *p.status != 0;                 // an earlier product gave up: no number is left to stand
    int acc = 0;
    uint32_t acc_phase = 0;
    int64_t u = 0;
    bool ok = true;
    for (int64_t w = w0; w < p.n_work && ok; w += dw) {
      float al = p.alpha, be = p.beta, bl = p.beta_lo;
      if (p.t_scale != nullptr) {
        const float ts = p.t_scale[ns_decode<MODE>(w, p.m_tiles, p.n_tiles).b];
        al *= MODE == NS_GRAM ? ts * ts : ts;
        be *= ts;
        bl *= ts;
      }
      ok = mbar_wait<true>(&tfull[acc], acc_phase, abort_flag);
      if (!ok) break;
      tc_fence_after();
#pragma unroll 1
      for (int g = 0; g < 4; ++g, ++u) {
        uint32_t r[2][32];
        tmem_ld32(lane_addr + acc * NS_T + g * 64, r[0]);
        tmem_ld32(lane_addr + acc * NS_T + g * 64 + 32, r[1]);
        ok = mbar_wait(&sfull[u & 1], (uint32_t)(u >> 1) & 1u, abort_flag);
        tmem_ld_wait();
        if (g == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_addr(map_to_cta(&tempty[acc], 0));
        }
        if (!ok) break;
        unsigned char* slot = smem + NS_OFF_SLOT + (u & 1) * 2 * C_SUB;
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
          uint4* hi = reinterpret_cast<uint4*>(slot + swz(row, jj));
          uint4* lo = reinterpret_cast<uint4*>(slot + C_SUB + swz(row, jj));
          const uint32_t* a = r[jj >> 2] + 8 * (jj & 3);
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = al * __uint_as_float(a[i]);
          if (p.has_s) {
            const uint4 s = *hi;
            const uint32_t* ps = reinterpret_cast<const uint32_t*>(&s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = unpack_f16(ps[i]);
              v[2 * i] = fmaf(be, f.x, v[2 * i]);
              v[2 * i + 1] = fmaf(be, f.y, v[2 * i + 1]);
            }
          }
          if (p.has_lo) {
            const uint4 s = *lo;
            const uint32_t* ps = reinterpret_cast<const uint32_t*>(&s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = unpack_f16(ps[i]);
              v[2 * i] = fmaf(bl, f.x, v[2 * i]);
              v[2 * i + 1] = fmaf(bl, f.y, v[2 * i + 1]);
            }
          }
          uint4 o;
          uint32_t* po = reinterpret_cast<uint32_t*>(&o);
          if (p.out_bf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              po[i] = poison ? 0x7fff7fffu : pack_bf16(v[2 * i] * (1.f / NS_ONE), v[2 * i + 1] * (1.f / NS_ONE));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) po[i] = pack_f16(v[2 * i], v[2 * i + 1]);
          }
          *hi = o;
          if (p.out_lo) {
            uint4 l;
            uint32_t* pl = reinterpret_cast<uint32_t*>(&l);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = unpack_f16(po[i]);
              pl[i] = pack_f16((v[2 * i] - f.x) * NS_LO, (v[2 * i + 1] - f.y) * NS_LO);
            }
            *lo = l;
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(&cfull[u & 1]);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {                             // a wait gave up: copies may still be in flight to this shared memory
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    if (threadIdx.x == 0) atomicExch(p.status, 112);
    if (p.out_bf16) {                            // its part of the caller's result is void
      for (int64_t w = w0; w < p.n_work; w += dw) {
        const NsTile t = ns_decode<MODE>(w, p.m_tiles, p.n_tiles);
        for (int i = threadIdx.x; i < BM * NS_T; i += NS_THREADS) {
          const int y = t.i * NS_T + pr * BM + i / NS_T, x = t.j * NS_T + i % NS_T;
          if (y < p.rows && x < p.cols) p.out[((int64_t)t.b * p.rows + y) * p.cols + x] = __ushort_as_bfloat16(0x7fff);
        }
      }
    }
  }
  cluster_sync_all();                            // nobody leaves while the pair's other CTA may still signal or read this one
  if (warp == 1) { tc_fence_after(); tmem_dealloc_cg2(tmem_base, 2 * NS_T); }
}

// ---- matrices with a side of at most 128: everything in one launch ------------------------------------------------------
// A cluster of 1-8 CTAs per matrix, each with a slice of up to 384 columns of x (m x n, m <= 128) for all the steps: x lives in
// tensor memory in fp32, times 2^24 and the next step's a, so that "a x + F x" is an accumulation onto it; its upper half in
// f16 is the operand of both products, in one shared-memory layout that is K-major for x x^T and MN-major for F x.  The Gram
// matrices of the slices are summed through distributed shared memory (each CTA reduces every C-th row and hands the rounded
// result to all); the m x m products are done by every CTA for itself.  The launches, not the flops, are what a small matrix
// costs: 64 x 2048 fp32 took 18 launches and 211 us.
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

template <typename T>
__global__ void __launch_bounds__(NS_SM_THREADS, 1)
ns_small_kernel(const __grid_constant__ NsSmallArgs p, int cluster) {
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
        v[i] = col + i < cols ? to_f32<T>(p.tall ? u[c * p.row_stride + row] : u[(int64_t)row * p.row_stride + c]) : 0.f;
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
  for (int g = half; g < groups; g += 2) {
    float v[32];
    load(g * 32, v);
#pragma unroll
    for (int i = 0; i < 32; ++i) ss = fmaf(v[i], v[i], ss);
    tmem_st32(tx + lane_off + g * 32, reinterpret_cast<const uint32_t*>(v));
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
    ss = 0.f;
    for (int c = 0; c < cluster; ++c) ss += ld_remote_f1(red + 8, c);
  }
  const float inv = 1.f / (sqrtf(ss) + p.eps);
  const float* co = p.coefficients;
  float a = p.joint ? co[0] * co[3] : co[0];
  for (int g = half; g < groups; g += 2) {
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
    for (int g = half; g < mp / 32; g += 2) {
      float v[32];
      get(tm + g * 32, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = groups > 0 ? v[i] + poison : 0.f;   // an empty slice has multiplied nothing
      if (cluster == 1) {
        put(mat, g * 32, v, 1.f / NS_ONE);
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
      for (int i = threadIdx.x; i < BM / cluster * quads; i += NS_SM_THREADS) {   // rows cta, cta + cluster, ...
        const int r = (int)cta + i / quads * cluster, k = i % quads;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4* at = reinterpret_cast<const float4*>(exch) + r * 32 + (k ^ (r & 7));
        for (int c = 0; c < cluster; ++c) {
          const float4 v = ld_remote_f4(at, c);
          s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        const float z = 1.f / NS_ONE;
        const uint2 o = make_uint2(pack_f16(s.x * z, s.y * z), pack_f16(s.z * z, s.w * z));
        unsigned char* dst = mat + (k >> 4) * C_SUB + swz(r, (k & 15) >> 1) + (k & 1) * 8;
        for (int c = 0; c < cluster; ++c) st_remote_u2(dst, c, o);
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
      }
      umma_commit(done);
    }
    wait_products();
    for (int g = half; g < mp / 32; g += 2) {
      float v[32];
      get(tm + g * 32, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] *= alpha / NS_ONE;
      add(mat + s * NS_MAT, g * 32, v, beta);
      if (s2 >= 0) add(mat + s2 * NS_MAT, g * 32, v, beta2);
      put(mat + to * NS_MAT, g * 32, v, 1.f);
    }
  };
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
        }
      }
      umma_commit(done);
    }
    wait_products();
    const bool failed = *abort_flag != 0;
    for (int g = half; g < groups; g += 2) {
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
      if (!p.tall && p.cols % 8 == 0 && aligned16_dev(p.out) && g * 32 + 32 <= cols) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          reinterpret_cast<uint4*>(o + (int64_t)row * p.cols + c)[k] =
              make_uint4(pack_bf16(v[8 * k], v[8 * k + 1]), pack_bf16(v[8 * k + 2], v[8 * k + 3]),
                         pack_bf16(v[8 * k + 4], v[8 * k + 5]), pack_bf16(v[8 * k + 6], v[8 * k + 7]));
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (g * 32 + i < cols) o[p.tall ? (c + i) * p.cols + row : (int64_t)row * p.cols + c + i] = __float2bfloat16_rn(v[i]);
      }
    }
    if (!last) tmem_st_wait();
  };

  int s = 0;
  if (p.joint) {                                                 // the first two steps as one, see above
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

// ---- way in: sum of squares, then f16 (two halves for fp32), in the orientation of u ----------------------------------
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
ns_enter_kernel(const T* __restrict__ u, int64_t batch_stride, int64_t row_stride, int rows, int cols, float eps,
                const float* __restrict__ partial, int n_parts, __half* __restrict__ hi, __half* __restrict__ lo, int ld,
                float* __restrict__ t_out, int* __restrict__ status) {
  __shared__ float q_s;
  const int64_t b = blockIdx.y;
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
    if (blockIdx.x == 0) {
      t_out[b] = NS_ONE / (norm * q);
      if (b == 0) *status = 0;
    }
  }
  __syncthreads();
  const float q = q_s;
  const T* src = u + b * batch_stride;
  for (int r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += 256) {
      const float v = q * to_f32<T>(src[(int64_t)r * row_stride + c]);
      const __half h = __float2half_rn(v);
      const int64_t at = (b * rows + r) * ld + c;
      hi[at] = h;
      if (lo != nullptr) lo[at] = __float2half_rn((v - __half2float(h)) * NS_LO);
    }
}

// ---- way out where the result's rows cannot be stored as tiles --------------------------------------------------------
__global__ void __launch_bounds__(256)
ns_leave_kernel(const __half* __restrict__ x, int ld, int rows, int cols, const int* __restrict__ status,
                __nv_bfloat16* __restrict__ out) {
  const int64_t b = blockIdx.y;
  const bool failed = *status != 0;              // a wait gave up: no number is left to stand
  for (int r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += 256) {
      const float v = __half2float(x[(b * rows + r) * ld + c]) * (1.f / NS_ONE);
      out[(b * rows + r) * (int64_t)cols + c] = __float2bfloat16_rn(failed ? __int_as_float(0x7fffffff) : v);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------
template <int MODE, bool TALL> static int ns_launch(NsArgs& p, int64_t batch, int k_dim, cudaStream_t st) {
  auto kern = ns_product_kernel<MODE, TALL>;
  static DeviceOnce once;
  const int rc = once.get([&](int*) {
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM));
    return (int)BIBO_OK;
  });
  if (rc) return rc;
  p.m_tiles = (p.rows + NS_T - 1) / NS_T;
  p.n_tiles = (p.cols + NS_T - 1) / NS_T;
  p.k_blocks = (k_dim + BK - 1) / BK;
  p.n_work = batch * (MODE == NS_APPLY ? (int64_t)p.m_tiles * p.n_tiles : (int64_t)p.m_tiles * (p.m_tiles + 1) / 2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)std::min<int64_t>(sm_count() / 2, p.n_work));
  cfg.blockDim = dim3(NS_THREADS);
  cfg.dynamicSmemBytes = NS_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BIBO_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  BIBO_CHECK_LAUNCH("ns_product_kernel");
  return BIBO_OK;
}
template <int MODE> static int ns_product(NsArgs& p, int tall, int64_t batch, int k_dim, cudaStream_t st) {
  return tall ? ns_launch<MODE, true>(p, batch, k_dim, st) : ns_launch<MODE, false>(p, batch, k_dim, st);
}

// workspace of `batch` matrices: x twice and its lower half, four m x m matrices (f16, rows of 16-byte multiples), partial sums, t,
// status
struct NsLayout {
  int m, n, rows, cols, ldx, ldg;
  int64_t x_bytes, g_bytes, off_g, off_part, off_t, off_status, bytes;
  NsLayout(int64_t batch, int rows_, int cols_) {
    rows = rows_; cols = cols_;
    m = std::min(rows, cols);
    n = std::max(rows, cols);
    ldx = (cols + 7) / 8 * 8;
    ldg = (m + 7) / 8 * 8;
    auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
    x_bytes = up(batch * rows * (int64_t)ldx * 2);
    g_bytes = up(batch * m * (int64_t)ldg * 2);
    off_g = 3 * x_bytes;
    off_part = off_g + 4 * g_bytes;
    off_t = off_part + up(batch * NS_MAX_PARTS * 4);
    off_status = off_t + up(batch * 4);
    bytes = off_status + 256;
  }
};
// matrices that run together: as many as a workspace of 2 GiB holds, one at least
static int64_t ns_chunk(int64_t batch, int rows, int cols) {
  const int64_t one = NsLayout(1, rows, cols).bytes;
  return std::max<int64_t>(1, std::min<int64_t>({batch, (2ll << 30) / one, 32768}));
}

// CTAs per matrix of the one-launch kernel, 0: it does not take these sizes.  Slices of at most NS_SM_COLS columns; beyond that as
// many CTAs as the machine has for the batch, while a slice keeps 128 columns.
static int ns_small_cluster(int64_t batch, int rows, int cols) {
  const int m = std::min(rows, cols), n = std::max(rows, cols);
  if (m > BM || n > NS_SM_COLS * NS_SM_MAX_CLUSTER) return 0;
  int c = 1;
  while ((int64_t)c * NS_SM_COLS < n) c *= 2;
  while (c < NS_SM_MAX_CLUSTER && n >= 256 * c && batch * 2 * c <= sm_count()) c *= 2;
  return c;
}
template <typename T>
static int ns_small(const void* u, int64_t batch, int64_t batch_stride, int rows, int cols, int64_t row_stride, int steps, bool joint,
                    const float* co, float eps, int cluster, void* out, cudaStream_t st) {
  auto kern = ns_small_kernel<T>;
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
    BIBO_CUDA(cudaLaunchKernelEx(&cfg, kern, p, cluster));
    BIBO_CHECK_LAUNCH("ns_small_kernel");
  }
  return BIBO_OK;
}

static int ns_maps(NsMaps* m, const void* base, int64_t batch, int rows, int cols, int ld) {
  const int rc = make_tmap_f16_3d(&m->r128, base, batch, rows, cols, ld, BM);
  return rc ? rc : make_tmap_f16_3d(&m->r64, base, batch, rows, cols, ld, 64);
}

}  // namespace tc
}  // namespace bibo

using namespace bibo;
using namespace bibo::tc;

extern "C" int64_t bibo_moe_orthogonalize_workspace(int64_t batch, int rows, int cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0 || ns_small_cluster(batch, rows, cols)) return 0;
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
  const int cluster = ns_small_cluster(batch, rows, cols);
  if (!u || (!workspace && !cluster) || !out) return fail(BIBO_ERR_ARG, "orthogonalize: null pointer");
  if ((reinterpret_cast<uintptr_t>(workspace) & 127u) != 0) return fail(BIBO_ERR_ALIGN, "orthogonalize: workspace not 128-byte aligned");
  if ((rows > 1 && row_stride < cols) || (batch > 1 && batch_stride < (rows - 1) * row_stride + cols))
    return fail(BIBO_ERR_ARG, "orthogonalize: overlapping rows or matrices");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int tall = rows > cols, size = dtype == BIBO_F32 ? 4 : 2;
  const int64_t chunk = ns_chunk(batch, rows, cols);
  const float* co = coefficients_host;
  // the first two steps as one, where their joint matrices stay in range (|T| <= a1^2, |R| <= a1 a2) and a step follows
  const bool joint = steps >= 3 && co[0] * co[0] <= 14.f && co[0] * co[3] <= 14.f && co[0] > 0.f && co[3] > 0.f;
  if (cluster)
    return dtype == BIBO_F32
               ? ns_small<float>(u, batch, batch_stride, rows, cols, row_stride, steps, joint, co, eps, cluster, out, st)
               : ns_small<__nv_bfloat16>(u, batch, batch_stride, rows, cols, row_stride, steps, joint, co, eps, cluster, out, st);
  for (int64_t b0 = 0; b0 < batch; b0 += chunk) {
    const int64_t nb = std::min(chunk, batch - b0);
    const NsLayout l(nb, rows, cols);
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    __half* x[3] = {reinterpret_cast<__half*>(ws), reinterpret_cast<__half*>(ws + l.x_bytes), reinterpret_cast<__half*>(ws + 2 * l.x_bytes)};
    float* partial = reinterpret_cast<float*>(ws + l.off_part);
    float* t = reinterpret_cast<float*>(ws + l.off_t);
    int* status = reinterpret_cast<int*>(ws + l.off_status);
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(out) + b0 * rows * cols;
    const unsigned char* src = static_cast<const unsigned char*>(u) + b0 * batch_stride * size;
    const int parts = std::min(NS_MAX_PARTS, rows);
    const dim3 sum_grid(parts, (unsigned)nb), row_grid(std::min(rows, 65535), (unsigned)nb);
    if (dtype == BIBO_F32) {
      ns_sumsq_kernel<float><<<sum_grid, 256, 0, st>>>(reinterpret_cast<const float*>(src), batch_stride, row_stride, rows, cols, partial);
      BIBO_CHECK_LAUNCH("ns_sumsq_kernel");
      ns_enter_kernel<float><<<row_grid, 256, 0, st>>>(reinterpret_cast<const float*>(src), batch_stride, row_stride, rows, cols, eps,
                                                      partial, parts, x[0], x[2], l.ldx, t, status);
    } else {
      ns_sumsq_kernel<__nv_bfloat16><<<sum_grid, 256, 0, st>>>(reinterpret_cast<const __nv_bfloat16*>(src), batch_stride, row_stride,
                                                              rows, cols, partial);
      BIBO_CHECK_LAUNCH("ns_sumsq_kernel");
      ns_enter_kernel<__nv_bfloat16><<<row_grid, 256, 0, st>>>(reinterpret_cast<const __nv_bfloat16*>(src), batch_stride, row_stride,
                                                              rows, cols, eps, partial, parts, x[0], nullptr, l.ldx, t, status);
    }
    BIBO_CHECK_LAUNCH("ns_enter_kernel");
    NsMaps mx[3], mm[4];                     // x, x', lower half;  m x m matrices
    CUtensorMap mout;
    int rc;
    for (int i = 0; i < 3; ++i)
      if ((rc = ns_maps(&mx[i], x[i], nb, rows, cols, l.ldx))) return rc;
    for (int i = 0; i < 4; ++i)
      if ((rc = ns_maps(&mm[i], ws + l.off_g + i * l.g_bytes, nb, l.m, l.m, l.ldg))) return rc;
    const bool direct = cols % 8 == 0 && aligned16(dst);        // the result's rows can be stored as tiles
    if (direct && (rc = make_tmap_f16_3d(&mout, dst, nb, rows, cols, cols, BM))) return rc;

    NsArgs base = {};
    base.status = status;
    auto gram = [&](int from, int to, const float* ts) {
      NsArgs p = base;
      p.a = p.b = mx[from];
      p.s_hi = p.s_lo = p.c_hi = p.c_lo = mm[to].r128;
      p.rows = p.cols = l.m;
      p.alpha = 1.f / NS_ONE;
      p.t_scale = ts;
      return ns_product<NS_GRAM>(p, tall, nb, l.n, st);
    };
    // mm[to] = alpha mm[a] mm[b] + beta mm[s] + beta2 mm[s2]
    auto sym = [&](int a, int b, float alpha, int s, float beta, int s2, float beta2, int to) {
      NsArgs p = base;
      p.a = mm[a];
      p.b = mm[b];
      p.s_hi = mm[s].r128;
      p.s_lo = mm[s2 < 0 ? s : s2].r128;
      p.c_hi = p.c_lo = mm[to].r128;
      p.rows = p.cols = l.m;
      p.has_s = 1;
      p.has_lo = s2 >= 0;
      p.alpha = alpha / NS_ONE;
      p.beta = beta;
      p.beta_lo = beta2;
      return ns_launch<NS_SYM, false>(p, nb, l.m, st);
    };
    // x[1 - from] = mm[f] x + a x
    auto apply = [&](int f, int from, float a, bool lo_in, bool lo_out, bool last, const float* ts) {
      NsArgs p = base;
      p.a = tall ? mx[from] : mm[f];
      p.b = tall ? mm[f] : mx[from];
      p.s_hi = mx[from].r128;
      p.s_lo = p.c_lo = mx[2].r128;
      p.c_hi = last && direct ? mout : mx[1 - from].r128;
      p.out_bf16 = last && direct;
      p.out = dst;
      p.rows = rows;
      p.cols = cols;
      p.has_s = 1;
      p.has_lo = lo_in;
      p.out_lo = lo_out;
      p.alpha = 1.f / NS_ONE;
      p.beta = a;
      p.beta_lo = a / NS_LO;
      p.t_scale = ts;
      return ns_product<NS_APPLY>(p, tall, nb, l.m, st);
    };
    int at = 0, s = 0;
    bool lo = dtype == BIBO_F32;             // x[2] holds the lower half of x[at]
    const float* ts = t;
    if (joint) {
      const float a1 = co[0], a2 = co[3];
      if ((rc = gram(0, 0, ts))) return rc;
      if ((rc = sym(0, 0, co[2], 0, co[1], -1, 0.f, 1))) return rc;       // F1 = b1 G + c1 G^2
      if ((rc = sym(1, 1, 1.f, 1, 2.f * a1, -1, 0.f, 2))) return rc;       // T  = F1^2 + 2 a1 F1
      if ((rc = sym(2, 0, 1.f, 0, a1 * a1, -1, 0.f, 3))) return rc;        // G' = a1^2 G + T G
      if ((rc = sym(3, 3, co[5], 3, co[4], -1, 0.f, 0))) return rc;       // F2 = b2 G' + c2 G'^2
      if ((rc = sym(0, 1, 1.f, 0, a1, 1, a2, 2))) return rc;              // R  = F2 F1 + a1 F2 + a2 F1
      if ((rc = apply(2, 0, a1 * a2, lo, true, false, ts))) return rc;
      at = 1;
      s = 2;
      lo = true;
      ts = nullptr;
    }
    for (; s < steps; ++s) {
      if ((rc = gram(at, 0, ts))) return rc;
      if ((rc = sym(0, 0, co[3 * s + 2], 0, co[3 * s + 1], -1, 0.f, 1))) return rc;
      if ((rc = apply(1, at, co[3 * s], lo, false, s == steps - 1, ts))) return rc;
      at = 1 - at;
      lo = false;
      ts = nullptr;
    }
    if (!direct) {
      ns_leave_kernel<<<row_grid, 256, 0, st>>>(x[at], l.ldx, rows, cols, status, dst);
      BIBO_CHECK_LAUNCH("ns_leave_kernel");
    }
  }
  return BIBO_OK;
}
