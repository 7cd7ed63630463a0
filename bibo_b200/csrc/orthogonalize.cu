// Newton-Schulz orthogonalisation of stacked matrices, the update of an optimiser that steps along the orthogonal
// factor of the momentum of the expert stacks [E,2I,H] / [E,H,I] and the router weight:
//   x_0 = u / (|u|_F + eps);   x_{k+1} = a x_k + (b G + c G^2) x_k,  G = x_k x_k^T   (m x n with m <= n; a tall u is used
//   as it lies, with G = x^T x and the products' sides swapped), out = bf16(x_steps)
// An odd polynomial of the singular values is applied and the singular vectors stay.
//
// Numbers.  The products run on the tensor cores with f16 operands and fp32 accumulators: bf16 operands would lose
// three bits more, tf32 would halve the rate for none, and the range is bounded (|x|_2 <= about 1.2 for the usual
// coefficients, so every entry of x, G and b G + c G^2 is below 16).  All three are kept times 2^12, which centres
// them in f16's range: an entry of 2^-26 is still a normal number.  u enters scaled by a power of two (exact for bf16)
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
// Error against 64 bits, relative in the Frobenius norm, five steps of the usual coefficients; the result's own rounding to bf16 is
// 0.0017 of it, and all that fp32 products leave.  Mean (largest) of 16-32 matrices with a momentum's decaying spectrum, then of
// Gaussian ones, whose singular values are alike and may all lie where the five steps are steep:
//   both sides 512 and more            0.0017 (0.0017)  0.0019-0.0022 (0.0023)
//   short side 129 to 511              0.0017-0.0019 (0.0019)  0.0021-0.0023 (0.0024)
//   short side 65 to 128               0.0018-0.0021 (0.0022)  0.0023-0.0026 (0.0028)
//   16 to 64, in one launch            0.0018-0.0022 (0.0025)  0.0021-0.0025 (0.0035)
//   16 to 64, longer than one launch takes (the m x m matrices are single f16 here)   0.0020-0.0026 (0.0032)  0.0022-0.0035 (0.0040)
//   8 by 8, 8 by 3200                  0.0024 (0.0030), 0.0033 (0.0047)  0.0028 (0.0036), 0.0030 (0.0039); one of 12 by 16384 0.0053
//   4 by 4, 2 by 2                     0.0031 (0.0059), 0.0022 (0.0045)  0.0034 (0.0052), 0.0031 (0.0119)
// Roundings of a matrix of many entries average out in its singular values, those of a few entries do not.
//
// Symmetric products (G, F, T, R, the second G) are computed and stored on and below the diagonal's 256 x 256 tiles only; an
// operand tile above it is read as the transposed tile below it, as an MN-major operand.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "orthogonalize_common.cuh"

namespace bibo {
namespace tc {

constexpr int NS_MAX_PARTS = 256;                // partial sums of squares per matrix

// ---- products ----------------------------------------------------------------------------------------------------
// 256 x 256 tiles: a CTA pair runs tcgen05.mma.cta_group::2 (256 x 256 x 16), each CTA staging its 128 rows of A and its half of
// B's rows, four or five stages of 32 KB.  Warps: 0 loads, 1 products (pair leader), 2 loads the sources of the drain and stores its
// results, 4-11 drain (two warps per quarter of the rows, 32 columns each: with one, a scheduler has nothing to run while its
// warp waits, and a sub-tile took 1600 cycles).  Results leave in sub-tiles of 64 columns through slots of 16 KB (32 KB where
// values come or go in two halves): source halves in, result halves out, in place.
constexpr int NS_GRAM = 0, NS_SYM = 1, NS_APPLY = 2;
constexpr int NS_T = 256, NS_STAGES = 5, NS_DRAIN = 256, NS_THREADS = 128 + NS_DRAIN;
constexpr int NS_OFF_A = 0;
constexpr int NS_OFF_B = NS_OFF_A + NS_STAGES * A_BYTES;
constexpr int NS_OFF_SLOT = NS_OFF_B + NS_STAGES * A_BYTES;      // 4 slots of {upper [128 x 64]} or 2 of {upper, lower}
constexpr int NS_OFF_BAR = NS_OFF_SLOT + 4 * C_SUB;
constexpr int NS_SMEM = NS_OFF_BAR + 256 + 1024;

struct NsMaps {            // a matrix of a batch with boxes of 128 rows (K-major operands, sources, results) and 64 rows (MN-major)
  CUtensorMap r128, r64;
};
struct NsArgs {
  NsMaps a, b;
  CUtensorMap s_hi, s_lo, c_hi, c_lo;
  int64_t n_work, batch;
  int m_tiles, n_tiles, k_blocks;
  int rows, cols;            // of the result
  int has_s, has_lo, out_lo; // source; source's or second source's map s_lo; result in two halves
  int backwards;             // the tiles in reverse: what the launch before wrote last is still in L2 and is read first
  int out_bf16;              // the last product: c_hi is the caller's bf16 result
  float alpha, beta, beta_lo;   // C = alpha A B + beta S_hi + beta_lo S_lo
  const float* t_scale;      // first products: t of each matrix
  int* status;
  __nv_bfloat16* out;        // with out_bf16: the result itself, for a run that gave up
};

struct NsTile { int b, i, j; };
template <int MODE> __device__ __forceinline__ NsTile ns_decode(int64_t w, const NsArgs& p) {
  const int m_tiles = p.m_tiles, n_tiles = p.n_tiles;
  if (p.backwards) w = p.n_work - 1 - w;
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

template <int MODE, bool TALL> struct NsOps {
  static constexpr int A = MODE == NS_GRAM ? (TALL ? OP_MN : OP_K) : MODE == NS_SYM ? OP_SYM : TALL ? OP_K : OP_SYM;
  static constexpr int B = MODE == NS_GRAM ? (TALL ? OP_MN : OP_K) : MODE == NS_SYM ? OP_SYM : TALL ? OP_SYM : OP_MN;
  // both operands of a CTA are the same rows of x
  static __device__ __forceinline__ bool same(const NsTile& t) { return MODE == NS_GRAM && t.i == t.j; }
};

struct NsBars {                                  // barriers and flags in shared memory
  uint64_t *full, *empty, *tfull, *tempty, *sfull, *cfull, *pfull;   // [stages], [stages], [2], [2], [6], [6], [1]
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  __device__ explicit NsBars(unsigned char* smem) {
    full = reinterpret_cast<uint64_t*>(smem + NS_OFF_BAR);   // pair leader
    empty = full + NS_STAGES;
    tfull = empty + NS_STAGES;
    tempty = tfull + 2;                                      // pair leader: the drain warps of both CTAs
    sfull = tempty + 2;                                      // a slot's sources have landed (and its last store has left)
    cfull = sfull + 6;                                       // a slot's results are written
    pfull = cfull + 6;                                       // the other pairs' partial sums have landed
    tmem_slot = reinterpret_cast<uint32_t*>(pfull + 1);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  }
  __device__ __forceinline__ void init() const {
    for (int s = 0; s < NS_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 2 * NS_DRAIN / 32); }
    for (int b = 0; b < 6; ++b) { mbar_init(&sfull[b], 1); mbar_init(&cfull[b], NS_DRAIN); }
    mbar_init(pfull, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
};

// k-blocks [k0, k1) of a tile into the stages; one thread of each CTA of the pair
template <int MODE, bool TALL, int STAGES = NS_STAGES>
__device__ __forceinline__ bool ns_produce(unsigned char* smem, const NsArgs& p, const NsBars& s, const NsTile& t, int k0, int k1,
                                           int pr, uint32_t leader, PipeState& ps) {
  using Ops = NsOps<MODE, TALL>;
  const bool same = Ops::same(t);
  for (int kb = k0; kb < k1; ++kb) {
    if (!mbar_wait<true>(&s.empty[ps.stage], ps.phase ^ 1, s.abort_flag)) return false;
    if (pr == 0) mbar_expect_tx(&s.full[ps.stage], same ? 2 * A_BYTES : 4 * A_BYTES);
    const uint32_t bar = map_to_cta(&s.full[ps.stage], leader);
    ns_load<Ops::A>(smem + NS_OFF_A + ps.stage * A_BYTES, p.a, bar, t.i, pr, kb, t.b);
    if (!same) ns_load<Ops::B>(smem + NS_OFF_A + (STAGES + ps.stage) * A_BYTES, p.b, bar, t.j, pr, kb, t.b);
    ps.next<STAGES>();
  }
  return true;
}
// ... and their products onto 256 accumulator columns; one thread of the pair leader
template <int MODE, bool TALL, int STAGES = NS_STAGES>
__device__ __forceinline__ bool ns_multiply(unsigned char* smem, const NsBars& s, const NsTile& t, int k0, int k1, uint32_t tmem_d,
                                            uint16_t pair_mask, PipeState& ps) {
  using Ops = NsOps<MODE, TALL>;
  const bool same = Ops::same(t);
  for (int kb = k0; kb < k1; ++kb) {
    if (!mbar_wait<true>(&s.full[ps.stage], ps.phase, s.abort_flag)) return false;
    tc_fence_after();
    const uint32_t sa = smem_u32(smem + NS_OFF_A + ps.stage * A_BYTES);
    const uint32_t sb = same ? sa : smem_u32(smem + NS_OFF_A + (STAGES + ps.stage) * A_BYTES);
    const bool amn = ns_mn_major<Ops::A>(t.i, kb), bmn = ns_mn_major<Ops::B>(t.j, kb);
    const uint64_t da = amn ? make_sdesc_mn128(sa) : make_sdesc_k128(sa);
    const uint64_t db = bmn ? make_sdesc_mn128(sb) : make_sdesc_k128(sb);
    const int a_step = amn ? (2048 >> 4) : (32 >> 4), b_step = bmn ? (2048 >> 4) : (32 >> 4);
    // bit 15: A is MN-major, bit 16: B is MN-major
    const uint32_t idesc = make_idesc_f16(2 * BM, NS_T) | (amn ? 1u << 15 : 0u) | (bmn ? 1u << 16 : 0u);
#pragma unroll
    for (int k = 0; k < BK / UK; ++k)
      umma_bf16_cg2(tmem_d, da + k * a_step, db + k * b_step, idesc, (kb > k0) | (k != 0));
    umma_commit_cg2_mc(&s.empty[ps.stage], pair_mask);
    ps.next<STAGES>();
  }
  return true;
}

struct NsScale { float al, be, bl; bool poison; };
template <int MODE> __device__ __forceinline__ NsScale ns_scale(const NsArgs& p, int b, bool poison) {
  NsScale c{p.alpha, p.beta, p.beta_lo, poison};
  if (p.t_scale != nullptr) {
    const float ts = p.t_scale[b];
    c.al *= MODE == NS_GRAM ? ts * ts : ts;
    c.be *= ts;
    c.bl *= ts;
  }
  return c;
}
// 32 accumulator columns of a row (half `h` of a sub-tile) and its sources -> results, in the slot
__device__ __forceinline__ void ns_finish(const NsArgs& p, const NsScale& c, const float (&acc)[32], unsigned char* slot, int row,
                                          int h) {
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) {
    uint4* hi = reinterpret_cast<uint4*>(slot + swz(row, 4 * h + jj));
    uint4* lo = reinterpret_cast<uint4*>(slot + C_SUB + swz(row, 4 * h + jj));
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c.al * acc[8 * jj + i];
    if (p.has_s) {
      const uint4 s = *hi;
      const uint32_t* ps = reinterpret_cast<const uint32_t*>(&s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_f16(ps[i]);
        v[2 * i] = fmaf(c.be, f.x, v[2 * i]);
        v[2 * i + 1] = fmaf(c.be, f.y, v[2 * i + 1]);
      }
    }
    if (p.has_lo) {
      const uint4 s = *lo;
      const uint32_t* ps = reinterpret_cast<const uint32_t*>(&s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_f16(ps[i]);
        v[2 * i] = fmaf(c.bl, f.x, v[2 * i]);
        v[2 * i + 1] = fmaf(c.bl, f.y, v[2 * i + 1]);
      }
    }
    uint4 o;
    uint32_t* po = reinterpret_cast<uint32_t*>(&o);
    if (p.out_bf16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        po[i] = c.poison ? 0x7fff7fffu : pack_bf16(v[2 * i] * (1.f / NS_ONE), v[2 * i + 1] * (1.f / NS_ONE));
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
}
// a wait gave up: lets copies in flight to this shared memory end, raises the status and voids this CTA's part of the caller's result
template <int MODE> __device__ __forceinline__ void ns_give_up(const NsArgs& p, int64_t w0, int64_t dw, int pr) {
  for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  if (threadIdx.x == 0) atomicExch(p.status, 112);
  if (!p.out_bf16) return;
  for (int64_t w = w0; w < p.n_work; w += dw) {
    const NsTile t = ns_decode<MODE>(w, p);
    for (int i = threadIdx.x; i < BM * NS_T; i += NS_THREADS) {
      const int y = t.i * NS_T + pr * BM + i / NS_T, x = t.j * NS_T + i % NS_T;
      if (y < p.rows && x < p.cols) p.out[((int64_t)t.b * p.rows + y) * p.cols + x] = __ushort_as_bfloat16(0x7fff);
    }
  }
}
__device__ __forceinline__ unsigned char* ns_smem() {
  extern __shared__ unsigned char smem_dyn[];
  return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
}

// Many tiles: persistent pairs, 2 x 256 accumulator columns, so the drain of a tile runs under the next one's products.  STAGES of 32 KB, the
// rest of the 224 KB are slots.
template <int MODE, bool TALL, int STAGES>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_product_kernel(const __grid_constant__ NsArgs p) {
  unsigned char* smem = ns_smem();
  const NsBars s(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pr = (int)(cluster_ctarank() & 1u);
  const int64_t w0 = blockIdx.x / 2, dw = gridDim.x / 2;
  pdl_launch_next();
  if (threadIdx.x == 0) {
    s.init();
    prefetch_tmap(&p.a.r128); prefetch_tmap(&p.a.r64); prefetch_tmap(&p.b.r128); prefetch_tmap(&p.b.r64);
    prefetch_tmap(&p.s_hi); prefetch_tmap(&p.c_hi);
  }
  if (warp == 1) { tmem_alloc_cg2(s.tmem_slot, 2 * NS_T); tmem_relinquish_cg2(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *s.tmem_slot;
  pdl_wait();
  const int halves = p.has_lo || p.out_lo ? 2 : 1, slots = (2 * NS_STAGES + 4 - 2 * STAGES) / halves;
  auto slot_at = [&](int i) { return smem + 2 * STAGES * A_BYTES + i * halves * C_SUB; };

  if (warp == 0) {
    if (elect_one()) {
      PipeState ps;
      bool ok = true;
      for (int64_t w = w0; w < p.n_work && ok; w += dw)
        ok = ns_produce<MODE, TALL, STAGES>(smem, p, s, ns_decode<MODE>(w, p), 0, p.k_blocks, pr, 0, ps);
    }
  } else if (warp == 1) {
    if (pr == 0 && elect_one()) {
      PipeState ps;
      int acc = 0;
      uint32_t acc_phase = 0;
      for (int64_t w = w0; w < p.n_work; w += dw) {
        if (!mbar_wait<true>(&s.tempty[acc], acc_phase ^ 1, s.abort_flag)) break;
        tc_fence_after();
        if (!ns_multiply<MODE, TALL, STAGES>(smem, s, ns_decode<MODE>(w, p), 0, p.k_blocks, tmem_base + acc * NS_T, 3, ps)) break;
        umma_commit_cg2_mc(&s.tfull[acc], 3);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else if (warp == 2) {
    if (elect_one()) {
      // sub-tile u of this CTA: tile w0 + (u / 4) * dw, columns (u % 4) * 64; a sub-tile outside the result is passed through
      const int64_t n_sub = w0 < p.n_work ? ((p.n_work - 1 - w0) / dw + 1) * 4 : 0;
      auto place = [&](int64_t u, NsTile& t, int& x, int& y) {
        t = ns_decode<MODE>(w0 + (u >> 2) * dw, p);
        x = t.j * NS_T + (int)(u & 3) * 64;
        y = t.i * NS_T + pr * BM;
        return x < p.cols && y < p.rows;
      };
      auto source = [&](int64_t u, int slot) {
        if (u >= n_sub) return;
        uint64_t* bar = &s.sfull[slot];
        NsTile t;
        int x, y;
        if (!p.has_s || !place(u, t, x, y)) { mbar_arrive(bar); return; }
        mbar_expect_tx(bar, p.has_lo ? 2 * C_SUB : C_SUB);
        tma_load_3d(slot_at(slot), &p.s_hi, bar, x, y, t.b);
        if (p.has_lo) tma_load_3d(slot_at(slot) + C_SUB, &p.s_lo, bar, x, y, t.b);
      };
      for (int u = 0; u < slots; ++u) source(u, u);
      int slot = 0;
      uint32_t phase = 0;
      for (int64_t u = 0; u < n_sub; ++u) {
        if (!mbar_wait(&s.cfull[slot], phase, s.abort_flag)) break;
        NsTile t;
        int x, y;
        if (place(u, t, x, y)) {
          tma_store_3d(&p.c_hi, slot_at(slot), x, y, t.b);
          if (p.out_lo) tma_store_3d(&p.c_lo, slot_at(slot) + C_SUB, x, y, t.b);
          tma_store_commit();
        }
        if (u + slots < n_sub) {
          tma_store_wait_read();
          source(u + slots, slot);
        }
        if (++slot == slots) { slot = 0; phase ^= 1; }
      }
      tma_store_wait_all();
    }
  } else if (warp >= 4) {
    const int row = (warp & 3) * 32 + lane;
    const int h = (warp - 4) >> 2;
    const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const bool poison = p.out_bf16 && *p.status != 0;                 // an earlier product gave up: no number is left to stand
    int acc = 0, slot = 0;
    uint32_t acc_phase = 0, phase = 0;
    bool ok = true;
    for (int64_t w = w0; w < p.n_work && ok; w += dw) {
      const NsScale c = ns_scale<MODE>(p, ns_decode<MODE>(w, p).b, poison);
      ok = mbar_wait<true>(&s.tfull[acc], acc_phase, s.abort_flag);
      if (!ok) break;
      __syncwarp();
      tc_fence_after();
#pragma unroll 1
      for (int g = 0; g < 4; ++g) {
        float r[32];
        tmem_ld32(lane_addr + acc * NS_T + g * 64 + h * 32, reinterpret_cast<uint32_t*>(r));
        ok = mbar_wait(&s.sfull[slot], phase, s.abort_flag);
        __syncwarp();
        tmem_ld_wait();
        if (g == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_addr(map_to_cta(&s.tempty[acc], 0));
        }
        if (!ok) break;
        ns_finish(p, c, r, slot_at(slot), row, h);
        fence_proxy_async_smem();
        mbar_arrive(&s.cfull[slot]);
        if (++slot == slots) { slot = 0; phase ^= 1; }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*s.abort_flag) ns_give_up<MODE>(p, w0, dw, pr);
  cluster_sync_all();                            // nobody leaves while the pair's other CTA may still signal or read this one
  if (warp == 1) { tc_fence_after(); tmem_dealloc_cg2(tmem_base, 2 * NS_T); }
}

// Few tiles and a long k: a cluster of S pairs per tile, each with a part of the k-blocks.  The partial sums cross the cluster as bulk copies
// between shared memories, a warp's 32 rows at a time (stores of the drain's threads, one row each, took 9400 of 24000 cycles);
// pair s finishes columns [s, s+1) * 256 / S and sums in pair order.  4096 x 1024: the Gram product (k = 4096) 29 us on ten pairs
// alone, 17 us split.
// Shared memory: three stages (the copies leave from them), the partial sums that arrive, slots.
constexpr int NS_SP_STAGES = 3, NS_OFF_PART = 2 * NS_SP_STAGES * A_BYTES;
template <int MODE, bool TALL, int S>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_split_kernel(const __grid_constant__ NsArgs p) {
  constexpr int G = 4 / S;                       // sub-tiles of 64 columns that a CTA finishes
  constexpr int PART = BM * 256;                 // bytes of a partial sub-tile: [128 rows][64 columns] fp32
  constexpr int OFF_SLOT = NS_OFF_PART + (S - 1) * G * PART;
  static_assert((S - 1) * G * PART <= NS_OFF_PART, "what leaves fits into the stages");
  static_assert(OFF_SLOT + G * 2 * C_SUB <= NS_OFF_BAR, "what arrives and the slots fit behind them");
  unsigned char* smem = ns_smem();
  const NsBars s(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pr = (int)(rank & 1u), sp = (int)(rank >> 1);
  const uint32_t leader = rank & ~1u;
  const uint16_t pair_mask = (uint16_t)(3u << leader);
  const int64_t w = blockIdx.x / (2 * S);
  pdl_launch_next();
  if (threadIdx.x == 0) {
    s.init();
    mbar_expect_tx(s.pfull, (S - 1) * G * PART);
    prefetch_tmap(&p.a.r128); prefetch_tmap(&p.a.r64); prefetch_tmap(&p.b.r128); prefetch_tmap(&p.b.r64);
    prefetch_tmap(&p.s_hi); prefetch_tmap(&p.c_hi);
  }
  if (warp == 1) { tmem_alloc_cg2(s.tmem_slot, NS_T); tmem_relinquish_cg2(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *s.tmem_slot;
  pdl_wait();
  const NsTile t = ns_decode<MODE>(w, p);
  const int k0 = p.k_blocks * sp / S, k1 = p.k_blocks * (sp + 1) / S;
  const int row = (warp & 3) * 32 + lane, h = (warp - 4) >> 2;
  const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
  const int y = t.i * NS_T + pr * BM, x0 = t.j * NS_T + sp * G * 64;
  auto slot_at = [&](int i) { return smem + OFF_SLOT + i * 2 * C_SUB; };
  auto exists = [&](int i) { return x0 + i * 64 < p.cols && y < p.rows; };
  // A partial sub-tile: 8 KB per warp pair (32 rows), in it 4 KB per half of the columns: a warp's [32 rows][8 pieces of 16 bytes],
  // the pieces swizzled by the row
  auto piece = [&](unsigned char* part, int k) { return part + (warp & 3) * 8192 + h * 4096 + lane * 128 + ((k ^ (lane & 7)) << 4); };

  if (warp == 0) {
    if (elect_one()) {
      PipeState ps;
      ns_produce<MODE, TALL, NS_SP_STAGES>(smem, p, s, t, k0, k1, pr, leader, ps);
    }
  } else if (warp == 1) {
    if (pr == 0 && elect_one()) {
      PipeState ps;
      if (ns_multiply<MODE, TALL, NS_SP_STAGES>(smem, s, t, k0, k1, tmem_base, pair_mask, ps))
        umma_commit_cg2_mc(&s.tfull[0], pair_mask);
    }
  } else if (warp == 2) {
    if (elect_one()) {
      for (int i = 0; i < G; ++i) {
        if (!p.has_s || !exists(i)) { mbar_arrive(&s.sfull[i]); continue; }
        mbar_expect_tx(&s.sfull[i], p.has_lo ? 2 * C_SUB : C_SUB);
        tma_load_3d(slot_at(i), &p.s_hi, &s.sfull[i], x0 + i * 64, y, t.b);
        if (p.has_lo) tma_load_3d(slot_at(i) + C_SUB, &p.s_lo, &s.sfull[i], x0 + i * 64, y, t.b);
      }
      for (int i = 0; i < G; ++i) {
        if (!mbar_wait(&s.cfull[i], 0, s.abort_flag)) break;
        if (!exists(i)) continue;
        tma_store_3d(&p.c_hi, slot_at(i), x0 + i * 64, y, t.b);
        if (p.out_lo) tma_store_3d(&p.c_lo, slot_at(i) + C_SUB, x0 + i * 64, y, t.b);
        tma_store_commit();
      }
      tma_store_wait_all();
    }
  } else if (warp >= 4) {
    bool ok = mbar_wait<true>(&s.tfull[0], 0, s.abort_flag);     // this pair's products are done: its stages are free
    __syncwarp();
    tc_fence_after();
    const float mine = k1 > k0 ? 1.f : 0.f;                     // without a k-block of its own nothing was accumulated
#pragma unroll 1
    for (int d = 1; d < S && ok; ++d) {
      const int to = (sp + d) % S;
      const int o = sp < to ? sp : sp - 1;       // this pair's place among the others of `to`
#pragma unroll 1
      for (int i = 0; i < G; ++i) {
        unsigned char* out = smem + ((d - 1) * G + i) * PART;
        float r[32];
        tmem_ld32(lane_addr + (to * G + i) * 64 + h * 32, reinterpret_cast<uint32_t*>(r));
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float4 v = make_float4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
          if (mine == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(piece(out, k)) = v;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          const int at = (warp & 3) * 8192 + h * 4096;
          const uint32_t cta = (uint32_t)(2 * to + pr);
          asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(map_to_cta(smem + NS_OFF_PART + (o * G + i) * PART + at, cta)), "r"(smem_u32(out + at)), "r"(4096),
                       "r"(map_to_cta(s.pfull, cta)) : "memory");
        }
      }
    }
    const NsScale c = ns_scale<MODE>(p, t.b, p.out_bf16 && *p.status != 0);
    ok = ok && mbar_wait<true>(s.pfull, 0, s.abort_flag);
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < G && ok; ++i) {
      float r[32], v[32];
      tmem_ld32(lane_addr + (sp * G + i) * 64 + h * 32, reinterpret_cast<uint32_t*>(r));
      tmem_ld_wait();
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = 0.f;
#pragma unroll
      for (int o = 0; o < S; ++o) {
        if (o == sp) {
          if (mine != 0.f)
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] += r[k];
        } else {
          unsigned char* part = smem + NS_OFF_PART + ((o < sp ? o : o - 1) * G + i) * PART;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 f = *reinterpret_cast<const float4*>(piece(part, k));
            v[4 * k] += f.x; v[4 * k + 1] += f.y; v[4 * k + 2] += f.z; v[4 * k + 3] += f.w;
          }
        }
      }
      ok = mbar_wait(&s.sfull[i], 0, s.abort_flag);
      __syncwarp();
      if (!ok) break;
      ns_finish(p, c, v, slot_at(i), row, h);
      fence_proxy_async_smem();
      mbar_arrive(&s.cfull[i]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*s.abort_flag) ns_give_up<MODE>(p, w, p.n_work, pr);
  cluster_sync_all();                            // nobody leaves while copies to or from its shared memory may be under way
  if (warp == 1) { tc_fence_after(); tmem_dealloc_cg2(tmem_base, NS_T); }
}

// Few tiles: one CTA per 128 x 128 tile.  The tiles of a 256 x 256 block on the diagonal are all computed, so that what the pairs'
// kernel reads is there.
constexpr int NS_ST_BN = 128;
template <int MODE> __device__ __forceinline__ NsTile ns_decode_single(int64_t w, const NsArgs& p) {
  NsTile t;
  if (MODE == NS_APPLY) {
    const int64_t per = (int64_t)p.m_tiles * p.n_tiles;
    t.b = (int)(w / per);
    const int r = (int)(w % per);
    t.i = r % p.m_tiles;
    t.j = r / p.m_tiles;
  } else {
    // rows 2 h and 2 h + 1 have 2 h + 2 tiles each (one less where the last row is alone): h (h + 1) * 2 tiles lie before them
    const int per = (int)(p.n_work / p.batch);
    t.b = (int)(w / per);
    const int r = (int)(w % per);
    int h = (int)((sqrtf(2.f * r + 1.f) - 1.f) * 0.5f);
    while (2 * (h + 1) * (h + 2) <= r) ++h;
    while (2 * h * (h + 1) > r) --h;
    const int q = r - 2 * h * (h + 1), width = min(2 * h + 2, p.m_tiles);
    t.i = 2 * h + q / width;
    t.j = q % width;
  }
  return t;
}
template <int OP>
__device__ __forceinline__ void ns_load_single(unsigned char* dst, const NsMaps& m, uint64_t* bar, int tile, int kb, int b) {
  const int r0 = tile * BM;
  if (OP == OP_MN || (OP == OP_SYM && kb / (BM / BK) > tile)) {
    tma_load_3d(dst, &m.r64, bar, r0, kb * BK, b);
    tma_load_3d(dst + MN_BOX, &m.r64, bar, r0 + 64, kb * BK, b);
  } else {
    tma_load_3d(dst, &m.r128, bar, kb * BK, r0, b);
  }
}
template <int MODE, bool TALL>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_single_kernel(const __grid_constant__ NsArgs p) {
  using Ops = NsOps<MODE, TALL>;
  unsigned char* smem = ns_smem();
  const NsBars s(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_next();
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS_STAGES; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
    mbar_init(&s.tfull[0], 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&s.sfull[i], 1); mbar_init(&s.cfull[i], NS_DRAIN / 2); }
    *s.abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&p.a.r128); prefetch_tmap(&p.a.r64); prefetch_tmap(&p.b.r128); prefetch_tmap(&p.b.r64);
    prefetch_tmap(&p.s_hi); prefetch_tmap(&p.c_hi);
  }
  if (warp == 1) { tmem_alloc(s.tmem_slot, NS_ST_BN); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *s.tmem_slot;
  const int64_t w = blockIdx.x;
  const NsTile t = ns_decode_single<MODE>(w, p);
  const bool same = Ops::same(t);
  const int y = t.i * BM, x0 = t.j * NS_ST_BN;
  auto slot_at = [&](int i) { return smem + NS_OFF_SLOT + i * 2 * C_SUB; };
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      PipeState ps;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        if (!mbar_wait(&s.empty[ps.stage], ps.phase ^ 1, s.abort_flag)) break;
        mbar_expect_tx(&s.full[ps.stage], same ? A_BYTES : 2 * A_BYTES);
        ns_load_single<Ops::A>(smem + NS_OFF_A + ps.stage * A_BYTES, p.a, &s.full[ps.stage], t.i, kb, t.b);
        if (!same) ns_load_single<Ops::B>(smem + NS_OFF_B + ps.stage * A_BYTES, p.b, &s.full[ps.stage], t.j, kb, t.b);
        ps.next<NS_STAGES>();
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      PipeState ps;
      bool ok = true;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        ok = mbar_wait(&s.full[ps.stage], ps.phase, s.abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + NS_OFF_A + ps.stage * A_BYTES);
        const uint32_t sb = same ? sa : smem_u32(smem + NS_OFF_B + ps.stage * A_BYTES);
        const bool amn = Ops::A == OP_MN || (Ops::A == OP_SYM && kb / (BM / BK) > t.i);
        const bool bmn = Ops::B == OP_MN || (Ops::B == OP_SYM && kb / (BM / BK) > t.j);
        const uint64_t da = amn ? make_sdesc_mn128(sa) : make_sdesc_k128(sa);
        const uint64_t db = bmn ? make_sdesc_mn128(sb) : make_sdesc_k128(sb);
        const int a_step = amn ? (2048 >> 4) : (32 >> 4), b_step = bmn ? (2048 >> 4) : (32 >> 4);
        const uint32_t idesc = make_idesc_f16(BM, NS_ST_BN) | (amn ? 1u << 15 : 0u) | (bmn ? 1u << 16 : 0u);
#pragma unroll
        for (int k = 0; k < BK / UK; ++k) umma_bf16(tmem_base, da + k * a_step, db + k * b_step, idesc, (kb | k) != 0);
        umma_commit(&s.empty[ps.stage]);
        ps.next<NS_STAGES>();
      }
      if (ok) umma_commit(&s.tfull[0]);
    }
  } else if (warp == 2) {
    if (elect_one()) {
      for (int i = 0; i < 2; ++i) {
        if (!p.has_s || x0 + i * 64 >= p.cols) { mbar_arrive(&s.sfull[i]); continue; }
        mbar_expect_tx(&s.sfull[i], p.has_lo ? 2 * C_SUB : C_SUB);
        tma_load_3d(slot_at(i), &p.s_hi, &s.sfull[i], x0 + i * 64, y, t.b);
        if (p.has_lo) tma_load_3d(slot_at(i) + C_SUB, &p.s_lo, &s.sfull[i], x0 + i * 64, y, t.b);
      }
      for (int i = 0; i < 2; ++i) {
        if (!mbar_wait(&s.cfull[i], 0, s.abort_flag)) break;
        if (x0 + i * 64 >= p.cols) continue;
        tma_store_3d(&p.c_hi, slot_at(i), x0 + i * 64, y, t.b);
        if (p.out_lo) tma_store_3d(&p.c_lo, slot_at(i) + C_SUB, x0 + i * 64, y, t.b);
        tma_store_commit();
      }
      tma_store_wait_all();
    }
  } else if (warp >= 4) {
    const int row = (warp & 3) * 32 + lane, i = (warp - 4) >> 2;       // four warps per sub-tile of 64 columns
    const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + i * 64;
    const NsScale c = ns_scale<MODE>(p, t.b, p.out_bf16 && *p.status != 0);
    bool ok = mbar_wait(&s.tfull[0], 0, s.abort_flag) && mbar_wait(&s.sfull[i], 0, s.abort_flag);
    __syncwarp();
    tc_fence_after();
    if (ok) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float r[32];
        tmem_ld32(lane_addr + h * 32, reinterpret_cast<uint32_t*>(r));
        tmem_ld_wait();
        ns_finish(p, c, r, slot_at(i), row, h);
      }
      fence_proxy_async_smem();
      mbar_arrive(&s.cfull[i]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*s.abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    if (threadIdx.x == 0) atomicExch(p.status, 112);
    if (p.out_bf16)
      for (int i = threadIdx.x; i < BM * NS_ST_BN; i += NS_THREADS) {
        const int r = y + i / NS_ST_BN, x = x0 + i % NS_ST_BN;
        if (r < p.rows && x < p.cols) p.out[((int64_t)t.b * p.rows + r) * p.cols + x] = __ushort_as_bfloat16(0x7fff);
      }
  }
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, NS_ST_BN); }
}

// ---- way in: sum of squares, then f16 (two halves for fp32), in the orientation of u ----------------------------------
// A unit is up to NS_UNIT elements of a row (of the whole matrix where its rows follow each other); a block takes units blockIdx.x,
// + gridDim.x, ...  16-byte accesses where rows and pointers allow them.
constexpr int NS_UNIT = 8192;
template <typename T, typename F>
__device__ __forceinline__ void ns_units(const T* src, int64_t row_stride, int64_t rows, int64_t cols, bool vec, F&& f) {
  constexpr int VE = 16 / sizeof(T);
  const int64_t per_row = (cols + NS_UNIT - 1) / NS_UNIT;
  for (int64_t i = blockIdx.x; i < rows * per_row; i += gridDim.x) {
    const int64_t r = per_row == 1 ? i : i / per_row, c0 = per_row == 1 ? 0 : i % per_row * NS_UNIT;
    const int64_t end = min(cols, c0 + NS_UNIT);
    const T* at = src + r * row_stride;
    if (vec) {
#pragma unroll 4
      for (int64_t c = c0 + threadIdx.x * VE; c < end; c += 256 * VE) {
        const uint4 w = *reinterpret_cast<const uint4*>(at + c);
        const uint32_t x4[4] = {w.x, w.y, w.z, w.w};
        float v[VE];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (sizeof(T) == 4) v[k] = __uint_as_float(x4[k]);
          else { v[2 * k] = bf16_lo(x4[k]); v[2 * k + 1] = bf16_hi(x4[k]); }
        }
        f(r, c, v, std::integral_constant<int, VE>());
      }
    } else {
#pragma unroll 4
      for (int64_t c = c0 + threadIdx.x; c < end; c += 256) {
        float v[1] = {to_f32<T>(at[c])};
        f(r, c, v, std::integral_constant<int, 1>());
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
ns_sumsq_kernel(const T* __restrict__ u, int64_t batch_stride, int64_t row_stride, int64_t rows, int64_t cols, int vec,
                float* __restrict__ partial) {
  __shared__ float red[8];
  pdl_launch_next();
  pdl_wait();
  float s = 0.f;
  ns_units(u + (int64_t)blockIdx.y * batch_stride, row_stride, rows, cols, vec != 0, [&](int64_t, int64_t, const float* v, auto n) {
#pragma unroll
    for (int i = 0; i < n.value; ++i) s = fmaf(v[i], v[i], s);
  });
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
ns_enter_kernel(const T* __restrict__ u, int64_t batch_stride, int64_t row_stride, int64_t rows, int64_t cols, int vec, float eps,
                const float* __restrict__ partial, int n_parts, __half* __restrict__ hi, __half* __restrict__ lo, int64_t ld,
                float* __restrict__ t_out, int* __restrict__ status) {
  __shared__ float q_s;
  pdl_launch_next();
  pdl_wait();
  const int64_t b = blockIdx.y;
  if (threadIdx.x < 32) {
    float s = 0.f;
    for (int p = threadIdx.x; p < n_parts; p += 32) s += partial[b * NS_MAX_PARTS + p];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) {
      const float norm = sqrtf(s) + eps;
      int e = 0;
      float q = 1.f;
      if (norm > 0.f && norm < 3e38f) {
        frexpf(norm, &e);                        // norm = f * 2^e, f in [0.5, 1)
        q = ldexpf(1.f, 12 - e < 120 ? 12 - e : 120);
      }
      q_s = q;
      if (blockIdx.x == 0) {
        t_out[b] = NS_ONE / (norm * q);
        if (b == 0 && status != nullptr) *status = 0;
      }
    }
  }
  __syncthreads();
  const float q = q_s;
  hi += b * rows * ld;
  if (lo != nullptr) lo += b * rows * ld;
  ns_units(u + b * batch_stride, row_stride, rows, cols, vec != 0, [&](int64_t r, int64_t c, float* v, auto n) {
    constexpr int N = decltype(n)::value;
    __half h[N];
#pragma unroll
    for (int i = 0; i < N; ++i) { v[i] *= q; h[i] = __float2half_rn(v[i]); }
    __half* at = hi + r * ld + c;
    if constexpr (N == 8) *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(h);
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(at) = *reinterpret_cast<uint2*>(h);
    else at[0] = h[0];
    if (lo == nullptr) return;
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = __float2half_rn((v[i] - __half2float(h[i])) * NS_LO);
    at = lo + r * ld + c;
    if constexpr (N == 8) *reinterpret_cast<uint4*>(at) = *reinterpret_cast<uint4*>(h);
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(at) = *reinterpret_cast<uint2*>(h);
    else at[0] = h[0];
  });
}

// ---- way out where the result's rows cannot be stored as tiles --------------------------------------------------------
__global__ void __launch_bounds__(256)
ns_leave_kernel(const __half* __restrict__ x, int ld, int rows, int cols, const int* __restrict__ status,
                __nv_bfloat16* __restrict__ out) {
  pdl_launch_next();
  pdl_wait();
  const int64_t b = blockIdx.y;
  const bool failed = *status != 0;              // a wait gave up: no number is left to stand
  for (int r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += 256) {
      const float v = __half2float(x[(b * rows + r) * ld + c]) * (1.f / NS_ONE);
      out[(b * rows + r) * (int64_t)cols + c] = __float2bfloat16_rn(failed ? __int_as_float(0x7fffffff) : v);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------
// a kernel that may start under the tail of the one before it
template <typename Kern, typename... Args>
static int ns_start(Kern kern, dim3 grid, int threads, int smem, int cluster, cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  BIBO_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  BIBO_CHECK_LAUNCH("orthogonalize");
  return BIBO_OK;
}
template <typename Kern> static int ns_attributes(DeviceOnce& once, Kern kern) {
  return once.get([&](int*) {
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM));
    return (int)BIBO_OK;
  });
}
// how many clusters of S pairs are resident at once
template <int MODE, bool TALL, int S> static int ns_split_resident(int* clusters) {
  static DeviceOnce once;
  return once.get([&](int* v) {
    auto kern = ns_split_kernel<MODE, TALL, S>;
    BIBO_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * S);
    cfg.blockDim = dim3(NS_THREADS);
    cfg.dynamicSmemBytes = NS_SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BIBO_CUDA(cudaOccupancyMaxActiveClusters(v, kern, &cfg));
    return (int)BIBO_OK;
  }, clusters);
}
template <int MODE, bool TALL, int S> static int ns_launch_split(const NsArgs& p, cudaStream_t st) {
  return ns_start(ns_split_kernel<MODE, TALL, S>, dim3((unsigned)p.n_work * 2 * S), NS_THREADS, NS_SMEM, 2 * S, st, p);
}
template <int MODE, bool TALL, int STAGES> static int ns_launch_pairs(const NsArgs& p, cudaStream_t st) {
  static DeviceOnce once;
  const int rc = ns_attributes(once, ns_product_kernel<MODE, TALL, STAGES>);
  return rc ? rc : ns_start(ns_product_kernel<MODE, TALL, STAGES>, dim3(2 * (unsigned)std::min<int64_t>(sm_count() / 2, p.n_work)),
                            NS_THREADS, NS_SMEM, 2, st, p);
}
template <int MODE, bool TALL> static int ns_launch(NsArgs& p, int64_t batch, int k_dim, cudaStream_t st) {
  p.m_tiles = (p.rows + NS_T - 1) / NS_T;
  p.n_tiles = (p.cols + NS_T - 1) / NS_T;
  p.k_blocks = (k_dim + BK - 1) / BK;
  p.n_work = batch * (MODE == NS_APPLY ? (int64_t)p.m_tiles * p.n_tiles : (int64_t)p.m_tiles * (p.m_tiles + 1) / 2);
  p.batch = batch;
  // 128 x 128 tiles where they need no more waves than the pairs' tiles (up to two: beyond that the pairs' drain under the next
  // tile's products wins), unless k is so long that splitting it over pairs gains more than the exchange costs.  A wave takes
  // about the same either way, a CTA of both kernels loads 32 KB per k-block.  All steps of 1024 x 1024: 151 us this way, 186
  // split, 218 with a pair per tile; of 512 x 8192: 249 us against 198 split.
  if (p.k_blocks <= 40) {
    const int mt = (p.rows + BM - 1) / BM, nt = (p.cols + NS_ST_BN - 1) / NS_ST_BN;
    int64_t tiles = (int64_t)mt * nt;
    if (MODE != NS_APPLY) {
      tiles = 0;
      for (int i = 0; i < mt; ++i) tiles += std::min(i / 2 * 2 + 2, mt);
    }
    const int64_t sms = sm_count(), waves = (batch * tiles + sms - 1) / sms;
    if (waves <= 2 && waves <= (p.n_work + sms / 2 - 1) / (sms / 2)) {
      NsArgs q = p;
      q.m_tiles = mt;
      q.n_tiles = nt;
      q.n_work = batch * tiles;
      static DeviceOnce once1;
      const int rc1 = ns_attributes(once1, ns_single_kernel<MODE, TALL>);
      return rc1 ? rc1 : ns_start(ns_single_kernel<MODE, TALL>, dim3((unsigned)q.n_work), NS_THREADS, NS_SMEM, 1, st, q);
    }
  }
  // tiles so few that clusters of four (two) pairs for each are resident together are split over them
  int four = 0, two = 0;
  int rc = ns_split_resident<MODE, TALL, 4>(&four);
  if (!rc) rc = ns_split_resident<MODE, TALL, 2>(&two);
  if (rc) return rc;
  if (p.n_work <= four) return ns_launch_split<MODE, TALL, 4>(p, st);
  if (p.n_work <= two) return ns_launch_split<MODE, TALL, 2>(p, st);
  // Short k: a tile's products are over before its drain, which then wants slots more than the products want stages.  All steps of
  // 64 x 2048 x 512: 773 us with four stages, 805 with five, in runs too short to reach the power limit (885 in a long one); of 64 x 1024 x 2048 (k = 1024 and more) 2195 against 2170.
  return p.k_blocks <= 8 ? ns_launch_pairs<MODE, TALL, NS_STAGES - 1>(p, st) : ns_launch_pairs<MODE, TALL, NS_STAGES>(p, st);
}
template <int MODE> static int ns_product(NsArgs& p, int tall, int64_t batch, int k_dim, cudaStream_t st) {
  return tall ? ns_launch<MODE, true>(p, batch, k_dim, st) : ns_launch<MODE, false>(p, batch, k_dim, st);
}

// sums of squares and scaled x of nb matrices, in groups whose u (48 MB at most) is still in L2 for the second reading
template <typename T>
static int ns_enter(const T* u, int64_t nb, int64_t batch_stride, int rows, int cols, int64_t row_stride, float eps, float* partial,
                    __half* hi, __half* lo, int ldx, float* t, int* status, cudaStream_t st) {
  const int64_t bytes = (int64_t)rows * cols * sizeof(T);
  const int64_t group = std::max<int64_t>(1, std::min<int64_t>(nb, (48 << 20) / bytes));
  const bool whole_in = row_stride == cols || rows == 1, whole = whole_in && ldx == cols;   // rows follow each other: one long row
  const bool vec = ((reinterpret_cast<uintptr_t>(u) | (uintptr_t)(batch_stride * sizeof(T))) & 15) == 0 && cols * sizeof(T) % 16 == 0 &&
                   (whole_in || row_stride * sizeof(T) % 16 == 0);
  auto blocks = [&](bool one, int64_t n) {
    const int64_t units = one ? ((int64_t)rows * cols + NS_UNIT - 1) / NS_UNIT : (int64_t)rows * ((cols + NS_UNIT - 1) / NS_UNIT);
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>({units, NS_MAX_PARTS, (8 * (int64_t)sm_count() + n - 1) / n}));
  };
  for (int64_t g0 = 0; g0 < nb; g0 += group) {
    const int64_t n = std::min(group, nb - g0);
    const T* src = u + g0 * batch_stride;
    const unsigned parts = blocks(whole_in, n);
    int rc = ns_start(ns_sumsq_kernel<T>, dim3(parts, (unsigned)n), 256, 0, 1, st, src, batch_stride, row_stride,
                      whole_in ? (int64_t)1 : (int64_t)rows, whole_in ? (int64_t)rows * cols : (int64_t)cols, (int)vec,
                      partial + g0 * NS_MAX_PARTS);
    if (rc) return rc;
    rc = ns_start(ns_enter_kernel<T>, dim3(blocks(whole, n), (unsigned)n), 256, 0, 1, st, src, batch_stride, row_stride,
                  whole ? (int64_t)1 : (int64_t)rows, whole ? (int64_t)rows * cols : (int64_t)cols, (int)vec, eps,
                  (const float*)(partial + g0 * NS_MAX_PARTS), (int)parts, hi + g0 * rows * ldx,
                  lo ? lo + g0 * rows * ldx : (__half*)nullptr, whole ? (int64_t)rows * ldx : (int64_t)ldx, t + g0,
                  g0 == 0 ? status : (int*)nullptr);
    if (rc) return rc;
  }
  return BIBO_OK;
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

// ---- ranges of the polynomials -----------------------------------------------------------------------------------------
// The singular values of x_0 lie in [0, 1], and an odd polynomial of them is continuous, so the magnitudes after a step fill
// [0, M] with M its largest magnitude: each step's range is exact.  What is stored as f16 times 2^12 has to stay below 16.
constexpr double NS_LIMIT = 15.8, NS_LIMIT_X = 3.97;             // of matrices, and of an x whose Gram matrix is formed (x^2 < 15.8)
struct NsRange { double lo, hi; double magnitude() const { return std::max(-lo, hi); } };
// b z + c z^2 over z in [0, top^2]
static NsRange ns_range_factor(double b, double c, double top) {
  const double z = top * top, end = z * (b + c * z);
  NsRange r{std::min(0.0, end), std::max(0.0, end)};
  const double at = c != 0 ? -b / (2 * c) : 0, v = at * (b + c * at);
  if (at > 0 && at < z) { r.lo = std::min(r.lo, v); r.hi = std::max(r.hi, v); }
  return r;
}
// the largest |a s + b s^3 + c s^5| over s in [0, top]
static double ns_range_x(double a, double b, double c, double top) {
  double most = 0;
  auto see = [&](double z) {                     // z = s^2
    if (z > 0 && z <= top * top) most = std::max(most, std::sqrt(z) * std::abs(a + z * (b + c * z)));
  };
  see(top * top);
  if (c != 0) {                                  // a + 3 b z + 5 c z^2 = 0
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0) { see((-3 * b + std::sqrt(d)) / (10 * c)); see((-3 * b - std::sqrt(d)) / (10 * c)); }
  } else if (b != 0) {
    see(-a / (3 * b));
  }
  return most;
}
// The first step that leaves the range (-1: none).  joint: the first two steps may be one, with a step behind them.
static int ns_check_steps(int steps, const float* co, bool* joint) {
  double top = 1;
  *joint = steps >= 3 && co[0] * co[0] <= 14.f && co[0] * co[3] <= 14.f && co[0] > 0.f && co[3] > 0.f;
  for (int s = 0; s < steps; ++s) {
    const double a = co[3 * s], b = co[3 * s + 1], c = co[3 * s + 2];
    const NsRange f = ns_range_factor(b, c, top);
    const double next = ns_range_x(a, b, c, top);
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c) || !(f.magnitude() <= NS_LIMIT) ||
        !(next <= (s + 1 < steps ? NS_LIMIT_X : NS_LIMIT)))
      return s;
    if (s == 0 && *joint) {
      // T = (a1 + F1)^2 - a1^2 and R = (a2 + F2) (a1 + F1) - a1 a2; where the first polynomial stretches (b > 0, say) neither is
      // bounded by a1 and a2
      const NsRange f2 = ns_range_factor(co[4], co[5], next);
      const double l1 = a + f.lo, h1 = a + f.hi, l2 = co[3] + f2.lo, h2 = co[3] + f2.hi;
      const double r_lo = std::min({l1 * l2, l1 * h2, h1 * l2, h1 * h2}) - a * co[3];
      const double r_hi = std::max({l1 * l2, l1 * h2, h1 * l2, h1 * h2}) - a * co[3];
      const double t = std::max(std::max(l1 * l1, h1 * h1) - a * a, a * a);
      *joint = t <= NS_LIMIT && std::max(-r_lo, r_hi) <= NS_LIMIT;
    }
    top = next;
  }
  return -1;
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
  if (!(eps >= 0.f)) return fail(BIBO_ERR_ARG, "orthogonalize: eps=%g", eps);
  bool joint;                                    // the first two steps as one
  const int wide = ns_check_steps(steps, coefficients_host, &joint);
  if (wide >= 0)
    return fail(BIBO_ERR_UNSUPPORTED, "orthogonalize: step %d takes singular values from [0, 1] out of range (below 4 before the last step, "
                "|b s^2 + c s^4| below 16)", wide);
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
  if (cluster)
    return ns_small_launch(u, dtype, batch, batch_stride, rows, cols, row_stride, steps, joint, co, eps, cluster, out, st);
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
    const int rc0 = dtype == BIBO_F32
                        ? ns_enter(reinterpret_cast<const float*>(src), nb, batch_stride, rows, cols, row_stride, eps, partial, x[0], x[2],
                                   l.ldx, t, status, st)
                        : ns_enter(reinterpret_cast<const __nv_bfloat16*>(src), nb, batch_stride, rows, cols, row_stride, eps, partial,
                                   x[0], nullptr, l.ldx, t, status, st);
    if (rc0) return rc0;
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
    base.backwards = 0;
    auto gram = [&](int from, int to, const float* ts) {
      NsArgs p = base;
      base.backwards ^= 1;
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
      base.backwards ^= 1;
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
      base.backwards ^= 1;
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
      if ((rc = ns_start(ns_leave_kernel, dim3(std::min(rows, 65535), (unsigned)nb), 256, 0, 1, st, (const __half*)x[at], l.ldx, rows,
                         cols, (const int*)status, dst)))
        return rc;
    }
  }
  return BIBO_OK;
}
