// Matrix products of 16-bit operands with a fused epilogue, for the gated feed-forward block and
// the Newton-Schulz iteration: D = A B in fp32 (tensor memory), then an element-wise step that
// reads D (and sometimes one more matrix) and writes one to three 16-bit matrices.
//
//   op              D[i,j]                          written
//   kOpGate         g = x Wg^T and u = x Wu^T       act(g) u  (and g, u)
//   kOpDown         h Wd^T                          D
//   kOpDact         dh = dy Wd                      dg = dh u act'(g), du = dh act(g), h = act(g) u
//   kOpDx           [dg du] [Wg; Wu]                D
//   kOpDw           dg^T x, du^T x (or dy^T h)      D
//   kOpGramWide     x x^T  (kOpGramTall: x^T x)     p = D / S, on both sides of the diagonal
//   kOpPoly         p p                             q = b p + c D / S, likewise; vec = a + what the
//                                                   rounding of q's diagonal lost, / S
//   kOpUpdateWide   q x    (kOpUpdateTall: x q)     vec x + D / S as a 16-bit pair (or bf16, / S)
//
// Structure: the GEMM family's (one persistent CTA, or CTA pair, per SM): a TMA producer warp
// fills a ring of 64-deep k-blocks, one thread issues tcgen05.mma, eight epilogue warps empty one
// of two accumulators while the other one fills. What is different from that family: both
// operands may be contiguous along k or along m / n, maps are 3-D (a batch of matrices, the two
// halves [dg du]), the reduction may run over two pairs of matrices (kOpDx), a tile's columns
// may come from two matrices (kOpGate: each half of the tile from one weight, so the thread
// that holds g[i,j] also holds u[i,j] and neither reaches memory unless it is asked for), only one
// triangle of a symmetric product is computed, and a tile's reduction may be cut into `nsplit`
// parts.
//
// Split reductions: with few rows there are few tiles, and a weight has to be streamed by all SMs
// to come at the memory's rate. Each part leaves its fp32 sums in a workspace and counts itself
// in; the part that arrives last adds all of them in the parts' order (so the result does not
// depend on who was last) and runs the epilogue. Nobody waits for anybody.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fused_gemm.h"
#include "ptx_sm100.cuh"

namespace rb200 {

template <int OP_, int CG_, int BN_, int DT_>
struct FusedCfg {
  static constexpr int OP = OP_, CG = CG_, BN = BN_, DT = DT_;
  static constexpr int BM = 128, BK = 64;
  static constexpr int TILE_M = BM * CG;
  static constexpr int BNL = BN / CG;            // tile columns staged by one CTA
  static constexpr bool A_MN = (OP == kOpDw || OP == kOpGramTall);
  static constexpr bool B_MN = (OP == kOpDact || OP == kOpDx || OP == kOpDw || OP == kOpGramTall ||
                                OP == kOpUpdateWide);
  static constexpr bool SYM = (OP == kOpGramWide || OP == kOpGramTall || OP == kOpPoly);
  static constexpr bool UPDATE = (OP == kOpUpdateWide || OP == kOpUpdateTall);
  static constexpr int A_BYTES = BM * 128, B_BYTES = BNL * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // columns of D one epilogue warp owns, and columns of one box it hands to the TMA unit
  static constexpr int OUT_COLS = (OP == kOpGate ? BN / 4 : BN / 2);
  static constexpr int BOX_COLS = (OP == kOpDact || OUT_COLS < 64) ? 32 : 64;
  static constexpr int BOX_BYTES = BOX_COLS * 2 * 32;
  static constexpr int SET_BOXES = OP == kOpDact ? 3 : (SYM || UPDATE) ? 2 : 1;
  static constexpr int SET_BYTES = SET_BOXES * BOX_BYTES;
  static constexpr int EPI_WARPS = 8;
  static constexpr int STAGING_BYTES = EPI_WARPS * SET_BYTES;
  static constexpr int CTRL_BYTES = 256;
  static constexpr int SMEM_LIMIT = 232448;      // 227 KiB opt-in maximum per CTA
  static constexpr int STAGES_FIT = (SMEM_LIMIT - 1024 - CTRL_BYTES - STAGING_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT > 8 ? 8 : STAGES_FIT;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + STAGING_BYTES + CTRL_BYTES + 1024;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int FIRST_EPI_WARP = 4;
  static constexpr int THREADS = (FIRST_EPI_WARP + EPI_WARPS) * 32;
  static_assert(BN == 256 || BN == 128, "tile widths");
  static_assert(!SYM || TILE_M == BN, "one triangle of square tiles");
  static_assert(STAGES >= 3 && SMEM_BYTES <= SMEM_LIMIT, "shared memory");
};

template <int DT>
__device__ __forceinline__ uint32_t fused_pack(float lo, float hi) {
  if constexpr (DT == 1) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int DT>
__device__ __forceinline__ float2 fused_unpack(uint32_t w) {
  if constexpr (DT == 1) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ float sigmoidf_(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// act(v) and its slope. tanh appears only as 1 + tanh(z) = 2 sigmoid(2 z): a difference of small
// numbers never occurs, and the 2^-11 error of the hardware tanh stays out of fp16 results.
template <int ACT>
__device__ __forceinline__ void activation(float v, float& y, float& slope) {
  if constexpr (ACT == kActSilu) {
    const float p = sigmoidf_(v);
    y = v * p;
    slope = p * (1.0f + v * (1.0f - p));
  } else if constexpr (ACT == kActGelu) {
    const float p = 0.5f + 0.5f * erff(v * 0.70710678118654752f);
    y = v * p;
    slope = p + v * 0.39894228040143268f * __expf(-0.5f * v * v);
  } else {
    constexpr float c = 0.79788456080286536f;
    const float w = v * v;
    const float p = sigmoidf_(2.0f * c * v * (1.0f + 0.044715f * w));
    y = v * p;
    slope = p + 2.0f * c * v * p * (1.0f - p) * (1.0f + 3.0f * 0.044715f * w);
  }
}

// Barrier among the 256 epilogue threads carrying a vote.
__device__ __forceinline__ bool fused_bar_any(bool mine) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, 256, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(out)
      : "r"(static_cast<uint32_t>(mine))
      : "memory");
  return out != 0;
}

struct FusedTile {
  int z, mb, nb;
};

// Tile order. Rectangular problems: panels of 8 tile rows, so that the tiles in flight share
// operand rows and columns in L2. Symmetric ones: the lower triangle, row by row.
template <bool SYM>
__device__ __forceinline__ FusedTile fused_tile(int t, int tiles_m, int tiles_n, int per_z) {
  FusedTile c;
  c.z = t / per_z;
  int r = t - c.z * per_z;
  if constexpr (SYM) {
    int i = static_cast<int>((sqrtf(8.0f * static_cast<float>(r) + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > r) --i;
    while ((i + 1) * (i + 2) / 2 <= r) ++i;
    c.mb = i;
    c.nb = r - i * (i + 1) / 2;
  } else {
    constexpr int kPanel = 8;
    const int per_panel = kPanel * tiles_n;
    const int panel = r / per_panel;
    const int first = panel * kPanel;
    const int rows = min(tiles_m - first, kPanel);
    r -= panel * per_panel;
    c.mb = first + r % rows;
    c.nb = r / rows;
  }
  return c;
}

// Loads `ROWS` m/n values x 64 k of an operand at (row0, k0, z) into shared memory.
template <int ROWS, bool MN, bool PAIR>
__device__ __forceinline__ void fused_load(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int row0,
                                           int k0, int z) {
  if constexpr (MN) {
#pragma unroll
    for (int j = 0; j < ROWS / 64; ++j) {   // boxes of 64 k-rows of 64 values
      if constexpr (PAIR) tma_load_3d_pair(dst + j * 8192, tm, bar, row0 + j * 64, k0, z);
      else tma_load_3d(dst + j * 8192, tm, bar, row0 + j * 64, k0, z);
    }
  } else {
    if constexpr (PAIR) tma_load_3d_pair(dst, tm, bar, k0, row0, z);
    else tma_load_3d(dst, tm, bar, k0, row0, z);
  }
}
template <bool MN>
__device__ __forceinline__ uint64_t fused_desc(uint32_t addr) {
  // k-contiguous: 8-row swizzle atoms 1024 B apart; m/n-contiguous: atoms of 8 k-rows 1024 B
  // apart, the next 64 m/n values one box (8192 B) further
  return MN ? make_smem_desc(addr, 8192, 1024, kLayoutSw128) : make_smem_desc(addr, 16, 1024, kLayoutSw128);
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
fused_gemm_kernel(const __grid_constant__ FusedParams p) {
  constexpr int BN = Cfg::BN, CG = Cfg::CG, STAGES = Cfg::STAGES, DT = Cfg::DT, OP = Cfg::OP;
  extern __shared__ uint8_t smem_dyn[];
  const uint32_t smem_base = (smem_addr(smem_dyn) + 1023u) & ~1023u;
  const uint32_t staging = smem_base + STAGES * Cfg::STAGE_BYTES;
  const uint32_t ctrl = staging + Cfg::STAGING_BYTES;
  auto full_bar = [&](int s) { return ctrl + 8u * s; };
  auto empty_bar = [&](int s) { return ctrl + 64u + 8u * s; };
  auto tmem_full_bar = [&](int a) { return ctrl + 128u + 8u * a; };
  auto tmem_empty_bar = [&](int a) { return ctrl + 144u + 8u * a; };
  const uint32_t mma_done_bar = ctrl + 160u;
  const uint32_t tmem_slot = ctrl + 176u;
  const uint32_t last_slot = ctrl + 180u;   // outcome of the count of a split reduction
  const WaitCtx wc{p.status, p.spin_limit};

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = (CG == 2) ? cluster_ctarank() : 0u;
  const bool is_leader = (cta_rank == 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar(a), 1);
      mbar_init(tmem_empty_bar(a), CG * Cfg::EPI_WARPS);
    }
    mbar_init(mma_done_bar, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc<CG>(tmem_slot, Cfg::TMEM_COLS);
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.a);
    tma_prefetch_desc(&p.b[0]);
    if (OP == kOpGate || OP == kOpDx) tma_prefetch_desc(&p.b[1]);
  }
  grid_launch_dependents();
  tcgen05_fence_before_sync();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tcgen05_fence_after_sync();
  grid_dependency_wait();   // everything below touches memory that the previous kernel may have

  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));

  const int workers = static_cast<int>(gridDim.x) / CG;
  const int worker = static_cast<int>(blockIdx.x) / CG;
  const int per_z = p.tiles_per_z;
  const int units = per_z * p.zcount * p.nsplit;
  const int total_kb = p.num_kb * (OP == kOpDx ? 2 : 1);

  if (warp == 0 && lane == 0) {
    // ---------------------------------------------------------------- TMA producer
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int u = worker; ok && u < units; u += workers) {
      const int t = u / p.nsplit, part = u - t * p.nsplit;
      const FusedTile c = fused_tile<Cfg::SYM>(t, p.tiles_m, p.tiles_n, per_z);
      const int kb0 = static_cast<int>(static_cast<long long>(total_kb) * part / p.nsplit);
      const int kb1 = static_cast<int>(static_cast<long long>(total_kb) * (part + 1) / p.nsplit);
      const int m0 = (c.mb * CG + static_cast<int>(cta_rank)) * Cfg::BM;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(empty_bar(s), ph ^ 1u, wc, kDevTimeoutEmpty)) { ok = false; break; }
        const uint32_t a_dst = smem_base + s * Cfg::STAGE_BYTES;
        const uint32_t b_dst = a_dst + Cfg::A_BYTES;
        uint32_t bar = full_bar(s);
        if constexpr (CG == 2) {
          // the leader's barrier counts the bytes of both CTAs; only the leader arms it
          if (is_leader) mbar_expect_tx(bar, 2 * (Cfg::A_BYTES + Cfg::B_BYTES));
          bar = map_to_cta(bar, 0);
        } else {
          mbar_expect_tx(bar, p.a_bytes + Cfg::B_BYTES);
        }
        const int phase = (OP == kOpDx && kb >= p.num_kb) ? 1 : 0;
        const int k0 = (kb - phase * p.num_kb) * Cfg::BK;
        const int az = OP == kOpDx ? phase : c.z;
        const int bz = (OP == kOpDw || OP == kOpDx) ? 0 : c.z;
        fused_load<Cfg::BM, Cfg::A_MN, CG == 2>(a_dst, &p.a, bar, m0, k0, az);
        if constexpr (OP == kOpGate) {
          // tile columns: BN/2 rows of Wg, then the same BN/2 rows of Wu
          const int f0 = c.nb * (BN / 2);
          if constexpr (CG == 2) {
            fused_load<Cfg::BNL, false, true>(b_dst, &p.b[cta_rank], bar, f0, k0, 0);
          } else {
            fused_load<BN / 2, false, false>(b_dst, &p.b[0], bar, f0, k0, 0);
            fused_load<BN / 2, false, false>(b_dst + Cfg::B_BYTES / 2, &p.b[1], bar, f0, k0, 0);
          }
        } else {
          const int n0 = c.nb * BN + static_cast<int>(cta_rank) * Cfg::BNL;
          fused_load<Cfg::BNL, Cfg::B_MN, CG == 2>(b_dst, &p.b[phase], bar, n0, k0, bz);
        }
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
    }
    // the MMA issuer's last releases must land in this CTA before it may exit
    for (int i = 0; i < STAGES && ok; ++i) {
      ok = mbar_wait(empty_bar(s), ph ^ 1u, wc, kDevTimeoutTail);
      if (++s == STAGES) { s = 0; ph ^= 1u; }
    }
    mbar_wait_drain(mma_done_bar, 0u, p.spin_limit);
  } else if (warp == 1 && lane == 0 && is_leader) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc = make_idesc_f16(Cfg::TILE_M, BN, Cfg::A_MN ? 1u : 0u, Cfg::B_MN ? 1u : 0u,
                                              DT == 1 ? 1u : 0u);
    // one MMA covers 16 k: 32 bytes along a k-contiguous row, or 16 rows of 128 bytes
    constexpr uint64_t a_step = Cfg::A_MN ? 128 : 2, b_step = Cfg::B_MN ? 128 : 2;
    int s = 0, acc = 0;
    uint32_t ph = 0, acc_ph = 0;
    bool ok = true;
    for (int u = worker; ok && u < units; u += workers) {
      const int part = u % p.nsplit;
      const int kb0 = static_cast<int>(static_cast<long long>(total_kb) * part / p.nsplit);
      const int kb1 = static_cast<int>(static_cast<long long>(total_kb) * (part + 1) / p.nsplit);
      if (!mbar_wait(tmem_empty_bar(acc), acc_ph ^ 1u, wc, kDevTimeoutTmemEmpty)) break;
      tcgen05_fence_after_sync();
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(full_bar(s), ph, wc, kDevTimeoutReady)) { ok = false; break; }
        tcgen05_fence_after_sync();
        const uint32_t stage = smem_base + s * Cfg::STAGE_BYTES;
        const uint64_t a = fused_desc<Cfg::A_MN>(stage);
        const uint64_t b = fused_desc<Cfg::B_MN>(stage + Cfg::A_BYTES);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_f16<CG>(d_tmem, a + kk * a_step, b + kk * b_step, idesc, (kb != kb0 || kk != 0) ? 1u : 0u);
        umma_commit<CG>(empty_bar(s));
        if (++s == STAGES) { s = 0; ph ^= 1u; }
      }
      if (ok) umma_commit<CG>(tmem_full_bar(acc));
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
    }
    // whatever was issued has to complete before tensor and shared memory are given up
    umma_commit<CG>(mma_done_bar);
    mbar_wait_drain(mma_done_bar, 0u, p.spin_limit);
  } else if (warp >= Cfg::FIRST_EPI_WARP) {
    // ---------------------------------------------------------------- epilogue
    const int quarter = warp & 3;                     // TMEM lanes 32 * (warp id mod 4)
    const int half = (warp - Cfg::FIRST_EPI_WARP) >> 2;
    const int et = static_cast<int>(threadIdx.x) - Cfg::FIRST_EPI_WARP * 32;
    const uint32_t boxes = staging + static_cast<uint32_t>(warp - Cfg::FIRST_EPI_WARP) * Cfg::SET_BYTES;
    const uint32_t tmem_lane = static_cast<uint32_t>(quarter * 32) << 16;
    int acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true;
    for (int u = worker; ok && u < units; u += workers) {
      const int t = u / p.nsplit, part = u - t * p.nsplit;
      const FusedTile c = fused_tile<Cfg::SYM>(t, p.tiles_m, p.tiles_n, per_z);
      const int row0 = (c.mb * CG + static_cast<int>(cta_rank)) * Cfg::BM + quarter * 32;
      const int row = row0 + lane;
      const bool row_ok = row < p.M;
      // a tile row of CTA rank `cta_rank` that lies wholly below the matrix has nothing to do but
      // to hand its accumulator back
      ok = __all_sync(0xffffffffu, mbar_wait(tmem_full_bar(acc), acc_ph, wc, kDevTimeoutTmemFull));
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN) + tmem_lane;
      bool finish = ok;
      // ---- split reduction: leave this part's sums, count in, go on only as the last one
      const size_t slot4 = static_cast<size_t>(32 * BN);   // float4 per CTA's partial tile
      const float4* parts4 = nullptr;
      if (p.nsplit > 1) {
        if (fused_bar_any(!ok)) { ok = false; break; }
        tcgen05_fence_after_sync();
        float4* tile4 = reinterpret_cast<float4*>(p.ws) + (static_cast<size_t>(t) * CG + cta_rank) * p.nsplit * slot4;
        float4* mine4 = tile4 + part * slot4 + quarter * 32 + lane;
        for (int c32 = half * (BN / 2); c32 < (half + 1) * (BN / 2); c32 += 32) {
          uint32_t r[32];
          tmem_ld_32x32(d_tmem + c32, r);
          tmem_ld_wait();
          if (row_ok) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              __stcg(mine4 + (c32 / 4 + j) * 128,
                     make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                                 __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])));
          }
        }
        __threadfence();
        fused_bar_any(false);
        if (et == 0) {
          uint32_t* counter = p.counters + static_cast<size_t>(t) * CG + cta_rank;
          const uint32_t before = atomicAdd(counter, 1u);
          const bool last = before == static_cast<uint32_t>(p.nsplit) - 1u;
          if (last) *counter = 0;    // ready for the next launch
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(last_slot), "r"(static_cast<uint32_t>(last)) : "memory");
          __threadfence();
        }
        fused_bar_any(false);
        uint32_t last;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(last) : "r"(last_slot) : "memory");
        finish = last != 0;
        __threadfence();
        parts4 = tile4 + quarter * 32 + lane;
      }
      if (!ok) break;
      tcgen05_fence_after_sync();

      // the 32 columns of D from tile column `col` on
      auto slab = [&](int col, float (&v)[32]) {
        if (p.nsplit == 1) {
          uint32_t r[32];
          tmem_ld_32x32(d_tmem + col, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.0f;
          if (row_ok) {
            for (int q = 0; q < p.nsplit; ++q) {
              const float4* src = parts4 + q * slot4 + (col / 4) * 128;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 x = __ldcg(src + j * 128);
                v[4 * j] += x.x; v[4 * j + 1] += x.y; v[4 * j + 2] += x.z; v[4 * j + 3] += x.w;
              }
            }
          }
        }
      };
      // 32 elements of this thread's row of an epilogue input
      auto input = [&](int which, int col, float (&v)[32]) {
        const uint16_t* src = static_cast<const uint16_t*>(p.in[which]) + c.z * p.in_zstride +
                              static_cast<long long>(row) * p.in_ld[which] + col;
        if (row_ok && p.in_vec && col + 32 <= p.in_cols) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(src) + j);
            float2 f;
            f = fused_unpack<DT>(w.x); v[8 * j] = f.x; v[8 * j + 1] = f.y;
            f = fused_unpack<DT>(w.y); v[8 * j + 2] = f.x; v[8 * j + 3] = f.y;
            f = fused_unpack<DT>(w.z); v[8 * j + 4] = f.x; v[8 * j + 5] = f.y;
            f = fused_unpack<DT>(w.w); v[8 * j + 6] = f.x; v[8 * j + 7] = f.y;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            uint32_t w = 0;
            if (row_ok && col + j < p.in_cols) w = __ldg(src + j);
            v[j] = fused_unpack<DT>(w).x;
          }
        }
      };
      // 32 columns as 16-bit values into half `s` of box `b` of the staging area
      auto put = [&](int b, int s, const float (&v)[32], bool as_bf16) {
        const uint32_t box = boxes + b * Cfg::BOX_BYTES;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = (as_bf16 && DT != 1) ? fused_pack<1>(v[8 * j + 2 * i], v[8 * j + 2 * i + 1])
                                        : fused_pack<DT>(v[8 * j + 2 * i], v[8 * j + 2 * i + 1]);
          const int chunk = Cfg::BOX_COLS == 64 ? ((s * 4 + j) ^ (lane & 7)) : (j ^ ((lane >> 1) & 3));
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                           box + lane * (Cfg::BOX_COLS * 2) + chunk * 16),
                       "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
        }
      };
      // the staging boxes may be written again once the TMA unit has read them
      auto boxes_free = [&]() {
        if (lane == 0) bulk_wait_read_all();
        __syncwarp();
      };
      auto boxes_written = [&]() {
        fence_proxy_async_smem();
        __syncwarp();
      };
      // box `b` to columns col0.. of output `o`
      auto emit = [&](int o, int b, int col0) {
        if (col0 >= p.out_cols || row0 >= p.M) return;
        const uint32_t box = boxes + b * Cfg::BOX_BYTES;
        const int oz = OP == kOpDw ? 0 : c.z;
        if (p.out_tma & (1 << o)) {
          if (lane == 0) tma_store_3d(&p.o[o], box, col0, row0, oz);
        } else {
          // rows that start anywhere: a warp writes 32 consecutive elements per instruction
          uint16_t* dst = static_cast<uint16_t*>(p.out[o]) + oz * p.out_zstride + col0;
          for (int r = 0; r < 32 && row0 + r < p.M; ++r) {
#pragma unroll
            for (int h = 0; h < Cfg::BOX_COLS / 32; ++h) {
              const int j = h * 32 + lane;
              const int chunk = Cfg::BOX_COLS == 64 ? ((j >> 3) ^ (r & 7)) : ((j >> 3) ^ ((r >> 1) & 3));
              uint16_t w;
              asm volatile("ld.shared.u16 %0, [%1];"
                           : "=h"(w)
                           : "r"(box + r * (Cfg::BOX_COLS * 2) + chunk * 16 + (j & 7) * 2)
                           : "memory");
              if (col0 + j < p.out_cols) dst[static_cast<long long>(row0 + r) * p.out_ld[o] + j] = w;
            }
          }
        }
      };
      auto emitted = [&]() {
        if (lane == 0) bulk_commit_group();
      };

      if (finish) {
        constexpr int SL = Cfg::BOX_COLS / 32;
        const int tcol0 = half * Cfg::OUT_COLS;                   // first column in the tile
        const int col_base = c.nb * (OP == kOpGate ? BN / 2 : BN) + tcol0;
        if constexpr (OP == kOpGate) {
          auto gate = [&](auto act_tag) {
            constexpr int ACT = decltype(act_tag)::value;
            const int outs = (p.flags & kFusedSave) ? 3 : 1;
            for (int o = 0; o < outs; ++o) {
#pragma unroll 1
              for (int cc = 0; cc < Cfg::OUT_COLS; cc += Cfg::BOX_COLS) {
                boxes_free();
#pragma unroll 1
                for (int s = 0; s < SL; ++s) {
                  const int tc = tcol0 + cc + s * 32;
                  float v[32];
                  if (o == 2) {
                    slab(tc + BN / 2, v);
                  } else {
                    slab(tc, v);
                    if (o == 0) {
                      float w[32];
                      slab(tc + BN / 2, w);
#pragma unroll
                      for (int j = 0; j < 32; ++j) {
                        float y, slope;
                        activation<ACT>(v[j], y, slope);
                        v[j] = y * w[j];
                      }
                    }
                  }
                  put(0, s, v, false);
                }
                boxes_written();
                emit(o, 0, col_base + cc);
                emitted();
              }
            }
          };
          if (p.act == kActSilu) gate(IntTag<kActSilu>{});
          else if (p.act == kActGelu) gate(IntTag<kActGelu>{});
          else gate(IntTag<kActGeluTanh>{});
        } else if constexpr (OP == kOpDact) {
          auto dact = [&](auto act_tag) {
            constexpr int ACT = decltype(act_tag)::value;
#pragma unroll 1
            for (int cc = 0; cc < Cfg::OUT_COLS; cc += 32) {
              const int col = col_base + cc;
              if (col >= p.out_cols) break;     // (uniform over the warp)
              float g[32], w[32], d[32];
              input(0, col, g);
              input(1, col, w);
              slab(tcol0 + cc, d);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                float y, slope;
                activation<ACT>(g[j], y, slope);
                const float dh = d[j], uu = w[j];
                g[j] = dh * uu * slope;    // dg
                d[j] = dh * y;             // du
                w[j] = y * uu;             // h
              }
              boxes_free();
              put(0, 0, g, false);
              put(1, 0, d, false);
              put(2, 0, w, false);
              boxes_written();
              emit(0, 0, col);
              emit(1, 1, col);
              emit(2, 2, col);
              emitted();
            }
          };
          if (p.act == kActSilu) dact(IntTag<kActSilu>{});
          else if (p.act == kActGelu) dact(IntTag<kActGelu>{});
          else dact(IntTag<kActGeluTanh>{});
        } else {
#pragma unroll 1
          for (int cc = 0; cc < Cfg::OUT_COLS; cc += 64) {
            const int col0 = col_base + cc;
            if (col0 >= p.out_cols) break;      // (uniform over the warp)
            boxes_free();
#pragma unroll 1
            for (int s = 0; s < 2; ++s) {
              const int col = col0 + s * 32;
              float v[32];
              slab(tcol0 + cc + s * 32, v);
              if constexpr (OP == kOpDown || OP == kOpDx || OP == kOpDw) {
                put(0, s, v, false);
              } else if constexpr (Cfg::SYM) {
                if constexpr (OP == kOpPoly) {
                  float pin[32];
                  input(0, col, pin);
#pragma unroll
                  for (int j = 0; j < 32; ++j) v[j] = p.coef_b * pin[j] + p.coef_c * v[j];
                  // what rounding q's diagonal to 16 bits loses is as large as the rest of
                  // that rounding together: it goes into the vector that scales x instead
                  const int dj = row - col;
                  if (row_ok && dj >= 0 && dj < 32) {
                    float x = 0.0f;
#pragma unroll
                    for (int j = 0; j < 32; ++j) x = (j == dj) ? v[j] : x;
                    p.vec[c.z * p.vec_ld + row] = p.coef_a + (x - __half2float(__float2half_rn(x))) * p.inv_scale;
                  }
                } else {
#pragma unroll
                  for (int j = 0; j < 32; ++j) v[j] *= p.inv_scale;
                }
                put(0, s, v, false);
                if (c.mb != c.nb) {
                  // the mirror image: 64 rows (this tile's columns) of 32 elements, unswizzled
                  const uint32_t box = boxes + Cfg::BOX_BYTES + s * 32 * 64 + lane * 2;
#pragma unroll
                  for (int j = 0; j < 32; ++j) {
                    const __half h = __float2half_rn(v[j]);
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(box + j * 64), "h"(__half_as_ushort(h)) : "memory");
                  }
                }
              } else {
                float hi[32], lo[32];
                input(0, col, hi);
                input(1, col, lo);
                const float dr = (OP == kOpUpdateWide && row_ok) ? p.vec[c.z * p.vec_ld + row] : 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  float dv = dr;
                  if constexpr (OP == kOpUpdateTall) dv = (col + j < p.out_cols) ? __ldg(p.vec + c.z * p.vec_ld + col + j) : 0.0f;
                  v[j] = dv * (hi[j] + lo[j]) + v[j] * p.inv_scale;
                }
                if (p.flags & kFusedLast) {
#pragma unroll
                  for (int j = 0; j < 32; ++j) v[j] *= p.inv_scale;
                  put(0, s, v, true);
                } else {
#pragma unroll
                  for (int j = 0; j < 32; ++j) lo[j] = v[j] - __half2float(__float2half_rn(v[j]));
                  put(0, s, v, false);
                  put(1, s, lo, false);
                }
              }
            }
            boxes_written();
            if constexpr (OP == kOpDw) {
              emit(c.z, 0, col0);
            } else {
              emit(0, 0, col0);
              if constexpr (Cfg::SYM) {
                // (rows of the mirror image that lie outside the matrix are clipped)
                if (c.mb != c.nb && row0 < p.M && lane == 0) tma_store_3d(&p.o[1], boxes + Cfg::BOX_BYTES, row0, col0, c.z);
              } else if constexpr (Cfg::UPDATE) {
                if (!(p.flags & kFusedLast)) emit(1, 1, col0);
              }
            }
            emitted();
          }
        }
      }
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(tmem_empty_bar(acc), 0);
        else mbar_arrive(tmem_empty_bar(acc));
      }
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
    }
    // stores handed to the TMA unit have to be performed before the CTA may go
    if (lane == 0) bulk_wait_all();
  }

  // ------------------------------------------------------------------ teardown
  __syncwarp();
  // after a failed wait some role left its loop early: let bulk copies on their way land
  if (*reinterpret_cast<volatile uint32_t*>(p.status) != kDevOk) abort_grace_period();
  tcgen05_fence_before_sync();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc<CG>(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace rb200
