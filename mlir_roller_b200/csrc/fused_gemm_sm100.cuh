// Matrix products of 16-bit operands with a fused epilogue, for the gated feed-forward block and
// the Newton-Schulz iteration: D = A B in fp32 (tensor memory), then an element-wise step that
// reads D (and sometimes one more matrix) and writes one to three 16-bit matrices.
//
//   op              D[i,j]                          written
//   kOpGate         g = x Wg^T and u = x Wu^T       act(g) u  (and g, u)
//   kOpDown         h Wd^T                          D
//   kOpDact         dh = dy Wd                      dg = dh u act'(g), du = dh act(g), h = act(g) u
//   kOpDx           [dg du] [Wg; Wu]                D
//   kOpDw           dg^T x, du^T x and dy^T h       D
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
// that holds g[i,j] also holds u[i,j] and neither reaches memory unless it is asked for), and only
// one triangle of a symmetric product is computed.
//
// With few rows or columns there are few tiles, and a weight has to be streamed by all SMs to come
// at the memory's rate. CTAs (or pairs) therefore also run in clusters of up to 8 CTAs that share
// one tile: each takes a part of k, and at the end each collects the others' sums of its share of
// the columns through distributed shared memory (the ring's, which is free by then), adds them in the
// order of k and runs the epilogue on its share. Results do not depend on timing.
//
// Epilogue inputs come and results go through the TMA unit in boxes of 32 rows x 32 (or 64) columns,
// one warp's slab. Loads and stores from registers, a thread per row, were measured beside it (whole
// 32-byte sectors): the pair kernels got a third slower with kOpDact and kOpUpdate*, because
// every access of a warp touches 32 lines.
//
// A launch may be scheduled while the previous one of its stream still runs (programmatic
// dependent launch). It touches memory only behind griddepcontrol.wait, with two exceptions:
//   * p.b_early: weights that the previous kernel does not write may be fetched before the wait;
//   * p.late_wait: a kernel that needs nothing from its predecessor (and writes nothing that one
//     touches) waits for it only before it ends, so that its CTAs fill the SMs that the
//     predecessor's last wave leaves idle. It ends after its predecessor, so what follows
//     in the stream still finds both complete.
// Both read what kernels before the predecessor wrote, and need these complete when they start. That holds
// if the predecessor let its successor start only after its own wait had returned, as a launch without
// late_wait does. It does not hold behind one with late_wait, behind late copies (AlignJobs::late), or
// behind a launch that is not of this call; there the two flags are taken back (LaunchOrder).
//
// Measured on B200 (whole calls by events, operands beyond L2; shares of the cycles in which an SM has
// work from counters on 4096 tokens x 2048 x 4096, one launch at a time):
//   kOpGate, kOpDown   8192 x 4096 x 8192, bf16: 1.19 ms = 1.39 PFLOP/s, what the power limit leaves the
//                      library's GEMM too. Tensor pipe busy 86 and 81 %, of all cycles 79 and 64 %
//                      (128 tiles of kOpDown on 74 pairs run as two waves).
//                      1 x 2048 x 8192: 25 us for 101 MB, of which the kernels' starts and ends and a second
//                      stream that begins when the first one has ended; 1 x 8192 x 32768: 6.4 TB/s.
//   kOpDact, kOpDx, kOpDw   8192 x 4096 x 8192, bf16: 2.58 ms together = 1.28 PFLOP/s. Tensor pipe 52,
//                      90, 92 %: with 2048 to reduce over, a tile of kOpDact is 19 us of epilogue beside 11 us of
//                      MMAs, and neither the memory (2.3 TB/s) nor the tensor pipe is busy then: inputs, arithmetic
//                      and results of 64 columns follow one another. 200 x 1024 x 2816: 30 us, three launches of
//                      which two overlap, the first one on 44 of 148 SMs.
//   kOpGram*, kOpPoly, kOpUpdate*   8192 x 4096, five steps: 2.19 ms = 1.10 PFLOP/s, triangles counted
//                      as such; 512 x 512: 95 us, 5 to 7 us a product, nearly all of it the way from one
//                      launch's results to the next one's loads.
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
  // Columns of the result one epilogue warp owns. They leave in boxes of 32 rows x 32 columns, or
  // 64 where an epilogue reads two matrices and writes two or three: half as many copies, worth
  // 3-6 % of a small orthogonalisation and under 2 % of kOpDact. These
  // boxes serve twice: a matrix read is replaced, in place, by one written.
  static constexpr int OUT_COLS = (OP == kOpGate ? BN / 4 : BN / 2);
  static constexpr int INPUTS = (OP == kOpDact || UPDATE) ? 2 : OP == kOpPoly ? 1 : 0;
  static constexpr bool WIDE = INPUTS == 2;
  static constexpr int BOX_BYTES = WIDE ? 32 * 128 : 32 * 64;
  static constexpr int EPI_WARPS = 8;
  // boxes of one warp: narrow: its inputs, and two results under way
  static constexpr int RING = 2;
  static constexpr int WARP_BOXES = OP == kOpDact ? 3 : UPDATE ? 2 : INPUTS + RING;
  static constexpr int STAGING_BYTES = EPI_WARPS * WARP_BOXES * BOX_BYTES;
  static constexpr int CTRL_BYTES = 384;
  static constexpr int SMEM_LIMIT = 232448;      // 227 KiB opt-in maximum per CTA
  static constexpr int STAGES_FIT = (SMEM_LIMIT - 1024 - CTRL_BYTES - STAGING_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT > 8 ? 8 : STAGES_FIT;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int SMEM_BYTES = RING_BYTES + STAGING_BYTES + CTRL_BYTES + 1024;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int FIRST_EPI_WARP = 4;
  static constexpr int THREADS = (FIRST_EPI_WARP + EPI_WARPS) * 32;
  static_assert(BN == 256 || BN == 128 || (BN == 64 && OP != kOpGate), "tile widths");
  static_assert(!WIDE || OUT_COLS % 64 == 0, "whole boxes");
  // triangle of tiles: tile rows per tile column, or minus tile columns per tile row; 0 = all tiles
  static constexpr int SYM_RATIO = !SYM ? 0 : BN >= TILE_M ? BN / TILE_M : -(TILE_M / BN);
  static_assert(SYM_RATIO >= -2 && SYM_RATIO <= 2, "triangle of tiles");
  // The exchange of partial sums in a splitting cluster goes through the ring's memory: each CTA
  // receives its share of the columns of 128 rows from every other part. (With more parts than
  // slabs of 32 columns, some only give.) Products whose epilogue reads matrices are not split: there is no
  // size at which the estimate would have it.
  static constexpr int SLABS = (OP == kOpGate ? BN / 2 : BN) / 32;
  static constexpr int MAX_SPLIT = INPUTS > 0 ? 1 : CG == 2 ? (OP == kOpGate ? 2 : 4) : OP == kOpGate ? 4 : 8;
  static constexpr int exchange_bytes(int split) {
    return (split - 1) * (SLABS > split ? SLABS / split : 1) * (OP == kOpGate ? 2 : 1) * 16384;
  }
  static_assert(exchange_bytes(MAX_SPLIT) <= STAGES * STAGE_BYTES && exchange_bytes(2) <= STAGES * STAGE_BYTES,
                "exchange area");
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

// act(v) and its slope. tanh appears only as 1 + tanh(z) = 2 sigmoid(2 z) and 1 + erf(z) as erfc(-z): a
// difference of nearly equal numbers never occurs, and the 2^-11 error of the hardware tanh stays out of fp16
// results. A factor act(v) / v under 2^-126 is zero.
template <int ACT>
__device__ __forceinline__ void activation(float v, float& y, float& slope) {
  if constexpr (ACT == kActSilu) {
    const float p = sigmoidf_(v);
    y = v * p;
    slope = p * (1.0f + v * (1.0f - p));
  } else if constexpr (ACT == kActGelu) {
    // Phi(-|v|) = e R with e = exp(-v^2 / 2), which the slope needs as well, and R = erfc(|v| / sqrt 2) / (2 e), a
    // smooth function: a polynomial in t = 1 / (1 + 0.3 |v|), fitted for the least largest relative error
    // over |v| < 14 (beyond, e is zero): 5e-7 in fp32. 1 - q is never under a half. erfcf in its place: 1.5-8 %
    // of the whole call (backward of 4096 x 1024 x 4096: 216 -> 234 us).
    const float t = __fdividef(1.0f, 1.0f + 0.3f * fabsf(v)), e = __expf(-0.5f * v * v);
    float r = 0.035674773f;
    r = fmaf(r, t, -0.157203078f);
    r = fmaf(r, t, 0.206353486f);
    r = fmaf(r, t, -0.0536836311f);
    r = fmaf(r, t, 0.128561616f);
    r = fmaf(r, t, 0.0999134928f);
    r = fmaf(r, t, 0.120753959f);
    r = fmaf(r, t, 0.119629301f);
    const float q = e * (r * t), p = v < 0.0f ? q : 1.0f - q;
    y = v * p;
    slope = p + v * 0.39894228040143268f * e;
  } else {
    constexpr float c = 0.79788456080286536f;
    const float w = fminf(v * v, 1e30f);     // (an infinite one would meet the slope's zero)
    const float p = sigmoidf_(2.0f * c * v * (1.0f + 0.044715f * w));
    y = v * p;
    // (p (1 - p) before v: it is zero where 2 c v may be infinite)
    slope = p + 2.0f * c * (v * (p * (1.0f - p))) * (1.0f + 3.0f * 0.044715f * w);
  }
}

struct FusedTile {
  int z, mb, nb;
};

// Tile order. Rectangular problems: panels of 8 tile rows, so that the tiles in flight share
// operand rows and columns in L2. Symmetric ones: the tiles that touch the lower triangle, row by
// row (RATIO: FusedCfg::SYM_RATIO).
template <int RATIO>
__device__ __forceinline__ FusedTile fused_tile(int t, int tiles_m, int tiles_n, int per_z) {
  FusedTile c;
  c.z = t / per_z;
  int r = t - c.z * per_z;
  if constexpr (RATIO < 0) {
    // row mb has 2 (mb + 1) tiles, mb (mb + 1) come before it
    int q = static_cast<int>((sqrtf(4.0f * static_cast<float>(r) + 1.0f) - 1.0f) * 0.5f);
    while (q * (q + 1) > r) --q;
    while ((q + 1) * (q + 2) <= r) ++q;
    c.mb = q;
    c.nb = r - q * (q + 1);
  } else if constexpr (RATIO > 0) {
    // RATIO rows have q + 1 tiles each, RATIO q (q + 1) / 2 tiles come before them
    int q = static_cast<int>((sqrtf(8.0f / RATIO * static_cast<float>(r) + 1.0f) - 1.0f) * 0.5f);
    while (RATIO * q * (q + 1) / 2 > r) --q;
    while (RATIO * (q + 1) * (q + 2) / 2 <= r) ++q;
    r -= RATIO * q * (q + 1) / 2;
    c.mb = RATIO * q + r / (q + 1);
    c.nb = r % (q + 1);
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

// Where a thread stands: addresses of the CTA's barriers and buffers, its role.
struct FusedCta {
  uint32_t smem_base, staging, ctrl, tmem_base;
  int warp, lane;
  int split;                  // parts of the cluster
  uint32_t cluster_rank, cta_rank, part, leader_rank;
  bool is_leader, epi;
  int quarter, half;          // epilogue: TMEM lanes 32 quarter .., which half of the tile's columns
  WaitCtx wc;
  __device__ uint32_t full_bar(int s) const { return ctrl + 8u * s; }
  __device__ uint32_t empty_bar(int s) const { return ctrl + 128u + 8u * s; }
  __device__ uint32_t tmem_full_bar(int a) const { return ctrl + 256u + 8u * a; }
  __device__ uint32_t tmem_empty_bar(int a) const { return ctrl + 272u + 8u * a; }
  __device__ uint32_t mma_done_bar() const { return ctrl + 288u; }
  __device__ uint32_t tmem_slot() const { return ctrl + 296u; }
  __device__ uint32_t in_bar(int w) const { return ctrl + 304u + 8u * w; }   // a warp's inputs have landed
};

// How far a role has come in the rings it works on (stage, accumulator, inputs, result boxes).
struct FusedRing {
  int s = 0, acc = 0, box_at = 0;
  uint32_t ph = 0, acc_ph = 0, in_ph = 0;
  bool ok = true;
};

// Sets the CTA up: barriers and tensor memory. (Touches no global memory.)
template <class Cfg>
__device__ __forceinline__ FusedCta fused_begin(uint8_t* smem_dyn, int split, uint32_t* status, long long spin_limit) {
  FusedCta x;
  x.smem_base = (smem_addr(smem_dyn) + 1023u) & ~1023u;
  x.staging = x.smem_base + Cfg::RING_BYTES;
  x.ctrl = x.staging + Cfg::STAGING_BYTES;
  x.wc = WaitCtx{status, spin_limit};
  // (the broadcast tells the compiler that the warp index is the same in all lanes)
  x.warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  x.lane = threadIdx.x & 31;
  // a cluster holds the `split` parts of one tile's k, each a CTA or a pair (ranks 2i and 2i + 1)
  x.split = split;
  x.cluster_rank = (Cfg::CG == 2 || split > 1) ? cluster_ctarank() : 0u;
  x.cta_rank = Cfg::CG == 2 ? (x.cluster_rank & 1u) : 0u;
  x.part = x.cluster_rank / Cfg::CG;
  x.leader_rank = x.cluster_rank - x.cta_rank;
  x.is_leader = x.cta_rank == 0;
  x.epi = x.warp >= Cfg::FIRST_EPI_WARP;
  x.quarter = x.warp & 3;
  x.half = (x.warp - Cfg::FIRST_EPI_WARP) >> 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(x.full_bar(s), 1);
      mbar_init(x.empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(x.tmem_full_bar(a), 1);
      mbar_init(x.tmem_empty_bar(a), Cfg::CG * Cfg::EPI_WARPS);
    }
    mbar_init(x.mma_done_bar(), 1);
    for (int w = 0; w < Cfg::EPI_WARPS; ++w) mbar_init(x.in_bar(w), 1);
    fence_barrier_init();
  }
  if (x.warp == 1) tmem_alloc<Cfg::CG>(x.tmem_slot(), Cfg::TMEM_COLS);
  tcgen05_fence_before_sync();
  if constexpr (Cfg::CG == 2) cluster_sync(); else __syncthreads();
  tcgen05_fence_after_sync();
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x.tmem_base) : "r"(x.tmem_slot()));
  return x;
}

// Ends the producer's work: the MMA issuer's last releases must land in this CTA before it may exit.
template <class Cfg>
__device__ __forceinline__ void fused_end_producer(const FusedCta& x, FusedRing& r) {
  for (int i = 0; i < Cfg::STAGES && r.ok; ++i) {
    r.ok = mbar_wait_warp(x.empty_bar(r.s), r.ph ^ 1u, x.wc, kDevTimeoutTail);
    if (++r.s == Cfg::STAGES) { r.s = 0; r.ph ^= 1u; }
  }
  mbar_wait_drain(x.mma_done_bar(), 0u, x.wc.limit);
}
// Ends the MMA issuer's: what was issued has to complete before tensor and shared memory are given up.
template <class Cfg>
__device__ __forceinline__ void fused_end_mma(const FusedCta& x, bool issues) {
  if (issues) {
    umma_commit_to<Cfg::CG>(x.mma_done_bar(), x.leader_rank);
    mbar_wait_drain(x.mma_done_bar(), 0u, x.wc.limit);
  }
}
template <class Cfg>
__device__ __forceinline__ void fused_end(const FusedCta& x) {
  // the TMA unit has to have read what it stores before the CTA may go (its stores are complete when
  // the grid is)
  if (x.epi && x.lane == 0) bulk_wait_read_all();
  __syncwarp();
  // after a failed wait some role left its loop early: let bulk copies on their way land
  if (*reinterpret_cast<volatile uint32_t*>(x.wc.status) != kDevOk) abort_grace_period();
  tcgen05_fence_before_sync();
  if constexpr (Cfg::CG == 2) cluster_sync(); else __syncthreads();
  if (x.warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc<Cfg::CG>(x.tmem_base, Cfg::TMEM_COLS);
  }
}

// One product, as the roles of a CTA see it.
template <class Cfg>
struct FusedWork {
  static constexpr int BN = Cfg::BN, CG = Cfg::CG, STAGES = Cfg::STAGES, DT = Cfg::DT, OP = Cfg::OP;
  const FusedParams& p;
  const FusedCta& me;
  int per_z, tiles, total_kb;
  // Tiles go round-robin to the CTAs, pairs or clusters; a CTA of a splitting cluster takes its part
  // of k, and its cluster has exactly one tile.
  int workers, worker, kb0, kb1;
  uint32_t in_boxes, boxes, tmem_lane;

  __device__ FusedWork(const FusedParams& p_, const FusedCta& me_) : p(p_), me(me_) {
    per_z = p.tiles_per_z;
    tiles = per_z * p.zcount + (OP == kOpDw ? p.tiles_m2 * p.tiles_n2 : 0);
    total_kb = p.num_kb * (OP == kOpDx ? 2 : 1);
    workers = static_cast<int>(gridDim.x) / (CG * me.split);
    worker = static_cast<int>(blockIdx.x) / (CG * me.split);
    kb0 = static_cast<int>(static_cast<long long>(total_kb) * me.part / me.split);
    kb1 = static_cast<int>(static_cast<long long>(total_kb) * (me.part + 1) / me.split);
    in_boxes = me.staging + static_cast<uint32_t>(me.warp - Cfg::FIRST_EPI_WARP) * (Cfg::WARP_BOXES * Cfg::BOX_BYTES);
    boxes = in_boxes + (Cfg::WIDE ? 0 : Cfg::INPUTS) * Cfg::BOX_BYTES;
    tmem_lane = static_cast<uint32_t>(me.quarter * 32) << 16;
  }

  // Where tile t is. (kOpDw: dWd's tiles, z = 2, come behind those of dWg and dWu.)
  __device__ __forceinline__ FusedTile tile(int t) const {
    if constexpr (OP == kOpDw) {
      const int behind = t - per_z * p.zcount;
      if (behind >= 0) {
        FusedTile c = fused_tile<0>(behind, p.tiles_m2, p.tiles_n2, p.tiles_m2 * p.tiles_n2);
        c.z = 2;
        return c;
      }
    }
    return fused_tile<Cfg::SYM_RATIO>(t, p.tiles_m, p.tiles_n, per_z);
  }
  __device__ __forceinline__ int rows(const FusedTile& c) const { return OP == kOpDw && c.z == 2 ? p.M2 : p.M; }
  __device__ __forceinline__ int cols(const FusedTile& c) const { return OP == kOpDw && c.z == 2 ? p.out_cols2 : p.out_cols; }
  // A worker's first tile, and the one after t. In kOpDw the first `head` workers, which find an SM while the
  // previous kernel's last wave is still busy, have the first head_tiles to themselves.
  // (Workers start in the order of their index; if they did not, only the balance would suffer.)
  __device__ __forceinline__ int first() const { return OP == kOpDw && worker >= p.head ? p.head_tiles + worker : worker; }
  __device__ __forceinline__ int next(int t) const {
    if (OP != kOpDw || t >= p.head_tiles) return t + workers;
    return t + p.head < p.head_tiles ? t + p.head : p.head_tiles + worker;
  }

  // ---------------------------------------------------------------- TMA producer (warp 0)
  // The whole warp walks the loop and one elected lane issues: with the loop's values the same in
  // all lanes they stay in uniform registers, where tcgen05.mma and the TMA instructions want
  // them. (Loops of one lane took 0.255 us a k-block whatever the tile's width.)
  // before_loads: what has to be waited for in front of the first load (but p.b_early's).
  template <class F>
  __device__ __forceinline__ void produce(FusedRing& r, bool issues, F before_loads) {
    auto load_a = [&](int s, uint32_t bar, const FusedTile& c, int kb) {
      const int phase = (OP == kOpDx && kb >= p.num_kb) ? 1 : 0;
      const int m0 = (c.mb * CG + static_cast<int>(me.cta_rank)) * Cfg::BM;
      const bool second = OP == kOpDw && c.z == 2;
      fused_load<Cfg::BM, Cfg::A_MN, CG == 2>(me.smem_base + s * Cfg::STAGE_BYTES, second ? &p.a2 : &p.a, bar, m0,
                                              (kb - phase * p.num_kb) * Cfg::BK, OP == kOpDx ? phase : second ? 0 : c.z);
    };
    auto load_b = [&](int s, uint32_t bar, const FusedTile& c, int kb) {
      const uint32_t b_dst = me.smem_base + s * Cfg::STAGE_BYTES + Cfg::A_BYTES;
      const int phase = (OP == kOpDx && kb >= p.num_kb) ? 1 : 0;
      const int k0 = (kb - phase * p.num_kb) * Cfg::BK;
      if constexpr (OP == kOpGate) {
        // tile columns: BN/2 rows of Wg, then the same BN/2 rows of Wu
        const int f0 = c.nb * (BN / 2);
        if constexpr (CG == 2) {
          fused_load<Cfg::BNL, false, true>(b_dst, &p.b[me.cta_rank], bar, f0, k0, 0);
        } else {
          fused_load<BN / 2, false, false>(b_dst, &p.b[0], bar, f0, k0, 0);
          fused_load<BN / 2, false, false>(b_dst + Cfg::B_BYTES / 2, &p.b[1], bar, f0, k0, 0);
        }
      } else {
        const int bz = (OP == kOpDw || OP == kOpDx) ? 0 : c.z;
        const int n0 = c.nb * BN + static_cast<int>(me.cta_rank) * Cfg::BNL;
        fused_load<Cfg::BNL, Cfg::B_MN, CG == 2>(b_dst, &p.b[OP == kOpDw ? c.z >> 1 : phase], bar, n0, k0, bz);
      }
    };
    // The barrier that counts the bytes of both operands (for a pair: of both CTAs, on the leader's,
    // which alone arms it).
    auto counts = [&](int s) { return CG == 2 ? map_to_cta(me.full_bar(s), me.leader_rank) : me.full_bar(s); };
    auto arm = [&](int s) {
      if constexpr (CG == 2) {
        if (me.is_leader) mbar_expect_tx(me.full_bar(s), 2 * (Cfg::A_BYTES + Cfg::B_BYTES));
      } else {
        mbar_expect_tx(me.full_bar(s), p.a_bytes + Cfg::B_BYTES);
      }
    };
    for (int t = first(); r.ok && t < tiles; t = next(t)) {
      const FusedTile c = tile(t);
      int kb = kb0;
      if (t == first()) {
        const int early = p.b_early ? min(STAGES, kb1 - kb0) : 0;    // (of a launch's first tiles)
        if (issues) {
          for (int i = 0; i < early; ++i) {
            arm(i);
            load_b(i, counts(i), c, kb + i);
          }
        }
        before_loads();
        if (issues)
          for (int i = 0; i < early; ++i) load_a(i, counts(i), c, kb + i);
        __syncwarp();
        kb += early;
        r.s += early;
        if (r.s == STAGES) { r.s = 0; r.ph ^= 1u; }
      }
      for (; kb < kb1; ++kb) {
        if (!mbar_wait_warp(me.empty_bar(r.s), r.ph ^ 1u, me.wc, kDevTimeoutEmpty)) { r.ok = false; break; }
        if (issues) {
          const uint32_t bar = counts(r.s);
          arm(r.s);
          load_a(r.s, bar, c, kb);
          load_b(r.s, bar, c, kb);
        }
        __syncwarp();
        if (++r.s == STAGES) { r.s = 0; r.ph ^= 1u; }
      }
    }
  }

  // ---------------------------------------------------------------- MMA issuer (warp 1 of the leader)
  __device__ __forceinline__ void multiply(FusedRing& r, bool issues) {
    constexpr uint32_t idesc = make_idesc_f16(Cfg::TILE_M, BN, Cfg::A_MN ? 1u : 0u, Cfg::B_MN ? 1u : 0u,
                                              DT == 1 ? 1u : 0u);
    // one MMA covers 16 k: 32 bytes along a k-contiguous row, or 16 rows of 128 bytes
    constexpr uint64_t a_step = Cfg::A_MN ? 128 : 2, b_step = Cfg::B_MN ? 128 : 2;
    for (int t = first(); r.ok && t < tiles; t = next(t)) {
      if (!mbar_wait_warp(me.tmem_empty_bar(r.acc), r.acc_ph ^ 1u, me.wc, kDevTimeoutTmemEmpty)) { r.ok = false; break; }
      tcgen05_fence_after_sync();
      const uint32_t d_tmem = me.tmem_base + static_cast<uint32_t>(r.acc * BN);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_warp(me.full_bar(r.s), r.ph, me.wc, kDevTimeoutReady)) { r.ok = false; break; }
        tcgen05_fence_after_sync();
        const uint32_t stage = me.smem_base + r.s * Cfg::STAGE_BYTES;
        const uint64_t a = fused_desc<Cfg::A_MN>(stage);
        const uint64_t b = fused_desc<Cfg::B_MN>(stage + Cfg::A_BYTES);
        if (issues) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f16<CG>(d_tmem, a + kk * a_step, b + kk * b_step, idesc, (kb != kb0 || kk != 0) ? 1u : 0u);
          umma_commit_to<CG>(me.empty_bar(r.s), me.leader_rank);
        }
        __syncwarp();
        if (++r.s == STAGES) { r.s = 0; r.ph ^= 1u; }
      }
      if (r.ok && issues) umma_commit_to<CG>(me.tmem_full_bar(r.acc), me.leader_rank);
      __syncwarp();
      r.acc ^= 1;
      if (r.acc == 0) r.acc_ph ^= 1u;
    }
  }

  // ---------------------------------------------------------------- epilogue (warps 4 .. 11), wide
  // 64 columns at a time, in two halves: a thread takes 32 elements of its row of both inputs out of
  // the boxes and puts 32 elements of the results in their place.
  template <class F>
  __device__ __forceinline__ void finish_wide(FusedRing& r, F before_loads) {
    const uint32_t bar = me.in_bar(me.warp - Cfg::FIRST_EPI_WARP);
    auto at = [&](int b, int half, int j) {      // 16 bytes: chunk j of a half, 128-byte swizzle
      return in_boxes + b * Cfg::BOX_BYTES + me.lane * 128 + (((half * 4 + j) ^ (me.lane & 7)) << 4);
    };
    auto fetch = [&](const FusedTile& c, int row0, int col) {
      if (me.lane == 0) {
        bulk_wait_read_all();        // the boxes' last results are on their way
        mbar_expect_tx(bar, 2 * Cfg::BOX_BYTES);
        tma_load_3d(in_boxes, &p.i[0], bar, col, row0, c.z);
        tma_load_3d(in_boxes + Cfg::BOX_BYTES, &p.i[1], bar, col, row0, c.z);
      }
    };
    auto take = [&](int q, int half, uint32_t (&raw)[16]) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(raw[4 * j]), "=r"(raw[4 * j + 1]), "=r"(raw[4 * j + 2]), "=r"(raw[4 * j + 3])
                     : "r"(at(q, half, j))
                     : "memory");
    };
    auto put = [&](int b, int half, const float (&v)[32], auto dt) {
      constexpr int T = decltype(dt)::value;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at(b, half, j)),
                     "r"(fused_pack<T>(v[8 * j], v[8 * j + 1])), "r"(fused_pack<T>(v[8 * j + 2], v[8 * j + 3])),
                     "r"(fused_pack<T>(v[8 * j + 4], v[8 * j + 5])), "r"(fused_pack<T>(v[8 * j + 6], v[8 * j + 7]))
                     : "memory");
    };
    // the first n boxes to outputs 0 .. n - 1, through the TMA unit
    auto hand_over = [&](int n, const FusedTile& c, int row0, int col) {
      if (me.lane == 0) {
        if (row0 < p.M)
          for (int o = 0; o < n; ++o) tma_store_3d(&p.o[o], in_boxes + o * Cfg::BOX_BYTES, col, row0, c.z);
        bulk_commit_group();
      }
    };
    // box 0 to rows that start or end anywhere: a warp writes 32 consecutive elements per instruction
    auto store_unaligned = [&](const FusedTile& c, int row0, int col) {
      uint16_t* dst = static_cast<uint16_t*>(p.out[0]) + c.z * p.out_zstride + static_cast<long long>(row0) * p.out_ld[0] + col + me.lane;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const int rows = col + h * 32 + me.lane < p.out_cols ? p.M - row0 : 0;
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += 8) {
          uint16_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            asm volatile("ld.shared.u16 %0, [%1];"
                         : "=h"(w[k])
                         : "r"(in_boxes + (r0 + k) * 128 + (((h * 4 + (me.lane >> 3)) ^ k) << 4) + (me.lane & 7) * 2)
                         : "memory");
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (r0 + k < rows) dst[(r0 + k) * p.out_ld[0] + h * 32] = w[k];
        }
      }
      __syncwarp();
    };

    before_loads();
    for (int t = first(); r.ok && t < tiles; t = next(t)) {
      const FusedTile c = tile(t);
      const int row0 = (c.mb * CG + static_cast<int>(me.cta_rank)) * Cfg::BM + me.quarter * 32;
      const int row = row0 + me.lane;
      const int col0 = c.nb * BN + me.half * Cfg::OUT_COLS;
      __syncwarp();
      if (col0 < p.out_cols) fetch(c, row0, col0);       // they do not depend on the product
      // vec of the thread's row (q x), or of every 32nd column of the warp's from `lane` on (x q);
      // asked for here, because in the loop below its way from L2 would be waited for
      [[maybe_unused]] float scale[OP == kOpUpdateTall ? Cfg::OUT_COLS / 32 : 1] = {};
      if constexpr (Cfg::UPDATE) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(scale) / sizeof(float)); ++i) {
          const int at = OP == kOpUpdateTall ? col0 + i * 32 + me.lane : row;
          if (at < (OP == kOpUpdateTall ? p.out_cols : p.M)) scale[i] = __ldcg(p.vec + c.z * p.vec_ld + at);
        }
      }
      r.ok = mbar_wait_warp(me.tmem_full_bar(r.acc), r.acc_ph, me.wc, kDevTimeoutTmemFull);
      if (!r.ok) break;
      tcgen05_fence_after_sync();
      const uint32_t d_tmem = me.tmem_base + static_cast<uint32_t>(r.acc * BN + me.half * Cfg::OUT_COLS) + tmem_lane;
      auto run = [&](auto act_tag) {
        [[maybe_unused]] constexpr int ACT = decltype(act_tag)::value;
#pragma unroll 1
        for (int k = 0; k < Cfg::OUT_COLS; k += 64) {
          const int col = col0 + k;
          if (col >= p.out_cols) break;     // (uniform over the warp)
          if (k > 0) {
            __syncwarp();
            fetch(c, row0, col);
          }
          r.ok = mbar_wait_warp(bar, r.in_ph, me.wc, kDevTimeoutFull) && r.ok;
          r.in_ph ^= 1u;
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            uint32_t d[32], raw0[16], raw1[16];
            float v[32];
            tmem_ld_32x32(d_tmem + k + half * 32, d);
            take(0, half, raw0);
            take(1, half, raw1);
            tmem_ld_wait();
            auto element = [&](const uint32_t (&raw)[16], int j) {
              const float2 f = fused_unpack<DT>(raw[j / 2]);
              return j & 1 ? f.y : f.x;
            };
            if constexpr (OP == kOpDact) {
              float du[32], h[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                float y, slope;
                activation<ACT>(element(raw0, j), y, slope);
                const float dh = __uint_as_float(d[j]), uu = element(raw1, j);
                v[j] = dh * slope * uu;    // dg (dh uu may overflow where the slope is zero)
                du[j] = dh * y;
                h[j] = y * uu;
              }
              put(0, half, v, IntTag<DT>{});
              put(1, half, du, IntTag<DT>{});
              put(2, half, h, IntTag<DT>{});
            } else {
              // x = vec x + D / S; vec belongs to rows (q x) or columns (x q)
              float of_columns = 0.0f;
              if constexpr (OP == kOpUpdateTall) {
#pragma unroll
                for (int i = 0; i < Cfg::OUT_COLS / 32; ++i) of_columns = i == k / 32 + half ? scale[i] : of_columns;
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float f = OP == kOpUpdateTall ? __shfl_sync(0xffffffffu, of_columns, j) : scale[0];
                v[j] = f * (element(raw0, j) + element(raw1, j)) + __uint_as_float(d[j]) * p.inv_scale;
              }
              if (p.flags & kFusedLast) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] *= p.inv_scale;
                put(0, half, v, IntTag<1>{});        // bf16
              } else {
                put(0, half, v, IntTag<DT>{});
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] -= __half2float(__float2half_rn(v[j]));
                put(1, half, v, IntTag<DT>{});
              }
            }
          }
          // what was put into the boxes comes before the TMA unit's next access, be it the store that reads
          // them or, behind ordinary stores, the next inputs that overwrite them
          fence_proxy_async_smem();
          __syncwarp();
          if (OP == kOpDact) hand_over(3, c, row0, col);
          else if (!(p.flags & kFusedLast)) hand_over(2, c, row0, col);
          else if ((p.out_tma & 1) && (col + 64 <= p.out_cols || (p.out_whole & 1))) hand_over(1, c, row0, col);
          else store_unaligned(c, row0, col);
        }
      };
      if (OP != kOpDact || p.act == kActSilu) run(IntTag<kActSilu>{});
      else if (p.act == kActGelu) run(IntTag<kActGelu>{});
      else run(IntTag<kActGeluTanh>{});
      tcgen05_fence_before_sync();
      __syncwarp();
      if (me.lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(me.tmem_empty_bar(r.acc), me.leader_rank);
        else mbar_arrive(me.tmem_empty_bar(r.acc));
      }
      r.acc ^= 1;
      if (r.acc == 0) r.acc_ph ^= 1u;
    }
  }

  // ---------------------------------------------------------------- epilogue (warps 4 .. 11)
  // split: the whole CTA calls this (it meets the cluster's others at barriers).
  template <class F>
  __device__ __forceinline__ void finish(FusedRing& r, F before_loads) {
    auto load_d = [&](uint32_t taddr, float (&v)[32]) {
      uint32_t r[32];
      tmem_ld_32x32(taddr, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
    };
    // The inputs of one slab are sent for, and later taken into registers (16-bit pairs).
    auto fetch = [&](const FusedTile& c, int row0, int col) {
      __syncwarp();      // (every lane has taken the previous slab's)
      if (me.lane == 0) {
        const uint32_t bar = me.in_bar(me.warp - Cfg::FIRST_EPI_WARP);
        mbar_expect_tx(bar, Cfg::INPUTS * Cfg::BOX_BYTES);
#pragma unroll
        for (int q = 0; q < Cfg::INPUTS; ++q) tma_load_3d(in_boxes + q * Cfg::BOX_BYTES, &p.i[q], bar, col, row0, c.z);
      }
    };
    auto take = [&](uint32_t (&raw)[Cfg::INPUTS ? Cfg::INPUTS : 1][16]) {
      const bool ok = __all_sync(0xffffffffu, mbar_wait(me.in_bar(me.warp - Cfg::FIRST_EPI_WARP), r.in_ph, me.wc, kDevTimeoutFull));
      r.in_ph ^= 1u;
#pragma unroll
      for (int q = 0; q < Cfg::INPUTS; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(raw[q][4 * j]), "=r"(raw[q][4 * j + 1]), "=r"(raw[q][4 * j + 2]), "=r"(raw[q][4 * j + 3])
                       : "r"(in_boxes + q * Cfg::BOX_BYTES + me.lane * 64 + (j ^ ((me.lane >> 1) & 3)) * 16)
                       : "memory");
      return ok;
    };
    // A staging box that the TMA unit has read (the one handed out RING boxes ago).
    auto free_box = [&]() {
      if (me.lane == 0) bulk_wait_read<Cfg::RING - 1>();
      __syncwarp();
      const uint32_t b = boxes + static_cast<uint32_t>(r.box_at) * Cfg::BOX_BYTES;
      r.box_at = r.box_at + 1 == Cfg::RING ? 0 : r.box_at + 1;
      return b;
    };
    // 32 columns of this warp's 32 rows, as 16-bit values, into a box ...
    auto put = [&](uint32_t box, const float (&v)[32]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = fused_pack<DT>(v[8 * j + 2 * i], v[8 * j + 2 * i + 1]);
        // 64-byte swizzle: 16-byte chunks of a 64-byte row, exchanged by bits 1..2 of the row
        const int chunk = j ^ ((me.lane >> 1) & 3);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + me.lane * 64 + chunk * 16),
                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
      }
    };
    // ... and from there to columns col.. of output `o`.
    auto emit = [&](int o, const FusedTile& c, int row0, int col, const float (&v)[32]) {
      const uint32_t box = free_box();
      put(box, v);
      const int oz = OP == kOpDw ? 0 : c.z;
      if (((col + 32 <= cols(c) ? p.out_tma : p.out_whole) >> o) & 1) {
        fence_proxy_async_smem();
        __syncwarp();
        if (me.lane == 0) {
          if (row0 < rows(c)) tma_store_3d(&p.o[o], box, col, row0, oz);
          bulk_commit_group();
        }
      } else {
        // rows that start or end anywhere: a warp writes 32 consecutive elements per instruction
        __syncwarp();
        uint16_t* dst = static_cast<uint16_t*>(p.out[o]) + oz * p.out_zstride + static_cast<long long>(row0) * p.out_ld[o] + col + me.lane;
        const int left = col + me.lane < cols(c) ? rows(c) - row0 : 0;
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += 8) {
          uint16_t x[8];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            asm volatile("ld.shared.u16 %0, [%1];"
                         : "=h"(x[r])
                         : "r"(box + (r0 + r) * 64 + (((me.lane >> 3) ^ (((r0 + r) >> 1) & 3)) * 16) + (me.lane & 7) * 2)
                         : "memory");
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r0 + r < left) dst[(r0 + r) * p.out_ld[o]] = x[r];
        }
        if (me.lane == 0) bulk_commit_group();   // (an empty group keeps the ring's count)
      }
    };
    // The mirror image of 32 x 32 elements of a symmetric fp16 matrix (its own box has no swizzle).
    // Neighbouring lanes exchange halves, so that each word holds two neighbouring columns.
    auto emit_mirror = [&](const FusedTile& c, int row0, int col, const float (&v)[32]) {
      const uint32_t box = free_box();
      const bool odd = me.lane & 1;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t ab = fused_pack<DT>(v[2 * j], v[2 * j + 1]);
        const uint32_t got = __shfl_xor_sync(0xffffffffu, ab, 1);
        const uint32_t word = odd ? __byte_perm(got, ab, 0x7632) : __byte_perm(ab, got, 0x5410);
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(box + (2 * j + odd) * 64 + (me.lane >> 1) * 4), "r"(word) : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (me.lane == 0) {
        if (row0 < p.M) tma_store_3d(&p.o[1], box, row0, col, c.z);
        bulk_commit_group();
      }
    };

    // Whether a slab has anything to do (it decides whether inputs are sent for).
    auto wanted = [&](const FusedTile& c, int row0, int col) { return col < cols(c) && (!Cfg::SYM || col <= row0); };

    // The epilogue of this warp's slabs slab0, slab0 + step, .. < slab_end of tile `c`. Slab i is the 32
    // result columns from tile column 32 i on; `sums(tile_col, v)` gives 32 columns of D.
    // The first slab's inputs have been sent for.
    auto epilogue = [&](const FusedTile& c, int slab0, int step, int slab_end, auto sums) {
      const int row0 = (c.mb * CG + static_cast<int>(me.cta_rank)) * Cfg::BM + me.quarter * 32;
      [[maybe_unused]] const int row = row0 + me.lane;
      const int col_base = c.nb * (OP == kOpGate ? BN / 2 : BN);
      auto run = [&](auto act_tag) {
        [[maybe_unused]] constexpr int ACT = decltype(act_tag)::value;
#pragma unroll 1
        for (int i = slab0; i < slab_end; i += step) {
          const int tc = i * 32, col = col_base + tc;
          // (uniform over the warp; above the diagonal a slab is the mirror image of another one)
          if (!wanted(c, row0, col)) break;
          float v[32];
          uint32_t raw[Cfg::INPUTS ? Cfg::INPUTS : 1][16] = {};
          if constexpr (Cfg::INPUTS > 0) {
            r.ok = take(raw) && r.ok;
            // the next slab's inputs are on their way while this one is worked on
            if (i + step < slab_end && wanted(c, row0, col + step * 32)) fetch(c, row0, col + step * 32);
          }
          auto input = [&](int q, int k) {      // element k of input q
            const float2 f = fused_unpack<DT>(raw[q][k / 2]);
            return k & 1 ? f.y : f.x;
          };
          if constexpr (OP == kOpGate) {
            float w[32];
            sums(tc, v);
            sums(tc + BN / 2, w);
            if (p.flags & kFusedSave) {
              emit(1, c, row0, col, v);
              emit(2, c, row0, col, w);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              float y, slope;
              activation<ACT>(v[j], y, slope);
              v[j] = y * w[j];
            }
            emit(0, c, row0, col, v);
          } else if constexpr (OP == kOpDown || OP == kOpDx || OP == kOpDw) {
            sums(tc, v);
            emit(OP == kOpDw ? c.z : 0, c, row0, col, v);
          } else if constexpr (Cfg::SYM) {
            if constexpr (OP == kOpPoly) {
              sums(tc, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = p.coef_b * input(0, j) + p.coef_c * v[j];
              // what rounding q's diagonal to 16 bits loses is as large as the rest of that
              // rounding together: it goes into the vector that scales x instead
              const int dj = row - col;
              if (row < p.M && dj >= 0 && dj < 32) {
                float x = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j) x = (j == dj) ? v[j] : x;
                p.vec[c.z * p.vec_ld + row] = p.coef_a + (x - __half2float(__float2half_rn(x))) * p.inv_scale;
              }
            } else {
              sums(tc, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] *= p.inv_scale;
            }
            emit(0, c, row0, col, v);
            if (col < row0) emit_mirror(c, row0, col, v);
          }
        }
      };
      if constexpr (OP == kOpGate) {
        if (p.act == kActSilu) run(IntTag<kActSilu>{});
        else if (p.act == kActGelu) run(IntTag<kActGelu>{});
        else run(IntTag<kActGeluTanh>{});
      } else {
        run(IntTag<0>{});
      }
    };

    constexpr int kSlabs = Cfg::OUT_COLS / 32;     // slabs of one warp of a whole tile

    if (Cfg::MAX_SPLIT == 1 || me.split == 1) {
      before_loads();
      for (int t = first(); r.ok && t < tiles; t = next(t)) {
        const FusedTile c = tile(t);
        if constexpr (Cfg::INPUTS > 0) {     // they do not depend on the product
          const int col = c.nb * BN + me.half * Cfg::OUT_COLS;
          const int row0 = (c.mb * CG + static_cast<int>(me.cta_rank)) * Cfg::BM + me.quarter * 32;
          if (wanted(c, row0, col)) fetch(c, row0, col);
        }
        r.ok = __all_sync(0xffffffffu, mbar_wait(me.tmem_full_bar(r.acc), r.acc_ph, me.wc, kDevTimeoutTmemFull));
        if (!r.ok) break;
        tcgen05_fence_after_sync();
        const uint32_t d_tmem = me.tmem_base + static_cast<uint32_t>(r.acc * BN) + tmem_lane;
        epilogue(c, me.half * kSlabs, 1, (me.half + 1) * kSlabs,
                 [&](int tc, float (&v)[32]) { load_d(d_tmem + tc, v); });
        tcgen05_fence_before_sync();
        __syncwarp();
        if (me.lane == 0) {
          if constexpr (CG == 2) mbar_arrive_cluster(me.tmem_empty_bar(r.acc), me.leader_rank);
          else mbar_arrive(me.tmem_empty_bar(r.acc));
        }
        r.acc ^= 1;
        if (r.acc == 0) r.acc_ph ^= 1u;
      }
    } else {
      // ---- the cluster holds the tile's parts: their sums are put together, each CTA taking a share
      // of the slabs: slab i is received by part i / share, or by every `apart`-th part
      const FusedTile c = tile(worker);
      const int row0 = (c.mb * CG + static_cast<int>(me.cta_rank)) * Cfg::BM + me.quarter * 32;
      const bool row_ok = row0 + me.lane < rows(c);
      const int share = max(Cfg::SLABS / me.split, 1), apart = max(me.split / Cfg::SLABS, 1);
      const int my_slab = static_cast<int>(me.part) / apart * share;
      const bool receives = static_cast<int>(me.part) % apart == 0 && me.half < share;
      if (me.epi) {
        before_loads();
        r.ok = __all_sync(0xffffffffu, mbar_wait(me.tmem_full_bar(0), 0u, me.wc, kDevTimeoutTmemFull));
      }
      __syncwarp();
      cluster_sync();      // all MMAs of the cluster are done: the rings' memory is free
      // Exchange area of a CTA: [sender][32-column group][4 columns][row] float4. The gate has two
      // groups per slab (g, then u).
      constexpr int kGroups = OP == kOpGate ? 2 : 1;
      const uint32_t sender_bytes = static_cast<uint32_t>(share * kGroups) * 16384u;
      const uint32_t lane_at = static_cast<uint32_t>(me.quarter * 32 + me.lane) * 16u;
      if (me.epi && r.ok) {
        tcgen05_fence_after_sync();
        for (int i = me.half; i < Cfg::SLABS; i += 2) {
          const uint32_t to = static_cast<uint32_t>(i / share * apart);
          if (to == me.part) continue;
          // senders in the order of k, the receiver itself left out
          const uint32_t place = me.part - (me.part > to ? 1u : 0u);
#pragma unroll
          for (int q = 0; q < kGroups; ++q) {
            float v[32];
            load_d(me.tmem_base + tmem_lane + i * 32 + q * (BN / 2), v);
            if (row_ok) {
              const uint32_t dst = map_to_cta(
                  me.smem_base + place * sender_bytes + static_cast<uint32_t>((i % share) * kGroups + q) * 16384u + lane_at,
                  to * CG + me.cta_rank);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + j * 2048u),
                             "f"(v[4 * j]), "f"(v[4 * j + 1]), "f"(v[4 * j + 2]), "f"(v[4 * j + 3])
                             : "memory");
            }
          }
        }
      }
      __syncwarp();
      cluster_sync();
      if (me.epi && r.ok && receives) {
        epilogue(c, my_slab + me.half, 2, my_slab + share, [&](int tc, float (&v)[32]) {
          const int q = (OP == kOpGate && tc >= BN / 2) ? 1 : 0;
          const int i = (tc - q * (BN / 2)) / 32 - my_slab;
          float own[32];
          load_d(me.tmem_base + tmem_lane + tc, own);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.0f;
          for (int r = 0; r < me.split; ++r) {
            if (r == static_cast<int>(me.part)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] += own[j];
            } else if (row_ok) {
              const uint32_t src = me.smem_base + static_cast<uint32_t>(r - (r > static_cast<int>(me.part) ? 1 : 0)) * sender_bytes +
                                   static_cast<uint32_t>(i * kGroups + q) * 16384u + lane_at;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float4 x;
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
                             : "r"(src + j * 2048u)
                             : "memory");
                v[4 * j] += x.x; v[4 * j + 1] += x.y; v[4 * j + 2] += x.z; v[4 * j + 3] += x.w;
              }
            }
          }
        });
      }
    }
  }
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
fused_gemm_kernel(const __grid_constant__ FusedParams p) {
  extern __shared__ uint8_t smem_dyn[];
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.a);
    tma_prefetch_desc(&p.b[0]);
    if (Cfg::OP == kOpGate || Cfg::OP == kOpDx || Cfg::OP == kOpDw) tma_prefetch_desc(&p.b[1]);
    tma_prefetch_desc(&p.o[0]);
  }
  const FusedCta x = fused_begin<Cfg>(smem_dyn, p.split, p.status, p.spin_limit);
  FusedWork<Cfg> work(p, x);
  FusedRing r;
  auto previous = [&]() {
    if (!p.late_wait) grid_dependency_wait();
  };
  if (x.warp == 0) {
    work.produce(r, elect_one(), [&]() {
      previous();
      grid_launch_dependents();
    });
    fused_end_producer<Cfg>(x, r);
  } else if (x.warp == 1 && x.is_leader) {
    const bool issues = elect_one();
    previous();
    work.multiply(r, issues);
    fused_end_mma<Cfg>(x, issues);
  }
  if constexpr (Cfg::WIDE) {
    if (x.epi) work.finish_wide(r, previous);
  } else {
    if (x.epi || x.split > 1) work.finish(r, previous);
  }
  if (p.late_wait) grid_dependency_wait();
  fused_end<Cfg>(x);
}

}  // namespace rb200
