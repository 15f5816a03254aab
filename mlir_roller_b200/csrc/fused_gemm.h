// Host-side interface of the fused 16-bit products (fused_gemm_sm100.cuh): launch parameters, the
// table of compiled kernels, and the choice of tile and reduction split.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace rb200 {

enum FusedOp : int {
  kOpGate = 0, kOpDown, kOpDact, kOpDx, kOpDw,
  kOpGramWide, kOpGramTall, kOpPoly, kOpUpdateWide, kOpUpdateTall,
  kFusedOps
};
enum Activation : int { kActSilu = 0, kActGelu = 1, kActGeluTanh = 2 };
template <int V>
struct IntTag {
  static constexpr int value = V;
};

constexpr int kFusedSave = 1;   // kOpGate: g and u are written too
constexpr int kFusedLast = 2;   // kOpUpdate*: the result leaves as bf16, divided by the scale

// Everything one launch needs. Matrices are [z][rows][columns]; leading dimensions in elements.
struct FusedParams {
  CUtensorMap a;        // first operand
  CUtensorMap a2;       // kOpDw: first operand of dWd
  CUtensorMap b[2];     // second operand (kOpGate: Wg, Wu; kOpDx: of each half; kOpDw: x, h)
  CUtensorMap o[3];     // outputs as store destinations, where out_tma says so
  void* out[3];
  long long out_ld[3];
  long long out_zstride;
  int out_cols;         // columns of the outputs (those beyond are not written)
  int out_tma;          // bit o: output o leaves through o[o] (16-byte aligned base and rows)
  int out_whole;        // bit o: and so do boxes that reach beyond the last column. A TMA store drops what lies
                        // there in units of 16 bytes only: up to 7 columns behind the last one are written, which
                        // must be none (a width of whole units) or the library's own padding.
  CUtensorMap i[2];     // element-wise inputs of the epilogue
  float* vec;           // kOpPoly writes, kOpUpdate* reads: one value per row of q, [z][vec_ld]
  int vec_ld;
  int M;                // rows of D
  int num_kb;           // k-blocks of 64 (of each half in kOpDx)
  int a_bytes;          // bytes one TMA load of A brings (fewer rows than 128 on single CTAs)
  int tiles_m, tiles_n, tiles_per_z, zcount;
  int M2, out_cols2, tiles_m2, tiles_n2;   // kOpDw: of dWd, whose tiles come behind the zcount others
  int head, head_tiles;                    // kOpDw: FusedWork::next
  int split;            // parts of a cluster that share a tile's k (1 = none)
  int b_early;          // the second operand may be read before the previous kernel is done ...
  int late_wait;        // ... or everything: that kernel is only waited for at the end
  int act;
  int flags;
  float coef_a, coef_b, coef_c, inv_scale;
  uint32_t* status;
  long long spin_limit;
};

// What a launch may take for granted about the launches before it in its call. `waited`: the last one let
// its successor start only after its own wait, so that everything before it is complete by then. Only then may
// the next one read operands early (b_early) or wait late (late_wait, AlignJobs::late); it says so here, and
// one that waits late itself, or a launch of somebody else (the start of a call), gives nothing for granted.
struct LaunchOrder {
  bool waited = false;
  // The liberties that the next launch wants, as far as it may take them.
  void next(int* b_early, int* late_wait) {
    if (!waited) {
      if (b_early) *b_early = 0;
      *late_wait = 0;
    }
    waited = *late_wait == 0;
  }
};

struct FusedVariant {
  int op, cta_group, block_n, dt;   // dt: 1 = bf16, 2 = fp16
  int threads, smem_bytes, max_split;
  const void* func;
  cudaError_t (*launch)(const FusedParams& p, int grid, cudaStream_t stream);
};

// The compiled kernels of one operand type (1 = bf16, 2 = fp16); fp16 also has the Newton-Schulz
// products. nullptr where none was compiled.
const FusedVariant* fused_variants_bf16(int* n);
const FusedVariant* fused_variants_f16(int* n);
const FusedVariant* fused_variants_ortho(int* n);
const FusedVariant* fused_find(int op, int cta_group, int block_n, int dt);

// A problem as the choice of a kernel sees it.
struct FusedShape {
  int op, dt;
  long long M, N;       // of D (kOpGate: of one weight's product; kOpDw: of dWg, and dWd is N x M)
  long long K;          // of one half in kOpDx
  int zcount;
};
struct FusedChoice {
  const FusedVariant* kv;
  int tiles_m, tiles_n, tiles_per_z, num_kb, split, grid;
  int tiles_m2, tiles_n2;   // kOpDw: of dWd
  int tiles, at_once;       // in all; clusters that run at once
  double tile_us;           // estimated time of a tile
};
// What the current device holds at once: CTAs of one per SM, and clusters of 2, 4 and 8.
struct FusedDevice {
  int sm_count;
  int clusters[4];     // [i]: clusters of 2^i CTAs
};
FusedChoice fused_choose(const FusedShape& s, const FusedDevice& d);
// How kOpDw's tiles are dealt when it starts beside the last wave of `before` (FusedWork::next).
void fused_deal(const FusedChoice& before, const FusedChoice& dw, const FusedDevice& d, int* head, int* head_tiles);
}  // namespace rb200
