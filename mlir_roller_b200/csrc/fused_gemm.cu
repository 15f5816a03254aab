// Which fused product kernel a problem runs on, and how its reduction is cut.
#include "fused_product.h"

namespace rb200 {

namespace {

const FusedVariant* table(int i, int* n) {
  switch (i) {
    case 0: return fused_variants_bf16(n);
    case 1: return fused_variants_f16(n);
    default: return fused_variants_ortho(n);
  }
}

struct TileCost {
  int cta_group, block_n;
  double kb_us;    // one k-block of one tile while every SM works
  double tile_us;  // what a tile costs besides (first accumulator's epilogue, fill)
};
constexpr TileCost kTiles[] = {{2, 256, 0.40, 3.0}, {1, 256, 0.40, 3.0}, {1, 128, 0.24, 2.0}};

}  // namespace

const FusedVariant* fused_find(int op, int cta_group, int block_n, int dt) {
  for (int i = 0; i < 3; ++i) {
    int n = 0;
    const FusedVariant* t = table(i, &n);
    for (int j = 0; j < n; ++j)
      if (t[j].op == op && t[j].cta_group == cta_group && t[j].block_n == block_n && t[j].dt == dt)
        return &t[j];
  }
  return nullptr;
}

// Raises the kernels' shared-memory limits on the current device and asks how many CTA pairs it
// can hold at once.
static cudaError_t bind_device(int* max_pairs) {
  *max_pairs = 0;
  for (int i = 0; i < 3; ++i) {
    int n = 0;
    const FusedVariant* t = table(i, &n);
    for (int j = 0; j < n; ++j) {
      cudaError_t e = cudaFuncSetAttribute(t[j].func, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           t[j].smem_bytes);
      if (e != cudaSuccess) return e;
      if (t[j].cta_group != 2 || *max_pairs > 0) continue;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(148, 1, 1);
      cfg.blockDim = dim3(static_cast<unsigned>(t[j].threads), 1, 1);
      cfg.dynamicSmemBytes = static_cast<size_t>(t[j].smem_bytes);
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(max_pairs, t[j].func, &cfg);
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

// The kernels have the same inner loop, so a launch takes about (k-blocks and tiles the busiest
// worker gets) x (their costs); the smallest estimate wins. Parts of a reduction cost a trip of
// the fp32 sums through L2 each.
FusedChoice fused_choose(const FusedShape& s, int sm_count, int max_pairs) {
  FusedChoice best = {};
  double best_us = 0.0;
  const bool sym = s.op == kOpGramWide || s.op == kOpGramTall || s.op == kOpPoly;
  for (const TileCost& c : kTiles) {
    const FusedVariant* kv = fused_find(s.op, c.cta_group, c.block_n, s.dt);
    if (!kv) continue;
    FusedChoice f = {};
    f.kv = kv;
    const int bm = 128 * c.cta_group, bn = s.op == kOpGate ? c.block_n / 2 : c.block_n;
    f.tiles_m = static_cast<int>((s.M + bm - 1) / bm);
    f.tiles_n = static_cast<int>((s.N + bn - 1) / bn);
    f.tiles_per_z = sym ? f.tiles_m * (f.tiles_m + 1) / 2 : f.tiles_m * f.tiles_n;
    f.num_kb = static_cast<int>((s.K + 63) / 64);
    const int kbs = f.num_kb * (s.op == kOpDx ? 2 : 1);
    const long long tiles = static_cast<long long>(f.tiles_per_z) * s.zcount;
    const int workers = c.cta_group == 2 ? max_pairs : sm_count;
    if (workers < 1) continue;
    for (int split = 1; split <= 32 && split <= kbs; ++split) {
      const long long units = tiles * split;
      if (split > 1 && (units * c.cta_group > kFusedMaxUnits || kbs / split < 4)) break;
      const long long waves = (units + workers - 1) / workers;
      const int part = (kbs + split - 1) / split;
      double us = static_cast<double>(waves) * (part * c.kb_us) + c.tile_us;
      if (split > 1) us += 2.0 + 0.6 * split;
      if (best.kv && us >= best_us) continue;
      best_us = us;
      best = f;
      best.nsplit = split;
      best.grid = static_cast<int>(units < workers ? units : workers) * c.cta_group;
    }
  }
  return best;
}

int fused_context_create(FusedContext* c) {
  memset(c, 0, sizeof(*c));
  FUSED_CUDA(cudaGetDevice(&c->device));
  cudaDeviceProp prop;
  FUSED_CUDA(cudaGetDeviceProperties(&prop, c->device));
  if (prop.major != 10) return ROLLER_ERR_DEVICE;
  c->sm_count = prop.multiProcessorCount;
  cudaError_t e = bind_device(&c->max_pairs);
  if (c->max_pairs > c->sm_count / 2) c->max_pairs = c->sm_count / 2;
  if (e == cudaSuccess) e = cudaMalloc(&c->ws, kFusedWsBytes);
  if (e == cudaSuccess) e = cudaMalloc(&c->counters, kFusedMaxUnits * sizeof(uint32_t));
  if (e == cudaSuccess) e = cudaMemset(c->counters, 0, kFusedMaxUnits * sizeof(uint32_t));
  if (e == cudaSuccess) e = cudaMalloc(&c->status, sizeof(uint32_t));
  if (e == cudaSuccess) e = cudaMemset(c->status, 0, sizeof(uint32_t));
  if (e == cudaSuccess) return ROLLER_OK;
  const int rc = e == cudaErrorMemoryAllocation ? ROLLER_ERR_NOMEM : report_cuda_error(e, "plan setup");
  cudaGetLastError();
  fused_context_destroy(c);
  return rc;
}

void fused_context_destroy(FusedContext* c) {
  cudaFree(c->ws);
  cudaFree(c->counters);
  cudaFree(c->status);
  c->ws = nullptr;
  c->counters = c->status = nullptr;
}

int fused_context_status(FusedContext* c, uint32_t* device_status) {
  uint32_t h = 0;
  FUSED_CUDA(cudaDeviceSynchronize());
  FUSED_CUDA(cudaMemcpy(&h, c->status, sizeof(h), cudaMemcpyDeviceToHost));
  if (device_status) *device_status = h;
  if (h == 0) return ROLLER_OK;
  // a launch that gave up may have left a split reduction half counted
  FUSED_CUDA(cudaMemset(c->status, 0, sizeof(uint32_t)));
  FUSED_CUDA(cudaMemset(c->counters, 0, kFusedMaxUnits * sizeof(uint32_t)));
  return ROLLER_ERR_TIMEOUT;
}

}  // namespace rb200
