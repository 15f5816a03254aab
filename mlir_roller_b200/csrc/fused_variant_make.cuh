// Turns one instantiation of the fused product kernel into an entry of the host-side table.
#pragma once

#include "fused_gemm_sm100.cuh"

namespace rb200 {

template <class Cfg>
static cudaError_t fused_launch(const FusedParams& p, int grid, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(Cfg::CG * p.split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  // scheduled while the previous kernel of the stream winds down; the kernel waits for that
  // kernel's completion before it touches global memory
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, fused_gemm_kernel<Cfg>, p);
}

template <int OP, int CG, int BN, int DT>
static FusedVariant fused_make() {
  using Cfg = FusedCfg<OP, CG, BN, DT>;
  FusedVariant v;
  v.op = OP;
  v.cta_group = CG;
  v.block_n = BN;
  v.dt = DT;
  v.threads = Cfg::THREADS;
  v.max_split = Cfg::MAX_SPLIT;
  v.smem_bytes = Cfg::SMEM_BYTES;
  v.func = reinterpret_cast<const void*>(&fused_gemm_kernel<Cfg>);
  v.launch = &fused_launch<Cfg>;
  return v;
}

// The feed-forward products of one operand type: the pair tiles 256 x 256 and 256 x 128 and, for few rows or
// columns, single CTAs of 128 x 256, 128 x 128 and 128 x 64.
template <int DT>
static const FusedVariant* fused_ffn_table(int* n) {
  static const FusedVariant t[] = {
      fused_make<kOpGate, 2, 256, DT>(), fused_make<kOpGate, 2, 128, DT>(), fused_make<kOpGate, 1, 256, DT>(), fused_make<kOpGate, 1, 128, DT>(),
      fused_make<kOpDown, 2, 256, DT>(), fused_make<kOpDown, 2, 128, DT>(), fused_make<kOpDown, 1, 256, DT>(), fused_make<kOpDown, 1, 128, DT>(),
      fused_make<kOpDown, 1, 64, DT>(),  fused_make<kOpDx, 1, 64, DT>(),
      fused_make<kOpDact, 2, 256, DT>(), fused_make<kOpDact, 2, 128, DT>(), fused_make<kOpDact, 1, 128, DT>(),
      fused_make<kOpDx, 2, 256, DT>(), fused_make<kOpDx, 2, 128, DT>(),   fused_make<kOpDx, 1, 256, DT>(), fused_make<kOpDx, 1, 128, DT>(),
      fused_make<kOpDw, 2, 256, DT>(), fused_make<kOpDw, 2, 128, DT>(),   fused_make<kOpDw, 1, 128, DT>(),
  };
  *n = static_cast<int>(sizeof(t) / sizeof(t[0]));
  return t;
}

}  // namespace rb200
