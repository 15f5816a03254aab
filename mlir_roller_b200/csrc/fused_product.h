// Builds the launch of one fused product: choice of kernel, tensor maps, parameters.
#pragma once

#include <cstring>

#include "../../include/roller_b200.h"
#include "fused_gemm.h"
#include "gemm_launch.h"
#include "host_util.h"

namespace rb200 {

#define FUSED_CUDA(call)                                               \
  do {                                                                 \
    cudaError_t e_ = (call);                                           \
    if (e_ != cudaSuccess) return rb200::report_cuda_error(e_, #call); \
  } while (0)
#define FUSED_OK(call)                \
  do {                                \
    int rc_ = (call);                 \
    if (rc_ != ROLLER_OK) return rc_; \
  } while (0)

inline long long up64(long long x) { return (x + 63) / 64 * 64; }

inline bool aligned16(const void* p, long long ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0;
}

// What the products of one plan share.
struct FusedContext {
  int device;
  FusedDevice dev;
  uint32_t* status;     // device status word
};
int fused_context_create(FusedContext* c);    // on the current device; a roller_status
void fused_context_destroy(FusedContext* c);
int fused_context_status(FusedContext* c, uint32_t* device_status);   // reads and clears; on its device

// One allocation for all workspaces of a plan: sizes are asked for first, pointers given afterwards
// (each on a 1024-byte boundary).
struct Arena {
  char* base = nullptr;
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += (n + 1023) / 1024 * 1024;
    return at;
  }
  cudaError_t allocate() { return cudaMalloc(&base, bytes); }
  template <class T>
  T* at(size_t offset) const { return reinterpret_cast<T*>(base + offset); }
};

// Operands whose rows do not start on 16 bytes are copied, all of a call's in one launch.
struct AlignJob {
  const uint16_t* src;
  uint16_t* dst;
  long long ld_src, ld_dst;
  int rows, cols;
  int blocks;       // set by align_rows
};
struct AlignJobs {
  AlignJob job[8];
  int n = 0;
  int late = 0;     // the previous kernel of the call has nothing to do with them (taken back if LaunchOrder says so)
};
cudaError_t align_rows(AlignJobs& jobs, LaunchOrder& order, int sm_count, cudaStream_t stream);

// D is M x N, reduced over K, for z matrices; operand matrices are [z][rows][cols] in memory.
struct Product {
  FusedParams p;
  FusedChoice c;
  int op;
  bool bf16;

  // `known`: the choice for an earlier product of these sizes.
  Product(const FusedContext& x, int op_, int dt, long long M, long long N, long long K, int z,
          const FusedChoice* known = nullptr)
      : op(op_), bf16(dt == 1) {
    memset(&p, 0, sizeof(p));
    c = known ? *known : fused_choose(FusedShape{op, dt, M, N, K, z}, x.dev);
    p.M = static_cast<int>(M);
    p.out_cols = static_cast<int>(N);
    p.num_kb = c.num_kb;
    p.tiles_m = c.tiles_m;
    p.tiles_n = c.tiles_n;
    p.tiles_per_z = c.tiles_per_z;
    p.M2 = static_cast<int>(N);
    p.out_cols2 = static_cast<int>(M);
    p.tiles_m2 = c.tiles_m2;
    p.tiles_n2 = c.tiles_n2;
    p.zcount = z;
    p.split = c.split;
    p.status = x.status;
    p.spin_limit = kSpinLimitCycles;
  }
  // First operand, rows along k.
  int a_k(const void* base, long long cols, long long rows, long long z, long long ld, long long zs) {
    // with few rows a load brings only those (the accumulator's rows beyond are never looked at)
    int box = 128;
    if (c.kv->cta_group == 1 && rows < 128) box = static_cast<int>((rows + 7) / 8 * 8);
    p.a_bytes = box * 128;
    return encode_batch16(&p.a, base, cols, rows, z, ld, zs, 64, box, CU_TENSOR_MAP_SWIZZLE_128B, bf16);
  }
  // First operand, rows along m (its memory rows are k).
  int a_mn(const void* base, long long cols, long long rows, long long z, long long ld, long long zs) {
    p.a_bytes = 128 * 128;
    return encode_batch16(&p.a, base, cols, rows, z, ld, zs, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B, bf16);
  }
  int a2_mn(const void* base, long long cols, long long rows, long long ld) {
    return encode_batch16(&p.a2, base, cols, rows, 1, ld, 0, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B, bf16);
  }
  int b_k(int i, const void* base, long long cols, long long rows, long long z, long long ld, long long zs) {
    const int box = op == kOpGate ? c.kv->block_n / 2 : c.kv->block_n / c.kv->cta_group;
    return encode_batch16(&p.b[i], base, cols, rows, z, ld, zs, 64, box, CU_TENSOR_MAP_SWIZZLE_128B, bf16);
  }
  int b_mn(int i, const void* base, long long cols, long long rows, long long z, long long ld, long long zs) {
    return encode_batch16(&p.b[i], base, cols, rows, z, ld, zs, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B, bf16);
  }
  // The boxes one epilogue warp reads and writes (FusedCfg::WIDE).
  int box_map(CUtensorMap* map, const void* base, long long z, long long ld, long long zs, bool as_bf16, bool second = false) const {
    const bool wide = op == kOpDact || op == kOpUpdateWide || op == kOpUpdateTall;
    return encode_batch16(map, base, second ? p.out_cols2 : p.out_cols, second ? p.M2 : p.M, z, ld, zs, wide ? 64 : 32, 32,
                          wide ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, as_bf16);
  }
  // padded: the rows are the library's own and have room up to the next 16 bytes.
  int output(int i, void* base, long long z, long long ld, long long zs, bool as_bf16, bool padded) {
    const bool second = op == kOpDw && i == 2;
    p.out[i] = base;
    p.out_ld[i] = ld;
    p.out_zstride = zs;
    if (!aligned16(base, ld) || (z > 1 && (zs % 8 != 0 || zs < ld * p.M))) return ROLLER_OK;
    p.out_tma |= 1 << i;
    if (padded || (second ? p.out_cols2 : p.out_cols) % 8 == 0) p.out_whole |= 1 << i;
    return box_map(&p.o[i], base, z, ld, zs, as_bf16, second);
  }
  // A matrix that the epilogue reads beside D.
  int input(int i, const void* base, long long z, long long ld, long long zs) {
    return box_map(&p.i[i], base, z, ld, zs, bf16);
  }
  // The mirror image of a symmetric output (always the library's own, aligned memory).
  int mirror(void* base, long long z, long long ld, long long zs) {
    return encode_batch16(&p.o[1], base, p.out_cols, p.M, z, ld, zs, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE, bf16);
  }
  int launch(cudaStream_t st) {
    FUSED_CUDA(c.kv->launch(p, c.grid, st));
    return ROLLER_OK;
  }
  int launch(LaunchOrder& order, cudaStream_t st) {
    order.next(&p.b_early, &p.late_wait);
    return launch(st);
  }
};

}  // namespace rb200
