// The Newton-Schulz iteration on a batch of matrices: norm, conversion, and three products a
// step. The products are in fused_gemm_sm100.cuh; the contract in include/roller_b200.h.
//
// With m the shorter side and x on that side (x x^T for a wide matrix, x^T x for a tall one):
//     p = x x^T          m m n / 2   multiplications (one triangle of a symmetric product)
//     q = b p + c p p    m m m / 2
//     x = a x + q x      m m n
// Numbers. Everything is scaled by S = 2^10, so that the entries of x (about 1 / sqrt(m n) at the
// start, 1 / sqrt(n) at the end), p and q sit in fp16's normal range. The operands of the products
// are fp16: 2^-12 a rounding, where bf16 would lose 2^-9. The iteration multiplies weak
// directions by a = 3.4 a step, and with them whatever was rounded off x in those directions, so a
// matrix of low rank would come out with 4e-2 (rank 8) to 1.5e-1 (rank 1) of noise; x is
// therefore carried as hi + lo, two fp16 numbers, and only q x reads hi alone: there a weak
// direction's error meets the weak direction's q, which is small. What rounding loses on q's
// diagonal (as large as all its other roundings together, once p is near the identity) goes into
// the fp32 factor of x. Against 64 bits: 0.3-2e-3 of |x| before the last rounding to bf16.
#include <cmath>
#include <new>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fused_product.h"
#include "ptx_sm100.cuh"

using namespace rb200;

namespace {

constexpr float kScale = 1024.0f;   // S
constexpr int kSumBlocks = 1184;    // blocks of the norm per matrix, at most
constexpr int kMaxSide = 65536, kMaxShort = 16384, kMaxBatch = 4096;

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

// Eight consecutive elements of a row (those beyond the row's end are zero). Ordinary loads, not those of
// constant data (ld.global.nc): the kernel before may still be writing them when this one starts.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int col, int cols, bool vec, float (&v)[8]) {
  if (vec && col + 8 <= cols) {
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(row + col)[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(t[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = col + j < cols ? to_float(row[col + j]) : 0.0f;
  }
}

struct Source {
  const void* g;
  long long ld, zs;
  int rows, cols;
  int vec;             // rows and matrices start on 16 bytes
  uint32_t per_row;    // groups of eight elements in a row
};

// A thread of the next two kernels takes every (grid's threads)-th group of eight elements of a
// matrix, four groups at a time, so that 64 to 128 bytes per thread are on their way.
constexpr int kGroupsAtOnce = 4;
struct Walk {
  uint32_t r, c, dr, dc, per_row;     // row and group in it; the step, likewise
  __device__ explicit Walk(uint32_t per_row_) : per_row(per_row_) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x, stride = gridDim.x * 256u;
    r = u / per_row;
    c = u - r * per_row;
    dr = stride / per_row;
    dc = stride - dr * per_row;
  }
  __device__ void step() {
    r += dr;
    c += dc;
    if (c >= per_row) {
      c -= per_row;
      ++r;
    }
  }
};

__device__ __forceinline__ double block_sum(double sum) {
  __shared__ double warp_sum[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < 8; ++i) sum += warp_sum[i];
  return sum;
}

// Sum of squares of each matrix, one partial sum per block. Eight elements at a time are scaled by a
// power of two to below 4, squared and added in fp32, and their sum goes on in fp64: neither
// tiny nor huge matrices leave the range, and the one conversion to fp64 per eight elements
// does not bound the read (one per element would: 4 a cycle and SM).
template <typename T>
__global__ void __launch_bounds__(256) ortho_sumsq(Source s, double* __restrict__ part) {
  grid_dependency_wait();
  grid_launch_dependents();
  const T* g = static_cast<const T*>(s.g) + blockIdx.y * s.zs;
  const uint32_t rows = static_cast<uint32_t>(s.rows);
  double sum = 0.0;
  Walk w(s.per_row);
  while (w.r < rows) {
    float v[kGroupsAtOnce][8];
#pragma unroll
    for (int i = 0; i < kGroupsAtOnce; ++i, w.step()) {
      if (w.r < rows) {
        load8(g + w.r * s.ld, static_cast<int>(w.c) * 8, s.cols, s.vec, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kGroupsAtOnce; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
      // exponent of the largest; 255 (not finite) passes through unscaled
      const uint32_t e = top >> 23;
      const uint32_t k = e < 253u ? e : 253u;
      const float scale = e == 255u ? 1.0f : __uint_as_float((254u - k) << 23);   // 2^(127 - k)
      float q = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = v[i][j] * scale;
        q = fmaf(f, f, q);
      }
      // times 2^(2 (k - 127))
      sum += static_cast<double>(q) * __hiloint2double(static_cast<int>((769u + 2u * k) << 20), 0);
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) part[blockIdx.y * kSumBlocks + blockIdx.x] = sum;
}

// x = S g / (|g| + eps) as hi + lo. Every block adds the partial sums in the same order. The factor
// itself can leave fp32's range (norms under 1e-35 or over 1e40), so a power of two goes first.
// Norm and scaling of 8192 x 4096 in fp32 take 48 us together, about what writing hi and lo and
// reading g twice take (403 MB, a part of the second time from L2).
template <typename T>
__global__ void __launch_bounds__(256)
ortho_scale(Source s, const double* part, int parts, double eps, __half* __restrict__ hi,
            __half* __restrict__ lo, long long ldx, long long zsx) {
  grid_dependency_wait();
  grid_launch_dependents();
  const T* g = static_cast<const T*>(s.g) + blockIdx.y * s.zs;
  const uint32_t rows = static_cast<uint32_t>(s.rows);
  Walk w(s.per_row);
  Walk back = w;
  float v[kGroupsAtOnce][8];
  auto load = [&]() {
    back = w;
#pragma unroll
    for (int i = 0; i < kGroupsAtOnce; ++i, w.step())
      if (w.r < rows) load8(g + w.r * s.ld, static_cast<int>(w.c) * 8, s.cols, s.vec, v[i]);
  };
  load();      // on their way while the norm is put together

  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) sum += __ldcg(part + blockIdx.y * kSumBlocks + i);
  sum = block_sum(sum);
  const double norm = sqrt(sum) + eps;
  const int e = ((__double2hiint(norm) >> 20) & 0x7FF) - 1023;
  const float near_one = __uint_as_float(static_cast<uint32_t>(127 - max(-100, min(100, e))) << 23);
  const float scale = static_cast<float>(static_cast<double>(kScale) / (norm * near_one));

  while (back.r < rows) {
#pragma unroll
    for (int i = 0; i < kGroupsAtOnce; ++i, back.step()) {
      if (back.r >= rows) break;
      alignas(16) __half h[8], l[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = v[i][j] * near_one * scale;
        h[j] = __float2half_rn(f);
        l[j] = __float2half_rn(f - __half2float(h[j]));
      }
      const long long at = blockIdx.y * zsx + back.r * ldx + back.c * 8;
      *reinterpret_cast<uint4*>(hi + at) = *reinterpret_cast<const uint4*>(h);
      *reinterpret_cast<uint4*>(lo + at) = *reinterpret_cast<const uint4*>(l);
    }
    load();
  }
}

template <typename T>
int convert(const Source& s, int batch, int sm_count, double* part, double eps, __half* hi, __half* lo,
            long long ldx, long long zsx, cudaStream_t st) {
  // about eight blocks per SM over the whole batch
  const long long groups = static_cast<long long>(s.per_row) * s.rows;
  long long blocks = (groups + 256 * kGroupsAtOnce - 1) / (256 * kGroupsAtOnce);
  const int most = (8 * sm_count + batch - 1) / batch;
  if (blocks > most) blocks = most;
  if (blocks > kSumBlocks) blocks = kSumBlocks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(batch), 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FUSED_CUDA(cudaLaunchKernelEx(&cfg, ortho_sumsq<T>, s, part));
  FUSED_CUDA(cudaLaunchKernelEx(&cfg, ortho_scale<T>, s, static_cast<const double*>(part), static_cast<int>(blocks), eps, hi,
                                lo, ldx, zsx));
  return ROLLER_OK;
}

// The largest |s (a + b s^2 + c s^4)| for s in [0, r], and the largest |b s^2 + c s^4|.
void polynomial_range(double a, double b, double c, double r, double* out, double* poly) {
  *out = *poly = 0.0;
  for (int i = 0; i <= 4096; ++i) {
    const double s = r * i / 4096.0, q = b * s * s + c * s * s * s * s;
    *out = fmax(*out, fabs(s * (a + q)));
    *poly = fmax(*poly, fabs(q));
  }
}

}  // namespace

struct roller_ortho_plan {
  FusedContext ctx;
  int batch, rows, cols, in_type, steps;
  int m, n;                // shorter and longer side
  bool tall;
  float a, b, c, eps;
  long long ldx, zsx, ldm, zsm;
  Arena arena;
  double* part;            // partial sums of squares
  __half* x[2][2];         // [which][hi, lo], [batch][rows][ldx]
  __half *pm, *qm;         // p and q, [batch][m][ldm]
  float* vec;              // [batch][ldm]
  // The launches of a step, built once: everything they touch is the plan's own, but for the last
  // step's output. [which x] reads x[which] and writes the other.
  Product *gram[2], *poly, *update[2], *last[2];
};

namespace {

// Tensor maps and parameters of the plan's launches.
int build_products(roller_ortho_plan* p) {
  const int R = p->rows, C = p->cols, Z = p->batch, m = p->m, n = p->n;
  for (int w = 0; w < 2; ++w) {
    __half *hi = p->x[w][0], *lo = p->x[w][1];
    p->gram[w] = new (std::nothrow) Product(p->ctx, p->tall ? kOpGramTall : kOpGramWide, 2, m, m, n, Z);
    if (!p->gram[w]) return ROLLER_ERR_NOMEM;
    Product& g = *p->gram[w];
    if (p->tall) {
      FUSED_OK(g.a_mn(hi, C, R, Z, p->ldx, p->zsx));
      FUSED_OK(g.b_mn(0, hi, C, R, Z, p->ldx, p->zsx));
    } else {
      FUSED_OK(g.a_k(hi, C, R, Z, p->ldx, p->zsx));
      FUSED_OK(g.b_k(0, hi, C, R, Z, p->ldx, p->zsx));
    }
    FUSED_OK(g.output(0, p->pm, Z, p->ldm, p->zsm, false, true));
    FUSED_OK(g.mirror(p->pm, Z, p->ldm, p->zsm));
    g.p.inv_scale = 1.0f / kScale;
    for (int final_step = 0; final_step < 2; ++final_step) {
      Product*& slot = final_step ? p->last[w] : p->update[w];
      slot = new (std::nothrow) Product(p->ctx, p->tall ? kOpUpdateTall : kOpUpdateWide, 2, R, C, m, Z);
      if (!slot) return ROLLER_ERR_NOMEM;
      Product& u = *slot;
      if (p->tall) {
        FUSED_OK(u.a_k(hi, C, R, Z, p->ldx, p->zsx));
        FUSED_OK(u.b_k(0, p->qm, m, m, Z, p->ldm, p->zsm));
      } else {
        FUSED_OK(u.a_k(p->qm, m, m, Z, p->ldm, p->zsm));
        FUSED_OK(u.b_mn(0, hi, C, R, Z, p->ldx, p->zsx));
      }
      FUSED_OK(u.input(0, hi, Z, p->ldx, p->zsx));
      FUSED_OK(u.input(1, lo, Z, p->ldx, p->zsx));
      u.p.vec = p->vec;
      u.p.vec_ld = static_cast<int>(p->ldm);
      u.p.inv_scale = 1.0f / kScale;
      if (final_step) {
        u.p.flags |= kFusedLast;      // (its output is set by each call)
      } else {
        FUSED_OK(u.output(0, p->x[1 - w][0], Z, p->ldx, p->zsx, false, true));
        FUSED_OK(u.output(1, p->x[1 - w][1], Z, p->ldx, p->zsx, false, true));
      }
    }
  }
  p->poly = new (std::nothrow) Product(p->ctx, kOpPoly, 2, m, m, m, Z);
  if (!p->poly) return ROLLER_ERR_NOMEM;
  Product& q = *p->poly;
  FUSED_OK(q.a_k(p->pm, m, m, Z, p->ldm, p->zsm));
  FUSED_OK(q.b_k(0, p->pm, m, m, Z, p->ldm, p->zsm));
  FUSED_OK(q.input(0, p->pm, Z, p->ldm, p->zsm));
  FUSED_OK(q.output(0, p->qm, Z, p->ldm, p->zsm, false, true));
  FUSED_OK(q.mirror(p->qm, Z, p->ldm, p->zsm));
  q.p.vec = p->vec;
  q.p.vec_ld = static_cast<int>(p->ldm);
  q.p.coef_a = p->a;
  q.p.coef_b = p->b;
  q.p.coef_c = p->c / kScale;
  q.p.inv_scale = 1.0f / kScale;
  return ROLLER_OK;
}

}  // namespace

extern "C" {

int roller_b200_ortho_create(int batch, int rows, int cols, int in_type, int steps, float a, float b,
                             float c, float eps, roller_ortho_plan** out) {
  if (!out) return ROLLER_ERR_INVALID;
  *out = nullptr;
  if (batch < 1 || batch > kMaxBatch || rows < 1 || cols < 1 || rows > kMaxSide || cols > kMaxSide)
    return ROLLER_ERR_INVALID;
  if ((rows < cols ? rows : cols) > kMaxShort) return ROLLER_ERR_TOO_LARGE;
  if (in_type < ROLLER_ORTHO_IN_F32 || in_type > ROLLER_ORTHO_IN_F16 || steps < 1 || steps > 32)
    return ROLLER_ERR_INVALID;
  if (!(eps >= 0.0f) || !std::isfinite(eps) || !std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c))
    return ROLLER_ERR_INVALID;
  double r = 1.0;
  for (int i = 0; i < steps; ++i) {
    double next, poly;
    polynomial_range(a, b, c, r, &next, &poly);
    if (!(poly < 32.0) || !(next < 4.0)) return ROLLER_ERR_INVALID;
    r = fmax(r, next);
  }
  roller_ortho_plan* p = new (std::nothrow) roller_ortho_plan();
  if (!p) return ROLLER_ERR_NOMEM;
  memset(static_cast<void*>(p), 0, sizeof(*p));
  const int rc = fused_context_create(&p->ctx);
  if (rc != ROLLER_OK) {
    delete p;
    return rc;
  }
  p->batch = batch;
  p->rows = rows;
  p->cols = cols;
  p->in_type = in_type;
  p->steps = steps;
  p->tall = rows > cols;
  p->m = p->tall ? cols : rows;
  p->n = p->tall ? rows : cols;
  p->a = a;
  p->b = b;
  p->c = c;
  p->eps = eps;
  p->ldx = up64(cols);
  p->zsx = p->ldx * rows;
  p->ldm = up64(p->m);
  p->zsm = p->ldm * p->m;
  size_t x[4];
  for (size_t& at : x) at = p->arena.take(sizeof(__half) * p->zsx * batch);
  const size_t pm = p->arena.take(sizeof(__half) * p->zsm * batch), qm = p->arena.take(sizeof(__half) * p->zsm * batch);
  const size_t vec = p->arena.take(sizeof(float) * p->ldm * batch);
  const size_t part = p->arena.take(sizeof(double) * kSumBlocks * batch);
  const cudaError_t e = p->arena.allocate();
  if (e != cudaSuccess) {
    const int failed = e == cudaErrorMemoryAllocation ? ROLLER_ERR_NOMEM : report_cuda_error(e, "ortho plan setup");
    cudaGetLastError();
    p->arena.base = nullptr;
    roller_b200_ortho_destroy(p);
    return failed;
  }
  for (int i = 0; i < 4; ++i) p->x[i / 2][i % 2] = p->arena.at<__half>(x[i]);
  p->pm = p->arena.at<__half>(pm);
  p->qm = p->arena.at<__half>(qm);
  p->vec = p->arena.at<float>(vec);
  p->part = p->arena.at<double>(part);
  const int built = build_products(p);
  if (built != ROLLER_OK) {
    roller_b200_ortho_destroy(p);
    return built;
  }
  *out = p;
  return ROLLER_OK;
}

// Whether rows of `cols` elements, `ld` apart in matrices `zs` apart, never overlap: matrices one
// after the other, or interleaved row by row.
static bool strides_ok(long long batch, long long rows, long long cols, long long ld, long long zs) {
  if (rows == 1) return batch == 1 || zs >= cols;
  if (ld < cols) return false;
  if (batch == 1) return true;
  return zs >= ld * (rows - 1) + cols || (zs >= cols && ld >= zs * (batch - 1) + cols);
}

int roller_b200_ortho_run(roller_ortho_plan* p, const void* g, long long ld_g, long long zs_g, void* out,
                          long long ld_out, long long zs_out, void* stream) {
  if (!p || !g || !out || g == out) return ROLLER_ERR_INVALID;
  int cur = -1;
  if (cudaGetDevice(&cur) != cudaSuccess || cur != p->ctx.device) return ROLLER_ERR_DEVICE;
  if (p->rows == 1) ld_g = ld_out = up64(p->cols);   // there is no second row to step to
  if (!strides_ok(p->batch, p->rows, p->cols, ld_g, zs_g) || !strides_ok(p->batch, p->rows, p->cols, ld_out, zs_out))
    return ROLLER_ERR_INVALID;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Source s;
  s.g = g;
  s.ld = ld_g;
  s.zs = zs_g;
  s.rows = p->rows;
  s.cols = p->cols;
  const int per16 = p->in_type == ROLLER_ORTHO_IN_F32 ? 4 : 8;
  s.vec = (reinterpret_cast<uintptr_t>(g) & 15) == 0 && ld_g % per16 == 0 && (p->batch == 1 || zs_g % per16 == 0);
  s.per_row = static_cast<uint32_t>((p->cols + 7) / 8);
  const int sms = p->ctx.dev.sm_count;
  if (p->in_type == ROLLER_ORTHO_IN_F32)
    FUSED_OK(convert<float>(s, p->batch, sms, p->part, p->eps, p->x[0][0], p->x[0][1], p->ldx, p->zsx, st));
  else if (p->in_type == ROLLER_ORTHO_IN_BF16)
    FUSED_OK(convert<__nv_bfloat16>(s, p->batch, sms, p->part, p->eps, p->x[0][0], p->x[0][1], p->ldx, p->zsx, st));
  else
    FUSED_OK(convert<__half>(s, p->batch, sms, p->part, p->eps, p->x[0][0], p->x[0][1], p->ldx, p->zsx, st));

  for (int i = 0; i < p->steps; ++i) {
    const int w = i & 1;
    FUSED_OK(p->gram[w]->launch(st));
    FUSED_OK(p->poly->launch(st));
    if (i + 1 < p->steps) {
      FUSED_OK(p->update[w]->launch(st));
      continue;
    }
    Product u = *p->last[w];
    FUSED_OK(u.output(0, out, p->batch, ld_out, zs_out, true, false));
    FUSED_OK(u.launch(st));
  }
  return ROLLER_OK;
}

int roller_b200_ortho_status(roller_ortho_plan* p, uint32_t* device_status) {
  if (!p) return ROLLER_ERR_INVALID;
  return fused_context_status(&p->ctx, device_status);
}

int roller_b200_ortho_destroy(roller_ortho_plan* p) {
  if (!p) return ROLLER_OK;
  for (Product* q : {p->gram[0], p->gram[1], p->poly, p->update[0], p->update[1], p->last[0], p->last[1]}) delete q;
  cudaFree(p->arena.base);
  fused_context_destroy(&p->ctx);
  cudaGetLastError();
  delete p;
  return ROLLER_OK;
}

}  // extern "C"
