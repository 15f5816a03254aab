// The gated feed-forward block: plan, workspaces and the order of its products. The arithmetic is
// in fused_gemm_sm100.cuh; the contract of the entry points in include/roller_b200.h.
//
//   forward    kOpGate:  h = act(x Wg^T) * (x Wu^T)        kOpDown:  y = h Wd^T
//   backward   kOpDact:  dh = dy Wd, from which dg, du and h leave together (dh itself stays in the
//                        accumulator, and h is made again from g and u rather than kept)
//              kOpDx:    dx = dg Wg + du Wu, one reduction over both
//              kOpDw:    dWg = dg^T x, dWu = du^T x and dWd = dy^T h in one launch: tiles of equal length
//              The last two launches need only what kOpDact wrote, so they overlap
//              (FusedParams::late_wait, LaunchOrder); kOpDx goes first, because its few long tiles leave SMs free.
#include <cstring>
#include <new>

#include "fused_product.h"

using namespace rb200;

namespace {

constexpr int kMaxExtent = 1 << 20;

enum { kPGate = 0, kPDown, kPDact, kPDx, kPDw, kProducts };
enum Operand { kX = 0, kWg, kWu, kWd, kDy, kG, kU, kOperands };

}  // namespace

struct roller_ffn_plan {
  FusedContext ctx;
  int max_tokens, d, f;
  int dt;                  // 1 = bf16, 2 = fp16
  int act;
  bool training;
  long long ldf;           // row stride of h, dg, du
  Arena arena;
  void* h;                 // [max_tokens, ldf]
  void* dgu;               // [2][max_tokens, ldf]
  void* pad[kOperands];    // copies of unaligned operands, in the arena ...
  void* own_pad[kOperands];  // ... or made when one turned out to be needed
  // The kernels chosen for the last number of tokens (choosing costs as much host time as a launch).
  int chosen_tokens;
  FusedChoice choice[kProducts];
};

namespace {

int rows_of(const roller_ffn_plan* p, int which) {
  return which == kWd ? p->d : (which == kWg || which == kWu) ? p->f : p->max_tokens;
}
int cols_of(const roller_ffn_plan* p, int which) {
  return which == kWd || which == kG || which == kU ? p->f : p->d;
}

size_t pad_bytes(const roller_ffn_plan* p, int which) {
  return static_cast<size_t>(rows_of(p, which)) * up64(cols_of(p, which)) * 2;
}

// The operand as the tensor maps may take it: itself, or a copy with aligned rows that `jobs` will make.
int usable(roller_ffn_plan* p, int which, const roller_mat& m, int rows, cudaStream_t st, AlignJobs* jobs,
           const void** ptr, long long* ld) {
  if (aligned16(m.ptr, m.ld)) {
    *ptr = m.ptr;
    *ld = m.ld;
    return ROLLER_OK;
  }
  const long long ldp = up64(cols_of(p, which));
  if (!p->pad[which]) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    FUSED_CUDA(cudaStreamIsCapturing(st, &cap));
    if (cap != cudaStreamCaptureStatusNone) return ROLLER_ERR_UNSUPPORTED;
    if (cudaMalloc(&p->own_pad[which], pad_bytes(p, which)) != cudaSuccess) {
      cudaGetLastError();
      p->own_pad[which] = nullptr;
      return ROLLER_ERR_NOMEM;
    }
    p->pad[which] = p->own_pad[which];
  }
  jobs->job[jobs->n++] = AlignJob{static_cast<const uint16_t*>(m.ptr), static_cast<uint16_t*>(p->pad[which]), m.ld,
                                  ldp, rows, cols_of(p, which), 0};
  *ptr = p->pad[which];
  *ld = ldp;
  return ROLLER_OK;
}

// The choices for `T` tokens.
const FusedChoice* choices(roller_ffn_plan* p, int T) {
  if (p->chosen_tokens != T) {
    const FusedShape shapes[kProducts] = {
        {kOpGate, p->dt, T, p->f, p->d, 1}, {kOpDown, p->dt, T, p->d, p->f, 1}, {kOpDact, p->dt, T, p->f, p->d, 1},
        {kOpDx, p->dt, T, p->d, p->f, 1},   {kOpDw, p->dt, p->f, p->d, T, 2}};
    for (int i = 0; i < (p->training ? kProducts : kPDact); ++i) p->choice[i] = fused_choose(shapes[i], p->ctx.dev);
    p->chosen_tokens = T;
  }
  return p->choice;
}

bool given(const roller_mat& m, long long cols) { return m.ptr && m.ld >= cols; }

int check_plan(const roller_ffn_plan* p, const roller_ffn_io* io) {
  if (!p || !io || io->tokens < 0) return ROLLER_ERR_INVALID;
  if (io->tokens > p->max_tokens) return ROLLER_ERR_TOO_LARGE;
  int cur = -1;
  if (cudaGetDevice(&cur) != cudaSuccess || cur != p->ctx.device) return ROLLER_ERR_DEVICE;
  return ROLLER_OK;
}

}  // namespace

extern "C" {

int roller_b200_ffn_create(int max_tokens, int d_model, int d_ff, int mode, int activation, int flags,
                           roller_ffn_plan** out) {
  if (!out) return ROLLER_ERR_INVALID;
  *out = nullptr;
  if (max_tokens < 1 || d_model < 1 || d_ff < 1 || max_tokens > kMaxExtent || d_model > kMaxExtent ||
      d_ff > kMaxExtent)
    return ROLLER_ERR_INVALID;
  if (mode != ROLLER_MODE_BF16 && mode != ROLLER_MODE_F16) return ROLLER_ERR_INVALID;
  if (activation < ROLLER_ACT_SILU || activation > ROLLER_ACT_GELU_TANH) return ROLLER_ERR_INVALID;
  if (flags & ~ROLLER_FFN_TRAINING) return ROLLER_ERR_INVALID;
  roller_ffn_plan* p = new (std::nothrow) roller_ffn_plan();
  if (!p) return ROLLER_ERR_NOMEM;
  memset(static_cast<void*>(p), 0, sizeof(*p));
  const int rc = fused_context_create(&p->ctx);
  if (rc != ROLLER_OK) {
    delete p;
    return rc;
  }
  p->max_tokens = max_tokens;
  p->d = d_model;
  p->f = d_ff;
  p->dt = mode == ROLLER_MODE_BF16 ? 1 : 2;
  p->act = activation;
  p->training = (flags & ROLLER_FFN_TRAINING) != 0;
  p->ldf = up64(d_ff);
  const size_t h_bytes = static_cast<size_t>(max_tokens) * p->ldf * 2;
  const size_t h = p->arena.take(h_bytes);
  const size_t dgu = p->training ? p->arena.take(2 * h_bytes) : 0;
  size_t pad[kOperands];
  bool padded[kOperands];      // operands that are unaligned when they are contiguous
  for (int i = 0; i < kOperands; ++i) {
    padded[i] = cols_of(p, i) % 8 != 0 && (i < kDy || p->training);
    pad[i] = padded[i] ? p->arena.take(pad_bytes(p, i)) : 0;
  }
  const cudaError_t e = p->arena.allocate();
  if (e != cudaSuccess) {
    const int failed = e == cudaErrorMemoryAllocation ? ROLLER_ERR_NOMEM : report_cuda_error(e, "ffn plan setup");
    cudaGetLastError();
    p->arena.base = nullptr;
    roller_b200_ffn_destroy(p);
    return failed;
  }
  p->h = p->arena.at<void>(h);
  if (p->training) p->dgu = p->arena.at<void>(dgu);
  for (int i = 0; i < kOperands; ++i)
    if (padded[i]) p->pad[i] = p->arena.at<void>(pad[i]);
  *out = p;
  return ROLLER_OK;
}

int roller_b200_ffn_forward(roller_ffn_plan* p, const roller_ffn_io* io, void* stream) {
  FUSED_OK(check_plan(p, io));
  const int T = io->tokens, D = p->d, F = p->f;
  if (T == 0) return ROLLER_OK;
  if (!given(io->x, D) || !given(io->wg, D) || !given(io->wu, D) || !given(io->wd, F) || !given(io->y, D))
    return ROLLER_ERR_INVALID;
  const bool save = io->g.ptr || io->u.ptr;
  if (save && (!given(io->g, F) || !given(io->u, F))) return ROLLER_ERR_INVALID;
  const void* outs[] = {io->y.ptr, io->g.ptr, io->u.ptr};
  const void* all[] = {io->x.ptr, io->wg.ptr, io->wu.ptr, io->wd.ptr, io->y.ptr, io->g.ptr, io->u.ptr};
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 4 + i; ++j)
      if (outs[i] && outs[i] == all[j]) return ROLLER_ERR_INVALID;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = p->dt == 1;
  const FusedChoice* choice = choices(p, T);
  const void *x, *wg, *wu, *wd;
  long long ldx, ldg, ldu, ldd;
  // Copies of unaligned operands: those of the first product before it, the others behind it, where
  // they run on the SMs that its last wave leaves idle.
  AlignJobs jobs, later;
  LaunchOrder order;
  later.late = 1;
  FUSED_OK(usable(p, kX, io->x, T, st, &jobs, &x, &ldx));
  FUSED_OK(usable(p, kWg, io->wg, F, st, &jobs, &wg, &ldg));
  FUSED_OK(usable(p, kWu, io->wu, F, st, &jobs, &wu, &ldu));
  FUSED_OK(usable(p, kWd, io->wd, D, st, &later, &wd, &ldd));
  FUSED_CUDA(align_rows(jobs, order, p->ctx.dev.sm_count, st));
  {
    Product g(p->ctx, kOpGate, p->dt, T, F, D, 1, &choice[kPGate]);
    g.p.act = p->act;
    FUSED_OK(g.a_k(x, D, T, 1, ldx, 0));
    FUSED_OK(g.b_k(0, wg, D, F, 1, ldg, 0));
    FUSED_OK(g.b_k(1, wu, D, F, 1, ldu, 0));
    FUSED_OK(g.output(0, p->h, 1, p->ldf, 0, bf16, true));
    if (save) {
      FUSED_OK(g.output(1, io->g.ptr, 1, io->g.ld, 0, bf16, false));
      FUSED_OK(g.output(2, io->u.ptr, 1, io->u.ld, 0, bf16, false));
      g.p.flags |= kFusedSave;
    }
    FUSED_OK(g.launch(order, st));
  }
  FUSED_CUDA(align_rows(later, order, p->ctx.dev.sm_count, st));
  Product d(p->ctx, kOpDown, p->dt, T, D, F, 1, &choice[kPDown]);
  d.p.b_early = later.n == 0;   // Wd comes neither from the gate kernel nor from a copy
  FUSED_OK(d.a_k(p->h, F, T, 1, p->ldf, 0));
  FUSED_OK(d.b_k(0, wd, F, D, 1, ldd, 0));
  FUSED_OK(d.output(0, io->y.ptr, 1, io->y.ld, 0, bf16, false));
  return d.launch(order, st);
}

int roller_b200_ffn_backward(roller_ffn_plan* p, const roller_ffn_io* io, void* stream) {
  FUSED_OK(check_plan(p, io));
  if (!p->training) return ROLLER_ERR_UNSUPPORTED;
  const int T = io->tokens, D = p->d, F = p->f;
  if (!given(io->dwg, D) || !given(io->dwu, D) || !given(io->dwd, F)) return ROLLER_ERR_INVALID;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    FUSED_CUDA(cudaMemset2DAsync(io->dwg.ptr, io->dwg.ld * 2, 0, static_cast<size_t>(D) * 2, F, st));
    FUSED_CUDA(cudaMemset2DAsync(io->dwu.ptr, io->dwu.ld * 2, 0, static_cast<size_t>(D) * 2, F, st));
    FUSED_CUDA(cudaMemset2DAsync(io->dwd.ptr, io->dwd.ld * 2, 0, static_cast<size_t>(F) * 2, D, st));
    return ROLLER_OK;
  }
  if (!given(io->x, D) || !given(io->wg, D) || !given(io->wu, D) || !given(io->wd, F) || !given(io->g, F) ||
      !given(io->u, F) || !given(io->dy, D) || !given(io->dx, D))
    return ROLLER_ERR_INVALID;
  const void* all[] = {io->x.ptr, io->wg.ptr, io->wu.ptr, io->wd.ptr, io->g.ptr,  io->u.ptr,
                       io->dy.ptr, io->dx.ptr, io->dwg.ptr, io->dwu.ptr, io->dwd.ptr};
  for (int i = 7; i < 11; ++i)
    for (int j = 0; j < i; ++j)
      if (all[i] == all[j]) return ROLLER_ERR_INVALID;
  const bool bf16 = p->dt == 1;
  const FusedChoice* choice = choices(p, T);
  const void *x, *wg, *wu, *wd, *dy, *g, *u;
  long long ldx, ldg, ldu, ldd, ldy, ldsg, ldsu;
  // Copies of unaligned operands: those of the first product before it, the others behind it, where
  // they run on the SMs that its last wave leaves idle.
  AlignJobs jobs, later;
  LaunchOrder order;
  later.late = 1;
  FUSED_OK(usable(p, kX, io->x, T, st, &later, &x, &ldx));
  FUSED_OK(usable(p, kWg, io->wg, F, st, &later, &wg, &ldg));
  FUSED_OK(usable(p, kWu, io->wu, F, st, &later, &wu, &ldu));
  FUSED_OK(usable(p, kWd, io->wd, D, st, &jobs, &wd, &ldd));
  FUSED_OK(usable(p, kDy, io->dy, T, st, &jobs, &dy, &ldy));
  FUSED_OK(usable(p, kG, io->g, T, st, &jobs, &g, &ldsg));
  FUSED_OK(usable(p, kU, io->u, T, st, &jobs, &u, &ldsu));
  FUSED_CUDA(align_rows(jobs, order, p->ctx.dev.sm_count, st));
  const long long zs = static_cast<long long>(p->max_tokens) * p->ldf;   // dg to du
  {
    Product a(p->ctx, kOpDact, p->dt, T, F, D, 1, &choice[kPDact]);
    a.p.act = p->act;
    FUSED_OK(a.a_k(dy, D, T, 1, ldy, 0));
    FUSED_OK(a.b_mn(0, wd, F, D, 1, ldd, 0));
    FUSED_OK(a.output(0, p->dgu, 1, p->ldf, 0, bf16, true));
    FUSED_OK(a.output(1, static_cast<uint16_t*>(p->dgu) + zs, 1, p->ldf, 0, bf16, true));
    FUSED_OK(a.output(2, p->h, 1, p->ldf, 0, bf16, true));
    FUSED_OK(a.input(0, g, 1, ldsg, 0));
    FUSED_OK(a.input(1, u, 1, ldsu, 0));
    FUSED_OK(a.launch(order, st));
  }
  FUSED_CUDA(align_rows(later, order, p->ctx.dev.sm_count, st));
  {
    Product r(p->ctx, kOpDx, p->dt, T, D, F, 1, &choice[kPDx]);
    r.p.b_early = later.n == 0;   // Wg and Wu come neither from the kernel above nor from a copy
    FUSED_OK(r.a_k(p->dgu, F, T, 2, p->ldf, zs));
    FUSED_OK(r.b_mn(0, wg, D, F, 1, ldg, 0));
    FUSED_OK(r.b_mn(1, wu, D, F, 1, ldu, 0));
    FUSED_OK(r.output(0, io->dx.ptr, 1, io->dx.ld, 0, bf16, false));
    FUSED_OK(r.launch(order, st));
  }
  Product w(p->ctx, kOpDw, p->dt, F, D, T, 2, &choice[kPDw]);
  w.p.late_wait = 1;   // dg, du and h were complete before the kernel above started
  fused_deal(choice[kPDx], choice[kPDw], p->ctx.dev, &w.p.head, &w.p.head_tiles);
  FUSED_OK(w.a_mn(p->dgu, F, T, 2, p->ldf, zs));
  FUSED_OK(w.b_mn(0, x, D, T, 1, ldx, 0));
  FUSED_OK(w.output(0, io->dwg.ptr, 1, io->dwg.ld, 0, bf16, false));
  FUSED_OK(w.output(1, io->dwu.ptr, 1, io->dwu.ld, 0, bf16, false));
  FUSED_OK(w.a2_mn(dy, D, T, ldy));
  FUSED_OK(w.b_mn(1, p->h, F, T, 1, p->ldf, 0));
  FUSED_OK(w.output(2, io->dwd.ptr, 1, io->dwd.ld, 0, bf16, false));
  return w.launch(order, st);
}

int roller_b200_ffn_status(roller_ffn_plan* p, uint32_t* device_status) {
  if (!p) return ROLLER_ERR_INVALID;
  return fused_context_status(&p->ctx, device_status);
}

int roller_b200_ffn_destroy(roller_ffn_plan* p) {
  if (!p) return ROLLER_OK;
  cudaFree(p->arena.base);
  for (void* b : p->own_pad) cudaFree(b);
  fused_context_destroy(&p->ctx);
  cudaGetLastError();
  delete p;
  return ROLLER_OK;
}

}  // extern "C"
