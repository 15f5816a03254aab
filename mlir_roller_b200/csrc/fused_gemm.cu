// Which fused product kernel a problem runs on, and how its reduction is cut.
#include <atomic>

#include "fused_product.h"
#include "ptx_sm100.cuh"

namespace rb200 {

namespace {

const FusedVariant* table(int i, int* n) {
  switch (i) {
    case 0: return fused_variants_bf16(n);
    case 1: return fused_variants_f16(n);
    default: return fused_variants_ortho(n);
  }
}

// Measured on B200 over widths 512 .. 8192, 1 .. 8192 rows (every kernel and split timed beside the
// others).
struct TileCost {
  int cta_group, block_n;
  double alone_us, busy_us;   // one k-block of one tile, on a few SMs and on all of them
  double epilogue_us;         // of one tile, plain; hidden behind the next tile's k-blocks
  double fixed_us;            // start, first loads, last epilogue
};
constexpr TileCost kTiles[] = {{2, 256, 0.26, 0.33, 4.1, 7.0},
                               {2, 128, 0.145, 0.20, 2.6, 4.8},
                               {1, 256, 0.285, 0.39, 3.2, 6.4},
                               {1, 128, 0.18, 0.23, 3.2, 3.7},
                               {1, 64, 0.155, 0.172, 1.5, 2.9}};
// The epilogues beside the plain one.
double epilogue_weight(int op) {
  switch (op) {
    case kOpDact: return 4.7;
    case kOpUpdateTall: return 2.0;
    case kOpUpdateWide: return 1.5;
    case kOpGate: return 0.9;
    case kOpDw: return 0.3;
    default: return 0.55;
  }
}

// Copies the jobs' 16-bit rows into rows that start on 16 bytes. A warp takes 256 words (of two
// elements) of a row at a time, a thread eight of them, all on their way together: a source row
// that starts between two words gives each word from two neighbouring ones, the second of which the
// next lane has. (A word that holds an element of the row may be read whole. Ordinary loads, not those of
// constant data: the kernel before may still be writing an operand when this one starts.)
// A 2048 x 5461 weight costs a forward call of 777 tokens 8 us of 72 (45 MB, overlapped with the first
// product's end).
// jobs.late: as FusedParams::late_wait, the copies need nothing from the previous kernel.
__global__ void __launch_bounds__(256) align_rows_kernel(const __grid_constant__ AlignJobs jobs) {
  if (!jobs.late) grid_dependency_wait();
  grid_launch_dependents();
  int b = static_cast<int>(blockIdx.x), i = 0;
  while (i + 1 < jobs.n && b >= jobs.job[i].blocks) b -= jobs.job[i++].blocks;
  const AlignJob& j = jobs.job[i];
  const int lane = threadIdx.x & 31;
  const int words = (j.cols + 1) / 2, runs = (words + 255) / 256;
  const long long units = static_cast<long long>(j.rows) * runs;
  for (long long u = b * 8 + static_cast<int>(threadIdx.x >> 5); u < units; u += j.blocks * 8) {
    const int row = static_cast<int>(u / runs), w0 = static_cast<int>(u - static_cast<long long>(row) * runs) * 256 + lane;
    const uintptr_t at = reinterpret_cast<uintptr_t>(j.src + row * j.ld_src);
    const uint32_t* src = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
    uint32_t* dst = reinterpret_cast<uint32_t*>(j.dst + row * j.ld_dst);
    const bool between = (at & 2) != 0;
    const int sources = (j.cols + (between ? 2 : 1)) / 2;
    uint32_t x[9];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = w0 + 32 * k < sources ? src[w0 + 32 * k] : 0u;
    x[8] = between && lane == 31 && w0 + 225 < sources ? src[w0 + 225] : 0u;   // (only lane 31's neighbour)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t next = __shfl_sync(0xffffffffu, lane == 0 ? x[k + 1] : x[k], (lane + 1) & 31);
      if (k == 7 && lane == 31) next = x[8];
      if (w0 + 32 * k < words) dst[w0 + 32 * k] = between ? __byte_perm(x[k], next, 0x5432) : x[k];
    }
  }
  if (jobs.late) grid_dependency_wait();
}

}  // namespace

cudaError_t align_rows(AlignJobs& jobs, LaunchOrder& order, int sm_count, cudaStream_t stream) {
  if (jobs.n == 0) return cudaSuccess;
  order.next(nullptr, &jobs.late);
  // blocks in proportion to the jobs' sizes, eight per SM in all
  double total = 0.0;
  for (int i = 0; i < jobs.n; ++i) total += static_cast<double>(jobs.job[i].rows) * jobs.job[i].cols;
  int blocks = 0;
  for (int i = 0; i < jobs.n; ++i) {
    AlignJob& j = jobs.job[i];
    const double most = (static_cast<double>(j.rows) * ((j.cols + 511) / 512) + 7) / 8;
    const double b = 8.0 * sm_count * j.rows * j.cols / total + 1;
    j.blocks = static_cast<int>(b < most ? b : most);
    blocks += j.blocks;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, align_rows_kernel, jobs);
}

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

// Raises the kernels' shared-memory limits on the current device and asks how many clusters of
// their CTAs it can hold at once.
static cudaError_t bind_device(FusedDevice* d) {
  int largest[2] = {0, 0};
  const void* func[2] = {nullptr, nullptr};
  int threads = 0;
  for (int i = 0; i < 3; ++i) {
    int n = 0;
    const FusedVariant* t = table(i, &n);
    for (int j = 0; j < n; ++j) {
      const cudaError_t e = cudaFuncSetAttribute(t[j].func, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 t[j].smem_bytes);
      if (e != cudaSuccess) return e;
      const int pair = t[j].cta_group == 2;
      if (t[j].smem_bytes > largest[pair]) {
        largest[pair] = t[j].smem_bytes;
        func[pair] = t[j].func;
        threads = t[j].threads;
      }
    }
  }
  d->clusters[0] = d->sm_count;
  for (int i = 1; i < 4; ++i) {
    const int pair = i == 1;     // (a pair and a splitting cluster of two occupy SMs alike)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(d->sm_count >> i << i), 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(largest[pair]);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << i;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&d->clusters[i], func[pair], &cfg);
    if (e != cudaSuccess) return e;
    if (d->clusters[i] > d->sm_count >> i) d->clusters[i] = d->sm_count >> i;
  }
  return cudaSuccess;
}

// The kernels have the same inner loop, so a launch takes about (k-blocks the busiest worker gets)
// x (their cost) + the fill and drain; the smallest estimate wins.
//   * whole tiles: the busiest CTA (or pair) gets ceil(tiles / workers) of them. (Dealing the tiles
//     that do not fill a last wave out along k was built and measured: writing and reading back the
//     fp32 sums of 256 x 256 tiles costs 13-26 us, more than an even share of k saves up to
//     K = 8192.)
//   * a cluster per tile: 1 / split of a tile's k-blocks per wave of clusters, and the exchange.
// No launch is shorter than its operands' way from memory: with few rows this decides, and the
// kernel with the smallest fixed cost that still has enough CTAs on the way wins.
FusedChoice fused_choose(const FusedShape& s, const FusedDevice& d) {
  FusedChoice best = {};
  double best_us = 0.0;
  const bool sym = s.op == kOpGramWide || s.op == kOpGramTall || s.op == kOpPoly;
  const double halves = s.op == kOpGate || s.op == kOpDx ? 2.0 : 1.0;
  const double stream_us = halves * s.K * (s.op == kOpGate ? s.M / 2.0 + s.N : s.op == kOpDw ? 1.5 * s.M + s.N : sym ? s.N : s.M + s.N) *
                           s.zcount * 2.0 / 6.2e6;
  for (const TileCost& c : kTiles) {
    const FusedVariant* kv = fused_find(s.op, c.cta_group, c.block_n, s.dt);
    if (!kv) continue;
    FusedChoice f = {};
    f.kv = kv;
    const int bm = 128 * c.cta_group, bn = s.op == kOpGate ? c.block_n / 2 : c.block_n;
    f.tiles_m = static_cast<int>((s.M + bm - 1) / bm);
    f.tiles_n = static_cast<int>((s.N + bn - 1) / bn);
    f.tiles_per_z = f.tiles_m * f.tiles_n;
    if (sym) {   // fused_tile: 1, 2, 3 .. tiles in each `ratio` tile rows, or 2, 4, 6 .. in a row
      const int ratio = bn / bm, q = ratio ? f.tiles_m / ratio : 0;
      f.tiles_per_z = ratio ? ratio * q * (q + 1) / 2 + f.tiles_m % ratio * (q + 1) : f.tiles_m * (f.tiles_m + 1);
    }
    f.num_kb = static_cast<int>((s.K + 63) / 64);
    const int kbs = f.num_kb * (s.op == kOpDx ? 2 : 1);
    if (s.op == kOpDw) {
      f.tiles_m2 = static_cast<int>((s.N + bm - 1) / bm);
      f.tiles_n2 = static_cast<int>((s.M + bn - 1) / bn);
    }
    const long long tiles = static_cast<long long>(f.tiles_per_z) * s.zcount + f.tiles_m2 * f.tiles_n2;
    for (int split = 1; split <= kv->max_split && split <= kbs; split *= 2) {
      const int ctas = c.cta_group * split;                       // of a cluster
      const long long at_once = d.clusters[ctas == 1 ? 0 : ctas == 2 ? 1 : ctas == 4 ? 2 : 3];
      if (at_once < 1) break;
      const long long waves = (tiles + at_once - 1) / at_once;
      const int part = (kbs + split - 1) / split;
      const double busy = tiles * ctas < d.sm_count ? static_cast<double>(tiles * ctas) / d.sm_count : 1.0;
      const double kb_us = c.alone_us + (c.busy_us - c.alone_us) * busy;
      // a cluster has one tile: from the second wave on every tile pays for its own start and end
      const double fixed = c.fixed_us + (split == 1 ? 0.0 : split == 2 ? 2.1 : 3.0);
      const double tile_us = part * kb_us, epilogue_us = c.epilogue_us * epilogue_weight(s.op);
      double us = split > 1 ? waves * (tile_us + fixed) : waves * (tile_us > epilogue_us ? tile_us : epilogue_us) + fixed;
      // (among kernels that all wait for memory, the one with the most to spare)
      us = (us < stream_us + 4.8 ? stream_us + 4.8 : us) + 0.05 * us;
      if (best.kv && us >= best_us) continue;
      best_us = us;
      best = f;
      best.split = split;
      best.tiles = static_cast<int>(tiles);
      best.at_once = static_cast<int>(at_once);
      best.tile_us = tile_us > epilogue_us ? tile_us : epilogue_us;
      best.grid = static_cast<int>(split > 1 ? tiles : tiles < at_once ? tiles : at_once) * ctas;
    }
  }
  return best;
}

// SMs that the last wave of `before` leaves idle start on kOpDw's tiles that much earlier, and take
// more of them: as many more as let the busiest worker end first. (Backward of 333 x 768 x 2048: 25.6 us
// dealt evenly, 23.9 so; 700 x 4096 x 1000: 59.7, 55.8; 1999 x 2048 x 5461 and longer: within 1 %.)
void fused_deal(const FusedChoice& before, const FusedChoice& dw, const FusedDevice& d, int* head, int* head_tiles) {
  *head = *head_tiles = 0;
  if (dw.split > 1) return;
  const int last = (before.tiles - 1) % before.at_once + 1;
  const int h = (d.sm_count - last * before.kv->cta_group * before.split) / dw.kv->cta_group;
  const int workers = dw.grid / dw.kv->cta_group;
  if (h < 1 || h >= workers) return;
  const double lead = before.tile_us / dw.tile_us;      // in tiles of kOpDw
  double best = 0.0;
  for (int more = 0; more <= lead + 1 && more * h <= dw.tiles; ++more) {
    const int rest = (dw.tiles - more * h + workers - 1) / workers;
    const double end = rest + (more > lead ? more : lead);
    if (more > 0 && end >= best) continue;
    best = end;
    *head = more ? h : 0;
    *head_tiles = more * h;
  }
}

// What bind_device found on each device: asking again costs every new plan the better part of a
// millisecond. (A thread that comes while another one is asking uses its own answer.)
static cudaError_t device_facts(int dev, FusedDevice* d) {
  constexpr int kDevices = 64;
  static std::atomic<int> state[kDevices];      // 0 = not asked, 1 = being written, 2 = known
  static FusedDevice known[kDevices];
  if (dev < kDevices && state[dev].load(std::memory_order_acquire) == 2) {
    *d = known[dev];
    return cudaSuccess;
  }
  cudaError_t e = cudaDeviceGetAttribute(&d->sm_count, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = bind_device(d);
  int expected = 0;
  if (e == cudaSuccess && dev < kDevices && state[dev].compare_exchange_strong(expected, 1)) {
    known[dev] = *d;
    state[dev].store(2, std::memory_order_release);
  }
  return e;
}

int fused_context_create(FusedContext* c) {
  memset(c, 0, sizeof(*c));
  FUSED_CUDA(cudaGetDevice(&c->device));
  int major = 0;
  FUSED_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, c->device));
  if (major != 10) return ROLLER_ERR_DEVICE;
  cudaError_t e = device_facts(c->device, &c->dev);
  if (e == cudaSuccess) e = cudaMalloc(&c->status, sizeof(uint32_t));
  if (e == cudaSuccess) e = zero_now(c->status, sizeof(uint32_t));
  if (e == cudaSuccess) return ROLLER_OK;
  const int rc = e == cudaErrorMemoryAllocation ? ROLLER_ERR_NOMEM : report_cuda_error(e, "plan setup");
  cudaGetLastError();
  fused_context_destroy(c);
  return rc;
}

void fused_context_destroy(FusedContext* c) {
  cudaFree(c->status);
  c->status = nullptr;
}

int fused_context_status(FusedContext* c, uint32_t* device_status) {
  uint32_t h = 0;
  int cur = -1;
  if (cudaGetDevice(&cur) != cudaSuccess || cur != c->device) return ROLLER_ERR_DEVICE;
  FUSED_CUDA(cudaDeviceSynchronize());
  FUSED_CUDA(cudaMemcpy(&h, c->status, sizeof(h), cudaMemcpyDeviceToHost));
  if (device_status) *device_status = h;
  if (h == 0) return ROLLER_OK;
  FUSED_CUDA(zero_now(c->status, sizeof(uint32_t)));
  return ROLLER_ERR_TIMEOUT;
}

}  // namespace rb200
