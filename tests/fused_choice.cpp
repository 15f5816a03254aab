// What the host side of the fused products decides, for tests without a GPU: prints the table of compiled
// kernels, then for each problem on standard input (op, type, M, N, K, matrices) the kernel chosen for it.
// argv: SMs, clusters of 2, 4 and 8 CTAs that the device holds at once.
#include <cstdio>
#include <cstdlib>

#include "fused_gemm.h"

using namespace rb200;

int main(int argc, char** argv) {
  if (argc != 5) return 2;
  FusedDevice d;
  d.sm_count = d.clusters[0] = atoi(argv[1]);
  for (int i = 1; i < 4; ++i) d.clusters[i] = atoi(argv[i + 1]);
  const FusedVariant* (*const tables[])(int*) = {fused_variants_bf16, fused_variants_f16, fused_variants_ortho};
  for (auto table : tables) {
    int n = 0;
    const FusedVariant* t = table(&n);
    for (int i = 0; i < n; ++i)
      printf("kernel %d %d %d %d %d\n", t[i].op, t[i].dt, t[i].cta_group, t[i].block_n, t[i].max_split);
  }
  FusedShape s;
  while (scanf("%d %d %lld %lld %lld %d", &s.op, &s.dt, &s.M, &s.N, &s.K, &s.zcount) == 6) {
    const FusedChoice c = fused_choose(s, d);
    printf("%d %d %d %d %d\n", s.op, s.dt, c.kv->cta_group, c.kv->block_n, c.split);
  }
  // the order of launches: nothing is read early, or waited for late, unless the launch before waited
  LaunchOrder o;
  int early = 1, late = 0;
  auto launch = [&](int e, int l) {
    early = e;
    late = l;
    o.next(&early, &late);
    return early * 10 + late;
  };
  printf("order %d", launch(1, 1));        // the first of a call: neither
  printf(" %d", launch(1, 0));             // behind one that waited: as it wants
  printf(" %d", launch(0, 1));
  printf(" %d", launch(1, 1));             // behind a late one: neither, but it waits
  late = 1;
  o.next(nullptr, &late);                  // a late copy
  printf(" %d", late);
  printf(" %d", launch(1, 0));             // behind it: nothing early
  printf(" %d\n", launch(0, 1));
  return 0;
}
