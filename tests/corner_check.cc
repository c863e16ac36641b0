// Reads rel0, a sequence's own position and a step, answers each three with the relative position that the kernels go on from.
#include <inttypes.h>
#include <stdio.h>

#include "../ps-lite_amd/csrc/relbias.h"

int main() {
  int64_t rel0, own, step;
  while (scanf("%" SCNd64 "%" SCNd64 "%" SCNd64, &rel0, &own, &step) == 3) printf("%d\n", pskv::nearer(rel0, own, step));
  return 0;
}
