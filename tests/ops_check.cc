// Host checks of what the operators on rows decide on the CPU. Reads lines, answers each with one line:
//   overlap at_a n k stride size  at_b n k stride size      0 or 1
//   border buckets max two_sided                            the borders of the buckets that widen
//   philox c0 c1 c2 c3 k0 k1                                four words
#include <inttypes.h>
#include <stdio.h>
#include <string.h>

#include "../ps-lite_amd/csrc/philox.h"
#include "../ps-lite_amd/csrc/relbias.h"
#include "../ps-lite_amd/csrc/row_span.h"

using namespace pskv;

int main() {
  char what[16];
  while (scanf("%15s", what) == 1) {
    if (!strcmp(what, "overlap")) {
      uint64_t x[10];
      for (uint64_t& v : x)
        if (scanf("%" SCNu64, &v) != 1) return 1;
      const RowSpan a{reinterpret_cast<void*>(x[0]), x[1], x[2], x[3], x[4]}, b{reinterpret_cast<void*>(x[5]), x[6], x[7], x[8], x[9]};
      printf("%d\n", rows_overlap(a, b) ? 1 : 0);
    } else if (!strcmp(what, "border")) {
      uint64_t buckets, far, sides;
      if (scanf("%" SCNu64 "%" SCNu64 "%" SCNu64, &buckets, &far, &sides) != 3) return 1;
      Buckets b;
      if (!make_buckets(&b, buckets, far, sides != 0)) {
        printf("refused\n");
        continue;
      }
      for (unsigned c = 1; c <= b.steps; ++c) printf("%u ", b.border[c]);
      printf("\n");
    } else if (!strcmp(what, "philox")) {
      uint32_t x[6];
      for (uint32_t& v : x)
        if (scanf("%" SCNx32, &v) != 1) return 1;
      const Drawn d = philox(x[0], x[1], x[2], x[3], x[4], x[5]);
      printf("%08x %08x %08x %08x\n", d.word[0], d.word[1], d.word[2], d.word[3]);
    } else {
      return 1;
    }
  }
  return 0;
}
