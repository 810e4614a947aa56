// CPU check of the sampling kernel's layout of a row: for every vocabulary,
// number of rows that changes the cluster, element size and start of a row,
// the CTAs' and warps' parts cover the row once, and the steps of a part fit
// the sums that the draw keeps of them.  Exit status 0 when all hold.
#include <algorithm>
#include <cstdio>

#include "sample_plan.h"

using namespace walsh;

int main() {
  const int rows_of[] = {1, 18, 19, 36, 37, 73, 74, 147, 148, 100000};
  int most = 0, failures = 0;
  for (int vec = 4; vec <= 8; vec *= 2)
    for (int vocab = 1; vocab <= kSampleMaxVocab; ++vocab)
      for (int rows : rows_of)
        for (int mis = 0; mis < vec; ++mis) {
          const int cs = sample_cluster(rows, vocab);
          const int chunks = sample_chunks(vocab, mis, vec), per_cta = sample_cta_chunks(chunks, cs);
          const int per_warp = sample_warp_chunks(per_cta);
          const int steps = sample_steps(std::min(per_warp, per_cta));
          most = std::max(most, steps);
          if (steps > kSampleSteps || (int64_t)per_cta * cs < chunks || (int64_t)per_warp * kSampleWarps < per_cta ||
              (int64_t)chunks * vec < mis + vocab) {
            if (failures++ < 10)
              std::printf("FAILED vec %d vocab %d rows %d start %d: %d steps of %d\n", vec, vocab, rows, mis, steps, kSampleSteps);
          }
        }
  if (most != kSampleSteps) std::printf("FAILED: the longest part has %d steps, not %d\n", most, kSampleSteps), ++failures;
  if (failures) return 1;
  std::printf("sample_plan ok\n");
  return 0;
}
