// Instances of the paged attention with a bias by distance.
#include "paged_kernel.h"

namespace fa {
int launch_scored_sloped(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st)
{
    return launch_scored_kind<kScoresSloped>(a, bf16, rows, blocks, st);
}
}  // namespace fa
