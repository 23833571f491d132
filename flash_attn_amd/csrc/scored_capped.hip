// Instances of the paged attention with scores capped by a tanh.
#include "paged_kernel.h"

namespace fa {
int launch_scored_capped(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st)
{
    return launch_scored_kind<kScoresCapped>(a, bf16, rows, blocks, st);
}
}  // namespace fa
