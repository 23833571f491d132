// Instances of the paged attention with a prefix, or a tree of drafted tokens, and nothing else.
#include "paged_kernel.h"

namespace fa {
int launch_scored_masked(const ScoredArgs& a, bool bf16, int rows, long long blocks, hipStream_t st)
{
    return launch_scored_kind<kScoresMasked>(a, bf16, rows, blocks, st);
}
}  // namespace fa
