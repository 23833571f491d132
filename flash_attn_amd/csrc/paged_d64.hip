// Instances of the paged attention for d <= 64.
#include "paged_kernel.h"

namespace fa {
int launch_paged_d64(const PagedArgs& a, bool bf16, int rows, long long blocks, hipStream_t st) { return launch_paged_bucket<64>(a, bf16, rows, blocks, st); }
}  // namespace fa
