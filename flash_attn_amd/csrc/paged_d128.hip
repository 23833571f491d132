// Instances of the paged attention for 64 < d <= 128, and the merge of its splits.
#include "paged_kernel.h"

namespace fa {
int launch_paged_d128(const PagedArgs& a, bool bf16, int rows, long long blocks, hipStream_t st) { return launch_paged_bucket<128>(a, bf16, rows, blocks, st); }

// Four waves per row where rows are few and splits many: a wave alone would walk them one pair after the other.
int launch_paged_merge(const PagedArgs& p, bool bf16, hipStream_t st)
{
    const PagedMergeArgs a = {p.O, p.LSE, p.O_partial, p.LSE_partial, p.cu, p.o_token, p.o_head, p.B, p.H, p.d, p.tokens, p.num_splits};
    const long long rows = (long long)a.tokens * a.H;
    const bool four = rows <= 4096 && a.num_splits > 8;
    const dim3 grid((unsigned)(four ? rows : (rows + 3) / 4));
    if (four) return (int)(bf16 ? launch_kernel(paged_merge_kernel<true, 4>, grid, dim3(256), 0, st, a) : launch_kernel(paged_merge_kernel<false, 4>, grid, dim3(256), 0, st, a));
    return (int)(bf16 ? launch_kernel(paged_merge_kernel<true, 1>, grid, dim3(256), 0, st, a) : launch_kernel(paged_merge_kernel<false, 1>, grid, dim3(256), 0, st, a));
}
}  // namespace fa
