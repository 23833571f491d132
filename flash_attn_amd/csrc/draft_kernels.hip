// Drafted tokens around the paged attention: masks and positions of a tree from its tokens' parents (flash_tree_mask), and the rows of the accepted path
// to their places in the cache (flash_keep_paged).  Both are short launches, bound by the chain of loads that they begin with and by the host's call.
#include "draft_kernels.h"

namespace fa {
namespace {

// ---- masks
//
// mask(i) = bit i | mask(parent(i)).  Pointers double: mask(i) |= mask(up(i)), up(i) = up(up(i)), so that a path of n tokens takes log2 n rounds in
// LDS, whose two halves take turns: one barrier a round.  A thread per token that the mask can name, a work-group per sequence: of 64 tokens it is one
// wave, whose barriers cost nothing.
template <int W>
__global__ void __launch_bounds__(64 * W) tree_mask_kernel(const TreeMaskArgs a)
{
    constexpr int kTokens = 64 * W;
    __shared__ uint64_t words[2][W][kTokens];
    __shared__ int up[2][kTokens];
    const int b = blockIdx.x, i = threadIdx.x;
    int c0 = a.cu[b], c1 = a.cu[b + 1], len = a.lens ? a.lens[b] : 0;
    c0 = c0 < 0 ? 0 : c0 > a.tokens ? a.tokens : c0;
    c1 = c1 < c0 ? c0 : c1 > a.tokens ? a.tokens : c1;
    const int n = c1 - c0, base = a.lens ? (int)((uint32_t)len - (uint32_t)n) : 0;
    const bool mine = i < n;
    int p = mine ? a.parents[c0 + i] : -1;
    if (p >= i || p < 0) p = -1;  // a parent stands in front of its children
    uint64_t w[W];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = i >> 6 == k ? 1ull << (i & 63) : 0ull;
    int half = 0;
    for (int reach = 1; reach < min(n, kTokens); reach *= 2) {  // paths of so many tokens are complete
#pragma unroll
        for (int k = 0; k < W; ++k) words[half][k][i] = w[k];
        up[half][i] = p;
        __syncthreads();
        if (p >= 0) {
#pragma unroll
            for (int k = 0; k < W; ++k) w[k] |= words[half][k][p];
            p = up[half][p];
        }
        half ^= 1;
    }
    if (mine) {
        int depth = -1;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            a.mask[(int64_t)(c0 + i) * a.mask_stride + k] = w[k];
            depth += __builtin_popcountll(w[k]);
        }
        if (a.positions) a.positions[c0 + i] = base + depth;
    }
    // tokens that the mask has no bits for
    for (int j = i + kTokens; j < n; j += kTokens) {
        for (int k = 0; k < W; ++k) a.mask[(int64_t)(c0 + j) * a.mask_stride + k] = 0;
        if (a.positions) a.positions[c0 + j] = base;
    }
}

// ---- accepted rows
//
// Row path[i] of the chunk goes to its row i.  Paths grow, so path[i] >= i, and a thread that walks the rows of its own 16 bytes of a head in this
// order writes no row that it has yet to read: kAhead rows are read, then written.  No thread reads what another one writes.
constexpr int kAhead = 8;

__global__ void __launch_bounds__(256) keep_kernel(const KeepArgs a)
{
    const int lane = threadIdx.x & 63, group = blockIdx.x;
    const int unit = a.by_parts.quotient(group), part = group - unit * a.parts;
    const int layer = a.by_b.quotient(unit), b = unit - layer * a.B;
    const int n = (int)max((int64_t)0, min((int64_t)a.cu[b + 1] - a.cu[b], (int64_t)1 << 30));
    int len = a.lens[b], want = a.accepted[b];
    int p = lane < a.most ? a.path[(int64_t)b * a.path_stride + lane] : -1;  // (asked for together with them)
    len = len < 0 ? 0 : len > a.capacity ? a.capacity : len;
    want = want < 0 ? 0 : want > a.most ? a.most : want;
    const int base = len - n;

    const int pieces = a.d / 8, half = a.Hk * pieces;
    const int column = part * 256 + threadIdx.x;
    const bool is_v = column >= half;
    const int c = is_v ? column - half : column, h = a.by_pieces.quotient(c), x = c - h * pieces;
    char* const at = is_v ? a.V + layer * a.v_layer + h * a.v_head + x * 16 : a.K + layer * a.k_layer + h * a.k_head + x * 16;
    const int64_t page_bytes = is_v ? a.v_page : a.k_page, row_bytes = is_v ? a.v_row : a.k_row;
    const bool moves = column < 2 * half;

    int kept = 0, last = -1;
    for (int i0 = 0; i0 < want; i0 += 64) {
        // a lane per entry of the path: how far it grows, and where its rows lie
        const int i = i0 + lane;
        if (i0 > 0) p = i < want ? a.path[(int64_t)b * a.path_stride + i] : -1;
        int before = __shfl_up(p, 1);
        if (lane == 0) before = last;
        const uint64_t bad = __builtin_amdgcn_ballot_w64(!(i < want && p > before && p < n));
        const int good = bad ? __builtin_ctzll(bad) : 64;
        int from = -1, to = -1, from_row = 0, to_row = 0;  // pages
        const int64_t s = (int64_t)base + p, t = (int64_t)base + i;
        if (lane < good && p != i && t >= 0 && s < a.capacity) {  // (t < s)
            const int sp = a.by_page.quotient((int)s), tp = a.by_page.quotient((int)t);
            from_row = (int)s - sp * a.page, to_row = (int)t - tp * a.page;
            from = a.table[b * a.table_stride + sp], to = a.table[b * a.table_stride + tp];
            if ((uint32_t)from >= (uint32_t)a.num_pages || (uint32_t)to >= (uint32_t)a.num_pages) from = -1;
        }
        for (int k0 = 0; k0 < good; k0 += kAhead) {
            v4u row[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int e = k0 + k;  // (below 64)
                const int pg = __builtin_amdgcn_readlane(from, e), r = __builtin_amdgcn_readlane(from_row, e);
                if (pg >= 0 && moves) row[k] = *reinterpret_cast<const v4u*>(at + pg * page_bytes + r * row_bytes);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int e = k0 + k;
                const int pg = __builtin_amdgcn_readlane(to, e), r = __builtin_amdgcn_readlane(to_row, e);
                if (__builtin_amdgcn_readlane(from, e) >= 0 && moves) *reinterpret_cast<v4u*>(at + pg * page_bytes + r * row_bytes) = row[k];
            }
        }
        kept = i0 + good;
        if (good < 64) break;
        last = __builtin_amdgcn_readlane(p, 63);
    }
    if (layer == 0 && part == 0 && threadIdx.x == 0) a.lens_out[b] = max(base + kept, 0);
}

}  // namespace

int launch_tree_mask(const TreeMaskArgs& a, hipStream_t st)
{
    const auto kern = a.words == 1 ? tree_mask_kernel<1> : a.words == 2 ? tree_mask_kernel<2> : a.words == 3 ? tree_mask_kernel<3> : tree_mask_kernel<4>;
    return (int)launch_kernel(kern, dim3((unsigned)a.B), dim3(64 * a.words), 0, st, a);
}

int launch_keep(const KeepArgs& p, hipStream_t st)
{
    KeepArgs a = p;
    const int pieces = a.d / 8;
    a.parts = (2 * a.Hk * pieces + 255) / 256;
    a.by_page = fast_div(a.page), a.by_pieces = fast_div(pieces), a.by_parts = fast_div(a.parts), a.by_b = fast_div(a.B);
    return (int)launch_kernel(keep_kernel, dim3((unsigned)((long long)a.parts * a.B * a.layers)), dim3(256), 0, st, a);
}

}  // namespace fa
