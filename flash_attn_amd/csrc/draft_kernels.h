#pragma once
#include "common.h"

namespace fa {

// Parents of drafted tokens -> masks and positions (flash_tree_mask)
struct TreeMaskArgs {
    const int32_t *parents, *cu, *lens;  // lens: nullptr where positions count from the chunk's begin
    uint64_t* mask;
    int32_t* positions;  // or nullptr
    int64_t mask_stride;
    int B, tokens, words;
};

// Accepted rows to their places (flash_keep_paged).  Strides in bytes.
struct KeepArgs {
    const int32_t *table, *lens, *cu, *path, *accepted;
    int32_t* lens_out;
    char *K, *V;
    int64_t k_layer, k_page, k_head, k_row, v_layer, v_page, v_head, v_row, table_stride, path_stride;
    int B, layers, Hk, d, num_pages, page, capacity, most, parts;  // most: entries of a row of path; parts: work-groups of a sequence and layer
    FastDiv by_page, by_pieces, by_parts, by_b;
};

int launch_tree_mask(const TreeMaskArgs& a, hipStream_t st);
int launch_keep(const KeepArgs& a, hipStream_t st);  // chooses a.parts and the divisors

}  // namespace fa
