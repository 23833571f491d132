#pragma once
#include "common.h"

namespace fa {

// Rows of flash_rotary.  Strides in elements.
struct RotaryArgs {
    const void* X;
    void* Y;
    const void* positions;
    const float* inv_freq;
    int64_t x_batch, x_head, x_row, y_batch, y_head, y_row, positions_batch;
    float factor;
    int B, H, N, d, rot, positions_64, interleaved, inverse, parts;
    FastDiv by_n, by_chunks;  // rows of a batch; chunks of a row
};

// New tokens of flash_append_paged.  Strides in elements.
struct AppendArgs {
    const void *Q, *K, *V, *positions;
    void *O, *K_cache, *V_cache;
    const int32_t *table, *lens, *cu;
    const float* inv_freq;  // nullptr: nothing turns
    int64_t q_token, q_head, o_token, o_head, k_token, k_head, v_token, v_head, kc_page, kc_head, kc_row, vc_page, vc_head, vc_row, table_stride;
    float factor;
    int B, H, Hk, d, rot, tokens, num_pages, page, capacity, positions_64, interleaved, parts;  // H: query heads to turn, 0 for none
    FastDiv by_page, by_chunks, by_copy_chunks;
};

// dtype: FLASH_FP16 / FLASH_BF16 / FLASH_FP32 of the public header; wide: elements that the strides and addresses allow a thread to move at
// once (8, 4 or 1).  The launchers choose a.parts and the divisors.
int launch_rotary(const RotaryArgs& a, int dtype, int wide, hipStream_t st);
int launch_append(const AppendArgs& a, int dtype, hipStream_t st);

}  // namespace fa
