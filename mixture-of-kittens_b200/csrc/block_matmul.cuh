// The 8-bit block-scaled product (block_matmul.cu) and its form for a few rows (block_matmul_few.cu).
#pragma once

#include "mok_common.cuh"

namespace mok {

struct BlockProduct {
    const uint8_t *a, *b;
    long long a_stride, b_stride;
    const float *sa, *sb;
    long long sa_row, sa_block, sb_row, sb_block;
    int b_tile_rows;   // 1 or 128
    int rows, cols, depth;
    bf16* out;
    long long out_stride;
    uint32_t* status;
};

// Most rows of A that the form for a few rows takes.
constexpr int kFewRows = 24;
int launch_block_matmul_few(const BlockProduct& p, cudaStream_t stream);

}  // namespace mok
