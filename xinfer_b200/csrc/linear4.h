// What the kernels of products with 4-bit weights share (linear4.cu says what they compute).
#pragma once
#include "codes4.cuh"

namespace xb4 {

struct LinearArgs {
    void* out;                     // [tokens, rows], rows `out_stride` elements apart
    const void* x;                 // [tokens, columns], rows `x_stride` elements apart
    const uint8_t* weight;         // [row tiles, column tiles, tile bytes]
    long long out_stride, x_stride;
    int tokens, rows, columns, per_row;      // per_row: groups of a tile's row (4, 2, 1)
    int early;                     // whatever wrote the weight has ended: it may be read before the kernel ahead has
};

int linear4_mma(const LinearArgs& A, cudaStream_t stream);                   // linear4_mma.cu
bool linear4_tc_takes(const LinearArgs& A);                                  // linear4_tc.cu
int linear4_tc(const LinearArgs& A, int* err, cudaStream_t stream);

}  // namespace xb4
