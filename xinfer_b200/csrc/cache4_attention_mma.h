// Few rows of a key/value head over 4-bit pages, in bfloat16 (cache4_attention_mma.cu).
#pragma once
#include "cache4_attention.cuh"

namespace xb4 {

bool mma_takes(int d);                        // whether it has a form for such heads
bool mma_takes(const AttendArgs& A);
// `rows`: of the request that has most, as far as it is known (TC_ROWS of more)
long long mma_scratch(int d, int rows);        // float32 numbers, on a 16-byte boundary
int mma_launch(const AttendArgs& A, int rows, float* scratch, cudaStream_t stream);

}  // namespace xb4
