// Many rows of a key/value head over 4-bit pages, in bfloat16 on tcgen05 (cache4_attention_tc.cu).
#pragma once
#include "cache4_attention.cuh"

namespace xb4 {

constexpr int TC_ROWS = 64;        // from so many rows of a request's key/value head on

bool tc_takes(int nh, int nkv, int d, int longest);                // whether it may, for a step's largest request
bool tc_takes(const AttendArgs& A, int longest);
long long tc_scratch(int d);                                       // float32 numbers, on a 16-byte boundary
int tc_launch(const AttendArgs& A, float* scratch, cudaStream_t stream);

}  // namespace xb4
