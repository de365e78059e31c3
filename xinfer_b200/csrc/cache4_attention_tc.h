// Many rows of a key/value head over 4-bit pages, in bfloat16 on tcgen05 (cache4_attention_tc.cu).
#pragma once
#include "cache4_attention.cuh"

namespace xb4 {

// A step whose largest request has TC_ROWS rows of a key/value head has this kernel; in it, requests of fewer than OWN_ROWS are left to the one for few.  Few-row
// kernel / this one (us, 32 heads over 8, up to 4,096 keys): 8 requests of up to 32 rows 34.4 / 34.1, 48 rows 38 / 34.5, 64 rows 45 / 34.8, 96 rows 55 / 36; 32 requests
// of 48 91 / 83; one of 48 at 1,024 keys 18.3 / 20.1.  The 8 requests of 64 took 58 with those below 64 rows left to the other kernel: a second launch reads
// lengths, places and parts again.
constexpr int TC_ROWS = 48, OWN_ROWS = 16;

bool tc_takes(int nh, int nkv, int d, int longest);                // whether it may, for a step's largest request
bool tc_takes(const AttendArgs& A, int longest);
long long tc_scratch(int d);                                       // float32 numbers, on a 16-byte boundary
const int* tc_wide(int d, const float* scratch);                   // where it says which requests it leaves to others (AttendArgs::wide)
int tc_launch(const AttendArgs& A, float* scratch, cudaStream_t stream);

}  // namespace xb4
