// Products of a step's rows with a weight in 4 bits: y[t, n] = sum_k x[t, k] (m + s code)[n, k], groups of 32, 64 or 128 columns (codes4.cuh).
//
// The weight lies in tiles of 16 rows and 128 columns, a tile's bytes together: 1,024 bytes of codes, then per row the words of its groups.
// Lane 4 g + t of a warp has rows g and g + 8 (two pieces of 16 bytes, 512 bytes apart) and in them the columns 32 j + 8 t + e of word j: as an
// MMA's lanes take them, each word's columns in one group whatever the group's size.  Column e of a word lies in its half byte 4 (e & 1) +
// e / 2, so that a mask takes out a pair of neighbours.  Rows and columns beyond the weight have codes and words of zeros.
//
// Three kernels: bfloat16 of up to 8 rows, up to 16 with small weights, and of any number off 16-byte boundaries, linear4_mma.cu; of more, linear4_tc.cu; float32
// the one below.
#include "linear4.h"

namespace {

using namespace xb4;

// float32: a block per tile of rows and eight tokens, its warps take the column tiles in turn.  Products and sums in float32.  Few blocks of few trips:
// five rows, 1,000 columns, 777 rows of the weight 5.8 us, a chain of codes, x, sums and launch.
constexpr int F32_WARPS = 8, F32_TOKENS = 8;

__global__ void __launch_bounds__(F32_WARPS * 32)
linear4_f32_kernel(const LinearArgs A) {
    __shared__ float part[F32_WARPS][F32_TOKENS][TILE_ROWS];
    pdl_overlap_few();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int col_tiles = (A.columns + TILE_COLS - 1) / TILE_COLS, tile_bytes = TILE_CODES + TILE_ROWS * A.per_row * 4;
    const int t0 = blockIdx.y * F32_TOKENS, many = min(F32_TOKENS, A.tokens - t0);
    const uint8_t* line = A.weight + (long long)blockIdx.x * col_tiles * tile_bytes;
    const float* x = static_cast<const float*>(A.x) + t0 * A.x_stride;
    float acc[F32_TOKENS][2] = {};
    for (int ct = warp; ct < col_tiles; ct += F32_WARPS) {
        const uint8_t* tile = line + (long long)ct * tile_bytes;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(tile + TILE_CODES);
        const uint4 a = reinterpret_cast<const uint4*>(tile)[lane], b = reinterpret_cast<const uint4*>(tile)[32 + lane];
        const uint32_t lo[4] = {a.x, a.y, a.z, a.w}, hi[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int grp = j * A.per_row / 4;
            const uint32_t wlo = words[g * A.per_row + grp], whi = words[(g + 8) * A.per_row + grp];
            const int c0 = ct * TILE_COLS + j * 32 + t * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (c0 + e >= A.columns) break;
                const int shift = 4 * ((e & 1) * 4 + e / 2);
                const float w0 = value_of((lo[j] >> shift) & 15, wlo), w1 = value_of((hi[j] >> shift) & 15, whi);
#pragma unroll
                for (int i = 0; i < F32_TOKENS; ++i)
                    if (i < many) {
                        const float v = x[i * A.x_stride + c0 + e];
                        acc[i][0] = fmaf(v, w0, acc[i][0]);
                        acc[i][1] = fmaf(v, w1, acc[i][1]);
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < F32_TOKENS; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float v = acc[i][r];
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            if (t == 0) part[warp][i][g + 8 * r] = v;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < many * TILE_ROWS; i += F32_WARPS * 32) {
        const int tok = i / TILE_ROWS, row = i % TILE_ROWS, n = blockIdx.x * TILE_ROWS + row;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < F32_WARPS; ++w) v += part[w][tok][row];
        if (n < A.rows) static_cast<float*>(A.out)[(t0 + tok) * A.out_stride + n] = v;
    }
}

int launch_f32(const LinearArgs& A, cudaStream_t stream) {
    const dim3 grid((A.rows + TILE_ROWS - 1) / TILE_ROWS, (A.tokens + F32_TOKENS - 1) / F32_TOKENS);
    return xb_launch_few(linear4_f32_kernel, grid, dim3(F32_WARPS * 32), 0, stream, A);
}

}  // namespace

static int linear4(int dtype, void* out, const void* x, const uint8_t* weight, long long out_stride, long long x_stride, int tokens, int rows, int columns,
                   int group, int early, int* err, cudaStream_t stream) {
    if (tokens <= 0 || rows <= 0) return 0;
    if (columns < 1 || (group != 32 && group != 64 && group != 128) || tokens > 65535 * F32_TOKENS) return (int)cudaErrorInvalidValue;
    const LinearArgs A{out, x, weight, out_stride, x_stride, tokens, rows, columns, TILE_COLS / group, early};
    if (dtype == XB_F32) return launch_f32(A, stream);
    // Few rows (us, few-row kernel / many-row kernel, the weight ready): 8 rows of 4,096 x 24,576 15.1 / 23.0, 9 rows 25.5 / 23.1, 16 rows of it 27.4 / 22.9, of 12,288 x 4,096
    // 14.4 / 11.2, of 2,048 x 2,048 5.0 / 4.1, but of 1,024 x 1,024 3.1 / 3.9; 17 of that 4,096 x 24,576 47 / 23, of 4,096 x 4,096 9.3 / 7.1.
    const bool many = A.tokens > 16 || (A.tokens > 8 && (long long)A.rows * A.columns > 1 << 20);
    return many && linear4_tc_takes(A) ? linear4_tc(A, err, stream) : linear4_mma(A, stream);
}
XB_EXPORT int xb_linear4(const long long* words, int n) { return xb_by_words(linear4, words, n); }
