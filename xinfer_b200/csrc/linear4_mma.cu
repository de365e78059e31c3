// Products of few rows (16 at a time) with a weight in 4 bits, in bfloat16 on matrix units (linear4.cu says what is computed and how a weight lies).
//
// The weight's rows are the rows of the products, the tokens their columns.  The bits c of a code under a mask of four bits are the bfloat16
// c 2^-133, in the next four bits 16 c 2^-133: a word of eight codes becomes eight operands by one shift and four masks, and nothing is subtracted.
// Every warp scales each token's x by a power of two (and by a 16th of it in front of the 16-fold codes), by which its sums are divided before they meet the others', so
// that they are ordinary float32 numbers whatever x's size is: the largest number of its first columns that are not all zero goes to 2^90 .. 2^91 (by 2^127 at
// most).  Where a later one is more than 2^37 above it a product is not finite, and such a sum is formed again number by number.  (Eight rows of 4,096 x 24,576 take
// 15.1 us, with one power for all 14.6, looking for the largest number of every 128 columns 16.0.)  Per group of columns
//   y += s (code . x) + m sum(x),   sum(x) by a product of the same x with ones; both in float32.
//
// Bound by reading the weight once.  A block's warps and the blocks of a cluster take a range of the columns each, for R tiles of rows at a time, and walk
// over the rows' tiles; the codes are fetched two or four stages ahead, over the ends of the rows' tiles too (where the caller says that the weight is
// complete, the first ones before the kernel in front has ended: 5.2 us instead of 6.1 for 4,096 x 6,144 and one row).  Sums meet in shared memory, warp by
// warp and block by block in their order.
#include "linear4.h"

namespace {

using namespace xb4;

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u, ONES = 0x00010001u, ONES16 = 0x00100010u;      // ones of the scale of the codes
constexpr int X_TOP = 90, UP_MOST = 127;   // where a token's largest number goes, and the largest power of two in bfloat16

constexpr int SLOTS = 2 * 148;             // blocks that the processors hold
__host__ __device__ constexpr int stages(int r) { return r == 4 ? 2 : 4; }
__host__ __device__ constexpr int tile_bytes(int per) { return TILE_CODES + TILE_ROWS * per * 4; }
__host__ __device__ constexpr int sums_stride(int r) { return r * TILE_ROWS + 4; }
__host__ __device__ constexpr int ring_bytes(int r, int per) { return WARPS * stages(r) * r * tile_bytes(per); }
__host__ __device__ constexpr int smem_bytes(int nt, int r, int per) { return ring_bytes(r, per) + WARPS * nt * 8 * sums_stride(r) * 4; }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// The larger sizes of two pairs of numbers, whatever their signs; one that is no number wins.
__device__ __forceinline__ uint32_t max_sizes(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }       // -126 <= e <= 127
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float of_rank(uint32_t addr, uint32_t rank) {
    uint32_t remote;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote));
    return v;
}

// The sum of a token and a row of the weight, whose first tile `tile` is, number by number.
template <int PER>
__device__ __noinline__ float sum_by_number(const __nv_bfloat16* x, const uint8_t* tile, int row, int columns) {
    float sum = 0.f;
    for (int c0 = 0; c0 < columns && fabsf(sum) < INFINITY; c0 += TILE_COLS, tile += tile_bytes(PER)) {       // (what is not finite stays so)
        float of_tile = 0.f;
#pragma unroll 1
        for (int c = 0; c < min(TILE_COLS, columns - c0); ++c) {
            const uint32_t codes = reinterpret_cast<const uint32_t*>(tile)[row * 16 + c % 32 / 8 * 4 + c / 32];
            const int half = (c & 1) * 4 + (c & 7) / 2;                                            // (the half byte of the word)
            of_tile = fmaf(__bfloat162float(x[c0 + c]), value_of(codes >> 4 * half & 15u, reinterpret_cast<const uint32_t*>(tile + TILE_CODES)[row * PER + c * PER / TILE_COLS]), of_tile);
        }
        sum += of_tile;
    }
    return sum;
}

template <int NT, int R, int PER>
__global__ void __launch_bounds__(THREADS, 2)
linear4_mma_kernel(const LinearArgs A, int cluster) {
    extern __shared__ __align__(128) char mem[];
    constexpr int STAGES = stages(R), TILE = tile_bytes(PER), JOIN = 4 / PER;       // JOIN: words of a row's group
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int row_tiles = (A.rows + TILE_ROWS - 1) / TILE_ROWS, col_tiles = (A.columns + TILE_COLS - 1) / TILE_COLS;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0, parts = cluster * WARPS, part = rank * WARPS + warp;
    const int from = (int)((long long)col_tiles * part / parts), to = (int)((long long)col_tiles * (part + 1) / parts);
    const int first = (int)blockIdx.x / cluster * R, stride = (int)gridDim.x / cluster * R;       // row tiles
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(mem) + warp * STAGES * R * TILE;
    const int t0 = blockIdx.y * NT * 8, many = min(NT * 8, A.tokens - t0);

    int put = from, put_row = first, put_slot = 0, take_slot = 0;
    const uint8_t* src[R];                                     // the next tile of each row of tiles
    auto to_row = [&]() {
#pragma unroll
        for (int r = 0; r < R; ++r)                            // (behind the weight's rows: the last one's again, nobody stores what comes of them)
            src[r] = A.weight + ((long long)min(put_row + r, row_tiles - 1) * col_tiles + from) * TILE + lane * 16;
    };
    to_row();
    auto fetch = [&]() {
        if (put < to && put_row < row_tiles) {
            const uint32_t dst = ring + put_slot * R * TILE + lane * 16;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                copy16(dst + r * TILE, src[r]);
                copy16(dst + r * TILE + 512, src[r] + 512);
                if (lane < PER * 4) copy16(dst + r * TILE + 1024, src[r] + 1024);
                src[r] += TILE;
            }
            if (++put == to) {
                put = from;
                put_row += stride;
                to_row();
            }
        }
        commit();
        put_slot = put_slot + 1 == STAGES ? 0 : put_slot + 1;
    };
    if (!A.early) pdl_wait();
#pragma unroll
    for (int i = 0; i < STAGES; ++i) fetch();
    pdl_launch_dependents();
    pdl_wait();

    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(A.x) + t0 * A.x_stride;
    const bool on16 = ((uintptr_t)A.x & 15) == 0 && A.x_stride % 8 == 0;
    // columns c .. c + 7 of the lane's token of column tile n of the products, some of them beyond the matrix or off 16 bytes
    auto load_x = [&](int n, int c) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (n * 8 + g < many) {
            const uint16_t* row = reinterpret_cast<const uint16_t*>(x) + (n * 8 + g) * A.x_stride;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < A.columns) w[e / 2] |= (uint32_t)row[c + e] << (16 * (e & 1));
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    const uint4* x16[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x16[n] = reinterpret_cast<const uint4*>(x + min(n * 8 + g, many - 1) * A.x_stride + t * 8);       // (columns without a token repeat the last one)

    auto x_of = [&](int ct, uint4 (&xv)[NT][4]) {
        if (on16 && (ct + 1) * TILE_COLS <= A.columns) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n) xv[n][j] = x16[n][ct * (TILE_COLS / 8) + j * 4];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n) xv[n][j] = load_x(n, ct * TILE_COLS + j * 32 + t * 8);
        }
    };
    uint32_t up[NT];                                           // the power of two of the lane's token, twice
#pragma unroll
    for (int n = 0; n < NT; ++n) up[n] = (127 + UP_MOST) * 0x00800080u;
    auto power_of = [&](int n) { return (int)(up[n] >> 23) - 127; };
    unsigned known = 0;                                        // tokens that have theirs: those whose columns so far are not all zero
    bool settled = false;
    for (int rt0 = first; rt0 < row_tiles; rt0 += stride) {
    float acc[R][NT][4] = {};
    for (int ct = from; ct < to; ++ct) {
        uint4 xv[NT][4];
        x_of(ct, xv);                                          // (asked for before the codes are waited for)
        if (!settled) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) top = max_sizes(top, max_sizes(max_sizes(xv[n][j].x, xv[n][j].y), max_sizes(xv[n][j].z, xv[n][j].w)));
                top = max_sizes(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max_sizes(top, __shfl_xor_sync(0xffffffffu, top, 2)) & 0x7fff7fffu;
                const int size = (int)max(top & 0xffffu, top >> 16);             // (sizes of bfloat16 numbers compare as whole numbers)
                if (size > 0 && !(known >> n & 1)) up[n] = (uint32_t)min(X_TOP + 254 - (size >> 7), 127 + UP_MOST) * 0x00800080u;
                known |= (size > 0 || n * 8 + g >= many ? 1u : 0u) << n;
            }
            settled = __all_sync(0xffffffffu, known == (1u << NT) - 1);
        }
        wait_but<STAGES - 1>();
        __syncwarp();
        const uint32_t at = ring + take_slot * R * TILE;
        take_slot = take_slot + 1 == STAGES ? 0 : take_slot + 1;
        float d[R][NT][4], ones[NT][4];
        uint4 lo[R], hi[R];
#pragma unroll
        for (int r = 0; r < R; ++r) lo[r] = shared16(at + r * TILE + lane * 16), hi[r] = shared16(at + r * TILE + 512 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j % JOIN == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ones[n][e] = 0.f;
#pragma unroll
                        for (int r = 0; r < R; ++r) d[r][n][e] = 0.f;
                    }
            }
            uint32_t b[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 v = xv[n][j];
                const uint32_t up16 = up[n] - 4 * 0x00800080u;
                b[n][0] = times(v.x, up[n]), b[n][1] = times(v.y, up16), b[n][2] = times(v.z, up[n]), b[n][3] = times(v.w, up16);
                mma(ones[n], ONES, ONES, ONES16, ONES16, b[n][0], b[n][1]);
                mma(ones[n], ONES, ONES, ONES16, ONES16, b[n][2], b[n][3]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t u = j == 0 ? lo[r].x : (j == 1 ? lo[r].y : (j == 2 ? lo[r].z : lo[r].w)), v = j == 0 ? hi[r].x : (j == 1 ? hi[r].y : (j == 2 ? hi[r].z : hi[r].w));
                const uint32_t u8 = u >> 8, v8 = v >> 8;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma(d[r][n], u & LOW, v & LOW, u & HIGH, v & HIGH, b[n][0], b[n][1]);
                    mma(d[r][n], u8 & LOW, v8 & LOW, u8 & HIGH, v8 & HIGH, b[n][2], b[n][3]);
                }
            }
            if (j % JOIN == JOIN - 1) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    uint32_t wl, wh;
                    const uint32_t words = at + r * TILE + TILE_CODES + (g * PER + j / JOIN) * 4;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(wl) : "r"(words) : "memory");
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(wh) : "r"(words + 8 * PER * 4) : "memory");
                    const float sl = scale_of(wl), ml = least_of(wl), sh = scale_of(wh), mh = least_of(wh);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        acc[r][n][0] = fmaf(sl, d[r][n][0], fmaf(ml, ones[n][0], acc[r][n][0]));
                        acc[r][n][1] = fmaf(sl, d[r][n][1], fmaf(ml, ones[n][1], acc[r][n][1]));
                        acc[r][n][2] = fmaf(sh, d[r][n][2], fmaf(mh, ones[n][0], acc[r][n][2]));
                        acc[r][n][3] = fmaf(sh, d[r][n][3], fmaf(mh, ones[n][1], acc[r][n][3]));
                    }
                }
            }
        }
        __syncwarp();                                          // (the stage has been read: the next codes may come)
        fetch();
    }
    // ---- sums: [warp][token][row]
    constexpr int STRIDE = sums_stride(R), ROWS = R * TILE_ROWS;
    float* sums = reinterpret_cast<float*>(mem + ring_bytes(R, PER));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // (6 to 171, in two steps that both go up: nothing is lost or too large on the way)
            const int of = 133 - __shfl_sync(0xffffffffu, power_of(n), (2 * t + e) * 4);
            const float half = power_of_two(of / 2), rest = power_of_two(of - of / 2);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h) sums[(warp * NT * 8 + n * 8 + 2 * t + e) * STRIDE + r * TILE_ROWS + g + 8 * h] = acc[r][n][2 * h + e] * half * rest;
        }
    __syncthreads();
    const int n0 = rt0 * TILE_ROWS, total = many * ROWS;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out);
    auto store = [&](int token, int row, float v) {
        if (n0 + row >= A.rows) return;
        if (!(fabsf(v) < INFINITY)) v = sum_by_number<PER>(x + token * A.x_stride, A.weight + (long long)(rt0 + row / TILE_ROWS) * col_tiles * TILE, row % TILE_ROWS, A.columns);
        out[(t0 + token) * A.out_stride + n0 + row] = __float2bfloat16_rn(v);
    };
    for (int i = threadIdx.x; i < total; i += THREADS) {
        const int token = i / ROWS, row = i % ROWS;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += sums[(w * NT * 8 + token) * STRIDE + row];
        if (cluster > 1) sums[token * STRIDE + row] = v;
        else store(token, row, v);
    }
    if (cluster > 1) {
        cluster_sync();
        const uint32_t base = (uint32_t)__cvta_generic_to_shared(sums);
        for (int i = total * rank / cluster + (int)threadIdx.x; i < total * (rank + 1) / cluster; i += THREADS) {
            const int token = i / ROWS, row = i % ROWS;
            float v = 0.f;
            for (int k = 0; k < cluster; ++k) v += of_rank(base + (token * STRIDE + row) * 4, k);
            store(token, row, v);
        }
        cluster_sync();                                        // (nobody leaves, or forms other sums, while its sums are read)
    } else {
        __syncthreads();
    }
    }
    wait_but<0>();
}

template <int NT, int R, int PER>
int launch(const LinearArgs& A, cudaStream_t stream) {
    constexpr int smem = smem_bytes(NT, R, PER);
    const int groups = ((A.rows + TILE_ROWS - 1) / TILE_ROWS + R - 1) / R, col_tiles = (A.columns + TILE_COLS - 1) / TILE_COLS, blocks_y = (A.tokens + NT * 8 - 1) / (NT * 8);
    // Columns are shared out among a cluster's blocks while all blocks are on the processors at once and a warp has two tiles.  Measured with one, two,
    // four and eight blocks (the weight ready): 4,096 x 4,096 (one row) 4.8, 4.8, 7.2, 15.7 us; 12,288 columns 11.9, 8.4, 10.9, 21.4; 4,096 x 6,144 5.1, 7.7, 11.7, 23.7.
    int cluster = 1;
    while (cluster < 8 && (long long)groups * blocks_y * cluster * 2 <= SLOTS && col_tiles >= 2 * WARPS * cluster) cluster *= 2;
    const int most = SLOTS / cluster / blocks_y, wide = groups < most ? groups : (most < 1 ? 1 : most);
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(linear4_mma_kernel<NT, R, PER>, smem, &roomy)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(wide * cluster, blocks_y);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = xb_pdl_enabled() ? 2 : 1;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, linear4_mma_kernel<NT, R, PER>, A, cluster);
    return rc != cudaSuccess ? (int)rc : xb_launch_status();
}

template <int NT, int R>
int with_group(const LinearArgs& A, cudaStream_t stream) {
    return A.per_row == 4 ? launch<NT, R, 4>(A, stream) : (A.per_row == 2 ? launch<NT, R, 2>(A, stream) : launch<NT, R, 1>(A, stream));
}

}  // namespace

namespace xb4 {

int linear4_mma(const LinearArgs& A, cudaStream_t stream) {
    // (sixteen columns for eight rows or fewer: 4,096 x 24,576 25 us instead of 15.1)
    if (A.tokens > 8) return with_group<2, 2>(A, stream);
    // Four tiles of rows at a time take x out of memory half as often as two, but leave processors idle where they do not go round: whichever has less to do in
    // its longest block, with a sixth more work for two.
    const long long tiles = (A.rows + TILE_ROWS - 1) / TILE_ROWS, four = (((tiles + 3) / 4 + SLOTS - 1) / SLOTS) * 4 * 6, two = (((tiles + 1) / 2 + SLOTS - 1) / SLOTS) * 2 * 7;
    return two < four ? with_group<1, 2>(A, stream) : with_group<1, 4>(A, stream);
}

}  // namespace xb4
