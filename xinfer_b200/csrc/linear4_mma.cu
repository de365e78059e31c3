// Products of few rows (16 at a time) with a weight in 4 bits, in bfloat16 on matrix units (linear4.cu says what is computed and how a weight lies).
//
// The weight's rows are the rows of the products, the tokens their columns.  The bits c of a code under a mask of four bits are the bfloat16
// c 2^-133, in the next four bits 16 c 2^-133: a word of eight codes becomes eight operands by one shift and four masks, and nothing is subtracted.
// x is scaled by 2^60 (2^56 in front of the 16-fold ones), so that sums are ordinary float32 numbers: 2^-73 of their value.  Per group of columns
//   y += s (code . x) + m sum(x),   sum(x) by a product of the same x with ones; both in float32.
// x may be up to 2^67 in size; below 2^-100 it loses digits.
//
// Bound by reading the weight once.  A block's warps and the blocks of a cluster take a range of the columns each, for R tiles of rows at a time, and walk
// over the rows' tiles; the codes are fetched two or four stages ahead, over the ends of the rows' tiles too (where the caller says that the weight is
// complete, the first ones before the kernel in front has ended: 5.1 us instead of 5.9 for 4,096 x 6,144 and one row).  Sums meet in shared memory, warp by
// warp and block by block in their order.
#include "linear4.h"

namespace {

using namespace xb4;

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u, ONES = 0x00010001u, ONES16 = 0x00100010u;      // ones of the scale of the codes
constexpr uint32_t UP = 0x5d805d80u, UP16 = 0x5b805b80u;           // 2^60 and 2^56, twice
constexpr float BACK = 0x1p73f;

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

    for (int rt0 = first; rt0 < row_tiles; rt0 += stride) {
    float acc[R][NT][4] = {};
    for (int ct = from; ct < to; ++ct) {
        uint4 xv[NT][4];
        // (asked for before the codes are waited for)
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
                b[n][0] = times(v.x, UP), b[n][1] = times(v.y, UP16), b[n][2] = times(v.z, UP), b[n][3] = times(v.w, UP16);
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
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[(warp * NT * 8 + n * 8 + 2 * t + (e & 1)) * STRIDE + r * TILE_ROWS + g + 8 * (e >> 1)] = acc[r][n][e] * BACK;
    __syncthreads();
    const int n0 = rt0 * TILE_ROWS, total = many * ROWS;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out);
    for (int i = threadIdx.x; i < total; i += THREADS) {
        const int token = i / ROWS, row = i % ROWS;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += sums[(w * NT * 8 + token) * STRIDE + row];
        if (cluster > 1) sums[token * STRIDE + row] = v;
        else if (n0 + row < A.rows) out[(t0 + token) * A.out_stride + n0 + row] = __float2bfloat16_rn(v);
    }
    if (cluster > 1) {
        cluster_sync();
        const uint32_t base = (uint32_t)__cvta_generic_to_shared(sums);
        for (int i = total * rank / cluster + (int)threadIdx.x; i < total * (rank + 1) / cluster; i += THREADS) {
            const int token = i / ROWS, row = i % ROWS;
            float v = 0.f;
            for (int k = 0; k < cluster; ++k) v += of_rank(base + (token * STRIDE + row) * 4, k);
            if (n0 + row < A.rows) out[(t0 + token) * A.out_stride + n0 + row] = __float2bfloat16_rn(v);
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
    // four and eight blocks: 4,096 x 4,096 (one row) 5.6, 4.9, 4.3, 7.4 us; 12,288 columns 19.2, 12.2, 8.9, 12.3; 4,096 x 6,144 6.6, 6.5, 8.0, 11.7.
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
    // (sixteen columns for eight rows or fewer: 4,096 x 24,576 23 us instead of 14.6)
    if (A.tokens > 8) return with_group<2, 2>(A, stream);
    // Four tiles of rows at a time take x out of memory half as often as two, but leave processors idle where they do not go round: whichever has less to do in
    // its longest block, with a sixth more work for two.
    const long long tiles = (A.rows + TILE_ROWS - 1) / TILE_ROWS, four = (((tiles + 3) / 4 + SLOTS - 1) / SLOTS) * 4 * 6, two = (((tiles + 1) / 2 + SLOTS - 1) / SLOTS) * 2 * 7;
    return two < four ? with_group<1, 2>(A, stream) : with_group<1, 4>(A, stream);
}

}  // namespace xb4
