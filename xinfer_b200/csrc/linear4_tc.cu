// Products of many rows with a weight in 4 bits, in bfloat16 on the 5th-generation tensor cores (linear4.cu says what is computed and how a weight
// lies).
//
// D[128 rows of the weight, up to 256 tokens] in tensor memory, and so is the weight's operand: a thread takes a row of a column tile out of its codes
// into 64 registers and stores them to its lane.  (Through shared memory the operand is written and read again at 128 bytes a cycle, which bound the
// kernel: 850 cycles a column tile with 64 tokens.)  Four teams of four warps take every fourth column tile each.  One thread fetches the tokens'
// columns by TMA, one warp issues the products.  A number of the weight becomes m + s code rounded to bfloat16 once, as a weight in bfloat16
// would be: the bits of a code under a mask are the bfloat16 c 2^-133 (16 times that in the next four bits), times 2^127 (2^123) they are c 2^-6, and a
// multiply-add of two numbers with s 2^6 and m gives both.  Numbers and sums are what they stand for, whatever their size; scales may be up to 2^121.
// K is split over a cluster's blocks where the row tiles alone do not fill the processors; their sums meet through distributed shared memory in
// rank order.
#include "linear4.h"
#include "tc_common.cuh"

namespace {

using namespace xb4;
using namespace xbtc;

constexpr int ROWS = 128, CODE_WARPS = 16, TEAMS = CODE_WARPS / 4, THREADS = (CODE_WARPS + 2) * 32;
constexpr int A_COLUMNS = TILE_COLS / 2;   // of tensor memory that a tile of the weight takes
constexpr int TOKENS_MOST = 256, STAGES_MOST = 4;
// Blocks of a cluster wait for each other while they hold all of their processors' tensor memory, and the waits for either have no limit: a block of
// another kernel that does both (gemm_skinny_tc.cu, 37 KB of shared memory at least) on the same processor could hold columns that this one waits for while its
// cluster waits for columns that this one's cluster holds elsewhere.  So a clustered launch takes so much of a processor's 228 KB of shared memory that no
// block of that kernel, and none of this one, is there beside it.
constexpr int SMEM_MOST = 201 * 1024, SMEM_CLUSTERED = SMEM_MOST;
constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;
constexpr uint32_t UP = 0x7f007f00u, UP16 = 0x7d007d00u, BACK = 0x42804280u;       // 2^127, 2^123, 2^6, twice

struct TcArgs {
    LinearArgs a;
    int mp, stages, tiles_per_split;       // tokens of a tile, padded
    int* err;
};

__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t fma_bf16(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
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

__device__ __forceinline__ uint32_t elected() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e;
}
// Products issued by one lane of a warp that stays together: their operands are then values of the warp (in a branch of one lane every operand is
// moved there, 100 cycles a product).
__device__ __forceinline__ void umma_of(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void commit_of(uint32_t one, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(bar), "r"(one) : "memory");
}

// A row's 128 codes in a column tile, and its words.
template <int PER>
struct Codes {
    uint4 c[4];
    uint32_t w[PER];
};

// grid: (row blocks, splits, token blocks); cluster (1, splits, 1)
template <int PER>
__global__ void __launch_bounds__(THREADS, 1)
linear4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const TcArgs T) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * STAGES_MOST + 2 * TEAMS + 1];
    __shared__ uint32_t s_tmem;
    const LinearArgs& A = T.a;
    constexpr int TILE = TILE_CODES + TILE_ROWS * PER * 4;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;       // (the swizzle repeats every 1024 bytes)
    float* sums = reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw)));
    const uint32_t x_atom = (uint32_t)T.mp * 128, stage_bytes = 2 * x_atom;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mp = T.mp, stages = T.stages;
    const int row_tiles = (A.rows + TILE_ROWS - 1) / TILE_ROWS, col_tiles = (A.columns + TILE_COLS - 1) / TILE_COLS;
    const int from = blockIdx.y * T.tiles_per_split, iters = max(0, min(col_tiles - from, T.tiles_per_split));
    const int t0 = blockIdx.z * mp, many = min(mp, A.tokens - t0);
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES_MOST]), a_full0 = smem_u32(&bars[2 * STAGES_MOST]), a_empty0 = a_full0 + 8 * TEAMS, accum = a_empty0 + 8 * TEAMS;
    const uint32_t tmem_cols = 512;        // D from the first on, the weight's tiles from 256 on
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int i = 0; i < TEAMS; ++i) mbar_init(a_full0 + 8 * i, 4), mbar_init(a_empty0 + 8 * i, 1);
        mbar_init(accum, 1);
        mbar_init_fence();
    }
    if (warp == CODE_WARPS) tmem_alloc(&s_tmem, tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();       // only now: see pdl_launch_dependents on tensor memory

    if (warp < CODE_WARPS) {
        // ---- codes to numbers: row 32 (warp % 4) + lane of the block
        if (!A.early) pdl_wait();
        const int team = warp >> 2, in_tile = lane & 15;
        const int row_tile = min((int)blockIdx.x * 8 + (warp & 3) * 2 + (lane >> 4), row_tiles - 1);       // (behind the last row: it again)
        const uint8_t* next = A.weight + ((long long)row_tile * col_tiles + from + team) * TILE;
        const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 256 + team * A_COLUMNS;
        int asked = team;
        auto fetch = [&](Codes<PER>& h) {
            if (asked < iters) {
#pragma unroll
                for (int t = 0; t < 4; ++t) h.c[t] = reinterpret_cast<const uint4*>(next + in_tile * 64)[t];       // (columns 32 j + 8 t + e of word j)
                const uint32_t* w = reinterpret_cast<const uint32_t*>(next + TILE_CODES) + in_tile * PER;
                if constexpr (PER == 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(w);
                    h.w[0] = v.x, h.w[1] = v.y, h.w[2] = v.z, h.w[3] = v.w;
                } else if constexpr (PER == 2) {
                    const uint2 v = *reinterpret_cast<const uint2*>(w);
                    h.w[0] = v.x, h.w[1] = v.y;
                } else {
                    h.w[0] = *w;
                }
            }
            asked += TEAMS;
            next += TEAMS * TILE;
        };
        Codes<PER> have[2];
        fetch(have[0]);
        fetch(have[1]);
        bool ok = true;
        uint32_t laps = 0;
        for (int it0 = team; it0 < iters && ok; it0 += 2 * TEAMS) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (it0 + i * TEAMS >= iters || !ok) break;
                if (laps > 0) ok = __all_sync(0xffffffffu, mbar_wait(a_empty0 + 8 * team, (laps - 1) & 1, T.err, true));
                if (!ok) break;
                ++laps;
                tc_fence_after();                          // (the products that read this part of tensor memory are done)
#pragma unroll
                for (int p = 0; p < 2; ++p) {              // columns 64 p .. 64 p + 63: words 2 p and 2 p + 1
                    uint32_t v[32];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t w = have[i].w[(2 * p + q) * PER / 4];
                        const uint32_t sc = times(__byte_perm(w, w, 0x1010), BACK), m = __byte_perm(w, w, 0x3232);
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            const uint4& c = have[i].c[t];
                            const uint32_t u = p == 0 ? (q == 0 ? c.x : c.y) : (q == 0 ? c.z : c.w), u8 = u >> 8;
                            v[q * 16 + t * 4] = fma_bf16(times(u & LOW, UP), sc, m), v[q * 16 + t * 4 + 1] = fma_bf16(times(u & HIGH, UP16), sc, m);
                            v[q * 16 + t * 4 + 2] = fma_bf16(times(u8 & LOW, UP), sc, m), v[q * 16 + t * 4 + 3] = fma_bf16(times(u8 & HIGH, UP16), sc, m);
                        }
                    }
                    tmem_st32_u(to + p * 32, v);
                }
                fetch(have[i]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(a_full0 + 8 * team);
            }
        }
    } else if (threadIdx.x == CODE_WARPS * 32) {
        // ---- the tokens' columns
        pdl_wait();
        int s = 0;
        uint32_t phase = 0;
        for (int it = 0; it < iters; ++it) {
            if (it >= stages && !mbar_wait(empty0 + 8 * s, phase ^ 1u, T.err)) break;
            const uint32_t dst = base + s * stage_bytes;
            mbar_expect_tx(full0 + 8 * s, 2 * x_atom);
            tma_load_2d(dst, &map_x, (from + it) * TILE_COLS, t0, full0 + 8 * s);
            tma_load_2d(dst + x_atom, &map_x, (from + it) * TILE_COLS + 64, t0, full0 + 8 * s);
            if (++s == stages) {
                s = 0;
                phase ^= 1u;
            }
        }
    } else if (warp == CODE_WARPS + 1) {
        // ---- products
        const uint32_t one = elected(), tmem_u = __shfl_sync(0xffffffffu, tmem, 0), idesc = umma_idesc(mp);
        const uint64_t bdesc0 = umma_desc(base);
        int s = 0;
        uint32_t phase = 0;
        for (int it = 0; it < iters; ++it) {
            const int slot = it % TEAMS;
            const bool ok = mbar_wait(a_full0 + 8 * slot, (it / TEAMS) & 1, T.err, true) && mbar_wait(full0 + 8 * s, phase, T.err, true);
            if (!__all_sync(0xffffffffu, ok)) {            // (reported; copies that are still on their way are waited for once more)
                for (int i = 0; i < stages; ++i) mbar_wait(full0 + 8 * i, i < s ? phase ^ 1u : phase, T.err);
                break;
            }
            tc_fence_after();
            const uint64_t bdesc = bdesc0 + (uint64_t)((s * stage_bytes) >> 4);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_of(one, tmem_u, tmem_u + 256 + slot * A_COLUMNS + p * 32 + kk * 8, bdesc + (uint64_t)(p * (x_atom >> 4) + kk * 2), idesc, (it | p | kk) ? 1u : 0u);
            commit_of(one, empty0 + 8 * s);
            commit_of(one, a_empty0 + 8 * slot);
            if (++s == stages) {
                s = 0;
                phase ^= 1u;
            }
        }
        commit_of(one, accum);
    }
    __syncwarp();
    pdl_wait();                    // nothing of the kernel before may still read what is written below
    const uint32_t csize = cluster_size(), crank = cluster_rank();
    const int n0 = blockIdx.x * ROWS;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out);
    const bool ready = mbar_wait(accum, 0, T.err) && iters > 0;
    tc_fence_after();
    if (warp < CODE_WARPS) {
        // warps of a quarter of the rows share the tokens
        const int row = (warp & 3) * 32 + lane;
        for (int c0 = (warp >> 2) * 16; c0 < mp; c0 += (CODE_WARPS / 4) * 16) {
            float v[16];
            if (ready) {
                tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c0, v);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0.f;
            }
            if (csize == 1) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (c0 + i < many && n0 + row < A.rows) out[(long long)(t0 + c0 + i) * A.out_stride + n0 + row] = __float2bfloat16_rn(v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) sums[(c0 + i) * ROWS + row] = v[i];
            }
        }
    }
    if (csize > 1) {
        cluster_sync();            // every block of the cluster has written its sums
        const int total = many * ROWS, per = (total + (int)csize - 1) / (int)csize, end = min(total, ((int)crank + 1) * per);
        for (int e = (int)crank * per + (int)threadIdx.x; e < end; e += THREADS) {
            float v = 0.f;
            for (uint32_t r = 0; r < csize; ++r) v += of_rank(base + (uint32_t)e * 4u, r);
            const int n = n0 + e % ROWS;
            if (n < A.rows) out[(long long)(t0 + e / ROWS) * A.out_stride + n] = __float2bfloat16_rn(v);
        }
        cluster_sync();            // nobody leaves while its sums are read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == CODE_WARPS) tmem_free(tmem, tmem_cols);
}

// [tokens, columns] through boxes of 64 columns and `box` tokens, 128-byte swizzle; what lies outside is zero.
bool map_of(CUtensorMap* map, const LinearArgs& A, int box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)A.columns, (cuuint64_t)A.tokens}, strides[1] = {(cuuint64_t)A.x_stride * 2};
    const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(A.x), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int PER>
int launch(const LinearArgs& A, int* err, cudaStream_t stream) {
    TcArgs T{A, 32, 0, 0, err};
    while (T.mp < A.tokens && T.mp < TOKENS_MOST) T.mp *= 2;
    const int blocks = (A.rows + ROWS - 1) / ROWS, col_tiles = (A.columns + TILE_COLS - 1) / TILE_COLS, token_blocks = (A.tokens + T.mp - 1) / T.mp;
    // blocks enough for the processors, four column tiles each at least
    int splits = 1;
    while (splits < 8 && (long long)blocks * token_blocks * splits * 2 <= 148 && col_tiles / (splits * 2) >= 4) splits *= 2;
    T.tiles_per_split = (col_tiles + splits - 1) / splits;
    const int stage_bytes = 2 * T.mp * 128;
    T.stages = 200 * 1024 / stage_bytes < STAGES_MOST ? 200 * 1024 / stage_bytes : STAGES_MOST;
    const int holds = (T.stages * stage_bytes > T.mp * ROWS * 4 ? T.stages * stage_bytes : T.mp * ROWS * 4) + 1024;        // (the sums lie where the stages did)
    const int smem = splits > 1 && holds < SMEM_CLUSTERED ? SMEM_CLUSTERED : holds;
    CUtensorMap map;
    if (!map_of(&map, A, T.mp)) return (int)cudaErrorInvalidValue;
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(linear4_tc_kernel<PER>, SMEM_MOST, &roomy)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, splits, token_blocks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = splits;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = xb_pdl_enabled() ? 2 : 1;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, linear4_tc_kernel<PER>, map, T);
    return rc != cudaSuccess ? (int)rc : xb_launch_status();
}

}  // namespace

namespace xb4 {

bool linear4_tc_takes(const LinearArgs& A) { return ((uintptr_t)A.x & 15) == 0 && A.x_stride % 8 == 0; }
int linear4_tc(const LinearArgs& A, int* err, cudaStream_t stream) {
    return A.per_row == 4 ? launch<4>(A, err, stream) : (A.per_row == 2 ? launch<2>(A, err, stream) : launch<1>(A, err, stream));
}

}  // namespace xb4
