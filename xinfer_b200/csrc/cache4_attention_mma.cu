// Attention over 4-bit pages for few rows of a key/value head (decoding, bfloat16) on matrix units (cache4_attention.cu says what is computed).
//
// A job is (request, key/value head, up to 8 NT rows); the rows, (token, query head of the group) pairs, are the columns of the products, 16 keys
// their rows: S^T = K Q^T and O^T = V^T P^T, so that the codes are the operand that lanes take apart in registers.
//
// Codes as numbers.  The bits c of a code under a mask of four bits are the bfloat16 c 2^-133, in the next four bits 16 c 2^-133 (below 2^-126, and
// in the first binade above it, bfloat16 numbers lie evenly): a word of eight codes becomes eight numbers by one shift and four masks, and
// nothing is subtracted.  Queries are scaled by a power of two of their own, so that their largest is near 2^120, probabilities times
// scales by 2^44: products and sums are ordinary float32 numbers.
//   score:  sum_groups s (q . code) + m sum(q), both in float32 per group;
//   output: sum_keys (p s) (code - 8) + p (m + 8 s): p s is rounded to bfloat16 once, and around the middle of the codes that rounding is no
//           larger than that of a probability times a value; the second sum is float32.  8 sum(p s) is a product with a constant operand.
// The softmax's reference is a number per column that moves only when a score is more than 2^8 above it.
//
// The tiles (64 keys) of all jobs are one line cut into equal shares, one a block, whatever the lengths are; a block's four warps take a quarter of
// its tiles of a job each, fetch them into rings of their own with bulk copies, and join in shared memory.  Parts of a job that several
// blocks share are joined by a second kernel in their order.
#include "cache4_attention_mma.h"
#include "tc_common.cuh"

namespace {

using namespace xb4;
using xbtc::smem_u32;

constexpr int KT = 64;                     // keys of a tile of the line
constexpr int STEP = 16;                   // keys of a warp's step
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int COST_TILE = 2, COST_JOB = 2; // a job's start and end take about as long as a tile
constexpr float RESCALE_STEP = 8.f;
constexpr int JOB_WORDS = 8;

__host__ __device__ constexpr int per_sm(int nt, int ng) { return nt == 1 && ng <= 4 ? 4 : (nt == 1 || ng <= 4 ? 2 : 1); }
__host__ __device__ constexpr int blocks_of(int nt, int ng) { return 148 * per_sm(nt, ng); }
__host__ __device__ constexpr int stages(int ng) { return ng <= 2 ? 8 : (ng <= 4 ? 5 : 4); }
__host__ __device__ constexpr int stage_bytes(int ng) { return 2 * STEP * 20 * ng; }
// a warp's result in shared memory: [rows][channels + 4], then the rows' maxima and sums
__host__ __device__ constexpr int result_floats(int nt, int ng) { return 8 * nt * (32 * ng + 4) + 16 * nt; }
__host__ __device__ constexpr int smem_bytes(int nt, int ng) {
    const int ring = WARPS * stages(ng) * stage_bytes(ng), joined = WARPS * result_floats(nt, ng) * 4;
    return (ring > joined ? ring : joined) + WARPS * stages(ng) * 8;
}

struct Line {
    float* part_o;                 // [blocks][2][rows][d]: a block's first segment, if its job began before it, and its last, if its job goes on
    float* part_ml;                // [blocks][2][rows][2]: maximum and sum
    int* jobs;                     // [blocks][2][8]: parts (0: there is no such part), block of the first, first row, rows, key/value head, request
    int min_share;
};

struct Walk {
    Request r;
    int b, g, piece;               // the job: request, key/value head, which of their pieces of rows
    int tile0, tiles, pieces;      // of the request
    int job, from, end, share;     // where the job begins in the line, the block's range, a block's share
    int i0, i1;                    // the block's tiles of the job's
    __device__ __forceinline__ int job_units() const { return tiles * COST_TILE + COST_JOB; }
};

template <int ROWS>
__device__ __forceinline__ void set_request(const AttendArgs& A, Walk& w, int b) {
    w.b = b;
    w.r = request_of(A, b);
    w.pieces = (w.r.nodes * (A.nh / A.nkv) + ROWS - 1) / ROWS;
    w.tile0 = first_seen(A, w.r.first_pos) / KT;
    // (a request that sees no key has a tile all the same: its rows are written)
    w.tiles = max(1, (w.r.keys + KT - 1) / KT - w.tile0);
}

// The block's place in the line before its first job; every warp of the block finds it for itself.
template <int ROWS>
__device__ __forceinline__ bool place_in_line(const AttendArgs& A, const Line& line, Walk& w) {
    const int lane = threadIdx.x & 31, each = (A.requests + 31) / 32, b0 = lane * each, b1 = min(b0 + each, A.requests);
    int mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        set_request<ROWS>(A, w, b);
        mine += A.nkv * w.pieces * w.job_units();
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    w.share = max(line.min_share, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    w.from = (int)min((long long)blockIdx.x * w.share, (long long)total);
    w.end = min(total, w.from + w.share);
    if (w.from >= w.end) return false;
    int before = incl - mine, b = b0;
    const int owner = __ffs(__ballot_sync(0xffffffffu, w.from >= before && w.from < incl)) - 1;
    if (lane == owner) {
#pragma unroll 1
        for (; b < b1; ++b) {
            set_request<ROWS>(A, w, b);
            const int n = A.nkv * w.pieces * w.job_units();
            if (w.from < before + n) break;
            before += n;
        }
    }
    set_request<ROWS>(A, w, __shfl_sync(0xffffffffu, b, owner));
    before = __shfl_sync(0xffffffffu, before, owner);
    const int at = (w.from - before) / w.job_units();
    w.g = at / w.pieces;
    w.piece = at % w.pieces;
    w.job = before + at * w.job_units();
    return true;
}

// The next job of which the block has tiles: those that begin in its share.
template <int ROWS>
__device__ __forceinline__ bool next_segment(const AttendArgs& A, Walk& w, bool first) {
    for (;; first = false) {
        if (!first) {
            w.job += w.job_units();
            if (w.job >= w.end) return false;
            if (++w.piece == w.pieces) {
                w.piece = 0;
                if (++w.g == A.nkv) {
                    w.g = 0;
                    do {
                        if (w.b + 1 >= A.requests) return false;
                        set_request<ROWS>(A, w, w.b + 1);
                    } while (w.pieces == 0);
                }
            }
        }
        w.i0 = w.from > w.job ? (w.from - w.job + COST_TILE - 1) / COST_TILE : 0;
        w.i1 = min(w.tiles, (w.end - w.job + COST_TILE - 1) / COST_TILE);
        if (w.i0 < w.i1) return true;
    }
}

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;
constexpr float BACK = 6.18970019642690137449e26f;       // 2^89: 2^133 of the codes over 2^44 of the probabilities
constexpr float UP = 17592186044416.f;                   // 2^44

template <int NT, int NG>
__global__ void __launch_bounds__(THREADS, per_sm(NT, NG))
cache4_attention_mma_kernel(const AttendArgs A, const Line line) {
    extern __shared__ __align__(128) char mem[];
    constexpr int ROWS = 8 * NT, STAGES = stages(NG), STAGE = stage_bytes(NG), HALF = STAGE / 2, CODES = NG * STEP * 16, DP = 32 * NG;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gi = lane >> 2, ti = lane & 3;
    const int group = A.nh / A.nkv, ps = A.page_size, piece_keys = ps % STEP == 0 ? STEP : STEP / 2;
    const uint32_t ring = smem_u32(mem) + warp * STAGES * STAGE;
    const uint32_t bars = smem_u32(mem) + smem_bytes(NT, NG) - WARPS * STAGES * 8 + warp * STAGES * 8;
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) xbtc::mbar_init(bars + 8 * i, 1);
        xbtc::mbar_init_fence();
    }
    __syncwarp();
    pdl_launch_dependents();
    pdl_wait();
    if (threadIdx.x < 2) line.jobs[((size_t)blockIdx.x * 2 + threadIdx.x) * JOB_WORDS] = 0;
    Walk w;
    if (!place_in_line<ROWS>(A, line, w)) return;
    const long long page_bytes = (long long)ps * 20 * NG;
    uint32_t issued = 0, taken = 0;            // steps of this warp's ring, over all segments
    bool failed = false;                       // a copy never came: nothing is waited for any more
    for (bool first = true; next_segment<ROWS>(A, w, first); first = false) {
        const int row0 = w.piece * ROWS, rows = min(ROWS, w.r.nodes * group - row0);
        const int pos0 = w.r.first_pos + row0 / group, pos1 = w.r.first_pos + (row0 + rows - 1) / group;
        const int low1 = first_seen(A, pos1);
        // this warp's steps of the segment, and of these the ones with keys that some row sees
        const int steps = (w.i1 - w.i0) * (KT / STEP), s0 = (w.tile0 + w.i0) * (KT / STEP);
        const int seen0 = first_seen(A, pos0) / STEP, seen1 = (min(pos1 + 1, w.r.keys) + STEP - 1) / STEP;
        const int from = max(s0 + steps * warp / WARPS, seen0), to = failed ? from : min(s0 + steps * (warp + 1) / WARPS, seen1);
        const int* table = A.block_table + (long long)w.b * A.table_stride;
        const uint8_t* k_pages = A.k_cache + w.g * page_bytes;
        const uint8_t* v_pages = A.v_cache + w.g * page_bytes;
        // ---- queries: columns of S^T; column gi of column tile j is row 8 j + gi
        uint32_t qf[NT][NG][4];
        float qsum[NT][NG][2], c1[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int row = j * 8 + gi;
            const bool live = row < rows;
            const long long t = w.r.first + (row0 + (live ? row : 0)) / group;
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(A.q) + t * A.q_stride + (long long)(w.g * group + (row0 + (live ? row : 0)) % group) * A.d;
            float x[NG][8], top = 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = 32 * n + 8 * ti + e;
                    x[n][e] = live && c < A.d ? __bfloat162float(q[c]) : 0.f;
                    top = max_nan(top, fabsf(x[n][e]));
                }
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the power of two that brings the row's largest number to 2^119 .. 2^120 (any for rows of zeros and of numbers that are not finite)
            const int e2 = top > 0.f && top < INFINITY ? 120 - (ilogbf(top) + 1) : 120;
            const float f1 = ldexpf(1.f, e2 / 2), f2 = ldexpf(1.f, e2 - e2 / 2);
            float sums[NG];
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                float y[8], sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[e] = x[n][e] * f1 * f2;
                    sum += y[e] * 0x1p-100f;
                }
                qf[j][n][0] = xbtc::pack_bf16(y[0], y[4]);
                qf[j][n][1] = xbtc::pack_bf16(y[1] * 0.0625f, y[5] * 0.0625f);
                qf[j][n][2] = xbtc::pack_bf16(y[2], y[6]);
                qf[j][n][3] = xbtc::pack_bf16(y[3] * 0.0625f, y[7] * 0.0625f);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sums[n] = sum * 0x1p-33f;
            }
            // what the lane's columns 2 ti and 2 ti + 1 of S^T need
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int from_lane = (2 * ti + e) * 4;
#pragma unroll
                for (int n = 0; n < NG; ++n) qsum[j][n][e] = __shfl_sync(0xffffffffu, sums[n], from_lane);
                const float back = ldexpf(A.scale * 1.4426950408889634f, 133 - __shfl_sync(0xffffffffu, e2, from_lane));
                c1[j][e] = fminf(fmaxf(back, -3.0e38f), 3.0e38f);      // (queries near 2^128: a sum of zero stays one)
            }
        }
        float o[NT][2 * NG][4] = {}, eight[NT][4] = {}, rest[NT][NG][2] = {}, ref[NT][2], l[NT][2] = {};
#pragma unroll
        for (int j = 0; j < NT; ++j) ref[j][0] = ref[j][1] = -INFINITY;

        // ---- fetching: a step's codes as [group][key][16 bytes], its words as [key][group]; keys, then values
        int ids = -1, ids_from = -1, put = from;           // a lane holds the page of one of 32 pieces
        unsigned long long bad = 0;                        // two bits a step, of the last 32: pieces without a page
        auto issue = [&]() {
            // (all lanes)
            const int pieces_a_step = STEP / piece_keys, at = (put - from) * pieces_a_step;
            if (at / 32 * 32 != ids_from) {
                ids_from = at / 32 * 32;
                const long long key = (long long)from * STEP + (long long)(ids_from + lane) * piece_keys;
                ids = -1;
                if (key < (long long)to * STEP && key < w.r.keys) {
                    ids = table[key / ps];
                    if (ids < 0 || ids >= A.num_pages) {
                        atomicOr(A.err, XB_ERR_BAD_PAGE);
                        ids = -1;
                    }
                }
            }
            const uint32_t bar = bars + 8 * (issued % STAGES), dst = ring + issued % STAGES * STAGE;
            const int id0 = __shfl_sync(0xffffffffu, ids, at & 31), id1 = pieces_a_step == 2 ? __shfl_sync(0xffffffffu, ids, (at & 31) + 1) : id0;
            const unsigned none = (id0 < 0 ? 1u : 0u) | (id1 < 0 ? 2u : 0u);
            bad = bad << 2 | none;
            const int key0 = put * STEP;
            if (pieces_a_step == 1) {
                if (lane == 0) xbtc::mbar_expect_tx(bar, none ? 0 : STAGE);
                __syncwarp();
                if (!none) {
                    const long long page = (long long)id0 * A.nkv * page_bytes;
                    if (ps == STEP) {
                        if (lane < 2) bulk_copy(dst + lane * HALF, (lane ? v_pages : k_pages) + page, HALF, bar);
                    } else if (lane < 2 * (NG + 1)) {
                        const int n = lane % (NG + 1), slot = key0 % ps;
                        const uint8_t* src = (lane > NG ? v_pages : k_pages) + page;
                        src += n < NG ? ((long long)n * ps + slot) * 16 : (long long)ps * 16 * NG + slot * NG * 4;
                        bulk_copy(dst + (lane > NG ? HALF : 0) + n * STEP * 16, src, n < NG ? STEP * 16 : STEP * NG * 4, bar);
                    }
                }
            } else {
                const int there = (id0 < 0 ? 0 : 1) + (id1 < 0 ? 0 : 1);
                if (lane == 0) xbtc::mbar_expect_tx(bar, there * (STAGE / 2));
                __syncwarp();
                for (int i = lane; i < 4 * (NG + 1); i += 32) {
                    const int half = i & 1, n = (i >> 1) % (NG + 1), v = (i >> 1) / (NG + 1), id = half ? id1 : id0;
                    if (id < 0) continue;
                    const int slot = (key0 + half * 8) % ps;
                    const uint8_t* src = (v ? v_pages : k_pages) + (long long)id * A.nkv * page_bytes;
                    src += n < NG ? ((long long)n * ps + slot) * 16 : (long long)ps * 16 * NG + slot * NG * 4;
                    const uint32_t to_smem = dst + v * HALF + (n < NG ? n * STEP * 16 + half * 128 : CODES + half * 8 * NG * 4);
                    bulk_copy(to_smem, src, n < NG ? 128 : 8 * NG * 4, bar);
                }
            }
            ++issued;
            ++put;
        };
        for (int i = 0; i < STAGES && put < to; ++i) issue();

        for (int s = from; s < to; ++s) {
            const uint32_t at = ring + taken % STAGES * STAGE;
            failed = !__all_sync(0xffffffffu, xbtc::mbar_wait(bars + 8 * (taken % STAGES), taken / STAGES & 1, A.err, true));
            if (failed) {
                while (++taken < issued) xbtc::mbar_wait(bars + 8 * (taken % STAGES), taken / STAGES & 1, A.err);
                break;
            }
            const unsigned none = (unsigned)(bad >> (2 * (put - 1 - s))) & 3u;
            const int key0 = s * STEP;
            // ---- scores
            float x[NT][4] = {};
            {
                const uint32_t row = at + (lane & 15) * 16 + (lane >> 4) * STEP * 16;      // matrices: keys 0..7 and 8..15 of a group, then of the next
                uint32_t wd[2][NG];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t words = at + CODES + (gi + 8 * h) * NG * 4;
                    if constexpr (NG % 4 == 0) {
#pragma unroll
                        for (int n = 0; n < NG; n += 4)
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(wd[h][n]), "=r"(wd[h][n + 1]), "=r"(wd[h][n + 2]), "=r"(wd[h][n + 3]) : "r"(words + n * 4) : "memory");
                    } else {
#pragma unroll
                        for (int n = 0; n < NG; ++n) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(wd[h][n]) : "r"(words + n * 4) : "memory");
                    }
                }
#pragma unroll
                for (int n = 0; n < NG; n += 2) {
                    uint32_t c[4];
                    ldmatrix_x4(n + 1 < NG ? row + n * STEP * 16 : at + (lane & 15) * 16 + n * STEP * 16, c);
#pragma unroll
                    for (int u = 0; u < 2 && n + u < NG; ++u) {
                        const uint32_t a = c[2 * u], b = c[2 * u + 1], a8 = a >> 8, b8 = b >> 8;
                        const float sa = scale_of(wd[0][n + u]), ma = least_of(wd[0][n + u]), sb = scale_of(wd[1][n + u]), mb = least_of(wd[1][n + u]);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            float d[4] = {0.f, 0.f, 0.f, 0.f};
                            mma(d, a & LOW, b & LOW, a & HIGH, b & HIGH, qf[j][n + u][0], qf[j][n + u][1]);
                            mma(d, a8 & LOW, b8 & LOW, a8 & HIGH, b8 & HIGH, qf[j][n + u][2], qf[j][n + u][3]);
                            x[j][0] = fmaf(sa, d[0], fmaf(ma, qsum[j][n + u][0], x[j][0]));
                            x[j][1] = fmaf(sa, d[1], fmaf(ma, qsum[j][n + u][1], x[j][1]));
                            x[j][2] = fmaf(sb, d[2], fmaf(mb, qsum[j][n + u][0], x[j][2]));
                            x[j][3] = fmaf(sb, d[3], fmaf(mb, qsum[j][n + u][1], x[j][3]));
                        }
                    }
                }
            }
            // ---- probabilities: element e of x is key gi + 8 (e / 2), column 2 ti + e % 2
            const bool masked = none || key0 < low1 || key0 + STEP - 1 > min(pos0, w.r.keys - 1);
            uint32_t seen = 0xffffffffu;                   // bit 4 j + e
            if (masked) {
                seen = 0;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + gi + 8 * (e >> 1), row = min(j * 8 + 2 * ti + (e & 1), rows - 1), pos = w.r.first_pos + (row0 + row) / group;
                        const bool there = !(none & (e >> 1 && piece_keys != STEP ? 2u : 1u));
                        if (there && key < w.r.keys && key <= pos && key >= first_seen(A, pos)) seen |= 1u << (4 * j + e);
                    }
            }
            bool higher = false;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[j][e] *= c1[j][e & 1];
                    if (!(seen >> (4 * j + e) & 1)) x[j][e] = -INFINITY;
                    higher |= !(x[j][e] <= ref[j][e & 1] + RESCALE_STEP);       // (a score that is no number is one too)
                }
            if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = max_nan(x[j][e], x[j][e + 2]);
                        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float now = max_nan(ref[j][e], top), f = ref[j][e] == -INFINITY ? 0.f : xbtc::ex2(ref[j][e] - now);
                        if (now != ref[j][e]) {
                            ref[j][e] = now;
                            l[j][e] *= f;
                            eight[j][e] *= f, eight[j][e + 2] *= f;
#pragma unroll
                            for (int n = 0; n < NG; ++n) rest[j][n][e] *= f;
#pragma unroll
                            for (int n = 0; n < 2 * NG; ++n) o[j][n][e] *= f, o[j][n][e + 2] *= f;
                        }
                    }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float base = ref[j][e & 1] == -INFINITY ? 0.f : ref[j][e & 1];
                    x[j][e] = xbtc::ex2(x[j][e] - base);
                    l[j][e & 1] += x[j][e];
                }
            // ---- values
            {
                const uint32_t row = at + HALF + (lane & 15) * 16 + (lane >> 4) * STEP * 16;
                uint32_t wd[2][NG];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t words = at + HALF + CODES + (gi + 8 * h) * NG * 4;
                    if constexpr (NG % 4 == 0) {
#pragma unroll
                        for (int n = 0; n < NG; n += 4)
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(wd[h][n]), "=r"(wd[h][n + 1]), "=r"(wd[h][n + 2]), "=r"(wd[h][n + 3]) : "r"(words + n * 4) : "memory");
                    } else {
#pragma unroll
                        for (int n = 0; n < NG; ++n) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(wd[h][n]) : "r"(words + n * 4) : "memory");
                    }
                }
#pragma unroll
                for (int n = 0; n < NG; n += 2) {
                    uint32_t c[4];
                    ldmatrix_x4_t(n + 1 < NG ? row + n * STEP * 16 : at + HALF + (lane & 15) * 16 + n * STEP * 16, c);
#pragma unroll
                    for (int u = 0; u < 2 && n + u < NG; ++u) {
                        const uint32_t a = c[2 * u], b = c[2 * u + 1], a8 = a >> 8, b8 = b >> 8;
                        const float sa = scale_of(wd[0][n + u]) * UP, sb = scale_of(wd[1][n + u]) * UP;
                        const float ma = fmaf(scale_of(wd[0][n + u]), 8.f, least_of(wd[0][n + u])), mb = fmaf(scale_of(wd[1][n + u]), 8.f, least_of(wd[1][n + u]));
                        const uint32_t mine = gi == n + u ? 0x00080008u : 0u;          // 8 2^-133 in the group's row
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            float y[4] = {x[j][0] * sa, x[j][1] * sa, x[j][2] * sb, x[j][3] * sb}, z[4] = {x[j][0] * ma, x[j][1] * ma, x[j][2] * mb, x[j][3] * mb};
                            if (masked) {                  // what is not seen adds nothing, whatever its scale is
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (!(seen >> (4 * j + e) & 1)) y[e] = z[e] = 0.f;
                            }
                            rest[j][n + u][0] += z[0] + z[2];
                            rest[j][n + u][1] += z[1] + z[3];
                            const uint32_t p0 = transposed(xbtc::pack_bf16(y[0], y[1])), p1 = transposed(xbtc::pack_bf16(y[2], y[3]));
                            mma(o[j][2 * (n + u)], a & LOW, a & HIGH, b & LOW, b & HIGH, p0, p1);
                            mma(o[j][2 * (n + u) + 1], a8 & LOW, a8 & HIGH, b8 & LOW, b8 & HIGH, p0, p1);
                            mma(eight[j], mine, 0u, mine, 0u, p0, p1);
                        }
                    }
                }
            }
            __syncwarp();
            ++taken;
            if (put < to) issue();
        }
        // ---- the warps' results, joined by the block
        __syncthreads();                                   // (the rings are empty: results may lie there)
        float* mine = reinterpret_cast<float*>(mem) + warp * result_floats(NT, NG);
        if (failed)
            for (int j = 0; j < NT; ++j) l[j][0] = l[j][1] = 0.f, ref[j][0] = ref[j][1] = -INFINITY;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[j][e];
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
                float* to_row = mine + (j * 8 + 2 * ti + e) * (DP + 4);
                float* ml = mine + ROWS * (DP + 4) + (j * 8 + 2 * ti + e) * 2;
                if (gi == 0) ml[0] = ref[j][e], ml[1] = sum;
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    float r = rest[j][n][e];
#pragma unroll
                    for (int s = 4; s < 32; s <<= 1) r += __shfl_xor_sync(0xffffffffu, r, s);
                    const float minus = __shfl_sync(0xffffffffu, eight[j][e], n * 4 + ti);
                    float4 v;
                    v.x = fmaf(o[j][2 * n][e] - minus, BACK, r);
                    v.y = fmaf(o[j][2 * n][e + 2] * 0.0625f - minus, BACK, r);
                    v.z = fmaf(o[j][2 * n + 1][e] - minus, BACK, r);
                    v.w = fmaf(o[j][2 * n + 1][e + 2] * 0.0625f - minus, BACK, r);
                    *reinterpret_cast<float4*>(to_row + 32 * n + 4 * gi) = v;
                }
            }
        __syncthreads();
        {
            const bool whole = w.i0 == 0 && w.i1 == w.tiles;
            const int which = w.from > w.job ? 0 : 1;
            const size_t part = (size_t)blockIdx.x * 2 + which;
            const float* all = reinterpret_cast<const float*>(mem);
            constexpr int FLOATS = result_floats(NT, NG);
            for (int i = threadIdx.x; i < rows * (DP / 4); i += THREADS) {
                const int row = i / (DP / 4), c = i % (DP / 4) * 4;
                float top = -INFINITY, f[WARPS], total = 0.f;
#pragma unroll
                for (int k = 0; k < WARPS; ++k) top = max_nan(top, all[k * FLOATS + ROWS * (DP + 4) + row * 2]);
                float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < WARPS; ++k) {
                    const float ref_k = all[k * FLOATS + ROWS * (DP + 4) + row * 2];
                    f[k] = ref_k == -INFINITY ? 0.f : xbtc::ex2(ref_k - top);
                    if (ref_k == -INFINITY) continue;
                    total = fmaf(f[k], all[k * FLOATS + ROWS * (DP + 4) + row * 2 + 1], total);
                    const float4 u = *reinterpret_cast<const float4*>(all + k * FLOATS + row * (DP + 4) + c);
                    v.x = fmaf(f[k], u.x, v.x), v.y = fmaf(f[k], u.y, v.y), v.z = fmaf(f[k], u.z, v.z), v.w = fmaf(f[k], u.w, v.w);
                }
                if (whole) {
                    const long long t = w.r.first + (row0 + row) / group;
                    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out) + t * A.out_stride + (long long)(w.g * group + (row0 + row) % group) * A.d;
                    const float inv = total == 0.f ? 0.f : 1.f / total;
                    const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < A.d) out[c + e] = __float2bfloat16_rn(y[e]);
                } else {
                    *reinterpret_cast<float4*>(line.part_o + (part * ROWS + row) * DP + c) = v;
                    if (c == 0) line.part_ml[(part * ROWS + row) * 2] = top, line.part_ml[(part * ROWS + row) * 2 + 1] = total;
                }
            }
            if (!whole && threadIdx.x == 0) {
                int* job = line.jobs + part * JOB_WORDS;
                const int first_block = w.job / w.share, last = (w.job + (w.tiles - 1) * COST_TILE) / w.share;
                job[1] = first_block, job[2] = row0, job[3] = rows, job[4] = w.g, job[5] = w.b;
                job[0] = last - first_block + 1;
            }
        }
        xbtc::fence_async_shared();
        __syncthreads();                                   // (the next segment's copies may write where the results lay)
    }
}

// A job's parts, joined in the order of the line: the blocks that left them share its numbers.
template <int NT, int NG>
__global__ void __launch_bounds__(THREADS)
cache4_attention_join_kernel(const AttendArgs A, const Line line) {
    constexpr int ROWS = 8 * NT, DP = 32 * NG, FOURS = DP / 4;
    pdl_launch_dependents();
    pdl_wait();
    const int* job = line.jobs + (size_t)blockIdx.x * JOB_WORDS;
    const int parts = job[0];
    if (parts < 1) return;
    const int first = job[1], row0 = job[2], rows = job[3], g = job[4], group = A.nh / A.nkv;
    const Request r = request_of(A, job[5]);
    const int mine = (int)blockIdx.x / 2 - first, total = rows * FOURS;
    auto part_of = [&](int i) { return (size_t)(first + i) * 2 + (i == 0 ? 1 : 0); };     // (the first part is its block's last segment)
    for (int i = total * mine / parts + (int)threadIdx.x; i < total * (mine + 1) / parts; i += THREADS) {
        const int row = i / FOURS, c = i % FOURS * 4;
        float top = -INFINITY, sum = 0.f;
        for (int k = 0; k < parts; ++k) top = max_nan(top, line.part_ml[(part_of(k) * ROWS + row) * 2]);
        float4 v = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < parts; ++k) {
            const size_t at = part_of(k) * ROWS + row;
            const float ref = line.part_ml[at * 2];
            if (ref == -INFINITY) continue;
            const float f = xbtc::ex2(ref - top);
            const float4 u = *reinterpret_cast<const float4*>(line.part_o + at * DP + c);
            sum = fmaf(f, line.part_ml[at * 2 + 1], sum);
            v.x = fmaf(f, u.x, v.x), v.y = fmaf(f, u.y, v.y), v.z = fmaf(f, u.z, v.z), v.w = fmaf(f, u.w, v.w);
        }
        const long long t = r.first + (row0 + row) / group;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out) + t * A.out_stride + (long long)(g * group + (row0 + row) % group) * A.d;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < A.d) out[c + e] = __float2bfloat16_rn(y[e]);
    }
}

template <int NT, int NG>
long long scratch_of() {
    return (long long)blocks_of(NT, NG) * 2 * (8 * NT * (32 * NG + 2) + JOB_WORDS);
}

template <int NT, int NG>
int launch(const AttendArgs& A, float* scratch, cudaStream_t stream) {
    constexpr int blocks = blocks_of(NT, NG);
    Line line;
    line.part_o = scratch;
    line.part_ml = scratch + (size_t)blocks * 2 * 8 * NT * 32 * NG;
    line.jobs = reinterpret_cast<int*>(line.part_ml + (size_t)blocks * 2 * 8 * NT * 2);
    line.min_share = COST_TILE;
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(cache4_attention_mma_kernel<NT, NG>, smem_bytes(NT, NG), &roomy)) return rc;
    const int rc = xb_launch(cache4_attention_mma_kernel<NT, NG>, dim3(blocks), dim3(THREADS), smem_bytes(NT, NG), stream, A, line);
    if (rc) return rc;
    return xb_launch(cache4_attention_join_kernel<NT, NG>, dim3(2 * blocks), dim3(THREADS), 0, stream, A, line);
}

template <typename F>
auto by_form(int rows, int groups, F f) {
    auto with = [&](auto nt) {
        switch (groups) {
            case 1: return f(nt, std::integral_constant<int, 1>());
            case 2: return f(nt, std::integral_constant<int, 2>());
            case 3: return f(nt, std::integral_constant<int, 3>());
            case 4: return f(nt, std::integral_constant<int, 4>());
            default: return f(nt, std::integral_constant<int, 8>());
        }
    };
    return rows <= 8 ? with(std::integral_constant<int, 1>()) : with(std::integral_constant<int, 2>());
}

int rows_of(int nh, int nkv, int longest) {
    const long long r = (long long)(nh / nkv) * longest;
    return r > 1 << 20 ? 1 << 20 : (int)r;
}

}  // namespace

namespace xb4 {

bool mma_takes(int d) { return groups_of(d) <= 4 || groups_of(d) == 8; }
bool mma_takes(const AttendArgs& A) {
    // the longest line that these shapes allow is counted in 32 bits
    const double jobs = (double)A.nkv * ((double)A.tokens * (A.nh / A.nkv) / 8 + A.requests), tiles = (double)A.table_stride * A.page_size / KT + 2;
    return mma_takes(A.d) && A.page_size % 8 == 0 && A.num_pages > 0 && jobs * (tiles * COST_TILE + COST_JOB) < 2147483648.0;
}
long long mma_scratch(int nh, int nkv, int d, int longest) {
    return by_form(rows_of(nh, nkv, longest), groups_of(d), [](auto nt, auto ng) { return scratch_of<decltype(nt)::value, decltype(ng)::value>(); });
}
int mma_launch(const AttendArgs& A, int longest, float* scratch, cudaStream_t stream) {
    return by_form(rows_of(A.nh, A.nkv, longest), groups_of(A.d),
                   [&](auto nt, auto ng) { return launch<decltype(nt)::value, decltype(ng)::value>(A, scratch, stream); });
}

}  // namespace xb4
