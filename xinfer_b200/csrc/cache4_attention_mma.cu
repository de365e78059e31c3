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
// The products of values are ordinary float32 numbers for values of up to 2^50 and sums of 2^-28 and more.  A segment with a row of smaller sums, with larger values or
// a group that is no number is known by its sums' sizes and done again number by number.  (A power of two that follows the values instead: 64 single tokens
// 51 us instead of 48, the loop has no register for it.)
//
// The tiles (32 keys) of all jobs are one line cut into equal shares, one a warp, whatever the lengths are: warps of a block have nothing to do with each
// other.  A warp fetches its keys and values into a ring of its own with bulk copies.  Parts of a job that several warps share are joined by a
// second kernel in their order.
//
// Bound by issued instructions: 377 for 16 keys of 128 channels, 2.2 to 2.4 a cycle of a processor's 4, of which the matrix instructions are 2 cycles each; then
// by what a segment costs to start and end (20,000 cycles) and by the join.  Bfloat16, 32 heads over 8 of 128 channels: 64 single tokens at up to 4,096 keys 48 us (2.5 TB/s of
// codes), 24 at up to 32,768 101 us (3.8 TB/s); one token of 16 heads at 1,024 keys 11 us, of which the join is 4.
#include "cache4_attention_mma.h"
#include "tc_common.cuh"

namespace {

using namespace xb4;
using xbtc::smem_u32;

constexpr int STEP = 16;                   // keys of a step
constexpr int STAGE_STEPS = 2;             // steps that are fetched together
constexpr int KT = STEP * STAGE_STEPS;     // keys of a tile of the line
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int COST_JOB = 3;                // a job's start and end take about as long as three tiles
constexpr float RESCALE_STEP = 8.f;
constexpr int JOB_WORDS = 8;

__host__ __device__ constexpr int per_sm(int nt, int ng) { return nt == 1 && ng <= 4 ? 4 : 2; }
__host__ __device__ constexpr int blocks_of(int nt, int ng) { return 148 * per_sm(nt, ng); }
__host__ __device__ constexpr int stages(int ng) { return ng <= 2 ? 4 : 2; }
__host__ __device__ constexpr int stage_bytes(int ng) { return STAGE_STEPS * 2 * STEP * 20 * ng; }
__host__ __device__ constexpr int smem_bytes(int ng) { return WARPS * stages(ng) * (stage_bytes(ng) + 8); }

struct Line {
    float* part_o;                 // [warps][2][rows][d]: a warp's first segment, if its job began before it, and its last, if its job goes on
    float* part_ml;                // [warps][2][rows][2]: maximum and sum
    int* jobs;                     // [warps][2][8]: parts (0: there is no such part), warp of the first, first row, rows, key/value head, the request's first token
};

struct Walk {
    Request r;
    int b, g, piece;               // the job: request, key/value head, which of their pieces of rows
    int tile0, tiles, pieces;      // of the request
    int job, from, end, share;     // where the job begins in the line, the warp's range, a warp's share
    int i0, i1;                    // the warp's tiles of the job's
    __device__ __forceinline__ int job_units() const { return tiles + COST_JOB; }
};

template <int ROWS>
__device__ __forceinline__ void set_request(const AttendArgs& A, Walk& w, int b) {
    w.b = b;
    w.r = request_of<true>(A, b);
    w.pieces = (w.r.nodes * A.group + ROWS - 1) / ROWS;
    w.tile0 = first_seen(A, w.r.first_pos) / KT;
    // (a request that sees no key has a tile all the same: its rows are written)
    w.tiles = max(1, (w.r.keys + KT - 1) / KT - w.tile0);
}

// The warp's place in the line before its first job.
template <int ROWS>
__device__ __forceinline__ bool place_in_line(const AttendArgs& A, const Line& line, int me, int warps, Walk& w) {
    const int lane = threadIdx.x & 31, each = (A.requests + 31) / 32, b0 = lane * each, b1 = min(b0 + each, A.requests);
    long long mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        set_request<ROWS>(A, w, b);
        mine += (long long)A.nkv * w.pieces * w.job_units();
    }
    int incl;
    const int total = prefix_of_lanes(A, mine, incl);
    if (total < 0) return false;
    w.share = (total + warps - 1) / warps;
    w.from = (int)min((long long)me * w.share, (long long)total);
    w.end = min(total, w.from + w.share);
    if (w.from >= w.end) return false;
    int before = incl - (int)mine, b = b0;
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

// The next job of which the warp has tiles: those that begin in its share.
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
        w.i0 = max(0, w.from - w.job);
        w.i1 = min(w.tiles, w.end - w.job);
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
// the same without a sum before it
__device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void ldmatrix_x2(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x2_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
// The halves of a word that are infinities or no numbers become zero.
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t packed) {        // what bfloat16 rounding left of a and b
    return xbtc::pack_bf16(a - scale_of(packed), b - least_of(packed));
}

constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;
constexpr float BACK = 6.18970019642690137449e26f;       // 2^89: 2^133 of the codes over 2^44 of the probabilities
constexpr float UP = 44.f, DOWN = 0x1p-44f;
constexpr float TOP = UP + RESCALE_STEP;

// The words of the groups of two keys, eight apart.
template <int NG>
__device__ __forceinline__ void load_words(uint32_t at, uint32_t (&w)[2][NG]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t key = at + 8 * h * NG * 4;
        if constexpr (NG % 4 == 0) {
#pragma unroll
            for (int n = 0; n < NG; n += 4)
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[h][n]), "=r"(w[h][n + 1]), "=r"(w[h][n + 2]), "=r"(w[h][n + 3]) : "r"(key + n * 4) : "memory");
        } else {
#pragma unroll
            for (int n = 0; n < NG; ++n) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[h][n]) : "r"(key + n * 4) : "memory");
        }
    }
}

// Eight channels of a query (zeros behind the head).
__device__ __forceinline__ void load_query(const __nv_bfloat16* q, int c, int d, bool on16, float (&x)[8]) {
    if (on16 && c + 8 <= d) {
        const uint4 v = *reinterpret_cast<const uint4*>(q + c);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = c + e < d ? __bfloat162float(q[c + e]) : 0.f;
    }
}

constexpr uint32_t VALUES_TO = (127 + 50) << 7, NO_NUMBER = 0x8000u;       // bits of 2^50 in bfloat16; above those of all sizes

// Bits of the largest scale or least value of a group's word, NO_NUMBER for one that is not finite.
__device__ __forceinline__ uint32_t size_of_word(uint32_t word) {
    const uint32_t size = max(word & 0x7fffu, word >> 16 & 0x7fffu);
    return size >= 0x7f80u ? NO_NUMBER : size;
}
// The largest of some keys' values, out of the cache.
template <int NG>
__device__ __noinline__ uint32_t size_of_values(const AttendArgs& A, int b, int g, int from, int to) {
    const int ps = A.page_size;
    const long long page_bytes = (long long)ps * 20 * NG;
    uint32_t most = 0;
    for (int key = from + (int)(threadIdx.x & 31); key < to; key += 32) {
        const int id = A.block_table[(long long)b * A.table_stride + key / ps];
        if (id < 0 || id >= A.num_pages) continue;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(A.v_cache + ((long long)id * A.nkv + g) * page_bytes + (long long)ps * 16 * NG) + key % ps * NG;
        for (int n = 0; n < NG; ++n) most = max(most, size_of_word(words[n]));
    }
    return __reduce_max_sync(0xffffffffu, most);
}
// Keys `from` .. `to` of some rows, number by number: whole rows, or a part where `part_o` is given.
template <int NG>
__device__ __noinline__ void rows_by_number(const AttendArgs& A, int b, int g, int row0, int rows, int from, int to, float* part_o, float* part_ml) {
    const int lane = threadIdx.x & 31, ps = A.page_size;
    const Request r = request_of<true>(A, b);
    const long long page_bytes = (long long)ps * 20 * NG;
    const int* table = A.block_table + (long long)b * A.table_stride;
    for (int row = 0; row < rows; ++row) {
        const int token = token_of(A, row0 + row), pos = r.first_pos + token;
        const long long head = g * A.group + (row0 + row - token * A.group);
        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(A.q) + (r.first + token) * A.q_stride + head * A.d;
        float qv[NG], o[NG] = {}, top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int n = 0; n < NG; ++n) qv[n] = 32 * n + lane < A.d ? __bfloat162float(q[32 * n + lane]) : 0.f;
        for (int key = max(from, first_seen(A, pos)); key < min(min(to, pos + 1), r.keys); ++key) {
            const int id = table[key / ps], slot = key % ps;
            if (id < 0 || id >= A.num_pages) continue;             // (reported where it was to be fetched)
            const uint8_t* page[2] = {A.k_cache + ((long long)id * A.nkv + g) * page_bytes, A.v_cache + ((long long)id * A.nkv + g) * page_bytes};
            float x[2][NG], score = 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int v = 0; v < 2; ++v)                        // (channels behind the head have codes nobody wrote)
                    x[v][n] = 32 * n + lane < A.d ? value_of(page[v][((long long)n * ps + slot) * 16 + lane / 2] >> 4 * (lane & 1) & 15u,
                                                             reinterpret_cast<const uint32_t*>(page[v] + (long long)ps * 16 * NG)[slot * NG + n]) : 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n) score = fmaf(qv[n], x[0][n], score);
            score = warp_sum(score) * (A.scale * 1.4426950408889634f);
            const float now = max_nan(top, score), a = top == -INFINITY ? 0.f : xbtc::ex2(top - now), p = now == -INFINITY ? 0.f : xbtc::ex2(score - now);
            top = now;
            sum = fmaf(sum, a, p);
#pragma unroll
            for (int n = 0; n < NG; ++n) o[n] = fmaf(p, x[1][n], o[n] * a);
        }
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out) + (r.first + token) * A.out_stride + head * A.d;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if (part_o) part_o[row * 32 * NG + 32 * n + lane] = o[n];
            else if (32 * n + lane < A.d) out[32 * n + lane] = __float2bfloat16_rn(sum == 0.f ? 0.f : o[n] / sum);
        }
        if (part_o && lane == 0) *reinterpret_cast<float2*>(part_ml + row * 2) = make_float2(top, sum);
    }
}

template <int NT, int NG>
__global__ void __launch_bounds__(THREADS, per_sm(NT, NG))
cache4_attention_mma_kernel(const __grid_constant__ AttendArgs A, const Line line) {
    extern __shared__ __align__(128) char mem[];
    constexpr int ROWS = 8 * NT, STAGES = stages(NG), STAGE = stage_bytes(NG), HALF = 20 * NG * STEP, CODES = NG * STEP * 16, DP = 32 * NG;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gi = lane >> 2, ti = lane & 3;
    const int group = A.group, ps = A.page_size;
    const bool by16 = ps % STEP == 0;                      // a step's keys lie in one page; else in two
    const uint32_t ring = smem_u32(mem) + warp * STAGES * STAGE;
    const uint32_t bars = smem_u32(mem) + WARPS * STAGES * STAGE + warp * STAGES * 8;
    // (shares one behind another lie in different blocks, so that few of them are spread over the processors)
    const int warps = (int)gridDim.x * WARPS, me = warp * (int)gridDim.x + (int)blockIdx.x;
    constexpr bool BY_WORDS = NG % 4 == 0;                 // a key's words are rows that ldmatrix takes
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) xbtc::mbar_init(bars + 8 * i, 1);
        xbtc::mbar_init_fence();
    }
    __syncwarp();
    pdl_launch_dependents();
    pdl_wait();
    if (lane < 2) line.jobs[((size_t)me * 2 + lane) * JOB_WORDS] = 0;
    __syncwarp();
    Walk w;
    if (!place_in_line<ROWS>(A, line, me, warps, w)) return;
    const long long page_bytes = (long long)ps * 20 * NG;
    const bool q16 = ((uintptr_t)A.q & 15) == 0 && A.q_stride % 8 == 0 && A.d % 8 == 0;
    const bool out8 = ((uintptr_t)A.out & 7) == 0 && A.out_stride % 4 == 0 && A.d % 4 == 0;
    uint32_t put_slot = 0, take_slot = 0, take_parity = 0; // of this warp's ring, over all segments
    bool failed = false;                                   // a copy never came: nothing is fetched any more
    for (bool first = true; next_segment<ROWS>(A, w, first); first = false) {
        const int row0 = w.piece * ROWS, rows = min(ROWS, w.r.nodes * group - row0);
        const int pos0 = w.r.first_pos + token_of(A, row0), pos1 = w.r.first_pos + token_of(A, row0 + rows - 1);
        // keys from `all0` on and below `all1` are seen by all rows
        const int all0 = first_seen(A, pos1), all1 = min(pos0 + 1, w.r.keys);
        // the segment's steps, of these the ones with keys that some row sees
        const int first_key = first_seen(A, pos0), seen0 = first_key / STEP, seen1 = (min(pos1 + 1, w.r.keys) + STEP - 1) / STEP;
        const int from = max((w.tile0 + w.i0) * STAGE_STEPS, seen0), to = failed ? from : min((w.tile0 + w.i1) * STAGE_STEPS, seen1);
        const int* table = A.block_table + (long long)w.b * A.table_stride;
        const uint8_t* k_pages = A.k_cache + w.g * page_bytes;
        const uint8_t* v_pages = A.v_cache + w.g * page_bytes;

        // ---- fetching: a stage holds two steps, each its keys' codes as [group][key][16 bytes] and words as [key][group], then its values'
        long long page_at = 0;                             // a lane holds the place of one of 32 pieces' pages (pieces: keys that lie in one page),
        unsigned have = 0;                                 // and this which of them there are
        int ids_from = -1, put = from;
        unsigned none_of = 0;                              // eight bits a stage, the last one lowest: pieces without a page
        auto issue = [&]() {
            const int shift = by16 ? 0 : 1, at = (put - from) << shift, in_use = min(STAGE_STEPS, to - put) << shift;
            if ((at & ~31) != ids_from) {
                ids_from = at & ~31;
                const int key = (from << 4) + ((ids_from + lane) << (4 - shift));
                int ids = -1;
                // (pieces in front of the first row's window: their pages may have been given back)
                if (key < to * STEP && key < w.r.keys && key + (STEP >> shift) > first_key) {
                    ids = table[key / ps];
                    if (ids < 0 || ids >= A.num_pages) {
                        atomicOr(A.err, XB_ERR_BAD_PAGE);
                        ids = -1;
                    }
                }
                have = __ballot_sync(0xffffffffu, ids >= 0);
                page_at = (long long)ids * A.nkv * page_bytes;
            }
            const uint32_t bar = bars + 8 * put_slot, dst = ring + put_slot * STAGE;
            // piece i of the stage is lane (at & 31) + i of ids
            const unsigned there = have >> (at & 31) & ((1u << in_use) - 1);
            none_of = none_of << 8 | (~there & 0xffu);
            if (lane == 0) xbtc::mbar_expect_tx(bar, __popc(there) * (by16 ? 2 * HALF : HALF));
            __syncwarp();
            if (ps == STEP) {                              // whole pages
                const long long page = __shfl_sync(0xffffffffu, page_at, (at & 31) + (lane >> 1 & 1));
                if (lane < 4 && (there >> (lane >> 1) & 1)) bulk_copy(dst + lane * HALF, (lane & 1 ? v_pages : k_pages) + page, HALF, bar);
            } else {
                const int each = 2 * (NG + 1), keys = by16 ? STEP : STEP / 2;      // copies of a piece
#pragma unroll 1
                for (int i = lane; i < ((in_use * each + 31) & ~31); i += 32) {
                    const int piece = min(i / each, 3), n = i % each % (NG + 1), v = i % each / (NG + 1);
                    const long long page = __shfl_sync(0xffffffffu, page_at, (at & 31) + piece);
                    if (i >= in_use * each || !(there >> piece & 1)) continue;
                    const int key = put * STEP + piece * keys, slot = key % ps, half = by16 ? 0 : piece & 1;
                    const uint8_t* src = (v ? v_pages : k_pages) + page;
                    src += n < NG ? ((long long)n * ps + slot) * 16 : (long long)ps * 16 * NG + slot * NG * 4;
                    const uint32_t to_smem = dst + (2 * (piece >> shift) + v) * HALF + (n < NG ? n * STEP * 16 + half * 128 : CODES + half * 8 * NG * 4);
                    bulk_copy(to_smem, src, n < NG ? keys * 16 : keys * NG * 4, bar);
                }
            }
            put_slot = put_slot + 1 == STAGES ? 0 : put_slot + 1;
            put += STAGE_STEPS;
        };
        for (int i = 0; i < STAGES && put < to; ++i) issue();

        // ---- queries: columns of S^T; column gi of column tile j is row 8 j + gi
        uint32_t qf[NT][NG][4];
        float qsum[NT][NG][2], c1[NT][2];                  // the columns' sums per group: as numbers, or in two parts as an operand beside the words
        uint32_t qw[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int row = min(j * 8 + gi, rows - 1);     // (columns without a row repeat the last one's)
            const long long t = w.r.first + token_of(A, row0 + row);
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(A.q) + t * A.q_stride + (long long)(w.g * group + (row0 + row - token_of(A, row0 + row) * group)) * A.d;
            float x[NG][8], top = 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                load_query(q, 32 * n + 8 * ti, A.d, q16, x[n]);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(x[n][e]));
            }
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the power of two that brings the row's largest number to 2^119 .. 2^120 (any for rows of zeros and of numbers that are not finite;
            // exponents of numbers below 2^-126 count as 2^-127's, which is no less exact)
            const int expo = (int)(__float_as_uint(top) >> 23), e2 = expo < 255 && top > 0.f ? 246 - max(expo, 1) : 120;
            const float f1 = __uint_as_float((uint32_t)(127 + e2 / 2) << 23), f2 = __uint_as_float((uint32_t)(127 + e2 - e2 / 2) << 23);
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
            if constexpr (BY_WORDS) {                      // in front of s: zero; in front of m: 16 bits of the sum in two parts
#pragma unroll
                for (int h = 0; h < NG / 4; ++h) {
                    const float sum = ti == 0 ? sums[4 * h] : (ti == 1 ? sums[4 * h + 1] : (ti == 2 ? sums[4 * h + 2] : sums[4 * h + 3]));
                    const uint32_t high = xbtc::pack_bf16(0.f, sum);
                    qw[j][2 * h] = high;
                    qw[j][2 * h + 1] = xbtc::pack_bf16(0.f, sum - least_of(high));
                }
            }
            // what the lane's columns 2 ti and 2 ti + 1 of S^T need
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int from_lane = (2 * ti + e) * 4;
                if constexpr (!BY_WORDS) {
#pragma unroll
                    for (int n = 0; n < NG; ++n) qsum[j][n][e] = __shfl_sync(0xffffffffu, sums[n], from_lane);
                }
                const float back = ldexpf(A.scale * 1.4426950408889634f, 133 - __shfl_sync(0xffffffffu, e2, from_lane));
                c1[j][e] = fminf(fmaxf(back, -3.0e38f), 3.0e38f);      // (queries near 2^128: a sum of zero stays one)
            }
        }
        // `base`: 44 minus a column's reference; an infinity before there is one, which makes every score one above it
        float o[NT][2 * NG][4] = {}, eight[NT][4] = {}, base[NT][2], l[NT][2] = {};
        float rest[NT][BY_WORDS ? 1 : NG][2] = {}, both[NT][4] = {};       // sums of p (m + 8 s) per group; of p s and p m in rows 2 group and 2 group + 1
#pragma unroll
        for (int j = 0; j < NT; ++j) base[j][0] = base[j][1] = INFINITY;

        for (int s = from; s < to; s += STAGE_STEPS) {
            const bool ok = xbtc::mbar_wait(bars + 8 * take_slot, take_parity, A.err, true);
            if (!__all_sync(0xffffffffu, ok)) {            // (reported: what comes out then does not count)
                failed = true;
                for (int i = s + STAGE_STEPS; i < put; i += STAGE_STEPS) {
                    take_slot = take_slot + 1 == STAGES ? 0 : take_slot + 1;
                    if (take_slot == 0) take_parity ^= 1;
                    xbtc::mbar_wait(bars + 8 * take_slot, take_parity, A.err);
                }
                break;
            }
            const int ahead = (put - s) / STAGE_STEPS - 1;           // stages issued behind this one
            const unsigned none = none_of >> (8 * ahead);
            auto step = [&](auto masks, const int sub, const unsigned lost) {
                constexpr bool MASKED = decltype(masks)::value;            // some row does not see all of the step's keys
                const uint32_t at = ring + take_slot * STAGE + sub * 2 * HALF;
                const int key0 = (s + sub) * STEP;
                // ---- scores
                float x[NT][4] = {};
                {
                    uint32_t wd[2][NG];
                    load_words<NG>(at + CODES + gi * NG * 4, wd);
                    if constexpr (BY_WORDS) {
                        uint32_t c[4];
                        if constexpr (NG == 4) ldmatrix_x2(at + CODES + (lane & 15) * 16, c);
                        else ldmatrix_x4(at + CODES + (lane & 15) * 32 + (lane >> 4) * 16, c);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            if constexpr (NG == 4) {
                                mma0(x[j], c[0], c[1], c[0], c[1], qw[j][0], qw[j][1]);
                            } else {
                                mma0(x[j], c[0], c[1], c[2], c[3], qw[j][0], qw[j][2]);
                                mma(x[j], c[0], c[1], c[2], c[3], qw[j][1], qw[j][3]);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NG; n += 2) {
                        uint32_t c[4];                     // keys 0..7 and 8..15 of a group, then of the next
                        ldmatrix_x4(at + (lane & 15) * 16 + (n + 1 < NG ? lane >> 4 : 0) * STEP * 16 + n * STEP * 16, c);
#pragma unroll
                        for (int u = 0; u < 2 && n + u < NG; ++u) {
                            const uint32_t a = c[2 * u], b = c[2 * u + 1], a8 = a >> 8, b8 = b >> 8;
                            const float sa = scale_of(wd[0][n + u]), sb = scale_of(wd[1][n + u]);
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                float d[4];
                                mma0(d, a & LOW, b & LOW, a & HIGH, b & HIGH, qf[j][n + u][0], qf[j][n + u][1]);
                                mma(d, a8 & LOW, b8 & LOW, a8 & HIGH, b8 & HIGH, qf[j][n + u][2], qf[j][n + u][3]);
                                if constexpr (!BY_WORDS) {
                                    const float ma = least_of(wd[0][n + u]), mb = least_of(wd[1][n + u]);
                                    x[j][0] = fmaf(ma, qsum[j][n + u][0], x[j][0]);
                                    x[j][1] = fmaf(ma, qsum[j][n + u][1], x[j][1]);
                                    x[j][2] = fmaf(mb, qsum[j][n + u][0], x[j][2]);
                                    x[j][3] = fmaf(mb, qsum[j][n + u][1], x[j][3]);
                                }
                                x[j][0] = fmaf(sa, d[0], x[j][0]);
                                x[j][1] = fmaf(sa, d[1], x[j][1]);
                                x[j][2] = fmaf(sb, d[2], x[j][2]);
                                x[j][3] = fmaf(sb, d[3], x[j][3]);
                            }
                        }
                    }
                }
                // ---- probabilities times 2^44: element e of x is key gi + 8 (e / 2), column 2 ti + e % 2
                uint32_t seen = 0xffffffffu;               // bit 4 j + e
                if constexpr (MASKED) {
                    seen = 0;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + gi + 8 * (e >> 1), row = min(j * 8 + 2 * ti + (e & 1), rows - 1), pos = w.r.first_pos + token_of(A, row0 + row);
                            const bool is = !(lost >> (e >> 1) & 1) && key < w.r.keys && key <= pos && key >= first_seen(A, pos);
                            seen |= is ? 1u << (4 * j + e) : 0u;
                        }
                }
                bool higher = false;
                float p[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[j][e] = fmaf(x[j][e], c1[j][e & 1], base[j][e & 1]);
                        higher |= !(p[j][e] <= TOP);       // (a score that is no number is one too)
                    }
                if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float x0 = seen >> (4 * j + e) & 1 ? x[j][e] * c1[j][e] : -INFINITY, x1 = seen >> (4 * j + e + 2) & 1 ? x[j][e + 2] * c1[j][e] : -INFINITY;
                            float top = max_nan(x0, x1);
                            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 4));
                            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 8));
                            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 16));
                            const float now = UP - top;
                            if (!(now >= base[j][e])) {    // (smaller, or no number)
                                const float f = base[j][e] == INFINITY ? 0.f : xbtc::ex2(now - base[j][e]);
                                base[j][e] = now;
                                l[j][e] *= f;
                                eight[j][e] *= f, eight[j][e + 2] *= f;
#pragma unroll
                                for (int n = 0; n < (BY_WORDS ? 0 : NG); ++n) rest[j][n][e] *= f;
                                both[j][e] *= f, both[j][e + 2] *= f;
#pragma unroll
                                for (int n = 0; n < 2 * NG; ++n) o[j][n][e] *= f, o[j][n][e + 2] *= f;
                            }
                            p[j][e] = base[j][e] == INFINITY ? -INFINITY : fmaf(x[j][e], c1[j][e], base[j][e]);
                            p[j][e + 2] = base[j][e] == INFINITY ? -INFINITY : fmaf(x[j][e + 2], c1[j][e], base[j][e]);
                        }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[j][e] = xbtc::ex2(p[j][e]);
                if constexpr (MASKED) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!(seen >> (4 * j + e) & 1)) p[j][e] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) l[j][0] += p[j][0] + p[j][2], l[j][1] += p[j][1] + p[j][3];
                // ---- values
                {
                    uint32_t wd[2][NG];
                    load_words<NG>(at + HALF + CODES + gi * NG * 4, wd);
                    // (what a row does not see must not reach it, whatever it is: zero times no number is no number)
                    if constexpr (BY_WORDS) {
                        uint32_t c[4];
                        if constexpr (NG == 4) ldmatrix_x2_t(at + HALF + CODES + (lane & 15) * 16, c);
                        else ldmatrix_x4_t(at + HALF + CODES + (lane & 15) * 32 + (lane >> 4) * 16, c);
                        if constexpr (MASKED) {            // those who see words that are no numbers get one by p s
#pragma unroll
                            for (int i = 0; i < NG / 2; ++i) c[i] = finite_halves(c[i]);
                        }
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const uint32_t h0 = xbtc::pack_bf16(p[j][0], p[j][1]), h1 = xbtc::pack_bf16(p[j][2], p[j][3]);
                            const uint32_t r0 = pack_rest(p[j][0], p[j][1], h0), r1 = pack_rest(p[j][2], p[j][3], h1);
                            const uint32_t p0 = transposed(h0), p1 = transposed(h1), q0 = transposed(r0), q1 = transposed(r1);
                            mma(both[j], c[0], NG == 4 ? 0u : c[2], c[1], NG == 4 ? 0u : c[3], p0, p1);
                            mma(both[j], c[0], NG == 4 ? 0u : c[2], c[1], NG == 4 ? 0u : c[3], q0, q1);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NG; n += 2) {
                        uint32_t c[4];
                        ldmatrix_x4_t(at + HALF + (lane & 15) * 16 + (n + 1 < NG ? lane >> 4 : 0) * STEP * 16 + n * STEP * 16, c);
#pragma unroll
                        for (int u = 0; u < 2 && n + u < NG; ++u) {
                            const uint32_t a = c[2 * u], b = c[2 * u + 1], a8 = a >> 8, b8 = b >> 8;
                            const float sa = scale_of(wd[0][n + u]), sb = scale_of(wd[1][n + u]);
                            const uint32_t mine = gi == n + u ? 0x00080008u : 0u;          // 8 2^-133 in the group's row
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                float y[4] = {p[j][0] * sa, p[j][1] * sa, p[j][2] * sb, p[j][3] * sb};
                                if constexpr (MASKED) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        const uint32_t word = wd[e >> 1][n + u];
                                        y[e] = !(seen >> (4 * j + e) & 1) ? 0.f : (finite_halves(word) == word ? y[e] : __uint_as_float(0x7fffffffu));
                                    }
                                }
                                if constexpr (!BY_WORDS) {
                                    const float ma = fmaf(sa, 8.f, least_of(wd[0][n + u])), mb = fmaf(sb, 8.f, least_of(wd[1][n + u]));
                                    if constexpr (!MASKED) {
                                        rest[j][n + u][0] = fmaf(p[j][0], ma, fmaf(p[j][2], mb, rest[j][n + u][0]));
                                        rest[j][n + u][1] = fmaf(p[j][1], ma, fmaf(p[j][3], mb, rest[j][n + u][1]));
                                    } else {
#pragma unroll
                                        for (int e = 0; e < 4; ++e)
                                            if (seen >> (4 * j + e) & 1) rest[j][n + u][e & 1] = fmaf(p[j][e], e < 2 ? ma : mb, rest[j][n + u][e & 1]);
                                    }
                                }
                                const uint32_t p0 = transposed(xbtc::pack_bf16(y[0], y[1])), p1 = transposed(xbtc::pack_bf16(y[2], y[3]));
                                mma(o[j][2 * (n + u)], a & LOW, a & HIGH, b & LOW, b & HIGH, p0, p1);
                                mma(o[j][2 * (n + u) + 1], a8 & LOW, a8 & HIGH, b8 & LOW, b8 & HIGH, p0, p1);
                                mma(eight[j], mine, 0u, mine, 0u, p0, p1);
                            }
                        }
                    }
                }
            };
#pragma unroll 1
            for (int sub = 0; sub < STAGE_STEPS && s + sub < to; ++sub) {
                const unsigned lost = by16 ? (none >> sub & 1) * 3u : none >> (2 * sub) & 3u;
                const int key0 = (s + sub) * STEP;
                if (lost || key0 < all0 || key0 + STEP > all1) step(std::true_type(), sub, lost);
                else step(std::false_type(), sub, 0u);
            }
            __syncwarp();
            take_slot = take_slot + 1 == STAGES ? 0 : take_slot + 1;
            if (take_slot == 0) take_parity ^= 1;
            if (put < to) issue();
        }
        // ---- the segment's result: whole rows, or a part
        const bool whole = w.i0 == 0 && w.i1 == w.tiles;
        const size_t part = (size_t)me * 2 + (w.from > w.job ? 0 : 1);
        // the sums' sizes: those of an ordinary column are finite, and not all below 2^-28 of its sum of probabilities
        bool large = false, small = false;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float of_words = 0.f, of_p = l[j][e];
                if constexpr (BY_WORDS) of_words = max_nan(fabsf(both[j][e]), fabsf(both[j][e + 2]));
#pragma unroll
                for (int n = 0; n < (BY_WORDS ? 0 : NG); ++n) of_words = max_nan(of_words, fabsf(rest[j][n][e]));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) of_words = max_nan(of_words, __shfl_xor_sync(0xffffffffu, of_words, o)), of_p += __shfl_xor_sync(0xffffffffu, of_p, o);
                // (2^120: the lanes' parts are added up yet)
                large |= !(max_nan(of_words, max_nan(fabsf(eight[j][e]), fabsf(eight[j][e + 2]))) < 0x1p120f);
                small |= of_p > 0.f && of_words <= 0x1p-28f * of_p;
            }
        large = __any_sync(0xffffffffu, large), small = __any_sync(0xffffffffu, small);
        bool ordinary = true;
        if (!failed && (large || small)) {
            const uint32_t most = size_of_values<NG>(A, w.b, w.g, max(from * STEP, first_key), min(min(to * STEP, pos1 + 1), w.r.keys));
            ordinary = large ? most < VALUES_TO : most == 0;       // (if it is not the values it is the queries or keys)
        }
        if (!ordinary) rows_by_number<NG>(A, w.b, w.g, row0, rows, max(from * STEP, first_key), to * STEP, whole ? nullptr : line.part_o + part * ROWS * DP, line.part_ml + part * ROWS * 2);
        if (ordinary) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = j * 8 + 2 * ti + e;
                float sum = l[j][e];
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
                sum *= DOWN;
                const float inv = whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
                const long long t = w.r.first + token_of(A, row0 + min(row, rows - 1));
                __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out) + t * A.out_stride + (long long)(w.g * group + (row0 + row - token_of(A, row0 + row) * group)) * A.d;
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    float r;
                    if constexpr (BY_WORDS) {
                        const float s8 = __shfl_sync(0xffffffffu, both[j][e + (n >= 4 ? 2 : 0)], (2 * n & 7) * 4 + ti);
                        r = fmaf(8.f, s8, __shfl_sync(0xffffffffu, both[j][e + (n >= 4 ? 2 : 0)], ((2 * n & 7) + 1) * 4 + ti));
                    } else {
                        r = rest[j][n][e];
#pragma unroll
                        for (int s = 4; s < 32; s <<= 1) r += __shfl_xor_sync(0xffffffffu, r, s);
                    }
                    r *= DOWN;
                    const float minus = __shfl_sync(0xffffffffu, eight[j][e], n * 4 + ti);
                    const float v[4] = {fmaf(o[j][2 * n][e] - minus, BACK, r) * inv, fmaf(o[j][2 * n][e + 2] * 0.0625f - minus, BACK, r) * inv,
                                        fmaf(o[j][2 * n + 1][e] - minus, BACK, r) * inv, fmaf(o[j][2 * n + 1][e + 2] * 0.0625f - minus, BACK, r) * inv};
                    const int c = 32 * n + 4 * gi;
                    if (row >= rows) continue;
                    if (!whole) {
                        *reinterpret_cast<float4*>(line.part_o + (part * ROWS + row) * DP + c) = make_float4(v[0], v[1], v[2], v[3]);
                    } else if (out8) {
                        if (c < A.d) *reinterpret_cast<uint2*>(out + c) = make_uint2(xbtc::pack_bf16(v[0], v[1]), xbtc::pack_bf16(v[2], v[3]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (c + i < A.d) out[c + i] = __float2bfloat16_rn(v[i]);
                    }
                }
                // (minus infinity: there is nothing)
                if (!whole && gi == 0 && row < rows) *reinterpret_cast<float2*>(line.part_ml + (part * ROWS + row) * 2) = make_float2(UP - base[j][e], sum);
            }
        }
        if (!whole && lane == 0) {
            int* job = line.jobs + part * JOB_WORDS;
            const int first_warp = w.job / w.share, last = (w.job + w.tiles - 1) / w.share;
            job[1] = first_warp, job[2] = row0, job[3] = rows, job[4] = w.g, job[5] = w.r.first;
            job[0] = last - first_warp + 1;
        }
    }
}

// A job's parts, joined in the order of the line: a warp for every part takes its share of the job's numbers, and as many lanes for a number as leave
// one trip.
template <int NT, int NG>
__global__ void __launch_bounds__(THREADS)
cache4_attention_join_kernel(const AttendArgs A, const Line line) {
    constexpr int ROWS = 8 * NT, DP = 32 * NG, FOURS = DP / 4;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, entry = (int)blockIdx.x * WARPS + ((int)threadIdx.x >> 5);
    const int* job = line.jobs + (size_t)entry * JOB_WORDS;
    const int4 head = *reinterpret_cast<const int4*>(job);
    const int2 more = *reinterpret_cast<const int2*>(job + 4);
    const int parts = head.x;
    if (parts < 1) return;
    const int first = head.y, row0 = head.z, rows = head.w, g = more.x, group = A.group, first_token = more.y;
    const int mine = entry / 2 - first, total = rows * FOURS;
    auto part_of = [&](int i) { return (size_t)(first + i) * 2 + (i == 0 ? 1 : 0); };     // (the first part is its warp's last segment)
    const int lo = (int)((long long)total * mine / parts), hi = (int)((long long)total * (mine + 1) / parts);
    int lanes = 1;
    while (lanes < 16 && lanes * 2 * (hi - lo) <= 32 && lanes < parts) lanes *= 2;
    const int sub = lane & (lanes - 1);
    for (int i0 = lo; i0 < hi; i0 += 32 / lanes) {
        const int i = min(i0 + lane / lanes, hi - 1), row = i / FOURS, c = i % FOURS * 4;
        float top = -INFINITY, sum = 0.f;
        float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = sub; k < parts; k += lanes) {
            const size_t at = part_of(k) * ROWS + row;
            const float2 ml = *reinterpret_cast<const float2*>(line.part_ml + at * 2);
            const float4 u = *reinterpret_cast<const float4*>(line.part_o + at * DP + c);
            if (ml.x == -INFINITY) continue;                   // (a part of nothing)
            const float now = max_nan(top, ml.x), a = xbtc::ex2(top - now), f = xbtc::ex2(ml.x - now);
            top = now;
            sum = fmaf(f, ml.y, sum * a);
            v.x = fmaf(f, u.x, v.x * a), v.y = fmaf(f, u.y, v.y * a), v.z = fmaf(f, u.z, v.z * a), v.w = fmaf(f, u.w, v.w * a);
        }
        for (int s = 1; s < lanes; s <<= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, top, s), now = max_nan(top, other);
            const float a = now == -INFINITY ? 0.f : xbtc::ex2(top - now), f = now == -INFINITY ? 0.f : xbtc::ex2(other - now);
            top = now;
            sum = sum * a + __shfl_xor_sync(0xffffffffu, sum, s) * f;
            v.x = v.x * a + __shfl_xor_sync(0xffffffffu, v.x, s) * f, v.y = v.y * a + __shfl_xor_sync(0xffffffffu, v.y, s) * f;
            v.z = v.z * a + __shfl_xor_sync(0xffffffffu, v.z, s) * f, v.w = v.w * a + __shfl_xor_sync(0xffffffffu, v.w, s) * f;
        }
        if (sub || i0 + lane / lanes >= hi) continue;
        const int token = token_of(A, row0 + row);
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out) + (long long)(first_token + token) * A.out_stride + (long long)(g * group + row0 + row - token * group) * A.d;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < A.d) out[c + e] = __float2bfloat16_rn(y[e]);
    }
}

template <int NT, int NG>
long long scratch_of() {
    return (long long)blocks_of(NT, NG) * WARPS * 2 * (8 * NT * (32 * NG + 2) + JOB_WORDS);
}

template <int NT, int NG>
int launch(const AttendArgs& A, float* scratch, cudaStream_t stream) {
    constexpr int blocks = blocks_of(NT, NG), parts = blocks * WARPS * 2;
    Line line;
    line.part_o = scratch;
    line.part_ml = scratch + (size_t)parts * 8 * NT * 32 * NG;
    line.jobs = reinterpret_cast<int*>(line.part_ml + (size_t)parts * 8 * NT * 2);
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(cache4_attention_mma_kernel<NT, NG>, smem_bytes(NG), &roomy)) return rc;
    const int rc = xb_launch(cache4_attention_mma_kernel<NT, NG>, dim3(blocks), dim3(THREADS), smem_bytes(NG), stream, A, line);
    if (rc) return rc;
    return xb_launch(cache4_attention_join_kernel<NT, NG>, dim3(parts / WARPS), dim3(THREADS), 0, stream, A, line);
}

// Eight rows a job where no request brings more, else sixteen (a cache read once for sixteen: 8 requests of up to 16 rows at up to 4,096 keys 26 us); heads of 256 channels always eight, whose sums alone are 64 registers a thread.
template <typename F>
auto by_form(int rows, int groups, F f) {
    const std::integral_constant<int, 1> one{};
    const std::integral_constant<int, 2> two{};
    auto with = [&](auto ng) { return rows <= 8 ? f(one, ng) : f(two, ng); };
    switch (groups) {
        case 1: return with(std::integral_constant<int, 1>());
        case 2: return with(std::integral_constant<int, 2>());
        case 3: return with(std::integral_constant<int, 3>());
        case 4: return with(std::integral_constant<int, 4>());
        default: return f(one, std::integral_constant<int, 8>());
    }
}

}  // namespace

namespace xb4 {

bool mma_takes(int d) { return groups_of(d) <= 4 || groups_of(d) == 8; }
bool mma_takes(const AttendArgs& A) {
    // the longest line that these shapes allow is counted in 32 bits
    const double jobs = (double)A.nkv * ((double)A.tokens * A.group / 8 + A.requests), tiles = (double)A.table_stride * A.page_size / KT + 2;
    return mma_takes(A.d) && tokens_of_rows(A) && A.page_size % 8 == 0 && A.num_pages > 0 && jobs * (tiles + COST_JOB) < LINE_MOST;
}
long long mma_scratch(int d, int rows) {
    return by_form(rows, groups_of(d), [](auto nt, auto ng) { return scratch_of<decltype(nt)::value, decltype(ng)::value>(); });
}
int mma_launch(const AttendArgs& A, int rows, float* scratch, cudaStream_t stream) {
    return by_form(rows, groups_of(A.d), [&](auto nt, auto ng) { return launch<decltype(nt)::value, decltype(ng)::value>(A, scratch, stream); });
}

}  // namespace xb4
