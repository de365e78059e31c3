// Attention over 4-bit pages for many rows of a key/value head (portions of prompts, bfloat16) on the 5th-generation tensor cores
// (cache4_attention.cu says what is computed).
//
// A job is (request, key/value head, up to two tiles of 128 rows): the rows are (token, query head of the group) pairs.  Warps 8..11 take tiles of 64
// keys and warps 12..15 tiles of 64 values out of their codes, once for the 256 rows, into operands in shared memory (128-byte swizzle); S = Q K^T is issued by
// warp 16, P = 2^(S - m) formed by a thread per row in warps 0..3 and 4..7, in the tensor memory of S, O += P V issued by warp 17.
//
// All operands are float16: 11 digits of m + s code and of a probability, where bfloat16's 8 would each move the result as much as its own rounding
// does.  float16's range is made up for by powers of two that are undone in float32: one per row of Q; one for every 16 keys of a tile, by which the
// scores are multiplied; one for every 16 values, by which probabilities are multiplied, relative to the largest so far (which moves O as a new
// maximum does).  Probabilities are held 2^6 times their size.  Keys and values much smaller than others lose digits, whoever sees those: keys beside ones of 2^24 times
// their size among sixteen; values beside ones of 2^r times theirs have probabilities that are off by 2^(r - 31) of the largest, which many small ones feel first
// (2,000 of 2^-13.4 at r = 16: 5 % of the result).  A block whose keys or values differ by more than K_RANGE and V_RANGE says so, and its requests are done again by
// the kernel that takes the rest of the step (cache4_attention.cu).
// A group's word that is no number is zero in the operand; rows that see its key get no number in the group's channels at the end, the others nothing.
//
// The tiles of all jobs are one line cut into equal shares, one a block; parts of a job that blocks share are joined by a second kernel in their order.
//
// Bound by the softmax warps, 3,400 cycles for a tile of 64 keys and 256 rows (1,500 of them the exponentials), and by a job's start and end, 20,000 cycles.  Four
// requests of up to 512 tokens at up to 4,096 keys, 32 heads over 8 of 128 channels: 106 us, a quarter of the products' rate.
#include <cuda_fp16.h>

#include "cache4_attention_tc.h"
#include "tc_common.cuh"

namespace {

using namespace xb4;
using namespace xbtc;

constexpr int RT = 128, ROWS = 2 * RT, KT = 64;
constexpr int BLOCKS = 148, THREADS = 576, NS = 3;
constexpr int COST_JOB = 6;                // a job's start and end take about as long as six tiles
constexpr float RESCALE_STEP = 8.f;
constexpr int JOB_WORDS = 8, INFOS = 8;    // (a tile's facts are read at most NS + 2 tiles after they are written)
constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;
constexpr float P_UP = 6.f;
constexpr int RAW = 3;                     // tiles whose codes are on their way

struct Line {
    float* part_o;                 // [blocks][2][DP / 4][256][4]: a block's first segment, if its job began before it, and its last, if its job goes on
    float* part_ml;                // [blocks][2][256][2]
    int* jobs;                     // [blocks][2][8]: parts (0: there is no such part), block of the first, first row, rows, key/value head, request
    int* wide;                     // AttendArgs::wide of the kernel that follows
};
// Exponents of the largest number that a key and a value holds may differ by that much among those that a block meets, and be that small (2^-100).
constexpr int K_RANGE = 22, V_RANGE = 12, LEAST = 127 - 100;

// What the softmax needs to know of a tile's keys and values.
struct __align__(16) Info {
    float k_back[4];               // what the scores of every 16 keys are multiplied by,
    float v_back[4];               // and what comes of every 16 values
    unsigned short there[4];       // keys that lie in a page
    unsigned short odd[4];         // keys whose values have a group that is no number,
    unsigned char groups[KT];      // and which groups
};

struct Walk {
    Request r;
    int b, g, piece, pieces;
    int tile0, tiles;              // of the job
    int job, from, end, share;
    int i0, i1;
};

// Keys and tiles of a request's piece of rows, from the places of its first and its last token.
__device__ __forceinline__ void set_tiles(const AttendArgs& A, Walk& w, int node0, int node1) {
    w.tile0 = first_seen(A, w.r.first_pos + node0) / KT;
    w.tiles = max(1, (min(w.r.first_pos + node1 + 1, w.r.keys) + KT - 1) / KT - w.tile0);       // (rows that see no key are written all the same)
}
__device__ __forceinline__ void set_piece(const AttendArgs& A, Walk& w) {
    const int row0 = w.piece * ROWS;
    set_tiles(A, w, token_of(A, row0), min(w.r.nodes - 1, token_of(A, row0 + ROWS - 1)));
}
__device__ __forceinline__ void set_request(const AttendArgs& A, Walk& w, int b) {
    w.b = b;
    w.r = request_of<false>(A, b);
    w.pieces = (w.r.nodes * A.group + ROWS - 1) / ROWS;
}
// The pieces one after another, until `f(piece)` is true: their tokens' places by sums.
template <typename F>
__device__ __forceinline__ void each_piece(const AttendArgs& A, Walk& w, F f) {
    const int group = A.group, quo = ROWS / group, rem = ROWS % group;
    int node = 0, over = 0;        // (256 * piece) / group and the remainder
#pragma unroll 1
    for (w.piece = 0; w.piece < w.pieces; ++w.piece) {
        int next = node + quo, left = over + rem;
        if (left >= group) left -= group, ++next;
        set_tiles(A, w, node, min(w.r.nodes - 1, left == 0 ? next - 1 : next));        // (the last row is one before the next piece's first)
        if (f()) return;
        node = next, over = left;
    }
}
__device__ __forceinline__ int head_units(const AttendArgs& A, Walk& w) {
    int sum = 0;
    each_piece(A, w, [&]() {
        sum += w.tiles + COST_JOB;
        return false;
    });
    return sum;
}

__device__ __forceinline__ bool place_in_line(const AttendArgs& A, Walk& w) {
    const int lane = threadIdx.x & 31, each = (A.requests + 31) / 32, b0 = lane * each, b1 = min(b0 + each, A.requests);
    long long mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        set_request(A, w, b);
        mine += (long long)A.nkv * head_units(A, w);
    }
    int incl;
    const int total = prefix_of_lanes(A, mine, incl);
    if (total < 0) return false;
    w.share = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    w.from = (int)min((long long)blockIdx.x * w.share, (long long)total);
    w.end = min(total, w.from + w.share);
    if (w.from >= w.end) return false;
    int before = incl - (int)mine, b = b0;
    const int owner = __ffs(__ballot_sync(0xffffffffu, w.from >= before && w.from < incl)) - 1;
    if (lane == owner) {
#pragma unroll 1
        for (; b < b1; ++b) {
            set_request(A, w, b);
            const int n = A.nkv * head_units(A, w);
            if (w.from < before + n) break;
            before += n;
        }
    }
    set_request(A, w, __shfl_sync(0xffffffffu, b, owner));
    before = __shfl_sync(0xffffffffu, before, owner);
    const int units = head_units(A, w);
    w.g = (w.from - before) / units;
    w.job = before + w.g * units;
    each_piece(A, w, [&]() {
        if (w.from < w.job + w.tiles + COST_JOB) return true;
        w.job += w.tiles + COST_JOB;
        return false;
    });
    return true;
}

// The next job of which the block has tiles: those that begin in its share.
__device__ __forceinline__ bool next_segment(const AttendArgs& A, Walk& w, bool first) {
    for (;; first = false) {
        if (!first) {
            w.job += w.tiles + COST_JOB;
            if (w.job >= w.end) return false;
            if (++w.piece == w.pieces) {
                w.piece = 0;
                if (++w.g == A.nkv) {
                    w.g = 0;
                    do {
                        if (w.b + 1 >= A.requests) return false;
                        set_request(A, w, w.b + 1);
                    } while (w.pieces == 0);
                }
            }
            set_piece(A, w);
        }
        w.i0 = max(0, w.from - w.job);
        w.i1 = min(w.tiles, w.end - w.job);
        if (w.i0 < w.i1) return true;
    }
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
// Products issued by one lane of a warp that stays together.
__device__ __forceinline__ void umma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.eq.b32 p, 0, 0;\n\t"
        "setp.ne.b32 q, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(one) : "memory");
}
__device__ __forceinline__ void commit(uint32_t one, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(bar), "r"(one) : "memory");
}
// D float32, A and B float16, both K-major, M = 128, N = n
__device__ __forceinline__ uint32_t idesc_f16(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }

__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* err) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, true)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void tmem_st16_u(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t fma_f16(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t add_f16(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ void store16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ bool half_not_finite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ int exponent_of(float power) { return (int)(__float_as_uint(power) >> 23) - 127; }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }       // -126 <= e <= 127

// Copies of a key's words to shared memory, and from there.
template <int NG>
__device__ __forceinline__ void copy_words(uint32_t dst, const uint8_t* src) {
    if constexpr (NG == 4) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    } else {
#pragma unroll
        for (int n = 0; n < NG; ++n) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * n), "l"(src + 4 * n) : "memory");
    }
}
template <int NG>
__device__ __forceinline__ void load_words(uint32_t at, uint32_t (&w)[NG]) {
    if constexpr (NG == 4) {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    } else {
#pragma unroll
        for (int n = 0; n < NG; ++n) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[n]) : "r"(at + 4 * n) : "memory");
    }
}
// Eight numbers m + s code from a word, in their order.  (1,024 + c and 1,024 + 16 c are float16 numbers with the code's bits.)
__device__ __forceinline__ void store_word(uint32_t at, uint32_t c, uint32_t s2, uint32_t m2) {
    const uint32_t u8 = c >> 8;
    const uint32_t a = fma_f16(add_f16((c & LOW) | 0x64006400u, 0xe400e400u), s2, m2), b = fma_f16(fma_f16((c & HIGH) | 0x64006400u, 0x2c002c00u, 0xd400d400u), s2, m2);
    const uint32_t x = fma_f16(add_f16((u8 & LOW) | 0x64006400u, 0xe400e400u), s2, m2), y = fma_f16(fma_f16((u8 & HIGH) | 0x64006400u, 0x2c002c00u, 0xd400d400u), s2, m2);
    // (they come as 0 4, 1 5, 2 6, 3 7)
    store16(at, __byte_perm(a, b, 0x5410), __byte_perm(x, y, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(x, y, 0x7632));
}
template <int NG>
__global__ void __launch_bounds__(THREADS, 1)
cache4_attention_tc_kernel(const AttendArgs A, const Line line, float scale_log2) {
    constexpr int DP = NG <= 2 ? 64 : 128, HALVES = DP / 64;
    constexpr uint32_t Q_ONE = HALVES * RT * 128, KV_HALF = KT * 128, KV_BYTES = HALVES * KV_HALF, STAGE_BYTES = 2 * KV_BYTES;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ __align__(8) unsigned long long bars[4 * NS + 16];
    __shared__ uint32_t s_tmem;
    __shared__ Info infos[INFOS];
    __shared__ unsigned sizes[4];                  // bits of the least and the largest number that a key holds, and a value
    __shared__ int met[2];                         // the first and the last request
    constexpr uint32_t RAW_CODES = NG * KT * 16, RAW_BYTES = RAW_CODES + KT * NG * 4;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, q_sm = base, kv_sm = base + 2 * Q_ONE, raw_sm = kv_sm + NS * STAGE_BYTES;
    const uint32_t bar0 = smem_u32(bars), k_full0 = bar0, k_empty0 = bar0 + 8 * NS, v_full0 = bar0 + 16 * NS, v_empty0 = bar0 + 24 * NS, rest = bar0 + 32 * NS;
    const uint32_t s_ready0 = rest, pv_done0 = rest + 32, p_ready0 = rest + 64, q_ready0 = rest + 96, drained0 = rest + 112;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = A.group, ps = A.page_size;
    int* const err = A.err;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(k_full0 + 8 * i, 4), mbar_init(k_empty0 + 8 * i, 1), mbar_init(v_full0 + 8 * i, 4), mbar_init(v_empty0 + 8 * i, 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_ready0 + 8 * i, 1);
            mbar_init(pv_done0 + 8 * i, 1);
            mbar_init(p_ready0 + 8 * i, 4);        // a warp each
        }
        for (int i = 0; i < 2; ++i) mbar_init(q_ready0 + 8 * i, 4), mbar_init(drained0 + 8 * i, 1);
        mbar_init_fence();
    }
    if (threadIdx.x < 4) sizes[threadIdx.x] = threadIdx.x & 1 ? 0u : 0x7f800000u;
    if (threadIdx.x == 0) met[0] = 1, met[1] = 0;
    if (warp == 8) tmem_alloc(&s_tmem, 512);
    if (NG * 32 < DP)                              // channels that no group has: zeros for good (the products of Q and K go over them)
        for (uint32_t i = threadIdx.x * 16; i < NS * STAGE_BYTES; i += THREADS * 16) store16(kv_sm + i, 0, 0, 0, 0);
    fence_async_shared();
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();       // only now: see pdl_launch_dependents on tensor memory
    if (threadIdx.x < 2) line.jobs[(blockIdx.x * 2 + threadIdx.x) * JOB_WORDS] = 0;
    Walk w;
    const bool any = place_in_line(A, w);
    const long long page_bytes = (long long)ps * 20 * NG;

    if (warp >= 8 && warp < 16) {
        const bool is_v = warp >= 12;
        const uint32_t full0 = is_v ? v_full0 : k_full0, empty0 = is_v ? v_empty0 : k_empty0, raw0 = raw_sm + (is_v ? RAW * RAW_BYTES : 0u);
        // ---- codes to operands: a quarter of a tile's keys (warps 8..11) or values a warp, two lanes a key (the first and the second half of its groups)
        const int quarter = warp & 3, key = quarter * 16 + (lane & 15), part = lane >> 4;
        constexpr int GP = (NG + 1) / 2;           // groups of a lane, at most
        const int n0 = part * GP, n1 = min(NG, n0 + GP), quo = KT / ps, rem = KT % ps;
        int st = 0, done = 0;                      // ring stage, tiles
        uint32_t ph = 0;
        unsigned least = 0x7f800000u, most = 0u;   // of the lane's keys or values that are not all zero
        bool ok = any;
        if (any && threadIdx.x == 8 * 32) met[0] = w.b;
        for (bool first = true; ok && next_segment(A, w, first); first = false) {
            const int* table = A.block_table + (long long)w.b * A.table_stride;
            const uint8_t* pages = (is_v ? A.v_cache : A.k_cache) + w.g * page_bytes;
            const int first_key = first_seen(A, w.r.first_pos + token_of(A, w.piece * ROWS));       // (pages in front of it may have been given back)
            // the lane's key: its place in the table and in its page, kept up by sums
            int k = (w.tile0 + w.i0) * KT + key, at = k / ps, slot = k % ps, asked = w.i0, slot_in = 0, slot_out = 0;       // tiles asked for, their places in the ring
            unsigned have = 0;                     // whether the key is there, a bit a tile, the last asked for lowest
            auto look = [&]() { return asked < w.i1 && k < w.r.keys && k >= first_key ? table[at] : -1; };
            int id = look();
            auto ask = [&]() {
                const bool there = id >= 0 && id < A.num_pages;
                if (!there && asked < w.i1 && k < w.r.keys && k >= first_key) atomicOr(err, XB_ERR_BAD_PAGE);
                have = have << 1 | (there ? 1u : 0u);
                if (there) {
                    const uint32_t to = raw0 + slot_in * RAW_BYTES;
                    const uint8_t* from = pages + (long long)id * A.nkv * page_bytes;
#pragma unroll
                    for (int g = 0; g < GP; ++g)
                        if (n0 + g < n1)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to + ((n0 + g) * KT + key) * 16), "l"(from + ((n0 + g) * ps + slot) * 16) : "memory");
                    if (part == 0) copy_words<NG>(to + RAW_CODES + key * NG * 4, from + ps * 16 * NG + slot * NG * 4);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                k += KT;
                slot += rem;
                at += quo;
                if (slot >= ps) slot -= ps, ++at;
                ++asked;
                slot_in = slot_in + 1 == RAW ? 0 : slot_in + 1;
                id = look();
            };
#pragma unroll
            for (int i = 0; i < RAW - 1; ++i) ask();
            for (int it = w.i0; it < w.i1; ++it) {
                ask();
                asm volatile("cp.async.wait_group %0;" ::"n"(RAW - 1) : "memory");
                __syncwarp();
                const bool there = have >> (RAW - 1) & 1u;
                const uint32_t raw = raw0 + slot_out * RAW_BYTES;
                slot_out = slot_out + 1 == RAW ? 0 : slot_out + 1;
                uint32_t words[NG];
                load_words<NG>(raw + RAW_CODES + key * NG * 4, words);
                // the power of two that brings the largest number that these 16 keys or values can hold below 2^15
                float top = 0.f;
                unsigned odd = 0;
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    if (!there) words[n] = 0u;
                    const bool strange = half_not_finite(words[n]);
                    top = fmaxf(top, strange ? 0.f : fmaf(15.f, fabsf(scale_of(words[n])), fabsf(least_of(words[n]))));
                    if (strange && is_v) odd |= 1u << n, words[n] = 0u;
                }
                most = max(most, __float_as_uint(top));
                least = min(least, top > 0.f ? __float_as_uint(top) : 0x7f800000u);
                const int expo = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23), e = expo == 0 ? 100 : min(141 - expo, 100);
                const float f = power_of_two(e);
                const unsigned bits = __ballot_sync(0xffffffffu, is_v ? odd != 0 : there);
                if (done >= NS) ok = wait_warp(empty0 + 8 * st, ph ^ 1u, err);
                if (!ok) break;
                Info& info = infos[done % INFOS];
                if (lane == 0) (is_v ? info.v_back : info.k_back)[quarter] = power_of_two(-e), (is_v ? info.odd : info.there)[quarter] = (unsigned short)bits;
                if (is_v && bits && part == 0) info.groups[key] = (unsigned char)odd;
                const uint32_t row = kv_sm + st * STAGE_BYTES + (is_v ? KV_BYTES : 0u) + key * 128;
#pragma unroll
                for (int g = 0; g < GP; ++g) {
                    const int n = n0 + g;
                    if (n < n1) {
                        const uint32_t wd = part ? words[min(GP + g, NG - 1)] : words[g];
                        uint32_t c[4];
                        const float sc = scale_of(wd) * f, m = least_of(wd) * f;
                        const uint32_t s2 = pack_f16(sc, sc), m2 = pack_f16(m, m);
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(raw + (n * KT + key) * 16) : "memory");
#pragma unroll
                        for (int i = 0; i < 4; ++i) store_word(row + (n >> 1) * KV_HALF + ((((n & 1) * 4 + i) ^ (key & 7)) << 4), c[i], s2, m2);
                    }
                }
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(full0 + 8 * st);
                ++done;
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
        }
        if (any && threadIdx.x == 8 * 32) met[1] = w.b;
        least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) atomicMin(&sizes[is_v ? 2 : 0], least), atomicMax(&sizes[is_v ? 3 : 1], most);
    } else if (warp == 16) {
        // ---- S = Q K^T of every tile
        const uint32_t one = elected(), tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t idesc = idesc_f16(KT);
        const uint64_t dq0 = umma_desc(q_sm, 16, 1024), dk0 = umma_desc(kv_sm, 16, 1024);
        int st = 0, Th[2] = {0, 0}, I = 0, I1 = 0;
        uint32_t ph = 0;
        bool ok = any;
        for (bool first = true; ok && next_segment(A, w, first); first = false, ++I) {
            const int halves = w.r.nodes * group - w.piece * ROWS > RT ? 2 : 1;
            ok = wait_warp(q_ready0, I & 1, err);
            if (halves == 2) ok = ok && wait_warp(q_ready0 + 8, I1++ & 1, err);
            for (int it = w.i0; it < w.i1 && ok; ++it) {
                ok = wait_warp(k_full0 + 8 * st, ph, err);
                const uint64_t dk = dk0 + (uint64_t)((st * STAGE_BYTES) >> 4);
                for (int hd = 0; hd < halves && ok; ++hd) {
                    const int th = Th[hd]++, sb = th & 1;
                    // these columns held the scores and then P of this half's last tile but one: its P V must have read them
                    ok = th < 2 || wait_warp(pv_done0 + 8 * (2 * hd + sb), ((th >> 1) - 1) & 1, err);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dq = dq0 + (uint64_t)((hd * Q_ONE) >> 4);
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk) {
                        const uint32_t off = (kk >> 2), inner = (kk & 3) * 32;
                        umma_ss(one, tmem_u + (uint32_t)(hd * 128 + sb * 64), dq + (uint64_t)((off * RT * 128 + inner) >> 4), dk + (uint64_t)((off * KV_HALF + inner) >> 4), idesc, kk ? 1u : 0u);
                    }
                    commit(one, s_ready0 + 8 * (2 * hd + sb));
                }
                if (!ok) break;
                commit(one, k_empty0 + 8 * st);
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        }
        commit(one, drained0);                   // no product is at work when the tensor memory is freed, however the block ends
        wait_warp(drained0, 0, err);
    } else if (warp == 17) {
        // ---- O += P V of every tile (O starts as zeros, by the softmax threads)
        const uint32_t one = elected(), tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t idesc = idesc_f16(DP) | 1u << 16;       // V lies channel by channel along its rows
        const uint64_t dv0 = umma_desc(kv_sm + KV_BYTES, KV_HALF, 1024);
        int st = 0, Th[2] = {0, 0};
        uint32_t ph = 0;
        bool ok = any;
        for (bool first = true; ok && next_segment(A, w, first); first = false) {
            const int halves = w.r.nodes * group - w.piece * ROWS > RT ? 2 : 1;
            for (int it = w.i0; it < w.i1 && ok; ++it) {
                ok = wait_warp(v_full0 + 8 * st, ph, err);
                const uint64_t dv = dv0 + (uint64_t)((st * STAGE_BYTES) >> 4);
                for (int hd = 0; hd < halves && ok; ++hd) {
                    const int th = Th[hd]++, sb = th & 1;
                    ok = wait_warp(p_ready0 + 8 * (2 * hd + sb), (th >> 1) & 1, err);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t tp = tmem_u + (uint32_t)(hd * 128 + sb * 64);
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        umma_ts(one, tmem_u + (uint32_t)(256 + hd * 128), tp + (uint32_t)(kk * 8), dv + (uint64_t)((kk * 2048) >> 4), idesc);
                    commit(one, pv_done0 + 8 * (2 * hd + sb));
                }
                if (!ok) break;
                commit(one, v_empty0 + 8 * st);
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        }
        commit(one, drained0 + 8);
        wait_warp(drained0 + 8, 0, err);
    } else {
        // ---- softmax: a row per thread
        const int hd = warp >> 2, r = (int)threadIdx.x & 127;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + (uint32_t)(hd * 128) + lane_addr, tmem_o = tmem + (uint32_t)(256 + hd * 128) + lane_addr;
        const uint32_t my_s_ready = s_ready0 + 16 * hd, my_p_ready = p_ready0 + 16 * hd, my_pv_done = pv_done0 + 16 * hd;
        const bool q16 = ((uintptr_t)A.q & 15) == 0 && A.q_stride % 8 == 0 && A.d % 8 == 0, out16 = ((uintptr_t)A.out & 15) == 0 && A.out_stride % 8 == 0 && A.d % 8 == 0;
        int T = 0, Th = 0;                       // tiles of all segments so far, of this half's
        bool alive = any;
        for (bool first = true; alive && next_segment(A, w, first); first = false) {
            const int row0 = w.piece * ROWS, rows = min(ROWS, w.r.nodes * group - row0);
            if (rows <= hd * RT) {               // there is no second tile of rows
                T += w.i1 - w.i0;
                continue;
            }
            const int row = hd * RT + r;
            const bool valid = row < rows;
            const int of_request = row0 + min(row, rows - 1), pos = w.r.first_pos + token_of(A, of_request);
            const int lo = first_seen(A, pos), hi = min(pos + 1, w.r.keys);              // the keys that the row sees
            const long long t = w.r.first + token_of(A, of_request);
            const int head = w.g * group + of_request - token_of(A, of_request) * group;
            // Q: the last tile's scores of the last segment are there, so nothing reads what lies there
            float c1;
            {
                // (VPR lanes have a row, eight channels each, so that lanes read what lies together; eight trips are on their way at a time)
                constexpr int VPR = DP / 8, RPI = 32 / VPR, TRIPS = 32 / RPI;
                const int c = (lane % VPR) * 8, sub = lane / VPR, warp_row = hd * RT + (warp & 3) * 32;
                int e2 = 0, of = row0 + min(warp_row + sub, rows - 1), token = token_of(A, of), of_head = of - token * group;
                const int last = row0 + rows - 1;
#pragma unroll 1
                for (int i0 = 0; i0 < TRIPS; i0 += 8) {
                    uint4 u[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(A.q) + (w.r.first + token) * A.q_stride + (long long)(w.g * group + of_head) * A.d;
                        for (int j = 0; j < RPI && of < last; ++j) {       // (rows behind the last repeat it)
                            ++of;
                            if (++of_head == group) of_head = 0, ++token;
                        }
                        uint32_t x[4] = {0, 0, 0, 0};
                        if (q16) {
                            if (c < A.d) {
                                const uint4 v = *reinterpret_cast<const uint4*>(q + c);
                                x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (c + e < A.d) x[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[c + e] << (16 * (e & 1));
                        }
                        u[i] = make_uint4(x[0], x[1], x[2], x[3]);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t x[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
                        float top = 0.f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = max3_nan(top, fabsf(scale_of(x[e])), fabsf(least_of(x[e])));
#pragma unroll
                        for (int o = 1; o < VPR; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                        // the power of two that brings the row's largest number to 2^13 .. 2^14
                        const int expo = (int)(__float_as_uint(top) >> 23), e = expo < 255 && expo > 0 ? 140 - expo : 0;
                        const float f1 = power_of_two(e / 2), f2 = power_of_two(e - e / 2);
                        uint32_t y[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = pack_f16(scale_of(x[j]) * f1 * f2, least_of(x[j]) * f1 * f2);
                        const int to = (warp & 3) * 32 + (i0 + i) * RPI + sub;
                        store16(q_sm + hd * Q_ONE + (c >> 6) * (RT * 128) + to * 128 + ((((c >> 3) & 7) ^ (to & 7)) << 4), y[0], y[1], y[2], y[3]);
                        const int mine = __shfl_sync(0xffffffffu, e, (lane % RPI) * VPR);          // of the row of this trip that the lane may have
                        if (lane / RPI == i0 + i) e2 = mine;
                    }
                }
                c1 = scale_log2 * power_of_two(-(e2 / 2)) * power_of_two(-(e2 - e2 / 2));
                float zero[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) zero[i] = 0.f;
#pragma unroll
                for (int c0 = 0; c0 < DP; c0 += 32) tmem_st32(tmem_o + c0, zero);
                tmem_st_wait();
                fence_async_shared();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_ready0 + 8 * hd);
            }
            float m_ref = -INFINITY, l = 0.f, v_back = 0.f, v_down = 0.f;
            unsigned poison = 0;                 // groups of channels that are no number
            // keys from all0 on and below all1 are seen by all rows of the job
            const int pos0 = w.r.first_pos + token_of(A, row0), pos1 = w.r.first_pos + token_of(A, row0 + rows - 1);
            const int all0 = first_seen(A, pos1), all1 = min(pos0 + 1, w.r.keys);
            for (int it = w.i0; it < w.i1; ++it, ++Th) {
                const int sb = Th & 1, key0 = (w.tile0 + it) * KT;
                if (!wait_warp(my_s_ready + 8 * sb, (Th >> 1) & 1, err)) {
                    alive = false;
                    break;
                }
                tc_fence_after();
                const int vst = (T + it - w.i0) % NS;
                if (!wait_warp(v_full0 + 8 * vst, ((T + it - w.i0) / NS) & 1, err)) {      // (what is known of the values)
                    alive = false;
                    break;
                }
                const uint32_t info_at = smem_u32(&infos[(T + it - w.i0) % INFOS]);
                float cf[4], vf[4], v_most = v_back;
                unsigned t0, t1, o0, o1;
                asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(cf[0]), "=f"(cf[1]), "=f"(cf[2]), "=f"(cf[3]) : "r"(info_at) : "memory");
                asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(vf[0]), "=f"(vf[1]), "=f"(vf[2]), "=f"(vf[3]) : "r"(info_at + 16) : "memory");
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(t0), "=r"(t1), "=r"(o0), "=r"(o1) : "r"(info_at + 32) : "memory");
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    cf[i] = fminf(fmaxf(c1 * cf[i], 1.2e-38f), 3.0e38f);   // (a sum of zero stays one, and one of a key that is not seen)
                    v_most = fmaxf(v_most, vf[i]);
                }
                const bool edge = key0 < all0 || key0 + KT > all1 || (t0 & t1) != 0xffffffffu || (o0 | o1);
                unsigned long long seen = ~0ull;
                if (edge) {
                    seen = (unsigned long long)t1 << 32 | t0;
                    if (hi - key0 < 64) seen &= hi > key0 ? (1ull << (hi - key0)) - 1 : 0ull;
                    if (lo > key0) seen = lo - key0 < 64 ? seen & (~0ull << (lo - key0)) : 0ull;
                    unsigned long long odd = ((unsigned long long)o1 << 32 | o0) & seen;
                    while (odd) {
                        poison |= reinterpret_cast<volatile Info*>(infos)[(T + it - w.i0) % INFOS].groups[__ffsll((long long)odd) - 1];
                        odd &= odd - 1;
                    }
                }
                // twice over the scores, 32 at a time, so that they need not stay in registers: the largest, then the exponentials
                auto scores = [&](int half, float (&sc)[32]) {
                    tmem_ld32(tmem_s + sb * 64 + half * 32, sc);
                    if (edge) {
                        const unsigned mine = (unsigned)(seen >> (32 * half));
#pragma unroll
                        for (int i = 0; i < 32; ++i) sc[i] = (mine >> i & 1u) ? sc[i] : -INFINITY;
                    }
                };
                float top = -INFINITY;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float sc[32];
                    scores(half, sc);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            m2[0] = max3_nan(m2[0], sc[h * 16 + i], sc[h * 16 + i + 1]);
                            m2[1] = max3_nan(m2[1], sc[h * 16 + i + 2], sc[h * 16 + i + 3]);
                        }
                        top = max_nan(top, max_nan(m2[0], m2[1]) * cf[2 * half + h]);
                    }
                }
                float corr = 1.f;
                bool moved = false;
                if (!(top <= m_ref + RESCALE_STEP)) {                    // (a score that is no number makes the row one)
                    corr = m_ref == -INFINITY ? 0.f : ex2(m_ref - top);
                    moved = m_ref != -INFINITY && valid;                 // (O is zero before)
                    m_ref = top;
                }
                float f_o = corr;                // O's part: it is also in another power of two from now on
                if (v_most != v_back) {          // (the same for all)
                    if (v_back != 0.f) f_o *= v_back * power_of_two(-exponent_of(v_most)), moved = true;
                    v_back = v_most;
                    v_down = power_of_two(-exponent_of(v_most));
                }
                const float m_neg = m_ref == -INFINITY ? 0.f : P_UP - m_ref;
                const f32x2 mneg2 = pack2(m_neg, m_neg);
                f32x2 sum_a = pack2(0.f, 0.f), sum_b = pack2(0.f, 0.f);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float sc[32];
                    uint32_t pk[16];
                    scores(half, sc);
#pragma unroll
                    for (int c8 = 0; c8 < 4; ++c8) {
                        const f32x2 scale2 = pack2(cf[2 * half + c8 / 2], cf[2 * half + c8 / 2]);
                        const float of_v = vf[2 * half + c8 / 2] * v_down;
                        float e[8];
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            float x0, x1;
                            unpack2(fma2(pack2(sc[c8 * 8 + i], sc[c8 * 8 + i + 1]), scale2, mneg2), x0, x1);
                            e[i] = ex2(x0), e[i + 1] = ex2(x1);
                        }
                        sum_a = add2(sum_a, add2(pack2(e[0], e[1]), pack2(e[2], e[3])));
                        sum_b = add2(sum_b, add2(pack2(e[4], e[5]), pack2(e[6], e[7])));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float p0, p1;
                            unpack2(mul2(pack2(e[2 * i], e[2 * i + 1]), pack2(of_v, of_v)), p0, p1);
                            pk[c8 * 4 + i] = pack_f16(p0, p1);
                        }
                    }
                    tmem_st16_u(tmem_s + sb * 64 + half * 16, pk);       // P goes where scores were that have been read
                }
                float s0, s1, s2, s3;
                unpack2(sum_a, s0, s1);
                unpack2(sum_b, s2, s3);
                l = l * corr + ((s0 + s1) + (s2 + s3));
                // O is touched only when the last tile's P V has completed
                if (__any_sync(0xffffffffu, moved)) {
                    if (it > w.i0 && !wait_warp(my_pv_done + 8 * (sb ^ 1), ((Th - 1) >> 1) & 1, err)) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const float f = moved ? f_o : 1.f;
#pragma unroll 1
                    for (int c0 = 0; c0 < DP; c0 += 32) {
                        float o[32];
                        tmem_ld32(tmem_o + c0, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= f;
                        tmem_st32(tmem_o + c0, o);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(my_p_ready + 8 * sb);
            }
            T += w.i1 - w.i0;
            // ---- O / l, or this part of a job that blocks share
            if (alive) alive = wait_warp(my_pv_done + 8 * ((Th - 1) & 1), ((Th - 1) >> 1) & 1, err);
            if (!alive) break;
            tc_fence_after();
            const bool whole = w.i0 == 0 && w.i1 == w.tiles;
            const size_t part = (size_t)blockIdx.x * 2 + (w.from > w.job ? 0 : 1);
            const float f = whole ? (l > 0.f || l != l ? v_back / l : 0.f) : v_back;
            float* part_to = line.part_o + (part * (DP / 4) * ROWS + row) * 4;
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out) + t * A.out_stride + (long long)head * A.d;
#pragma unroll 1
            for (int c0 = 0; c0 < min(DP, NG * 32); c0 += 32) {
                float o[32];
                tmem_ld32(tmem_o + c0, o);
                const bool bad = poison >> (c0 / 32) & 1u;
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = bad ? __uint_as_float(0x7fffffffu) : o[i] * f;
                if (!valid) continue;
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(part_to + (size_t)(c0 + i) * ROWS) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else if (out16) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        if (c0 + i < A.d) *reinterpret_cast<uint4*>(out + c0 + i) = make_uint4(pack_bf16(o[i], o[i + 1]), pack_bf16(o[i + 2], o[i + 3]), pack_bf16(o[i + 4], o[i + 5]), pack_bf16(o[i + 6], o[i + 7]));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c0 + i < A.d) out[c0 + i] = __float2bfloat16_rn(o[i]);
                }
            }
            if (!whole && valid) *reinterpret_cast<float2*>(line.part_ml + (part * ROWS + row) * 2) = make_float2(m_ref, l);
            if (!whole && threadIdx.x == 0) {
                int* job = line.jobs + part * JOB_WORDS;
                const int first_block = w.job / w.share, last = (w.job + w.tiles - 1) / w.share;
                job[1] = first_block, job[2] = row0, job[3] = rows, job[4] = w.g, job[5] = w.b;
                job[0] = last - first_block + 1;
            }
            tc_fence_before();                   // (O has been read before it is written again)
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) tmem_free(tmem, 512);
    if (threadIdx.x == 0) {
        const int k0 = sizes[0] >> 23, v0 = sizes[2] >> 23;
        const bool wide = (int)(sizes[1] >> 23) - k0 > K_RANGE || (int)(sizes[3] >> 23) - v0 > V_RANGE || min(k0, v0) < LEAST;
        *reinterpret_cast<int2*>(line.wide + 2 + 2 * blockIdx.x) = wide ? make_int2(met[0], met[1]) : make_int2(1, 0);
    }
}

// A job's parts, joined in the order of the line: every part's blocks take a share of the job's numbers.
constexpr int JOIN_THREADS = 256, JOIN_BLOCKS = 4;

template <int NG>
__global__ void __launch_bounds__(JOIN_THREADS)
cache4_attention_tc_join_kernel(const AttendArgs A, const Line line) {
    constexpr int DP = NG <= 2 ? 64 : 128, FOURS = NG * 8;
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        const int2 met = threadIdx.x < BLOCKS ? *reinterpret_cast<const int2*>(line.wide + 2 + 2 * threadIdx.x) : make_int2(1, 0);
        const int any = __syncthreads_or(met.x <= met.y);
        if (threadIdx.x == 0) line.wide[0] = any;
    }
    const int* job = line.jobs + (size_t)blockIdx.x * JOB_WORDS;
    const int4 head = *reinterpret_cast<const int4*>(job);
    const int parts = head.x;
    if (parts < 1) return;
    const int first = head.y, row0 = head.z, rows = head.w, g = job[4], group = A.group;
    const Request r = request_of<false>(A, job[5]);
    // pieces of eight rows and sixteen channels, 32 lanes
    const int mine = ((int)blockIdx.x / 2 - first) * JOIN_BLOCKS + (int)blockIdx.y, shares = parts * JOIN_BLOCKS, total = (rows + 7) / 8 * (FOURS / 4);
    const int lane = threadIdx.x & 31;
    auto part_of = [&](int i) { return (size_t)(first + i) * 2 + (i == 0 ? 1 : 0); };     // (the first part is its block's last segment)
    for (int i = total * mine / shares + (int)(threadIdx.x >> 5); i < total * (mine + 1) / shares; i += JOIN_THREADS / 32) {
        const int row = i / (FOURS / 4) * 8 + (lane & 7), four = i % (FOURS / 4) * 4 + (lane >> 3), c = four * 4;
        if (row >= rows) continue;
        float top = -INFINITY, sum = 0.f;
        for (int k = 0; k < parts; ++k) top = max_nan(top, line.part_ml[(part_of(k) * ROWS + row) * 2]);
        float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < parts; ++k) {
            const size_t at = part_of(k) * ROWS + row;
            const float2 ml = *reinterpret_cast<const float2*>(line.part_ml + at * 2);
            const float4 u = *reinterpret_cast<const float4*>(line.part_o + ((part_of(k) * (DP / 4) + four) * ROWS + row) * 4);
            const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
            sum = fmaf(f, ml.y, sum);
            v.x = fmaf(f, u.x, v.x), v.y = fmaf(f, u.y, v.y), v.z = fmaf(f, u.z, v.z), v.w = fmaf(f, u.w, v.w);
        }
        const long long t = r.first + token_of(A, row0 + row);
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(A.out) + t * A.out_stride + (long long)(g * group + (row0 + row - token_of(A, row0 + row) * group)) * A.d;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < A.d) out[c + e] = __float2bfloat16_rn(y[e]);
    }
}

constexpr int dp_of(int d) { return d <= 64 ? 64 : 128; }

template <int NG>
int launch(const AttendArgs& A, float* scratch, cudaStream_t stream) {
    constexpr int DP = NG <= 2 ? 64 : 128, smem = (DP / 64) * (2 * RT * 128 + NS * 2 * KT * 128) + RAW * 2 * (NG * KT * 16 + KT * NG * 4) + 1024;
    Line line;
    line.part_o = scratch;
    line.part_ml = scratch + (size_t)BLOCKS * 2 * ROWS * DP;
    line.jobs = reinterpret_cast<int*>(line.part_ml + (size_t)BLOCKS * 2 * ROWS * 2);
    line.wide = const_cast<int*>(xb4::tc_wide(A.d, scratch));
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(cache4_attention_tc_kernel<NG>, smem, &roomy)) return rc;
    const int rc = xb_launch(cache4_attention_tc_kernel<NG>, dim3(BLOCKS), dim3(THREADS), smem, stream, A, line, A.scale * 1.4426950408889634f);
    if (rc) return rc;
    return xb_launch(cache4_attention_tc_join_kernel<NG>, dim3(2 * BLOCKS, JOIN_BLOCKS), dim3(JOIN_THREADS), 0, stream, A, line);
}

}  // namespace

namespace xb4 {

bool tc_takes(int nh, int nkv, int d, int longest) { return d <= 128 && (long long)longest * (nh / nkv) >= TC_ROWS; }
bool tc_takes(const AttendArgs& A, int longest) {
    // the longest line that these shapes allow is counted in 32 bits
    const double jobs = (double)A.nkv * ((double)A.tokens * A.group / ROWS + A.requests), tiles = (double)A.table_stride * A.page_size / KT + 2;
    return tc_takes(A.nh, A.nkv, A.d, longest) && tokens_of_rows(A) && A.scale > 0.f && A.num_pages > 0 && (long long)A.page_size * row_bytes(A.d) % 16 == 0 && jobs * (tiles + COST_JOB) < LINE_MOST;
}
static_assert(WIDE_PAIRS == BLOCKS && (2 + 2 * BLOCKS + 2) % 4 == 0 && BLOCKS <= JOIN_THREADS);
static long long wide_at(int d) { return (long long)BLOCKS * 2 * (ROWS * (dp_of(d) + 2) + JOB_WORDS); }
long long tc_scratch(int d) { return wide_at(d) + 2 + 2 * BLOCKS + 2; }
const int* tc_wide(int d, const float* scratch) { return reinterpret_cast<const int*>(scratch + wide_at(d)); }
int tc_launch(const AttendArgs& A, float* scratch, cudaStream_t stream) {
    switch (groups_of(A.d)) {
        case 1: return launch<1>(A, scratch, stream);
        case 2: return launch<2>(A, scratch, stream);
        case 3: return launch<3>(A, scratch, stream);
        default: return launch<4>(A, scratch, stream);
    }
}

}  // namespace xb4
