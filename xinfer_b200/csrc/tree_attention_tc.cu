// Attention of a tree of drafted tokens on the 5th-generation tensor cores, in bfloat16 (tree_attention.cu says what is computed).
//
// The nodes of a tree and the query heads of a key/value head are the rows of the products: a job is (request, key/value head, up to
// two tiles of 128 rows), so a tile of keys and values is read once for 256 rows.  Its keys are walked over in tiles of 64, the cached
// ones first, then the drafted ones, with a running maximum and sum per row (one thread a row) and O in tensor memory.
// Which rows see a drafted key is a bit per key: the row's words of ancestors.
//
// The tiles of all jobs are one line that is cut into equal shares, one per block (tree_attention.cuh).  A job that several blocks share
// leaves an unnormalised O with its maximum and sum per block; tree_merge_kernel joins them in their order.  One warp of a block forms the
// line, from three numbers per request, and tells the others of the block's parts of jobs.
//
// Per tile: S = Q K^T by warp 9, P = 2^(S - m) by warps 0..3 (first row tile) and 4..7 (second), in the tensor memory of S, O += P V by
// warp 11; warps 8 and 10 fetch keys and values, by page boxes from the cache and by boxes of 64 rows from the drafted rows.
// Barriers carry on from segment to segment, as do the rings.
//
// A value that a row does not see must not reach it, whatever it holds, but a product takes 0 * inf for NaN.  In tiles that not all rows
// see alike (drafted keys, the edge of a window) the value rows are looked at: those that hold an infinity or NaN are zeroed for the
// product, and the rows that do see them add their share to O by hand.  Value rows that nobody sees are zeroed too.
//
// What bounds it, and what it measured (bfloat16, 32 heads over 8 of 128 channels, pages of 16; both kernels, calls in a row):
//   48 trees of 24 nodes, up to 32,768 keys   391 us, 5.6 TB/s: the cache's bytes (tiles of one row tile take 1,350 cycles, the memory's rate).
//                                             Calls for seconds on end run into the power limit: at 1,450 MHz the cycles a tile are the bound, 466 us
//   64 trees of 8, up to 4,096                84 us, 4.6 TB/s: the same, with a job's start every 28 tiles
//   32 trees of 64, up to 8,192               113 us: jobs of two row tiles take about 2,000 cycles a tile of keys: exponentials (a quarter of them
//                                             by a polynomial), maxima and conversions of 64 scores a thread, two such warps to an issue slot
//   8 trees of 64, up to 4,096                33 to 35 us: 5 until the first scores, 14 of tiles, 2.4 to write the parts (19 MB at the L2's rate), 2.3
//                                             until the join's blocks are there, 7 of join
//   1 tree of 16, 1,024 keys (16 heads)       13.6 us: a chain of trips to memory.  In cycles: lengths 1,300, the place in the line 1,000, the
//                                             first segment 1,650, pages and the first tile 1,300, then four tiles, the part and the join
// A block reads 32 KB a tile with at least three tiles on their way, so boxes of both halves of a page (half as many copies) were no faster, and
// 5 % slower where memory is the bound.
#include "tc_common.cuh"
#include "tree_attention.cuh"

#include <type_traits>

namespace {

using namespace xbtc;
using namespace xbtree;

constexpr int RT = 128;                    // rows of a tile
constexpr int KT = 64;                     // keys of a tile
constexpr int LINE_BLOCKS = 148;           // a block per SM
constexpr float RESCALE_STEP = 8.f;        // a row's maximum moves only when it grows by more than 2^8
constexpr int THREADS = 384;
__host__ __device__ constexpr int stages(int dp) { return dp <= 64 ? 8 : 4; }

__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
    tmem_ld_wait();
    return r;
}

__host__ __device__ __forceinline__ bool rows_on_16_bytes(const void* p, long long stride) { return ((uintptr_t)p & 15) == 0 && stride % 8 == 0; }
__device__ __forceinline__ void store8(__nv_bfloat16* dst, const uint4& v, bool on16) {
    if (on16) {
        *reinterpret_cast<uint4*>(dst) = v;
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<uint16_t*>(dst)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
}

// where four channels of a part's row lie, in float4: those of eight rows together, as a warp writes and reads them
__device__ __forceinline__ size_t part_four(const Line& line, int d, size_t row, int c4) { return ((row >> 3) * (d >> 2) + c4) * 8 + (row & 7); }

// One lane of the warp, chosen by the hardware.
__device__ __forceinline__ uint32_t elected() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e;
}
// Products issued by one lane of a warp that stays together: their operands are then values of the warp, and an issue takes a few
// instructions (with the issue in a branch of one lane every operand is moved there, 100 cycles a product).
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
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// Whether one of eight bfloat16 is not finite: times zero it is no number, and stays so in a sum.
__device__ __forceinline__ bool any_not_finite(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(w[i]), "r"(0u));
    return (sum & 0x7fff7fffu) != 0u;
}
// The largest of three; one that is no number wins.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Bounded waits, with the way that is taken when the barrier is not yet there outside the loops' code.
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, int* err) { return mbar_wait(bar, parity, err); }
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int* err) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok ? true : wait_long(bar, parity, err);
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* err) { return __all_sync(0xffffffffu, wait(bar, parity, err)); }

// A block's part of a job, as the warp that walks the line tells it the others: a ring of these lies in shared memory.
struct __align__(16) Segment {
    int i0, i1, old_tiles, key0;       // tiles of the job from i0 to i1; cached ones; the first cached key that is walked over
    int context, tree, first, node0;   // cached keys, the request's nodes and the row of the first, the job's first node
    int nodes, g, b, whole;            // the job's nodes (0: there is no segment any more), key/value head, request; whether this is all of the job
    int deep_lo, pad[3];               // where the deepest node's window begins (0: none)
};
constexpr int SEGMENTS = 8;
constexpr int READERS = 11;            // warps that read a segment

template <int DP>
__global__ void __launch_bounds__(THREADS)
tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                         const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_vn, const TreeArgs A, const Line line,
                         int ps_shift, float scale_log2) {
    constexpr int HALVES = DP / 64, NS = stages(DP);
    constexpr uint32_t Q_ONE = HALVES * RT * 128, Q_BYTES = 2 * Q_ONE, KV_HALF = KT * 128, KV_BYTES = HALVES * KV_HALF, STAGE_BYTES = 2 * KV_BYTES;
    constexpr uint32_t BAR_OFF = Q_BYTES + NS * STAGE_BYTES, RING = 8 * NS, OUT_OFF = BAR_OFF + 1024, STATS_OFF = OUT_OFF + 8 * 2048;
    constexpr uint32_t SEG_OFF = STATS_OFF + 2048;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t base = smem_u32(smem_raw), q_sm = base, kv_sm = base + Q_BYTES, bars = base + BAR_OFF;
    const uint32_t k_full0 = bars, k_empty0 = bars + RING, v_full0 = bars + 2 * RING, v_empty0 = bars + 3 * RING, rest = bars + 4 * RING;
    const uint32_t s_ready0 = rest, pv_done0 = rest + 32, p_ready0 = rest + 64, q_full = rest + 96, q_empty = rest + 104, looked0 = rest + 112,
                   told = rest + 144, joined = rest + 152, seg_full0 = rest + 160, seg_empty0 = seg_full0 + 8 * SEGMENTS,
                   drained = seg_empty0 + 8 * SEGMENTS + 136;    // (behind the words)
    volatile uint32_t* words = reinterpret_cast<volatile uint32_t*>(smem_raw + BAR_OFF + 4 * RING + 160 + 16 * SEGMENTS);   // tmem, -, then the value rows
    volatile uint32_t* odd_rows = words + 2;                                                                                // that are not finite: [4][warp][2]
    Segment* const segments = reinterpret_cast<Segment*>(smem_raw + SEG_OFF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = A.nh / A.nkv, half_nodes = line.two_from;
    int* const err = A.err;

    Walk w;
    bool gave_up = false;
    if (warp == 8) {
        pdl_wait();                // lengths, rows and masks may come from the kernel before
        if (base & 1023u) atomicOr(err, XB_ERR_WAIT);                                  // the swizzle needs a 1024-byte aligned window
        const int word = lane == 0 ? *reinterpret_cast<volatile int*>(err) : 0;        // or an earlier block gave up: do not pile on
        w = place_in_line<KT>(A, line);
        gave_up = __any_sync(0xffffffffu, word & XB_ERR_WAIT);
    } else {
        if (threadIdx.x == 9 * 32) {
            for (int i = 0; i < 4 * NS; ++i) mbar_init(bars + 8 * i, 1);
            for (int i = 0; i < 4; ++i) {
                mbar_init(s_ready0 + 8 * i, 1);
                mbar_init(pv_done0 + 8 * i, 1);
                mbar_init(p_ready0 + 8 * i, 4);        // a warp each
                mbar_init(looked0 + 8 * i, 4);
            }
            mbar_init(q_full, 1);
            mbar_init(q_empty, 1);
            mbar_init(told, 8);
            mbar_init(joined, 8);
            mbar_init(drained, 1);
            mbar_init(drained + 8, 1);
            for (int i = 0; i < SEGMENTS; ++i) mbar_init(seg_full0 + 8 * i, 1), mbar_init(seg_empty0 + 8 * i, READERS);
            mbar_init_fence();
        }
        if (warp == 10) tmem_alloc(const_cast<uint32_t*>(&words[0]), 512);
        pdl_wait();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = words[0];
    pdl_launch_dependents();       // only now: see pdl_launch_dependents on tensor memory

    int seg = 0;                   // segments so far
    // The next segment from the ring; nodes == 0: there is none, or a wait gave up.
    auto read_segment = [&]() -> Segment {
        Segment s;
        s.nodes = 0;
        const int at = seg % SEGMENTS;
        if (wait_warp(seg_full0 + 8 * at, (seg / SEGMENTS) & 1, err)) {
            const int4* from = reinterpret_cast<const int4*>(segments + at);
            int4* to = reinterpret_cast<int4*>(&s);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = from[i];
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_empty0 + 8 * at);
        }
        ++seg;
        return s;
    };

    const int box_rows = min(A.page_size, KT);
    if (warp == 8 || warp == 10) {
        // ---- keys (warp 8, which also walks the line) and values (warp 10), a lane per box --------------------------------------
        const bool is_v = warp == 10;
        const uint32_t full0 = is_v ? v_full0 : k_full0, empty0 = is_v ? v_empty0 : k_empty0;
        const CUtensorMap* map = is_v ? &map_v : &map_k;
        const CUtensorMap* map_new = is_v ? &map_vn : &map_kn;
        const int boxes = KT / box_rows * HALVES, bi = lane / HALVES, hf = lane % HALVES;
        int st = 0;
        uint32_t ph = 0;
        bool rounds = false, ok = true;
        if (gave_up) w.job = w.end;
        bool first = true;
        int told_of = 0;           // the parts of shared jobs that the join knows of
        while (ok) {
            Segment s;
            if (is_v) {
                s = read_segment();
                if (!s.nodes) break;
            } else {
                const bool more = next_segment<KT>(A, line, w, first);
                first = false;
                if (more) {
                    const RequestLine& r = w.r;
                    s.i0 = w.i0;
                    s.i1 = w.i1;
                    s.old_tiles = r.old_tiles;
                    s.key0 = r.tile0 * KT;
                    s.context = r.context;
                    s.tree = r.nodes;
                    s.first = r.first;
                    s.node0 = w.piece * line.row_div;
                    s.nodes = min(line.row_div, r.nodes - s.node0);
                    s.g = w.g;
                    s.b = w.b;
                    s.whole = w.i1 - w.i0 == r.tiles;
                    s.deep_lo = 0;
                    if (A.window > 0) {
                        int deepest = 0;
                        for (int i = lane; i < r.nodes; i += 32) deepest = max(deepest, A.depth[r.first + i]);
                        s.deep_lo = r.context + __reduce_max_sync(0xffffffffu, deepest) - A.window + 1;
                    }
                } else {
                    s.nodes = 0;
                    for (int which = 0; which < 2; ++which)
                        if (lane == 0 && !(told_of >> which & 1)) line.shared_jobs[(blockIdx.x * 2 + which) * 8] = 0;
                }
                const int at = seg % SEGMENTS;
                if (seg >= SEGMENTS) ok = wait_warp(seg_empty0 + 8 * at, ((seg / SEGMENTS) - 1) & 1, err);
                if (!ok) break;
                if (lane == 0) {
                    int4* to = reinterpret_cast<int4*>(segments + at);
                    const int4* from = reinterpret_cast<const int4*>(&s);
#pragma unroll
                    for (int i = 0; i < 4; ++i) to[i] = from[i];
                    mbar_arrive(seg_full0 + 8 * at);
                }
                __syncwarp();
                ++seg;
                if (!more) break;
            }
            // 32 entries of the block table at a time, a lane each, and the next 32 on their way; a tile's entries lie in one such run
            const int* table = A.block_table + (size_t)s.b * A.table_stride;
            const int entries = (min(s.context, s.key0 + min(s.i1, s.old_tiles) * KT) + A.page_size - 1) >> ps_shift;
            int entry0 = (s.key0 + s.i0 * KT) >> ps_shift;
            auto entry = [&](int i) { return i < entries ? table[i] : 0; };
            int run = entry(entry0 + lane), next_run = entry(entry0 + 32 + lane);
            for (int it = s.i0; it < s.i1; ++it) {
                int page = -1;                             // of this lane's box, -1: nothing to load
                if (it < s.old_tiles) {
                    const int at = (s.key0 + it * KT) >> ps_shift;
                    if (at - entry0 >= 32) {
                        run = next_run;
                        entry0 += 32;
                        next_run = entry(entry0 + 32 + lane);
                    }
                    page = __shfl_sync(0xffffffffu, run, (at - entry0 + bi) & 31);
                    if (lane >= boxes || s.key0 + it * KT + bi * box_rows >= s.context) {
                        page = -1;
                    } else if (page < 0 || page >= A.num_pages) {
                        atomicOr(err, XB_ERR_BAD_PAGE);
                        page = A.num_pages;                // behind the last page: the box reads as zeros
                    }
                }
                if (rounds && !wait_warp(empty0 + 8 * st, ph ^ 1u, err)) {
                    ok = false;
                    break;
                }
                const uint32_t dst0 = kv_sm + st * STAGE_BYTES + (is_v ? KV_BYTES : 0u);
                if (it < s.old_tiles) {
                    const uint32_t nb = __popc(__ballot_sync(0xffffffffu, page >= 0));
                    if (lane == 0) mbar_expect_tx(full0 + 8 * st, nb * box_rows * 128);
                    __syncwarp();
                    if (page >= 0) {
                        const int j = it * KT + bi * box_rows;             // (key0 is a multiple of the tile, so of the smaller pages too)
                        tma_load_2d(dst0 + hf * KV_HALF + bi * box_rows * 128, map, hf * 64, (page * A.nkv + s.g) * A.page_size + ((s.key0 + j) & (A.page_size - 1)), full0 + 8 * st);
                    }
                } else {
                    if (lane == 0) mbar_expect_tx(full0 + 8 * st, KV_BYTES);
                    __syncwarp();
                    if (lane < HALVES) tma_load_3d(dst0 + lane * KV_HALF, map_new, lane * 64, s.g, s.first + (it - s.old_tiles) * KT, full0 + 8 * st);
                }
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                    rounds = true;
                }
            }
            if (!is_v && !s.whole && lane == 0) {          // what the join needs to know
                const int which = s.i0 > 0 ? 0 : 1;
                int from;
                const int parts = job_parts(w, from);
                int4* job = reinterpret_cast<int4*>(line.shared_jobs + (blockIdx.x * 2 + which) * 8);
                job[0] = make_int4(parts, from, s.first + s.node0, s.nodes);
                job[1].x = s.g;
                told_of |= 1 << which;
            }
        }
        // nothing of this warp's is on its way when the block ends, however it ends
        for (int i = 0; i < NS; ++i)
            if (rounds || i < st) wait_warp(full0 + 8 * i, i < st ? ph : ph ^ 1u, err);
    } else if (warp == 9) {
        // ---- Q, then S = Q K^T of every tile --------------------------------------------------------------------------------
        const uint32_t one = elected(), tmem_u = uniform(tmem);
        const uint32_t idesc_s = umma_idesc(KT, 0);
        const uint64_t dq0 = umma_desc(q_sm, 16, 1024), dk0 = umma_desc(kv_sm, 16, 1024);
        int st = 0, Th[2] = {0, 0};              // ring stage, tiles of either half so far
        uint32_t ph = 0;
        bool ok = true;
        while (ok) {
            const Segment s = read_segment();
            const int nodes = uniform(s.nodes), iters = uniform(s.i1 - s.i0);
            if (!nodes) break;
            const int halves = nodes > half_nodes ? 2 : 1, I = seg - 1;
            if (I > 0) {                         // Q lies where the last one lay: once every product that reads that has completed
                commit(one, q_empty);
                ok = wait_warp(q_empty, (uint32_t)(I - 1) & 1u, err);
                if (!ok) break;
            }
            if (one) {
                mbar_expect_tx(q_full, (uint32_t)(halves * HALVES * half_nodes * G * 128));
                for (int hd = 0; hd < halves; ++hd)
#pragma unroll
                    for (int hf = 0; hf < HALVES; ++hf)
                        tma_load_3d(q_sm + hd * Q_ONE + hf * RT * 128, &map_q, hf * 64, s.g * G, s.first + s.node0 + hd * half_nodes, q_full);
            }
            __syncwarp();
            ok = wait_warp(q_full, (uint32_t)I & 1u, err);
            for (int it = 0; it < iters && ok; ++it) {
                ok = wait_warp(k_full0 + 8 * st, ph, err);
                const uint64_t dk = dk0 + (uint64_t)((st * STAGE_BYTES) >> 4);
#pragma unroll
                for (int hd = 0; hd < 2; ++hd) {
                    if (halves == 1 && (it & 1) != hd) continue;
                    const int th = Th[hd]++, sb = th & 1;
                    // these columns held the scores and then P of this half's last tile but one: its P V must have read them
                    ok = ok && (th < 2 || wait_warp(pv_done0 + 8 * (2 * hd + sb), ((th >> 1) - 1) & 1, err));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dq = dq0 + (uint64_t)((halves == 1 ? 0u : hd * Q_ONE) >> 4);
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk) {
                        const uint32_t off = (kk >> 2), inner = (kk & 3) * 32;
                        umma_ss(one, tmem_u + (uint32_t)(hd * 128 + sb * 64), dq + (uint64_t)((off * RT * 128 + inner) >> 4),
                                dk + (uint64_t)((off * KV_HALF + inner) >> 4), idesc_s, kk ? 1u : 0u);
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
        commit(one, drained);                    // no product is at work when the tensor memory is freed, however the block ends
        wait_warp(drained, 0, err);
    } else if (warp == 11) {
        // ---- O += P V of every tile (O starts as zeros, by the softmax threads) -----------------------------------------------
        const uint32_t one = elected(), tmem_u = uniform(tmem);
        const uint32_t idesc_o = umma_idesc(DP, 1);
        const uint64_t dv0 = umma_desc(kv_sm + KV_BYTES, KV_HALF, 1024);
        int st = 0, Th[2] = {0, 0};
        uint32_t ph = 0;
        bool ok = true;
        while (ok) {
            const Segment s = read_segment();
            const int nodes = uniform(s.nodes), iters = uniform(s.i1 - s.i0);
            if (!nodes) break;
            const int halves = nodes > half_nodes ? 2 : 1;
            for (int it = 0; it < iters && ok; ++it) {
                ok = wait_warp(v_full0 + 8 * st, ph, err);
                const uint64_t dv = dv0 + (uint64_t)((st * STAGE_BYTES) >> 4);
#pragma unroll
                for (int hd = 0; hd < 2; ++hd) {
                    if (halves == 1 && (it & 1) != hd) continue;
                    const int th = Th[hd]++, sb = th & 1;
                    ok = ok && wait_warp(p_ready0 + 8 * (2 * hd + sb), (th >> 1) & 1, err);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t tp = tmem_u + (uint32_t)(hd * 128 + sb * 64);
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        umma_ts(one, tmem_u + (uint32_t)(256 + hd * 128), tp + (uint32_t)(kk * 8), dv + (uint64_t)((kk * 2048) >> 4), idesc_o);
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
        commit(one, drained + 8);
        wait_warp(drained + 8, 0, err);
    } else {
        // ---- softmax: a row per thread ---------------------------------------------------------------------------------------------
        const int hd = warp >> 2, r = (int)threadIdx.x & 127;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + (uint32_t)(hd * 128) + lane_addr, tmem_o = tmem + (uint32_t)(256 + hd * 128) + lane_addr;
        const uint32_t my_s_ready = s_ready0 + 16 * hd, my_p_ready = p_ready0 + 16 * hd, my_pv_done = pv_done0 + 16 * hd;
        const int node_r = r / G, head_r = r % G;
        const int window = A.window;
        const bool out16 = rows_on_16_bytes(A.out, A.out_stride);
        // the rows whose results this thread stores, one of every eight of the warp's: their nodes, and where they lie from the job's first on
        int st_node[4];
        long long st_at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int in_half = (warp & 3) * 32 + k * 8 + (lane >> 2);
            st_node[k] = in_half / G;
            st_at[k] = st_node[k] * A.out_stride + (in_half % G) * A.d + (lane & 3) * 8;
        }
        int T = 0, Th = 0, looks = 0, joins = 0;   // tiles of all segments so far, of this half's, tiles that were looked at, segments of one tile of rows
        bool alive = true;
        while (alive) {
            const Segment s = read_segment();
            if (!s.nodes) break;
            // one tile of rows: both halves work on it, each on every other tile of keys
            const bool split = s.nodes <= half_nodes;
            const int half_first = split ? 0 : hd * half_nodes;
            const int node = s.node0 + half_first + node_r;              // in its tree
            const bool valid = node_r < half_nodes && node < s.node0 + s.nodes;
            const bool working = __any_sync(0xffffffffu, valid);
            const int t = s.first + node;
            const int my_depth = valid && window > 0 ? max(0, A.depth[t]) : 0;
            const int my_lo = window > 0 ? max(0, s.context + my_depth - window + 1) : 0;
            const int* my_words = A.ancestors + (size_t)(valid ? t : s.first) * A.words;
            uint32_t word_lo = 0, word_hi = 0;            // of the first drafted tile
            if (valid && s.i1 > s.old_tiles) {
                word_lo = A.words > 0 ? (uint32_t)my_words[0] : 0u;
                word_hi = A.words > 1 ? (uint32_t)my_words[1] : 0u;
            }
            if (working) {
                float zero[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) zero[i] = 0.f;
#pragma unroll
                for (int c0 = 0; c0 < DP; c0 += 32) tmem_st32(tmem_o + c0, zero);
                tmem_st_wait();
            }
            float m_ref = -INFINITY, l = 0.f;
            // cached tiles before `mixed` begin before the deepest node's window does; those from `full` on go beyond the context
            const int mixed = s.deep_lo > s.key0 ? min(s.old_tiles, (s.deep_lo - s.key0 + KT - 1) / KT) : 0, full = (s.context - s.key0) / KT;
            // the looks at tiles that not all rows see alike, up to tile `it`
            auto looks_at = [&](int it) { return looks + min(it, mixed) - min(s.i0, mixed) + max(it, s.old_tiles) - max(s.i0, s.old_tiles); };

            // One tile; EDGE: not all of its keys are seen by all rows.
            auto tile = [&](auto edge_c, int it, int th) -> bool {
                constexpr bool EDGE = decltype(edge_c)::value;
                const int sb = th & 1;
                const bool drafted = EDGE && it >= s.old_tiles, look = EDGE && (drafted || it < mixed);
                const int key0 = !EDGE ? 0 : drafted ? (it - s.old_tiles) * KT : s.key0 + it * KT;
                const int keys = drafted ? s.tree : s.context;            // keys from here on belong to nobody
                const int n_look = look ? looks_at(it) : 0;
                if (!wait_warp(my_s_ready + 8 * sb, (th >> 1) & 1, err)) return false;
                float corr = 1.f;
                int moved = 0;
                unsigned long long seen = ~0ull;
                if (working) {
                    tc_fence_after();
                    float sc[64];
                    {
                        uint32_t ra[32], rb[32];
                        tmem_ld32_nowait(tmem_s + sb * 64, ra);
                        tmem_ld32_nowait(tmem_s + sb * 64 + 32, rb);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            sc[i] = __uint_as_float(ra[i]);
                            sc[32 + i] = __uint_as_float(rb[i]);
                        }
                    }
                    if (EDGE) {
                        if (drafted) {
                            const int at = key0 / 32;
                            seen = at == 0 ? ((unsigned long long)word_hi << 32 | word_lo) : 0ull;
                            if (at > 0 && valid) {
                                if (at < A.words) seen = (uint32_t)my_words[at];
                                if (at + 1 < A.words) seen |= (unsigned long long)(uint32_t)my_words[at + 1] << 32;
                            }
                            if (keys - key0 < 64) seen &= (1ull << (keys - key0)) - 1;
                            if (window > 0)
                                for (int i = 0; i < min(64, keys - key0); ++i)
                                    if (my_depth - max(0, A.depth[s.first + key0 + i]) >= window) seen &= ~(1ull << i);
                        } else {
                            if (keys - key0 < 64) seen = (1ull << (keys - key0)) - 1;
                            if (my_lo > key0) seen = my_lo - key0 < 64 ? seen & (~0ull << (my_lo - key0)) : 0ull;
                        }
#pragma unroll
                        for (int i = 0; i < 64; ++i) sc[i] = (seen >> i & 1ull) ? sc[i] : -INFINITY;
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 64; i += 8) {
                        mx4[0] = max3_nan(mx4[0], sc[i], sc[i + 1]);
                        mx4[1] = max3_nan(mx4[1], sc[i + 2], sc[i + 3]);
                        mx4[2] = max3_nan(mx4[2], sc[i + 4], sc[i + 5]);
                        mx4[3] = max3_nan(mx4[3], sc[i + 6], sc[i + 7]);
                    }
                    const float mx = max3_nan(mx4[0], mx4[1], max3_nan(mx4[2], mx4[3], mx4[3])) * scale_log2;
                    if (!(mx <= m_ref + RESCALE_STEP)) {                 // (a score that is no number makes the row one)
                        corr = m_ref == -INFINITY ? 0.f : ex2(m_ref - mx);
                        moved = m_ref != -INFINITY && valid;             // (O is zero before)
                        m_ref = mx;
                    }
                    const float m_neg = m_ref == -INFINITY ? 0.f : -m_ref;
                    const f32x2 scale2 = pack2(scale_log2, scale_log2), mneg2 = pack2(m_neg, m_neg);
                    f32x2 sum_a = pack2(0.f, 0.f), sum_b = pack2(0.f, 0.f);
                    uint32_t pk[32];
#pragma unroll
                    for (int c8 = 0; c8 < 8; ++c8) {
                        float x[8], e[8];
#pragma unroll
                        for (int i = 0; i < 8; i += 2) unpack2(fma2(pack2(sc[c8 * 8 + i], sc[c8 * 8 + i + 1]), scale2, mneg2), x[i], x[i + 1]);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if ((i & 3) != 3) e[i] = ex2(x[i]);
                        ex2_poly2(x[3], x[7], e[3], e[7]);
                        if (EDGE) {                // the polynomial ends at 2^-126: a key that is not seen has no weight at all
                            if (x[3] == -INFINITY) e[3] = 0.f;
                            if (x[7] == -INFINITY) e[7] = 0.f;
                        }
                        sum_a = add2(sum_a, add2(pack2(e[0], e[1]), pack2(e[2], e[3])));
                        sum_b = add2(sum_b, add2(pack2(e[4], e[5]), pack2(e[6], e[7])));
                        pk[c8 * 4] = pack_bf16(e[0], e[1]);
                        pk[c8 * 4 + 1] = pack_bf16(e[2], e[3]);
                        pk[c8 * 4 + 2] = pack_bf16(e[4], e[5]);
                        pk[c8 * 4 + 3] = pack_bf16(e[6], e[7]);
                    }
                    float s0, s1, s2, s3;
                    unpack2(sum_a, s0, s1);
                    unpack2(sum_b, s2, s3);
                    l = l * corr + ((s0 + s1) + (s2 + s3));
                    tmem_st32_u(tmem_s + sb * 64, pk);                   // P goes where the scores were
                }
                if (EDGE && (split || hd == 0)) {
                    // the value rows: zeroed where nobody may see them, and in tiles that are not seen alike where they are not finite.
                    // Eight lanes have a row's half, a warp every fourth group of four rows.
                    const int gt = T + it - s.i0, st = gt % NS;
                    const bool here = wait_warp(v_full0 + 8 * st, (gt / NS) & 1, err);     // orders these accesses after the copy
                    unsigned char* const rows = smem_raw + Q_BYTES + st * STAGE_BYTES + KV_BYTES;
                    const int dead_to = !drafted && window > 0 ? s.context - window + 1 - key0 : 0, dead_from = keys - key0;
                    uint32_t odd_lo = 0, odd_hi = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int rr = k * 16 + (warp & 3) * 4 + (lane >> 3);
                        uint4* at = reinterpret_cast<uint4*>(rows + rr * 128 + (lane & 7) * 16);
                        const bool drop = rr >= dead_from || rr < dead_to;
                        bool odd = false;
                        if (look && !drop) {
#pragma unroll
                            for (int hf = 0; hf < HALVES; ++hf) odd |= any_not_finite(at[hf * (KV_HALF / 16)]);
                        }
                        uint32_t mask = __ballot_sync(0xffffffffu, odd);                   // eight bits to a row
                        mask = (mask & 0xffu ? 1u : 0u) | (mask & 0xff00u ? 2u : 0u) | (mask & 0xff0000u ? 4u : 0u) | (mask & 0xff000000u ? 8u : 0u);
                        if (here && (drop || (mask >> (lane >> 3) & 1u))) {
#pragma unroll
                            for (int hf = 0; hf < HALVES; ++hf) at[hf * (KV_HALF / 16)] = make_uint4(0, 0, 0, 0);
                        }
                        if (k < 2) odd_lo |= mask << (k * 16 + (warp & 3) * 4);
                        else odd_hi |= mask << ((k - 2) * 16 + (warp & 3) * 4);
                    }
                    fence_async_shared();          // the zeroed rows: visible to the product
                    __syncwarp();
                    if (look && lane == 0) {
                        odd_rows[(n_look & 3) * 8 + (warp & 3) * 2] = odd_lo;
                        odd_rows[(n_look & 3) * 8 + (warp & 3) * 2 + 1] = odd_hi;
                        mbar_arrive(looked0 + 8 * (n_look & 3));
                    }
                    if (!here) return false;
                }
                // O is touched only when the last tile's P V has completed
                if (EDGE || __any_sync(0xffffffffu, moved)) {
                    if (th > Th && !wait_warp(my_pv_done + 8 * (sb ^ 1), ((th - 1) >> 1) & 1, err)) return false;
                }
                if (__any_sync(0xffffffffu, moved)) {
                    tc_fence_after();
                    const float f = moved ? corr : 1.f;
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
                if (look) {
                    if (!wait_warp(looked0 + 8 * (n_look & 3), (n_look >> 2) & 1, err)) return false;
                    uint32_t odd_lo = 0, odd_hi = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) odd_lo |= odd_rows[(n_look & 3) * 8 + 2 * i], odd_hi |= odd_rows[(n_look & 3) * 8 + 2 * i + 1];
                    if ((odd_lo | odd_hi) && working) {    // (rare) the same for all lanes
                        tc_fence_after();
                        for (int i = 0; i < 64; ++i) {
                            if (!((i < 32 ? odd_lo >> i : odd_hi >> (i - 32)) & 1u)) continue;
                            const uint32_t two = tmem_ld1(tmem_s + sb * 64 + (uint32_t)(i >> 1));
                            const float p = __uint_as_float((i & 1) ? two & 0xffff0000u : two << 16);
                            const bool mine = valid && (seen >> i & 1ull);
                            const __nv_bfloat16* v;
                            if (drafted) {
                                v = (const __nv_bfloat16*)A.v_new + (size_t)(s.first + key0 + i) * A.v_stride + (size_t)s.g * A.d;
                            } else {
                                const int j = key0 + i, page = A.block_table[(size_t)s.b * A.table_stride + (j >> ps_shift)];
                                v = (const __nv_bfloat16*)A.v_cache + (((size_t)page * A.nkv + s.g) * A.page_size + (j & (A.page_size - 1))) * A.d;
                            }
#pragma unroll 1
                            for (int c0 = 0; c0 < DP; c0 += 32) {
                                float o[32];
                                tmem_ld32(tmem_o + c0, o);
#pragma unroll
                                for (int c = 0; c < 32; ++c)
                                    if (mine && c0 + c < A.d) o[c] = fmaf(p, __bfloat162float(v[c0 + c]), o[c]);
                                tmem_st32(tmem_o + c0, o);
                            }
                            tmem_st_wait();
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(my_p_ready + 8 * sb);
                return true;
            };
            int th = Th;
            const int step = split ? 2 : 1;
            for (int it = s.i0 + (split ? hd : 0); it < s.i1 && alive; it += step, ++th)
                alive = it >= mixed && it < full ? tile(std::false_type{}, it, th) : tile(std::true_type{}, it, th);
            const int n_it = th - Th;
            // ---- O / l, or this part of a job that blocks share ---------------------------------------------------------------------
            Th = th;
            T += s.i1 - s.i0;
            looks = looks_at(s.i1);
            if (alive && n_it > 0) alive = wait_warp(my_pv_done + 8 * ((Th - 1) & 1), ((Th - 1) >> 1) & 1, err);
            alive = __all_sync(0xffffffffu, alive);
            float f_mine = 1.f, f_other = 0.f;
            if (split && alive) {
                // the halves' sums come together: each of them takes half of the channels of both
                volatile float2* stats = reinterpret_cast<volatile float2*>(smem_raw + STATS_OFF);
                stats[hd * 128 + r].x = m_ref;
                stats[hd * 128 + r].y = l;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(told);
                alive = wait_warp(told, joins & 1, err);
                tc_fence_after();
                const float m_o = stats[(hd ^ 1) * 128 + r].x, l_o = stats[(hd ^ 1) * 128 + r].y;
                const float m_all = max3_nan(m_ref, m_o, m_o);
                f_mine = m_all == -INFINITY ? 0.f : ex2(m_ref - m_all);
                f_other = m_all == -INFINITY ? 0.f : ex2(m_o - m_all);
                l = f_mine * l + f_other * l_o;
                m_ref = m_all;
            }
            if (alive && working) {
                tc_fence_after();
                if (s.whole) {
                    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
                    f_mine *= inv;
                    f_other *= inv;
                }
                const uint32_t o_other = tmem + (uint32_t)(256 + (hd ^ 1) * 128) + lane_addr;
                const int c_from = split ? hd * (DP / 2) : 0, c_to = min(A.d, split ? c_from + DP / 2 : DP);
                const size_t part = part_row(line, blockIdx.x, s.i0 > 0 ? 0 : 1, (half_first + node_r) * G + head_r);
                float4* part_to = reinterpret_cast<float4*>(line.part_o) + part_four(line, A.d, part, c_from / 4);
                __nv_bfloat16* out_to = (__nv_bfloat16*)A.out + (size_t)(s.first + s.node0 + half_first) * A.out_stride + (size_t)s.g * G * A.d + c_from;
                uint4* const stage = reinterpret_cast<uint4*>(smem_raw + OUT_OFF + warp * 2048);
                const int st_nodes = min(half_nodes, s.nodes - half_first);
#pragma unroll 1
                for (int c0 = c_from; c0 < c_to; c0 += 32) {
                    float o[32];
                    tmem_ld32(tmem_o + c0, o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= f_mine;
                    if (split) {
                        float o2[32];
                        tmem_ld32(o_other + c0, o2);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = fmaf(o2[i], f_other, o[i]);
                    }
                    if (s.whole) {
                        // through shared memory, so that neighbouring lanes write neighbouring addresses: 64 bytes of a row lie in
                        // four pieces of 16, at places that differ from row to row
                        __syncwarp();
#pragma unroll
                        for (int c8 = 0; c8 < 4; ++c8) {
                            uint4 v;
                            v.x = pack_bf16(o[c8 * 8], o[c8 * 8 + 1]);
                            v.y = pack_bf16(o[c8 * 8 + 2], o[c8 * 8 + 3]);
                            v.z = pack_bf16(o[c8 * 8 + 4], o[c8 * 8 + 5]);
                            v.w = pack_bf16(o[c8 * 8 + 6], o[c8 * 8 + 7]);
                            stage[lane * 4 + (c8 ^ ((lane >> 1) & 3))] = v;
                        }
                        __syncwarp();
                        const bool in = c0 + (lane & 3) * 8 < A.d;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int rr = k * 8 + (lane >> 2);
                            if (in && st_node[k] < st_nodes) store8(out_to + st_at[k], stage[rr * 4 + ((lane & 3) ^ ((rr >> 1) & 3))], out16);
                        }
                        out_to += 32;
                    } else if (valid) {
#pragma unroll
                        for (int c4 = 0; c4 < 8; ++c4)
                            if (c0 + c4 * 4 < A.d) part_to[c4 * 8] = make_float4(o[c4 * 4], o[c4 * 4 + 1], o[c4 * 4 + 2], o[c4 * 4 + 3]);
                        part_to += 64;
                    }
                }
                if (valid && !s.whole && !(split && hd)) *reinterpret_cast<float2*>(line.part_ml + part * 2) = make_float2(m_ref, l);
            }
            if (split) {
                // O is not written again before both halves have read it
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(joined);
                if (alive) alive = wait_warp(joined, joins & 1, err);
                tc_fence_after();
                ++joins;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 10) tmem_free(tmem, 512);
}

// Joins the parts of a job that several blocks shared, in the order of the parts: with M the largest of their maxima,
// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.  Grid (block and which of its parts, MERGE_Y): as many of the job's rows as the part is
// of the job, so that there are as many blocks at work as there are parts.  A thread has four channels of a row in every group of eight
// rows and requests eight numbers of four at once: P parts of 8 / P groups.  Bound by trips to the L2 (the told job, maxima and sums, the
// parts): 7 us for 64 jobs of 256 rows in 211 parts (27 MB), 2.5 us for 8 jobs of 32 rows.  Two blocks a part with twice the work, more
// blocks a processor, or the parts asked for before the factors: 1 to 8 % longer.
constexpr int MERGE_Y = 4;
constexpr int MERGE_ROWS = 32;     // rows whose factors lie in shared memory

struct MergeJob {
    int parts, c_first, t0, rows, g, G;
};

template <int P>
__device__ __forceinline__ void merge_groups(const TreeArgs& A, const Line& line, const MergeJob& job, const float (*factors)[MERGE_ROWS],
                                             const float* inverse, int base, int end, int in, int c4) {
    constexpr int K = 8 / P;
    const float4* o = reinterpret_cast<const float4*>(line.part_o);
    const bool out16 = rows_on_16_bytes(A.out, A.out_stride);
    for (int g0 = base; g0 < end; g0 += K) {
        float4 acc[K];
#pragma unroll
        for (int k = 0; k < K; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < job.parts; i0 += P) {
            float4 v[K][P];
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int row = (g0 + k) * 8 + in;
                    v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (g0 + k < end && i0 + i < job.parts)
                        v[k][i] = __ldcg(o + part_four(line, A.d, part_row(line, job.c_first + i0 + i, i0 + i > 0 ? 0 : 1, row), c4));
                }
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float f = g0 + k < end && i0 + i < job.parts ? factors[i0 + i][(g0 + k - base) * 8 + in] : 0.f;
                    acc[k].x = fmaf(f, v[k][i].x, acc[k].x);
                    acc[k].y = fmaf(f, v[k][i].y, acc[k].y);
                    acc[k].z = fmaf(f, v[k][i].z, acc[k].z);
                    acc[k].w = fmaf(f, v[k][i].w, acc[k].w);
                }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int row = (g0 + k) * 8 + in;
            if (g0 + k >= end || row >= job.rows) continue;
            const float inv = inverse[(g0 + k - base) * 8 + in];
            __nv_bfloat16* dst = (__nv_bfloat16*)A.out + (size_t)(job.t0 + row / job.G) * A.out_stride + (size_t)(job.g * job.G + row % job.G) * A.d + c4 * 4;
            const uint2 two = make_uint2(pack_bf16(acc[k].x * inv, acc[k].y * inv), pack_bf16(acc[k].z * inv, acc[k].w * inv));
            if (out16) {
                *reinterpret_cast<uint2*>(dst) = two;
            } else {
                reinterpret_cast<uint16_t*>(dst)[0] = (uint16_t)two.x;
                reinterpret_cast<uint16_t*>(dst)[1] = (uint16_t)(two.x >> 16);
                reinterpret_cast<uint16_t*>(dst)[2] = (uint16_t)two.y;
                reinterpret_cast<uint16_t*>(dst)[3] = (uint16_t)(two.y >> 16);
            }
        }
    }
}

template <int DP>
__global__ void __launch_bounds__(DP * 2)
tree_merge_kernel(const TreeArgs A, const Line line) {
    __shared__ float factors[LINE_BLOCKS][MERGE_ROWS], inverse[MERGE_ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const int4 told = *reinterpret_cast<const int4*>(line.shared_jobs + blockIdx.x * 8);    // parts, first block, first node's row, nodes
    const int G = A.nh / A.nkv;
    const MergeJob job{told.x, told.y, told.z, told.w * G, line.shared_jobs[blockIdx.x * 8 + 4], G};
    if (job.parts < 2) return;
    // this block's groups of eight rows
    const int groups = (job.rows + 7) / 8, shares = job.parts * MERGE_Y, mine = ((int)blockIdx.x / 2 - job.c_first) * MERGE_Y + blockIdx.y;
    const int g0 = groups * mine / shares, g1 = groups * (mine + 1) / shares;
    if (g0 >= g1 || (*reinterpret_cast<volatile int*>(A.err) & XB_ERR_WAIT)) return;
    const int in = threadIdx.x & 7, c4 = threadIdx.x >> 3;
    const float2* ml = reinterpret_cast<const float2*>(line.part_ml);
    for (int base = g0; base < g1; base += MERGE_ROWS / 8) {
        const int end = min(g1, base + MERGE_ROWS / 8);
        for (int t = threadIdx.x; t < (end - base) * 64; t += DP * 2) {    // eight lanes to a row
            const int r8 = t >> 3, q = t & 7, row = min(base * 8 + r8, job.rows - 1);
            auto at = [&](int i) { return ml + part_row(line, job.c_first + i, i > 0 ? 0 : 1, row); };
            const float2 first = q < job.parts ? __ldcg(at(q)) : make_float2(-INFINITY, 0.f);
            float M = first.x, W = 0.f;
            for (int i = q + 8; i < job.parts; i += 8) M = fmaxf(M, __ldcg(at(i)).x);
#pragma unroll
            for (int k = 1; k < 8; k <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
            if (M == -INFINITY) M = 0.f;
            for (int i = q; i < job.parts; i += 8) {
                const float2 x = i == q ? first : __ldcg(at(i));
                const float f = exp2f(x.x - M);
                factors[i][r8] = f;
                W = fmaf(f, x.y, W);
            }
#pragma unroll
            for (int k = 1; k < 8; k <<= 1) W += __shfl_xor_sync(0xffffffffu, W, k);
            if (q == 0) inverse[r8] = W > 0.f || W != W ? 1.f / W : 0.f;
        }
        __syncthreads();
        if (c4 * 4 < A.d) {
            if (job.parts == 2) merge_groups<2>(A, line, job, factors, inverse, base, end, in, c4);
            else if (job.parts <= 4) merge_groups<4>(A, line, job, factors, inverse, base, end, in, c4);
            else merge_groups<8>(A, line, job, factors, inverse, base, end, in, c4);
        }
        __syncthreads();           // the factors are written anew
    }
}

// Rows that do not start on 16-byte boundaries, which the copies into shared memory want, are laid out densely first.
__global__ void tree_dense_rows_kernel(__nv_bfloat16* to, const TreeArgs A) {
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, nq = A.nh * A.d, nk = A.nkv * A.d;
    const __nv_bfloat16 *q = (const __nv_bfloat16*)A.q + (size_t)t * A.q_stride, *k = (const __nv_bfloat16*)A.k_new + (size_t)t * A.k_stride,
                        *v = (const __nv_bfloat16*)A.v_new + (size_t)t * A.v_stride;
    for (int i = threadIdx.x; i < nq; i += blockDim.x) to[(size_t)t * nq + i] = q[i];
    to += (size_t)A.tokens * nq;
    for (int i = threadIdx.x; i < nk; i += blockDim.x) {
        to[(size_t)t * nk + i] = k[i];
        to[(size_t)(A.tokens + t) * nk + i] = v[i];
    }
}

// A bfloat16 tensor of `RANK` dimensions, innermost first, `strides` elements apart, through boxes in the 128-byte swizzle.
template <int RANK>
bool map_of(CUtensorMap* out, const void* ptr, const long long (&dims)[RANK], const long long (&strides)[RANK - 1], const int (&box)[RANK]) {
    const EncodeTiledFn fn = encode_fn();
    cuuint64_t dim[RANK], stride[RANK - 1];
    cuuint32_t boxes[RANK], each[RANK];
    for (int i = 0; i < RANK; ++i) dim[i] = (cuuint64_t)dims[i], boxes[i] = (cuuint32_t)box[i], each[i] = 1;
    for (int i = 0; i + 1 < RANK; ++i) stride[i] = (cuuint64_t)strides[i] * 2;
    return fn && fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, RANK, const_cast<void*>(ptr), dim, stride, boxes, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP>
int launch_tc(const TreeArgs& A, const Line& line, cudaStream_t stream) {
    constexpr int NS = stages(DP);
    constexpr size_t smem = 2 * (DP / 64) * RT * 128 + NS * 2 * (DP / 64) * KT * 128 + 1024 + 8 * 2048 + 2048 + SEGMENTS * sizeof(Segment);
    static unsigned long long roomy = 0;
    if (const int rc = xb_more_smem(tree_attention_tc_kernel<DP>, (int)smem, &roomy)) return rc;
    const int G = A.nh / A.nkv, box_rows = A.page_size < KT ? A.page_size : KT;
    int shift = 0;
    while ((1 << shift) < A.page_size) ++shift;
    CUtensorMap mq, mk, mv, mkn, mvn;
    const long long rows = (long long)A.num_pages * A.nkv * A.page_size;
    if (!map_of<3>(&mq, A.q, {A.d, A.nh, A.tokens}, {A.d, A.q_stride}, {64, G, line.two_from}) || !map_of<2>(&mk, A.k_cache, {A.d, rows}, {A.d}, {64, box_rows}) ||
        !map_of<2>(&mv, A.v_cache, {A.d, rows}, {A.d}, {64, box_rows}) || !map_of<3>(&mkn, A.k_new, {A.d, A.nkv, A.tokens}, {A.d, A.k_stride}, {64, 1, KT}) ||
        !map_of<3>(&mvn, A.v_new, {A.d, A.nkv, A.tokens}, {A.d, A.v_stride}, {64, 1, KT}))
        return (int)cudaErrorInvalidValue;
    const int rc = xb_launch(tree_attention_tc_kernel<DP>, dim3(LINE_BLOCKS), dim3(THREADS), smem, stream, mq, mk, mv, mkn, mvn, A, line, shift, A.scale * 1.4426950408889634f);
    if (rc) return rc;
    return xb_launch(tree_merge_kernel<DP>, dim3(2 * LINE_BLOCKS, MERGE_Y), dim3(DP * 2), 0, stream, A, line);
}

}  // namespace

namespace xbtree {

// (Unseen keys are set to -inf before the scores are scaled, so the factor has to be above zero, and by so much that no product with it is
// taken for zero; the other kernel scales first.  A cache without pages has no tensor map.)
bool tree_tc_takes(const TreeArgs& A) {
    return A.scale >= 1.17549435e-38f && A.d % 16 == 0 && A.d >= 16 && A.d <= 128 && A.nh / A.nkv <= RT && A.page_size >= 8 &&
           (A.page_size & (A.page_size - 1)) == 0 && A.num_pages > 0 && ((long long)A.num_pages + 1) * A.nkv * A.page_size < (1LL << 31) &&
           rows_on_16_bytes(A.k_cache, 0) && rows_on_16_bytes(A.v_cache, 0);
}

static int part_rows_of(int tokens, int group) {
    const int nodes = 2 * (RT / (group < RT ? group : RT));
    return ((tokens < nodes ? tokens : nodes) * group + 7) / 8 * 8;
}

long long tree_tc_scratch(int tokens, int nh, int nkv, int d) {
    return line_floats(LINE_BLOCKS, part_rows_of(tokens, nh / nkv), d, ((long long)tokens * (nh + 2 * nkv) * d + 1) / 2);
}

int tree_tc_launch(const TreeArgs& given, float* scratch, cudaStream_t stream) {
    TreeArgs A = given;
    Line line;
    line.two_from = RT / (A.nh / A.nkv);
    line.min_share = 8;
    line.row_mul = 1;
    line.row_div = 2 * line.two_from;
    line.part_rows = part_rows_of(A.tokens, A.nh / A.nkv);
    lay_out(line, LINE_BLOCKS, A.d, scratch);
    if (!rows_on_16_bytes(A.q, A.q_stride) || !rows_on_16_bytes(A.k_new, A.k_stride) || !rows_on_16_bytes(A.v_new, A.v_stride)) {
        __nv_bfloat16* dense = reinterpret_cast<__nv_bfloat16*>(line.dense);
        const int rc = xb_launch(tree_dense_rows_kernel, dim3(A.tokens), dim3(256), 0, stream, dense, A);
        if (rc) return rc;
        A.q = dense;
        A.k_new = dense + (size_t)A.tokens * A.nh * A.d;
        A.v_new = dense + (size_t)A.tokens * (A.nh + A.nkv) * A.d;
        A.q_stride = (long long)A.nh * A.d;
        A.k_stride = A.v_stride = (long long)A.nkv * A.d;
    }
    return A.d <= 64 ? launch_tc<64>(A, line, stream) : launch_tc<128>(A, line, stream);
}

}  // namespace xbtree
