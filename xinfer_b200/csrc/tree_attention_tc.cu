// Attention of a tree of drafted tokens on the 5th-generation tensor cores, in bfloat16 (tree_attention.cu says what is computed).
//
// The nodes of a tree and the query heads of a key/value head are the rows of the products: a job is (request, key/value head, up to
// two tiles of 128 rows), so a tile of keys and values is read once for 256 rows.  Its keys are walked over in tiles of 64, the cached
// ones first, then the drafted ones, with a running maximum and sum per row (one thread a row) and O in tensor memory.
// Which rows see a drafted key is a bit per key: the row's words of ancestors.
//
// The tiles of all jobs, in order of the requests, are one line that is cut into equal shares, one per block: blocks finish together
// whatever the lengths are, and nobody has to know the lengths on the host.  A job that several blocks share leaves an unnormalised O with
// its maximum and sum per block; tree_merge_kernel joins them in their order.  Every block forms the line for itself, from two numbers
// per request.
//
// Per tile: S = Q K^T by warp 9, P = 2^(S - m) by warps 0..3 (first row tile) and 4..7 (second), in the tensor memory of S, O += P V by
// warp 11; warps 8 and 10 fetch keys and values, by page boxes from the cache and by boxes of 64 rows from the drafted rows.
// Barriers carry on from segment to segment, as do the rings.
//
// A value that a row does not see must not reach it, whatever it holds, but a product takes 0 * inf for NaN.  In tiles that not all rows
// see alike (drafted keys, the edge of a window) the value rows are looked at: those that hold an infinity or NaN are zeroed for the
// product, and the rows that do see them add their share to O by hand.  Value rows that nobody sees are zeroed too.
#include "tc_common.cuh"
#include "tree_attention.cuh"

namespace {

using namespace xbtc;
using namespace xbtree;

constexpr int RT = TILE_ROWS;              // rows of a tile
constexpr float RESCALE_STEP = 8.f;        // a row's maximum moves only when it grows by more than 2^8
constexpr int THREADS = 384;
__host__ __device__ constexpr int stages(int dp) { return dp <= 64 ? 8 : 5; }

// A block's part of a job.
struct Segment {
    int b, g, node0, t0;           // request, key/value head, first node of the job and its row
    int nodes;                     // of the job (both tiles)
    int tree0, tree_n, context;    // the request's first node's row, its nodes, its cached keys
    int tile0, old_tiles;          // the first cached tile, cached tiles from there on
    int i0, i1, tiles;             // this segment's tiles of the job's
};

struct Walk {                      // where a role stands in the line
    int b, before, unit, end;      // request, units before it, the next unit, the block's end
};

__device__ __forceinline__ bool next_segment(const TreeArgs& A, const Line& line, Walk& w, Segment& s) {
    if (w.unit >= w.end) return false;
    RequestLine r = request_line(A, line, w.b);
    while (w.unit >= w.before + r.jobs * r.tiles) {       // (requests without work have no units)
        w.before += r.jobs * r.tiles;
        r = request_line(A, line, ++w.b);
    }
    const int job = (w.unit - w.before) / r.tiles, pieces = r.jobs / A.nkv;
    s.b = w.b;
    s.g = job / pieces;
    s.tree0 = r.first;
    s.tree_n = r.nodes;
    s.context = r.context;
    s.node0 = job % pieces * line.job_nodes;
    s.t0 = r.first + s.node0;
    s.nodes = min(line.job_nodes, r.nodes - s.node0);
    s.tile0 = r.tile0;
    s.old_tiles = r.old_tiles;
    s.tiles = r.tiles;
    s.i0 = w.unit - w.before - job * r.tiles;
    s.i1 = min(r.tiles, s.i0 + w.end - w.unit);
    w.unit += s.i1 - s.i0;
    return true;
}

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

// The largest of three; one that is no number wins.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <int DP>
__global__ void __launch_bounds__(THREADS)
tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                         const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_vn, const TreeArgs A, const Line line,
                         int ps_shift, float scale_log2) {
    constexpr int HALVES = DP / 64, NS = stages(DP);
    constexpr uint32_t Q_ONE = HALVES * RT * 128, Q_BYTES = 2 * Q_ONE, KV_HALF = KT * 128, KV_BYTES = HALVES * KV_HALF, STAGE_BYTES = 2 * KV_BYTES;
    constexpr uint32_t BAR_OFF = Q_BYTES + NS * STAGE_BYTES, RING = 8 * NS;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t base = smem_u32(smem_raw), q_sm = base, kv_sm = base + Q_BYTES, bars = base + BAR_OFF;
    const uint32_t k_full0 = bars, k_empty0 = bars + RING, v_full0 = bars + 2 * RING, v_empty0 = bars + 3 * RING, rest = bars + 4 * RING;
    const uint32_t s_ready0 = rest, pv_done0 = rest + 32, p_ready0 = rest + 64, q_full = rest + 80, q_empty = rest + 96, looked0 = rest + 104;
    volatile uint32_t* words = reinterpret_cast<volatile uint32_t*>(smem_raw + BAR_OFF + 4 * RING + 120);   // tmem, dead, then the value rows that are
    volatile uint32_t* odd_rows = words + 2;                                                                // not finite: [4 looks][2 words]
    LineShared& line_sh = *reinterpret_cast<LineShared*>(smem_raw + BAR_OFF + 512);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4 * NS; ++i) mbar_init(bars + 8 * i, 1);
        for (int i = 0; i < 4; ++i) mbar_init(s_ready0 + 8 * i, 1), mbar_init(pv_done0 + 8 * i, 1);
        mbar_init(p_ready0, 128);
        mbar_init(p_ready0 + 8, 128);
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(looked0, 2);
        mbar_init(looked0 + 8, 2);
        mbar_init_fence();
    }
    constexpr uint32_t TMEM_COLS = 512;
    if (warp == 0) tmem_alloc(const_cast<uint32_t*>(&words[0]), TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = words[0];
    pdl_launch_dependents();       // only now: see pdl_launch_dependents on tensor memory
    pdl_wait();                    // lengths, rows and masks may come from the kernel before
    if (threadIdx.x == 0) {
        if (base & 1023u) atomicOr(A.err, XB_ERR_WAIT);                                        // the swizzle needs a 1024-byte aligned window
        words[1] = (*reinterpret_cast<volatile int*>(A.err) & XB_ERR_WAIT) ? 1u : 0u;          // or an earlier block gave up: do not pile on
    }
    const LinePlace at = place_in_line(A, line, line_sh);
    const Walk start{at.request, at.before, at.unit, words[1] ? at.unit : at.end};
    const bool out16 = rows_on_16_bytes(A.out, A.out_stride);
    const int G = A.nh / A.nkv, half_nodes = line.half_nodes;
    const int box_rows = min(A.page_size, KT);
    int* err = A.err;

    if (warp == 8 || warp == 10) {
        // ---- keys (warp 8) and values (warp 10), a lane per box ----------------------------------------------------------
        const bool is_v = warp == 10;
        const uint32_t full0 = is_v ? v_full0 : k_full0, empty0 = is_v ? v_empty0 : k_empty0;
        const CUtensorMap* map = is_v ? &map_v : &map_k;
        const CUtensorMap* map_new = is_v ? &map_vn : &map_kn;
        const int boxes = KT / box_rows * HALVES, bi = lane / HALVES, hf = lane % HALVES;
        int st = 0;
        uint32_t ph = 0;
        bool rounds = false, ok = true;
        Walk w = start;
        Segment s;
        while (ok && next_segment(A, line, w, s)) {
            const int* table = A.block_table + (size_t)s.b * A.table_stride;
            auto page_of = [&](int it) -> int {            // the page of this lane's box, -1: nothing to load
                if (it >= s.i1 || it >= s.old_tiles || lane >= boxes) return -1;
                const int j = (s.tile0 + it) * KT + bi * box_rows;
                if (j >= s.context) return -1;
                const int page = table[j >> ps_shift];
                if (page < 0 || page >= A.num_pages) {
                    atomicOr(err, XB_ERR_BAD_PAGE);
                    return A.num_pages;                    // behind the last page: the box reads as zeros
                }
                return page;
            };
            int page_next = page_of(s.i0);
            for (int it = s.i0; it < s.i1; ++it) {
                const int page = page_next;
                if (rounds && !__all_sync(0xffffffffu, mbar_wait(empty0 + 8 * st, ph ^ 1u, err))) {
                    words[1] = 1;
                    ok = false;
                    break;
                }
                const uint32_t dst0 = kv_sm + st * STAGE_BYTES + (is_v ? KV_BYTES : 0u);
                if (it < s.old_tiles) {
                    const uint32_t nb = __popc(__ballot_sync(0xffffffffu, page >= 0));
                    if (lane == 0) mbar_expect_tx(full0 + 8 * st, nb * box_rows * 128);
                    __syncwarp();
                    if (page >= 0) {
                        const int j = (s.tile0 + it) * KT + bi * box_rows;
                        tma_load_2d(dst0 + hf * KV_HALF + bi * box_rows * 128, map, hf * 64, (page * A.nkv + s.g) * A.page_size + (j & (A.page_size - 1)), full0 + 8 * st);
                    }
                } else {
                    if (lane == 0) mbar_expect_tx(full0 + 8 * st, KV_BYTES);
                    __syncwarp();
                    if (lane < HALVES) tma_load_3d(dst0 + lane * KV_HALF, map_new, lane * 64, s.g, s.tree0 + (it - s.old_tiles) * KT, full0 + 8 * st);
                }
                page_next = page_of(it + 1);
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                    rounds = true;
                }
            }
        }
    } else if (warp == 9) {
        // ---- Q, then S = Q K^T of every tile --------------------------------------------------------------------------------
        const bool leader = lane == 0;
        const uint32_t idesc_s = umma_idesc(KT, 0);
        const uint64_t dq0 = umma_desc(q_sm, 16, 1024), dk0 = umma_desc(kv_sm, 16, 1024);
        int st = 0, Th[2] = {0, 0}, I = 0;       // ring stage, tiles of either row tile so far, segments so far
        uint32_t ph = 0;
        bool ok = true;
        Walk w = start;
        Segment s;
        while (ok && next_segment(A, line, w, s)) {
            const int halves = s.nodes > half_nodes ? 2 : 1;
            if (I > 0) {                         // Q lies where the last one lay: once every product that reads that has completed
                if (leader) umma_commit(q_empty);
                __syncwarp();
                ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (uint32_t)(I - 1) & 1u, err, true));
                if (!ok) break;
            }
            if (leader) {
                mbar_expect_tx(q_full, (uint32_t)(halves * HALVES * half_nodes * G * 128));
                for (int hd = 0; hd < halves; ++hd)
#pragma unroll
                    for (int hf = 0; hf < HALVES; ++hf)
                        tma_load_3d(q_sm + hd * Q_ONE + hf * RT * 128, &map_q, hf * 64, s.g * G, s.t0 + hd * half_nodes, q_full);
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, mbar_wait(q_full, (uint32_t)I & 1u, err, true));
            ++I;
            for (int it = s.i0; it < s.i1 && ok; ++it) {
                ok = __all_sync(0xffffffffu, mbar_wait(k_full0 + 8 * st, ph, err, true));
                const uint64_t dk = dk0 + (uint64_t)((st * STAGE_BYTES) >> 4);
#pragma unroll
                for (int hd = 0; hd < 2; ++hd) {
                    if (hd >= halves) break;
                    const int th = Th[hd]++, sb = th & 1;
                    // these columns held the scores and then P of this row tile's last tile but one: its P V must have read them
                    ok = ok && (th < 2 || __all_sync(0xffffffffu, mbar_wait(pv_done0 + 8 * (2 * hd + sb), ((th >> 1) - 1) & 1, err, true)));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dq = dq0 + (uint64_t)((hd * Q_ONE) >> 4);
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < DP / 16; ++kk) {
                            const uint32_t off = (kk >> 2), inner = (kk & 3) * 32;
                            umma_bf16(tmem + (uint32_t)(hd * 128 + sb * 64), dq + (uint64_t)((off * RT * 128 + inner) >> 4),
                                      dk + (uint64_t)((off * KV_HALF + inner) >> 4), idesc_s, kk ? 1u : 0u);
                        }
                        umma_commit(s_ready0 + 8 * (2 * hd + sb));
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (leader) umma_commit(k_empty0 + 8 * st);
                __syncwarp();
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        }
        if (!ok) words[1] = 1;
    } else if (warp == 11) {
        // ---- O += P V of every tile (O starts as zeros, by the softmax threads) -----------------------------------------------
        const bool leader = lane == 0;
        const uint32_t idesc_o = umma_idesc(DP, 1);
        const uint64_t dv0 = umma_desc(kv_sm + KV_BYTES, KV_HALF, 1024);
        int st = 0, Th[2] = {0, 0};
        uint32_t ph = 0;
        bool ok = true;
        Walk w = start;
        Segment s;
        while (ok && next_segment(A, line, w, s)) {
            const int halves = s.nodes > half_nodes ? 2 : 1;
            for (int it = s.i0; it < s.i1 && ok; ++it) {
                ok = __all_sync(0xffffffffu, mbar_wait(v_full0 + 8 * st, ph, err, true));
                const uint64_t dv = dv0 + (uint64_t)((st * STAGE_BYTES) >> 4);
#pragma unroll
                for (int hd = 0; hd < 2; ++hd) {
                    if (hd >= halves) break;
                    const int th = Th[hd]++, sb = th & 1;
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(p_ready0 + 8 * hd, th & 1, err, true));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t tp = tmem + (uint32_t)(hd * 128 + sb * 64);
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < KT / 16; ++kk)
                            umma_bf16_ta(tmem + (uint32_t)(256 + hd * 128), tp + (uint32_t)(kk * 8), dv + (uint64_t)((kk * 2048) >> 4), idesc_o, 1u);
                        umma_commit(pv_done0 + 8 * (2 * hd + sb));
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (leader) umma_commit(v_empty0 + 8 * st);
                __syncwarp();
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        }
        if (!ok) words[1] = 1;
    } else {
        // ---- softmax: a row per thread ---------------------------------------------------------------------------------------------
        const int hd = warp >> 2, r = (int)threadIdx.x & 127;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem + (uint32_t)(hd * 128), tmem_o = tmem + (uint32_t)(256 + hd * 128);
        const uint32_t my_s_ready = s_ready0 + 16 * hd, my_p_ready = p_ready0 + 8 * hd, my_pv_done = pv_done0 + 16 * hd;
        const int node_r = r / G, head_r = r % G;
        const bool warp_rows = (warp & 3) * 32 < half_nodes * G;
        int T = 0, Th = 0, looks = 0;            // tiles of all segments so far, of this row tile's, tiles that were looked at
        bool alive = true;
        Walk w = start;
        Segment s;
        while (alive && next_segment(A, line, w, s)) {
            const int window = A.window, iters = s.i1 - s.i0;
            // whether the tile's keys are not seen alike by all rows (the windows of deeper nodes begin later)
            int deep_lo = 0;                              // where the deepest node's begins
            if (window > 0) {
                int deepest = 0;
                for (int i = lane; i < s.tree_n; i += 32) deepest = max(deepest, A.depth[s.tree0 + i]);
                deep_lo = s.context + __reduce_max_sync(0xffffffffu, deepest) - window + 1;
            }
            auto mixed = [&](int it) { return it >= s.old_tiles || (window > 0 && (s.tile0 + it) * KT < deep_lo); };
            if (hd == 1 && s.nodes <= half_nodes) {       // a segment of one row tile: the second one's threads sit it out
                for (int it = s.i0; it < s.i1; ++it) looks += mixed(it) ? 1 : 0;
                T += iters;
                continue;
            }
            const int node = s.node0 + hd * half_nodes + node_r;         // in its tree
            const bool valid = node_r < half_nodes && node < s.node0 + s.nodes;
            const bool working = warp_rows && __any_sync(0xffffffffu, valid);
            const int t = s.tree0 + node, h = s.g * G + head_r;
            const int my_depth = valid && window > 0 ? max(0, A.depth[t]) : 0;
            const int my_lo = window > 0 ? max(0, s.context + my_depth - window + 1) : 0;
            const int* my_words = A.ancestors + (size_t)(valid ? t : s.t0) * A.words;
            uint32_t word_lo = 0, word_hi = 0;            // of the first drafted tile
            if (valid && s.i1 > s.old_tiles) {
                word_lo = A.words > 0 ? (uint32_t)my_words[0] : 0u;
                word_hi = A.words > 1 ? (uint32_t)my_words[1] : 0u;
            }
            {
                float zero[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) zero[i] = 0.f;
#pragma unroll
                for (int c0 = 0; c0 < DP; c0 += 32) tmem_st32(tmem_o + lane_addr + c0, zero);
            }
            float m_ref = -INFINITY, l = 0.f;
            for (int it = s.i0; it < s.i1; ++it) {
                const int n_it = it - s.i0, th = Th + n_it, sb = th & 1, gt = T + n_it, st = gt % NS;
                const bool drafted = it >= s.old_tiles, look = mixed(it);
                const int key0 = drafted ? (it - s.old_tiles) * KT : (s.tile0 + it) * KT;
                const int keys = drafted ? s.tree_n : s.context;          // keys from here on belong to nobody
                const bool edge = look || key0 + KT > keys;
                // the value rows: zeroed where nobody may see them, and in tiles that are not seen alike where they are not finite
                if (hd == 0 && edge && r < KT) {
                    alive = __all_sync(0xffffffffu, mbar_wait(v_full0 + 8 * st, (gt / NS) & 1, err));   // orders these accesses after the copy
                    uint4* row = reinterpret_cast<uint4*>(smem_raw + Q_BYTES + st * STAGE_BYTES + KV_BYTES + r * 128);
                    bool drop = key0 + r >= keys || (!drafted && key0 + r < (window > 0 ? max(0, s.context - window + 1) : 0)), odd = false;
                    if (look && !drop) {
#pragma unroll
                        for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
                            for (int c8 = 0; c8 < 8; ++c8) odd |= bf16_not_finite(row[hf * (KV_HALF / 16) + c8]);
                    }
                    if (alive && (drop || odd)) {
#pragma unroll
                        for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll
                            for (int c8 = 0; c8 < 8; ++c8) row[hf * (KV_HALF / 16) + c8] = make_uint4(0, 0, 0, 0);
                    }
                    const uint32_t odd_mask = __ballot_sync(0xffffffffu, odd);
                    fence_async_shared();          // the zeroed rows: visible to the product
                    __syncwarp();
                    if (look && lane == 0) {
                        odd_rows[(looks & 3) * 2 + warp] = odd_mask;
                        mbar_arrive(looked0 + 8 * (looks & 1));
                    }
                    if (!alive) break;
                }
                if (!__all_sync(0xffffffffu, mbar_wait(my_s_ready + 8 * sb, (th >> 1) & 1, err))) {
                    alive = false;
                    break;
                }
                float corr = 1.f;
                int moved = 0;
                unsigned long long seen = ~0ull;
                if (working) {
                    tc_fence_after();
                    float sc[64];
                    {
                        uint32_t ra[32], rb[32];
                        tmem_ld32_nowait(tmem_s + sb * 64 + lane_addr, ra);
                        tmem_ld32_nowait(tmem_s + sb * 64 + lane_addr + 32, rb);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            sc[i] = __uint_as_float(ra[i]);
                            sc[32 + i] = __uint_as_float(rb[i]);
                        }
                    }
                    if (edge) {
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
                                    if (my_depth - max(0, A.depth[s.tree0 + key0 + i]) >= window) seen &= ~(1ull << i);
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
                        m_ref = mx;
                        moved = n_it > 0 && valid;
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
                        if (edge) {                // the polynomial ends at 2^-126: a key that is not seen has no weight at all
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
                    tmem_st32_u(tmem_s + sb * 64 + lane_addr, pk);       // P goes where the scores were
                }
                // O is not touched, and this tile not announced, before the last tile's P V has completed: the issuer waits for
                // announcements by their parity, so none may be two of them ahead
                if (n_it > 0 && !__all_sync(0xffffffffu, mbar_wait(my_pv_done + 8 * (sb ^ 1), ((th - 1) >> 1) & 1, err))) {
                    alive = false;
                    break;
                }
                if (__any_sync(0xffffffffu, moved)) {
                    tc_fence_after();
                    const float f = moved ? corr : 1.f;
#pragma unroll
                    for (int c0 = 0; c0 < DP; c0 += 32) {
                        float o[32];
                        tmem_ld32(tmem_o + lane_addr + c0, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= f;
                        tmem_st32(tmem_o + lane_addr + c0, o);
                    }
                }
                tmem_st_wait();
                if (look) {
                    if (!__all_sync(0xffffffffu, mbar_wait(looked0 + 8 * (looks & 1), (looks >> 1) & 1, err))) {
                        alive = false;
                        break;
                    }
                    const uint32_t odd_lo = odd_rows[(looks & 3) * 2], odd_hi = odd_rows[(looks & 3) * 2 + 1];
                    ++looks;
                    if ((odd_lo | odd_hi) && working) {    // (rare) the same for all lanes
                        tc_fence_after();
                        for (int i = 0; i < 64; ++i) {
                            if (!((i < 32 ? odd_lo >> i : odd_hi >> (i - 32)) & 1u)) continue;
                            const uint32_t two = tmem_ld1(tmem_s + sb * 64 + lane_addr + (uint32_t)(i >> 1));
                            const float p = __uint_as_float((i & 1) ? two & 0xffff0000u : two << 16);
                            const bool mine = valid && (seen >> i & 1ull);
                            const __nv_bfloat16* v;
                            if (drafted) {
                                v = (const __nv_bfloat16*)A.v_new + (size_t)(s.tree0 + key0 + i) * A.v_stride + (size_t)s.g * A.d;
                            } else {
                                const int j = key0 + i, page = A.block_table[(size_t)s.b * A.table_stride + (j >> ps_shift)];
                                v = (const __nv_bfloat16*)A.v_cache + (((size_t)page * A.nkv + s.g) * A.page_size + (j & (A.page_size - 1))) * A.d;
                            }
#pragma unroll 1
                            for (int c0 = 0; c0 < DP; c0 += 32) {
                                float o[32];
                                tmem_ld32(tmem_o + lane_addr + c0, o);
#pragma unroll
                                for (int c = 0; c < 32; ++c)
                                    if (mine && c0 + c < A.d) o[c] = fmaf(p, __bfloat162float(v[c0 + c]), o[c]);
                                tmem_st32(tmem_o + lane_addr + c0, o);
                            }
                            tmem_st_wait();
                        }
                    }
                }
                tc_fence_before();
                mbar_arrive(my_p_ready);
            }
            // ---- O / l, or this part of a job that blocks share -----------------------------------------------------------------------
            if (alive) alive = mbar_wait(my_pv_done + 8 * ((Th + iters - 1) & 1), ((Th + iters - 1) >> 1) & 1, err);
            alive = __all_sync(0xffffffffu, alive);
            if (alive && working) {
                tc_fence_after();
                const bool whole = iters == s.tiles;
                const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
                const size_t part = part_row(line, blockIdx.x, s.i0 > 0 ? 0 : 1, (node - s.node0) * G + head_r);
#pragma unroll
                for (int c0 = 0; c0 < DP; c0 += 32) {
                    float o[32];
                    tmem_ld32(tmem_o + lane_addr + c0, o);
                    if (!valid) continue;
                    if (whole) {
                        __nv_bfloat16* dst = (__nv_bfloat16*)A.out + (size_t)t * A.out_stride + (size_t)h * A.d;
#pragma unroll
                        for (int c8 = 0; c8 < 4; ++c8) {
                            const int c = c0 + c8 * 8;
                            if (c < A.d) {
                                uint4 v;
                                v.x = pack_bf16(o[c8 * 8] * inv, o[c8 * 8 + 1] * inv);
                                v.y = pack_bf16(o[c8 * 8 + 2] * inv, o[c8 * 8 + 3] * inv);
                                v.z = pack_bf16(o[c8 * 8 + 4] * inv, o[c8 * 8 + 5] * inv);
                                v.w = pack_bf16(o[c8 * 8 + 6] * inv, o[c8 * 8 + 7] * inv);
                                store8(dst + c, v, out16);
                            }
                        }
                    } else {
                        float* dst = line.part_o + part * A.d;
#pragma unroll
                        for (int c4 = 0; c4 < 8; ++c4) {
                            const int c = c0 + c4 * 4;
                            if (c < A.d) *reinterpret_cast<float4*>(dst + c) = make_float4(o[c4 * 4], o[c4 * 4 + 1], o[c4 * 4 + 2], o[c4 * 4 + 3]);
                        }
                    }
                }
                if (valid && !whole) {
                    line.part_ml[part * 2] = m_ref;
                    line.part_ml[part * 2 + 1] = l;
                }
            }
            T += iters;
            Th += iters;
        }
        if (!alive) words[1] = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_free(tmem, TMEM_COLS);
}

// Joins the parts of rows that several blocks shared, in the order of the parts: with M the largest of their maxima,
// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.  A warp per row.
__global__ void __launch_bounds__(128)
tree_merge_kernel(const TreeArgs A, const Line line) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(item / A.nh), h = (int)(item % A.nh);
    if (t >= A.tokens || (*reinterpret_cast<volatile int*>(A.err) & XB_ERR_WAIT)) return;
    const int b = request_of(A, t);
    if (b < 0) return;
    const RequestLine r = request_line(A, line, b);
    const int share = line.starts[A.requests], G = A.nh / A.nkv, node = t - r.first, piece = node / line.job_nodes;
    const int unit0 = line.starts[b] + (h / G * (r.jobs / A.nkv) + piece) * r.tiles, c0 = unit0 / share, c1 = (unit0 + r.tiles - 1) / share;
    if (c0 == c1) return;
    const int row = (node - piece * line.job_nodes) * G + h % G, parts = c1 - c0 + 1;
    auto at = [&](int i) { return part_row(line, c0 + i, i > 0 ? 0 : 1, row); };
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 32) M = fmaxf(M, __ldcg(line.part_ml + at(i) * 2));
    M = warp_max(M);
    const float base = M == -INFINITY ? 0.f : M;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, W = 0.f;
    const int c = lane * 4;
    for (int i = 0; i < parts; ++i) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(line.part_ml + at(i) * 2));
        const float f = exp2f(ml.x - base);
        W = fmaf(f, ml.y, W);
        if (c < A.d) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(line.part_o + at(i) * A.d + c));
            acc[0] = fmaf(f, v.x, acc[0]);
            acc[1] = fmaf(f, v.y, acc[1]);
            acc[2] = fmaf(f, v.z, acc[2]);
            acc[3] = fmaf(f, v.w, acc[3]);
        }
    }
    const float inv = W > 0.f || W != W ? 1.f / W : 0.f;
    if (c < A.d) {
        __nv_bfloat16* dst = (__nv_bfloat16*)A.out + (size_t)t * A.out_stride + (size_t)h * A.d + c;
        if (rows_on_16_bytes(A.out, A.out_stride)) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = __float2bfloat16_rn(acc[i] * inv);
        }
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

template <int DP>
int launch_tc(const TreeArgs& A, const Line& line, cudaStream_t stream) {
    constexpr int NS = stages(DP);
    constexpr size_t smem = 2 * (DP / 64) * RT * 128 + NS * 2 * (DP / 64) * KT * 128 + 1024;
    static const cudaError_t room = cudaFuncSetAttribute(tree_attention_tc_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (room != cudaSuccess) return (int)room;
    const int G = A.nh / A.nkv, box_rows = A.page_size < KT ? A.page_size : KT;
    int shift = 0;
    while ((1 << shift) < A.page_size) ++shift;
    CUtensorMap mq, mk, mv, mkn, mvn;
    const long long rows = (long long)A.num_pages * A.nkv * A.page_size;
    const long long dq[3] = {A.d, A.nh, A.tokens}, dn[3] = {A.d, A.nkv, A.tokens};
    const long long sq[2] = {A.d, A.q_stride}, sk[2] = {A.d, A.k_stride}, sv[2] = {A.d, A.v_stride};
    const int bq[3] = {64, G, line.half_nodes}, bn[3] = {64, 1, KT};
    if (!tensor_map_bf16(&mq, A.q, 3, dq, sq, bq) || !tensor_map_2d(&mk, A.k_cache, rows, A.d, box_rows) || !tensor_map_2d(&mv, A.v_cache, rows, A.d, box_rows) ||
        !tensor_map_bf16(&mkn, A.k_new, 3, dn, sk, bn) || !tensor_map_bf16(&mvn, A.v_new, 3, dn, sv, bn))
        return (int)cudaErrorInvalidValue;
    const int rc = xb_launch(tree_attention_tc_kernel<DP>, dim3(line.blocks), dim3(THREADS), smem, stream, mq, mk, mv, mkn, mvn, A, line, shift, A.scale * 1.4426950408889634f);
    if (rc) return rc;
    return xb_launch(tree_merge_kernel, dim3((unsigned)(((long long)A.tokens * A.nh + 3) / 4)), dim3(128), 0, stream, A, line);
}

}  // namespace

namespace xbtree {

bool tree_tc_takes(const TreeArgs& A) {
    return A.d % 16 == 0 && A.d >= 16 && A.d <= 128 && A.nh / A.nkv <= RT && A.page_size >= 8 && (A.page_size & (A.page_size - 1)) == 0 &&
           ((long long)A.num_pages + 1) * A.nkv * A.page_size < (1LL << 31) && rows_on_16_bytes(A.k_cache, 0) && rows_on_16_bytes(A.v_cache, 0);
}

int tree_tc_launch(const TreeArgs& given, float* scratch, cudaStream_t stream) {
    TreeArgs A = given;
    const Line line = make_line(A, scratch);
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
