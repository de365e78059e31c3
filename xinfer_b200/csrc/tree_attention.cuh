// What the kernels of attention over a tree of drafted tokens share (tree_attention.cu says what they compute).
#pragma once
#include "common.cuh"

namespace xbtree {

struct TreeArgs {
    void* out;                     // [tokens, nh, d], tokens `out_stride` elements apart; q, k_new and v_new alike
    const void* q;
    const void* k_new;             // [tokens, nkv, d]: the drafted tokens' own keys and values
    const void* v_new;
    const void* k_cache;           // [pages, nkv, page_size, d]
    const void* v_cache;
    const int* context;            // [requests]: cached keys
    const int* token_start;        // [requests + 1]
    const int* ancestors;          // [tokens, words]: bit i of the words, lowest first: the node sees node i of its own tree
    const int* depth;              // [tokens], null without a window
    const int* block_table;        // [requests, table_stride]
    long long out_stride, q_stride, k_stride, v_stride;
    int tokens, requests, words, table_stride, nh, nkv, d, page_size, num_pages, window;
    float scale;
    int* err;
};

// Starts outside the tokens would be reads outside the rows: they count as the nearest bound.
__device__ __forceinline__ int clamp_start(const TreeArgs& A, int start) { return min(max(start, 0), A.tokens); }

// A context beyond the row of the block table is reported and cut to it.
__device__ __forceinline__ int context_of(const TreeArgs& A, int b) {
    const int c = A.context[b];
    const long long most = (long long)A.table_stride * A.page_size;
    if (c > most) atomicOr(A.err, XB_ERR_BAD_PAGE);
    return c < 0 ? 0 : (int)(c > most ? most : c);
}

// The request that token t belongs to: the last one that starts at or before it; -1 for a token behind them all.
__device__ __forceinline__ int request_of(const TreeArgs& A, int t) {
    if (t < A.token_start[0] || t >= A.token_start[A.requests]) return -1;
    int lo = 0, hi = A.requests;             // token_start[lo] <= t < token_start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (A.token_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---- the line of all jobs' tiles -------------------------------------------------------------------------------------------
// A job is (request, key/value head, up to job_nodes nodes); its tiles of KT keys are the cached ones from the first that a node sees
// and the drafted ones.  The line holds all jobs' tiles, request by request, each as long as it costs: block c takes the tiles that begin
// in c * share .. (c + 1) * share - 1.
constexpr int KT = 64;
constexpr int LINE_BLOCKS = 148;   // a block per SM
constexpr int LINE_REQUESTS = 8192;
constexpr int MIN_SHARE = 4;       // tiles that a block takes at least: below that its start and the join cost more than they save
constexpr int TILE_ROWS = 128;     // rows (node, query head of the group) of a product; a job has up to two such tiles
constexpr int COST_ONE = 2;        // what a tile of keys costs a job of one tile of rows, and of two: 1,400 and 2,150 cycles measured
constexpr int COST_TWO = 3;
constexpr int COST_JOB = 8;        // what a job costs beside its tiles: its last, drafted keys and its result

struct Line {
    int half_nodes, job_nodes;     // nodes of a tile of rows and of a job
    int part_rows;                 // rows of a part that is kept for the join: a multiple of 8
    float* part_o;                 // [blocks][2][part_rows / 8][d / 4][8][4]: a block's first segment, if its job began before it, and its last,
                                   // if its job goes on; four channels of eight rows lie together, as a warp writes and reads them
    float* part_ml;                // [blocks][2][part_rows][2]: maximum and sum
    int* shared_jobs;              // [blocks][2][8]: the jobs of these parts: parts (0: there is no such part), block of the first, first node's
                                   // row, nodes, key/value head
    float* dense;                  // room for q, k_new and v_new as dense rows of bfloat16
};

struct RequestLine {
    int first, nodes, context, tile0, old_tiles, tiles, pieces;
    int per_tile;                  // what a tile costs each of its jobs
    __device__ __forceinline__ int job_units() const { return tiles * per_tile + COST_JOB; }
    __device__ __forceinline__ int units(int nkv) const { return nkv * pieces * job_units(); }
};

__device__ __forceinline__ RequestLine request_line(const TreeArgs& A, const Line& line, int b) {
    RequestLine r;
    r.first = clamp_start(A, A.token_start[b]);
    r.nodes = max(0, clamp_start(A, A.token_start[b + 1]) - r.first);
    r.context = context_of(A, b);
    r.tile0 = A.window > 0 ? max(0, r.context - A.window + 1) / KT : 0;    // (the root's window begins first)
    r.old_tiles = max(0, (r.context + KT - 1) / KT - r.tile0);
    r.tiles = r.old_tiles + (r.nodes + KT - 1) / KT;
    r.pieces = (r.nodes + line.job_nodes - 1) / line.job_nodes;
    r.per_tile = r.nodes > line.half_nodes ? COST_TWO : COST_ONE;
    return r;
}

// Where a block stands in the line; walked by one warp, whose lanes hold the same values.
struct Walk {
    RequestLine r;                 // of request b
    int b, g, piece;               // the job: request, key/value head, which of their pieces
    int job, from, end, share;     // where the job begins in the line, the block's range, a block's share
    int i0, i1;                    // the block's tiles of the job's
};

// (x > 0) / cost, upwards
__device__ __forceinline__ int tiles_of_cost(int x, int cost) { return cost == COST_TWO ? (x + COST_TWO - 1) / COST_TWO : (x + COST_ONE - 1) / COST_ONE; }

// The block's place before its first job: every lane sums a run of the requests.
__device__ __forceinline__ Walk place_in_line(const TreeArgs& A, const Line& line) {
    const int lane = threadIdx.x & 31, each = (A.requests + 31) / 32, b0 = lane * each, b1 = min(b0 + each, A.requests);
    Walk w;
    int mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        w.r = request_line(A, line, b);
        mine += w.r.units(A.nkv);
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    w.share = max(MIN_SHARE * COST_TWO, (total + LINE_BLOCKS - 1) / LINE_BLOCKS);
    w.from = (int)min((long long)blockIdx.x * w.share, (long long)total);
    w.end = min(total, w.from + w.share);
    w.job = w.end;
    w.b = w.g = w.piece = w.i0 = w.i1 = 0;
    if (w.from >= w.end) return w;
    int before = incl - mine, b = b0;
    const unsigned who = __ballot_sync(0xffffffffu, w.from >= before && w.from < incl);
    const int owner = __ffs(who) - 1;
    if (lane == owner) {
#pragma unroll 1
        for (; b < b1; ++b) {
            if (each > 1) w.r = request_line(A, line, b);
            const int n = w.r.units(A.nkv);
            if (w.from < before + n) break;
            before += n;
        }
    }
    w.b = __shfl_sync(0xffffffffu, b, owner);
    before = __shfl_sync(0xffffffffu, before, owner);
    w.r = request_line(A, line, w.b);
    const int length = w.r.job_units(), at = (w.from - before) / length;
    w.g = at / w.r.pieces;
    w.piece = at % w.r.pieces;
    w.job = before + at * length;
    return w;
}

// The next job of which the block has a part; false: there is none.  (The first tile that begins at or behind `from` may be the next
// job's, or the next request's first.)
__device__ __forceinline__ bool next_segment(const TreeArgs& A, const Line& line, Walk& w, bool first) {
    for (;; first = false) {
        if (!first) w.job += w.r.job_units();
        if (w.job >= w.end) return false;
        if (!first && ++w.piece == w.r.pieces) {
            w.piece = 0;
            if (++w.g == A.nkv) {
                w.g = 0;
                do {
                    if (++w.b >= A.requests) return false;
                    w.r = request_line(A, line, w.b);
                } while (w.r.nodes == 0);                          // (a request without nodes has no jobs)
            }
        }
        w.i0 = w.from > w.job ? tiles_of_cost(w.from - w.job, w.r.per_tile) : 0;
        w.i1 = min(w.r.tiles, tiles_of_cost(w.end - w.job, w.r.per_tile));
        if (w.i0 < w.i1) return true;
    }
}

__device__ __forceinline__ size_t part_row(const Line& line, int block, int which, int row) { return ((size_t)block * 2 + which) * line.part_rows + row; }
// where four channels of a part's row lie, in float4
__device__ __forceinline__ size_t part_four(const Line& line, int d, size_t row, int c4) { return ((row >> 3) * (d >> 2) + c4) * 8 + (row & 7); }

// host: the scratch in float32 numbers, and its layout (every part is a multiple of 4 numbers long)
inline int line_part_rows(int tokens, int group) {
    const int nodes = 2 * (TILE_ROWS / (group < TILE_ROWS ? group : TILE_ROWS));
    return ((tokens < nodes ? tokens : nodes) * group + 7) / 8 * 8;
}
inline long long line_floats(int tokens, int nh, int nkv, int d) {
    return (long long)LINE_BLOCKS * (2 * line_part_rows(tokens, nh / nkv) * (long long)(d + 2) + 16) + ((long long)tokens * (nh + 2 * nkv) * d + 1) / 2;
}
inline Line make_line(const TreeArgs& A, float* scratch) {
    const int G = A.nh / A.nkv;
    Line line;
    line.half_nodes = TILE_ROWS / G;
    line.job_nodes = 2 * line.half_nodes;
    line.part_rows = line_part_rows(A.tokens, G);
    line.part_o = scratch;
    line.part_ml = scratch + (size_t)LINE_BLOCKS * 2 * line.part_rows * A.d;
    line.shared_jobs = reinterpret_cast<int*>(line.part_ml + (size_t)LINE_BLOCKS * 2 * line.part_rows * 2);
    line.dense = reinterpret_cast<float*>(line.shared_jobs) + LINE_BLOCKS * 16;
    return line;
}

// tree_attention_tc.cu
bool tree_tc_takes(const TreeArgs& A);
int tree_tc_launch(const TreeArgs& A, float* scratch, cudaStream_t stream);

}  // namespace xbtree
