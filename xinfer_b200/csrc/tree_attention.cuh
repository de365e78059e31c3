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
// and the drafted ones.  The line holds all jobs' tiles, request by request; block c takes the units c * share .. (c + 1) * share - 1.
constexpr int KT = 64;
constexpr int LINE_BLOCKS = 148;   // a block per SM
constexpr int LINE_REQUESTS = 8192;
constexpr int MIN_SHARE = 4;       // tiles that a block takes at least: below that its start and the join cost more than they save

struct Line {
    int half_nodes, job_nodes;     // nodes of a tile of rows and of a job
    int blocks, part_rows;         // rows of a part that is kept for the join
    float* part_o;                 // [blocks][2][part_rows][d]: a block's first segment, if its job began before it, and its last, if its job goes on
    float* part_ml;                // [blocks][2][part_rows][2]: maximum and sum
    int* starts;                   // [requests + 1]: units before each request, then the share
    float* dense;                  // room for q, k_new and v_new as dense rows of bfloat16
};

struct RequestLine {
    int first, nodes, context, tile0, old_tiles, tiles, jobs;
};

__device__ __forceinline__ RequestLine request_line(const TreeArgs& A, const Line& line, int b) {
    RequestLine r;
    r.first = clamp_start(A, A.token_start[b]);
    r.nodes = max(0, clamp_start(A, A.token_start[b + 1]) - r.first);
    r.context = context_of(A, b);
    r.tile0 = A.window > 0 ? max(0, r.context - A.window + 1) / KT : 0;    // (the root's window begins first)
    r.old_tiles = max(0, (r.context + KT - 1) / KT - r.tile0);
    r.tiles = r.old_tiles + (r.nodes + KT - 1) / KT;
    r.jobs = A.nkv * ((r.nodes + line.job_nodes - 1) / line.job_nodes);
    return r;
}

__device__ __forceinline__ size_t part_row(const Line& line, int block, int which, int row) { return ((size_t)block * 2 + which) * line.part_rows + row; }

struct LineShared {
    int of_warps[32];
    int request, before;
};
struct LinePlace {
    int request, before, unit, end;    // the request of the block's first unit, the units before it, the block's units
};

// Where this block begins; every thread of the block takes part.  Block 0 writes line.starts.
__device__ __forceinline__ LinePlace place_in_line(const TreeArgs& A, const Line& line, LineShared& sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int each = (A.requests + blockDim.x - 1) / blockDim.x, b0 = (int)threadIdx.x * each, b1 = min(b0 + each, A.requests);
    auto units = [&](int b) {
        const RequestLine r = request_line(A, line, b);
        return r.jobs * r.tiles;
    };
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += units(b);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) sh.of_warps[warp] = incl;
    __syncthreads();
    int before = incl - mine, total = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) before += sh.of_warps[w];
        total += sh.of_warps[w];
    }
    const int share = max(MIN_SHARE, (total + line.blocks - 1) / line.blocks), unit = min((long long)blockIdx.x * share, (long long)total);
    for (int b = b0; b < b1; ++b) {
        const int n = units(b);
        if (unit >= before && unit < before + n) {
            sh.request = b;
            sh.before = before;
        }
        if (blockIdx.x == 0) line.starts[b] = before;
        before += n;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) line.starts[A.requests] = share;
    __syncthreads();
    return LinePlace{sh.request, sh.before, unit, min(total, unit + share)};
}

// host: the scratch in float32 numbers, and its layout
constexpr int TILE_ROWS = 128;
inline int line_part_rows(int tokens, int group) {
    const int nodes = 2 * (TILE_ROWS / (group < TILE_ROWS ? group : TILE_ROWS));
    return (tokens < nodes ? tokens : nodes) * group;
}
inline long long line_floats(int tokens, int nh, int nkv, int d) {
    return (long long)LINE_BLOCKS * 2 * line_part_rows(tokens, nh / nkv) * (d + 2) + LINE_REQUESTS + 4 + ((long long)tokens * (nh + 2 * nkv) * d + 1) / 2;
}
inline Line make_line(const TreeArgs& A, float* scratch) {
    const int G = A.nh / A.nkv;
    Line line;
    line.half_nodes = TILE_ROWS / G;
    line.job_nodes = 2 * line.half_nodes;
    line.blocks = LINE_BLOCKS;
    line.part_rows = line_part_rows(A.tokens, G);
    line.part_o = scratch;
    line.part_ml = scratch + (size_t)line.blocks * 2 * line.part_rows * A.d;
    line.starts = reinterpret_cast<int*>(line.part_ml + (size_t)line.blocks * 2 * line.part_rows * 2);
    line.dense = reinterpret_cast<float*>(line.starts) + LINE_REQUESTS + 4;      // (every part before it is a multiple of 4 numbers long)
    return line;
}

// tree_attention_tc.cu
bool tree_tc_takes(const TreeArgs& A);
int tree_tc_launch(const TreeArgs& A, float* scratch, cudaStream_t stream);

}  // namespace xbtree
