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

// ---- the line of all jobs' tiles -------------------------------------------------------------------------------------------
// A job is (request, key/value head, some of the rows that a node and a query head of the group make); its tiles of KT keys are the cached
// ones from the first that a node sees and the drafted ones.  The line holds all jobs' tiles, request by request, each as long as it
// costs: block c takes the tiles that begin in c * share .. (c + 1) * share - 1, whatever the lengths are, so that blocks finish together and
// nobody has to know the lengths on the host.
constexpr int LINE_REQUESTS = 8192;
constexpr int COST_ONE = 2;        // what a tile of keys costs a job of one tile of rows, and of two: 1,350 and 2,000 cycles measured
constexpr int COST_TWO = 3;
constexpr int COST_JOB = 12;       // what a job costs beside its tiles: its last, drafted keys and its result

struct Line {
    int row_mul, row_div;          // a request's jobs of a head: nodes * row_mul / row_div, upwards
    int two_from;                  // jobs of more nodes have two tiles of rows
    int min_share;                 // what a block takes at least: below that its start and the join cost more than they save
    int part_rows;                 // rows of a part that is kept for the join
    float* part_o;                 // [blocks][2][part_rows][d]: a block's first segment, if its job began before it, and its last, if its job
                                   // goes on; how rows and channels lie is each kernel's own
    float* part_ml;                // [blocks][2][part_rows][2]: maximum and sum
    int* shared_jobs;              // [blocks][2][8]: the jobs of these parts: parts (0: there is no such part), block of the first, first row
                                   // or node, rows or nodes, key/value head, request
    float* dense;                  // room for q, k_new and v_new as dense rows of bfloat16
};

struct RequestLine {
    int first, nodes, context, tile0, old_tiles, tiles, pieces;
    int per_tile;                  // what a tile costs each of its jobs
    __device__ __forceinline__ int job_units() const { return tiles * per_tile + COST_JOB; }
    __device__ __forceinline__ int units(int nkv) const { return nkv * pieces * job_units(); }
    __device__ __forceinline__ RequestLine of_lane(int l) const {
        auto from = [&](int v) { return __shfl_sync(0xffffffffu, v, l); };
        return RequestLine{from(first), from(nodes), from(context), from(tile0), from(old_tiles), from(tiles), from(pieces), from(per_tile)};
    }
};

template <int KT>
__device__ __forceinline__ RequestLine request_line(const TreeArgs& A, const Line& line, int b) {
    RequestLine r;
    r.first = clamp_start(A, A.token_start[b]);
    r.nodes = max(0, clamp_start(A, A.token_start[b + 1]) - r.first);
    r.context = context_of(A, b);
    r.tile0 = A.window > 0 ? max(0, r.context - A.window + 1) / KT : 0;    // (the root's window begins first)
    r.old_tiles = max(0, (r.context + KT - 1) / KT - r.tile0);
    r.tiles = r.old_tiles + (r.nodes + KT - 1) / KT;
    r.pieces = (r.nodes * line.row_mul + line.row_div - 1) / line.row_div;
    r.per_tile = r.nodes > line.two_from ? COST_TWO : COST_ONE;
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
template <int KT>
__device__ __forceinline__ Walk place_in_line(const TreeArgs& A, const Line& line) {
    const int lane = threadIdx.x & 31, each = (A.requests + 31) / 32, b0 = lane * each, b1 = min(b0 + each, A.requests);
    Walk w;
    int mine = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        w.r = request_line<KT>(A, line, b);
        mine += w.r.units(A.nkv);
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
    w.job = w.end;
    w.b = w.g = w.piece = w.i0 = w.i1 = 0;
    if (w.from >= w.end) return w;
    int before = incl - mine, b = b0;
    const unsigned who = __ballot_sync(0xffffffffu, w.from >= before && w.from < incl);
    const int owner = __ffs(who) - 1;
    if (each > 1) {
        if (lane == owner) {
#pragma unroll 1
            for (; b < b1; ++b) {
                w.r = request_line<KT>(A, line, b);
                const int n = w.r.units(A.nkv);
                if (w.from < before + n) break;
                before += n;
            }
        }
        w.b = __shfl_sync(0xffffffffu, b, owner);
        w.r = request_line<KT>(A, line, w.b);
    } else {                           // a lane has one request: the owner's, without another trip
        w.b = owner;
        w.r = w.r.of_lane(owner);
    }
    before = __shfl_sync(0xffffffffu, before, owner);
    const int length = w.r.job_units(), at = (w.from - before) / length;
    w.g = at / w.r.pieces;
    w.piece = at % w.r.pieces;
    w.job = before + at * length;
    return w;
}

// The next job of which the block has a part; false: there is none.  (The first tile that begins at or behind `from` may be the next
// job's, or the next request's first.)
template <int KT>
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
                    w.r = request_line<KT>(A, line, w.b);
                } while (w.r.nodes == 0);                          // (a request without nodes has no jobs)
            }
        }
        w.i0 = w.from > w.job ? tiles_of_cost(w.from - w.job, w.r.per_tile) : 0;
        w.i1 = min(w.r.tiles, tiles_of_cost(w.end - w.job, w.r.per_tile));
        if (w.i0 < w.i1) return true;
    }
}

// In how many blocks the job's tiles begin, and the first of them.
__device__ __forceinline__ int job_parts(const Walk& w, int& first) {
    first = w.job / w.share;
    return (w.job + (w.r.tiles - 1) * w.r.per_tile) / w.share - first + 1;
}

__device__ __forceinline__ size_t part_row(const Line& line, int block, int which, int row) { return ((size_t)block * 2 + which) * line.part_rows + row; }

// host: the layout of a line's scratch, in float32 numbers (every part is a multiple of 4 numbers long)
inline long long line_floats(int blocks, int part_rows, int d, long long dense) { return (long long)blocks * 2 * (part_rows * (long long)(d + 2) + 8) + dense; }
inline void lay_out(Line& line, int blocks, int d, float* scratch) {
    line.part_o = scratch;
    line.part_ml = scratch + (size_t)blocks * 2 * line.part_rows * d;
    line.shared_jobs = reinterpret_cast<int*>(line.part_ml + (size_t)blocks * 2 * line.part_rows * 2);
    line.dense = reinterpret_cast<float*>(line.shared_jobs) + (size_t)blocks * 16;
}

// tree_attention_tc.cu
bool tree_tc_takes(const TreeArgs& A);
long long tree_tc_scratch(int tokens, int nh, int nkv, int d);
int tree_tc_launch(const TreeArgs& A, float* scratch, cudaStream_t stream);

}  // namespace xbtree
