// What the kernels of attention over a cache of 4-bit codes share (cache4_attention.cu says what they compute and which of them takes a call).
#pragma once
#include "codes4.cuh"

namespace xb4 {

struct AttendArgs {
    void* out;                     // [tokens, nh, d], tokens `out_stride` elements apart; q alike
    const void* q;
    const uint8_t* k_cache;        // [pages, nkv, page_size * row_bytes(d)]
    const uint8_t* v_cache;
    const int* lengths;            // [requests]: tokens with the step's own
    const int* token_start;        // [requests + 1]
    const int* block_table;        // [requests, table_stride]
    long long out_stride, q_stride;
    int tokens, requests, table_stride, nh, nkv, d, page_size, num_pages, window;
    int group;                     // query heads of a key/value head
    unsigned long long group_inv;  // 2^32 / group, upwards
    int rows_from, rows_to;        // requests of other numbers of rows (tokens times query heads of a key/value head) are another kernel's
    float scale;
    int* err;
    const int* wide;               // null, or: whether the kernel for many rows has left requests to this one, then pairs of the first and the last of some (WIDE_PAIRS)
};
constexpr int WIDE_PAIRS = 148;            // a pair for each of its blocks; the first behind the last: none

static __device__ __noinline__ bool in_wide_pairs(const int* wide, int b) {
    for (int i = 0; i < WIDE_PAIRS; ++i)
        if (b >= wide[2 + 2 * i] && b <= wide[3 + 2 * i]) return true;
    return false;
}

// The token that a row (token, query head of the group) of a request belongs to: row / group, right for rows below 2^32 / group.
__device__ __forceinline__ int token_of(const AttendArgs& A, int row) { return (int)((unsigned)row * A.group_inv >> 32); }
inline bool tokens_of_rows(const AttendArgs& A) { return (double)A.tokens * A.group * A.group < 4294967296.0; }

constexpr int REQUESTS_MAX = 8192;
constexpr int ROWS_MOST = 0x7ffff000;            // rows of a step: their numbers, rounded up to blocks, are 32 bits
constexpr int LINE_MOST = 0x70000000;            // tiles of a step's line of jobs (a share more is 32 bits still)
constexpr long long KEYS_MOST = 0x7fff0000;      // keys that a row of the table may hold: their numbers, rounded up to tiles, are 32 bits

// A request of the step.  Its token i stands at position first_pos + i and sees the keys up to there, of these the last `window`.
struct Request {
    int first, nodes;              // its tokens in the step
    int first_pos;
    int keys;                      // keys that lie in the table's row
};
// LEFT: with those that the kernel for many rows has left.
template <bool LEFT>
__device__ __forceinline__ Request request_of(const AttendArgs& A, int b) {
    Request r;
    r.first = min(max(A.token_start[b], 0), A.tokens);               // (starts outside the tokens count as the nearest bound)
    r.nodes = max(0, min(max(A.token_start[b + 1], 0), A.tokens) - r.first);
    const int len = A.lengths[b];
    const long long most = (long long)A.table_stride * A.page_size;
    if (len > most && r.nodes > 0) atomicOr(A.err, XB_ERR_BAD_PAGE);
    r.keys = len < 0 ? 0 : (int)(len > most ? most : len);
    r.first_pos = max(len, 0) - r.nodes;
    const int rows = r.nodes * A.group;
    if ((rows < A.rows_from || rows >= A.rows_to) && !(LEFT && A.wide && A.wide[0] && in_wide_pairs(A.wide, b))) r.nodes = 0;
    return r;
}
// The sum of the lanes' numbers up to each lane, and of all.  Requests whose tokens overlap can be more work than 32 bits count (others cannot, the
// host has seen to that): reported, and nothing is done (-1).
__device__ __forceinline__ int prefix_of_lanes(const AttendArgs& A, long long mine, int& incl) {
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if ((int)(threadIdx.x & 31) >= o) sum += v;
    }
    incl = (int)sum;
    const long long total = __shfl_sync(0xffffffffu, sum, 31);
    if (total > LINE_MOST) {
        atomicOr(A.err, XB_ERR_BAD_ROW);
        return -1;
    }
    return (int)total;
}
// The first key that a token at `pos` sees.
__device__ __forceinline__ int first_seen(const AttendArgs& A, int pos) { return A.window > 0 ? max(0, pos - A.window + 1) : 0; }

}  // namespace xb4
