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

}  // namespace xbtree
