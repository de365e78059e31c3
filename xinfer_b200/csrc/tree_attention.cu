// Attention of a tree of drafted tokens over the paged cache.  Request b has `context[b]` cached keys and the nodes
// token_start[b] .. token_start[b + 1] - 1, whose keys and values lie in rows of their own beside the cache.  With scale s, node
// i of depth p_i sees the keys
//     cached j < context[b]                          (window w: and j > context[b] + p_i - w)
//     drafted i' with bit i' of ancestors[i] set     (window w: and p_i - p_i' < w)
// and its result is  sum_j exp(s q.k_j - m) v_j / sum_j exp(s q.k_j - m),  m the largest score;  zeros where it sees no key.
// A value that a node does not see is not part of its result, whatever it holds.
#include "tree_attention.cuh"

namespace {

using namespace xbtree;

constexpr int WARPS = 4;

// The simple form, for every type, head size and layout: a warp per (node, head), 32 keys at a time.  A lane scores a key, the
// warp forms the tile's maximum and sum, then the lanes hold channels and the tile's weights come by shuffle.
template <typename T, int CH>
__global__ void __launch_bounds__(WARPS * 32)
tree_attention_kernel(const TreeArgs A) {
    extern __shared__ float q_rows[];        // [WARPS][d]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = (long long)blockIdx.x * WARPS + warp;
    const int t = (int)(item / A.nh), h = (int)(item % A.nh);
    if (t >= A.tokens) return;
    const int b = request_of(A, t);
    T* out = (T*)A.out + (size_t)t * A.out_stride + (size_t)h * A.d;
    if (b < 0) return;                       // a row of no request is left as it is
    const int g = h / (A.nh / A.nkv), first = clamp_start(A, A.token_start[b]), n = clamp_start(A, A.token_start[b + 1]) - first;
    const int context = context_of(A, b);
    const int my_depth = A.window > 0 ? max(0, A.depth[t]) : 0, my_pos = context + my_depth;
    const int lo = A.window > 0 ? max(0, my_pos - A.window + 1) : 0;
    float* qs = q_rows + (size_t)warp * A.d;
    const T* q = (const T*)A.q + (size_t)t * A.q_stride + (size_t)h * A.d;
    for (int c = lane; c < A.d; c += 32) qs[c] = to_f32<T>(q[c]);
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) o[i] = 0.f;
    const int* table = A.block_table + (size_t)b * A.table_stride;
    const int old_tiles = (context + 31) / 32, tiles = old_tiles + (n + 31) / 32;
    for (int tile = lo / 32; tile < tiles; ++tile) {
        const bool drafted = tile >= old_tiles;
        const int j = (drafted ? tile - old_tiles : tile) * 32 + lane;
        bool seen;
        long long row = 0;                   // of the key, in elements of its tensor
        if (drafted) {
            seen = j < n && (A.ancestors[(size_t)t * A.words + (j >> 5)] >> (j & 31) & 1);
            if (seen && A.window > 0) seen = my_depth - max(0, A.depth[first + j]) < A.window;
        } else {
            seen = j >= lo && j < context;
            if (seen) {
                const int page = table[j / A.page_size];
                if (page < 0 || page >= A.num_pages) {
                    atomicOr(A.err, XB_ERR_BAD_PAGE);
                    seen = false;
                } else {
                    row = (((long long)page * A.nkv + g) * A.page_size + j % A.page_size) * A.d;
                }
            }
        }
        const T* k = drafted ? (const T*)A.k_new + (size_t)(first + j) * A.k_stride + (size_t)g * A.d : (const T*)A.k_cache + row;
        const T* v = drafted ? (const T*)A.v_new + (size_t)(first + j) * A.v_stride + (size_t)g * A.d : (const T*)A.v_cache + row;
        float s = -INFINITY;
        if (seen) {
            s = 0.f;
            for (int c = 0; c < A.d; ++c) s = fmaf(qs[c], to_f32<T>(k[c]), s);
            s *= A.scale;
        }
        const unsigned live = __ballot_sync(0xffffffffu, seen);
        if (!live) continue;
        const float top = fmaxf(m, warp_max(s)), base = top == -INFINITY ? 0.f : top;
        const float p = seen ? expf(s - base) : 0.f, corr = expf(m - base);
        l = l * corr + warp_sum(p);
        m = top;
#pragma unroll
        for (int i = 0; i < CH; ++i) o[i] *= corr;
        for (unsigned left = live; left; left &= left - 1) {
            const int who = __ffs(left) - 1;
            const float w = __shfl_sync(0xffffffffu, p, who);
            const T* vr = (const T*)__shfl_sync(0xffffffffu, (unsigned long long)v, who);
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (lane + 32 * i < A.d) o[i] = fmaf(w, to_f32<T>(vr[lane + 32 * i]), o[i]);
        }
    }
    const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (lane + 32 * i < A.d) out[lane + 32 * i] = from_f32<T>(o[i] * inv);
}

template <typename T>
int launch(const TreeArgs& A, cudaStream_t stream) {
    const unsigned blocks = (unsigned)(((long long)A.tokens * A.nh + WARPS - 1) / WARPS);
    const size_t smem = (size_t)WARPS * A.d * 4;
    if (A.d <= 64) tree_attention_kernel<T, 2><<<blocks, WARPS * 32, smem, stream>>>(A);
    else if (A.d <= 128) tree_attention_kernel<T, 4><<<blocks, WARPS * 32, smem, stream>>>(A);
    else tree_attention_kernel<T, 16><<<blocks, WARPS * 32, smem, stream>>>(A);
    return xb_launch_status();
}

}  // namespace

XB_EXPORT int xb_tree_attention(int dtype, void* out, const void* q, const void* k_new, const void* v_new, const void* k_cache, const void* v_cache,
                                const int* context, const int* token_start, const int* ancestors, const int* depth, const int* block_table,
                                long long out_stride, long long q_stride, long long k_stride, long long v_stride, int tokens, int requests, int words,
                                int table_stride, int nh, int nkv, int d, int page_size, int num_pages, int window, float scale, float* scratch,
                                int* err, cudaStream_t stream) {
    if (tokens <= 0 || requests <= 0) return 0;
    if (requests > LINE_REQUESTS || d < 1 || d > 512 || nkv < 1 || nh % nkv || page_size < 1 || (window > 0 && !depth)) return (int)cudaErrorInvalidValue;
    const TreeArgs A{out, q, k_new, v_new, k_cache, v_cache, context, token_start, ancestors, depth, block_table, out_stride, q_stride, k_stride, v_stride,
                     tokens, requests, words, table_stride, nh, nkv, d, page_size, num_pages, window, scale, err};
    if (dtype == XB_BF16 && scratch && ((uintptr_t)scratch & 15) == 0 && tree_tc_takes(A)) return tree_tc_launch(A, scratch, stream);
    return dtype == XB_F32 ? launch<float>(A, stream) : launch<__nv_bfloat16>(A, stream);
}

// float32 numbers of scratch for a step of `tokens` drafted tokens (0: none is used)
XB_EXPORT long long xb_tree_attention_scratch(int dtype, int tokens, int nh, int nkv, int d) {
    if (dtype != XB_BF16 || tokens <= 0 || nkv <= 0 || nh < nkv) return 0;
    return line_floats(tokens, nh, nkv, d);
}
